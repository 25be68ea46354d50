// Values joined over the 64 lanes of a wave, and a barrier that leaves loads from memory in flight.
#pragma once

#include <hip/hip_runtime.h>

namespace tsac_hip
{
// One step of a butterfly over the lanes, from stride 1 on: every group of `stride` lanes holds one value, so that any lane of
// the neighbouring group will do and no step goes through LDS. `join` commutes.
template <int stride, class V, class Join> __device__ __forceinline__ V join_neighbours(V value, Join join)
{
    const int bits = __builtin_bit_cast(int, value);
    if constexpr (stride < 16)
    {
        // quad_perm [1,0,3,2] and [2,3,0,1], row_half_mirror, row_mirror
        constexpr int control = stride == 1 ? 0xb1 : stride == 2 ? 0x4e : stride == 4 ? 0x141 : 0x140;
        return join(value, __builtin_bit_cast(V, __builtin_amdgcn_mov_dpp(bits, control, 0xf, 0xf, false)));
    }
    else if constexpr (stride == 16)
    {
        // An exchange of a value with itself leaves the lower group's in one result, the upper group's in the other.
        const auto r = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
        return join(__builtin_bit_cast(V, int(r[0])), __builtin_bit_cast(V, int(r[1])));
    }
    else
    {
        const auto r = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
        return join(__builtin_bit_cast(V, int(r[0])), __builtin_bit_cast(V, int(r[1])));
    }
}

// The values of all lanes, or of each group of 16 or 32, joined, in every lane of them.
template <int Lanes = 64, class V, class Join> __device__ __forceinline__ V over_lanes(V value, Join join)
{
    static_assert(sizeof(V) == 4 && (Lanes == 16 || Lanes == 32 || Lanes == 64));
    value = join_neighbours<2>(join_neighbours<1>(value, join), join);
    value = join_neighbours<8>(join_neighbours<4>(value, join), join);
    if constexpr (Lanes > 16)
    {
        value = join_neighbours<16>(value, join);
    }
    if constexpr (Lanes > 32)
    {
        value = join_neighbours<32>(value, join);
    }
    return value;
}

// A workgroup's barrier for what lies in LDS.
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
} // namespace tsac_hip
