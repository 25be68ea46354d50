"""A model's step around the paged attention on the MI355X: tokens to 8 bits, their products, norms around a block,
rotated rows into pages, rules on logits; and a run of them together with the attention and the verification. Against
plain implementations in 64 bits written from the definitions.

h = 2^-24 is half a step of 32 bits and u that of the result's type (2^-8 for BF16, 2^-11 for half, 2^-24 for single); a
result of half's subnormal range is off by 2^-25 more. Every tolerance below counts roundings from these."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}
TINY = {"bfloat16": 2.0 ** -133, "float16": 2.0 ** -25, "float32": 2.0 ** -126}
H = 2.0 ** -24
KINDS = ["bfloat16", "float16", "float32"]


@pytest.fixture(scope="module")
def torch():
    import torch

    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    return torch


@pytest.fixture(scope="module")
def native():
    from tsac_hip import native

    native.library()
    return native


def ints(torch, values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def floats(torch, values):
    return torch.tensor(np.asarray(values), dtype=torch.float32, device="cuda")


def normal(torch, shape, seed, kind, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(getattr(torch, kind))


class Inside:
    """A matrix inside of a larger buffer, whose other parts have to stay."""

    def __init__(self, torch, rows, width, kind, pad=16, offset=0, fill=7):
        self.torch, self.fill = torch, fill
        pitch = -(-width // 16) * 16 + pad
        self.buffer = torch.full((rows + 2, pitch), fill, dtype=getattr(torch, kind), device="cuda")
        self.at = (slice(1, rows + 1), slice(offset, offset + width))
        self.view = self.buffer[self.at]

    def rest_stays(self):
        rest = self.buffer.clone()
        rest[self.at] = self.fill
        assert bool((rest == self.fill).all())


def near(torch, got, want, room):
    """Elementwise |got - want| <= room, and the same places that are not numbers."""
    got = got.double()
    nan = want.isnan()
    assert bool((got.isnan() == nan).all()), "not a number in other places"
    bad = ~((got - want).abs() <= room) & ~nan & (got != want)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[0].tolist(), float(((got - want).abs() - room)[bad].max()))


# ---------------------------------------------------------------- tokens to 8 bits

def quantised(torch, x):
    """(q, scales) from the definition: a scale is a product of two floats, a quotient of numbers of 24 bits is told
    from a border between whole numbers by 64 bits."""
    top = x.double().abs().amax(1)
    scale = (top * float(np.float32(1) / np.float32(127))).float()  # 48 bits: rounded once
    finite = top.isfinite()
    q = torch.where(((scale > 0) & finite)[:, None], (x.double() / scale.double()[:, None]).round(), 0.0)
    return q.nan_to_num(0.0).clamp(-127, 127), torch.where(finite, scale, math.nan)


def check_quantised(torch, native, x):
    rows, width = x.shape
    out = Inside(torch, rows, width, "int8")
    scales = torch.full((rows + 1,), 5.0, device="cuda")
    native.quantize_tokens(x, out.view, scales)
    q, s = quantised(torch, x)
    assert torch.equal(scales[:rows].nan_to_num(-1.0), s.nan_to_num(-1.0)) and float(scales[rows]) == 5.0
    assert torch.equal(out.view.double(), q)
    out.rest_stays()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 63, 100, 511, 512, 513, 1024, 1025, 2048, 2049, 4096, 5003, 8192, 8200,
                                   16384, 16385, 32768, 65535, 65536])
def test_tokens_to_8_bits(torch, native, kind, width):
    for rows in (1, 5):
        check_quantised(torch, native, normal(torch, (rows, width), width, kind, 3.0))
    # Rows at an odd pitch, from an odd place on.
    wide = normal(torch, (4, width + 3), width + 1, kind)
    check_quantised(torch, native, wide[1:, 1:width + 1])


@pytest.mark.parametrize("kind", KINDS)
def test_tokens_on_borders_between_whole_numbers(torch, native, kind):
    """Halves of steps, which go to the even number, and what lies just beside them."""
    half = torch.arange(-127, 127, device="cuda") + 0.5
    x = torch.stack([torch.cat([half, torch.tensor([t], device="cuda")]) for t in (127.0, -127.0, 128.0, 130.0, 254.0)])
    x = torch.cat([x, x * 2.0 ** -9, x[:, :] * 0.5]).to(getattr(torch, kind))
    q, s = quantised(torch, x)
    ties = ((x.double() / s.double()[:, None] * 2) % 2 == 1).sum()
    assert int(ties) > 100
    check_quantised(torch, native, x)
    if kind == "float32":
        for bits in (1, -1):
            check_quantised(torch, native, (x.view(torch.int32) + bits).view(torch.float32))


@pytest.mark.parametrize("kind", KINDS)
def test_tokens_that_are_zero_tiny_huge_or_not_numbers(torch, native, kind):
    x = normal(torch, (12, 200), 3, kind)
    info = torch.finfo(x.dtype)
    x[0] = 0
    x[1] *= info.tiny  # subnormal
    x[2] = 0
    x[2, 7] = info.smallest_normal
    x[3, 199] = math.inf
    x[4, 0] = -math.inf
    x[5, 100] = math.nan
    x[6] = info.max
    x[7] = -0.0
    x[8] = torch.sign(x[8].float()).to(x.dtype) * info.max
    x[9] = 0
    x[9, 3] = 2.0 ** -149 if kind == "float32" else 2.0 ** -133 if kind == "bfloat16" else 2.0 ** -24
    check_quantised(torch, native, x)


# ---------------------------------------------------------------- products

def linear_of(torch, native, outputs, inputs, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randint(-128, 128, (outputs, inputs), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    c = (0.5 + torch.rand(outputs, generator=g, device="cuda")) / 64
    b = torch.randn(outputs, generator=g, device="cuda") if bias else None
    return native.ChannelLinear(w, c, b), w, c, b


def tokens_of(torch, rows, inputs, seed):
    """q inside of a buffer whose other bytes are anything, and scales."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pitch = -(-inputs // 16) * 16 + 16
    q = torch.randint(-128, 128, (rows, pitch), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    s = (0.5 + torch.rand(rows, generator=g, device="cuda")) / (64 * math.sqrt(inputs))
    return q[:, :inputs], s


def product(torch, q, s, w, c, b, kind):
    """(result, tolerance): the sum as a float, the scales' product and theirs are rounded, then the sum with the bias."""
    exact = (q.double() @ w.double().T) * (s.double()[:, None] * c.double())
    y = exact if b is None else exact + b.double()
    return y, 3.01 * H * exact.abs() + H * y.abs() + UNIT[kind] * (1 + 4 * H) * y.abs() + TINY[kind]


def check_product(torch, native, rows, inputs, outputs, kind, seed=0, bias=True, linear=None):
    linear, w, c, b = linear or linear_of(torch, native, outputs, inputs, seed, bias)
    q, s = tokens_of(torch, rows, inputs, seed + 1)
    out = Inside(torch, rows, outputs, kind, offset=3 if rows % 2 else 0)
    linear.apply(q, s, out.view)
    y, room = product(torch, q, s, w, c, b, kind)
    near(torch, out.view, y, room)
    out.rest_stays()
    return out.view


ROWS = [1, 2, 3, 16, 17, 31, 32, 33, 48, 63, 64, 65, 96, 127, 128, 129, 192, 200, 255, 256, 257, 300, 511, 513, 1000, 2049]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("inputs,outputs", [(1, 1), (15, 5), (128, 32), (129, 33), (256, 31), (1000, 257), (4096, 96),
                                            (333, 1100)])
def test_products_of_odd_sizes(torch, native, rows, inputs, outputs):
    kind = KINDS[(rows + inputs + outputs) % 3]
    check_product(torch, native, rows, inputs, outputs, kind, seed=rows, bias=rows % 3 != 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,inputs,outputs", [(3, 1024, 4096), (12, 512, 1536), (64, 2048, 512), (40, 16000, 64),
                                                 (130, 8192, 640), (700, 1024, 1024), (1024, 640, 3000), (3000, 3001, 801)])
def test_products_of_model_sizes(torch, native, kind, rows, inputs, outputs):
    check_product(torch, native, rows, inputs, outputs, kind, seed=5)


# Sizes for which each variant of many rows has workgroups that go on from one tile to the next, of 256 units: tiles of outputs
# x rows, and tiles a workgroup at most.
SEVERAL_TILES = [(1000, 20000),  # 128 x 128, 5
                 (128, 70000),  # 128 x 128, one row tile, 3
                 (700, 30000),  # 128 x 256, 3
                 (256, 90000),  # 128 x 256, one row tile, 3
                 (8190, 4096),  # 256 x 256, 2
                 (4999, 5001),  # 256 x 256, 2
                 (240, 120000),  # 256 x 256, one row tile, 2
                 (12000, 300)]  # 64 x 64, 2


@pytest.mark.parametrize("rows,outputs", SEVERAL_TILES)
def test_products_of_several_tiles_a_workgroup(torch, native, rows, outputs):
    """Every element, of one stage a tile to more than a ring holds, in all types, stored in whole vectors and one by one."""
    for i, inputs in enumerate((1, 64, 100, 128, 129, 256, 700)):
        linear, w, c, b = linear_of(torch, native, outputs, inputs, i, bias=i % 2 == 0)
        q, s = tokens_of(torch, rows, inputs, i + 1)
        exact = (q.double() @ w.double().T) * (s.double()[:, None] * c.double())
        y = exact if b is None else exact + b.double()
        for j, kind in enumerate(KINDS):
            out = Inside(torch, rows, outputs, kind, offset=3 if (i + j) % 4 == 3 else 0)
            linear.apply(q, s, out.view)
            near(torch, out.view, y, 3.01 * H * exact.abs() + H * y.abs() + UNIT[kind] * (1 + 4 * H) * y.abs() + TINY[kind])
            out.rest_stays()


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_products_of_the_longest_sums(torch, native, rows):
    """Sums up to 128 x 128 x 131071 = 2^31 - 16384."""
    inputs = 131071
    w = torch.full((40, inputs), -128, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    linear = native.ChannelLinear(w, torch.ones(40, device="cuda"))
    q = torch.full((rows, inputs + 1), -128, dtype=torch.int8, device="cuda")[:, :inputs]
    out = torch.empty(rows, 40, device="cuda")
    linear.apply(q, torch.ones(rows, device="cuda"), out)
    want = torch.where(torch.arange(40, device="cuda") % 2 == 0, 128 * 128 * inputs, -128 * 127 * inputs).double()
    assert bool(((out.double() - want).abs() <= H * want.abs()).all())


def test_products_are_the_same_in_every_batch(torch, native):
    """A row alone and among others, in 32 bits: the same bits."""
    linear, *_ = linear_of(torch, native, 515, 1100, 1)
    q, s = tokens_of(torch, 1500, 1100, 2)
    q = torch.nn.functional.pad(q, (0, 4))[:, :1100]
    every = torch.empty(1500, 515, device="cuda")
    linear.apply(q, s, every)
    for rows in (1, 7, 33, 64, 100, 140, 256, 400, 777):
        some = torch.empty(rows, 515, device="cuda")
        linear.apply(q[:rows], s[:rows], some)
        assert torch.equal(some, every[:rows]), rows


def test_products_of_rows_without_a_scale(torch, native):
    linear, w, c, b = linear_of(torch, native, 70, 100, 1)
    x = normal(torch, (5, 100), 2, "bfloat16")
    x[1, 3], x[3] = math.inf, 0
    q, s = torch.zeros(5, 112, dtype=torch.int8, device="cuda")[:, :100], torch.empty(5, device="cuda")
    native.quantize_tokens(x, q, s)
    out = torch.empty(5, 70, dtype=torch.bfloat16, device="cuda")
    linear.apply(q, s, out)
    assert bool(out[1].isnan().all()) and torch.equal(out[3].float(), b.bfloat16().float())
    assert not bool(out[[0, 2, 4]].isnan().any())


def test_linears_from_host_and_device_memory(torch, native):
    _, w, c, b = linear_of(torch, native, 77, 130, 1)
    q, s = tokens_of(torch, 9, 130, 2)
    outs = []
    side = torch.cuda.Stream()
    for parts in ((w, c, b), (w.cpu(), c.cpu(), b.cpu()), (w.cpu().numpy(), c.cpu().numpy(), b.cpu().numpy()),
                  (w.T.contiguous().T, c, b)):
        outs.append(torch.empty(9, 77, device="cuda"))
        native.ChannelLinear(*parts).apply(q, s, outs[-1])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        linear = native.ChannelLinear(w * 1, c * 1, b * 1)
        outs.append(torch.empty(9, 77, device="cuda"))
        linear.apply(q, s, outs[-1])
    side.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_products_of_more_than_2_to_the_31_elements(torch, native):
    """Outputs past 32 bits of offset, and rows of q past 2^31 bytes."""
    linear, w, c, b = linear_of(torch, native, 4099, 64, 3)
    rows = 530000
    q = torch.randint(-128, 128, (rows, 4112), device="cuda", dtype=torch.int8)[:, :64]
    s = torch.rand(rows, device="cuda") / 256
    out = torch.empty(rows, 4112, dtype=torch.bfloat16, device="cuda")[:, :4099]
    linear.apply(q, s, out)
    for first in (0, 260000, 522000, rows - 40):
        part = slice(first, first + 40)
        y, room = product(torch, q[part], s[part], w, c, b, "bfloat16")
        near(torch, out[part], y, room)


# ---------------------------------------------------------------- norms around a block

def normed(torch, v, e, norm, gain, bias, epsilon):
    """(result, bound of its error) of values v that are off by e. Sums of n terms of one sign are off by (n + 24) H
    relative, with n the terms that one thread adds, at most 64, and 24 levels at most behind them."""
    if norm == 0:
        return v, e
    sums = (64 + 24) * H
    width = v.shape[1]
    mean = v.mean(1, keepdim=True) if norm == 2 else torch.zeros_like(v[:, :1])
    shift = (sums * v.abs().mean(1, keepdim=True) + e.mean(1, keepdim=True) + 2 * H * mean.abs()) if norm == 2 else 0 * mean
    d = v - mean
    off = e + shift + H * d.abs()  # of a deviation
    variance = (d * d).mean(1, keepdim=True)
    wrong = 2 * (d.abs() * off).mean(1, keepdim=True) + (off * off).mean(1, keepdim=True) + (sums + 2 * H) * variance
    bottom = variance + epsilon
    factor = 1 / bottom.sqrt()
    # 1/sqrt moves by half of what its argument does and, where that is much, by no more than to its end.
    relative = 0.5 * wrong / (bottom - wrong).clamp(min=1e-300) + 4 * H
    out = d * factor
    error = (off + d.abs() * relative) * factor * (1 + 2.0 ** -10) + H * out.abs()
    if gain is not None:
        out, error = out * gain.double(), error * gain.double().abs() + H * (out * gain.double()).abs()
    if bias is not None:
        out = out + bias.double()
        error = error + H * out.abs()
    return out, error


class Block:
    def __init__(self, torch, rows, width, kind, wide, post, norm, gate, seed, aligned=True, mean=0.0):
        place = (lambda t: t) if aligned else (lambda t: torch.nn.functional.pad(t, (1, 2))[:, 1:-2])
        self.torch, self.rows, self.width, self.kind, self.wide = torch, rows, width, kind, wide
        self.x = place(normal(torch, (rows, width), seed, kind) + mean)
        self.r = place(normal(torch, (rows, width), seed + 1, wide, 2.0))
        vector = lambda i: normal(torch, (width + 1,), seed + i, kind)[0 if aligned else 1:][:width].contiguous()  # noqa: E731
        self.post, self.norm = post, norm
        self.post_gain, self.gain = (vector(2) if post else None), (vector(3) if norm else None)
        self.post_bias, self.bias = (vector(4) if post == 2 else None), (vector(5) if norm == 2 else None)
        self.gate = None if gate == 0 else place(normal(torch, (1 if gate == 1 else rows, width), seed + 6, kind))
        self.scale, self.epsilon = 0.37, 1e-5

    def expected(self):
        torch = self.torch
        u, e = normed(torch, self.x.double(), torch.zeros_like(self.x.double()), self.post, self.post_gain, self.post_bias,
                      self.epsilon)
        scale = float(np.float32(self.scale))
        if self.gate is not None:
            u, e = u * self.gate.double(), (e + H * u.abs()) * self.gate.double().abs()
        u, e = u * scale, (e + H * u.abs()) * scale
        total = u if self.r is None else self.r.double() + u
        e = e + H * total.abs()
        out, error = normed(torch, total, e, self.norm, self.gain, self.bias, self.epsilon)
        return total, e, out, error

    def run(self, native, sum=None, out=None, out_scales=None):
        native.block_norm(self.x, post=self.post, post_gain=self.post_gain, post_bias=self.post_bias, gate=self.gate,
                          scale=self.scale, residual=self.r, sum=sum, norm=self.norm, gain=self.gain, bias=self.bias,
                          epsilon=self.epsilon, out=out, out_scales=out_scales)

    def check(self, native, offset=0):
        torch = self.torch
        total, e, h, error = self.expected()
        s, out = (Inside(torch, self.rows, self.width, k, offset=offset) for k in (self.wide, self.kind))
        self.run(native, s.view, out.view)
        near(torch, s.view, total, e + UNIT[self.wide] * (total.abs() + e) + TINY[self.wide])
        near(torch, out.view, h, error + UNIT[self.kind] * (h.abs() + error) + TINY[self.kind])
        s.rest_stays()
        out.rest_stays()
        # To 8 bits: the scale is off by what the largest is, a value by half a step and what it was.
        q, scales = Inside(torch, self.rows, self.width, "int8"), torch.zeros(self.rows, device="cuda")
        self.run(native, None, q.view, scales)
        top = h.abs().amax(1)
        assert bool(((scales.double() - top / 127).abs() <= error.amax(1) / 127 + 2 * H * top / 127 + 2.0 ** -149).all())
        assert bool(((q.view.double() * scales.double()[:, None] - h).abs() <=
                     (0.5 + 2.0 ** -16) * scales.double()[:, None] + error).all())
        assert int(q.view.int().abs().max()) <= 127
        q.rest_stays()


@pytest.mark.parametrize("kind,wide", [("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", "float16"),
                                       ("float16", "float32"), ("float32", "float32")])
@pytest.mark.parametrize("width", [1, 3, 8, 100, 512, 1000, 1024, 2048, 4100, 8192, 9000, 20000, 65536])
def test_norms_around_a_block(torch, native, kind, wide, width):
    for i, (post, norm, gate) in enumerate([(0, 1, 0), (1, 1, 1), (2, 2, 2), (0, 2, 0), (1, 0, 1), (2, 1, 2)]):
        Block(torch, 5 if i % 2 else 1, width, kind, wide, post, norm, gate, width + i).check(native)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width", [1, 77, 1024, 3001])
def test_norms_of_rows_at_odd_places(torch, native, kind, width):
    Block(torch, 6, width, kind, kind, 2, 2, 2, 3, aligned=False).check(native, offset=5)


@pytest.mark.parametrize("width", [64, 1024, 5000])
def test_norms_of_values_far_from_their_mean(torch, native, width):
    """A mean of 100 deviations: squares around it, not around 0."""
    for norm in (1, 2):
        Block(torch, 4, width, "float32", "float32", 0, norm, 0, 9, mean=100.0).check(native)


def test_norms_of_constant_zero_and_broken_rows(torch, native):
    b = Block(torch, 5, 300, "bfloat16", "bfloat16", 0, 2, 0, 1)
    b.x[0], b.r[0] = 1.0, 0  # constant: its norm is the bias
    b.x[1], b.r[1] = 0, 0
    b.x[2, 7] = math.nan
    b.r[3, 0] = math.inf
    out, total = torch.zeros(2, 5, 300, dtype=torch.bfloat16, device="cuda")
    b.run(native, total, out)
    assert torch.equal(out[1], b.bias) and bool(((out[0].float() - b.bias.float()).abs() <= 2e-3 + b.bias.float().abs() * 2.0 ** -8).all())
    assert bool(out[2].isnan().all()) and bool(out[3].isnan().all()) and not bool(out[4].isnan().any())
    assert int(total.isnan().sum()) == 1
    q, scales = torch.zeros(5, 304, dtype=torch.int8, device="cuda"), torch.zeros(5, device="cuda")
    b.run(native, None, q[:, :300], scales)
    assert scales.isnan().tolist() == [False, False, True, True, False] and not bool(q[2:4].any())


def test_norms_without_their_parts_and_in_place(torch, native):
    b = Block(torch, 7, 1500, "bfloat16", "bfloat16", 1, 1, 0, 2)
    b.gain = b.post_gain = None
    b.check(native)
    b.r = None
    b.check(native)
    b = Block(torch, 7, 1500, "float16", "float32", 2, 2, 1, 2)
    b.bias = b.post_bias = None
    total, e, h, error = b.expected()
    kept = torch.empty_like(b.r)
    b.run(native, kept, None)  # no norm of it
    near(torch, kept, total, e + UNIT["float32"] * total.abs() + TINY["float32"])
    want = torch.empty_like(b.x)
    b.run(native, kept, want)
    b.run(native, b.r, b.x)  # the sum over the residual, the norm over the input
    assert torch.equal(b.r, kept) and torch.equal(b.x, want)


@pytest.mark.parametrize("width", [60, 130, 512, 1000, 2048, 4100, 8192, 10000])
def test_norms_are_the_same_in_every_batch(torch, native, width):
    """A row alone, among others, and in rows that lie at odd places: the same bits."""
    b = Block(torch, 5000, width, "bfloat16", "float32", 2, 2, 1, 4)
    total, out = torch.empty(5000, width, device="cuda"), torch.empty(5000, width, dtype=torch.bfloat16, device="cuda")
    b.run(native, total, out)
    x, r, gate = b.x, b.r, b.gate
    for first, rows in ((0, 1), (3, 2), (4000, 999)):
        part = slice(first, first + rows)
        for odd in (False, True):
            place = (lambda t: torch.nn.functional.pad(t, (1, 2))[:, 1:-2]) if odd else (lambda t: t)  # noqa: E731
            b.x, b.r, b.gate = place(x[part]), place(r[part]), place(gate)
            some, other = torch.empty_like(total[part]), torch.empty_like(out[part])
            b.run(native, some, other)
            assert torch.equal(some, total[part]) and torch.equal(other, out[part]), (first, odd)


def test_calls_of_no_rows(torch, native):
    """Nothing is written, and nothing is refused."""
    empty = lambda *shape, kind=torch.bfloat16: torch.empty(*shape, dtype=kind, device="cuda")  # noqa: E731
    native.quantize_tokens(empty(0, 64), empty(0, 64, kind=torch.int8), empty(0, kind=torch.float32))
    linear, *_ = linear_of(torch, native, 32, 64, 1)
    linear.apply(empty(0, 64, kind=torch.int8), empty(0, kind=torch.float32), empty(0, 32))
    native.block_norm(empty(0, 64), norm=native.NORM_RMS, out=empty(0, 64))
    native.adjust_logits(empty(0, 100), empty(0, 100), ints(torch, [0, 0, 0]))
    logits = normal(torch, (3, 100), 1, "float32")
    out = torch.full((3, 100), 7.0, device="cuda")
    native.adjust_logits(logits, out, ints(torch, [0]))  # no sequence
    native.adjust_logits(logits, out, ints(torch, [2, 2, 2]))  # none with a row
    assert bool((out == 7).all())


def test_norms_of_more_than_2_to_the_31_elements(torch, native):
    rows, width = 270000, 8192
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in range(0, rows, 30000):
        x[i:i + 30000] = torch.randn(30000, width, generator=g, device="cuda").bfloat16()
    out = torch.empty_like(x)
    native.block_norm(x, norm=native.NORM_RMS, out=out)
    for first in (0, 262140, rows - 4):
        h, error = normed(torch, x[first:first + 4].double(), torch.zeros(4, width, dtype=torch.float64, device="cuda"), 1, None,
                          None, 1e-5)
        near(torch, out[first:first + 4], h, error + UNIT["bfloat16"] * h.abs())


# ---------------------------------------------------------------- rotated rows into pages

class Pages:
    def __init__(self, torch, native, lengths, counts, heads=4, kv=2, width=64, page_rows=16, kind="bfloat16", layers=2,
                 seed=0, spare=3):
        self.torch, self.native, self.lengths, self.counts = torch, native, lengths, counts
        self.page_rows, self.kind, self.kv, self.width, self.heads = page_rows, kind, kv, width, heads
        rng = np.random.default_rng(seed)
        held = [-(-(a + b) // page_rows) for a, b in zip(lengths, counts)]
        pages = sum(held) + spare
        order = rng.permutation(pages)
        self.table_list = -np.ones((len(lengths), max(held + [1]) + 1), np.int64)
        at = 0
        for s, h in enumerate(held):
            self.table_list[s, :h] = order[at:at + h]
            at += h
        references = np.zeros(pages, np.int64)
        references[order[:at]] = 1
        self.keys = normal(torch, (layers, pages, page_rows, kv, width), seed + 1, kind)
        self.values = normal(torch, (layers, pages, page_rows, kv, width), seed + 2, kind)
        self.table, self.held, self.references = ints(torch, self.table_list), ints(torch, held), ints(torch, references)
        self.starts_list = [0] + np.cumsum(counts).tolist()
        self.rows, self.starts = self.starts_list[-1], ints(torch, self.starts_list)
        self.cache = native.PagedCache(self.keys, self.values, self.table, self.held, ints(torch, lengths), self.references)
        qkv = normal(torch, (max(self.rows, 1), heads + 2 * kv, width), seed + 3, kind)[:self.rows]
        self.query, self.new_keys, self.new_values = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        self.max_rows = max(counts + [1])

    def turned(self, x, positions, frequencies, interleaved, amplitude):
        """(result, tolerance). A sine is off by the last turn's narrowing, pi 2^-25, and by two steps of its own, 2^-23, so
        by 2^-22 with the amplitude's product; a pair's two products and their sum round three times."""
        torch = self.torch
        x = x.double()
        rotary = 2 * len(frequencies)
        angle = positions.double()[:, None] * torch.tensor(frequencies, dtype=torch.float64, device="cuda")
        a = float(np.float32(amplitude))
        cos, sin = angle.cos()[:, None] * a, angle.sin()[:, None] * a
        even, odd = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
        p, q, out, room = x[..., even], x[..., odd], x.clone(), torch.zeros_like(x)
        out[..., even], out[..., odd] = p * cos - q * sin, p * sin + q * cos
        spread = (p.abs() + q.abs()) * abs(a) * (2.0 ** -22 + 4 * H)
        room[..., even] = room[..., odd] = spread
        room[..., :rotary] += UNIT[self.kind] * (out[..., :rotary].abs() + room[..., :rotary]) + TINY[self.kind]
        return out, room

    def check(self, frequencies, interleaved=False, amplitude=1.0, layer=0, positions=None, mask=None, depth=None,
              max_rows=None, in_place=False, missing=()):
        torch = self.torch
        most = self.max_rows if max_rows is None else max_rows
        rows = [(s, i) for s, c in enumerate(self.counts) for i in range(c)]
        if positions is not None:
            where = positions
        else:
            down = depth if depth is not None else [i for _, i in rows]
            where = [self.lengths[s] + d for (s, _), d in zip(rows, down)]
        where_t = torch.tensor(where, dtype=torch.int64, device="cuda")
        want_q, room_q = self.turned(self.query, where_t, frequencies, interleaved, amplitude)
        want_k, room_k = self.turned(self.new_keys, where_t, frequencies, interleaved, amplitude)
        before_k, before_v = self.keys.clone(), self.values.clone()
        buffer = torch.full((self.rows + 2, self.heads + 1, self.width), 7.0, dtype=self.query.dtype, device="cuda")
        out = buffer[1:self.rows + 1, :self.heads]
        if in_place:
            out.copy_(self.query)
        status = ints(torch, [0])
        self.cache.append(layer, out if in_place else self.query, self.new_keys, self.new_values, self.starts, most,
                          torch.tensor(frequencies, dtype=torch.float64, device="cuda"), out, interleaved=interleaved,
                          amplitude=amplitude, positions=None if positions is None else ints(torch, positions), mask=mask,
                          status=status)
        assert bool((buffer[:, self.heads:] == 7).all()) and bool((buffer[[0, -1]] == 7).all())
        here = torch.tensor([i < most for _, i in rows], device="cuda")
        near(torch, out[here], want_q[here], room_q[here])
        left = self.query if in_place else torch.full_like(out, 7.0)
        assert torch.equal(out[~here], left[~here])
        there = [r for r, (s, i) in enumerate(rows) if i < most and (s, i) not in missing]
        page = [int(self.table_list[rows[r][0], (self.lengths[rows[r][0]] + rows[r][1]) // self.page_rows]) for r in there]
        within = [(self.lengths[rows[r][0]] + rows[r][1]) % self.page_rows for r in there]
        got = self.keys[layer, page, within]
        near(torch, got, want_k[there], room_k[there])
        assert torch.equal(self.values[layer, page, within], self.new_values[there])
        self.keys[layer, page, within] = before_k[layer, page, within]
        self.values[layer, page, within] = before_v[layer, page, within]
        assert torch.equal(self.keys, before_k) and torch.equal(self.values, before_v), "another place was written"
        assert int(status) == (self.native.PAGES_INVALID if missing else 0)


LENGTHS = [0, 1, 15, 16, 17, 100, 255]


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("heads,kv,width", [(16, 16, 64), (8, 2, 128), (3, 1, 64), (1, 1, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_appended_rows(torch, native, kind, heads, kv, width, interleaved):
    for rotary in (2, 16, 20, width // 2, width - 2, width):
        counts = [3, 0, 20, 1, 16, 5, 33]
        p = Pages(torch, native, LENGTHS, counts, heads, kv, width, kind=kind, seed=rotary)
        p.check(native.rotary_frequencies(rotary), interleaved, layer=1)
        p.check(native.rotary_frequencies(rotary, base=500000.0), interleaved, amplitude=1.3, in_place=True)


@pytest.mark.parametrize("page_rows", [16, 64, 1024])
def test_appended_trees(torch, native, page_rows):
    """Positions down the lines of drafted trees, over more than one word of bits."""
    rng = np.random.default_rng(page_rows)
    counts = [70, 1, 0, 130, 12]
    p = Pages(torch, native, [5, 0, 9, 1000, 63], counts, page_rows=page_rows)
    parents, depth = [], []
    for c in counts:
        tree = [-1 if i < 2 else int(rng.integers(max(0, i - 6), i)) for i in range(c)]
        down = []
        for q in tree:
            down.append(0 if q < 0 else down[q] + 1)
        parents += tree
        depth += down
    mask = torch.zeros(p.rows, 3, dtype=torch.int64, device="cuda")
    native.tree_mask(ints(torch, parents), p.starts, p.max_rows, mask)
    p.check(native.rotary_frequencies(64), mask=mask, depth=depth)
    p.check(native.rotary_frequencies(64), mask=mask, depth=depth, max_rows=13)


def test_appended_rows_at_given_and_far_positions(torch, native):
    """Far positions, whose angles 32 bits would not hold, and negative ones."""
    p = Pages(torch, native, [0, 40], [4, 3], heads=2, kv=1, width=128, kind="float16")
    where = [(1 << 31) - 1, 0, 131071, -7, 1048575, 999983, -(1 << 31)]
    for interleaved in (False, True):
        p.check(native.rotary_frequencies(128), interleaved, positions=where)
        p.check(native.rotary_frequencies(128, scaling=native.ROTARY_TURNS, factor=8.0, context=8192.0, slow=1.0, fast=4.0),
                interleaved, positions=where)


def test_appended_rows_without_a_page(torch, native):
    """Pages that are not held, out of range or another sequence's too: queries turn, keys stay away."""
    p = Pages(torch, native, [30, 30, 30, 5], [4, 4, 4, 4])
    p.held[0] = 2                    # rows at 32 and 33 have none
    p.table[1, 2] = 9999
    p.references[int(p.table_list[2, 2])] = 2
    missing = [(s, i) for s in (0, 1, 2) for i in (2, 3)]
    p.check(native.rotary_frequencies(64), missing=missing)
    p.lengths = [30, 30, 30, -9]
    p.cache.tensors[4][3] = -9
    p.check(native.rotary_frequencies(64), missing=missing + [(3, i) for i in range(4)])


def test_appended_rows_of_few_and_many_announced(torch, native):
    """A batch in which one sequence has most rows, and one that announces more rows than it has."""
    counts = [1] * 60 + [700] + [0] * 5 + [2]
    p = Pages(torch, native, [7 * i for i in range(len(counts))], counts)
    p.check(native.rotary_frequencies(64))
    p = Pages(torch, native, LENGTHS, [2] * 7)
    p.check(native.rotary_frequencies(64), max_rows=50)
    p = Pages(torch, native, [3, 4], [0, 0])
    p.cache.append(0, p.query, p.new_keys, p.new_values, p.starts, 4, torch.ones(32, dtype=torch.float64, device="cuda"),
                   p.query)


def test_appended_rows_past_2_to_the_31_elements(torch, native):
    """A pool of 5 GiB, the last pages of the last layer."""
    layers, pages = 5, 2100
    keys = torch.zeros(layers, pages, 256, 8, 128, dtype=torch.bfloat16, device="cuda")
    values = torch.zeros_like(keys)
    references = torch.ones(pages, dtype=torch.int32, device="cuda")
    cache = native.PagedCache(keys, values, ints(torch, [[3, pages - 1]]), ints(torch, [2]), ints(torch, [510]), references)
    qkv = normal(torch, (2, 24, 128), 1, "bfloat16")
    out = torch.empty(2, 8, 128, dtype=torch.bfloat16, device="cuda")
    cache.append(4, qkv[:, :8], qkv[:, 8:16], qkv[:, 16:], ints(torch, [0, 2]), 2,
                 torch.zeros(64, dtype=torch.float64, device="cuda"), out)
    assert torch.equal(keys[4, pages - 1, 254:], qkv[:, 8:16]) and torch.equal(values[4, pages - 1, 254:], qkv[:, 16:])
    assert torch.equal(out, qkv[:, :8]) and not bool(keys[:4].any()) and not bool(keys[4, :pages - 1].any())


# ---------------------------------------------------------------- rules on logits

class Logits:
    """Rows of sequences with every rule, and the definition."""

    def __init__(self, torch, counts, alphabet, kind, history=50, seed=0, biases=9, allowed="rows", temperature=True,
                 prompt=True, penalties=True, drafted=True, aligned=True):
        self.torch, self.counts, self.alphabet, self.kind = torch, counts, alphabet, kind
        rng = np.random.default_rng(seed)
        n = len(counts)
        self.starts_list = [0] + np.cumsum(counts).tolist()
        rows = self.rows = self.starts_list[-1]
        pitch = -(-alphabet // 16) * 16 + 16 if aligned else alphabet + 3
        self.logits = normal(torch, (rows, pitch), seed, kind, 4.0)[:, :alphabet]
        if not aligned:
            self.logits = normal(torch, (rows + 1, alphabet + 3), seed, kind, 4.0)[1:, 1:alphabet + 1]
        self.rules = {}
        if history is not None:
            tokens = (rng.random((n, max(history, 1))) ** 3 * alphabet).astype(np.int64)
            tokens[rng.random(tokens.shape) < 0.05] = alphabet + 5  # not of this alphabet
            tokens[rng.random(tokens.shape) < 0.05] = -1
            lengths = rng.integers(0, history + 1, n)
            lengths[0] = history
            self.history, self.lengths = tokens, lengths
            self.rules.update(history=ints(torch, tokens), history_lengths=ints(torch, lengths))
            self.prompts = rng.integers(0, history + 1, n) if prompt else np.zeros(n, np.int64)
            if prompt:
                self.rules["prompt_lengths"] = ints(torch, self.prompts)
        else:
            self.history, self.lengths, self.prompts = np.zeros((n, 1), np.int64), np.zeros(n, int), np.zeros(n, int)
        self.tokens, self.lines = None, None
        if drafted:
            self.tokens = (rng.random(rows) ** 2 * alphabet).astype(np.int64)
            self.rules["tokens"] = ints(torch, self.tokens)
            self.lines = [set(range(i + 1)) for c in counts for i in range(c)]
            if drafted == "trees":
                words = max(1, -(-max(counts) // 64))
                self.lines, bits = [], np.zeros((rows, words), np.uint64)
                for c in counts:
                    lines = []
                    for i in range(c):
                        lines.append({i} | (lines[int(rng.integers(max(0, i - 5), i))] if i else set()))
                    self.lines += lines
                for r, line in enumerate(self.lines):
                    for j in line:
                        bits[r, j // 64] |= np.uint64(1) << np.uint64(j % 64)
                self.rules["mask"] = torch.from_numpy(bits.view(np.int64)).cuda()
        self.repetition = 1 + rng.random(n).astype(np.float32) if penalties else np.ones(n, np.float32)
        self.presence = rng.random(n).astype(np.float32) if penalties else np.zeros(n, np.float32)
        self.frequency = rng.random(n).astype(np.float32) if penalties else np.zeros(n, np.float32)
        if penalties:
            self.rules.update({k: floats(torch, getattr(self, k)) for k in ("repetition", "presence", "frequency")})
        self.bias = np.zeros((n, alphabet))
        if biases:
            sizes = rng.integers(0, biases + 1, n)
            starts = [0] + np.cumsum(sizes).tolist()
            tokens = rng.integers(0, alphabet + 2, starts[-1])  # some twice, some of no alphabet
            values = rng.normal(size=starts[-1]).astype(np.float32) * 3
            for s in range(n):
                for i in range(starts[s], starts[s + 1]):
                    if tokens[i] < alphabet:
                        self.bias[s, tokens[i]] = values[i]
            self.rules.update(bias_starts=ints(torch, starts), bias_tokens=ints(torch, tokens), bias_values=floats(torch, values))
        words = -(-alphabet // 32)
        self.ok = np.ones((rows, alphabet), bool)
        if allowed:
            bits = rng.integers(0, 1 << 32, (rows if allowed == "rows" else 1, words), dtype=np.uint64)
            if allowed == "rows" and rows > 2:
                bits[1], bits[2] = 0, (1 << 32) - 1
            every = (bits[:, :, None] >> np.arange(32, dtype=np.uint64) & np.uint64(1)).reshape(len(bits), -1)[:, :alphabet]
            self.ok[:] = every.astype(bool)
            self.rules["allowed"] = torch.from_numpy(bits.astype(np.uint32).view(np.int32)).cuda()
        self.temperature = (0.4 + rng.random(n)).astype(np.float32) if temperature else np.ones(n, np.float32)
        if temperature:
            self.rules["temperature"] = floats(torch, self.temperature)
        self.starts = ints(torch, self.starts_list)

    def adjusted(self):
        """(x, bound of its error) [rows][alphabet]: each step rounds once."""
        torch = self.torch
        x = self.logits.double().cpu().numpy()
        e = np.zeros_like(x)
        for s, c in enumerate(self.counts):
            past, prompt = self.history[s, :self.lengths[s]], min(self.prompts[s], self.lengths[s])
            had, said = np.zeros(self.alphabet, bool), np.zeros(self.alphabet, np.int64)
            for i, t in enumerate(past):
                if 0 <= t < self.alphabet:
                    had[t] = True
                    said[t] += i >= prompt
            for r in range(self.starts_list[s], self.starts_list[s + 1]):
                count, seen = said.copy(), had.copy()
                if self.tokens is not None:
                    for j in self.lines[r]:
                        t = self.tokens[self.starts_list[s] + j]
                        count[t] += 1
                        seen[t] = True
                v, w = x[r].copy(), e[r]
                v = np.where(seen, np.where(v > 0, v / float(self.repetition[s]), v * float(self.repetition[s])), v)
                # A positive one is taken times a reciprocal: two roundings, (1 + H)^2 - 1 < 2.01 H.
                w = w + np.where(seen, 2.01 * H * np.abs(v), 0)
                f = float(self.frequency[s]) * count
                v = v - f
                w = w + np.where(count > 0, H * np.abs(f) + H * np.abs(v), 0)
                v = v - np.where(count > 0, float(self.presence[s]), 0)
                w = w + np.where(count > 0, H * np.abs(v), 0)
                v = v + self.bias[s]
                w = w + np.where(self.bias[s] != 0, H * np.abs(v), 0)
                x[r], e[r] = np.where(self.ok[r], v, -np.inf), np.where(self.ok[r], w, 0)
        return torch.from_numpy(x).cuda(), torch.from_numpy(np.nan_to_num(e)).cuda()

    def sequence(self):
        return np.repeat(np.arange(len(self.counts)), self.counts)

    def probabilities(self):
        """(p, tolerance). An exponent (x - m) / t is off by the errors of x and m, by the difference's rounding, and
        relative by those of log2 e / t, of that quotient and of the product, 4 h; the exponential by 2^-22. A sum of at most
        2^15 numbers, one thread's 64 first, is off by 88 h, joined ones by as much again, and its reciprocal and the
        last product by 2 h."""
        torch = self.torch
        x, e = self.adjusted()
        t = torch.from_numpy(self.temperature.astype(np.float64)).cuda()[torch.from_numpy(self.sequence()).cuda()][:, None]
        m = x.amax(1, keepdim=True)
        empty = (m == -math.inf)
        d = torch.where(x == -math.inf, 0.0, x - torch.where(empty, 0.0, m)).abs()
        off = (e + e.amax(1, keepdim=True) + H * d) / t + 4 * H * d / t + 2.0 ** -22
        p = torch.where(empty, 0.0, torch.softmax(x / t, 1).nan_to_num(0.0))
        total = (p * off).sum(1, keepdim=True) + 180 * H
        return p, p * (off + total) * (1 + 2.0 ** -8) + 2.0 ** -120

    def run(self, native, out, probabilities=True, workspace=None):
        rules = dict(self.rules)
        if not probabilities:
            rules.pop("temperature", None)
        native.adjust_logits(self.logits, out, self.starts, probabilities=probabilities, workspace=workspace, **rules)

    def check(self, native, out_kind, probabilities=True, offset=0):
        torch = self.torch
        out = Inside(torch, self.rows, self.alphabet, out_kind, offset=offset)
        self.run(native, out.view, probabilities)
        want, room = self.probabilities() if probabilities else self.adjusted()
        room = room + UNIT[out_kind] * (torch.where(want.isinf(), 0.0, want.abs()) + room) + TINY[out_kind]
        near(torch, out.view, want, room)
        out.rest_stays()


ALPHABETS = [1, 2, 7, 8, 31, 33, 100, 512, 1000, 1024, 4095, 4097, 8200]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("alphabet", ALPHABETS)
def test_rules_and_probabilities(torch, native, kind, alphabet):
    out_kind = KINDS[(KINDS.index(kind) + alphabet) % 3]
    for i, drafted in enumerate((False, True, "trees")):
        logits = Logits(torch, [3, 1, 0, 7, 2], alphabet, kind, seed=alphabet + i, drafted=drafted,
                        allowed=("rows", "one", None)[i])
        logits.check(native, out_kind)
        logits.check(native, out_kind, probabilities=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("alphabet", [16384, 16385, 32000, 32768, 32769, 50001, 128001])
def test_rules_on_wide_alphabets(torch, native, kind, alphabet):
    logits = Logits(torch, [2, 1, 0, 3], alphabet, kind, history=3000, seed=alphabet, biases=300, drafted="trees")
    logits.check(native, "float32")
    logits.check(native, kind, probabilities=False)


def test_the_widest_alphabet(torch, native):
    Logits(torch, [1, 1], 1 << 20, "bfloat16", history=900, seed=1, biases=40).check(native, "float32")


@pytest.mark.parametrize("aligned", [True, False])
def test_rules_one_at_a_time(torch, native, aligned):
    none = dict(history=None, biases=0, allowed=None, temperature=False, penalties=False, drafted=False, aligned=aligned)
    for changes in ({}, dict(history=40), dict(history=40, penalties=True), dict(history=40, penalties=True, prompt=False),
                    dict(biases=20), dict(allowed="rows"), dict(allowed="one"), dict(temperature=True),
                    dict(drafted=True, penalties=True), dict(drafted="trees", penalties=True)):
        logits = Logits(torch, [2, 3], 777, "float16", **dict(none, **changes))
        logits.check(native, "float32", offset=0 if aligned else 5)
        logits.check(native, "bfloat16", probabilities=False, offset=0 if aligned else 5)


def test_long_histories_and_many_nodes(torch, native):
    logits = Logits(torch, [200, 1, 90], 300, "float32", history=30000, seed=4, drafted="trees")
    logits.check(native, "float32")


@pytest.mark.parametrize("past,words", [(32703, 1), (32704, 1), (32767, 0), (32768, 0)])
def test_counts_at_the_end_of_16_bits(torch, native, past, words):
    """One token all along a history, on both sides of the sizes at which a count and a bias no longer share a word."""
    alphabet, rows = 300, 64 if words else 1
    x = normal(torch, (rows, alphabet), past, "float32", 4.0)
    rules = dict(history=ints(torch, [[7] * past]), history_lengths=ints(torch, [past]), frequency=floats(torch, [2.0 ** -10]),
                 presence=floats(torch, [0.25]), bias_starts=ints(torch, [0, 2]), bias_tokens=ints(torch, [7, 8]),
                 bias_values=floats(torch, [0.5, -0.5]))
    if words:  # each node of the same token, on the line of those in front of it
        mask = [(1 << (r + 1)) - 1 for r in range(rows)]
        rules.update(tokens=ints(torch, [7] * rows), mask=torch.from_numpy(np.array(mask, np.uint64).view(np.int64))[:, None].cuda())
    counts = past + (torch.arange(rows, device="cuda").double() + 1 if words else torch.zeros(1, device="cuda").double())
    want = x.double()
    want[:, 7] = want[:, 7] - counts / 1024 - 0.25 + 0.5
    want[:, 8] -= 0.5
    out = torch.empty_like(x)
    native.adjust_logits(x, out, ints(torch, [0, rows]), probabilities=False, **rules)
    # The count's product, then two sums more of numbers below 2^6.
    near(torch, out, want, torch.full_like(want, 3 * H * 64))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("alphabet", [300, 8200, 16384, 32000, 50001, 128001])
def test_histories_past_16_bits_of_count(torch, native, kind, alphabet):
    """Counts and biases in words of their own, in each number of a thread's eights."""
    logits = Logits(torch, [2, 1, 0, 3], alphabet, kind, history=40000, seed=alphabet, biases=300, drafted="trees",
                    aligned=alphabet != 8200)
    logits.check(native, "float32")
    logits.check(native, kind, probabilities=False)


def test_more_biases_than_16_bits(torch, native):
    """Tokens that are listed many times, past the 65,535th bias of a sequence: the last one counts."""
    logits = Logits(torch, [2, 1], 20000, "float32", history=100, seed=5, biases=0)
    rng = np.random.default_rng(6)
    starts, tokens = [0, 90000, 160000], rng.integers(0, 20002, 160000)
    values = rng.normal(size=160000).astype(np.float32)
    for s in range(2):
        for i in range(starts[s], starts[s + 1]):
            if tokens[i] < 20000:
                logits.bias[s, tokens[i]] = values[i]
    logits.rules.update(bias_starts=ints(torch, starts), bias_tokens=ints(torch, tokens), bias_values=floats(torch, values))
    logits.check(native, "float32")
    logits.check(native, "bfloat16", probabilities=False)


def test_lengths_of_histories_out_of_range(torch, native):
    """Taken as 0, or as what there is room for; a prompt longer than its history is all of it."""
    logits = Logits(torch, [1, 2, 1], 60, "float32", history=20, seed=2)
    logits.rules["history_lengths"] = ints(torch, [-5, 1 << 30, 7])
    logits.rules["prompt_lengths"] = ints(torch, [3, -8, 1 << 30])
    logits.lengths, logits.prompts = np.array([0, 20, 7]), np.array([0, 0, 7])
    logits.check(native, "float32")


@pytest.mark.parametrize("alphabet", [50, 1000, 8200, 32001, 40001])
def test_tokens_out_of_range_are_passed_over(torch, native, alphabet):
    """In the history, among the nodes and among the biases, whatever the rules would make of them."""
    x = normal(torch, (6, alphabet), 1, "float32", 4.0)
    within = [0, alphabet // 2, alphabet - 1]
    outside = [alphabet, alphabet + 1, alphabet + 6, alphabet + 9, -1, -alphabet, 2 ** 31 - 1, -2 ** 31]
    starts, nodes = ints(torch, [0, 2, 4, 6]), ints(torch, [0, alphabet, 0, -1, 0, alphabet + 3])
    for repetition in (0.0, -0.5, 1.5, math.nan):
        rules = dict(repetition=floats(torch, [repetition] * 3), presence=floats(torch, [0.5] * 3),
                     frequency=floats(torch, [0.25] * 3), bias_starts=ints(torch, [0, 2, 2, 4]),
                     bias_tokens=ints(torch, [alphabet, alphabet + 2, 1, alphabet + 5]),
                     bias_values=floats(torch, [math.nan, math.inf, 0.0, math.inf]))
        lone = torch.where(torch.arange(6, device="cuda") % 2 == 0, 0, -1).int()  # the nodes that are of the alphabet
        for probabilities in (False, True):
            got, want = torch.empty_like(x), torch.empty_like(x)
            for out, tokens, past in ((got, nodes, within + outside), (want, lone, within + [-1] * len(outside))):
                native.adjust_logits(x, out, starts, probabilities=probabilities, history=ints(torch, [past] * 3),
                                     history_lengths=ints(torch, [len(past)] * 3), tokens=tokens, **rules)
            assert torch.equal(got.nan_to_num(-7.0), want.nan_to_num(-7.0)), (repetition, probabilities)
            assert repetition not in (-0.5, 1.5) or not bool(want.isnan().any())


@pytest.mark.parametrize("alphabet", [50, 1000, 40000])
def test_the_likeliest_token(torch, native, alphabet):
    """Temperature 0 and below, ties, rows without a token, infinities and what is not a number."""
    x = normal(torch, (9, alphabet), 1, "float32")
    x[0, [7, 3, alphabet - 1]] = 30.0
    x[1] = 2.5
    x[2] = -math.inf
    x[3, 11] = math.nan
    x[4, [20, 9]] = math.inf
    x[5, alphabet - 1] = 99.0
    allowed = torch.full((9, -(-alphabet // 32)), -1, dtype=torch.int32, device="cuda")
    allowed[6] = 0
    x[7, 0] = math.nan
    allowed[7, 0] = -2  # the one that is not a number is not allowed
    want = torch.zeros(9, alphabet)
    for r, t in ((0, 3), (1, 0), (4, 9), (5, alphabet - 1)):
        want[r, t] = 1
    want[3] = math.nan
    want[7, int(x[7, 1:].argmax()) + 1] = 1
    want[8, int(x[8].argmax())] = 1
    for t in (0.0, -1.0):
        out = torch.empty(9, alphabet, dtype=torch.bfloat16, device="cuda")
        native.adjust_logits(x, out, ints(torch, list(range(10))), allowed=allowed, temperature=torch.full((9,), t, device="cuda"))
        assert torch.equal(out.float().cpu().nan_to_num(-5.0), want.nan_to_num(-5.0))


@pytest.mark.parametrize("alphabet", [50, 1000, 40000])
def test_rows_that_are_empty_or_broken(torch, native, alphabet):
    """Masked places do not matter, whatever they hold; a row without a place is 0; the type's lowest number is one."""
    x = normal(torch, (7, alphabet), 1, "bfloat16")
    allowed = torch.full((7, -(-alphabet // 32)), -1, dtype=torch.int32, device="cuda")
    x[0, 3], x[1, 3], x[2, 3] = math.nan, math.inf, -math.inf
    x[3, 3], x[3, 4], allowed[3, 0] = math.nan, math.inf, ~0b11000
    allowed[4] = 0
    x[5] = torch.finfo(torch.bfloat16).min
    x[6] = -math.inf
    out = torch.empty(7, alphabet, device="cuda")
    native.adjust_logits(x, out, ints(torch, [0, 7]), allowed=allowed)
    assert bool(out[:2].isnan().all()) and not bool(out[2:].isnan().any())
    assert not bool(out[4].any()) and not bool(out[6].any()) and float(out[2, 3]) == 0.0 and not bool(out[3, 3:5].any())
    assert bool(((out[5].double() * alphabet - 1).abs() < 200 * H).all())
    assert bool(((out[[2, 3]].double().sum(1) - 1).abs() < 1e-5).all())


@pytest.mark.parametrize("alphabet", [4096, 32000, 70001])
def test_shares_far_below_the_largest(torch, native, alphabet):
    """A probability over the largest one, which leaves the sum out: e^((x - m) / t). The difference is rounded, and its product
    with the factor: 2 h of the exponent. The exponential is off by 2^-22 at most and the factor, joined from two floats, by less
    than h / 8 of the exponent; the largest's weight is 1, and both are rounded as they are scaled and stored, 4 h."""
    temperatures = [0.3, 0.37, 0.5, 0.61, 0.7, 0.77, 0.9, 1.0, 1.1, 1.3, 1.7, 2.3]
    x = normal(torch, (len(temperatures), alphabet), 7, "float32", 3.0)
    out = torch.empty_like(x)
    t = floats(torch, temperatures)
    native.adjust_logits(x, out, ints(torch, list(range(len(temperatures) + 1))), temperature=t)
    exponent = (x.double() - x.double().amax(1, keepdim=True)) / t.double()[:, None]
    want = exponent.exp()
    got = out.double() / out.double().amax(1, keepdim=True)
    room = want * (2.125 * H * exponent.abs() + 2.0 ** -22 + 4 * H) * (1 + 2.0 ** -12)
    normal_numbers = want > 2.0 ** -100
    assert bool(((got - want).abs() <= room)[normal_numbers].all()), float(((got - want).abs() / room)[normal_numbers].max())


@pytest.mark.parametrize("kind", KINDS)
def test_a_repeated_logit_is_divided(torch, native, kind):
    """x / r of a positive one and x r of another are each rounded once; h / 64 for what stands in for the quotient."""
    alphabet = 5000
    factors = [1.0, 1.1, 1.15, 1.2, 1.3, 1.5, 2.0, 3.0, 0.7, 7.3]
    x = normal(torch, (len(factors), alphabet), 9, kind, 4.0)
    out = torch.empty(x.shape, device="cuda")
    r = floats(torch, factors)
    history = torch.arange(alphabet, dtype=torch.int32, device="cuda").repeat(len(factors), 1)
    native.adjust_logits(x, out, ints(torch, list(range(len(factors) + 1))), probabilities=False, history=history,
                         history_lengths=ints(torch, [alphabet] * len(factors)), repetition=r)
    v, by = x.double(), r.double()[:, None]
    want = torch.where(v > 0, v / by, v * by)
    near(torch, out, want, H * (1 + 1 / 64) * want.abs())
    x[:, ::7], x[:, 1::7], x[:, 2::7] = math.inf, -math.inf, 0.0
    native.adjust_logits(x, out, ints(torch, list(range(len(factors) + 1))), probabilities=False, history=history,
                         history_lengths=ints(torch, [alphabet] * len(factors)), repetition=r)
    assert torch.equal(out.sign(), x.float().sign()) and torch.equal(out.isinf(), x.isinf())


def test_temperatures_at_their_ends(torch, native):
    """So small that its reciprocal overflows: the largest share it all; so large that all are alike."""
    x = floats(torch, [[1.0, 3.0, 3.0, -2.0]] * 4)
    t = floats(torch, [1e-44, 2.0 ** -126, 3e38, math.inf])
    out = torch.empty(4, 4, device="cuda")
    native.adjust_logits(x, out, ints(torch, [0, 1, 2, 3, 4]), temperature=t)
    assert out[:2].tolist() == [[0, 0.5, 0.5, 0]] * 2
    assert out[2:].tolist() == [[0.25] * 4] * 2


def test_logits_in_place_and_rows_of_no_sequence(torch, native):
    for alphabet, probabilities in ((1000, True), (1000, False), (70001, True), (70001, False)):
        logits = Logits(torch, [3, 2], alphabet, "float32", seed=alphabet)
        want = torch.empty(5, alphabet, device="cuda")
        logits.run(native, want, probabilities)
        wide = torch.full((8, alphabet), 7.0, device="cuda")
        wide[1:6] = logits.logits
        rules = {k: v for k, v in logits.rules.items() if probabilities or k != "temperature"}
        for name, fill in (("allowed", -1), ("tokens", 0)):
            old = rules[name]
            rules[name] = torch.full((8,) + tuple(old.shape[1:]), fill, dtype=old.dtype, device="cuda")
            rules[name][1:6] = old
        native.adjust_logits(wide, wide, logits.starts + 1, probabilities=probabilities, **rules)
        assert torch.equal(wide[1:6].nan_to_num(-1.0), want.nan_to_num(-1.0))
        assert bool((wide[[0, 6, 7]] == 7).all())


@pytest.mark.parametrize("alphabet", [50001, 128001])
def test_a_workspace_for_the_largest_batch(torch, native, alphabet):
    """One workspace for batches that shrink, across the numbers of rows at which a row has another number of parts."""
    need = native.library().tsac_hip_adjust_logits_workspace
    space = torch.full((need(64, alphabet) + 16,), 77, dtype=torch.uint8, device="cuda")
    for counts in ([40, 24], [63], [20, 17], [36], [31], [16], [15], [1]):
        logits = Logits(torch, counts, alphabet, "bfloat16", seed=sum(counts), biases=0, allowed=None)
        out = torch.empty(logits.rows, alphabet, device="cuda")
        logits.run(native, out, workspace=space[:need(64, alphabet)])
        want, room = logits.probabilities()
        near(torch, out, want, room + H * want + TINY["float32"])
        assert bool((space[-16:] == 77).all())


def test_logits_past_2_to_the_31_elements(torch, native):
    rows, alphabet = 17000, 131072
    x = torch.zeros(rows, alphabet, dtype=torch.bfloat16, device="cuda")
    x[-1, -1] = x[0, 5] = 20.0
    starts = ints(torch, [0, rows])
    native.adjust_logits(x, x, starts)
    top = math.exp(20) / (math.exp(20) + alphabet - 1)
    for r, t in ((0, 5), (rows - 1, alphabet - 1)):
        assert abs(float(x[r, t]) - top) < 2.0 ** -8 and float(x[r, (t + 1) % alphabet]) < 1e-8
    assert abs(float(x[9000].float().sum()) - 1) < 2.0 ** -7


# ---------------------------------------------------------------- streams, graphs, a run together

class Step:
    """A layer of a small model over a paged cache: norm, projection, rotation, attention, projection, the norm behind it,
    logits, rules, verification."""

    def __init__(self, torch, native, seed=0, counts=(5, 1, 12), lengths=(20, 0, 33)):
        self.torch, self.native = torch, native
        width, heads, kv, hw, alphabet = 256, 4, 2, 64, 500
        self.p = p = Pages(torch, native, list(lengths), list(counts), heads, kv, hw, seed=seed)
        rows, self.alphabet, self.dims = p.rows, alphabet, (width, heads, kv, hw)
        bf = torch.bfloat16
        self.x = normal(torch, (rows, width), seed + 5, "float32", 2.0)
        self.gain = normal(torch, (width,), seed + 6, "bfloat16", 0.2) + 1
        self.qkv_linear, self.out_linear, self.head = (linear_of(torch, native, n, k, seed + i) for i, (n, k) in enumerate(
            (((heads + 2 * kv) * hw, width), (width, heads * hw), (alphabet, width))))
        rng = np.random.default_rng(seed)
        self.parents = [-1 if i == 0 else int(rng.integers(0, i)) for c in counts for i in range(c)]
        self.parents_t = ints(torch, self.parents)
        empty = lambda *shape, kind=bf: torch.zeros(shape, dtype=kind, device="cuda")  # noqa: E731
        self.mask = empty(rows, 1, kind=torch.int64)
        self.q, self.s = empty(rows, width, kind=torch.int8), empty(rows, kind=torch.float32)
        self.qkv, self.turned, self.mixed = empty(rows, (heads + 2 * kv) * hw), empty(rows, heads, hw), empty(rows, heads, hw)
        self.q2, self.s2 = empty(rows, heads * hw, kind=torch.int8), empty(rows, kind=torch.float32)
        self.block, self.after = empty(rows, width), empty(rows, width, kind=torch.float32)
        self.q3, self.s3 = empty(rows, width, kind=torch.int8), empty(rows, kind=torch.float32)
        self.logits, self.probs = empty(rows, alphabet, kind=torch.float32), empty(rows, alphabet, kind=torch.float32)
        self.frequencies = torch.from_numpy(native.rotary_frequencies(hw)).cuda()
        self.history, self.history_lengths = ints(torch, rng.integers(0, alphabet, (len(counts), 64))), ints(torch, list(lengths))
        self.tokens = ints(torch, rng.integers(0, alphabet, rows))
        self.penalty = floats(torch, [1.2] * len(counts))
        self.uniforms, self.draws = floats(torch, rng.random(rows)), floats(torch, rng.random(len(counts)))
        self.path = ints(torch, -np.ones((len(counts), p.max_rows)))
        self.accepted, self.next = ints(torch, [0] * len(counts)), ints(torch, [0] * len(counts))
        self.longest = max(a + b for a, b in zip(lengths, counts))
        self.spaces = [torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for n in (
            native.attention_paged_workspace(p.cache, rows, heads, p.max_rows, self.longest),
            native.library().tsac_hip_adjust_logits_workspace(rows, alphabet),
            native.library().tsac_hip_verify_drafts_workspace(len(counts), alphabet))]

    def run(self):
        native, p, (width, heads, kv, hw) = self.native, self.p, self.dims
        native.tree_mask(self.parents_t, p.starts, p.max_rows, self.mask)
        native.block_norm(self.x.bfloat16(), norm=native.NORM_RMS, gain=self.gain, out=self.q, out_scales=self.s)
        self.qkv_linear[0].apply(self.q, self.s, self.qkv)
        parts = self.qkv.view(-1, heads + 2 * kv, hw)
        p.cache.append(0, parts[:, :heads], parts[:, heads:heads + kv], parts[:, heads + kv:], p.starts, p.max_rows,
                       self.frequencies, self.turned, mask=self.mask)
        native.attention_paged(p.cache, 0, self.turned, p.starts, p.max_rows, self.longest, self.mask, 0.125, self.mixed,
                               workspace=self.spaces[0])
        native.quantize_tokens(self.mixed.view(-1, heads * hw), self.q2, self.s2)
        self.out_linear[0].apply(self.q2, self.s2, self.block)
        native.block_norm(self.block, post=native.NORM_RMS, post_gain=self.gain, scale=0.5, residual=self.x, sum=self.after,
                          norm=native.NORM_LAYER, out=self.q3, out_scales=self.s3)
        self.head[0].apply(self.q3, self.s3, self.logits)
        native.adjust_logits(self.logits, self.probs, p.starts, history=self.history, history_lengths=self.history_lengths,
                             tokens=self.tokens, mask=self.mask, repetition=self.penalty, workspace=self.spaces[1])
        native.verify_drafts(self.probs, None, self.tokens, self.parents_t, p.starts, p.max_rows, self.uniforms, self.draws,
                             self.path, self.accepted, self.next, workspace=self.spaces[2])

    def results(self):
        return [t.clone() for t in (self.qkv, self.turned, self.p.keys, self.p.values, self.mixed, self.block, self.after,
                                    self.q3, self.s3, self.logits, self.probs, self.path, self.accepted, self.next)]


def test_a_step_of_a_model(torch, native):
    """Each stage against its definition on what the stage before it gave."""
    step = Step(torch, native)
    p, (width, heads, kv, hw) = step.p, step.dims
    step.run()
    qkv_linear, w, c, b = step.qkv_linear
    y, room = product(torch, step.q, step.s, w, c, b, "bfloat16")
    near(torch, step.qkv, y, room)
    down = []
    for s, count in enumerate(p.counts):
        mine = []
        for i in range(count):
            parent = step.parents[p.starts_list[s] + i]
            mine.append(0 if parent < 0 else mine[parent] + 1)
        down += [p.lengths[s] + d for d in mine]
    where = torch.tensor(down, device="cuda")
    parts = step.qkv.view(-1, heads + 2 * kv, hw)
    want, room = p.turned(parts[:, :heads], where, step.frequencies.tolist(), False, 1.0)
    near(torch, step.turned, want, room)
    # A row's own key is the one it is to see: its line's keys as they lie in the cache.
    for s, count in enumerate(p.counts):
        for i in range(count):
            row = p.starts_list[s] + i
            line, j = [], i
            while j >= 0:
                line.append(j)
                j = step.parents[p.starts_list[s] + j]
            spots = list(range(p.lengths[s])) + [p.lengths[s] + j for j in line]
            page = [int(p.table_list[s, t // 16]) for t in spots]
            within = [t % 16 for t in spots]
            k, v = p.keys[0, page, within].double(), p.values[0, page, within].double()
            k, v = (t.repeat_interleave(heads // kv, 1) for t in (k, v))
            weights = torch.softmax((k * step.turned[row].double()).sum(2) * 0.125, 0)
            mixed = (weights[:, :, None] * v).sum(0)
            # Two roundings of 2^-8 of an attention in 16 bits, each at most of the values' size.
            assert bool(((step.mixed[row].double() - mixed).abs() <= 3 * 2.0 ** -8 * (weights[:, :, None] * v.abs()).sum(0)).all())
    q, s = quantised(torch, step.mixed.view(-1, heads * hw))
    assert torch.equal(step.q2.double(), q) and torch.equal(step.s2, s)
    _, w, c, b = step.out_linear
    y, room = product(torch, step.q2, step.s2, w, c, b, "bfloat16")
    near(torch, step.block, y, room)
    _, w, c, b = step.head
    y, room = product(torch, step.q3, step.s3, w, c, b, "float32")
    near(torch, step.logits, y, room)
    assert bool(((step.probs.double().sum(1) - 1).abs() < 1e-5).all())
    assert bool((step.accepted >= 1).all()) and bool((step.next >= 0).all())
    assert step.path[:, 0].tolist() == [0] * len(p.counts)


def to_8_bits(q, scales, h, error):
    """Rows h that are off by at most `error`, as 8 bits and a scale each."""
    top = h.abs().amax(1)
    assert bool(((scales.double() - top / 127).abs() <= error.amax(1) / 127 + 2 * H * top / 127 + 2.0 ** -149).all())
    off = (q.double() * scales.double()[:, None] - h).abs()
    assert bool((off <= (0.5 + 2.0 ** -16) * scales.double()[:, None] + error).all())


def test_norms_rules_and_verification_of_a_step(torch, native):
    """What one stage hands to the next, each held against its definition on what it was given."""
    from test_gpu_drafts import verify_plain

    step = Step(torch, native, seed=7, counts=(6, 1, 12))
    p, (width, heads, kv, hw) = step.p, step.dims
    step.run()
    # Some drafted tokens are the likeliest behind their parents, so that there is something to accept.
    likely = step.probs.argmax(1).tolist()
    tokens = step.tokens.tolist()
    for s, count in enumerate(p.counts):
        for i in range(1, count, 2):
            tokens[p.starts_list[s] + i] = likely[p.starts_list[s] + step.parents[p.starts_list[s] + i]]
    step.tokens.copy_(ints(torch, tokens))
    step.uniforms.mul_(2.0 ** -12)
    step.run()
    rms = step.x.bfloat16().double()
    to_8_bits(step.q, step.s, *normed(torch, rms, torch.zeros_like(rms), native.NORM_RMS, step.gain, None, 1e-5))
    block = step.block.double()
    u, e = normed(torch, block, torch.zeros_like(block), native.NORM_RMS, step.gain, None, 1e-5)
    total = step.x.double() + 0.5 * u
    e = 0.5 * e + H * total.abs()  # halves are exact
    near(torch, step.after, total, e + H * (total.abs() + e) + TINY["float32"])
    to_8_bits(step.q3, step.s3, *normed(torch, total, e, native.NORM_LAYER, None, None, 1e-5))
    rules = Logits(torch, p.counts, step.alphabet, "float32", biases=0, allowed=None, temperature=False, prompt=False)
    n = len(p.counts)
    rules.logits, rules.history, rules.lengths = step.logits, step.history.cpu().numpy(), step.history_lengths.cpu().numpy()
    rules.prompts, rules.tokens, rules.lines = np.zeros(n, np.int64), np.array(tokens), []
    for s, count in enumerate(p.counts):
        lines = []
        for i in range(count):
            parent = step.parents[p.starts_list[s] + i]
            lines.append({i} | (lines[parent] if parent >= 0 else set()))
        rules.lines += lines
    rules.repetition, rules.presence, rules.frequency = np.full(n, 1.2, np.float32), np.zeros(n), np.zeros(n)
    want, room = rules.probabilities()
    near(torch, step.probs, want, room + H * want + TINY["float32"])
    probs, uniforms, draws = (t.cpu().numpy() for t in (step.probs, step.uniforms, step.draws))
    for s, count in enumerate(p.counts):
        part = slice(p.starts_list[s], p.starts_list[s] + count)
        path, following = verify_plain(probs[part], None, tokens[part], step.parents[part], uniforms[part], draws[s])
        got = int(step.accepted[s])
        assert (step.path[s, :got].tolist(), int(step.next[s])) == (path, following)
        assert step.path[s, got:].tolist() == [-1] * (p.max_rows - got)
    assert int(step.accepted.max()) > 2


def test_a_captured_step(torch, native):
    """Replays between other work give what the calls give, on new inputs too."""
    step = Step(torch, native, seed=3)
    before = step.p.keys.clone(), step.p.values.clone()
    step.run()
    want = step.results()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step.run()
    inputs = [step.x.clone(), step.x * 0.7 + 0.1]
    wants = [want]
    step.x.copy_(inputs[1])
    step.p.keys.copy_(before[0])
    step.p.values.copy_(before[1])
    step.run()
    wants.append(step.results())
    for i in (0, 1, 1, 0, 1):
        step.x.copy_(inputs[i])
        step.p.keys.copy_(before[0])
        step.p.values.copy_(before[1])
        torch.randn(1000, 1000, device="cuda").sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step.results(), wants[i])), i


def test_steps_on_two_streams(torch, native):
    """Two models' steps at once, each on its own stream with its own workspaces."""
    steps = [Step(torch, native, seed=i, counts=(7, 3, 2)) for i in (1, 2)]
    wants = []
    for step in steps:
        step.run()
        wants.append(step.results())
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(5):
        for step, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                step.run()
    torch.cuda.synchronize()
    for step, want in zip(steps, wants):
        assert all(torch.equal(a, b) for a, b in zip(step.results(), want))
