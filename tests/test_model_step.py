"""Refusals of the calls of a model's step, without a GPU: every check of sizes, pointers and strides comes before any
device work, as a status and a message. And the frequencies of rotated positions, which are computed on the host."""
import ctypes
import math

import numpy as np
import pytest

from tsac_hip import native

POINTER = 1 << 40  # never read: the calls below are refused on the host


def refused(status, text):
    assert status != 0
    assert text in native.library().tsac_hip_last_error().decode()


def cache(**changes):
    fields = dict(keys=POINTER, values=POINTER, layer_stride=4096, page_stride=2048, row_stride=128, layers=2, pages=8,
                  page_rows=16, heads=2, head_width=64, type=native.TYPE_BF16, table=POINTER, table_stride=4, held=POINTER,
                  lengths=POINTER, references=POINTER, sequences=3)
    fields.update(changes)
    return ctypes.byref(native.PagedCacheDesc(**fields))


def test_linears():
    lib = native.library()
    handle = ctypes.c_void_p()

    def create(values=POINTER, scales=POINTER, inputs=64, outputs=64, to=ctypes.byref(handle)):
        return lib.tsac_hip_channel_linear_create(values, scales, None, inputs, outputs, None, to)

    refused(create(values=None), "missing")
    refused(create(scales=None), "missing")
    refused(create(to=None), "missing")
    for inputs, outputs in ((0, 64), (131072, 64), (64, 0), (64, (1 << 24) + 1)):
        refused(create(inputs=inputs, outputs=outputs), "inputs")
    refused(lib.tsac_hip_channel_linear_apply(None, POINTER, 64, POINTER, 4, POINTER, 64, 0, None), "missing")
    lib.tsac_hip_channel_linear_destroy(None)


@pytest.mark.parametrize("changes,text", [
    (dict(x=None), "missing"), (dict(q=None), "missing"), (dict(scales=None), "missing"), (dict(type_=3), "type"),
    (dict(type_=-1), "type"), (dict(rows=1 << 24), "size"), (dict(width=0), "size"), (dict(width=65537), "size"),
    (dict(x=POINTER + 1), "misaligned"), (dict(type_=2, x=POINTER + 2), "misaligned"), (dict(x_stride=63), "overlap"),
    (dict(q=POINTER + 8), "16-byte"), (dict(q_stride=72), "16-byte"), (dict(q_stride=48), "apart"), (dict(q_stride=1 << 23), "apart"),
])
def test_quantised_tokens(changes, text):
    call = dict(x=POINTER, x_stride=64, type_=0, rows=4, width=64, q=POINTER, q_stride=64, scales=POINTER)
    call.update(changes)
    refused(native.library().tsac_hip_quantize_tokens(*call.values(), None), text)


@pytest.mark.parametrize("changes,text", [
    (dict(type=3), "type"), (dict(residual_type=4), "type"), (dict(type=0, residual_type=1), "residual"),
    (dict(type=2, residual_type=0), "residual"), (dict(rows=1 << 24), "size"), (dict(width=0), "size"),
    (dict(width=65537), "size"), (dict(input=None), "missing"), (dict(out=None, out_scales=POINTER), "scales"),
    (dict(post=3), "norm"), (dict(norm=-1), "norm"), (dict(input_stride=32), "overlap"), (dict(sum_stride=63), "overlap"),
    (dict(residual_stride=1), "overlap"), (dict(gate_stride=63), "overlap"), (dict(out_stride=63), "overlap"),
    (dict(input=POINTER + 1), "misaligned"), (dict(gain=POINTER + 1), "misaligned"), (dict(sum=POINTER + 1), "misaligned"),
    (dict(residual_type=2, residual=POINTER + 2), "misaligned"), (dict(out_scales=POINTER, out=POINTER + 8), "16-byte"),
    (dict(out_scales=POINTER, out_stride=72), "16-byte"),
])
def test_block_rows(changes, text):
    fields = dict(rows=4, width=64, type=0, residual_type=0, input=POINTER, input_stride=64, post=1, post_gain=POINTER,
                  gate=POINTER, gate_stride=64, scale=1.0, residual=POINTER, residual_stride=64, sum=POINTER, sum_stride=64,
                  norm=2, gain=POINTER, bias=POINTER, epsilon=1e-5, out=POINTER, out_stride=64)
    fields.update(changes)
    refused(native.library().tsac_hip_block_norm(ctypes.byref(native.BlockRows(**fields)), None), text)
    refused(native.library().tsac_hip_block_norm(None, None), "missing")


@pytest.mark.parametrize("changes,text", [
    (dict(heads=65537), "heads"), (dict(rows=1 << 24), "too many"), (dict(max_rows=1 << 24), "too many"),
    (dict(rotary=0), "rotated"), (dict(rotary=66), "rotated"), (dict(rotary=7), "rotated"), (dict(starts=None), "missing"),
    (dict(frequencies=None), "missing"), (dict(keys=None), "missing"), (dict(values=None), "missing"),
    (dict(query=None), "missing"), (dict(out=None), "missing"), (dict(positions=POINTER, mask=POINTER, words=1), "both"),
    (dict(mask=POINTER), "mask words"), (dict(mask=POINTER, words=1025), "mask words"), (dict(keys=POINTER + 8), "aligned"),
    (dict(row_stride=132), "aligned"), (dict(query_stride=130), "aligned"), (dict(out=POINTER + 2), "aligned"),
    (dict(row_stride=64), "overlap"), (dict(query_stride=128), "overlap"), (dict(out_stride=128), "overlap"),
])
def test_appended_rows(changes, text):
    fields = dict(query=POINTER, query_stride=256, out=POINTER, out_stride=256, heads=4, keys=POINTER, values=POINTER,
                  row_stride=128, rows=5, max_rows=5, starts=POINTER, frequencies=POINTER, rotary=64, amplitude=1.0)
    lib = native.library()
    refused(lib.tsac_hip_pages_append(cache(), 2, ctypes.byref(native.RotaryRows(**fields)), None, None), "layer")
    refused(lib.tsac_hip_pages_append(cache(), 0, None, None, None), "missing")
    refused(lib.tsac_hip_pages_append(cache(type=2), 0, ctypes.byref(native.RotaryRows(**fields)), None, None), "type")
    fields.update(changes)
    refused(lib.tsac_hip_pages_append(cache(), 0, ctypes.byref(native.RotaryRows(**fields)), None, None), text)


@pytest.mark.parametrize("changes,call,text", [
    (dict(starts=None), {}, "missing"), (dict(sequences=65536), {}, "sequences"),
    (dict(history=POINTER), {}, "history"), (dict(history=POINTER, history_lengths=POINTER, history_stride=1 << 40), {}, "history"),
    (dict(mask=POINTER), {}, "mask words"), (dict(mask=POINTER, words=1025), {}, "mask words"),
    (dict(bias_starts=POINTER, biases=3), {}, "biases"), (dict(bias_starts=POINTER, biases=1 << 31, bias_tokens=POINTER,
                                                               bias_values=POINTER), {}, "biases"),
    (dict(allowed=POINTER, allowed_stride=31), {}, "allowed"), (dict(temperature=POINTER), dict(probabilities=0), "temperature"),
    ({}, dict(logits=None), "missing"), ({}, dict(out=None), "missing"), ({}, dict(type_=3), "type"),
    ({}, dict(out_type=-1), "type"), ({}, dict(rows=1 << 24), "rows"), ({}, dict(alphabet=0), "alphabets"),
    ({}, dict(alphabet=(1 << 20) + 1), "alphabets"), ({}, dict(stride=999), "overlap"), ({}, dict(out_stride=999), "overlap"),
    ({}, dict(logits=POINTER + 1), "misaligned"), ({}, dict(out_type=2, out=POINTER + 2), "misaligned"),
    ({}, dict(out=POINTER, out_type=2), "in place"), ({}, dict(out=POINTER, out_stride=1024), "in place"),
    ({}, dict(workspace=POINTER + 8), "workspace"), ({}, dict(alphabet=40000, stride=40000, out_stride=40000), "workspace"),
])
def test_logit_rules(changes, call, text):
    arguments = dict(logits=POINTER, stride=1000, type_=0, rows=4, alphabet=1000, rules=None, probabilities=1,
                     out=POINTER + (1 << 30), out_stride=1000, out_type=0, workspace=None, size=0)
    arguments.update(call)
    fields = dict(starts=POINTER, sequences=2)
    fields.update(changes)
    arguments["rules"] = ctypes.byref(native.LogitRules(**fields))
    lib = native.library()
    refused(lib.tsac_hip_adjust_logits(*arguments.values(), None), text)
    arguments["rules"] = None
    assert lib.tsac_hip_adjust_logits(*arguments.values(), None) != 0
    assert lib.tsac_hip_adjust_logits_workspace(4, 0) == 0


def test_workspaces_of_logits():
    """One asked for once, for a program's largest batch, is enough for every smaller one; and the query grows with both sizes."""
    need = native.library().tsac_hip_adjust_logits_workspace
    for alphabet in (1, 32768, 32769, 50001, 65537, 128001, 1 << 20):
        sizes = [need(rows, alphabet) for rows in range(600)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])), alphabet
    for rows in (1, 3, 15, 16, 31, 32, 63, 64, 255, 256, 5000):
        sizes = [need(rows, alphabet) for alphabet in range(1, 1 << 20, 509)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])), rows


def test_frequencies():
    """Plain ones, divided ones, those of a larger base and those chosen by their turns, from the formulas."""
    for rotary in (2, 4, 20, 96, 128):
        plain = [10000.0 ** (-2 * i / rotary) for i in range(rotary // 2)]
        close = dict(rtol=1e-14, atol=0)
        assert np.allclose(native.rotary_frequencies(rotary), plain, **close)
        assert np.allclose(native.rotary_frequencies(rotary, scaling=native.ROTARY_LINEAR, factor=4), np.array(plain) / 4, **close)
        if rotary > 2:
            scaled = native.rotary_frequencies(rotary, scaling=native.ROTARY_BASE, factor=8.0)
            assert scaled[0] == 1.0 and math.isclose(scaled[-1], plain[-1] / 8, rel_tol=1e-13)
            assert all(a < b for a, b in zip(scaled[1:], plain[1:]))
        turned = native.rotary_frequencies(rotary, scaling=native.ROTARY_TURNS, factor=8.0, context=8192, slow=1.0, fast=4.0)
        for f, p in zip(turned, plain):
            turns = 8192 * p / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1) / 3))
            assert math.isclose(f, p * (keep + (1 - keep) / 8), rel_tol=1e-14)


@pytest.mark.parametrize("arguments,text", [
    (dict(rotary=0), "even"), (dict(rotary=3), "even"), (dict(rotary=130), "even"), (dict(base=0.0), "base"),
    (dict(base=float("nan")), "base"), (dict(scaling=4), "scaling"), (dict(scaling=1, factor=0.0), "factor"),
    (dict(rotary=2, scaling=2, factor=2.0), "one pair"), (dict(scaling=3, factor=2.0), "context"),
    (dict(scaling=3, factor=2.0, context=64.0, slow=2.0, fast=2.0), "turns"),
])
def test_frequencies_that_are_none(arguments, text):
    with pytest.raises(native.HipError, match=text):
        native.rotary_frequencies(**dict(dict(rotary=64), **arguments))


def test_bindings_check_their_tensors():
    torch = pytest.importorskip("torch")

    def ints(*shape):
        return torch.zeros(shape, dtype=torch.int32)

    x, q = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 64, dtype=torch.int8)
    floats = torch.zeros(4)
    for bad in [(x, q[:3], floats), (x, q.float(), floats), (x.T, q, floats), (x.double(), q, floats),
                (x, q, floats[:3]), (x, q, floats.half()), (x, q, floats)]:  # the last: not on a GPU
        with pytest.raises(native.HipError):
            native.quantize_tokens(*bad)
    for bad in [(q.float(), floats), (q[0], floats), (q, torch.zeros(3)), (q, floats.half()), (q, None)]:
        with pytest.raises(native.HipError):
            native.ChannelLinear(*bad)
    for bad in [dict(residual=x.half()), dict(sum=x.double()), dict(residual=x.float(), sum=x), dict(gate=x[:2]),
                dict(gate=x.float()), dict(out=x.float()), dict(out=x, out_scales=floats), dict(out_scales=floats),
                dict(gain=floats), dict(gain=x), dict(norm=native.NORM_RMS, out=x)]:  # the last: not on a GPU
        with pytest.raises(native.HipError):
            native.block_norm(x, **bad)
    pool = torch.zeros(2, 8, 16, 2, 64, dtype=torch.bfloat16)
    paged = native.PagedCache(pool, pool.clone(), ints(3, 4), ints(3), ints(3), ints(8))
    query, rows = torch.zeros(5, 4, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    good = dict(layer=0, query=query, keys=rows, values=rows, starts=ints(4), max_rows=5,
                frequencies=torch.zeros(32, dtype=torch.float64), out=query)
    for bad in [dict(query=query.half()), dict(out=query[:4]), dict(keys=rows[:4]), dict(values=query), dict(starts=ints(3)),
                dict(frequencies=torch.zeros(32)), dict(positions=ints(4)), dict(mask=torch.zeros(5, dtype=torch.int64)),
                dict(mask=torch.zeros(4, 1, dtype=torch.int64)), dict(values=torch.zeros(5, 3, 64, dtype=torch.bfloat16)[:, :2]),
                {}]:
        with pytest.raises(native.HipError):
            paged.append(**dict(good, **bad))
    logits = torch.zeros(4, 100)
    for bad in [dict(out=logits[:, :99]), dict(out=logits.double()), dict(history=ints(2, 5), history_lengths=ints(1)),
                dict(history=ints(10), history_lengths=ints(2)), dict(tokens=ints(3)), dict(mask=torch.zeros(4, dtype=torch.int64)),
                dict(repetition=torch.zeros(1)), dict(temperature=ints(2)), dict(bias_starts=ints(2)), dict(allowed=ints(4, 3)),
                dict(allowed=ints(3, 4)), dict(allowed=ints(4)), {}]:
        with pytest.raises(native.HipError):
            native.adjust_logits(**dict(dict(logits=logits, out=logits.clone(), starts=ints(3)), **bad))


def test_biases_come_with_their_starts():
    """Tokens and values alone are no biases of any sequence: refused, not passed over."""
    torch = pytest.importorskip("torch")
    logits, starts = torch.zeros(4, 100), torch.zeros(3, dtype=torch.int32)
    tokens, values = torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    for some in (dict(bias_tokens=tokens, bias_values=values), dict(bias_tokens=tokens), dict(bias_values=values),
                 dict(bias_starts=starts, bias_tokens=tokens), dict(bias_starts=starts, bias_values=values)):
        with pytest.raises(native.HipError, match="biases"):
            native.adjust_logits(logits, logits.clone(), starts, **some)
