"""Drafted decoding on the MI355X: pages, attention over them, tree masks and verification,
through the C ABI, against plain implementations in 64 bits written from the definitions.

Attention's tolerance, element by element, with u half a step of the 16-bit type (2^-8 for BF16,
2^-11 for half): the output's rounding is u |out|; each weight's rounding before the second product
u sum w|v|, and as the rounded weights are summed, sum w e v - out sum w e with |e| <= u, u |out| more; a
score's error (32-bit sums of head_width products, their scaling and the exponential's argument) d = (head_width + 8) 2^-24 sum|q k| scale log2(e) moves a weight and its share of the sum by 2 d,
the exponential itself and 32-bit sums of T terms by (T + 16) 2^-24:
|error| <= 2 u |out| + (u + 2 d + (T + 16) 2^-24) sum w|v|, times 1 + 2^-6 for products of these."""
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


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
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def random_tree(rng, nodes, roots=1):
    return [-1 if i < roots else int(rng.integers(max(0, i - 6), i)) for i in range(nodes)]


def line(parents, i):
    """The node and those above it."""
    found = set()
    while i >= 0:
        found.add(i)
        i = parents[i] if 0 <= parents[i] < i else -1
    return found


def pack_masks(torch, rows, words):
    """int64 [rows][words] of sets of bits."""
    out = np.zeros((len(rows), words), np.uint64)
    for r, bits in enumerate(rows):
        for b in bits:
            out[r, b // 64] |= np.uint64(1) << np.uint64(b % 64)
    return torch.from_numpy(out.view(np.int64)).cuda()


class Batch:
    """A paged cache of random keys and values, new rows of each sequence, and the definition."""

    def __init__(self, torch, native, lengths, counts, heads=4, kv_heads=2, width=64, page_rows=16, kind="bfloat16",
                 layers=1, seed=0, scale=None, spare=3, magnitude=1.0):
        self.torch, self.native = torch, native
        self.lengths, self.counts, self.heads, self.kv, self.width = lengths, counts, heads, kv_heads, width
        self.page_rows, self.kind = page_rows, kind
        self.rng = rng = np.random.default_rng(seed)
        held = [-(-(a + b) // page_rows) for a, b in zip(lengths, counts)]
        pages = sum(held) + spare
        order = rng.permutation(pages)
        table = -np.ones((len(lengths), max(held + [1]) + 1), np.int32)
        at = 0
        for s, h in enumerate(held):
            table[s, :h] = order[at:at + h]
            at += h
        references = np.zeros(pages, np.int32)
        references[order[:at]] = 1
        dtype = getattr(torch, kind)
        g = torch.Generator(device="cuda").manual_seed(seed + 1)

        def normal(*shape, m=1.0):
            return (torch.randn(*shape, generator=g, device="cuda") * m).to(dtype)

        self.keys = normal(layers, pages, page_rows, kv_heads, width, m=magnitude)
        self.values = normal(layers, pages, page_rows, kv_heads, width)
        self.table, self.held = ints(torch, table), ints(torch, held)
        self.starts_list = [0] + np.cumsum(counts).tolist()
        self.starts, self.rows = ints(torch, self.starts_list), self.starts_list[-1]
        self.cache = native.PagedCache(self.keys, self.values, self.table, self.held, ints(torch, lengths),
                                       ints(torch, references))
        self.qkv = normal(max(self.rows, 1), heads + 2 * kv_heads, width, m=magnitude)[:self.rows]
        self.query = self.qkv[:, :heads]
        self.scale = 1 / math.sqrt(width) if scale is None else scale
        self.max_rows = max(counts + [1])
        self.max_length = max([a + b for a, b in zip(lengths, counts)] + [1])

    def attend(self, mask=None, layer=0, max_length=None, workspace=None, query=None):
        torch = self.torch
        # Rows of a wider buffer, whose other parts have to stay.
        self.buffer = torch.full((self.rows + 2, self.heads + 1, self.width), 7.0, dtype=self.query.dtype, device="cuda")
        out = self.buffer[1:self.rows + 1, :self.heads]
        self.native.attention_paged(self.cache, layer, self.query if query is None else query, self.starts,
                                    self.max_rows, max_length or self.max_length, mask, self.scale, out,
                                    workspace=workspace)
        torch.cuda.synchronize()
        assert bool((self.buffer[:, self.heads:] == 7).all()) and bool((self.buffer[[0, -1]] == 7).all())
        return out

    def position(self, s, t, layer=0):
        """(keys, values) [kv][width] at a position, None where there is no page."""
        index = t // self.page_rows
        table = self.table.cpu()
        if index >= min(int(self.held[s]), table.shape[1]):
            return None
        page = int(table[s, index])
        if not 0 <= page < self.keys.shape[1]:
            return None
        return self.keys[layer, page, t % self.page_rows], self.values[layer, page, t % self.page_rows]

    def expected(self, sees, layer=0):
        """(out, tolerance) [rows][heads][width]; sees(s, i) is the set of the new rows that row i sees."""
        torch = self.torch
        u = UNIT[self.kind]
        out = torch.zeros(self.rows, self.heads, self.width, dtype=torch.float64)
        room = torch.zeros_like(out)
        group = self.heads // self.kv
        for s, (length, count) in enumerate(zip(self.lengths, self.counts)):
            if not count:
                continue
            where = [self.position(s, t, layer) for t in range(length + count)]
            there = [t for t, w in enumerate(where) if w is not None]
            if not there:
                continue
            k = torch.stack([where[t][0] for t in there]).double().cpu()
            v = torch.stack([where[t][1] for t in there]).double().cpu()
            q = self.query[self.starts_list[s]:self.starts_list[s + 1]].double().cpu()
            for i in range(count):
                mine = sees(s, i)
                keep = [a for a, t in enumerate(there) if t < length or t - length in mine]
                if not keep:
                    continue
                for h in range(self.heads):
                    kk, vv = k[keep, h // group], v[keep, h // group]
                    score = kk @ q[i, h] * self.scale
                    top = score.max()
                    if top == -math.inf:
                        continue
                    w = torch.exp(score - top)
                    w = w / w.sum()
                    row = self.starts_list[s] + i
                    out[row, h] = w @ vv
                    spread = w @ vv.abs()
                    d = (self.width + 8) * 2.0 ** -24 * float((kk.abs() @ q[i, h].abs()).max()) * abs(self.scale) * 1.4427
                    room[row, h] = (2 * u * out[row, h].abs() + (u + 2 * d + (len(keep) + 16) * 2.0 ** -24) * spread) * (
                        1 + 2.0 ** -6)
        return out, room

    def check(self, got, sees, layer=0):
        out, room = self.expected(sees, layer)
        got = got.double().cpu()
        nan = out.isnan()
        assert bool((got.isnan() == nan).all()), "not a number in other places"
        bad = ((got - out).abs() > room) & ~nan & (got != out)
        assert not bool(bad.any()), (int(bad.sum()), float(((got - out).abs() - room)[~nan].max()))


def chain(_, i):
    return set(range(i + 1))


# ---------------------------------------------------------------- attention

LENGTHS = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300]


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("heads,kv_heads,width", [(16, 16, 64), (4, 4, 128), (8, 2, 128), (6, 1, 64), (5, 1, 128)])
@pytest.mark.parametrize("nodes", [1, 3, 12, 40])
def test_attention_of_chains(torch, native, kind, heads, kv_heads, width, nodes):
    """Single tokens and chains, ragged, over every boundary of pages and blocks, some sequences empty."""
    counts = [(nodes - i % 3) if i % 5 != 3 else 0 for i in range(len(LENGTHS))]
    counts = [max(c, 0) for c in counts]
    b = Batch(torch, native, LENGTHS, counts, heads, kv_heads, width, 16, kind, seed=nodes)
    b.check(b.attend(), chain)


@pytest.mark.parametrize("kind,width", [("bfloat16", 64), ("float16", 128)])
@pytest.mark.parametrize("page_rows", [16, 32, 64, 256])
@pytest.mark.parametrize("nodes", [2, 25, 64, 70, 130])
def test_attention_of_trees(torch, native, kind, width, page_rows, nodes):
    lengths = [0, 1, 31, 50, 100, 333]
    counts = [max(1, nodes - 7 * i) for i in range(len(lengths))]
    b = Batch(torch, native, lengths, counts, 4, 2, width, page_rows, kind, layers=2, seed=nodes)
    trees = [random_tree(b.rng, n, roots=1 + n % 2) for n in counts]
    words = -(-max(counts) // 64)
    mask = torch.zeros(b.rows, words, dtype=torch.int64, device="cuda")
    native.tree_mask(ints(torch, sum(trees, [])), b.starts, b.max_rows, mask)
    rows = [line(t, i) for t in trees for i in range(len(t))]
    assert torch.equal(mask, pack_masks(torch, rows, words))
    for layer in range(2):
        b.check(b.attend(mask, layer), lambda s, i: line(trees[s], i), layer)


@pytest.mark.parametrize("lengths,nodes,heads,kv_heads,width", [
    ([5000, 1, 2049], 1, 8, 2, 128), ([20011], 5, 4, 4, 64), ([9000, 8191, 8193, 3], 20, 2, 1, 64), ([0, 7], 300, 2, 2, 64)])
def test_attention_over_many_chunks(torch, native, lengths, nodes, heads, kv_heads, width):
    """Long contexts are split over workgroups; the launch's guess of the longest does not matter."""
    b = Batch(torch, native, lengths, [max(1, nodes - i) for i in range(len(lengths))], heads, kv_heads, width, 64, seed=3)
    out, room = b.expected(chain)
    for guess in (None, 1, 700, 100000):
        got = b.attend(max_length=guess).double().cpu()
        assert bool(((got - out).abs() <= room).all()), guess


@pytest.mark.parametrize("kind,heads,kv_heads,width", [("bfloat16", 32, 16, 64), ("float16", 32, 8, 128)])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_many_tall_tiles(torch, native, kind, heads, kv_heads, width, tree):
    """As many (sequence, head) pairs as units, each of more than 128 query rows; a sequence's garbage behind
    its end, a value of one node that is not finite."""
    lengths = [(37 * i) % 301 for i in range(32)]
    counts = [70 - i if i != 9 else 0 for i in range(32)]
    b = Batch(torch, native, lengths, counts, heads, kv_heads, width, 16, kind, seed=21)
    trees = [random_tree(b.rng, n) for n in counts]
    used = torch.zeros(b.keys.shape[1:3], dtype=torch.bool)
    table = b.table.cpu()
    for s in range(32):
        for t in range(lengths[s] + counts[s]):
            used[int(table[s, t // 16]), t % 16] = True
    b.keys[0][~used] = math.nan
    b.values[0][~used] = math.inf
    if tree:
        page, row = int(table[3, (lengths[3] + 9) // 16]), (lengths[3] + 9) % 16
        b.values[0, page, row, 0, 5] = math.inf
    rows = [line(t, i) for t in trees for i in range(len(t))]
    got = b.attend(pack_masks(torch, rows, 2) if tree else None)
    if tree:
        reached = torch.zeros(got.shape, dtype=torch.bool)
        for i in range(counts[3]):
            reached[b.starts_list[3] + i, :heads // kv_heads, 5] = 9 in line(trees[3], i)
        assert torch.equal(got.cpu() == math.inf, reached) and bool(got.cpu()[~reached].isfinite().all())
        b.values[0, page, row, 0, 5] = 0.0
        out, room = b.expected(lambda s, i: line(trees[s], i))
        assert bool((((got.double().cpu() - out).abs() <= room) | reached).all())
    else:
        b.check(got, chain)


@pytest.mark.parametrize("kind,heads,kv_heads,width", [("bfloat16", 16, 8, 128), ("float16", 32, 16, 64)])
@pytest.mark.parametrize("nodes,longest", [(1, 400), (12, 100), (20, 150), (31, 33)])
@pytest.mark.parametrize("guess", [300, 8000])
def test_attention_of_many_short_sequences(torch, native, kind, heads, kv_heads, width, nodes, longest, guess):
    """More (sequence, head) pairs than units: of one to four 16-row parts each, empty ones among them, whether the
    launch is shaped for short sequences or for long ones."""
    rng = np.random.default_rng(nodes)
    lengths = [int(x) for x in rng.integers(0, longest, 36)]
    counts = [0 if i % 7 == 3 else max(1, nodes - i % 4) for i in range(36)]
    b = Batch(torch, native, lengths, counts, heads, kv_heads, width, 16, kind, seed=41)
    trees = [random_tree(b.rng, n) for n in counts]
    mask = pack_masks(torch, [line(t, i) for t in trees for i in range(len(t))], 1)
    b.values[0, int(b.table[5, 0]), 0, 0, 3] = math.nan if lengths[5] else 0.0  # cached: reaches all of its rows
    b.check(b.attend(mask, max_length=guess), lambda s, i: line(trees[s], i))


def test_attention_of_more_workgroups_than_a_launch_holds(torch, native):
    """A batch of single rows and one prompt, announced as 65,536 rows a sequence: the tiles that have rows are
    those of the smaller announcement, the last sequences in a second launch."""
    rng = np.random.default_rng(7)
    sequences = 2100
    lengths = [int(x) for x in rng.integers(0, 30, sequences)]
    counts = [1] * sequences
    counts[-3], counts[5], counts[2050] = 300, 0, 40
    b = Batch(torch, native, lengths, counts, 16, 8, 64, 16, seed=51)
    want = b.attend().clone()
    assert b.max_rows == 300 and bool((want != 7).all())
    b.max_rows = 65536
    assert torch.equal(b.attend(), want)


def test_attention_of_more_workgroups_than_a_call_holds(torch, native):
    sequences, heads = 65535, 16384
    keys = torch.zeros(1, 1, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    table, held, lengths = (torch.zeros(*shape, dtype=torch.int32, device="cuda")
                            for shape in ((sequences, 1), (sequences,), (sequences,)))
    cache = native.PagedCache(keys, keys.clone(), table, held, lengths, ints(torch, [0]))
    query = torch.zeros(1, heads, 64, dtype=torch.bfloat16, device="cuda")
    out, starts = torch.full_like(query, 7.0), torch.zeros(sequences + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(native.HipError, match="too many"):
        native.attention_paged(cache, 0, query, starts, 65536, 64, None, 1.0, out)
    torch.cuda.synchronize()
    assert bool((out == 7).all())


@pytest.mark.parametrize("kind,heads,kv_heads,width", [("bfloat16", 32, 8, 128), ("float16", 24, 4, 64)])
@pytest.mark.parametrize("tree", [False, True])
def test_tall_tiles_over_chunks(torch, native, kind, heads, kv_heads, width, tree):
    """A launch that is shaped for a long context takes tiles of 256 rows over chunks of it, whatever there is."""
    b = Batch(torch, native, [4900, 2303], [41, 36], heads, kv_heads, width, 64, kind, seed=31)
    trees = [random_tree(b.rng, n) for n in b.counts]
    mask = pack_masks(torch, [line(t, i) for t in trees for i in range(len(t))], 1) if tree else None
    out, room = b.expected((lambda s, i: line(trees[s], i)) if tree else chain)
    for guess in (70000, 140000):
        got = b.attend(mask, max_length=guess).double().cpu()
        assert bool(((got - out).abs() <= room).all()), guess


@pytest.mark.parametrize("nodes", [3, 40])
def test_rows_behind_the_last_sequence_stay(torch, native, nodes):
    b = Batch(torch, native, [50, 20, 9], [nodes, nodes, nodes], 4, 2, 64, 16, seed=6)
    full = b.attend().clone()
    b.starts = ints(torch, [0, nodes, 2 * nodes, 2 * nodes])
    got = b.attend()
    assert torch.equal(got[:2 * nodes], full[:2 * nodes]) and bool((got[2 * nodes:] == 7).all())


@pytest.mark.parametrize("magnitude,scale", [(30.0, None), (1.0, 0.0), (1.0, -1.0), (60.0, 1.0)])
def test_attention_of_large_and_equal_scores(torch, native, magnitude, scale):
    """Scores far apart move the reference many times; equal ones weigh the same."""
    b = Batch(torch, native, [700, 64, 3], [3, 20, 9], 4, 2, 64, 32, "float16", seed=5, magnitude=magnitude, scale=scale)
    b.check(b.attend(), chain)


@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("nodes,tree", [(1, False), (12, True), (40, False), (40, True)])
@pytest.mark.parametrize("gap", [10.0, 14.0, 16.0, 17.5, 18.0])
def test_small_weights_in_half_precision_count(torch, native, width, nodes, tree, gap):
    """Every sixteenth key scores `gap` above the others and has a value of 0, so that all of the output comes
    from weights of e^-gap. As operands in half, of which the largest is 2^7 or more, they are off by half a step:
    2^-11 of them or, below the smallest normal number, 2^-25, which is 2^-32 of the largest weight. Everything else
    as above, with f the weights against the largest one and u_f = max(u f, 2^-32): the output's rounding is u |out|
    (no outputs are subnormal here) and
    |error| <= u |out| + sum (u_f + f (2 d + (T + 16) 2^-24)) |v| / sum f + |out| sum u_f / sum f, times 1 + 2^-6."""
    heads, kv = 4, 2
    b = Batch(torch, native, [600, 33], [nodes, nodes], heads, kv, width, 16, "float16", seed=61)
    g = torch.Generator(device="cuda").manual_seed(62)
    # Scores are the keys' first coordinates: exact but for the scale, a power of two or one rounding.
    b.query.zero_()
    b.query[:, :, 0] = 8.0
    b.scale = 0.125
    b.keys[..., 0] = torch.rand(b.keys.shape[:-1], generator=g, device="cuda").half() * 0.25
    b.keys[0, :, 3, :, 0] = gap
    b.values.copy_(8000 + 22000 * torch.rand(b.values.shape, generator=g, device="cuda"))
    b.values[0, :, 3] = 0
    trees = [random_tree(b.rng, n) for n in b.counts]
    sees = (lambda s, i: line(trees[s], i)) if tree else chain
    got = b.attend(pack_masks(torch, [line(t, i) for t in trees for i in range(len(t))], 1) if tree else None)
    got = got.double().cpu()
    for s, (length, count) in enumerate(zip(b.lengths, b.counts)):
        where = [b.position(s, t) for t in range(length + count)]
        keys, values = (torch.stack([w[side] for w in where]).double().cpu() for side in range(2))
        for i in range(count):
            keep = [t for t in range(length + count) if t < length or t - length in sees(s, i)]
            for h in range(heads):
                score, v = keys[keep, h // 2, 0], values[keep, h // 2]
                f = torch.exp(score - score.max())
                out = f @ v / f.sum()
                d = (width + 8) * 2.0 ** -24 * gap * 1.4427
                step = torch.clamp(f * UNIT["float16"], min=2.0 ** -32)
                room = ((step + f * (2 * d + (len(keep) + 16) * 2.0 ** -24)) @ v + out * step.sum()) / f.sum()
                room = (room + UNIT["float16"] * out) * (1 + 2.0 ** -6)
                error = (got[b.starts_list[s] + i, h] - out).abs()
                assert float(out.min()) > 2.0 ** -14 and bool((error <= room).all()), (s, i, h, float((error / out).max()))


@pytest.mark.parametrize("nodes", [1, 70])
def test_attention_past_32_bits_of_offset(torch, native, nodes):
    """Two layers of 2,100 pages of 2^20 elements: the second's last page lies past 2^32 elements, and 2^33 bytes."""
    b = Batch(torch, native, [3000, 900], [nodes, nodes], 16, 8, 128, 1024, layers=2, seed=71, spare=2094)
    b.table[0, 0] = b.keys.shape[1] - 1
    assert b.keys[1].storage_offset() + b.keys.stride(1) * int(b.table[0, 0]) > 2 ** 32
    b.check(b.attend(layer=1), chain, layer=1)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("nodes,tree", [(1, False), (40, False), (40, True)])
@pytest.mark.parametrize("size", [10, 23, 25, 26])
def test_scores_that_are_large_and_close(torch, native, kind, width, nodes, tree, size):
    """Scores 2^size + 8 j, j from 0 to 5, rising with the position, exact in 32 bits, though as powers of two their
    neighbours lie up to 8 apart. With f the weights against the largest and u_f = max(u f, 2^-32) in half, u f in
    BF16, exponents of up to 58 are off by half a step of theirs and the factor log2 e by one: d = 58 * 2^-23, and
    |error| <= u |out| + sum (u_f + f (d + (T + 16) 2^-24)) |v| / sum f + |out| sum u_f / sum f, times 1 + 2^-6."""
    heads, kv, u = 4, 2, UNIT[kind]
    b = Batch(torch, native, [1500, 33], [nodes, nodes], heads, kv, width, 16, kind, seed=81, scale=1.0)
    g = torch.Generator(device="cuda").manual_seed(82)
    b.query.zero_()
    b.query[:, :, 0], b.query[:, :, 1] = 2.0 ** 15, 1.0
    b.keys.zero_()
    b.keys[..., 0] = 2.0 ** (size - 15)
    b.keys[..., 1] = 8.0 * torch.randint(0, 6, b.keys.shape[:-1], generator=g, device="cuda").to(b.keys.dtype)
    for i, page in enumerate(b.table[0].tolist()):  # rising, so that every wave or team meets one after another
        b.keys[0, page, :, :, 1] = 8.0 * min(5, i // 16) if page >= 0 else 0.0
    trees = [random_tree(b.rng, n) for n in b.counts]
    sees = (lambda s, i: line(trees[s], i)) if tree else chain
    got = b.attend(pack_masks(torch, [line(t, i) for t in trees for i in range(len(t))], 1) if tree else None)
    got = got.double().cpu()
    for s, (length, count) in enumerate(zip(b.lengths, b.counts)):
        where = [b.position(s, t) for t in range(length + count)]
        keys, values = (torch.stack([w[side] for w in where]).double().cpu() for side in range(2))
        for i in range(0, count, 7):
            keep = [t for t in range(length + count) if t < length or t - length in sees(s, i)]
            for h in range(heads):
                score, v = keys[keep, h // 2, 1], values[keep, h // 2]
                f = torch.exp(score - score.max())
                out = f @ v / f.sum()
                step = torch.clamp(f * u, min=2.0 ** -32) if kind == "float16" else f * u
                room = (step + f * (58 * 2.0 ** -23 + (len(keep) + 16) * 2.0 ** -24)) @ v.abs() / f.sum()
                room = (room + (u + step.sum() / f.sum()) * out.abs()) * (1 + 2.0 ** -6)
                error = (got[b.starts_list[s] + i, h] - out).abs()
                assert bool((error <= room).all()), (s, i, h, float((error / room).max()))


def test_rows_without_keys_are_zero(torch, native):
    b = Batch(torch, native, [0, 40, 0], [6, 6, 40], 4, 2, 64)
    seen = {(0, 2): {2}, (0, 5): {0, 3}, (2, 39): {0}}
    mask = pack_masks(torch, [seen.get((s, i), set()) for s, n in enumerate(b.counts) for i in range(n)], 1)
    got = b.attend(mask)
    b.check(got, lambda s, i: seen.get((s, i), set()))
    assert bool((got[0] == 0).all()) and bool((got[12:51] == 0).all()) and bool((got[2] != 0).any())


@pytest.mark.parametrize("kind,width", [("bfloat16", 64), ("bfloat16", 128), ("float16", 64), ("float16", 128)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_a_row_does_not_see_does_not_reach_it(torch, native, kind, width, bad):
    """Pages hold garbage behind a sequence's end; a drafted row that is not finite reaches only the rows below it."""
    lengths, counts = [37, 0, 64, 90], [11, 20, 33, 7]
    b = Batch(torch, native, lengths, counts, 4, 2, width, 32, kind, seed=8)
    trees = [random_tree(b.rng, n) for n in counts]
    table = b.table.cpu()

    def at(s, t):
        return int(table[s, t // 32]), t % 32

    used = {at(s, t) for s in range(4) for t in range(lengths[s] + counts[s])}
    for page in range(b.keys.shape[1]):
        for row in range(32):
            if (page, row) not in used:
                b.keys[0, page, row] = bad
                b.values[0, page, row] = bad
    broken = {0: 4, 1: 13, 2: 1, 3: 6}
    for s, node in broken.items():
        page, row = at(s, lengths[s] + node)
        b.values[0, page, row, :, 3::5] = bad
        if s == 3:
            b.keys[0, page, row] = math.nan
    mask = pack_masks(torch, [line(t, i) for t in trees for i in range(len(t))], 1)
    got = b.attend(mask).double().cpu()
    out, room = b.expected(lambda s, i: line(trees[s], i))
    finite = out.isfinite()
    reached = torch.zeros_like(finite)
    for s, node in broken.items():
        for i in range(counts[s]):
            if node in line(trees[s], i):
                row = b.starts_list[s] + i
                reached[row, :, slice(None) if s == 3 else slice(3, None, 5)] = True
    assert bool((finite == ~reached).all()), "the definition itself"
    assert bool((got.isfinite() == finite).all())
    assert bool(((got - out).abs() <= room)[finite].all())
    assert bool((got.isnan() == out.isnan()).all()) and bool((got[out.isinf()] == out[out.isinf()]).all())


def test_a_cached_value_that_is_not_finite_reaches_all_rows(torch, native):
    b = Batch(torch, native, [100], [5], 4, 2, 64, 16, seed=2)
    b.values[0, int(b.table[0, 2]), 5, 1, 7] = math.inf
    got = b.attend()
    assert bool((got[:, 2:, 7] == math.inf).all())
    assert int((~got.isfinite()).sum()) == 5 * 2


@pytest.mark.parametrize("number", [-1, 1 << 30, "pool"])
def test_positions_without_a_page_are_not_seen(torch, native, number):
    """Pages out of the pool, and positions past what is held, in the middle and at the end."""
    b = Batch(torch, native, [200, 70, 40], [9, 9, 9], 4, 2, 64, 16, seed=4)
    b.table[0, 3] = b.keys.shape[1] if number == "pool" else number
    b.table[1, 0] = -2
    b.held[2] = 1  # of 4
    b.check(b.attend(), chain)
    b.held.zero_()
    assert bool((b.attend() == 0).all())


def test_numbers_out_of_range_stay_inside(torch, native):
    """Lengths and row ranges that make no sense give something, and touch nothing else."""
    b = Batch(torch, native, [50, 50, 50], [4, 4, 4], 4, 2, 64, 16, seed=4)
    good = b.attend().clone()
    b.cache.tensors[4].copy_(ints(torch, [-5, 50, 1 << 30]))
    got = b.attend()
    assert torch.equal(got[4:8], good[4:8])
    b.cache.tensors[4].copy_(ints(torch, [50, 50, 50]))
    for starts in ([0, 4, 2, 12], [-3, 4, 8, 12], [0, 4, 8, 1000], [8, 4, 0, 0]):
        b.starts = ints(torch, starts)
        b.attend()


@pytest.mark.parametrize("nodes", [1, 60])
@pytest.mark.parametrize("length", [49, 5000, 1 << 30, 2 ** 31 - 1])
def test_a_length_past_what_is_held_ends_there(torch, native, nodes, length):
    b = Batch(torch, native, [48, 20], [nodes, nodes], 8, 4, 128, 16, seed=12)
    want, room = b.expected(lambda s, i: set() if s == 0 else chain(s, i))
    b.held[0] = 3
    b.cache.tensors[4].copy_(ints(torch, [length, 20]))
    got = b.attend(max_length=9000).double().cpu()
    assert bool(((got - want).abs() <= room).all())


@pytest.mark.parametrize("nodes,lengths", [(1, [5000, 70]), (30, [5000, 70]), (60, [9, 4100])])
def test_wide_heads_in_graphs(torch, native, nodes, lengths):
    """Two captured calls with a workspace each, replayed one after the other and side by side with eager ones."""
    batches = [Batch(torch, native, lengths, [nodes, max(1, nodes - 3)], 8, 4, 128, 32, kind, seed=13 + i)
               for i, kind in enumerate(("bfloat16", "float16"))]
    need = [native.attention_paged_workspace(b.cache, b.rows, b.heads, b.max_rows, b.max_length) for b in batches]
    spaces = [torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for n in need]
    outs = [torch.zeros(b.rows, b.heads, b.width, dtype=b.query.dtype, device="cuda") for b in batches]
    queries = [b.query.clone() for b in batches]

    def call(i):
        b = batches[i]
        native.attention_paged(b.cache, 0, queries[i], b.starts, b.max_rows, b.max_length, None, b.scale, outs[i],
                               workspace=spaces[i])

    eager = [b.attend().clone() for b in batches]
    graphs = []
    for i in range(2):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            call(i)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            call(i)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(4):
        for i in range(2):
            queries[i].copy_(batches[i].query)
            outs[i].zero_()
            spaces[i].fill_(255)
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        again = batches[step % 2].attend()
        torch.cuda.synchronize()
        assert torch.equal(again, eager[step % 2])
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1]), step


def test_more_rows_than_announced_are_left_alone(torch, native):
    b = Batch(torch, native, [50, 20], [10, 3], 4, 2, 64, 16, seed=4)
    full = b.attend().clone()
    b.max_rows = 4
    got = b.attend()
    assert torch.equal(got[:4], full[:4]) and torch.equal(got[10:], full[10:]) and bool((got[4:10] == 7).all())


def test_layouts(torch, native):
    """Keys and values interleaved in one pool, past 2^32 bytes and 2^31 elements of offset, in a layer of many."""
    lengths, counts, rows, kv, width, layers = [45, 100], [3, 8], 16, 2, 64, 3
    b = Batch(torch, native, lengths, counts, 4, kv, width, rows, seed=9)
    page = 2 * rows * kv * width
    apart = 1 << 28  # elements from page to page
    pages = b.keys.shape[1]
    pool = torch.empty((pages - 1) * apart + layers * 2 * page + 64, dtype=torch.bfloat16, device="cuda")
    assert (pages - 1) * apart > 1 << 31

    def view(at):
        return torch.as_strided(pool, (layers, pages, rows, kv, width), (2 * page, apart, 2 * kv * width, width, 1), at)

    keys, values = view(0), view(kv * width)
    keys[2], values[2] = b.keys[0], b.values[0]
    got = b.attend()
    b.cache = native.PagedCache(keys, values, b.table, b.held, b.cache.tensors[4], b.cache.tensors[5])
    assert torch.equal(b.attend(layer=2), got)
    b.check(got, chain)
    # A query whose rows do not lie one after the other, as int16.
    wide = torch.zeros(b.rows, 3, 4, width, dtype=torch.bfloat16, device="cuda")
    wide[:, 1] = b.query
    assert torch.equal(b.attend(layer=2, query=wide[:, 1]), got)


def test_calls_on_other_streams_and_in_graphs(torch, native):
    """Captured calls replay on changed data; calls on two streams with workspaces of their own do not mix."""
    b = Batch(torch, native, [3000, 50], [4, 9], 4, 2, 64, 64, seed=6)
    other = Batch(torch, native, [2500, 90], [4, 9], 4, 2, 64, 64, seed=7)
    want, want_other = b.attend().clone(), other.attend().clone()
    out, out_other = torch.zeros_like(want), torch.zeros_like(want)

    def call(x, to):
        native.attention_paged(x.cache, 0, x.query, x.starts, x.max_rows, x.max_length, None, x.scale, to)

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for stream, x, to in zip(streams, (b, other), (out, out_other)):
            with torch.cuda.stream(stream):
                to.zero_()
                call(x, to)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(out_other, want_other)
    with torch.cuda.stream(streams[0]):
        call(b, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(b, out)
    for step in range(4):
        b.query.mul_(0.5 + step)
        out.zero_()
        graph.replay()
        got = out.clone()
        assert torch.equal(got, b.attend()), step


def test_workspace_is_checked(torch, native):
    b = Batch(torch, native, [9000], [4], 4, 2, 64, 64)
    need = native.attention_paged_workspace(b.cache, b.rows, b.heads, b.max_rows, b.max_length)
    assert need > 0
    with pytest.raises(native.HipError, match="workspace"):
        b.attend(workspace=torch.empty(need - 16, dtype=torch.uint8, device="cuda"))
    dirty = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(b.attend(workspace=dirty).clone(), b.attend())


def test_masks_at_word_boundaries(torch, native):
    """Nodes of trees over 16 words, as many as a mask may have, and lines that skip whole words."""
    nodes = 1024
    parents = [-1] + [i - 1 if i % 65 else max(0, i - 200) for i in range(1, nodes)]
    bad = [5, -7, 3, 2, 9]  # not in front of their nodes: roots
    starts = ints(torch, [0, nodes, nodes, nodes + 5])
    mask = torch.full((nodes + 5, 16), -1, dtype=torch.int64, device="cuda")
    native.tree_mask(ints(torch, parents + bad), starts, nodes, mask)
    rows = [line(parents, i) for i in range(nodes)] + [line(bad, i) for i in range(5)]
    assert torch.equal(mask, pack_masks(torch, rows, 16))
    # Rows past the announced ones, and the last sequence's end, stay.
    mask.fill_(-1)
    native.tree_mask(ints(torch, parents + bad), ints(torch, [0, 300]), 100, mask[:, :])
    assert bool((mask[100:] == -1).all()) and torch.equal(mask[:100], pack_masks(torch, rows[:100], 16))


def test_masks_of_a_thousand_nodes(torch, native):
    rng = np.random.default_rng(1)
    trees = [list(range(-1, 1023)), [-1] + [0] * 1023, random_tree(rng, 1000)]
    mask = torch.full((3050, 16), -1, dtype=torch.int64, device="cuda")
    native.tree_mask(ints(torch, sum(trees, []) + [0] * 2), ints(torch, [0, 1024, 2048, 3048]), 1024, mask)
    rows = [line(t, i) for t in trees for i in range(len(t))]
    assert torch.equal(mask[:3048], pack_masks(torch, rows, 16)) and bool((mask[3048:] == -1).all())


# ---------------------------------------------------------------- pages

class Model:
    """The cache's bookkeeping and contents in plain Python."""

    def __init__(self, sequences, pages, width, rows):
        self.table = [[-1] * width for _ in range(sequences)]
        self.held, self.lengths, self.references = [0] * sequences, [0] * sequences, [0] * pages
        self.rows, self.width = rows, width

    def take(self, count):
        free = [p for p, r in enumerate(self.references) if r == 0][:count]
        return free if len(free) == count else None

    def reserve(self, sequences, rows):
        if len(set(sequences)) < len(sequences) or any(not 0 <= s < len(self.held) for s in sequences) or min(rows) < 0:
            return 1
        need = [max(0, -(-(self.lengths[s] + n) // self.rows) - self.held[s]) for s, n in zip(sequences, rows)]
        if any(self.held[s] + n > self.width for s, n in zip(sequences, need)):
            return 1
        got = self.take(sum(need))
        if got is None:
            return 2
        for s, n in zip(sequences, need):
            for _ in range(n):
                page = got.pop(0)
                self.table[s][self.held[s]] = page
                self.references[page] = 1
                self.held[s] += 1
        return 0

    def fork(self, sources, targets):
        """(status, pages copied: [(from, to, rows)])"""
        everything = range(len(self.held))
        if (len(set(targets)) < len(targets) or any(t not in everything or self.held[t] for t in targets) or
                any(s not in everything or s in targets for s in sources)):
            return 1, []
        got = self.take(sum(self.lengths[s] % self.rows > 0 for s in sources))
        if got is None:
            return 2, []
        copies = []
        for s, t in zip(sources, targets):
            full, rest = divmod(self.lengths[s], self.rows)
            for j in range(full):
                self.table[t][j] = self.table[s][j]
                self.references[self.table[s][j]] += 1
            if rest:
                page = got.pop(0)
                self.references[page] = 1
                self.table[t][full] = page
                copies.append((self.table[s][full], page, rest))
            self.held[t], self.lengths[t] = full + (rest > 0), self.lengths[s]
        return 0, copies

    def free(self, sequences):
        status = 0
        for s in sequences:
            if not 0 <= s < len(self.held):
                status = 1
                continue
            for j in range(self.held[s]):
                self.references[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.held[s] = self.lengths[s] = 0
        return status


class Pool:
    def __init__(self, torch, native, sequences=7, pages=40, width=9, rows=16, layers=2, heads=2, kind="bfloat16"):
        self.torch, self.model = torch, Model(sequences, pages, width, rows)
        shape = (layers, pages, rows, heads, 64)
        g = torch.Generator(device="cuda").manual_seed(1)
        self.keys = torch.randn(shape, generator=g, device="cuda").to(getattr(torch, kind))
        self.values = torch.randn(shape, generator=g, device="cuda").to(getattr(torch, kind))
        self.table = ints(torch, self.model.table)
        self.held, self.lengths, self.references = (ints(torch, [0] * n) for n in (sequences, sequences, pages))
        self.cache = native.PagedCache(self.keys, self.values, self.table, self.held, self.lengths, self.references)
        self.status = ints(torch, [0])
        self.want_keys, self.want_values = self.keys.clone(), self.values.clone()

    def same(self, status=0):
        m = self.model
        assert int(self.status) == status
        self.status.zero_()
        assert self.held.tolist() == m.held and self.lengths.tolist() == m.lengths
        assert self.references.tolist() == m.references
        table = self.table.tolist()
        for s, h in enumerate(m.held):
            assert table[s][:h] == m.table[s][:h], s
        assert self.torch.equal(self.keys, self.want_keys) and self.torch.equal(self.values, self.want_values)

    def reserve(self, sequences, rows):
        self.cache.reserve(ints(self.torch, rows), ints(self.torch, sequences), status=self.status)
        self.same(self.model.reserve(sequences, rows))

    def fork(self, sources, targets):
        self.cache.fork(ints(self.torch, sources), ints(self.torch, targets), status=self.status)
        status, copies = self.model.fork(sources, targets)
        for old, new, rows in copies:
            self.want_keys[:, new, :rows] = self.want_keys[:, old, :rows]
            self.want_values[:, new, :rows] = self.want_values[:, old, :rows]
        self.same(status)

    def free(self, sequences):
        self.cache.free(ints(self.torch, sequences), status=self.status)
        self.same(self.model.free(sequences))

    def grow(self, s, rows):
        """Rows of a sequence become its own, as keep() would make them."""
        self.model.lengths[s] += rows
        self.lengths[s] += rows


def test_pages_are_taken_lowest_first_and_given_back(torch, native):
    p = Pool(torch, native)
    p.reserve([3, 0], [40, 16])
    assert p.table.tolist()[3][:3] == [0, 1, 2] and p.table.tolist()[0][0] == 3
    p.reserve([3, 0], [40, 16])  # there already
    p.grow(3, 40)
    p.reserve([3], [8])
    p.reserve([3], [9])
    p.free([3])
    p.reserve([1, 2], [100, 1])  # the holes first, in order
    assert p.table.tolist()[1][:7] == [0, 1, 2, 4, 5, 6, 7] and p.table.tolist()[2][0] == 8
    p.free([0, 1, 2])
    assert not p.references.any() and bool((p.table == -1).all())


def test_calls_that_cannot_be_met_change_nothing(torch, native):
    p = Pool(torch, native, pages=12)
    p.reserve([0, 1], [100, 20])
    p.grow(0, 100)
    p.grow(1, 20)
    p.reserve([2, 3], [40, 1])       # exhausted: 3 of 4 are left
    p.reserve([2, 2], [1, 1])        # twice
    p.reserve([2, 7], [1, 1])        # out of range
    p.reserve([-1], [1])
    p.reserve([2, 3], [1, -1])
    p.reserve([2], [16 * 9 + 1])     # longer than the table
    p.reserve([2], [2 ** 31 - 1])
    p.fork([0, 1], [4, 4])
    p.fork([0, 1], [4, 1])           # holds pages
    p.fork([0, 4], [4, 5])           # source and target
    p.fork([9], [4])
    p.fork([0], [9])
    p.fork([0, 1, 0, 1], [2, 3, 4, 5])  # exhausted
    p.fork([0, 1, 0], [2, 3, 4])
    p.fork([6, 6], [5, 1])           # refused, though empty
    p.free([9, 2, -4])
    p.free([])


def test_a_refused_fork_leaves_numbers_that_make_no_sense(torch, native):
    """What a target holds may look like anything; nothing is shared, copied or counted for it."""
    p = Pool(torch, native)
    p.reserve([0], [40])
    p.grow(0, 40)
    for held, length in (((1 << 30) | 3, 1 << 29), ((1 << 30) | 2, 40), (2 ** 31 - 1, 2 ** 31 - 1), ((1 << 30) | 9, -5)):
        p.held[4], p.lengths[4] = held, length
        p.model.held[4], p.model.lengths[4] = 0, length
        p.cache.fork(ints(torch, [0]), ints(torch, [4]), status=p.status)
        assert p.held.tolist()[4] == held
        p.held[4] = 0
        p.same(native.PAGES_INVALID)


def test_forks_share_full_pages_and_copy_the_last(torch, native):
    p = Pool(torch, native, kind="float16")
    for s, n in ((0, 50), (1, 32), (2, 5)):
        p.reserve([s], [n + 20])
        p.grow(s, n)
    p.fork([0, 0, 1, 2], [6, 3, 4, 5])
    assert p.references.tolist()[:3] == [3, 3, 3]
    p.free([0])
    p.free([6, 6, 3])  # twice is once
    p.fork([3], [0])   # an empty one
    p.fork([4], [3])
    p.free([1, 4, 3, 2, 5])
    assert not p.references.any()


def test_freed_sequences_have_no_length(torch, native):
    """Whatever they held: a length without pages, a negative number of them, a sequence listed twice."""
    p = Pool(torch, native)
    p.reserve([0, 1], [40, 20])
    p.grow(0, 40)
    p.held[2], p.lengths[2] = 0, 50
    p.held[3], p.lengths[3] = -3, -8
    p.cache.free(ints(torch, [2, 0, 3, 0]), status=p.status)
    p.model.free([0])
    p.same()


@pytest.mark.parametrize("number", [-1, 1 << 30, "pool"])
@pytest.mark.parametrize("index", [1, 3])  # a full page, the last one of two rows
def test_a_fork_passes_on_entries_out_of_range(torch, native, number, index):
    """As -1, without a page in their place: what the source does not see the fork does not either."""
    p = Pool(torch, native)
    p.reserve([0], [50])
    p.grow(0, 50)
    bad = p.keys.shape[1] if number == "pool" else number
    p.table[0, index] = p.model.table[0][index] = bad
    p.cache.fork(ints(torch, [0]), ints(torch, [4]), status=p.status)
    m = p.model
    m.table[4] = [-1 if i == index else page for i, page in enumerate(m.table[0])]
    m.held[4], m.lengths[4] = 4, 50
    for page in m.table[4][:3]:
        if page >= 0:
            m.references[page] += 1
    if index != 3:
        m.table[4][3] = 4
        m.references[4] = 1
        p.want_keys[:, 4, :2], p.want_values[:, 4, :2] = p.want_keys[:, 3, :2], p.want_values[:, 3, :2]
    p.same(native.PAGES_INVALID)
    query = torch.randn(2, 2, 64, device="cuda").to(p.keys.dtype)
    query[1] = query[0]
    out = torch.full_like(query, 7.0)
    cached = torch.zeros(2, 1, dtype=torch.int64, device="cuda")  # of the new rows none is seen
    native.attention_paged(p.cache, 1, query, ints(torch, [0, 1, 1, 1, 1, 2, 2, 2]), 1, 51, cached, 0.125, out)
    assert torch.equal(out[0], out[1]) and bool((out[0] != 7).any())
    p.cache.free(ints(torch, [4]), status=p.status)
    for page in m.table[4][:4]:
        if page >= 0:
            m.references[page] -= 1
    m.table[4], m.held[4], m.lengths[4] = [-1] * 9, 0, 0
    p.same(native.PAGES_INVALID)


@pytest.mark.parametrize("seed", range(4))
def test_pages_through_many_calls(torch, native, seed):
    """A random history against the plain bookkeeping, refusals among it."""
    rng = random.Random(seed)
    p = Pool(torch, native, sequences=9, pages=rng.choice([20, 60]), rows=rng.choice([16, 32]))
    for _ in range(60):
        what = rng.random()
        some = rng.sample(range(9), rng.randint(1, 5))
        if what < 0.4:
            p.reserve(some, [rng.randint(0, 60) for _ in some])
            for s in some:
                room = p.model.held[s] * p.model.rows - p.model.lengths[s]
                if room > 0:
                    p.grow(s, rng.randint(0, room))
        elif what < 0.7:
            p.fork([rng.choice([s for s in range(10) if s not in some] + some[:1]) for _ in some], some)
        else:
            p.free(some)


def test_large_pools_and_lists(torch, native):
    """More pages than one step of the scan, and thousands of sequences in a call."""
    sequences, pages = 8192, 40000
    keys = torch.zeros(1, pages, 16, 1, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.full((sequences, 8), -1, dtype=torch.int32, device="cuda")
    held, lengths = (torch.zeros(sequences, dtype=torch.int32, device="cuda") for _ in range(2))
    references = torch.zeros(pages, dtype=torch.int32, device="cuda")
    references[::3] = 1
    cache = native.PagedCache(keys, keys.clone(), table, held, lengths, references)
    status = ints(torch, [0])
    rows = torch.arange(sequences, device="cuda", dtype=torch.int32) % 64
    free = (references == 0).nonzero()[:, 0].tolist()
    cache.reserve(rows, status=status)
    need = ((rows + 15) // 16).tolist()
    assert int(status) == 0 and held.tolist() == need
    got, at = table.tolist(), 0
    for s in range(sequences):
        assert got[s] == free[at:at + need[s]] + [-1] * (8 - need[s]), s
        at += need[s]
    before = references.clone(), table.clone(), held.clone()
    cache.reserve(rows + 64, status=status)  # more than there is
    assert int(status) == native.PAGES_EXHAUSTED
    assert all(torch.equal(a, b) for a, b in zip(before, (references, table, held)))
    cache.free()
    assert int(references.sum()) == -(-pages // 3) and not held.any()


@pytest.mark.parametrize("kind,layers", [("bfloat16", 1), ("float16", 3)])
def test_written_rows_lie_behind_the_length(torch, native, kind, layers):
    p = Pool(torch, native, layers=3, kind=kind)
    for s, n in ((0, 50), (1, 32), (2, 0), (5, 15)):
        p.reserve([s], [n + 20])
        p.grow(s, n)
    counts = [7, 20, 3, 0, 2, 1, 0]  # sequence 4 holds no page
    starts = [0] + np.cumsum(counts).tolist()
    g = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn(layers, starts[-1], 6, 64, generator=g, device="cuda").to(p.keys.dtype)
    keys, values = qkv[:, :, 2:4], qkv[:, :, 4:]
    if layers == 1:
        keys, values = keys[0], values[0]
    first = 2 if layers == 1 else 0
    p.cache.write(keys, values, ints(torch, starts), 20, layer=first, status=p.status)
    for s, n in enumerate(counts):
        for i in range(n):
            t = p.model.lengths[s] + i
            page = p.model.table[s][t // 16]
            if s != 4:
                p.want_keys[first:first + layers, page, t % 16] = qkv[:, starts[s] + i, 2:4]
                p.want_values[first:first + layers, page, t % 16] = qkv[:, starts[s] + i, 4:]
    p.same(native.PAGES_INVALID)
    # No more than announced: the rows past it keep what was there.
    p.cache.write(keys * 0, values * 0, ints(torch, starts), 1, layer=first, status=p.status)
    assert int(p.status) == native.PAGES_INVALID
    page, row = p.model.table[1][2], 1
    assert torch.equal(p.keys[:, page, row], p.want_keys[:, page, row]) and not p.keys[first, page, 0].any()


@pytest.mark.parametrize("announced", [700, 5, 1 << 20])
def test_written_rows_of_ragged_batches(torch, native, announced):
    """Most sequences with a row or none and one with hundreds, by a search over starts 64 at a time; rows in front
    of the first sequence and behind the last one are nobody's."""
    rng = np.random.default_rng(3)
    n, rows = 4200, 16
    counts = [int(c) for c in rng.integers(0, 3, n)]
    counts[64], counts[63], counts[4097], counts[-1] = 700, 0, 9, 4
    starts = 3 + np.concatenate([[0], np.cumsum(counts)])
    lengths = [int(x) for x in rng.integers(0, 20, n)]
    held = [-(-(a + b) // rows) for a, b in zip(lengths, counts)]
    pages = sum(held)
    table, at = -np.ones((n, max(held)), np.int32), 0
    order = rng.permutation(pages)
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
    keys = torch.zeros(2, pages, rows, 1, 64, dtype=torch.bfloat16, device="cuda")
    cache = native.PagedCache(keys, torch.zeros_like(keys), ints(torch, table), ints(torch, held), ints(torch, lengths),
                              ints(torch, [1] * pages))
    fresh = torch.randn(2, 2, int(starts[-1]) + 5, 1, 64, device="cuda").bfloat16()
    status = ints(torch, [0])
    cache.write(fresh[0], fresh[1], ints(torch, starts), announced, status=status)
    assert int(status) == 0
    want = torch.zeros_like(keys), torch.zeros_like(keys)
    to = [(table[s, (lengths[s] + i) // rows], (lengths[s] + i) % rows, starts[s] + i)
          for s in range(n) for i in range(min(counts[s], announced))]
    page, place, row = (torch.tensor(np.array(x), device="cuda") for x in zip(*to))
    for side in range(2):
        want[side][:, page, place] = fresh[side][:, row]
        assert torch.equal(cache.tensors[side], want[side])


def test_shared_pages_are_not_written(torch, native):
    p = Pool(torch, native)
    p.reserve([0], [48])
    p.grow(0, 48)
    p.fork([0], [1])
    p.lengths[0] = 40  # wound back into a page that sequence 1 reads
    rows = torch.ones(4, 2, 64, dtype=p.keys.dtype, device="cuda")
    p.cache.write(rows, rows.clone(), ints(torch, [0, 4, 4, 4, 4, 4, 4, 4]), 4, status=p.status)
    p.lengths[0] = 48
    p.same(native.PAGES_INVALID)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("heads,rows", [(2, 16), (1, 64)])
def test_accepted_rows_are_kept(torch, native, in_place, heads, rows):
    p = Pool(torch, native, sequences=6, pages=60, width=12, rows=rows, heads=heads, layers=3)
    lengths, counts = [5, 0, 47, 16, 30, 9], [30, 1, 64, 20, 0, 33]
    paths = [[0, 2, 3, 17, 29], [0], sorted(random.Random(1).sample(range(64), 40)), [], [], list(range(33))]
    for s, (n, c) in enumerate(zip(lengths, counts)):
        p.reserve([s], [n + c])
        p.grow(s, n)
    path = -np.ones((6, 64), np.int32)
    for s, nodes in enumerate(paths):
        path[s, :len(nodes)] = nodes
    accepted = [len(x) for x in paths]
    starts = ints(torch, [0] + np.cumsum(counts).tolist())
    old_keys, old_values = p.want_keys.clone(), p.want_values.clone()
    for s, nodes in enumerate(paths):
        for k, node in enumerate(nodes):
            a, b = lengths[s] + node, lengths[s] + k
            pa, pb = p.model.table[s][a // rows], p.model.table[s][b // rows]
            p.want_keys[:, pb, b % rows], p.want_values[:, pb, b % rows] = (old_keys[:, pa, a % rows],
                                                                           old_values[:, pa, a % rows])
    out = torch.zeros(6, dtype=torch.int32, device="cuda")
    p.cache.keep(starts, ints(torch, path), ints(torch, accepted), None if in_place else out, status=p.status)
    after = [a + b for a, b in zip(lengths, accepted)]
    if in_place:
        p.model.lengths = after
    else:
        assert out.tolist() == after
    p.same()


@pytest.mark.parametrize("heads", [3, 20, 40])
def test_rows_of_any_width_are_written_forked_and_kept(torch, native, heads):
    """24, 160 and 320 vectors a row: threads without one, several a thread, more than one workgroup has in keep().
    One tree of 1,024 nodes of which more are kept than are looked up at a time, one in place but for its end."""
    p = Pool(torch, native, sequences=4, pages=170, width=80, heads=heads, layers=2)
    lengths, counts = [7, 33, 0, 0], [1024, 600, 0, 0]
    paths = [sorted(random.Random(5).sample(range(1024), 700)), list(range(515)) + [530, 599], [], []]
    for s in range(2):
        p.reserve([s], [lengths[s] + counts[s]])
        p.grow(s, lengths[s])
    starts = [0] + np.cumsum(counts).tolist()
    fresh = torch.randn(2, 2, starts[-1], heads, 64, device="cuda").bfloat16()
    p.cache.write(fresh[0], fresh[1], ints(torch, starts), 1024, status=p.status)
    path = -np.ones((4, 1024), np.int32)
    for s, nodes in enumerate(paths):
        path[s, :len(nodes)] = nodes
        for i in range(counts[s]):
            t = lengths[s] + i
            p.want_keys[:, p.model.table[s][t // 16], t % 16] = fresh[0, :, starts[s] + i]
            p.want_values[:, p.model.table[s][t // 16], t % 16] = fresh[1, :, starts[s] + i]
    p.same()
    p.cache.keep(ints(torch, starts), ints(torch, path), ints(torch, [len(x) for x in paths]), status=p.status)
    for s, nodes in enumerate(paths):
        for k, node in enumerate(nodes):
            t = lengths[s] + k
            p.want_keys[:, p.model.table[s][t // 16], t % 16] = fresh[0, :, starts[s] + node]
            p.want_values[:, p.model.table[s][t // 16], t % 16] = fresh[1, :, starts[s] + node]
        p.model.lengths[s] += len(nodes)
    p.same()
    p.fork([0, 1], [3, 2])


def test_pages_past_32_bits_of_offset(torch, native):
    """Rows written, kept and forked in the last pages of a pool of 2^32 elements and more a layer."""
    layers, pages, rows = 2, 2100, 1024
    keys, values = (torch.empty(layers, pages, rows, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    references = torch.ones(pages, dtype=torch.int32, device="cuda")
    references[-3:] = 0
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    held, lengths, status = ints(torch, [0, 0]), ints(torch, [0, 0]), ints(torch, [0])
    cache = native.PagedCache(keys, values, table, held, lengths, references)
    cache.reserve(ints(torch, [1100]), ints(torch, [1]), status=status)
    assert table[1].tolist() == [pages - 3, pages - 2, -1, -1]
    fresh = torch.randn(2, layers, 1100, 8, 128, device="cuda").bfloat16()
    starts = ints(torch, [0, 0, 1100])
    cache.write(fresh[0], fresh[1], starts, 1100, status=status)
    path = ints(torch, [[0] * 1030, [*range(1020), *range(1090, 1100)]])
    cache.keep(starts, path, ints(torch, [0, 1030]), status=status)
    cache.fork(ints(torch, [1]), ints(torch, [0]), status=status)
    assert int(status) == 0 and lengths.tolist() == [1030] * 2 and table[0].tolist() == [pages - 3, pages - 1, -1, -1]
    kept = fresh[:, :, path[1].long()]
    for side, pool in enumerate((keys, values)):
        for page in (pages - 2, pages - 1):
            assert torch.equal(torch.cat([pool[:, pages - 3], pool[:, page, :6]], 1), kept[side])


def test_hundreds_of_forks(torch, native):
    p = Pool(torch, native, sequences=700, pages=640, width=5, heads=3, layers=1)
    for s, n in ((0, 50), (1, 32), (2, 5)):
        p.reserve([s], [n])
        p.grow(s, n)
    targets = list(range(699, 99, -1))
    p.fork([t % 3 for t in targets], targets)
    assert int(p.references.max()) == 201
    p.free(targets[::2] + targets[1:400:2])
    p.fork([699 - 2 * 250] * 300, targets[:600:2])  # of those still held
    p.free(list(range(700)))
    assert not p.references.any()


def test_paths_that_are_none_move_nothing(torch, native):
    p = Pool(torch, native, sequences=6)
    lengths = [20] * 6
    for s in range(6):
        p.reserve([s], [40])
        p.grow(s, 20)
    path = ints(torch, [[0, 2, 2, 3], [0, 3, 1, -1], [0, 1, 9, -1], [-1, 2, 3, 4], [0, 1, 2, 3], [0, 2, -1, -1]])
    accepted = ints(torch, [4, 3, 3, 2, 5, 2])
    out = torch.zeros(6, dtype=torch.int32, device="cuda")
    p.cache.keep(ints(torch, [0, 8, 16, 24, 32, 40, 48]), path, accepted, out, status=p.status)
    page = [p.model.table[5][t // 16] for t in (21, 22)]
    p.want_keys[:, page[0], 5], p.want_values[:, page[0], 5] = (p.want_keys[:, page[1], 6].clone(),
                                                               p.want_values[:, page[1], 6].clone())
    assert out.tolist() == lengths[:5] + [22]
    p.same(native.PAGES_INVALID)
    p.cache.keep(ints(torch, [0, 8, 16, 24, 32, 40, 48]), path, ints(torch, [4, 3, 3, 2, -1, 0]), status=p.status)
    p.same(native.PAGES_INVALID)


@pytest.mark.parametrize("in_place", [False, True])
def test_a_negative_length_is_kept_as_it_is(torch, native, in_place):
    p = Pool(torch, native, sequences=2)
    p.reserve([0, 1], [40, 40])
    p.grow(1, 20)
    p.lengths[0] = p.model.lengths[0] = -7
    out = p.lengths if in_place else torch.zeros(2, dtype=torch.int32, device="cuda")
    p.cache.keep(ints(torch, [0, 4, 8]), ints(torch, [[0, 1], [0, 1]]), ints(torch, [2, 2]), None if in_place else out,
                 status=p.status)
    assert out.tolist() == [-7, 22]
    p.model.lengths[1] = 22 if in_place else 20
    p.same(native.PAGES_INVALID)


# ---------------------------------------------------------------- verification

def verify_plain(p, q, tokens, parents, uniforms, draw):
    """(path, next) of one sequence, in 64 bits, from the definition: residuals renormalised one by one
    are the closed form's, which decides here."""
    def clean(row):
        row = row.astype(np.float64)
        return np.where((row > 0) & (row < np.inf), row, 0.0)

    if not len(tokens):
        return [], -1
    node, path = 0, [0]
    while True:
        row, drafts = clean(p[node]), clean(q[node]) if q is not None else None
        left, weight, shift, taken = row.copy(), 1.0, 0.0, None
        value = lambda a, x: a[x] if 0 <= x < len(a) else 0.0  # noqa: E731
        for c in range(node + 1, len(tokens)):
            if parents[c] != node:
                continue
            x, u = tokens[c], float(uniforms[c])
            if u * (value(drafts, x) if q is not None else 1.0) * weight < value(left, x):
                taken = c
                break
            if q is not None:
                shift += weight
                left = np.maximum(row - shift * drafts, 0.0)
                weight = left.sum()
            else:
                weight -= value(left, x)
                if 0 <= x < len(left):
                    left[x] = 0.0
        if taken is None:
            break
        node = taken
        path.append(node)
    if not left.sum() > 0:
        left = row
    sums = np.cumsum(left)
    if not sums[-1] > 0:
        return path, -1
    return path, int(np.searchsorted(sums, float(draw) * sums[-1], side="right"))


def run_verify(torch, native, p, q, trees, tokens, uniforms, draws, kind="float32", pad=0, max_nodes=None):
    """p, q [rows][alphabet] (float arrays) through the library: [(path, next)]."""
    rows, alphabet = p.shape
    counts = [len(t) for t in trees]
    starts = ints(torch, [0] + np.cumsum(counts).tolist())
    dtype = getattr(torch, kind)

    def table(values):
        wide = torch.full((rows, alphabet + pad), 0.25, dtype=dtype, device="cuda")
        wide[:, :alphabet] = torch.from_numpy(values).cuda().to(dtype)
        return wide[:, :alphabet]

    target, draft = table(p), None if q is None else table(q)
    nodes = max_nodes or max(counts + [1])
    n = len(trees)
    path, accepted, following = (torch.full(s, 99, dtype=torch.int32, device="cuda") for s in ((n, nodes), (n,), (n,)))
    native.verify_drafts(target, draft, ints(torch, tokens), ints(torch, sum(trees, [])), starts, nodes,
                         torch.from_numpy(uniforms).cuda(), torch.from_numpy(draws).cuda(), path, accepted, following)
    got = []
    for line_, count, token in zip(path.tolist(), accepted.tolist(), following.tolist()):
        assert line_[count:] == [-1] * (nodes - count)
        got.append((line_[:count], token))
    back = target.double().cpu().numpy()
    return got, back, None if draft is None else draft.double().cpu().numpy()


def softmax(x):
    e = np.exp(x - x.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


def drafted(rng, counts, alphabet, children, drafts, spread=2.0):
    """Distributions, trees and tokens drawn as a drafter draws them."""
    trees = []
    for n in counts:
        parents = [-1] * min(n, 1)
        for i in range(1, n):
            open_ = [v for v in range(max(0, i - 8), i) if sum(x == v for x in parents) < children]
            parents.append(int(rng.choice(open_)))
        trees.append(parents)
    rows = sum(counts)
    logits = rng.standard_normal((rows, alphabet)) * spread
    p = softmax(logits).astype(np.float32)
    q = softmax(logits + 0.8 * rng.standard_normal((rows, alphabet))).astype(np.float32) if drafts else None
    tokens, first = [], 0
    for t in trees:
        for i, v in enumerate(t):
            source = (q if drafts else p)[first + max(v, 0)].astype(np.float64)
            tokens.append(int(rng.choice(alphabet, p=source / source.sum())))
        first += len(t)
    return p, q, trees, tokens


@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("alphabet,pad", [(2, 0), (7, 2), (513, 7), (1024, 0), (4099, 5)])
@pytest.mark.parametrize("children", [1, 3])
def test_verification_follows_the_definition(torch, native, kind, drafts, alphabet, pad, children):
    """Chains and trees, alphabets that end inside a lane's values, rows at any alignment, empty sequences."""
    rng = np.random.default_rng(alphabet + children)
    counts = [1, 12, 0, 30, 2, 70, 5]
    p, q, trees, tokens = drafted(rng, counts, alphabet, children, drafts)
    uniforms, draws = rng.random(sum(counts), np.float32), rng.random(len(counts), np.float32)
    got, p, q = run_verify(torch, native, p, q, trees, tokens, uniforms, draws, kind, pad)
    first = 0
    for s, n in enumerate(counts):
        part = slice(first, first + n)
        want = verify_plain(p[part], q[part] if drafts else None, tokens[part], trees[s], uniforms[part], draws[s])
        assert got[s] == want, (s, got[s], want)
        first += n


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("alphabet", [50257, 131071])
def test_verification_of_wide_alphabets(torch, native, drafts, alphabet):
    rng = np.random.default_rng(alphabet)
    counts = [4, 9, 1]
    p, q, trees, tokens = drafted(rng, counts, alphabet, 3, drafts, spread=4.0)
    for trial in range(4):
        uniforms = rng.random(14, np.float32) if trial else np.full(14, 0.999, np.float32)
        draws = rng.random(3, np.float32) if trial < 3 else np.array([0, 1 - 2.0 ** -24, 0.5], np.float32)
        got, back, drafts_back = run_verify(torch, native, p, q, trees, tokens, uniforms, draws, "bfloat16", trial)
        first = 0
        for s, n in enumerate(counts):
            part = slice(first, first + n)
            assert got[s] == verify_plain(back[part], drafts_back[part] if drafts else None, tokens[part], trees[s],
                                          uniforms[part], draws[s])
            first += n


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("sequences", [40, 70, 140])
def test_verification_of_many_sequences_over_wide_alphabets(torch, native, drafts, sequences):
    """As many as fill the units in several chunks of the alphabet each, or by themselves."""
    rng = np.random.default_rng(sequences)
    counts, alphabet = [5 if s % 9 else 0 for s in range(sequences)], 33001
    p, q, trees, tokens = drafted(rng, counts, alphabet, 3, drafts, spread=4.0)
    uniforms, draws = rng.random(sum(counts), np.float32), rng.random(sequences, np.float32)
    got, back, drafts_back = run_verify(torch, native, p, q, trees, tokens, uniforms, draws, "bfloat16", 7)
    first = 0
    for s, n in enumerate(counts):
        part = slice(first, first + n)
        assert got[s] == verify_plain(back[part], drafts_back[part] if drafts else None, tokens[part], trees[s],
                                      uniforms[part], draws[s]), s
        first += n


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("alphabet", [1, 40000, 65537])
def test_verification_of_sparse_rows(torch, native, drafts, alphabet):
    """Alphabets of one token, and wide ones whose mass lies in few places, all sums exact: at the ends, around the
    boundaries of what is summed together, nowhere."""
    def row(*places):
        values = np.zeros(alphabet, np.float32)
        for at, value in places:
            values[at % alphabet] = value
        return values

    last = alphabet - 1
    rows = [row((0, 1.0)), row((last, 1.0)), row((0, 0.5), (last, 0.5)), row(), row((0, math.nan), (last, math.inf)),
            row((8191, 0.25), (8192, 0.25), (32767, 0.25), (last, 0.25)), row((511, 0.5), (512, 0.25), (513, 0.25))]
    trees, tokens, p, q, uniforms, draws = [], [], [], [], [], []
    for i, target in enumerate(rows):
        for j, draft in enumerate(rows):
            for token, u, d in ((0, 0.0, 0.0), (last, 0.5, 0.5), (8192 % alphabet, 0.75, 1 - 2.0 ** -24)):
                trees.append([-1, 0, 0])
                tokens += [0, token, last]
                p += [target, draft, target]
                q += [draft, draft, draft]
                uniforms += [0.0, u, 0.25]
                draws.append(d)
    for at in range(0, len(trees), 21):
        nodes = slice(3 * at, 3 * (at + 21))
        args = [np.stack(p[nodes]), np.stack(q[nodes]) if drafts else None]
        u, d = np.array(uniforms[nodes], np.float32), np.array(draws[at:at + 21], np.float32)
        got, back, drafts_back = run_verify(torch, native, *args, trees[at:at + 21], tokens[nodes], u, d)
        for s in range(21):
            part = slice(3 * s, 3 * s + 3)
            want = verify_plain(back[part], drafts_back[part] if drafts else None, tokens[nodes][part], [-1, 0, 0],
                                u[part], d[s])
            assert got[s] == want, (at + s, got[s], want)


def test_the_workspace_of_verification_is_checked(torch, native):
    rows, alphabet = 3, 70000
    p = torch.full((rows, alphabet), 1.0 / alphabet, device="cuda")
    outputs = [torch.full(shape, 99, dtype=torch.int32, device="cuda") for shape in ((1, 3), (1,), (1,))]
    need = native.library().tsac_hip_verify_drafts_workspace(1, alphabet)
    assert need > 0 and native.library().tsac_hip_verify_drafts_workspace(1, 1000) == 0

    def call(space):
        native.verify_drafts(p, None, ints(torch, [0, 5, 6]), ints(torch, [-1, 0, 0]), ints(torch, [0, 3]), 3,
                             torch.full((3,), 0.5, device="cuda"), torch.tensor([0.25], device="cuda"), *outputs,
                             workspace=space)
        torch.cuda.synchronize()
        return [x.tolist() for x in outputs]

    with pytest.raises(native.HipError, match="workspace"):
        call(torch.empty(need - 16, dtype=torch.uint8, device="cuda"))
    assert outputs[0].tolist() == [[99] * 3]
    dirty = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    assert call(dirty) == call(None) == call(dirty)


def test_verification_at_the_edges(torch, native):
    """Ties and zeros, equal distributions, siblings of one token, tokens and parents out of range, rows that
    are no distributions."""
    half = np.array([0.5, 0.25, 0.25, 0.0], np.float32)
    other = np.array([0.25, 0.5, 0.0, 0.25], np.float32)
    nan = np.array([np.nan, -1.0, np.inf, 0.25], np.float32)
    zero = np.zeros(4, np.float32)
    cases = [  # rows of p, rows of q, parents, tokens, uniforms, draw
        ([half, half], [half, half], [-1, 0], [0, 0], [0, 0.999], 0.0),          # p = q: accepted
        ([half, half], [half, half], [-1, 0], [0, 3], [0, 0.0], 0.5),            # neither draws it: refused, row of p
        ([half, other], [other, half], [-1, 0], [0, 1], [0, 0.5], 0.999),        # u q = p: refused (not below)
        ([half, other], [other, half], [-1, 0], [0, 1], [0, 0.49], 0.75),
        ([half, half, other], None, [-1, 0, 0], [0, 0, 0], [0, 0.5, 0.0], 0.5),  # a sibling of the refused token
        ([half, half, other], None, [-1, 0, 0], [0, 0, 1], [0, 0.5, 0.499], 0.0),
        ([half, half, other], None, [-1, 0, 0], [0, 0, 1], [0, 0.5, 0.5], 0.0),
        ([half, half, half], None, [-1, 0, 0], [0, 4, -1], [0, 0.0, 0.0], 0.75),  # tokens of no alphabet
        ([half, half, half], [other] * 3, [-1, 0, 1], [0, 4, 1 << 30], [0, 0.0, 0.0], 0.75),
        ([half, other, half], None, [5, 1, 7], [0, 0, 0], [0, 0, 0], 0.25),      # parents that are none
        ([half, other, half], None, [-1, -1, 1], [0, 0, 0], [0, 0, 0], 0.25),
        ([nan, other], [nan, other], [-1, 0], [0, 3], [0, 0.9], 0.5),
        ([nan, other], None, [-1, 0], [0, 2], [0, 0.0], 0.5),
        ([zero, other], None, [-1, 0], [0, 2], [0, 0.0], 0.5),                   # nothing to draw from
        ([zero, zero], [zero, half], [-1, 0], [0, 2], [0, 0.0], 0.5),
    ]
    for p, q, parents, tokens, uniforms, draw in cases:
        uniforms, draws = np.array(uniforms, np.float32), np.array([draw], np.float32)
        p, q = np.stack(p), np.stack(q) if q is not None else None
        got, _, _ = run_verify(torch, native, p, q, [parents], tokens, uniforms, draws)
        reached = [v if 0 <= v < i else -1 for i, v in enumerate(parents)]
        assert got[0] == verify_plain(p, q, tokens, reached, uniforms, draw), (parents, tokens)


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("alphabet", [1500, 33001])
@pytest.mark.parametrize("last", [True, False])
def test_verification_of_a_thousand_siblings(torch, native, drafts, alphabet, last):
    """A root of 1,023 children, repeated tokens among them, all refused or all but the last. Every sum is exact:
    half of p lies on 1,024 tokens that q has twice as often, half on one that q lacks."""
    places = np.arange(1024) * ((alphabet - 1) // 1024) % (alphabet - 1)
    p, q = np.zeros((1024, alphabet), np.float32), np.zeros((1024, alphabet), np.float32)
    p[:, places], p[:, -1], q[:, places] = 2.0 ** -11, 0.5, 2.0 ** -10
    rng = np.random.default_rng(alphabet)
    tokens = [0] + [int(places[i]) for i in rng.integers(0, 700, 1022)] + [alphabet - 1 if last else int(places[3])]
    trees, uniforms = [[-1] + [0] * 1023], np.full(1024, 0.999, np.float32)
    if last and not drafts:
        uniforms[-1] = 0.25  # of what is left, 0.5 and what was not drafted
    for draw in (0.0, 0.3, 0.77, 1 - 2.0 ** -24):
        draws = np.array([draw], np.float32)
        got, back, back_q = run_verify(torch, native, p, q if drafts else None, trees, tokens, uniforms, draws, "bfloat16")
        want = verify_plain(p, q if drafts else None, tokens, trees[0], uniforms, draws[0])
        assert want[0] == ([0, 1023] if last else [0]) and got[0] == want


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("alphabet", [41, 33001])
def test_verification_of_deep_trees(torch, native, drafts, alphabet):
    """A chain and a tree of 1,024 nodes each, followed to the end and as far as random numbers go."""
    rng = np.random.default_rng(alphabet)
    rows, counts = 2048, [1024, 1024]
    p = np.zeros((rows, alphabet), np.float32)
    q = np.zeros((rows, alphabet), np.float32)
    tokens = rng.integers(0, alphabet, rows)
    places = rng.integers(0, alphabet, (rows, 8))
    tree = [-1] + [int(rng.integers(max(0, i - 200), i)) for i in range(1, 1024)]
    trees = [list(range(-1, 1023)), tree]
    for r in range(rows):
        np.add.at(p[r], places[r], rng.integers(1, 9, 8).astype(np.float32) / 64)
        np.add.at(q[r], places[r], rng.integers(1, 9, 8).astype(np.float32) / 64)
    for first, parents in ((0, trees[0]), (1024, trees[1])):
        for i in range(1, 1024):
            p[first + parents[i], tokens[first + i]] += 0.25
            q[first + parents[i], tokens[first + i]] += 0.25
    for scale in (0.0, 0.3, 1.0):
        uniforms = (rng.random(rows, np.float32) * scale).astype(np.float32)
        draws = rng.random(2, np.float32)
        got, back, _ = run_verify(torch, native, p, q if drafts else None, trees, tokens.tolist(), uniforms, draws)
        for s in range(2):
            part = slice(1024 * s, 1024 * s + 1024)
            want = verify_plain(p[part], q[part] if drafts else None, tokens[part], trees[s], uniforms[part], draws[s])
            assert got[s] == want, (scale, s)
        assert scale or len(got[0][0]) == 1024


@pytest.mark.parametrize("drafts", [True, False])
def test_verification_past_32_bits_of_offset(torch, native, drafts):
    """The last rows of 4,100 over 2^20 tokens: their values lie past 2^32 elements."""
    rng = np.random.default_rng(9)
    rows, alphabet, nodes = 4100, 1 << 20, 4
    p, q, trees, tokens = drafted(rng, [nodes], alphabet, 3, drafts, spread=6.0)
    target = torch.empty(rows, alphabet, dtype=torch.bfloat16, device="cuda")
    draft = torch.empty_like(target) if drafts else None
    target[-nodes:] = torch.from_numpy(p).cuda()
    if drafts:
        draft[-nodes:] = torch.from_numpy(q).cuda()
    uniforms, draws = rng.random(rows, np.float32), rng.random(1, np.float32)
    ids, parents = np.zeros(rows, np.int32), np.zeros(rows, np.int32)
    ids[-nodes:], parents[-nodes:] = tokens, trees[0]
    path, accepted, following = ints(torch, [[9] * nodes]), ints(torch, [9]), ints(torch, [9])
    native.verify_drafts(target, draft, ints(torch, ids), ints(torch, parents), ints(torch, [rows - nodes, rows]), nodes,
                         torch.from_numpy(uniforms).cuda(), torch.from_numpy(draws).cuda(), path, accepted, following)
    back, back_q = (None if x is None else x[-nodes:].double().cpu().numpy() for x in (target, draft))
    want, token = verify_plain(back, back_q, tokens, trees[0], uniforms[-nodes:], draws[0])
    assert path[0, :int(accepted)].tolist() == want and int(following) == token


def test_nodes_past_the_announced_ones_are_not_looked_at(torch, native):
    rng = np.random.default_rng(3)
    p, q, trees, tokens = drafted(rng, [20, 3], 40, 1, True)
    uniforms, draws = np.zeros(23, np.float32), rng.random(2, np.float32)  # all are accepted
    got, back, drafts_back = run_verify(torch, native, p, q, trees, tokens, uniforms, draws, max_nodes=8)
    assert [len(g[0]) for g in got] == [8, 3]
    assert got[0] == verify_plain(back[:8], drafts_back[:8], tokens[:8], trees[0][:8], uniforms[:8], draws[0])


@pytest.mark.parametrize("drafts", [True, False])
def test_what_follows_is_distributed_as_the_target(torch, native, drafts):
    """The first token behind the root, accepted or drawn, over 40,000 sequences with three drafted children
    each: within five standard deviations of the target's probabilities."""
    rng = np.random.default_rng(11)
    n, alphabet = 40000, 6
    p = np.array([0.05, 0.4, 0.1, 0.25, 0.15, 0.05], np.float32)
    q = np.array([0.3, 0.1, 0.1, 0.05, 0.15, 0.3], np.float32)
    tokens = rng.choice(alphabet, (n, 4), p=q.astype(np.float64) / q.sum(dtype=np.float64))
    if not drafts:
        tokens[:, 1:] = [3, 0, 3]
    rows = np.broadcast_to(p, (4 * n, alphabet)).copy()
    got, _, _ = run_verify(torch, native, rows, np.broadcast_to(q, rows.shape).copy() if drafts else None,
                           [[-1, 0, 0, 0]] * n, tokens.reshape(-1).tolist(), rng.random(4 * n, np.float32),
                           rng.random(n, np.float32))
    first = [tokens[s][path[1]] if len(path) > 1 else token for s, (path, token) in enumerate(got)]
    share = np.bincount(first, minlength=alphabet) / n
    assert np.all(np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / n)), share
    assert 0.2 < np.mean([len(path) > 1 for path, _ in got]) < 0.99


def test_verification_in_a_graph_and_on_a_stream(torch, native):
    rng = np.random.default_rng(5)
    counts = [9, 30]
    p, q, trees, tokens = drafted(rng, counts, 1000, 3, True)
    target, draft = torch.from_numpy(p).cuda(), torch.from_numpy(q).cuda()
    arguments = [ints(torch, tokens), ints(torch, sum(trees, [])), ints(torch, [0, 9, 39]), 30]
    uniforms, draws = torch.rand(39, device="cuda"), torch.rand(2, device="cuda")
    outputs = [torch.zeros(2, 30, dtype=torch.int32, device="cuda")] + [ints(torch, [0, 0]) for _ in range(2)]

    def call():
        native.verify_drafts(target, draft, *arguments, uniforms, draws, *outputs)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(5):
        uniforms.uniform_()
        draws.uniform_()
        graph.replay()
        got = [x.clone() for x in outputs]
        u, d, first = uniforms.cpu().numpy(), draws.cpu().numpy(), 0
        for s, n in enumerate(counts):
            part = slice(first, first + n)
            path, token = verify_plain(p[part], q[part], tokens[part], trees[s], u[part], d[s])
            assert got[0][s].tolist()[:len(path)] == path and int(got[1][s]) == len(path) and int(got[2][s]) == token
            first += n


def test_a_path_wider_than_the_trees_is_kept_from(torch, native):
    """One buffer of 64 nodes a sequence for trees of fewer, written by verification and read by keep; another
    width than what is announced is refused, as a call would write it at one pitch and the other read it at
    another."""
    rng = np.random.default_rng(12)
    p = Pool(torch, native, sequences=3, pages=30, layers=2)
    counts, lengths = [12, 20, 9], [5, 0, 30]
    for s in range(3):
        p.reserve([s], [lengths[s] + counts[s]])
        p.grow(s, lengths[s])
    q, _, trees, tokens = drafted(rng, counts, 50, 3, False)
    target = torch.from_numpy(q).cuda()
    starts, uniforms = ints(torch, [0] + np.cumsum(counts).tolist()), torch.zeros(sum(counts), device="cuda")
    buffer = torch.full((3, 64), 77, dtype=torch.int32, device="cuda")
    accepted, following = ints(torch, [0] * 3), ints(torch, [0] * 3)

    def verify(max_nodes):
        native.verify_drafts(target, None, ints(torch, tokens), ints(torch, sum(trees, [])), starts, max_nodes,
                             uniforms, torch.rand(3, device="cuda"), buffer, accepted, following)

    with pytest.raises(native.HipError, match="path"):
        verify(20)
    assert bool((buffer == 77).all())
    verify(64)
    p.cache.keep(starts, buffer, accepted, status=p.status)
    old_keys, old_values = p.want_keys.clone(), p.want_values.clone()
    first = 0
    for s, n in enumerate(counts):
        path, _ = verify_plain(q[first:first + n], None, tokens[first:first + n], trees[s], np.zeros(n), 0.5)
        assert len(path) > 1 and buffer[s].tolist() == path + [-1] * (64 - len(path))
        for k, node in enumerate(path):
            a, b = lengths[s] + node, lengths[s] + k
            to, frm = (p.model.table[s][b // 16], b % 16), (p.model.table[s][a // 16], a % 16)
            p.want_keys[:, to[0], to[1]] = old_keys[:, frm[0], frm[1]]
            p.want_values[:, to[0], to[1]] = old_values[:, frm[0], frm[1]]
        p.model.lengths[s] += len(path)
        first += n
    p.same()


# ---------------------------------------------------------------- together

def test_a_drafted_decode(torch, native):
    """Steps as a program takes them (room, rows, masks, attention of two layers, verification, what is kept),
    eager and captured, with a fork in the middle: the cache ends with the rows of the accepted tokens in
    order, and a step over it equals attention over them."""
    torch.manual_seed(0)
    heads, kv, width, layers, rows, alphabet, sequences = 4, 2, 64, 2, 16, 97, 4
    g = torch.Generator(device="cuda").manual_seed(2)
    pool = torch.full((2, layers, 64, rows, kv, width), math.nan, device="cuda").bfloat16()
    table = torch.full((sequences, 16), -1, dtype=torch.int32, device="cuda")
    held, lengths = (torch.zeros(sequences, dtype=torch.int32, device="cuda") for _ in range(2))
    cache = native.PagedCache(pool[0], pool[1], table, held, lengths, ints(torch, [0] * 64))
    status = ints(torch, [0])
    embed = torch.randn(2, layers, alphabet, kv, width, generator=g, device="cuda").bfloat16()
    to_query = torch.randn(alphabet, heads, width, generator=g, device="cuda").bfloat16()
    to_logits = torch.randn(heads * width, alphabet, generator=g, device="cuda") * 0.2
    rng = np.random.default_rng(1)
    history = [[] for _ in range(sequences)]
    last = [3, 5, -1, 7]  # sequence 2 joins as a fork
    counts = [6, 9, 0, 1]

    def step(last, counts, seed):
        trees = [random_tree(np.random.default_rng(seed + s), n) for s, n in enumerate(counts)]
        tokens = [int(last[s]) if i == 0 else int(rng.integers(alphabet)) for s, t in enumerate(trees)
                  for i in range(len(t))]
        starts = ints(torch, [0] + np.cumsum(counts).tolist())
        ids, parents, most = ints(torch, tokens), ints(torch, sum(trees, [])), max(counts)
        n = len(tokens)
        mask = torch.zeros(n, 1, dtype=torch.int64, device="cuda")
        outs = [torch.zeros(n, heads, width, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]
        uniforms, draws = (torch.from_numpy(rng.random(k, np.float32)).cuda() for k in (n, sequences))
        path = torch.zeros(sequences, most, dtype=torch.int32, device="cuda")
        accepted, following = (torch.zeros(sequences, dtype=torch.int32, device="cuda") for _ in range(2))
        room = ints(torch, counts)
        space = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
        probabilities = torch.zeros(n, alphabet, device="cuda")

        def model():
            cache.reserve(room, status=status)
            native.tree_mask(parents, starts, most, mask)
            for layer in range(layers):
                cache.write(embed[0, layer, ids.long()], embed[1, layer, ids.long()], starts, most, layer, status=status)
                native.attention_paged(cache, layer, to_query[ids.long()], starts, most, 256, mask, 0.125, outs[layer],
                                       workspace=space)
            hidden = outs[0].float() + outs[1].float()
            probabilities.copy_(torch.softmax((hidden.view(n, -1)[:, :, None] * to_logits).sum(1), 1))
            native.verify_drafts(probabilities, None, ids, parents, starts, most, uniforms, draws, path, accepted,
                                 following)

        if seed % 2:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                model()
                cache.keep(starts, path, accepted, status=status)
            graph.replay()
        else:
            model()
            cache.keep(starts, path, accepted, status=status)
        torch.cuda.synchronize()
        p, at = probabilities.cpu().numpy(), starts.tolist()
        after = list(last)
        for s, tree in enumerate(trees):
            part = slice(at[s], at[s + 1])
            want, token = verify_plain(p[part], None, tokens[part], tree, uniforms.cpu().numpy()[part], float(draws[s]))
            assert path[s].tolist()[:len(want)] == want and int(accepted[s]) == len(want)
            if tree:
                assert int(following[s]) == token
                history[s] += [tokens[at[s] + i] for i in want]
                after[s] = token
        assert int(status) == 0 and lengths.tolist() == [len(h) for h in history]
        return after

    for seed in range(4):
        last = step(last, counts, seed)
    cache.fork(ints(torch, [1]), ints(torch, [2]), status=status)
    history[2], last[2] = list(history[1]), last[1]
    counts = [4, 9, 9, 1]
    for seed in range(4, 10):
        last = step(last, counts, seed)
        counts = counts[1:] + counts[:1]
    held_list, table_list = held.tolist(), table.tolist()
    for s, tokens in enumerate(history):
        assert len(tokens) >= 10
        for layer in range(layers):
            for side in range(2):
                got = torch.stack([pool[side, layer, table_list[s][t // rows], t % rows] for t in range(len(tokens))])
                assert torch.equal(got, embed[side, layer, torch.tensor(tokens, device="cuda")]), (s, layer)
    cache.free(status=status)
    assert int(status) == 0 and not cache.tensors[5].any() and held_list != held.tolist()
