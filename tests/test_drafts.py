"""Refusals of the drafted-decoding calls, without a GPU: every check of sizes, pointers and
strides comes before any device work, as a status and a message."""
import ctypes

import pytest

from tsac_hip import native

POINTER = 1 << 40  # never read: the calls below are refused on the host


def desc(**changes):
    fields = dict(keys=POINTER, values=POINTER, layer_stride=4096, page_stride=2048, row_stride=128, layers=2, pages=8,
                  page_rows=16, heads=2, head_width=64, type=native.TYPE_BF16, table=POINTER, table_stride=4, held=POINTER,
                  lengths=POINTER, references=POINTER, sequences=3)
    fields.update(changes)
    return ctypes.byref(native.PagedCacheDesc(**fields))


def refused(status, text):
    assert status != 0
    assert text in native.library().tsac_hip_last_error().decode()


@pytest.mark.parametrize("changes,text", [
    (dict(type=2), "type"), (dict(head_width=96), "head width"), (dict(page_rows=8), "page rows"),
    (dict(page_rows=48), "page rows"), (dict(page_rows=2048), "page rows"), (dict(heads=0), "size"),
    (dict(layers=0), "size"), (dict(layers=256), "size"), (dict(pages=0), "size"), (dict(sequences=65536), "size"),
    (dict(table_stride=0), "table"), (dict(table_stride=(1 << 20) + 1), "table"), (dict(row_stride=120), "strides"),
    (dict(row_stride=132), "strides"), (dict(page_stride=2049), "strides"), (dict(layer_stride=4), "strides"),
    (dict(keys=None), "missing"), (dict(references=None), "missing"), (dict(values=POINTER + 8), "aligned"),
])
def test_cache_descriptions(changes, text):
    lib = native.library()
    refused(lib.tsac_hip_pages_reserve(desc(**changes), None, POINTER, 1, None, None), text)
    refused(lib.tsac_hip_pages_free(desc(**changes), POINTER, 1, None, None), text)
    refused(lib.tsac_hip_pages_keep(desc(**changes), POINTER, POINTER, 4, POINTER, POINTER, None, None), text)
    refused(lib.tsac_hip_attention_paged(desc(**changes), 0, POINTER, 128, 4, 2, POINTER, 4, 64, None, 0, 1.0, POINTER,
                                         128, POINTER, 1 << 30, None), text)
    assert lib.tsac_hip_attention_paged_workspace(desc(**changes), 4, 2, 4, 64) == 0


def test_page_calls():
    lib = native.library()
    refused(lib.tsac_hip_pages_reserve(None, None, POINTER, 1, None, None), "missing")
    refused(lib.tsac_hip_pages_reserve(desc(), None, None, 1, None, None), "missing")
    refused(lib.tsac_hip_pages_reserve(desc(), POINTER, POINTER, 8193, None, None), "too many")
    refused(lib.tsac_hip_pages_reserve(desc(), None, POINTER, 4, None, None), "too many")  # of 3 sequences
    refused(lib.tsac_hip_pages_fork(desc(), POINTER, None, 1, None, None), "missing")
    refused(lib.tsac_hip_pages_fork(desc(), POINTER, POINTER, 8193, None, None), "too many")
    refused(lib.tsac_hip_pages_free(desc(), None, 4, None, None), "too many")

    def write(layer=0, layers=1, keys=POINTER, values=POINTER, layer_stride=0, row_stride=128, rows=4, starts=POINTER,
              max_rows=4):
        return lib.tsac_hip_pages_write(desc(), layer, layers, keys, values, layer_stride, row_stride, rows, starts,
                                        max_rows, None, None)

    refused(write(keys=None), "missing")
    refused(write(starts=None), "missing")
    refused(write(layer=2), "layers")
    refused(write(layer=1, layers=2), "layers")
    refused(write(layer=3, layers=0), "layers")
    refused(write(rows=1 << 24), "too many")
    refused(write(row_stride=130), "aligned")
    refused(write(layer_stride=4), "aligned")
    refused(write(keys=POINTER + 2), "aligned")
    refused(lib.tsac_hip_pages_keep(desc(), POINTER, POINTER, 4, POINTER, None, None, None), "missing")


def test_tree_masks():
    lib = native.library()

    def mask(parents=POINTER, rows=8, starts=POINTER, sequences=2, max_rows=4, bits=POINTER, words=1):
        return lib.tsac_hip_tree_mask(parents, rows, starts, sequences, max_rows, bits, words, None)

    refused(mask(parents=None), "missing")
    refused(mask(bits=None), "missing")
    refused(mask(starts=None), "missing")
    refused(mask(words=0), "words")
    refused(mask(words=17), "words")
    refused(mask(max_rows=65), "words")
    refused(mask(sequences=65536), "size")


def test_attention_arguments():
    lib = native.library()

    def attend(layer=0, query=POINTER, stride=128, rows=4, heads=2, starts=POINTER, max_rows=4, max_length=64, mask=None,
               words=0, out=POINTER, out_stride=128, space=POINTER, size=1 << 30, cache=None):
        return lib.tsac_hip_attention_paged(cache or desc(), layer, query, stride, rows, heads, starts, max_rows,
                                            max_length, mask, words, 1.0, out, out_stride, space, size, None)

    refused(attend(layer=2), "layer")
    refused(attend(query=None), "missing")
    refused(attend(out=None), "missing")
    refused(attend(starts=None), "missing")
    refused(attend(heads=3), "multiple")
    refused(attend(heads=0), "multiple")
    refused(attend(rows=1 << 24), "range")
    refused(attend(max_rows=65537), "range")
    refused(attend(max_length=1 << 30), "range")
    refused(attend(mask=POINTER, words=0), "mask words")
    refused(attend(mask=POINTER, words=1025), "mask words")
    refused(attend(query=POINTER + 4), "aligned")
    refused(attend(stride=132), "aligned")
    refused(attend(out_stride=129), "aligned")
    refused(attend(space=POINTER + 8), "aligned")
    refused(attend(stride=64), "overlap")
    refused(attend(out_stride=64), "overlap")


def test_verification_arguments():
    lib = native.library()

    def verify(target=POINTER, stride=1024, draft=POINTER, draft_stride=1024, type_=0, alphabet=1024, rows=4,
               tokens=POINTER, starts=POINTER, sequences=2, nodes=4, path=POINTER, following=POINTER):
        return lib.tsac_hip_verify_drafts(target, stride, draft, draft_stride, type_, alphabet, rows, tokens, POINTER,
                                          starts, sequences, nodes, POINTER, POINTER, path, POINTER, following, None, 0,
                                          None)

    refused(verify(type_=3), "type")
    refused(verify(type_=-1), "type")
    refused(verify(alphabet=0), "alphabets")
    refused(verify(alphabet=(1 << 20) + 1, stride=1 << 21, draft_stride=1 << 21), "alphabets")
    refused(verify(nodes=0), "nodes")
    refused(verify(nodes=1025), "nodes")
    refused(verify(target=None), "missing")
    refused(verify(tokens=None), "missing")
    refused(verify(starts=None), "missing")
    refused(verify(path=None), "missing")
    refused(verify(following=None), "missing")
    refused(verify(rows=1 << 24), "rows")
    refused(verify(stride=1000), "overlap")
    refused(verify(draft_stride=1000), "overlap")
    refused(verify(target=POINTER + 1), "misaligned")
    refused(verify(type_=2, target=POINTER + 2), "misaligned")


def test_bindings_check_their_tensors():
    torch = pytest.importorskip("torch")

    def ints(*shape):
        return torch.zeros(shape, dtype=torch.int32)

    pool = torch.zeros(2, 8, 16, 2, 64, dtype=torch.bfloat16)
    table = ints(3, 4)
    cache = native.PagedCache(pool, pool.clone(), table, ints(3), ints(3), ints(8))
    assert (cache.desc.layer_stride, cache.desc.page_stride, cache.desc.row_stride) == (16384, 2048, 128)
    for bad in [(pool.float(), pool.float(), table, ints(3), ints(3), ints(8)),
                (pool, pool[:, :4], table, ints(3), ints(3), ints(8)),
                (pool, pool.half(), table, ints(3), ints(3), ints(8)),
                (pool, pool.clone(), table.long(), ints(3), ints(3), ints(8)),
                (pool, pool.clone(), table.T, ints(4), ints(4), ints(8)),
                (pool, pool.clone(), table, ints(2), ints(3), ints(8)),
                (pool, pool.clone(), table, ints(3), ints(3), ints(7))]:
        with pytest.raises(native.HipError):
            native.PagedCache(*bad)
    with pytest.raises(native.HipError, match="current device"):
        cache.reserve(ints(3))
    with pytest.raises(native.HipError, match="one target"):
        cache.fork(ints(2), ints(3))
    rows = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(native.HipError, match="starts"):
        cache.write(rows, rows.clone(), ints(3), 5)
    with pytest.raises(native.HipError):
        cache.write(rows.half(), rows.half(), ints(4), 5)
    with pytest.raises(native.HipError, match="elements"):
        cache.keep(ints(4), ints(2, 5), ints(3))
    with pytest.raises(native.HipError, match="must be"):
        native.attention_paged(cache, 0, torch.zeros(5, 4, 32, dtype=torch.bfloat16), ints(4), 5, 64, None, 1.0, rows)
    with pytest.raises(native.HipError, match="query's rows"):
        native.attention_paged(cache, 0, rows, ints(4), 5, 64, None, 1.0, rows[:4])
    with pytest.raises(native.HipError, match="draft"):
        native.verify_drafts(torch.zeros(4, 9), torch.zeros(4, 8), ints(4), ints(4), ints(2), 4, torch.zeros(4),
                             torch.zeros(1), ints(1, 4), ints(1), ints(1))


def test_bindings_check_what_is_read_at_a_pitch():
    """A path of another width than the nodes announced would be written at one pitch and kept at another; words
    of a mask are its second axis."""
    torch = pytest.importorskip("torch")

    def ints(*shape):
        return torch.zeros(shape, dtype=torch.int32)

    def verify(path, max_nodes):
        native.verify_drafts(torch.zeros(4, 9), None, ints(4), ints(4), ints(3), max_nodes, torch.zeros(4),
                             torch.zeros(2), path, ints(2), ints(2))

    for path, max_nodes in ((ints(2, 64), 32), (ints(4, 4), 8), (ints(64), 32), (ints(2, 4, 8), 4)):
        with pytest.raises(native.HipError, match="path"):
            verify(path, max_nodes)
    with pytest.raises(native.HipError, match="path: 4 elements"):
        verify(ints(1, 4), 4)
    pool = torch.zeros(2, 8, 16, 2, 64, dtype=torch.bfloat16)
    cache = native.PagedCache(pool, pool.clone(), ints(3, 4), ints(3), ints(3), ints(8))
    rows = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    for mask in (torch.zeros(5, dtype=torch.int64), torch.zeros(5, 1, 2, dtype=torch.int64)):
        with pytest.raises(native.HipError, match="mask"):
            native.attention_paged(cache, 0, rows, ints(4), 5, 64, mask, 1.0, rows.clone())
        with pytest.raises(native.HipError, match="mask"):
            native.tree_mask(ints(5), ints(4), 5, mask)


def test_attention_of_too_many_rows():
    """More query rows of a cached head than the kernels count."""
    lib = native.library()

    def attend(sequences, heads, max_rows, stride):
        return lib.tsac_hip_attention_paged(desc(sequences=sequences), 0, POINTER, stride, 4, heads, POINTER, max_rows, 64,
                                            None, 0, 1.0, POINTER, stride, POINTER, 1 << 30, None)

    refused(attend(1, 32768, 65536, 32768 * 64), "rows")  # 2^30 of each of two heads
    assert lib.tsac_hip_attention_paged_workspace(desc(sequences=1), 4, 32768, 65536, 64) == 0
