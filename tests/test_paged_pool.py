"""Host side of the paged cache: the pool's bookkeeping against a plain model of
it, and the refusals of the device entry points (which come before any HIP
call, so they run without a GPU)."""
import numpy as np
import pytest


def test_pages_are_handed_out_lowest_first_and_come_back(yuear_lib):
    pool = yuear_lib.PagePool(6, 32)
    a, b = pool.open(), pool.open()
    assert pool.extend(a, 33) == ([], []) and pool.extend(b, 32) == ([], [])
    assert pool.table([a, b], 3).tolist() == [[0, 1, -1], [2, -1, -1]]
    assert (pool.length(a), pool.length(b), pool.unused) == (33, 32, 3)
    assert pool.extend(b, 1) == ([], [])  # a full last page needs no copy
    pool.close_sequence(a)
    assert pool.unused == 4
    c = pool.open()
    pool.extend(c, 65)
    assert pool.table([c], 3).tolist() == [[0, 1, 4]]
    with pytest.raises(ValueError, match="no such sequence"):
        pool.length(a)


@pytest.mark.parametrize("length,copies", [(1, True), (31, True), (32, False), (40, True), (64, False)])
def test_a_fork_shares_pages_until_it_writes(yuear_lib, length, copies):
    pool = yuear_lib.PagePool(16, 32)
    a = pool.open()
    pool.extend(a, length)
    held = (length + 31) // 32
    b, c = pool.fork(a), pool.fork(a)
    assert pool.unused == 16 - held
    assert pool.extend(b, 0) == ([], [])
    src, dst = pool.extend(b, 1)
    assert (src, dst) == (([held - 1], [held]) if copies else ([], []))
    rows = pool.table([a, b, c], 4)
    assert (rows[0] == rows[2]).all() and (rows[0][:length // 32] == rows[1][:length // 32]).all()
    assert rows[1][length // 32] == held
    # the last holder writes in place; the others' copies are their own
    assert pool.extend(c, 1)[1] == ([held + 1] if copies else [])
    assert pool.extend(a, 1) == ([], [])
    for s in (a, b, c):
        pool.close_sequence(s)
    assert pool.unused == 16


def test_out_of_pages_changes_nothing(yuear_lib):
    pool = yuear_lib.PagePool(3, 64)
    a = pool.open()
    pool.extend(a, 65)
    b = pool.fork(a)
    with pytest.raises(MemoryError, match="out of pages"):
        pool.extend(b, 64)  # its own last page and one more
    assert pool.length(b) == 65 and pool.unused == 1
    assert pool.table([b], 2).tolist() == [[0, 1]]
    assert pool.extend(b, 63) == ([1], [2])
    with pytest.raises(MemoryError):
        pool.extend(a, 64)
    assert pool.extend(a, 63) == ([], [])


def test_truncate_and_trim(yuear_lib):
    pool = yuear_lib.PagePool(20, 32)
    a = pool.open()
    pool.extend(a, 300)
    pool.truncate(a, 257)
    assert pool.table([a], 10).tolist() == [[0, 1, 2, 3, 4, 5, 6, 7, 8, -1]]
    # the token at 257 sees (157, 257] and [0, 33): pages 2 and 3 end at 127, page 4 at 159
    pool.trim(a, 100, 33)
    assert pool.table([a], 9).tolist() == [[0, 1, -1, -1, 4, 5, 6, 7, 8]]
    pool.trim(a, 98, 33)  # 160 is the first it sees
    assert pool.table([a], 9).tolist() == [[0, 1, -1, -1, -1, 5, 6, 7, 8]]
    assert pool.unused == 20 - 6
    with pytest.raises(ValueError, match="given back"):
        pool.truncate(a, 256)
    b = pool.fork(a)
    pool.close_sequence(a)
    assert pool.unused == 20 - 6
    pool.extend(b, 100)  # pages given back are taken again
    assert pool.table([b], 12).tolist() == [[0, 1, -1, -1, -1, 5, 6, 7, 8, 2, 3, 4]]
    pool.truncate(b, 257)
    pool.truncate(b, 257)
    assert pool.length(b) == 257


def test_compaction_moves_the_highest_pages_into_the_holes(yuear_lib):
    rng = np.random.default_rng(4)
    pool = yuear_lib.PagePool(64, 32)
    seqs = [pool.open() for _ in range(12)]
    for s in seqs:
        pool.extend(s, int(rng.integers(1, 150)))
    forks = [pool.fork(s) for s in seqs[::3]]
    for s in seqs[1::2]:
        pool.close_sequence(s)
    live = [s for i, s in enumerate(seqs) if i % 2 == 0] + forks
    before, unused = pool.table(live, 8), pool.unused
    src, dst = pool.compact()
    move = dict(zip(src, dst))
    held = 64 - unused
    assert pool.unused == unused and src and not set(src) & set(dst) and len(set(dst)) == len(dst)
    assert all(p >= held for p in src) and all(p < held for p in dst)
    after = pool.table(live, 8)
    assert (after == np.vectorize(lambda p: move.get(p, p))(before)).all()
    assert sorted(set(after.ravel()) - {-1}) == list(range(held))
    assert pool.compact() == ([], [])
    s = pool.open()
    pool.extend(s, 1)
    assert pool.table([s], 1)[0, 0] == held


def test_pool_refusals(yuear_lib):
    for pages, slots in ((0, 32), (-1, 64), (4, 16), (4, 48), (4, 0)):
        with pytest.raises(ValueError):
            yuear_lib.PagePool(pages, slots)
    pool = yuear_lib.PagePool(4, 32)
    a = pool.open()
    pool.extend(a, 64)
    for bad in (lambda: pool.extend(a, -1), lambda: pool.extend(7, 1), lambda: pool.fork(7),
                lambda: pool.truncate(a, 65), lambda: pool.truncate(a, -1), lambda: pool.trim(a, 0, 0),
                lambda: pool.trim(a, 3, -1), lambda: pool.table([a], 1), lambda: pool.close_sequence(9),
                lambda: pool.extend(a, 2 ** 31 - 1)):
        with pytest.raises(ValueError):
            bad()
    assert pool.length(a) == 64 and pool.unused == 2
    lib = yuear_lib.lib
    assert lib.yuear_pages_length(None, 0) == -1 and lib.yuear_pages_unused(None) == -1
    assert lib.yuear_pages_open(None, None, None) == 2


P = 1 << 20  # stands for a device pointer: no refused call reads it
APPEND = dict(qkv=P, qkv_stride=640, q_norm=P, k_norm=P, eps=1e-5, cos=P, sin=P, positions=64, k=P, v=P, pages=4,
              slots=32, table=P, width=2, table_stride=2, starts=P, pos0=P, batch=1, rows=3, heads=3, kv_heads=1,
              q_out=P, q_stride=384, stream=None)
PREFILL = dict(q=P, q_stride=384, k=P, v=P, pages=4, slots=32, table=P, width=2, table_stride=2, starts=P, pos0=P,
               batch=1, rows=3, heads=3, kv_heads=1, window=0, sinks=0, workspace=P, bytes=1 << 40, out=P,
               out_stride=384, stream=None)
DECODE = dict(qkv=P, qkv_stride=640, q_norm=P, k_norm=P, eps=1e-5, cos=P, sin=P, positions=64, k=P, v=P, pages=4,
              slots=32, table=P, width=2, table_stride=2, pos=P, batch=1, heads=3, kv_heads=1, window=0, sinks=0,
              workspace=P, bytes=1 << 40, out=P, out_stride=384, stream=None)
BAD = dict(qkv=(None, P + 8), q=(None, P + 2), k=(None, P + 8), v=(None, P + 4), cos=(None, P + 8), sin=(None, P + 8),
           q_norm=(P + 2,), k_norm=(P + 8,), positions=(0, -1), pages=(0, -4), slots=(0, 16, 33, 96, -32), table=(None,),
           width=(0, -1), table_stride=(1,), starts=(None,), pos0=(None,), pos=(None,), batch=(-1,), rows=(-1,),
           heads=(0, 5, 7, -3), kv_heads=(0, 2, -1), window=(-1,), sinks=(-1,), workspace=(None, P + 4),
           bytes=(0, 1024), out=(None, P + 8), q_out=(None, P + 8), qkv_stride=(632, 644), q_stride=(376, 388),
           out_stride=(376, 388))


@pytest.mark.parametrize("name,args", [("yuear_op_paged_append", APPEND), ("yuear_op_paged_attention_prefill", PREFILL),
                                       ("yuear_op_paged_attention_decode", DECODE)])
def test_device_entry_points_refuse_invalid_arguments(yuear_lib, name, args):
    fn = getattr(yuear_lib.lib, name)
    for key in args:
        for value in BAD.get(key, ()):
            assert fn(*{**args, key: value}.values()) == 1, (key, value)
    for empty in ("batch", "rows"):
        if empty in args:
            assert fn(*{**args, empty: 0}.values()) == 0


def test_passes_of_a_decode_call_are_counted_in_31_bits(yuear_lib):
    fn = yuear_lib.lib.yuear_op_paged_attention_decode
    assert fn(*{**DECODE, "batch": 1 << 20, "positions": 2 ** 31 - 1, "width": 1 << 20, "table_stride": 1 << 20,
                "slots": 1024}.values()) == 1


def test_page_copies_refuse_pages_written_twice_or_also_read(yuear_lib):
    i32 = lambda v: np.ascontiguousarray(v, np.int32).ctypes.data_as(yuear_lib.i32p)

    def call(src, dst, k=P, v=P, layers=2, stride=1 << 20, pages=8, kv_heads=2, slots=32):
        return yuear_lib.lib.yuear_op_pages_copy(k, v, layers, stride, pages, kv_heads, slots, i32(src), i32(dst),
                                                 len(dst), None)
    for src, dst in (([0, 1], [2, 2]), ([0, 2], [2, 3]), ([1], [1]), ([8], [1]), ([-1], [1]), ([1], [8]), ([1], [-1])):
        assert call(src, dst) == 1, (src, dst)
    good = dict(src=[0], dst=[1])
    for bad in (dict(k=None), dict(v=P + 8), dict(layers=0), dict(stride=8 * 2 * 32 * 128 - 8), dict(stride=(1 << 20) + 4),
                dict(pages=0), dict(kv_heads=0), dict(slots=40)):
        assert call(**{**good, **bad}) == 1, bad
    assert call([], []) == 0


def test_workspace_size(yuear_lib):
    size = yuear_lib.lib.yuear_op_paged_workspace_bytes
    assert size(1, 24, 8, 0) > 0 and size(8, 64, 8, 0) >= size(1, 24, 8, 0)
    assert size(1, 24, 8, 5000) >= size(1, 24, 8, 0)
    for bad in ((-1, 24, 8, 0), (1, 24, 0, 0), (1, 20, 8, 0), (1, 24, 8, -1), (1, 0, 1, 0)):
        assert size(*bad) == 0


def test_pool_refuses_numbers_past_32_bits_and_calls_after_close(yuear_lib):
    pool = yuear_lib.PagePool(8, 32)
    a = pool.open()
    for call in (lambda: pool.extend(a, 2 ** 32 + 1), lambda: pool.fork(a + 2 ** 32), lambda: pool.trim(a, 2 ** 32, 0)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        yuear_lib.PagePool(2 ** 32 + 8, 32)
    assert pool.length(a) == 0 and pool.unused == 8
    pool.close()
    with pytest.raises(ValueError):
        pool.open()


@pytest.mark.parametrize("past", [2 ** 32, -2 ** 32, 2 ** 31, 2 ** 40])
def test_pool_reads_name_no_other_sequence(yuear_lib, past):
    """Sequence numbers whose low 32 bits are a sequence's are not that sequence."""
    pool = yuear_lib.PagePool(8, 32)
    a, b = pool.open(), pool.open()
    pool.extend(b, 40)
    with pytest.raises(ValueError):
        pool.length(b + past)
    for ids in ([b + past], np.array([b + past], np.int64), np.array([[a], [b + past]], np.int64),
                np.array([b + past], np.float64), np.array([b + 0.5])):
        with pytest.raises(ValueError):
            pool.table(ids, 4)
    if past > 0:
        with pytest.raises(ValueError):
            pool.table(np.array([b + past], np.uint64), 4)
    with pytest.raises(ValueError):
        pool.table([b], 2 ** 32 + 2)
    for ids in ([b], np.array([b], np.int64), np.array([[b]], np.uint8), (np.int32(b),)):
        assert pool.table(ids, 3).tolist() == [[0, 1, -1]]
    assert pool.length(np.int64(b)) == 40
    assert pool.table([], 4).shape == (0, 4) and pool.table(np.empty(0), 4).shape == (0, 4)


@pytest.mark.parametrize("sizes", [(2 ** 32 + 1, 24, 8, 0), (1, 2 ** 32 + 24, 8, 0), (1, 24, 2 ** 32 + 8, 0),
                                   (1, 24, 8, 2 ** 32 + 100), (2 ** 31, 24, 8, 0), (1 - 2 ** 32, 24, 8, 0)])
def test_workspace_sizes_past_32_bits_are_refused(yuear_lib, sizes):
    """Not answered with the workspace of their low 32 bits."""
    with pytest.raises(ValueError, match="paged_workspace"):
        yuear_lib.paged_workspace(*sizes)


@pytest.mark.parametrize("pages", [2 ** 25 + 1, 2 ** 31 - 1])
def test_a_pool_of_more_pages_than_a_gpu_holds_is_refused(yuear_lib, pages):
    """Its bookkeeping would take the host's memory."""
    with pytest.raises(ValueError, match="2\\^25 pages"):
        yuear_lib.PagePool(pages, 32)
