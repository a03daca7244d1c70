"""Paged cache operators on the GPU against their plain 64-bit forms
(paged_ref.py), at the sizes and masks where they can go wrong. Slots that no
token wrote, and pages that no table holds, are NaN throughout."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def torch():
    import torch as t
    t.cuda.init()
    return t


def normal(torch, rng, *shape, mean=0.0, std=1.0):
    a = rng.standard_normal(shape, dtype=np.float32) * std + mean
    return torch.from_numpy(a).to(torch.bfloat16).cuda()


def ints(torch, v):
    return torch.tensor(np.ascontiguousarray(v, np.int32)).cuda()


def rope(torch, yuear_lib, n):
    c, s = yuear_lib.rope_table(n, 128, 5e5)
    return tuple(torch.from_numpy(t.view(np.int16)).cuda().view(torch.bfloat16) for t in (c, s))


def gains(torch, rng, on=True):
    return [normal(torch, rng, 128, mean=1.3, std=0.1) if on else None for _ in range(2)]


def same_bits(torch, a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


# ---- append ----

@pytest.mark.parametrize("heads,kv,slots,lens,pos0,gain", [
    (3, 1, 32, [1], [0], True),
    (24, 8, 64, [97], [40], True),
    (16, 8, 32, [5, 0, 33, 64, 1, 200], [0, 7, 31, 32, 63, 95], True),
    (4, 4, 128, [31, 32, 65], [1, 127, 96], False),
    (8, 1, 256, [300], [255], True),
    (2, 1, 32, [1 + i % 3 for i in range(150)], [i % 70 for i in range(150)], True),
])
def test_append(torch, yuear_lib, heads, kv, slots, lens, pos0, gain):
    rng = np.random.default_rng(len(lens) * 7 + heads)
    table = ref.tables([p + n for p, n in zip(pos0, lens)], slots, 400, rng, 24)
    pages = ref.Pages(400, kv, slots, "cuda")
    rows = sum(lens)
    wide = normal(torch, rng, rows + 2, (heads + 2 * kv) * 128 + 64)
    qkv = wide[:, :(heads + 2 * kv) * 128]
    qn, kn = gains(torch, rng, gain)
    cos, sin = rope(torch, yuear_lib, 2000)
    starts = np.concatenate([[1], 1 + np.cumsum(lens)])  # a row before the first sequence, one behind the last
    q_wide = torch.full((rows + 2, heads + 1, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    want = ref.Pages(400, kv, slots, "cuda")
    want.k.copy_(pages.k), want.v.copy_(pages.v)
    q = yuear_lib.paged_append(qkv, pages.k, pages.v, ints(torch, table), ints(torch, starts), ints(torch, pos0), cos,
                               sin, q_norm=qn, k_norm=kn, eps=EPS, out=q_wide[:, :heads])
    assert q.data_ptr() == q_wide.data_ptr()
    torch.cuda.synchronize()
    k_bound = torch.zeros_like(want.k, dtype=torch.float64)
    k_want = torch.zeros_like(k_bound)
    for b, (p, n) in enumerate(zip(pos0, lens)):
        if not n:
            continue
        x = qkv[starts[b]:starts[b + 1]].reshape(n, -1, 128)
        at = slice(p, p + n)
        y, size = ref.turn(x[:, :heads], qn, cos[at, None], sin[at, None], EPS)
        ref.check(q[starts[b]:starts[b + 1]], y, ref.HALF * y.abs() + ref.FINE * size, f"q of sequence {b}")
        y, size = ref.turn(x[:, heads:heads + kv], kn, cos[at, None], sin[at, None], EPS)
        bound = ref.HALF * y.abs() + ref.FINE * size
        v = x[:, heads + kv:]
        want.put(table[b], p, y.transpose(0, 1).to(torch.bfloat16), v.transpose(0, 1))
        for i in range(n):
            page, slot = table[b][(p + i) // slots], (p + i) % slots
            k_want[page, :, slot], k_bound[page, :, slot] = y[i], bound[i]
    written = ~torch.isnan(want.k)
    assert torch.equal(torch.isnan(pages.k), ~written)  # no other slot is touched
    ref.check(torch.where(written, pages.k, 0.0), k_want, k_bound, "keys")
    assert same_bits(torch, pages.v, want.v)
    # rows of no sequence and columns beside the output keep their contents
    assert (q_wide[0] == 7).all() and (q_wide[-1] == 7).all() and (q_wide[:, heads:] == 7).all()


def test_append_leaves_out_rows_outside_the_table_and_pages_that_are_not_there(torch, yuear_lib):
    rng = np.random.default_rng(1)
    heads, kv, slots = 3, 1, 32
    lens, pos0 = [40, 10, 10, 40, 8], [40, -1, 64, 0, 2 ** 31 - 1]  # the table ends at 64
    table = np.array([[0, 1], [2, 3], [4, 5], [-1, 6], [7, 8]], np.int32)
    pages = ref.Pages(9, kv, slots, "cuda")
    qkv = normal(torch, rng, sum(lens), (heads + 2 * kv) * 128)
    cos, sin = rope(torch, yuear_lib, 100)
    starts = np.concatenate([[0], np.cumsum(lens)])
    out = torch.full((sum(lens), heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    yuear_lib.paged_append(qkv, pages.k, pages.v, ints(torch, table), ints(torch, starts), ints(torch, pos0), cos, sin,
                           out=out)
    torch.cuda.synchronize()
    left = (out == 7).all(-1).all(-1).cpu().numpy()
    assert not left[:24].any() and left[24:60].all() and not left[60:100].any() and left[100:].all()
    wrote = ~torch.isnan(pages.k).all(-1)[:, 0].cpu().numpy()
    assert wrote[0].sum() == 0 and not wrote[1][:8].any() and wrote[1][8:].all()
    assert not wrote[2:6].any() and wrote[6][:8].all() and not wrote[6][8:].any() and not wrote[7:].any()
    assert np.array_equal(~torch.isnan(pages.v[:, 0, 0, 5]).cpu().numpy(), wrote)


# ---- decode ----

def decode_inputs(torch, yuear_lib, rng, heads, kv, slots, pos, pages_n, width=None, gain=True, std=1.0):
    lens = [max(p, 0) + 1 for p in pos]
    table = ref.tables(lens, slots, pages_n, rng, width)
    pages = ref.Pages(pages_n, kv, slots, "cuda")
    for b, n in enumerate(lens):
        if n > 1:
            pages.put(table[b], 0, normal(torch, rng, kv, n - 1, 128, std=std), normal(torch, rng, kv, n - 1, 128))
    qkv = normal(torch, rng, len(pos), (heads + 2 * kv) * 128)
    return dict(qkv=qkv, pages=pages, table=table, gains=gains(torch, rng, gain), pos=list(pos), heads=heads, kv=kv,
                rope=rope(torch, yuear_lib, max(lens)))


def decode(torch, yuear_lib, s, window=0, sinks=0, **kw):
    return yuear_lib.paged_attention_decode(
        s["qkv"], s["pages"].k, s["pages"].v, ints(torch, s["table"]), ints(torch, s["pos"]), *s["rope"],
        q_norm=s["gains"][0], k_norm=s["gains"][1], eps=EPS, window=window, sinks=sinks, **kw)


def check_decode(torch, s, out, window=0, sinks=0, own=None):
    """Output and appended rows of every sequence of a decode call; `own`:
    (key, value) rows to take for the token where the table does not keep it."""
    heads, kv = s["heads"], s["kv"]
    for b, p in enumerate(s["pos"]):
        x = s["qkv"][b].reshape(-1, 128)
        c, n = s["rope"][0][p], s["rope"][1][p]
        q, _ = ref.turn(x[:heads], s["gains"][0], c, n, EPS)
        new, size = ref.turn(x[heads:heads + kv], s["gains"][1], c, n, EPS)
        k, v, present = ref.gather(s["pages"].k, s["pages"].v, s["table"][b], p + 1)
        if present[p]:
            ref.check(k[:, p], new, ref.HALF * new.abs() + ref.FINE * size, f"key of sequence {b}")
            assert torch.equal(v[:, p], x[heads + kv:].double())
        else:  # the token sees itself all the same
            k[:, p], v[:, p], present[p] = new.to(torch.bfloat16).double(), x[heads + kv:].double(), True
        seen = ref.visible(p, p + 1, window, sinks) & present
        want, bound = ref.attend(q, k, v, seen, 2.0 ** -16)
        ref.check(out[b], want, bound, f"sequence {b} at {p}")


@pytest.mark.parametrize("heads,kv,slots,pos,window,sinks,gain", [
    (24, 8, 64, [0], 0, 0, True),
    (24, 8, 64, [332], 0, 0, True),
    (24, 8, 64, [4095], 0, 0, True),
    (16, 8, 32, [0, 1, 31, 32, 33, 127, 128, 700], 0, 0, True),
    (1, 1, 32, [5, 3000], 0, 0, False),
    (8, 1, 128, [129, 9000, 64], 0, 0, True),
    (6, 1, 256, [1000, 255, 256], 0, 0, True),
    (32, 8, 64, [511, 1024], 0, 0, False),
    (24, 8, 64, [0, 40, 63, 64, 65, 500, 2000], 1, 0, True),
    (24, 8, 64, [0, 40, 63, 64, 65, 500, 2000], 64, 1, True),
    (16, 8, 32, [10, 99, 100, 131, 132, 133, 640, 1501], 100, 33, True),
    (4, 2, 32, [3000, 2999], 1000, 32, True),
    (3, 1, 64, [800], 30, 5000, True),       # more sinks than keys
    (2, 1, 32, [777], 2 ** 31 - 1, 3, True),  # a window over everything
])
def test_decode(torch, yuear_lib, heads, kv, slots, pos, window, sinks, gain):
    rng = np.random.default_rng(heads + kv + len(pos) + window % 997)
    s = decode_inputs(torch, yuear_lib, rng, heads, kv, slots, pos, 700, gain=gain)
    before_k, before_v = s["pages"].k.clone(), s["pages"].v.clone()
    out = decode(torch, yuear_lib, s, window, sinks)
    torch.cuda.synchronize()
    check_decode(torch, s, out, window, sinks)
    # nothing else of the pages changed
    for b, p in enumerate(pos):
        page, slot = int(s["table"][b][p // slots]), p % slots
        before_k[page, :, slot] = s["pages"].k[page, :, slot]
        before_v[page, :, slot // 32, :, slot % 32] = s["pages"].v[page, :, slot // 32, :, slot % 32]
    assert same_bits(torch, before_k, s["pages"].k) and same_bits(torch, before_v, s["pages"].v)


def test_decode_of_many_sequences(torch, yuear_lib):
    rng = np.random.default_rng(3)
    pos = [int(p) for p in np.exp(rng.uniform(0, np.log(600), 300))]
    s = decode_inputs(torch, yuear_lib, rng, 3, 1, 32, pos, 4000)
    ws = yuear_lib.paged_workspace(300, 3, 1)
    out = decode(torch, yuear_lib, s, workspace=ws)
    check_decode(torch, s, out)
    assert not ws[:512 * 64].any()  # the counters are ready for the next call


def test_decode_of_large_scores(torch, yuear_lib):
    """Scores of hundreds: the weights are those of the largest few keys."""
    rng = np.random.default_rng(5)
    s = decode_inputs(torch, yuear_lib, rng, 6, 2, 64, [700, 90], 40, std=30.0, gain=False)
    s["qkv"][:, :6 * 128] *= 10
    check_decode(torch, s, decode(torch, yuear_lib, s))


def test_decode_leaves_out_sequences_outside_the_table(torch, yuear_lib):
    rng = np.random.default_rng(6)
    s = decode_inputs(torch, yuear_lib, rng, 3, 1, 32, [40, 10, 63, 5], 30, width=2)
    k, v = s["pages"].k.clone(), s["pages"].v.clone()
    s["pos"] = [-1, 64, 2 ** 31 - 1, -2 ** 31]
    out = torch.full((4, 3, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    decode(torch, yuear_lib, s, out=out)
    torch.cuda.synchronize()
    assert (out == 7).all() and same_bits(torch, k, s["pages"].k) and same_bits(torch, v, s["pages"].v)
    s["pos"], s["rope"] = [40, 10, 63, 5], tuple(t[:41].contiguous() for t in s["rope"])  # 63 has no rope row
    decode(torch, yuear_lib, s, out=out)
    torch.cuda.synchronize()
    assert (out[2] == 7).all() and not (out[[0, 1, 3]] == 7).all(-1).any()


@pytest.mark.parametrize("bad", [-1, 30, 2 ** 31 - 1, -2 ** 31])
def test_decode_sees_no_key_of_a_page_that_is_not_there(torch, yuear_lib, bad):
    rng = np.random.default_rng(7)
    s = decode_inputs(torch, yuear_lib, rng, 24, 8, 64, [800, 64, 63, 200], 30)
    s["table"][0, [0, 3, 4, 9]] = bad
    s["table"][1, 1] = bad   # the token's own page: it sees itself and the first page
    s["table"][2, 0] = bad   # ... and here nothing else
    s["table"][3, 0:4] = bad
    out = decode(torch, yuear_lib, s)
    check_decode(torch, s, out)


def test_decode_ignores_infinities_that_it_does_not_see(torch, yuear_lib):
    rng = np.random.default_rng(8)
    s = decode_inputs(torch, yuear_lib, rng, 6, 2, 32, [500], 30)
    for fill in (float("inf"), float("-inf"), float("nan")):
        for t in list(range(35, 396)):  # between the sinks and the window
            page, slot = int(s["table"][0][t // 32]), t % 32
            s["pages"].k[page, :, slot] = fill
            s["pages"].v[page, :, slot // 32, :, slot % 32] = fill
        out = decode(torch, yuear_lib, s, 105, 35)
        assert torch.isfinite(out).all()
    for t in range(35, 396):
        page, slot = int(s["table"][0][t // 32]), t % 32
        s["pages"].k[page, :, slot] = 0
        s["pages"].v[page, :, slot // 32, :, slot % 32] = 0
    check_decode(torch, s, out, 105, 35)


def test_decode_of_strided_rows_on_another_stream(torch, yuear_lib):
    rng = np.random.default_rng(9)
    s = decode_inputs(torch, yuear_lib, rng, 3, 1, 64, [100, 300, 7], 30)
    wide = torch.zeros(3, 5 * 128 + 40, dtype=torch.bfloat16, device="cuda")
    wide[:, :640] = s["qkv"]
    s["qkv"] = wide[:, :640]
    out = torch.full((3, 5, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = yuear_lib.paged_workspace(3, 3, 1)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with pytest.raises(ValueError, match="another stream"):
        decode(torch, yuear_lib, s, stream=stream.cuda_stream)
    table, pos = ints(torch, s["table"]), ints(torch, s["pos"])
    torch.cuda.synchronize()
    yuear_lib.paged_attention_decode(s["qkv"], s["pages"].k, s["pages"].v, table, pos, *s["rope"],
                                     q_norm=s["gains"][0], k_norm=s["gains"][1], eps=EPS, workspace=ws,
                                     out=out[:, 1:4], stream=stream.cuda_stream)
    stream.synchronize()
    check_decode(torch, s, out[:, 1:4])
    assert (out[:, 0] == 7).all() and (out[:, 4] == 7).all()


def test_decode_replayed_from_a_graph(torch, yuear_lib):
    """One captured call serves every length: positions, rows and tables change
    between replays, and each equals the eager call's bits."""
    rng = np.random.default_rng(10)
    s = decode_inputs(torch, yuear_lib, rng, 24, 8, 64, [900, 5, 400], 60, width=40)
    table, pos = ints(torch, s["table"]), ints(torch, s["pos"])
    ws, out = yuear_lib.paged_workspace(3, 24, 8), torch.empty(3, 24, 128, dtype=torch.bfloat16, device="cuda")
    cos, sin = rope(torch, yuear_lib, 2000)

    def call(qkv, k, v, o, w):
        yuear_lib.paged_attention_decode(qkv, k, v, table, pos, cos, sin, eps=EPS, window=512, sinks=70, workspace=w,
                                         out=o)
    call(s["qkv"], s["pages"].k, s["pages"].v, out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(s["qkv"], s["pages"].k, s["pages"].v, out, ws)
    ws2 = yuear_lib.paged_workspace(3, 24, 8)
    for step in range(5):
        pos.copy_(ints(torch, [900 + step, 5 + 40 * step, max(-1, 400 - 150 * step)]))
        s["qkv"].copy_(normal(torch, rng, *s["qkv"].shape))
        k, v, want = s["pages"].k.clone(), s["pages"].v.clone(), out.clone()
        graph.replay()
        call(s["qkv"], k, v, want, ws2)
        torch.cuda.synchronize()
        assert same_bits(torch, out, want) and same_bits(torch, k, s["pages"].k) and same_bits(torch, v, s["pages"].v)


def test_calls_of_unlike_shapes_take_turns_on_a_workspace(torch, yuear_lib):
    rng = np.random.default_rng(11)
    shapes = [(24, 8, [4000]), (2, 1, [3000, 50]), (8, 1, [2500]), (16, 8, [100] * 9)]
    ws = yuear_lib.paged_workspace(9, 64, 8, 600)
    for heads, kv, pos in shapes * 2:
        s = decode_inputs(torch, yuear_lib, rng, heads, kv, 64, pos, 120)
        check_decode(torch, s, decode(torch, yuear_lib, s, workspace=ws))
        t = prefill_inputs(torch, rng, heads, kv, 64, [60, 9], [700, 3], 120)
        check_prefill(torch, t, prefill(torch, yuear_lib, t, workspace=ws))


# ---- prompt attention ----

def prefill_inputs(torch, rng, heads, kv, slots, lens, pos0, pages_n, width=None, std=1.0):
    ends = [p + n for p, n in zip(pos0, lens)]
    table = ref.tables(ends, slots, pages_n, rng, width)
    pages = ref.Pages(pages_n, kv, slots, "cuda")
    for b, n in enumerate(ends):
        if n:
            pages.put(table[b], 0, normal(torch, rng, kv, n, 128, std=std), normal(torch, rng, kv, n, 128, mean=0.1))
    return dict(q=normal(torch, rng, sum(lens), heads, 128, std=1.5), pages=pages, table=table, pos0=list(pos0),
                starts=np.concatenate([[0], np.cumsum(lens)]), heads=heads, kv=kv)


def prefill(torch, yuear_lib, s, window=0, sinks=0, **kw):
    return yuear_lib.paged_attention_prefill(s["q"], s["pages"].k, s["pages"].v, ints(torch, s["table"]),
                                             ints(torch, s["starts"]), ints(torch, s["pos0"]), window=window,
                                             sinks=sinks, **kw)


def check_prefill(torch, s, out, window=0, sinks=0, some=40, seed=0):
    """Rows of a prompt call: the first, the last and `some` others of each sequence."""
    rng = np.random.default_rng(seed)
    heads, kv = s["heads"], s["kv"]
    for b, p0 in enumerate(s["pos0"]):
        a, e = int(s["starts"][b]), int(s["starts"][b + 1])
        if a == e:
            continue
        k, v, present = ref.gather(s["pages"].k, s["pages"].v, s["table"][b], p0 + e - a)
        for i in sorted({0, e - a - 1} | set(rng.integers(0, e - a, some).tolist())):
            p = p0 + i
            seen = ref.visible(p, p + 1, window, sinks) & present[:p + 1]
            want, bound = ref.attend(s["q"][a + i].double(), k[:, :p + 1], v[:, :p + 1], seen, ref.HALF)
            ref.check(out[a + i], want, bound, f"row {i} of sequence {b}")


@pytest.mark.parametrize("heads,kv,slots,lens,pos0,window,sinks", [
    (24, 8, 64, [1], [0], 0, 0),
    (24, 8, 64, [1], [1000], 0, 0),
    (24, 8, 64, [300], [0], 0, 0),
    (24, 8, 64, [97], [2000], 0, 0),
    (16, 8, 32, [5, 0, 33, 64, 1, 200], [0, 7, 31, 32, 63, 95], 0, 0),
    (1, 1, 32, [500], [77], 0, 0),
    (4, 4, 128, [31, 32, 65], [1, 127, 96], 0, 0),
    (6, 1, 256, [300], [255], 0, 0),
    (8, 1, 64, [130, 41], [20, 0], 0, 0),
    (32, 8, 32, [257], [63], 0, 0),
    (24, 8, 64, [700], [0], 1, 0),
    (24, 8, 64, [700], [3], 64, 1),
    (16, 8, 32, [400, 1, 700], [0, 900, 350], 100, 33),
    (3, 1, 64, [1000], [100], 333, 130),
    (2, 1, 32, [200], [1500], 30, 5000),
    (2, 1, 32, [77], [700], 2 ** 31 - 1, 3),
    (3, 1, 32, [1 + i % 3 for i in range(150)], [i % 70 for i in range(150)], 40, 2),
    (24, 8, 64, [3000], [0], 0, 0),
])
def test_prefill(torch, yuear_lib, heads, kv, slots, lens, pos0, window, sinks):
    rng = np.random.default_rng(heads + kv + len(lens) + window % 997)
    s = prefill_inputs(torch, rng, heads, kv, slots, lens, pos0, 500)
    check_prefill(torch, s, prefill(torch, yuear_lib, s, window, sinks), window, sinks, 40 if len(lens) < 20 else 1)


@pytest.mark.parametrize("heads,kv,slots,lens,pos0,window,sinks", [
    (24, 8, 64, [1], [0], 0, 0),
    (24, 8, 64, [97], [4000], 0, 0),
    (24, 8, 64, [43, 42], [41, 4000], 0, 0),
    (16, 8, 32, [5, 0, 33, 64, 1, 200], [0, 7, 31, 32, 63, 95], 0, 0),
    (1, 1, 32, [500], [77], 0, 0),
    (4, 4, 128, [31, 32, 65], [1, 127, 96], 0, 0),
    (6, 1, 256, [300], [255], 0, 0),
    (8, 1, 64, [130, 41], [20, 3000], 0, 0),
    (16, 8, 32, [400, 1, 300], [0, 3000, 350], 1000, 33),
    (3, 1, 64, [1000], [100], 700, 130),
    (2, 1, 32, [200], [1500], 30, 5000),
    (2, 1, 32, [77], [700], 2 ** 31 - 1, 3),
    (3, 1, 32, [1 + i % 3 for i in range(16)], [i % 70 for i in range(16)], 0, 0),
    (3, 1, 32, [1 + i % 3 for i in range(17)], [i % 70 for i in range(17)], 0, 0),
    (3, 1, 32, [i % 4 for i in range(32)], [i % 70 for i in range(32)], 0, 0),
    (3, 1, 32, [i % 4 for i in range(33)], [i % 70 for i in range(33)], 0, 0),
])
def test_prefill_in_a_table_with_room(torch, yuear_lib, heads, kv, slots, lens, pos0, window, sinks):
    """A table of 16384 slots, where steps are dealt out however few keys there are."""
    rng = np.random.default_rng(heads + kv + len(lens) + window % 997)
    s = prefill_inputs(torch, rng, heads, kv, slots, lens, pos0, 500, width=16384 // slots)
    check_prefill(torch, s, prefill(torch, yuear_lib, s, window, sinks), window, sinks)


def test_prefill_of_large_scores(torch, yuear_lib):
    """Rows whose largest score grows by hundreds along the keys, and rows whose
    scores all lie far below zero."""
    rng = np.random.default_rng(15)
    s = prefill_inputs(torch, rng, 3, 1, 64, [400, 90], [30, 0], 30, std=10.0)
    s["q"] *= 10
    check_prefill(torch, s, prefill(torch, yuear_lib, s), some=60)
    s["q"] = s["q"].abs()
    s["pages"].k = -s["pages"].k.abs()
    check_prefill(torch, s, prefill(torch, yuear_lib, s), some=60)


@pytest.mark.parametrize("bad", [-1, 30, 2 ** 31 - 1, -2 ** 31])
def test_prefill_sees_no_key_of_a_page_that_is_not_there(torch, yuear_lib, bad):
    rng = np.random.default_rng(16)
    s = prefill_inputs(torch, rng, 24, 8, 32, [200, 40, 33], [300, 0, 20], 30)
    s["table"][0, [0, 3, 4, 12]] = bad
    s["table"][1, :] = bad          # rows that see nothing
    s["table"][2, 0] = bad          # ... until the second page
    out = prefill(torch, yuear_lib, s)
    check_prefill(torch, s, out)
    assert not out[200:240].any() and not out[240:252].any() and out[252:].any()


@pytest.mark.parametrize("width", [8, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3)])
def test_prefill_keeps_infinities_from_rows_that_do_not_see_them(torch, yuear_lib, width, window, sinks):
    """Values of some keys are infinities and NaNs: rows that see them give those,
    the rows beside them in a tile what they give with zeros there."""
    rng = np.random.default_rng(23)
    heads, kv, n, before = 24, 8, 150, 130
    s = prefill_inputs(torch, rng, heads, kv, 64, [n], [before], 30, width=width)
    inf = float("inf")
    marks = {131: inf, 170: float("nan"), 171: -inf, 200: inf, 201: -inf, 279: inf}
    v = normal(torch, rng, kv, before + n, 128)
    odd = torch.zeros_like(v)
    for t, x in marks.items():
        odd[:, t, 5:100:7] = x
        if t in (170, 201):
            odd[:, t] = x
    k = normal(torch, rng, kv, before + n, 128)
    s["pages"].put(s["table"][0], 0, k, torch.where(odd == 0, v, torch.zeros_like(v)))
    clean = prefill(torch, yuear_lib, s, window, sinks)
    check_prefill(torch, s, clean, window, sinks)
    s["pages"].put(s["table"][0], 0, k, torch.where(odd == 0, v, odd))
    out = prefill(torch, yuear_lib, s, window, sinks).float()
    want = clean.float()
    for i in range(n):
        for t in marks:
            if ref.visible(before + i, before + n, window, sinks)[t]:
                want[i] += odd[:, t].float().repeat_interleave(heads // kv, 0)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~finite].nan_to_num(), want[~finite].nan_to_num())
    s["pages"].put(s["table"][0], 0, k, torch.where(odd == 0, v, torch.zeros_like(v)))
    check_prefill(torch, s, torch.where(finite, out, want.nan_to_num(0, 0, 0) + clean), window, sinks, some=150)


@pytest.mark.parametrize("width", [8, 128])
def test_prefill_gives_nan_for_a_row_whose_query_is_nan(torch, yuear_lib, width):
    rng = np.random.default_rng(24)
    s = prefill_inputs(torch, rng, 24, 8, 64, [150], [130], 30, width=width)
    s["pages"].v[int(s["table"][0, 4]), 3, 0, 5, 20] = float("inf")  # key 276 of kv head 3: a tile with an odd value
    clean = prefill(torch, yuear_lib, s)
    s["q"][70, 4] = float("nan")
    s["q"][148, 9:12] = float("nan")
    out = prefill(torch, yuear_lib, s)
    nan = torch.isnan(s["q"])
    assert torch.isnan(out[nan]).all() and same_bits(torch, out[~nan], clean[~nan])


@pytest.mark.parametrize("width", [8, 128])
def test_prefill_with_decreasing_starts_stays_in_its_workspace(torch, yuear_lib, width):
    rng = np.random.default_rng(25)
    lens, n = [20] * 16, 320
    s = prefill_inputs(torch, rng, 8, 8, 64, lens, [3] * 16, 300, width=width)
    s["starts"] = np.array([0, n] * 8 + [0])  # every second sequence takes all rows
    need = yuear_lib.lib.yuear_op_paged_workspace_bytes(16, 8, 8, n)
    ws = yuear_lib.paged_workspace(16, 8, 8, n)
    assert ws.numel() * 4 == need
    guarded = torch.full((need // 4 + 4096,), 7, dtype=torch.int32, device="cuda")
    guarded[:need // 4] = 0
    prefill(torch, yuear_lib, s, workspace=guarded)
    torch.cuda.synchronize()
    assert (guarded[need // 4:] == 7).all() and not guarded[:131072 // 4].any()
    # the workspace is fit for the next call
    t = prefill_inputs(torch, rng, 8, 8, 64, lens, [3] * 16, 300, width=width)
    check_prefill(torch, t, prefill(torch, yuear_lib, t, workspace=guarded))


def test_prefill_leaves_other_rows_as_they_are(torch, yuear_lib):
    rng = np.random.default_rng(17)
    s = prefill_inputs(torch, rng, 3, 1, 32, [40, 10, 10, 40], [40, 0, 3, 0], 30, width=3)
    s["table"] = np.ascontiguousarray(s["table"][:, :2])  # ends at 64
    s["pos0"] = [40, -1, 64, 0]
    wide = torch.zeros(102, 4, 128, dtype=torch.bfloat16, device="cuda")
    wide[1:101, 1:] = s["q"]
    s["q"], s["starts"] = wide[:, 1:], s["starts"] + 1
    out = torch.full((102, 5, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    prefill(torch, yuear_lib, s, out=out[:, 1:4])
    torch.cuda.synchronize()
    left = (out == 7).all(-1).cpu().numpy()
    assert left[:, 0].all() and left[:, 4].all()
    rows = left[:, 1:4].all(-1)
    assert rows[0] and not rows[1:25].any() and rows[25:61].all() and not rows[61:101].any() and rows[101]
    s.update(pos0=[40, 0], starts=np.array([1, 25, 25]), table=s["table"][:2])
    check_prefill(torch, s, out[:, 1:4])


def test_prefill_replayed_from_a_graph(torch, yuear_lib):
    rng = np.random.default_rng(18)
    s = prefill_inputs(torch, rng, 24, 8, 64, [130, 20], [700, 0], 60, width=20)
    table, starts, pos0 = ints(torch, s["table"]), ints(torch, s["starts"]), ints(torch, s["pos0"])
    ws = [yuear_lib.paged_workspace(2, 24, 8, 150) for _ in range(2)]
    out = torch.empty_like(s["q"])

    def call(o, w):
        yuear_lib.paged_attention_prefill(s["q"], s["pages"].k, s["pages"].v, table, starts, pos0, workspace=w, out=o)
    call(out, ws[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, ws[0])
    for step in range(4):
        starts.copy_(ints(torch, [0, 130 - 40 * step, 150 - 10 * step]))
        pos0.copy_(ints(torch, [700 - 200 * step, step]))
        s["q"].copy_(normal(torch, rng, *s["q"].shape))
        want = out.clone()
        graph.replay()
        call(want, ws[1])
        torch.cuda.synchronize()
        assert same_bits(torch, out, want)


# ---- copies, and pages far into a pool ----

@pytest.mark.parametrize("layers,kv,slots,pairs", [(1, 1, 32, 1), (3, 8, 64, 17), (2, 2, 128, 300), (28, 4, 32, 5)])
def test_pages_copy(torch, yuear_lib, layers, kv, slots, pairs):
    rng = np.random.default_rng(pairs)
    n = 2 * pairs + 3
    k = normal(torch, rng, layers, n, kv, slots, 128)
    v = normal(torch, rng, layers, n, kv, slots // 32, 128, 32)
    k[0, 0], v[0, 1] = float("nan"), float("inf")
    ids = rng.permutation(n)
    src, dst = rng.choice(ids[:pairs], pairs).tolist(), ids[pairs:2 * pairs].tolist()
    want_k, want_v = k.clone(), v.clone()
    want_k[:, dst], want_v[:, dst] = want_k[:, src], want_v[:, src]
    yuear_lib.pages_copy(k, v, src, dst)
    assert same_bits(torch, k, want_k) and same_bits(torch, v, want_v)
    yuear_lib.pages_copy(k, v, [], [])
    if layers == 1:
        yuear_lib.pages_copy(k[0], v[0], [dst[0]], [src[0]])
        assert same_bits(torch, k, want_k)
    with pytest.raises(ValueError):
        yuear_lib.pages_copy(k, v, [0, 1], [2, 2])


def test_pages_past_32_bit_offsets(torch, yuear_lib):
    """Pages whose first element lies past 2^32 (8 kv heads of 64 slots)."""
    rng = np.random.default_rng(20)
    n, kv, slots = 66000, 8, 64
    assert (n - 400) * kv * slots * 128 > 2 ** 32
    k = torch.empty(n, kv, slots, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.empty(n, kv, slots // 32, 128, 32, dtype=torch.bfloat16, device="cuda")
    k[-400:], v[-400:] = float("nan"), float("nan")
    lens, pos0 = [150, 70], [0, 0]
    table = ref.tables([200, 200], slots, 300, rng) + (n - 310)
    qkv = normal(torch, rng, sum(lens), 40 * 128)
    cos, sin = rope(torch, yuear_lib, 300)
    starts = np.array([0, 150, 220])
    q = yuear_lib.paged_append(qkv, k, v, ints(torch, table), ints(torch, starts), ints(torch, pos0), cos, sin)
    out = yuear_lib.paged_attention_prefill(q, k, v, ints(torch, table), ints(torch, starts), ints(torch, pos0))
    pages = ref.Pages(1, kv, slots, "cuda")
    pages.k, pages.v = k, v
    check_prefill(torch, dict(q=q, pages=pages, table=table, pos0=pos0, starts=starts, heads=24, kv=8), out)
    s = dict(qkv=normal(torch, rng, 2, 40 * 128), pages=pages, table=table, gains=[None, None], pos=[150, 70], heads=24,
             kv=8, rope=(cos, sin))
    check_decode(torch, s, decode(torch, yuear_lib, s))
    src, dst = [int(table[0][0]), int(table[1][0])], [n - 1, n - 2]
    yuear_lib.pages_copy(k, v, src, dst)
    assert same_bits(torch, k[dst], k[src]) and same_bits(torch, v[dst], v[src])


# ---- a server's life: prompts, forks, decoding, windows, compaction ----

def test_a_run_of_requests(torch, yuear_lib):
    rng = np.random.default_rng(21)
    heads, kv, slots, layers, window, sinks = 6, 2, 32, 2, 150, 20
    pool = yuear_lib.PagePool(80, slots)
    pages = [ref.Pages(80, kv, slots, "cuda") for _ in range(layers)]
    k = torch.stack([p.k for p in pages])
    v = torch.stack([p.v for p in pages])
    qn, kn = gains(torch, rng)
    cos, sin = rope(torch, yuear_lib, 600)
    kept = {}  # sequence -> per layer [keys, values] of all its tokens, as the pages should hold them

    def copies(c):
        yuear_lib.pages_copy(k, v, *c)

    def rows_of(seqs, width=20):
        return pool.table(seqs, width)

    def prompts(seqs, lens):
        pos0 = [pool.length(s) for s in seqs]
        for s, n in zip(seqs, lens):
            copies(pool.extend(s, n))
        table, starts = rows_of(seqs), np.concatenate([[0], np.cumsum(lens)])
        args = ints(torch, table), ints(torch, starts), ints(torch, pos0)
        for layer in range(layers):
            qkv = normal(torch, rng, sum(lens), (heads + 2 * kv) * 128)
            q = yuear_lib.paged_append(qkv, k[layer], v[layer], *args, cos, sin, q_norm=qn, k_norm=kn, eps=EPS)
            out = yuear_lib.paged_attention_prefill(q, k[layer], v[layer], *args, window=window, sinks=sinks)
            for b, s in enumerate(seqs):
                x = qkv[starts[b]:starts[b + 1]].reshape(lens[b], -1, 128)
                at = slice(pos0[b], pos0[b] + lens[b])
                y, size = ref.turn(x[:, heads:heads + kv], kn, cos[at, None], sin[at, None], EPS)
                got, values, present = ref.gather(k[layer], v[layer], table[b], pos0[b] + lens[b])
                ref.check(got[:, at].transpose(0, 1), y, ref.HALF * y.abs() + ref.FINE * size, "keys")
                old = kept.setdefault(s, {}).get(layer, [got[:, :0], values[:, :0]])
                kept[s][layer] = [torch.cat((old[0], got[:, at]), 1),
                                  torch.cat((old[1], x[:, heads + kv:].double().transpose(0, 1)), 1)]
                for i in range(0, lens[b], 7):
                    p = pos0[b] + i
                    want, bound = ref.attend(q[starts[b] + i].double(), *(t[:, :p + 1] for t in kept[s][layer]),
                                             ref.visible(p, p + 1, window, sinks), ref.HALF)
                    ref.check(out[starts[b] + i], want, bound, f"prompt of {s}")

    def step(seqs, ws):
        pos = [pool.length(s) for s in seqs]
        for s in seqs:
            pool.trim(s, window, sinks)  # before the new token's room: it is the next one
            copies(pool.extend(s, 1))
        table = rows_of(seqs)
        for layer in range(layers):
            qkv = normal(torch, rng, len(seqs), (heads + 2 * kv) * 128)
            out = yuear_lib.paged_attention_decode(qkv, k[layer], v[layer], ints(torch, table), ints(torch, pos), cos,
                                                   sin, q_norm=qn, k_norm=kn, eps=EPS, window=window, sinks=sinks,
                                                   workspace=ws)
            for b, s in enumerate(seqs):
                x = qkv[b].reshape(-1, 128)
                page, slot = int(table[b][pos[b] // slots]), pos[b] % slots
                y, size = ref.turn(x[heads:heads + kv], kn, cos[pos[b]], sin[pos[b]], EPS)
                new = k[layer][page, :, slot].double()
                ref.check(new, y, ref.HALF * y.abs() + ref.FINE * size, "key")
                kept[s][layer] = [torch.cat((kept[s][layer][0], new[:, None]), 1),
                                  torch.cat((kept[s][layer][1], x[heads + kv:].double()[:, None]), 1)]
                q, _ = ref.turn(x[:heads], qn, cos[pos[b]], sin[pos[b]], EPS)
                want, bound = ref.attend(q, *kept[s][layer], ref.visible(pos[b], pos[b] + 1, window, sinks), 2.0 ** -16)
                ref.check(out[b], want, bound, f"step of {s} at {pos[b]}")

    def fork(s):
        new = pool.fork(s)
        kept[new] = {layer: list(kv_) for layer, kv_ in kept[s].items()}
        return new

    def done(s):
        pool.close_sequence(s)
        del kept[s]

    a, b = pool.open(), pool.open()
    prompts([a, b], [200, 45])
    takes = [fork(b) for _ in range(3)]     # shared pages, then a page of their own each
    prompts([a, takes[0]], [30, 61])        # the rest of a prompt, after a shared one
    ws = yuear_lib.paged_workspace(6, heads, kv)
    for _ in range(3):
        step([a, b, *takes], ws)
    done(b)
    copies(pool.compact())                  # holes are filled, tables move
    for _ in range(40):
        step([*takes, a], ws)
    done(a)
    src, dst = pool.compact()
    assert src
    copies((src, dst))
    step(takes, ws)
    for s in takes:
        done(s)
    assert pool.unused == 80


# ---- refusals of the binding ----

def test_binding_refuses_tensors_that_do_not_fit(torch, yuear_lib):
    rng = np.random.default_rng(22)
    s = decode_inputs(torch, yuear_lib, rng, 3, 1, 32, [40, 10], 30)
    good = dict(qkv=s["qkv"], k_pages=s["pages"].k, v_pages=s["pages"].v, table=ints(torch, s["table"]),
                pos=ints(torch, s["pos"]), cos=s["rope"][0], sin=s["rope"][1])
    bad = dict(qkv=[s["qkv"].float(), s["qkv"][:, :600], s["qkv"].cpu(), s["qkv"][0], s["qkv"][:1]],
               k_pages=[s["pages"].k.float(), s["pages"].k[:, :, :, :64], s["pages"].k[:, :, ::2]],
               v_pages=[s["pages"].v[:-1], s["pages"].v.transpose(-1, -2)],
               table=[good["table"].long(), good["table"].t().contiguous().t(), good["table"][:1], good["table"].cpu()],
               pos=[good["pos"].long(), good["pos"][:1], good["pos"].cpu()],
               cos=[s["rope"][0].float(), s["rope"][0][:, :32], s["rope"][0][:10]])
    for key, values in bad.items():
        for value in values:
            with pytest.raises(ValueError):
                yuear_lib.paged_attention_decode(**{**good, key: value})
    for kw in (dict(window=-1), dict(sinks=-1), dict(q_norm=s["qkv"][0, :64]),
               dict(out=torch.empty(2, 4, 128, dtype=torch.bfloat16, device="cuda")),
               dict(workspace=torch.zeros(16, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            yuear_lib.paged_attention_decode(**good, **kw)
    empty = yuear_lib.paged_attention_decode(s["qkv"][:0], s["pages"].k, s["pages"].v, good["table"][:0],
                                             good["pos"][:0], *s["rope"])
    assert empty.shape == (0, 3, 128)


def test_binding_refuses_numbers_past_32_bits(torch, yuear_lib):
    """Such a number is refused, not cut to its low bits."""
    rng = np.random.default_rng(26)
    s = prefill_inputs(torch, rng, 3, 1, 32, [40], [0], 30)
    for kw in (dict(window=2 ** 32 + 1), dict(window=1, sinks=2 ** 32 + 1), dict(window=2 ** 31)):
        with pytest.raises(ValueError):
            prefill(torch, yuear_lib, s, **kw)
    for src, dst in (([2 ** 32], [1]), ([0], [2 ** 32 + 1]), ([0], [30]), ([-1], [1]), ([0, 1], [2])):
        with pytest.raises(ValueError):
            yuear_lib.pages_copy(s["pages"].k, s["pages"].v, src, dst)
    yuear_lib.pages_copy(s["pages"].k, s["pages"].v, [], [])
