"""Paged cache operators on the GPU where their plans and their arithmetic meet an
edge: infinities that are seen, scores past 2^24, workgroups that walk several
items or tiles, one long sequence among short ones, and the same cache through
the contiguous operators. Bounds are paged_ref.py's."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import (check_decode, check_prefill, decode, decode_inputs, ints, normal, prefill, prefill_inputs,
                            rope, same_bits, torch)  # noqa: F401 (torch: the fixture)

pytestmark = pytest.mark.gpu
INF = float("inf")
COUNTERS = 131072 // 4  # int32 words of a workspace before its partial sums
UNSET = 0x7F123456      # no sum of these tests


def put_v(s, b, t, head, dims, x):
    page, slot = int(s["table"][b][t // s["pages"].slots]), t % s["pages"].slots
    s["pages"].v[page, head, slot // 32, dims, slot % 32] = x


def put_k(s, b, t, head, dims, x):
    page, slot = int(s["table"][b][t // s["pages"].slots]), t % s["pages"].slots
    s["pages"].k[page, head, slot, dims] = x


def marked_workspace(torch, yuear_lib, *sizes):
    ws = yuear_lib.paged_workspace(*sizes)
    ws[COUNTERS:] = UNSET
    return ws


def written_slots(torch, ws, group):
    """Which partial sums of a decode call its workgroups left: [512, 2], for each
    workgroup that of an item that began before it and that of one that begins in it."""
    words = group * 130
    part = ws[COUNTERS:COUNTERS + 1024 * words].view(1024, words)
    return (part != UNSET).any(1).cpu().numpy().reshape(512, 2)


# ---- infinities that a row sees ----

@pytest.mark.parametrize("pos", [[40], [500, 40, 31, 700], [5000], [20 + 9 * i for i in range(70)]])
def test_decode_gives_the_infinities_that_it_sees(torch, yuear_lib, pos):
    """An infinite value gives an infinity of its sign whatever its key's weight is."""
    rng = np.random.default_rng(len(pos))
    heads, kv = 6, 2
    s = decode_inputs(torch, yuear_lib, rng, heads, kv, 64, pos, 200 if len(pos) < 9 else 500)
    first, middle, own, last = slice(0, 30, 7), slice(31, 60, 7), slice(61, 90, 7), slice(91, 120, 7)
    rows = s["qkv"].view(len(pos), heads + 2 * kv, 128)

    def marks(scale):
        for b, p in enumerate(pos):
            put_v(s, b, 0, 0, first, INF * scale if scale else 0.0)
            put_v(s, b, p // 2, 1, middle, -INF * scale if scale else 0.0)
            rows[b, heads + kv, own] = INF if scale else 0.0
            put_v(s, b, p - 1, 1, last, INF if scale else 0.0)
    marks(0)
    check_decode(torch, s, decode(torch, yuear_lib, s))
    marks(1)
    out = decode(torch, yuear_lib, s)
    want = torch.zeros(len(pos), kv, heads // kv, 128, device="cuda")
    want[:, 0, :, first], want[:, 1, :, middle], want[:, 0, :, own], want[:, 1, :, last] = INF, -INF, INF, INF
    want = want.view(len(pos), heads, 128)
    odd = want != 0
    assert torch.equal(out[odd].float(), want[odd])
    marks(0)
    plain = decode(torch, yuear_lib, s)
    check_decode(torch, s, torch.where(odd, plain, out))


@pytest.mark.parametrize("batch", [1, 70])
def test_decode_keeps_unseen_slots_out_beside_infinities_that_it_sees(torch, yuear_lib, batch):
    """Window, sinks, a page that is not there and slots past the token, all of them
    NaN, in blocks that hold a seen infinity."""
    rng = np.random.default_rng(39)
    heads, kv, window, sinks = 8, 2, 105, 35
    pos = [500 + i for i in range(batch)]
    s = decode_inputs(torch, yuear_lib, rng, heads, kv, 32, pos, 20 * batch)
    s["table"][:, 13] = -1  # keys 416 to 447 are not there
    dims = slice(3, 128, 11)
    marks = {0: [34], 1: [398 + batch, 500]}  # of a kv head: keys that every sequence sees

    def fill(x):
        for b, p in enumerate(pos):
            for h, keys in marks.items():
                for t in keys:
                    if t < p:
                        put_v(s, b, t, h, dims, x)
    for b, p in enumerate(pos):
        for t in [35, 63, p - window, p - window - 1]:
            put_k(s, b, t, slice(None), slice(None), float("nan"))
            put_v(s, b, t, slice(None), slice(None), float("nan"))
    marks[1] = [t for t in marks[1] if t > pos[-1] - window]
    fill(0.0)
    plain = decode(torch, yuear_lib, s, window, sinks)
    fill(INF)
    out = decode(torch, yuear_lib, s, window, sinks)
    odd = torch.zeros(batch, kv, heads // kv, 128, dtype=torch.bool, device="cuda")
    odd[:, 0, :, dims] = True
    for b, p in enumerate(pos):
        odd[b, 1, :, dims] = any(t < p for t in marks[1])
    odd = odd.view(batch, heads, 128)
    assert torch.equal(out == INF, odd)
    fill(0.0)
    for b, p in enumerate(pos):
        for t in [35, 63, p - window, p - window - 1]:
            put_k(s, b, t, slice(None), slice(None), 0.0)
            put_v(s, b, t, slice(None), slice(None), 0.0)
    check_decode(torch, s, torch.where(odd, plain, out), window, sinks)


@pytest.mark.parametrize("pos", [[40], [500, 40, 31, 700], [5000]])
def test_decode_weighs_keys_with_an_infinity(torch, yuear_lib, pos):
    """A key whose score is -inf weighs nothing; one of +inf makes its rows NaN."""
    rng = np.random.default_rng(40 + len(pos))
    heads, kv = 6, 2
    s = decode_inputs(torch, yuear_lib, rng, heads, kv, 64, pos, 200)
    for b, p in enumerate(pos):
        x = s["qkv"][b].reshape(-1, 128)
        q, _ = ref.turn(x[:heads], s["gains"][0], s["rope"][0][p], s["rope"][1][p], 1e-5)
        d = int(q.abs().amin(0).argmax())  # no head's query is near zero there
        at = {0: p // 3, 1: p - 1}
        for h, t in at.items():
            put_k(s, b, t, h, d, INF if h else -INF)
        out = decode(torch, yuear_lib, s)[b]
        for h, t in at.items():
            put_k(s, b, t, h, d, 0.0)
        k, v, present = ref.gather(s["pages"].k, s["pages"].v, s["table"][b], p + 1)
        for n in range(heads):
            h = n // (heads // kv)
            if (float(q[n, d]) > 0) == (h == 1):
                assert torch.isnan(out[n]).all(), (b, n)
                continue
            seen = present.copy()
            seen[at[h]] = False
            want, bound = ref.attend(q[n:n + 1], k[h:h + 1], v[h:h + 1], seen, 2.0 ** -16)
            ref.check(out[n:n + 1], want, bound, f"sequence {b}, head {n}")


@pytest.mark.parametrize("width", [8, 256])
@pytest.mark.parametrize("odd", [False, True])
def test_prefill_weighs_keys_with_an_infinity(torch, yuear_lib, width, odd):
    """Keys 0 to 200 have an infinity, so their scores are infinite: rows that see
    -inf scores alone have no softmax (NaN, as for +inf), rows that see others too
    do not count those keys. odd: with an infinite value at the causal edge, too."""
    rng = np.random.default_rng(41)
    heads, kv, n, last = 6, 2, 330, 200
    s = prefill_inputs(torch, rng, heads, kv, 64, [n], [0], 30, width=width)
    for t in range(last + 1):
        put_k(s, 0, t, slice(None), 9, INF)
    s["q"][:, :, 9] = -s["q"][:, :, 9].abs() - 0.125
    up = {5: 1, 210: 4, 300: 2}  # rows of a head whose query has the other sign
    for i, h in up.items():
        s["q"][i, h, 9] *= -1
    if odd:
        put_v(s, 0, 290, 0, 100, INF)
    out = prefill(torch, yuear_lib, s)
    for t in range(last + 1):
        put_k(s, 0, t, slice(None), 9, 0.0)
    if odd:
        put_v(s, 0, 290, 0, 100, 0.0)
        assert (out[290:300, :3, 100] == INF).all() and torch.isfinite(out[201:290, :, 100]).sum() == 89 * 6 - 1
    k, v, present = ref.gather(s["pages"].k, s["pages"].v, s["table"][0], n)
    assert torch.isnan(out[:last + 1]).all()
    for i in [201, 202, 255, 256, 289, 290, n - 1] + [i for i in up if i > last]:
        seen = ref.visible(i, n, 0, 0) & (np.arange(n) > last)
        want, bound = ref.attend(s["q"][i].double(), k, v, seen, ref.HALF)
        bad = up.get(i)
        for h in range(heads):
            if h == bad:
                assert torch.isnan(out[i, h]).all()
                continue
            dims = [d for d in range(128) if not (odd and d == 100 and i >= 290 and h < 3)]
            ref.check(out[i, h, dims], want[h, dims], bound[h, dims], f"row {i}, head {h}")


@pytest.mark.parametrize("width", [6, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3), (1, 64)])
def test_prefill_rows_that_see_no_page_stay_zeros_beside_ones_without_a_softmax(torch, yuear_lib, width, window, sinks):
    rng = np.random.default_rng(42)
    s = prefill_inputs(torch, rng, 3, 1, 64, [200], [40], 30, width=width)
    s["table"][0, 0] = -1              # rows at 40 to 63 see nothing
    for t in range(64, 128):
        put_k(s, 0, t, 0, 3, -INF)
    s["q"][:, :, 3] = s["q"][:, :, 3].abs() + 0.125  # rows at 64 to 127 see scores of -inf alone
    out = prefill(torch, yuear_lib, s, window, sinks)
    assert not out[:24].any() and torch.isnan(out[24:88]).all() and torch.isfinite(out[88:]).all()


# ---- scores far past the fp32 integers ----

@pytest.mark.parametrize("size", [2.0 ** 8, 3.0e7, 1.0e12, 1.0e25])
@pytest.mark.parametrize("width", [5, 128])
@pytest.mark.parametrize("odd", [False, True])
def test_prefill_gives_equal_keys_equal_weights(torch, yuear_lib, size, width, odd):
    """Equal keys in different steps, behind smaller ones, weigh the same whatever
    their score is. Every weight is 1, so what is rounded is the output (half a
    step) and a few fp32 sums."""
    rng = np.random.default_rng(43)
    heads, kv, n, before = 3, 1, 90, 200
    s = prefill_inputs(torch, rng, heads, kv, 64, [n], [before], 20, width=width)
    s["q"][:] = torch.tensor([1.0, 1.171875, 2.96875], device="cuda")[None, :, None]  # of a head, all dims
    s["pages"].k[:] = 0
    small, big = [3, 66, 130], [70, 133, 190, 201, 250]
    for t in small:
        put_k(s, 0, t, 0, slice(None), size * 0.4453125)
    for t in big:
        put_k(s, 0, t, 0, slice(None), size)
    if odd:
        put_v(s, 0, 280, 0, 0, INF)  # of weight 0: a NaN, in this dim of rows that see it
    out = prefill(torch, yuear_lib, s)
    v = ref.gather(s["pages"].k, s["pages"].v, s["table"][0], before + n)[1][0]
    for i in range(0, n, 5):
        at = [t for t in big if t <= before + i]
        want = v[at].mean(0)
        bound = ref.HALF * want.abs() + ref.FINE * v[at].abs().mean(0)
        dims = slice(1, None) if odd else slice(None)
        for h in range(heads):
            ref.check(out[i, h, dims], want[dims], bound[dims], f"row {i}, head {h}")


@pytest.mark.parametrize("size", [2.0 ** 8, 3.0e7, 1.0e12, 1.0e25])
@pytest.mark.parametrize("pos", [[290], [3000, 290]])
def test_decode_gives_equal_keys_equal_weights(torch, yuear_lib, size, pos):
    rng = np.random.default_rng(44)
    heads = kv = 2
    s = decode_inputs(torch, yuear_lib, rng, heads, kv, 64, pos, 100, gain=False)
    s["pages"].k[:] = 0
    s["qkv"].view(len(pos), -1, 128)[:, heads:heads + kv] = 0
    small, big = [3, 66, 130], [70, 133, 190, 201, 250]
    for b, p in enumerate(pos):
        q, _ = ref.turn(s["qkv"][b].view(-1, 128)[:heads], None, s["rope"][0][p], s["rope"][1][p], 1e-5)
        for t in small + big:
            put_k(s, b, t, slice(None), slice(None), q.sign().to(torch.bfloat16) * (size * (0.4453125 if t in small else 1)))
    out = decode(torch, yuear_lib, s)
    for b, p in enumerate(pos):
        v = ref.gather(s["pages"].k, s["pages"].v, s["table"][b], p + 1)[1]
        want = v[:, big].mean(1)
        ref.check(out[b], want, ref.HALF * want.abs() + ref.FINE * v[:, big].abs().mean(1), f"sequence {b}")


# ---- workgroups that walk several items or tiles ----

def decode_on_gpu(torch, yuear_lib, heads, kv, slots, pos, absent, seed):
    """decode_inputs() of many keys: one draw for the whole pool, NaN in slots that
    no token wrote; `absent`: (sequence, page of it) pairs that the table does not have."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    lens = [max(p, 0) + 1 for p in pos]
    n = sum((x + slots - 1) // slots for x in lens) + 3
    s = dict(table=ref.tables(lens, slots, n, rng), pages=ref.Pages(n, kv, slots, "cuda"), pos=list(pos), heads=heads,
             kv=kv, gains=[normal(torch, rng, 128, mean=1.3, std=0.1) for _ in range(2)],
             qkv=normal(torch, rng, len(pos), (heads + 2 * kv) * 128), rope=rope(torch, yuear_lib, max(lens)))
    pages = s["pages"]
    pages.k = torch.randn(pages.k.shape, generator=gen, device="cuda").to(torch.bfloat16)
    pages.v = torch.randn(pages.v.shape, generator=gen, device="cuda").to(torch.bfloat16)
    held = set(s["table"].ravel().tolist()) - {-1}
    loose = [p for p in range(n) if p not in held]
    pages.k[loose], pages.v[loose] = float("nan"), float("nan")
    for b, x in enumerate(lens):  # slots at and past the token's own
        page, slot = int(s["table"][b][(x - 1) // slots]), (x - 1) % slots
        pages.k[page, :, slot:] = float("nan")
        blocks = pages.v[page].transpose(-1, -2).reshape(kv, slots, 128)
        blocks[:, slot:] = float("nan")
        pages.v[page] = blocks.reshape(kv, slots // 32, 32, 128).transpose(-1, -2)
    for b, j in absent:
        s["table"][b, j] = -1
    return s


def check_some(torch, s, out, window, sinks, idle):
    """check_decode() of the sequences that the call has, and the others' rows as they were."""
    live = [b for b, p in enumerate(s["pos"]) if p >= 0]
    assert sorted(set(range(len(s["pos"]))) - set(live)) == sorted(idle)
    assert (out[idle] == 7).all()
    part = dict(s, qkv=s["qkv"][live], table=s["table"][live], pos=[s["pos"][b] for b in live])
    check_decode(torch, part, out[live], window, sinks)


@pytest.mark.parametrize("heads,kv,batch,longest,window,sinks,both", [
    (24, 8, 90, 1500, 0, 0, 50),
    (24, 8, 90, 3000, 700, 37, 60),
    (16, 8, 40, 4000, 0, 0, 200),   # up to 64 sequences, past 24 * 512 blocks
    (6, 1, 200, 3000, 0, 0, 80),
    (8, 1, 300, 1500, 0, 0, 80),
    (4, 2, 300, 400, 0, 0, 20),
])
def test_decode_runs_that_cross_items(torch, yuear_lib, heads, kv, batch, longest, window, sinks, both):
    """Equal runs of blocks whose workgroups end one item and begin the next, over
    sequences, kv heads, absent pages and idle sequences."""
    rng = np.random.default_rng(batch)
    pos = [int(p) for p in np.exp(rng.uniform(0, np.log(longest), batch))]
    pos[batch // 3] = longest
    if batch <= 64 or kv == 1:
        pos = [int(p) for p in rng.uniform(longest / 2 if batch <= 64 else 0, longest, batch)]
    idle = [0, 1, batch // 2, batch - 1]
    for b in idle:
        pos[b] = -1
    absent = [(b, j) for b in range(2, batch - 1, 7) for j in ([0, 2] if pos[b] > 300 else [0])]
    s = decode_on_gpu(torch, yuear_lib, heads, kv, 64, pos, absent, batch + heads)
    ws = marked_workspace(torch, yuear_lib, batch, heads, kv)
    k, v = s["pages"].k.clone(), s["pages"].v.clone()
    out = torch.full((batch, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    decode(torch, yuear_lib, s, window, sinks, workspace=ws, out=out)
    check_some(torch, s, out, window, sinks, idle)
    slots = written_slots(torch, ws, heads // kv)
    assert slots.all(1).sum() >= both and not ws[:COUNTERS].any()
    # nothing but the tokens' own slots changed, and an equal call gives equal bits
    for b, p in enumerate(pos):
        page, slot = (int(s["table"][b][p // 64]), p % 64) if p >= 0 else (-1, 0)
        if page >= 0:
            k[page, :, slot] = s["pages"].k[page, :, slot]
            v[page, :, slot // 32, :, slot % 32] = s["pages"].v[page, :, slot // 32, :, slot % 32]
    assert same_bits(torch, k, s["pages"].k) and same_bits(torch, v, s["pages"].v)
    again = torch.full_like(out, 7.0)
    decode(torch, yuear_lib, s, window, sinks, workspace=ws, out=again)
    assert same_bits(torch, out, again)


@pytest.mark.parametrize("kv,batch,short,longest", [(8, 64, 370, 24570), (16, 32, 370, 12270)])
def test_decode_of_one_long_sequence_among_short_ones(torch, yuear_lib, kv, batch, short, longest):
    """The long one's keys are shared out over many workgroups."""
    pos = [short] * batch
    pos[batch // 2] = longest
    s = decode_on_gpu(torch, yuear_lib, kv, kv, 128, pos, [], 45)
    ws = marked_workspace(torch, yuear_lib, batch, kv, kv)
    out = decode(torch, yuear_lib, s, workspace=ws)
    check_decode(torch, s, out)
    # its heads take at least half of the work and so of the 512 workgroups
    assert written_slots(torch, ws, 1).any(1).sum() >= 200 and not ws[:COUNTERS].any()
    assert same_bits(torch, out, decode(torch, yuear_lib, s, workspace=ws))


@pytest.mark.parametrize("heads,kv,lens,pos0,window,sinks,cross", [
    (24, 8, [400], [3000], 0, 0, 5),
    (24, 8, [200, 0, 700, 33], [2500, 5, 1500, 4000], 0, 0, 5),
    (24, 8, [70, 0, 300, 33], [2500, 5, 0, 4000], 0, 0, 0),  # runs of about a tile's cost
    (12, 6, [500], [2500], 0, 0, 5),
    (16, 8, [400, 1, 300], [1000, 3000, 350], 1500, 33, 5),
    (8, 1, [700, 500], [3000, 1200], 0, 0, 5),
])
@pytest.mark.parametrize("odd", [False, True])
def test_prefill_runs_that_cross_tiles(torch, yuear_lib, heads, kv, lens, pos0, window, sinks, cross, odd):
    """Dealt steps whose workgroups end one tile and begin the next, also of another
    kv head; odd: some of the tiles hold infinite values that some rows see."""
    rng = np.random.default_rng(heads + sum(lens) + odd)
    rows, batch, group = sum(lens), len(lens), heads // kv
    s = prefill_inputs(torch, rng, heads, kv, 64, lens, pos0, 300)
    marks = []  # sequence, key, kv head
    if odd:
        marks = [(b, p + n * i // 7, h) for b, (p, n) in enumerate(zip(pos0, lens)) if n > 30 for i in (1, 3, 6)
                 for h in range(0, kv, 3)]
    for b, t, h in marks:
        put_v(s, b, t, h, slice(0, 128, 9), 0.0)
    clean = prefill(torch, yuear_lib, s, window, sinks)
    check_prefill(torch, s, clean, window, sinks, some=12)
    for b, t, h in marks:
        put_v(s, b, t, h, slice(0, 128, 9), INF)
    ws = marked_workspace(torch, yuear_lib, batch, heads, kv, rows)
    out = prefill(torch, yuear_lib, s, window, sinks, workspace=ws)
    seen = torch.zeros(rows, kv, dtype=torch.bool, device="cuda")
    for b, t, h in marks:
        p = np.arange(pos0[b], pos0[b] + lens[b])
        sees = (t <= p) & ((p - t < window) | (t < sinks) if window else True)
        seen[int(s["starts"][b]):int(s["starts"][b + 1]), h] |= torch.from_numpy(sees).cuda()
    inf = torch.zeros(rows, heads, 128, dtype=torch.bool, device="cuda")
    inf[:, :, ::9] = seen.repeat_interleave(group, 1)[:, :, None]
    assert torch.equal(out == INF, inf)
    for b, t, h in marks:
        put_v(s, b, t, h, slice(0, 128, 9), 0.0)
    check_prefill(torch, s, torch.where(inf, clean, out), window, sinks, some=12)
    for b, t, h in marks:
        put_v(s, b, t, h, slice(0, 128, 9), INF)
    assert same_bits(torch, out, prefill(torch, yuear_lib, s, window, sinks, workspace=ws))
    # the records of the tiles: their first and last run
    tiles = rows * group // 128 + min(batch, rows)
    info = ws[COUNTERS + 1024 * 16640:].cpu().numpy()
    assert info[0] == sum((n * group + 127) // 128 for n in lens)
    held = [set() for _ in range(512)]
    for h in range(kv):
        for i in range(info[0]):
            first, last = info[8 * (1 + h * tiles + i):][:2]
            for run in range(first, last + 1):
                held[run].add((h, i))
    assert sum(len(x) > 1 for x in held) >= cross
    assert kv != 6 or sum(len({h for h, _ in x}) > 1 for x in held) >= 1


def test_prefill_rounds_each_weight_once(torch, yuear_lib):
    """Relative error of a whole call. A bf16 rounding of values with a mantissa m
    of even logarithm leaves 2^-8 sqrt(E[1 / m^2] / 3) = 0.00166 (E = 3 / (8 ln 2));
    values around zero take the outputs' one and the weights', independent of it:
    0.00235 together, and a tenth for how the mantissas fall."""
    rng = np.random.default_rng(46)
    for lens, pos0 in (([97], [1000]), ([600], [0]), ([33, 210], [400, 7])):
        s = prefill_inputs(torch, rng, 24, 8, 64, lens, pos0, 60)
        s["pages"].v = normal(torch, rng, *s["pages"].v.shape)
        out = prefill(torch, yuear_lib, s).double()
        off = total = 0.0
        for b, p0 in enumerate(pos0):
            a, n = int(s["starts"][b]), lens[b]
            k, v, _ = ref.gather(s["pages"].k, s["pages"].v, s["table"][b], p0 + n)
            for i in range(0, n, 5):
                want, _ = ref.attend(s["q"][a + i].double(), k[:, :p0 + i + 1], v[:, :p0 + i + 1], np.ones(p0 + i + 1, bool),
                                     ref.HALF)
                off += float(((out[a + i] - want) ** 2).sum())
                total += float((want ** 2).sum())
        assert (off / total) ** 0.5 <= 1.1 * 0.00235, (lens, (off / total) ** 0.5)


# ---- beside the contiguous operators ----

@pytest.mark.parametrize("heads,kv,n,before", [(24, 8, 130, 0), (24, 8, 1, 400), (16, 8, 77, 200), (8, 1, 33, 479)])
def test_one_page_holds_what_a_contiguous_cache_does(torch, yuear_lib, heads, kv, n, before):
    """A page of 512 slots is the contiguous cache of as many: both operators read
    the same memory."""
    rng = np.random.default_rng(heads + n)
    pages = ref.Pages(1, kv, 512, "cuda")
    pages.k[:], pages.v[:] = 0, 0
    pages.put(np.zeros(1, np.int32), 0, normal(torch, rng, kv, before + n, 128), normal(torch, rng, kv, before + n, 128))
    q = normal(torch, rng, n, heads, 128, std=1.5)
    s = dict(q=q, pages=pages, table=np.zeros((1, 1), np.int32), pos0=[before], starts=np.array([0, n]), heads=heads, kv=kv)
    paged = prefill(torch, yuear_lib, s)
    other = torch.empty_like(paged)
    assert yuear_lib.lib.yuear_op_attention_prefill(q.data_ptr(), pages.k.data_ptr(), pages.v.data_ptr(), n, before, heads,
                                                    kv, 512, other.data_ptr(), None) == 0
    torch.cuda.synchronize()
    check_prefill(torch, s, paged)
    check_prefill(torch, s, other)


@pytest.mark.parametrize("heads,kv,pos", [(24, 8, 0), (24, 8, 400), (16, 8, 95), (8, 1, 511)])
def test_a_step_on_one_page_is_one_on_a_contiguous_cache(torch, yuear_lib, heads, kv, pos):
    """Rotation by nothing, no norm: both take the same queries and keep the same keys."""
    rng = np.random.default_rng(heads + pos)
    one, none = (torch.full((512, 64), x, dtype=torch.bfloat16, device="cuda") for x in (1.0, 0.0))
    s = dict(qkv=normal(torch, rng, 1, (heads + 2 * kv) * 128), pages=ref.Pages(1, kv, 512, "cuda"),
             table=np.zeros((1, 1), np.int32), gains=[None, None], pos=[pos], heads=heads, kv=kv, rope=(one, none))
    if pos:
        s["pages"].put(s["table"][0], 0, normal(torch, rng, kv, pos, 128), normal(torch, rng, kv, pos, 128))
    k, v = s["pages"].k.clone(), s["pages"].v.clone()
    paged = decode(torch, yuear_lib, s)
    other = torch.empty_like(paged)
    assert yuear_lib.lib.yuear_op_attention_decode(
        s["qkv"].data_ptr(), None, None, 1e-5, one.data_ptr(), none.data_ptr(), k.data_ptr(), v.data_ptr(),
        ints(torch, [pos]).data_ptr(), heads, kv, 512, 1, 16, other.data_ptr(), None) == 0
    torch.cuda.synchronize()
    check_decode(torch, s, paged)
    check_decode(torch, s, other)
    assert torch.equal(k.nan_to_num(7), s["pages"].k.nan_to_num(7))
    # (V's slots after the token's in its block are the contiguous operator's own)
    rows = [t[0].transpose(-1, -2).reshape(kv, 512, 128)[:, :pos + 1] for t in (v, s["pages"].v)]
    assert torch.equal(rows[0], rows[1])


def test_a_fork_decodes_into_a_page_of_its_own(torch, yuear_lib):
    """A prompt, a second take of it, and a step of both: the tables are made after
    the pool has given each its room."""
    rng = np.random.default_rng(47)
    heads, kv, slots, n = 6, 2, 32, 45
    pool = yuear_lib.PagePool(10, slots)
    pages = ref.Pages(10, kv, slots, "cuda")
    cos, sin = rope(torch, yuear_lib, 100)
    a = pool.open()
    pool.extend(a, n)
    table = pool.table([a], 3)
    qkv = normal(torch, rng, n, (heads + 2 * kv) * 128)
    yuear_lib.paged_append(qkv, pages.k, pages.v, ints(torch, table), ints(torch, [0, n]), ints(torch, [0]), cos, sin)
    b = pool.fork(a)
    takes = [a, b]
    pos = [pool.length(t) for t in takes]
    for t in takes:
        yuear_lib.pages_copy(pages.k, pages.v, *pool.extend(t, 1))
    both = pool.table(takes, 3)
    assert both[0, 0] == both[1, 0] and both[0, 1] != both[1, 1]
    s = dict(qkv=normal(torch, rng, 2, (heads + 2 * kv) * 128), pages=pages, table=both, gains=[None, None], pos=pos,
             heads=heads, kv=kv, rope=(cos, sin))
    check_decode(torch, s, decode(torch, yuear_lib, s))
    x = s["qkv"].view(2, -1, 128)[:, heads + kv:]
    for t in range(2):  # each take's page has its own token behind the shared prompt
        values = ref.gather(pages.k, pages.v, both[t], n + 1)[1]
        assert torch.equal(values[:, n], x[t].double())
        assert torch.equal(values[:, :n], qkv.view(n, -1, 128)[:, heads + kv:].double().transpose(0, 1))


# ---- calls at once, in place, and through slices ----

def test_calls_on_two_streams_at_once(torch, yuear_lib):
    """Each with a workspace of its own, over one pool: equal bits to one after the other."""
    rng = np.random.default_rng(48)
    heads, kv = 24, 8
    sizes = [([900, 5, 3000, 40], [70, 33], [2500, 400]), ([2000, 2100, 60, 7], [120, 5], [1500, 30])]
    calls = []
    for pos, lens, pos0 in sizes:
        s = decode_inputs(torch, yuear_lib, rng, heads, kv, 64, pos, 150)
        t = prefill_inputs(torch, rng, heads, kv, 64, lens, pos0, 150)
        ws = yuear_lib.paged_workspace(4, heads, kv, sum(lens))
        out = [torch.empty(4, heads, 128, dtype=torch.bfloat16, device="cuda"), torch.empty_like(t["q"])]
        fixed = [ints(torch, x) for x in (s["table"], s["pos"], t["table"], t["starts"], t["pos0"])]
        calls.append((s, t, ws, out, fixed))

    def both(call, stream):
        s, t, ws, out, (table, pos, table2, starts, pos0) = call
        yuear_lib.paged_attention_decode(s["qkv"], s["pages"].k, s["pages"].v, table, pos, *s["rope"], workspace=ws,
                                         out=out[0], stream=stream)
        yuear_lib.paged_attention_prefill(t["q"], t["pages"].k, t["pages"].v, table2, starts, pos0, workspace=ws,
                                          out=out[1], stream=stream)
    want = []
    for call in calls:
        both(call, None)
        want.append([o.clone() for o in call[3]])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for call in calls:
            for o in call[3]:
                o.zero_()
        torch.cuda.synchronize()
        for _ in range(10):
            for call, stream in zip(calls, streams):
                both(call, stream.cuda_stream)
        for stream in streams:
            stream.synchronize()
        for call, w in zip(calls, want):
            assert all(same_bits(torch, a, b) for a, b in zip(call[3], w)) and not call[2][:COUNTERS].any()


def test_two_graphs_take_turns_on_a_workspace(torch, yuear_lib):
    rng = np.random.default_rng(49)
    heads, kv = 16, 8
    ws = yuear_lib.paged_workspace(3, heads, kv, 100)
    s = decode_inputs(torch, yuear_lib, rng, heads, kv, 64, [3000, 50, 700], 100)
    t = prefill_inputs(torch, rng, heads, kv, 64, [60, 9], [2700, 3], 100)
    table, pos = ints(torch, s["table"]), ints(torch, s["pos"])
    table2, starts, pos0 = (ints(torch, t[x]) for x in ("table", "starts", "pos0"))
    out = torch.empty(3, heads, 128, dtype=torch.bfloat16, device="cuda"), torch.empty_like(t["q"])

    def step(w, o):
        yuear_lib.paged_attention_decode(s["qkv"], s["pages"].k, s["pages"].v, table, pos, *s["rope"], workspace=w, out=o)

    def prompt(w, o):
        yuear_lib.paged_attention_prefill(t["q"], t["pages"].k, t["pages"].v, table2, starts, pos0, workspace=w, out=o)
    graphs = []
    for call, o in ((step, out[0]), (prompt, out[1])):
        call(ws, o)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(ws, o)
        graphs.append(g)
    own = yuear_lib.paged_workspace(3, heads, kv, 100)
    for i in range(6):
        s["qkv"].copy_(normal(torch, rng, *s["qkv"].shape))
        t["q"].copy_(normal(torch, rng, *t["q"].shape))
        for g in graphs[::1 - 2 * (i & 1)]:
            g.replay()
        want = [torch.empty_like(o) for o in out]
        step(own, want[0])
        prompt(own, want[1])
        torch.cuda.synchronize()
        assert all(same_bits(torch, a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("batch", [3, 70])
def test_outputs_over_the_inputs(torch, yuear_lib, batch):
    """Queries that the call turns into its output, in the same rows."""
    rng = np.random.default_rng(50)
    heads, kv, slots = 6, 2, 32
    cos, sin = rope(torch, yuear_lib, 3100)
    lens, before = [40 + i % 9 for i in range(batch)], [(500 if batch > 3 else 2900) - i for i in range(batch)]
    rows = sum(lens)
    ends = [n + p + 1 for n, p in zip(lens, before)]
    n = sum((e + slots - 1) // slots for e in ends)
    wide = torch.full((batch, n // batch + 9), -1, dtype=torch.int32)
    table = ref.tables(ends, slots, n, rng)
    wide[:, 3:3 + table.shape[1]] = torch.from_numpy(table)
    table = wide.cuda()[:, 3:3 + table.shape[1]]  # rows of a wider table
    starts, pos0 = ints(torch, np.concatenate([[0], np.cumsum(lens)])), ints(torch, before)
    pos = ints(torch, [p + n_ for p, n_ in zip(before, lens)])
    k = torch.randn(n, kv, slots, 128, device="cuda").to(torch.bfloat16)
    v = torch.randn(n, kv, 1, 128, 32, device="cuda").to(torch.bfloat16)
    qkv, new = normal(torch, rng, rows, (heads + 2 * kv) * 128), normal(torch, rng, batch, (heads + 2 * kv) * 128)
    got = []
    for over in (False, True):
        a, b, k2, v2 = qkv.clone(), new.clone(), k.clone(), v.clone()
        place = a[:, :heads * 128].unflatten(1, (heads, 128)) if over else None
        q = yuear_lib.paged_append(a, k2, v2, table, starts, pos0, cos, sin, out=place)
        y = yuear_lib.paged_attention_prefill(q, k2, v2, table, starts, pos0, out=place)
        place = b[:, :heads * 128].unflatten(1, (heads, 128)) if over else None
        z = yuear_lib.paged_attention_decode(b, k2, v2, table, pos, cos, sin, out=place)
        got.append((y, z, k2, v2))
        assert not over or (torch.equal(a[:, heads * 128:], qkv[:, heads * 128:])
                            and torch.equal(b[:, heads * 128:], new[:, heads * 128:]))
    assert torch.isfinite(got[0][0]).all() and torch.isfinite(got[0][1]).all()
    assert all(torch.equal(x, y) for x, y in zip(*got))
