"""Paged cache operators on the GPU where their plans and their arithmetic meet an
edge. Bounds are paged_ref.py's."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import (check_decode, decode, decode_inputs, normal, prefill, prefill_inputs, rope, same_bits,
                            torch)  # noqa: F401 (torch: the fixture)

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
def test_prefill_rows_that_see_no_page_stay_zeros_beside_ones_without_a_softmax(torch, yuear_lib, width):
    rng = np.random.default_rng(42)
    s = prefill_inputs(torch, rng, 3, 1, 64, [200], [40], 30, width=width)
    s["table"][0, 0] = -1              # rows at 40 to 63 see nothing
    for t in range(64, 128):
        put_k(s, 0, t, 0, 3, -INF)
    s["q"][:, :, 3] = s["q"][:, :, 3].abs() + 0.125  # rows at 64 to 127 see scores of -inf alone
    out = prefill(torch, yuear_lib, s)
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
