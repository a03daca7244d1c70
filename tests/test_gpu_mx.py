"""Block-scaled rows on the GPU against their 64-bit definition (mx_ref.py): codes
and scales bit for bit, norms within the reach of 32-bit arithmetic, products
within derived bounds, at the sizes, strides and values where they can go wrong."""
import numpy as np
import pytest

import mx_ref as ref

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def torch():
    import torch as t
    t.cuda.init()
    return t


def bf16(torch, bits):
    return torch.from_numpy(np.ascontiguousarray(bits, np.uint16).view(np.int16)).cuda().view(torch.bfloat16)


def bits_of(torch, t):
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def raw(torch, t):
    return t.view(torch.uint8).cpu().numpy()


def random_rows(rng, rows, k, kind):
    """bf16 bits [rows, k]: "wide" any finite pattern, "near" values within 2^-14 of their block's
    largest, on and beside the codes' midpoints, "plain" normal with channels of unlike size."""
    if kind == "wide":
        return rng.integers(0, 1 << 16, (rows, k), dtype=np.uint16) & np.uint16(0xBFFF)
    if kind == "near":
        e = np.repeat(rng.integers(1, 254, (rows, k // 32)), 32, 1) - rng.integers(0, 15, (rows, k))
        sign = rng.integers(0, 2, (rows, k)) << 15
        mantissa = rng.choice(np.array([0, 1, 7, 8, 9, 24, 31, 32, 33, 40, 56, 64, 72, 95, 96, 97, 100, 127]), (rows, k))
        return (sign | np.maximum(e, 0) << 7 | mantissa).astype(np.uint16)
    return ref.to_bf16(rng.standard_normal((rows, k)) * np.exp(0.8 * rng.standard_normal(k)))


def pair_in(torch, rows, k, bits, gap=0, fill=0x5A):
    """A pair whose rows lie `gap` 16-byte pieces (scales: 4 bytes) apart in wider buffers."""
    wide = torch.full((rows, k * bits // 8 + 16 * gap), fill, dtype=torch.uint8, device="cuda")
    wide_s = torch.full((rows, k // 32 + 4 * gap), fill, dtype=torch.uint8, device="cuda")
    codes, scales = wide[:, :k * bits // 8], wide_s[:, :k // 32]
    if bits == 8:
        codes = codes.view(torch.float8_e4m3fn)
    return (codes, scales.view(torch.float8_e8m0fnu)), (wide, wide_s)


def untouched(wides, k, bits, fill=0x5A):
    return bool((wides[0][:, k * bits // 8:] == fill).all() and (wides[1][:, k // 32:] == fill).all())


def pair_of(torch, stored, scales, bits):
    codes = torch.from_numpy(np.ascontiguousarray(stored)).cuda()
    if bits == 8:
        codes = codes.view(torch.float8_e4m3fn)
    return codes, torch.from_numpy(np.ascontiguousarray(scales)).cuda().view(torch.float8_e8m0fnu)


# ---- quantise, dequantise ----

@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kind", ["wide", "near", "plain"])
@pytest.mark.parametrize("rows,k,gap", [(1, 32, 0), (3, 96, 0), (257, 1056, 1), (1027, 32, 2), (37, 2048, 0), (2, 16384, 0)])
def test_quantize_and_back(torch, yuear_lib, bits, kind, rows, k, gap):
    rng = np.random.default_rng(rows * 31 + k + bits)
    x = random_rows(rng, rows, k, kind)
    t = bf16(torch, x)
    if gap:
        wide = torch.full((rows, k + 8 * gap), 7.0, dtype=torch.bfloat16, device="cuda")
        wide[:, :k] = t
        t = wide[:, :k]
    out, wides = pair_in(torch, rows, k, bits, gap)
    got = yuear_lib.mx_quantize(t, bits, out=out)
    assert got[0].data_ptr() == out[0].data_ptr() and untouched(wides, k, bits)
    codes, scales = ref.quantize(ref.from_bf16(x), bits)
    np.testing.assert_array_equal(raw(torch, got[1].contiguous()), scales)
    np.testing.assert_array_equal(raw(torch, got[0].contiguous()), codes)
    back = torch.full((rows, k + 8 * gap), 9.0, dtype=torch.bfloat16, device="cuda")
    yuear_lib.mx_dequantize(got, out=back[:, :k])
    np.testing.assert_array_equal(bits_of(torch, back[:, :k]), ref.to_bf16(ref.values(codes, scales, bits)))
    assert (back[:, k:] == 9).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_quantize_every_bf16_value(torch, yuear_lib, bits):
    """All finite patterns, each in a block of its own exponent, of one 4 and of one 13 above it; zeros."""
    e = np.arange(255)[:, None, None]
    m = np.arange(128)[None, :, None]
    sign = np.arange(2)[None, None, :] << 15
    v = (sign | e << 7 | m).reshape(255, 256).astype(np.uint16)
    rows = []
    for up in (0, 4, 13):
        top = (np.minimum(np.arange(255) + up, 254) << 7).astype(np.uint16)
        block = np.concatenate([v, np.zeros((255, 23), np.uint16)], 1).reshape(255, 9, 31)  # 31 values and the top
        rows.append(np.concatenate([block, np.broadcast_to(top[:, None, None], (255, 9, 1))], 2).reshape(255, 288))
    x = np.concatenate(rows + [np.zeros((1, 288), np.uint16), np.full((1, 288), 0x8000, np.uint16)])
    got = yuear_lib.mx_quantize(bf16(torch, x), bits)
    codes, scales = ref.quantize(ref.from_bf16(x), bits)
    np.testing.assert_array_equal(raw(torch, got[1]), scales)
    np.testing.assert_array_equal(raw(torch, got[0]), codes)


@pytest.mark.parametrize("bits", [8, 4])
def test_not_finite_blocks(torch, yuear_lib, bits):
    """An infinity or NaN, wherever in its block, makes that block alone NaN."""
    rng = np.random.default_rng(3)
    x = random_rows(rng, 96, 96, "plain")
    for i in range(96):
        x[i, i] = (0x7F80, 0xFF80, 0x7FC0, 0xFFFF, 0x7F81)[i % 5]
    got = yuear_lib.mx_quantize(bf16(torch, x), bits)
    codes, scales = ref.quantize(ref.from_bf16(x), bits)
    assert (scales == 255).sum() == 96
    np.testing.assert_array_equal(raw(torch, got[1]), scales)
    np.testing.assert_array_equal(raw(torch, got[0]), codes)
    back = yuear_lib.mx_dequantize(got)
    np.testing.assert_array_equal(torch.isnan(back).cpu().numpy(), np.repeat(scales == 255, 32, 1))


@pytest.mark.parametrize("bits", [8, 4])
def test_dequantize_every_code_and_scale(torch, yuear_lib, bits):
    codes = np.tile(np.arange(256, dtype=np.uint8), 256 // (2 if bits == 4 else 1)).reshape(-1, 32 * bits // 8)
    codes = np.repeat(codes[:16 if bits == 4 else 8], 256, 0)
    scales = np.tile(np.arange(256, dtype=np.uint8), codes.shape[0] // 256)[:, None]
    got = yuear_lib.mx_dequantize(pair_of(torch, codes, scales, bits))
    want = ref.to_bf16(ref.values(codes, scales, bits))
    g = bits_of(torch, got)
    nan = (want & 0x7FFF) > 0x7F80
    assert ((g & 0x7FFF) > 0x7F80)[nan].all()
    np.testing.assert_array_equal(g[~nan], want[~nan])


# ---- norm ----

# Wider than needed: what y has with all of it in 32 bits, the squares' sum (k / 256 additions in a lane, 8 across) and
# its root, quotient and two products, each half a step of 2^-24 of the value, the sum's halved by the root: under
# (8192 / 256 * 8 + 24) * 2^-25 = 2^-16.9. (The kernel's codes are those of 64 bits: the tests of every code below.)
NORM_FINE = 2.0 ** -16


def check_norm(torch, got, h, gain, bits):
    """codes of y = h / sqrt(mean h^2 + eps) gain, for some y within NORM_FINE of the exact one."""
    y = h / np.sqrt((h ** 2).mean(-1, keepdims=True) + EPS) * gain
    rows, k = y.shape
    scales = raw(torch, got[1].contiguous())
    top = np.abs(y).reshape(rows, -1, 32).max(-1)
    low, high = ref.scale_bytes(top * (1 - NORM_FINE), bits), ref.scale_bytes(top * (1 + NORM_FINE), bits)
    assert ((scales == low) | (scales == high)).all()
    s = np.repeat(ref.power(scales), 32, 1)
    codes = ref.unpack(raw(torch, got[0].contiguous()), bits)
    a = np.abs(y) / s
    low, high = ref.nearest(a * (1 - NORM_FINE), bits), ref.nearest(a * (1 + NORM_FINE), bits)
    magnitude = codes & ((1 << (bits - 1)) - 1)
    assert ((magnitude >= low) & (magnitude <= high)).all()
    assert (magnitude == ref.nearest(a, bits)).mean() > 0.999
    nonzero = y != 0
    assert ((codes >> (bits - 1) != 0) == np.signbit(y))[nonzero].all()


@pytest.mark.parametrize("rows,k,gap,bits,residual", [
    (1, 32, 0, 8, True), (1, 3072, 0, 8, True), (7, 96, 1, 8, True), (5, 512, 0, 4, False), (9, 544, 0, 8, True),
    (3, 2048, 2, 8, False), (4, 2080, 0, 8, True), (3, 4096, 1, 4, True), (2, 4128, 0, 8, True), (3, 8192, 0, 8, True),
    (2, 8224, 0, 8, False), (3, 16384, 0, 8, True), (1030, 64, 0, 8, True), (300, 2048, 0, 8, True),
])
def test_norm(torch, yuear_lib, rows, k, gap, bits, residual):
    rng = np.random.default_rng(rows + k)
    x, r = random_rows(rng, rows, k, "plain"), random_rows(rng, rows, k, "plain")
    gain = ref.to_bf16(1 + 0.2 * rng.standard_normal(k))
    wide = torch.zeros(rows, k + 8 * gap, dtype=torch.bfloat16, device="cuda")
    t = wide[:, :k]
    t.copy_(bf16(torch, x))
    total = torch.full((rows, k + 16), 5.0, dtype=torch.bfloat16, device="cuda")
    out, wides = pair_in(torch, rows, k, bits, gap)
    got, h = yuear_lib.mx_rms_norm(t, bf16(torch, gain), EPS, residual=bf16(torch, r) if residual else None, bits=bits,
                                   out=out, sum_out=total[:, :k] if residual else None)
    want = ref.from_bf16(x)
    if residual:
        want = ref.from_bf16(ref.to_bf16(want + ref.from_bf16(r)))
        np.testing.assert_array_equal(ref.from_bf16(bits_of(torch, h)), want)
        assert (total[:, k:] == 5).all()
    else:
        assert h is None and (total == 5).all()
    assert untouched(wides, k, bits)
    check_norm(torch, got, want, ref.from_bf16(gain), bits)


@pytest.mark.parametrize("rows,k,bits", [(1500, 3072, 8), (1500, 3072, 4), (9000, 256, 8), (300, 16384, 4)])
def test_norm_codes_are_those_of_64_bits(torch, yuear_lib, rows, k, bits):
    """Every code, of millions; a product would have to come within 2^-45 of a tie to differ."""
    rng = np.random.default_rng(rows + bits)
    x, gain = random_rows(rng, rows, k, "plain"), ref.to_bf16(1 + 0.2 * rng.standard_normal(k))
    got, _ = yuear_lib.mx_rms_norm(bf16(torch, x), bf16(torch, gain), EPS, bits=bits)
    h = ref.from_bf16(x)
    codes, scales = ref.quantize(h / np.sqrt((h ** 2).mean(-1, keepdims=True) + EPS) * ref.from_bf16(gain), bits)
    np.testing.assert_array_equal(raw(torch, got[1]), scales)
    np.testing.assert_array_equal(raw(torch, got[0]), codes)


@pytest.mark.parametrize("bits", [8, 4])
def test_norm_ties_where_the_factor_is_exact(torch, yuear_lib, bits):
    """Rows of +-1, +-2, +-0.25 without eps: the products are the gains, ties among them."""
    rng = np.random.default_rng(5)
    k = 2080
    x = np.where(rng.integers(0, 2, (6, k)), 1.0, -1.0) * np.array([1, 2, 0.25, 1, 2.0 ** 20, 2.0 ** -20])[:, None]
    gain = ref.from_bf16(ref.to_bf16(rng.integers(128, 256, k) / 128.0 * 2.0 ** rng.integers(-6, 3, k)))
    gain[::7] = 0
    got, _ = yuear_lib.mx_rms_norm(bf16(torch, ref.to_bf16(x)), bf16(torch, ref.to_bf16(gain)), 0.0, bits=bits)
    codes, scales = ref.quantize(np.sign(x) * gain, bits)
    np.testing.assert_array_equal(raw(torch, got[1]), scales)
    np.testing.assert_array_equal(raw(torch, got[0]), codes)


def test_norm_in_place(torch, yuear_lib):
    """The sum over the residual, and over x, give the same bits as apart."""
    rng = np.random.default_rng(8)
    x, r = (bf16(torch, random_rows(rng, 33, 1024, "plain")) for _ in range(2))
    gain = bf16(torch, ref.to_bf16(1 + 0.1 * rng.standard_normal(1024)))
    want, h = yuear_lib.mx_rms_norm(x, gain, residual=r)
    for over in (0, 1):
        a, b = x.clone(), r.clone()
        got, s = yuear_lib.mx_rms_norm(a, gain, residual=b, sum_out=(a, b)[over])
        assert s.data_ptr() == (a, b)[over].data_ptr() and torch.equal(s, h)
        assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(got, want))


def test_norm_rows_that_are_not_finite(torch, yuear_lib):
    """An infinity or NaN spoils its row alone; a sum that overflows is one; zeros stay zeros."""
    rng = np.random.default_rng(9)
    x, r = random_rows(rng, 6, 256, "plain"), random_rows(rng, 6, 256, "plain")
    x[1, 3], x[2, 200], x[4, 7], r[4, 7] = 0x7F80, 0x7FC0, 0x7F7F, 0x7F7F
    x[5] = r[5] = 0
    gain = bf16(torch, np.full(256, 0x3F80))
    got, h = yuear_lib.mx_rms_norm(bf16(torch, x), gain, residual=bf16(torch, r))
    scales, codes = raw(torch, got[1]), raw(torch, got[0])
    # an infinity's row: inf * 0 in its own block is NaN, the other values are 0
    assert scales[1, 0] == 255 and (codes[1, 32:] & 0x7F == 0).all() and torch.isinf(h[1, 3])
    assert (scales[2] == 255).all() and scales[4, 0] == 255 and torch.isinf(h[4, 7])
    assert not codes[5].any() and not scales[5].any()
    sound = [0, 3]
    check_norm(torch, (got[0][sound], got[1].view(torch.uint8)[sound].view(torch.float8_e8m0fnu)),
               ref.from_bf16(bits_of(torch, h[sound])), np.ones(256), 8)


# ---- product ----

def random_pair(rng, rows, k, bits, kind="codes"):
    """(stored codes, scales) of random codes with scales near 1, or of quantised normal rows."""
    if kind == "codes":
        n = 127 if bits == 8 else 8
        c = rng.integers(0, n, (rows, k)).astype(np.uint8) | (rng.integers(0, 2, (rows, k)) << (bits - 1)).astype(np.uint8)
        return ref.pack(c, bits), rng.integers(121, 132, (rows, k // 32)).astype(np.uint8)
    return ref.quantize(rng.standard_normal((rows, k)) * np.exp(0.8 * rng.standard_normal(k)), bits)


def check_gemm(torch, out, a, w, a_bits, epilogue, r=None):
    y, off = ref.product(a, w, a_bits)
    got = ref.from_bf16(bits_of(torch, out))
    if epilogue == "residual":
        y = y + r
        off = off + 2.0 ** -24 * np.abs(y)
    elif epilogue == "swiglu":
        g, u = y[:, 0::2], y[:, 1::2]
        dg, du = off[:, 0::2], off[:, 1::2]
        sig = 1 / (1 + np.exp(-g))
        y = g * sig * u
        # |d silu| <= 1.1, exp and the quotient 2^-21 of the result (expf within 2 units, at |g| up to 88)
        off = 1.1 * dg * np.abs(u) + (np.abs(g * sig) + 1.1 * dg) * du + 2.0 ** -20 * np.abs(y)
    bound = (1 + ref.HALF_BF16) * off + ref.HALF_BF16 * np.abs(y) + 2.0 ** -133
    err = np.abs(got - y)
    assert (err <= bound).all(), f"{(err > bound).sum()} of {err.size} off, worst {np.nanmax(err / bound):.3g}"


GEMMS = [
    (1, 1, 128, 8, "store"), (1, 16, 128, 4, "store"), (1, 256, 1024, 8, "store"), (2, 50, 384, 8, "swiglu"),
    (5, 33, 640, 4, "residual"), (8, 512, 512, 8, "swiglu"), (15, 17, 256, 8, "residual"), (16, 96, 896, 4, "swiglu"),
    (17, 130, 128, 8, "store"), (31, 64, 1152, 8, "residual"), (32, 258, 256, 4, "store"), (33, 100, 512, 8, "swiglu"),
    (48, 16, 2048, 8, "store"), (64, 192, 384, 8, "residual"), (65, 66, 768, 4, "swiglu"), (97, 301, 512, 8, "store"),
    (128, 128, 256, 8, "swiglu"), (130, 257, 640, 4, "residual"), (197, 384, 1024, 8, "residual"),
    (255, 510, 128, 8, "store"), (257, 514, 384, 8, "swiglu"), (300, 700, 256, 4, "store"), (513, 258, 128, 8, "residual"),
    (1, 3, 8192, 8, "store"), (600, 130, 512, 4, "swiglu"), (1030, 520, 256, 8, "store"),
]


@pytest.mark.parametrize("m,n,k,bits,epilogue", GEMMS)
@pytest.mark.parametrize("kind", ["codes", "quantised"])
def test_gemm(torch, yuear_lib, m, n, k, bits, epilogue, kind):
    rng = np.random.default_rng(m * 7 + n + k)
    a, w = random_pair(rng, m, k, bits, kind), random_pair(rng, n, k, 4, kind)
    width = n // 2 if epilogue == "swiglu" else n
    wide = torch.full((m + 1, width + 3), 3.0, dtype=torch.bfloat16, device="cuda")
    r = ref.to_bf16(4 * rng.standard_normal((m, n))) if epilogue == "residual" else None
    out = yuear_lib.mx_gemm(pair_of(torch, *a, bits), pair_of(torch, *w, 4), swiglu=epilogue == "swiglu",
                            residual=bf16(torch, r) if r is not None else None, out=wide[:m, :width])
    assert out.data_ptr() == wide.data_ptr() and (wide[m:] == 3).all() and (wide[:, width:] == 3).all()
    check_gemm(torch, out, ref.values(*a, bits), ref.values(*w, 4), bits, epilogue,
               ref.from_bf16(r) if r is not None else None)


def forced(torch, yuear_lib, form, a, w, a_bits, out, residual=None, swiglu=False, expect=0):
    (ac, asc), (wc, wsc) = a, w
    status = yuear_lib.lib.yuear_op_mx_gemm_form(
        ac.data_ptr(), ac.stride(0), asc.data_ptr(), asc.stride(0), a_bits, wc.data_ptr(), wc.stride(0),
        wsc.data_ptr(), wsc.stride(0), ac.shape[0], wc.shape[0], asc.shape[1] * 32,
        residual.data_ptr() if residual is not None else None, residual.stride(0) if residual is not None else 0,
        out.data_ptr(), out.stride(0), int(swiglu), form, torch.cuda.current_stream().cuda_stream)
    assert status == expect


# tokens, features, K: one and two rounds of a ring, odd numbers of 128s and of 512s, tiles with one
# row or column; each workgroup has one tile (test_tiles_one_after_another has more of them)
FORMS = [(1, 2, 128), (5, 40, 384), (16, 66, 640), (33, 34, 1152), (65, 130, 512), (130, 62, 1664), (257, 300, 896),
         (40, 514, 2304), (300, 130, 4224)]


@pytest.mark.parametrize("form", range(8))
@pytest.mark.parametrize("m,n,k", FORMS)
@pytest.mark.parametrize("bits", [8, 4])
def test_every_form(torch, yuear_lib, form, m, n, k, bits):
    """Each form at any shape, stored rows and their surroundings, with each epilogue in turn."""
    rng = np.random.default_rng(form + m + k)
    a, w = random_pair(rng, m, k, bits), random_pair(rng, n, k, 4)
    va, vw = ref.values(*a, bits), ref.values(*w, 4)
    pa, pw = pair_of(torch, *a, bits), pair_of(torch, *w, 4)
    r = ref.to_bf16(4 * rng.standard_normal((m, n)))
    for epilogue, pad in (("store", 8), ("swiglu", 0), ("residual", 3)):
        width = n // 2 if epilogue == "swiglu" else n
        wide = torch.full((m + 2, width + pad), 3.0, dtype=torch.bfloat16, device="cuda")
        forced(torch, yuear_lib, form, pa, pw, bits, wide[:m, :width], bf16(torch, r) if epilogue == "residual" else None,
               epilogue == "swiglu")
        assert (wide[m:] == 3).all() and (wide[:, width:] == 3).all()
        check_gemm(torch, wide[:m, :width], va, vw, bits, epilogue, ref.from_bf16(r) if epilogue == "residual" else None)


@pytest.mark.parametrize("bits,k", [(8, 640), (8, 1024), (4, 768), (4, 896), (4, 1024)])
@pytest.mark.parametrize("epilogue", ["store", "swiglu", "residual"])
def test_tiles_one_after_another(torch, yuear_lib, bits, k, epilogue):
    """More tiles of 256 x 256 and 192 x 192 than CUs: the ring runs on into the next tile (ragged last
    ones), the same bits as the tiles of 128 x 128, whose sums have the same order."""
    rng = np.random.default_rng(k)
    m, n = 300, 35002
    a, w = pair_of(torch, *random_pair(rng, m, k, bits), bits), pair_of(torch, *random_pair(rng, n, k, 4), 4)
    width = n // 2 if epilogue == "swiglu" else n
    r = bf16(torch, ref.to_bf16(rng.standard_normal((m, n)))) if epilogue == "residual" else None
    outs = []
    for form in (7, 6, 5):
        for ld in (width, width + (-width) % 8 + 8):
            out = torch.full((m, ld), 7.0, dtype=torch.bfloat16, device="cuda")[:, :width]
            forced(torch, yuear_lib, form, a, w, bits, out, r, epilogue == "swiglu")
            outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    rows = [0, 1, 255, 256, 299]
    check_gemm(torch, outs[0][rows][:, :2000], ref.values(raw(torch, a[0])[rows], raw(torch, a[1])[rows], bits),
               ref.values(raw(torch, w[0])[:2000 * n // width], raw(torch, w[1])[:2000 * n // width], 4), bits, epilogue,
               ref.from_bf16(bits_of(torch, r))[rows][:, :2000] if r is not None else None)


@pytest.mark.parametrize("form", [8, 9])
@pytest.mark.parametrize("m,n,k,bits", [(1, 2, 128, 8), (5, 40, 384, 4), (16, 66, 640, 8), (3, 20002, 1152, 8),
                                        (7, 70034, 640, 4), (15, 9000, 512, 8), (2, 16390, 4096, 4)])
@pytest.mark.parametrize("epilogue", ["store", "swiglu", "residual"])
def test_streamed_rows(torch, yuear_lib, form, m, n, k, bits, epilogue):
    """Features one workgroup after another: the sums of the rows form (0), whose order is the same."""
    rng = np.random.default_rng(n)
    a, w = pair_of(torch, *random_pair(rng, m, k, bits), bits), pair_of(torch, *random_pair(rng, n, k, 4), 4)
    width = n // 2 if epilogue == "swiglu" else n
    r = bf16(torch, ref.to_bf16(rng.standard_normal((m, n)))) if epilogue == "residual" else None
    wide = torch.full((m + 1, width + 5), 3.0, dtype=torch.bfloat16, device="cuda")
    want = torch.empty(m, width, dtype=torch.bfloat16, device="cuda")
    if (form, k) == (9, 4096):  # two buffers of 32 rows for eight waves do not fit a CU's LDS
        forced(torch, yuear_lib, form, a, w, bits, wide[:m, :width], r, epilogue == "swiglu", expect=1)
        return
    forced(torch, yuear_lib, form, a, w, bits, wide[:m, :width], r, epilogue == "swiglu")
    forced(torch, yuear_lib, 0, a, w, bits, want, r, epilogue == "swiglu")
    assert torch.equal(wide[:m, :width], want) and (wide[m:] == 3).all() and (wide[:, width:] == 3).all()


@pytest.mark.parametrize("form", [8, 9])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("epilogue", ["store", "swiglu", "residual"])
def test_streamed_weights_past_the_cache(torch, yuear_lib, form, bits, epilogue):
    """More than 64 MiB of weights: the same bits as by form 0, whose last columns are checked."""
    rng = np.random.default_rng(31)
    m, n, k = 3, 140_002, 1024
    a, rows = random_pair(rng, m, k, bits), random_pair(rng, 1009, k, 4)
    w = tuple(t.view(torch.uint8)[torch.arange(n, device="cuda") * 7 % 1009] for t in pair_of(torch, *rows, 4))
    w = (w[0], w[1].view(torch.float8_e8m0fnu))
    width = n // 2 if epilogue == "swiglu" else n
    r = bf16(torch, ref.to_bf16(rng.standard_normal((m, width)))) if epilogue == "residual" else None
    out, want = (torch.empty(m, width, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    forced(torch, yuear_lib, form, pair_of(torch, *a, bits), w, bits, out, r, epilogue == "swiglu")
    forced(torch, yuear_lib, 0, pair_of(torch, *a, bits), w, bits, want, r, epilogue == "swiglu")
    assert torch.equal(out, want)
    last = 202
    at = width - (last // 2 if epilogue == "swiglu" else last)
    check_gemm(torch, want[:, at:], ref.values(*a, bits),
               ref.values(raw(torch, w[0][-last:]), raw(torch, w[1].view(torch.uint8)[-last:]), 4), bits, epilogue,
               ref.from_bf16(bits_of(torch, r[:, at:])) if r is not None else None)


@pytest.mark.parametrize("m,n,k,bits", [(3, 40, 256, 8), (70, 140, 384, 4), (300, 300, 256, 8)])
def test_gemm_rows_apart(torch, yuear_lib, m, n, k, bits):
    """Operands that are columns of wider buffers; what lies between their rows is NaN."""
    rng = np.random.default_rng(k)
    a, w = random_pair(rng, m, k, bits), random_pair(rng, n, k, 4)
    pairs = []
    for (codes, scales), b in ((a, bits), (w, 4)):
        p, _ = pair_in(torch, codes.shape[0], k, b, 3, fill=0xFF)
        p[0].view(torch.uint8).copy_(torch.from_numpy(codes))
        p[1].view(torch.uint8).copy_(torch.from_numpy(scales))
        pairs.append(p)
    out = yuear_lib.mx_gemm(*pairs)
    check_gemm(torch, out, ref.values(*a, bits), ref.values(*w, 4), bits, "store")
    same = yuear_lib.mx_gemm(pair_of(torch, *a, bits), pair_of(torch, *w, 4))
    assert torch.equal(out, same)
    for form in range(8):
        forced(torch, yuear_lib, form, *pairs, bits, out)
        check_gemm(torch, out, ref.values(*a, bits), ref.values(*w, 4), bits, "store")


@pytest.mark.parametrize("m,n,form", [(1, 38, 0), (9, 70, 1), (9, 70, 8), (16, 102, 9), (33, 71, 2), (65, 133, 3), (66, 262, 4),
                                      (130, 263, 5), (200, 390, 6), (261, 519, 7)])
@pytest.mark.parametrize("epilogue", ["store", "swiglu", "residual"])
@pytest.mark.parametrize("at,more", [(1, 2), (2, 1), (3, 5), (4, 4)])
def test_outputs_at_any_even_address(torch, yuear_lib, m, n, form, epilogue, at, more):
    """Outputs and residuals that are columns of wider arrays of odd and even widths."""
    if epilogue == "swiglu":
        n -= n % 2
    rng = np.random.default_rng(n + at)
    a, w = random_pair(rng, m, 384, 8), random_pair(rng, n, 384, 4)
    width = n // 2 if epilogue == "swiglu" else n
    wide = torch.full((m + 1, at + width + more), 3.0, dtype=torch.bfloat16, device="cuda")
    r = rng.standard_normal((m, width))
    resid = torch.full((m, width + 3 + at), float("nan"), dtype=torch.bfloat16, device="cuda")
    r = resid[:, 3:3 + width].copy_(torch.from_numpy(r))
    out = wide[:m, at:at + width]
    forced(torch, yuear_lib, form, pair_of(torch, *a, 8), pair_of(torch, *w, 4), 8, out,
           r if epilogue == "residual" else None, epilogue == "swiglu")
    check_gemm(torch, out, ref.values(*a, 8), ref.values(*w, 4), 8, epilogue, ref.from_bf16(bits_of(torch, r)))
    assert (wide[m:] == 3).all() and (wide[:, :at] == 3).all() and (wide[:, at + width:] == 3).all()


@pytest.mark.parametrize("m,form", [(3, 0), (3, 1), (3, 8), (3, 9), (40, 2), (40, 3), (40, 4), (300, 5), (300, 6), (300, 7)])
def test_gemm_not_finite(torch, yuear_lib, m, form):
    """NaN scales and NaN codes reach their rows and columns, nothing else. Sums past 2^128 are not finite:
    infinities, or NaN where partial sums of either sign overflow."""
    rng = np.random.default_rng(m)
    n, k = 50, 512
    a, w = random_pair(rng, m, k, 8), random_pair(rng, n, k, 4)
    a[0][1, 100] = 0x7F
    a[1][2, 15] = 255
    w[1][7, 3] = 255
    a[1][0], w[1][9] = 200, 200  # 2^73 each
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    forced(torch, yuear_lib, form, pair_of(torch, *a, 8), pair_of(torch, *w, 4), 8, out)
    nan = torch.isnan(out).cpu().numpy()
    want = np.zeros((m, n), bool)
    want[1], want[2], want[:, 7] = True, True, True
    assert not torch.isfinite(out[0, 9])
    nan[0, 9] = False
    np.testing.assert_array_equal(nan, want)
    fine = np.ones((m, n), bool)
    fine[0], fine[:, 9], fine[want] = False, False, False
    rows, cols = [i for i in range(m) if i > 2], [j for j in range(n) if j not in (7, 9)]
    if rows:
        y, off = ref.product(ref.values(a[0][rows], a[1][rows], 8), ref.values(w[0][cols], w[1][cols], 4), 8)
        got = ref.from_bf16(bits_of(torch, out))[np.ix_(rows, cols)]
        assert (np.abs(got - y) <= ref.HALF_BF16 * np.abs(y) + (1 + ref.HALF_BF16) * off).all()


@pytest.mark.parametrize("m", [1, 9, 70, 300])
@pytest.mark.parametrize("bits", [8, 4])
def test_swiglu_at_far_gates(torch, yuear_lib, m, bits):
    """Gates down to where e^-gate leaves 32 bits, and up; the sums are one product each, exact."""
    gates = np.array([-104, -96, -88, -80, -64, -40, -16, -2, 0, 1, 12, 80, 96, 104]) if bits == 8 else np.array(
        [-96, -64, -48, -24, -4, -1, 0, 2, 32, 96])
    x = np.zeros((m, 128))
    x[:, 0] = np.resize(gates, m)
    x[:, 32] = 1
    w = np.zeros((64, 128))
    w[0::2, 0], w[1::2, 32] = 1, np.resize(2.0 ** np.arange(-12, 20, 3), 32)
    a, w = yuear_lib.mx_quantize(bf16(torch, ref.to_bf16(x)), bits), yuear_lib.mx_quantize(bf16(torch, ref.to_bf16(w)), 4)
    got = ref.from_bf16(bits_of(torch, yuear_lib.mx_gemm(a, w, swiglu=True)))
    g = x[:, :1]
    want = g / (1 + np.exp(-g)) * ref.values(raw(torch, w[0]), raw(torch, w[1].view(torch.uint8)), 4)[1::2, 32]
    # of the result: the argument's roundings, exp2's, the reciprocal's and five more of 32 bits, then bf16's
    near = np.abs(got - want) <= np.abs(want) * (np.abs(g) * 7.4e-8 + 9 * 2.0 ** -24 + ref.HALF_BF16) * (1 + 2.0 ** -8) + 2.0 ** -134
    lost = g < -88.7  # e^-gate is infinite in 32 bits
    assert (near | (lost & (got == 0))).all()


def test_gemm_into_its_residual(torch, yuear_lib):
    rng = np.random.default_rng(4)
    for m in (2, 90, 400):
        a, w = pair_of(torch, *random_pair(rng, m, 256, 8), 8), pair_of(torch, *random_pair(rng, 200, 256, 4), 4)
        r = bf16(torch, ref.to_bf16(rng.standard_normal((m, 200))))
        want = yuear_lib.mx_gemm(a, w, residual=r)
        got = yuear_lib.mx_gemm(a, w, residual=r, out=r)
        assert got is r and torch.equal(got, want)


def test_refused_on_the_gpu(torch, yuear_lib):
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    a, w = yuear_lib.mx_quantize(x), yuear_lib.mx_quantize(x, 4)
    other = yuear_lib.mx_quantize(torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda"), 4)
    for call in (
            lambda: yuear_lib.mx_quantize(x.float()), lambda: yuear_lib.mx_quantize(x, 6),
            lambda: yuear_lib.mx_quantize(x[:, :40]), lambda: yuear_lib.mx_quantize(x.T),
            lambda: yuear_lib.mx_quantize(x[:, 4:100]), lambda: yuear_lib.mx_quantize(x, 4, out=a),
            lambda: yuear_lib.mx_dequantize((a[0], a[1][:2])), lambda: yuear_lib.mx_dequantize((x, a[1])),
            lambda: yuear_lib.mx_dequantize(a, out=x.float()), lambda: yuear_lib.mx_rms_norm(x, x[0, :64]),
            lambda: yuear_lib.mx_rms_norm(x, x[0], sum_out=x), lambda: yuear_lib.mx_rms_norm(x, x[0], residual=x[:2]),
            lambda: yuear_lib.mx_gemm(a, a), lambda: yuear_lib.mx_gemm(a, other), lambda: yuear_lib.mx_gemm(x, w),
            lambda: yuear_lib.mx_gemm(a, w, residual=x), lambda: yuear_lib.mx_gemm(a, w, swiglu=True, residual=x),
            lambda: yuear_lib.mx_gemm((a[0][:, :32], a[1][:, :1]), (w[0][:, :16], w[1][:, :1])),
            lambda: yuear_lib.mx_quantize(x, stream=torch.cuda.Stream().cuda_stream),
    ):
        with pytest.raises((ValueError, TypeError)):
            call()


def test_rows_past_32_bits_of_values_are_refused(torch, yuear_lib):
    """k of 2^32 + 32 is not taken for 32."""
    k = 2 ** 32 + 32
    x = torch.empty(1, k, dtype=torch.bfloat16, device="cuda")
    pair = (x.view(torch.uint8)[:, :k].view(torch.float8_e4m3fn), x.view(torch.uint8)[:, :k // 32].view(torch.float8_e8m0fnu))
    small = pair_of(torch, *random_pair(np.random.default_rng(1), 2, 128, 4), 4)
    for call in (lambda: yuear_lib.mx_quantize(x), lambda: yuear_lib.mx_dequantize(pair),
                 lambda: yuear_lib.mx_rms_norm(x, x[0]), lambda: yuear_lib.mx_gemm(pair, small)):
        with pytest.raises(ValueError):
            call()


def test_empty(torch, yuear_lib):
    x = torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda")
    gain = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    a = yuear_lib.mx_quantize(x)
    w = yuear_lib.mx_quantize(torch.zeros(6, 128, dtype=torch.bfloat16, device="cuda"), 4)
    assert yuear_lib.mx_dequantize(a).shape == (0, 128) and yuear_lib.mx_gemm(a, w).shape == (0, 6)
    assert yuear_lib.mx_rms_norm(x, gain, residual=x)[1].shape == (0, 128)
    some = yuear_lib.mx_quantize(torch.ones(3, 128, dtype=torch.bfloat16, device="cuda"))
    assert yuear_lib.mx_gemm(some, (w[0][:0], w[1][:0])).shape == (3, 0)


def test_rows_past_32_bits(torch, yuear_lib):
    """More than 2^31 chunks of 8 values, 2^35 bytes: the last rows' codes, norm, values and products."""
    rng = np.random.default_rng(21)
    rows, k, n = 2_200_000, 8192, 24
    tail = random_rows(rng, 40, k, "plain")
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-40:] = bf16(torch, tail)
    codes, scales = ref.quantize(ref.from_bf16(tail), 8)
    a = yuear_lib.mx_quantize(x)
    assert a[0].numel() > 2 ** 34
    np.testing.assert_array_equal(raw(torch, a[0][-40:]), codes)
    np.testing.assert_array_equal(raw(torch, a[1].view(torch.uint8)[-40:]), scales)
    assert not a[0].view(torch.uint8)[:-40].any()
    w = random_pair(rng, n, k, 4)
    out = yuear_lib.mx_gemm(a, pair_of(torch, *w, 4))
    assert not out[:-40].any()
    check_gemm(torch, out[-40:], ref.values(codes, scales, 8), ref.values(*w, 4), 8, "store")
    back = yuear_lib.mx_dequantize(a, out=x)
    np.testing.assert_array_equal(bits_of(torch, back[-40:]), ref.to_bf16(ref.values(codes, scales, 8)))
    x[-40:] = bf16(torch, tail)
    got, _ = yuear_lib.mx_rms_norm(x, torch.ones(k, dtype=torch.bfloat16, device="cuda"), EPS, out=a)
    check_norm(torch, (got[0][-40:], got[1].view(torch.uint8)[-40:].view(torch.float8_e8m0fnu)), ref.from_bf16(tail),
               np.ones(k), 8)
    assert not got[0].view(torch.uint8)[:-40].any()


def test_outputs_past_32_bits(torch, yuear_lib):
    """A product of more than 2^31 values, each form's last rows and columns."""
    rng = np.random.default_rng(22)
    m, n, k = 40_000, 65_600, 128
    a, w = pair_of(torch, *random_pair(rng, m, k, 8), 8), pair_of(torch, *random_pair(rng, n, k, 4), 4)
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    rows, cols = slice(m - 300, m), slice(n - 300, n)
    va = ref.values(raw(torch, a[0][rows]), raw(torch, a[1].view(torch.uint8)[rows]), 8)
    vw = ref.values(raw(torch, w[0][cols]), raw(torch, w[1].view(torch.uint8)[cols]), 4)
    for form in (-1, 2, 4, 5, 6, 7):
        out[rows].zero_()
        forced(torch, yuear_lib, form, a, w, 8, out)
        check_gemm(torch, out[rows, cols], va, vw, 8, "store")


# ---- together ----

def mlp(yuear_lib, x, stream, gain, w_up, w_down, **kw):
    """A decoder layer's second half: norm of the sum, gate/up, down into the residual stream."""
    a, h = yuear_lib.mx_rms_norm(x, gain, EPS, residual=stream)
    y = yuear_lib.mx_gemm(a, w_up, swiglu=True)
    return yuear_lib.mx_gemm(yuear_lib.mx_quantize(y), w_down, residual=h)


def mlp_inputs(torch, rng, m, h=512, f=1024):
    x, stream = (bf16(torch, random_rows(rng, m, h, "plain")) for _ in range(2))
    gain = bf16(torch, ref.to_bf16(1 + 0.1 * rng.standard_normal(h)))
    up = bf16(torch, ref.to_bf16(0.04 * rng.standard_normal((2 * f, h))))
    down = bf16(torch, ref.to_bf16(0.04 * rng.standard_normal((h, f))))
    return x, stream, gain, up, down


@pytest.mark.parametrize("m", [1, 8, 70, 300])
def test_mlp_together(torch, yuear_lib, m):
    """The run of operators against the same steps in 64 bits, each from the one before as it was stored."""
    rng = np.random.default_rng(m)
    x, stream, gain, up, down = mlp_inputs(torch, rng, m)
    w_up, w_down = yuear_lib.mx_quantize(up, 4), yuear_lib.mx_quantize(down, 4)
    a, h = yuear_lib.mx_rms_norm(x, gain, EPS, residual=stream)
    want_h = ref.from_bf16(ref.to_bf16(ref.from_bf16(bits_of(torch, x)) + ref.from_bf16(bits_of(torch, stream))))
    np.testing.assert_array_equal(ref.from_bf16(bits_of(torch, h)), want_h)
    check_norm(torch, a, want_h, ref.from_bf16(bits_of(torch, gain)), 8)

    def held(pair, bits):
        return ref.values(raw(torch, pair[0]), raw(torch, pair[1]), bits)

    y = yuear_lib.mx_gemm(a, w_up, swiglu=True)
    check_gemm(torch, y, held(a, 8), held(w_up, 4), 8, "swiglu")
    q = yuear_lib.mx_quantize(y)
    codes, scales = ref.quantize(ref.from_bf16(bits_of(torch, y)), 8)
    np.testing.assert_array_equal(raw(torch, q[0]), codes)
    np.testing.assert_array_equal(raw(torch, q[1]), scales)
    out = yuear_lib.mx_gemm(q, w_down, residual=h)
    check_gemm(torch, out, held(q, 8), held(w_down, 4), 8, "residual", want_h)
    assert torch.equal(out, mlp(yuear_lib, x, stream, gain, w_up, w_down))


@pytest.mark.parametrize("m", [2, 200])
def test_captured_and_replayed(torch, yuear_lib, m):
    """A captured run of them, replayed with eager work and other inputs between, gives the eager bits."""
    rng = np.random.default_rng(11)
    x, stream, gain, up, down = mlp_inputs(torch, rng, m)
    w_up, w_down = yuear_lib.mx_quantize(up, 4), yuear_lib.mx_quantize(down, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mlp(yuear_lib, x, stream, gain, w_up, w_down)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(yuear_lib, x, stream, gain, w_up, w_down)
    for i in range(4):
        x.copy_(bf16(torch, random_rows(rng, m, 512, "plain")))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mlp(yuear_lib, x, stream, gain, w_up, w_down))


def test_two_streams_and_given_outputs(torch, yuear_lib):
    """Calls on a given stream with given outputs, two streams at once, against calls in order."""
    rng = np.random.default_rng(12)
    streams = [torch.cuda.Stream() for _ in range(2)]
    w = yuear_lib.mx_quantize(bf16(torch, ref.to_bf16(rng.standard_normal((640, 512)))), 4)
    gain = bf16(torch, np.full(512, 0x3F80))
    rows = [bf16(torch, random_rows(rng, m, 512, "plain")) for m in (9, 150)]
    want = [yuear_lib.mx_gemm(yuear_lib.mx_rms_norm(x, gain)[0], w) for x in rows]
    outs = [(yuear_lib.mx_quantize(x), torch.empty(x.shape[0], 640, dtype=torch.bfloat16, device="cuda")) for x in rows]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, x, (pair, out) in zip(streams, rows, outs):
            yuear_lib.mx_rms_norm(x, gain, out=pair, stream=st.cuda_stream)
            yuear_lib.mx_gemm(pair, w, out=out, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(out, y) for (_, out), y in zip(outs, want))


def test_equal_calls_give_equal_bits(torch, yuear_lib):
    rng = np.random.default_rng(13)
    w = pair_of(torch, *random_pair(rng, 1000, 1024, 4), 4)
    for m in (1, 20, 100, 500):
        a = pair_of(torch, *random_pair(rng, m, 1024, 8), 8)
        first = yuear_lib.mx_gemm(a, w)
        assert all(torch.equal(first, yuear_lib.mx_gemm(a, w)) for _ in range(3))
