"""Block-scaled rows on the GPU where rounding, range or order meet an edge: norms whose
values lie on the middle of two codes or on a power of two, values past 32 bits, gates
whose exponential leaves 32 bits, and tiles that a workgroup takes after its first."""
import numpy as np
import pytest

import mx_ref as ref
from test_gpu_mx import (bf16, bits_of, forced, pair_in, pair_of, random_pair, random_rows, raw,
                         torch, untouched)  # noqa: F401 (torch: the fixture)

pytestmark = pytest.mark.gpu


def check_codes(torch, got, y, bits):
    """The codes and scales of y in 64 bits, each of them."""
    codes, scales = ref.quantize(y, bits)
    np.testing.assert_array_equal(raw(torch, got[1].contiguous()), scales)
    np.testing.assert_array_equal(raw(torch, got[0].contiguous()), codes)


def tied_gains(rng, k):
    """Gains of which one in sixteen is the middle of two codes, some of them powers of two, some zeros."""
    gain = rng.integers(128, 256, k) / 128.0 * 2.0 ** rng.integers(-6, 3, k)
    gain[5::11] = 2.0 ** rng.integers(-6, 3, gain[5::11].size)
    gain[::7] = 0
    return gain


# ---- norm ----

@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("k", [1568, 2080, 3136, 3296, 5152])
def test_norm_of_a_mean_that_is_exact(torch, yuear_lib, k, bits):
    """Rows of +-1, +-2, +-0.25: their mean is exact, whatever k is, and the products are the gains."""
    rng = np.random.default_rng(k)
    x = np.where(rng.integers(0, 2, (4, k)), 1.0, -1.0)
    gain = tied_gains(rng, k)
    got, _ = yuear_lib.mx_rms_norm(bf16(torch, ref.to_bf16(x * np.array([[1], [2], [0.25], [1]]))),
                                   bf16(torch, ref.to_bf16(gain)), 0.0, bits=bits)
    check_codes(torch, got, x * gain, bits)


# Rows of one magnitude: their root is that magnitude, its reciprocal no float, and y is sign * gain.
# The last row's eps adds to a square: sqrt(2 * 2 + 2.25) is 2.5.
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("k,residual", [(1024, False), (2080, True), (3072, False), (3136, True), (16384, False)])
@pytest.mark.parametrize("magnitude,eps", [(3, 0.0), (1.5, 0.0), (7 * 2.0 ** 20, 0.0), (0.625, 0.0), (100, 0.0), (2, 2.25)])
def test_norm_ties_where_the_factor_is_not_exact(torch, yuear_lib, k, residual, magnitude, eps, bits):
    rng = np.random.default_rng(k)
    x = np.where(rng.integers(0, 2, (5, k)), 1.0, -1.0)
    root = np.sqrt(magnitude ** 2 + eps)
    gain = tied_gains(rng, k) * (1.25 if eps else 1.0)  # 2 * 1.25 / 2.5 = 1
    gain = ref.from_bf16(ref.to_bf16(gain))
    h = x * magnitude
    part = np.where(rng.integers(0, 2, (5, k)), 0.25 * magnitude, -magnitude) if residual else 0 * h
    got, total = yuear_lib.mx_rms_norm(bf16(torch, ref.to_bf16(h - part)), bf16(torch, ref.to_bf16(gain)), eps,
                                       residual=bf16(torch, ref.to_bf16(part)) if residual else None, bits=bits)
    if residual:
        np.testing.assert_array_equal(ref.from_bf16(bits_of(torch, total)), h)
    check_codes(torch, got, h * gain / root, bits)  # exact wherever it is a tie


@pytest.mark.parametrize("bits", [8, 4])
def test_norm_of_one_value_in_nine(torch, yuear_lib, bits):
    """32 of 288 values are 1: a mean of 1/9, which no float is, and y is three times the gain."""
    rng = np.random.default_rng(2)
    x = np.zeros((3, 288))
    x[0, ::9], x[1, 4::9], x[2, 8::9] = 1, -2, 0.5
    gain = tied_gains(rng, 288)
    gain[gain == 0] = 1
    got, _ = yuear_lib.mx_rms_norm(bf16(torch, ref.to_bf16(x)), bf16(torch, ref.to_bf16(gain)), 0.0, bits=bits)
    check_codes(torch, got, 3 * np.sign(x) * gain, bits)


@pytest.mark.parametrize("rows,k,gap,bits,eps", [
    (1500, 3072, 0, 8, 1e-5), (1500, 2048, 0, 4, 1e-6), (700, 3136, 1, 8, 1e-5), (9000, 256, 0, 8, 1e-5),
    (300, 16384, 0, 4, 1e-5), (5, 8224, 2, 8, 0.0), (1, 3072, 0, 8, 1e-5),
])
def test_norm_of_a_sum_has_the_codes_of_64_bits(torch, yuear_lib, rows, k, gap, bits, eps):
    """With a residual, rows apart, the eps as the float that the call takes."""
    rng = np.random.default_rng(rows + k)
    x, r = random_rows(rng, rows, k, "plain"), random_rows(rng, rows, k, "plain")
    gain = ref.to_bf16(1 + 0.2 * rng.standard_normal(k))
    wide = torch.full((rows, k + 8 * gap), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:, :k] = bf16(torch, x)
    out, wides = pair_in(torch, rows, k, bits, gap)
    got, total = yuear_lib.mx_rms_norm(wide[:, :k], bf16(torch, gain), eps, residual=bf16(torch, r), bits=bits, out=out)
    h = ref.from_bf16(ref.to_bf16(ref.from_bf16(x) + ref.from_bf16(r)))
    np.testing.assert_array_equal(ref.from_bf16(bits_of(torch, total)), h)
    mean = (h ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps))
    check_codes(torch, got, h / np.sqrt(mean) * ref.from_bf16(gain), bits)
    assert untouched(wides, k, bits)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("ones", [1, 2])
def test_norm_of_values_past_32_bits(torch, yuear_lib, bits, ones):
    """A row of few values has a factor of 128 (ones = 1) or 90.5: values from 2^128 on count as infinite and
    make their block NaN, those below keep their codes."""
    k = 16384
    x, gain = np.zeros((4, k)), np.ones(k)
    x[0, :ones], x[1, 64:64 + ones], x[2, 128:128 + ones], x[3, 5000:5000 + ones] = 1, -1, 1, -3
    gain[:64], gain[64:128], gain[128:192], gain[4992:5024] = 2.0 ** 122 * 1.5, 2.0 ** 127, 2.0 ** 120 * 1.25, 2.0 ** 126
    got, _ = yuear_lib.mx_rms_norm(bf16(torch, ref.to_bf16(x)), bf16(torch, ref.to_bf16(gain)), 0.0, bits=bits)
    y = x / np.sqrt((x ** 2).mean(-1, keepdims=True)) * gain
    past = np.abs(y) >= 2.0 ** 128
    assert past.any(1).tolist() == [True, True, False, True]
    check_codes(torch, got, np.where(past, np.copysign(np.inf, y), y), bits)


# ---- product ----

@pytest.mark.parametrize("m,form", [(m, form) for m in (1, 5, 40, 70, 130, 300) for form in range(-1, 10 if m <= 16 else 8)])
def test_swiglu_where_the_exponential_leaves_32_bits(torch, yuear_lib, m, form):
    """Gates from -64 to -224 beside ups that make ordinary numbers of their results again, and beside
    ordinary gates of the same waves; the sums are one product each, exact."""
    gates = np.array([-64, -80, -88, -96, -104, -112, 2, -128, -144, -160, 0, -176, -192, -208, -224, 12])
    x = np.zeros((m, 128))
    x[:, 0], x[:, 32] = np.resize(gates if m > 1 else [-96], m), 1
    ups = np.resize(np.concatenate([2.0 ** np.arange(-24, 125, 7), -2.0 ** np.arange(3, 127, 11)]), 96)
    w = np.zeros((192, 128))
    w[0::2, 0], w[1::2, 32] = 1, ups
    a, wq = ref.quantize(x, 8), ref.quantize(w, 4)
    assert (ref.values(*a, 8) == x).all() and (ref.values(*wq, 4) == w).all()
    out = torch.empty(m, 96, dtype=torch.bfloat16, device="cuda")
    forced(torch, yuear_lib, form, pair_of(torch, *a, 8), pair_of(torch, *wq, 4), 8, out, swiglu=True)
    got, g = ref.from_bf16(bits_of(torch, out)), x[:, :1]
    want = g / (1 + np.exp(-g)) * ups
    # of the result: the exponent's roundings, of t and of its constant, ln 2 |t| 2^-23 = |g| 2^-23; one unit each of
    # three exponentials; eight roundings of half a step; then bf16's. Below its least number: half a step of that.
    off = np.abs(want) * (np.abs(g) * 2.0 ** -23 + 3 * 2.0 ** -23 + 8 * 2.0 ** -24)
    assert (np.abs(got - want) <= off * (1 + 2.0 ** -8) + np.abs(want) * ref.HALF_BF16 + 2.0 ** -134).all()
    assert (np.abs(want)[g[:, 0] < -88.7] > 2.0 ** -120).any()


@pytest.mark.parametrize("form", [5, 6, 7])
@pytest.mark.parametrize("bits,k", [(8, 640), (8, 1152), (4, 768), (4, 896)])
@pytest.mark.parametrize("epilogue", ["store", "swiglu", "residual"])
def test_every_value_of_tiles_after_the_first(torch, yuear_lib, form, bits, k, epilogue):
    """300 x 35002 are 274 tiles of 256 x 256 and more of the smaller ones, past the 256 workgroups of a launch:
    all of them against 64 bits, whose products are those of 1009 rows of W (an odd number, so that tiles differ)."""
    rng = np.random.default_rng(k + form)
    m, n, some = 300, 35002, 1009
    a, w = random_pair(rng, m, k, bits), random_pair(rng, some, k, 4)
    which = np.arange(n) * 7 % some
    width = n // 2 if epilogue == "swiglu" else n
    r = bf16(torch, ref.to_bf16(rng.standard_normal((m, n)))) if epilogue == "residual" else None
    out = torch.full((m, width), 7.0, dtype=torch.bfloat16, device="cuda")
    forced(torch, yuear_lib, form, pair_of(torch, *a, bits), pair_of(torch, w[0][which], w[1][which], 4), bits, out, r,
           epilogue == "swiglu")
    y, off = ref.product(ref.values(*a, bits), ref.values(*w, 4), bits)
    y, off = y[:, which], off[:, which]
    if epilogue == "residual":
        y = y + ref.from_bf16(bits_of(torch, r))
        off = off + 2.0 ** -24 * np.abs(y)
    elif epilogue == "swiglu":
        g, u, dg, du = y[:, 0::2], y[:, 1::2], off[:, 0::2], off[:, 1::2]
        with np.errstate(over="ignore"):
            silu = g / (1 + np.exp(-g))
        # |d silu| <= 1.1; the exponential and the quotient 2^-20 of the result, its argument's roundings |g| 2^-23
        y = silu * u
        off = 1.1 * dg * np.abs(u) + (np.abs(silu) + 1.1 * dg) * du + (2.0 ** -20 + np.abs(g) * 2.0 ** -23) * np.abs(y)
    bound = (1 + ref.HALF_BF16) * off + ref.HALF_BF16 * np.abs(y) + 2.0 ** -133
    err = np.abs(ref.from_bf16(bits_of(torch, out)) - y)
    assert (err <= bound).all(), f"{(err > bound).sum()} of {err.size} off, first at {np.argwhere(err > bound)[0]}"
