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
