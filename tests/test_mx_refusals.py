"""What the block-scaled entry points refuse, before anything is launched: runs without a GPU."""
import numpy as np
import pytest

import mx_ref as ref

BASE = 1 << 40  # addresses that nothing reads


def quantize(lib, x=BASE, x_stride=64, rows=4, k=64, bits=8, codes=BASE + (1 << 20), codes_stride=64,
             scales=BASE + (2 << 20), scales_stride=2):
    return lib.yuear_op_mx_quantize(x, x_stride, rows, k, bits, codes, codes_stride, scales, scales_stride, None)


def dequantize(lib, x=BASE, x_stride=64, rows=4, k=64, bits=8, codes=BASE + (1 << 20), codes_stride=64,
               scales=BASE + (2 << 20), scales_stride=2):
    return lib.yuear_op_mx_dequantize(codes, codes_stride, scales, scales_stride, rows, k, bits, x, x_stride, None)


BAD_ROWS = [
    dict(x=0), dict(codes=0), dict(scales=0), dict(x=BASE + 2), dict(codes=BASE + (1 << 20) + 8), dict(rows=-1),
    dict(k=0), dict(k=48), dict(k=-32), dict(k=(1 << 20) + 32, x_stride=1 << 21, codes_stride=1 << 21),
    dict(bits=6), dict(bits=0), dict(x_stride=56), dict(x_stride=60), dict(x_stride=-64), dict(codes_stride=48),
    dict(codes_stride=72), dict(scales_stride=1), dict(x_stride=(1 << 22) + 8), dict(codes_stride=(1 << 22) + 16),
    dict(scales_stride=(1 << 22) + 1), dict(codes=BASE), dict(codes=BASE + 480), dict(scales=BASE + 511),
    dict(bits=4, codes_stride=16), dict(rows=0x7FFFFFFF, k=1 << 20, x_stride=1 << 20, codes_stride=1 << 20,
                                        scales_stride=1 << 15, codes=BASE + (1 << 53), scales=BASE + (1 << 54)),
]


@pytest.mark.parametrize("bad", BAD_ROWS, ids=[str(i) for i in range(len(BAD_ROWS))])
@pytest.mark.parametrize("call", [quantize, dequantize])
def test_rows_refused(yuear_lib, call, bad):
    assert call(yuear_lib.lib, **bad) == 1


def test_quantize_refuses_codes_over_scales(yuear_lib):
    assert quantize(yuear_lib.lib, scales=BASE + (1 << 20) + 64) == 1


def norm(lib, x=BASE, x_stride=64, residual=BASE + (1 << 20), residual_stride=64, gain=BASE + (5 << 20), rows=4, k=64,
         bits=8, codes=BASE + (2 << 20), codes_stride=64, scales=BASE + (3 << 20), scales_stride=2,
         total=BASE + (4 << 20), sum_stride=64):
    return lib.yuear_op_mx_rms_norm(x, x_stride, residual, residual_stride, gain, 1e-5, rows, k, bits, codes,
                                    codes_stride, scales, scales_stride, total, sum_stride, None)


@pytest.mark.parametrize("bad", [
    dict(x=0), dict(gain=0), dict(gain=BASE + (5 << 20) + 2), dict(residual=0), dict(total=0), dict(codes=0),
    dict(scales=0), dict(k=16416, x_stride=16416, residual_stride=16416, sum_stride=16416, codes_stride=16416,
                         scales_stride=513), dict(k=33), dict(rows=-5), dict(rows=1 << 23), dict(bits=16),
    dict(sum_stride=32), dict(residual_stride=60), dict(total=BASE + 16), dict(total=BASE, sum_stride=72),
    dict(total=BASE + (1 << 20) + 128), dict(total=BASE + (5 << 20)), dict(codes=BASE + (5 << 20)),
    dict(codes=BASE + (4 << 20)), dict(codes=BASE + (1 << 20)), dict(scales=BASE + 6), dict(codes=BASE + (3 << 20) - 64),
])
def test_norm_refused(yuear_lib, bad):
    assert norm(yuear_lib.lib, **bad) == 1


def gemm(lib, a=BASE, a_stride=256, a_scales=BASE + (1 << 20), a_scales_stride=8, a_bits=8, w=BASE + (2 << 20),
         w_stride=128, w_scales=BASE + (3 << 20), w_scales_stride=8, m=4, n=6, k=256, residual=None,
         residual_stride=0, c=BASE + (4 << 20), ldc=6, swiglu=0):
    return lib.yuear_op_mx_gemm(a, a_stride, a_scales, a_scales_stride, a_bits, w, w_stride, w_scales, w_scales_stride,
                                m, n, k, residual, residual_stride, c, ldc, swiglu, None)


@pytest.mark.parametrize("bad", [
    dict(a=0), dict(w=0), dict(c=0), dict(a_scales=0), dict(w_scales=0), dict(a=BASE + 8), dict(w=BASE + (2 << 20) + 4),
    dict(a_scales=BASE + (1 << 20) + 2), dict(w_scales=BASE + (3 << 20) + 1), dict(a_scales_stride=10),
    dict(w_scales_stride=9), dict(a_scales_stride=4), dict(c=BASE + (4 << 20) + 1), dict(k=64), dict(k=0), dict(k=-128),
    dict(k=192), dict(k=(1 << 20) + 128), dict(a_bits=16), dict(a_stride=128), dict(w_stride=64), dict(a_stride=264),
    dict(m=-1), dict(n=-1), dict(ldc=5), dict(swiglu=2), dict(n=5, swiglu=1), dict(swiglu=1, ldc=2),
    dict(swiglu=1, residual=BASE + (5 << 20), residual_stride=6), dict(residual=BASE + (5 << 20), residual_stride=5),
    dict(residual=BASE + (4 << 20) + 2, residual_stride=6), dict(residual=BASE + (4 << 20), residual_stride=8),
    dict(c=BASE), dict(c=BASE + (1 << 20)), dict(c=BASE + (2 << 20) - 16), dict(c=BASE + (3 << 20) + 4),
    dict(ldc=1 << 31), dict(m=(1 << 30) + 1), dict(n=(1 << 30) + 1, ldc=1 << 31), dict(w_stride=(1 << 22) + 16),
])
def test_gemm_refused(yuear_lib, bad):
    assert gemm(yuear_lib.lib, **bad) == 1


def test_forms_refused(yuear_lib):
    for form in (-2, 10):
        assert yuear_lib.lib.yuear_op_mx_gemm_form(BASE, 256, BASE + (1 << 20), 8, 8, BASE + (2 << 20), 128, BASE + (3 << 20),
                                                   8, 4, 6, 256, None, 0, BASE + (4 << 20), 6, 0, form, None) == 1


def test_empty_calls(yuear_lib):
    lib = yuear_lib.lib
    assert quantize(lib, rows=0) == 0 and dequantize(lib, rows=0) == 0 and norm(lib, rows=0) == 0
    assert gemm(lib, m=0) == 0 and gemm(lib, n=0) == 0


def test_python_calls_are_checked(yuear_lib):
    """The binding's own checks: CPU tensors, types, shapes and pairs."""
    import torch
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    pair = torch.zeros(4, 128, dtype=torch.float8_e4m3fn), torch.zeros(4, 4, dtype=torch.float8_e8m0fnu)
    w = torch.zeros(6, 64, dtype=torch.uint8), torch.zeros(6, 4, dtype=torch.float8_e8m0fnu)
    for call in (lambda: yuear_lib.mx_quantize(x), lambda: yuear_lib.mx_dequantize(pair),
                 lambda: yuear_lib.mx_rms_norm(x, x[0]), lambda: yuear_lib.mx_gemm(pair, w)):
        with pytest.raises(ValueError, match="on the GPU"):
            call()


def test_formats():
    """The grids against the formats' known values."""
    g = ref.grid(8)
    assert g[0] == 0 and g[1] == 2.0 ** -9 and g[8] == 2.0 ** -6 and g[0x38] == 1 and g[126] == 448
    assert list(ref.grid(4)) == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    x = np.zeros((1, 64))
    x[0, :4], x[0, 32:35] = [7.9, -5, 2.5, 0.25], [np.inf, 1, 2]
    codes, scales = ref.quantize(x, 4)
    assert list(scales[0]) == [127, 255] and list(ref.unpack(codes, 4)[0, :4]) == [7, 14, 4, 0]
    assert not ref.unpack(codes, 4)[0, 32:].any()
