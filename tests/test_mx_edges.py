"""Block-scaled rows where no GPU is needed: the binding on a torch without the types of their
scales, numbers of rows past 32 bits, and sizes that a launch takes."""
import pytest


@pytest.fixture
def old_torch(yuear_lib, monkeypatch):
    """torch without float8_e8m0fnu, met for the first time by the binding."""
    import torch
    monkeypatch.delattr(torch, "float8_e8m0fnu")
    for name in ("_T", "_BF16", "_INT32", "_UINT8", "_E4M3", "_E8M0"):
        monkeypatch.setattr(yuear_lib, name, None)
    return torch


def test_paged_operators_need_no_scale_type(yuear_lib, old_torch):
    """They come as far as their own checks (here: tensors on the CPU)."""
    pages = old_torch.zeros(1, 1, 32, 128, dtype=old_torch.bfloat16), old_torch.zeros(1, 1, 1, 128, 32, dtype=old_torch.bfloat16)
    with pytest.raises(ValueError, match="pages_copy"):
        yuear_lib.pages_copy(*pages, [0], [0])


def test_block_scaled_rows_without_their_types_are_refused(yuear_lib, old_torch):
    x = old_torch.zeros(4, 128, dtype=old_torch.bfloat16)
    yuear_lib._torch()
    with pytest.raises(ValueError, match="float8_e8m0fnu"):
        yuear_lib._mx_out(x, 4, 128, 8, None, 0, "mx_quantize")
    pair = old_torch.zeros(4, 128, dtype=old_torch.float8_e4m3fn), old_torch.zeros(4, 4, dtype=old_torch.uint8)
    with pytest.raises(ValueError, match="block-scaled rows"):
        yuear_lib._mx_rows(pair, -1, "mx_dequantize")


def test_products_of_the_largest_sizes_are_not_refused(yuear_lib):
    """257 x (2^29 + 256) in SwiGLU, 138 GB of outputs, are more than 2^22 tiles of 256 x 256. (Without a GPU the
    launch itself fails, with another error than that of invalid arguments.)"""
    import torch
    if torch.cuda.device_count():
        pytest.skip("nothing is to be launched on these addresses")
    base, m, n = 1 << 40, 257, (1 << 29) + 256
    for k in (128, 512, 640):
        status = yuear_lib.lib.yuear_op_mx_gemm(base, k, base + (1 << 20), k // 32, 8, base + (1 << 41), k // 2,
                                                base + (1 << 40), k // 32, m, n, k, None, 0, base + (1 << 43), n // 2, 1, None)
        assert status not in (0, 1)


@pytest.mark.parametrize("rows", [1 << 31, (1 << 32) + 5])
def test_rows_that_32_bits_do_not_count_are_refused(yuear_lib, rows):
    """2^32 + 5 rows (of weights in 4 bits with k 128: 292 GB) are not taken for 5."""
    import torch
    yuear_lib._torch()
    codes, scales = torch.zeros(1, 64, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.float8_e8m0fnu)
    assert yuear_lib._mx_rows((codes, scales), -1, "mx_gemm")[:3] == (1, 128, 4)
    with pytest.raises(ValueError, match="2.31"):
        yuear_lib._mx_rows((codes.expand(rows, 64), scales.expand(rows, 4)), -1, "mx_gemm")
    with pytest.raises(ValueError, match="2.31"):
        yuear_lib._mx_shape(torch.zeros(1, 32, dtype=torch.bfloat16).expand(rows, 32), "mx_quantize")
