"""Block-scaled rows where no GPU is needed: the binding on a torch without the types of their
scales."""
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
