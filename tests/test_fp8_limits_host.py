"""Row counts and dimensions at the end of 32 bits, on the CPU: the library refuses what its tiles would carry past it, before
anything is launched, and the Python layer refuses what 32 bits do not hold (no memory is behind these tensors)."""
import pytest
import torch

from moe_llava_amd import _lib, fp8

SHAPE = -2
MOST, PAST = 2 ** 31 - 512, (2 ** 31 - 511, 2 ** 31 - 1)


@pytest.mark.parametrize("n", PAST)
def test_library_refuses(n):
    lib = _lib.load()
    big = n // 16 * 16                                     # a multiple of 16 where the operator wants one
    assert lib.moe_add_rms_norm_fwd(16, 64, None, 0, 16, 0, 1e-6, n, 64, 16, 64, None, 0, None, None, 0, None, 0, 0, None) == SHAPE
    assert lib.moe_add_rms_norm_bwd(16, 64, None, 0, 16, 64, 16, 0, 16, n, 64, 16, 64, 16, 16, 2 ** 40, 0, None) == SHAPE
    assert lib.moe_quantize_rows_fp8(16, 64, n, 64, 16, 64, 16, 4, 0, None) == SHAPE
    assert lib.moe_quantize_blocks_fp8(16, 1, n, 16, 16, 16, 0, None) == SHAPE
    gemm = lambda rows, N: lib.moe_grouped_gemm_fp8_fwd(16, 16, 16, 4, None, 0, 16, 16, None, None, 1, 1, rows, 16, N, 0, 16, N, 0, None)
    assert gemm(n, 16) == SHAPE and gemm(16, n) == SHAPE
    linear = lambda rows, N: lib.moe_grouped_linear_fp8_fwd(16, 16, 16, 16, None, None, 1, 1, rows, 16, N, 0, 16, 2 ** 62, 16, N, 0, None)
    assert linear(n, 16) == SHAPE and linear(16, n) == SHAPE
    ffn = lambda src, rows: lib.moe_expert_ffn_fp8_fwd(1, 16, 16, src, None, 0, None, 0, 16, 1, 16, 16, None, 16, 16, None, 16, 1, 1, rows,
                                                       16, 16, -1, 16, 2 ** 62, 16, 0, None)
    assert ffn(16, n) == SHAPE and ffn(n, 16) == SHAPE
    if big > MOST:
        assert lib.moe_quantize_rows_fp8(16, big, 1, big, 16, big, 16, 2 ** 25, 0, None) == SHAPE
        assert lib.moe_quantize_blocks_fp8(16, 1, 16, big, 16, 16, 0, None) == SHAPE
        assert lib.moe_transpose_blocks_fp8(16, 16, 1, big, 16, 16, 16, None) == SHAPE
        assert lib.moe_transpose_blocks_fp8(16, 16, 1, 16, big, 16, 16, None) == SHAPE


def test_python_layer_refuses(monkeypatch):
    monkeypatch.setattr(fp8, "_gpu", lambda t, name: None)
    x = torch.zeros((1, 16), dtype=torch.bfloat16)
    row = torch.zeros((1, 1), dtype=torch.bfloat16)
    for bad in (x.expand(MOST + 1, 16), row.expand(1, 2 ** 32 + 16), x.expand(2 ** 32, 16)):
        with pytest.raises(ValueError, match="at most"):
            fp8.quantize_rows(bad)
    q = torch.zeros(1, dtype=torch.uint8).view(fp8.E4M3)
    s = torch.zeros(1, dtype=torch.uint8).view(fp8.E8M0)
    monkeypatch.setattr(torch.Tensor, "is_contiguous", lambda self, *a, **k: True)
    N = 2 ** 32 + 16
    with pytest.raises(ValueError, match="at most"):
        fp8._check_weight(q.expand(N, 16), s.expand((N + 127) // 128, 1), "w", 0, None)
