"""CPU tests of the 8-bit operators: the entry points refuse what they cannot do before anything is launched, the Python
layer refuses CPU tensors, and the reference of the GPU tests agrees with torch's own e4m3 conversion."""
import pytest
import torch

from moe_llava_amd import _lib, fp8, norm
from tests import _fp8_ref as R

ARG, SHAPE, ALIGN, WS = -1, -2, -3, -4


def test_norm_entry_refuses():
    f = _lib.load().moe_add_rms_norm_fwd

    def call(x=16, ldx=64, r=16, ldr=64, w=16, wd=0, S=4, M=64, y=16, ldy=64, s=16, lds=64, q=None, ldq=0, sc=None, lsc=0, dt=0):
        return f(x, ldx, r, ldr, w, wd, 1e-6, S, M, y, ldy, s, lds, None, q, ldq, sc, lsc, dt, None)
    assert call(S=0) == 0                                      # nothing to do, nothing launched
    assert call(x=None) == ARG and call(w=None) == ARG and call(y=None) == ARG and call(dt=2) == ARG
    assert call(wd=2, dt=0) == ARG and call(wd=1, dt=1) == ARG and call(s=None) == ARG and call(q=16) == ARG
    assert call(M=0) == SHAPE and call(M=65537, ldx=70000, ldr=70000, ldy=70000, lds=70000) == SHAPE and call(S=-1) == SHAPE
    assert call(ldx=63) == SHAPE and call(lds=60) == SHAPE
    assert call(q=16, sc=16, ldq=63, lsc=4) == SHAPE and call(q=16, sc=16, ldq=64, lsc=0) == SHAPE
    assert call(q=16, sc=16, ldq=64, lsc=4, M=56) == SHAPE
    assert call(x=17) == ALIGN and call(q=20, sc=16, ldq=64, lsc=4) == ALIGN and call(w=18) == ALIGN


def test_norm_backward_entry_refuses():
    lib = _lib.load()
    f = lib.moe_add_rms_norm_bwd
    n = lib.moe_add_rms_norm_bwd_workspace_bytes(4, 64)
    assert n == 4 * 64 * 4 and lib.moe_add_rms_norm_bwd_workspace_bytes(0, 64) == 0

    def call(dy=16, s=16, w=16, rstd=16, S=4, M=64, dx=16, dw=16, ws=16, nb=n, dt=0, lds=64):
        return f(dy, 64, None, 0, s, lds, w, 0, rstd, S, M, dx, 64, dw, ws, nb, dt, None)
    assert call(s=None) == ARG and call(rstd=None) == ARG and call(dw=None) == ARG and call(dt=5) == ARG
    assert call(S=0) == SHAPE and call(M=0) == SHAPE and call(lds=8) == SHAPE
    assert call(dx=17) == ALIGN and call(nb=n - 1) == WS


def test_quantise_and_transpose_entries_refuse():
    lib = _lib.load()
    f = lib.moe_quantize_rows_fp8
    assert f(16, 64, 0, 64, 16, 64, 16, 4, 0, None) == 0
    assert f(None, 64, 4, 64, 16, 64, 16, 4, 0, None) == ARG and f(16, 64, 4, 64, 16, 64, 16, 4, 9, None) == ARG
    assert f(16, 64, 4, 60, 16, 64, 16, 4, 0, None) == SHAPE and f(16, 63, 4, 64, 16, 64, 16, 4, 0, None) == SHAPE
    assert f(16, 64, 4, 64, 16, 60, 16, 4, 0, None) == SHAPE and f(16, 64, 4, 64, 16, 64, 16, 0, 0, None) == SHAPE
    assert f(17, 64, 4, 64, 16, 64, 16, 4, 0, None) == ALIGN and f(16, 64, 4, 64, 20, 64, 16, 4, 0, None) == ALIGN
    b = lib.moe_quantize_blocks_fp8
    assert b(None, 1, 4, 16, 16, 16, 0, None) == ARG and b(16, 0, 4, 16, 16, 16, 0, None) == SHAPE
    assert b(16, 1, 4, 24, 16, 16, 0, None) == SHAPE and b(24, 1, 4, 16, 16, 16, 0, None) == ALIGN
    t = lib.moe_transpose_blocks_fp8
    assert t(None, 16, 1, 16, 16, 16, 16, None) == ARG and t(16, 16, 1, 20, 16, 16, 16, None) == SHAPE
    assert t(16, 16, 1, 16, 8, 16, 16, None) == SHAPE and t(24, 16, 1, 16, 16, 16, 16, None) == ALIGN


def test_product_entry_refuses():
    f = _lib.load().moe_grouped_gemm_fp8_fwd

    def call(a=16, lda=128, s=16, lds=4, sh=0, w=16, ws=16, offs=16, G=2, E=2, rows=8, K=128, N=64, out=16, ldo=64, dt=0):
        return f(a, lda, s, lds, None, sh, w, ws, None, offs, G, E, rows, K, N, 0, out, ldo, dt, None)
    assert call(rows=0) == 0
    assert call(a=None) == ARG and call(w=None) == ARG and call(out=None) == ARG and call(offs=None) == ARG and call(dt=3) == ARG
    assert call(K=120) == SHAPE and call(K=0) == SHAPE and call(K=65552, lda=65552, lds=1024) == SHAPE
    assert call(N=0) == SHAPE and call(G=0) == SHAPE and call(G=5000) == SHAPE and call(E=0) == SHAPE and call(rows=-1) == SHAPE
    assert call(lda=112) == SHAPE and call(lda=136) == SHAPE and call(lds=3) == SHAPE and call(lds=0) == SHAPE
    assert call(sh=2) == SHAPE and call(ldo=63) == SHAPE
    assert call(a=24) == ALIGN and call(w=24) == ALIGN and call(s=18) == ALIGN and call(out=17) == ALIGN


def test_ffn_entry_refuses():
    lib = _lib.load()
    need = lib.moe_expert_ffn_fp8_workspace_bytes(8, 16, 128, 256)
    assert need >= 16 * 256 + 16 * 4 + 8 * 128 + 8 * 4 and lib.moe_expert_ffn_fp8_workspace_bytes(-1, 1, 16, 16) == 0

    def call(act=0, x=16, a=None, asc=None, w1=16, w2=16, offs=16, G=2, rows=16, M=128, I=256, ws=16, nb=need, y=16, dt=0, sh=1):
        return lib.moe_expert_ffn_fp8_fwd(act, x, 128, 8, a, 128, asc, 4, 16, sh, w1, 16, None, w2, 16, None, offs, G, 2, rows,
                                          M, I, -1, ws, nb, y, dt, None)
    assert call(rows=0) == 0
    assert call(act=4) == ARG and call(dt=7) == ARG and call(a=16, asc=16) == ARG and call(x=None) == ARG
    assert call(w1=None) == ARG and call(w2=None) == ARG and call(offs=None) == ARG and call(ws=None) == ARG and call(y=None) == ARG
    assert call(M=120) == SHAPE and call(I=200) == SHAPE and call(G=0) == SHAPE and call(sh=3) == SHAPE and call(rows=-2) == SHAPE
    assert call(ws=24) == ALIGN and call(y=24) == ALIGN and call(w1=24) == ALIGN
    assert call(nb=need - 1) == WS


def test_python_layer_refuses_cpu_tensors():
    x = torch.zeros((4, 128), dtype=torch.bfloat16)
    q, s = torch.zeros((64, 128), dtype=R.E4M3), torch.zeros((1, 1), dtype=torch.uint8).view(R.E8M0)
    for f in (lambda: fp8.quantize_rows(x), lambda: fp8.quantize_weight(x), lambda: fp8.linear(x, q, s),
              lambda: fp8.grouped_linear(x, q[None], s[None], torch.zeros(2, dtype=torch.int32)),
              lambda: fp8.expert_ffn("gelu_new", x, q[None], s[None], q.t().contiguous()[None], s[None], torch.zeros(2, dtype=torch.int32), 4),
              lambda: norm.rms_norm(x, x[0]), lambda: norm.add_rms_norm(x, x, x[0]), lambda: norm.add_rms_norm_fp8(x, x, x[0])):
        with pytest.raises(_lib.MoEKernelError):
            f()
    with pytest.raises(TypeError):
        fp8.quantize_rows([1.0])
    with pytest.raises(ValueError):
        norm.add_rms_norm(x, None, x[0])


def test_reference_rounds_like_the_type():
    v = torch.linspace(-448, 448, 40001, dtype=torch.float64)
    v = torch.cat([v, v * 2.0 ** -10, v * 2.0 ** -16]).to(torch.float32).to(torch.float64)     # torch converts from fp32
    assert torch.equal(R.e4m3(v), v.to(torch.float32).to(R.E4M3).to(torch.float32).to(torch.float64))
    top = torch.tensor([0.0, 448.0, 448.0001, 1.75, 1.7500001, 896.0, 1e-40], dtype=torch.float64)
    assert R.scale_byte(top).tolist() == [1, 127, 128, 119, 120, 128, 1]


def test_forward_normed_refuses_other_norms():
    """A LayerNorm has a weight and an eps as well, but is another norm."""
    import moe_llava_amd
    from tests.expert_mlps import StableLMMLP
    moe = moe_llava_amd.MoE(64, StableLMMLP(64, 64), num_experts=2, k=2)
    x = torch.zeros((2, 64))
    with pytest.raises(TypeError):
        moe.forward_normed(x, None, torch.nn.LayerNorm(64))
    with pytest.raises(TypeError):
        moe.forward_normed(x, None, torch.nn.LayerNorm(64, elementwise_affine=False))
