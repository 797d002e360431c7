"""The block scales of the hidden values of gated 8-bit experts whose width is not a multiple of 128.

The second product's weights are an identity, so the output is the hidden values as the kernel quantised them: 1.0 is 256
times the scale 2^-8 of its block, a power of two times an e4m3 value is exact in every step up to a 16-bit output, and the
other terms are zeros.  So y is compared with the definition itself: the e4m3 value of h with the smallest scale that brings
the block's largest |h| to 448, where h lies within d of its 64-bit value and quantisation is monotone for a given scale.

d: the pre-activations are off by at most t (_fp8_ref: the instruction's truncation and the fp32 additions, of which the bias
is one more term); silu moves between its values at the interval's ends (and by at most t^2 / 4 beyond them where the interval
holds the minimum of silu at -1.2785, as |silu''| <= 1/2); fp32 exponential and reciprocal are good for 2^-18 of the product at
|a| <= 32 (the argument's rounding is 32 log2(e) 2^-24 = 2^-18.5, the functions' own two units 2^-22)."""
import pytest
import torch

from moe_llava_amd import fp8, ops
from tests import _fp8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = torch.float64
M = 384


def _silu(a):
    return a * torch.sigmoid(a)


def _operands(I, kind, dt):
    """(x, w1, b1): gates near -16 everywhere, or open ones with a closed gate on a large last column."""
    g = torch.Generator().manual_seed(I)
    w = torch.randn((2 * I, M), generator=g) * M ** -0.5
    b = torch.zeros(2 * I)
    w[:I] *= 2.0 ** -4
    if kind == "closed":
        b[:I] = -16.0
    else:
        b[I - 1] = -16.0
        w[2 * I - 1] *= 64.0
    return w.to(torch.bfloat16), b.to(dt)


def _rows(S, dt):
    return torch.randn((S, M), generator=torch.Generator().manual_seed(S)).to(dt)


def _hidden(x, q1, s1, b1, I, ng):
    """(h, d) in 64 bits from the stored operands."""
    xd, wd = R.deq(x), R.deq_stored(q1, s1, 2)
    a, t = R.product(xd, wd)
    bias = b1.to(D)
    a, t = a + bias, t + (M / 8 + 16) * 2.0 ** -24 * bias.abs()
    u, v, tu, tv = a[:, :I], a[:, I:], t[:, :I], t[:, I:]
    lo, hi, mid = _silu(u - tu), _silu(u + tu), _silu(u)
    du = torch.maximum((lo - mid).abs(), (hi - mid).abs()) + torch.where((u + 1.2785).abs() <= tu + 1e-4, tu * tu / 4, 0.0)
    gated = torch.arange(I) < (I if ng < 0 else ng)
    h = torch.where(gated, mid, torch.ones((), dtype=D)) * v
    d = torch.where(gated, du * (v.abs() + tv) + mid.abs() * tv + 2.0 ** -18 * h.abs(), tv)
    return h, d


def _check(y, h, d):
    top, e = R._top(h), R._top(d)
    got = y.cpu().to(D)
    ok = torch.zeros(h.shape, dtype=torch.bool)
    for b in (R.scale_byte((top - e).clamp_min(0)), R.scale_byte(top + e)):
        sc = R.spread(torch.exp2(b.to(D) - 127), *h.shape)
        q = lambda v: R.e4m3((v / sc).clamp(-448.0, 448.0)) * sc
        ok |= (got >= q(h - d)) & (got <= q(h + d))
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} hidden values are not the e4m3 values of their block"


@pytest.mark.parametrize("kind,dt", [("closed", torch.bfloat16), ("large_last", torch.float16), ("large_last", torch.bfloat16)])
@pytest.mark.parametrize("I", [16, 112, 128, 176, 320])
@pytest.mark.parametrize("S,tile", [(1, None), (70, None), (300, "256,256"), (300, "192,256"), (300, "128,256"), (300, "64,256"),
                                    (300, "32,256")])
def test_hidden_scales_of_a_short_block(S, tile, I, kind, dt, monkeypatch):
    w1, b1 = _operands(I, kind, dt)
    x = _rows(S, dt)
    q1, s1 = fp8.quantize_weight(w1.to(DEV), 2)
    q2, s2 = fp8.quantize_weight(torch.eye(M, I, dtype=torch.bfloat16, device=DEV))
    offs = torch.tensor([0, S], dtype=torch.int32, device=DEV)
    try:
        if tile:
            monkeypatch.setenv("MOE_GEMM_TILE", tile)
            ops.reload_knobs()
        for ng in (-1, I, I - 5, I // 2):
            y = fp8.expert_ffn("swiglu", x.to(DEV), q1[None], s1[None], q2[None], s2[None], offs, S, b1=b1.to(DEV)[None], n_gated=ng)
            h, d = _hidden(x, q1.cpu(), s1.cpu(), b1, I, ng)
            _check(y[:, :I], h, d)
            assert not bool(y[:, I:].any())
    finally:
        if tile:
            monkeypatch.delenv("MOE_GEMM_TILE")
            ops.reload_knobs()
