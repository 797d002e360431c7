"""The 8-bit expert MLP against 64 bits in the 2-norm, as tight as the format and the matrix instruction allow.

Two errors remain in y.  (1) Its rounding: uniform within half a step, u = eps / 2 of the value at most, so u / sqrt(3) in the
2-norm.  (2) Hidden values that go to the neighbouring e4m3 value.  The first product is off by 1.4e-5 of its size in the 2-norm
(the instruction cuts terms 13 bits below the largest of 8), a gated hidden value, a product of two of them, by d = 2^-15 at
most.  An error e of a value h crosses a rounding tie with the probability |e| / step and then moves it by one step, at most
2^-3 |h|: the expected square is sum |e| 2^-3 |h| <= 2^-3 d |h|^2 (Cauchy-Schwarz), 2^-9 of |h| in the 2-norm, and as much of
y, to within a quarter at these sizes (thousands of values, a random second matrix).  The two are independent."""
import pytest
import torch

from moe_llava_amd import fp8
from tests import _fp8_ref as R
from tests.test_gpu_fp8 import _ffn_ref, _rows

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,E,S,M,I", [("swiglu", 2, 64, 2048, 512), ("swiglu", 4, 200, 1024, 1408), ("swiglu", 2, 300, 512, 176),
                                         ("swiglu", 3, 48, 1024, 320), ("gelu_new", 2, 120, 1280, 2560), ("gelu_new", 3, 33, 2560, 272)])
def test_expert_ffn_in_the_2_norm(act, E, S, M, I, dt):
    g = torch.Generator().manual_seed(S + M + I)
    parts = 2 if act == "swiglu" else 1
    x = _rows(g, S, M, dt)
    q1, s1 = R.weights(g, E, I, M, parts)
    q2, s2 = R.weights(g, E, M, I)
    cut = [S * e // E for e in range(E + 1)]
    y = fp8.expert_ffn(act, x.to(DEV), *[t.to(DEV) for t in (q1, s1, q2, s2)], torch.tensor(cut, dtype=torch.int32, device=DEV), S)
    ref = torch.cat([_ffn_ref(x[cut[e]:cut[e + 1]], q1[e], s1[e], q2[e], s2[e], None, None, act)[0] for e in range(E)])
    rel = float((y.cpu().to(torch.float64) - ref).norm() / ref.norm())
    limit = (R.half_step(dt) ** 2 / 3 + (1.25 * 2.0 ** -9) ** 2) ** 0.5
    assert rel <= limit, (rel, limit)
