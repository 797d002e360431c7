"""Which norms MoE.forward_normed runs as kernels and which it calls, on the CPU: the block itself and the kernels are replaced
by stand-ins."""
import pytest
import torch
from torch import nn

import moe_llava_amd
from moe_llava_amd import norm as norm_ops
from tests.expert_mlps import StableLMMLP

M = 64


class _Llama(nn.Module):
    """A norm of the usual form, with the usual names."""
    def __init__(self):
        super().__init__()
        self.weight = nn.Parameter(torch.randn(M))
        self.variance_epsilon = 1e-5

    def forward(self, x):
        return self.weight * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.variance_epsilon)


class _OnePlus(_Llama):
    def forward(self, x):
        return (1 + self.weight) * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.variance_epsilon)


class _Property(_Llama):
    """An eps that is a property, and a forward of its own."""
    eps = property(lambda self: 2e-5)

    def forward(self, x):
        return super().forward(x)


@pytest.fixture
def moe(monkeypatch):
    class Block(moe_llava_amd.MoE):
        def forward(self, x, used_token=None):
            return x * 3, "l_aux", "counts"

    block = Block(M, StableLMMLP(M, M), num_experts=2, k=2)
    block.kernels = []

    def rms_norm(x, weight, eps):
        block.kernels.append((weight, eps))
        return x

    monkeypatch.setattr(norm_ops, "rms_norm", rms_norm)
    monkeypatch.setattr(norm_ops, "add_rms_norm", lambda x, r, w, e: (rms_norm(x + r, w, e), x + r))
    monkeypatch.setattr(norm_ops, "_FORWARDS", set(getattr(norm_ops, "_FORWARDS", ())), raising=False)
    return block


def _x(seed):
    return torch.randn((5, M), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("make", [_Llama, _OnePlus, lambda: nn.RMSNorm(M), lambda: nn.RMSNorm(M, elementwise_affine=False),
                                  lambda: nn.RMSNorm(M, 1e-5, elementwise_affine=False)])
@pytest.mark.parametrize("res", [False, True])
def test_other_norms_are_called(moe, make, res):
    """Not declared, or an eps or a weight that only the module's forward knows."""
    nm, x, r = make(), _x(1), _x(2) if res else None
    s = x + r if res else x
    out = moe.forward_normed(x, r, nm)
    assert torch.equal(out[0], nm(s) * 3) and out[1:3] == ("l_aux", "counts") and torch.equal(out[3], s) and not moe.kernels


@pytest.mark.parametrize("make,eps", [(lambda: norm_ops.RMSNorm(M, 1e-4), 1e-4), (lambda: nn.RMSNorm(M, 1e-3), 1e-3),
                                      (lambda: norm_ops.register_rms_norm(_Llama)(), 1e-5),
                                      (lambda: norm_ops.register_rms_norm(_Property)(), 2e-5)])
@pytest.mark.parametrize("res", [False, True])
def test_known_norms_run_as_kernels(moe, make, eps, res):
    nm = make()
    moe.forward_normed(_x(1), _x(2) if res else None, nm)
    assert len(moe.kernels) == 1 and moe.kernels[0][0] is nm.weight and moe.kernels[0][1] == eps


def test_what_is_around_a_known_norm_is_kept(moe):
    """Hooks, a forward set on the module, and a subclass with a forward of its own."""
    x = _x(1)
    nm = nn.RMSNorm(M, 1e-5)
    seen = []
    h = nm.register_forward_hook(lambda m, a, o: seen.append(1) or o * 2)
    assert torch.equal(moe.forward_normed(x, None, nm)[0], nm(x) * 3) and seen
    h.remove()
    nm.forward = lambda t: t * 5
    assert torch.equal(moe.forward_normed(x, None, nm)[0], x * 5 * 3)
    norm_ops.register_rms_norm(_Llama)
    nm = _OnePlus()
    assert torch.equal(moe.forward_normed(x, None, nm)[0], nm(x) * 3) and not moe.kernels
