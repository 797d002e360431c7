"""The state that 8-bit experts keep between calls (the packed 16-bit weights, the 8-bit copy of them), on the CPU: the
quantisation itself is replaced by a stand-in that records what it was asked to do."""
import pytest
import torch

import moe_llava_amd
from moe_llava_amd import fp8
from tests.expert_mlps import PhiMLP, StableLMMLP

CPU = torch.device("cpu")


@pytest.fixture
def made(monkeypatch):
    """List of the quantisations that were run: (weights, out)."""
    log = []

    def quantize_weight(w, projections=1, out=None):
        log.append((w, out))
        return out if out is not None else (w.to(torch.float32), torch.zeros(w.shape[0], dtype=torch.uint8))

    monkeypatch.setattr(fp8, "quantize_weight", quantize_weight)
    return log


def _experts(form=StableLMMLP, eight=True):
    torch.manual_seed(0)
    ex = moe_llava_amd.MoE(64, form(64, 64).to(torch.bfloat16), num_experts=2, k=2).deepspeed_moe.experts
    if eight:
        ex.quantize_fp8()
    return ex


@pytest.mark.parametrize("form", [StableLMMLP, PhiMLP])
def test_change_in_inference_mode_is_seen(made, form):
    """A module made as usual whose first call runs in inference mode: changes in place, inside that mode and outside it,
    are quantised again, and calls without one are not."""
    ex = _experts(form)
    with torch.inference_mode():
        ex.packed_fp8(CPU)
        n = len(made)
        ex.packed_fp8(CPU)
        assert n == 2 and len(made) == n
        for p in ex.parameters():
            p.mul_(2)
        ex.packed_fp8(CPU)
        assert len(made) == n + 2
    with torch.no_grad():
        ex.packed_fp8(CPU)
        assert len(made) == n + 2


def test_packing_in_inference_mode_leaves_trainable_parameters():
    ex = _experts(eight=False)
    with torch.inference_mode():
        ex.packed(CPU)
    for p in ex.parameters():
        assert not p.is_inference()
        p.float().square().sum().backward()
        assert p.grad is not None


@pytest.mark.parametrize("first", [torch.inference_mode, torch.no_grad])
@pytest.mark.parametrize("then", [torch.inference_mode, torch.no_grad])
def test_refill_in_another_mode(made, first, then):
    """The copy made in one mode is filled again in the other, biases included, and stays the same tensors."""
    ex = _experts(PhiMLP)
    with first():
        a = ex.packed_fp8(CPU)
    with torch.no_grad():
        for e in ex.deepspeed_experts:
            e.fc1.weight.mul_(2)
            e.fc2.bias.fill_(3)
    with then():
        b = ex.packed_fp8(CPU)
    assert b is a and len(made) == 4 and all(bool((t == 3).all()) for t in b[6])
    assert not any(t.is_inference() for t in b[1:] if t is not None)
