"""MoE blocks on 8-bit experts (MoE.quantize_experts, MoE.forward_normed): routing identical to the 16-bit block, outputs
against 64 bits, the pieces against the whole, staleness, refusals."""
import pytest
import torch

import moe_llava_amd
from moe_llava_amd import fp8, norm
from moe_llava_amd.graph import GraphedMoE
from tests import _fp8_ref as R
from tests.expert_mlps import PhiMLP, RePaMLP, StableLMMLP
from tests.test_gpu_fp8 import _check_ffn, _ffn_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = torch.float64


def _moe(M=256, I=320, E=4, form="swiglu", dt=torch.bfloat16, **kw):
    torch.manual_seed(0)
    proto = (StableLMMLP if form == "swiglu" else PhiMLP)(M, I).to(dt)
    args = dict(num_experts=E, k=2, capacity_factor=1.0, eval_capacity_factor=2.0, min_capacity=0,
                top2_2nd_expert_sampling=False)
    args.update(kw)
    moe = moe_llava_amd.MoE(M, proto, **args).to(DEV)
    with torch.no_grad():
        for n, p in moe.named_parameters():
            p.copy_((torch.randn(p.shape) * (0.3 if "wg" in n else 0.08)).to(p.dtype))
    return moe.to(dt).eval()


def _x(S, M, dt=torch.bfloat16, seed=1):
    x = torch.randn((S, M), generator=torch.Generator().manual_seed(seed))
    x[:, 7] *= 9
    return x.to(dt).to(DEV)


def _reference(moe, x, r):
    """Outputs and bounds of the block on 8-bit experts, given the routing."""
    specs = moe.deepspeed_moe.experts._specs()
    S, M = x.shape
    slot, idx, w = r.slot.cpu(), r.expert_idx.cpu(), r.weight.cpu()
    ref, tol = torch.zeros((S, M), dtype=D), torch.zeros((S, M), dtype=D)
    for e, sp in enumerate(specs):
        q1, s1, q2, s2 = [], [], None, None
        for lin in sp.fc1:
            v, b = R.quant(lin.weight.detach().cpu(), 128)
            q1.append(v.to(torch.float32).to(R.E4M3))
            s1.append(b.to(torch.uint8))
        v, b = R.quant(sp.fc2.weight.detach().cpu(), 128)
        q2, s2 = v.to(torch.float32).to(R.E4M3), b.to(torch.uint8).view(R.E8M0)
        b1 = torch.cat([lin.bias.detach().cpu() for lin in sp.fc1]) if sp.fc1[0].bias is not None else None
        b2 = sp.fc2.bias.detach().cpu() if sp.fc2.bias is not None else None
        for j in range(r.top_k):
            t = torch.nonzero((idx[:, j] == e) & (slot[:, j] >= 0)).flatten()
            if not t.numel():
                continue
            y, d = _ffn_ref(x.cpu()[t], torch.cat(q1), torch.cat(s1).view(R.E8M0), q2, s2, b1, b2,
                            "swiglu" if len(sp.fc1) == 2 else "gelu_new")
            d = d + R.half_step(x.dtype) * (y.abs() + d)                    # y is rounded before the combine
            g = w[t, j].to(x.dtype).to(D)[:, None]
            ref[t] += g * y
            tol[t] += g.abs() * d
    return ref, tol


@pytest.mark.parametrize("S", [1, 5, 33, 64, 65, 300])
@pytest.mark.parametrize("form,dt", [("swiglu", torch.bfloat16), ("gelu_new", torch.float16)])
def test_block_against_64_bits(S, form, dt):
    moe = _moe(form=form, dt=dt, eval_capacity_factor=0.6 if S == 300 else 2.0)     # at 300 tokens rows are dropped
    x = _x(S, 256, dt)
    with torch.no_grad():
        out16, la16, ec16 = moe(x)
        r16 = moe.deepspeed_moe.last_routing
        logits16, idx16, slot16 = moe.deepspeed_moe.gate.last_logits.clone(), r16.expert_idx.clone(), r16.slot.clone()
        la16, ec16 = la16.clone(), ec16.clone()
        moe.quantize_experts()
        out8, la8, ec8 = moe(x)
    r = moe.deepspeed_moe.last_routing
    assert torch.equal(moe.deepspeed_moe.gate.last_logits, logits16) and torch.equal(r.expert_idx, idx16) and torch.equal(r.slot, slot16)
    assert torch.equal(la8, la16) and torch.equal(ec8, ec16)
    ref, tol = _reference(moe, x, r)
    _check_ffn(out8, ref, tol)
    # 8 bits against 16: half a step of e4m3 on each of three operands in two products
    assert float((out8 - out16).float().norm() / out16.float().norm()) <= 5 * 2.0 ** -4
    with torch.no_grad():
        moe.quantize_experts(False)
        again = moe(x)[0]
    assert torch.equal(again, out16)


def test_general_path_and_top1():
    """Calls that the one-call path does not take: a hook on wg, a phase timer, top-1."""
    x = _x(40, 256)
    moe = _moe().quantize_experts()
    with torch.no_grad():
        want = moe(x)[0].clone()
        seen = []
        h = moe.deepspeed_moe.gate.wg.register_forward_hook(lambda m, i, o: seen.append(o.shape))
        assert torch.equal(moe(x)[0], want) and seen
        h.remove()
        top1 = _moe(k=1, use_rts=False).quantize_experts()
        out = top1(x)[0]
        ref, tol = _reference(top1, x, top1.deepspeed_moe.last_routing)
        _check_ffn(out, ref, tol)


@pytest.mark.parametrize("S", [1, 48, 200])
def test_normed_block_is_its_parts(S):
    moe = _moe().quantize_experts()
    nm = norm.RMSNorm(256, eps=1e-5, dtype=torch.bfloat16, device=DEV)
    with torch.no_grad():
        nm.weight.copy_(1 + 0.1 * torch.randn(256))
        x, r = _x(S, 256, seed=3).view(1, S, 256), _x(S, 256, seed=4).view(1, S, 256)
        out, la, ec, s = moe.forward_normed(x, r, nm)
        la, ec = la.clone(), ec.clone()
        rows, y, s2 = norm.add_rms_norm_fp8(x, r, nm.weight, 1e-5)
        lay = moe.deepspeed_moe
        ref = fp8.block_top2(y.view(S, 256), lay.gate.wg.weight, lay.last_routing.capacity, None, 0, True,
                             lay.experts.packed_fp8(x.device), -1, None, rows)
        assert torch.equal(out.view(S, 256), ref[0]) and torch.equal(s, s2) and torch.equal(ec, ref[2].exp_counts)
        moe.quantize_experts(False)
        o16, l16, e16, s16 = moe.forward_normed(x, r, nm)
        y16, _ = norm.add_rms_norm(x, r, nm.weight, 1e-5)
        assert torch.equal(o16, moe(y16)[0]) and torch.equal(s16, s) and torch.equal(e16, ec)
    # with gradients (16-bit experts): through the block, the norm and both inputs
    xg, rg = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
    o, la, ec, s = moe.forward_normed(xg, rg, nm)
    (o.float().sum() + s.float().sum() + la).backward()
    assert torch.equal(xg.grad, rg.grad) and bool(torch.isfinite(xg.grad).all()) and nm.weight.grad is not None


def test_changed_weights_are_quantised_again():
    moe = _moe().quantize_experts()
    x = _x(24, 256)
    with torch.no_grad():
        a = moe(x)[0].clone()
        first = moe.deepspeed_moe.experts._fp8
        assert torch.equal(moe(x)[0], a) and moe.deepspeed_moe.experts._fp8 is first
        sd = {k: v.clone() * (2 if "down_proj" in k else 1) for k, v in moe.state_dict().items()}
        moe.load_state_dict(sd)
        assert torch.equal(moe(x)[0], (a.float() * 2).to(a.dtype))         # a power of two moves only the exponents
        for p in moe.deepspeed_moe.experts.parameters():
            p.mul_(0)
        assert not bool(moe(x)[0].any())


def test_graphed_step_on_eight_bit_experts():
    moe = _moe(top2_2nd_expert_sampling=True).quantize_experts()
    x = _x(8, 256)
    g = GraphedMoE(moe, x, seed=77)
    g2 = GraphedMoE(moe, x, seed=77)
    for k in range(4):
        xk = (x.float() * (k + 1)).to(torch.bfloat16)
        a = [t.clone() for t in g(xk)]
        with torch.no_grad():
            moe(xk)                                                          # eager work between the replays
        torch.cuda.synchronize()
        b = g2(xk)
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])


def test_graph_follows_the_weights():
    moe = _moe().quantize_experts()
    x = _x(8, 256)
    g = GraphedMoE(moe, x)
    with torch.no_grad():
        a = g(x)[0].clone()
        assert torch.equal(a, moe(x)[0])
        for e in moe.deepspeed_moe.experts.deepspeed_experts:
            e.down_proj.weight.mul_(2)
        junk = [torch.full((1 << 20,), 77, dtype=torch.uint8, device=DEV) for _ in range(8)]    # what a freed copy would hold
        for _ in range(3):
            assert torch.equal(g(x)[0], (a.float() * 2).to(a.dtype))
            assert torch.equal(moe(x)[0], (a.float() * 2).to(a.dtype))
        del junk
        moe.quantize_experts(False)
        with pytest.raises(ValueError):
            g(x)
        moe.quantize_experts()
        with pytest.raises(ValueError):
            g(x)                                                             # another 8-bit copy


def test_refusals():
    moe = _moe().quantize_experts()
    x = _x(8, 256)
    with pytest.raises(NotImplementedError):
        moe(x)                                                               # gradients are on
    with torch.no_grad():
        out, la, ec = moe(x[:0])
        assert out.shape == (0, 256)
        with pytest.raises(NotImplementedError):
            moe.deepspeed_moe.experts(torch.zeros((1, 4, 2, 256), dtype=torch.bfloat16, device=DEV))
    with pytest.raises(NotImplementedError):
        moe_llava_amd.MoE(256, StableLMMLP(256, 320).to(torch.bfloat16), num_experts=4, ep_size=2, k=2).quantize_experts()


@pytest.mark.parametrize("S", [5, 130])
def test_masked_experts_follow_their_mask(S):
    """Experts with a channel mask: the number of gated channels can change between two calls of the same size."""
    torch.manual_seed(0)
    moe = moe_llava_amd.MoE(256, RePaMLP(256, 320).to(torch.bfloat16), num_experts=4, k=2, eval_capacity_factor=2.0,
                            min_capacity=0, top2_2nd_expert_sampling=False).to(DEV)
    with torch.no_grad():
        for n, p in moe.named_parameters():
            p.copy_((torch.randn(p.shape) * (0.3 if "wg" in n else 0.08)).to(p.dtype))
    moe = moe.to(torch.bfloat16).eval().quantize_experts()
    x = _x(S, 256)
    specs = moe.deepspeed_moe.experts
    with torch.no_grad():
        seen = []
        for ratio in (1.0, 0.5, 0.25, 1.0):
            for e in specs.deepspeed_experts:
                e.adjust_gated_ratio(ratio)
            out = moe(x)[0].clone()
            lay, r = moe.deepspeed_moe, moe.deepspeed_moe.last_routing
            ng = int(320 * ratio) if ratio < 1 else -1
            want = fp8.block_top2(x, lay.gate.wg.weight, r.capacity, None, 0, True, specs.packed_fp8(x.device), ng)[0]
            assert torch.equal(out, want)
            seen.append(out)
        assert torch.equal(seen[0], seen[3]) and not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
        if S == 5:
            g = GraphedMoE(moe, x)
            assert torch.equal(g(x)[0], seen[0])
            for e in specs.deepspeed_experts:
                e.adjust_gated_ratio(0.5)
            with pytest.raises(ValueError):
                g(x)


@pytest.mark.parametrize("eight", [False, True])
def test_two_graphs_of_one_layer_share_no_buffer(eight):
    moe = _moe()
    if eight:
        moe.quantize_experts()
    a, b = _x(8, 256, seed=5), _x(8, 256, seed=6)
    g1, g2 = GraphedMoE(moe, a), GraphedMoE(moe, a)
    with torch.no_grad():
        ra = [t.clone() for t in moe(a)[:3]]
        rb = [t.clone() for t in moe(b)[:3]]
        for _ in range(3):
            o1 = g1(a)
            torch.cuda.synchronize()
            o2 = g2(b)
            torch.cuda.synchronize()
            moe(a)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(o1, ra)) and all(torch.equal(p, q) for p, q in zip(o2, rb))


def test_a_forced_tile_that_the_products_lack(monkeypatch):
    """A tile forced for the 16-bit products that the 8-bit ones do not have leaves those to their rule."""
    from moe_llava_amd import ops
    moe = _moe().quantize_experts()
    x = _x(200, 256)
    with torch.no_grad():
        want = moe(x)[0].clone()
        try:
            monkeypatch.setenv("MOE_GEMM_TILE", "256,64")
            ops.reload_knobs()
            assert torch.equal(moe(x)[0], want)
        finally:
            monkeypatch.delenv("MOE_GEMM_TILE")
            ops.reload_knobs()


def test_flattened_parameters_are_followed():
    """Parameters that are views into somebody else's buffer: copied and quantised for each call."""
    moe, x = _moe(), _x(24, 256)
    ps = list(moe.deepspeed_moe.experts.parameters())
    flat = torch.cat([p.detach().reshape(-1) for p in ps])
    at = 0
    for p in ps:
        p.data = flat[at:at + p.numel()].view(p.shape)
        at += p.numel()
    same = _moe().quantize_experts()
    with torch.no_grad(), pytest.warns(UserWarning):
        moe.quantize_experts()
        a = moe(x)[0].clone()
    with torch.no_grad():
        assert torch.equal(a, same(x)[0])
        flat.mul_(0)
        assert not bool(moe(x)[0].any())


def test_two_streams_and_a_second_module():
    """The same layer on two streams, and another layer between: every call its own buffers."""
    m1, m2 = _moe().quantize_experts(), _moe(form="gelu_new", I=448).quantize_experts()
    x1, x2 = _x(32, 256, seed=8), _x(600, 256, seed=9)
    st = [torch.cuda.Stream() for _ in range(2)]
    with torch.no_grad():
        want = [m(x)[0].clone() for m, x in ((m1, x1), (m2, x2), (m2, x1), (m1, x2))]
        torch.cuda.synchronize()
        got = []
        for k in range(6):
            with torch.cuda.stream(st[k % 2]):
                got.append([m(x)[0] for m, x in ((m1, x1), (m2, x2), (m2, x1), (m1, x2))])
        torch.cuda.synchronize()
        for row in got:
            assert all(torch.equal(a, b) for a, b in zip(row, want))


@pytest.mark.parametrize("S", [3, 90])
def test_normed_block_shapes_and_fallbacks(S):
    """forward_normed without a residual, on rows with a stride, on 16-bit experts, top-1 and a width of 8-bit tails."""
    for M, kw in ((320, {}), (256, dict(k=1, use_rts=False))):
        moe = _moe(M=M, **kw).quantize_experts()
        nm = norm.RMSNorm(M, eps=1e-5, dtype=torch.bfloat16, device=DEV)
        x = _x(S, 2 * M, seed=12)[:, :M]
        with torch.no_grad():
            out, la, ec, s = moe.forward_normed(x, None, nm)
            la, ec = la.clone(), ec.clone()
            assert torch.equal(s, x)
            if not kw:                       # the norm's launch quantises its fp32 values, not the rounded 16-bit ones
                lay = moe.deepspeed_moe
                rows, y, _ = norm.add_rms_norm_fp8(x, None, nm.weight, 1e-5)
                want = fp8.block_top2(y, lay.gate.wg.weight, lay.last_routing.capacity, None, 0, True,
                                      lay.experts.packed_fp8(x.device), -1, None, rows)[0]
                assert torch.equal(out, want)
            want = moe(nm(x))
            assert (not kw or torch.equal(out, want[0])) and torch.equal(la, want[1]) and torch.equal(ec, want[2])
            moe.quantize_experts(False)
            out = moe.forward_normed(x, None, nm)[0]
            assert torch.equal(out, moe(nm(x))[0])


def test_normed_block_keeps_what_is_around_the_forward():
    """A subclass with a forward of its own and hooks on the module are not passed by."""
    class Scaled(moe_llava_amd.MoE):
        def forward(self, x, *args, **kwargs):
            out, l_aux, counts = super().forward(x, *args, **kwargs)
            return out * 2, l_aux, counts

    moe = _moe().quantize_experts()
    nm = norm.RMSNorm(256, eps=1e-5, dtype=torch.bfloat16, device=DEV)
    x, r = _x(20, 256, seed=3), _x(20, 256, seed=4)
    with torch.no_grad():
        want = moe(norm.add_rms_norm(x, r, nm.weight, 1e-5)[0])[0].clone()
        seen = []
        h = moe.register_forward_hook(lambda m, i, o: seen.append(1))
        assert torch.equal(moe.forward_normed(x, r, nm)[0], want) and seen
        h.remove()
        moe.__class__ = Scaled
        assert torch.equal(moe.forward_normed(x, r, nm)[0], want * 2)


@pytest.mark.parametrize("S", [8, 100])
def test_parameters_made_in_inference_mode_are_followed(S):
    """Such parameters keep no version: a change in place is found because they are quantised for every call."""
    with torch.inference_mode():
        moe = _moe().quantize_experts()
        x = _x(S, 256)
        a = moe(x)[0].clone()
        for e in moe.deepspeed_moe.experts.deepspeed_experts:
            e.down_proj.weight.mul_(2)
        assert torch.equal(moe(x)[0], (a.float() * 2).to(a.dtype))
