"""What 8-bit experts keep between calls, on the GPU: streams, modes, graphs."""
import pytest
import torch

from moe_llava_amd import norm
from moe_llava_amd.graph import GraphedMoE
from tests.test_gpu_fp8_block import _moe, _x

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("S", [8, 300])
@pytest.mark.parametrize("form", ["swiglu", "gelu_new"])
def test_first_call_and_refill_seen_from_two_streams(S, form):
    """No call before the streams part: the second stream's call is behind the filling that the first one launched."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x = _x(S, 1024)
    want = _moe(M=1024, I=2048, form=form).quantize_experts()
    moe = _moe(M=1024, I=2048, form=form).quantize_experts()
    torch.cuda.synchronize()
    with torch.no_grad():
        for _ in range(3):
            ref = want(x)[0].clone()
            torch.cuda.synchronize()
            with torch.cuda.stream(a):
                y = moe(x)[0]
            with torch.cuda.stream(b):
                z = moe(x)[0]
            torch.cuda.synchronize()
            assert torch.equal(y, ref) and torch.equal(z, ref)
            for m in (want, moe):
                for p in m.deepspeed_moe.experts.parameters():
                    p.mul_(0.5)
            torch.cuda.synchronize()


@pytest.mark.parametrize("S", [8, 100])
@pytest.mark.parametrize("form", ["swiglu", "gelu_new"])
def test_modes_mixed(S, form):
    """First call in inference mode, weights changed in it and outside, calls and replays in either mode."""
    moe, want = _moe(form=form).quantize_experts(), _moe(form=form).quantize_experts()
    x = _x(S, 256)
    with torch.inference_mode():
        assert torch.equal(moe(x)[0], want(x)[0])
        g = GraphedMoE(moe, x)
        for m in (moe, want):
            for p in m.deepspeed_moe.experts.parameters():
                p.mul_(2)
        assert torch.equal(moe(x)[0], want(x)[0]) and torch.equal(g(x)[0], want(x)[0])
    with torch.no_grad():
        for m in (moe, want):
            for p in m.deepspeed_moe.experts.parameters():
                p.mul_(0.5)
        ref = want(x)[0].clone()
        assert torch.equal(moe(x)[0], ref) and torch.equal(g(x)[0], ref)
    for p in moe.deepspeed_moe.experts.parameters():
        assert not p.is_inference()


def test_graphed_step_takes_inputs_of_any_mode():
    """Captured in inference mode, called outside it and with an input that requires a gradient (none is recorded)."""
    for eight in (False, True):
        moe = _moe()
        if eight:
            moe.quantize_experts()
        x = _x(8, 256)
        with torch.inference_mode():
            g = GraphedMoE(moe, x)
        with torch.no_grad():
            ref = moe(x)[0].clone()
        for _ in range(3):
            out = g(x.clone().requires_grad_(True))[0]
            assert torch.equal(out, ref) and not out.requires_grad and g.x.grad_fn is None


def _capture(fn):
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        out = fn()
    return g, out


@pytest.mark.parametrize("S", [8, 100])
def test_capture_without_an_eager_call_in_8_bits(S):
    """16-bit calls, then 8-bit experts whose first call is captured: eager calls before and between the replays are right,
    and the graph, which quantises at every replay, follows the weights."""
    moe, want = _moe(form="gelu_new"), _moe(form="gelu_new").quantize_experts()
    x = _x(S, 256)
    with torch.no_grad():
        moe(x)
        moe.quantize_experts()
        g, (out, _, _) = _capture(lambda: moe(x))
        for k in range(3):
            ref = want(x)[0].clone()
            assert torch.equal(moe(x)[0], ref)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ref) and torch.equal(moe(x)[0], ref)
            for m in (moe, want):
                for p in m.deepspeed_moe.experts.parameters():
                    p.mul_(0.5)


def test_first_call_is_not_captured():
    moe, x = _moe(), _x(8, 256)
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(g):
            moe(x)
    with torch.no_grad():
        assert torch.equal(moe(x)[0], _moe()(x)[0])                          # the module is as it was


@pytest.mark.parametrize("S", [8, 100])
@pytest.mark.parametrize("eight", [False, True])
def test_two_graphs_captured_by_hand(S, eight):
    """Two steps of one layer captured on one stream: neither writes what the other returned, and eager calls (here of enough
    different sizes that the kept plans are dropped) leave both alone."""
    moe = _moe()
    if eight:
        moe.quantize_experts()
    a, b = _x(S, 256, seed=5), _x(S, 256, seed=6)
    with torch.no_grad():
        ra, rb = [t.clone() for t in moe(a)], [t.clone() for t in moe(b)]
        (g1, o1), (g2, o2) = _capture(lambda: moe(a)), _capture(lambda: moe(b))
        for _ in range(3):
            g1.replay(), g2.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(o1, ra)) and all(torch.equal(p, q) for p, q in zip(o2, rb))
            g2.replay()
            for s in range(1, 40):
                moe(a[:s])
            g1.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(o1, ra)) and all(torch.equal(p, q) for p, q in zip(o2, rb))


def test_two_captured_steps_of_16_bit_experts_on_two_streams():
    """Sizes whose products cut their last round along K: each graph has a workspace of its own."""
    moe = _moe(M=1024, I=4096)
    a, b = _x(1500, 1024, seed=5), _x(1500, 1024, seed=6)
    with torch.no_grad():
        ra, rb = moe(a)[0].clone(), moe(b)[0].clone()
        (g1, o1), (g2, o2) = _capture(lambda: moe(a)), _capture(lambda: moe(b))
        st = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(5):
            for s, g in zip(st, (g1, g2)):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o1[0], ra) and torch.equal(o2[0], rb)


@pytest.mark.parametrize("S", [8, 100])
def test_normed_block_keeps_what_is_around_the_inner_layer(S):
    """A hook on, or a forward of, the layer inside the module may change what the experts get: the rows that the norm's launch
    wrote in 8 bits are not theirs then."""
    moe = _moe().quantize_experts()
    nm = norm.RMSNorm(256, eps=1e-5, dtype=torch.bfloat16, device=DEV)
    x, r = _x(S, 256, seed=3), _x(S, 256, seed=4)
    layer = moe.deepspeed_moe
    with torch.no_grad():
        y = norm.add_rms_norm(x, r, nm.weight, 1e-5)[0]
        want = moe(y * 2)[0].clone()
        h = layer.register_forward_pre_hook(lambda m, args: (args[0] * 2,) + args[1:])
        assert torch.equal(moe.forward_normed(x, r, nm)[0], want)
        h.remove()
        inner = layer.forward
        layer.forward = lambda a, used_token=None: inner(a * 2, used_token)
        assert torch.equal(moe.forward_normed(x, r, nm)[0], want)


@pytest.mark.parametrize("eight", [False, True])
def test_norms_in_front_of_the_block(eight):
    """torch's own norm with an eps runs as the kernel; without one, and a norm that scales by 1 + weight, as they are."""
    class OnePlus(torch.nn.RMSNorm):
        def forward(self, x):
            return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-5) * (1 + self.weight.float())).to(x.dtype)

    moe = _moe()
    if eight:
        moe.quantize_experts()
    x, r = _x(20, 256, seed=3), _x(20, 256, seed=4)
    mk = dict(dtype=torch.bfloat16, device=DEV)
    with torch.no_grad():
        w = (1 + 0.1 * torch.randn(256)).to(torch.bfloat16).to(DEV)
        own, theirs = norm.RMSNorm(256, 1e-5, **mk), torch.nn.RMSNorm(256, 1e-5, **mk)
        for nm in (own, theirs):
            nm.weight.copy_(w)
        a, b = moe.forward_normed(x, r, own), moe.forward_normed(x, r, theirs)
        assert torch.equal(a[0], b[0]) and torch.equal(a[3], b[3])
        for nm in (torch.nn.RMSNorm(256, **mk), torch.nn.RMSNorm(256, elementwise_affine=False), OnePlus(256, **mk)):
            out, la, ec, s = moe.forward_normed(x, r, nm)
            assert torch.equal(s, x + r) and torch.equal(out, moe(nm(x + r))[0])


@pytest.mark.parametrize("eight", [False, True])
def test_a_used_module_can_be_copied(eight):
    import copy
    moe, x = _moe(), _x(8, 256)
    if eight:
        moe.quantize_experts()
    with torch.no_grad():
        ref = moe(x)[0].clone()
        other = copy.deepcopy(moe)
        for p in other.deepspeed_moe.experts.parameters():
            p.mul_(0.5)
        assert torch.equal(moe(x)[0], ref) and not torch.equal(other(x)[0], ref)


@pytest.mark.parametrize("S", [8, 200])
@pytest.mark.parametrize("eight", [False, True])
def test_threads_with_streams_of_their_own(S, eight):
    """Four threads call one layer, first call included, each on its stream."""
    import threading
    ref, moe = _moe(), _moe()
    if eight:
        ref.quantize_experts(), moe.quantize_experts()
    xs = [_x(S, 256, seed=20 + i) for i in range(4)]
    with torch.no_grad():
        want = [ref(x)[0].clone() for x in xs]
    torch.cuda.synchronize()
    got, go = [None] * 4, threading.Barrier(4)

    def run(i):
        st = torch.cuda.Stream()
        go.wait()
        with torch.no_grad(), torch.cuda.stream(st):
            got[i] = [moe(xs[i])[0] for _ in range(20)]
        st.synchronize()

    ts = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    for g, w in zip(got, want):
        assert all(torch.equal(y, w) for y in g)
