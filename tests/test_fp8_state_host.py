"""The state that 8-bit experts keep between calls (the packed 16-bit weights, the 8-bit copy of them), on the CPU: the
quantisation itself is replaced by a stand-in that records what it was asked to do."""
import copy
import pickle

import pytest
import torch

import moe_llava_amd
from moe_llava_amd import fp8, ops
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


class _Stream:
    """Stand-in of a stream: what was launched on it, in order, with the waits between."""
    def __init__(self, log, name):
        self.log, self.name, self.past = log, name, set()

    def run(self, what):
        self.past.add(what)
        self.log.append((self.name, what))

    def record_event(self):
        return frozenset(self.past)

    def wait_event(self, past):
        self.past |= past

    def wait_stream(self, other):
        self.past |= other.past


@pytest.fixture
def streams(monkeypatch, made):
    """Three streams of a pretended device; ``use(i)`` makes one current, fillings are launched on the current one."""
    st = [_Stream([], i) for i in range(3)]
    now = [0]
    monkeypatch.setattr(ops, "_stream_key", lambda dev: now[0])
    monkeypatch.setattr(ops, "_torch_stream", lambda dev: st[now[0]])
    fill = fp8.quantize_weight

    def quantize_weight(w, projections=1, out=None):
        res = fill(w, projections, out)
        st[now[0]].run(("fill", len(made)))
        return res

    monkeypatch.setattr(fp8, "quantize_weight", quantize_weight)

    def use(i):
        now[0] = i
        return st[i]

    return use


def test_another_stream_is_behind_the_first_filling(streams, made):
    ex = _experts()
    streams(0)
    ex.packed_fp8(CPU)
    for i in (1, 2, 1, 0):
        s = streams(i)
        ex.packed_fp8(CPU)
        assert {("fill", 1), ("fill", 2)} <= s.past and len(made) == 2


def test_refilling_is_ordered_both_ways(streams, made):
    """A refill runs behind what other streams launched before it, and in front of what they launch after it."""
    ex = _experts()
    streams(0)
    ex.packed_fp8(CPU)
    s1 = streams(1)
    ex.packed_fp8(CPU)
    s1.run("product")
    with torch.no_grad():
        ex.deepspeed_experts[0].up_proj.weight.mul_(2)
    s2 = streams(2)
    ex.packed_fp8(CPU)
    assert "product" in s2.past and len(made) == 4
    for i in (0, 1):
        s = streams(i)
        ex.packed_fp8(CPU)
        assert {("fill", 3), ("fill", 4)} <= s.past and len(made) == 4


def test_a_copy_of_the_module_makes_its_own(made):
    ex = _experts()
    a = ex.packed_fp8(CPU)
    ex._fp8[4].done = lambda: None                       # stands for an event, which no copy can hold
    for other in (copy.deepcopy(ex), pickle.loads(pickle.dumps(ex))):
        assert other.fp8 and other._fp8 is None and ex._fp8[2] is a
        b = other.packed_fp8(CPU)
        assert b is not a and torch.equal(b[1], a[1])


@pytest.mark.parametrize("again", ["packed", "packed_unchanged", "packed_fp8"])
def test_another_stream_is_behind_the_packing(streams, monkeypatch, again):
    ex = _experts(eight=again == "packed_fp8")
    s0 = streams(0)
    copy_in = ex._copy_in
    monkeypatch.setattr(ex, "_copy_in", lambda *a: (copy_in(*a), s0.run("pack"))[0])
    pk = ex.packed(CPU)
    ex._remember_fast(ex._specs(), pk)
    s1 = streams(1)
    assert "pack" not in s1.past
    getattr(ex, again)(*(() if again == "packed_unchanged" else (CPU,)))
    assert "pack" in s1.past


def test_a_capture_leaves_the_copy_alone(monkeypatch, made):
    """Quantised in a capture (no copy yet, or a stale one): tensors of the graph's own, never what other calls read."""
    ex = _experts()
    capture = lambda on: monkeypatch.setattr(ops, "_capturing", lambda dev: on)
    capture(True)
    with pytest.raises(RuntimeError, match="capture"):
        ex.packed(CPU)
    with pytest.raises(RuntimeError, match="capture"):
        ex.packed_fp8(CPU)
    capture(False)
    ex.packed(CPU)
    capture(True)
    a = ex.packed_fp8(CPU)
    assert ex._fp8 is None and len(made) == 2
    capture(False)
    b = ex.packed_fp8(CPU)
    assert b is not a and len(made) == 4
    capture(True)
    assert ex.packed_fp8(CPU) is b and len(made) == 4                        # up to date: the graph reads the copy
    with torch.no_grad():
        ex.deepspeed_experts[1].down_proj.weight.mul_(2)
    c = ex.packed_fp8(CPU)
    assert c is not b and all(out is None for _, out in made[4:])
    capture(False)
    assert ex.packed_fp8(CPU) is b and len(made) == 8


@pytest.mark.parametrize("eight", [False, True])
def test_captured_decode_steps_keep_no_plan(monkeypatch, made, eight):
    """Every captured step gets a plan (the step's buffers) of its own; steps outside a capture share theirs."""
    from moe_llava_amd import sharded_moe
    plans = []

    class Plan:
        def __init__(self, layer, x, packed, st):
            self.packed, self.logits, self.exp_counts, self.routing, self.l_aux = packed, None, None, None, None
            plans.append(self)

        def run(self, gate, x, rows8=None):
            self.ran = True
            return x

    monkeypatch.setattr(sharded_moe, "_DecodePlan", Plan)
    monkeypatch.setattr(ops, "_stream_ptr", lambda t: 5)
    moe = moe_llava_amd.MoE(64, StableLMMLP(64, 64).to(torch.bfloat16), num_experts=2, k=2)
    layer = moe.quantize_experts(eight).deepspeed_moe
    x = torch.zeros((1, 64), dtype=torch.bfloat16)
    step = lambda: layer._decode_step(x, x, 1)
    step(), step()
    assert len(plans) == 1
    monkeypatch.setattr(ops, "_capturing", lambda dev: True)
    step(), step()
    assert len(plans) == 3 and all(p.ran for p in plans)
    assert list(layer.__dict__["_decode_plans"].values()) == plans[:1]
    monkeypatch.setattr(ops, "_capturing", lambda dev: False)
    step()
    assert len(plans) == 3


@pytest.mark.parametrize("eight", [False, True])
def test_a_decode_step_runs_on_its_device(monkeypatch, eight):
    """The library launches on the current device, which need not be the one that the tokens are on."""
    import contextlib
    from moe_llava_amd import _lib, sharded_moe
    current, ran_on = ["other"], []

    @contextlib.contextmanager
    def on(dev):
        current.append(dev)
        yield
        current.pop()

    monkeypatch.setattr(ops, "_on", on)
    plan = object.__new__(sharded_moe._DecodePlan)
    plan.args, plan.refs = _lib.BlockTop2Args(), (None,)
    plan.q = _lib.Fp8Experts() if eight else None
    plan.S, plan.M, plan.dtype, plan.dev, plan.sampling = 1, 64, torch.bfloat16, CPU, False
    plan.fn = lambda *a: ran_on.append(current[-1]) or 0
    gate = moe_llava_amd.TopKGate(64, 2, k=2)
    plan.run(gate, torch.zeros((1, 64), dtype=torch.bfloat16))
    assert ran_on == [CPU]


def test_captured_launches_share_no_splitk_workspace(monkeypatch):
    from types import SimpleNamespace
    monkeypatch.setattr(ops, "_SPLITK_BYTES", 4096)
    monkeypatch.setattr(ops, "_SPLITK_WS", ops._Workspaces())
    t = SimpleNamespace(is_cuda=True, device=CPU)
    eager = ops._splitk_ws(t, 7)
    assert ops._splitk_ws(t, 7)[0] == eager[0] != ops._splitk_ws(t, 8)[0]
    monkeypatch.setattr(ops, "_capturing", lambda dev: True)
    held = [ops._splitk_ws(t, 7) for _ in range(2)]
    assert len({eager[0], held[0][0], held[1][0]}) == 3 and all(h[2].data_ptr() == h[0] for h in held)
    assert len(ops._SPLITK_WS.kept) == 2


def test_a_copy_of_the_layer_has_no_plans():
    from moe_llava_amd import _lib
    moe = moe_llava_amd.MoE(64, StableLMMLP(64, 64).to(torch.bfloat16), num_experts=2, k=2)
    plans = moe.deepspeed_moe.__dict__["_decode_plans"] = {0: _lib.BlockTop2Args()}
    for other in (copy.deepcopy(moe), pickle.loads(pickle.dumps(moe))):
        assert "_decode_plans" not in other.deepspeed_moe.__dict__
        assert all(torch.equal(a, b) for a, b in zip(other.parameters(), moe.parameters()))
    assert moe.deepspeed_moe._decode_plans is plans


def _threads(n, fn):
    """fn(i) in n threads at once; what they returned."""
    import threading
    out, go = [None] * n, threading.Barrier(n)

    def run(i):
        go.wait()
        out[i] = fn(i)

    ts = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    return out


@pytest.mark.parametrize("eight", [False, True])
def test_first_calls_of_several_threads(monkeypatch, made, eight):
    """One packing and one quantisation, and parameters that all lie in the buffers that the calls got."""
    import time
    ex = _experts(eight=eight)
    ref = [p.detach().clone() for p in ex.parameters()]
    copy_in = ex._copy_in
    monkeypatch.setattr(ex, "_copy_in", lambda *a: (time.sleep(0.05), copy_in(*a)))      # the threads meet in here
    got = _threads(4, lambda i: ex.packed_fp8(CPU) if eight else ex.packed(CPU))
    assert all(a is b for g in got for a, b in zip(g, got[0])) and len(made) == (2 if eight else 0)
    own = {t.untyped_storage().data_ptr() for t in ex._packed.values() if t is not None}
    assert all(p.untyped_storage().data_ptr() in own for p in ex.parameters())
    assert all(torch.equal(a, b) for a, b in zip(ref, ex.parameters()))


def test_a_thread_keeps_its_stream(monkeypatch):
    """The stream that a forward looks up once is that thread's, whatever other threads run meanwhile."""
    import threading
    from types import SimpleNamespace
    mine = threading.local()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: SimpleNamespace(cuda_stream=mine.stream))
    t = SimpleNamespace(is_cuda=True, device=SimpleNamespace(index=0))
    both = threading.Barrier(2)

    def run(i):
        mine.stream = 100 + i
        with ops.stream_scope(t):
            both.wait()
            got = ops._stream_ptr(t)
            both.wait()
        return got

    assert _threads(2, run) == [100, 101]


@pytest.mark.parametrize("eight", [False, True])
def test_threads_on_one_stream_have_plans_of_their_own(monkeypatch, made, eight):
    from moe_llava_amd import sharded_moe

    class Plan:
        def __init__(self, layer, x, packed, st):
            self.packed, self.logits, self.exp_counts, self.routing, self.l_aux = packed, None, None, None, None

        def run(self, gate, x, rows8=None):
            seen.append(self)
            return x

    seen = []
    monkeypatch.setattr(sharded_moe, "_DecodePlan", Plan)
    monkeypatch.setattr(ops, "_stream_ptr", lambda t: 5)
    layer = moe_llava_amd.MoE(64, StableLMMLP(64, 64).to(torch.bfloat16), num_experts=2, k=2).quantize_experts(eight).deepspeed_moe
    x = torch.zeros((1, 64), dtype=torch.bfloat16)
    layer._decode_step(x, x, 1)
    _threads(2, lambda i: (layer._decode_step(x, x, 1), layer._decode_step(x, x, 1)))
    assert len(seen) == 5 and len(set(map(id, seen))) == 3


def test_threads_on_one_stream_share_no_splitk_workspace(monkeypatch):
    from types import SimpleNamespace
    monkeypatch.setattr(ops, "_SPLITK_BYTES", 4096)
    t = SimpleNamespace(is_cuda=True, device=CPU)
    mine = ops._splitk_ws(t, 7)
    held = _threads(3, lambda i: (ops._splitk_ws(t, 7), ops._splitk_ws(t, 7)))
    assert all(a[0] == b[0] for a, b in held) and len({mine[0]} | {a[0] for a, _ in held}) == 4
