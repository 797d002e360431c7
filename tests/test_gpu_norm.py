"""Residual addition + root-mean-square norm (moe_add_rms_norm_fwd / _bwd, moe_llava_amd.norm) against 64 bits.

Bounds.  s is one fp32 addition and one rounding: exact.  Everything behind it is fp32: a sum of M squares in a tree
(at most 64 sequential + 10 tree additions), a square root, a division and two products, together below 2^-18 relative (the
sum's relative error 74 * 2^-24 enters rstd halved); then half a step of the output's type."""
import pytest
import torch

from moe_llava_amd import _lib, norm
from tests import _fp8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = torch.float64
REL = 2.0 ** -18


def _data(S, M, dt, seed, wdt=None, big=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((S, M), generator=g)
    r = torch.randn((S, M), generator=g) * 3
    if big and M > 8:
        x[:, M // 3] *= 40
    w = 1 + 0.2 * torch.randn(M, generator=g)
    return x.to(dt), r.to(dt), w.to(wdt or dt)


def _ref(x, r, w, eps):
    s = (x.float() + r.float()).to(x.dtype) if r is not None else x
    f = s.to(D)
    rstd = 1.0 / torch.sqrt((f * f).mean(dim=1, keepdim=True) + eps)
    return s, f * rstd * w.to(D), rstd


SIZES = [(1, 1), (1, 7), (2, 16), (3, 64), (1, 2048), (5, 2560), (33, 1000), (4, 4096), (7, 4104), (2, 20000), (1, 65536),
         (4097, 512), (4099, 520), (5000, 2040), (4100, 4096), (4100, 2555)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,M", SIZES)
def test_forward(S, M, dt):
    for res in (True, False):
        x, r, w = _data(S, M, dt, S * 7 + M, torch.float32 if S % 2 else dt)
        xg, rg, wg = x.to(DEV), r.to(DEV), w.to(DEV)
        if res:
            y, s = norm.add_rms_norm(xg, rg, wg, eps=1e-5)
        else:
            y, s = norm.rms_norm(xg, wg, eps=1e-5), None
        rs, ry, _ = _ref(x, r if res else None, w, 1e-5)
        if res:
            assert torch.equal(s.cpu(), rs)
        R.check16(y, ry, REL * ry.abs(), f"y res={res}")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,M", [(1, 16), (1, 2048), (3, 144), (6, 2560), (2, 5632), (4099, 1040), (4100, 2048), (1, 20000)])
def test_eight_bit_output(S, M, dt):
    x, r, w = _data(S, M, dt, S + M)
    if S > 2:
        r[1] = -x[1]                            # a row of zeros
    rows, y, s = norm.add_rms_norm_fp8(x.to(DEV), r.to(DEV), w.to(DEV), eps=1e-6)
    rs, ry, _ = _ref(x, r, w, 1e-6)
    assert torch.equal(s.cpu(), rs)
    R.check16(y, ry, REL * ry.abs(), "y")
    assert tuple(rows.q.shape) == (S, M) and tuple(rows.scale.shape) == (S, R.nb(M))
    b = rows.scale.cpu().view(torch.uint8).to(torch.int64)
    lo, hi = R.scale_byte(R._top(ry) * (1 - REL)), R.scale_byte(R._top(ry) * (1 + REL))
    assert bool(((b >= lo) & (b <= hi)).all())
    # with the stored scale, every element is the rounding of a value within REL of the exact one (rounding is monotone)
    sc = R.spread(torch.exp2(b.to(D) - 127), S, M)
    q = rows.q.cpu().to(torch.float32).to(D)
    a, c = ry * (1 - REL) / sc, ry * (1 + REL) / sc
    assert bool((q >= R.e4m3(torch.minimum(a, c))).all()) and bool((q <= R.e4m3(torch.maximum(a, c))).all())
    only, none, _ = norm.add_rms_norm_fp8(x.to(DEV), r.to(DEV), w.to(DEV), want_y=False)
    assert none is None and torch.equal(only.q.view(torch.uint8), rows.q.view(torch.uint8))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S,M", [(1, 1), (1, 2048), (3, 17), (700, 2560), (5000, 512), (4100, 2043), (2, 20000)])
def test_gradients(S, M, dt):
    x, r, w = _data(S, M, dt, S * 3 + M, torch.float32 if M % 2 else dt)
    g = torch.Generator().manual_seed(S)
    dy, ds = torch.randn((S, M), generator=g).to(dt), torch.randn((S, M), generator=g).to(dt)
    xg, rg, wg = (t.to(DEV).requires_grad_(True) for t in (x, r, w))
    y, s = norm.add_rms_norm(xg, rg, wg, eps=1e-5)
    dx, dr, dw = torch.autograd.grad((y, s), (xg, rg, wg), (dy.to(DEV), ds.to(DEV)))
    assert torch.equal(dx, dr)
    # the formula, in 64 bits, by autograd of the definition (independent of the closed form in the kernel)
    s64 = (x.float() + r.float()).to(dt).to(D).requires_grad_(True)
    w64 = w.to(D).requires_grad_(True)
    y64 = s64 / torch.sqrt((s64 * s64).mean(dim=1, keepdim=True) + 1e-5) * w64
    rx, rw = torch.autograd.grad((y64, s64 * 1.0), (s64, w64), (dy.to(D), ds.to(D)))
    f = s64.detach()
    rstd = 1.0 / torch.sqrt((f * f).mean(dim=1, keepdim=True) + 1e-5)
    n, gg = f * rstd, dy.to(D) * w.to(D)
    # terms of dx, each within 2^-17 (twice the forward's bound: rstd enters twice)
    size = rstd * (gg.abs() + n.abs() * (gg * n).abs().mean(dim=1, keepdim=True)) + ds.to(D).abs()
    R.check16(dx, rx, 2.0 ** -17 * size, "dx")
    tol = 2.0 ** -17 * (dy.to(D) * n).abs().sum(dim=0)      # <= 74 sequential and tree additions, + rstd
    if w.dtype == torch.float32:
        assert bool(((dw.cpu().to(D) - rw).abs() <= tol).all())
    else:
        R.check16(dw, rw, tol, "dw")
    # and against differences of the 64-bit function, along one direction
    d = torch.randn((S, M), generator=g, dtype=D)
    h = 1e-5

    def loss(v):
        return (v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-5) * w.to(D) * dy.to(D)).sum() + (v * ds.to(D)).sum()
    diff = (loss(f + h * d) - loss(f - h * d)) / (2 * h)
    lim = ((2.0 ** -17 * size + R.half_step(dt) * rx.abs()) * d.abs()).sum() + 1e-6 * (rx * d).abs().sum() + 1e-6
    if M > 1:       # the third derivative of a one-column norm near zero is not small against h^2
        assert abs(float((dx.cpu().to(D) * d).sum() - diff)) <= float(lim) * 1.01 + 1e-5 * S * M


def test_gradients_of_one_output_only():
    x, r, w = _data(9, 264, torch.bfloat16, 5)
    xg, rg, wg = (t.to(DEV).requires_grad_(True) for t in (x, r, w))
    y, s = norm.add_rms_norm(xg, rg, wg)
    dy = torch.ones_like(y)
    a = torch.autograd.grad(y, (xg, rg, wg), dy, retain_graph=True)
    b = torch.autograd.grad((y, s), (xg, rg, wg), (dy, torch.zeros_like(s)), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    c = torch.autograd.grad(s, (xg, rg), torch.full_like(s, 2.0), retain_graph=True)
    assert bool((c[0] == 2).all()) and bool((c[1] == 2).all())
    dw, = torch.autograd.grad(s, (wg,), torch.ones_like(s), allow_unused=True, retain_graph=True)
    assert dw is None or not bool(dw.any())
    z = norm.rms_norm(xg, wg)
    gx, = torch.autograd.grad(z.float().sum(), xg)
    f = x.to(D).requires_grad_(True)
    ref, = torch.autograd.grad((f / torch.sqrt((f * f).mean(1, keepdim=True) + 1e-6) * w.to(D)).sum(), f)
    rstd = 1 / torch.sqrt((f * f).mean(1, keepdim=True) + 1e-6).detach()
    n = f.detach() * rstd
    size = rstd * (w.to(D).abs() + n.abs() * (w.to(D) * n).abs().mean(1, keepdim=True))
    R.check16(gx, ref, 2.0 ** -17 * size, "dx without residual")


def test_strides_shapes_and_empty():
    x, r, w = _data(24, 256, torch.bfloat16, 3)
    y0, s0 = norm.add_rms_norm(x.to(DEV), r.to(DEV), w.to(DEV))
    y3, s3 = norm.add_rms_norm(x.to(DEV).view(2, 3, 4, 256), r.to(DEV).view(2, 3, 4, 256), w.to(DEV))
    assert y3.shape == (2, 3, 4, 256) and torch.equal(y3.view(24, 256), y0) and torch.equal(s3.view(24, 256), s0)
    for pad, off in ((8, 0), (3, 0), (16, 1), (5, 3)):          # row strides and starts that rule wide loads out, or not
        xb = torch.zeros((24, 256 + pad + off), dtype=torch.bfloat16, device=DEV)
        xb[:, off:off + 256] = x.to(DEV)
        y, s = norm.add_rms_norm(xb[:, off:off + 256], r.to(DEV), w.to(DEV))
        assert torch.equal(y, y0) and torch.equal(s, s0)
        rows, y, s = norm.add_rms_norm_fp8(xb[:, off:off + 256], r.to(DEV), w.to(DEV))
        assert torch.equal(y, y0)
    yt, _ = norm.add_rms_norm(x.to(DEV).t().contiguous().t(), r.to(DEV), w.to(DEV))
    assert torch.equal(yt, y0)
    ye, se = norm.add_rms_norm(x.to(DEV)[:1].expand(24, 256), r.to(DEV), w.to(DEV))    # rows that share their memory
    assert torch.equal(ye[0], y0[0]) and tuple(ye.shape) == (24, 256)
    y, s = norm.add_rms_norm(torch.empty((0, 256), dtype=torch.bfloat16, device=DEV), torch.empty((0, 256), dtype=torch.bfloat16, device=DEV), w.to(DEV))
    assert y.shape == s.shape == (0, 256)
    xe = torch.empty((0, 256), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    wg = w.to(DEV).requires_grad_(True)
    gw, = torch.autograd.grad(norm.rms_norm(xe, wg).sum(), wg)
    assert not bool(gw.any())


def test_extreme_rows():
    x = torch.zeros((6, 512), dtype=torch.bfloat16)
    x[1] = 3e38                                  # squares overflow fp32: y = x * 0
    x[2, 5] = float("inf")
    x[3, 300] = float("nan")
    x[4] = 1e-30
    x[5] = torch.linspace(-1, 1, 512).to(torch.bfloat16)
    w = torch.ones(512, dtype=torch.bfloat16)
    rows, y, _ = norm.add_rms_norm_fp8(x.to(DEV), None, w.to(DEV), eps=1e-6)
    y, q, b = y.cpu().float(), rows.q.cpu().float(), rows.scale.cpu().view(torch.uint8)
    assert not bool(y[0].any()) and not bool(q[0].any())
    assert not bool(y[1].any())
    assert bool(torch.isnan(y[2, 5])) and not bool(y[2, :5].any())
    assert bool(torch.isnan(q[2, :128]).all()) and int(b[2, 0]) == 255 and not bool(torch.isnan(q[2, 128:]).any())
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(q[3]).all()) and bool((b[3] == 255).all())
    ref = _ref(x[4:], None, w, 1e-6)[1]
    R.check16(y[4:].to(torch.bfloat16), ref, REL * ref.abs())


def test_graph_replay_and_streams():
    x, r, w = (t.to(DEV) for t in _data(65, 1040, torch.bfloat16, 11))
    want = norm.add_rms_norm_fp8(x, r, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm.add_rms_norm_fp8(x, r, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.cuda.graph(graph):
        rows, y, s = norm.add_rms_norm_fp8(xs, r, w)
    for k in range(4):
        xk = (x.float() * (k + 1)).to(torch.bfloat16)
        xs.copy_(xk)
        graph.replay()
        torch.cuda.synchronize()
        want = norm.add_rms_norm_fp8(xk, r, w)
        assert torch.equal(y, want[1]) and torch.equal(s, want[2])
        assert torch.equal(rows.q.view(torch.uint8), want[0].q.view(torch.uint8))
        assert torch.equal(rows.scale.view(torch.uint8), want[0].scale.view(torch.uint8))


def test_weight_gradient_is_the_same_every_time():
    x, r, w = _data(9000, 512, torch.bfloat16, 2)
    xg, rg, wg = (t.to(DEV).requires_grad_(True) for t in (x, r, w.float()))
    got = []
    for _ in range(3):
        y, s = norm.add_rms_norm(xg, rg, wg)
        got.append(torch.autograd.grad(y.float().square().sum(), wg)[0])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_refusals_on_the_gpu():
    x, r, w = (t.to(DEV) for t in _data(4, 64, torch.bfloat16, 1))
    with pytest.raises(ValueError):
        norm.add_rms_norm(x, r[:3], w)
    with pytest.raises(ValueError):
        norm.add_rms_norm(x, r.half(), w)
    with pytest.raises(ValueError):
        norm.add_rms_norm(x, r, w[:32])
    with pytest.raises(TypeError):
        norm.add_rms_norm(x, r, w.half())
    with pytest.raises(TypeError):
        norm.rms_norm(x.float(), w)
    with pytest.raises(ValueError):
        norm.add_rms_norm_fp8(x[:, :40], r[:, :40], w[:40])        # 40 columns: not a multiple of 16
    with pytest.raises(NotImplementedError):
        norm.add_rms_norm_fp8(x.clone().requires_grad_(True), r, w)
    with pytest.raises(_lib.MoEKernelError):
        norm.rms_norm(x.cpu(), w)


def test_gradients_of_both_inputs_are_their_own():
    """x and residual have the same gradient, but neither owns the other's; one leaf in both places gets it twice."""
    x, r, w = (t.to(DEV) for t in _data(9, 264, torch.bfloat16, 6))
    xg, rg = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
    y, s = norm.add_rms_norm(xg, rg, w)
    (y.float().sum() + s.float().sum()).backward()
    assert torch.equal(xg.grad, rg.grad) and xg.grad.data_ptr() != rg.grad.data_ptr()
    keep = rg.grad.clone()
    xg.grad.zero_()
    assert torch.equal(rg.grad, keep)
    both = x.clone().requires_grad_(True)
    y, s = norm.add_rms_norm(both, both, w)
    d1, = torch.autograd.grad(y.float().sum(), both, retain_graph=True)
    xa, xb = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    da, db = torch.autograd.grad(norm.add_rms_norm(xa, xb, w)[0].float().sum(), (xa, xb))
    assert torch.equal(d1, da + db)
    # the new stream is saved for the backward pass: changing it in place is refused
    y, s = norm.add_rms_norm(xg, rg, w)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError):
        y.float().sum().backward()


def test_offsets_past_32_bits():
    """More than 2^32 elements: every copy of the same 1024 rows gets the same result, forward, 8-bit output and backward."""
    S, M, P = 2 ** 21 + 5, 2064, 1024
    x, r, w = (t.to(DEV) for t in _data(P, M, torch.bfloat16, 7))
    big_x, big_r = (t.repeat(S // P + 1, 1)[:S] for t in (x, r))

    def same(t, u):
        assert torch.equal(t[:S // P * P].view((S // P, P) + t.shape[1:]), u.expand((S // P,) + u.shape))
        assert torch.equal(t[S // P * P:], u[:S % P])

    with torch.no_grad():
        rows, y, s = norm.add_rms_norm_fp8(big_x, big_r, w)
        # 4096 rows and more take the one-wave form: the copies are compared with its own first rows
        for t in (rows.q.view(torch.uint8), rows.scale.view(torch.uint8), y, s):
            same(t, t[:P].clone())
        small = norm.add_rms_norm_fp8(x, r, w)
        assert torch.equal(s[:P], small[2])
        R.check16(y[-P:], small[1].roll(-(S % P), 0).cpu().to(D), 2.0 ** -7 * small[1].roll(-(S % P), 0).cpu().to(D).abs(), "y")
        del rows, y, s, big_r
    xg = big_x.requires_grad_(True)
    y = norm.rms_norm(xg, w)
    dx, = torch.autograd.grad(y, xg, big_x.detach())
    same(dx, dx[:P].clone())
