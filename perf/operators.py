"""Measured cases of the 8-bit operators around the expert MLP.

Three families, in the order in which a decoder layer runs them:

* ``norm``: residual addition and root-mean-square norm of the hidden states in front of the MLP, leaving 16-bit rows, or
  8-bit rows with a scale for every 128 columns, or (training) the gradients of inputs and weight;
* ``linear``: one matrix product, or one per expert over ragged groups of rows, with e4m3 operands, a scale for every
  1 x 128 block of the activations and every 128 x 128 block of the weights; forward, and the input gradient through
  frozen 8-bit weights (scales are powers of two, held as exponents in 8 bits: the smallest that brings the block's
  largest magnitude to 448 or below, so scaling rounds nothing);
* ``ffn``: the whole expert MLP of a routed batch (rows gathered through the dispatch index, first products, SwiGLU or
  gelu_new, requantisation, second product).

``own`` chooses between the plain form below (elementary torch operations in 32 bits) and the package's operators.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 128           # columns (activations) or rows x columns (weights) that share a scale
E4M3_MAX = 448.0
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
MOST_FLOPS = 3.2e12   # a pass of the largest listed case


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decode step in front of an 8-bit MoE block (StableLM width): pure latency
        dict(name="norm_fp8_decode", op="norm", mode="fp8", S=1, M=2048, dt="bf16"),
        # a prompt of 4 x 576 image tokens + 128 text tokens less a few, Phi width, fp16 checkpoint
        dict(name="norm_fp8_prompt", op="norm", mode="fp8", S=2411, M=2560, dt="f16"),
        # 64 prompts of 576 + 128 tokens, 16-bit output (a block whose experts stay in 16 bits)
        dict(name="norm_batch", op="norm", mode="plain", S=45056, M=2048, dt="bf16"),
        # a training step over 32 prompts: outputs and the gradients of both inputs and the norm's weight
        dict(name="norm_train", op="norm", mode="train", S=22528, M=2048, dt="bf16"),
        # a projection of odd sizes on the rows of a short prompt, rows strided inside a wider buffer
        dict(name="linear_odd", op="linear", mode="forward", G=1, S=333, K=1008, N=1003, dt="bf16", bias=True, pad=16),
        # the dense MLP's up projection of a residual MoE layer over 32 prompts
        dict(name="linear_batch", op="linear", mode="forward", G=1, S=22528, K=2048, N=5632, dt="bf16", bias=False, pad=0),
        # ragged groups of 8 experts, forward and input gradient (adapters trained around frozen 8-bit experts)
        dict(name="linear_grouped_train", op="linear", mode="train", G=8, S=11264, K=2560, N=2048, dt="bf16", bias=True, pad=0),
        # the expert MLP of one decode step: one token, two of four experts
        dict(name="ffn_decode_1", op="ffn", S=1, M=2048, I=5632, E=4, act="swiglu", dt="bf16", bias=False),
        # a decode step of 32 requests
        dict(name="ffn_decode_32", op="ffn", S=32, M=2048, I=5632, E=4, act="swiglu", dt="bf16", bias=False),
        # one prompt of 576 image + 128 text tokens
        dict(name="ffn_prompt", op="ffn", S=704, M=2048, I=5632, E=4, act="swiglu", dt="bf16", bias=False),
        # Phi-form experts (biases, gelu_new) on 729 image tokens + text, 4 prompts, fp16
        dict(name="ffn_phi", op="ffn", S=3427, M=2560, I=10240, E=4, act="gelu_new", dt="f16", bias=True),
        # 32 prompts of 576 + 128 tokens: the batch that the 16-bit block is benchmarked on
        dict(name="ffn_batch", op="ffn", S=22528, M=2048, I=5632, E=4, act="swiglu", dt="bf16", bias=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "linear", "linear", "ffn", "ffn"))
    dt = rng.choice(("bf16", "bf16", "f16"))
    if op == "norm":
        mode = rng.choice(("fp8", "plain", "train"))
        M = rng.choice((256, 2048, 2560, 4096, _log(rng, 64, 5120), 16 * _log(rng, 4, 320)))
        if mode == "fp8":
            M = (M + 15) // 16 * 16
        return dict(op=op, mode=mode, S=_log(rng, 1, 45056 * 2048 // max(M, 2048)), M=M, dt=dt)
    if op == "linear":
        mode = rng.choice(("forward", "train"))
        G = rng.choice((1, 1, 2, 4, 8))
        K = 16 * _log(rng, 4, 640)
        N = _log(rng, 64, 10240)
        if mode == "train":
            N = (N + 15) // 16 * 16
        passes = 2 if mode == "train" else 1
        most = max(1, min(45056, int(MOST_FLOPS / (2.0 * K * N * passes * 4))))
        return dict(op=op, mode=mode, G=G, S=_log(rng, 1, most), K=K, N=N, dt=dt, bias=rng.random() < 0.5,
                    pad=rng.choice((0, 0, 8, 64)))
    act = rng.choice(("swiglu", "swiglu", "gelu_new"))
    M, I = rng.choice(((2048, 5632), (2560, 10240), (2048, 5504), (16 * _log(rng, 8, 128), 16 * _log(rng, 8, 256))))
    E = rng.choice((2, 4, 4, 8))
    per = 2.0 * 2 * M * I * (3 if act == "swiglu" else 2)          # flops of one token
    return dict(op=op, S=_log(rng, 1, max(1, min(22528, int(MOST_FLOPS / per)))), M=M, I=I, E=E, act=act, dt=dt,
                bias=act == "gelu_new")


def _up(n, m):
    return (n + m - 1) // m


def work(case):
    if case["op"] == "norm":
        S, M = case["S"], case["M"]
        el = S * M
        if case["mode"] == "fp8":       # x, residual in; residual, rows in 16 bits, rows in 8 bits and their scales out
            return {"bytes": el * (2 + 2 + 2 + 2 + 1) + S * _up(M, BLOCK), "flops": 6 * el}
        if case["mode"] == "plain":
            return {"bytes": el * 8, "flops": 5 * el}
        # forward: x, residual in, y, sum out; backward: dy, dsum, sum in, dx out
        return {"bytes": el * 16 + 8 * M, "flops": 14 * el}
    if case["op"] == "linear":
        G, S, K, N = case["G"], case["S"], case["K"], case["N"]
        b = S * K * 2 + G * N * K + G * _up(N, BLOCK) * _up(K, BLOCK) + S * N * 2 + (G * N * 2 if case["bias"] else 0)
        f = 2.0 * S * K * N
        if case["mode"] == "train":     # dy in, dx out, the weights a second time
            b += S * N * 2 + S * K * 2 + G * N * K
            f *= 2
        return {"bytes": b, "flops": f}
    S, M, I, E = case["S"], case["M"], case["I"], case["E"]
    n1 = 2 * I if case["act"] == "swiglu" else I
    active = min(E, 2 * S)
    rows = 2 * S
    b = S * M * 2 + active * (n1 * M + M * I) + rows * M * 2 + rows * 4
    return {"bytes": b, "flops": 2.0 * rows * (n1 * M + M * I)}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _exponent(top):
    """Exponents of the scales of blocks whose largest magnitude is `top`: 448 = 0.875 * 2**9."""
    m, ex = torch.frexp(top)
    return torch.where(top > 0, ex - 9 + (m > E4M3_MAX / 512).to(ex.dtype), -126).clamp_min(-126)


def _pow2(ex):
    """2**ex in fp32, exactly, for -126 <= ex <= 127."""
    return ((ex + 127).to(torch.int32) << 23).view(torch.float32)


def _weight(g, groups, n, k, parts=1):
    """e4m3 weights [groups, parts * n, k] and the exponents of their scales [groups, parts * ceil(n/128), ceil(k/128)],
    as a checkpoint holds them (each part quantised by itself)."""
    nb, kb = _up(n, BLOCK), _up(k, BLOCK)
    q = torch.empty((groups, parts * n, k), dtype=torch.float8_e4m3fn, device=DEV)
    s = torch.empty((groups, parts * nb, kb), dtype=torch.uint8, device=DEV)
    for e in range(groups):
        for p in range(parts):
            w = torch.randn((n, k), generator=g, device=DEV) * (0.6 / math.sqrt(k))
            w *= torch.exp(0.3 * torch.randn((n, 1), generator=g, device=DEV))      # rows of different size
            wp = torch.zeros((nb * BLOCK, kb * BLOCK), device=DEV)
            wp[:n, :k] = w
            blk = wp.view(nb, BLOCK, kb, BLOCK)
            ex = _exponent(blk.abs().amax(dim=(1, 3)))
            q[e, p * n:(p + 1) * n] = ((blk * _pow2(-ex)[:, None, :, None])
                                       .view(nb * BLOCK, kb * BLOCK)[:n, :k].to(torch.float8_e4m3fn))
            s[e, p * nb:(p + 1) * nb] = (ex + 127).to(torch.uint8)
    return q, s.view(torch.float8_e8m0fnu)


def _hidden(g, S, M, dt, pad=0):
    """Hidden states: normal, with a few channels far larger than the rest, rows inside a buffer `pad` columns wider."""
    x = torch.randn((S, M + pad), generator=g, device=DEV)
    x[:, torch.randint(0, M, (max(1, M // 256),), generator=g, device=DEV)] *= 12.0
    return x.to(dt)[:, :M]


def _ragged(g, rows, groups):
    """`rows` split over `groups` unevenly; the third group of a longer list stays empty."""
    p = torch.rand(groups, generator=g, device=DEV) + 0.2
    if groups > 3:
        p[2] = 0.0
    c = (p / p.sum() * rows).floor().to(torch.int64)
    c[0] += rows - c.sum()
    return [int(v) for v in c.tolist()]


def prepare(case, seed):
    g = _gen(seed)
    dt = DT[case["dt"]]
    st = dict(case=case)
    if case["op"] == "norm":
        S, M = case["S"], case["M"]
        st["x"] = _hidden(g, S, M, dt)
        st["res"] = (_hidden(g, S, M, dt).float() * 2).to(dt)
        st["w"] = (1.0 + 0.1 * torch.randn(M, generator=g, device=DEV)).to(dt)
        if case["mode"] == "train":
            st["dy"] = (torch.randn((S, M), generator=g, device=DEV) * 0.1).to(dt)
            st["ds"] = (torch.randn((S, M), generator=g, device=DEV) * 0.1).to(dt)
            for n in ("x", "res", "w"):
                st[n].requires_grad_(True)
        return st
    if case["op"] == "linear":
        G, S, K, N = case["G"], case["S"], case["K"], case["N"]
        st["x"] = _hidden(g, S, K, dt, case["pad"])
        st["q"], st["s"] = _weight(g, G, N, K)
        st["b"] = (torch.randn((G, N), generator=g, device=DEV) * 0.1).to(dt) if case["bias"] else None
        st["counts"] = _ragged(g, S, G)
        st["offs"] = torch.tensor([sum(st["counts"][:i]) for i in range(G + 1)], dtype=torch.int32, device=DEV)
        if case["mode"] == "train":
            st["x"] = st["x"].detach().requires_grad_(True)
            st["dy"] = (torch.randn((S, N), generator=g, device=DEV) * 0.1).to(dt)
        return st
    S, M, I, E = case["S"], case["M"], case["I"], case["E"]
    swiglu = case["act"] == "swiglu"
    st["x"] = _hidden(g, S, M, dt)
    st["q1"], st["s1"] = _weight(g, E, I, M, 2 if swiglu else 1)
    st["q2"], st["s2"] = _weight(g, E, M, I)
    st["b1"] = (torch.randn((E, I), generator=g, device=DEV) * 0.1).to(dt) if case["bias"] else None
    st["b2"] = (torch.randn((E, M), generator=g, device=DEV) * 0.1).to(dt) if case["bias"] else None
    # two different experts a token, some experts busier than others; rows sorted by expert, token order inside
    z = torch.randn((S, E), generator=g, device=DEV) + torch.linspace(0.5, 0.0, E, device=DEV)
    two = z.topk(2, dim=1).indices.reshape(-1)
    order = torch.sort(two, stable=True).indices
    st["perm"] = order.to(torch.int32)
    cnt = torch.bincount(two, minlength=E)
    st["counts"] = [int(v) for v in cnt.tolist()]
    st["offs"] = torch.tensor([sum(st["counts"][:i]) for i in range(E + 1)], dtype=torch.int32, device=DEV)
    return st


# ------------------------------------------------------------------------------------------------ plain form
def _quant(x):
    """Rows in fp32 -> (e4m3 [R, K], exponents [R, ceil(K/128)])."""
    R, K = x.shape
    kb = _up(K, BLOCK)
    xp = torch.nn.functional.pad(x, (0, kb * BLOCK - K)).view(R, kb, BLOCK)
    ex = _exponent(xp.abs().amax(dim=2))
    q = (xp * _pow2(-ex)[:, :, None]).reshape(R, kb * BLOCK)[:, :K].to(torch.float8_e4m3fn)
    return q, ex


def _rows(x):
    """Rows in fp32 as their e4m3 form holds them."""
    q, ex = _quant(x)
    return q.float() * _pow2(ex).repeat_interleave(BLOCK, dim=1)[:, :x.shape[1]]


def _blocks(q, s, parts=1):
    """One expert's weights in fp32."""
    n, k = q.shape[0] // parts, q.shape[1]
    w = q.float().view(parts, n, k)
    sc = _pow2(s.view(torch.uint8).to(torch.int32).view(parts, -1, s.shape[1]) - 127)
    return (w * sc.repeat_interleave(BLOCK, dim=1)[:, :n].repeat_interleave(BLOCK, dim=2)[:, :, :k]).view(parts * n, k)


def _act(a, I, act):
    if act == "swiglu":
        u, v = a[:, :I], a[:, I:]
        return u / (1 + torch.exp(-u)) * v
    return 0.5 * a * (1 + torch.tanh(0.7978845608028654 * (a + 0.044715 * a * a * a)))


def _plain_norm(st):
    c = st["case"]
    dt = DT[c["dt"]]
    with torch.no_grad():
        s = (st["x"].float() + st["res"].float()).to(dt)
        f = s.float()
        rstd = torch.rsqrt(f.square().mean(dim=1, keepdim=True) + 1e-6)
        y = f * rstd * st["w"].float()
        if c["mode"] == "plain":
            return dict(y=y.to(dt), s=s)
        if c["mode"] == "fp8":
            q, ex = _quant(y)
            return dict(y=y.to(dt), s=s, q=q, scale=(ex + 127).to(torch.uint8).view(torch.float8_e8m0fnu))
        dy = st["dy"].float()
        n = f * rstd
        gw = dy * st["w"].float()
        dx = ((gw - n * (gw * n).mean(dim=1, keepdim=True)) * rstd + st["ds"].float()).to(dt)
        return dict(y=y.to(dt), s=s, dx=dx, dres=dx, dw=(dy * n).sum(dim=0).to(dt))


def _plain_linear(st):
    c = st["case"]
    dt = DT[c["dt"]]
    with torch.no_grad():
        x = _rows(st["x"].float())
        ys, dxs = [], []
        dy = _rows(st["dy"].float()) if c["mode"] == "train" else None
        r = 0
        for e, n in enumerate(st["counts"]):                # one product per group
            w = _blocks(st["q"][e], st["s"][e])
            y = x[r:r + n] @ w.t()
            ys.append((y + st["b"][e].float() if st["b"] is not None else y).to(dt))
            if dy is not None:
                dxs.append((dy[r:r + n] @ w).to(dt))
            r += n
        out = dict(y=torch.cat(ys))
        if dy is not None:
            out["dx"] = torch.cat(dxs)
        return out


def _plain_ffn(st):
    c = st["case"]
    dt = DT[c["dt"]]
    parts = 2 if c["act"] == "swiglu" else 1
    with torch.no_grad():
        x = _rows(st["x"].float())[st["perm"].long() >> 1]
        ys = []
        r = 0
        for e, n in enumerate(st["counts"]):                # one MLP per expert that got rows
            if n == 0:
                continue
            a = x[r:r + n] @ _blocks(st["q1"][e], st["s1"][e], parts).t()
            if st["b1"] is not None:
                a = a + st["b1"][e].float()
            y = _rows(_act(a, c["I"], c["act"])) @ _blocks(st["q2"][e], st["s2"][e]).t()
            ys.append((y + st["b2"][e].float() if st["b2"] is not None else y).to(dt))
            r += n
        return dict(y=torch.cat(ys))


# ------------------------------------------------------------------------------------------------ the package's operators
def _own_norm(st):
    from moe_llava_amd import norm
    c = st["case"]
    if c["mode"] == "fp8":
        with torch.no_grad():
            rows, y, s = norm.add_rms_norm_fp8(st["x"], st["res"], st["w"], eps=1e-6)
        return dict(y=y, s=s, q=rows.q, scale=rows.scale)
    if c["mode"] == "plain":
        with torch.no_grad():
            y, s = norm.add_rms_norm(st["x"], st["res"], st["w"], eps=1e-6)
        return dict(y=y, s=s)
    y, s = norm.add_rms_norm(st["x"], st["res"], st["w"], eps=1e-6)
    dx, dres, dw = torch.autograd.grad((y, s), (st["x"], st["res"], st["w"]), (st["dy"], st["ds"]))
    return dict(y=y.detach(), s=s.detach(), dx=dx, dres=dres, dw=dw)


def _own_linear(st):
    from moe_llava_amd import fp8
    c = st["case"]
    if c["G"] == 1:
        y = fp8.linear(st["x"], st["q"][0], st["s"][0], st["b"][0] if st["b"] is not None else None)
    else:
        y = fp8.grouped_linear(st["x"], st["q"], st["s"], st["offs"], st["b"])
    if c["mode"] != "train":
        return dict(y=y)
    dx, = torch.autograd.grad(y, st["x"], st["dy"])
    return dict(y=y.detach(), dx=dx)


def _own_ffn(st):
    from moe_llava_amd import fp8
    c = st["case"]
    with torch.no_grad():
        y = fp8.expert_ffn(c["act"], st["x"], st["q1"], st["s1"], st["q2"], st["s2"], st["offs"], 2 * c["S"],
                           gather=st["perm"], gather_shift=1, b1=st["b1"], b2=st["b2"])
    return dict(y=y)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "linear": _own_linear, "ffn": _own_ffn}[op](state)
    return {"norm": _plain_norm, "linear": _plain_linear, "ffn": _plain_ffn}[op](state)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _e4m3(v):
    """Nearest value of the 8-bit format (3 bits behind the leading one, smallest exponent -6), ties to even."""
    ex = torch.frexp(v.abs())[1].to(torch.float64) - 1
    step = torch.exp2(ex.clamp_min(-6.0) - 3)
    return torch.round(v / step) * step


def _exact_rows(x):
    R, K = x.shape
    out = torch.empty_like(x)
    scales = torch.empty((R, _up(K, BLOCK)), dtype=torch.float64, device=x.device)
    for b in range(_up(K, BLOCK)):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        big = part.abs().max(dim=1).values / E4M3_MAX
        sc = torch.exp2(torch.ceil(torch.log2(big.clamp(min=2.0 ** -126))))
        out[:, b * BLOCK:(b + 1) * BLOCK] = _e4m3(part / sc[:, None])
        scales[:, b] = sc
    return out, scales


def _exact_value(x):
    q, s = _exact_rows(x)
    cols = torch.arange(x.shape[1], device=x.device) // BLOCK
    return q * s[:, cols]


def _exact_weight(q, s, parts=1):
    n = q.shape[0] // parts
    rows = torch.arange(q.shape[0], device=q.device)
    rb = rows // n * _up(n, BLOCK) + rows % n // BLOCK
    cb = torch.arange(q.shape[1], device=q.device) // BLOCK
    return q.to(torch.float64) * torch.exp2(s.view(torch.uint8).to(torch.float64) - 127)[rb][:, cb]


def exact(case, seed):
    st = prepare(case, seed)
    D = torch.float64
    with torch.no_grad():
        if case["op"] == "norm":
            x, r, w = (st[k].to(D) for k in ("x", "res", "w"))
            s = (x + r).to(DT[case["dt"]]).to(D)        # the sum is held in the rows' own type
            inv = 1.0 / torch.sqrt((s * s).mean(dim=1, keepdim=True) + 1e-6)
            y = s * inv * w
            if case["mode"] == "plain":
                return dict(y=y, s=s)
            if case["mode"] == "fp8":
                q, sc = _exact_rows(y)
                return dict(y=y, s=s, q=q, scale=sc)
            dy, ds = st["dy"].to(D), st["ds"].to(D)
            t = dy * w
            dot = (t * s).sum(dim=1, keepdim=True)
            dx = t * inv - s * dot * inv ** 3 / case["M"] + ds
            return dict(y=y, s=s, dx=dx, dres=dx, dw=(dy * s * inv).sum(dim=0))
        offs = [0]
        for n in st["counts"]:
            offs.append(offs[-1] + n)
        if case["op"] == "linear":
            x = _exact_value(st["x"].to(D))
            y = torch.empty((case["S"], case["N"]), dtype=D, device=DEV)
            dx = torch.empty((case["S"], case["K"]), dtype=D, device=DEV) if case["mode"] == "train" else None
            dy = _exact_value(st["dy"].to(D)) if dx is not None else None
            for e in range(case["G"]):
                w = _exact_weight(st["q"][e], st["s"][e])
                rows = slice(offs[e], offs[e + 1])
                y[rows] = torch.mm(x[rows], w.t())
                if st["b"] is not None:
                    y[rows] += st["b"][e].to(D)
                if dx is not None:
                    dx[rows] = torch.mm(dy[rows], w)
            return dict(y=y) if dx is None else dict(y=y, dx=dx)
        I = case["I"]
        x = _exact_value(st["x"].to(D))
        tok = torch.div(st["perm"], 2, rounding_mode="floor").long()
        y = torch.empty((2 * case["S"], case["M"]), dtype=D, device=DEV)
        for e in range(case["E"]):
            rows = slice(offs[e], offs[e + 1])
            if offs[e] == offs[e + 1]:
                continue
            a = torch.mm(x[tok[rows]], _exact_weight(st["q1"][e], st["s1"][e], 2 if case["act"] == "swiglu" else 1).t())
            if st["b1"] is not None:
                a += st["b1"][e].to(D)
            if case["act"] == "swiglu":
                h = a[:, :I] * torch.sigmoid(a[:, :I]) * a[:, I:]
            else:
                h = 0.5 * a * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (a + 0.044715 * a ** 3)))
            y[rows] = torch.mm(_exact_value(h), _exact_weight(st["q2"][e], st["s2"][e]).t())
            if st["b2"] is not None:
                y[rows] += st["b2"][e].to(D)
        return dict(y=y)
