"""8-bit experts: products and expert MLPs on e4m3 operands with power-of-two scales per block of 128.

Format (``include/moe_gfx950.h``): e4m3 elements (``torch.float8_e4m3fn``) and, for every 1 x 128 block of a row and every
128 x 128 block of a weight matrix, one scale 2^e held as ``torch.float8_e8m0fnu``; e is the smallest exponent that brings
the block's largest magnitude to 448 or below, so that scaling rounds nothing.

    w, ws = fp8.quantize_weight(weight)              # [.., N, K] bf16 / fp16 -> e4m3 + scales, once
    y = fp8.linear(x, w, ws, bias)                   # x [.., K]; differentiable with respect to x (weights are frozen)
    y = fp8.grouped_linear(x, w, ws, group_offsets)  # rows of group g with expert g % E
    y = fp8.expert_ffn("swiglu", x, w1, ws1, w2, ws2, group_offsets, max_rows, gather, 1)      # inference

Inputs are 16-bit tensors, quantised in front of the product, or ``Fp8Rows`` (``quantize_rows``, ``norm.add_rms_norm_fp8``).
The reference has no counterpart: its experts run in 16 bits.  As in ``ops``, nothing here computes on the CPU.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib, ops

BLOCK = 128
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
MAX_K = 65536            # columns of a product's operands
MAX_ROWS = 2 ** 31 - 512  # row counts and matrix dimensions: rounded up to a tile they stay within the library's 32 bits
_ACTS = {"swiglu": ops.ACT_SWIGLU, "gelu_new": ops.ACT_GELU_NEW, ops.ACT_SWIGLU: ops.ACT_SWIGLU,
         ops.ACT_GELU_NEW: ops.ACT_GELU_NEW}


class Fp8Rows(NamedTuple):
    """Rows in 8 bits: ``q`` [S, K] e4m3 and ``scale`` [S, ceil(K/128)] e8m0.  The scales' row stride is a multiple of 4
    bytes (``scale`` is a view of a padded buffer), as the kernels read them 4 at a time."""
    q: Tensor
    scale: Tensor


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _empty_rows(S: int, K: int, dev) -> Fp8Rows:
    kb = (K + BLOCK - 1) // BLOCK
    q = torch.empty((S, K), dtype=E4M3, device=dev)
    if not kb % 4:
        return Fp8Rows(q, torch.empty((S, kb), dtype=E8M0, device=dev))
    return Fp8Rows(q, torch.empty((S, (kb + 3) // 4 * 4), dtype=E8M0, device=dev)[:, :kb])


#: pointer of the current stream of a device, by index (torch.cuda.current_stream builds a Stream object per call: 1.9 us
#: of a decode step's host time against 0.1)
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _gpu(t, name: str) -> None:
    if not isinstance(t, Tensor):
        raise TypeError(f"{name}: expected a tensor")
    if not t.is_cuda:
        raise _lib.MoEKernelError(f"{name}: must live on the GPU (got {t.device}); there is no CPU path")


def _half_rows(x: Tensor, name: str) -> Tensor:
    """x [.., K] as rows [S, K] whose last dimension is dense (other strides stay; a copy only where they cannot)."""
    _gpu(x, name)
    if x.dtype not in ops.HALF_DTYPES:
        raise TypeError(f"{name}: expected bf16 or fp16, got {x.dtype}")
    d = x.dim()
    if d < 1:
        raise ValueError(f"{name}: expected at least one dimension")
    if d != 2:
        x = x.reshape(-1, x.shape[-1]) if x.numel() else x.reshape(x.shape[:-1].numel(), x.shape[-1])
    if x.shape[0] > MAX_ROWS or x.shape[1] > MAX_ROWS:
        raise ValueError(f"{name}: {tuple(x.shape)}: rows and columns of at most {MAX_ROWS}")
    if d == 2 and x.is_contiguous():
        return x
    if x.shape[1] > 1 and x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()                  # transposed, or rows that overlap (an expanded row)
    return x


def _check_rows(a: Fp8Rows, name: str) -> Fp8Rows:
    q, sc = a
    _gpu(q, f"{name}.q")
    _gpu(sc, f"{name}.scale")
    if q.dtype != E4M3 or sc.dtype != E8M0 or q.dim() != 2 or sc.dim() != 2:
        raise TypeError(f"{name}: expected e4m3 rows [S, K] and e8m0 scales [S, ceil(K/128)]")
    S, K = q.shape
    if S > MAX_ROWS:
        raise ValueError(f"{name}: {S} rows: at most {MAX_ROWS}")
    if tuple(sc.shape) != (S, _blocks(K)) or sc.device != q.device:
        raise ValueError(f"{name}: scales {tuple(sc.shape)} on {sc.device} do not match rows {tuple(q.shape)} on {q.device}")
    if q.stride(1) != 1 or (S > 1 and (q.stride(0) % 16 or q.stride(0) < K)) or q.data_ptr() % 16:
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
    kb4 = (sc.shape[1] + 3) // 4 * 4
    room = sc.untyped_storage().nbytes() - sc.storage_offset()      # e8m0: one byte per element
    st = sc.stride(0) if S > 1 else kb4
    if sc.stride(1) != 1 and sc.shape[1] > 1 or st % 4 or st < kb4 or sc.data_ptr() % 4 or room < (S - 1) * st + kb4:
        pad = torch.empty((S, kb4), dtype=E8M0, device=q.device)
        pad.view(torch.uint8)[:, :sc.shape[1]].copy_(sc.view(torch.uint8))
        sc = pad[:, :sc.shape[1]]
    return Fp8Rows(q, sc)


def _lead(t: Tensor, width: int) -> int:
    """Row stride of a 2-d tensor; that of a single row is arbitrary in torch."""
    return t.stride(0) if t.shape[0] > 1 else width


def _lead_scale(sc: Tensor) -> int:
    return sc.stride(0) if sc.shape[0] > 1 else (sc.shape[1] + 3) // 4 * 4


def _check_weight(w: Tensor, ws: Tensor, name: str, E: int, N: Optional[int], parts: int = 1) -> Tuple[int, int]:
    """w [E, parts*N, K] (E == 0: [N, K]) with scales [E, parts*ceil(N/128), ceil(K/128)]; returns (N, K)."""
    _gpu(w, name)
    _gpu(ws, f"{name}_scale")
    if w.dtype != E4M3 or ws.dtype != E8M0:
        raise TypeError(f"{name}: expected {E4M3} with {E8M0} scales, got {w.dtype} with {ws.dtype}")
    if not (w.is_contiguous() and ws.is_contiguous()):
        raise ValueError(f"{name} and its scales must be contiguous")
    sh, sc = w.shape, ws.shape
    nd = 3 if E else 2
    if len(sh) != nd or len(sc) != nd:
        raise ValueError(f"{name}: {tuple(sh)} with scales {tuple(sc)}: need {'[E, N, K]' if E else '[N, K]'}")
    n, K = sh[-2], sh[-1]
    if n < parts or n % parts or (N is not None and n != parts * N):
        raise ValueError(f"{name}: {tuple(sh)} does not hold {parts} projection(s) of the expected width")
    n //= parts
    if K % 16 or not 16 <= K <= MAX_K:
        raise ValueError(f"{name}: K={K} must be a multiple of 16 and at most {MAX_K}")
    if n > MAX_ROWS:
        raise ValueError(f"{name}: N={n}: at most {MAX_ROWS}")
    if sc[-2] != parts * ((n + 127) // BLOCK) or sc[-1] != (K + 127) // BLOCK or (E and (sh[0] != E or sc[0] != E)) \
            or ws.device != w.device:
        raise ValueError(f"{name}_scale: {tuple(sc)} on {ws.device} does not match {name} {tuple(sh)} on {w.device}")
    if w.data_ptr() % 16:
        raise ValueError(f"{name}: must be 16-byte aligned")
    return n, K


def _check_bias(b: Tensor, name: str, shape, dtype, dev) -> None:
    if not isinstance(b, Tensor) or b.dtype != dtype or tuple(b.shape) != tuple(shape) or b.device != dev \
            or not b.is_contiguous():
        raise ValueError(f"{name}: need a contiguous {dtype} tensor of shape {tuple(shape)} on {dev}")


def _check_index(t: Tensor, name: str, dev) -> None:
    _gpu(t, name)
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{name}: need a contiguous 1-d int32 tensor on {dev}")


# ------------------------------------------------------------------------------------------------ quantisation
def quantize_rows(x: Tensor) -> Fp8Rows:
    """16-bit rows [.., K] (any row stride, K % 16 == 0) -> ``Fp8Rows`` of shape [S, K]."""
    x = _half_rows(x, "x")
    S, K = x.shape
    if K % 16 or K < 16:
        raise ValueError(f"x: K={K} must be a multiple of 16")
    out = _empty_rows(S, K, x.device)
    if S:
        with ops._on(x.device):
            rc = _lib.load().moe_quantize_rows_fp8(x.data_ptr(), _lead(x, K), S, K, out.q.data_ptr(), K, out.scale.data_ptr(),
                                                   _lead_scale(out.scale), ops._dt(x), _stream(x.device.index))
        _lib.check(rc, "moe_quantize_rows_fp8")
    return out


def quantize_weight(w: Tensor, projections: int = 1, out=None) -> Tuple[Tensor, Tensor]:
    """16-bit weights [.., N, K] (K % 16 == 0) -> (e4m3 [.., N, K], scales [.., projections * ceil(N'/128), ceil(K/128)]).
    ``projections`` = 2 for a gated W1 [.., 2I, M]: each half gets blocks of its own (N' = I).
    ``out``: (weights, scales) of an earlier call of the same shape, filled again."""
    _gpu(w, "w")
    if w.dtype not in ops.HALF_DTYPES:
        raise TypeError(f"w: expected bf16 or fp16, got {w.dtype}")
    if w.dim() < 2 or w.numel() == 0 or w.shape[-2] % projections or w.shape[-1] % 16:
        raise ValueError(f"w: {tuple(w.shape)}: need [.., N, K] with K % 16 == 0 and N a multiple of {projections}")
    w = w.contiguous()
    if w.data_ptr() % 16:
        w = w.clone()
    n, k = w.shape[-2] // projections, w.shape[-1]
    batch = w.numel() // (n * k)
    if max(batch, n, k) > MAX_ROWS:
        raise ValueError(f"w: {tuple(w.shape)}: dimensions of at most {MAX_ROWS}")
    shape_s = tuple(w.shape[:-2]) + (projections * _blocks(n), _blocks(k))
    if out is None:
        q = torch.empty(w.shape, dtype=E4M3, device=w.device)
        sc = torch.empty(shape_s, dtype=E8M0, device=w.device)
    else:
        q, sc = out
        for t, dt, shape in ((q, E4M3, tuple(w.shape)), (sc, E8M0, shape_s)):
            if t.dtype != dt or tuple(t.shape) != shape or t.device != w.device or not t.is_contiguous():
                raise ValueError(f"out: need a contiguous {dt} tensor of shape {shape} on {w.device}")
    with ops._on(w.device):
        rc = _lib.load().moe_quantize_blocks_fp8(w.data_ptr(), batch, n, k, q.data_ptr(), sc.data_ptr(), ops._dt(w),
                                                 _stream(w.device.index))
    _lib.check(rc, "moe_quantize_blocks_fp8")
    if out is not None:                     # the library's writes are invisible to autograd: a graph that saved them must see
        torch.autograd.graph.increment_version([t for t in (q, sc) if not t.is_inference()])
    return q, sc


def _frozen(*ts) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise NotImplementedError("8-bit experts are frozen: weights, scales and biases with requires_grad are not supported "
                                  "(torch.no_grad() runs them)")


# ------------------------------------------------------------------------------------------------ products
def _gemm(a: Fp8Rows, w: Tensor, ws: Tensor, bias: Optional[Tensor], offs: Optional[Tensor], E: int, N: int, K: int, dtype,
          zero_tail: bool) -> Tensor:
    S = a.q.shape[0]
    out = torch.empty((S, N), dtype=dtype, device=a.q.device)
    if S == 0:
        return out
    G = offs.numel() - 1 if offs is not None else 1
    with ops._on(a.q.device):
        rc = _lib.load().moe_grouped_gemm_fp8_fwd(
            a.q.data_ptr(), _lead(a.q, K), a.scale.data_ptr(), _lead_scale(a.scale), None, 0, w.data_ptr(), ws.data_ptr(),
            bias.data_ptr() if bias is not None else None, offs.data_ptr() if offs is not None else None, G, E, S, K, N,
            int(zero_tail), out.data_ptr(), N, ops.DTYPE_F16 if dtype == torch.float16 else ops.DTYPE_BF16,
            _stream(a.q.device.index))
    _lib.check(rc, "moe_grouped_gemm_fp8_fwd")
    return out


def _linear16(x: Tensor, w: Tensor, ws: Tensor, bias: Optional[Tensor], offs: Optional[Tensor], E: int, N: int, K: int) -> Tensor:
    """16-bit rows x [S, K]: quantised and multiplied in one library call."""
    S = x.shape[0]
    dev = x.device
    out = torch.empty((S, N), dtype=x.dtype, device=dev)
    if S == 0:
        return out
    lib = _lib.load()
    nws = lib.moe_grouped_linear_fp8_workspace_bytes(S, K)
    buf = torch.empty((nws,), dtype=torch.uint8, device=dev)
    with ops._on(dev):
        rc = lib.moe_grouped_linear_fp8_fwd(
            x.data_ptr(), _lead(x, K), w.data_ptr(), ws.data_ptr(), bias.data_ptr() if bias is not None else None,
            offs.data_ptr() if offs is not None else None, offs.numel() - 1 if offs is not None else 1, E, S, K, N,
            int(offs is not None), buf.data_ptr(), nws, out.data_ptr(), N, ops._dt(x), _stream(dev.index))
    _lib.check(rc, "moe_grouped_linear_fp8_fwd")
    return out


class _LinearFn(torch.autograd.Function):
    """y = Q(x) W^T + b over groups of rows; dx = Q(dy) W with W's blocks transposed on the fly (frozen weights: no copy of
    them is kept).  The rounding of x to 8 bits is passed through as the identity; a gradient of ``bias`` is the column sum
    of dy and is refused here (8-bit experts are frozen)."""

    @staticmethod
    def forward(ctx, x: Tensor, w: Tensor, ws: Tensor, bias, offs, E: int, N: int, K: int):
        ctx.save_for_backward(w, ws, offs)
        ctx.meta = (E, N, K, x.shape, x.dtype)
        return _linear16(x, w, ws, bias, offs, E, N, K)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy: Tensor):
        w, ws, offs = ctx.saved_tensors
        E, N, K, shape, dtype = ctx.meta
        wt = torch.empty((E, K, N), dtype=E4M3, device=w.device)
        wst = torch.empty((E, _blocks(K), _blocks(N)), dtype=E8M0, device=w.device)
        with ops._on(w.device):
            rc = _lib.load().moe_transpose_blocks_fp8(w.data_ptr(), ws.data_ptr(), E, N, K, wt.data_ptr(), wst.data_ptr(),
                                                      _stream(w.device.index))
        _lib.check(rc, "moe_transpose_blocks_fp8")
        dx = _linear16(_half_rows(dy, "dy"), wt, wst, None, offs, E, K, N)
        return dx.reshape(shape), None, None, None, None, None, None, None


def _linear(x, w: Tensor, ws: Tensor, bias: Optional[Tensor], offs: Optional[Tensor], dtype) -> Tensor:
    grouped = offs is not None
    _gpu(w, "w")
    E = (w.shape[0] if w.dim() == 3 else -1) if grouped else 0
    N, K = _check_weight(w, ws, "w", E, None)
    dev = w.device
    rows = None
    if isinstance(x, Fp8Rows):
        if dtype is None:
            dtype = bias.dtype if bias is not None else torch.bfloat16
        if dtype not in ops.HALF_DTYPES:
            raise TypeError(f"out_dtype: expected bf16 or fp16, got {dtype}")
        rows = _check_rows(x, "x")
        x2 = rows.q
    else:
        x2 = _half_rows(x, "x")
        if dtype is not None and dtype != x.dtype:
            raise TypeError("out_dtype is the input's type for 16-bit inputs")
        dtype = x.dtype
    if x2.shape[1] != K or x2.device != dev:
        raise ValueError(f"x {tuple(x2.shape)} on {x2.device} does not match w {tuple(w.shape)} on {dev}")
    if bias is not None:
        _check_bias(bias, "bias", (E, N) if grouped else (N,), dtype, dev)
    if grouped:
        _check_index(offs, "group_offsets", dev)
        if not 2 <= offs.numel() <= 4097:
            raise ValueError("group_offsets needs 2 to 4097 entries")
    E = E or 1
    _frozen(w, ws, bias)
    if rows is not None:
        return _gemm(rows, w, ws, bias, offs, E, N, K, dtype, grouped)
    grad = torch.is_grad_enabled() and x.requires_grad
    if grad and (N % 16 or N > MAX_K):
        raise NotImplementedError(f"the input gradient needs N % 16 == 0 and N <= {MAX_K} (N={N})")
    y = (_LinearFn.apply if grad else _linear16)(x2, w, ws, bias, offs, E, N, K)
    return y if x.dim() == 2 else y.reshape(x.shape[:-1] + (N,))


def linear(x: Union[Tensor, Fp8Rows], w: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, out_dtype=None) -> Tensor:
    """``x @ w.T + bias`` with w [N, K] in 8 bits.  x [.., K] bf16 / fp16 (the output's type), or ``Fp8Rows`` (``out_dtype``,
    by default the bias' type, else bf16).  fp32 accumulation, one rounding.  Differentiable with respect to a 16-bit x when
    N % 16 == 0: the gradient is quantised like any rows and multiplied by the transposed 8-bit weights."""
    return _linear(x, w, w_scale, bias, None, out_dtype)


def grouped_linear(x: Union[Tensor, Fp8Rows], w: Tensor, w_scale: Tensor, group_offsets: Tensor,
                   bias: Optional[Tensor] = None, out_dtype=None) -> Tensor:
    """``linear`` for ragged groups of rows: rows [group_offsets[g], group_offsets[g+1]) of x [S, K] use expert g % E of
    w [E, N, K] (bias [E, N]).  ``group_offsets`` [G+1] int32 stays on the device (ascending, within [0, S]); rows of no
    group give 0, and get no gradient."""
    if not isinstance(x, Fp8Rows) and isinstance(x, Tensor) and x.dim() != 2:
        raise ValueError(f"x: expected [S, K], got {tuple(x.shape)}")
    if group_offsets is None:
        raise ValueError("group_offsets is missing")
    return _linear(x, w, w_scale, bias, group_offsets, out_dtype)


# ------------------------------------------------------------------------------------------------ expert MLP
def expert_ffn(act, x: Union[Tensor, Fp8Rows], w1: Tensor, w1_scale: Tensor, w2: Tensor, w2_scale: Tensor,
               group_offsets: Tensor, max_rows: int, gather: Optional[Tensor] = None, gather_shift: int = 0,
               b1: Optional[Tensor] = None, b2: Optional[Tensor] = None, n_gated: int = -1, out_dtype=None) -> Tensor:
    """``ops.expert_ffn`` on 8-bit experts (inference): y [max_rows, M] for the compact rows of the groups; compact row p
    reads row ``gather[p] >> gather_shift`` of x (row p without ``gather``); rows past ``group_offsets[G]`` are left
    unwritten.  ``act`` "swiglu" (w1 [E, 2I, M], scales [E, 2*ceil(I/128), ceil(M/128)]) or "gelu_new" (w1 [E, I, M]);
    w2 [E, M, I].  M and I are multiples of 16.  The activation is evaluated in fp32 on the first product's accumulators and
    quantised per 128 hidden channels."""
    act = _ACTS.get(act, -1)
    if act < 0:
        raise ValueError("act: 'swiglu' or 'gelu_new'")
    _gpu(w2, "w2")
    if w2.dim() != 3 or w2.shape[0] < 1:
        raise ValueError(f"w2: {tuple(w2.shape)}: need [E, M, I]")
    E = w2.shape[0]
    M, I = _check_weight(w2, w2_scale, "w2", E, None)
    parts = 2 if act == ops.ACT_SWIGLU else 1
    if _check_weight(w1, w1_scale, "w1", E, I, parts)[1] != M or M % 16 or I % 16:
        raise ValueError(f"w1 {tuple(w1.shape)} / w2 {tuple(w2.shape)} do not match (multiples of 16)")
    dev = w1.device
    eight = isinstance(x, Fp8Rows)
    if eight:
        x = _check_rows(x, "x")
        src = x.q
        dtype = out_dtype or (b2.dtype if b2 is not None else torch.bfloat16)
        if dtype not in ops.HALF_DTYPES:
            raise TypeError(f"out_dtype: expected bf16 or fp16, got {dtype}")
    else:
        x = src = _half_rows(x, "x")
        dtype = x.dtype
        if out_dtype is not None and out_dtype != dtype:
            raise TypeError("out_dtype is the input's type for 16-bit inputs")
        if torch.is_grad_enabled() and x.requires_grad:
            raise NotImplementedError("fp8.expert_ffn is for inference: wrap it in torch.no_grad(), or compose "
                                      "fp8.grouped_linear, which is differentiable")
    if src.shape[1] != M or src.device != dev or w2.device != dev:
        raise ValueError(f"x {tuple(src.shape)} on {src.device} does not match w1 {tuple(w1.shape)} on {dev}")
    if b1 is not None:
        _check_bias(b1, "b1", (E, parts * I), dtype, dev)
    if b2 is not None:
        _check_bias(b2, "b2", (E, M), dtype, dev)
    _frozen(w1, w1_scale, b1, w2, w2_scale, b2)
    _check_index(group_offsets, "group_offsets", dev)
    G = group_offsets.numel() - 1
    if not 1 <= G <= 4096 or not 0 <= max_rows <= MAX_ROWS:
        raise ValueError("group_offsets needs 2 to 4097 entries, max_rows >= 0")
    if gather is not None:
        _check_index(gather, "gather", dev)
        if gather.numel() < max_rows:
            raise ValueError("gather shorter than max_rows")
        if gather_shift not in (0, 1):
            raise ValueError("gather_shift: 0 or 1")
    elif src.shape[0] < max_rows:
        raise ValueError("x has fewer rows than max_rows")
    y = torch.empty((max_rows, M), dtype=dtype, device=dev)
    if max_rows == 0:
        return y
    S = src.shape[0]
    lib = _lib.load()
    nws = lib.moe_expert_ffn_fp8_workspace_bytes(0 if eight else S, max_rows, M, I)
    ws = torch.empty((nws,), dtype=torch.uint8, device=dev)
    if eight:
        args = (None, 0, 0, src.data_ptr(), _lead(src, M), x.scale.data_ptr(), _lead_scale(x.scale))
    else:
        args = (src.data_ptr(), _lead(src, M), S, None, 0, None, 0)
    with ops._on(dev):
        rc = lib.moe_expert_ffn_fp8_fwd(
            act, *args, gather.data_ptr() if gather is not None else None, gather_shift, w1.data_ptr(), w1_scale.data_ptr(),
            b1.data_ptr() if b1 is not None else None, w2.data_ptr(), w2_scale.data_ptr(),
            b2.data_ptr() if b2 is not None else None, group_offsets.data_ptr(), G, E, max_rows, M, I, n_gated,
            ws.data_ptr(), nws, y.data_ptr(), ops.DTYPE_F16 if dtype == torch.float16 else ops.DTYPE_BF16,
            _stream(dev.index))
    _lib.check(rc, "moe_expert_ffn_fp8_fwd")
    return y


# ------------------------------------------------------------------------------------------------ whole block
def check_experts(x: Tensor, experts) -> Tuple[int, int, int]:
    """(M, I, E) of what ``Experts.packed_fp8`` returns, checked against the rows x [S, M]."""
    act, w1, s1, b1, w2, s2, b2 = experts
    ops._need(x, "x", ops.HALF_DTYPES, 2)
    S, M = x.shape
    E = w2.shape[0]
    if _check_weight(w2, s2, "w2", E, M)[1] % 16 or S < 1:
        raise ValueError(f"w2 {tuple(w2.shape)} / x {tuple(x.shape)}: need multiples of 16, and at least one token")
    I = w2.shape[2]
    parts = 2 if act == ops.ACT_SWIGLU else 1
    dev = x.device
    if _check_weight(w1, s1, "w1", E, I, parts)[1] != M or w1.device != dev or w2.device != dev:
        raise ValueError(f"w1 {tuple(w1.shape)} / w2 {tuple(w2.shape)} do not match x {tuple(x.shape)} on {dev}")
    if b1 is not None:
        _check_bias(b1, "b1", (E, parts * I), x.dtype, dev)
    if b2 is not None:
        _check_bias(b2, "b2", (E, M), x.dtype, dev)
    return M, I, E


def row_pointers(rows: Fp8Rows, S: int, M: int, dev):
    """(q, row stride, scales, their row stride) for a library call on rows [S, M]."""
    rows = _check_rows(rows, "rows")
    if tuple(rows.q.shape) != (S, M) or rows.q.device != dev:
        raise ValueError(f"rows {tuple(rows.q.shape)} do not match x {(S, M)}")
    return rows.q.data_ptr(), _lead(rows.q, M), rows.scale.data_ptr(), _lead_scale(rows.scale)


def block_top2(x: Tensor, wg_weight: Tensor, capacity: int, noise: Optional[Tensor], noise_seed: int, drop_tokens: bool,
               experts, n_gated: int = -1, noise_seed_dev: Optional[Tensor] = None, rows: Optional[Fp8Rows] = None):
    """``ops.block_top2`` on 8-bit experts: gate -> top-2 routing -> expert MLPs -> combine in one library call.  ``experts``:
    what ``Experts.packed_fp8`` returns; ``rows``: x in 8 bits (the gate reads x).  Returns (out, logits, Routing)."""
    M, I, E = check_experts(x, experts)
    act, w1, s1, b1, w2, s2, b2 = experts
    S, dev = x.shape[0], x.device
    wgd = ops._wg_dt(wg_weight, x)
    ops._need(wg_weight, "wg.weight", wg_weight.dtype, 2)
    if tuple(wg_weight.shape) != (E, M) or wg_weight.device != dev:
        raise ValueError("wg.weight does not match x and the experts")
    if noise is not None:
        ops._need(noise, "noise", torch.float32, 2)
        if tuple(noise.shape) != (S, E) or noise.device != dev:
            raise ValueError("noise must be [S, E] on x's device")
    if noise_seed_dev is not None:
        ops._need(noise_seed_dev, "noise_seed_dev", torch.int64)
        if noise is not None or noise_seed_dev.numel() != 1 or noise_seed_dev.device != dev:
            raise ValueError("noise_seed_dev: one int64 on x's device, and no noise tensor with it")
    if rows is not None:
        rows = _check_rows(rows, "rows")
    max_rows = min(2 * S, E * int(capacity)) if drop_tokens else 2 * S
    lib = _lib.load()
    wsr = lib.moe_routing_workspace_bytes(S, E)
    r = ops.Routing.allocate(S, E, 2, max_rows, int(capacity), wsr, dev)
    logits = torch.empty((S, E), dtype=torch.float32, device=dev)
    nws = max(lib.moe_expert_ffn_fp8_workspace_bytes(0 if rows is not None else S, max_rows, M, I), 256)
    ybytes = (max(max_rows, 1) * M * 2 + 255) // 256 * 256
    buf = torch.empty((ybytes + nws,), dtype=torch.uint8, device=dev)    # y, then the experts' workspace
    out = torch.empty((S, M), dtype=x.dtype, device=dev)
    a = _lib.BlockTop2Args()
    a.x, a.wg, a.wg_dtype, a.logits = x.data_ptr(), wg_weight.data_ptr(), wgd, logits.data_ptr()
    a.noise = noise.data_ptr() if noise is not None else None
    a.noise_seed = int(noise_seed) & 0xFFFFFFFFFFFFFFFF
    a.noise_seed_dev = noise_seed_dev.data_ptr() if noise_seed_dev is not None else None
    a.S, a.M, a.E, a.I, a.act, a.capacity = S, M, E, I, act, int(capacity)
    a.drop_tokens, a.n_gated = int(bool(drop_tokens)), n_gated
    for name in ("expert_idx", "slot", "weight", "exp_counts", "kept_counts", "expert_offsets", "perm", "l_aux"):
        setattr(a, name, r.ptr(name))
    a.routing_ws, a.routing_ws_bytes = r.ptr("workspace"), wsr
    a.y, a.out, a.dtype, a.stream = buf.data_ptr(), out.data_ptr(), ops._dt(x), _stream(dev.index)
    q = _lib.Fp8Experts()
    q.w1, q.w1_scale, q.b1 = w1.data_ptr(), s1.data_ptr(), b1.data_ptr() if b1 is not None else None
    q.w2, q.w2_scale, q.b2 = w2.data_ptr(), s2.data_ptr(), b2.data_ptr() if b2 is not None else None
    if rows is not None:
        q.xq, q.ld_xq, q.xq_scale, q.ld_xs = row_pointers(rows, S, M, dev)
    q.workspace, q.ws_bytes = buf.data_ptr() + ybytes, nws
    with ops._on(dev):
        rc = lib.moe_block_top2_fp8_fwd(ctypes.byref(a), ctypes.byref(q))
    _lib.check(rc, "moe_block_top2_fp8_fwd")
    r._keep = buf
    return out, logits, r
