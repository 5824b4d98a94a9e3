"""Linear layers in 8 bits and over ragged groups (csrc/norm_fp8.hip, csrc/linear.hip).

8-bit values are float8_e4m3fn codes with one f32 scale for each block of 128 columns, either of one
row (activations, embeddings) or of 128 rows (weights).  Codes have shape [.., rows, cols] (a row is
padded with zeros to a multiple of 16 bytes), scales [.., rows or ceil(rows / 128), ceil(cols / 128)]
with the rows next to each other in memory.  A call takes scales of any strides.

    q, s, h = rms_norm_fp8(x, weight, residual=r)        # normalise what a layer reads, in 8 bits
    wq, ws = quantize_fp8(w, block_rows=128)             # once, when the weights are loaded
    y = matmul_fp8(q, s, wq, ws)                         # [rows, N]
    y = matmul_grouped(x, w, counts)                     # rows sorted by stream, one weight for each

Every call runs on the current stream of its inputs' device and never waits for it; each may be
captured into a graph.  The 16- and 32-bit norm and the 16-bit grouped product have gradients; the
8-bit forms are for serving and refuse inputs that require one.  Forward-mode derivatives are refused by all.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib
from .ops import _need_gpu, _raw_stream

__all__ = ["rms_norm", "rms_norm_fp8", "quantize_fp8", "matmul_fp8", "matmul_grouped"]

_P, _I, _I64, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
_lib.register({
    "trk_rms_norm": ([_P, _I64, _P, _I64, _P, _F, _I64, _I64, _I, _P, _I64, _P, _I64, _P, _P], _I),
    "trk_rms_norm_fp8": ([_P, _I64, _P, _I64, _P, _F, _I64, _I64, _I, _P, _I64, _P, _I64, _P, _I64, _P], _I),
    "trk_rms_norm_bwd_parts": ([_I64, _I64], _I64),
    "trk_rms_norm_bwd": ([_P, _I64, _P, _P, _P, _I64, _P, _I64, _I64, _I64, _I, _P, _I64, _P, _I64, _P, _P], _I),
    "trk_quantize_fp8": ([_P, _I64, _I64, _I64, _I64, _I64, _I, _I, _P, _I64, _I64, _P, _I64, _I64, _P], _I),
    "trk_matmul_fp8": ([_P, _I64, _P, _I64, _I64, _P, _I64, _P, _I64, _I64, _I, _P, _I64, _I64, _I64, _P, _I64, _I,
                        _P, _I64, _P], _I),
    "trk_matmul_fp8_parts": ([_I64, _I64, _I64], _I64),
    "trk_matmul_grouped": ([_P, _I64, _P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I64, _I, _P, _I64, _I64, _I64,
                            _I64, _I, _P, _I64, _I, _I, _P], _I),
    "trk_matmul_grouped_split": ([_P, _I64, _P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I64, _I, _P, _I64, _I64, _I64,
                                  _I64, _I, _P, _I64, _I, _I, _P, _I64, _P], _I),
    "trk_matmul_grouped_parts": ([_I64, _I64, _I64, _I64, _I], _I64),
    "trk_matmul_grouped_bwd": ([_P, _I64, _P, _I64, _P, _I64, _I64, _P, _I64, _I64, _I64, _I64, _I, _P, _I64, _P, _I64,
                                _I64, _P, _I64, _P], _I),
    "trk_matmul_grouped_bwd_parts": ([_I64, _I64, _I64, _I64], _I64),
})

FP8 = torch.float8_e4m3fn
_FLOAT = {torch.float32: _lib.TRK_F32, torch.bfloat16: _lib.TRK_BF16, torch.float16: _lib.TRK_F16}
_HALF = {torch.bfloat16: _lib.TRK_BF16, torch.float16: _lib.TRK_F16}


def _public_stream(idx: int) -> int:
    return torch.cuda.current_stream(idx).cuda_stream


# the raw accessors are one C call each; a torch without them has the public ones
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_stream_of = _raw_stream or _public_stream


def _launch(what: str, fn: str, x: torch.Tensor, *args):
    """lib().fn(*args, stream) on the current stream of x's device, which is made current for the launch"""
    idx = x.get_device()
    f = getattr(lib(), fn)
    if idx == _device():
        rc = f(*args, _stream_of(idx))
    else:
        with torch.cuda.device(idx):
            rc = f(*args, _stream_of(idx))
    if rc:
        check(rc, what)


def _type(t: torch.Tensor, of: dict, what: str, name: str) -> int:
    dt = of.get(t.dtype)
    if dt is None:
        raise TypeError(f"{what}: {name} must be one of {', '.join(str(k)[6:] for k in of)}, got {t.dtype}")
    return dt


def _on(x: torch.Tensor, what: str) -> int:
    """index of the device x is on"""
    if not isinstance(x, torch.Tensor) or x.get_device() < 0:
        _need_gpu(x, what)
    return x.get_device()


def _elsewhere(x: torch.Tensor, t: torch.Tensor, what: str, name: str):
    """error of a tensor that is not on x's device"""
    _need_gpu(t, what)
    raise ValueError(f"{what}: {name} is on {t.device}, x on {x.device}")


def _no_grad(what: str, *ts):
    for t in ts:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError(f"{what}: the 8-bit form has no gradient; call it under torch.no_grad()")


def _no_tangent(what: str, *ts):
    """error of a dual tensor: the kernels know no forward-mode derivative, and a result without one reads as zero"""
    if getattr(forward_ad, "_current_level", 0) < 0:  # (no level is open, so no tensor has a tangent)
        return
    for t in ts:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what}: no forward-mode derivative")


def _rows(t: torch.Tensor):
    """(t [.., D] as [R, D] with unit column stride and a row stride >= D, that stride); a view where t allows it"""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t, t.shape[1] or 1
    R, D = t.shape
    if (D > 1 and t.stride(1) != 1) or (R > 1 and t.stride(0) < D):
        t = t.contiguous()
    elif R > 1:
        return t, t.stride(0)
    return t, D or 1


def _at(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _codes(shape, x):
    """e4m3 codes of `shape`, rows padded to 16 bytes: (tensor, row stride)"""
    ld = (shape[-1] + 15) // 16 * 16
    q = x.new_empty((*shape[:-1], ld), dtype=FP8)
    return (q if ld == shape[-1] else q[..., :shape[-1]]), ld


# ------------------------------------------------------------------------------------------- norm
def _norm_inputs(what, x, weight, residual, eps):
    dev = _on(x, what)
    dt = _FLOAT.get(x.dtype)
    if dt is None:
        _type(x, _FLOAT, what, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: x must be [.., D] with D >= 1")
    if weight is not None:
        if weight.get_device() != dev:
            _elsewhere(x, weight, what, "weight")
        if weight.dtype != x.dtype:
            raise TypeError(f"{what}: weight is {weight.dtype}, x {x.dtype}")
        if weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
            raise ValueError(f"{what}: weight must be [{x.shape[-1]}], got {list(weight.shape)}")
    if residual is not None:
        if residual.get_device() != dev:
            _elsewhere(x, residual, what, "residual")
        if residual.dtype != x.dtype:
            raise TypeError(f"{what}: residual is {residual.dtype}, x {x.dtype}")
        if residual.shape != x.shape:
            raise ValueError(f"{what}: residual is {list(residual.shape)}, x {list(x.shape)}")
    if not eps >= 0:
        raise ValueError(f"{what}: eps must not be negative")
    _no_tangent(what, x, weight, residual)
    return dt


def _like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _norm_forward(dt, x, weight, residual, eps, want_rstd):
    x2, ldx = _rows(x)
    R, D = x2.shape
    r2, ldr = (None, 0) if residual is None else _rows(residual)
    w = None if weight is None else weight.contiguous()
    y = _like(x)
    h = None if residual is None else _like(x)
    rstd = x.new_empty(R, dtype=torch.float32) if want_rstd else None
    _launch("rms_norm", "trk_rms_norm", x, x2.data_ptr(), ldx, _at(r2), ldr, _at(w), eps, R, D, dt, y.data_ptr(), D, _at(h),
            D, _at(rstd))
    return y, h, rstd


class _Tied(torch.autograd.Function):
    """The n first tensors, hung on all of them: whoever differentiates them gets an error."""
    @staticmethod
    def forward(ctx, what, n, *ts):
        ctx.what = what
        return ts[:n]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.what}: no second derivative (its backward pass is once_differentiable)")


def _backward_once(what):
    """For a backward pass (ctx, saved tensors, gradients) without a derivative.  Where a graph of it is asked for, its gradients are hung on what came in and
    on every saved input: a second derivative is then an error for each of them.  (torch's own mark looks at
    what came in only: after a sum, whose gradient is a constant, the second derivative would silently be zero.)"""
    def mark(backward):
        def call(ctx, *grads):
            saved = ctx.saved_tensors  # once: a checkpoint computes them again for each reading
            if not torch.is_grad_enabled():
                return backward(ctx, saved, *grads)
            with torch.no_grad():
                out = backward(ctx, saved, *grads)
            of = [t for t in (*grads, *saved, *ctx.links) if t is not None and t.requires_grad]
            given = [t for t in out if t is not None]
            if not of or not given:
                return out
            tied = iter(_Tied.apply(what, len(given), *given, *of))
            return tuple(None if t is None else next(tied) for t in out)

        return call

    return mark


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, dt, eps):
        y, h, rstd = _norm_forward(dt, x, weight, residual, eps, True)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.dt, ctx.links = dt, ()
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @_backward_once("rms_norm")
    def backward(ctx, saved, dy, dh=None):
        h, weight, rstd = saved
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if dy is None:  # only the sum was used
            return dh if need_x else None, None, dh if need_r else None, None, None
        h2, ldh = _rows(h)
        y2, ldy = _rows(dy)
        R, D = h2.shape
        want = need_x or need_r
        e2, lde = (None, 0) if dh is None or not want else _rows(dh)
        w = None if weight is None else weight.contiguous()
        dx = _like(h) if want else None
        part = dw = None
        parts = 1
        if need_w:
            parts = lib().trk_rms_norm_bwd_parts(R, D)
            part = h.new_empty((parts, D), dtype=torch.float32)
            dw = h.new_empty(D)
        _launch("rms_norm backward", "trk_rms_norm_bwd", h, h2.data_ptr(), ldh, _at(w), rstd.data_ptr(), y2.data_ptr(), ldy,
                _at(e2), lde, R, D, ctx.dt, _at(dx), D, _at(part), parts, _at(dw))
        return dx if need_x else None, dw, dx if need_r else None, None, None


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension, h = x (+ residual).

    x, residual [.., D] and weight [D] in bfloat16, float16 or float32 (one type).  Returns y, or with a
    residual (y, h): h is what the next layer adds to.  Sums are f32, the norm is of the unrounded f32
    sum; y and h are rounded once.  Differentiable (backwards, once) in all three inputs, and through
    both outputs."""
    dt = _norm_inputs("rms_norm", x, weight, residual, eps)
    if (x.requires_grad or (weight is not None and weight.requires_grad) or
            (residual is not None and residual.requires_grad)) and torch.is_grad_enabled():
        return _RmsNorm.apply(x, weight, residual, dt, eps)
    y, h, _ = _norm_forward(dt, x, weight, residual, eps, False)
    return y if h is None else (y, h)


def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
                 eps: float = 1e-6):
    """rms_norm whose y is quantised as quantize_fp8(block_rows=1) does it, from f32: (q, scale), or with a
    residual (q, scale, h).  q [.., D] float8_e4m3fn, scale [.., ceil(D / 128)] f32."""
    what = "rms_norm_fp8"
    dt = _norm_inputs(what, x, weight, residual, eps)
    _no_grad(what, x, weight, residual)
    x2, ldx = _rows(x)
    R, D = x2.shape
    r2, ldr = (None, 0) if residual is None else _rows(residual)
    w = None if weight is None else weight.contiguous()
    q, ldq = _codes((R, D), x)
    s = torch.empty_strided((R, (D + 127) // 128), (1, max(R, 1)), dtype=torch.float32, device=x.device)
    h = None if residual is None else _like(x)
    _launch(what, "trk_rms_norm_fp8", x, x2.data_ptr(), ldx, _at(r2), ldr, _at(w), eps, R, D, dt, q.data_ptr(), ldq,
            s.data_ptr(), max(R, 1), _at(h), D)
    if x.dim() > 2:
        q, s = q.unflatten(0, x.shape[:-1]), s.unflatten(0, x.shape[:-1])
    elif x.dim() == 1:
        q, s = q[0], s[0]
    return (q, s) if h is None else (q, s, h)


# ---------------------------------------------------------------------------------------- quantise
def quantize_fp8(x: torch.Tensor, *, block_rows: int = 1):
    """x [rows, cols] (or a batch [B, rows, cols]) in bfloat16, float16 or float32 -> (q, scale): e4m3 codes and
    the f32 scales of blocks of block_rows (1 or 128) x 128 values.

    scale = max(|x|, 2^-117) / 448 over the block, q = x * 448 / max rounded to the nearest code (ties to
    even).  NaN values keep a NaN code and are left out of the maximum; a block that holds an infinity has an
    infinite scale, so that all of it reads back as NaN."""
    what = "quantize_fp8"
    _on(x, what)
    dt = _FLOAT.get(x.dtype)
    if dt is None:
        _type(x, _FLOAT, what, "x")
    if block_rows not in (1, 128):
        raise ValueError(f"{what}: block_rows must be 1 or 128")
    if x.dim() not in (2, 3) or x.shape[-1] < 1:
        raise ValueError(f"{what}: x must be [rows, cols] or [B, rows, cols] with cols >= 1")
    _no_grad(what, x)
    _no_tangent(what, x)
    R, D = x.shape[-2:]
    B = x.shape[0] if x.dim() == 3 else 1
    if not x.is_contiguous() and ((D > 1 and x.stride(-1) != 1) or (R > 1 and x.stride(-2) < D)):
        x = x.contiguous()
    ldx = x.stride(-2) if R > 1 else D
    q, ldq = _codes(x.shape, x)
    rb, kb = (R if block_rows == 1 else (R + 127) // 128), (D + 127) // 128
    one = (1, max(rb, 1))
    s = torch.empty_strided((rb, kb) if x.dim() == 2 else (B, rb, kb), one if x.dim() == 2 else (kb * rb, *one),
                            dtype=torch.float32, device=x.device)
    _launch(what, "trk_quantize_fp8", x, x.data_ptr(), ldx, x.stride(0) if x.dim() == 3 else 0, B, R, D, block_rows, dt,
            q.data_ptr(), ldq, R * ldq, s.data_ptr(), max(rb, 1), kb * rb)
    return q, s


# ---------------------------------------------------------------------------------------- products
def _scales(what, t, name, x, dev, shape, few):
    """rows of a block (1 or 128) of the scales of an operand: shape has one for each row, `few` one for 128"""
    if t is None:
        raise TypeError(f"{what}: {name} is required with 8-bit operands")
    if t.get_device() != dev:
        _elsewhere(x, t, what, name)
    if t.dtype != torch.float32:
        raise TypeError(f"{what}: {name} must be float32, got {t.dtype}")
    if t.shape == shape:
        return 1
    if few is not None and t.shape == few:
        return 128
    raise ValueError(f"{what}: {name} must be {list(shape)}{f' or {list(few)}' if few else ''}, got {list(t.shape)}")


def _out(what, out, out_dtype, x, M, N, default):
    if out is None:
        dt = out_dtype or default
        if dt not in _FLOAT:
            raise TypeError(f"{what}: out_dtype must be one of {', '.join(str(k)[6:] for k in _FLOAT)}, got {dt}")
        return x.new_empty((M, N), dtype=dt)
    if out.get_device() != x.get_device():
        _elsewhere(x, out, what, "out")
    _type(out, _FLOAT, what, "out")
    if out_dtype is not None and out.dtype != out_dtype:
        raise TypeError(f"{what}: out is {out.dtype}, out_dtype {out_dtype}")
    if tuple(out.shape) != (M, N) or (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
        raise ValueError(f"{what}: out must be [{M}, {N}] with unit column stride")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: out must not require a gradient")
    return out


def _wrote(out) -> None:
    """tells autograd that the caller's `out` was written: a graph that saved it before refuses to go back over it"""
    if out is not None:
        torch.autograd.graph.increment_version(out)


def matmul_fp8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *,
               bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [M, N] = x [M, K] @ w [N, K]^T (+ bias [N] f32) of float8_e4m3fn codes with their scales: x_scale
    [M, ceil(K / 128)]; w_scale [N, ceil(K / 128)] (block_rows 1) or [ceil(N / 128), ceil(K / 128)] (128).

    Each block's sum is scaled by the product of its two scales, taken in f32 (beyond f32's range an infinity, NaN
    with a sum of zero), and added in f32, and y is rounded once to out_dtype (bfloat16 by default; float16, float32).
    For float32 the products of a block are summed in f32.  For the 16-bit types the 8-bit matrix instruction sums
    them: in each 8 columns (8 i .. 8 i + 7) it cuts every product, towards zero, by less than 2^-13 of the largest
    one.  That is 1.5e-5 of an ordinary sum, far below a rounding of y; but where large products cancel, small
    ones beside them are lost, and float32 is the type to ask for.

    out: written in place of a new tensor (it must not overlap an input)."""
    what = "matmul_fp8"
    dev = _on(x, what)
    if w.get_device() != dev:
        _elsewhere(x, w, what, "w")
    if x.dtype != FP8 or w.dtype != FP8:
        raise TypeError(f"{what}: x and w must be float8_e4m3fn, got {x.dtype} and {w.dtype}")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"{what}: x must be [M, K] and w [N, K], got {list(x.shape)} and {list(w.shape)}")
    M, K = x.shape
    N = w.shape[0]
    kb = (K + 127) // 128
    _scales(what, x_scale, "x_scale", x, dev, (M, kb), None)
    wb = _scales(what, w_scale, "w_scale", x, dev, (N, kb), ((N + 127) // 128, kb))
    _no_grad(what, x, x_scale, w, w_scale, bias)
    if bias is not None:
        if bias.get_device() != dev:
            _elsewhere(x, bias, what, "bias")
        if bias.dtype != torch.float32 or bias.dim() != 1 or bias.shape[0] != N:
            raise ValueError(f"{what}: bias must be float32 [{N}]")
        bias = bias.contiguous()
    y = _out(what, out, out_dtype, x, M, N, torch.bfloat16)
    _no_tangent(what, x, x_scale, w, w_scale, bias, out)
    x, ldx = _rows(x)
    w, ldw = _rows(w)
    part, parts = None, 1
    if K > 24 * 128:  # (one part always, else)
        parts = lib().trk_matmul_fp8_parts(M, N, K)
        if parts > 1:
            part = x.new_empty((parts, M, N), dtype=torch.float32)
    _launch(what, "trk_matmul_fp8", x, x.data_ptr(), ldx, x_scale.data_ptr(), *x_scale.stride(), w.data_ptr(), ldw,
            w_scale.data_ptr(), *w_scale.stride(), wb, _at(bias), M, N, K, y.data_ptr(), y.stride(0) if M > 1 else max(N, 1),
            _FLOAT[y.dtype], _at(part), parts)
    _wrote(out)
    return y


def _weights(w: torch.Tensor):
    """(w [G, N, K] with unit column stride, its row stride)"""
    if not w.is_contiguous() and ((w.shape[2] > 1 and w.stride(2) != 1) or (w.shape[1] > 1 and w.stride(1) < w.shape[2])):
        w = w.contiguous()
    return w, w.stride(1) if w.shape[1] > 1 else max(w.shape[2], 1)


def _grouped_forward(what, x, x_scale, w, w_scale, wb, counts, in_dt, y, zero_tail):
    x, ldx = _rows(x)
    w, ldw = _weights(w)
    M, K = x.shape
    G, N = w.shape[:2]
    if x_scale is None:
        sx, sw = (None, 0, 0), (None, 0, 0, 0)
    else:
        sx = (x_scale.data_ptr(), *x_scale.stride())
        sw = (w_scale.data_ptr(), w_scale.stride(1), w_scale.stride(2), w_scale.stride(0))
    args = (x.data_ptr(), ldx, *sx, w.data_ptr(), ldw, w.stride(0), *sw, wb, counts.data_ptr(), G, M, N, K, in_dt,
            y.data_ptr(), y.stride(0) if M > 1 else max(N, 1), _FLOAT[y.dtype], zero_tail)
    item = x.element_size()
    if K * item > 24 * 128:  # (one part always, else)
        parts = lib().trk_matmul_grouped_parts(G, M, N, K, in_dt)
        # rows off the multiples of 16 bytes that were not copied are bound by their way through the registers (64 x
        # 6000 x 3500: strips 32 us, 47 in 6 parts)
        if parts > 1 and (x.data_ptr() | w.data_ptr() | ldx * item | ldw * item | w.stride(0) * item) % 16 == 0:
            part = x.new_empty((parts, M, N), dtype=torch.float32)
            _launch(what, "trk_matmul_grouped_split", x, *args, part.data_ptr(), parts)
            return
    _launch(what, "trk_matmul_grouped", x, *args)


def _laid(t: torch.Tensor) -> bool:
    """whether every row of t [.., K] of 16-bit values starts at a multiple of 16 bytes"""
    return t.data_ptr() % 16 == 0 and t.stride(-1) == 1 and all(s % 8 == 0 for s in t.stride()[:-1])


def _lay(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it with padded rows, so that _laid holds"""
    if _laid(t):
        return t
    return t.new_empty((*t.shape[:-1], (t.shape[-1] + 7) // 8 * 8))[..., :t.shape[-1]].copy_(t)


def _lay_pays(M: int, N: int, K: int, G: int) -> bool:
    """Whether x and w with rows off the multiples of 16 bytes are copied first (_lay).  The tiles take such rows
    through registers, about 1.5 us a step of 64 columns slower (8 groups of 16384 x 1501 x 1203 in all: 239 us,
    117 with the copies, 81 for aligned rows); the copies cost two launches and their bytes.  Few strips of rows
    are read at any alignment at no loss."""
    if -(-N // 16) * max(-(-M // 64), min(G, M)) <= 512:
        return False
    rounds = -(-(M // 128 + min(G, M)) * -(-N // 128) // 512)
    return 1.5 * (K // 64) * rounds > 10 + (M + G * N) * K / 750_000


def _lay_pays_backward(M: int, N: int, K: int, G: int, x, w, dy) -> bool:
    """The same for the gradients, of the operands they read (x: dw is wanted, w: dx is).  dx goes over dy and w in steps of
    64 columns of dy, about 3.5 us a step slower off the multiples of 16 bytes; dw over dy and x in steps of 64 rows of
    a group's part, about 5.5 us a step; even groups.  Below 50 us the kernels run under the host's part of a call,
    and the copies' host part is what counts.  us without / with copies of all operands, dx, dw, both: 8 groups of 16384 x
    1501 x 1203 in all 243 / 122, 265 / 119, 399 / 222; 3 of 3105 x 1301 x 1111 120 / 68, 96 / 71, 193 / 98; 64 of 4096 x
    511 x 513 55 / 67, 51 / 67, 81 / 84; 2 of 214 x 755 x 943 66 / 67, 51 / 67, 67 / 86."""
    if not (M and N and K):
        return False
    used, wide = min(G, M), -(-K // 256)
    slower = 0.0
    if w is not None:
        slower += 3.5 * (N // 64) * -(-used * -(-M // (used * 256)) * wide // 256)
    if x is not None:
        tiles = -(-N // 256) * wide * G
        split = max(1, min(256 // tiles, M // (256 * G)))
        slower += 5.5 * (M // (64 * G * split)) * -(-tiles * split // 256)
    both = x is not None and w is not None
    if slower + (1 + both) * M * N * K / 300_000_000 <= 50:
        return False
    copied = [t.numel() for t in (x, w, dy) if t is not None and not _laid(t)]
    return slower > 7 * len(copied) + sum(copied) / 1_270_000


class _Grouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, counts, dt, out_dtype, lay, links):
        want_x, want_w = ctx.needs_input_grad[:2]
        ctx.dt, ctx.sizes, ctx.links = dt, (x.shape[0], *w.shape), links
        if lay:
            x, w = _lay(x), _lay(w)
        # What the wanted gradients read; where x and w were copied, the copies: made again in the backward pass they would
        # cost 454 us a training step against 374 (16 groups of 8192 x 2047 x 2047), kept they cost their bytes till then
        ctx.save_for_backward(x if want_w else None, w if want_x else None, counts)
        y = x.new_empty((x.shape[0], w.shape[1]), dtype=out_dtype)
        _grouped_forward("matmul_grouped", x, None, w, None, 128, counts, dt, y, 1)
        return y

    @staticmethod
    @_backward_once("matmul_grouped")
    def backward(ctx, saved, dy):
        x, w, counts = saved
        M, G, N, K = ctx.sizes
        read = w if x is None else x
        if dy.dtype != read.dtype:
            dy = dy.to(read.dtype)
        if _lay_pays_backward(M, N, K, G, x, w, dy):
            x, w, dy = (None if t is None else _lay(t) for t in (x, w, dy))
        dy, ldy = _rows(dy)
        px, pw = (None, 0), (None, 0, 0)
        dx = dw = part = None
        parts = 1
        if w is not None:
            w, ldw = _weights(w)
            pw = (w.data_ptr(), ldw, w.stride(0))
            dx = dy.new_empty((M, K))
        if x is not None:
            x, ldx = _rows(x)
            px = (x.data_ptr(), ldx)
            dw = dy.new_empty((G, N, K))
            parts = lib().trk_matmul_grouped_bwd_parts(G, M, N, K)
            if parts > 1:
                part = dy.new_empty((parts, G, N, K), dtype=torch.float32)
        _launch("matmul_grouped backward", "trk_matmul_grouped_bwd", dy, dy.data_ptr(), ldy, *px, *pw, counts.data_ptr(), G, M, N, K,
                ctx.dt, _at(dx), max(K, 1), _at(dw), max(K, 1), N * K, _at(part), parts)
        return dx, dw, None, None, None, None, None


def matmul_grouped(x: torch.Tensor, w: torch.Tensor, counts: torch.Tensor, *, x_scale: Optional[torch.Tensor] = None,
                   w_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [R, N] = x [R, K] @ w[g]^T with the rows of x sorted by group: the first counts[0] rows belong to
    w[0], the next counts[1] to w[1], ..  w [G, N, K]; counts [G] int32 on the device (never read by the
    host; values below 0 count as 0 and their sum is cut at R).

    bfloat16 / float16 x and w (one type; differentiable in both, a gradient of another type is rounded to
    theirs), or float8_e4m3fn with x_scale
    [R, ceil(K / 128)] and w_scale [G, N or ceil(N / 128), ceil(K / 128)], summed as matmul_fp8 does it.  16-bit
    products are summed in f32.  y is rounded once to out_dtype
    (x's type, or bfloat16 for 8 bits; float16, float32).  Rows behind the last group are zeros in a new y;
    with `out` (which must not overlap an input) they are left as they were."""
    what = "matmul_grouped"
    dev = _on(x, what)
    if w.get_device() != dev:
        _elsewhere(x, w, what, "w")
    if counts.get_device() != dev:
        _elsewhere(x, counts, what, "counts")
    if x.dtype != w.dtype:
        raise TypeError(f"{what}: x is {x.dtype}, w {w.dtype}")
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2] or w.shape[0] < 1:
        raise ValueError(f"{what}: x must be [R, K] and w [G >= 1, N, K], got {list(x.shape)} and {list(w.shape)}")
    G, N, K = w.shape
    M = x.shape[0]
    if counts.dtype != torch.int32 or counts.dim() != 1 or counts.shape[0] != G:
        raise ValueError(f"{what}: counts must be int32 [{G}]")
    counts = counts.contiguous()
    _no_tangent(what, x, x_scale, w, w_scale, out)
    if x.dtype == FP8:
        kb = (K + 127) // 128
        _scales(what, x_scale, "x_scale", x, dev, (M, kb), None)
        wb = _scales(what, w_scale, "w_scale", x, dev, (G, N, kb), (G, (N + 127) // 128, kb))
        _no_grad(what, x, x_scale, w, w_scale)
        y = _out(what, out, out_dtype, x, M, N, torch.bfloat16)
        _grouped_forward(what, x, x_scale, w, w_scale, wb, counts, _lib.TRK_E4M3, y, int(out is None))
        _wrote(out)
        return y
    dt = _type(x, _HALF, what, "x")
    if x_scale is not None or w_scale is not None:
        raise TypeError(f"{what}: scales go with float8_e4m3fn operands only")
    if (x.requires_grad or w.requires_grad) and torch.is_grad_enabled():
        if out is not None:
            raise ValueError(f"{what}: `out` has no gradient; call without it, or under torch.no_grad()")
        if out_dtype is not None and out_dtype not in _FLOAT:
            raise TypeError(f"{what}: out_dtype must be one of {', '.join(str(k)[6:] for k in _FLOAT)}, got {out_dtype}")
        lay = _lay_pays(M, N, K, G)
        # (empty tensors with the history of x and w, which their padded copies lack)
        links = tuple(t[:0].clone() for t in (x, w) if t.requires_grad) if lay else ()
        return _Grouped.apply(x, w, counts, dt, out_dtype or x.dtype, lay, links)
    y = _out(what, out, out_dtype, x, M, N, x.dtype)
    if _lay_pays(M, N, K, G):
        x, w = _lay(x), _lay(w)
    _grouped_forward(what, x, None, w, None, 128, counts, dt, y, int(out is None))
    _wrote(out)
    return y
