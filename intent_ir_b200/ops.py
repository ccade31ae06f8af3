"""Device-resident entry points: torch CUDA tensors in, torch CUDA tensors out, no host
copies, no synchronisation.  Each function checks its tensors the way the reference's
generated launch wrapper does (``is_cuda`` / ``is_contiguous`` / dtype,
frontends/cuda/runtime.py:641-669), enqueues the kernel on torch's current stream
(:723, :731) through the C ABI and returns.  PyTorch only allocates the buffers.
"""

from __future__ import annotations

import ctypes as C
import functools
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import _lib
from .errors import B200LoweringError, B200RuntimeError

_TORCH_CODE = {
    torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.int32: _lib.I32,
    torch.int64: _lib.I64, torch.bool: _lib.BOOL, torch.uint8: _lib.U8, torch.int8: _lib.I8, torch.int16: _lib.I16,
    torch.float64: _lib.F64,
}
TORCH_OF_DTYPE = {
    "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32, "i64": torch.int64,
    "bool": torch.bool, "i1": torch.bool, "u8": torch.uint8, "i8": torch.int8, "i16": torch.int16, "f64": torch.float64,
}


def _check(rc: int, what: str) -> None:
    if rc == _lib.OK:
        return
    msg = f"{what}: {_lib.last_error()} (status {rc})"
    if rc == _lib.ERR_UNSUPPORTED:
        raise B200LoweringError(msg)
    raise B200RuntimeError(msg)


def _dev(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise B200RuntimeError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise B200RuntimeError(f"{name} must be contiguous")
    return t


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else (t.data_ptr() or None)


def _stream() -> int:
    # the handle of torch.cuda.current_stream(), without building the Stream object (3 us of a 10 us call)
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def code_of(t: torch.Tensor) -> int:
    try:
        return _TORCH_CODE[t.dtype]
    except KeyError:
        raise B200LoweringError(f"unsupported tensor dtype {t.dtype}") from None


# ---- device status word for the bounded waits of the tensor-core GEMM -----------------------
_status: Dict[int, torch.Tensor] = {}


def status_word() -> torch.Tensor:
    dev = torch.cuda.current_device()
    if dev not in _status:
        if torch.cuda.is_current_stream_capturing():
            # memory of the graph's own pool may be written by its other nodes, and a node that zeroes the word would wipe out what
            # earlier replays reported: the library's built-in word is neither
            _status[dev] = torch.as_tensor(_BuiltInWord(), device=f"cuda:{dev}")
        else:
            _status[dev] = torch.zeros(1, dtype=torch.int32, device=f"cuda:{dev}")
    return _status[dev]


class _BuiltInWord:
    """The library's status word on the current device, as torch takes foreign device memory."""

    def __init__(self) -> None:
        at = _lib.load().ib200_status_word()
        if not at:
            raise B200RuntimeError("the library has no status word on this device")
        self.__cuda_array_interface__ = {"shape": (1,), "typestr": "<i4", "data": (at, False), "version": 2}


def check_device_status() -> None:
    """Synchronise the current stream and raise if a bounded device-side wait expired."""
    dev = torch.cuda.current_device()
    if dev not in _status:
        return
    rc = _lib.load().ib200_check_status(_status[dev].data_ptr(), _stream())
    if rc != _lib.OK:
        msg = _lib.last_error()
        _status[dev].zero_()
        raise B200RuntimeError(msg)


# ---- ops ------------------------------------------------------------------------------------

def normalise_axes(dims: Sequence[int], rank: int) -> Tuple[int, ...]:
    axes = sorted({d + rank if d < 0 else d for d in dims})
    if any(a < 0 or a >= rank for a in axes):
        raise B200LoweringError(f"reduce axes {list(dims)} out of range for rank {rank}")
    return tuple(axes)


def reduce(x: torch.Tensor, kind: str, dims: Sequence[int], keepdims: bool = False, scale: float = 1.0,
           out_dtype: Optional[torch.dtype] = None, split: bool = True) -> torch.Tensor:
    """``reduce_sum`` / ``reduce_max`` / ``reduce_any`` over a contiguous run of axes.  With
    ``split`` (default) shapes with too few results to fill the GPU get scratch memory and are
    split along the reduced axis; the result does not vary from run to run either way."""
    _dev(x, "x")
    axes = normalise_axes(dims, x.dim())
    if not axes:
        raise B200LoweringError("reduce needs at least one axis")
    if axes != tuple(range(axes[0], axes[-1] + 1)):
        raise B200LoweringError(f"reduce axes {axes} are not adjacent")
    shape = list(x.shape)
    outer = int(torch.Size(shape[: axes[0]]).numel())
    red = int(torch.Size(shape[axes[0]: axes[-1] + 1]).numel())
    inner = int(torch.Size(shape[axes[-1] + 1:]).numel())
    kinds = {"sum": _lib.REDUCE_SUM, "max": _lib.REDUCE_MAX, "any": _lib.REDUCE_ANY}
    if out_dtype is None:
        out_dtype = torch.bool if kind == "any" else x.dtype
    out_shape = [1 if i in axes else d for i, d in enumerate(shape)] if keepdims else [d for i, d in enumerate(shape) if i not in axes]
    out = torch.empty(out_shape, dtype=out_dtype, device=x.device)
    lib = _lib.load()
    need = int(lib.ib200_reduce_scratch_bytes(outer, red, inner)) if split else 0
    if need:
        scratch = torch.empty(need, dtype=torch.uint8, device=x.device)  # freed stream-ordered by the caching allocator
        rc = lib.ib200_reduce_ws(_ptr(x), _ptr(out), code_of(x), code_of(out), kinds[kind], outer, red, inner, float(scale),
                                 _ptr(scratch), need, _stream())
    else:
        rc = lib.ib200_reduce(_ptr(x), _ptr(out), code_of(x), code_of(out), kinds[kind], outer, red, inner, float(scale), _stream())
    _check(rc, f"reduce_{kind}")
    return out


def softmax(x: torch.Tensor, out: Optional[torch.Tensor] = None, row_max: Optional[torch.Tensor] = None,
            row_sum: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Softmax over the last axis.  ``out_dtype`` (or the dtype of ``out``) may be float32 for
    bf16 / f16 inputs."""
    _dev(x, "x")
    cols = x.shape[-1] if x.dim() else 1
    rows = x.numel() // cols if cols else 0
    if out is None:
        out = torch.empty_like(x, dtype=out_dtype or x.dtype)
    _dev(out, "out")
    for t, n in ((row_max, "row_max"), (row_sum, "row_sum")):
        if t is not None and (_dev(t, n).dtype != torch.float32 or t.numel() != rows):
            raise B200RuntimeError(f"{n} must be f32 with one element per row")
    rc = _lib.load().ib200_softmax_io(_ptr(x), _ptr(out), _ptr(row_max), _ptr(row_sum), code_of(x), code_of(out), rows, cols, _stream())
    _check(rc, "softmax")
    return out


def softmax_masked(x: torch.Tensor, mask: torch.Tensor, fill: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(where(mask, x, fill))`` over the last axis of an f32 tensor in one kernel.  ``mask``
    (bool / uint8) has the shape of ``x`` or of its last axis (one vector shared by all rows)."""
    _dev(x, "x")
    _dev(mask, "mask")
    if x.dtype != torch.float32 or mask.dtype not in (torch.bool, torch.uint8):
        raise B200RuntimeError("softmax_masked: x must be float32 and mask bool or uint8")
    cols = x.shape[-1] if x.dim() else 1
    rows = x.numel() // cols if cols else 0
    if tuple(mask.shape) == tuple(x.shape):
        stride = cols
    elif mask.numel() == cols:
        stride = 0
    else:
        raise B200RuntimeError(f"softmax_masked: mask shape {tuple(mask.shape)} matches neither x {tuple(x.shape)} nor its last axis")
    if out is None:
        out = torch.empty_like(x)
    _dev(out, "out")
    rc = _lib.load().ib200_softmax_masked(_ptr(x), _ptr(mask), stride, float(fill), _ptr(out), None, None, rows, cols, _stream())
    _check(rc, "softmax_masked")
    return out


def norm_rows(x, w, b, rows: int, cols: int, affine_inner: int, affine_period: int, eps: float, want_stats: bool = True):
    _dev(x, "x")
    y = torch.empty_like(x)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device) if want_stats else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if want_stats else None
    aff = w if w is not None else b
    if w is not None and b is not None and w.dtype != b.dtype:
        raise B200LoweringError("norm: weight and bias must share a dtype")
    for t, n in ((w, "w"), (b, "b")):
        if t is not None:
            _dev(t, n)
    rc = _lib.load().ib200_norm_rows(
        _ptr(x), _ptr(w), _ptr(b), _ptr(y), _ptr(mean), _ptr(rstd), code_of(x), code_of(aff) if aff is not None else code_of(x),
        rows, cols, affine_inner, affine_period, float(eps), _stream())
    _check(rc, "norm_rows")
    return y, mean, rstd


def layernorm(x: torch.Tensor, w: Optional[torch.Tensor], b: Optional[torch.Tensor], eps: float = 1e-5):
    """y, mean[rows], rstd[rows] over the last axis of x."""
    cols = x.shape[-1]
    return norm_rows(x, w, b, x.numel() // max(cols, 1), cols, 1, cols, eps)


def groupnorm(x: torch.Tensor, w: Optional[torch.Tensor], b: Optional[torch.Tensor], groups: int, eps: float = 1e-5):
    """x is [N, C, *spatial]; returns y, mean[N, G], rstd[N, G]."""
    n, c = x.shape[0], x.shape[1]
    hw = x.numel() // max(n * c, 1)
    if groups <= 0 or c % groups:
        raise B200LoweringError(f"groupnorm: C={c} is not a multiple of groups={groups}")
    y, mean, rstd = norm_rows(x, w, b, n * groups, (c // groups) * hw, max(hw, 1), max(c, 1), eps)
    return y, mean.view(n, groups), rstd.view(n, groups)


_gemm_scratch: Dict[int, torch.Tensor] = {}


def gemm_bias_act(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
                  transpose_b: bool = False, out_dtype: Optional[torch.dtype] = None, allow_tf32: bool = False,
                  split_tail: bool = True, cta_pairs: Optional[bool] = None, narrow_tail: bool = False) -> torch.Tensor:
    """act(a @ b + bias) with fp32 accumulation; ``b`` is [K,N], or [N,K] with transpose_b.  bf16 / f16 operands
    (and f32 operands with ``allow_tf32``) whose K and N are multiples of 8 run on the tensor cores.  ``split_tail``
    gives the kernel scratch memory (kept per device, grown on demand) so that a last, mostly empty round of tiles
    is split along K.  ``cta_pairs``: True / False force the two-CTA (cta_group::2) or the one-CTA kernel; None lets the
    library choose (pairs for large products).  ``narrow_tail`` runs the pair kernel's last-round tiles as two half-width units each when they fill at most half of the pairs."""
    _dev(a, "a"), _dev(b, "b")
    if a.dim() != 2 or b.dim() != 2 or a.dtype != b.dtype:
        raise B200LoweringError("gemm: a and b must be rank-2 tensors of one dtype")
    m, k = a.shape
    n = b.shape[0] if transpose_b else b.shape[1]
    if (b.shape[1] if transpose_b else b.shape[0]) != k:
        raise B200LoweringError(f"gemm: inner extents differ: {tuple(a.shape)} x {tuple(b.shape)}")
    out_dtype = out_dtype or a.dtype
    c = torch.empty((m, n), dtype=out_dtype, device=a.device)
    if bias is not None:
        _dev(bias, "bias")
        if bias.dtype != out_dtype or bias.numel() != n:
            raise B200LoweringError("gemm: bias must have the output dtype and N elements")
    lib = _lib.load()
    flags = (_lib.GEMM_ALLOW_TF32 if allow_tf32 else 0) | (_lib.GEMM_CTA_PAIRS if cta_pairs else _lib.GEMM_ONE_CTA if cta_pairs is False else 0)
    flags |= _lib.GEMM_NARROW_TAIL if narrow_tail else 0
    need = lib.ib200_gemm_scratch_bytes(code_of(a), code_of(c), m, n, k, int(transpose_b), flags) if split_tail else 0
    scratch = None
    if need:
        dev = a.device.index if a.device.index is not None else torch.cuda.current_device()
        scratch = _gemm_scratch.get(dev)
        if scratch is None or scratch.numel() < need + 256:
            scratch = _gemm_scratch[dev] = torch.empty(need + 256, dtype=torch.uint8, device=a.device)
    rc = lib.ib200_gemm_bias_act_ws(
        _ptr(a), _ptr(b), _ptr(bias), _ptr(c), code_of(a), code_of(c), m, n, k, int(transpose_b),
        {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU}[act], flags, ((scratch.data_ptr() + 255) & ~255) if need else None, need,
        status_word().data_ptr(), _stream())
    _check(rc, "gemm_bias_act")
    return c


def transpose2d(x: torch.Tensor) -> torch.Tensor:
    _dev(x, "x")
    if x.dim() != 2:
        raise B200LoweringError("transpose2d needs a rank-2 tensor")
    out = torch.empty((x.shape[1], x.shape[0]), dtype=x.dtype, device=x.device)
    rc = _lib.load().ib200_transpose2d(_ptr(x), _ptr(out), x.element_size(), x.shape[0], x.shape[1], _stream())
    _check(rc, "transpose2d")
    return out


# ---- a decoder layer's serving step: activations, weights and the key / value cache in 8 or 4 bits ------------
# One-token steps are launch-bound, so these calls test all their arguments in one expression and look for the one
# to name only when it fails.

_FLOAT_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_HALF_CODE = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_HELD_CODE = {torch.float8_e4m3fn: _lib.E4M3, torch.int8: _lib.I8}


# what torch.cuda.current_device asks, once CUDA is up (there is a CUDA tensor by then), and the handle of torch.cuda.current_stream(device); a torch built
# without CUDA has neither, nor a tensor that would get as far
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _on_device(index: int, **tensors: Optional[torch.Tensor]) -> None:
    for name, t in tensors.items():
        if t is not None and (not isinstance(t, torch.Tensor) or t.get_device() != index):
            raise B200RuntimeError(f"{name} must be a tensor on cuda:{index}")


def _first(name: str, t) -> int:
    """The device of a call's first tensor."""
    if isinstance(t, torch.Tensor):
        index = t.get_device()
        if index >= 0:
            return index
    raise B200RuntimeError(f"{name} must be a CUDA tensor")


def _dense(name: str, t: torch.Tensor, shape: Sequence[int], dtype: torch.dtype) -> None:
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise B200RuntimeError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}, not {t.dtype} {tuple(t.shape)}")


def _row_stride(name: str, t: torch.Tensor) -> int:
    """The row stride of a contiguous tensor, or of a matrix of evenly spaced contiguous rows."""
    if t.dim() > 0:
        if t.is_contiguous():
            return t.shape[-1]
        if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
            return t.stride(0)
    raise B200RuntimeError(f"{name} must be contiguous, or a matrix of evenly spaced contiguous rows")


def _code(name: str, t: torch.Tensor, codes: Dict[torch.dtype, int]) -> int:
    try:
        return codes[t.dtype]
    except KeyError:
        raise B200LoweringError(f"{name}: unsupported dtype {t.dtype}") from None


def _address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _dense_empty(shape: Tuple[int, ...], dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    # of the ways to allocate without another tensor as a pattern this is the fastest (1.5 us; new_empty 2.1 - 2.5, empty 2.5)
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=dev)
    if len(shape) == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=dev)
    return torch.empty(shape, dtype=dtype, device=dev)


def rmsnorm(x: torch.Tensor, w: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
            out_dtype: Optional[torch.dtype] = None, group: int = 0, residual_out: Optional[torch.Tensor] = None):
    """``h = x + residual`` and ``y = h / sqrt(mean(h * h) + eps) * w`` over the last axis, in f32 from the unrounded sum; returns
    ``(y, scale, h)``.  ``h`` has the type of ``x`` and is None without a residual; ``residual_out`` says where it goes (it may be
    ``residual`` or ``x`` itself).  ``out_dtype`` float8_e4m3fn or int8 holds y in 8 bits, ``y * scale`` standing for the result,
    with one f32 scale for each row (``group`` 0) or for each 32, 64, 128 or 256 columns (``max|y| / Q``; y times ``Q / max|y|``, in f32, is
    rounded to nearest); otherwise y has the type of x and scale is None.  x is f32, bf16 or f16; w has its type or f32; x, residual and
    residual_out may be matrices of spaced rows.  A row's last bits may differ between calls of different shapes."""
    index = _first("x", x)
    if index != _current_device():
        with torch.cuda.device(index):
            return rmsnorm(x, w, residual, eps, out_dtype, group, residual_out)
    stride = _row_stride("x", x)
    shape, dtype = x.shape, x.dtype
    cols = shape[-1]
    code = w_code = _code("x", x, _FLOAT_CODE)
    if w is not None:
        if not isinstance(w, torch.Tensor) or w.get_device() != index or w.numel() != cols or not w.is_contiguous():
            raise B200RuntimeError(f"w must be contiguous on cuda:{index} with one element per column ({cols})")
        w_code = _code("w", w, _FLOAT_CODE)
    res_stride = h_stride = 0
    h = residual_out
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.get_device() != index or residual.shape != shape or residual.dtype != dtype:
            raise B200RuntimeError(f"residual must be on cuda:{index} with the shape and dtype of x")
        res_stride = _row_stride("residual", residual)
        if h is None:
            h = torch.empty_like(x) if stride == cols else _dense_empty(shape, dtype, x.device)
            h_stride = cols
        else:
            if not isinstance(h, torch.Tensor) or h.get_device() != index or h.shape != shape or h.dtype != dtype:
                raise B200RuntimeError(f"residual_out must be on cuda:{index} with the shape and dtype of x")
            h_stride = _row_stride("residual_out", h)
    elif h is not None:
        raise B200RuntimeError("residual_out needs a residual")
    scale = None
    out_code = code
    if out_dtype is None or out_dtype == dtype:
        y = torch.empty_like(x) if stride == cols else _dense_empty(shape, dtype, x.device)
    else:
        out_code = _HELD_CODE.get(out_dtype)
        if out_code is None:
            raise B200LoweringError(f"rmsnorm: the result is {dtype}, float8_e4m3fn or int8, not {out_dtype}")
        y = torch.empty_like(x, dtype=out_dtype) if stride == cols else _dense_empty(shape, out_dtype, x.device)
        scale = _dense_empty(shape[:-1] + ((cols + group - 1) // group if group > 0 else 1,), torch.float32, x.device)
    args = _lib.RMSNORM_ARGS.pack(x.data_ptr(), _address(residual), _address(w), y.data_ptr(), _address(h), _address(scale), stride, res_stride, h_stride,
                                  code, w_code, out_code, shape[:-1].numel(), cols, group, eps)
    rc = _lib.load().ib200_rmsnorm(args, _stream_of(index))
    if rc:
        _check(rc, "rmsnorm")
    return y, scale, h


def w4_matmul(x: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
              bias: Optional[torch.Tensor] = None, x_scale: Optional[torch.Tensor] = None, group: int = 128,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x @ w.T + bias`` for weights of 4 bits, ``w[n, k] = scales[n, k // group] * (q[n, k] - zeros[n, k // group])``, with f32 sums.
    ``q`` is uint8 [N, K/2] with the even k of a byte in its low half, ``scales`` [N, ceil(K / group)] f32 / bf16 / f16, ``zeros``
    uint8 of that shape (default 8), 0 to 127: one above makes its row of weights, a column of the result, NaN.  ``x`` [.., K] is
    bf16 or f16, or float8_e4m3fn / int8 with ``x_scale`` f32 [.., 1] or [.., ceil(K / group)], as ``rmsnorm`` returns them.
    ``out_dtype`` (default: the type of x, bf16 for 8-bit x) is also the bias's.  K is a multiple of 32 (up to 2^30 for more than 16
    rows, or 8 in groups of 128), the group 32, 64 or 128.  A wait inside the kernel that runs out is reported by ``check_device_status``."""
    index = _first("x", x)
    if index != _current_device():
        with torch.cuda.device(index):
            return w4_matmul(x, q, scales, zeros, bias, x_scale, group, out_dtype)
    for t in (q, scales, zeros, bias, x_scale):
        if t is not None and (not isinstance(t, torch.Tensor) or t.get_device() != index):
            _on_device(index, q=q, scales=scales, zeros=zeros, bias=bias, x_scale=x_scale)
    if q is None or scales is None or q.dim() != 2 or group not in (32, 64, 128):
        raise B200LoweringError("w4_matmul: q is a matrix, the group 32, 64 or 128")
    stride = _row_stride("x", x)
    front, k, n = x.shape[:-1], x.shape[-1], q.shape[0]
    if k % 32:
        raise B200LoweringError(f"w4_matmul: K = {k} is not a multiple of 32")
    groups = (k + group - 1) // group
    if q.dtype is not torch.uint8 or q.shape[1] * 2 != k or not q.is_contiguous():
        _dense("q", q, (n, k // 2), torch.uint8)
    if scales.shape != (n, groups) or not scales.is_contiguous():
        _dense("scales", scales, (n, groups), scales.dtype)
    if zeros is not None:
        _dense("zeros", zeros, (n, groups), torch.uint8)
    x_code = _HELD_CODE.get(x.dtype)
    x_groups = 0
    if x_code is not None:
        if x_scale is None or x_scale.dim() != x.dim() or x_scale.shape[:-1] != front or x_scale.shape[-1] not in (1, groups):
            raise B200RuntimeError(f"w4_matmul: 8-bit x needs x_scale of shape {tuple(front)} + (1 or {groups},)")
        _dense("x_scale", x_scale, x_scale.shape, torch.float32)
        x_groups = x_scale.shape[-1]
    else:
        x_code = _code("x", x, _HALF_CODE)
        if x_scale is not None:
            raise B200RuntimeError("w4_matmul: x_scale belongs to 8-bit x")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if x.dtype in _HELD_CODE else x.dtype
    elif out_dtype not in _FLOAT_CODE:
        raise B200LoweringError(f"w4_matmul: the result is float32, bfloat16 or float16, not {out_dtype}")
    y = _dense_empty(front + (n,), out_dtype, x.device)
    if bias is not None:
        _dense("bias", bias, (n,), out_dtype)
    m = front.numel()
    need = _w4_scratch(x_code, m, n, k, group)
    scratch = _dense_empty((need,), torch.uint8, x.device) if need else None
    args = _lib.W4_ARGS.pack(x.data_ptr(), _address(x_scale), q.data_ptr(), scales.data_ptr(), _address(zeros), _address(bias), y.data_ptr(), _address(scratch),
                             _status_address(index), stride, x_groups, x_code, _code("scales", scales, _FLOAT_CODE), _FLOAT_CODE[out_dtype], m, n, k, group, need)
    rc = _lib.load().ib200_w4_matmul(args, _stream_of(index))
    if rc:
        _check(rc, "w4_matmul")
    return y


def _status_address(index: int) -> int:
    """The status word of the current device, `index`."""
    word = _status.get(index)
    return (status_word() if word is None else word).data_ptr()


@functools.lru_cache(maxsize=4096)
def _w4_scratch(*extents: int) -> int:
    return _lib.load().ib200_w4_scratch_bytes(*extents)


@functools.lru_cache(maxsize=4096)
def _attention_scratch(*extents: int) -> int:
    return _lib.load().ib200_attention_kv8_scratch_bytes(*extents)


def _cache_extents(index: int, name: str, x, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_new):
    """The checked extents of the paged cache's arguments: held type's code, pages, heads, block, dim, batch, table_blocks."""
    try:
        pages, heads, block, dim = cache = k_cache.shape
        batch, table_blocks = block_table.shape
        f32, i32 = torch.float32, torch.int32
        good = (x.dim() == 3 and x.shape[2] == dim and x.stride(2) == 1 and v_cache.shape == cache and k_scale.shape == (pages, heads)
                and v_scale.shape == (pages, heads) and seq_lens.shape == (batch,)
                and v_cache.dtype is k_cache.dtype and k_scale.dtype is f32 and v_scale.dtype is f32 and block_table.dtype is i32 and seq_lens.dtype is i32
                and k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()
                and block_table.is_contiguous() and seq_lens.is_contiguous()
                and k_cache.get_device() == index and v_cache.get_device() == index and k_scale.get_device() == index and v_scale.get_device() == index
                and block_table.get_device() == index and seq_lens.get_device() == index
                and (cu_new is None or (cu_new.shape == (batch + 1,) and cu_new.dtype is i32 and cu_new.is_contiguous() and cu_new.get_device() == index)))
    except (AttributeError, ValueError):
        good = False
    if not good:
        _name_the_fault(index, name, x, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_new)
    return _code("k_cache", k_cache, _HELD_CODE), pages, heads, block, dim, batch, table_blocks


def _name_the_fault(index: int, name: str, x, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_new) -> None:
    _on_device(index, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, block_table=block_table, seq_lens=seq_lens, cu_new=cu_new)
    if any(t is None for t in (k_cache, v_cache, k_scale, v_scale, block_table, seq_lens)):
        raise B200RuntimeError("the caches, their scales, block_table and seq_lens are needed")
    if k_cache.dim() != 4 or block_table.dim() != 2 or x.dim() != 3:
        raise B200RuntimeError(f"{name} is [tokens, heads, dim], the caches [pages, heads, block, dim], block_table [sequences, blocks]")
    pages, heads = k_cache.shape[:2]
    batch = block_table.shape[0]
    _dense("k_cache", k_cache, k_cache.shape, k_cache.dtype)
    _dense("v_cache", v_cache, k_cache.shape, k_cache.dtype)
    _dense("k_scale", k_scale, (pages, heads), torch.float32)
    _dense("v_scale", v_scale, (pages, heads), torch.float32)
    _dense("block_table", block_table, block_table.shape, torch.int32)
    _dense("seq_lens", seq_lens, (batch,), torch.int32)
    if cu_new is not None:
        _dense("cu_new", cu_new, (batch + 1,), torch.int32)
    raise B200RuntimeError(f"{name} must have the cache's width {k_cache.shape[3]} as its last, adjacent axis")


def kv8_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, cu_new: Optional[torch.Tensor] = None) -> None:
    """Writes new tokens' keys and values ``k``, ``v`` [tokens, heads, dim] (bf16 / f16, last axis adjacent) into the caches
    [pages, heads, block, dim] (float8_e4m3fn or int8) with one f32 scale for each page and head, ``k_scale`` / ``v_scale``
    [pages, heads].  ``block_table`` [sequences, blocks] int32 names the pages, ``seq_lens`` [sequences] int32 the lengths with the
    new tokens, ``cu_new`` [sequences + 1] int32 where each sequence's new tokens lie (None: the same number for each).  A scale
    grows with its block's largest value, and the values held before are rounded again; slots behind the end, tokens behind
    ``cu_new[-1]``, and pages or tokens outside the cache and the table are left alone.  No page may take new tokens twice in a call, from two
    sequences or two blocks of one."""
    index = _first("k", k)
    if index != _current_device():
        with torch.cuda.device(index):
            return kv8_append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_new)
    held, pages, heads, block, dim, batch, table_blocks = _cache_extents(index, "k", k, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_new)
    if (not isinstance(v, torch.Tensor) or v.get_device() != index or v.shape != k.shape or v.dtype != k.dtype or k.shape[1] != heads
            or v.stride(2) != 1):
        raise B200RuntimeError(f"k and v must be [tokens, {heads}, {dim}] tensors of one dtype on cuda:{index} with adjacent last axes")
    k_token, k_head, _ = k.stride()
    v_token, v_head, _ = v.stride()
    args = _lib.KV8_APPEND_ARGS.pack(k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                     block_table.data_ptr(), seq_lens.data_ptr(), _address(cu_new), k_token, k_head, v_token, v_head,
                                     _code("k", k, _HALF_CODE), held, k.shape[0], batch, heads, dim, pages, block, table_blocks)
    rc = _lib.load().ib200_kv8_append(args, _stream_of(index))
    if rc:
        _check(rc, "kv8_append")


def attention_kv8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                  block_table: torch.Tensor, seq_lens: torch.Tensor, cu_new: Optional[torch.Tensor] = None,
                  scale: Optional[float] = None, window: int = 0, return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of the new tokens' queries ``q`` [tokens, query heads, dim] over the cache that ``kv8_append`` has put their keys
    and values into (same arguments): token i of a sequence's n new ones sees the keys up to its own place, seq_len - n + i, and
    with ``window`` > 0 only the last that many of them.  ``scale`` defaults to 1 / sqrt(dim); consecutive query heads share a key
    head.  Returns ``o`` of q's shape and dtype (``out``, if given), with ``return_lse`` also the f32 [tokens, query heads] logs of
    the softmax's denominators.  The softmax's numerators are rounded to f16 once (2^-12) for bf16 results and held in two f16 parts for f16
    ones, whatever scales the pages that a row does not see have; sums are f32.  Rows without keys are 0 (lse -inf); rows that need a
    page outside the cache or a token outside the table are NaN; tokens behind ``cu_new[-1]`` are not written."""
    index = _first("q", q)
    if index != _current_device():
        with torch.cuda.device(index):
            return attention_kv8(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_new, scale, window, return_lse, out)
    held, pages, heads, block, dim, batch, table_blocks = _cache_extents(index, "q", q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_new)
    tokens, q_heads, _ = shape = q.shape
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else _dense_empty(shape, q.dtype, q.device)
    else:
        _on_device(index, out=out)
        _dense("out", out, shape, q.dtype)
    dev = q.device
    lse = torch.empty_strided((tokens, q_heads), (q_heads, 1), dtype=torch.float32, device=dev) if return_lse else None
    need = _attention_scratch(tokens, batch, q_heads, heads, dim, block, table_blocks, cu_new is None)
    scratch = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=dev) if need else None
    q_token, q_head, _ = q.stride()
    args = _lib.ATTENTION_KV8_ARGS.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(),
                                        seq_lens.data_ptr(), _address(cu_new), out.data_ptr(), _address(lse), _address(scratch), q_token, q_head,
                                        _code("q", q, _HALF_CODE), held, tokens, batch, q_heads, heads, dim, pages, block, table_blocks, window, need,
                                        max(dim, 1) ** -0.5 if scale is None else scale)
    rc = _lib.load().ib200_attention_kv8(args, _stream_of(index))
    if rc:
        _check(rc, "attention_kv8")
    return (out, lse) if return_lse else out
