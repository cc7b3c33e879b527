"""torch-facing wrappers of the C ABI.

torch provides device memory and the current stream only; every computation
runs in the library's sm_100a kernels.  Tensors must be CUDA tensors with a
unit stride along their last dimension.  Calls are asynchronous on the given
stream (default: torch's current stream of the tensor's device).
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib

OUT_CODE = {torch.bfloat16: _lib.OUT_BF16, torch.float16: _lib.OUT_F16, torch.float32: _lib.OUT_F32}
QUANT_CODE = {"int8": _lib.QUANT_INT8, "fp8_e4m3": _lib.QUANT_FP8_E4M3}
QUANT_DTYPE = {"int8": torch.int8, "fp8_e4m3": torch.float8_e4m3fn}
F8_E4M3_MAX = 448.0


# torch's current raw cudaStream_t without building a Stream object (2 us -> 0.1 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_handle(device, stream=None) -> int:
    if stream is None:
        idx = device.index if isinstance(device, torch.device) else device
        if idx is None:
            idx = torch.cuda.current_device()
        if _raw_stream is not None:
            return _raw_stream(idx)
        return torch.cuda.current_stream(idx).cuda_stream
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(fn, idx: int, *args) -> None:
    """fn(*args, current stream or the given one) with CUDA device `idx` current; `args` ends with the
    stream (None: torch's current stream of that device).  Raises on a nonzero status."""
    stream = args[-1]
    if stream is None and _raw_stream is not None:
        handle = _raw_stream(idx)
    else:
        handle = _stream_handle(idx, stream)
    if _current_device() == idx:
        rc = fn(*args[:-1], handle)
    else:
        with _on(idx):
            rc = fn(*args[:-1], handle)
    if rc:
        _lib.check(rc)


class _on:
    """Makes `device` the current CUDA device inside the block (a no-op when it already is)."""
    __slots__ = ("idx", "prev")

    def __init__(self, device):
        self.idx = device.index if isinstance(device, torch.device) else device

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.idx is not None and self.idx != self.prev:
            torch.cuda.set_device(self.idx)

    def __exit__(self, *exc):
        if self.idx is not None and self.idx != self.prev:
            torch.cuda.set_device(self.prev)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need_cuda(name, t, dtype=None, ndim=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the library has no CPU path)")
    if dtype is not None and t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D, got shape {tuple(t.shape)}")
    if t.dim() >= 1 and t.numel() and t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit stride in its last dimension")


def gemm_dequant(x: torch.Tensor, w: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor,
                 bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 out_dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """out = cast(((f32(x @ w^T) * x_scale[:, None]) * w_scale) + bias).

    x [M, K] and w [N, K] are both int8 (exact int32 accumulation) or both
    float8_e4m3fn (fp32 accumulation); x_scale [M] float32; w_scale [N] or [1]
    float32; bias [N] in the output dtype or None/empty; out [M, N] bf16/fp16/fp32.
    """
    if out is None and isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor) and x.dim() == 2 and w.dim() == 2:
        out = torch.empty(x.shape[0], w.shape[0], dtype=out_dtype, device=x.device)
    if not _gemm_args_ok(x, w, x_scale, w_scale, bias, out):
        _gemm_args_explain(x, w, x_scale, w_scale, bias, out)
    M, K = x.shape
    N = w.shape[0]
    nb = 0 if bias is None else bias.numel()
    fn = _lib.load().t8g_gemm_i8_dequant if x.dtype is torch.int8 else _lib.load().t8g_gemm_fp8_dequant
    idx = x.get_device()
    with _on(idx):
        rc = fn(x.data_ptr(), w.data_ptr(), x_scale.data_ptr(), w_scale.data_ptr(), w_scale.numel(),
                bias.data_ptr() if nb else None, nb, out.data_ptr(), OUT_CODE[out.dtype], M, N, K, x.stride(0),
                w.stride(0), out.stride(0), _stream_handle(idx, stream))
    if rc:
        _lib.check(rc)
    return out


_GEMM_IN = (torch.int8, torch.float8_e4m3fn)


def _gemm_args_ok(x, w, xs, ws, bias, out) -> bool:
    """The common case of gemm_dequant's argument rules, checked cheaply; a False sends the
    call through _gemm_args_explain, which raises the precise error."""
    try:
        xd = x.dtype
        if xd not in _GEMM_IN or w.dtype is not xd or x.dim() != 2 or w.dim() != 2 or out is None or out.dim() != 2:
            return False
        M, K = x.shape
        N, Kw = w.shape
        if Kw != K or out.shape[0] != M or out.shape[1] != N or out.dtype not in OUT_CODE:
            return False
        if not (x.is_cuda and w.is_cuda and xs.is_cuda and ws.is_cuda and out.is_cuda):
            return False
        d = x.get_device()
        if w.get_device() != d or xs.get_device() != d or ws.get_device() != d or out.get_device() != d:
            return False
        if (M and K and x.stride(1) != 1) or (N and K and w.stride(1) != 1) or (M and N and out.stride(1) != 1):
            return False
        if xs.dtype is not torch.float32 or ws.dtype is not torch.float32:
            return False
        if xs.numel() != M or not xs.is_contiguous() or ws.numel() not in (1, N) or not ws.is_contiguous():
            return False
        if bias is not None and bias.numel():
            if (not bias.is_cuda or bias.get_device() != d or bias.dtype is not out.dtype or bias.numel() != N
                    or not bias.is_contiguous()):
                return False
        return True
    except (AttributeError, TypeError, ValueError):
        return False


def _gemm_args_explain(x, w, x_scale, w_scale, bias, out) -> None:
    _need_cuda("x", x, _GEMM_IN, 2)
    _need_cuda("w", w, x.dtype, 2)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"w has K={w.shape[1]}, x has K={K}")
    _need_cuda("x_scale", x_scale, torch.float32)
    _need_cuda("w_scale", w_scale, torch.float32)
    if x_scale.numel() != M or not x_scale.is_contiguous():
        raise ValueError("x_scale must be a contiguous float32 tensor with M elements")
    if w_scale.numel() not in (1, N) or not w_scale.is_contiguous():
        raise ValueError("w_scale must be a contiguous float32 tensor with 1 or N elements")
    _need_cuda("out", out, tuple(OUT_CODE), 2)
    if tuple(out.shape) != (M, N):
        raise ValueError(f"out has shape {tuple(out.shape)}, expected {(M, N)}")
    if bias is not None and bias.numel():
        _need_cuda("bias", bias, out.dtype)
        if bias.numel() != N or not bias.is_contiguous():
            raise ValueError("bias must be contiguous with N elements, in the output dtype")
    ts = [x, w, x_scale, w_scale, out] + ([bias] if bias is not None and bias.numel() else [])
    if len({t.get_device() for t in ts}) != 1:
        raise ValueError("x, w, the scales, bias and out must be on one CUDA device")
    raise ValueError("gemm_dequant: arguments rejected")   # the fast check and this one disagree


SWIGLU_BLOCK = 128


def interleave_gate_up(t: torch.Tensor, block: int = SWIGLU_BLOCK) -> torch.Tensor:
    """Reorder an fc1 parameter whose first half (along dim 0) is gate and second half up
    into the layout of gemm_swiglu: blocks of `block` gate rows followed by the matching
    `block` up rows.  Works for the weight [2F, K], its per-channel scales [2F] and the
    bias [2F]; done once when the weights are loaded."""
    n = t.shape[0]
    if n % (2 * block):
        raise ValueError(f"dim 0 ({n}) must be a multiple of {2 * block}")
    F = n // 2
    g = t[:F].reshape(F // block, block, *t.shape[1:])
    u = t[F:].reshape(F // block, block, *t.shape[1:])
    return torch.stack([g, u], dim=1).reshape(t.shape).contiguous()


def gemm_swiglu(x: torch.Tensor, w_il: torch.Tensor, x_scale: torch.Tensor, w_scale_il: torch.Tensor,
                bias_il: torch.Tensor | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """act = bf16(silu(gate) * up) of the fc1 GEMM, fused: gate / up are the bf16 outputs
    the plain gemm_dequant would produce for fc1 channels j and F + j.  w_il, w_scale_il
    (numel 2F, or 1) and bias_il (bf16, 2F) come from interleave_gate_up; x int8 [M, K] or
    float8_e4m3fn; out [M, F] bf16."""
    _need_cuda("x", x, (torch.int8, torch.float8_e4m3fn), 2)
    _need_cuda("w", w_il, x.dtype, 2)
    M, K = x.shape
    N = w_il.shape[0]
    if w_il.shape[1] != K:
        raise ValueError(f"w has K={w_il.shape[1]}, x has K={K}")
    if N % (2 * SWIGLU_BLOCK):
        raise ValueError(f"w must have 2F rows with F a multiple of {SWIGLU_BLOCK}")
    F = N // 2
    _need_cuda("x_scale", x_scale, torch.float32)
    _need_cuda("w_scale", w_scale_il, torch.float32)
    if x_scale.numel() != M or not x_scale.is_contiguous():
        raise ValueError("x_scale must be a contiguous float32 tensor with M elements")
    if w_scale_il.numel() not in (1, N) or not w_scale_il.is_contiguous():
        raise ValueError("w_scale must be a contiguous float32 tensor with 1 or 2F elements")
    if out is None:
        out = torch.empty(M, F, dtype=torch.bfloat16, device=x.device)
    _need_cuda("out", out, torch.bfloat16, 2)
    if tuple(out.shape) != (M, F):
        raise ValueError(f"out has shape {tuple(out.shape)}, expected {(M, F)}")
    nb = 0 if bias_il is None else bias_il.numel()
    if nb:
        _need_cuda("bias", bias_il, torch.bfloat16)
        if nb != N or not bias_il.is_contiguous():
            raise ValueError("bias must be contiguous bf16 with 2F elements")
    lib = _lib.load()
    fn = lib.t8g_gemm_i8_swiglu if x.dtype == torch.int8 else lib.t8g_gemm_fp8_swiglu
    with _on(x.device):
        rc = fn(_ptr(x), _ptr(w_il), _ptr(x_scale), _ptr(w_scale_il), w_scale_il.numel(),
                _ptr(bias_il) if nb else None, nb, _ptr(out), M, F, K, x.stride(0), w_il.stride(0), out.stride(0),
                _stream_handle(x.device, stream))
    _lib.check(rc)
    return out


def gemm_swiglu_quant(x: torch.Tensor, w_il: torch.Tensor, x_scale: torch.Tensor, w_scale_il: torch.Tensor,
                      bias_il: torch.Tensor | None = None, kind: str = "int8", act: torch.Tensor | None = None,
                      stream=None):
    """fc1 + SwiGLU + per-token quantisation of act in one call -> (q, q_scale, act): the SwiGLU
    epilogue also reports each row's max |act|, so the quantiser streams act once (equal bit
    for bit to quant_rows(gemm_swiglu(...)))."""
    _need_cuda("x", x, (torch.int8, torch.float8_e4m3fn), 2)
    _need_cuda("w", w_il, x.dtype, 2)
    M, K = x.shape
    N = w_il.shape[0]
    if w_il.shape[1] != K:
        raise ValueError(f"w has K={w_il.shape[1]}, x has K={K}")
    if N % (2 * SWIGLU_BLOCK):
        raise ValueError(f"w must have 2F rows with F a multiple of {SWIGLU_BLOCK}")
    F = N // 2
    _need_cuda("x_scale", x_scale, torch.float32)
    _need_cuda("w_scale", w_scale_il, torch.float32)
    if x_scale.numel() != M or not x_scale.is_contiguous():
        raise ValueError("x_scale must be a contiguous float32 tensor with M elements")
    if w_scale_il.numel() not in (1, N) or not w_scale_il.is_contiguous():
        raise ValueError("w_scale must be a contiguous float32 tensor with 1 or 2F elements")
    if act is None:
        act = torch.empty(M, F, dtype=torch.bfloat16, device=x.device)
    _need_cuda("act", act, torch.bfloat16, 2)
    if tuple(act.shape) != (M, F):
        raise ValueError(f"act has shape {tuple(act.shape)}, expected {(M, F)}")
    nb = 0 if bias_il is None else bias_il.numel()
    if nb:
        _need_cuda("bias", bias_il, torch.bfloat16)
        if nb != N or not bias_il.is_contiguous():
            raise ValueError("bias must be contiguous bf16 with 2F elements")
    amax = torch.empty(M, dtype=torch.float32, device=x.device)
    q = torch.empty(M, F, dtype=QUANT_DTYPE[kind], device=x.device)
    q_scale = torch.empty(M, dtype=torch.float32, device=x.device)
    lib = _lib.load()
    fn = lib.t8g_gemm_i8_swiglu_quant if x.dtype == torch.int8 else lib.t8g_gemm_fp8_swiglu_quant
    with _on(x.device):
        rc = fn(_ptr(x), _ptr(w_il), _ptr(x_scale), _ptr(w_scale_il), w_scale_il.numel(),
                _ptr(bias_il) if nb else None, nb, _ptr(act), act.stride(0), _ptr(amax), _ptr(q), q.stride(0),
                _ptr(q_scale), M, F, K, x.stride(0), w_il.stride(0), QUANT_CODE[kind], _stream_handle(x.device, stream))
    _lib.check(rc)
    return q, q_scale, act


def gemm_gated(x: torch.Tensor, w: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor,
               bias: torch.Tensor | None, res: torch.Tensor, gate: torch.Tensor, *,
               rows_per_gate: int | None = None, gate_index: torch.Tensor | None = None,
               out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The DiT block's gated residual with the projection GEMM fused in front of it:
    out = res + gate[g] * y in torch's bf16 order (t = bf16(gate * y), out = bf16(res + t)),
    y = gemm_dequant(x, w, x_scale, w_scale, bias) as bf16, never stored.  g is
    gate_index[m] (int32 [M]) or m // rows_per_gate (default: M // gate rows, which must
    divide M).  res [M, N] bf16; gate [n_gate, N] bf16; out [M, N] bf16, may be res itself
    (in-place update)."""
    _need_cuda("x", x, (torch.int8, torch.float8_e4m3fn), 2)
    _need_cuda("w", w, x.dtype, 2)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"w has K={w.shape[1]}, x has K={K}")
    _need_cuda("x_scale", x_scale, torch.float32)
    _need_cuda("w_scale", w_scale, torch.float32)
    if x_scale.numel() != M or not x_scale.is_contiguous():
        raise ValueError("x_scale must be a contiguous float32 tensor with M elements")
    if w_scale.numel() not in (1, N) or not w_scale.is_contiguous():
        raise ValueError("w_scale must be a contiguous float32 tensor with 1 or N elements")
    _need_cuda("res", res, torch.bfloat16, 2)
    if tuple(res.shape) != (M, N):
        raise ValueError(f"res has shape {tuple(res.shape)}, expected {(M, N)}")
    if gate.dim() == 1:
        gate = gate.view(1, -1)
    _need_cuda("gate", gate, torch.bfloat16, 2)
    if gate.shape[1] != N or gate.shape[0] < 1:
        raise ValueError(f"gate must be [n_gate, {N}], got {tuple(gate.shape)}")
    if gate_index is not None:
        _need_cuda("gate_index", gate_index, torch.int32, 1)
        if gate_index.numel() != M or not gate_index.is_contiguous():
            raise ValueError("gate_index must be a contiguous int32 tensor with M elements")
        rpg = 0
    else:
        if rows_per_gate is None:
            if M % gate.shape[0]:
                raise ValueError(f"{M} rows do not split evenly over {gate.shape[0]} gate rows; pass gate_index")
            rows_per_gate = max(1, M // gate.shape[0])
        rpg = int(rows_per_gate)
        if rpg < 1 or (M and (M - 1) // rpg >= gate.shape[0]):
            raise ValueError(f"rows_per_gate={rpg} maps rows past the {gate.shape[0]} gate rows")
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
    _need_cuda("out", out, torch.bfloat16, 2)
    if tuple(out.shape) != (M, N):
        raise ValueError(f"out has shape {tuple(out.shape)}, expected {(M, N)}")
    nb = 0 if bias is None else bias.numel()
    if nb:
        _need_cuda("bias", bias, torch.bfloat16)
        if nb != N or not bias.is_contiguous():
            raise ValueError("bias must be contiguous bf16 with N elements")
    lib = _lib.load()
    fn = lib.t8g_gemm_i8_gated if x.dtype == torch.int8 else lib.t8g_gemm_fp8_gated
    with _on(x.device):
        rc = fn(_ptr(x), _ptr(w), _ptr(x_scale), _ptr(w_scale), w_scale.numel(), _ptr(bias) if nb else None, nb,
                _ptr(res), res.stride(0), _ptr(gate), gate.stride(0), _ptr(gate_index), rpg, _ptr(out),
                M, N, K, x.stride(0), w.stride(0), out.stride(0), _stream_handle(x.device, stream))
    _lib.check(rc)
    return out


def quant_rows(x: torch.Tensor, kind: str = "int8", q: torch.Tensor | None = None,
               q_scale: torch.Tensor | None = None, stream=None):
    """Per-token quantisation of a bf16 [S, D] matrix -> (q [S, D], q_scale [S] float32)."""
    _need_cuda("x", x, torch.bfloat16, 2)
    S, D = x.shape
    if q is None:
        q = torch.empty(S, D, dtype=QUANT_DTYPE[kind], device=x.device)
    if q_scale is None:
        q_scale = torch.empty(S, dtype=torch.float32, device=x.device)
    _need_cuda("q", q, QUANT_DTYPE[kind], 2)
    with _on(x.device):
        rc = _lib.load().t8g_quant_rows(_ptr(x), x.stride(0), _ptr(q), q.stride(0), _ptr(q_scale), S, D,
                                        QUANT_CODE[kind], _stream_handle(x.device, stream))
    _lib.check(rc)
    return q, q_scale


def _mod_args(x, shift, scale, mod_index, rows_per_mod):
    S, D = x.shape
    for name, t in (("shift", shift), ("scale", scale)):
        _need_cuda(name, t, torch.bfloat16)
        if t.dim() == 1:
            if t.shape[0] != D:
                raise ValueError(f"{name} must have D={D} elements")
        elif t.dim() != 2 or t.shape[1] != D:
            raise ValueError(f"{name} must be [n_mod, D]")
    shift2 = shift.reshape(-1, D)
    scale2 = scale.reshape(-1, D)
    if shift2.stride(0) != scale2.stride(0):
        raise ValueError("shift and scale must share a row stride")
    if mod_index is not None:
        _need_cuda("mod_index", mod_index, torch.int32, 1)
        if mod_index.numel() != S or not mod_index.is_contiguous():
            raise ValueError("mod_index must be a contiguous int32 tensor with S elements")
        rows_per_mod = 1
    elif rows_per_mod is None:
        n_mod = shift2.shape[0]
        if S and (not n_mod or S % n_mod):
            raise ValueError(f"{S} rows do not split evenly over {n_mod} modulation rows; pass mod_index")
        rows_per_mod = max(S // max(n_mod, 1), 1)
    return shift2, scale2, rows_per_mod


def rms_mod_quant(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *, w: torch.Tensor | None = None,
                  mod_index: torch.Tensor | None = None, rows_per_mod: int | None = None,
                  scale_is_multiplier: bool = False, eps: float = 1e-6, kind: str = "fp8_e4m3",
                  return_h: bool = False, return_res: bool = False, stream=None):
    """One-pass RMSNorm + adaLN modulation + per-token quantisation of x [S, D] bf16.

    h = rms_norm(x) * w * s + shift[row], s = bf16(1 + scale[row]) (or scale itself
    when scale_is_multiplier); the modulation row of token r is mod_index[r], or
    r // rows_per_mod (default: S split evenly over the rows of shift/scale).
    Returns (q, q_scale[, h][, res]).
    """
    _need_cuda("x", x, torch.bfloat16, 2)
    S, D = x.shape
    shift2, scale2, rpm = _mod_args(x, shift, scale, mod_index, rows_per_mod)
    if w is not None:
        _need_cuda("w", w, torch.bfloat16, 1)
        if w.numel() != D:
            raise ValueError("w must have D elements")
    q = torch.empty(S, D, dtype=QUANT_DTYPE[kind], device=x.device)
    q_scale = torch.empty(S, dtype=torch.float32, device=x.device)
    h = torch.empty_like(x) if return_h else None
    res = torch.empty_like(x) if return_res else None
    with _on(x.device):
        rc = _lib.load().t8g_rms_mod_quant(
            _ptr(x), x.stride(0), _ptr(w), _ptr(shift2), _ptr(scale2), shift2.stride(0), _ptr(mod_index), rpm,
            int(scale_is_multiplier), float(eps), _ptr(q), q.stride(0), _ptr(q_scale), _ptr(h), D, _ptr(res), D,
            S, D, QUANT_CODE[kind], _stream_handle(x.device, stream))
    _lib.check(rc)
    out = [q, q_scale]
    if return_h:
        out.append(h)
    if return_res:
        out.append(res)
    return tuple(out)


def rms_mod_quant_tensorwise(x, shift, scale, *, w=None, mod_index=None, rows_per_mod=None,
                             scale_is_multiplier=False, eps=1e-5, kind="fp8_e4m3", want_res=True, stream=None):
    """The reference's two-phase form: (q, scale 0-d tensor, h, res); one scale for the tensor."""
    _need_cuda("x", x, torch.bfloat16, 2)
    S, D = x.shape
    shift2, scale2, rpm = _mod_args(x, shift, scale, mod_index, rows_per_mod)
    if w is not None:
        _need_cuda("w", w, torch.bfloat16, 1)
    q = torch.empty(S, D, dtype=QUANT_DTYPE[kind], device=x.device)
    h = torch.empty_like(x)
    res = torch.empty_like(x) if want_res else None
    amax = torch.zeros((), dtype=torch.float32, device=x.device)
    qs = torch.empty((), dtype=torch.float32, device=x.device)
    with _on(x.device):
        rc = _lib.load().t8g_rms_mod_quant_tensorwise(
            _ptr(x), x.stride(0), _ptr(w), _ptr(shift2), _ptr(scale2), shift2.stride(0), _ptr(mod_index), rpm,
            int(scale_is_multiplier), float(eps), _ptr(q), q.stride(0), _ptr(h), D, _ptr(res), D, _ptr(amax),
            _ptr(qs), S, D, QUANT_CODE[kind], _stream_handle(x.device, stream))
    _lib.check(rc)
    return q, qs, h, res


def swiglu_quant(gate: torch.Tensor, up: torch.Tensor, kind: str = "int8", return_act: bool = False, stream=None):
    """act = bf16(silu(gate) * up), per-token quantised -> (q, q_scale[, act]).

    gate and up are [M, F] bf16 views with the same row stride (for example the
    two halves of a [M, 2F] fc1 output, read in place)."""
    _need_cuda("gate", gate, torch.bfloat16, 2)
    _need_cuda("up", up, torch.bfloat16, 2)
    if gate.shape != up.shape or gate.stride() != up.stride():
        raise ValueError("gate and up must have the same shape and strides")
    M, F = gate.shape
    q = torch.empty(M, F, dtype=QUANT_DTYPE[kind], device=gate.device)
    q_scale = torch.empty(M, dtype=torch.float32, device=gate.device)
    act = torch.empty(M, F, dtype=torch.bfloat16, device=gate.device) if return_act else None
    with _on(gate.device):
        rc = _lib.load().t8g_swiglu_quant(_ptr(gate), _ptr(up), gate.stride(0), _ptr(q), q.stride(0), _ptr(q_scale),
                                          _ptr(act), F, M, F, QUANT_CODE[kind], _stream_handle(gate.device, stream))
    _lib.check(rc)
    return (q, q_scale, act) if return_act else (q, q_scale)


def swiglu_quant_fc1(y: torch.Tensor, kind: str = "int8", return_act: bool = False, stream=None):
    """SwiGLU + quant of a [M, 2F] fc1 output whose first half is the gate."""
    F = y.shape[-1] // 2
    return swiglu_quant(y[:, :F], y[:, F:], kind=kind, return_act=return_act, stream=stream)


def swiglu_quant_tensorwise(gate, up, kind="fp8_e4m3", stream=None):
    """The reference's two-phase form: (q, scale 0-d tensor, act)."""
    _need_cuda("gate", gate, torch.bfloat16, 2)
    _need_cuda("up", up, torch.bfloat16, 2)
    if gate.shape != up.shape or gate.stride() != up.stride():
        raise ValueError("gate and up must have the same shape and strides")
    M, F = gate.shape
    q = torch.empty(M, F, dtype=QUANT_DTYPE[kind], device=gate.device)
    act = torch.empty(M, F, dtype=torch.bfloat16, device=gate.device)
    amax = torch.zeros((), dtype=torch.float32, device=gate.device)
    qs = torch.empty((), dtype=torch.float32, device=gate.device)
    with _on(gate.device):
        rc = _lib.load().t8g_swiglu_quant_tensorwise(_ptr(gate), _ptr(up), gate.stride(0), _ptr(q), q.stride(0),
                                                     _ptr(act), F, _ptr(amax), _ptr(qs), M, F, QUANT_CODE[kind],
                                                     _stream_handle(gate.device, stream))
    _lib.check(rc)
    return q, qs, act


# ---------------------------------------------------------------- microscaled 4-bit formats
# A 4-bit matrix [S, D] is (q, sf, q_scale): q uint8 [S, D / 2], two e2m1 codes a byte (the even column in
# the low half) at a row pitch that is a multiple of 16 bytes; sf uint8, the block scales in tiles of
# 128 rows x 4 blocks (`fp4_scale_rows` gives them row by row); q_scale float32 [S], or None (mxfp4).
# The tiles' rows past S are never written nor read into a result: compare operands by `fp4_scale_rows`, not by sf.
# A call with `stream` is as the same call with that stream current: its outputs are that stream's.
FP4_CODE = {"mxfp4": _lib.QUANT_MXFP4, "nvfp4": _lib.QUANT_NVFP4}
FP4_BLOCK = {"mxfp4": 32, "nvfp4": 16}


class _NoCallPath:
    """In the compiled call path's place where that module is not built (or for another Python): every call
    takes the general path."""

    @staticmethod
    def _declines(*args) -> bool:
        return False

    gemm = gated = quant_rows = swiglu_fc1 = rms_mod_quant = dequant = _declines


_fp4_module = None


def _fp4_fast():
    """The compiled call path of the common case (csrc/fp4_call.c); each of its functions returns True
    when it launched, False for the general path below, or the library's status."""
    global _fp4_module
    if _fp4_module is None:
        _lib.load()   # raises where the library itself is missing
        try:
            from . import _t8g_fp4
        except ImportError:
            _fp4_module = _NoCallPath
            return _fp4_module
        raw = _raw_stream or (lambda idx: torch.cuda.current_stream(idx).cuda_stream)
        _t8g_fp4.setup(torch.uint8, torch.float32, torch.bfloat16, raw)
        _fp4_module = _t8g_fp4
    return _fp4_module


def _fp4_launched(r) -> bool:
    if r is True or r is False:
        return r
    _lib.check(r)
    return True


def _raw(stream):
    return stream if stream is None or isinstance(stream, int) else _stream_handle(None, stream)


def _fp4_code(kind: str) -> int:
    if kind not in FP4_CODE:
        raise ValueError(f"kind {kind!r} is not a 4-bit format ({', '.join(FP4_CODE)})")
    return FP4_CODE[kind]


def fp4_scale_bytes(rows: int, D: int, kind: str) -> int:
    """Bytes of the block scales of a [rows, D] 4-bit matrix (as t8g_fp4_scale_bytes)."""
    _fp4_code(kind)
    if rows < 0 or D < 0:
        raise ValueError(f"bad sizes {rows} x {D}")
    return _fp4_scale_bytes(rows, D, kind)


def _fp4_scale_bytes(rows: int, D: int, kind: str) -> int:
    return (rows + 127) // 128 * ((D + 127) // 128 if kind == "mxfp4" else (D + 63) // 64) * 512


def fp4_scale_rows(sf: torch.Tensor, rows: int, D: int, kind: str) -> torch.Tensor:
    """The block scales as a [rows, ceil(D / block)] uint8 matrix (e8m0 or e4m3 bytes)."""
    _fp4_code(kind)
    blocks = -(-D // FP4_BLOCK[kind])
    groups = -(-rows // 128)
    words = -(-blocks // 4)
    t = sf[:fp4_scale_bytes(rows, D, kind)].view(groups, words, 32, 4, 4)
    return t.permute(0, 3, 2, 1, 4).reshape(groups * 128, 4 * words)[:rows, :blocks]


def _stream_memory(stream, device):
    """Context for allocating the outputs of a call on `stream`: from the memory that torch keeps for that
    stream.  A block freed by work on the current stream may still be written there, and an output is not given
    back to that work while `stream` runs."""
    if device.type != "cuda":
        return contextlib.nullcontext()   # the call is refused later
    if not isinstance(stream, torch.cuda.Stream):
        handle = int(stream)
        stream = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
    return torch.cuda.stream(stream)


def _empty(M: int, N: int, dtype: torch.dtype, device, stream) -> torch.Tensor:
    if stream is not None:
        with _stream_memory(stream, device):
            return torch.empty(M, N, dtype=dtype, device=device)
    return torch.empty(M, N, dtype=dtype, device=device)


def _empty_like(t: torch.Tensor, stream) -> torch.Tensor:
    if stream is not None:
        with _stream_memory(stream, t.device):
            return torch.empty_like(t, memory_format=torch.contiguous_format)
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _fp4_empty(S: int, D: int, kind: str, device, stream):
    if stream is not None:
        with _stream_memory(stream, device):
            return _fp4_empty(S, D, kind, device, None)
    if D % 32:
        q = torch.empty(S, -(-D // 32) * 16, dtype=torch.uint8, device=device)[:, :D // 2]
    else:
        q = torch.empty(S, D // 2, dtype=torch.uint8, device=device)
    sf = torch.empty(_fp4_scale_bytes(S, D, kind), dtype=torch.uint8, device=device)
    q_scale = torch.empty(S, dtype=torch.float32, device=device) if kind == "nvfp4" else None
    return q, sf, q_scale


def _pitch(t: torch.Tensor, rows: int, width: int, multiple: int) -> int:
    """Row stride in elements of a [rows, width] matrix; a single row has none of its own."""
    return t.stride(0) if rows > 1 else -(-width // multiple) * multiple


def _one_device(**tensors) -> None:
    seen = {n: t.get_device() for n, t in tensors.items() if t is not None}
    if len(set(seen.values())) > 1:
        raise ValueError(f"tensors on different CUDA devices: {seen}")


def _fp4_operand(name: str, q: torch.Tensor, sf: torch.Tensor, kind: str):
    try:
        if q.dtype is torch.uint8 and sf.dtype is torch.uint8 and q.is_cuda and sf.is_cuda and sf.dim() == 1:
            rows, half = q.shape
            if ((q.stride(1) == 1 or not rows or not half) and sf.is_contiguous()
                    and sf.shape[0] >= _fp4_scale_bytes(rows, 2 * half, kind)):
                return rows, 2 * half
    except (AttributeError, ValueError):
        pass
    _need_cuda(name, q, torch.uint8, 2)
    rows, D = q.shape[0], 2 * q.shape[1]
    _need_cuda(f"{name}_sf", sf, torch.uint8, 1)
    if not sf.is_contiguous() or sf.numel() < fp4_scale_bytes(rows, D, kind):
        raise ValueError(f"{name}_sf must be contiguous with at least {fp4_scale_bytes(rows, D, kind)} bytes "
                         f"({kind}, {rows} x {D}), got {sf.numel()}")
    return rows, D


def _fp4_bf16_rows(name: str, t: torch.Tensor):
    """A CUDA bf16 matrix with rows of a multiple of 8 elements -> its shape."""
    try:
        if t.dtype is torch.bfloat16 and t.is_cuda:
            S, D = t.shape
            if not D % 8 and (t.stride(1) == 1 or not S or not D):
                return S, D
    except (AttributeError, ValueError):
        pass
    _need_cuda(name, t, torch.bfloat16, 2)
    if t.shape[1] % 8:
        raise ValueError(f"{name} has rows of {t.shape[1]} elements, not a multiple of 8")
    return t.shape


def quant_rows_fp4(x: torch.Tensor, kind: str = "nvfp4", stream=None):
    """4-bit quantisation of a bf16 [S, D] matrix (D a multiple of 8) -> (q, sf, q_scale).

    mxfp4: blocks of 32 with a power-of-two scale, q_scale None; nvfp4: blocks of 16 with an
    e4m3 scale, and a power of two per row.  A block (mxfp4) or row (nvfp4) that holds a NaN or an
    infinity stands for NaN."""
    code = _fp4_code(kind)
    if isinstance(x, torch.Tensor) and x.dim() == 2:
        out = _fp4_empty(*x.shape, kind, x.device, stream)
        if _fp4_launched(_fp4_fast().quant_rows(x, *out, code, _raw(stream))):
            return out
    S, D = _fp4_bf16_rows("x", x)
    q, sf, q_scale = _fp4_empty(S, D, kind, x.device, stream)
    idx = x.get_device()
    _call(_lib.load().t8g_quant_rows_fp4, idx, x.data_ptr(), _pitch(x, S, D, 8), q.data_ptr(), _pitch(q, S, D // 2, 16),
          sf.data_ptr(), _ptr(q_scale), S, D, code, stream)
    return q, sf, q_scale


def dequant_rows_fp4(q: torch.Tensor, sf: torch.Tensor, q_scale: torch.Tensor | None = None, kind: str = "nvfp4",
                     out_dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """What a 4-bit matrix stands for: (code * block scale) * q_scale as bf16, fp16 or fp32 [S, D]."""
    code = _fp4_code(kind)
    if out_dtype not in OUT_CODE:
        raise TypeError(f"out_dtype {out_dtype} is not one of {tuple(OUT_CODE)}")
    if isinstance(q, torch.Tensor) and q.dim() == 2:
        out = _empty(q.shape[0], 2 * q.shape[1], out_dtype, q.device, stream)
        if _fp4_launched(_fp4_fast().dequant(q, sf, q_scale, out, OUT_CODE[out_dtype], code, _raw(stream))):
            return out
    S, D = _fp4_operand("q", q, sf, kind)
    if D % 8:
        raise ValueError(f"q has rows of {D} elements, not a multiple of 8")
    idx = q.get_device()
    if q_scale is not None and not _vector_ok(q_scale, torch.float32, (S,), idx):
        _need_cuda("q_scale", q_scale, torch.float32, 1)
        if q_scale.numel() != S or not q_scale.is_contiguous():
            raise ValueError("q_scale must be a contiguous float32 tensor with S elements")
    if sf.get_device() != idx or (q_scale is not None and q_scale.get_device() != idx):
        _one_device(q=q, sf=sf, q_scale=q_scale)
    out = _empty(S, D, out_dtype, q.device, stream)
    _call(_lib.load().t8g_dequant_rows_fp4, idx, q.data_ptr(), _pitch(q, S, D // 2, 16), sf.data_ptr(), _ptr(q_scale),
          out.data_ptr(), OUT_CODE[out_dtype], D, S, D, code, stream)
    return out


def rms_mod_quant_fp4(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *, w: torch.Tensor | None = None,
                      mod_index: torch.Tensor | None = None, rows_per_mod: int | None = None,
                      scale_is_multiplier: bool = False, eps: float = 1e-6, kind: str = "nvfp4", stream=None):
    """rms_mod_quant with 4-bit output -> (q, sf, q_scale): quant_rows_fp4 of its bf16 h, bit for
    bit, without storing h.  Values of mod_index are trusted to be rows of shift / scale."""
    code = _fp4_code(kind)
    if w is None and mod_index is None and rows_per_mod and isinstance(x, torch.Tensor) and x.dim() == 2:
        out = _fp4_empty(*x.shape, kind, x.device, stream)
        if _fp4_launched(_fp4_fast().rms_mod_quant(x, shift, scale, rows_per_mod, int(scale_is_multiplier), eps, *out, code,
                                                   _raw(stream))):
            return out
    S, D = _fp4_bf16_rows("x", x)
    idx = x.get_device()
    if not (rows_per_mod and mod_index is None and shift.dim() == 2 and scale.dim() == 2 and shift.shape == scale.shape
            and shift.shape[1] == D and shift.dtype is torch.bfloat16 and scale.dtype is torch.bfloat16
            and shift.stride() == scale.stride() and (not D or shift.stride(1) == 1) and shift.get_device() == idx
            and scale.get_device() == idx):
        shift, scale, rows_per_mod = _mod_args(x, shift, scale, mod_index, rows_per_mod)
        if shift.shape[0] != scale.shape[0]:
            raise ValueError(f"shift has {shift.shape[0]} rows, scale {scale.shape[0]}")
        _one_device(x=x, shift=shift, scale=scale, mod_index=mod_index)
    rpm = int(rows_per_mod)
    if mod_index is None and (rpm < 1 or (S and (S - 1) // rpm >= shift.shape[0])):
        raise ValueError(f"rows_per_mod={rpm} maps rows past the {shift.shape[0]} modulation rows")
    if w is not None:
        _need_cuda("w", w, torch.bfloat16, 1)
        if w.numel() != D:
            raise ValueError("w must have D elements")
        _one_device(x=x, w=w)
    q, sf, q_scale = _fp4_empty(S, D, kind, x.device, stream)
    _call(_lib.load().t8g_rms_mod_quant_fp4, idx, x.data_ptr(), _pitch(x, S, D, 8), _ptr(w), shift.data_ptr(),
          scale.data_ptr(), _pitch(shift, shift.shape[0], D, 8), _ptr(mod_index), rpm, int(scale_is_multiplier), float(eps),
          q.data_ptr(), _pitch(q, S, D // 2, 16), sf.data_ptr(), _ptr(q_scale), S, D, code, stream)
    return q, sf, q_scale


def swiglu_quant_fp4(gate: torch.Tensor, up: torch.Tensor, kind: str = "nvfp4", stream=None):
    """swiglu_quant with 4-bit output -> (q, sf, q_scale): quant_rows_fp4 of act = bf16(silu(gate) *
    up), bit for bit, without storing act."""
    M, F = _fp4_bf16_rows("gate", gate)
    _need_cuda("up", up, torch.bfloat16, 2)
    if gate.shape != up.shape or (M > 1 and gate.stride(0) != up.stride(0)):
        raise ValueError("gate and up must have the same shape and strides")
    _one_device(gate=gate, up=up)
    return _swiglu_fp4(gate.data_ptr(), up.data_ptr(), _pitch(gate, M, F, 8), M, F, kind, gate.device, stream)


def _swiglu_fp4(gate: int, up: int, ld: int, M: int, F: int, kind: str, device, stream):
    code = _fp4_code(kind)
    q, sf, q_scale = _fp4_empty(M, F, kind, device, stream)
    _call(_lib.load().t8g_swiglu_quant_fp4, device.index, gate, up, ld, q.data_ptr(), _pitch(q, M, F // 2, 16), sf.data_ptr(),
          _ptr(q_scale), M, F, code, stream)
    return q, sf, q_scale


def swiglu_quant_fp4_fc1(y: torch.Tensor, kind: str = "nvfp4", stream=None):
    """swiglu_quant_fp4 of a [M, 2F] fc1 output whose first half is the gate (read in place)."""
    code = _fp4_code(kind)
    if isinstance(y, torch.Tensor) and y.dim() == 2:
        out = _fp4_empty(y.shape[0], y.shape[1] // 2, kind, y.device, stream)
        if _fp4_launched(_fp4_fast().swiglu_fc1(y, *out, code, _raw(stream))):
            return out
    M, F2 = _fp4_bf16_rows("y", y)
    if F2 % 16:
        raise ValueError(f"y has rows of {F2} elements: two halves of a multiple of 8 are wanted")
    p = y.data_ptr()
    # the up half starts F2 / 2 elements of two bytes in
    return _swiglu_fp4(p, p + F2 if p else p, _pitch(y, M, F2, 8), M, F2 // 2, kind, y.device, stream)


def _vector_ok(t, dtype, sizes, device) -> bool:
    return t is None or (t.dtype is dtype and t.numel() in sizes and t.is_contiguous() and t.get_device() == device)


def _fp4_product_args(x, w, x_sf, w_sf, x_scale, w_scale, bias, kind, out_dtype):
    """Argument rules of the 4-bit products -> (device, M, N, K, w_scale numel, bias numel)."""
    M, K = _fp4_operand("x", x, x_sf, kind)
    N, Kw = _fp4_operand("w", w, w_sf, kind)
    if Kw != K:
        raise ValueError(f"w has K={Kw}, x has K={K}")
    if K < 8 or K % 8:
        raise ValueError(f"K={K} must be a positive multiple of 8")
    if x_scale is not None:
        _need_cuda("x_scale", x_scale, torch.float32)
        if x_scale.numel() != M or not x_scale.is_contiguous():
            raise ValueError("x_scale must be a contiguous float32 tensor with M elements")
    if w_scale is not None:
        _need_cuda("w_scale", w_scale, torch.float32)
        if w_scale.numel() not in (1, N) or not w_scale.is_contiguous():
            raise ValueError("w_scale must be a contiguous float32 tensor with 1 or N elements")
    nb = 0 if bias is None else bias.numel()
    if nb:
        _need_cuda("bias", bias, out_dtype)
        if nb != N or not bias.is_contiguous():
            raise ValueError("bias must be contiguous with N elements, in the output dtype")
    _one_device(x=x, w=w, x_sf=x_sf, w_sf=w_sf, x_scale=x_scale, w_scale=w_scale, bias=bias if nb else None)
    return x.get_device(), M, N, K, 0 if w_scale is None else w_scale.numel(), nb


def _out_matrix(M: int, N: int, dtype: torch.dtype, device, stream) -> torch.Tensor:
    """[M, N] with rows at a multiple of 16 bytes (contiguous when N allows)."""
    if stream is not None:
        with _stream_memory(stream, device):
            return _out_matrix(M, N, dtype, device, None)
    per = 16 // dtype.itemsize
    if N % per == 0:
        return torch.empty(M, N, dtype=dtype, device=device)
    return torch.empty(M, -(-N // per) * per, dtype=dtype, device=device)[:, :N]


def gemm_fp4(x: torch.Tensor, w: torch.Tensor, x_sf: torch.Tensor, w_sf: torch.Tensor,
             x_scale: torch.Tensor | None = None, w_scale: torch.Tensor | None = None,
             bias: torch.Tensor | None = None, kind: str = "nvfp4", out: torch.Tensor | None = None,
             out_dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """out = cast(((acc * x_scale[:, None]) * w_scale) + bias), acc the product of the 4-bit matrices
    x [M, K] and w [N, K] (codes times block scales) accumulated in fp32.

    x, w: codes, uint8 [., K / 2]; x_scale float32 [M] or None; w_scale [N], [1] or None; bias [N] in
    the output dtype or None / empty; out [M, N] bf16 / fp16 / fp32 (allocated with rows at
    a multiple of 16 bytes when not given)."""
    code = _fp4_code(kind)
    if out is not None:
        out_dtype = out.dtype
    if out_dtype not in OUT_CODE:
        raise TypeError(f"out_dtype {out_dtype} is not one of {tuple(OUT_CODE)}")
    fast = out
    if out is None and isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor) and x.dim() == 2 and w.dim() == 2:
        fast = out = _out_matrix(x.shape[0], w.shape[0], out_dtype, x.device, stream)
    if fast is not None and _fp4_launched(_fp4_fast().gemm(x, w, x_sf, w_sf, x_scale, w_scale, bias, out, out_dtype,
                                                           OUT_CODE[out_dtype], 16 // out_dtype.itemsize, code,
                                                           _raw(stream))):
        return out
    d, M, N, K, nws, nb = _fp4_product_args(x, w, x_sf, w_sf, x_scale, w_scale, bias, kind, out_dtype)
    if out is None:
        out = _out_matrix(M, N, out_dtype, x.device, stream)
    else:
        _need_cuda("out", out, out_dtype, 2)
        if tuple(out.shape) != (M, N):
            raise ValueError(f"out has shape {tuple(out.shape)}, expected {(M, N)}")
        _one_device(x=x, out=out)
    _call(_lib.load().t8g_gemm_fp4, d, x.data_ptr(), x_sf.data_ptr(), None if x_scale is None else x_scale.data_ptr(),
          w.data_ptr(), w_sf.data_ptr(), None if w_scale is None else w_scale.data_ptr(), nws,
          bias.data_ptr() if nb else None, nb, out.data_ptr(), OUT_CODE[out_dtype], M, N, K, _pitch(x, M, K // 2, 16),
          _pitch(w, N, K // 2, 16), _pitch(out, M, N, 16), code, stream)
    return out


def gemm_fp4_gated(x: torch.Tensor, w: torch.Tensor, x_sf: torch.Tensor, w_sf: torch.Tensor,
                   x_scale: torch.Tensor | None, w_scale: torch.Tensor | None, bias: torch.Tensor | None,
                   res: torch.Tensor, gate: torch.Tensor, *, rows_per_gate: int | None = None,
                   gate_index: torch.Tensor | None = None, kind: str = "nvfp4", out: torch.Tensor | None = None,
                   stream=None) -> torch.Tensor:
    """gemm_fp4 as the DiT block's gated residual: out = bf16(res + gate[g] * y), y the product in
    float32 (one rounding, where gemm_gated keeps torch's three), g = gate_index[m] (trusted to be
    rows of gate) or m // rows_per_gate; out may be res itself (in-place update)."""
    code = _fp4_code(kind)
    if rows_per_gate and gate_index is None and isinstance(res, torch.Tensor):
        to = out if out is not None else _empty_like(res, stream)
        if _fp4_launched(_fp4_fast().gated(x, w, x_sf, w_sf, x_scale, w_scale, bias, res, gate, to, rows_per_gate, code,
                                           _raw(stream))):
            return to
    idx, M, N, K, nws, nb = _fp4_product_args(x, w, x_sf, w_sf, x_scale, w_scale, bias, kind, torch.bfloat16)
    if gate.dim() == 1:
        gate = gate.view(1, -1)
    if not (res.dtype is torch.bfloat16 and gate.dtype is torch.bfloat16 and res.dim() == 2 and gate.dim() == 2
            and res.shape[0] == M and res.shape[1] == N and gate.shape[1] == N and gate.shape[0] and res.is_cuda
            and gate.is_cuda and (not M or not N or (res.stride(1) == 1 and gate.stride(1) == 1))):
        _need_cuda("res", res, torch.bfloat16, 2)
        if tuple(res.shape) != (M, N):
            raise ValueError(f"res has shape {tuple(res.shape)}, expected {(M, N)}")
        _need_cuda("gate", gate, torch.bfloat16, 2)
        if gate.shape[1] != N or gate.shape[0] < 1:
            raise ValueError(f"gate must be [n_gate, {N}], got {tuple(gate.shape)}")
    if gate_index is not None:
        _need_cuda("gate_index", gate_index, torch.int32, 1)
        if gate_index.numel() != M or not gate_index.is_contiguous():
            raise ValueError("gate_index must be a contiguous int32 tensor with M elements")
        rpg = 0
    else:
        if rows_per_gate is None:
            if M % gate.shape[0]:
                raise ValueError(f"{M} rows do not split evenly over {gate.shape[0]} gate rows; pass gate_index")
            rows_per_gate = max(1, M // gate.shape[0])
        rpg = int(rows_per_gate)
        if rpg < 1 or (M and (M - 1) // rpg >= gate.shape[0]):
            raise ValueError(f"rows_per_gate={rpg} maps rows past the {gate.shape[0]} gate rows")
    if out is None:
        out = _empty(M, N, torch.bfloat16, x.device, stream)
    elif out is not res:
        _need_cuda("out", out, torch.bfloat16, 2)
        if tuple(out.shape) != (M, N):
            raise ValueError(f"out has shape {tuple(out.shape)}, expected {(M, N)}")
    if (res.get_device() != idx or gate.get_device() != idx or out.get_device() != idx
            or (gate_index is not None and gate_index.get_device() != idx)):
        _one_device(x=x, res=res, gate=gate, gate_index=gate_index, out=out)
    _call(_lib.load().t8g_gemm_fp4_gated, idx, x.data_ptr(), x_sf.data_ptr(), _ptr(x_scale), w.data_ptr(),
          w_sf.data_ptr(), _ptr(w_scale), nws, bias.data_ptr() if nb else None, nb, res.data_ptr(), _pitch(res, M, N, 8),
          gate.data_ptr(), _pitch(gate, gate.shape[0], N, 8), _ptr(gate_index), rpg, out.data_ptr(), M, N, K,
          _pitch(x, M, K // 2, 16), _pitch(w, N, K // 2, 16), _pitch(out, M, N, 8), code, stream)
    return out


def device_status(device=None, stream=None) -> int:
    """Synchronise and read/clear the device status word (0 = no wait ran out)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    st = ctypes.c_int(0)
    with _on(device):
        rc = _lib.load().t8g_device_status(_stream_handle(device, stream), ctypes.byref(st))
    _lib.check(rc)
    return st.value


_status_words = {}


def status_mirror(device=None):
    """The host-visible mirror of the device status word (a ctypes pointer to one int, shared by
    every device), set up for `device` on first use: nonzero once any kernel's bounded wait ran
    out.  Read it with `[0]`, clear it by assigning 0; no synchronisation or CUDA call involved."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    word = _status_words.get(device.index)
    if word is None:
        word = ctypes.POINTER(ctypes.c_int)()
        with _on(device):
            rc = _lib.load().t8g_status_mirror(ctypes.byref(word))
        _lib.check(rc)
        _status_words[device.index] = word
    return word


def wait_selftest(limit_ns: int = 20_000_000, device=None) -> int:
    """Run the bounded-wait self-test kernel; returns 1 if the wait gave up."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    flag = torch.zeros(1, dtype=torch.int32, device=device)
    with _on(device):
        rc = _lib.load().t8g_wait_selftest(limit_ns, _ptr(flag), _stream_handle(device))
    _lib.check(rc)
    return int(flag.item())
