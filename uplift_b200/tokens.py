"""Token-sequence operators over the C ABI of include/uplift_tokens.h: the
attention of transformer tokens and the per-head norm with position rotation
that feeds it (sm_100a kernels in uplift_b200/csrc/tok_*.cu).

They stand beside the Local Attender (`ops.local_attender`, a softmax over K
neighbours of a pixel) and the fast mode's layer norm (`glue.layernorm_act_`):

  norm_rotate        RMS norm of every query and key head and the rotation of
                     its channel pairs by position, in one pass
  packed_attention   softmax attention over packed sequences of different
                     lengths (prompts, images, or one new token per sequence
                     on a long history), grouped heads, causal or not

Tensors are [rows, heads, D] on an sm_100 device in float32, bfloat16 or
float16; views into a fused projection output are read in place.  Both are
differentiable (gradients are deterministic) and registered as torch custom
ops, so torch.compile and other tracers record them.  Launches go to the
current stream of the tensors' device; workspaces come from torch's allocator,
so calls on several streams and in captured graphs share nothing.  As with
every differentiable call, capture a backward pass into a CUDA graph only when
no result of an eager call on the same leaves is alive: their gradients would be
summed on the stream of that call, which is not being captured.
"""
from __future__ import annotations

import functools
import math
import struct
from contextlib import nullcontext
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native

_DTYPES = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}

# the argument structs of include/uplift_tokens.h (a token tensor: pointer, row stride, head stride)
_NR_ARGS = struct.Struct("@q" + 6 * "Pqq" + 7 * "P" + "qq" + "iiii" + "f" + "iiiii")
_PA_ARGS = struct.Struct("@q" + 9 * "Pqq" + 6 * "P" + "qqq" + "iiii" + "f" + "iii")
_NO_ROWS = (0, 0, 0)

try:  # without making Stream and device objects: microseconds count in a decoding step
    _raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
except AttributeError:  # pragma: no cover
    _current_device = torch.cuda.current_device

    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream

_HERE = nullcontext()


def _on(index: int):
    """Context in which `index` (the device of CUDA tensors, so CUDA is initialised) is the current device."""
    return _HERE if _current_device() == index else torch.cuda.device(index)


_PLAIN = (torch.Tensor, torch.nn.Parameter)
_modes, _tracing, _transforms = (torch._C._len_torch_dispatch_stack, torch._C._get_tracing_state,
                                 torch._C._functorch.maybe_current_level)


def _recorded(*tensors) -> bool:
    """Whether somebody follows the calls of torch's operators -- a compiler or tracer, a dispatch mode, a function
    transform, a tensor subclass -- and so has to be shown the custom op; else it is left out, since it costs more
    microseconds than some of the kernels take."""
    if torch.compiler.is_compiling() or _modes() or _tracing() is not None or _transforms() is not None:
        return True
    for t in tensors:
        if t.__class__ not in _PLAIN:
            return True
    return False


def _refuse_tangents(what: str, *tensors) -> None:
    """Raises in forward-mode differentiation, which torch would leave out without a word."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative (it is differentiable by backward)")


def _device(what: str, names: str, *tensors) -> int:
    """The common CUDA device index of the tensors (None: left out); raises where they differ or are not on CUDA."""
    index = tensors[0].get_device()
    same = index >= 0
    for t in tensors:
        same = same and (t is None or t.get_device() == index)
    if same:
        return index
    for name, t in zip(names.split(), tensors):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"uplift_b200 {what} runs on CUDA (sm_100) tensors only; {name} is a "
                               f"{t.device} tensor (there is no CPU fallback)")
        if t.get_device() != index:
            raise ValueError(f"{what}: tensors on different devices: {tensors[0].device} vs {t.device} ({name})")
    raise AssertionError


def _check_rows(what: str, names: str, *tensors) -> None:
    first = tensors[0]
    dtype, D = first.dtype, first.shape[-1] if first.dim() else 0
    fine = dtype in _DTYPES
    for t in tensors:
        shape = t.shape
        fine = fine and len(shape) == 3 and t.dtype is dtype and shape[2] == D and D > 0 and shape[1] > 0
    if fine:
        return
    if dtype not in _DTYPES:
        raise ValueError(f"{what}: unsupported dtype {dtype} (float32, bfloat16, float16)")
    names = names.split()
    for name, t in zip(names, tensors):
        if t.dim() != 3:
            raise ValueError(f"{what}: {name} must be [rows, heads, D], got {tuple(t.shape)}")
        if t.dtype is not dtype:
            raise ValueError(f"{what}: {name} is {t.dtype}, {names[0]} is {dtype}")
        if t.shape[2] != D:
            raise ValueError(f"{what}: {name} has head dimension {t.shape[2]}, {names[0]} has {D}")
        if t.shape[1] < 1 or D < 1:
            raise ValueError(f"{what}: {name} has no heads or channels: {tuple(t.shape)}")


def _rows(t: torch.Tensor):
    """(pointer, row stride, head stride) of t and the tensor that owns them: t, or a contiguous copy where the
    kernels cannot read it in place (channel stride 1 and, in 16 bits, 16-byte aligned rows whose stride is a
    multiple of the heads')."""
    r, h, c = t.stride()
    rows, heads, D = t.shape
    ok = c == 1 or D == 1
    p = t.data_ptr()
    if ok and t.dtype is not torch.float32:
        ok = p & 15 == 0 and (rows <= 1 or (r > 0 and r % 8 == 0)) and (
            heads <= 1 or (h > 0 and h % 8 == 0 and (rows <= 1 or r % h == 0)))
    if ok:
        return (p, r, h), t
    t = t.clone(memory_format=torch.contiguous_format)
    return (t.data_ptr(), heads * D, D), t


def _new_rows(t: torch.Tensor):
    """A new contiguous tensor like t, as _rows gives it."""
    n = torch.empty_like(t, memory_format=torch.contiguous_format)
    _, heads, D = t.shape
    return (n.data_ptr(), heads * D, D), n


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


# ------------------------------------------------------------- norm_rotate
def _norm_rotate_args(q, k, q_weight, k_weight, cos, sin, positions):
    """Checks the arguments: (device index, weights' type)."""
    what = "norm_rotate"
    _check_rows(what, "q k", q, k)
    T, _, D = q.shape
    if k.shape[0] != T:
        raise ValueError(f"{what}: q has {T} tokens, k has {k.shape[0]}")
    if D > 256:
        raise ValueError(f"{what}: head dimension {D} is above 256")
    wdt = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if w.shape != (D,) or w.dtype not in _DTYPES:
            raise ValueError(f"{what}: weights must be [{D}] in float32, bfloat16 or float16, got "
                             f"{tuple(w.shape)} {w.dtype}")
        if wdt is not None and w.dtype is not wdt:
            raise ValueError(f"{what}: q_weight is {wdt}, k_weight is {w.dtype}")
        wdt = w.dtype
    table = cos.shape
    if len(table) != 2 or table != sin.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise ValueError(f"{what}: cos and sin must be float32 [P, R / 2] tables of one shape, got "
                         f"{tuple(cos.shape)} {cos.dtype} and {tuple(sin.shape)} {sin.dtype}")
    if 2 * table[1] > D:
        raise ValueError(f"{what}: tables rotate {2 * table[1]} channels, heads have {D}")
    if positions is None:
        if table[1] > 0 and table[0] < T:
            raise ValueError(f"{what}: {table[0]} table rows for {T} tokens without positions")
    elif positions.shape != (T,) or (positions.dtype is not torch.int32 and positions.dtype is not torch.int64):
        raise ValueError(f"{what}: positions must be int32 or int64 [{T}], got {tuple(positions.shape)} "
                         f"{positions.dtype}")
    index = _device(what, "q k q_weight k_weight cos sin positions", q, k, q_weight, k_weight, cos, sin, positions)
    return index, (_native.F32 if wdt is None else _DTYPES[wdt])


def _c(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.contiguous()


def _weight_dtype(q_weight, k_weight) -> torch.dtype:
    return q_weight.dtype if q_weight is not None else k_weight.dtype if k_weight is not None else torch.float32


@functools.lru_cache(maxsize=None)
def _partial_floats(D: int) -> int:
    return _native.load().uplift_tok_norm_rotate_partial_floats(D)


def norm_rotate_raw(q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6, interleaved=False):
    """Launch uplift_tok_norm_rotate (no autograd)."""
    index, wt = _norm_rotate_args(q, k, q_weight, k_weight, cos, sin, positions)
    return _norm_rotate(index, wt, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)


def _norm_rotate(index, wt, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    T, Hq, D = q.shape
    P, half = cos.shape
    lib = _native.load()
    q_weight, k_weight, cos, sin, positions = _c(q_weight), _c(k_weight), _c(cos), _c(sin), _c(positions)
    with _on(index):
        rq, q = _rows(q)
        rk, k = _rows(k)
        ro, q_out = _new_rows(q)
        rp, k_out = _new_rows(k)
        rc = lib.uplift_tok_norm_rotate(
            _NR_ARGS.pack(_NR_ARGS.size, *rq, *rk, *ro, *rp, *_NO_ROWS, *_NO_ROWS, _ptr(q_weight), _ptr(k_weight),
                          cos.data_ptr(), sin.data_ptr(), _ptr(positions), 0, 0, T, P, Hq, k.shape[1], D, 2 * half,
                          eps, interleaved, wt, positions is not None and positions.dtype is torch.int64,
                          _DTYPES[q.dtype], 0), _raw_stream(index))
    if rc:
        _native.check(rc, "uplift_tok_norm_rotate")
    return q_out, k_out


def norm_rotate_backward_raw(gq, gk, q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6,
                             interleaved=False, need_weights=True):
    """Launch uplift_tok_norm_rotate_backward: (dq, dk, dweights [2, D] in the weights' type; empty when not needed)."""
    index, wt = _norm_rotate_args(q, k, q_weight, k_weight, cos, sin, positions)
    return _norm_rotate_backward(index, wt, gq.to(q.dtype), gk.to(q.dtype), q, k, q_weight, k_weight, cos, sin,
                                 positions, eps, interleaved, need_weights)


def _norm_rotate_backward(index, wt, gq, gk, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved,
                          need_weights):
    T, Hq, D = q.shape
    P, half = cos.shape
    lib = _native.load()
    q_weight, k_weight, cos, sin, positions = _c(q_weight), _c(k_weight), _c(cos), _c(sin), _c(positions)
    with _on(index):
        rq, q = _rows(q)
        rk, k = _rows(k)
        rg, gq = _rows(gq)
        rh, gk = _rows(gk)
        rdq, dq = _new_rows(q)
        rdk, dk = _new_rows(k)
        dw = torch.empty((2, D) if need_weights else (0,), dtype=_weight_dtype(q_weight, k_weight), device=q.device)
        partial = torch.empty(_partial_floats(D), dtype=torch.float32, device=q.device) if need_weights else None
        rc = lib.uplift_tok_norm_rotate_backward(
            _NR_ARGS.pack(_NR_ARGS.size, *rq, *rk, *rg, *rh, *rdq, *rdk, _ptr(q_weight), _ptr(k_weight),
                          cos.data_ptr(), sin.data_ptr(), _ptr(positions), dw.data_ptr() if need_weights else 0,
                          _ptr(partial), T, P, Hq, k.shape[1], D, 2 * half, eps, interleaved, wt,
                          positions is not None and positions.dtype is torch.int64, _DTYPES[q.dtype], 0),
            _raw_stream(index))
    if rc:
        _native.check(rc, "uplift_tok_norm_rotate_backward")
    return dq, dk, dw


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.checked = index, wt = _norm_rotate_args(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.set_materialize_grads(False)
        return _norm_rotate(index, wt, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        nq, nk, nqw, nkw = ctx.needs_input_grad[:4]
        if gq is None:  # an output that is not used
            gq = torch.zeros_like(q)
        if gk is None:
            gk = torch.zeros_like(k)
        dq, dk, dw = _norm_rotate_backward(*ctx.checked, gq, gk, q, k, q_weight, k_weight, cos, sin, positions,
                                           ctx.eps, ctx.interleaved, nqw or nkw)
        return (dq if nq else None, dk if nk else None, dw[0] if nqw else None, dw[1] if nkw else None, None, None,
                None, None, None)


@torch.library.custom_op("uplift_b200::norm_rotate", mutates_args=())
def _norm_rotate_op(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                    k_weight: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor,
                    positions: Optional[torch.Tensor], eps: float,
                    interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return norm_rotate_raw(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)


@_norm_rotate_op.register_fake
def _(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("uplift_b200::norm_rotate_backward", mutates_args=())
def _norm_rotate_backward_op(gq: torch.Tensor, gk: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                             q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                             cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor], eps: float,
                             interleaved: bool, need_weights: bool
                             ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return norm_rotate_backward_raw(gq, gk, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved,
                                    need_weights)


@_norm_rotate_backward_op.register_fake
def _(gq, gk, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, need_weights):
    return (q.new_empty(q.shape), k.new_empty(k.shape),
            q.new_empty((2, q.shape[2]) if need_weights else (0,), dtype=_weight_dtype(q_weight, k_weight)))


def _nr_setup_context(ctx, inputs, output):
    q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved = inputs
    ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
    ctx.eps, ctx.interleaved = eps, interleaved


def _nr_backward(ctx, gq, gk):
    q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
    nq, nk, nqw, nkw = ctx.needs_input_grad[:4]
    dq, dk, dw = torch.ops.uplift_b200.norm_rotate_backward(gq, gk, q, k, qw, kw, cos, sin, positions, ctx.eps,
                                                            ctx.interleaved, nqw or nkw)
    # the op's outputs must not alias each other, so the rows of dw are copied
    return (dq if nq else None, dk if nk else None, dw[0].clone() if nqw else None, dw[1].clone() if nkw else None,
            None, None, None, None, None)


torch.library.register_autograd("uplift_b200::norm_rotate", _nr_backward, setup_context=_nr_setup_context)


def norm_rotate(q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6, interleaved=False):
    """RMS norm of query and key heads and position rotation, in one pass.

    q [T, Hq, D] and k [T, Hk, D] -> new contiguous tensors of these shapes:

        y = x / sqrt(mean(x**2) + eps) * weight                   (per token and head)
        (a, b) -> (a cos - b sin, b cos + a sin)                  (per pair of channels)

    q_weight, k_weight: [D], or None for ones.  cos, sin: float32 [P, R / 2]
    tables (R <= D; channels from R on are not rotated); token t uses row
    positions[t] (int32 or int64), or row t without positions.  A negative
    position leaves the token unrotated (class tokens); one beyond the table
    makes its rotated channels NaN.  Pairs are (i, i + R/2), or (2i, 2i + 1)
    when interleaved.  Arithmetic in fp32, one rounding per result.
    Differentiable in q, k and the weights (once); the tables are constants.
    """
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("norm_rotate: cos and sin are constants and must not require gradients")
    if forward_ad._current_level >= 0:
        _refuse_tangents("norm_rotate", q, k, q_weight, k_weight, cos, sin)
    eps, interleaved = float(eps), bool(interleaved)
    if _recorded(q, k):
        return torch.ops.uplift_b200.norm_rotate(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or
                                    (q_weight is not None and q_weight.requires_grad) or
                                    (k_weight is not None and k_weight.requires_grad)):
        return _NormRotate.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    return norm_rotate_raw(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)


# -------------------------------------------------------- packed_attention
_MAX_SEQUENCES = (1 << 31) - 65536 - 1  # the kernels count them in 32 bits


def _starts(what: str, name: str, t: torch.Tensor, entries: int) -> None:
    if (t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != entries or entries < (name != "used_k") or
            entries > _MAX_SEQUENCES + 1):
        raise ValueError(f"{what}: {name} must be an int32 vector of {entries} entries (sequences" +
                         (")" if name == "used_k" else " + 1)") + f", at most {_MAX_SEQUENCES} sequences, "
                         f"got {tuple(t.shape)} {t.dtype}")


def _scale(q: torch.Tensor, scale: Optional[float]) -> float:
    if scale is not None:
        return float(scale)
    D = q.shape[-1] if q.dim() else 0
    return D ** -0.5 if D != 0 else 1.0  # (heads without channels are refused)


def _attention_args(q, k, v, cu_q, cu_k, used_k, scale):
    """Checks the arguments: the device index."""
    what = "packed_attention"
    _check_rows(what, "q k v", q, k, v)
    if k.shape != v.shape:
        raise ValueError(f"{what}: k is {tuple(k.shape)}, v is {tuple(v.shape)}")
    _, Hq, D = q.shape
    if Hq % k.shape[1] != 0:
        raise ValueError(f"{what}: {Hq} query heads are not a multiple of {k.shape[1]} key heads")
    if D > 128 or (D % 8 != 0 and q.dtype is not torch.float32):
        raise ValueError(f"{what}: head dimension {D} (at most 128; a multiple of 8 in 16 bits)")
    n = cu_q.numel()
    _starts(what, "cu_q", cu_q, n)
    _starts(what, "cu_k", cu_k, n)
    if used_k is not None:
        _starts(what, "used_k", used_k, n - 1)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"{what}: scale must be positive and finite, got {scale}")
    return _device(what, "q k v cu_q cu_k used_k", q, k, v, cu_q, cu_k, used_k)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(B, T, S, Hq, Hk, D, dtype) -> int:
    return _native.load().uplift_tok_attention_workspace(B, T, S, Hq, Hk, D, dtype)


def packed_attention_raw(q, k, v, cu_q, cu_k, used_k=None, causal=True, scale=None, need_lse=False, need_lo=False):
    """Launch uplift_tok_attention_forward (no autograd): (out, lse [Hq, T] fp32, out_lo: what the rounding of a
    16-bit out left); lse and out_lo are None when not needed."""
    scale = _scale(q, scale)
    index = _attention_args(q, k, v, cu_q, cu_k, used_k, scale)
    (T, Hq, D), (S, Hk, _) = q.shape, k.shape
    B = cu_q.shape[0] - 1
    dt = _DTYPES[q.dtype]
    lib = _native.load()
    _native.host_status.raise_if_set()
    cu_q, cu_k, used_k = cu_q.contiguous(), cu_k.contiguous(), _c(used_k)
    nbytes = _workspace_bytes(B, T, S, Hq, Hk, D, dt)
    with _on(index):
        rq, q = _rows(q)
        rk, k = _rows(k)
        rv, v = _rows(v)
        ro, out = _new_rows(q)
        rl, lo = _new_rows(q) if need_lo and q.dtype is not torch.float32 else (_NO_ROWS, None)
        lse = torch.empty((Hq, T), dtype=torch.float32, device=q.device) if need_lse else None
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        rc = lib.uplift_tok_attention_forward(
            _PA_ARGS.pack(_PA_ARGS.size, *rq, *rk, *rv, *ro, *rl, *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, _ptr(lse), 0,
                          cu_q.data_ptr(), cu_k.data_ptr(), _ptr(used_k), _ptr(ws), nbytes, T, S, B, Hq, Hk, D,
                          scale, causal, dt, 0), _raw_stream(index))
    if rc:
        _native.check(rc, "uplift_tok_attention_forward")
    return out, lse, lo


def packed_attention_backward_raw(g, q, k, v, out, lse, lo, cu_q, cu_k, used_k=None, causal=True, scale=None):
    """Launch uplift_tok_attention_backward: (dq, dk, dv)."""
    scale = _scale(q, scale)
    index = _attention_args(q, k, v, cu_q, cu_k, used_k, scale)
    return _packed_attention_backward(index, g.to(q.dtype), q, k, v, out, lse, lo, cu_q, cu_k, used_k, causal, scale)


def _packed_attention_backward(index, g, q, k, v, out, lse, lo, cu_q, cu_k, used_k, causal, scale):
    (T, Hq, D), (S, Hk, _) = q.shape, k.shape
    lib = _native.load()
    _native.host_status.raise_if_set()
    cu_q, cu_k, used_k, lse = cu_q.contiguous(), cu_k.contiguous(), _c(used_k), lse.contiguous()
    with _on(index):
        rg, g = _rows(g)
        rq, q = _rows(q)
        rk, k = _rows(k)
        rv, v = _rows(v)
        ro, out = _rows(out)
        rl, lo = _rows(lo) if lo is not None else (_NO_ROWS, None)
        rdq, dq = _new_rows(q)
        rdk, dk = _new_rows(k)
        rdv, dv = _new_rows(v)
        delta = torch.empty(Hq * T + 16, dtype=torch.float32, device=q.device)
        rc = lib.uplift_tok_attention_backward(
            _PA_ARGS.pack(_PA_ARGS.size, *rq, *rk, *rv, *ro, *rl, *rg, *rdq, *rdk, *rdv, lse.data_ptr(), delta.data_ptr(),
                          cu_q.data_ptr(), cu_k.data_ptr(), _ptr(used_k), 0, 0, T, S, cu_q.shape[0] - 1, Hq, Hk, D,
                          scale, causal, _DTYPES[q.dtype], 0), _raw_stream(index))
    if rc:
        _native.check(rc, "uplift_tok_attention_backward")
    return dq, dk, dv


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, used_k, causal, scale):
        out, lse, lo = packed_attention_raw(q, k, v, cu_q, cu_k, used_k, causal, scale, need_lse=True, need_lo=True)
        ctx.save_for_backward(q, k, v, out, lse, lo, cu_q, cu_k, used_k)
        ctx.causal, ctx.scale = causal, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 8
        q, k, v, out, lse, lo, cu_q, cu_k, used_k = ctx.saved_tensors
        grads = _packed_attention_backward(q.get_device(), g, q, k, v, out, lse, lo, cu_q, cu_k, used_k, ctx.causal,
                                           ctx.scale)
        return (*(d if n else None for d, n in zip(grads, ctx.needs_input_grad)), None, None, None, None, None)


@torch.library.custom_op("uplift_b200::packed_attention", mutates_args=())
def _packed_attention_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor,
                         used_k: Optional[torch.Tensor], causal: bool, scale: float, need_lse: bool,
                         need_lo: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    out, lse, lo = packed_attention_raw(q, k, v, cu_q, cu_k, used_k, causal, scale, need_lse, need_lo)
    return (out, lse if lse is not None else out.new_empty(0, dtype=torch.float32),
            lo if lo is not None else out.new_empty(0))


@_packed_attention_op.register_fake
def _(q, k, v, cu_q, cu_k, used_k, causal, scale, need_lse, need_lo):
    return (q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0]) if need_lse else 0, dtype=torch.float32),
            q.new_empty(q.shape if need_lo and q.dtype is not torch.float32 else 0))


@torch.library.custom_op("uplift_b200::packed_attention_backward", mutates_args=())
def _packed_attention_backward_op(g: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                                  out: torch.Tensor, lse: torch.Tensor, lo: torch.Tensor, cu_q: torch.Tensor,
                                  cu_k: torch.Tensor, used_k: Optional[torch.Tensor], causal: bool,
                                  scale: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return packed_attention_backward_raw(g, q, k, v, out, lse, lo if lo.dim() == 3 else None, cu_q, cu_k, used_k,
                                         causal, scale)


@_packed_attention_backward_op.register_fake
def _(g, q, k, v, out, lse, lo, cu_q, cu_k, used_k, causal, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _pa_setup_context(ctx, inputs, output):
    q, k, v, cu_q, cu_k, used_k, causal, scale, _, _ = inputs
    out, lse, lo = output
    ctx.save_for_backward(q, k, v, out, lse, lo, cu_q, cu_k, used_k)
    ctx.causal, ctx.scale = causal, scale


def _pa_backward(ctx, g, _lse, _lo):
    q, k, v, out, lse, lo, cu_q, cu_k, used_k = ctx.saved_tensors
    grads = torch.ops.uplift_b200.packed_attention_backward(g, q, k, v, out, lse, lo, cu_q, cu_k, used_k, ctx.causal,
                                                            ctx.scale)
    return (*(d if n else None for d, n in zip(grads, ctx.needs_input_grad)), *(None,) * 7)


torch.library.register_autograd("uplift_b200::packed_attention", _pa_backward, setup_context=_pa_setup_context)


def packed_attention(q, k, v, cu_q, cu_k=None, used_k=None, causal=True, scale=None, return_lse=False):
    """Softmax attention over packed sequences with grouped heads.

    q [T, Hq, D], k and v [S, Hk, D] (Hq a multiple of Hk; query head h reads
    key head h // (Hq // Hk)) -> out [T, Hq, D], contiguous.

    cu_q, cu_k: int32 vectors of B + 1 ascending row numbers on the device;
    sequence b owns the rows cu[b] .. cu[b + 1] - 1 (cu_k defaults to cu_q).
    used_k: int32 [B], how many rows of each key segment hold keys (a cache
    with room to grow); all of them by default.  A causal query i of n_q sees
    the keys j <= i + n_k - n_q, so the last query sees all n_k.  scale
    defaults to D ** -0.5.  Queries that see no key, and rows of no sequence,
    get zeros (lse -inf) and gradients zero.

    One form of the kernels serves the whole call, by its average tokens per
    sequence: prompts and single tokens are faster in calls of their own.
    Tensors are read in place, but for 16-bit ones whose rows are not 16-byte
    aligned or whose row stride is not a multiple of the head stride (a cache
    laid out [Hk, S, D]): these are copied on every call.

    With return_lse also returns log(sum_j exp(scale q_i . k_j)), fp32
    [Hq, T], a constant for autograd.  Differentiable in q, k, v (once).
    """
    if cu_k is None:
        if q.shape[:1] != k.shape[:1]:
            raise ValueError(f"packed_attention: q is {tuple(q.shape)} and k is {tuple(k.shape)}, not of the same rows: "
                             f"pass cu_k")
        cu_k = cu_q
    if forward_ad._current_level >= 0:
        _refuse_tangents("packed_attention", q, k, v)
    scale, causal = _scale(q, scale), bool(causal)
    train = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if _recorded(q, k, v):
        out, lse, _ = torch.ops.uplift_b200.packed_attention(q, k, v, cu_q, cu_k, used_k, causal, scale,
                                                             train or return_lse, train)
        lse = lse.detach()
    elif train:
        out, lse = _PackedAttention.apply(q, k, v, cu_q, cu_k, used_k, causal, scale)
    else:
        out, lse, _ = packed_attention_raw(q, k, v, cu_q, cu_k, used_k, causal, scale, need_lse=return_lse)
    return (out, lse) if return_lse else out
