"""
Sequence operators around the adapted Linears: the norm, rotary positions and attention of a pre-norm block over tokens of text,
images or video, as hand-written HIP kernels (C-ABI ``include/sam3_seq_amd.h``, ``csrc/seq_rows.hip``, ``csrc/seq_attention.hip``).

  rms_norm, rms_norm_q8   root-mean-square norm with the residual's addition, differentiable; the same with an 8-bit output and
                          its scales (the counterparts of ``vit.layer_norm`` and its fp8 image), which ``fp8.fp8_linear_q`` multiplies
  rotary_axes             rotary positions with several axes (time, height, width, ...) on q and k, differentiable (the general
                          form of the trunk's 2-D tables, ``vit.axial_rope_table``)
  packed_attention        attention over packed sequences of different lengths, causal or not, with grouped heads, differentiable;
                          one token against a long cache is the same call

Activations are bf16 or fp32 on an AMD GPU; there is no CPU fallback.  Calls run on the current stream of the tensors' device, never
wait for the GPU, keep nothing between calls, and can be captured into a graph.
"""
from __future__ import annotations

import contextlib
import ctypes
import operator
from functools import lru_cache
from numbers import Integral
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _ffi
from ._ffi import LoRAKernelError

__all__ = ["rms_norm", "rms_norm_q8", "rotary_axes", "packed_attention", "FP8_E4M3", "FP8_E5M2"]

FP8_E4M3, FP8_E5M2 = _ffi.FP8_E4M3, _ffi.FP8_E5M2
_FP8_TYPES = {FP8_E4M3: torch.float8_e4m3fn, FP8_E5M2: torch.float8_e5m2}
_TYPE_CODES = {torch.bfloat16: _ffi.DT_BF16, torch.float32: _ffi.DT_F32}
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise LoRAKernelError(f"{what} failed (code {rc}): {(_ffi.load().sam3_seq_last_error() or b'').decode()}")


def _activation(name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None) -> None:
    """Checks an activation; its place and type are ``like``'s.  (The messages are made where they are needed only: a small call is
    over in about 15 us.)"""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if like is not None:
        if t.dtype is not like.dtype or t.device != like.device:
            raise ValueError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
        return
    if t.dtype not in _TYPE_CODES:
        raise LoRAKernelError(f"sam3_lora_amd: activations must be bfloat16 or float32, got {t.dtype} for {name}")
    if not t.is_cuda:
        raise LoRAKernelError(f"sam3_lora_amd: the sequence operators run only on an AMD GPU (got a {t.device} tensor for {name}); "
                              "there is no CPU fallback.")


def _recorded(a: torch.Tensor, b: Optional[torch.Tensor], c: Optional[torch.Tensor] = None) -> bool:
    """Whether a call has to be made through its autograd function: a gradient is recorded; or derivatives run forward, which these functions
    do not have and say so; or the call is traced, and would not be seen otherwise."""
    return (torch.is_grad_enabled() and (a.requires_grad or (b is not None and b.requires_grad) or (c is not None and c.requires_grad))) \
        or forward_ad._current_level >= 0 or torch._C._is_tracing()


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """The tensors' device as the current one, where it is not."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)      # torch.cuda.current_stream() without the objects around it


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` with unit stride inside a row, and its address and other strides in multiples of 16 bytes (a copy where it has not); its
    last dimension is a multiple of 8."""
    if t.data_ptr() & 15 == 0:
        if t.is_contiguous():
            return t
        per = 16 // t.element_size()
        if t.stride(-1) == 1 and all(s % per == 0 and s >= 0 for s in t.stride()[:-1]):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor) -> Tuple[int, int]:
    """Strides of [tokens, heads, D] between tokens and between heads; 0 in place of a dimension of one's, which may be anything."""
    n, heads, _ = t.shape
    st, sh, _ = t.stride()
    return st if n > 1 else 0, sh if heads > 1 else 0


def _near(t: torch.Tensor, groups: bool) -> torch.Tensor:
    """:func:`_aligned` for q and the gradient of out: a copy too where rows that share a tile are 2^22 elements apart or more (each head's
    tokens side by side over very many of them; the copy is small beside the attention of so many)."""
    t = _aligned(t)
    st, sh = _strides(t)
    return t if st < 1 << 22 and (sh < 1 << 22 or not groups) else t.contiguous()


def _new(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of ``t``'s shape (the cheapest way to one)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ----------------------------------------------------------------------------------------------------------- RMS norm
def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    t = _aligned(t if t.dim() == 2 else t.reshape(-1, width))
    return t if t.shape[0] <= 1 or t.stride(0) >= width else t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _norm_fwd(x, residual, weight, eps, want_y, want_rstd, q8=None):
    """(y, h, low, rstd, image, scales) of contiguous outputs; q8 = (group, fmt) or None.  low and rstd are for the backward."""
    width = x.shape[-1]
    x2 = _rows(x, width)
    m = x2.shape[0]
    r2, ldr, h, low = None, 0, None, None
    if residual is not None:
        r2 = _rows(residual, width)
        ldr, h = _pitch(r2), _new(x)
        if want_rstd and x.dtype is torch.bfloat16:
            low = x.new_empty((m, width // 8), dtype=torch.int16)
    w = _aligned(weight)
    y = _new(x) if want_y else None
    rstd = x.new_empty(m, dtype=torch.float32) if want_rstd else None
    image = scales = None
    group, fmt = q8 or (0, FP8_E4M3)
    if q8 is not None:
        image = x.new_empty(x.shape, dtype=_FP8_TYPES[fmt])
        scales = x.new_empty(x.shape[:-1] + (width // group if group else 1,), dtype=torch.float32)
    with _on(x.device):
        _check(_ffi.load().sam3_seq_rms_norm_fwd(
            x2.data_ptr(), _pitch(x2), _ptr(r2), ldr, w.data_ptr(), _ptr(y), _ptr(h), _ptr(low), _ptr(rstd), _ptr(image), _ptr(scales), group, fmt,
            m, width, eps, _TYPE_CODES[x.dtype], _stream(x.device)), "sam3_seq_rms_norm_fwd")
    return y, h, low, rstd, image, scales


class _RMSNorm(torch.autograd.Function):
    """``(y, h)``; saves the stream h (x itself without a residual), two bits more of it than bf16 holds, and rstd."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, low, rstd, _, _ = _norm_fwd(x, residual, weight, eps, True, True)
        ctx.save_for_backward(x if residual is None else h, low, weight, rstd)
        ctx.with_residual = residual is not None
        ctx.set_materialize_grads(False)
        return (y, h) if ctx.with_residual else y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gh=None):
        h, low, weight, rstd = ctx.saved_tensors
        need_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        if gy is None:      # only the stream was used
            return gh if ctx.needs_input_grad[0] else None, gh if ctx.needs_input_grad[1] else None, None, None
        width = h.shape[-1]
        h2, w = _rows(h, width), _aligned(weight)
        gy2 = _aligned(gy.contiguous())
        gh2 = None if gh is None or not need_x else _aligned(gh.contiguous())
        gx = _new(h) if need_x else None
        gw = torch.empty_like(weight, memory_format=torch.contiguous_format) if ctx.needs_input_grad[2] else None
        m = h2.shape[0]
        if m == 0:
            return gx if ctx.needs_input_grad[0] else None, gx if ctx.needs_input_grad[1] else None, None if gw is None else gw.zero_(), None
        lib = _ffi.load()
        ws = None
        if gw is not None:
            ws = h.new_empty(lib.sam3_seq_rms_norm_bwd_workspace_bytes(m, width), dtype=torch.uint8)
        with _on(h.device):
            _check(lib.sam3_seq_rms_norm_bwd(
                gy2.data_ptr(), _ptr(gh2), h2.data_ptr(), _pitch(h2), _ptr(low), w.data_ptr(), rstd.data_ptr(), _ptr(gx), _ptr(gw), m, width,
                _TYPE_CODES[h.dtype], _ptr(ws), 0 if ws is None else ws.numel(), _stream(h.device)),
                "sam3_seq_rms_norm_bwd")
        return gx if ctx.needs_input_grad[0] else None, gx if ctx.needs_input_grad[1] else None, gw, None


def _norm_args(x, weight, residual, eps):
    _activation("x", x)
    _activation("weight", weight, x)
    if x.dim() == 0 or weight.dim() != 1 or x.shape[-1] != weight.shape[0]:
        raise ValueError(f"weight must have x's last dimension: got x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    if not 0 < x.shape[-1] <= 16384 or x.shape[-1] % 8:
        raise ValueError(f"the normalised dimension must be a multiple of 8 up to 16384, got {x.shape[-1]}")
    if residual is not None:
        _activation("residual", residual, x)
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    if not 0.0 <= eps < 3e38:
        raise ValueError(f"eps must be finite and not negative, got {eps}")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, with ``h = x + residual``.

    x, residual: [..., C] (rows may be strided), weight: [C], one type (bf16 or fp32); C a multiple of 8, at most 16384.  Returns y, or
    ``(y, h)`` with a residual: h, rounded, is the stream that the next block adds to, and its gradient joins the norm's in one pass.
    The statistics and y come from the unrounded fp32 h; squares that leave fp32 (elements over 1.8e19) give zeros.  Differentiable in x,
    residual and weight.
    """
    _norm_args(x, weight, residual, eps)
    if _recorded(x, weight, residual):
        return _RMSNorm.apply(x, residual, weight, eps)
    y, h, _, _, _, _ = _norm_fwd(x, residual, weight, eps, True, False)
    return y if residual is None else (y, h)


def rms_norm_q8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6, group: int = 0,
                fmt: int = FP8_E4M3):
    """:func:`rms_norm` with an 8-bit output: ``(image, scales)``, or ``(image, scales, h)`` with a residual.  With one scale for a row,
    ``fp8.fp8_linear_q(image, scales, w, b)`` (rows of a 2-D e4m3 image) is the frozen Linear behind it; scales of groups are for a product that
    applies them group by group, which this package has not.

    image: [..., C] ``float8_e4m3fn`` (``fmt=FP8_E5M2``: ``float8_e5m2``) of ``y / scale``; scales: fp32 [..., 1], or [..., C / group] with one
    scale for every ``group`` (32, 64 or 128, a divisor of C) neighbouring columns.  A scale is the largest ``|y|`` of its part, at
    least 2^-24, over the format's largest value, so nothing is clipped; y is rounded once, to 8 bits.  For inference: tensors that
    require a gradient are refused where gradients are recorded.
    """
    _norm_args(x, weight, residual, eps)
    if fmt not in _FP8_TYPES:
        raise ValueError(f"fmt must be FP8_E4M3 or FP8_E5M2, got {fmt}")
    if group != 0 and (group not in (32, 64, 128) or x.shape[-1] % group):
        raise ValueError(f"group must be 0, or 32, 64 or 128 and divide {x.shape[-1]}, got {group}")
    if _recorded(x, weight, residual):
        raise ValueError("rms_norm_q8 has no gradient and no traced form: call it under torch.no_grad(), or rms_norm for training")
    _, h, _, _, image, scales = _norm_fwd(x, residual, weight, eps, False, False, (group, fmt))
    return (image, scales) if residual is None else (image, scales, h)


# --------------------------------------------------------------------------------------------------- rotary positions
@lru_cache(maxsize=256)
def _rotation_table(sections: Tuple[int, ...], theta: float, spectrum: str, d: int):
    """(turns per position step, axis) of each pair as the C arrays that a call reads, and their number."""
    if not (0 < len(sections) <= 256 and all(n >= 0 for n in sections) and 0 < 2 * sum(sections) <= d):
        raise ValueError(f"sections {sections} do not fit a head of {d}")
    if spectrum not in ("shared", "per_axis"):
        raise ValueError(f"spectrum must be 'shared' or 'per_axis', got {spectrum!r}")
    if not 0.0 < theta < float("inf"):
        raise ValueError(f"theta must be positive and finite, got {theta}")
    pairs = sum(sections)
    two_pi = 6.283185307179586476925286766559
    turns, axis = [], []
    for a, n in enumerate(sections):
        for i in range(n):
            exponent = len(axis) / pairs if spectrum == "shared" else i / n
            turns.append(theta ** -exponent / two_pi)
            axis.append(a)
    return (ctypes.c_double * pairs)(*turns), (ctypes.c_ubyte * pairs)(*axis), pairs


def _tokens(t: torch.Tensor) -> torch.Tensor:
    """[..., heads, D] -> [tokens, heads, D], a view where it can be, with strides that the kernel takes."""
    return _aligned(t if t.dim() == 3 else t.reshape(-1, t.shape[-2], t.shape[-1]))


def _rotate(q, k, positions, table, halves, inverse):
    turns, axis, pairs = table
    q3 = _tokens(q)
    t, hq, d = q3.shape
    qs = _strides(q3)
    k3, hk, ks, ko = None, 0, (0, 0), None
    if k is not None:
        k3 = _tokens(k)
        hk, ks, ko = k3.shape[1], _strides(k3), _new(k)
    pos = positions if positions.dim() == 2 else positions.reshape(positions.shape[0], -1)
    qo = _new(q)
    with _on(q.device):
        _check(_ffi.load().sam3_seq_rotary(
            q3.data_ptr(), qs[0], qs[1], _ptr(k3), ks[0], ks[1], qo.data_ptr(), _ptr(ko), pos.data_ptr(), pos.stride(0), pos.stride(1),
            _POSITION_TYPES[pos.dtype], pos.shape[0], turns, axis, pairs, halves, inverse, t, hq, hk, d, _TYPE_CODES[q.dtype],
            _stream(q.device)), "sam3_seq_rotary")
    return qo, ko


class _RotaryAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, table, halves):
        qo, ko = _rotate(q, k, positions, table, halves, False)
        ctx.save_for_backward(positions)
        ctx.table, ctx.halves = table, halves
        ctx.set_materialize_grads(False)
        return qo if k is None else (qo, ko)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk=None):
        positions, = ctx.saved_tensors
        gq = gq if ctx.needs_input_grad[0] else None
        gk = gk if ctx.needs_input_grad[1] else None
        if gq is None and gk is None:
            return None, None, None, None, None
        if gq is None:
            return None, _rotate(gk, None, positions, ctx.table, ctx.halves, True)[0], None, None, None
        return _rotate(gq, gk, positions, ctx.table, ctx.halves, True) + (None, None, None)


def rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, sections: Sequence[int], theta: float = 10000.0,
                pairing: str = "adjacent", spectrum: str = "shared"):
    """Rotary positions with one or several axes on the heads of q and k; returns ``(q', k')``, or q' where k is None.

    q: [..., Hq, D], k: [..., Hk, D], the same leading (token) dimensions and type, any strides; D a multiple of 8, at most 256.
    positions: [axes, ...] of the tokens' positions on each axis: int32, int64, or fp32 (fractions for interpolated grids).
    sections: how many pairs of elements each axis turns; ``2 * sum(sections) <= D``, and the elements behind stay as they are.
    spectrum: ``"shared"``: pair i of n in all turns by ``theta ** (-i / n)`` per step, whatever its axis; ``"per_axis"``: each axis
    starts its own spectrum (``vit.axial_rope_table`` is ``sections=(D/4, D/4)``, per axis).
    pairing: ``"adjacent"``: elements (2i, 2i + 1), the trunk's convention; ``"halves"``: elements (i, i + n).
    Angles are reduced in 64 bits: they are good to fp32 at positions up to 2^30, and off by 2^-54 of a turn times the position behind that.
    Differentiable in q and k.
    """
    _activation("q", q)
    if q.dim() < 2 or not 0 < q.shape[-1] <= 256 or q.shape[-1] % 8:
        raise ValueError(f"q must be [..., heads, D] with D a multiple of 8 up to 256, got {tuple(q.shape)}")
    if k is not None:
        _activation("k", k, q)
        if k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
            raise ValueError(f"k must have q's tokens and head size: got q {tuple(q.shape)}, k {tuple(k.shape)}")
    if q.shape[-2] == 0 or (k is not None and k.shape[-2] == 0):
        raise ValueError("q and k must have heads")
    if type(sections) is not tuple:
        sections = tuple(operator.index(n) for n in sections)
    table = _rotation_table(sections, float(theta), spectrum, q.shape[-1])
    if pairing not in ("adjacent", "halves"):
        raise ValueError(f"pairing must be 'adjacent' or 'halves', got {pairing!r}")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in _POSITION_TYPES:
        raise TypeError("positions must be an int32, int64 or float32 tensor")
    if positions.device != q.device or positions.dim() == 0 or positions.shape[0] != len(sections) or positions.shape[1:] != q.shape[:-2]:
        raise ValueError(f"positions must be {(len(sections),) + tuple(q.shape[:-2])} on {q.device}, got {tuple(positions.shape)} on "
                         f"{positions.device}")
    if positions.requires_grad:
        raise ValueError("positions have no gradient")
    halves = pairing == "halves"
    if _recorded(q, k):
        return _RotaryAxes.apply(q, k, positions, table, halves)
    qo, ko = _rotate(q, k, positions, table, halves, False)
    return qo if k is None else (qo, ko)


# ---------------------------------------------------------------------------------------------------------- attention
def _attn_fwd(q, k, v, cu_q, cu_k, len_k, max_q, max_k, causal, scale, want_lse, want_stats=False):
    tq, hq, d = q.shape
    tk, hk = k.shape[:2]
    q, k, v = _near(q, hq > hk), _aligned(k), _aligned(v)
    out = _new(q)
    lse = q.new_empty((tq, hq), dtype=torch.float32) if want_lse else None
    stats = q.new_empty((tq, hq, 2), dtype=torch.float32) if want_stats else None
    dt = _TYPE_CODES[q.dtype]
    lib = _ffi.load()
    b = cu_q.shape[0] - 1
    nbytes = lib.sam3_seq_attn_fwd_workspace_bytes(tq, b, hq, hk, d, max_q, max_k, dt)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    qs, ks, vs = _strides(q), _strides(k), _strides(v)
    with _on(q.device):
        _check(lib.sam3_seq_attn_fwd(
            q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], cu_q.data_ptr(), cu_k.data_ptr(),
            _ptr(len_k), out.data_ptr(), _ptr(lse), _ptr(stats), tq, tk, b, hq, hk, d, max_q, max_k, causal, scale, dt, _ptr(ws), nbytes,
            _stream(q.device)), "sam3_seq_attn_fwd")
    return out, lse, stats, (q, k, v), qs + ks + vs


class _PackedAttention(torch.autograd.Function):
    """``(out, lse)``, lse None where it is not wanted.  What does not change until the backward is worked out here: that runs in
    another thread, where Python is slower."""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, max_q, max_k, causal, scale, want_lse):
        out, lse, stats, (q, k, v), strides = _attn_fwd(q, k, v, cu_q, cu_k, None, max_q, max_k, causal, scale, want_lse, True)
        ctx.save_for_backward(q, k, v, out, stats, cu_q, cu_k)
        tq, hq, d = q.shape
        tk, hk = k.shape[:2]
        ctx.strides = strides
        ctx.nbytes = _ffi.load().sam3_seq_attn_bwd_workspace_bytes(tq, hq)
        ctx.shape = tq, tk, cu_q.shape[0] - 1, hq, hk, d, max_q, max_k, causal, scale, _TYPE_CODES[q.dtype]
        ctx.set_materialize_grads(False)
        if lse is not None:
            ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, go, _):
        if go is None:
            return (None,) * 10
        q, k, v, out, stats, cu_q, cu_k = ctx.saved_tensors
        go = _near(go, q.shape[1] > k.shape[1])
        need = ctx.needs_input_grad
        gq, gk, gv = (_new(q), _new(k), _new(v)) if need[1] or need[2] else (_new(q), None, None)
        qt, qh, kt, kh, vt, vh = ctx.strides
        gs = _strides(go)
        ws = q.new_empty(ctx.nbytes, dtype=torch.uint8)
        with _on(q.device):
            _check(_ffi.load().sam3_seq_attn_bwd(
                q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, go.data_ptr(), gs[0], gs[1], out.data_ptr(),
                stats.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), gq.data_ptr(), _ptr(gk), _ptr(gv), *ctx.shape, ws.data_ptr(),
                ctx.nbytes, _stream(q.device)), "sam3_seq_attn_bwd")
        return (gq if need[0] else None, gk if need[1] else None, gv if need[2] else None) + (None,) * 7


def _index(name: str, t: torch.Tensor, n: int, device) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 tensor")
    if t.dim() != 1 or t.shape[0] != n or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{n}] on {device}, got {tuple(t.shape)} on {t.device}")


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: Optional[torch.Tensor] = None, *,
                     max_q: Optional[int] = None, max_k: Optional[int] = None, len_k: Optional[torch.Tensor] = None, causal: bool = True,
                     scale: Optional[float] = None, return_lse: bool = False):
    """Softmax attention over sequences of different lengths that lie one behind the other; returns out [Tq, Hq, D].

    q: [Tq, Hq, D], k, v: [Tk, Hk, D], one type (bf16 or fp32), strided as they come (views of a fused projection, or of a cache with
    its heads inside or outside; tokens of k and v less than 2^22 elements apart); Hq a multiple of Hk: head h of q reads head
    ``h // (Hq / Hk)`` of k and v.  D a multiple of 8, at most 128.
    cu_q, cu_k: int32 [B + 1] on the GPU; sequence b is rows ``cu_q[b]:cu_q[b + 1]`` of q and ``cu_k[b]:cu_k[b + 1]`` of k and v
    (cu_k None: the same rows).  They do not decrease; sequences may be empty.  Rows in front of the first and behind the last sequence
    give zeros.
    causal: the last query of a sequence sees all its keys, the one before it all but the last, and so on; False: all see all.  A query
    that sees no key gives zeros.  One new token per request over its cache is ``cu_q = arange(B + 1)``, with ``max_q=1`` and ``max_k``.
    len_k: int32 [B], for caches with room behind each request: only the first ``len_k[b]`` of the rows from ``cu_k[b]`` count (without
    gradients).  max_q, max_k: the longest lengths where the caller knows them: they choose the kernels and size the launch (longer ones still come out
    right; without them one token over long caches takes 1.8 times as long).
    scale: of the scores, 1 / sqrt(D) if None.  return_lse: also the logarithm of each row's sum, fp32 [Tq, Hq], without a gradient.

    Keys and values that a query does not see do not enter its result, whatever they hold; an infinity or NaN that it does see gives what the
    formulas give.  Sums and statistics are fp32; for bf16 the
    probabilities are rounded to bf16 for the product with v, but for calls of few rows, where they keep 16 bits.  Gradients come out the
    same in every run.
    """
    _activation("q", q)
    _activation("k", k, q)
    _activation("v", v, q)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[2] != k.shape[2]:
        raise ValueError(f"q must be [Tq, Hq, D] and k, v [Tk, Hk, D]: got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    (tq, hq, d), (tk, hk) = q.shape, k.shape[:2]
    if hq == 0 or hk == 0 or hq % hk:
        raise ValueError(f"{hq} query heads do not share {hk} key heads")
    if d == 0 or d % 8 or d > 128:
        raise ValueError(f"the head size must be a multiple of 8 up to 128, got {d}")
    if not isinstance(cu_q, torch.Tensor) or cu_q.dim() != 1 or cu_q.numel() < 1:
        raise TypeError("cu_q must be an int32 tensor [B + 1]")
    n = cu_q.numel()
    _index("cu_q", cu_q, n, q.device)
    if cu_k is None:
        if tk != tq:
            raise ValueError(f"without cu_k, k and v must have q's {tq} rows, got {tk}")
        cu_k = cu_q
    else:
        _index("cu_k", cu_k, n, q.device)
    if len_k is not None:
        _index("len_k", len_k, n - 1, q.device)
    for name, m in (("max_q", max_q), ("max_k", max_k)):
        if m is not None and not ((type(m) is int or isinstance(m, Integral)) and 0 <= m < 2 ** 31):
            raise ValueError(f"{name} must be a length, got {m}")
    max_q, max_k = tq if max_q is None else min(int(max_q), tq), tk if max_k is None else min(int(max_k), tk)
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 3e38:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if _recorded(q, k, v):
        if len_k is not None:
            raise ValueError("len_k has no gradient and no traced form: call packed_attention under torch.no_grad()")
        out, lse = _PackedAttention.apply(q, k, v, cu_q, cu_k, max_q, max_k, bool(causal), scale, return_lse)
    else:
        out, lse, _, _, _ = _attn_fwd(q, k, v, cu_q, cu_k, len_k, max_q, max_k, bool(causal), scale, return_lse)
    return (out, lse) if return_lse else out
