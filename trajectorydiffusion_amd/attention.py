"""Sequence operators for long tracks on the GPU (csrc/rotary.hip, csrc/window_attention.hip): rotary positions with several axes and
attention with a window and a few first tokens that stay visible.  Both are functions of tensors (batch, token, head, channel), fp32 or
bf16, differentiable through torch.autograd, and may be recorded into a HIP graph.  The reference has neither: its attention takes the
13 tokens of TrajUNet's middle block.

Training or prompts (rotate q and k, then attend):

    q, k, v = qkv.view(B, L, 3, heads, C // heads).unbind(2)
    pos = torch.stack([minutes, lon_cell, lat_cell], dim=2)                 # (B, L, 3) fp32
    q, k = (rotary_axes(x, pos, sections=(32, 16, 16)) for x in (q, k))
    out = window_attention(q, k, v, left=512, right=512, sinks=7)           # the 7 tokens in front stay visible to every point

Single tokens over a cache (B, capacity, Hkv, D) that holds k_lens[b] keys, the new one included:

    out = window_attention(q, k_cache, v_cache, left=4095, right=0, sinks=4, k_lens=k_lens)    # q (B, 1, Hq, D)

Everything runs on torch's current stream of the tensors' device; results are allocated by torch.  No CPU fallback: CPU tensors raise
TdxError, like shapes, types and limits the kernels do not take.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import RotaryDesc, TdxError, WindowAttnDesc

_LAYOUTS = {"halves": 0, "pairs": 1}
_CODES = {torch.float32: _lib.TDX_F32, torch.bfloat16: _lib.TDX_BF16}
_MAX = 1 << 28     # lengths and limits the kernels count in


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


class _On:
    """The tensors' device as the current one (the library launches on the current device), switched only when it is another."""
    __slots__ = ("dev", "old")

    def __init__(self, t: torch.Tensor):
        self.dev = t.device.index

    def __enter__(self):
        self.old = torch.cuda.current_device()
        if self.old != self.dev:
            torch.cuda.set_device(self.dev)

    def __exit__(self, *exc):
        if self.old != self.dev:
            torch.cuda.set_device(self.old)
        return False


def _strides(t: torch.Tensor) -> Tuple[int, int, int]:
    """Element strides of batch, token and head; a dimension of one element has none that matters."""
    return tuple(st if n > 1 else 0 for n, st in zip(t.shape[:3], t.stride()[:3]))


def _check4(t: torch.Tensor, name: str, fn: str) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise TdxError(f"{fn}: {name} must be a (batch, token, head, channel) tensor, got {tuple(t.shape) if isinstance(t, torch.Tensor) else type(t)}")
    if t.dtype not in _CODES:
        raise TdxError(f"{fn}: {name} is {t.dtype}; use torch.float32 or torch.bfloat16")
    _lib.require_device(t, f"{fn}: {name}")


# ---- rotary positions ---------------------------------------------------------------------------------------------------------------
def _rotary_launch(x, pos, sections, bases, layout, inverse, out) -> None:
    d = RotaryDesc()
    d.x, d.out, d.pos = x.data_ptr(), out.data_ptr(), pos.data_ptr()
    d.x_bs, d.x_ts, d.x_hs = _strides(x)
    d.out_bs, d.out_ts, d.out_hs = _strides(out)
    d.pos_bs, d.pos_ts, d.pos_as = pos.stride()
    d.B, d.T, d.H, d.D = x.shape
    d.dtype, d.layout, d.inverse, d.naxes = _CODES[x.dtype], layout, int(inverse), len(sections)
    d.sections[:len(sections)] = sections
    d.base[:len(sections)] = bases
    with _On(x):
        _lib.check(_lib.lib().tdx_rotary_axes(C.byref(d), _stream(x)), "tdx_rotary_axes")


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, sections, bases, layout, inverse):
        ctx.save_for_backward(pos)
        ctx.args = (sections, bases, layout, inverse)
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        _rotary_launch(x, pos, sections, bases, layout, inverse, out)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        pos, = ctx.saved_tensors
        sections, bases, layout, inverse = ctx.args
        if dout.stride(3) != 1 and dout.shape[3] != 1:
            dout = dout.contiguous()
        dx = torch.empty(dout.shape, dtype=dout.dtype, device=dout.device)
        _rotary_launch(dout, pos, sections, bases, layout, not inverse, dx)   # a rotation's transpose is its inverse
        return dx, None, None, None, None, None


def rotary_axes(x: torch.Tensor, pos: torch.Tensor, sections: Sequence[int], base: Union[float, Sequence[float]] = 10000.0, layout: str = "halves",
                inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turns the channel pairs of every head of x (B, T, H, D <= 256) by angles of the token's position.

    pos       (B, T, axes), (1, T, axes) or (T, axes) fp32: time, longitude, latitude, ...; angles are formed in 64 bits
    sections  pairs of each axis (their sum P <= D / 2; channels from 2 P on are copied)
    base      pair i of n of an axis turns by pos * base^(-i / n); one number, or one for each axis
    layout    "halves": channels (m, m + P) are pair m; "pairs": channels (2 m, 2 m + 1)
    inverse   turn back
    out       write here (x itself: in place); not differentiable
    Differentiable in x.  Returns a contiguous tensor of x's type."""
    fn = "rotary_axes"
    _check4(x, "x", fn)
    if layout not in _LAYOUTS:
        raise TdxError(f"{fn}: layout {layout!r}; use 'halves' or 'pairs'")
    sections = tuple(int(n) for n in sections)
    if not 1 <= len(sections) <= 8 or min(sections) < 0 or not 1 <= sum(sections) <= x.shape[3] // 2:
        raise TdxError(f"{fn}: sections {sections} do not fit heads of {x.shape[3]} channels (1 to 8 axes, at most D / 2 pairs)")
    bases = tuple(float(b) for b in base) if isinstance(base, (list, tuple)) else (float(base),) * len(sections)
    if len(bases) != len(sections) or not all(math.isfinite(b) and b > 0 for b in bases):
        raise TdxError(f"{fn}: base {base!r} for {len(sections)} axes (finite, > 0)")
    if not isinstance(pos, torch.Tensor) or pos.dtype != torch.float32 or pos.device != x.device:
        raise TdxError(f"{fn}: pos must be an fp32 tensor on {x.device}")
    if pos.requires_grad:
        raise TdxError(f"{fn}: positions have no gradient; detach them")
    if pos.dim() == 2:
        pos = pos.unsqueeze(0)
    if pos.dim() != 3 or pos.shape[0] not in (1, x.shape[0]) or pos.shape[1:] != (x.shape[1], len(sections)):
        raise TdxError(f"{fn}: pos {tuple(pos.shape)} for x {tuple(x.shape)} and {len(sections)} axes")
    if pos.shape[0] != x.shape[0]:
        pos = pos.expand(x.shape[0], -1, -1)
    if x.stride(3) != 1 and x.shape[3] != 1:
        if out is x:
            raise TdxError(f"{fn}: in place needs contiguous channels")
        x = x.contiguous()
    code = _LAYOUTS[layout]
    if out is not None:
        _check4(out, "out", fn)
        if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or out.stride(3) != 1:
            raise TdxError(f"{fn}: out must be like x, with contiguous channels")
        if torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
            raise TdxError(f"{fn}: out= is not differentiable")
        if 0 in out.stride() and any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise TdxError(f"{fn}: out must not repeat its own memory")
        if x.numel():
            _rotary_launch(x.detach(), pos, sections, bases, code, inverse, out)
        return out
    if x.requires_grad and torch.is_grad_enabled():
        return _Rotary.apply(x, pos, sections, bases, code, bool(inverse))
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        _rotary_launch(x, pos, sections, bases, code, inverse, out)
    return out


# ---- attention ------------------------------------------------------------------------------------------------------------------------
def _fits(t: torch.Tensor, most_token_bytes: int) -> torch.Tensor:
    """t itself when the kernels can take it as it lies, else a contiguous copy."""
    bs, ts, hs = _strides(t)
    es = t.element_size()
    if (t.stride(3) != 1 or t.data_ptr() % 16 or (bs * es) % 16 or (ts * es) % 16 or (hs * es) % 16 or ts * es >= most_token_bytes
            or (33 * ts + t.shape[2] * hs) * es >= 1 << 31):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _desc(q, k, v, out, lse, left, right, sinks, scale, q_lens, k_lens) -> WindowAttnDesc:
    d = WindowAttnDesc()
    d.q, d.k, d.v, d.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    d.lse = None if lse is None else lse.data_ptr()
    d.q_bs, d.q_ts, d.q_hs = _strides(q)
    d.k_bs, d.k_ts, d.k_hs = _strides(k)
    d.v_bs, d.v_ts, d.v_hs = _strides(v)
    d.out_bs, d.out_ts, d.out_hs = _strides(out)
    d.B, d.Tq, d.Hq, d.D = q.shape
    d.Tk, d.Hkv = k.shape[1], k.shape[2]
    d.dtype, d.left, d.right, d.sinks, d.scale = _CODES[q.dtype], left, right, sinks, scale
    d.q_lens, d.k_lens = _lib.ptr(q_lens), _lib.ptr(k_lens)
    return d


def _forward(q, k, v, left, right, sinks, scale, q_lens, k_lens, want_lse):
    B, Tq, Hq, D = q.shape
    out = torch.empty((B, Tq, Hq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, Hq, Tq), dtype=torch.float32, device=q.device) if want_lse else None
    if out.numel() == 0:
        return out, lse
    d = _desc(q, k, v, out, lse, left, right, sinks, scale, q_lens, k_lens)
    lib = _lib.lib()
    with _On(q):
        n = lib.tdx_window_attention_ws_bytes(C.byref(d))
        if n:
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)
            d.ws, d.ws_bytes = ws.data_ptr(), n
        _lib.check(lib.tdx_window_attention(C.byref(d), _stream(q)), "tdx_window_attention")
    return out, lse


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, left, right, sinks, scale, q_lens, k_lens):
        out, lse = _forward(q, k, v, left, right, sinks, scale, q_lens, k_lens, True)
        ctx.save_for_backward(q, k, v, out, lse, q_lens, k_lens)
        ctx.args = (left, right, sinks, scale)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _dlse):
        q, k, v, out, lse, q_lens, k_lens = ctx.saved_tensors
        left, right, sinks, scale = ctx.args
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        if dq.numel() == 0 or k.shape[1] == 0:
            return dq.zero_(), dk.zero_(), dv.zero_(), None, None, None, None, None, None
        dout = _fits(dout, 1 << 31)
        d = _desc(q, k, v, out, lse, left, right, sinks, scale, q_lens, k_lens)
        d.dout, d.dq, d.dk, d.dv = dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        d.dout_bs, d.dout_ts, d.dout_hs = _strides(dout)
        d.dq_bs, d.dq_ts, d.dq_hs = _strides(dq)
        d.dk_bs, d.dk_ts, d.dk_hs = _strides(dk)
        d.dv_bs, d.dv_ts, d.dv_hs = _strides(dv)
        lib = _lib.lib()
        with _On(q):
            n = lib.tdx_window_attention_bwd_ws_bytes(C.byref(d))
            ws = torch.empty(max(n, 1), dtype=torch.uint8, device=q.device)
            d.ws, d.ws_bytes = ws.data_ptr(), n
            _lib.check(lib.tdx_window_attention_bwd(C.byref(d), _stream(q)), "tdx_window_attention_bwd")
        return dq, dk, dv, None, None, None, None, None, None


def _limit(n: Optional[int], name: str) -> int:
    if n is None:
        return -1
    if isinstance(n, bool) or not isinstance(n, int) or n < 0:
        raise TdxError(f"window_attention: {name}={n!r} (None: no limit, or a number of tokens >= 0)")
    return min(n, _MAX)


def _lengths(t: Optional[torch.Tensor], name: str, q: torch.Tensor) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64) or t.shape != (q.shape[0],) or t.device != q.device:
        raise TdxError(f"window_attention: {name} must be an int32 or int64 tensor of {q.shape[0]} lengths on {q.device}")
    if t.dtype == torch.int64:
        t = t.clamp(-1, _MAX).to(torch.int32)
    return t.contiguous()


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, left: Optional[int] = None, right: Optional[int] = None, sinks: int = 0,
                     q_lens: Optional[torch.Tensor] = None, k_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """softmax(scale q k^T) v over the keys each query sees: q (B, Tq, Hq, D), k and v (B, Tk, Hkv, D) -> (B, Tq, Hq, D).

    Query i of a sequence with q_len queries and k_len keys stands at position p = i + k_len - q_len (the last query at the last key) and
    sees key j iff  j < k_len,  j <= p + right  and  (j >= p - left or j < sinks).  right = 0 is causal; None: no limit on that side.
    q_lens, k_lens  device lengths (B) of padded batches and partly filled caches, clamped to [0, Tq] / [0, Tk]; None: all
    scale           D ** -0.5 by default
    return_lse      also the logarithm of the sum of exponentials (B, Hq, Tq) fp32 (not differentiable)
    Hq a multiple of Hkv (query head h reads key head h // (Hq / Hkv)); D a multiple of 8, at most 128.  Queries that see nothing, and
    those behind q_len, get zeros (lse -inf) and pass no gradient; gradients of keys behind k_len are zero.  Whatever stands at keys a
    query does not see, NaN and infinities too, does not reach it.  Strided tensors are taken as they lie when their channels are
    contiguous and their strides multiples of 16 bytes, else copied.  Differentiable in q, k, v; results are reproducible."""
    fn = "window_attention"
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _check4(t, n, fn)
    B, Tq, Hq, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D or k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise TdxError(f"{fn}: q {tuple(q.shape)} {q.dtype}, k {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype} do not go together")
    if Hq < 1 or k.shape[2] < 1 or Hq % k.shape[2]:
        raise TdxError(f"{fn}: {Hq} query heads over {k.shape[2]} key heads")
    if D % 8 or not 8 <= D <= 128:
        raise TdxError(f"{fn}: heads of {D} channels (a multiple of 8, at most 128)")
    left, right = _limit(left, "left"), _limit(right, "right")
    if isinstance(sinks, bool) or not isinstance(sinks, int) or sinks < 0:
        raise TdxError(f"{fn}: sinks={sinks!r} (a number of tokens >= 0)")
    sinks = min(sinks, _MAX)
    scale = D ** -0.5 if scale is None else float(scale)
    if not (math.isfinite(scale) and scale > 0):
        raise TdxError(f"{fn}: scale={scale} (finite, > 0)")
    q_lens, k_lens = _lengths(q_lens, "q_lens", q), _lengths(k_lens, "k_lens", q)
    q, k, v = _fits(q, 1 << 31), _fits(k, 1 << 24), _fits(v, 1 << 24)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _WindowAttention.apply(q, k, v, left, right, sinks, scale, q_lens, k_lens)
    else:
        out, lse = _forward(q, k, v, left, right, sinks, scale, q_lens, k_lens, return_lse)
    return (out, lse) if return_lse else out
