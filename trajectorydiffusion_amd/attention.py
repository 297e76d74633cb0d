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
TdxError, like shapes, types and limits the kernels do not take, and like a trace (make_fx, torch.export, torch.jit), which would hold the
empty result and not the launch.
"""
from __future__ import annotations

import ctypes as C
import math
import threading
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import RotaryDesc, TdxError, WindowAttnDesc

_LAYOUTS = {"halves": 0, "pairs": 1}
_CODES = {torch.float32: _lib.TDX_F32, torch.bfloat16: _lib.TDX_BF16}
_MAX = 1 << 28     # lengths and limits the kernels count in

# Filled descriptors by what they were filled from (shapes, strides, types, limits: no addresses), one set per thread: a call of a form that
# was seen before sets its pointers and launches.  The library reads a descriptor during the call only.
_seen = threading.local()
_MOST_SEEN = 256


def _known(kind: str) -> dict:
    got = _seen.__dict__.setdefault(kind, {})
    if len(got) > _MOST_SEEN:
        got.clear()
    return got


def _launch(fn, name: str, d, index: int) -> None:
    """fn(descriptor, stream) on the current stream of device `index` (the library launches on the current device)."""
    old = torch._C._cuda_getDevice()
    if old == index:
        rc = fn(C.byref(d), torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(C.byref(d), torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


# What a call asks before anything else: may a trace be recorded?  Proxies come with a dispatch mode, ahead of dispatch with a stack of their own and, in the
# forward pass, a function mode (whose stack is counted in a third of the time).
_modes, _function_modes, _jit = torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack, torch._C._is_tracing
_modes_ahead = torch._ops._len_torch_dispatch_stack_pre_dispatch
_PROXY = torch._C._TorchDispatchModeKey.PROXY


def _refuse_traces(fn: str) -> None:
    """Raises under a trace, which holds torch's operators and not the launch: its result would be memory that nothing wrote."""
    if _jit() or torch._C._get_dispatch_mode(_PROXY) is not None or torch._ops._get_dispatch_mode_pre_dispatch(_PROXY) is not None:
        raise TdxError(f"{fn}: cannot be traced; call it outside of the traced function")


def _refuse_tangents(fn: str, *tensors: Optional[torch.Tensor]) -> None:
    """Raises where a tensor carries a forward-mode tangent: the launches would drop it."""
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise TdxError(f"{fn}: forward-mode derivatives are not provided")


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
def _rotary_desc(x, pos, sections, bases, layout, inverse, out) -> RotaryDesc:
    d = RotaryDesc()
    d.x_bs, d.x_ts, d.x_hs = _strides(x)
    d.out_bs, d.out_ts, d.out_hs = _strides(out)
    d.pos_bs, d.pos_ts, d.pos_as = pos.stride()
    if pos.shape[0] != x.shape[0]:
        d.pos_bs = 0
    d.B, d.T, d.H, d.D = x.shape
    d.dtype, d.layout, d.inverse, d.naxes = _CODES[x.dtype], layout, int(inverse), len(sections)
    d.sections[:len(sections)] = sections
    d.base[:len(sections)] = bases
    return d


def _rotary_launch(x, pos, sections, bases, layout, inverse, out, given=False) -> None:
    """given: out is the caller's, and may lie over pos"""
    key = (x.shape, x.stride(), x.dtype, pos.shape, pos.stride(), sections, bases, layout, inverse, None if out.is_contiguous() else out.stride())
    known = _known("rotary")
    d = known.get(key)
    if d is None:
        d = known[key] = _rotary_desc(x, pos, sections, bases, layout, inverse, out)
        d.out_bytes, d.pos_bytes = _bytes(out), _bytes(pos)
    at, pos_at = out.data_ptr(), pos.data_ptr()
    if given and at < pos_at + d.pos_bytes and pos_at < at + d.out_bytes and _touch(out, pos):
        raise TdxError("rotary_axes: out overlaps pos")
    d.x, d.out, d.pos = x.data_ptr(), at, pos_at
    _launch(_lib.lib().tdx_rotary_axes, "tdx_rotary_axes", d, x.get_device())


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, sections, bases, layout, inverse):
        ctx.save_for_backward(pos)
        ctx.args = (sections, bases, layout, inverse)
        out = x.new_empty(x.shape)
        _rotary_launch(x, pos, sections, bases, layout, inverse, out)
        return out

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():
            raise TdxError("rotary_axes: second derivatives are not provided")
        if _modes() or _modes_ahead() or _jit():
            _refuse_traces("rotary_axes")
        pos, = ctx.saved_tensors
        sections, bases, layout, inverse = ctx.args
        if dout.stride(3) != 1 and dout.shape[3] != 1:
            dout = dout.contiguous()
        dx = dout.new_empty(dout.shape)
        if dx.numel():
            _rotary_launch(dout, pos, sections, bases, layout, not inverse, dx)   # a rotation's transpose is its inverse
        return dx, None, None, None, None, None


def _rotary_args(x, pos, sections, base, layout) -> Tuple:
    """(sections, bases, layout code) of a call whose arguments go together; raises otherwise."""
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
    if pos.dim() not in (2, 3) or (pos.dim() == 3 and pos.shape[0] not in (1, x.shape[0])) or pos.shape[-2:] != (x.shape[1], len(sections)):
        raise TdxError(f"{fn}: pos {tuple(pos.shape)} for x {tuple(x.shape)} and {len(sections)} axes")
    return sections, bases, _LAYOUTS[layout]


def _bytes(t: torch.Tensor) -> int:
    """From t's first element to behind its last."""
    return (sum((n - 1) * st for st, n in zip(t.stride(), t.shape)) + 1) * t.element_size()


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory between the first and the last element of each has bytes in common."""
    return a.numel() > 0 and b.numel() > 0 and a.data_ptr() < b.data_ptr() + _bytes(b) and b.data_ptr() < a.data_ptr() + _bytes(a)


def _reached(far: int, dims: Sequence[Tuple[int, int, int]]) -> bool:
    """Whether a sum of stride * i with i in [lo, hi], over the (stride, lo, hi) of dims, is `far`."""
    merged = {}
    for st, lo, hi in dims:                    # equal strides are one dimension
        if st == 0:
            continue
        was = merged.get(st, (0, 0))
        merged[st] = (was[0] + lo, was[1] + hi)
    dims = sorted(((st, lo, hi) for st, (lo, hi) in merged.items()), reverse=True)

    def search(far: int, at: int) -> bool:
        if at == len(dims):
            return far == 0
        st, lo, hi = dims[at]
        least, most = (sum(t * n[k] for t, *n in dims[at + 1:]) for k in (0, 1))    # of the dimensions behind
        return any(search(far - i * st, at + 1) for i in range(max(lo, -((most - far) // st)), min(hi, (far - least) // st) + 1))
    return search(far, 0)


def _touch(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the two, which have elements, share a byte."""
    ea, eb = a.element_size(), b.element_size()
    dims = [(st * ea, 0, n - 1) for st, n in zip(a.stride(), a.shape)] + [(st * eb, 1 - n, 0) for st, n in zip(b.stride(), b.shape)]
    return _reached(b.data_ptr() - a.data_ptr(), dims + [(1, 1 - eb, ea - 1)])


def _clash(x: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether `out` holds an element of x's memory at another place than x does (of one form and type).
    Equal strides: some difference of indices leads from one address to the other.  Other strides: the spans meet."""
    if not _meet(x, out):
        return False
    dims = [(st, n) for st, n in zip(x.stride(), x.shape) if n > 1]
    far, part = divmod(out.data_ptr() - x.data_ptr(), x.element_size())
    if part or dims != [(st, n) for st, n in zip(out.stride(), out.shape) if n > 1]:
        return True
    return far != 0 and _reached(far, [(st, 1 - n, n - 1) for st, n in dims])


def rotary_axes(x: torch.Tensor, pos: torch.Tensor, sections: Sequence[int], base: Union[float, Sequence[float]] = 10000.0, layout: str = "halves",
                inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turns the channel pairs of every head of x (B, T, H, D <= 256) by angles of the token's position.

    pos       (B, T, axes), (1, T, axes) or (T, axes) fp32: time, longitude, latitude, ...; angles are formed in 64 bits
    sections  pairs of each axis (their sum P <= D / 2; channels from 2 P on are copied)
    base      pair i of n of an axis turns by pos * base^(-i / n); one number, or one for each axis
    layout    "halves": channels (m, m + P) are pair m; "pairs": channels (2 m, 2 m + 1)
    inverse   turn back
    out       write here (x itself: in place; no other overlap with x, none with pos); not differentiable
    Differentiable in x (backward only).  Returns a contiguous tensor of x's type."""
    fn = "rotary_axes"
    if _modes() or _function_modes() or _jit():
        _refuse_traces(fn)
    if forward_ad._current_level >= 0:
        _refuse_tangents(fn, x, pos, out)
    try:   # a form of call that was checked before?
        sections = tuple(map(int, sections))   # (numbers, not what they come from: a tensor's value may change)
        base = base if base.__class__ is float else tuple(map(float, base)) if isinstance(base, (list, tuple)) else float(base)
        key = (x.shape, x.dtype, x.device, pos.shape, pos.dtype, pos.device, sections, base, layout)
        args = _known("rotary_args").get(key)
    except (AttributeError, TypeError, ValueError):
        key = args = None
    if args is None:
        args = _rotary_args(x, pos, sections, base, layout)
        if key is not None:
            _known("rotary_args")[key] = args
    sections, bases, code = args
    if pos.requires_grad:
        raise TdxError(f"{fn}: positions have no gradient; detach them")
    if pos.dim() == 2:
        pos = pos.unsqueeze(0)
    if x.stride(3) != 1 and x.shape[3] != 1:
        if out is x:
            raise TdxError(f"{fn}: in place needs contiguous channels")
        x = x.contiguous()
    if out is not None:
        _check4(out, "out", fn)
        if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or out.stride(3) != 1:
            raise TdxError(f"{fn}: out must be like x, with contiguous channels")
        if torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
            raise TdxError(f"{fn}: out= is not differentiable")
        if any(n > 1 and st == 0 for n, st in zip(out.shape, out.stride())):
            raise TdxError(f"{fn}: out must not repeat its own memory")
        if out is not x and _clash(x, out):
            raise TdxError(f"{fn}: out overlaps x other than in place")
        if x.numel():
            _rotary_launch(x, pos, sections, bases, code, bool(inverse), out, given=True)
            torch.autograd.graph.increment_version(out)   # the launch writes behind autograd's back
        return out
    if x.requires_grad and torch.is_grad_enabled():
        if x.numel() == 0:
            return x.clone()
        return _Rotary.apply(x, pos, sections, bases, code, bool(inverse))
    out = x.new_empty(x.shape)
    if x.numel():
        _rotary_launch(x, pos, sections, bases, code, bool(inverse), out)
    return out


# ---- attention ------------------------------------------------------------------------------------------------------------------------
def _lies_well(t: torch.Tensor, most_token_bytes: int) -> bool:
    """Whether the kernels can take t as it lies, its address aside."""
    bs, ts, hs = _strides(t)
    es = t.element_size()
    return t.stride(3) == 1 and not ((bs | ts | hs) * es) % 16 and ts * es < most_token_bytes and (65 * ts + t.shape[2] * hs) * es < 1 << 31


def _fits(t: torch.Tensor, most_token_bytes: int) -> torch.Tensor:
    """t itself when the kernels can take it as it lies, else a contiguous copy."""
    return t if t.data_ptr() % 16 == 0 and _lies_well(t, most_token_bytes) else t.clone(memory_format=torch.contiguous_format)


def _desc(q, k, v, out, left, right, sinks, scale) -> WindowAttnDesc:
    d = WindowAttnDesc()
    d.q_bs, d.q_ts, d.q_hs = _strides(q)
    d.k_bs, d.k_ts, d.k_hs = _strides(k)
    d.v_bs, d.v_ts, d.v_hs = _strides(v)
    d.out_bs, d.out_ts, d.out_hs = _strides(out)
    d.B, d.Tq, d.Hq, d.D = q.shape
    d.Tk, d.Hkv = k.shape[1], k.shape[2]
    d.dtype, d.left, d.right, d.sinks, d.scale = _CODES[q.dtype], left, right, sinks, scale
    return d


class _Form:
    """What a call's shapes, strides, types and limits come to: the filled descriptors and the bytes of scratch memory."""
    __slots__ = ("desc", "ws", "lse_shape", "bwd", "bwd_key", "bwd_ws")


def _form(q, k, v, left, right, sinks, scale) -> _Form:
    key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), v.stride(), left, right, sinks, scale)
    known = _known("attention")
    f = known.get(key)
    if f is None:
        f = _Form()
        out = torch.empty(q.shape, dtype=q.dtype, device="meta")
        f.desc = _desc(q, k, v, out, left, right, sinks, scale)
        f.lse_shape = (q.shape[0], q.shape[2], q.shape[1])
        f.bwd = f.bwd_key = None
        d = f.desc
        d.q, d.k, d.v, d.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr()   # (checked for alignment; set again by every call)
        with torch.cuda.device(q.device):
            f.ws = _lib.lib().tdx_window_attention_ws_bytes(C.byref(d))
        known[key] = f
    return f


def _forward(q, k, v, left, right, sinks, scale, q_lens, k_lens, want_lse, out_lo=None):
    out = q.new_empty(q.shape)
    if out.numel() == 0:
        return out, q.new_empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32) if want_lse else None
    f = _form(q, k, v, left, right, sinks, scale)
    lse = q.new_empty(f.lse_shape, dtype=torch.float32) if want_lse else None
    d = f.desc
    d.q, d.k, d.v, d.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    d.lse, d.out_lo = None if lse is None else lse.data_ptr(), None if out_lo is None else out_lo.data_ptr()
    d.q_lens, d.k_lens = None if q_lens is None else q_lens.data_ptr(), None if k_lens is None else k_lens.data_ptr()
    if f.ws:
        ws = q.new_empty(f.ws, dtype=torch.uint8)
        d.ws, d.ws_bytes = ws.data_ptr(), f.ws
    _launch(_lib.lib().tdx_window_attention, "tdx_window_attention", d, q.get_device())
    return out, lse


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, left, right, sinks, scale, q_lens, k_lens):
        # what bf16 leaves of the result, for the backward pass's row sums of dout times out
        out_lo = q.new_empty(q.shape) if q.dtype == torch.bfloat16 else None
        out, lse = _forward(q, k, v, left, right, sinks, scale, q_lens, k_lens, True, out_lo)
        ctx.save_for_backward(q, k, v, out, lse, q_lens, k_lens, out_lo)
        ctx.args = (left, right, sinks, scale)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    def backward(ctx, dout, _dlse):
        if torch.is_grad_enabled():
            raise TdxError("window_attention: second derivatives are not provided")
        if _modes() or _modes_ahead() or _jit():
            _refuse_traces("window_attention")
        none = (None,) * 6
        if dout is None:
            return (None, None, None) + none
        q, k, v, out, lse, q_lens, k_lens, out_lo = ctx.saved_tensors
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        if dq.numel() == 0 or dk.numel() == 0:
            return (dq.zero_(), dk.zero_(), dv.zero_()) + none
        dout = _fits(dout, 1 << 31)
        f = _form(q, k, v, *ctx.args)
        lib = _lib.lib()
        key = dout.stride()
        if f.bwd_key != key:
            d = f.bwd = _desc(q, k, v, out, *ctx.args)
            d.dout_bs, d.dout_ts, d.dout_hs = _strides(dout)
            d.dq_bs, d.dq_ts, d.dq_hs = _strides(dq)
            d.dk_bs, d.dk_ts, d.dk_hs = _strides(dk)
            d.dv_bs, d.dv_ts, d.dv_hs = _strides(dv)
            d.q, d.k, d.v, d.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
            with torch.cuda.device(q.device):
                f.bwd_ws = lib.tdx_window_attention_bwd_ws_bytes(C.byref(d))
            f.bwd_key = key
        d = f.bwd
        ws = q.new_empty(f.bwd_ws, dtype=torch.uint8)
        d.q, d.k, d.v, d.out, d.lse = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr()
        d.q_lens, d.k_lens = None if q_lens is None else q_lens.data_ptr(), None if k_lens is None else k_lens.data_ptr()
        d.dout, d.dq, d.dk, d.dv, d.ws, d.ws_bytes = dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), f.bwd_ws
        d.out_lo = None if out_lo is None else out_lo.data_ptr()
        _launch(lib.tdx_window_attention_bwd, "tdx_window_attention_bwd", d, q.get_device())
        return (dq, dk, dv) + none


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


def _attention_args(q, k, v, left, right, sinks, scale) -> Tuple:
    """(left, right, sinks, scale, whether the tensors can be taken as they lie) of a call whose arguments go together; raises otherwise."""
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
    scale = D ** -0.5 if scale is None else float(scale)
    if not (math.isfinite(scale) and scale > 0):
        raise TdxError(f"{fn}: scale={scale} (finite, > 0)")
    as_it_lies = _lies_well(q, 1 << 31) and _lies_well(k, 1 << 24) and _lies_well(v, 1 << 24)
    return left, right, min(sinks, _MAX), scale, as_it_lies


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
    contiguous and their strides multiples of 16 bytes, else copied.  Differentiable in q, k, v (backward only); results are reproducible."""
    if _modes() or _function_modes() or _jit():
        _refuse_traces("window_attention")
    if forward_ad._current_level >= 0:
        _refuse_tangents("window_attention", q, k, v)
    try:   # a form of call that was checked before?
        if scale is not None and scale.__class__ is not float:
            scale = float(scale)
        key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device, left, right, sinks, scale,
               left.__class__, right.__class__, sinks.__class__)
        args = _known("attention_args").get(key)
    except (AttributeError, TypeError, ValueError, RuntimeError):
        key = args = None
    if args is None:
        args = _attention_args(q, k, v, left, right, sinks, scale)
        if key is not None:
            _known("attention_args")[key] = args
    left, right, sinks, scale, as_it_lies = args
    if q_lens is not None:
        q_lens = _lengths(q_lens, "q_lens", q)
    if k_lens is not None:
        k_lens = _lengths(k_lens, "k_lens", q)
    if not as_it_lies or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        q, k, v = _fits(q, 1 << 31), _fits(k, 1 << 24), _fits(v, 1 << 24)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _WindowAttention.apply(q, k, v, left, right, sinks, scale, q_lens, k_lens)
    else:
        out, lse = _forward(q, k, v, left, right, sinks, scale, q_lens, k_lens, return_lse)
    return (out, lse) if return_lse else out
