"""CPU: what the sequence operators tell autograd, and the contexts they refuse.  The launch itself is replaced by a note of its name."""
import contextlib

import pytest
import torch


class _Library:
    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def launches(monkeypatch):
    """The names of the launches that a call makes; CPU tensors pass for device tensors."""
    from trajectorydiffusion_amd import _lib, attention
    names = []
    monkeypatch.setattr(_lib, "require_device", lambda t, name: None)
    monkeypatch.setattr(_lib, "lib", lambda: _Library())
    monkeypatch.setattr(attention, "_launch", lambda fn, name, d, index: names.append(name))
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    attention._seen.__dict__.clear()
    yield names
    attention._seen.__dict__.clear()


def test_a_rotation_into_a_tensor_counts_as_a_change_in_place(launches):
    from trajectorydiffusion_amd import attention as A
    x, pos = torch.randn(1, 4, 2, 16), torch.zeros(1, 4, 1)
    for out in (x, torch.empty_like(x), torch.empty(1, 4, 6, 16)[:, :, 2:4]):
        weight = torch.ones_like(out, requires_grad=True)
        y = (weight * out).sum()                          # keeps `out` for the gradient of weight
        A.rotary_axes(x, pos, (8,), out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.no_grad():                                 # a tensor that requires grad may be rotated where nothing is recorded
        leaf = torch.randn(1, 4, 2, 16, requires_grad=True)
        before = leaf._version
        A.rotary_axes(leaf, pos, (8,), out=leaf)
        assert leaf._version == before + 1
    assert launches == ["tdx_rotary_axes"] * 4
    with torch.inference_mode():                          # these count no versions
        t = torch.randn(1, 4, 2, 16)
        A.rotary_axes(t, pos, (8,), out=t)
    empty = torch.empty(0, 4, 2, 16)
    assert A.rotary_axes(empty, torch.zeros(4, 1), (8,), out=empty) is empty


def _both(A, pos):
    return {"rotary_axes": lambda t: A.rotary_axes(t, pos, (8,)), "window_attention": lambda t: A.window_attention(t, t, t, 2, 2)}


@pytest.mark.parametrize("name", ["rotary_axes", "window_attention"])
def test_forward_mode_derivatives_are_refused(launches, name):
    import torch.autograd.forward_ad as forward_ad

    from trajectorydiffusion_amd import attention as A
    x, pos = torch.randn(1, 4, 2, 16), torch.zeros(1, 4, 1)
    f = _both(A, pos)[name]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for t in (dual, forward_ad.make_dual(x.clone().requires_grad_(), torch.ones_like(x))):
            with pytest.raises(A.TdxError, match=f"{name}: forward-mode"):
                f(t)
        others = [lambda: A.window_attention(x, dual, x, 2, 2), lambda: A.window_attention(x, x, dual, 2, 2),
                  lambda: A.rotary_axes(x, forward_ad.make_dual(pos, torch.ones_like(pos)), (8,)), lambda: A.rotary_axes(x, pos, (8,), out=forward_ad.make_dual(x.clone(), x))]
        for g in others:
            with pytest.raises(A.TdxError, match="forward-mode"):
                g()
        assert not launches
        f(x)                                              # no tangent: an ordinary call
    f(x)
    assert len(launches) == 2


@pytest.mark.parametrize("name", ["rotary_axes", "window_attention"])
def test_tracing_is_refused(launches, name):
    """A trace holds torch's operators alone: without the launch its result is memory that nothing wrote."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from trajectorydiffusion_amd import attention as A
    x, pos = torch.randn(1, 4, 2, 16), torch.zeros(1, 4, 1)
    f = _both(A, pos)[name]
    ways = {"proxies": lambda t: make_fx(f)(t), "proxies ahead of dispatch": lambda t: make_fx(f, pre_dispatch=True)(t),
            "proxies over fake tensors": lambda t: make_fx(f, tracing_mode="fake")(t), "jit": lambda t: torch.jit.trace(f, t, check_trace=False),
            "proxies of a copy": lambda t: make_fx(lambda u: f(u.detach().clone()))(t)}
    for way, g in ways.items():
        for t in (x, x.clone().requires_grad_()):
            with pytest.raises(A.TdxError, match=f"{name}: cannot be traced"):
                g(t)
    assert not launches
    leaf = x.clone().requires_grad_()
    y = f(leaf)
    for ahead in (False, True):
        with pytest.raises(A.TdxError, match=f"{name}: cannot be traced"):
            make_fx(lambda g: torch.autograd.grad(y, leaf, g, retain_graph=True), pre_dispatch=ahead)(torch.ones_like(y))
    assert len(launches) == 1


def test_modes_that_only_watch_are_no_trace(launches):
    from torch.utils.checkpoint import checkpoint
    from torch.utils.flop_counter import FlopCounterMode

    from trajectorydiffusion_amd import attention as A
    x, pos = torch.randn(1, 4, 2, 16), torch.zeros(1, 4, 1)
    with FlopCounterMode(display=False), torch.device("cpu"):
        for f in _both(A, pos).values():
            f(x)
    assert launches == ["tdx_rotary_axes", "tdx_window_attention"]
    y = checkpoint(_both(A, pos)["window_attention"], x.clone().requires_grad_(), use_reentrant=False)
    y.sum().backward()
    assert launches[2:] == ["tdx_window_attention"] * 2 + ["tdx_window_attention_bwd"]


def test_a_result_over_the_positions_is_refused(launches):
    from trajectorydiffusion_amd import attention as A
    room = torch.zeros(2 * 4 * 32)
    x = torch.randn(1, 4, 2, 16)
    whole = room.view(2, 4, 2, 16)
    for out, pos in ((whole[:1], room[3:19].view(4, 4)[:, :1]), (whole[:1], room[127:131].view(4, 1)), (whole[1:], room[127:131].view(4, 1)),
                     (whole[1:], room[250:251].expand(4, 1))):
        with pytest.raises(A.TdxError, match="overlaps pos"):
            A.rotary_axes(x, pos, (8,), out=out)
    with pytest.raises(A.TdxError, match="overlaps pos"):                     # views that share memory without sharing a storage
        A.rotary_axes(x, torch.from_dlpack(room[120:124]).view(4, 1), (8,), out=whole[:1])
    with pytest.raises(A.TdxError, match="overlaps x"):
        A.rotary_axes(torch.from_dlpack(room[8:136]).view(1, 4, 2, 16), torch.zeros(4, 1), (8,), out=whole[:1])
    assert not launches
    A.rotary_axes(x, room[128:132].view(4, 1), (8,), out=whole[:1])
    A.rotary_axes(x, room[:4].view(4, 1), (8,), out=whole[1:])
    A.rotary_axes(torch.from_dlpack(room[128:]).view(1, 4, 2, 16), torch.zeros(4, 1), (8,), out=whole[:1])
    assert len(launches) == 3
    rows = torch.zeros(2, 5, 3 + 32 + 3)                                        # positions and heads side by side in each row
    A.rotary_axes(torch.randn(2, 5, 2, 16), rows[:, :, :3], (4, 2, 2), out=rows[:, :, 3:35].unflatten(2, (2, 16)))
    assert len(launches) == 4


def test_shared_bytes_are_told_from_bytes_between_each_other():
    """Against the byte numbers themselves, over drawn forms."""
    from trajectorydiffusion_amd import attention as A
    gen = torch.Generator().manual_seed(7)
    draw = lambda n: int(torch.randint(0, n, (1,), generator=gen))  # noqa: E731
    room = torch.zeros(800, dtype=torch.uint8)
    ids = torch.arange(800)
    found = [0, 0]
    for _ in range(600):
        views, held = [], []
        for es, rank in ((2 if draw(2) else 4, 4), (4, 3)):
            shape, stride, at = tuple(1 + draw(3) for _ in range(rank)), tuple((0, 1, 3, 4, 7, 12, 20)[draw(7)] for _ in range(rank)), draw(20)
            views.append(room.view({2: torch.bfloat16, 4: torch.float32}[es]).as_strided(shape, stride, at))
            held.append(set((ids.as_strided(shape + (es,), tuple(es * s for s in stride) + (1,), es * at)).flatten().tolist()))
        assert A._touch(*views) == bool(held[0] & held[1])
        found[bool(held[0] & held[1])] += 1
    assert min(found) > 50


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38, float("inf"), 1e39])
def test_scales_that_leave_32_bits_are_refused(scale):
    """Exponents are formed as 2^(s scale log2 e)."""
    import ctypes as C

    from test_sequence_cpu import P, _attn_desc

    from trajectorydiffusion_amd import _lib
    lib = _lib.lib()
    for d, f in ((_attn_desc(scale=scale), lib.tdx_window_attention), (_attn_desc(scale=scale, ws=16 * P, ws_bytes=1 << 40), lib.tdx_window_attention_bwd)):
        assert f(C.byref(d), None) == 1 and b"scale" in lib.tdx_last_error()
    assert lib.tdx_window_attention_bwd_ws_bytes(C.byref(_attn_desc(scale=2.3e38))) > 0


def test_a_block_pickled_before_there_were_windows_attends_as_it_did():
    import io

    from trajectorydiffusion_amd import AttnBlock
    old = AttnBlock(64, 32)
    del old.__dict__["window_spec"]                       # as such a pickle holds it
    held = io.BytesIO()
    torch.save(old, held)
    held.seek(0)
    assert torch.load(held, weights_only=False).window_spec is None
    assert AttnBlock(64, 32, window=5).window_spec.window == 5
