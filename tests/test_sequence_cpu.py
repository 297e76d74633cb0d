"""CPU: refusals and plans of the sequence operators (rotary positions, windowed attention), through Python and through the C ABI.  Every C call
here is refused before a launch, or only asks for a size."""
import ctypes as C

import pytest
import torch

import _sequence_ref as R


def _mod():
    from trajectorydiffusion_amd import _lib, attention
    return _lib, attention


def test_python_functions_refuse_what_they_do_not_take():
    _lib, A = _mod()
    t = torch.zeros(2, 4, 2, 64)
    pos = torch.zeros(2, 4, 1)
    for f in (lambda: A.window_attention(t, t, t), lambda: A.rotary_axes(t, pos, (32,)), lambda: A.window_attention(t[0], t, t),
              lambda: A.window_attention("q", t, t), lambda: A.window_attention(t.double(), t, t), lambda: A.rotary_axes(None, pos, (32,)),
              lambda: A.rotary_axes(t.half(), pos, (32,))):
        with pytest.raises(_lib.TdxError):
            f()


class _Cuda(torch.Tensor):
    """A CPU tensor that says it lies on a GPU, so that the checks behind the device check are reached (they touch no data)."""
    is_cuda = True


def _fake(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Cuda)


@pytest.mark.parametrize("what,kwargs", [
    ("not go together", dict(k=(2, 4, 2, 64), v=(2, 5, 2, 64))),
    ("not go together", dict(k=(3, 4, 2, 64), v=(3, 4, 2, 64))),
    ("not go together", dict(k=(2, 4, 2, 32), v=(2, 4, 2, 32))),
    ("query heads", dict(k=(2, 4, 4, 64), v=(2, 4, 4, 64))),
    ("query heads", dict(q=(2, 4, 3, 64))),
    ("channels", dict(q=(2, 4, 2, 136), k=(2, 4, 2, 136), v=(2, 4, 2, 136))),
    ("channels", dict(q=(2, 4, 2, 20), k=(2, 4, 2, 20), v=(2, 4, 2, 20))),
    ("left", dict(left=-1)), ("left", dict(left=2.0)), ("left", dict(left=True)), ("right", dict(right=-5)), ("sinks", dict(sinks=-1)),
    ("sinks", dict(sinks=None)), ("sinks", dict(sinks=True)), ("scale", dict(scale=0.0)), ("scale", dict(scale=float("inf"))), ("scale", dict(scale=-1.0)),
])
def test_attention_arguments(what, kwargs):
    _lib, A = _mod()
    shapes = {n: kwargs.pop(n, (2, 4, 2, 64)) for n in "qkv"}
    q, k, v = (_fake(*shapes[n]) for n in "qkv")
    args = dict(left=None, right=None, sinks=0, scale=None)
    args.update(kwargs)
    with pytest.raises(_lib.TdxError, match=what):
        A._attention_args(q, k, v, args["left"], args["right"], args["sinks"], args["scale"])


def test_attention_types_and_lengths():
    _lib, A = _mod()
    q = _fake(2, 4, 2, 64)
    with pytest.raises(_lib.TdxError, match="not go together"):
        A._attention_args(q, _fake(2, 4, 2, 64, dtype=torch.bfloat16), q, None, None, 0, None)
    assert A._attention_args(q, q, q, None, 3, 5, None) == (-1, 3, 5, 0.125, True)
    for bad in (torch.zeros(3, dtype=torch.int32), torch.zeros(2), torch.zeros(2, 1, dtype=torch.int32), [4, 4], 4):
        with pytest.raises(_lib.TdxError, match="k_lens"):
            A._lengths(bad, "k_lens", q)
    assert A._lengths(torch.tensor([1 << 40, -3]), "k_lens", q).tolist() == [1 << 28, -1]


@pytest.mark.parametrize("what,kwargs", [
    ("layout", dict(layout="rows")), ("sections", dict(sections=())), ("sections", dict(sections=(33,))), ("sections", dict(sections=(0, 0))),
    ("sections", dict(sections=(-1, 4))), ("sections", dict(sections=(1,) * 9)), ("base", dict(base=0.0)), ("base", dict(base=(1.0, 2.0))),
    ("base", dict(base=float("nan"))), ("pos", dict(pos=torch.zeros(2, 4, 1, dtype=torch.float64))), ("pos", dict(pos=torch.zeros(2, 4, 2))),
    ("pos", dict(pos=torch.zeros(3, 4, 1))), ("pos", dict(pos=torch.zeros(4))), ("pos", dict(pos=torch.zeros(2, 5, 1))), ("pos", dict(pos=None)),
])
def test_rotary_arguments(what, kwargs):
    _lib, A = _mod()
    args = dict(pos=torch.zeros(2, 4, 1), sections=(32,), base=10000.0, layout="halves")
    args.update(kwargs)
    with pytest.raises(_lib.TdxError, match=what):
        A._rotary_args(_fake(2, 4, 2, 64), args["pos"], args["sections"], args["base"], args["layout"])


P = 1 << 20     # an address that is aligned and never touched


def _rotary_desc(**kw):
    _lib, _ = _mod()
    d = _lib.RotaryDesc()
    d.x, d.out, d.pos = P, 2 * P, 3 * P
    d.x_bs = d.out_bs = 4 * 128
    d.x_ts = d.out_ts = 128
    d.x_hs = d.out_hs = 64
    d.pos_bs, d.pos_ts, d.pos_as = 4, 1, 1
    d.B, d.T, d.H, d.D, d.naxes = 2, 4, 2, 64, 1
    d.sections[0], d.base[0] = 32, 10000.0
    for n, v in kw.items():
        if n in ("sections", "base"):
            for i, x in enumerate(v):
                getattr(d, n)[i] = x
        else:
            setattr(d, n, v)
    return d


@pytest.mark.parametrize("kw", [dict(x=None), dict(out=None), dict(pos=None), dict(dtype=2), dict(layout=2), dict(naxes=0), dict(naxes=9), dict(sections=[33]),
                                dict(sections=[0]), dict(sections=[-1]), dict(base=[0.0]), dict(base=[float("nan")]), dict(D=257), dict(D=0), dict(B=-1),
                                dict(H=65537), dict(out=P, out_ts=256)])
def test_c_rotary_refuses(kw):
    _lib, _ = _mod()
    assert _lib.lib().tdx_rotary_axes(C.byref(_rotary_desc(**kw)), None) == 1
    assert b"tdx_rotary_axes" in _lib.lib().tdx_last_error()
    assert _lib.lib().tdx_rotary_axes(None, None) == 1


def test_c_rotary_of_nothing_is_no_launch():
    _lib, _ = _mod()
    for kw in (dict(B=0), dict(T=0), dict(H=0)):
        assert _lib.lib().tdx_rotary_axes(C.byref(_rotary_desc(x=None, out=None, pos=None, **kw)), None) == 0


def _attn_desc(B=2, Tq=4, Tk=4, Hq=4, Hkv=2, D=64, **kw):
    _lib, _ = _mod()
    d = _lib.WindowAttnDesc()
    d.q, d.k, d.v, d.out, d.lse, d.dout, d.dq, d.dk, d.dv = (P * (n + 1) for n in range(9))
    d.B, d.Tq, d.Tk, d.Hq, d.Hkv, d.D = B, Tq, Tk, Hq, Hkv, D
    for n, T, H in (("q", Tq, Hq), ("k", Tk, Hkv), ("v", Tk, Hkv), ("out", Tq, Hq), ("dout", Tq, Hq), ("dq", Tq, Hq), ("dk", Tk, Hkv), ("dv", Tk, Hkv)):
        for suffix, v in (("_bs", T * H * D), ("_ts", H * D), ("_hs", D)):
            setattr(d, n + suffix, v)
    d.left, d.right, d.sinks, d.scale = 2, 0, 1, 0.125
    for n, v in kw.items():
        setattr(d, n, v)
    return d


BAD = [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=P + 4), dict(k=P + 8), dict(out=P + 2), dict(dtype=7), dict(B=-1), dict(Hq=3), dict(Hkv=0), dict(D=4),
       dict(D=12), dict(D=136), dict(scale=0.0), dict(scale=float("nan")), dict(scale=-1.0), dict(sinks=-1), dict(q_ts=130), dict(k_hs=66), dict(v_bs=2),
       dict(out_ts=1), dict(q_ts=-128), dict(k_ts=1 << 22), dict(v_ts=1 << 22), dict(q_ts=1 << 25), dict(q_hs=1 << 29), dict(Tq=1 << 28), dict(Tk=1 << 28), dict(q_lens=P + 2)]


@pytest.mark.parametrize("kw", BAD)
def test_c_attention_refuses(kw):
    _lib, _ = _mod()
    lib = _lib.lib()
    assert lib.tdx_window_attention(C.byref(_attn_desc(**kw)), None) == 1
    assert b"tdx_window_attention" in lib.tdx_last_error()
    assert lib.tdx_window_attention_ws_bytes(C.byref(_attn_desc(**kw))) == 0
    d = _attn_desc(**kw)
    d.ws, d.ws_bytes = 16 * P, 1 << 40
    assert lib.tdx_window_attention_bwd(C.byref(d), None) == 1


@pytest.mark.parametrize("kw", [dict(lse=None), dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=P + 4), dict(dout_ts=3), dict(dq_bs=1), dict(dk_hs=2),
                                dict(dout_ts=1 << 25), dict(ws=None), dict(ws=16 * P + 4), dict(ws_bytes=15), dict(Tq=0)])
def test_c_attention_backward_refuses(kw):
    _lib, _ = _mod()
    lib = _lib.lib()
    d = _attn_desc()
    d.ws, d.ws_bytes = 16 * P, int(lib.tdx_window_attention_bwd_ws_bytes(C.byref(d)))
    assert d.ws_bytes > 0
    for n, v in kw.items():
        setattr(d, n, v)
    assert lib.tdx_window_attention_bwd(C.byref(d), None) == 1
    assert b"tdx_window_attention_bwd" in lib.tdx_last_error()


def test_an_output_that_overlaps_x_is_told_from_one_beside_it():
    _, att = _mod()
    room = torch.zeros(4 * 3 * 2 * 16)
    whole = room.view(1, 4, 6, 16)
    q, k = whole[:, :, :2], whole[:, :, 2:4]
    assert not att._clash(q, k) and not att._clash(k, q) and not att._clash(q, q) and not att._clash(q, whole[:, :, :2])
    assert att._clash(whole[:, :-1], whole[:, 1:]) and att._clash(whole[:, 1:], whole[:, :-1]) and att._clash(whole[:, :, :2], whole[:, :, 1:3])
    assert not att._clash(whole[:, :2], whole[:, 2:]) and att._clash(whole[..., :8], whole[..., 4:12]) and not att._clash(whole[..., :8], whole[..., 8:])
    assert att._clash(whole.view(1, 4, 6, 16), room.view(1, 6, 4, 16).transpose(1, 2))      # other strides
    assert not att._clash(whole, torch.zeros_like(whole))
    # against the element numbers themselves
    ids = torch.arange(200)
    gen = torch.Generator().manual_seed(5)
    draw = lambda n: int(torch.randint(0, n, (1,), generator=gen))
    for _ in range(400):
        shape = tuple(1 + draw(3) for _ in range(4))
        stride = tuple([1, 3, 4, 7, 12, 20][draw(6)] for _ in range(4))
        x, out = (ids.as_strided(shape, stride, draw(40)) for _ in range(2))
        pairs = {a: i for i, a in enumerate(x.flatten().tolist())}
        if len(pairs) < x.numel():
            continue                                            # x repeats its own memory
        want = any(pairs.get(a, i) != i for i, a in enumerate(out.flatten().tolist()))
        assert att._clash(x, out) == want, (shape, stride, x.storage_offset(), out.storage_offset())


def test_token_strides_beyond_a_stage_are_refused_or_copied():
    # dK / dV reads 64 rows from one address with 31-bit offsets: 64 token strides must stay below 2 GiB, also where 33 do
    _lib, att = _mod()
    lib = _lib.lib()
    ts = (1 << 30) // 48                                       # elements; x 2 bytes: 33 strides are 1.4 GiB, 65 are 2.7 GiB
    ts -= ts % 8
    for kw in (dict(q_ts=ts), dict(dout_ts=ts)):
        d = _attn_desc(B=1, Tq=64, Tk=64, Hq=1, Hkv=1, dtype=_lib.TDX_BF16, ws=16 * P, ws_bytes=1 << 40, **kw)
        assert lib.tdx_window_attention_bwd(C.byref(d), None) == 1 and b"too large" in lib.tdx_last_error()
    t = torch.empty(1, dtype=torch.bfloat16, device="meta").as_strided((1, 64, 1, 32), (64 * ts, ts, 32, 1))
    assert not att._lies_well(t, 1 << 31)


def test_c_launches_of_more_threads_than_a_launch_counts_are_refused():
    _lib, _ = _mod()
    lib = _lib.lib()
    many = 1 << 24                                             # workgroups of 256 threads: 2^32
    assert lib.tdx_rotary_axes(C.byref(_rotary_desc(B=many, T=8, H=1)), None) == 1 and b"too many" in lib.tdx_last_error()
    d = _attn_desc(B=many, Tq=1, Tk=4096, Hq=1, Hkv=1, left=-1, sinks=0)
    assert lib.tdx_window_attention(C.byref(d), None) == 1 and b"too many" in lib.tdx_last_error()
    for kw in (dict(Tq=1, Tk=8), dict(Tq=1, Tk=8, D=32), dict(Tq=1, Tk=100, sinks=9, left=2, B=many // 8)):
        d = _attn_desc(**dict(dict(B=many, Hq=1, Hkv=1, ws=16 * P, ws_bytes=1 << 60), **kw))
        assert lib.tdx_window_attention_bwd(C.byref(d), None) == 1 and b"too many" in lib.tdx_last_error()


def test_c_attention_workspaces():
    _lib, _ = _mod()
    lib = _lib.lib()
    for f in (lib.tdx_window_attention_ws_bytes, lib.tdx_window_attention_bwd_ws_bytes):
        assert f(None) == 0 and f(C.byref(_attn_desc(B=0))) == 0
    assert lib.tdx_window_attention(None, None) == 1 and lib.tdx_window_attention_bwd(None, None) == 1
    assert lib.tdx_window_attention(C.byref(_attn_desc(B=0, q=None, k=None, v=None, out=None)), None) == 0
    # few rows over a long cache: splits, which need scratch memory that the call insists on
    d = _attn_desc(B=1, Tq=1, Tk=32768, left=-1, sinks=0)
    need = int(lib.tdx_window_attention_ws_bytes(C.byref(d)))
    assert need > 0
    d.ws, d.ws_bytes = 16 * P, need - 1
    assert lib.tdx_window_attention(C.byref(d), None) == 1 and b"workspace" in lib.tdx_last_error()
    d.ws, d.ws_bytes = None, need
    assert lib.tdx_window_attention(C.byref(d), None) == 1
    # sinks: their shares come on top of the row statistics
    a = int(lib.tdx_window_attention_bwd_ws_bytes(C.byref(_attn_desc(Tq=1000, Tk=1000, sinks=0))))
    b = int(lib.tdx_window_attention_bwd_ws_bytes(C.byref(_attn_desc(Tq=1000, Tk=1000, sinks=7))))
    assert b > a > 0
    # sinks or windows that hold every key are no window at all (the rows that see a key, and so its shares, depend on the window)
    a = int(lib.tdx_window_attention_bwd_ws_bytes(C.byref(_attn_desc(Tq=1000, Tk=1000, left=-1, sinks=0))))
    assert int(lib.tdx_window_attention_bwd_ws_bytes(C.byref(_attn_desc(Tq=1000, Tk=1000, sinks=1000)))) == a
    assert int(lib.tdx_window_attention_bwd_ws_bytes(C.byref(_attn_desc(Tq=1000, Tk=1000, sinks=7, left=1000)))) == a


@pytest.mark.parametrize("kw", [dict(attn_heads=2), dict(attn_sinks=1), dict(attn_rotary=100.0), dict(attn_window=-1), dict(attn_window=4, attn_heads=3),
                                dict(attn_window=4, attn_heads=16), dict(attn_window=4, attn_heads=0), dict(attn_window=4, attn_sinks=-1), dict(attn_window=2.5),
                                dict(attn_window=4, attn_rotary=0.0), dict(attn_window=True)])
def test_model_refuses_attention_options(kw):
    from trajectorydiffusion_amd import TrajUNet
    _lib, _ = _mod()
    with pytest.raises(_lib.TdxError, match="AttnBlock"):
        TrajUNet([32, 32, 64], diffusion_steps=10, **kw)


def test_model_refuses_one_wide_head_and_keeps_its_parameters():
    from trajectorydiffusion_amd import AttnBlock, TrajUNet
    _lib, _ = _mod()
    with pytest.raises(_lib.TdxError, match="at most 128"):
        AttnBlock(256, 32, window=10)
    torch.manual_seed(0)
    a = TrajUNet([32, 32, 64], diffusion_steps=10)
    torch.manual_seed(0)
    b = TrajUNet([32, 32, 64], diffusion_steps=10, attn_heads=4, attn_window=9, attn_sinks=3, attn_rotary=500.0)
    assert list(a.state_dict()) == list(b.state_dict()) and all(torch.equal(x, y) for x, y in zip(a.state_dict().values(), b.state_dict().values()))


def test_a_block_takes_windows_and_sinks_beyond_every_length():
    from trajectorydiffusion_amd import engine
    rows, out = torch.zeros(1, 6, 3 * 64), torch.zeros(1, 6, 64)
    for n in (6, 1 << 31, (1 << 32) + 2, 1 << 40):               # (a descriptor counts in 32 bits)
        d = engine.WindowSpec.check(64, 2, n, n, None).attn_desc(rows, out, None, 1, 6, 64, 0)
        assert d.left >= 6 and d.right >= 6 and d.sinks >= 6


def test_the_reference_statement_itself():
    """The 64-bit statement against a loop over single rows, and its gradients against autograd."""
    g = torch.Generator().manual_seed(0)
    B, Tq, Tk, Hq, Hkv, D = 2, 9, 11, 4, 2, 8
    q, k, v, do = (torch.randn(B, T, H, D, generator=g, dtype=torch.float64) for T, H in ((Tq, Hq), (Tk, Hkv), (Tk, Hkv), (Tq, Hq)))
    ql, kl = torch.tensor([9, 6]), torch.tensor([8, 11])
    ok = R.seen(B, Tq, Tk, 3, 1, 2, ql, kl)
    R.HALF[torch.float64] = 0.0
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    ref = R.attention(*(t.detach() for t in x), ok, dout=do)
    out = torch.zeros_like(q)
    rows = []
    for b in range(B):
        for i in range(Tq):
            for h in range(Hq):
                keys = [j for j in range(Tk) if j < kl[b] and i < ql[b] and j <= i + kl[b] - ql[b] + 1 and (j >= i + kl[b] - ql[b] - 3 or j < 2)]
                assert [bool(t) for t in ok[b, i]] == [j in keys for j in range(Tk)]
                if keys:
                    w = torch.softmax(torch.stack([(x[0][b, i, h] * x[1][b, j, h // 2]).sum() for j in keys]) * D ** -0.5, 0)
                    o = sum(w[n] * x[2][b, j, h // 2] for n, j in enumerate(keys))
                    out[b, i, h] = o.detach()
                    rows.append((o * do[b, i, h]).sum())
    assert torch.allclose(out, ref["out"][0], atol=1e-12)
    for n, got in zip(("dq", "dk", "dv"), torch.autograd.grad(sum(rows), x)):
        assert torch.allclose(got, ref[n][0], atol=1e-12), n
    del R.HALF[torch.float64]
