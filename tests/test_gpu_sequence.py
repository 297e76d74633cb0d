"""GPU: rotary positions with several axes and windowed attention with visible first tokens, against plain statements in 64 bits.  Tolerances
are bounds derived in tests/_sequence_ref.py."""
import math

import pytest
import torch

import _sequence_ref as R

pytestmark = pytest.mark.gpu

DT = [torch.float32, torch.bfloat16]


def _att():
    from trajectorydiffusion_amd import attention
    return attention


def _normal(*shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- rotary ----------------------------------------------------------------------------------------------------------------------------
ROT = [  # B, T, H, D, sections, base, layout
    (2, 5, 3, 128, (32, 16, 16), 10000.0, "halves"),
    (1, 1, 1, 8, (4,), 10000.0, "pairs"),
    (3, 7, 10, 64, (10, 6), (10000.0, 500.0), "halves"),       # 16 pairs of 32: channels 32 .. 63 are copied
    (2, 33, 2, 96, (24, 24), (10000.0, 100.0), "pairs"),
    (1, 9, 5, 20, (3, 0, 2), 50.0, "halves"),                   # no whole vectors: the element path; an axis without pairs
    (1, 9, 5, 21, (3, 2), 50.0, "pairs"),                       # odd head width
    (1, 4100, 1, 256, (128,), 10000.0, "halves"),
    (70, 1, 12, 64, (32,), 10000.0, "pairs"),
]


def _rot_case(B, T, H, D, sections, dtype, seed=0):
    x = _normal(B, T, H, D, dtype=dtype, seed=seed)
    pos = torch.rand(B, T, len(sections), generator=torch.Generator().manual_seed(seed + 1)) * 3e5 - 1e3
    return x, pos.round() if seed % 2 else pos


def _rot_bound(x, P, layout):
    # each result is x0 c - x1 s: the angle's last rounding (2^-25 turns, 2^-22.3 rad) and sincospi (4 units) come to at most 2^-21 of |x0| + |x1|
    u = R.HALF[x.dtype]
    a = x.double().abs()
    both = torch.zeros_like(a)
    if layout == "halves":
        both[..., :P] = both[..., P:2 * P] = a[..., :P] + a[..., P:2 * P]
    else:
        s = a[..., 0:2 * P:2] + a[..., 1:2 * P:2]
        both[..., 0:2 * P:2] = both[..., 1:2 * P:2] = s
    return both * (2.0 ** -21 + 1.01 * u)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,T,H,D,sections,base,layout", ROT)
def test_rotary_matches_the_formula_both_ways(B, T, H, D, sections, base, layout, dtype):
    A = _att()
    bases = base if isinstance(base, tuple) else (base,) * len(sections)
    for seed in (0, 1):
        x, pos = _rot_case(B, T, H, D, sections, dtype, seed)
        P = sum(sections)
        for inverse in (False, True):
            got = A.rotary_axes(x.cuda(), pos.cuda(), sections, base, layout, inverse=inverse)
            assert got.dtype == dtype
            R.check("out", got, R.rotary(x, pos, sections, bases, layout, inverse), _rot_bound(x, P, layout))
        assert torch.equal(got[..., 2 * P:].cpu(), x[..., 2 * P:])


@pytest.mark.parametrize("dtype", DT)
def test_rotary_strides_shared_positions_in_place_and_out(dtype):
    A = _att()
    B, T, H, D, sec = 3, 6, 4, 64, (16, 16)
    rows = _normal(B, T, 3 * H * D, dtype=dtype, seed=3).cuda()
    pos = torch.arange(T * 2).float().reshape(T, 2).cuda() * 1000.5
    x = rows.view(B, T, 3, H, D)[:, :, 1]                       # the k slice of a q | k | v row matrix
    want = R.rotary(x.cpu(), pos.cpu()[None].expand(B, T, 2), sec, (10000.0,) * 2, "halves")
    bound = _rot_bound(x.cpu(), 32, "halves")
    R.check("slice", A.rotary_axes(x, pos, sec), want, bound)
    R.check("(1, T, axes)", A.rotary_axes(x, pos[None], sec), want, bound)
    R.check("head-major", A.rotary_axes(x.transpose(1, 2).contiguous().transpose(1, 2), pos, sec), want, bound)
    R.check("channels apart", A.rotary_axes(x.transpose(2, 3).contiguous().transpose(2, 3), pos, sec), want, bound)
    R.check("misaligned", A.rotary_axes(torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].view(B, T, H, D), pos, sec), want, bound)
    R.check("positions by their transpose", A.rotary_axes(x, pos.t().contiguous().t(), sec), want, bound)
    out = torch.full((B, T, H, D + 8), 7.0, dtype=dtype, device="cuda")
    assert A.rotary_axes(x, pos, sec, out=out[..., :D]).data_ptr() == out.data_ptr()
    R.check("out", out[..., :D], want, bound)
    assert (out[..., D:] == 7).all()
    before = rows.clone()
    A.rotary_axes(x, pos, sec, out=x)
    R.check("in place", x, want, bound)
    v = rows.view(B, T, 3, H, D)
    assert torch.equal(v[:, :, 0], before.view(B, T, 3, H, D)[:, :, 0]) and torch.equal(v[:, :, 2], before.view(B, T, 3, H, D)[:, :, 2])
    for empty in ((0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)):
        e = torch.empty(empty, dtype=dtype, device="cuda")
        assert A.rotary_axes(e, torch.zeros(empty[0], empty[1], 2, device="cuda"), sec).shape == empty


def test_rotary_out_beside_x_and_across_it():
    A = _att()
    qk = _normal(2, 6, 4, 32, dtype=torch.float32, seed=4).cuda()
    pos = torch.arange(6.0, device="cuda")[:, None]
    want = A.rotary_axes(qk[:, :, :2], pos, (16,))
    A.rotary_axes(qk[:, :, :2], pos, (16,), out=qk[:, :, 2:])          # between each other in one buffer
    assert torch.equal(qk[:, :, 2:], want)
    with pytest.raises(A.TdxError, match="overlaps"):
        A.rotary_axes(qk[:, :-1], pos[:-1], (16,), out=qk[:, 1:])


@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_rotary_gradient(layout):
    A = _att()
    B, T, H, D, sec = 2, 5, 3, 40, (9, 7)
    x, pos = _rot_case(B, T, H, D, sec, torch.float32)
    g = _normal(B, T, H, D, dtype=torch.float32, seed=9)
    xd = x.cuda().requires_grad_()
    out = A.rotary_axes(xd, pos.cuda(), sec, layout=layout)
    out.backward(g.cuda())
    R.check("dx", xd.grad, R.rotary(g, pos, sec, (10000.0,) * 2, layout, inverse=True), _rot_bound(g, 16, layout))
    # against differences: the map is linear, so one step of any size is exact up to rounding
    step = _normal(B, T, H, D, dtype=torch.float32, seed=10)
    lhs = (A.rotary_axes(x.cuda() + step.cuda(), pos.cuda(), sec, layout=layout).double() - out.detach().double()).mul(g.cuda().double()).sum()
    rhs = (xd.grad.double() * step.cuda().double()).sum()
    assert abs(float(lhs - rhs)) < 2.0 ** -20 * 3 * float((x.abs().sum() + step.abs().sum()) * 2) * float(g.abs().max())
    # an expanded gradient, and a broadcast input
    y = torch.randn(1, T, H, D, device="cuda", requires_grad=True)
    A.rotary_axes(y.expand(B, T, H, D), pos.cuda(), sec, layout=layout).sum().backward()
    want = R.rotary(torch.ones(B, T, H, D), pos, sec, (10000.0,) * 2, layout, inverse=True).sum(0, keepdim=True)
    R.check("dx of a broadcast input", y.grad, want, B * (2.0 ** -21 + 2.0 ** -24) * 2 + 2.0 ** -23 * B)


# ---- attention -------------------------------------------------------------------------------------------------------------------------
CASES = [  # B, Tq, Tk, Hq, Hkv, D, left, right, sinks, q_lens, k_lens
    (1, 1, 1, 1, 1, 8, None, None, 0, None, None),
    (2, 13, 13, 8, 8, 128, None, None, 0, None, None),
    (2, 13, 13, 2, 1, 24, 2, 1, 3, None, None),
    (1, 33, 33, 3, 3, 40, 0, 0, 0, None, None),                      # every point sees itself alone
    (1, 70, 70, 4, 2, 64, 5, 0, 1, None, None),
    (2, 130, 130, 2, 2, 32, 17, 9, 4, None, None),
    (1, 200, 200, 6, 2, 96, 40, 0, 7, None, None),                  # three heads of a group: rows that no power of two divides
    (1, 257, 257, 5, 1, 80, 64, 64, 33, None, None),                # sinks over more than one key tile
    (3, 129, 129, 4, 4, 64, 30, 0, 7, [129, 65, 1], [129, 65, 1]),
    (4, 40, 100, 4, 2, 64, 20, 5, 3, [40, 7, 0, 40], [100, 50, 30, 0]),   # empty queries, empty keys
    (2, 90, 40, 2, 2, 128, 10, 0, 2, None, None),                   # more queries than keys: the first see nothing
    (2, 64, 30, 2, 1, 64, None, 0, 0, [64, 10], [3, 30]),
    (1, 50, 50, 2, 2, 48, 3, 0, 200, None, None),                   # every key is a sink
    (1, 96, 96, 1, 1, 128, None, 4, 5, None, None),
    (1, 96, 96, 1, 1, 128, 4, None, 5, None, None),
    (2, 1, 300, 8, 2, 128, 100, 0, 4, None, [300, 37]),
    (1, 1, 2000, 4, 4, 64, None, 0, 0, None, None),                 # splits
    (2, 3, 1500, 16, 2, 96, 700, 0, 9, None, [1500, 2]),
    (1, 2, 1111, 40, 1, 128, 900, 0, 64, None, [1000]),             # 80 rows of one key head
    (1, 300, 300, 8, 1, 64, 100, 30, 16, None, None),
    (70, 150, 150, 4, 2, 64, 50, 10, 5, "ragged", "ragged"),        # enough workgroups for the many-row kernel
    (40, 140, 140, 8, 8, 128, 70, 0, 40, "ragged", "ragged"),
    (300, 130, 170, 1, 1, 32, 33, 20, 5, None, "ragged"),
    (1, 700, 700, 8, 1, 128, None, 0, 0, None, None),               # few keys, many rows: the rows of a key tile are cut into shares
    (2, 520, 600, 12, 2, 48, 200, None, 3, [520, 77], [600, 300]),
]


def _case(B, Tq, Tk, Hq, Hkv, D, dtype, q_lens, k_lens, seed=0):
    q, k, v, do = (_normal(B, T, H, D, dtype=dtype, seed=seed + n) for n, (T, H) in enumerate(((Tq, Hq), (Tk, Hkv), (Tk, Hkv), (Tq, Hq))))
    if k_lens == "ragged":
        k_lens = [Tk - (b * 37) % Tk for b in range(B)]
        q_lens = [min(Tq, n) for n in k_lens] if q_lens == "ragged" else q_lens
    lens = [None if n is None else torch.tensor(n, dtype=torch.int32) for n in (q_lens, k_lens)]
    return q, k, v, do, lens[0], lens[1]


def _cuda(t):
    return None if t is None else t.cuda()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,D,left,right,sinks,q_lens,k_lens", CASES)
def test_attention_forward(B, Tq, Tk, Hq, Hkv, D, left, right, sinks, q_lens, k_lens, dtype):
    A = _att()
    q, k, v, _, ql, kl = _case(B, Tq, Tk, Hq, Hkv, D, dtype, q_lens, k_lens)
    ref = R.attention(q, k, v, R.seen(B, Tq, Tk, left, right, sinks, ql, kl))
    out, lse = A.window_attention(q.cuda(), k.cuda(), v.cuda(), left, right, sinks, _cuda(ql), _cuda(kl), return_lse=True)
    assert out.dtype == dtype and lse.dtype == torch.float32
    R.check("out", out, *ref["out"])
    R.check("lse", lse, *ref["lse"])
    again = A.window_attention(q.cuda(), k.cuda(), v.cuda(), left, right, sinks, _cuda(ql), _cuda(kl))
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,D,left,right,sinks,q_lens,k_lens", CASES)
def test_attention_backward(B, Tq, Tk, Hq, Hkv, D, left, right, sinks, q_lens, k_lens, dtype):
    A = _att()
    q, k, v, do, ql, kl = _case(B, Tq, Tk, Hq, Hkv, D, dtype, q_lens, k_lens, seed=5)
    ref = R.attention(q, k, v, R.seen(B, Tq, Tk, left, right, sinks, ql, kl), dout=do)
    x = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, lse = A.window_attention(*x, left, right, sinks, _cuda(ql), _cuda(kl), return_lse=True)
    grads = torch.autograd.grad(out, x, do.cuda(), retain_graph=True)
    R.check("out", out, *ref["out"])
    R.check("lse", lse, *ref["lse"])
    for n, g in zip(("dq", "dk", "dv"), grads):
        R.check(n, g, *ref[n])
    for a, b in zip(grads, torch.autograd.grad(out, x, do.cuda())):
        assert torch.equal(a, b)


def test_attention_gradient_against_differences():
    A = _att()
    B, Tq, Tk, Hq, Hkv, D = 1, 40, 52, 4, 2, 32
    q, k, v, do, ql, kl = _case(B, Tq, Tk, Hq, Hkv, D, torch.float32, [37], [49], seed=11)
    f = lambda *x: (A.window_attention(*x, 9, 3, 2, ql.cuda(), kl.cuda()).double() * do.cuda().double()).sum()  # noqa: E731
    x = [t.cuda().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(f(*x), x)
    h = 2.0 ** -6
    for n in range(3):
        step = _normal(*x[n].shape, dtype=torch.float32, seed=20 + n).cuda()
        at = lambda s: f(*[t.detach() + (s * step if m == n else 0) for m, t in enumerate(x)])  # noqa: E731
        # fourth order: the error is h^4 / 30 of the fifth derivative (a few hundred) plus rounding 2^-20 |out| |do| / h
        diff = float((8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h))
        want = float((grads[n].double() * step.double()).sum())
        size = float((grads[n].double() * step.double()).abs().sum())
        assert abs(diff - want) < 2e-3 * size, (n, diff, want)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Tq,Tk", [(1, 400), (150, 150)])
def test_attention_takes_slices_and_odd_strides(dtype, Tq, Tk):
    A = _att()
    B, H, D = 2, 4, 64
    q, k, v, do, _, _ = _case(B, Tq, Tk, H, H, D, dtype, None, None, seed=2)
    want = R.attention(q, k, v, R.seen(B, Tq, Tk, 60, 7, 3), dout=do)
    forms = {
        "rows of q | k | v": lambda t: torch.cat([t, t, t], dim=2).cuda()[:, :, H:2 * H],
        "heads before tokens": lambda t: t.transpose(1, 2).contiguous().cuda().transpose(1, 2),
        "tokens before batch": lambda t: t.transpose(0, 1).contiguous().cuda().transpose(0, 1),
        "channels apart": lambda t: t.transpose(2, 3).contiguous().cuda().transpose(2, 3),
        "misaligned": lambda t: torch.cat([t.reshape(-1)[:3], t.reshape(-1)]).cuda()[3:].view(t.shape),
        "odd row pitch": lambda t: torch.cat([t, t[..., :5]], dim=3).cuda()[..., :D],
    }
    for name, form in forms.items():
        x = [form(t).detach().requires_grad_() for t in (q, k, v)]
        out = A.window_attention(*x, 60, 7, 3)
        R.check(name, out, *want["out"])
        for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, x, form(do))):
            R.check(f"{name}: {n}", g, *want[n])


def test_numbers_given_as_tensors_count_by_their_value():
    A = _att()
    x = _normal(2, 40, 2, 32, dtype=torch.float32, seed=6).cuda()
    pos = torch.arange(40.0, device="cuda")[:, None]
    scale, base, pairs = torch.tensor(0.25), torch.tensor(100.0), torch.tensor(16)
    for _ in range(2):
        assert torch.equal(A.window_attention(x, x, x, 5, 5, 1, scale=scale), A.window_attention(x, x, x, 5, 5, 1, scale=float(scale)))
        for b in (base, [base]):
            assert torch.equal(A.rotary_axes(x, pos, [pairs], base=b), A.rotary_axes(x, pos, (int(pairs),), base=float(base)))
        scale.mul_(3)
        base.mul_(7)
        pairs.sub_(4)


def test_rows_far_apart_in_memory():
    # 64 rows of q and of dout span 2.6 GB: as far as one tile's offsets do not reach
    A = _att()
    T, ts = 64, 20 * 1024 * 1024
    room = torch.empty(T * ts, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    x = [torch.randn(1, T, 1, 32, generator=g, device="cuda").bfloat16() for _ in range(4)]
    far = [room[o:].as_strided((1, T, 1, 32), (T * ts, ts, 32, 1)) for o in (0, 1024)]
    for f, t in zip(far, (x[0], x[3])):
        f.copy_(t)
    results = []
    for q, dout in ((x[0], x[3]), far):
        q, k, v = (t.detach().requires_grad_() for t in (q, x[1], x[2]))
        out = A.window_attention(q, k, v, 20, 4, 3)
        results.append((out.detach(),) + torch.autograd.grad(out, (q, k, v), dout))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("Tq,Tk,few", [(1, 700, True), (150, 150, True), (150, 150, False)])
def test_what_is_not_seen_does_not_reach_a_row(dtype, bad, Tq, Tk, few):
    """Not-a-numbers and infinities behind the lengths and outside the windows, in every input; gradients too."""
    A = _att()
    B, H, G, D = (2, 2, 2, 64) if few else (80, 2, 2, 64)
    q, k, v, do, _, _ = _case(B, Tq, Tk, H * G, H, D, dtype, None, None, seed=4)
    kl = torch.full((B,), Tk - 11, dtype=torch.int32)
    ql = torch.full((B,), max(1, Tq - 11) if Tq > 1 else 1, dtype=torch.int32)
    ok = R.seen(B, Tq, Tk, 20, 2, 3, ql, kl)
    ref = R.attention(q, k, v, ok, dout=do)
    kd, vd, qd, dd = k.clone(), v.clone(), q.clone(), do.clone()
    for t in (kd, vd):
        t[:, Tk - 11:] = bad
    for t in (qd, dd):
        t[:, int(ql[0]):] = bad
    x = [t.cuda().requires_grad_() for t in (qd, kd, vd)]
    out, lse = A.window_attention(*x, 20, 2, 3, ql.cuda(), kl.cuda(), return_lse=True)
    R.check("out", out, *ref["out"])
    R.check("lse", lse, *ref["lse"])
    for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, x, dd.cuda())):
        R.check(n, g, *ref[n])
    # inside the lengths: one key and value that only some rows see; the others keep their results
    j = 50
    kd, vd = k.clone(), v.clone()
    vd[:, j] = bad
    hit = ok[0, :, j]
    x = [t.cuda().requires_grad_() for t in (q, kd, vd)]
    out = A.window_attention(*x, 20, 2, 3, ql.cuda(), kl.cuda())
    R.check("rows that do not see it", out[:, ~hit], ref["out"][0][:, ~hit], ref["out"][1][:, ~hit])
    assert not torch.isfinite(out[:, hit]).any()
    grads = torch.autograd.grad(out, x, do.cuda())
    R.check("dq of rows that do not see it", grads[0][:, ~hit], ref["dq"][0][:, ~hit], ref["dq"][1][:, ~hit])
    far = ~ok[0][hit].any(0)                                          # keys that none of the hit rows sees
    for n in (1, 2):
        name = ("dq", "dk", "dv")[n]
        R.check(name, grads[n][:, far], ref[name][0][:, far], ref[name][1][:, far])
    kd[:, j] = bad
    out = A.window_attention(q.cuda(), kd.cuda(), v.cuda(), 20, 2, 3, ql.cuda(), kl.cuda())
    R.check("key: rows that do not see it", out[:, ~hit], ref["out"][0][:, ~hit], ref["out"][1][:, ~hit])
    # a row of its own that is not a number: its neighbours keep theirs, and so do keys that it does not see
    if Tq > 1:
        qd = q.clone()
        qd[:, 30] = math.nan
        x = [t.cuda().requires_grad_() for t in (qd, k, v)]
        out = A.window_attention(*x, 20, 2, 3, ql.cuda(), kl.cuda())
        rest = torch.arange(Tq) != 30
        R.check("other rows", out[:, rest], ref["out"][0][:, rest], ref["out"][1][:, rest])
        assert torch.isnan(out[:, 30]).all()
        grads = torch.autograd.grad(out, x, do.cuda())
        R.check("dq of other rows", grads[0][:, rest], ref["dq"][0][:, rest], ref["dq"][1][:, rest])
        far = ~ok[0][30]
        for n in (1, 2):
            name = ("dq", "dk", "dv")[n]
            R.check(f"{name} of keys it does not see", grads[n][:, far], ref[name][0][:, far], ref[name][1][:, far])
            assert torch.isnan(grads[n][:, ~far]).all()


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_shares_keep_out_what_is_not_seen(dtype, D):
    """Few key heads: rows and keys are cut into shares, and the launches that join them take bad rows again."""
    import ctypes as C

    from test_sequence_cpu import _attn_desc

    from trajectorydiffusion_amd import _lib
    A = _att()
    T, G, window = 900, 8, (400, 0, 3)
    desc = _attn_desc(B=1, Tq=T, Tk=T, Hq=G, Hkv=1, D=D, dtype=A._CODES[dtype], left=400, right=0, sinks=0)
    rows, keys = -(-T * G // 128) * 128 * 8, T * D * 8            # bytes of the row statistics, of a share of dK and dV
    assert int(_lib.lib().tdx_window_attention_bwd_ws_bytes(C.byref(desc))) >= rows + 2 * keys
    q, k, v, do, _, _ = _case(1, T, T, G, 1, D, dtype, None, None, seed=8)
    ok = R.seen(1, T, T, *window)
    ref = R.attention(q, k, v, ok, dout=do)

    def grads(q, k, v):
        x = [t.cuda().requires_grad_() for t in (q, k, v)]
        out = A.window_attention(*x, *window)
        g = torch.autograd.grad(out, x, do.cuda(), retain_graph=True)
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(g, torch.autograd.grad(out, x, do.cuda())))
        return (out,) + g

    names = ("out", "dq", "dk", "dv")
    for n, g in zip(names, grads(q, k, v)):
        R.check(n, g, *ref[n])
    for bad in (math.nan, math.inf):
        vd = v.clone()
        vd[:, 50] = bad
        hit = ok[0, :, 50]
        far = ~ok[0][hit].any(0)
        assert (~hit).any() and far.any()
        got = grads(q, k, vd)
        for n, g, keep in zip(names, got, (~hit, ~hit, far, far)):
            R.check(f"{n}, {bad} in a value", g[:, keep], ref[n][0][:, keep], ref[n][1][:, keep])
    qd = q.clone()
    qd[:, 700] = math.nan
    others, far = torch.arange(T) != 700, ~ok[0][700]
    got = grads(qd, k, v)
    for n, g, keep in zip(names, got, (others, others, far, far)):
        R.check(f"{n}, a row of NaN", g[:, keep], ref[n][0][:, keep], ref[n][1][:, keep])
        assert torch.isnan(g[:, ~keep]).all()
