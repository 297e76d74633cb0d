"""GPU: the sequence operators where values or offsets are extreme, and where autograd has to be told: against plain statements in 64 bits."""
import math

import pytest
import torch

import _sequence_ref as R

pytestmark = pytest.mark.gpu

DT = [torch.float32, torch.bfloat16]


def _att():
    from trajectorydiffusion_amd import attention
    return attention


def _normal(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- what autograd is told --------------------------------------------------------------------------------------------------------------
def test_a_key_that_attention_kept_may_not_be_rotated_before_the_backward_pass():
    A = _att()
    q, k, v = (_normal(1, 20, 2, 32, seed=n).cuda() for n in range(3))
    pos = torch.arange(20.0, device="cuda")[:, None]
    q.requires_grad_()
    out = A.window_attention(q, k, v, 5, 0, 1)
    A.rotary_axes(k, pos, (16,), out=k)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


# ---- scores of every size ----------------------------------------------------------------------------------------------------------------
# A probability is rebuilt in the backward pass as 2^(s c - lse2) while |lse2| <= T (T = 128 for fp32, 2048 for bf16), from a log-sum lse2 that has been
# rounded four times (m scale, + log l, log2 e, c) and two more of this size in the exponent: 6 v T ln 2 off; beyond, from the distance to the row's maximum
# and the row's own sum, which are exact where one key, or several alike, hold all of a row.
BUILT = {torch.float32: 6 * R.V * 128 * math.log(2), torch.bfloat16: 6 * R.V * 2048 * math.log(2)}


def _tops(q, table, which, ok):
    """(highest score of each row, the keys that have it, the largest |q| |k| scale, whether the next score is further away than what 32-bit scores may be off,
    and 100)"""
    B, Tq, Hq, D = q.shape
    Q, each = q.double().permute(0, 2, 1, 3), table.double().permute(0, 2, 1, 3).repeat_interleave(Hq // table.shape[2], dim=1)
    scale, m = D ** -0.5, ok[:, None].expand(B, Hq, Tq, len(which))
    S = torch.where(m, (Q @ each.transpose(2, 3) * scale)[..., which], torch.full((1,), -math.inf, dtype=torch.float64))
    a = float((Q.abs() @ each.abs().transpose(2, 3) * scale).max())
    top = S.amax(-1, keepdim=True)
    near = (S == top) & m
    gap = torch.where(near, torch.full_like(S, -math.inf), S).amax(-1, keepdim=True)
    return top, near, a, ((top - gap) > 2 * (D + 4) * R.V * a + 100)[..., 0] | ~m.any(-1)


def _peaked(q, table, which, v, ok, do):
    """name -> (value, bound) like R.attention, for keys table[which]: every row's probabilities are 1 / n at n equal keys and 0 elsewhere."""
    u = R.HALF[q.dtype]
    u1 = u if q.dtype != torch.float32 else 0.0
    e = BUILT[q.dtype] + 2.0 ** -18
    B, Tq, Hq, D = q.shape
    Tk, Hkv = v.shape[1], v.shape[2]
    G, scale = Hq // Hkv, D ** -0.5
    Q, dO = (t.double().permute(0, 2, 1, 3) for t in (q, do))
    W, K = (t.double().permute(0, 2, 1, 3).repeat_interleave(G, dim=1) for t in (v, table[:, which]))
    m = ok[:, None].expand(B, Hq, Tq, Tk)
    top, near, a, sure = _tops(q, table, which, ok)
    assert sure.all(), "a row whose probabilities are not certain"
    n = near.sum(-1, keepdim=True)
    P = near.double() / n.clamp(min=1)
    lse = torch.where(n > 0, top + n.double().log(), top)[..., 0]
    out, PW = P @ W, P @ W.abs()
    e_out = u * out.abs() + (u1 + e + Tk * R.V) * PW * (1 + u)
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    got = {"out": (back(out), back(e_out)), "lse": (lse, 2 * (D + 4) * R.V * a + 4 * R.V * lse.abs().nan_to_num(0, 0, 0) + e)}
    dO = dO * m.any(-1)[..., None]
    dP, delta = dO @ W.transpose(2, 3), (dO * out).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    e_dp = D * R.V * (dO.abs() @ W.abs().transpose(2, 3)) + (dO.abs() * (e_out + D * R.V * out.abs())).sum(-1, keepdim=True) + 4 * R.V * (dP.abs() + delta.abs())
    e_ds = (u1 + e) * dS.abs() + (1 + u1 + e) * P * e_dp
    group = lambda t: t.reshape(B, Hkv, G, *t.shape[2:]).sum(2)  # noqa: E731
    rows = Tq * G * R.V
    dq, e_dq = dS @ K * scale, (e_ds + Tk * R.V * dS.abs()) @ K.abs() * scale
    dk, e_dk = group(dS.transpose(2, 3) @ Q) * scale, group((e_ds + rows * dS.abs()).transpose(2, 3) @ Q.abs()) * scale
    dv, e_dv = group(P.transpose(2, 3) @ dO), group(((u1 + e + rows) * P).transpose(2, 3) @ dO.abs())
    for name, g, eg in (("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv)):
        got[name] = (back(g), back(u * (g.abs() + eg) + eg + 4 * R.V * g.abs()))
    return got


FORMS = [  # B, Tq, Tk, Hq, Hkv, D, left, right, sinks
    (2, 13, 13, 8, 8, 128, None, None, 0),
    (2, 13, 13, 2, 1, 24, 2, 1, 3),
    (2, 130, 130, 2, 2, 32, 17, 9, 4),
    (1, 70, 70, 4, 2, 64, 5, 0, 3),
    (1, 300, 300, 8, 1, 96, 100, 30, 16),
    (1, 900, 900, 8, 1, 64, 400, 0, 3),              # rows and keys in shares
    (1, 900, 900, 8, 1, 128, None, 0, 0),
    (80, 150, 150, 4, 2, 64, 20, 2, 3),              # enough workgroups for the many-row kernel
    (40, 140, 140, 8, 4, 128, 70, 0, 40),
    (300, 130, 130, 1, 1, 32, 33, 20, 5),
]


def _sized(B, Tq, Tk, Hq, Hkv, D, size, dtype, kinds, seed):
    """q, table of keys, which key stands where, v, dout: scaled scores of about `size`."""
    q, table = (_normal(B, T, H, D, seed=seed + n) * size ** 0.5 for n, (T, H) in enumerate(((Tq, Hq), (kinds, Hkv))))
    v, do = (_normal(B, T, H, D, seed=seed + 2 + n) for n, (T, H) in enumerate(((Tk, Hkv), (Tq, Hq))))
    which = torch.randint(0, kinds, (Tk,), generator=torch.Generator().manual_seed(seed)) if kinds < Tk else torch.arange(Tk)
    return q.to(dtype), table.to(dtype), which, v.to(dtype), do.to(dtype)


def _settled(q, table, which, ok, size, seed):
    """q with other rows in the place of those whose probabilities are not certain."""
    for turn in range(20):
        sure = _tops(q, table, which, ok)[3].transpose(1, 2)
        if sure.all():
            break
        other = (_normal(*q.shape, seed=1000 + 20 * seed + turn) * size ** 0.5).to(q.dtype)
        q = torch.where(sure[..., None], q, other)
    return q


def _compare(ref, q, k, v, do, args, **kwargs):
    """The bounds hold for normal numbers; the hardware's exp2 gives 0 for results below 2^-126, and so may the rounding of a score gradient to bf16.  A probability
    is therefore off by another 2^-126, a score gradient by that times 1 + |dP - delta|, and sums by as much for each of their terms."""
    A, tiny = _att(), 2.0 ** -126
    most = [float(t.double().abs().nan_to_num(0, 0, 0).max()) for t in (q, k, v, do)]
    grads, scale = 1 + 2 * q.shape[3] * most[2] * most[3], kwargs.get("scale") or q.shape[3] ** -0.5
    rows = q.shape[1] * q.shape[2] // k.shape[2]
    for n, more in (("out", k.shape[1] * most[2]), ("dq", k.shape[1] * grads * most[1] * scale), ("dk", rows * grads * most[0] * scale), ("dv", rows * most[3])):
        ref[n] = (ref[n][0], ref[n][1] + tiny * more)
    x = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, lse = A.window_attention(*x, *args, return_lse=True, **kwargs)
    R.check("out", out, *ref["out"])
    R.check("lse", lse, *ref["lse"])
    grads = torch.autograd.grad(out, x, do.cuda(), retain_graph=True)
    for n, g in zip(("dq", "dk", "dv"), grads):
        R.check(n, g, *ref[n])
    for a, b in zip(grads, torch.autograd.grad(out, x, do.cuda())):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("size", [1.0, 1e3, 1e7, 1e30])
@pytest.mark.parametrize("form", FORMS)
def test_rows_that_see_one_key(form, size, dtype):
    """Their probability is 1, so dv is dout, and dq and dk are what rounding leaves of nothing."""
    B, Tq, Tk, Hq, Hkv, D = form[:6]
    q, table, which, v, do = _sized(B, Tq, Tk, Hq, Hkv, D, size, dtype, Tk, 3)
    _compare(_peaked(q, table, which, v, R.seen(B, Tq, Tk, 0, 0, 0), do), q, table, v, do, (0, 0, 0))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("size", [1e7, 1e30])
@pytest.mark.parametrize("form", FORMS)
def test_gradients_of_huge_scores(form, size, dtype):
    """Rows over several keys, some of them alike: these share the probability."""
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = form
    q, table, which, v, do = _sized(B, Tq, Tk, Hq, Hkv, D, size, dtype, min(Tk, 8), 11)
    k, ok = table[:, which].contiguous(), R.seen(B, Tq, Tk, left, right, sinks)
    q = _settled(q, table, which, ok, size, 11)
    _compare(_peaked(q, table, which, v, ok, do), q, k, v, do, (left, right, sinks))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("size", [1e3])
@pytest.mark.parametrize("form", FORMS)
def test_gradients_of_large_scores(form, size, dtype):
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = form
    q, table, which, v, do = _sized(B, Tq, Tk, Hq, Hkv, D, size, dtype, Tk, 17)
    _compare(R.attention(q, table, v, R.seen(B, Tq, Tk, left, right, sinks), dout=do), q, table, v, do, (left, right, sinks))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("size", [1.0, 1e10])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("form", [(2, 130, 130, 2, 2, 32, 17, 9, 4), (1, 900, 900, 8, 1, 64, 400, 0, 3), (80, 150, 150, 4, 2, 64, 20, 2, 3), (40, 140, 140, 8, 4, 128, 50, 0, 40),
                                  (2, 1, 700, 4, 2, 128, 20, 2, 3)])
def test_what_is_not_seen_does_not_reach_a_row_of_huge_scores(form, bad, size, dtype):
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = form
    A = _att()
    q, table, which, v, do = _sized(B, Tq, Tk, Hq, Hkv, D, size, dtype, Tk if size == 1 else 8, 23)
    k = table[:, which].contiguous()
    kl = torch.full((B,), Tk - 11, dtype=torch.int32)
    ql = torch.full((B,), max(1, Tq - 11), dtype=torch.int32)
    ok = R.seen(B, Tq, Tk, left, right, sinks, ql, kl)
    q = q if size == 1 else _settled(q, table, which, ok, size, 23)
    ref = R.attention(q, k, v, ok, dout=do) if size == 1 else _peaked(q, table, which, v, ok, do)
    for t in (k, v):
        t[:, Tk - 11:] = bad
    for t in (q, do):
        t[:, int(ql[0]):] = bad
    _compare(ref, q, k, v, do, (left, right, sinks), q_lens=ql.cuda(), k_lens=kl.cuda())
    # a value that some rows see: the others keep their results, and so do keys that none of these rows sees
    v[:, 60], hit = bad, ok[0, :, 60]
    far = ~ok[0][hit].any(0)
    x = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = A.window_attention(*x, left, right, sinks, ql.cuda(), kl.cuda())
    got = (out,) + torch.autograd.grad(out, x, do.cuda())
    for name, g, keep in zip(("out", "dq", "dk", "dv"), got, (~hit, ~hit, far, far)):
        R.check(f"{name}, {bad} in a value", g[:, keep], ref[name][0][:, keep], ref[name][1][:, keep])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("scale", [1.2e-38, 1e-39, 3e-42, 1.5e-45])
@pytest.mark.parametrize("form", [(2, 13, 13, 2, 2, 64, 5, 2, 1), (1, 1, 3000, 2, 2, 64, None, 0, 0), (80, 150, 150, 4, 2, 64, 20, 2, 3), (1, 900, 900, 8, 1, 32, 400, 0, 3)])
def test_the_smallest_scales(form, scale, dtype):
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = form
    q, k, v, do = (_normal(B, T, H, D, seed=n) for n, (T, H) in enumerate(((Tq, Hq), (Tk, Hkv), (Tk, Hkv), (Tq, Hq))))
    # Products of up to 1e38.  A scale below 2^-126 holds fewer bits: scale log2 e is off by half a step of 2^-149, which at these scores (3e37 scale, times 5
    # at most) is below 2^-23 and so part of what the bound gives exponentials (2^-20).
    q, k, v, do = (q * 2e18).to(dtype), (k * 2e18).to(dtype), v.to(dtype), do.to(dtype)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    _compare(R.attention(q, k, v, R.seen(B, Tq, Tk, left, right, sinks), scale=scale, dout=do), q, k, v, do, (left, right, sinks), scale=scale)


# ---- values next to the largest --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("form", [(2, 13, 13, 2, 2, 64, None, None, 0), (1, 1, 3000, 2, 2, 64, None, 0, 0), (1, 70, 70, 4, 2, 64, 5, 0, 3), (80, 150, 150, 4, 2, 64, 20, 2, 3),
                                  (40, 140, 140, 8, 4, 128, 50, 0, 40), (300, 130, 130, 1, 1, 32, 33, 20, 5)])
def test_averages_of_values_next_to_the_largest(form, dtype):
    """A weighted mean of numbers is a number, also where the sum of them all is none."""
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = form
    A = _att()
    q, k, v = (_normal(B, T, H, D, seed=n, dtype=dtype) for n, (T, H) in enumerate(((Tq, Hq), (Tk, Hkv), (Tk, Hkv))))
    most = 3.4e38 if dtype == torch.float32 else 3.0e38
    for v in (torch.full_like(v, most), (v.float().sign() * most).to(dtype), (v.float() * 1e37).to(dtype)):
        ref = R.attention(q, k, v, R.seen(B, Tq, Tk, left, right, sinks))
        R.check("out", A.window_attention(q.cuda(), k.cuda(), v.cuda(), left, right, sinks), *ref["out"])


@pytest.mark.parametrize("form", [(2, 13, 13, 2, 2, 64), (80, 150, 150, 4, 4, 64), (40, 140, 140, 8, 8, 128), (300, 130, 130, 1, 1, 32), (1, 900, 900, 1, 1, 64)])
def test_fp32_numbers_between_the_largest_of_bf16_and_of_fp32(form):
    """In every operand in turn, its partner small: each row sees one key, so dv is dout."""
    B, Tq, Tk, Hq, Hkv, D = form
    parts = [_normal(B, T, H, D, seed=n) for n, (T, H) in enumerate(((Tq, Hq), (Tk, Hkv), (Tk, Hkv), (Tq, Hq)))]
    small = lambda t: t * 2.0 ** -100                                                       # noqa: E731
    big = lambda t: torch.where(t > 0, 3.4e38, -3.395e38) * torch.where(t.abs() < 1, 1.0, 0.5)   # noqa: E731
    ok = R.seen(B, Tq, Tk, 0, 0, 0)
    for forms in ((big, small, None, None), (small, big, None, None), (None, None, big, small), (None, None, small, big)):
        q, k, v, do = (t if f is None else f(t) for f, t in zip(forms, parts))
        scale = 2.0 ** -30 if forms[0] else D ** -0.5
        _compare(R.attention(q, k, v, ok, scale=scale, dout=do), q, k, v, do, (0, 0, 0), scale=scale)


@pytest.mark.parametrize("form", [(2, 13, 13, 2, 2, 64, 5, 2, 1), (80, 150, 150, 4, 2, 64, 20, 2, 3), (40, 140, 140, 8, 4, 128, 50, 0, 40)])
def test_fp32_numbers_next_to_the_smallest(form):
    """Around 2^-118 the second and third bf16 plane of a number have exponents below bf16's normal numbers, whose step is 2^-133: half of it is lost of each
    number.  As q (k 2^118 times as large) that is 2^-16 sum |k| scale of a score, below 2^-13 here, so 2^-12 of a probability, once more for their sum."""
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = form
    q, k, v = (_normal(B, T, H, D, seed=n) for n, (T, H) in enumerate(((Tq, Hq), (Tk, Hkv), (Tk, Hkv))))
    ok = R.seen(B, Tq, Tk, left, right, sinks)
    A = _att()
    tiny = 2.0 ** -118
    assert float(k.abs().sum(-1).max()) * D ** -0.5 < 8 * 1.6
    for f, more in (((tiny, 1 / tiny, 1), 2.0 ** -11 * float(v.abs().max())), ((1 / tiny, tiny, 1), 2.0 ** -11 * float(v.abs().max())), ((1, 1, tiny), 2.0 ** -133)):
        x = [t * n for t, n in zip((q, k, v), f)]
        want, bound = R.attention(*x, ok)["out"]
        R.check(f"out {f}", A.window_attention(*(t.cuda() for t in x), left, right, sinks), want, bound + more)


# ---- a value that is not a number in a long causal sequence -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_one_channel_of_one_value_spoils_one_channel_of_its_rows(bad, dtype):
    A = _att()
    B, T, H, D = 2, 1500, 8, 64
    q, k, v = (_normal(B, T, H, D, dtype=dtype, seed=n) for n in range(3))
    ref = R.attention(q, k, v, R.seen(B, T, T, None, 0, 0))["out"]
    v[:, 700, :, 5] = bad
    out = A.window_attention(q.cuda(), k.cuda(), v.cuda(), None, 0).cpu()
    keep = torch.ones(T, D, dtype=torch.bool)
    keep[700:, 5] = False
    for b in range(B):
        for h in range(H):
            R.check("out", out[b, :, h][keep], ref[0][b, :, h][keep], ref[1][b, :, h][keep])
            assert not torch.isfinite(out[b, 700:, h, 5]).any()


# ---- offsets beyond 32 bits in the backward pass --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
def test_gradients_at_offsets_beyond_32_bits(dtype):
    """Batches 2^31 elements and more apart, and tokens whose indexes times their stride pass 2^31 elements; results are those of packed tensors."""
    A = _att()
    B, T, H, D, es = 2, 300, 2, 32, 2 if dtype == torch.bfloat16 else 4
    x = [_normal(B, T, H, D, dtype=dtype, seed=n).cuda() for n in range(4)]
    far_token = (1 << 24) // es - 64                           # just below 16 MiB
    ts = far_token - far_token % 8
    assert es == 4 or T * ts > 1 << 31
    room = torch.empty(max((1 << 31) + 64 + T * H * D, (T * ts if es == 2 else 0) + 1024), dtype=dtype, device="cuda")

    def run(q, k, v, do):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        out = A.window_attention(q, k, v, 40, 9, 5)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), do)
    want = run(*x)
    strides = {"batches": ((1 << 31) + 64, H * D, D)}
    if es == 2:
        strides["tokens"] = (512, ts, D)
    for name, st in strides.items():
        for n in range(4):                                      # one operand at a time
            far = room.as_strided((B, T, H, D), st + (1,))
            far.copy_(x[n])
            got = run(*(far if m == n else t for m, t in enumerate(x)))
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (name, n)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("form", [(2, 13, 13, 2, 2, 8, 2, 1, 0), (1, 1, 3000, 2, 2, 8, None, 0, 0), (1, 300, 300, 8, 1, 8, 100, 30, 16), (300, 130, 130, 1, 1, 8, 33, 20, 5)])
def test_rows_whose_scaled_scores_all_lie_below_32_bits(form, dtype):
    """Their log-sum is none that 32 bits hold, but they see keys: all alike here, so each gets an equal share.  Sums of products are -2.4e38, times a scale of 2."""
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = form
    A = _att()
    q, k = (torch.full((B, T, H, D), x).to(dtype) for T, H, x in ((Tq, Hq, 3e18), (Tk, Hkv, -1e19)))
    v, do = (_normal(B, T, H, D, seed=n, dtype=dtype) for n, (T, H) in enumerate(((Tk, Hkv), (Tq, Hq))))
    zero = torch.zeros_like(q)
    ref = R.attention(zero, k * 0, v, R.seen(B, Tq, Tk, left, right, sinks), dout=do)      # equal scores
    x = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, lse = A.window_attention(*x, left, right, sinks, scale=2.0, return_lse=True)
    R.check("out", out, *ref["out"])
    assert (lse < -3.4e38).all() and torch.isfinite(lse).all()
    R.check("dv", torch.autograd.grad(out, x, do.cuda())[2], *ref["dv"])
