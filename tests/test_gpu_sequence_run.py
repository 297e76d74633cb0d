"""GPU: the sequence operators as they are used: together (prompt, then single tokens over a cache), on other streams, in captured graphs, at the
ends of their ranges, and inside TrajUNet (forward, sampling, training) against the oracle with its middle attention restated."""
import ctypes as C
import math

import pytest
import torch
import torch.nn.functional as F

import _sequence_ref as R

pytestmark = pytest.mark.gpu

DT = [torch.float32, torch.bfloat16]


def _att():
    from trajectorydiffusion_amd import attention
    return attention


def _normal(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- together ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
def test_prompt_then_single_tokens_over_a_cache(dtype):
    """Rotate and attend over a padded prompt, fill a cache, then append one token at a time to sequences of different lengths: every token's
    result is the row of one causal pass over the whole sequence."""
    A = _att()
    B, Hq, Hkv, D, cap, sec = 3, 4, 2, 64, 96, (16, 8, 8)
    lens, new = [40, 17, 1], 12
    T = 64
    q, k, v = (_normal(B, T, H, D, dtype=dtype, seed=n) for n, H in enumerate((Hq, Hkv, Hkv)))
    pos = torch.stack([torch.arange(T).float().expand(B, T) * 60, (_normal(B, T, seed=5) * 40).round(), (_normal(B, T, seed=6) * 40).round()], dim=2)
    left, sinks = 14, 3
    qc, kc, vc, pc = (t.cuda() for t in (q, k, v, pos))
    qr, kr = A.rotary_axes(qc, pc, sec), A.rotary_axes(kc, pc, sec)
    ref = R.attention(qr.cpu(), kr.cpu(), v, R.seen(B, T, T, left, 0, sinks))["out"]
    cache_k = torch.full((B, cap, Hkv, D), math.nan, dtype=dtype, device="cuda")
    cache_v = torch.full_like(cache_k, math.inf)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = A.window_attention(qr, kr, vc, left, 0, sinks, q_lens=n, k_lens=n)
    rows = torch.arange(B, device="cuda")
    for b, length in enumerate(lens):
        R.check("prompt", out[b, :length], ref[0][b, :length], ref[1][b, :length])
        assert not out[b, length:].any()
        cache_k[b, :length], cache_v[b, :length] = kr[b, :length], vc[b, :length]
    for _ in range(new):
        at = n.long()
        q1, k1 = (A.rotary_axes(t[rows, at][:, None], pc[rows, at][:, None], sec) for t in (qc, kc))
        cache_k[rows, at], cache_v[rows, at] = k1[:, 0], vc[rows, at]
        n = n + 1
        out = A.window_attention(q1, cache_k, cache_v, left, 0, sinks, k_lens=n)
        for b in range(B):
            R.check("token", out[b, 0], ref[0][b, int(at[b])], ref[1][b, int(at[b])])


def test_two_kernels_give_the_same_answer():
    """The few-row kernel (one sequence) and the many-row kernel (that sequence among many) agree within their bounds' sum."""
    A = _att()
    q, k, v = (_normal(1, 200, 8, 64, dtype=torch.bfloat16, seed=n) for n in range(3))
    ref = R.attention(q, k, v, R.seen(1, 200, 200, 33, 5, 2))["out"]
    few = A.window_attention(q.cuda(), k.cuda(), v.cuda(), 33, 5, 2)
    many = A.window_attention(*(t.cuda().expand(64, -1, -1, -1) for t in (q, k, v)), 33, 5, 2)
    for t in (few, many[:1], many[63:]):
        R.check("out", t, *ref)
    assert torch.equal(many[0], many[63])


# ---- ends of the ranges -------------------------------------------------------------------------------------------------------------------
def test_lengths_are_clamped_and_may_be_64_bit():
    A = _att()
    B, T, H, D = 4, 50, 2, 32
    q, k, v, do = (_normal(B, T, H, D, seed=n) for n in range(4))
    given = [torch.tensor([-5, 50, 51, 1 << 40]), torch.tensor([7, 0, 1 << 33, 20])]
    ref = R.attention(q, k, v, R.seen(B, T, T, 9, 2, 1, given[0].clamp(0, T), given[1].clamp(0, T)), dout=do)
    for cast in (lambda t: t, lambda t: t.clamp(-5, 1000).to(torch.int32)):
        x = [t.cuda().requires_grad_() for t in (q, k, v)]
        out, lse = A.window_attention(*x, 9, 2, 1, *(cast(t).cuda() for t in given), return_lse=True)
        R.check("out", out, *ref["out"])
        R.check("lse", lse, *ref["lse"])
        for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, x, do.cuda())):
            R.check(n, g, *ref[n])


def test_nothing_to_do():
    A = _att()
    for B, Tq, Tk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v = (torch.randn(B, T, 2, 32, device="cuda", requires_grad=True) for T in (Tq, Tk, Tk))
        out, lse = A.window_attention(q, k, v, 1, 1, 1, return_lse=True)
        assert out.shape == (B, Tq, 2, 32) and lse.shape == (B, 2, Tq) and not out.any() and (lse == -math.inf).all()
        out.sum().backward()
        assert not any(t.grad.any() for t in (q, k, v))


def test_huge_limits_scales_and_scores():
    A = _att()
    q, k, v = (_normal(2, 40, 2, 32, seed=n) for n in range(3))
    ref = R.attention(q, k, v, R.seen(2, 40, 40, None, None, 0))["out"]
    for left, right, sinks in ((1 << 40, 1 << 40, 0), (0, 0, 1 << 40), (39, 39, 0), (None, 39, 1 << 50)):
        want = ref if right != 0 else R.attention(q, k, v, R.seen(2, 40, 40, None, 0, 0))["out"]
        R.check(f"{left} {right} {sinks}", A.window_attention(q.cuda(), k.cuda(), v.cuda(), left, right, sinks), *want)
    for scale in (1e-6, 30.0):
        want = R.attention(q, k, v, R.seen(2, 40, 40, 5, 0, 1), scale=scale)
        out, lse = A.window_attention(q.cuda(), k.cuda(), v.cuda(), 5, 0, 1, scale=scale, return_lse=True)
        R.check("out", out, *want["out"])
        R.check("lse", lse, *want["lse"])
    big = A.window_attention(q.cuda() * 1e15, k.cuda() * 1e15, v.cuda(), 5, 0, 1)     # scores of 1e30: one key takes all
    assert torch.isfinite(big).all()


def test_offsets_beyond_32_bits():
    """A cache of 2^31 + elements (bf16, 4.4 GB): the last keys, and the sinks at the other end."""
    A = _att()
    T, H, D = (1 << 25) + 200, 1, 64
    cache = torch.empty((1, T, H, D), dtype=torch.bfloat16, device="cuda")
    tail = _normal(1, 100, H, D, dtype=torch.bfloat16, seed=1)
    first = _normal(1, 3, H, D, dtype=torch.bfloat16, seed=2)
    cache[:, T - 100:] = tail.cuda()
    cache[:, :3] = first.cuda()
    q = _normal(1, 2, H, D, dtype=torch.bfloat16, seed=3)
    ref = R.attention(q, torch.cat([first, tail], 1), torch.cat([first, tail], 1), R.seen(1, 2, 103, 90, 0, 3))["out"]
    R.check("out", A.window_attention(q.cuda(), cache, cache, 90, 0, 3), *ref)
    do = _normal(1, 2, H, D, dtype=torch.bfloat16, seed=4).cuda()
    x = cache[:, T - 4000:].requires_grad_()
    out = A.window_attention(q.cuda(), x, x, 90, 0, 0)
    torch.autograd.grad(out, x, do)
    pos = torch.full((1, T - 1000, 1), 3.0, device="cuda").as_strided((1, T, 1), (0, 0, 0))
    y = A.rotary_axes(cache, pos, (32,), out=cache)
    want = R.rotary(tail, torch.full((1, 100, 1), 3.0), (32,), (10000.0,), "halves")
    R.check("rotary", y[:, T - 100:], want, tail.double().abs().amax() * 2 * (2.0 ** -21 + 1.01 * 2.0 ** -8))


def test_rotary_of_far_positions():
    """2^24 - 1 is the last whole number fp32 holds next to its neighbours; a 32-bit product would be off by a radian there."""
    A = _att()
    x = _normal(1, 3, 2, 32)
    pos = torch.tensor([[[2.0 ** 24 - 1], [-(2.0 ** 23) - 0.5], [1e7 + 1]]])
    got = A.rotary_axes(x.cuda(), pos.cuda(), (16,))
    R.check("out", got, R.rotary(x, pos, (16,), (10000.0,), "halves"), 2.0 ** -19 * x.abs().max().double())
    for bad in (math.nan, math.inf):
        y = A.rotary_axes(x.cuda(), torch.tensor([[[1.0], [bad], [2.0]]], device="cuda"), (8,))
        assert torch.isnan(y[:, 1, :, :16]).all() and torch.equal(y[:, 1, :, 16:].cpu(), x[:, 1, :, 16:]) and torch.isfinite(y[:, (0, 2)]).all()


# ---- streams, graphs, refusals ------------------------------------------------------------------------------------------------------------
def test_tensors_of_another_stream():
    A = _att()
    q, k, v = (_normal(2, 300, 4, 64, seed=n) for n in range(3))
    want = A.window_attention(q.cuda(), k.cuda(), v.cuda(), 30, 0, 2)
    turned = A.rotary_axes(q.cuda(), torch.arange(300.0).cuda()[:, None], (32,))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)                                    # the inputs are late on their stream
            x = [t.cuda(non_blocking=True) for t in (q, k, v)]
            got = A.window_attention(*x, 30, 0, 2)
            rot = A.rotary_axes(x[0], torch.arange(300.0).cuda()[:, None], (32,))
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(rot, turned)


def test_captured_graphs_replayed_between_eager_work():
    """Forward and backward of several forms in two graphs, replayed in turn and at the same time on two streams, with eager calls between."""
    A = _att()
    forms = [(1, 4, 2000, 8, 2, 64, None, 0, 4, torch.bfloat16), (2, 300, 300, 4, 4, 64, 40, 0, 5, torch.float32), (4, 200, 200, 8, 2, 128, 60, 10, 3, torch.bfloat16)]
    sets, graphs = [], []
    pool = torch.cuda.Stream()

    def once(x, do, pos, form):
        qr = A.rotary_axes(x[0], pos, (form[5] // 2,))
        out, lse = A.window_attention(qr, x[1], x[2], form[6], form[7], form[8], return_lse=True)
        return (out, lse) + torch.autograd.grad(out, x, do)
    for n, form in enumerate(forms):
        B, Tq, Tk, Hq, Hkv, D, _, _, _, dt = form
        x = [_normal(B, T, H, D, dtype=dt, seed=n + m).cuda() for m, (T, H) in enumerate(((Tq, Hq), (Tk, Hkv), (Tk, Hkv)))]
        sets.append((x, _normal(B, Tq, Hq, D, dtype=dt, seed=9).cuda(), torch.arange(float(Tq)).cuda()[:, None]))
    for half in range(2):
        with torch.cuda.stream(pool):
            for (x, do, pos), form in zip(sets, forms):
                once([t.detach().requires_grad_() for t in x], do, pos, form)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=pool):
            outs = [once([t.detach().requires_grad_() for t in x], do, pos, form) for (x, do, pos), form in zip(sets, forms)]
        graphs.append((g, outs))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for n, (x, do, pos) in enumerate(sets):
            for t in x:
                t.copy_(_normal(*t.shape, dtype=t.dtype, seed=100 * turn + n).cuda())
        want = [once([t.detach().requires_grad_() for t in x], do, pos, form) for (x, do, pos), form in zip(sets, forms)]
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, outs in graphs:
            for form, a, b in zip(forms, outs, want):
                assert all(torch.equal(p, q) for p, q in zip(a, b)), (turn, form)
        _ = torch.randn(1 << 20, device="cuda").sum().item()
    del graphs, g, outs
    torch.cuda.synchronize()


def test_refusals_on_the_device():
    from trajectorydiffusion_amd._lib import TdxError
    A = _att()
    t = torch.randn(2, 4, 2, 64, device="cuda")
    pos = torch.zeros(2, 4, 1, device="cuda")
    for f in (lambda: A.window_attention(t, t.cpu(), t), lambda: A.window_attention(t, t, t, k_lens=torch.tensor([4, 4])),
              lambda: A.window_attention(t, t, t, q_lens=torch.tensor([4.0, 4.0], device="cuda")), lambda: A.window_attention(t, t, t, left=True),
              lambda: A.rotary_axes(t, pos.cpu(), (32,)), lambda: A.rotary_axes(t, pos.clone().requires_grad_(), (32,)),
              lambda: A.rotary_axes(t, pos, (32,), out=torch.empty(2, 4, 2, 64, device="cuda", dtype=torch.bfloat16)),
              lambda: A.rotary_axes(t, pos, (32,), out=torch.empty(1, 4, 2, 64, device="cuda").expand(2, 4, 2, 64)),
              lambda: A.rotary_axes(t.clone().requires_grad_(), pos, (32,), out=torch.empty_like(t))):
        with pytest.raises(TdxError):
            f()
    A.window_attention(t, t, t, left=1)                                      # (a form that was taken does not open the door to one that is not)
    with pytest.raises(TdxError):
        A.window_attention(t, t, t, left=True)
    x = t.clone().requires_grad_()
    for out in (A.window_attention(x, t, t, 1, 1), A.rotary_axes(x, pos, (32,))):
        with pytest.raises(TdxError, match="second derivatives"):
            torch.autograd.grad(out.sum(), x, create_graph=True)
    y = t.clone().requires_grad_()
    z = y * 1
    out = A.window_attention(z, t, t, 1, 1)
    with torch.no_grad():
        z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_gradients_of_one_tensor_in_three_places_and_of_broadcasts():
    A = _att()
    x = _normal(2, 30, 2, 32)
    do = _normal(2, 30, 2, 32, seed=1)
    ref = R.attention(x, x, x, R.seen(2, 30, 30, 6, 6, 2), dout=do)
    t = x.cuda().requires_grad_()
    A.window_attention(t, t, t, 6, 6, 2).backward(do.cuda())
    R.check("sum of three", t.grad, sum(ref[n][0] for n in ("dq", "dk", "dv")), sum(ref[n][1] for n in ("dq", "dk", "dv")) + 2.0 ** -22 * ref["dv"][0].abs().max())
    one = _normal(1, 30, 2, 32, seed=2)
    kv = one.cuda().requires_grad_()
    ref = R.attention(x, one.expand(2, -1, -1, -1), one.expand(2, -1, -1, -1), R.seen(2, 30, 30, 6, 6, 2), dout=torch.ones_like(x))
    A.window_attention(x.cuda(), kv.expand(2, -1, -1, -1), kv.expand(2, -1, -1, -1), 6, 6, 2).sum().backward()
    R.check("broadcast", kv.grad, (ref["dk"][0] + ref["dv"][0]).sum(0, keepdim=True), (ref["dk"][1] + ref["dv"][1]).sum(0, keepdim=True) + 2.0 ** -21 * ref["dv"][0].abs().max())


# ---- inside the model ---------------------------------------------------------------------------------------------------------------------
SCHED, T_MODEL = [128, 128, 128], 20
OPTIONS = [dict(attn_heads=4, attn_window=11, attn_sinks=5, attn_rotary=500.0), dict(attn_heads=1, attn_window=40), dict(attn_heads=2, attn_window=0, attn_sinks=70)]


def _attn_block(heads, window, sinks, rotary):
    from oracle.trajunet_oracle import resnet_block

    def block(sd, p, x, emb, groups=32):
        x = resnet_block(sd, p + "res1.", x, emb, groups)
        B, Cn, L = x.shape
        h = F.group_norm(x, groups, sd[p + "qkv_getter.0.weight"], sd[p + "qkv_getter.0.bias"], eps=1e-6)
        qkv = F.conv1d(h, sd[p + "qkv_getter.1.weight"], sd[p + "qkv_getter.1.bias"]).transpose(1, 2)
        q, k, v = (t.reshape(B, L, heads, Cn // heads) for t in torch.split(qkv, Cn, dim=2))
        if rotary is not None:
            n = Cn // heads // 2
            ang = torch.arange(L, dtype=torch.float64)[:, None] * rotary ** (-torch.arange(n, dtype=torch.float64) / n)
            c, s = ang.cos().to(x.dtype)[:, None], ang.sin().to(x.dtype)[:, None]
            q, k = (torch.cat([t[..., :n] * c - t[..., n:] * s, t[..., :n] * s + t[..., n:] * c], dim=-1) for t in (q, k))
        i, j = torch.arange(L)[:, None], torch.arange(L)[None, :]
        ok = (j <= i + window) & ((j >= i - window) | (j < sinks))
        sc = (q.permute(0, 2, 1, 3) @ k.permute(0, 2, 3, 1)) * (Cn // heads) ** -0.5
        o = torch.softmax(sc.masked_fill(~ok, -math.inf), dim=-1) @ v.permute(0, 2, 1, 3)
        o = o.transpose(1, 2).reshape(B, L, Cn).transpose(1, 2)
        x = x + F.conv1d(o, sd[p + "project_out.weight"], sd[p + "project_out.bias"])
        return resnet_block(sd, p + "res2.", x, emb, groups)
    return block


def _model(seed, **options):
    from trajectorydiffusion_amd import TrajUNet
    torch.manual_seed(seed)
    return TrajUNet(SCHED, diffusion_steps=T_MODEL, res_blocks=2, **options)


def _oracle(monkeypatch, sd, x, t, cat, num, o):
    import oracle.trajunet_oracle as O
    monkeypatch.setattr(O, "attn_block", _attn_block(o["attn_heads"], o["attn_window"], o.get("attn_sinks", 0), o.get("attn_rotary")))
    table = O.positional_table
    monkeypatch.setattr(O, "positional_table", lambda n: table(n).to(x.dtype))
    return O.trajunet_forward(sd, x, t, cat, num, SCHED, T_MODEL)


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("L", [4, 150, 1201])      # 1, 38 and 301 tokens in the middle: 64 is the reference form's limit
def test_model_forward(monkeypatch, options, L):
    from _synth import synth_inputs
    m = _model(L, **options).eval()
    sd = {k: v.detach().clone() for k, v in m.state_dict().items()}
    x, t, cat, num = synth_inputs(2, L, T_MODEL, seed=1)
    with torch.no_grad():
        want = _oracle(monkeypatch, sd, x, t, cat, num, options)
    m = m.cuda()
    got = m(x.cuda(), t.cuda(), cat.cuda(), num.cuda()).cpu()
    assert float((got - want).abs().max() / want.abs().max()) < 1e-4               # the fp32 tolerance of the model tests
    # bf16 rounds every activation of some 30 layers: what it is off by in the end has no bound worth asserting (its attention launches have
    # one: the next test)
    assert torch.isfinite(m.set_compute_dtype(torch.bfloat16)(x.cuda(), t.cuda(), cat.cuda(), num.cuda())).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("heads,window,sinks,rotary", [(4, 11, 5, 500.0), (1, 40, 0, None), (2, 0, 70, 50.0)])
@pytest.mark.parametrize("B,L", [(2, 1), (2, 301), (40, 150)])
def test_attention_launches_of_a_program(B, L, heads, window, sinks, rotary, dtype):
    """What AttnBlock records between its projections: rotation in place and attention on slices of qkv rows."""
    from trajectorydiffusion_amd import engine
    Cn = 128
    D = Cn // heads
    rows = _normal(B, L, 3 * Cn, dtype=dtype, seed=L)
    pg = engine.Program(torch.device("cuda"), dtype)
    dev, out = rows.cuda(), torch.full((B, L, Cn), math.nan, dtype=dtype, device="cuda")
    engine.WindowSpec.check(Cn, heads, window, sinks, rotary).emit(pg, "attention", dev, out, None, B, L, Cn)
    pg.run()
    q, k, v = (t.reshape(B, L, heads, D) for t in rows.split(Cn, dim=2))
    if rotary is not None:
        pos = torch.arange(float(L)).reshape(1, L, 1).expand(B, L, 1)
        got = dev.cpu().split(Cn, dim=2)
        for t, w in ((q, got[0]), (k, got[1])):
            both = t.double().abs()
            both = torch.cat([both[..., :D // 2] + both[..., D // 2:]] * 2, dim=3)
            R.check("rotated", w.reshape(B, L, heads, D), R.rotary(t, pos, (D // 2,), (rotary,), "halves"), both * (2.0 ** -21 + 1.01 * R.HALF[dtype]))
        q, k = (t.reshape(B, L, heads, D) for t in got[:2])
    assert torch.equal(dev[..., 2 * Cn:].cpu(), rows[..., 2 * Cn:])
    ref = R.attention(q, k, v, R.seen(B, L, L, window, window, sinks))["out"]
    R.check("out", out.reshape(B, L, heads, D), *ref)


def test_a_window_over_all_tokens_is_the_reference_attention():
    from _synth import synth_inputs
    a, b = _model(3).eval().cuda(), _model(3, attn_window=10 ** 6).eval().cuda()
    x = [t.cuda() for t in synth_inputs(3, 200, T_MODEL, seed=2)]
    ya, yb = a(*x), b(*x)
    assert float((ya - yb).abs().max() / ya.abs().max()) < 2e-5


def test_attn_block_alone_and_sampling_with_a_graph(monkeypatch):
    from _synth import synth_inputs
    from trajectorydiffusion_amd import AttnBlock, DiffusionManager
    torch.manual_seed(5)
    blk = AttnBlock(128, 32, heads=4, window=9, sinks=2, rotary=100.0).eval()
    sd = {k: v.detach().clone() for k, v in blk.state_dict().items()}
    x, emb = _normal(2, 128, 130, seed=1), _normal(2, 256, 1, seed=2)
    with torch.no_grad():
        want = _attn_block(4, 9, 2, 100.0)(sd, "", x, emb)
    got = blk.cuda()(x.cuda(), emb.cuda()).cpu()
    assert float((got - want).abs().max() / want.abs().max()) < 1e-4
    m = _model(6, **OPTIONS[0]).eval().cuda()
    x, t, cat, num = (v.cuda() for v in synth_inputs(4, 1201, T_MODEL, seed=3))
    dm = DiffusionManager(1e-4, 0.05, T_MODEL, device="cuda")
    dm.seed = 11
    a = dm.diffusionBackward(x, cat, num, m, max_t=6, use_graph=True)
    b = dm.diffusionBackward(x, cat, num, m, max_t=6, use_graph=False)
    again = dm.diffusionBackward(x, cat, num, m, max_t=6, use_graph=True)
    assert torch.isfinite(a).all() and torch.equal(a, b) and torch.equal(a, again)
    dm.release_samplers()


@pytest.mark.parametrize("options", OPTIONS)
def test_model_training_step_gradients(monkeypatch, options):
    from _synth import synth_inputs, synth_noise
    from trajectorydiffusion_amd.training import TrainStep
    B, L = 2, 1201
    m = _model(7, **options)
    sd = {k: v.detach().double().requires_grad_() for k, v in m.state_dict().items()}
    x, t, cat, num = synth_inputs(B, L, T_MODEL, seed=4)
    eps = synth_noise(0, x.shape, seed=4)
    pred = _oracle(monkeypatch, sd, x.double(), t, cat, num.double(), options)
    loss = F.mse_loss(pred, eps.double())
    loss.backward()
    ts = TrainStep(m.cuda(), B, L, torch.device("cuda"), dropout=0.0)
    got = ts.forward_backward(x.cuda(), t.cuda(), cat.cuda(), num.cuda(), eps.cuda())
    assert abs(float(got) - float(loss)) < 2e-5 * float(loss)
    grads = {n: g.clone() for n, g in ts.named_gradients().items()}
    assert sorted(grads) == sorted(n for n, v in sd.items() if v.grad is not None)
    for n, g in grads.items():
        want = sd[n].grad
        err = float((g.cpu().double() - want).abs().max() / want.abs().max().clamp_min(1e-12))
        assert err < 1e-4, (n, err)                                              # GRAD_TOL of the training tests
    ts.forward_backward(x.cuda(), t.cuda(), cat.cuda(), num.cuda(), eps.cuda())
    assert all(torch.equal(grads[n], g) for n, g in ts.named_gradients().items())
    # behind torch.autograd, as a training loop calls it
    m.train()
    for blk in m.modules():
        if hasattr(blk, "dropout"):
            blk.dropout = 0.0
    out = m(x.cuda(), t.cuda(), cat.cuda(), num.cuda())
    F.mse_loss(out, eps.cuda()).backward()
    for n, p in m.named_parameters():
        if n in grads:
            assert float((p.grad - grads[n]).abs().max()) <= 1e-5 * float(grads[n].abs().max()) + 1e-12, n
