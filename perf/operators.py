"""The sequence operators that are timed: rotary positions with several axes, and attention with a window and visible first tokens.

Where `own` is false, run() computes them in their plain form, from elementary torch operations in 32 bits (angles in 64);
where it is true, run() makes the calls a user of trajectorydiffusion_amd makes.  exact() is the definition in 64 bits.

Notation: a query row i of a sequence with q_len queries and k_len keys stands at position p = i + k_len - q_len and sees key j iff
j < k_len, j <= p + right and (j >= p - left or j < sinks).  left / right = -1 in a case: no limit on that side.
"""
import math

import torch

own = False

FAR = 1 << 30            # a limit that no position reaches
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _rotary(name, dtype, B, T, H, D, axes, layout, train):
    case = {"op": "rotary", "dtype": dtype, "B": B, "T": T, "H": H, "D": D, "axes": axes, "layout": layout, "train": train}
    return {"name": name, **case} if name else case


def _attend(name, dtype, B, Tq, Tk, Hq, Hkv, D, left, right, sinks, ragged, train):
    case = {"op": "attend", "dtype": dtype, "B": B, "Tq": Tq, "Tk": Tk, "Hq": Hq, "Hkv": Hkv, "D": D, "left": left, "right": right, "sinks": sinks,
            "ragged": ragged, "train": train}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one new point for each of 64 tracks: the q and k heads of a serving step, rotated by its index alone
        _rotary("rotary, one point a track", "bf16", 64, 1, 10, 128, 1, "halves", False),
        # the q and k heads of long prompts, rotated by (time, longitude cell, latitude cell)
        _rotary("rotary, long prompts", "bf16", 8, 4096, 20, 128, 3, "halves", False),
        # a training step's rotation, forward and backward, in the framework's training type, head width not a power of two
        _rotary("rotary, training", "fp32", 32, 1250, 8, 96, 3, "pairs", True),
        # TrajUNet's middle block at 200 points: 13 tokens, 8 heads of 128
        _attend("13 tokens", "fp32", 64, 13, 13, 8, 8, 128, -1, -1, 0, False, False),
        # causal prompts with grouped key heads
        _attend("causal prompts", "bf16", 2, 4096, 4096, 16, 4, 128, 1023, 0, 4, False, False),
        # one long track, looked at from both sides, 16 anchor tokens
        _attend("one long track", "bf16", 1, 16384, 16384, 8, 8, 64, 512, 512, 16, False, False),
        # tracks of 20 000 points behind four stride-2 stages, padded to one length, 7 condition tokens in front of them
        _attend("padded tracks", "fp32", 8, 1250, 1250, 8, 8, 64, 128, 128, 7, True, False),
        # training steps: the causal prompts above, tracks of 10 000 points in the framework's training type, one long track
        _attend("causal prompts, training", "bf16", 2, 4096, 4096, 16, 4, 128, 1023, 0, 4, False, True),
        _attend("padded tracks, training", "fp32", 16, 625, 625, 8, 8, 128, 64, 64, 7, True, True),
        _attend("one long track, training", "bf16", 1, 8192, 8192, 8, 8, 64, 256, 256, 16, False, True),
        # single new points over caches of different lengths, and one stream alone, where latency counts
        _attend("64 streams, one point", "bf16", 64, 1, 8192, 16, 4, 128, 4095, 0, 4, True, False),
        _attend("one stream, one point", "bf16", 1, 1, 32768, 16, 4, 128, 16383, 0, 4, False, False),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    what = rng.choice(["rotary", "rotary", "attend", "attend", "attend", "train", "train", "token", "token"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    D = rng.choice([32, 40, 48, 64, 64, 80, 96, 128, 128])
    if what == "rotary":
        B, T, H = _spread(rng, 1, 64), _spread(rng, 1, 8192), _spread(rng, 1, 40)
        T = max(1, min(T, 80_000_000 // (B * H * D)))
        return _rotary(None, dtype, B, T, H, D, rng.choice([1, 2, 3]), rng.choice(["halves", "pairs"]), rng.random() < 0.4)
    Hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4, 8])
    Hq = Hkv * group
    sinks = rng.choice([0, 1, 4, 7, 16, 64, 100])
    ragged = rng.random() < 0.5
    if what == "token":
        B, Tk, Tq = _spread(rng, 1, 64), _spread(rng, 1, 32768), rng.choice([1, 1, 1, 2, 4])
        Tk = max(Tq, min(Tk, 260_000_000 // (B * Hkv * D)))
        return _attend(None, dtype, B, Tq, Tk, Hq, Hkv, D, rng.choice([-1, _spread(rng, 1, 16384)]), 0, sinks, ragged, False)
    most = 2_000_000_000 if what == "attend" else 500_000_000   # scores of the plain form, which holds them all
    T = _spread(rng, 16, 8192)
    Hkv = max(1, min(Hkv, most // (T * T * group)))
    Hq = Hkv * group
    B = _spread(rng, 1, max(1, min(64, most // (T * T * Hq))))
    left = rng.choice([-1, _spread(rng, 1, 2048), _spread(rng, 1, 2048), _spread(rng, 1, 2048)])
    right = rng.choice([0, 0, -1, left, _spread(rng, 1, 512)])
    return _attend(None, dtype, B, T, T, Hq, Hkv, D, left, right, sinks, ragged, what == "train")


def _sections(case):
    """Pairs of channels for each axis: the first axis (time) has what the others leave."""
    pairs, n = case["D"] // 2, case["axes"]
    rest = [pairs // (n + 1)] * (n - 1)
    return [pairs - sum(rest)] + rest


def _lengths(case):
    """Lengths of the sequences of a ragged case, before prepare() puts them in another order: from the whole length down to a third."""
    B, T = case["B"], case["Tk"]
    return [max(min(case["Tq"], T), T - (2 * T * b) // (3 * B)) for b in range(B)] if case["ragged"] else [T] * B


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    B = case["B"]
    if case["op"] == "rotary":
        T, H, D, axes = case["T"], case["H"], case["D"], case["axes"]
        state = {"x": normal(B, T, H, D), "sections": _sections(case), "layout": case["layout"], "train": case["train"]}
        # minutes since the track began (or a point's index), and cells of the 256 x 256 grid
        first = torch.randint(0, 20000, (B, 1), generator=gen, device="cuda")
        time = (first + torch.arange(T, device="cuda")).float()
        cells = [torch.randint(0, 256, (B, T), generator=gen, device="cuda").float() for _ in range(axes - 1)]
        state["pos"] = torch.stack([time] + cells, dim=2)
        if case["train"]:
            state["dout"] = normal(B, T, H, D)
        return state
    Tq, Tk, Hq, Hkv, D = case["Tq"], case["Tk"], case["Hq"], case["Hkv"], case["D"]
    state = {"q": normal(B, Tq, Hq, D), "k": normal(B, Tk, Hkv, D), "v": normal(B, Tk, Hkv, D), "train": case["train"], "sinks": case["sinks"],
             "left": None if case["left"] < 0 else case["left"], "right": None if case["right"] < 0 else case["right"], "q_lens": None, "k_lens": None}
    if case["ragged"]:
        order = torch.randperm(B, generator=gen, device="cuda")
        state["k_lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
        if Tq == Tk:
            state["q_lens"] = state["k_lens"]
    if case["train"]:
        state["dout"] = normal(B, Tq, Hq, D)
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------------------
def _plain_rotary(x, pos, sections, layout):
    D = x.shape[-1]
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=x.device)
    rate = torch.tensor([10000.0 ** (-i / n) for n in sections for i in range(n)], device=x.device, dtype=torch.float64)
    angle = pos.double()[:, :, axis] * rate                      # (B, T, D / 2): 32 bits lose the angles of far positions
    c, s = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    xf = x.float()
    if layout == "halves":
        a, b = xf[..., :D // 2], xf[..., D // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], dim=-1).to(x.dtype)
    a, b = xf[..., 0::2], xf[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], dim=-1).reshape(x.shape).to(x.dtype)


def _plain_attend(q, k, v, left, right, sinks, q_lens, k_lens):
    """(out (B, Tq, Hq, D), log of the sum of exponentials (B, Hq, Tq) in 32 bits); rows that see nothing: 0 and -inf."""
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    ql = torch.full((B,), Tq, device=q.device) if q_lens is None else q_lens.long()
    kl = torch.full((B,), Tk, device=q.device) if k_lens is None else k_lens.long()
    i, j = torch.arange(Tq, device=q.device)[None, :, None], torch.arange(Tk, device=q.device)[None, None, :]
    ql, kl = ql[:, None, None], kl[:, None, None]
    p = i + (kl - ql)
    seen = (i < ql) & (j < kl) & (j <= p + (FAR if right is None else right)) & ((j >= p - (FAR if left is None else left)) | (j < sinks))
    seen = seen[:, None, None]                                    # (B, 1, 1, Tq, Tk)
    qf = q.float().reshape(B, Tq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    kf, vf = k.float().permute(0, 2, 3, 1)[:, :, None], v.float().permute(0, 2, 1, 3)[:, :, None]
    score = (qf @ kf) * (1.0 / math.sqrt(D))
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top).detach()
    e = (score - top).exp()
    total = e.sum(-1, keepdim=True)
    out = (e / torch.where(total == 0, torch.ones_like(total), total)) @ vf
    out = out.permute(0, 3, 1, 2, 4).reshape(B, Tq, Hq, D).to(q.dtype)
    return out, (top + total.log()).reshape(B, Hq, Tq)


# ---- one pass ---------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        from trajectorydiffusion_amd.attention import rotary_axes, window_attention
    if "x" in state:
        def rotate(x):
            if own:
                return rotary_axes(x, state["pos"], state["sections"], layout=state["layout"])
            return _plain_rotary(x, state["pos"], state["sections"], state["layout"])
        if not state["train"]:
            return {"out": rotate(state["x"])}
        x = state["x"].detach().requires_grad_()
        out = rotate(x)
        return {"out": out.detach(), "dx": torch.autograd.grad(out, x, state["dout"])[0]}

    def attend(q, k, v):
        if own:
            return window_attention(q, k, v, left=state["left"], right=state["right"], sinks=state["sinks"], q_lens=state["q_lens"],
                                    k_lens=state["k_lens"], return_lse=True)
        return _plain_attend(q, k, v, state["left"], state["right"], state["sinks"], state["q_lens"], state["k_lens"])
    if not state["train"]:
        out, lse = attend(state["q"], state["k"], state["v"])
        return {"out": out, "lse": lse}
    q, k, v = (state[n].detach().requires_grad_() for n in "qkv")
    out, lse = attend(q, k, v)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["dout"])
    return {"out": out.detach(), "lse": lse.detach(), "dq": dq, "dk": dk, "dv": dv}


# ---- work -------------------------------------------------------------------------------------------------------------------------
def _pairs(case):
    """(pairs (query row, key) that see each other, keys that some row sees), summed over the sequences, for one head."""
    left, right = (FAR if case[n] < 0 else case[n] for n in ("left", "right"))
    pairs = keys = 0
    for length in _lengths(case):
        rows = length if case["Tq"] == case["Tk"] else case["Tq"]
        p = torch.arange(rows) + (length - rows)
        hi = (p + right).clamp(max=length - 1)                     # the last key of each row, the first of its window, its sinks before that
        lo = (p - left).clamp(min=0)
        first = torch.minimum(torch.minimum(lo, hi + 1), torch.full_like(lo, case["sinks"])).clamp(min=0)
        pairs += int(((hi - lo + 1).clamp(min=0) + first).sum())
        if rows:
            keys += int(hi[-1]) + 1 - int(lo[0]) + min(case["sinks"], int(lo[0]))
    return pairs, keys


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    passes = 2 if case["train"] else 1
    if case["op"] == "rotary":
        n = case["B"] * case["T"] * case["H"] * case["D"]
        return {"bytes": passes * 2 * n * size + case["B"] * case["T"] * case["axes"] * 4, "flops": passes * 3 * n}
    pairs, keys = _pairs(case)
    rows = sum(n if case["Tq"] == case["Tk"] else case["Tq"] for n in _lengths(case))
    wide_q, wide_k = case["Hq"] * case["D"] * size, case["Hkv"] * case["D"] * size
    got = {"bytes": 2 * rows * wide_q + 2 * keys * wide_k + rows * case["Hq"] * 4, "flops": 4 * pairs * case["Hq"] * case["D"]}
    if case["train"]:                                              # reads q, k, v, out and its gradient, writes three gradients; five products
        got["bytes"] += 4 * rows * wide_q + 4 * keys * wide_k
        got["flops"] += 10 * pairs * case["Hq"] * case["D"]
    return got


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------
def _exact_rotation(x, pos, sections, layout, sign):
    """Each pair of channels as a complex number, times exp(sign * i * angle)."""
    B, T, H, D = x.shape
    phase, at = [], 0
    for a, n in enumerate(sections):
        rate = torch.exp(torch.arange(n, dtype=torch.float64, device=x.device) * (-math.log(10000.0) / n))
        phase.append(pos[:, :, a].double().unsqueeze(-1) * rate)
        at += n
    turn = torch.polar(torch.ones((B, T, 1, at), dtype=torch.float64, device=x.device), sign * torch.cat(phase, dim=-1).unsqueeze(2))
    z = x.double()
    z = z.view(B, T, H, 2, at).transpose(3, 4) if layout == "halves" else z.view(B, T, H, at, 2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    return (z.transpose(3, 4) if layout == "halves" else z).reshape(B, T, H, D)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        got = {"out": _exact_rotation(s["x"], s["pos"], s["sections"], s["layout"], 1.0)}
        if case["train"]:
            got["dx"] = _exact_rotation(s["dout"], s["pos"], s["sections"], s["layout"], -1.0)
        return got
    B, Tq, Hq, D = s["q"].shape
    Tk, Hkv = s["k"].shape[1], s["k"].shape[2]
    group, scale = Hq // Hkv, D ** -0.5
    dev = s["q"].device
    left, right = FAR if s["left"] is None else s["left"], FAR if s["right"] is None else s["right"]
    got = {"out": torch.zeros((B, Tq, Hq, D), dtype=torch.float64, device=dev), "lse": torch.full((B, Hq, Tq), -math.inf, dtype=torch.float64, device=dev)}
    if case["train"]:
        got.update({n: torch.zeros(s[n[1]].shape, dtype=torch.float64, device=dev) for n in ("dq", "dk", "dv")})
    for b in range(B):
        kn = Tk if s["k_lens"] is None else int(s["k_lens"][b])
        qn = Tq if s["q_lens"] is None else int(s["q_lens"][b])
        for h in range(Hkv):
            K, V = s["k"][b, :kn, h].double(), s["v"][b, :kn, h].double()
            key = torch.arange(kn, device=dev)
            step = max(1, 60_000_000 // max(1, kn * group))
            for r0 in range(0, qn, step):
                r1 = min(qn, r0 + step)
                heads = slice(h * group, (h + 1) * group)
                Q = s["q"][b, r0:r1, heads].double()               # (rows, group, D)
                place = torch.arange(r0, r1, device=dev) + (kn - qn)
                away = key[None, :] - place[:, None]               # how far each key is ahead of the row
                hidden = (away > right) | ((away < -left) & (key[None, :] >= s["sinks"]))
                score = torch.einsum("rgd,kd->rgk", Q, K) * scale
                score[hidden[:, None].expand_as(score)] = -math.inf
                lse = torch.logsumexp(score, dim=-1)               # -inf where nothing is seen
                prob = torch.exp(score - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
                out = torch.einsum("rgk,kd->rgd", prob, V)
                got["out"][b, r0:r1, heads] = out
                got["lse"][b, heads, r0:r1] = lse.transpose(0, 1)
                if case["train"]:
                    dO = s["dout"][b, r0:r1, heads].double()
                    dP = torch.einsum("rgd,kd->rgk", dO, V)
                    dS = prob * (dP - (dO * out).sum(-1, keepdim=True)) * scale
                    got["dv"][b, :kn, h] += torch.einsum("rgk,rgd->kd", prob, dO)
                    got["dk"][b, :kn, h] += torch.einsum("rgk,rgd->kd", dS, Q)
                    got["dq"][b, r0:r1, heads] = torch.einsum("rgk,kd->rgd", dS, K)
    return got
