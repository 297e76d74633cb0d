"""Plain statements of the sequence operators in 64 bits on the CPU, with bounds on what the kernels' arithmetic may be off.

u is half a step of the storage type (bf16 2^-8, fp32 2^-24), v = 2^-24 half a step of the 32-bit sums.  With a = |q| |k|^T scale, n keys and D
channels, a score is off by at most (D + 4) v a (sum, scale, the factor log2 e, the subtraction of the maximum or of the log-sum), the
exponential by 2^-20 relative (hardware exp2, 2 units, and its argument), the sum of exponentials by n v; so a probability is off by at
most e = 2 ((D + 4) v max a + 2^-20) + n v relative, whichever way it is normalised.  Each product's sum adds n v (or D v) of its terms' sizes.
"""
import math

import torch

V = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def rotary(x, pos, sections, bases, layout, inverse=False):
    x, pos = x.double(), pos.double()
    out = x.clone()
    P = sum(sections)
    m = 0
    for a, n in enumerate(sections):
        for i in range(n):
            t = pos[:, :, a] * bases[a] ** (-i / n)
            c, s = torch.cos(t)[:, :, None], torch.sin(t)[:, :, None] * (-1 if inverse else 1)
            d0, d1 = (m, m + P) if layout == "halves" else (2 * m, 2 * m + 1)
            out[..., d0] = x[..., d0] * c - x[..., d1] * s
            out[..., d1] = x[..., d0] * s + x[..., d1] * c
            m += 1
    return out


def seen(B, Tq, Tk, left, right, sinks, q_lens=None, k_lens=None):
    """(B, Tq, Tk) truth values, one statement per pair."""
    far = 1 << 40
    ok = torch.zeros((B, Tq, Tk), dtype=torch.bool)
    for b in range(B):
        ql = Tq if q_lens is None else min(max(int(q_lens[b]), 0), Tq)
        kl = Tk if k_lens is None else min(max(int(k_lens[b]), 0), Tk)
        i, j = torch.arange(ql)[:, None], torch.arange(kl)[None, :]
        p = i + kl - ql
        ok[b, :ql, :kl] = (j <= p + (far if right is None else right)) & ((j >= p - (far if left is None else left)) | (j < sinks))
    return ok


def attention(q, k, v, ok, scale=None, dout=None):
    """dict name -> (value, bound on the kernels' error) for out, lse and, with dout, dq, dk, dv; all (B, T, H, D) but lse (B, H, Tq)."""
    u = HALF[q.dtype]
    u1 = u if q.dtype != torch.float32 else 0.0                        # rounding of the probabilities and score gradients to the type
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    Q = q.double().permute(0, 2, 1, 3)
    K, W = (t.double().permute(0, 2, 1, 3).repeat_interleave(G, dim=1) for t in (k, v))
    m = ok[:, None].expand(B, Hq, Tq, Tk)
    K0, W0 = K, W
    S = torch.matmul(Q, K.transpose(2, 3)) * scale
    S = torch.where(m, S, torch.full_like(S, -math.inf))
    lse = torch.logsumexp(S, dim=-1)
    none = lse == -math.inf
    P = torch.exp(S - torch.where(none, torch.zeros_like(lse), lse)[..., None])
    P = torch.where(m, P, torch.zeros_like(P))
    out = torch.matmul(P, W)
    a = float((torch.matmul(Q.abs(), K0.abs().transpose(2, 3)) * scale * m).max()) if m.any() else 0.0
    e = 2 * ((D + 4) * V * a + 2.0 ** -20) + Tk * V
    PW = torch.matmul(P, W0.abs())
    e_out = u * out.abs() + (u1 + e + Tk * V) * PW * (1 + u)
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    got = {"out": (back(out), back(e_out)), "lse": (lse, e + 4 * V * lse.abs().nan_to_num(0, 0, 0))}
    if dout is None:
        return got
    dO = dout.double().permute(0, 2, 1, 3) * (~none)[..., None]
    dP = torch.matmul(dO, W.transpose(2, 3))
    delta = (dO * out).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    e_dp = (D * V) * torch.matmul(dO.abs(), W0.abs().transpose(2, 3)) + (dO.abs() * (e_out + D * V * out.abs())).sum(-1, keepdim=True) + 4 * V * (dP.abs() + delta.abs())
    e_ds = (u1 + e) * dS.abs() + (1 + u1 + e) * P * e_dp
    group = lambda t: t.reshape(B, Hkv, G, *t.shape[2:]).sum(2)  # noqa: E731
    n = Tq * G * V
    dq, e_dq = torch.matmul(dS, K) * scale, torch.matmul(e_ds + Tk * V * dS.abs(), K.abs()) * scale
    dk, e_dk = group(torch.matmul(dS.transpose(2, 3), Q)) * scale, group(torch.matmul((e_ds + n * dS.abs()).transpose(2, 3), Q.abs())) * scale
    dv, e_dv = group(torch.matmul(P.transpose(2, 3), dO)), group(torch.matmul(((u1 + e + n) * P).transpose(2, 3), dO.abs()))
    for name, g, eg in (("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv)):
        got[name] = (back(g), back(u * (g.abs() + eg) + eg + 4 * V * g.abs()))
    return got


def check(name, got, want, bound):
    """Every element within its bound; what is not a number (or infinite) in one is so in the other."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)} != {tuple(want.shape)}"
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN at other places"
    odd = ~finite & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), f"{name}: infinities differ"
    off = (got - want).abs()[finite]
    lim = bound.expand_as(want)[finite] if torch.is_tensor(bound) else torch.full_like(off, bound)
    if off.numel():
        worst = float((off / (lim + 1e-38)).max())
        assert worst <= 1.0, f"{name}: {worst:.3f} of its bound (|err| {float(off.max()):.3e})"
