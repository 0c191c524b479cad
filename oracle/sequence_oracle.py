"""CPU restatements in float64 of the sequence-model operators (autovc_amd/sequence.py), with bounds
on what fp32 arithmetic may differ by.

Every bound is a first-order error analysis in units of U = 2^-24, the half step of fp32, run
beside the value it bounds; a value stored in a type adds half a step of that type (`rounded`).
"""
import math

import numpy as np
import torch

U = 2.0 ** -24


def rounded(x, dtype):
    """Half a step of dtype at x (its smallest subnormal's half where that is more)."""
    i = torch.finfo(dtype)
    return x.abs() * (i.eps / 2) + i.smallest_normal * i.eps / 2


# ---- gated linear recurrence --------------------------------------------------------------------
def recurrence(gates, T, B, h0=None, lengths=None, dirs=1):
    """y [T*B][D*H] and hT [D][B][H] by the definition, frame by frame (differentiable)."""
    D = 2 if dirs == 3 else 1
    H = gates.shape[1] // (3 * D)
    g = gates.double().view(T, B, D, 3, H).unbind(0)  # (a frame taken by its index would cost its gradient T frames)
    length = [T] * B if lengths is None else [max(0, min(T, int(v))) for v in lengths]
    live = torch.tensor([[t < length[b] for b in range(B)] for t in range(T)]).view(T, B, 1)
    ys, hs = [], []
    for d in range(D):
        rev = dirs == 2 or d == 1
        h = torch.zeros(B, H, dtype=torch.float64) if h0 is None else h0[d].double()
        y = [None] * T
        for t in (range(T - 1, -1, -1) if rev else range(T)):
            pre = torch.where(live[t][:, None], g[t][:, d], torch.zeros((), dtype=torch.float64))
            f, z, o = torch.sigmoid(pre[:, 0]), torch.tanh(pre[:, 1]), torch.sigmoid(pre[:, 2])
            h = torch.where(live[t], f * h + torch.sigmoid(-pre[:, 0]) * z, h)
            y[t] = torch.where(live[t], o * h, torch.zeros((), dtype=torch.float64))
        ys.append(torch.stack(y))
        hs.append(h)
    return torch.stack(ys, 2).reshape(T * B, D * H), torch.stack(hs)


def recurrence_bounds(gates, T, B, h0=None, lengths=None, dirs=1, dy=None, dhT=None):
    """Bounds on the fp32 error of (y, hT, dgates, dh0) before the stored values' own rounding.

    A gate's exponential takes its argument with an error of |g| U, and with it and the additions
    and reciprocal that follow, a gate is off by at most (|g| + 8) U relative (z and a gate's
    complement too: neither is formed by a subtraction that cancels).  C = max |g| + 12 leaves 4
    units for the products and sums of one frame, in whatever order the frames are joined: a
    product of gates is off by the sum of its factors' relative errors, as it is frame by frame."""
    D = 2 if dirs == 3 else 1
    H = gates.shape[1] // (3 * D)
    g = gates.double().view(T, B, D, 3, H)
    length = [T] * B if lengths is None else [max(0, min(T, int(v))) for v in lengths]
    dead = torch.tensor([[t >= length[b] for b in range(B)] for t in range(T)]).view(T, B, 1, 1, 1)
    g = torch.where(dead, torch.zeros((), dtype=torch.float64), g)
    C = (min(g.abs().max().item(), 100.0) + 12) * U
    z0 = torch.zeros(T, B, D, H, dtype=torch.float64)
    f, i, z, o = torch.sigmoid(g[..., 0, :]), torch.sigmoid(-g[..., 0, :]), torch.tanh(g[..., 1, :]), torch.sigmoid(g[..., 2, :])
    dead = dead[..., 0]
    f, i = torch.where(dead, z0 + 1, f), torch.where(dead, z0, i)
    live = torch.where(dead, z0, z0 + 1)
    dyv = z0 if dy is None else dy.double().view(T, B, D, H) * live
    Ey, EdG, EhT, Edh0 = z0.clone(), torch.zeros(T, B, D, 3, H, dtype=torch.float64), [], []
    for d in range(D):
        rev = dirs == 2 or d == 1
        order = list(range(T - 1, -1, -1) if rev else range(T))
        h = torch.zeros(B, H, dtype=torch.float64) if h0 is None else h0[d].double()
        E = torch.zeros_like(h)
        before, after, Eb, Ea = {}, {}, {}, {}
        for t in order:
            before[t], Eb[t] = h, E
            ft, it, zt = f[t, :, d], i[t, :, d], z[t, :, d]
            E = ft * E + live[t, :, d] * C * (ft * h.abs() + it * zt.abs())
            h = ft * h + it * zt
            after[t], Ea[t] = h, E
            Ey[t, :, d] = live[t, :, d] * (o[t, :, d] * E + C * (o[t, :, d] * h).abs())
        EhT.append(E)
        c = torch.zeros_like(h) if dhT is None else dhT[d].double()
        Ec = torch.zeros_like(h)
        for t in reversed(order):
            ft, it, zt, ot, dyt = f[t, :, d], i[t, :, d], z[t, :, d], o[t, :, d], dyv[t, :, d]
            e = ot * dyt + c
            Ee = Ec + C * ((ot * dyt).abs() + c.abs())
            dif = before[t] - zt
            # f (1 - f) and the like carry 2 C, a difference the errors of its operands
            EdG[t, :, d, 0] = ft * it * (Ee * dif.abs() + e.abs() * (Eb[t] + C * (before[t].abs() + zt.abs())) + 3 * C * (e * dif).abs())
            EdG[t, :, d, 1] = it * (Ee * (1 - zt * zt) + e.abs() * (2 * C * zt * zt + 3 * C))
            EdG[t, :, d, 2] = dyt.abs() * ot * (Ea[t] + 3 * C * after[t].abs())
            c = ft * e
            Ec = ft * Ee + C * live[t, :, d] * c.abs()
        Edh0.append(Ec + C * c.abs())
    return Ey.reshape(T * B, D * H), torch.stack(EhT), (EdG * live[:, :, :, None]).reshape(T * B, D * 3 * H), torch.stack(Edh0)


# ---- log-probabilities of given classes -----------------------------------------------------------
def log_softmax(z):
    """From the differences to the maximum (at logits of -3e38 even float64 holds no z - lse), and with
    the largest class kept out of the sum (a confident row's rest is below its 1's last bit)."""
    d = z - z.max()
    others = torch.ones_like(d, dtype=torch.bool)
    others[d.argmax()] = False
    return d - torch.log1p(torch.exp(d[others]).sum())


def entropy_of(lp):
    """Of log-probabilities along the last dimension (0 log 0 = 0; a NaN makes it NaN)."""
    p = torch.exp(lp)
    return -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(-1)


def log_probs(logits, tokens, top=0, ignore_index=-100):
    """(logp [N], entropy [N], top_logp [N][top], top_ids [N][top]) of rows [N][V]."""
    z = logits.double()
    N, V = z.shape
    lp = torch.full((N, V), -math.inf, dtype=torch.float64)
    for r in range(N):
        if not bool((z[r] == -math.inf).all()):
            lp[r] = log_softmax(z[r])
    entropy = entropy_of(lp)
    logp = torch.zeros(N, dtype=torch.float64)
    for r, t in enumerate(tokens.tolist()):
        if t != ignore_index:
            logp[r] = lp[r, t] if 0 <= t < V else math.nan
    rank = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z).numpy()
    ids = np.stack([np.lexsort((np.arange(V), -row))[:top] for row in rank]) if N else np.zeros((0, top))
    ids = torch.from_numpy(ids.astype(np.int64))
    return logp, entropy, torch.gather(lp, 1, ids) if N else lp[:, :top], ids


def log_probs_grad(logits, tokens, dlogp, dentropy, ignore_index=-100):
    """The gradient's formula: dlogp (onehot - p) - dentropy p (log p + entropy)."""
    z = logits.double()
    N, V = z.shape
    d = torch.zeros(N, V, dtype=torch.float64)
    for r, t in enumerate(tokens.tolist()):
        gl = 0.0 if t == ignore_index else float(dlogp[r]) if 0 <= t < V else math.nan
        if bool((z[r] == -math.inf).all()):
            d[r] = gl if gl != gl else 0.0
            continue
        lp = log_softmax(z[r])
        p = torch.exp(lp)
        plus = float(dentropy[r]) * p * (torch.where(p > 0, lp, torch.zeros_like(lp)) + entropy_of(lp))
        d[r] = -gl * p - plus
        if 0 <= t < V:
            d[r, t] = -gl * torch.expm1(lp[t]) - plus[t]  # gl (1 - p), not from 1 - p
    return d


def log_probs_bounds(logits, tokens, dlogp=None, dentropy=None, adds=300):
    """Bounds on the fp32 errors of (logp at every class, entropy, gradient), in the order above.

    adds: the longest chain of additions in a row's sums (a thread's own elements, then the joins).
    With d = z - max: e^d is off by (|d| + 3) U relative, the sum s of them by (adds + 3 + mean |d|) U,
    u = sum e^d d by (adds + 5) U of itself and mean d^2 U of s; the maximum being moved costs one
    more such exponential, which `adds` holds too."""
    z = logits.double()
    m = z.max(1, keepdim=True).values
    d = torch.where(z == -math.inf, torch.full_like(z, -math.inf), z - m)
    p = torch.softmax(d, 1)
    pd = torch.where(p > 0, p * d.abs(), torch.zeros_like(p))
    mean, mean2 = pd.sum(1), torch.where(p > 0, p * d * d, torch.zeros_like(p)).sum(1)
    logs = torch.logsumexp(d, 1)
    Es = (adds + 3 + mean) * U
    Elogs = Es + 2 * U * logs.abs()
    dd = torch.where(d == -math.inf, torch.zeros_like(d), d.abs())
    Elp = U * (dd + (dd + logs[:, None])) + Elogs[:, None]
    EH = Elogs + ((adds + 5) * mean + mean2) * U + mean * Es + 2 * U * (logs + mean)
    Eg = None
    if dlogp is not None or dentropy is not None:
        gl = torch.zeros(z.shape[0], dtype=torch.float64) if dlogp is None else dlogp.double().abs()
        ge = torch.zeros_like(gl) if dentropy is None else dentropy.double().abs()
        H = torch.special.entr(p).sum(1)
        Ep = p * ((dd + 6) * U + Es[:, None])
        inner = gl[:, None] + ge[:, None] * (torch.where(p > 0, (torch.log(p.clamp_min(1e-300))).abs(), torch.zeros_like(p)) + H[:, None])
        Eg = Ep * inner + p * ge[:, None] * (Elp + EH[:, None]) + 6 * U * p * inner + 2 * U * gl[:, None]
    return Elp, EH, Eg


# ---- counter-based dropout --------------------------------------------------------------------------
def dropout_keep(n, p, seed, steps, layer):
    """The first n decisions of the stream (seed, steps, layer), one Python integer at a time."""
    M, G = (1 << 64) - 1, 0x9E3779B97F4A7C15

    def mix(v):
        v = ((v ^ (v >> 30)) * 0xBF58476D1CE4E5B9) & M
        v = ((v ^ (v >> 27)) * 0x94D049BB133111EB) & M
        return v ^ (v >> 31)

    key = mix((mix((mix((seed + G) & M) + steps) & M) + layer) & M)
    keep = np.zeros(n + 1, dtype=bool)
    least = int(p * 2.0 ** 32)
    for j in range((n + 1) // 2):
        w = mix((key + (j + 1) * G) & M)
        keep[2 * j] = (w & 0xFFFFFFFF) >= least
        keep[2 * j + 1] = (w >> 32) >= least
    return torch.from_numpy(keep[:n].copy())
