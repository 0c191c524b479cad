"""Sequence-model operators over the HIP C-ABI: the gated linear recurrence, log-probabilities of
given classes, and counter-based dropout (kernels: csrc/recurrence.hip, class_probs.hip, dropout.hip).

They take fp32, bf16 and fp16 tensors; statistics, sums and recurrent states are fp32.  Rows may be
column slices of a wider buffer (any row stride); other layouts are made contiguous.  Every call
runs on the current stream of its tensors' device and allocates what it needs through torch, so it
may be captured into a graph and used from several streams.  Public names are re-exported by
`autovc_amd.ops`.

On small tensors a call costs what the host spends on it, and a backward more than the same code
elsewhere: it runs on a thread whose core has none of these objects in its caches.  So the common
layouts take a short path through here.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import DTYPES

MAX_TOP = 32
_F32 = torch.float32


def _check(t, name, like=None, dtypes=DTYPES):
    """t is a tensor on a GPU (like's) of one of dtypes."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"autovc_amd runs on the GPU only (HIP kernels); {name} is a CPU tensor")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}")


def _rows(t):
    """(tensor, row stride) of a matrix whose rows the kernels can walk: t itself unless its rows
    are not dense or overlap."""
    n, c = t.shape
    if t.is_contiguous():
        return t, c
    s = t.stride()
    if (c > 1 and s[1] != 1) or (n > 1 and s[0] < c):
        return t.contiguous(), c
    return t, (s[0] if n > 1 else c)


def _launch(dev, name, *args):
    """The library's call of that name on dev's current stream, with dev current."""
    if dev.index == torch.cuda.current_device():
        status = getattr(_lib.load(), name)(*args, _lib.stream(dev))
    else:
        with torch.cuda.device(dev):
            status = getattr(_lib.load(), name)(*args, _lib.stream(dev))
    if status:
        _lib.check(status, name)


def _wants_grad(a, b=None):
    return (a.requires_grad or (b is not None and b.requires_grad)) and torch.is_grad_enabled()


def _backward(grads, ctx, *d):
    """A backward that is not differentiable itself: where a graph of it is asked for
    (create_graph), using that graph is an error; without one, grads runs as it is."""
    if torch.is_grad_enabled():
        return once_differentiable(grads)(ctx, *d)
    return grads(ctx, *d)


# ---- gated linear recurrence --------------------------------------------------------------------
def _recurrence(gates, T, B, H, h0, lengths, dirs, save):
    dt, dev, lib = DTYPES[gates.dtype], gates.device, _lib.load()
    D = 2 if dirs == 3 else 1
    g, ldg = _rows(gates)
    y = torch.empty((T * B, D * H), dtype=gates.dtype, device=dev)
    hT = torch.empty((D, B, H), dtype=_F32, device=dev)
    states = torch.empty(lib.avc_gated_recurrence_states(T, B, H, dirs), dtype=_F32, device=dev) if save else None
    wb = lib.avc_gated_recurrence_workspace(dt, T, B, H, dirs)
    ws = torch.empty(wb, dtype=torch.uint8, device=dev) if wb else None
    _launch(dev, "avc_gated_recurrence_forward", dt, T, B, H, dirs, g.data_ptr(), ldg,
            None if h0 is None else h0.data_ptr(), None if lengths is None else lengths.data_ptr(), y.data_ptr(), D * H,
            hT.data_ptr(), states.data_ptr() if save else None, ws.data_ptr() if wb else None, wb)
    return y, hT, states


def _recurrence_grads(ctx, dy, dhT):
    gates, lengths, states = ctx.saved_tensors
    T, B, H, dirs, want_h0 = ctx.dims
    dt, dev = DTYPES[gates.dtype], gates.device
    D = 2 if dirs == 3 else 1
    g, ldg = _rows(gates)
    dy, lddy = _rows(torch.zeros((T * B, D * H), dtype=gates.dtype, device=dev) if dy is None else dy)
    dhT = None if dhT is None else dhT.contiguous()
    dg = torch.empty((T * B, D * 3 * H), dtype=gates.dtype, device=dev)
    dh0 = torch.empty((D, B, H), dtype=_F32, device=dev) if want_h0 else None
    wb = _lib.load().avc_gated_recurrence_workspace(dt, T, B, H, dirs)
    ws = torch.empty(wb, dtype=torch.uint8, device=dev) if wb else None
    _launch(dev, "avc_gated_recurrence_backward", dt, T, B, H, dirs, g.data_ptr(), ldg,
            None if lengths is None else lengths.data_ptr(), states.data_ptr(), dy.data_ptr(), lddy,
            None if dhT is None else dhT.data_ptr(), dg.data_ptr(), D * 3 * H, dh0.data_ptr() if want_h0 else None,
            ws.data_ptr() if wb else None, wb)
    return dg, dh0, None, None, None, None, None


class GatedRecurrence(torch.autograd.Function):
    """Autograd of gated_recurrence; the forward keeps the state before every 64th frame."""

    @staticmethod
    def forward(ctx, gates, h0, T, B, H, lengths, dirs):
        y, hT, states = _recurrence(gates, T, B, H, h0, lengths, dirs, True)
        ctx.save_for_backward(gates, lengths, states)
        ctx.dims = (T, B, H, dirs, ctx.needs_input_grad[1])
        ctx.set_materialize_grads(False)
        return y, hT

    @staticmethod
    def backward(ctx, dy, dhT):
        return _backward(_recurrence_grads, ctx, dy, dhT)


def gated_recurrence(gates, T, B, h0=None, lengths=None, dirs=1):
    """Gated linear recurrence over time-major frames: f = sigmoid(g_f), z = tanh(g_c),
    o = sigmoid(g_o);  h_t = f h_{t-1} + (1 - f) z,  y_t = o h_t.

    gates    [T*B][D*3*H], a row holding [D][f, c, o][H] (one projection of the layer's input)
    h0       [D][B][H] fp32, or None for zero
    lengths  [B] integers or None: frames at or behind a sequence's length are not used (whatever
             they hold), give y = 0 and no gradient; values are held to 0 .. T
    dirs     1 forward in time, 2 reverse, 3 both (D = 2; y holds forward || reverse)
    Returns y [T*B][D*H] in gates' type and the last states hT [D][B][H] fp32; differentiable in
    gates and h0."""
    _check(gates, "gates")
    T, B, dirs = int(T), int(B), int(dirs)
    if dirs not in (1, 2, 3):
        raise ValueError("dirs is 1 (forward), 2 (reverse) or 3 (both)")
    D = 2 if dirs == 3 else 1
    if T < 0 or B < 0 or gates.dim() != 2 or gates.shape[0] != T * B or gates.shape[1] == 0 or gates.shape[1] % (3 * D):
        raise ValueError(f"gates must be [T*B = {T * B}][{3 * D} * H], got {tuple(gates.shape)}")
    H = gates.shape[1] // (3 * D)
    if h0 is not None:
        _check(h0, "h0", gates, (_F32,))
        if tuple(h0.shape) != (D, B, H):
            raise ValueError(f"h0 must be {(D, B, H)}, got {tuple(h0.shape)}")
        h0 = h0.contiguous()
    if lengths is not None:
        _check(lengths, "lengths", gates, (torch.int32, torch.int64))
        if tuple(lengths.shape) != (B,):
            raise ValueError(f"lengths must be {(B,)}, got {tuple(lengths.shape)}")
        lengths = lengths.clamp(0, T).to(torch.int32) if lengths.dtype == torch.int64 else lengths.contiguous()
    if T * B == 0:
        hT = h0.clone() if h0 is not None else torch.zeros((D, B, H), dtype=_F32, device=gates.device)
        return gates[:, :D * H].contiguous(), hT
    if _wants_grad(gates, h0):
        return GatedRecurrence.apply(gates, h0, T, B, H, lengths, dirs)
    return _recurrence(gates, T, B, H, h0, lengths, dirs, False)[:2]


def gated_recurrence_step(gates, state, out_state=None):
    """One frame of gated_recurrence for every row, as a serving loop calls it: gates [B][3*H],
    state [B][H] fp32 -> (y [B][H], new state).  The new state goes to out_state (which may be
    `state` itself) or to a fresh tensor.  No autograd."""
    _check(gates, "gates")
    _check(state, "state", gates, (_F32,))
    if gates.dim() != 2 or gates.shape[1] == 0 or gates.shape[1] % 3:
        raise ValueError(f"gates must be [B][3 * H], got {tuple(gates.shape)}")
    if _wants_grad(gates, state):
        raise RuntimeError("gated_recurrence_step builds no autograd graph; use gated_recurrence")
    B, H = gates.shape[0], gates.shape[1] // 3
    if tuple(state.shape) != (B, H):
        raise ValueError(f"state must be {(B, H)}, got {tuple(state.shape)}")
    dev = gates.device
    if out_state is None:
        out_state = torch.empty((B, H), dtype=_F32, device=dev)
    else:
        _check(out_state, "out_state", gates, (_F32,))
        if tuple(out_state.shape) != (B, H) or not out_state.is_contiguous():
            raise ValueError(f"out_state must be a contiguous {(B, H)}")
        if out_state is not state and _overlap(out_state, state) and not (
                out_state.data_ptr() == state.data_ptr() and state.is_contiguous()):
            raise ValueError("out_state overlaps state without being it")
    y = torch.empty((B, H), dtype=gates.dtype, device=dev)
    if B:
        g, ldg = _rows(gates)
        state = state.contiguous()
        _launch(dev, "avc_gated_recurrence_step", DTYPES[gates.dtype], B, H, g.data_ptr(), ldg, state.data_ptr(),
                out_state.data_ptr(), y.data_ptr(), H)
    return y, out_state


def _overlap(a, b):
    """Whether a's (contiguous) bytes and the span of b's meet."""
    span = 1 + sum((n - 1) * s for n, s in zip(b.shape, b.stride())) if b.numel() else 0
    return a.data_ptr() < b.data_ptr() + span * b.element_size() and \
        b.data_ptr() < a.data_ptr() + a.numel() * a.element_size()


# ---- log-probabilities of given classes -----------------------------------------------------------
def _log_probs(logits, tokens, top, ignore, save):
    dt, dev = DTYPES[logits.dtype], logits.device
    N, V = logits.shape
    z, ldz = _rows(logits)
    logp = torch.empty(N, dtype=_F32, device=dev)
    entropy = torch.empty(N, dtype=_F32, device=dev)
    top_logp = torch.empty((N, top), dtype=_F32, device=dev)
    top_ids = torch.empty((N, top), dtype=torch.int64, device=dev)
    stats = torch.empty((N, 3), dtype=_F32, device=dev) if save else None
    wb = _lib.load().avc_token_log_probs_workspace(dt, N, V, top)
    ws = torch.empty(wb, dtype=torch.uint8, device=dev) if wb else None
    if N:
        _launch(dev, "avc_token_log_probs_forward", dt, N, V, z.data_ptr(), ldz, tokens.data_ptr(), ignore, top,
                logp.data_ptr(), entropy.data_ptr(), stats.data_ptr() if save else None, top_logp.data_ptr(),
                top_ids.data_ptr(), ws.data_ptr() if wb else None, wb)
    return logp, entropy, top_logp, top_ids, stats


def _log_probs_grads(ctx, dlogp, dentropy, _top_logp, _top_ids):
    logits, tokens, stats = ctx.saved_tensors
    N, V = logits.shape
    z, ldz = _rows(logits)
    d = torch.empty((N, V), dtype=logits.dtype, device=logits.device)
    dlogp = None if dlogp is None else dlogp.contiguous()
    dentropy = None if dentropy is None else dentropy.contiguous()
    if N:
        _launch(logits.device, "avc_token_log_probs_backward", DTYPES[logits.dtype], N, V, z.data_ptr(), ldz,
                tokens.data_ptr(), ctx.ignore, stats.data_ptr(), None if dlogp is None else dlogp.data_ptr(),
                None if dentropy is None else dentropy.data_ptr(), d.data_ptr(), V)
    return d, None, None, None


class TokenLogProbs(torch.autograd.Function):
    """Autograd of token_log_probs over rows [N][V]; keeps three statistics a row."""

    @staticmethod
    def forward(ctx, logits, tokens, top, ignore):
        logp, entropy, top_logp, top_ids, stats = _log_probs(logits, tokens, top, ignore, True)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.ignore = ignore
        ctx.mark_non_differentiable(top_logp, top_ids)
        ctx.set_materialize_grads(False)
        return logp, entropy, top_logp, top_ids

    @staticmethod
    def backward(ctx, *d):
        return _backward(_log_probs_grads, ctx, *d)


def token_log_probs(logits, tokens, top=0, ignore_index=-100):
    """Log-probabilities of given classes under softmax(logits), each row's entropy, and its `top`
    most probable classes.

    logits  [..., V]; -inf rules a class out
    tokens  [...] integers.  ignore_index gives 0 and no gradient through it; another value outside
            0 .. V-1 gives NaN
    Returns (logp [...], entropy [...], top_logp [..., top], top_ids [..., top]): fp32 and int64, the
    alternatives most probable first, equal ones by the lower class.  logp and entropy are
    differentiable in logits; the alternatives are not.  A row with every class ruled out gives
    log-probability -inf, entropy 0 and gradient 0."""
    _check(logits, "logits")
    _check(tokens, "tokens", logits, (torch.int64, torch.int32))
    if logits.dim() < 1 or logits.shape[-1] < 1 or logits.shape[:-1] != tokens.shape:
        raise ValueError(f"logits [..., V >= 1] and tokens [...] must agree, got {tuple(logits.shape)} and {tuple(tokens.shape)}")
    V = logits.shape[-1]
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must be 0 .. {min(MAX_TOP, V)}, got {top}")
    if tokens.dtype != torch.int64 or not tokens.is_contiguous():
        tokens = tokens.to(torch.int64).contiguous()
    lead = None
    if logits.dim() != 2:
        lead = tokens.shape
        logits, tokens = logits.reshape(-1, V), tokens.reshape(-1)
    if _wants_grad(logits):
        out = TokenLogProbs.apply(logits, tokens, top, int(ignore_index))
    else:
        out = _log_probs(logits, tokens, top, int(ignore_index), False)[:4]
    if lead is None:
        return out
    return out[0].view(lead), out[1].view(lead), out[2].view(*lead, top), out[3].view(*lead, top)


# ---- counter-based dropout --------------------------------------------------------------------------
def _drop(x, residual, p, rng, layer):
    if x.is_contiguous() and (residual is None or residual.is_contiguous()):
        y = torch.empty_like(x)
        n = c = ldx = ldr = ldy = x.numel()
        if n == 0:
            return y
        n = 1
    else:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if x.numel() == 0:
            return y
        c = ldy = x.shape[-1]
        x, ldx = _rows(x if x.dim() == 2 else x.reshape(-1, c))
        n, ldr = x.shape[0], 0
        if residual is not None:
            residual, ldr = _rows(residual if residual.dim() == 2 else residual.reshape(-1, c))
    _launch(x.device, "avc_dropout", DTYPES[x.dtype], n, c, x.data_ptr(), ldx,
            None if residual is None else residual.data_ptr(), ldr, p, rng.data_ptr(), layer, y.data_ptr(), ldy)
    return y


def _dropout_grads(ctx, dy):
    (rng,) = ctx.saved_tensors
    need_x, need_residual = ctx.needs_input_grad[:2]
    return _drop(dy, None, ctx.p, rng, ctx.layer) if need_x else None, dy if need_residual else None, None, None, None


class Dropout(torch.autograd.Function):
    """Autograd of dropout: the backward forms the mask again from rng (saved, so that changing it
    in place before the backward is an error and not another mask)."""

    @staticmethod
    def forward(ctx, x, residual, p, rng, layer):
        ctx.save_for_backward(rng)
        ctx.p, ctx.layer = p, layer
        return _drop(x, residual, p, rng, layer)

    @staticmethod
    def backward(ctx, dy):
        return _backward(_dropout_grads, ctx, dy)


def dropout(x, p, rng, residual=None, layer=0):
    """residual + x keep / (1 - p) with a mask that is a function of (rng, layer, element) and never
    stored; a fresh mask for every step count.

    x         any shape; element i of the mask is x's i-th element in row-major order
    p         probability of dropping an element, 0 <= p < 1
    rng       [2] int64 on x's device: a seed and the count of steps done.  Advance the count in
              place after the step's backward (`rng[1] += 1`), also inside a captured step
    layer     0 .. 2^32 - 1: tells the dropouts of one step apart
    residual  added after the dropout, x's shape and type, or None
    Differentiable in x and residual."""
    _check(x, "x")
    _check(rng, "rng", x, (torch.int64,))
    p, layer = float(p), int(layer)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"p must be 0 <= p < 1, got {p}")
    if not 0 <= layer < 1 << 32:
        raise ValueError(f"layer must be 0 .. 2^32 - 1, got {layer}")
    if rng.dim() != 1 or rng.shape[0] != 2 or not rng.is_contiguous():
        raise ValueError(f"rng must be a contiguous [2], got {tuple(rng.shape)}")
    if residual is not None:
        _check(residual, "residual", x, (x.dtype,))
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    if _wants_grad(x, residual):
        return Dropout.apply(x, residual, p, rng, layer)
    return _drop(x, residual, p, rng, layer)
