"""Sequence-model operators over the HIP C-ABI: the gated linear recurrence, log-probabilities of
given classes, and counter-based dropout (kernels: csrc/recurrence.hip, class_probs.hip, dropout.hip).

They take fp32, bf16 and fp16 tensors; statistics, sums and recurrent states are fp32.  Rows may be
column slices of a wider buffer (any row stride); other layouts are made contiguous.  Every call
runs on the current stream of its tensors' device and allocates what it needs through torch, so it
may be captured into a graph and used from several streams.  Public names are re-exported by
`autovc_amd.ops`.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call

MAX_TOP = 32


def _check(t, name, like=None, dtypes=None):
    """t is a tensor on a GPU (like's) of one of dtypes."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"autovc_amd runs on the GPU only (HIP kernels); {name} is a CPU tensor")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    if t.dtype not in (_lib.DTYPES if dtypes is None else dtypes):
        raise TypeError(f"{name} has dtype {t.dtype}")
    return t


def _rows(t):
    """(tensor, row stride) of a matrix whose rows the kernels can walk: t itself unless its rows
    are not dense or overlap."""
    n, c = t.shape
    s = t.stride()
    if (c > 1 and s[1] != 1) or (n > 1 and s[0] < c):
        t = t.contiguous()
        s = t.stride()
    return t, (s[0] if n > 1 else c)


def _launch(t, name, *args):
    """call(name, *args, stream) with t's device current."""
    dev = t.device
    if dev.index == torch.cuda.current_device():
        call(name, *args, _lib.stream(dev))
    else:
        with torch.cuda.device(dev):
            call(name, *args, _lib.stream(dev))


def _p(t):
    return None if t is None else t.data_ptr()


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ---- gated linear recurrence --------------------------------------------------------------------
def _recurrence_forward(gates, T, B, D, H, h0, lengths, dirs, save):
    dt = _lib.DTYPES[gates.dtype]
    lib = _lib.load()
    g, ldg = _rows(gates)
    y = torch.empty((T * B, D * H), dtype=gates.dtype, device=gates.device)
    hT = torch.empty((D, B, H), dtype=torch.float32, device=gates.device)
    states = None
    if save:
        states = torch.empty(lib.avc_gated_recurrence_states(T, B, H, dirs), dtype=torch.float32, device=gates.device)
    wb = lib.avc_gated_recurrence_workspace(dt, T, B, H, dirs)
    ws = torch.empty(wb, dtype=torch.uint8, device=gates.device) if wb else None
    _launch(gates, "avc_gated_recurrence_forward", dt, T, B, H, dirs, g.data_ptr(), ldg, _p(h0), _p(lengths),
            y.data_ptr(), D * H, hT.data_ptr(), _p(states), _p(ws), wb)
    return y, hT, states


class GatedRecurrence(torch.autograd.Function):
    """Autograd of gated_recurrence; the forward keeps the state before every 64th frame."""

    @staticmethod
    def forward(ctx, gates, h0, T, B, D, H, lengths, dirs):
        y, hT, states = _recurrence_forward(gates, T, B, D, H, h0, lengths, dirs, True)
        ctx.save_for_backward(gates, lengths, states)
        ctx.dims = (T, B, D, H, dirs, h0 is not None)
        ctx.set_materialize_grads(False)
        return y, hT

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dhT):
        gates, lengths, states = ctx.saved_tensors
        T, B, D, H, dirs, has_h0 = ctx.dims
        g, ldg = _rows(gates)
        dy, lddy = _rows(torch.zeros((T * B, D * H), dtype=gates.dtype, device=gates.device) if dy is None else dy)
        dhT = None if dhT is None else dhT.contiguous()
        dg = torch.empty((T * B, D * 3 * H), dtype=gates.dtype, device=gates.device)
        dh0 = torch.empty((D, B, H), dtype=torch.float32, device=gates.device) if has_h0 and ctx.needs_input_grad[1] else None
        dt = _lib.DTYPES[gates.dtype]
        wb = _lib.load().avc_gated_recurrence_workspace(dt, T, B, H, dirs)
        ws = torch.empty(wb, dtype=torch.uint8, device=gates.device) if wb else None
        _launch(gates, "avc_gated_recurrence_backward", dt, T, B, H, dirs, g.data_ptr(), ldg, _p(lengths),
                states.data_ptr(), dy.data_ptr(), lddy, _p(dhT), dg.data_ptr(), D * 3 * H, _p(dh0), _p(ws), wb)
        return dg, dh0, None, None, None, None, None, None


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
        _check(h0, "h0", gates, (torch.float32,))
        if tuple(h0.shape) != (D, B, H):
            raise ValueError(f"h0 must be {(D, B, H)}, got {tuple(h0.shape)}")
        h0 = h0.contiguous()
    if lengths is not None:
        _check(lengths, "lengths", gates, (torch.int32, torch.int64))
        if tuple(lengths.shape) != (B,):
            raise ValueError(f"lengths must be {(B,)}, got {tuple(lengths.shape)}")
        lengths = lengths.clamp(0, T).to(torch.int32) if lengths.dtype == torch.int64 else lengths.contiguous()
    if T * B == 0:
        hT = h0.clone() if h0 is not None else torch.zeros((D, B, H), dtype=torch.float32, device=gates.device)
        return gates[:, :D * H].contiguous(), hT
    if _wants_grad(gates, h0):
        return GatedRecurrence.apply(gates, h0, T, B, D, H, lengths, dirs)
    return _recurrence_forward(gates, T, B, D, H, h0, lengths, dirs, False)[:2]


def gated_recurrence_step(gates, state, out_state=None):
    """One frame of gated_recurrence for every row, as a serving loop calls it: gates [B][3*H],
    state [B][H] fp32 -> (y [B][H], new state).  The new state goes to out_state (which may be
    `state` itself) or to a fresh tensor.  No autograd."""
    _check(gates, "gates")
    _check(state, "state", gates, (torch.float32,))
    if gates.dim() != 2 or gates.shape[1] == 0 or gates.shape[1] % 3:
        raise ValueError(f"gates must be [B][3 * H], got {tuple(gates.shape)}")
    if _wants_grad(gates, state):
        raise RuntimeError("gated_recurrence_step builds no autograd graph; use gated_recurrence")
    B, H = gates.shape[0], gates.shape[1] // 3
    if tuple(state.shape) != (B, H):
        raise ValueError(f"state must be {(B, H)}, got {tuple(state.shape)}")
    if out_state is None:
        out_state = torch.empty((B, H), dtype=torch.float32, device=gates.device)
    else:
        _check(out_state, "out_state", gates, (torch.float32,))
        if tuple(out_state.shape) != (B, H) or not out_state.is_contiguous():
            raise ValueError(f"out_state must be a contiguous {(B, H)}")
        if out_state.data_ptr() != state.data_ptr() and _overlap(out_state, state):
            raise ValueError("out_state overlaps state without being it")
    y = torch.empty((B, H), dtype=gates.dtype, device=gates.device)
    if B:
        g, ldg = _rows(gates)
        state = state.contiguous()
        _launch(gates, "avc_gated_recurrence_step", _lib.DTYPES[gates.dtype], B, H, g.data_ptr(), ldg,
                state.data_ptr(), out_state.data_ptr(), y.data_ptr(), H)
    return y, out_state


def _overlap(a, b):
    """Whether a's (contiguous) bytes and the span of b's meet."""
    span = 1 + sum((n - 1) * s for n, s in zip(b.shape, b.stride())) if b.numel() else 0
    return a.data_ptr() < b.data_ptr() + span * b.element_size() and \
        b.data_ptr() < a.data_ptr() + a.numel() * a.element_size()


# ---- log-probabilities of given classes -----------------------------------------------------------
def _log_probs_forward(logits, tokens, top, ignore, save):
    dt = _lib.DTYPES[logits.dtype]
    dev = logits.device
    N, V = logits.shape
    z, ldz = _rows(logits)
    logp, entropy = torch.empty((2, N), dtype=torch.float32, device=dev).unbind(0)
    top_logp = torch.empty((N, top), dtype=torch.float32, device=dev)
    top_ids = torch.empty((N, top), dtype=torch.int64, device=dev)
    stats = torch.empty((N, 3), dtype=torch.float32, device=dev) if save else None
    wb = _lib.load().avc_token_log_probs_workspace(dt, N, V, top)
    ws = torch.empty(wb, dtype=torch.uint8, device=dev) if wb else None
    if N:
        _launch(logits, "avc_token_log_probs_forward", dt, N, V, z.data_ptr(), ldz, tokens.data_ptr(), ignore, top,
                logp.data_ptr(), entropy.data_ptr(), _p(stats), top_logp.data_ptr(), top_ids.data_ptr(), _p(ws), wb)
    return logp, entropy, top_logp, top_ids, stats


class TokenLogProbs(torch.autograd.Function):
    """Autograd of token_log_probs over rows [N][V]; keeps three statistics a row."""

    @staticmethod
    def forward(ctx, logits, tokens, top, ignore):
        logp, entropy, top_logp, top_ids, stats = _log_probs_forward(logits, tokens, top, ignore, True)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.ignore = ignore
        ctx.mark_non_differentiable(top_logp, top_ids)
        ctx.set_materialize_grads(False)
        return logp, entropy, top_logp, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dentropy, _top_logp, _top_ids):
        logits, tokens, stats = ctx.saved_tensors
        N, V = logits.shape
        z, ldz = _rows(logits)
        d = torch.empty((N, V), dtype=logits.dtype, device=logits.device)
        dlogp = None if dlogp is None else dlogp.contiguous()
        dentropy = None if dentropy is None else dentropy.contiguous()
        if N:
            _launch(logits, "avc_token_log_probs_backward", _lib.DTYPES[logits.dtype], N, V, z.data_ptr(), ldz,
                    tokens.data_ptr(), ctx.ignore, stats.data_ptr(), _p(dlogp), _p(dentropy), d.data_ptr(), V)
        return d, None, None, None


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
    V, lead = logits.shape[-1], tokens.shape
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must be 0 .. {min(MAX_TOP, V)}, got {top}")
    tokens = tokens.to(torch.int64).contiguous()
    flat = logits.dim() == 2
    if not flat:
        logits, tokens = logits.reshape(-1, V), tokens.reshape(-1)
    if _wants_grad(logits):
        out = TokenLogProbs.apply(logits, tokens, top, int(ignore_index))
    else:
        out = _log_probs_forward(logits, tokens, top, int(ignore_index), False)[:4]
    if flat:
        return out
    return out[0].view(lead), out[1].view(lead), out[2].view(*lead, top), out[3].view(*lead, top)


# ---- counter-based dropout --------------------------------------------------------------------------
def _drop(x, residual, p, rng, layer):
    shape = x.shape
    if x.dim() != 2 or residual is not None and residual.dim() != 2:
        c = shape[-1] if x.dim() else 1
        x = x.reshape(-1, c) if c else x.reshape(0, 0)
        residual = None if residual is None else residual.reshape(x.shape)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        x, ldx = _rows(x)
        ldr = 0
        if residual is not None:
            residual, ldr = _rows(residual)
        n, c = x.shape
        _launch(x, "avc_dropout", _lib.DTYPES[x.dtype], n, c, x.data_ptr(), ldx, _p(residual), ldr, p, rng.data_ptr(),
                layer, y.data_ptr(), c)
    return y.view(shape)


class Dropout(torch.autograd.Function):
    """Autograd of dropout: the backward forms the mask again from rng (saved, so that changing it
    in place before the backward is an error and not another mask)."""

    @staticmethod
    def forward(ctx, x, residual, p, rng, layer):
        ctx.save_for_backward(rng)
        ctx.cfg = (p, layer)
        return _drop(x, residual, p, rng, layer)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        dx = _drop(dy, None, ctx.cfg[0], rng, ctx.cfg[1]) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


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
    if tuple(rng.shape) != (2,) or not rng.is_contiguous():
        raise ValueError(f"rng must be a contiguous [2], got {tuple(rng.shape)}")
    if residual is not None:
        _check(residual, "residual", x, (x.dtype,))
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    if _wants_grad(x, residual):
        return Dropout.apply(x, residual, p, rng, layer)
    return _drop(x, residual, p, rng, layer)
