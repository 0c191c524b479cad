"""Sequence-model operators over the HIP C-ABI: the gated linear recurrence, log-probabilities of
given classes, and counter-based dropout (kernels: csrc/recurrence.hip, class_probs.hip, dropout.hip;
checks, allocation and autograd: csrc_torch/sequence.cpp).

They take fp32, bf16 and fp16 tensors; statistics, sums and recurrent states are fp32.  Rows may be
column slices of a wider buffer (any row stride); other layouts are made contiguous.  Every call
runs on the current stream of its tensors' device and allocates what it needs through torch, so it
may be captured into a graph and used from several streams.  (A backward pass is captured only while no
graph that was built outside the capture from the same leaves is alive, as torch asks for any of
its own.)  Gradients are differentiable once; forward-mode derivatives and
tracing (torch.jit.trace, make_fx, fake tensors) are refused.
Public names are re-exported by `autovc_amd.ops`.
"""
from __future__ import annotations

from . import _lib

MAX_TOP = 32
_ext = None


def _load():
    """The torch functions (autovc_amd/_sequence.so), bound to the library.  Raises if either is absent."""
    global _ext
    _lib.load()
    try:
        from . import _sequence
    except ImportError as e:
        raise _lib.HipLibraryError(f"autovc_amd/_sequence.so is not there or not for this torch ({e}); build it with `make`")
    _sequence.bind(_lib.LIB_PATH, _lib.HipLibraryError)
    _ext = _sequence
    return _ext


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
    return (_ext or _load()).gated_recurrence(gates, T, B, h0, lengths, dirs)


def gated_recurrence_step(gates, state, out_state=None):
    """One frame of gated_recurrence for every row, as a serving loop calls it: gates [B][3*H],
    state [B][H] fp32 -> (y [B][H], new state).  The new state goes to out_state (which may be
    `state` itself) or to a fresh tensor.  No autograd."""
    return (_ext or _load()).gated_recurrence_step(gates, state, out_state)


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
    return (_ext or _load()).token_log_probs(logits, tokens, top, ignore_index)


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
    return (_ext or _load()).dropout(x, p, rng, residual, layer)
