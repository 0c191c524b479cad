"""CPU: the float64 oracle of the sequence-model operators against differences and torch, and the
refusals of the entry points that need no GPU."""
import ctypes
import math

import pytest
import torch

from autovc_amd import _lib, ops
from oracle import sequence_oracle as so


@pytest.mark.parametrize("dirs,lengths", [(1, None), (2, [4, 0, 2]), (3, [5, 3, 0])])
def test_recurrence_gradient_matches_differences(dirs, lengths):
    T, B, H, D = 5, 3, 2, 2 if dirs == 3 else 1
    gen = torch.Generator().manual_seed(dirs)
    g = torch.randn(T * B, D * 3 * H, generator=gen, dtype=torch.float64, requires_grad=True)
    h0 = torch.randn(D, B, H, generator=gen, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a, b: so.recurrence(a, T, B, b, lengths, dirs), (g, h0), eps=1e-6, atol=1e-7)


def test_recurrence_of_unit_gates_is_a_running_mean():
    """f = 1/2 everywhere: h_t = h_{t-1}/2 + z/2."""
    T, H = 6, 1
    g = torch.zeros(T, 3 * H, dtype=torch.float64)
    g[:, 1] = 0.7
    y, hT = so.recurrence(g, T, 1)
    z = math.tanh(0.7)
    assert torch.allclose(hT.flatten(), torch.tensor([z * (1 - 2.0 ** -T)], dtype=torch.float64), atol=1e-15)
    assert torch.allclose(y[:, 0], torch.tensor([0.5 * z * (1 - 2.0 ** -(t + 1)) for t in range(T)], dtype=torch.float64), atol=1e-15)


def test_log_probs_gradient_matches_differences():
    gen = torch.Generator().manual_seed(3)
    z = torch.randn(4, 6, generator=gen, dtype=torch.float64)
    z[1, 2] = -math.inf
    tok = torch.tensor([0, 5, -100, 3])
    gl, ge = torch.randn(4, generator=gen, dtype=torch.float64), torch.randn(4, generator=gen, dtype=torch.float64)

    def value(v):
        lp, H, _, _ = so.log_probs(v, tok)
        return float((lp * gl).sum() + (H * ge).sum())

    d = so.log_probs_grad(z, tok, gl, ge)
    for r in range(4):
        for c in range(6):
            if z[r, c] == -math.inf:
                assert d[r, c] == 0
                continue
            up, dn = z.clone(), z.clone()
            up[r, c] += 1e-6
            dn[r, c] -= 1e-6
            assert abs((value(up) - value(dn)) / 2e-6 - d[r, c].item()) < 1e-8


def test_dropout_stream_is_fair_and_apart():
    a = so.dropout_keep(20000, 0.3, 5, 0, 0)
    # 20000 draws at 0.7: 5 standard deviations are 5 sqrt(n p q) = 324
    assert abs(int(a.sum()) - 14000) < 324
    for other in ((6, 0, 0), (5, 1, 0), (5, 0, 1)):
        b = so.dropout_keep(20000, 0.3, *other)
        # independent masks agree with probability p^2 + q^2 = 0.58; 5 sigma = 349
        assert abs(int((a == b).sum()) - 11600) < 349
    assert so.dropout_keep(8, 0.0, 1, 2, 3).all()


def test_python_entries_refuse_cpu_tensors():
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.gated_recurrence(torch.zeros(4, 6), 2, 2)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.gated_recurrence_step(torch.zeros(4, 6), torch.zeros(4, 2))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.token_log_probs(torch.zeros(4, 6), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.dropout(torch.zeros(4), 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        ops.dropout([1.0], 0.5, torch.zeros(2, dtype=torch.int64))


P = 4096  # stands for a device pointer: the refusals below come before any launch


def _refused(name, *args):
    status = getattr(_lib.load(), name)(*args)
    assert status == 1, f"{name}{args} gave {status}"
    assert b"invalid argument" in _lib.load().avc_last_error()


@pytest.mark.parametrize("change", [
    dict(dtype=3), dict(dtype=-1), dict(T=0), dict(T=-1), dict(B=-1), dict(H=0), dict(dirs=0), dict(dirs=4), dict(ldg=11),
    dict(ldy=3), dict(gates=None), dict(y=None), dict(T=(1 << 30) + 1), dict(B=1 << 30, H=1 << 28, ldg=1 << 40, ldy=1 << 40)])
def test_recurrence_forward_refusals(change):
    a = dict(dtype=0, T=8, B=2, H=4, dirs=1, gates=P, ldg=12, ldy=4, y=P) | change
    _refused("avc_gated_recurrence_forward", a["dtype"], a["T"], a["B"], a["H"], a["dirs"], a["gates"], a["ldg"], None, None,
             a["y"], a["ldy"], None, None, None, 0, None)


def test_recurrence_needs_its_workspace():
    need = _lib.load().avc_gated_recurrence_workspace(0, 1 << 16, 1, 4, 1)
    assert need > 0
    _refused("avc_gated_recurrence_forward", 0, 1 << 16, 1, 4, 1, P, 12, None, None, P, 4, None, None, P, need - 1, None)
    _refused("avc_gated_recurrence_forward", 0, 1 << 16, 1, 4, 1, P, 12, None, None, P, 4, None, None, None, need, None)
    _refused("avc_gated_recurrence_backward", 0, 1 << 16, 1, 4, 1, P, 12, None, P, P, 4, None, P, 12, None, P, need - 1, None)


@pytest.mark.parametrize("change", [dict(states=None), dict(dy=None), dict(dgates=None), dict(lddg=11), dict(lddy=3), dict(dirs=3)])
def test_recurrence_backward_refusals(change):
    a = dict(dirs=1, states=P, dy=P, lddy=4, dgates=P, lddg=12) | change
    _refused("avc_gated_recurrence_backward", 0, 8, 2, 4, a["dirs"], P, 12, None, a["states"], a["dy"], a["lddy"], None,
             a["dgates"], a["lddg"], None, None, 0, None)


def test_recurrence_step_refusals():
    for bad in ((3, 2, 4, P, 12, P, P, P, 4), (0, -1, 4, P, 12, P, P, P, 4), (0, 2, 0, P, 12, P, P, P, 4), (0, 2, 4, P, 11, P, P, P, 4),
                (0, 2, 4, P, 12, P, P, P, 3), (0, 2, 4, None, 12, P, P, P, 4), (0, 2, 4, P, 12, None, P, P, 4), (0, 2, 4, P, 12, P, None, P, 4)):
        _refused("avc_gated_recurrence_step", *bad, None)


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(N=-1), dict(V=0), dict(ldz=9), dict(top=-1), dict(top=33), dict(top=11), dict(z=None), dict(tok=None),
    dict(top=2, topv=None), dict(N=(1 << 40) + 1), dict(V=(1 << 30) + 1, ldz=1 << 31)])
def test_log_probs_forward_refusals(change):
    a = dict(dtype=0, N=4, V=10, z=P, ldz=10, tok=P, top=0, topv=P) | change
    _refused("avc_token_log_probs_forward", a["dtype"], a["N"], a["V"], a["z"], a["ldz"], a["tok"], -100, a["top"], P, P, None,
             a["topv"], P, None, 0, None)


def test_log_probs_needs_its_workspace():
    need = _lib.load().avc_token_log_probs_workspace(0, 2, 100000, 5)
    assert need > 0
    _refused("avc_token_log_probs_forward", 0, 2, 100000, P, 100000, P, -100, 5, P, P, None, P, P, P, need - 1, None)
    _refused("avc_token_log_probs_forward", 0, 2, 100000, P, 100000, P, -100, 5, P, P, None, P, P, None, need, None)


def test_log_probs_backward_refusals():
    for z, ldz, tok, st, d, ldd in ((None, 10, P, P, P, 10), (P, 9, P, P, P, 10), (P, 10, None, P, P, 10), (P, 10, P, None, P, 10),
                                    (P, 10, P, P, None, 10), (P, 10, P, P, P, 9)):
        _refused("avc_token_log_probs_backward", 0, 4, 10, z, ldz, tok, -100, st, P, P, d, ldd, None)


@pytest.mark.parametrize("change", [
    dict(dtype=3), dict(rows=-1), dict(cols=-1), dict(p=1.0), dict(p=-0.1), dict(p=math.nan), dict(x=None), dict(rng=None), dict(y=None),
    dict(ldx=4), dict(ldy=4), dict(res=P, ldr=4), dict(rows=1 << 41), dict(rows=1 << 30, cols=1 << 30, ldx=1 << 30, ldy=1 << 30)])
def test_dropout_refusals(change):
    a = dict(dtype=0, rows=3, cols=5, x=P, ldx=5, res=None, ldr=0, p=0.5, rng=P, y=P, ldy=5) | change
    _refused("avc_dropout", a["dtype"], a["rows"], a["cols"], a["x"], a["ldx"], a["res"], a["ldr"], ctypes.c_double(a["p"]), a["rng"], 0,
             a["y"], a["ldy"], None)


def test_empty_calls_are_done():
    lib = _lib.load()
    assert lib.avc_gated_recurrence_forward(0, 4, 0, 3, 1, None, 9, None, None, None, 3, None, None, None, 0, None) == 0
    assert lib.avc_gated_recurrence_step(0, 0, 3, None, 9, None, None, None, 3, None) == 0
    assert lib.avc_token_log_probs_forward(0, 0, 3, None, 3, None, -100, 0, None, None, None, None, None, None, 0, None) == 0
    assert lib.avc_dropout(0, 0, 5, None, 5, None, 0, ctypes.c_double(0.5), None, 0, None, 5, None) == 0
