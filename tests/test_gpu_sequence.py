"""The sequence-model operators on the GPU against float64 restatements (oracle/sequence_oracle.py),
within the oracle's own error bounds plus the stored type's half step."""
import math

import numpy as np
import pytest
import torch

from autovc_amd import ops
from oracle import sequence_oracle as so

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def _near(got, ref, bound, what):
    got, ref = got.detach().cpu().double(), ref.detach()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got - ref).abs() - bound
    assert not torch.isnan(off).any(), what
    assert off.max().item() <= 0 if off.numel() else True, f"{what}: over the bound by {off.max().item():.3g} (bound {bound.max().item():.3g})"


def _gates(gen, T, B, D, H, dtype, dev, pad=0):
    g = torch.randn(T * B, D, 3, H, generator=gen)
    g[:, :, 0] = g[:, :, 0] * 1.5 + 1.5
    g = g.reshape(T * B, D * 3 * H).to(dtype)
    if not pad:
        return g, g.to(dev)
    wide = torch.full((T * B, D * 3 * H + pad), math.nan, dtype=dtype, device=dev)
    wide[:, 3:3 + D * 3 * H] = g.to(dev)
    return g, wide[:, 3:3 + D * 3 * H]


def _check_recurrence(dev, dtype, T, B, H, dirs, lengths=None, h0=False, pad=0, seed=0):
    D = 2 if dirs == 3 else 1
    gen = torch.Generator().manual_seed(1000 * T + 100 * B + H + dirs + seed)
    g, gd = _gates(gen, T, B, D, H, dtype, dev, pad)
    if lengths is not None:
        # whatever stands behind a sequence's end must not be seen
        for b, n in enumerate(lengths):
            for k, t in enumerate(range(max(n, 0), T)):
                gd[t * B + b] = (math.nan, math.inf, -math.inf, torch.finfo(dtype).min)[k % 4]
    h = torch.rand(D, B, H, generator=gen) * 2 - 1 if h0 else None
    dy = torch.randn(T * B, D * H, generator=gen).to(dtype)
    dhT = torch.randn(D, B, H, generator=gen)
    L = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)

    gr = g.double().requires_grad_(True)
    hr = h.double().requires_grad_(True) if h0 else None
    y, hT = so.recurrence(gr, T, B, hr, lengths, dirs)
    ref = torch.autograd.grad((y, hT), (gr, hr) if h0 else (gr,), (dy.double(), dhT.double()))
    Ey, EhT, Eg, Eh0 = so.recurrence_bounds(g, T, B, h, lengths, dirs, dy, dhT)

    # (the gates enter as a leaf's view, so that a column slice stays one)
    leaf = gd.detach().requires_grad_(True)
    hd = h.to(dev).requires_grad_(True) if h0 else None
    yd, hTd = ops.gated_recurrence(leaf, T, B, h0=hd, lengths=L, dirs=dirs)
    assert yd.dtype == dtype and hTd.dtype == torch.float32
    _near(yd, y, Ey + so.rounded(y.detach(), dtype), "y")
    _near(hTd, hT, EhT, "hT")
    with torch.no_grad():
        y2, hT2 = ops.gated_recurrence(gd, T, B, h0=None if h is None else h.to(dev), lengths=L, dirs=dirs)
    assert torch.equal(y2, yd) and torch.equal(hT2, hTd)
    got = torch.autograd.grad((yd, hTd), (leaf, hd) if h0 else (leaf,), (dy.to(dev), dhT.to(dev)))
    _near(got[0], ref[0], Eg + so.rounded(ref[0], dtype), "dgates")
    if h0:
        _near(got[1], ref[1], Eh0, "dh0")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T,B,H,dirs", [
    (1, 1, 1, 1), (1, 3, 5, 3), (2, 1, 3, 2), (7, 2, 4, 1), (8, 1, 2, 3), (9, 5, 7, 2), (63, 2, 50, 1), (64, 3, 32, 3),
    (65, 1, 33, 2), (128, 2, 130, 1), (130, 4, 16, 3), (200, 1, 257, 1), (20, 70, 9, 3)])
def test_recurrence(cuda_device, dtype, T, B, H, dirs):
    _check_recurrence(cuda_device, dtype, T, B, H, dirs, h0=(T + B) % 2 == 0)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T,B,H,dirs,lengths", [
    (5, 4, 6, 3, [0, 5, 1, 3]), (70, 3, 9, 2, [64, 0, 65]), (70, 3, 40, 1, [64, 70, 1]), (1, 2, 3, 3, [0, 1]),
    (129, 2, 3, 3, [128, 63]), (9, 3, 4, 3, [0, 0, 0]), (6, 3, 4, 1, [-3, 100, 2])])
@pytest.mark.parametrize("h0", [False, True])
def test_recurrence_ragged(cuda_device, dtype, T, B, H, dirs, lengths, h0):
    _check_recurrence(cuda_device, dtype, T, B, H, dirs, lengths, h0)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T,B,H,dirs,lengths", [
    (1000, 1, 5, 1, None), (1537, 2, 66, 3, [1537, 700]), (3000, 1, 1, 2, None), (5000, 2, 3, 3, [4999, 0])])
def test_recurrence_time_split_over_workgroups(cuda_device, dtype, T, B, H, dirs, lengths):
    from autovc_amd import _lib
    assert _lib.load().avc_gated_recurrence_workspace(_lib.DTYPES[dtype], T, B, H, dirs) > 0
    _check_recurrence(cuda_device, dtype, T, B, H, dirs, lengths, True)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("dirs", [1, 3])
def test_recurrence_of_column_slices(cuda_device, dtype, dirs):
    _check_recurrence(cuda_device, dtype, 40, 3, 21, dirs, [40, 2, 17], True, pad=7)


def test_recurrence_gates_at_their_ends(cuda_device):
    """Saturated and infinite gates: f = 1 keeps the state, f = 0 takes the candidate; the types'
    lowest and highest values are not special."""
    for dtype in TYPES:
        big = torch.finfo(dtype).max
        ends = [-math.inf, -big, -90.0, -85.0, 0.0, 85.0, 90.0, big, math.inf]
        g = torch.tensor([[f, c, 0.5] for f in ends for c in (-math.inf, -big, 1e-4, big, math.inf)], dtype=dtype)
        T = g.shape[0]
        y, hT = so.recurrence(g, T, 1, torch.full((1, 1, 1), 0.25))
        yd, hTd = ops.gated_recurrence(g.to(cuda_device), T, 1, h0=torch.full((1, 1, 1), 0.25, device=cuda_device))
        # |g| counts up to 90 here (beyond, f or 1 - f is below 1e-38): 102 + 12 units a frame
        _near(yd, y, torch.full_like(y, T * 114 * so.U) + so.rounded(y, dtype), "y")
        _near(hTd, hT, torch.full_like(hT, T * 114 * so.U), "hT")
        leaf = g.to(cuda_device).requires_grad_(True)
        out, _ = ops.gated_recurrence(leaf, T, 1)
        assert torch.isfinite(torch.autograd.grad(out.float().sum(), leaf)[0]).all()


def test_recurrence_nan_stays_in_its_channel(cuda_device):
    T, B, H = 40, 2, 9
    g = torch.randn(T * B, 3 * H, device=cuda_device)
    clean, _ = ops.gated_recurrence(g, T, B)
    for k in range(3):
        bad = g.clone()
        bad[10 * B + 1, k * H + 4] = math.nan
        y, hT = ops.gated_recurrence(bad, T, B)
        y, c = y.view(T, B, H), clean.view(T, B, H)
        hit = torch.zeros(T, B, H, dtype=torch.bool, device=cuda_device)
        hit[10:(11 if k == 2 else T), 1, 4] = True
        assert torch.equal(torch.isnan(y), hit)
        assert torch.equal(y[~hit], c[~hit])
        assert bool(torch.isnan(hT[0, 1, 4])) == (k != 2)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_recurrence_continues_from_its_state(cuda_device, dtype):
    """Two calls in turn, then single frames, give what one call over all frames gives."""
    T, B, H = 150, 3, 37
    gen = torch.Generator().manual_seed(5)
    g, gd = _gates(gen, T, B, 1, H, dtype, cuda_device)
    y, hT = so.recurrence(g, T, B)
    Ey, EhT, _, _ = so.recurrence_bounds(g, T, B)
    y1, h = ops.gated_recurrence(gd[:100 * B], 100, B)
    y2, h = ops.gated_recurrence(gd[100 * B:140 * B], 40, B, h0=h)
    state, ys = h[0].clone(), [y1, y2]
    for t in range(140, T):
        out, new = ops.gated_recurrence_step(gd[t * B:(t + 1) * B], state)
        same, inplace = ops.gated_recurrence_step(gd[t * B:(t + 1) * B], state, out_state=state)
        assert inplace is state and torch.equal(state, new) and torch.equal(out, same)
        ys.append(out)
    _near(torch.cat(ys), y, Ey + so.rounded(y, dtype), "y")
    _near(state[None], hT, EhT, "hT")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("B,H", [(1, 1), (1, 512), (5, 3), (70, 130), (3, 7)])
def test_recurrence_step(cuda_device, dtype, B, H):
    gen = torch.Generator().manual_seed(B * H)
    g, gd = _gates(gen, 1, B, 1, H, dtype, cuda_device, pad=5)
    h = torch.rand(B, H, generator=gen) * 2 - 1
    y, hT = so.recurrence(g, 1, B, h[None])
    Ey, EhT, _, _ = so.recurrence_bounds(g, 1, B, h[None])
    yd, hd = ops.gated_recurrence_step(gd, h.to(cuda_device))
    _near(yd, y, Ey + so.rounded(y, dtype), "y")
    _near(hd[None], hT, EhT, "state")


def test_recurrence_only_one_of_its_gradients(cuda_device):
    T, B, H = 30, 2, 5
    gen = torch.Generator().manual_seed(1)
    g, gd = _gates(gen, T, B, 1, H, torch.float32, cuda_device)
    dy, dhT = torch.randn(T * B, H, generator=gen), torch.randn(1, B, H, generator=gen)
    for which in (0, 1):
        gr = g.double().requires_grad_(True)
        out = so.recurrence(gr, T, B)[which]
        d = (dy, dhT)[which]
        ref = torch.autograd.grad(out, gr, d.double())[0]
        bound = so.recurrence_bounds(g, T, B, dy=dy if which == 0 else None, dhT=dhT if which == 1 else None)[2]
        leaf = gd.clone().requires_grad_(True)
        got = torch.autograd.grad(ops.gated_recurrence(leaf, T, B)[which], leaf, d.to(cuda_device))[0]
        _near(got, ref, bound + so.rounded(ref, torch.float32), "dgates")
    # a gradient that is one number spread over y (its rows overlap)
    leaf = gd.clone().requires_grad_(True)
    ops.gated_recurrence(leaf, T, B)[0].sum().backward()
    gr = g.double().requires_grad_(True)
    so.recurrence(gr, T, B)[0].sum().backward()
    bound = so.recurrence_bounds(g, T, B, dy=torch.ones(T * B, H))[2]
    _near(leaf.grad, gr.grad, bound + so.rounded(gr.grad, torch.float32), "dgates")


def test_recurrence_empty(cuda_device):
    h0 = torch.rand(1, 3, 4, device=cuda_device, requires_grad=True)
    y, hT = ops.gated_recurrence(torch.zeros(0, 12, device=cuda_device), 0, 3, h0=h0)
    assert y.shape == (0, 4) and torch.equal(hT, h0)
    y, hT = ops.gated_recurrence(torch.zeros(0, 24, device=cuda_device), 5, 0, dirs=3)
    assert y.shape == (0, 8) and hT.shape == (2, 0, 4)
    y, s = ops.gated_recurrence_step(torch.zeros(0, 12, device=cuda_device), torch.zeros(0, 4, device=cuda_device))
    assert y.shape == (0, 4) and s.shape == (0, 4)


def test_recurrence_past_32_bit_offsets(cuda_device):
    """Gate elements beyond 2^31: the last rows are what a call over those rows alone gives."""
    T, B, H = 3, 480_000, 512
    g = torch.empty(T * B, 3 * H, dtype=torch.bfloat16, device=cuda_device)
    assert g.numel() > 2 ** 31
    g.normal_(generator=torch.Generator(device=cuda_device).manual_seed(2))
    y, hT = ops.gated_recurrence(g, T, B, dirs=2)
    tail = g.view(T, B, 3 * H)[:, B - 5:].reshape(T * 5, 3 * H).contiguous()
    y2, hT2 = ops.gated_recurrence(tail, T, 5, dirs=2)
    assert torch.equal(y.view(T, B, H)[:, B - 5:].reshape(T * 5, H), y2) and torch.equal(hT[:, B - 5:], hT2)
    assert torch.isfinite(hT).all()


# ---- log-probabilities of given classes -----------------------------------------------------------
def _logits(gen, N, V, dtype, masked):
    z = torch.randn(N, V, generator=gen) * 2
    z[torch.arange(N), torch.randint(0, V, (N,), generator=gen)] += 6
    if masked:
        z[torch.rand(N, V, generator=gen) < 0.3] = -math.inf
        z[N - 1] = -math.inf
        if N > 2:
            z[1, :] = torch.finfo(dtype).min  # a mask of the type's lowest value over a whole row
            z[2, : V // 2] = torch.finfo(dtype).min
    return z.to(dtype)


def _check_log_probs(dev, z, tok, top, zd=None, ignore=-100):
    N, V = z.shape
    dtype = z.dtype
    gen = torch.Generator().manual_seed(N + V)
    gl, ge = torch.randn(N, generator=gen), torch.randn(N, generator=gen)
    logp, H, tl, ti = so.log_probs(z, tok, top, ignore)
    empty = (z == -math.inf).all(1)
    Elp, EH, Eg = so.log_probs_bounds(z, tok, gl, ge)
    d = so.log_probs_grad(z, tok, gl, ge, ignore)
    leaf = (z.to(dev) if zd is None else zd).detach().requires_grad_(True)
    got = ops.token_log_probs(leaf, tok.to(dev), top=top, ignore_index=ignore)
    at = tok.clamp(0, V - 1)
    b_lp = torch.where(tok == ignore, torch.zeros((), dtype=torch.float64), Elp.gather(1, at[:, None])[:, 0])
    fin = torch.isfinite(logp)
    lp = got[0].detach().cpu().double()
    assert torch.equal(torch.isnan(lp), torch.isnan(logp)) and torch.equal(lp == -math.inf, logp == -math.inf)
    _near(lp[fin], logp[fin], b_lp[fin] + so.rounded(logp[fin], torch.float32), "logp")
    _near(got[1][~empty], H[~empty], EH[~empty] + so.rounded(H[~empty], torch.float32), "entropy")
    assert (got[1].detach().cpu()[empty] == 0).all()
    if top:
        assert torch.equal(got[3].cpu(), ti)
        t = got[2].cpu().double()
        f = torch.isfinite(tl)
        assert torch.equal(t == -math.inf, tl == -math.inf)
        _near(t[f], tl[f], Elp.gather(1, ti)[f] + so.rounded(tl[f], torch.float32), "top_logp")
    dz = torch.autograd.grad((got[0], got[1]), leaf, (gl.to(dev), ge.to(dev)))[0]
    assert dz.dtype == dtype
    dz = dz.cpu().double()
    live = ~empty & ~torch.isnan(d).any(1)
    _near(dz[live], d[live], Eg[live] + so.rounded(d[live], dtype), "dlogits")
    assert torch.equal(torch.isnan(dz).all(1), torch.isnan(d).all(1)) and (dz[empty & ~torch.isnan(d).any(1)] == 0).all()
    with torch.no_grad():
        again = ops.token_log_probs(leaf, tok.to(dev), top=top, ignore_index=ignore)
    for a, b in zip(got, again):
        assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N,V,top", [
    (1, 1, 1), (3, 2, 2), (5, 18, 3), (2, 63, 32), (4, 64, 1), (7, 512, 5), (3, 1000, 0), (2, 2048, 32), (2, 2049, 32),
    (3, 4097, 8), (600, 2100, 2), (1, 20001, 20), (4, 70003, 32), (300, 40, 0)])
@pytest.mark.parametrize("masked", [False, True])
def test_log_probs(cuda_device, dtype, N, V, top, masked):
    gen = torch.Generator().manual_seed(N * V + top)
    z = _logits(gen, N, V, dtype, masked)
    tok = torch.randint(0, V, (N,), generator=gen)
    if N > 3:
        tok[0], tok[3] = -100, -100
    _check_log_probs(cuda_device, z, tok, top)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N,V,top", [
    (4096, 1, 1), (4097, 7, 0), (4099, 40, 32), (4100, 128, 9), (4111, 129, 0), (4096, 256, 16), (4101, 257, 5), (4096, 300, 8),
    (4098, 512, 20), (4096, 511, 32), (4097, 513, 3)])
@pytest.mark.parametrize("masked", [False, True])
def test_log_probs_many_short_rows(cuda_device, dtype, N, V, top, masked):
    gen = torch.Generator().manual_seed(N * V + top)
    z = _logits(gen, N, V, dtype, masked)
    tok = torch.randint(0, V, (N,), generator=gen)
    tok[0], tok[3] = -100, -100
    _check_log_probs(cuda_device, z, tok, top)


@pytest.mark.parametrize("top", [0, 1, 8, 16, 32])
def test_log_probs_many_short_rows_of_every_kind(cuda_device, top):
    """Neighbouring rows that share a wave and need different things: equal classes, fewer classes left
    than are wanted, none, the largest classes side by side or rising, NaN and infinity, confident rows."""
    N, V = 4099, 500
    gen = torch.Generator().manual_seed(top)
    z = torch.randn(N, V, generator=gen)
    z[1::11] = 0.25
    z[2::11] = torch.randint(0, 3, (len(z[2::11]), V), generator=gen).float()
    z[3::11, 5:] = -math.inf
    z[4::11] = -math.inf
    z[5::11] = torch.linspace(-4, 4, V)
    for c in range(8):  # the classes that one lane of 16 holds in fours
        z[6::11, 24 + 64 * c:min(28 + 64 * c, V)] += 9.0
    z[7::11] = torch.where(torch.rand(len(z[7::11]), V, generator=gen) < 0.97, torch.tensor(-math.inf), z[7::11])
    z[8::11, 100] = 25.0
    z[9::11, 3] = -0.0
    z[9::11, 2] = 0.0
    z[9::11, 4:] = -1.0
    tok = torch.randint(0, V, (N,), generator=gen)
    _check_log_probs(cuda_device, z, tok, top)
    z[10::11, 7] = math.nan
    z[21::11, 400] = math.inf
    tok[::5], tok[1::5] = V, -1
    logp, H, tl, ti = so.log_probs(z, tok, top)
    got = ops.token_log_probs(z.to(cuda_device), tok.to(cuda_device), top=top)
    assert torch.equal(torch.isnan(got[0].cpu()), torch.isnan(logp)) and torch.equal(torch.isnan(got[1].cpu()), torch.isnan(H))
    assert torch.equal(got[3].cpu(), ti) and torch.equal(torch.isnan(got[2].cpu()), torch.isnan(tl))


@pytest.mark.parametrize("top", [8, 16, 32])
def test_log_probs_many_short_rows_with_their_classes_in_few_lanes(cuda_device, top):
    """More classes left than a row's list holds, all in three of its 16 lanes, beside rows with none
    ruled out."""
    N, V = 4096, 512
    gen = torch.Generator().manual_seed(top)
    z = torch.randn(N, V, generator=gen)
    lane = torch.arange(V) // 4 % 16
    z[1::3] = torch.where((lane >= 1) & (lane <= 3), z[1::3], torch.tensor(-math.inf))
    z[5::9] = torch.where(lane == 9, z[5::9].round(), z[5::9] - 20.0)
    _check_log_probs(cuda_device, z, torch.randint(0, V, (N,), generator=gen), top)


def test_log_probs_of_many_confident_short_rows(cuda_device):
    """As test_log_probs_of_confident_rows: 64 classes a lane at most and four joins."""
    N, V = 4096, 400
    gen = torch.Generator().manual_seed(V)
    z = torch.randn(N, V, generator=gen)
    top = torch.randint(0, V, (N,), generator=gen)
    z[torch.arange(N), top] = z.max() + torch.linspace(2.0, 22.0, N) + math.log(V)
    logp, H, _, _ = so.log_probs(z, top)
    got = ops.token_log_probs(z.to(cuda_device), top.to(cuda_device))
    rel = 350 * so.U
    _near(got[0], logp, rel * logp.abs(), "logp")
    _near(got[1], H, rel * H, "entropy")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_log_probs_ties_go_to_the_lower_class(cuda_device, dtype):
    for V in (40, 512, 3001, 50001):
        z = torch.zeros(3, V, dtype=dtype)
        z[1, ::7] = 1.0
        z[2] = torch.where(torch.arange(V) % 2 == 0, torch.tensor(0.0), torch.tensor(-0.0)).to(dtype)
        _check_log_probs(cuda_device, z, torch.zeros(3, dtype=torch.int64), 32)


@pytest.mark.parametrize("V", [2000, 30000, 300000])
def test_log_probs_with_large_classes_in_few_slices(cuda_device, V):
    """Every large class in the slices of a few threads, more of them than are ranked at once."""
    dtype = torch.float32
    for period in (256, 1024):  # a wave's and a workgroup's stride over fp32 vectors
        z = torch.full((2, V), -3.0, dtype=dtype)
        c = torch.arange(V)
        for k in range(2):
            hot = (c % period) < 32
            z[k, hot] = (c[hot] % 977).to(dtype) / 977 + k
        _check_log_probs(cuda_device, z, torch.tensor([5, 6]), 32)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_log_probs_rows_of_a_wider_buffer(cuda_device, dtype):
    gen = torch.Generator().manual_seed(8)
    for N, V in ((5, 33), (3, 5001)):
        z = _logits(gen, N, V, dtype, False)
        wide = torch.full((N, V + 9), math.nan, dtype=dtype, device=cuda_device)
        wide[:, 3:3 + V] = z.to(cuda_device)
        _check_log_probs(cuda_device, z, torch.randint(0, V, (N,), generator=gen), 4, wide[:, 3:3 + V])


def test_log_probs_nan_inf_and_bad_tokens(cuda_device):
    for V in (50, 9000):
        z = torch.randn(6, V, generator=torch.Generator().manual_seed(V))
        z[1, 7], z[2, V - 1], z[3, 0] = math.nan, math.inf, math.nan
        z[3, 1:] = -math.inf
        tok = torch.tensor([3, 3, 3, 3, V, -1])
        leaf = z.to(cuda_device).requires_grad_(True)
        logp, H, tl, ti = ops.token_log_probs(leaf, tok.to(cuda_device), top=5)
        assert torch.isnan(logp).tolist() == [False, True, True, True, True, True]
        assert torch.isnan(H).tolist() == [False, True, True, True, False, False]
        assert torch.equal(ti.cpu(), so.log_probs(z, tok, 5)[3])
        assert torch.isnan(tl).all(1).tolist() == [False, True, True, True, False, False]
        d = torch.autograd.grad(logp.sum(), leaf)[0]
        assert torch.isnan(d).all(1).tolist() == [False, True, True, True, True, True]
        # a token outside that is the ignored one is no mistake
        assert ops.token_log_probs(z[:1].to(cuda_device), torch.tensor([-1], device=cuda_device), ignore_index=-1)[0].item() == 0


@pytest.mark.parametrize("V", [2, 40, 3000, 40000])
def test_log_probs_of_confident_rows(cuda_device, V):
    """Rows whose largest class leaves the others 1e-2 .. 1e-14: entropy, log-probability and gradient
    keep their relative precision (in a sum that begins with the largest class's 1 they would not)."""
    gen = torch.Generator().manual_seed(V)
    z = torch.randn(16, V, generator=gen)
    top = torch.randint(0, V, (16,), generator=gen)
    z[torch.arange(16), top] = z.max() + torch.linspace(2.0, 22.0, 16) + math.log(V)
    logp, H, _, _ = so.log_probs(z, top)
    leaf = z.to(cuda_device).requires_grad_(True)
    got = ops.token_log_probs(leaf, top.to(cuda_device))
    # every term of these sums of like signs is off by (|d| + 3) U and each of at most 300 additions by
    # one: all of it relative to the result, |d| <= 45 here
    rel = 350 * so.U
    _near(got[0], logp, rel * logp.abs(), "logp")
    _near(got[1], H, rel * H, "entropy")
    ones = torch.ones(16)
    for gl, ge in ((ones, 0 * ones), (0 * ones, ones)):
        d = torch.autograd.grad((got[0], got[1]), leaf, (gl.to(cuda_device), ge.to(cuda_device)), retain_graph=True)[0].cpu().double()
        ref = so.log_probs_grad(z, top, gl, ge)
        hot = torch.zeros(16, V, dtype=torch.bool)
        hot[torch.arange(16), top] = True
        # dlogp: 1 - p at the token, -p elsewhere; dentropy: p (|d| - mean) with |d| far above mean
        # elsewhere, p mean at the token
        assert ((d - ref).abs() <= 2 * rel * ref.abs())[hot if gl[0] else ~hot].all()
        assert ((d - ref).abs() <= 2 * rel * ref.abs())[hot].all()


def test_log_probs_shapes_and_gradients_of_one_output(cuda_device):
    gen = torch.Generator().manual_seed(4)
    z, tok = torch.randn(2, 3, 20, generator=gen), torch.randint(0, 20, (2, 3), generator=gen)
    leaf = z.to(cuda_device).requires_grad_(True)
    logp, H, tl, ti = ops.token_log_probs(leaf, tok.to(cuda_device, torch.int32), top=2)
    assert logp.shape == H.shape == (2, 3) and tl.shape == ti.shape == (2, 3, 2)
    assert not tl.requires_grad and not ti.requires_grad
    zr = z.view(6, 20)
    for out, gl, ge in ((logp, 1.0, 0.0), (H, 0.0, 1.0)):
        d = torch.autograd.grad(out.sum(), leaf, retain_graph=True)[0]
        one = torch.full((6,), 1.0)
        ref = so.log_probs_grad(zr, tok.view(6), one * gl, one * ge)
        bound = so.log_probs_bounds(zr, tok.view(6), one * gl, one * ge)[2]
        _near(d.view(6, 20), ref, bound + so.rounded(ref, torch.float32), "dlogits")
    one = ops.token_log_probs(leaf[0, 0], tok[0, 0].to(cuda_device))
    assert one[0].shape == () and torch.equal(one[0], logp[0, 0])
    e = ops.token_log_probs(torch.zeros(0, 5, device=cuda_device), torch.zeros(0, dtype=torch.int64, device=cuda_device), top=2)
    assert e[0].shape == (0,) and e[3].shape == (0, 2)


@pytest.mark.parametrize("V", [3, 600])
def test_log_probs_of_more_rows_than_a_launch_takes(cuda_device, V):
    """Rows go in several launches: every row has what it has in a call of its neighbours alone."""
    N = 2 ** 25 + 11
    z = torch.empty(N, V, dtype=torch.float16, device=cuda_device)
    z.normal_(generator=torch.Generator(device=cuda_device).manual_seed(9)).requires_grad_(True)
    tok = torch.arange(N, device=cuda_device) % V
    got = ops.token_log_probs(z, tok, top=2)
    gl = torch.linspace(-1, 1, N, device=cuda_device)
    dz, = torch.autograd.grad((got[0], got[1]), z, (gl, gl.flip(0)))
    edges = [-(-N // -(-N // most)) for most in (2 ** 23, 2 ** 25)]  # the first parts' ends, forward and backward
    for lo in (0, edges[0] - 2500, edges[1] - 2500, N - 5000):
        rows = slice(lo, lo + 5000)
        part = z.detach()[rows].clone().requires_grad_(True)
        want = ops.token_log_probs(part, tok[rows], top=2)
        for a, b in zip(got, want):
            assert torch.equal(a[rows], b)
        d, = torch.autograd.grad(want[:2], part, (gl[rows], gl.flip(0)[rows]))
        assert torch.equal(dz[rows], d)
    assert bool((got[0] <= 0).all()) and bool((got[1] > 0).all())


def test_log_probs_past_32_bit_offsets(cuda_device):
    N, V = 45_000, 50_001
    z = torch.empty(N, V, dtype=torch.bfloat16, device=cuda_device)
    assert z.numel() > 2 ** 31
    z.normal_(generator=torch.Generator(device=cuda_device).manual_seed(2))
    tok = torch.full((N,), V - 1, device=cuda_device)
    a, b = ops.token_log_probs(z, tok, top=3), ops.token_log_probs(z[-600:].clone(), tok[-600:], top=3)
    assert torch.equal(a[3][-600:], b[3])
    # the two calls may lay rows over the chip differently: each is within the oracle's bound of the
    # exact value, so they are within twice that of each other
    Elp, EH, _ = so.log_probs_bounds(z[-20:].cpu(), tok[-20:].cpu())
    half = [so.rounded(x[-20:].cpu().double(), torch.float32) for x in a[:3]]
    _near(a[0][-20:], b[0][-20:].cpu().double(), 2 * (Elp[:, V - 1] + half[0]), "logp")
    _near(a[1][-20:], b[1][-20:].cpu().double(), 2 * (EH + half[1]), "entropy")
    _near(a[2][-20:], b[2][-20:].cpu().double(), 2 * (Elp.gather(1, a[3][-20:].cpu()) + half[2]), "top_logp")


# ---- counter-based dropout --------------------------------------------------------------------------
def _rng(dev, seed=12345, steps=3):
    return torch.tensor([seed, steps], dtype=torch.int64, device=dev)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1,), (7,), (3, 5), (1, 8), (64, 33), (5, 1), (1000, 3), (2, 3, 11), (17, 1025), (3, 9000), ()])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(cuda_device, dtype, shape, residual):
    p, layer = 0.3, 9
    gen = torch.Generator().manual_seed(len(shape) + (shape[-1] if shape else 0))
    x = torch.randn(shape, generator=gen).to(dtype)
    r = torch.randn(shape, generator=gen).to(dtype) if residual else None
    dy = torch.randn(shape, generator=gen).to(dtype)
    keep = so.dropout_keep(x.numel(), p, 12345, 3, layer).view(shape).double() / (1 - p)
    leaf = x.to(cuda_device).requires_grad_(True)
    res = r.to(cuda_device).requires_grad_(True) if residual else None
    y = ops.dropout(leaf, p, _rng(cuda_device), residual=res, layer=layer)
    ref = x.double() * keep + (r.double() if residual else 0)
    # the scale's rounding, the product's and the sum's
    bound = 2 * so.U * (x.double() * keep).abs() + so.U * ref.abs()
    _near(y, ref, bound + so.rounded(ref, dtype), "y")
    assert residual or torch.equal(y.detach().cpu() == 0, (keep == 0) | (x == 0))
    got = torch.autograd.grad(y, (leaf, res) if residual else (leaf,), dy.to(cuda_device))
    ref = dy.double() * keep
    _near(got[0], ref, 2 * so.U * ref.abs() + so.rounded(ref, dtype), "dx")
    if residual:
        assert torch.equal(got[1].cpu(), dy)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(5, 3), (9, 16), (33, 777), (4, 2), (700, 21)])
def test_dropout_mask_goes_by_element_not_by_place(cuda_device, dtype, rows, cols):
    """Column slices of wider buffers, transposed tensors and dense ones get the same mask."""
    x = torch.randn(rows, cols + 5, generator=torch.Generator().manual_seed(rows)).to(dtype).to(cuda_device)
    part = x[:, 3:3 + cols]
    want = ops.dropout(part.contiguous(), 0.5, _rng(cuda_device))
    assert torch.equal(ops.dropout(part, 0.5, _rng(cuda_device)), want)
    assert torch.equal(ops.dropout(part, 0.5, _rng(cuda_device), residual=part), want + part)
    turned = part.t().contiguous().t()
    assert torch.equal(ops.dropout(turned, 0.5, _rng(cuda_device)), want)
    leaf = part.detach().requires_grad_(True)
    d = torch.autograd.grad(ops.dropout(leaf, 0.5, _rng(cuda_device)), leaf, part)[0]
    assert torch.equal(d, want)


def test_dropout_words_and_ends(cuda_device):
    x = torch.ones(4099, device=cuda_device)
    base = ops.dropout(x, 0.5, _rng(cuda_device))
    assert torch.equal(base, ops.dropout(x, 0.5, _rng(cuda_device)))
    for other in (ops.dropout(x, 0.5, _rng(cuda_device, steps=4)), ops.dropout(x, 0.5, _rng(cuda_device, seed=-1)),
                  ops.dropout(x, 0.5, _rng(cuda_device), layer=1)):
        # independent masks differ at half of 4099 elements; 5 standard deviations are 160
        assert abs(int((other != base).sum()) - 2050) < 160
    assert torch.equal(ops.dropout(x, 0.0, _rng(cuda_device)), x)
    odd = torch.full((6,), math.inf, device=cuda_device)
    got = ops.dropout(odd, 0.5, _rng(cuda_device))  # a dropped infinity is 0, not NaN
    assert torch.equal(got == 0, base[:6] == 0) and not torch.isnan(got).any()
    assert ops.dropout(torch.zeros(0, 5, device=cuda_device), 0.5, _rng(cuda_device)).shape == (0, 5)
    assert ops.dropout(torch.zeros(3, 0, device=cuda_device), 0.5, _rng(cuda_device)).shape == (3, 0)
    seed = -(1 << 63)
    keep = so.dropout_keep(4099, 0.25, seed & ((1 << 64) - 1), (1 << 64) - 1, (1 << 32) - 1)
    got = ops.dropout(x, 0.25, _rng(cuda_device, seed=seed, steps=-1), layer=(1 << 32) - 1)
    assert torch.equal(got.cpu() != 0, keep)


def test_dropout_refuses_a_changed_stream_in_the_backward(cuda_device):
    x = torch.ones(8, device=cuda_device, requires_grad=True)
    rng = _rng(cuda_device)
    y = ops.dropout(x, 0.5, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_dropout_past_32_bit_offsets(cuda_device):
    n = (1 << 32) + 4099
    x = torch.ones(n, dtype=torch.float16, device=cuda_device)
    y = ops.dropout(x, 0.5, _rng(cuda_device, 7, 1))
    M, G = (1 << 64) - 1, 0x9E3779B97F4A7C15

    def mix(v):
        v = ((v ^ (v >> 30)) * 0xBF58476D1CE4E5B9) & M
        v = ((v ^ (v >> 27)) * 0x94D049BB133111EB) & M
        return v ^ (v >> 31)

    key = mix((mix((mix((7 + G) & M) + 1) & M)) & M)
    tail = y[-4099:].cpu().tolist()
    for k in (0, 1, 2, 2047, 4096, 4097, 4098):
        e = n - 4099 + k
        w = mix((key + (e // 2 + 1) * G) & M)
        assert (tail[k] != 0) == (((w >> 32 if e & 1 else w & 0xFFFFFFFF)) >= 1 << 31)


# ---- together, and as programs run them -------------------------------------------------------------
def _stack(params, x, tok, rng, T, B, lengths, double=None):
    """projection -> recurrence in both directions -> dropout on the residual path -> class scores."""
    w1, b1, w2, b2 = params
    if double is None:
        g = ops.Linear.apply(x, w1, b1)
        y, hT = ops.gated_recurrence(g, T, B, lengths=lengths, dirs=3)
        y = ops.dropout(y, 0.25, rng, residual=x, layer=1)
        z = ops.Linear.apply(y, w2, b2)
        logp, H, _, _ = ops.token_log_probs(z, tok)
        return -(logp.sum() + 0.05 * H.sum()) / (T * B) + hT.square().sum() * 0.01
    y, hT = so.recurrence(x @ w1.t() + b1, T, B, None, lengths, 3)
    z = (x + y * double) @ w2.t() + b2
    lp = torch.log_softmax(z, 1)
    picked = torch.stack([lp[r, t] if t >= 0 else lp[r, 0] * 0 for r, t in enumerate(tok.tolist())])
    H = -(lp.exp() * lp).sum(1)
    return -(picked.sum() + 0.05 * H.sum()) / (T * B) + hT.square().sum() * 0.01


def _stack_inputs(T, B, H, V):
    gen = torch.Generator().manual_seed(11)
    x = torch.randn(T * B, 2 * H, generator=gen)
    params = [torch.randn(6 * H, 2 * H, generator=gen) / math.sqrt(2 * H), torch.randn(6 * H, generator=gen),
              torch.randn(V, 2 * H, generator=gen) / math.sqrt(2 * H), torch.zeros(V)]
    tok = torch.randint(0, V, (T * B,), generator=gen)
    tok[5] = -100
    return x, params, tok


def test_operators_together(cuda_device):
    """One training step of a layer made of them: loss and every gradient against float64."""
    T, B, H, V = 70, 3, 16, 40
    lengths = [70, 0, 33]
    x, params, tok = _stack_inputs(T, B, H, V)
    keep = so.dropout_keep(T * B * 2 * H, 0.25, 77, 2, 1).view(T * B, 2 * H).double() / 0.75
    ref_p = [p.double().requires_grad_(True) for p in params]
    ref_x = x.double().requires_grad_(True)
    ref = _stack(ref_p, ref_x, tok, None, T, B, lengths, keep)
    ref_g = torch.autograd.grad(ref, ref_p + [ref_x])
    dp = [p.to(cuda_device).requires_grad_(True) for p in params]
    dx = x.to(cuda_device).requires_grad_(True)
    loss = _stack(dp, dx, tok.to(cuda_device), _rng(cuda_device, 77, 2), T, B, torch.tensor(lengths, device=cuda_device))
    got = torch.autograd.grad(loss, dp + [dx])
    # three products of K <= 210 terms and the operators in fp32, each off by at most a few hundred
    # units of the largest sum of magnitudes: 2000 units of each tensor's own largest value
    assert abs(loss.item() - ref.item()) <= 2000 * so.U * abs(ref.item())
    for a, b in zip(got, ref_g):
        _near(a, b, torch.full_like(b, 2000 * so.U * b.abs().max().item()), "gradient")


def test_operators_captured_and_replayed(cuda_device):
    """A captured training step (forward, backward, the generator's count) replayed with eager work
    between: every replay is what the eager step gives, with a new mask each time."""
    T, B, H, V = 200, 2, 8, 3000
    x, params, tok = _stack_inputs(T, B, H, V)
    dev = cuda_device
    x, tok = x.to(dev), tok.to(dev)
    lengths = torch.tensor([200, 150], dtype=torch.int32, device=dev)
    p_eager = [p.to(dev).requires_grad_(True) for p in params]
    rng_e, rng = _rng(dev, 5, 0), _rng(dev, 5, 0)

    def recurrent(g, xx, r):
        y, hT = ops.gated_recurrence(g, T, B, lengths=lengths, dirs=3)
        y = ops.dropout(y, 0.25, r, residual=xx, layer=1)
        z = y.repeat(1, V // (2 * H) + 1)[:, :V]
        logp, ent, tl, ti = ops.token_log_probs(z, tok, top=4)
        return y, hT, logp, ent, tl, ti

    def step(g, r):
        out = recurrent(g, x, r)
        d = torch.autograd.grad((out[2], out[3], out[1]), g, (ones, ones, torch.ones_like(out[1])))[0]
        r[1] += 1
        return [o.detach() for o in out] + [d]

    ones = torch.ones(T * B, device=dev)
    gates = torch.randn(T * B, 6 * H, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step(gates.clone().requires_grad_(True), _rng(dev))
    torch.cuda.current_stream().wait_stream(s)
    static = gates.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static, rng)
    del p_eager
    seen = []
    for k in range(4):
        fresh = torch.randn(T * B, 6 * H, device=dev)
        with torch.no_grad():
            static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        want = step(fresh.clone().requires_grad_(True), rng_e)
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), k
        assert rng.tolist() == rng_e.tolist() == [5, k + 1]
        seen.append((outs[0] == x).clone())
    assert not torch.equal(seen[0], seen[1])


def test_operators_on_two_streams(cuda_device):
    """Two streams at once, each with its own workspaces: what one after the other gives."""
    dev = cuda_device
    jobs = []
    for k in range(2):
        gen = torch.Generator(device=dev).manual_seed(k)
        jobs.append((torch.randn(4000, 30, device=dev, generator=gen), torch.randn(3, 40001, device=dev, generator=gen),
                     torch.arange(3, device=dev)))

    def work(g, z, tok):
        return list(ops.gated_recurrence(g, 4000, 1)) + list(ops.token_log_probs(z, tok, top=6)) + [ops.dropout(g, 0.5, _rng(dev))]

    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(work(*jobs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for run in got[k]:
            for a, b in zip(run, want[k]):
                assert torch.equal(a, b)


def test_refusals(cuda_device):
    dev = cuda_device
    g, tok = torch.zeros(8, 12, device=dev), torch.zeros(8, dtype=torch.int64, device=dev)
    for bad in (dict(T=3), dict(B=3), dict(dirs=0), dict(dirs=4), dict(h0=torch.zeros(1, 2, 5, device=dev)), dict(h0=torch.zeros(2, 4, device=dev)),
                dict(lengths=torch.zeros(3, dtype=torch.int32, device=dev)), dict(T=-4, B=-2)):
        with pytest.raises(ValueError):
            ops.gated_recurrence(g, **({"T": 4, "B": 2} | bad))
    for bad in (dict(h0=torch.zeros(1, 2, 4, dtype=torch.float16, device=dev)), dict(lengths=torch.zeros(2, device=dev))):
        with pytest.raises(TypeError):
            ops.gated_recurrence(g, 4, 2, **bad)
    with pytest.raises(TypeError):
        ops.gated_recurrence(g.double(), 4, 2)
    with pytest.raises(RuntimeError):
        ops.gated_recurrence(g, 4, 2, lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.gated_recurrence(torch.zeros(8, 11, device=dev), 4, 2)
    with pytest.raises(ValueError):
        ops.gated_recurrence(torch.zeros(8, 0, device=dev), 4, 2)
    s = torch.zeros(8, 4, device=dev)
    for bad in (dict(state=torch.zeros(8, 5, device=dev)), dict(out_state=torch.zeros(7, 4, device=dev)),
                dict(out_state=torch.zeros(4, 8, device=dev).t())):
        with pytest.raises(ValueError):
            ops.gated_recurrence_step(g, **({"state": s} | bad))
    buf = torch.zeros(9, 4, device=dev)
    with pytest.raises(ValueError):
        ops.gated_recurrence_step(g, buf[:8], out_state=buf[1:])
    with pytest.raises(RuntimeError):
        ops.gated_recurrence_step(g.clone().requires_grad_(True), s)
    for bad in (dict(top=-1), dict(top=13), dict(top=33), dict(tokens=tok[:7]), dict(tokens=tok.view(2, 4))):
        with pytest.raises(ValueError):
            ops.token_log_probs(g, **({"tokens": tok} | bad))
    with pytest.raises(ValueError):
        ops.token_log_probs(torch.zeros(8, 0, device=dev), tok)
    with pytest.raises(TypeError):
        ops.token_log_probs(g, tok.float())
    with pytest.raises(TypeError):
        ops.token_log_probs(g.double(), tok)
    r = _rng(dev)
    for bad in (dict(p=1.0), dict(p=-0.5), dict(p=math.nan), dict(layer=-1), dict(layer=1 << 32), dict(rng=r[:1]),
                dict(residual=torch.zeros(8, 11, device=dev))):
        with pytest.raises(ValueError):
            ops.dropout(g, **({"p": 0.5, "rng": r} | bad))
    for bad in (dict(rng=r.float()), dict(residual=torch.zeros(8, 12, dtype=torch.float16, device=dev))):
        with pytest.raises(TypeError):
            ops.dropout(g, **({"p": 0.5, "rng": r} | bad))


def test_gradients_are_differentiable_once(cuda_device):
    """create_graph is allowed; using the graph of a gradient is an error, not a silent zero."""
    dev = cuda_device
    g = torch.randn(12, 9, device=dev, requires_grad=True)
    w = torch.randn(12, 3, device=dev, requires_grad=True)
    calls = [lambda: ops.gated_recurrence(g, 6, 2)[0] * w, lambda: ops.dropout(g, 0.5, _rng(dev))[:, :3] * w,
             lambda: ops.token_log_probs(g, torch.zeros(12, dtype=torch.int64, device=dev))[0][:, None] * w]
    for call in calls:
        d = torch.autograd.grad(call().sum(), g)[0]
        d2 = torch.autograd.grad(call().sum(), g, create_graph=True)[0]
        assert torch.equal(d, d2.detach()) and d2.requires_grad
        with pytest.raises(RuntimeError, match="differentiate twice"):
            torch.autograd.grad(d2.sum(), w)


def test_dropout_hands_the_residuals_gradient_through(cuda_device):
    """The incoming gradient is the residual's own: it stays what it was (a leaf here), and a graph
    through it goes on."""
    dev = cuda_device
    x, res, w = (torch.randn(4, 6, device=dev, requires_grad=True) for _ in range(3))
    y = ops.dropout(x, 0.5, _rng(dev), residual=res)
    dx, dres = torch.autograd.grad(y, (x, res), w, create_graph=True)
    assert w.is_leaf and w.grad_fn is None
    assert torch.equal(dres, w)
    dw, = torch.autograd.grad((dres * dres).sum(), w)
    assert torch.equal(dw, 2 * w)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        torch.autograd.grad(dx.sum(), w)


def test_step_refuses_an_out_state_that_requires_a_gradient(cuda_device):
    dev = cuda_device
    s = torch.zeros(2, 4, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="out_state"):
        ops.gated_recurrence_step(torch.zeros(2, 12, device=dev), torch.zeros(2, 4, device=dev), out_state=s)
    with torch.no_grad():
        ops.gated_recurrence_step(torch.zeros(2, 12, device=dev), torch.ones(2, 4, device=dev), out_state=s)
    assert torch.equal(s.detach(), torch.full((2, 4), 0.5, device=dev))
