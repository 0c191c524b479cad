"""The sequence-model operators at the edges of their range, against the float64 oracle."""
import math

import pytest
import torch

from autovc_amd import _lib, ops
from oracle import sequence_oracle as so
from tests.test_gpu_sequence import IDS, TYPES, _check_log_probs, _check_recurrence, _near, _rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("N,V", [(5, 512), (6, 2048), (5, 4097), (5, 70003), (4096, 512), (4097, 700)])
def test_log_probs_of_classes_a_subnormal_apart(cuda_device, dtype, N, V):
    """Differences to the row's largest logit below 2^-126: every class counts, whichever thread has it."""
    gen = torch.Generator().manual_seed(V)
    z = torch.full((N, V), -100.0)
    z[0, 0], z[0, V // 2] = 0.0, -2.0 ** -127
    z[1] = -math.inf
    z[1, 0], z[1, [8 * k + 3 for k in range(1, 8)]] = 0.0, -2.0 ** -127
    z[2, [5, V // 3, V // 2, V - 2]] = torch.tensor([2.0e-38, 1.4e-38, 1.5e-38, 1.6e-38])  # all normal numbers
    z[3:] = torch.rand(N - 3, V, generator=gen) * 2.0 ** -126
    z[4] = torch.where(torch.rand(V, generator=gen) < 0.9, torch.tensor(-math.inf), z[4])
    tok = torch.randint(0, V, (N,), generator=gen)
    tok[:3] = torch.tensor([V // 2, 11, 5])
    _check_log_probs(cuda_device, z.to(dtype), tok, 4)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N,V", [(1, 130), (2, 200), (3, 248), (2, 124), (3, 3 * 4096 + 200), (2, 2 ** 16 + 216)])
def test_log_probs_with_fewer_slices_than_alternatives(cuda_device, dtype, N, V):
    """Rows, and last segments of rows, of fewer vectors than alternatives, with and without equal classes."""
    gen = torch.Generator().manual_seed(V)
    tok = torch.randint(0, V, (N,), generator=gen)
    for z in (torch.randn(N, V, generator=gen), torch.randint(0, 3, (N, V), generator=gen).float(),
              torch.linspace(-2, 2, V).expand(N, V), torch.randn(N, V, generator=gen).masked_fill(torch.arange(V) % 3 > 0, -math.inf)):
        for top in (17, 31, 32):
            _check_log_probs(cuda_device, z.to(dtype), tok, top)


@pytest.mark.parametrize("dtype,N,V", [(torch.float32, 12007, 440), (torch.float32, 12000, 300), (torch.bfloat16, 8200, 500),
                                       (torch.float16, 8192, 512), (torch.float16, 4100, 384)])
@pytest.mark.parametrize("top", [17, 32])
def test_log_probs_many_short_rows_with_many_alternatives(cuda_device, dtype, N, V, top):
    """Neighbouring rows of different kinds where 16 lanes hold a row and rank from their four largest each."""
    gen = torch.Generator().manual_seed(V + top)
    z = torch.randn(N, V, generator=gen)
    z[1::9] = 0.25
    z[2::9] = torch.randint(0, 3, (len(z[2::9]), V), generator=gen).float()
    z[3::9, 5:] = -math.inf
    z[4::9] = -math.inf
    z[5::9] = torch.linspace(-4, 4, V)
    lane = torch.arange(V) // (4 if dtype == torch.float32 else 8) % 16
    z[6::9] = torch.where((lane >= 1) & (lane <= 3), z[6::9], torch.tensor(-math.inf))
    z[7::9] = torch.where(lane == 9, z[7::9].round(), z[7::9] - 20.0)
    z[8::9, 100] = 25.0
    _check_log_probs(cuda_device, z.to(dtype), torch.randint(0, V, (N,), generator=gen), top)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_recurrence_state_of_small_candidates(cuda_device, dtype):
    """The fp32 state of one frame is as exact for 16-bit gates as for fp32 ones: with the forget gate at 1/2
    the state is tanh(c) / 2, off by at most 16 units: the candidate's 12 (a reciprocal, a sum and an
    exponential with its argument's rounding are off by 5.8, on 2 r = 0.66 of z = 0.34 where its two forms
    meet, and its own rounding), the gate's 3 and the product's."""
    steps = torch.arange(1, 64, dtype=torch.float64) / 64
    c = torch.cat([2.0 ** e * (1 + steps) for e in range(-13, 1)]).to(dtype)
    c = torch.cat([c, -c])
    g = torch.zeros(1, 3, len(c), dtype=dtype)
    g[0, 1] = c
    want = torch.tanh(c.double()) / 2
    y, hT = ops.gated_recurrence(g.view(1, -1).to(cuda_device), 1, 1)
    _near(hT.flatten(), want, 16 * so.U * want.abs(), "hT")
    y, state = ops.gated_recurrence_step(g.view(1, -1).to(cuda_device), torch.zeros(1, len(c), device=cuda_device))
    _near(state.flatten(), want, 16 * so.U * want.abs(), "state")


def test_a_gradient_of_a_gradient_is_an_error(cuda_device):
    """A penalty on a gradient, in whose graph nothing but the operator's own input needs a gradient."""
    dev = cuda_device
    g = torch.randn(12, 9, device=dev, requires_grad=True)
    h0 = torch.randn(1, 2, 3, device=dev, requires_grad=True)
    tok = torch.zeros(12, dtype=torch.int64, device=dev)
    for out, leaf in ((ops.gated_recurrence(g, 6, 2)[0], g), (ops.gated_recurrence(g, 6, 2)[1], g),
                      (ops.gated_recurrence(g.detach(), 6, 2, h0=h0)[0], h0),
                      (ops.token_log_probs(g, tok)[0], g), (ops.token_log_probs(g, tok)[1], g)):
        loss = out.sum()
        d, = torch.autograd.grad(loss, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            (loss + d.square().sum()).backward()
    # of a dropout the gradient does not depend on x: nothing is missing from the penalty's
    loss = ops.dropout(g, 0.5, _rng(dev)).sum()
    d, = torch.autograd.grad(loss, g, create_graph=True)
    want, = torch.autograd.grad(ops.dropout(g, 0.5, _rng(dev)).sum(), g)
    (loss + d.square().sum()).backward()
    assert torch.equal(g.grad, want)


@pytest.mark.parametrize("dtype,H", [(torch.float32, 65), (torch.bfloat16, 129)], ids=["f32", "bf16"])
def test_recurrence_of_more_row_tiles_than_a_grid_takes(cuda_device, dtype, H):
    """Rows go in several launches: every row has what it has in a call of its neighbours alone."""
    B = 2 ** 22 + 1003  # two channel tiles a row
    g = torch.empty(B, 3 * H, dtype=dtype, device=cuda_device)
    g.normal_(generator=torch.Generator(device=cuda_device).manual_seed(3)).requires_grad_(True)
    y, hT = ops.gated_recurrence(g, 1, B)
    d, = torch.autograd.grad((y, hT), g, (y.detach(), hT.detach()))
    for lo in (0, B // 2 - 500, B - 1000):
        rows = slice(lo, lo + 1000)
        part = g.detach()[rows].clone().requires_grad_(True)
        y2, hT2 = ops.gated_recurrence(part, 1, 1000)
        assert torch.equal(y[rows], y2) and torch.equal(hT[:, rows], hT2)
        assert torch.equal(d[rows], torch.autograd.grad((y2, hT2), part, (y2.detach(), hT2.detach()))[0])
    assert bool((hT.abs() <= 1).all())


def test_recurrence_of_few_columns_in_a_very_wide_buffer(cuda_device):
    """Row strides past what the kernels' 32-bit offsets reach."""
    T, B, H = 3, 2, 1
    wide = torch.full((T * B, (1 << 23) + 5), math.nan, device=cuda_device)
    wide[:, 3:6] = torch.randn(T * B, 3, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    dense = wide[:, 3:6].clone()
    got, want = [], []
    for g, out in ((wide[:, 3:6], got), (dense, want)):
        leaf = g.detach().requires_grad_(True)
        y, hT = ops.gated_recurrence(leaf, T, B)
        out += [y, hT, *torch.autograd.grad((y, hT), leaf, (y.detach(), hT.detach()))]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_negated_views(cuda_device):
    """The imaginary part of a conjugate is a view whose memory holds the opposite sign."""
    dev = cuda_device

    def pair(*shape):
        z = torch.randn(*shape, dtype=torch.complex64, generator=torch.Generator().manual_seed(len(shape))).to(dev)
        v = z.conj().imag
        assert v.is_neg()
        return v, v.resolve_neg().contiguous()

    tok = torch.zeros(1, dtype=torch.int64, device=dev)
    v, p = pair(4, 1)
    assert torch.equal(ops.dropout(v, 0.0, _rng(dev)), p)
    assert torch.equal(ops.dropout(p, 0.0, _rng(dev), residual=v), p + p)
    lone = torch._neg_view(p)
    assert torch.equal(ops.dropout(lone, 0.0, _rng(dev)), -p)
    v, p = pair(6, 9)
    v, p = torch._neg_view(p), -p
    leaf, dense = v.detach().requires_grad_(True), p.detach().requires_grad_(True)
    s = torch._neg_view(torch.rand(1, 2, 3, device=dev))
    y, hT = ops.gated_recurrence(leaf, 3, 2, h0=s)
    y2, hT2 = ops.gated_recurrence(dense, 3, 2, h0=s.resolve_neg())
    assert torch.equal(y, y2) and torch.equal(hT, hT2)
    dy, dh = torch._neg_view(y2.detach()), torch._neg_view(hT2.detach())
    d, = torch.autograd.grad((y, hT), leaf, (dy, dh))
    d2, = torch.autograd.grad((y2, hT2), dense, (dy.resolve_neg(), dh.resolve_neg()))
    assert torch.equal(d, d2)
    a, b = ops.gated_recurrence_step(v[:2].detach(), s[0]), ops.gated_recurrence_step(p[:2], s[0].resolve_neg())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(ValueError, match="out_state"):
        ops.gated_recurrence_step(p[:2], torch.zeros(2, 3, device=dev), out_state=torch._neg_view(torch.zeros(2, 3, device=dev)))
    tok = torch.arange(6, device=dev)
    a, b = ops.token_log_probs(leaf, tok, top=2), ops.token_log_probs(dense, tok, top=2)
    for k in range(4):
        assert torch.equal(a[k], b[k])
    gl, ge = torch._neg_view(torch.rand(6, device=dev)), torch._neg_view(torch.rand(6, device=dev))
    d, = torch.autograd.grad(a[:2], leaf, (gl, ge))
    d2, = torch.autograd.grad(b[:2], dense, (gl.resolve_neg(), ge.resolve_neg()))
    assert torch.equal(d, d2)


def _segments(dtype, T, B, H, dirs):
    """Segments that time is cut into, of the pass that cuts it finer."""
    D = 2 if dirs == 3 else 1
    return _lib.load().avc_gated_recurrence_workspace(_lib.DTYPES[dtype], T, B, H, dirs) // (2 * D * B * H * 4)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T,B,H,dirs,ragged", [
    (1100, 60, 66, 1, False), (1100, 60, 66, 3, True), (1030, 64, 130, 2, True), (1024, 64, 130, 1, False), (2050, 20, 34, 3, True)])
def test_recurrence_segments_of_several_chunks(cuda_device, dtype, T, B, H, dirs, ragged):
    """Segments of 2 to 9 chunks, so that a wave's run of a segment is longer than its frames in flight, with
    and without a rest, and a workgroup goes on over several chunks behind the joined segments."""
    n = _segments(dtype, T, B, H, dirs)
    chunk = 64 if dtype == torch.float32 else 32  # the finer pass's
    assert n > 1 and -(-T // chunk) >= 2 * n
    lengths = [(T, 0, T - 1, T // 2 + 3, 1, 700, 63)[b % 7] for b in range(B)] if ragged else None
    _check_recurrence(cuda_device, dtype, T, B, H, dirs, lengths, h0=True)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T,B,H,dirs,pad", [(20, 40, 130, 1, 0), (9, 31, 200, 3, 7), (70, 16, 128, 2, 5), (600, 11, 130, 3, 7)])
def test_recurrence_of_many_channel_tiles(cuda_device, dtype, T, B, H, dirs, pad):
    """Rows of several channel tiles that begin inside a cache line, in a grid that is reordered in part."""
    _check_recurrence(cuda_device, dtype, T, B, H, dirs, [T - b % 5 for b in range(B)], True, pad)


def test_a_compiled_backward(cuda_device):
    """Run by a compiled graph, where no autograd node is current."""
    g = torch.randn(12, 9, device=cuda_device, requires_grad=True)
    tok = torch.zeros(12, dtype=torch.int64, device=cuda_device)

    def loss():
        y, hT = ops.gated_recurrence(g, 6, 2)
        logp, entropy, _, _ = ops.token_log_probs(ops.dropout(g, 0.5, _rng(cuda_device)), tok)
        return y.sum() + hT.sum() + logp.sum() + entropy.sum()

    want, = torch.autograd.grad(loss(), g)
    value = loss()
    with torch._dynamo.compiled_autograd._enable(torch.compile(backend="eager")):
        value.backward()
    assert torch.equal(g.grad, want)
