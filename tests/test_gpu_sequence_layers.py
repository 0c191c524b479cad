"""The sequence-model operators where the package's own layers and models call them."""
import math

import pytest
import torch

from autovc_amd.auto_encoder.net_layers import GatedRecurrence
from autovc_amd.wavernn import WaveRNN
from oracle import sequence_oracle as so

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["forward", "reverse", "both"])
def test_gated_recurrence_layer(cuda_device, kind):
    T, B, din, H = 75, 3, 20, 24
    torch.manual_seed(3)
    layer = GatedRecurrence(din, H, bidirectional=kind == "both", reverse=kind == "reverse")
    lengths = torch.tensor([75, 0, 40])
    x = torch.randn(T * B, din)
    w, b = (p.detach().double().requires_grad_(True) for p in (layer.weight_ih, layer.bias_ih))
    xr = x.double().requires_grad_(True)
    y, hT = so.recurrence(xr @ w.t() + b, T, B, None, lengths.tolist(), layer.dirs)
    dy, dh = torch.randn(y.shape), torch.randn(hT.shape)
    ref = torch.autograd.grad((y, hT), (xr, w, b), (dy.double(), dh.double()))
    layer.to(cuda_device)
    xd = x.to(cuda_device).requires_grad_(True)
    yd, hd = layer(xd, T, B, lengths=lengths.to(cuda_device))
    got = torch.autograd.grad((yd, hd), (xd, layer.weight_ih, layer.bias_ih), (dy.to(cuda_device), dh.to(cuda_device)))
    # a projection of 20 terms, the recurrence, and a product of up to 225 terms, each off by at most a
    # few hundred units of the largest sum of magnitudes
    for a, r in zip((yd, hd) + got, (y, hT) + ref):
        r = r.detach()
        assert (a.detach().cpu().double() - r).abs().max() <= 1000 * so.U * max(r.abs().max().item(), 1.0)


def test_gated_recurrence_layer_stepped(cuda_device):
    T, B, din, H = 20, 2, 8, 12
    torch.manual_seed(4)
    layer = GatedRecurrence(din, H).to(cuda_device)
    x = torch.randn(T * B, din, device=cuda_device)
    with torch.no_grad():
        y, hT = layer(x, T, B)
    state = torch.zeros(B, H, device=cuda_device)
    ys = torch.cat([layer.step(x[t * B:(t + 1) * B].contiguous(), state) for t in range(T)])
    # 20 frames of at most (|g| + 12) units and the projection's few, both ways of running
    assert (ys - y).abs().max().item() <= 2000 * so.U and (state - hT[0]).abs().max().item() <= 2000 * so.U
    with pytest.raises(ValueError):
        GatedRecurrence(din, H, reverse=True).to(cuda_device).step(x[:B], state)
    with pytest.raises(ValueError):
        GatedRecurrence(din, H, bidirectional=True, reverse=True)


def test_gated_recurrence_layer_trains(cuda_device):
    """A step of its own gradients changes every parameter and stays finite; fresh gates remember."""
    torch.manual_seed(5)
    for widths in ((6, 12), (8, 10)):
        with pytest.raises(ValueError, match="multiples of 4"):
            GatedRecurrence(*widths)
    layer = GatedRecurrence(8, 12, bidirectional=True).to(cuda_device)
    assert layer.bias_ih.view(2, 3, 12)[:, 0].mean() > 0.5 > layer.bias_ih.view(2, 3, 12)[:, 1:].mean()
    y, hT = layer(torch.randn(30 * 2, 8, device=cuda_device), 30, 2)
    (y.square().sum() + hT.sum()).backward()
    for p in layer.parameters():
        assert torch.isfinite(p.grad).all() and (p.grad != 0).any()


def test_wavernn_log_probs(cuda_device):
    torch.manual_seed(6)
    net = WaveRNN(device=cuda_device, mode="RAW")
    net.eval()
    T = 6
    L = (T - 2 * net.pad) * net.hop_length
    x = torch.rand(1, L) * 2 - 1
    mels = torch.rand(1, net.feat_dims, T)
    classes = torch.randint(0, net.n_classes, (1, L))
    classes[0, 3] = -100
    logits = net(x, mels).cpu().double()[0]
    logp, entropy, top_logp, top_ids = net.log_probs(x, mels, classes, top=3)
    assert logp.shape == entropy.shape == (1, L) and top_ids.shape == (1, L, 3)
    ref = so.log_probs(logits, classes[0], 3)
    Elp, EH, _ = so.log_probs_bounds(logits, classes[0])
    at = classes[0].clamp_min(0)[:, None]
    assert ((logp[0].cpu().double() - ref[0]).abs() <= Elp.gather(1, at)[:, 0] + so.rounded(ref[0], torch.float32)).all()
    assert ((entropy[0].cpu().double() - ref[1]).abs() <= EH + so.rounded(ref[1], torch.float32)).all()
    assert torch.equal(top_ids[0].cpu(), ref[3]) and logp[0, 3] == 0
    assert math.isfinite(top_logp.sum().item())
    with pytest.raises(ValueError):
        WaveRNN(device=cuda_device, mode="MOL").log_probs(x, mels, classes)


@pytest.mark.parametrize("T,B", [(0, 3), (5, 0)])
def test_gated_recurrence_layer_without_frames(cuda_device, T, B):
    layer = GatedRecurrence(8, 12, bidirectional=True).to(cuda_device)
    h0 = torch.rand(2, B, 12, device=cuda_device)
    y, hT = layer(torch.zeros(0, 8, device=cuda_device, requires_grad=True), T, B, h0=h0)
    assert y.shape == (0, 24) and torch.equal(hT, h0)
    (y.sum() + hT.sum()).backward()
    assert all((p.grad == 0).all() for p in layer.parameters())
    y = GatedRecurrence(8, 12).to(cuda_device).step(torch.zeros(0, 8, device=cuda_device), torch.zeros(0, 12, device=cuda_device))
    assert y.shape == (0, 12)
