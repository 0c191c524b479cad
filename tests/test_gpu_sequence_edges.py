"""The sequence-model operators at the edges of their range, against the float64 oracle."""
import math

import pytest
import torch

from autovc_amd import ops
from tests.test_gpu_sequence import _check_log_probs, _rng

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
