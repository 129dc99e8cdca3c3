"""ops.top_distill(tail=True) of confident teachers: what the list leaves of 1 is 1e-4 to 1e-8, or nothing, and the classes outside the list
take their gradient from it."""
import math

import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
import scores_oracle as O

pytestmark = pytest.mark.gpu


def _teacher(rows, classes, k, rest, gen):
    """A list whose first class has nearly everything: its log probability is close to 0, where float32 steps are far below the rest."""
    index = torch.stack([torch.randperm(classes, generator=gen)[:k] for _ in range(rows)])
    others = torch.softmax(torch.randn(rows, k - 1, generator=gen, dtype=torch.float64), 1) * 1e-3 if k > 1 else torch.zeros(rows, 0, dtype=torch.float64)
    first = 1 - rest - others.sum(1, keepdim=True)
    return index, torch.log(torch.cat([first, others], 1)).float()


def _want(x, index, value, temperature):
    """(rest, share of each class outside the list, p, p of them all, loss, gradient) in 64 bits."""
    z = x.double() / temperature
    listed = torch.zeros_like(z, dtype=torch.bool).scatter_(1, index, True)
    q = torch.exp(value.double())
    rest = (1 - q.sum(1)).clamp(min=0)
    lse = torch.logsumexp(z, 1, keepdim=True)
    outside = torch.where(listed, -math.inf, z)
    lse_out = torch.logsumexp(outside, 1, keepdim=True)
    share, p, log_p_rest = torch.exp(outside - lse_out), torch.exp(z - lse), (lse_out - lse)[:, 0]
    loss = (q * (value.double() - (z - lse).gather(1, index))).sum(1)
    loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - log_p_rest), 0.0)
    all_ = torch.where(rest > 0, 1.0, q.sum(1))[:, None]
    grad = p * all_ - torch.zeros_like(z).scatter_(1, index, q) - rest[:, None] * share
    return rest, listed, share, p, torch.exp(log_p_rest), log_p_rest, loss, grad / temperature


@pytest.mark.parametrize("temperature", [1.0, 1.5])
@pytest.mark.parametrize("rest", [1e-4, 1e-6, 1e-8, 0.0])
@pytest.mark.parametrize("gap", [4.0, 14.0, 60.0])
@pytest.mark.parametrize("rows,classes,k", [(3, 101, 1), (4, 400, 20), (2, 2049, 64), (3, 5000, 10), (1, 40001, 256)])
def test_small_rests_hold(rows, classes, k, gap, rest, temperature):
    from vitta_amd import ops
    gen = torch.Generator().manual_seed(k)
    index, value = _teacher(rows, classes, k, rest, gen)
    x = torch.randn(rows, classes, generator=gen)
    x.scatter_add_(1, index, torch.full((rows, k), gap * temperature))
    leaf = x.cuda().requires_grad_()
    loss = ops.top_distill(leaf, index.cuda(), value.cuda(), temperature=temperature, tail=True)
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    real, listed, share, p, p_rest, log_p_rest, want, grad_want = _want(x, index, value, temperature)
    assert rest == 0 or bool(((real - rest).abs() < 0.2 * rest).all())
    # u = 2^-24.  The rest is 1 - (k terms) in 64 bits, k 2^-52 of the 1 in all, and rounded once; the sums of the student are off by
    # u (depth + 40 + 8 |x - m| / T) and every factor by a few u
    spread = (x.double().amax(1, keepdim=True) - x.double()).abs().amax(1, keepdim=True) / temperature
    off_p = O.U * (O.depth(classes) + 60 + 8 * spread)
    off_rest = 2 * O.U * real + (k + 4) * 2.0 ** -52
    q = torch.exp(value.double())
    bound = torch.where(listed, (p + torch.zeros_like(p).scatter_(1, index, q)) * off_p,
                        share * ((real + p_rest)[:, None] * off_p + off_rest[:, None])) / temperature
    got = grad.double().cpu()
    off = (got - grad_want).abs() - bound - O.U * grad_want.abs() - 2.0 ** -149
    assert float(off.max()) <= 0, ("gradient", float(off.max()), int(off.argmax()), float((got - grad_want).abs()[~listed].max()))
    far = value.double().abs() + log_p_rest.abs()[:, None] + gap + 10
    bound = (q * off_p * (1 + far)).sum(1) + (off_rest + real * off_p[:, 0]) * (log_p_rest.abs() + torch.log(real.clamp(min=1e-9)).abs() + 2) + O.U * want.abs()
    off = (loss.detach().double().cpu() - want).abs() - bound
    assert float(off.max()) <= 0, ("loss", float(off.max()))


def test_one_class_that_leaves_almost_nothing():
    """A log probability of -2e-8 leaves 2e-8, which 32 bits of 1 - exp would round to 0."""
    from vitta_amd import ops
    value = torch.tensor([[-2e-8]])
    rest = 1 - math.exp(float(value))
    loss = ops.top_distill(torch.zeros(1, 9, device="cuda"), torch.tensor([[4]]).cuda(), value.cuda(), tail=True)
    want = (1 - rest) * (float(value) + math.log(9)) + rest * (math.log(rest) - math.log(8 / 9))
    assert abs(float(loss) - want) < 60 * O.U  # (a sum of nine terms and its logarithm, 2.2)
    student = torch.full((1, 9), -60.0, device="cuda")
    student[0, 4] = 0.0
    leaf = student.requires_grad_()
    (grad,) = torch.autograd.grad(ops.top_distill(leaf, torch.tensor([[4]]).cuda(), value.cuda(), tail=True).sum(), leaf)
    want = -rest / 8
    assert float((grad[0, :4].double().cpu() - want).abs().max()) <= 1e-6 * abs(want)
