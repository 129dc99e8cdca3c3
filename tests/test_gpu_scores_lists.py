"""ops.top_distill on lists that name a class more than once: it counts as one class with the sum of its probabilities, in the loss as in the
gradient.  Compared with the divergence over all classes in 64 bits, and with the list that names each class once."""
import math

import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
import scores_oracle as O

pytestmark = pytest.mark.gpu


def dense_loss(x, index, value, temperature, tail):
    """The definition over all classes, in 64 bits: q (rows, V), then sum q (log q - log p), and the remaining mass as one class."""
    rows, classes = x.shape
    inside = (index >= 0) & (index < classes)
    v = torch.where(inside, value.double(), -math.inf)
    each = torch.exp(v) if tail else torch.softmax(v / temperature, 1)
    q = torch.zeros(rows, classes, dtype=torch.float64).scatter_add_(1, torch.where(inside, index, 0), torch.where(inside, each, 0.0))
    lp = torch.log_softmax(x.double() / temperature, 1)
    loss = torch.where(q > 0, q * (torch.log(q) - lp), 0.0).sum(1)
    if tail:
        listed = torch.zeros(rows, classes + 1, dtype=torch.bool).scatter_(1, torch.where(inside, index, classes), True)[:, :classes]
        rest, p_rest = (1 - q.sum(1)).clamp(min=0), torch.where(listed, 0.0, torch.exp(lp)).sum(1)
        loss = loss + torch.where((rest > 0) & (p_rest > 0), rest * (torch.log(rest) - torch.log(p_rest)), 0.0)
    return loss


def bound(x, index, value, temperature):
    """u = 2^-24.  log p is off by u (depth + 40 + 8 |x - m| / T), a probability of the list by u (K + 16 + 8 |v| / T), its logarithm by as much
    and 2 u of itself; the loss weighs these with probabilities whose sum is at most 1, and adds up K terms.  The rest carries the sum's error
    times its logarithms (|log| <= 20 for the rests used here)."""
    k = index.shape[1]
    spread = float((x.double().amax(1) - x.double().amin(1)).max()) / temperature
    far = float(value.double().abs().max()) / min(temperature, 1.0)
    log_p = spread + math.log(x.shape[1] + 1)
    return O.U * (O.depth(x.shape[1]) + k + 80 + 8 * far + 8 * spread) * (3 + log_p + far + 20)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,classes,k", [(3, 5, 4), (5, 40, 16), (4, 700, 64), (3, 2049, 65), (2, 5000, 256), (1, 131072, 200)])
def test_repeated_classes_count_as_one(rows, classes, k, tail):
    from vitta_amd import ops
    gen = torch.Generator().manual_seed(k)
    for temperature in (1.0, 1.7):
        x = torch.randn(rows, classes, generator=gen) * 2
        index = torch.randint(min(classes, k // 2), (rows, k), generator=gen)
        index[0] = index[0, 0]  # one class throughout
        index[-1, ::2] = index[-1, (k - 1) // 2 * 2]  # every other entry, across the lanes' chunks
        index[-1, 1] = -1
        value = torch.randn(rows, k, generator=gen)
        if tail:  # a rest of about a third
            value = torch.log_softmax(torch.cat([value, torch.logsumexp(value, 1, keepdim=True) - 0.7], 1), 1)[:, :k]
        leaf = x.cuda().requires_grad_()
        loss = ops.top_distill(leaf, index.cuda(), value.cuda(), temperature=temperature, tail=tail)
        want = dense_loss(x, index, value, temperature, tail)
        off = (loss.detach().double().cpu() - want).abs()
        assert float(off.max()) <= bound(x, index, value, temperature), (float(off.max()), int(off.argmax()))


@pytest.mark.parametrize("tail", [False, True])
def test_a_class_split_in_two_has_the_loss_of_the_whole(tail):
    from vitta_amd import ops
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(6, 90, generator=gen)
    index = torch.stack([torch.randperm(90, generator=gen)[:8] for _ in range(6)])
    value = torch.log_softmax(torch.randn(6, 9, generator=gen), 1)[:, :8]
    part = torch.rand(6, 8, generator=gen) * 0.8 + 0.1
    twice = torch.cat([index, index], 1)
    split = torch.cat([value + torch.log(part), value + torch.log1p(-part)], 1)
    leaf = x.cuda().requires_grad_()
    a, b = [ops.top_distill(leaf, i.cuda(), v.cuda(), tail=tail) for i, v in ((index, value), (twice, split))]
    assert float((a - b).abs().max()) <= 2 * bound(x, twice, split, 1.0)
    ga, gb = [torch.autograd.grad(t.sum(), leaf)[0] for t in (a, b)]
    assert float((ga - gb).abs().max()) <= 2 * bound(x, twice, split, 1.0)


def test_a_teacher_that_the_student_equals_has_no_divergence():
    from vitta_amd import ops
    x = torch.zeros(2, 2).cuda()
    index = torch.tensor([[0, 0, 1, 1], [0, 1, 1, 1]]).cuda()
    value = torch.tensor([[0.0, 0.0, 0.0, 0.0], [math.log(3.0), 0.0, 0.0, 0.0]]).cuda()
    for tail, v in ((False, value), (True, torch.log_softmax(value, 1))):
        assert float(ops.top_distill(x, index, v, tail=tail).abs().max()) <= 40 * O.U


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("low", [-80.0, -88.0, -95.0, -103.0, -200.0, -math.inf])
def test_repeats_of_next_to_no_probability(low, tail):
    """A repeated class whose probabilities are subnormal or 0: it adds nothing that 32 bits show, and no infinity."""
    from vitta_amd import ops
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(4, 30, generator=gen)
    index = torch.tensor([[3, 5, 5, 5], [5, 5, 3, 5], [7, 7, 7, 3], [0, 0, 0, 3]])
    value = torch.where(index == 3, -0.25 if tail else 0.0, low)
    leaf = x.cuda().requires_grad_()
    loss = ops.top_distill(leaf, index.cuda(), value.cuda(), tail=tail)
    off = (loss.detach().double().cpu() - dense_loss(x, index, value, 1.0, tail)).abs()
    assert float(off.max()) <= bound(x, index, torch.zeros(4, 4), 1.0)
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    assert bool(torch.isfinite(grad).all())


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("kind", ["one slot", "strided", "neighbours"])
def test_lists_whose_classes_meet_when_repeats_are_looked_for(kind, tail):
    """Classes that the multiplicative hash sends to one of its 1024 slots, and regular ones, some of them twice."""
    from vitta_amd import ops
    classes, k = 131072, 128
    number = torch.arange(classes)
    one = number[((number * 2654435769) % 2 ** 32) >> 22 == 5]
    pick = {"one slot": one[:100], "strided": number[::1024][:100], "neighbours": number[7:107]}[kind]
    assert len(pick) == 100
    gen = torch.Generator().manual_seed(4)
    index = torch.stack([torch.cat([pick, pick[:28]])[torch.randperm(k, generator=gen)] for _ in range(3)])
    value = torch.log_softmax(torch.randn(3, k + 40, generator=gen), 1)[:, :k]
    x = torch.randn(3, classes, generator=gen)
    loss = ops.top_distill(x.cuda(), index.cuda(), value.cuda(), tail=tail)
    off = (loss.double().cpu() - dense_loss(x, index, value, 1.0, tail)).abs()
    assert float(off.max()) <= bound(x, index, value, 1.0)
    for _ in range(3):
        assert torch.equal(ops.top_distill(x.cuda(), index.cuda(), value.cuda(), tail=tail), loss)
