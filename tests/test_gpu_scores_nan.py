"""Gradients of rows that have no distribution (NaN or +inf among the scores, a teacher's list of NaN or of -inf only): NaN in every class where
the loss uses the row, through whichever result, and zeros in every class where it does not."""
import math

import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)

pytestmark = pytest.mark.gpu

KINDS = ["nan", "inf", "nan among -inf"]


def _scores(kind, classes):
    x = torch.randn(3, classes, generator=torch.Generator().manual_seed(classes))
    if kind == "nan among -inf":
        x[1] = -math.inf
    x[1, classes // 2] = math.inf if kind == "inf" else math.nan
    return x.cuda()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("classes", [5, 101, 3000, 20001])
def test_a_row_without_a_distribution_poisons_its_gradient(classes, kind):
    from vitta_amd import ops
    leaf = _scores(kind, classes).requires_grad_()
    o = ops.label_logprobs(leaf, torch.zeros(3, dtype=torch.long, device="cuda"), top=3, lse=True)
    one, none = torch.ones(3, device="cuda"), torch.zeros(3, device="cuda")
    only = torch.zeros(3, 3, device="cuda")
    only[:, 2] = 1
    for outs, ups in (([o.logprob], [one]), ([o.entropy], [one]), ([o.lse], [one]), ([o.top_logprob], [only]),
                      ([o.top_logprob], [only - only.roll(1, 1)]), ([o.logprob, o.lse], [one, one])):
        (grad,) = torch.autograd.grad(outs, leaf, ups, retain_graph=True)
        assert bool(torch.isnan(grad[1]).all()) and bool(torch.isfinite(grad[::2]).all())
    (grad,) = torch.autograd.grad([o.logprob, o.entropy, o.lse, o.top_logprob], leaf, [none, none, none, 0 * only], retain_graph=True)
    assert bool((grad == 0).all())


@pytest.mark.parametrize("classes", [101, 5000])
def test_labels_that_are_no_class_in_rows_that_are_not_used(classes):
    from vitta_amd import ops
    leaf = torch.randn(2, classes, device="cuda").requires_grad_()
    o = ops.label_logprobs(leaf, torch.tensor([classes, -7], device="cuda"), entropy=False)
    (grad,) = torch.autograd.grad(o.logprob, leaf, torch.tensor([0.0, 1.0], device="cuda"))
    assert bool((grad[0] == 0).all()) and bool(torch.isnan(grad[1]).all())


LISTS = ["-inf", "nan", "some nan"]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("kind", KINDS + LISTS)
@pytest.mark.parametrize("classes", [5, 101, 3000, 20001])
def test_distillation_without_a_distribution(classes, kind, tail):
    from vitta_amd import ops
    x = _scores(kind, classes) if kind in KINDS else torch.randn(3, classes, generator=torch.Generator().manual_seed(classes)).cuda()
    index = torch.tensor([[0, classes // 2, -1]] * 3).cuda()
    value = torch.tensor([[-1.0, -2.0, -3.0]] * 3)
    if kind in LISTS:
        value[1] = -math.inf if kind == "-inf" else math.nan
    if kind == "some nan":
        value[1, 0] = -1.0
    leaf = x.requires_grad_()
    loss = ops.top_distill(leaf, index, value.cuda(), tail=tail)
    lost = not (kind == "-inf" and tail)  # (a teacher who leaves everything to the classes outside its list)
    assert bool(torch.isnan(loss[1])) == lost and bool(torch.isfinite(loss[::2]).all())
    (grad,) = torch.autograd.grad(loss.sum(), leaf, retain_graph=True)
    assert bool(torch.isnan(grad[1]).all() if lost else torch.isfinite(grad[1]).all()) and bool(torch.isfinite(grad[::2]).all())
    (grad,) = torch.autograd.grad(loss, leaf, torch.tensor([1.0, 0.0, 1.0], device="cuda"))
    assert bool((grad[1] == 0).all()) and bool((grad[::2] != 0).any())


@pytest.mark.parametrize("tail", [False, True])
def test_neither_student_nor_teacher_has_a_distribution(tail):
    from vitta_amd import ops
    leaf = torch.full((1, 50), -math.inf, device="cuda").requires_grad_()
    loss = ops.top_distill(leaf, torch.tensor([[3, 4]]).cuda(), torch.tensor([[math.nan, 0.0]]).cuda(), tail=tail)
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    assert bool(torch.isnan(loss).all()) and bool(torch.isnan(grad).all())
