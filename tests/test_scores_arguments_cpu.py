"""Arguments of the score operators that the C interface's types do not hold: refused, not wrapped around."""
from types import SimpleNamespace

import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
from test_scores_cpu import _bwd, _distil, _fwd
from test_scores_saved_cpu import launches  # noqa: F401  (a fixture)
from vitta_amd import _lib, ops


@pytest.mark.parametrize("classes", [2 ** 24 + 1, 2 ** 31 + 1, 2 ** 32 + 5, 2 ** 40])
@pytest.mark.parametrize("rows", [1, 3])
def test_more_classes_than_the_operators_take(rows, classes):
    """2^32 + 5 classes would arrive as five of them."""
    x = SimpleNamespace(is_cuda=True, dtype=torch.float16, device=torch.device("cuda", 0), dim=lambda: 2, shape=torch.Size((rows, classes)),
                        stride=lambda d=None: (classes, 1) if d is None else (classes, 1)[d], numel=lambda: rows * classes)
    with pytest.raises(_lib.VittaHipError, match="unsupported"):
        ops._score_rows(x, "logits", 1.0)


@pytest.mark.parametrize("ignore", [2 ** 63, 2 ** 64 - 100, -2 ** 63 - 1])
def test_ignored_labels_that_are_no_64_bit_number(launches, ignore):  # noqa: F811
    with pytest.raises(ValueError, match="ignore_index"):
        ops.label_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long), ignore_index=ignore)
    assert launches == []


@pytest.mark.parametrize("ignore", [2 ** 63 - 1, -2 ** 63, 0])
def test_ignored_labels_at_the_ends(launches, ignore):  # noqa: F811
    ops.label_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long), ignore_index=ignore)
    assert ignore in launches[-1][1]


def _distil_bwd(**kw):
    a = dict(x=4096, dtype=0, rows=2, classes=10, stride=10, inner=2, outer=0, t=1.0, index=4096, list=3, stats=4096, q=4096, g=4096, s_g=1, dx=4096)
    a.update(kw)
    return _lib.lib().vitta_top_distill_bwd(*a.values(), None)


@pytest.mark.parametrize("call", [_fwd, _bwd, _distil, _distil_bwd])
@pytest.mark.parametrize("temperature", [1e-45, 1e-39, 9e-31, 1.1e30, 3e38])
def test_temperatures_whose_reciprocal_or_differences_overflow(call, temperature):
    """1 / T is infinite below 3e-39 (0 times it is NaN), and two finite scores lie further apart than 32 bits reach, which a T of 1e38 would
    bring near again: the C interface refuses what the Python one refuses.  (A class count that is refused as well keeps the call from launching.)"""
    assert call(t=temperature, classes=(1 << 24) + 1, stride=1 << 25) == -1
    assert call(t=1.0, classes=(1 << 24) + 1, stride=1 << 25) == -4
