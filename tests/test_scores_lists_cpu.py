"""The distillation oracle on lists that name a class more than once, against the divergence over all classes."""
import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
import scores_oracle as O
from test_gpu_scores_lists import dense_loss


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_oracle_counts_a_repeated_class_once(tail, temperature):
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(6, 12, generator=gen)
    index = torch.randint(6, (6, 7), generator=gen)
    index[0], index[1, 3], index[2, 5] = 4, -1, 99
    value = torch.randn(6, 7, generator=gen)
    value = torch.log_softmax(value, 1) - 0.2 if tail else value
    torch.testing.assert_close(O.distill(x, index, value, temperature, tail)[0], dense_loss(x, index, value, temperature, tail), rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("tail", [False, True])
def test_oracle_of_a_list_that_says_what_the_student_says(tail):
    x = torch.zeros(1, 2)
    loss = O.distill(x, torch.tensor([[0, 0, 1, 1]]), torch.full((1, 4), -1.3862943611198906, dtype=torch.float64), 1.0, tail)[0]
    assert abs(float(loss)) < 1e-12
