"""What the score operators do under forward-mode differentiation and under tracers, which they have no rule for: an error, never a result
without its tangent or a recorded program without the launches.  The launches are replaced by a recorder: no GPU is needed."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
from test_scores_saved_cpu import launches  # noqa: F401  (a fixture)
from vitta_amd import _lib, ops

LABELS = torch.zeros(3, dtype=torch.long)
CALLS = {"label_logprobs": lambda x: ops.label_logprobs(x, LABELS, top=2).entropy,
         "one result": lambda x: ops.label_logprobs(x, LABELS, entropy=False).logprob,
         "top_distill": lambda x: ops.top_distill(x, LABELS[:, None], torch.zeros(3, 1))}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call", CALLS)
def test_a_tangent_is_refused(launches, call, grad):  # noqa: F811
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.randn(3, 10).requires_grad_(grad), torch.ones(3, 10))
        with pytest.raises(NotImplementedError, match="jvp"):
            CALLS[call](x)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
            CALLS[call](x)


def test_a_tangent_of_the_teacher_is_refused(launches):  # noqa: F811
    with forward_ad.dual_level():
        value = forward_ad.make_dual(torch.zeros(3, 1), torch.ones(3, 1))
        with pytest.raises(ValueError, match="teacher_value"):
            ops.top_distill(torch.randn(3, 10), LABELS[:, None], value)


@pytest.mark.parametrize("call", CALLS)
def test_scores_without_a_tangent_are_read_in_a_dual_level(launches, call):  # noqa: F811
    x = torch.randn(3, 10)
    with forward_ad.dual_level():
        out = CALLS[call](x)
        assert len(launches) == 1 and not out.requires_grad and forward_ad.unpack_dual(out).tangent is None
        leaf = x.clone().requires_grad_()
        (grad,) = torch.autograd.grad(CALLS[call](leaf).sum(), leaf)
        assert grad.shape == x.shape and len(launches) == 3


@pytest.mark.filterwarnings("ignore")  # (the tracer's own, on its deprecation and on what it takes for constants)
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call", CALLS)
def test_a_trace_is_refused(launches, call, grad):  # noqa: F811
    x = torch.randn(3, 10).requires_grad_(grad)
    with pytest.raises(_lib.VittaHipError, match="traced"):
        torch.jit.trace(CALLS[call], (x,), check_trace=False)
    with pytest.raises(_lib.VittaHipError, match="traced"):
        make_fx(CALLS[call])(x)
    assert launches == []
