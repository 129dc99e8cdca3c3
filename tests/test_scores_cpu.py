"""The score operators without a GPU: the oracle's gradients against differences of its losses, and what the entry points refuse."""
import ctypes
import math

import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
import scores_oracle as O
from vitta_amd import _lib, ops


def _differences(f, x, h=1e-5):
    """Central differences of the 64-bit function f at x (rows, V) -> (rows, V): f gives a number per row."""
    g = torch.zeros_like(x)
    for j in range(x.shape[1]):
        a, b = x.clone(), x.clone()
        a[:, j] += h
        b[:, j] -= h
        g[:, j] = (f(a) - f(b)) / (2 * h)
    return g


@pytest.mark.parametrize("temperature", [1.0, 0.6, 2.5])
def test_oracle_readout_gradient_equals_differences(temperature):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(4, 9, generator=gen, dtype=torch.float64) * 2
    labels = torch.tensor([0, 8, -100, 3])
    up = {k: torch.randn(4, generator=gen, dtype=torch.float64) for k in ("logprob", "entropy", "lse")}
    up_top = torch.randn(4, 3, generator=gen, dtype=torch.float64)

    def f(a):
        o = O.readout(a, labels, 3, temperature)
        return sum(up[k] * o[k] for k in up) + (up_top * o["top_logprob"]).sum(1)

    grad, _ = O.readout_grad(x, labels, 3, temperature, up["logprob"], up["entropy"], up["lse"], up_top)
    # differences of step h lose third derivatives (h^2, times 1/T^3) and 2^-53 / h
    torch.testing.assert_close(grad, _differences(f, x), rtol=0, atol=1e-8)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_oracle_distillation_gradient_equals_differences(tail, temperature):
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(5, 11, generator=gen, dtype=torch.float64) * 2
    index = torch.tensor([[0, 3, 10], [2, 2, 5], [7, -1, 1], [-1, -1, -1], [4, 99, 6]])  # (a double, padding, a number that is no class)
    value = torch.randn(5, 3, generator=gen, dtype=torch.float64) - (3.5 if tail else 0)
    _, grad, _, _ = O.distill(x, index, value, temperature, tail)
    torch.testing.assert_close(grad, _differences(lambda a: O.distill(a, index, value, temperature, tail)[0], x), rtol=0, atol=1e-8)
    assert (grad[3] == 0).all()


def test_oracle_agrees_with_torch():
    x = torch.randn(6, 50, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    labels = torch.arange(6)
    o = O.readout(x, labels, 4, 0.5)
    lp = torch.log_softmax(x / 0.5, 1)
    torch.testing.assert_close(o["logprob"], lp[torch.arange(6), labels])
    torch.testing.assert_close(o["entropy"], torch.distributions.Categorical(logits=x / 0.5).entropy())
    assert torch.equal(o["top_index"], torch.topk(x, 4).indices)
    index, value = torch.topk(torch.randn(6, 50, generator=torch.Generator().manual_seed(6), dtype=torch.float64), 8).indices, torch.randn(6, 8)
    loss = O.distill(x, index, value, 2.0)[0]
    target = torch.zeros(6, 50, dtype=torch.float64).scatter_(1, index, torch.softmax(value.double() / 2.0, 1))
    torch.testing.assert_close(loss, torch.nn.functional.kl_div(torch.log_softmax(x / 2.0, 1), target, reduction="none").sum(1))


def test_operators_refuse_host_tensors():
    x = torch.zeros(2, 5)
    with pytest.raises(_lib.VittaHipError, match="GPU"):
        ops.label_logprobs(x, torch.zeros(2, dtype=torch.long))
    with pytest.raises(_lib.VittaHipError, match="GPU"):
        ops.top_distill(x, torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 1))


def _fwd(**kw):
    a = dict(x=4096, dtype=0, rows=2, classes=10, stride=10, inner=2, outer=0, t=1.0, labels=4096, ignore=-100, top=0, logprob=4096, entropy=None, lse=4096,
             top_logprob=None, top_index=None, stats=None, ws=None, ws_bytes=1 << 40, tickets=None)
    a.update(kw)
    return _lib.lib().vitta_label_logprobs_fwd(*a.values(), None)


# every call below is refused before any launch: no pointer is read
@pytest.mark.parametrize("bad", [dict(x=None), dict(dtype=3), dict(dtype=-1), dict(rows=0), dict(rows=-1), dict(classes=0), dict(stride=-1), dict(inner=0), dict(inner=-3), dict(outer=-1),
                                 dict(t=0.0), dict(t=-1.0), dict(t=math.nan), dict(t=math.inf), dict(x=4097), dict(x=4098), dict(top=-1),
                                 dict(top=11), dict(top=65, classes=100, top_logprob=4096, top_index=4096), dict(top=3),
                                 dict(top=3, top_logprob=4096), dict(labels=None), dict(logprob=None), dict(stats=4104),
                                 dict(labels=None, logprob=None, lse=None)])
def test_readout_refusals(bad):
    assert _fwd(**bad) == -1


def test_layouts_of_rows():
    """What _row_layout says of a layout names the rows' addresses, over random views; None only where two strides do not do."""
    gen = torch.Generator().manual_seed(1)
    said = 0
    for _ in range(400):
        n = int(torch.randint(1, 5, (1,), generator=gen))
        x = torch.arange(4 * 5 * 3 * 6).view(4, 5, 3, 6)
        for d in range(3):
            lo = int(torch.randint(0, 2, (1,), generator=gen))
            hi = x.shape[d] - int(torch.randint(0, 2, (1,), generator=gen))
            x = x.narrow(d, lo, max(1, hi - lo))
        x = x[..., :4] if n == 1 else x.transpose(0, 1) if n == 2 else x[:, :1].expand(-1, 5, -1, -1) if n == 3 else x[:, 0]
        got = ops._row_layout(x.shape, x.stride())
        if got is None:
            continue
        said += 1
        stride, inner, outer = got
        base = x.storage_offset()
        rows = x.numel() // x.shape[-1]
        want = x.reshape(rows, -1)[:, 0]
        have = torch.tensor([base + (r // inner) * outer + (r % inner) * stride for r in range(rows)])
        assert torch.equal(want, have)
    assert said > 200
    assert ops._row_layout((3, 4), (1, 3)) is None and ops._row_layout((2, 2, 2, 5), (100, 30, 7, 1)) is None


def test_sizes_beyond_a_launch_are_refused():
    assert _fwd(rows=1 << 40) == -4
    assert _fwd(classes=(1 << 24) + 1, stride=1 << 25) == -4


def _bwd(**kw):
    a = dict(x=4096, dtype=0, rows=2, classes=10, stride=10, inner=2, outer=0, t=1.0, labels=4096, ignore=-100, top=0, top_index=None, stats=4096, g1=4096,
             s1=1, g2=None, s2=0, g3=None, s3=0, gtop=None, dx=4096)
    a.update(kw)
    return _lib.lib().vitta_label_logprobs_bwd(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(stats=None), dict(stats=4104), dict(dx=None), dict(dx=4097), dict(labels=None),
                                 dict(gtop=4096), dict(gtop=4096, top_index=4096), dict(gtop=4096, top_index=4096, top=65), dict(dtype=7), dict(t=0.0)])
def test_readout_gradient_refusals(bad):
    assert _bwd(**bad) == -1


def _distil(**kw):
    a = dict(x=4096, dtype=0, rows=2, classes=10, stride=10, inner=2, outer=0, t=1.0, index=4096, value=4096, value_dtype=0, list=3, tail=0, loss=4096,
             stats=4096, q=4096, ws=None, ws_bytes=1 << 40, tickets=None)
    a.update(kw)
    return _lib.lib().vitta_top_distill_fwd(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(index=None), dict(value=None), dict(loss=None), dict(stats=None), dict(stats=4104), dict(q=None),
                                 dict(list=0), dict(list=257), dict(value_dtype=3), dict(dtype=9), dict(t=math.nan), dict(classes=-3)])
def test_distillation_refusals(bad):
    assert _distil(**bad) == -1


@pytest.mark.parametrize("bad", [dict(x=None), dict(index=None), dict(stats=None), dict(stats=4104), dict(q=None), dict(g=None), dict(dx=None),
                                 dict(dx=4097), dict(list=0), dict(list=257)])
def test_distillation_gradient_refusals(bad):
    a = dict(x=4096, dtype=0, rows=2, classes=10, stride=10, inner=2, outer=0, t=1.0, index=4096, list=3, stats=4096, q=4096, g=4096, s_g=1, dx=4096)
    a.update(bad)
    assert _lib.lib().vitta_top_distill_bwd(*a.values(), None) == -1


def test_library_is_built_without_packed_float32_instructions():
    from vitta_amd import build
    flags = " ".join(build.CFLAGS)
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in flags and "-ffast-math" not in flags


def test_workspace_is_plain_host_arithmetic():
    f = _lib.lib().vitta_scores_workspace_bytes
    assert isinstance(f(1, 131072, 1, 64), int) and f(4096, 101, 0, 5) >= 0 and ctypes.sizeof(ctypes.c_size_t) == 8
