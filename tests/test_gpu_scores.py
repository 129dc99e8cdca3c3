"""The score operators on the GPU (ops.label_logprobs, ops.top_distill) against the 64-bit restatement in scores_oracle.py, with the bounds
derived there; a gradient is rounded once more, by half a step of the scores' type."""
import math

import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
import scores_oracle as O

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda"


def _scores(rows, classes, dtype, seed, pad=0, start=0, scale=2.0):
    """(rows, classes) scores cut from a matrix that is `pad` wider and whose first used element is number `start`."""
    gen = torch.Generator().manual_seed(seed)
    whole = (torch.randn(rows, classes + pad + start, generator=gen) * scale).to(dtype)
    return whole.to(DEV)[:, start:start + classes], whole[:, start:start + classes]


def _close(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * math.inf, want)  # (what 32 bits do not hold)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = (got - want).abs()[fine] - torch.as_tensor(bound, dtype=torch.float64).expand_as(want)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), int(off.argmax()))


def _readout_bounds(x, o, temperature):
    """Bounds of logprob / top_logprob (as a function of the log probability), entropy and lse."""
    far = (x.double().amax(1) / temperature).abs()
    far = torch.where(torch.isfinite(far), far, torch.zeros_like(far))
    classes = x.shape[1]
    # log s: the terms' errors (8 |a| u weighted by p: below 8 (H + log V)) and the additions; the score's own difference 8 u |a|
    log_s = O.U * (O.depth(classes) + 40 + 8 * 2 * math.log(classes + 1))
    return (lambda lp: log_s + 12 * O.U * (lp.abs() + math.log(classes + 1) + 1)), \
        (2 * log_s + 8 * O.U) * (2 + 2 * math.log(classes + 1)), log_s + 8 * O.U * (far + math.log(classes + 1) + 1)


def _check_readout(got, x, labels, top, temperature, ignore_index=-100):
    o = O.readout(x, labels, top, temperature, ignore_index)
    b_lp, b_h, b_lse = _readout_bounds(x, o, temperature)
    if labels is not None:
        _close(got.logprob, o["logprob"], b_lp(o["logprob"]), "logprob")
    if got.entropy is not None:
        _close(got.entropy, o["entropy"], b_h, "entropy")
    if got.lse is not None:
        _close(got.lse, o["lse"], b_lse, "lse")
    if top:
        assert torch.equal(got.top_index.cpu(), o["top_index"]), "top_index"
        _close(got.top_logprob, o["top_logprob"], b_lp(o["top_logprob"]), "top_logprob")
    return o


SHAPES = [(1, 1, 1), (2, 2, 1), (3, 7, 7), (5, 63, 20), (4, 64, 64), (9, 101, 5), (33, 174, 10), (6, 400, 64), (3, 513, 3), (2, 1000, 33),
          (5, 2048, 5), (2, 2049, 64), (3, 4096, 17), (3, 4097, 17), (2, 8200, 1), (1, 16385, 64), (2, 32003, 20), (1, 131072, 64), (1, 131075, 5)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,top", SHAPES)
def test_readout(rows, classes, top, dtype):
    from vitta_amd import ops
    for pad, start, temperature in ((0, 0, 1.0), (5, 1, 0.7), (8, 3, 2.5)):
        dx, x = _scores(rows, classes, dtype, classes + rows, pad, start)
        labels = torch.randint(classes, (rows,), generator=torch.Generator().manual_seed(rows))
        labels[rows // 2] = -100
        got = ops.label_logprobs(dx, labels.to(DEV), top=top, lse=True, temperature=temperature)
        _check_readout(got, x, labels, top, temperature)


def test_readout_parts_that_are_not_asked():
    from vitta_amd import ops
    dx, x = _scores(4, 300, torch.float32, 1)
    a = ops.label_logprobs(dx, lse=True)
    assert a.logprob is None and a.top_index is None and a.top_logprob is None
    b = ops.label_logprobs(dx, torch.zeros(4, dtype=torch.int32, device=DEV), entropy=False, top=2)
    assert b.entropy is None
    assert b.lse is None
    full = ops.label_logprobs(dx, torch.zeros(4, dtype=torch.int64, device=DEV), top=2, lse=True)
    assert torch.equal(a.entropy, full.entropy) and torch.equal(a.lse, full.lse)
    assert torch.equal(b.logprob, full.logprob) and torch.equal(b.top_index, full.top_index)


def test_readout_leading_dimensions_and_empty_ones():
    from vitta_amd import ops
    dx, x = _scores(12, 37, torch.bfloat16, 2)
    labels = torch.arange(12, device=DEV)
    flat = ops.label_logprobs(dx, labels, top=3, lse=True)
    deep = ops.label_logprobs(dx.view(2, 3, 2, 37), labels.view(2, 3, 2), top=3, lse=True)
    for a, b in zip(flat, deep):
        assert b.shape[:3] == (2, 3, 2) and torch.equal(a.reshape(-1), b.reshape(-1))
    one = ops.label_logprobs(dx[0], labels[0], top=3, lse=True)
    assert one.logprob.shape == () and one.top_index.shape == (3,) and torch.equal(one.top_index, flat.top_index[0])
    none = ops.label_logprobs(dx[:0], labels[:0], top=3, lse=True)
    assert none.logprob.shape == (0,) and none.top_index.shape == (0, 3)
    turned = ops.label_logprobs(dx.t().contiguous().t(), labels, top=3, lse=True)  # (classes are not the innermost dimension)
    same = ops.label_logprobs(dx[:1].expand(5, 37), labels[:1].expand(5), top=3, lse=True)  # (rows of stride 0)
    for a, b, c in zip(flat, turned, same):
        assert torch.equal(a, b) and torch.equal(c, a[:1].expand_as(c))


@pytest.mark.parametrize("classes", [37, 5001, 40003])
def test_rows_cut_from_sequences(classes):
    """Shifted sequences, transposed leading dimensions and broadcast ones, without a copy of the scores where two strides say it all."""
    from vitta_amd import ops
    whole = (torch.randn(3, 6, classes + 2, generator=torch.Generator().manual_seed(classes)) * 2).bfloat16()
    on = whole.to(DEV)
    labels = torch.randint(classes, (3, 5), generator=torch.Generator().manual_seed(1))
    for make in (lambda t: t[:, :-1, :classes], lambda t: t[:, 1:, 2:].transpose(0, 1), lambda t: t[:, :1, 1:classes + 1].expand(-1, 5, -1),
                 lambda t: t[:, ::2, :classes].unsqueeze(1)):
        x, leaf = make(whole), on.clone().requires_grad_()
        cut = make(leaf)
        y = labels.t().contiguous() if x.shape[:2] == (5, 3) else labels if x.shape[:2] == (3, 5) else labels[:, None, :3].contiguous()
        assert ops._score_rows(cut, "x", 1.0)[0] is cut
        o = ops.label_logprobs(cut, y.to(DEV), top=3, lse=True)
        flat = x.reshape(-1, classes)
        assert o.logprob.shape == x.shape[:-1] and o.top_index.shape == x.shape[:-1] + (3,)
        _check_readout(ops.LabelLogprobs(*[t.flatten(0, x.dim() - 2) for t in o]), flat, y.reshape(-1), 3, 1.0)
        up = torch.randn(flat.shape[0], generator=torch.Generator().manual_seed(2))
        index, value = _list(flat.shape[0], classes, 4, 3, True)
        lead = x.shape[:-1] + (4,)
        loss = ops.top_distill(cut, index.view(lead).to(DEV), value.view(lead).to(DEV), tail=True)
        want, grad_want, b_loss, b_grad = O.distill(flat, index, value, 1.0, True)
        _close(loss.flatten(), want, b_loss, "loss")
        (grad,) = torch.autograd.grad((o.entropy, loss), cut, (up.view(x.shape[:-1]).to(DEV), torch.ones(x.shape[:-1], device=DEV)), retain_graph=True)
        want, bound = O.readout_grad(flat, None, 0, 1.0, None, up)
        # two gradients, each rounded to bfloat16, and their sum
        _check_grad(grad.reshape(-1, classes), want + grad_want, bound + b_grad + 2 * O.half_step(torch.bfloat16) * (want.abs() + grad_want.abs()), torch.bfloat16)
        (grad,) = torch.autograd.grad(o.logprob.sum(), leaf)
        assert grad.shape == whole.shape
    deep = on.view(3, 2, 3, classes + 2)[:, :, :2, :classes]  # three groups: a copy, the same answers
    a = ops.label_logprobs(deep.transpose(0, 2), top=2)
    b = ops.label_logprobs(deep.transpose(0, 2).contiguous(), top=2)
    assert torch.equal(a.entropy, b.entropy) and torch.equal(a.top_index, b.top_index)


ROWS = ["-inf", "one", "two", "lowest", "some lowest", "equal", "zeros", "rising", "falling", "nan", "nan last", "inf", "huge"]


def _odd_rows(classes, dtype):
    """A row of each kind that a mask, a constant model or an overflow leaves."""
    gen = torch.Generator().manual_seed(9)
    x = (torch.randn(len(ROWS), classes, generator=gen) * 2).to(dtype)
    low = torch.finfo(dtype).min
    for r, kind in enumerate(ROWS):
        if kind == "-inf":
            x[r] = -math.inf
        elif kind == "one":
            x[r] = -math.inf
            x[r, classes // 3] = -3.0
        elif kind == "two":
            x[r] = -math.inf
            x[r, [0, classes - 1]] = torch.tensor([1.0, 2.0], dtype=dtype) if classes > 1 else 1.0
        elif kind == "lowest":
            x[r] = low
        elif kind == "some lowest":
            x[r, ::2] = low
        elif kind == "equal":
            x[r] = 1.5
        elif kind == "zeros":
            x[r] = 0.0
            x[r, ::2] = -0.0
        elif kind == "rising":
            x[r] = torch.linspace(-8, 8, classes).to(dtype)
        elif kind == "falling":
            x[r] = torch.linspace(8, -8, classes).to(dtype)
        elif kind == "nan":
            x[r, classes // 2] = math.nan
        elif kind == "nan last":
            x[r, classes - 1] = math.nan
        elif kind == "inf":
            x[r, classes // 4] = math.inf
        elif kind == "huge":
            x[r] = torch.finfo(dtype).max
            x[r, 0] = low
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [1, 3, 64, 101, 700, 4097, 20001])
def test_readout_of_odd_rows(classes, dtype):
    from vitta_amd import ops
    x = _odd_rows(classes, dtype)
    labels = torch.full((len(ROWS),), classes // 3)
    for top in {1, min(classes, 5), min(classes, 64)}:
        for temperature in (1.0, 2.0):
            got = ops.label_logprobs(x.to(DEV), labels.to(DEV), top=top, lse=True, temperature=temperature)
            _check_readout(got, x, labels, top, temperature)


@pytest.mark.parametrize("rows,classes", [(6, 4090), (4, 300001), (530, 20001)])
@pytest.mark.parametrize("top", [1, 5, 64])
def test_rows_that_hide_their_best(rows, classes, top):
    """Rows whose first classes say nothing of the best ones: rising scores, a masked first part, equal scores, one plateau, late spikes."""
    from vitta_amd import ops
    gen = torch.Generator().manual_seed(classes)
    x = torch.randn(rows, classes, generator=gen)
    for r in range(rows):
        kind = r % 6
        if kind == 0:
            x[r] = torch.arange(classes) * 1e-3
        elif kind == 1:
            x[r, : classes * 2 // 3] = -math.inf
        elif kind == 2:
            x[r] = 0.25
        elif kind == 3:
            x[r, classes // 2:] = 9.0
        elif kind == 4:
            x[r, -100:] += 20.0
        else:
            x[r] = torch.sort(x[r]).values
    x = x.bfloat16() if rows < 100 else x
    got = ops.label_logprobs(x.to(DEV), top=top)
    _check_readout(got, x, None, top, 1.0)


@pytest.mark.parametrize("classes", [101, 5000])
def test_labels_that_are_no_class(classes):
    from vitta_amd import ops
    dx, x = _scores(6, classes, torch.float32, 3)
    labels = torch.tensor([-100, -1, classes, 2 ** 40, -2 ** 62, 0])
    leaf = dx.clone().requires_grad_()
    got = ops.label_logprobs(leaf, labels.to(DEV))
    _check_readout(got, x, labels, 0, 1.0)
    (grad,) = torch.autograd.grad(got.logprob, leaf, torch.ones(6, device=DEV))
    assert (grad[0] == 0).all() and torch.isnan(grad[1:5]).all() and torch.isfinite(grad[5]).all()
    other = ops.label_logprobs(dx, labels.to(DEV), ignore_index=-1)
    assert other.logprob[1] == 0 and torch.isnan(other.logprob[0])


def _check_grad(got, want, bound, dtype):
    # one rounding to the type; below its smallest normal the step is fixed
    bound = bound + O.half_step(dtype) * (want.abs() + bound) + torch.finfo(dtype).tiny * O.half_step(dtype)
    _close(got, want, bound, "gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,top", SHAPES)
def test_readout_gradient(rows, classes, top, dtype):
    from vitta_amd import ops
    gen = torch.Generator().manual_seed(7)
    for pad, start, temperature in ((0, 0, 1.0), (3, 1, 0.7)):
        dx, x = _scores(rows, classes, dtype, 11 + classes, pad, start)
        labels = torch.randint(classes, (rows,), generator=gen)
        labels[rows // 2] = -100
        up = [torch.randn(rows, generator=gen) for _ in range(3)] + [torch.randn(rows, top, generator=gen)]
        leaf = dx.detach().requires_grad_()
        o = ops.label_logprobs(leaf, labels.to(DEV), top=top, lse=True, temperature=temperature)
        for use in ((0,), (1,), (0, 1), (0, 1, 2, 3), (3,)):
            outs, ups = zip(*[((o.logprob, o.entropy, o.lse, o.top_logprob)[i], up[i].to(DEV)) for i in use])
            (grad,) = torch.autograd.grad(outs, leaf, ups, retain_graph=True)
            assert grad.dtype == dtype and grad.is_contiguous()
            want, bound = O.readout_grad(x, labels, top, temperature, *[up[i] if i in use else None for i in range(4)])
            _check_grad(grad, want, bound, dtype)


@pytest.mark.parametrize("classes", [3, 101, 4097, 20001])
def test_readout_gradient_of_odd_rows(classes):
    from vitta_amd import ops
    x = _odd_rows(classes, torch.float32)
    labels = torch.full((len(ROWS),), classes // 3)
    top = min(classes, 5)
    leaf = x.to(DEV).requires_grad_()
    o = ops.label_logprobs(leaf, labels.to(DEV), top=top)
    gen = torch.Generator().manual_seed(1)
    up = [torch.randn(len(ROWS), generator=gen), torch.randn(len(ROWS), generator=gen), None, torch.randn(len(ROWS), top, generator=gen)]
    (grad,) = torch.autograd.grad((o.logprob, o.entropy, o.top_logprob), leaf, [u.to(DEV) for u in up if u is not None])
    want, bound = O.readout_grad(x, labels, top, 1.0, *up)
    keep = [r for r, k in enumerate(ROWS) if "nan" not in k and k != "inf"]
    _check_grad(grad[keep], want[keep], bound[keep], torch.float32)
    assert (grad[ROWS.index("-inf")] == 0).all()
    for k in ("nan", "nan last", "inf"):
        assert torch.isnan(grad[ROWS.index(k)]).all()
    # rows that the loss leaves out get zeros, whatever they hold
    (grad,) = torch.autograd.grad((ops.label_logprobs(leaf, torch.full_like(labels, -100).to(DEV)).logprob,), leaf, torch.ones(len(ROWS), device=DEV))
    assert (grad == 0).all()


def test_gradient_of_broadcast_upstreams_and_shared_leaves():
    from vitta_amd import ops
    dx, x = _scores(7, 333, torch.float32, 5)
    labels = torch.arange(7)
    leaf = dx.detach().requires_grad_()
    o = ops.label_logprobs(leaf, labels.to(DEV))
    (-o.logprob.mean() + 0.3 * o.entropy.sum()).backward()
    want, bound = O.readout_grad(x, labels, 0, 1.0, torch.full((7,), -1 / 7), torch.full((7,), 0.3))
    _check_grad(leaf.grad, want, bound, torch.float32)
    # the same leaf twice: the gradients add up
    ops.label_logprobs(leaf, labels.to(DEV)).logprob.sum().backward()
    again, b2 = O.readout_grad(x, labels, 0, 1.0, torch.ones(7))
    _check_grad(leaf.grad, want + again, bound + b2 + O.U * (want + again).abs(), torch.float32)
    # rows of stride 0: one row's gradient is the sum of its uses
    row = dx[0].detach().requires_grad_()
    ops.label_logprobs(row.expand(5, 333), labels[:5].to(DEV)).logprob.sum().backward()
    want, bound = O.readout_grad(x[:1].expand(5, 333).contiguous(), labels[:5], 0, 1.0, torch.ones(5))
    _check_grad(row.grad, want.sum(0), bound.sum(0) + 5 * O.U * want.abs().sum(0), torch.float32)


def test_gradient_against_differences():
    from vitta_amd import ops
    dx, x = _scores(3, 13, torch.float32, 6)
    labels = torch.tensor([1, 12, 5])
    up = torch.randn(3, generator=torch.Generator().manual_seed(2)), torch.randn(3, generator=torch.Generator().manual_seed(3))
    leaf = dx.detach().requires_grad_()
    o = ops.label_logprobs(leaf, labels.to(DEV), temperature=0.8)
    (grad,) = torch.autograd.grad((o.logprob, o.entropy), leaf, [u.to(DEV) for u in up])
    h = 1e-5
    for j in range(13):
        a, b = x.double(), x.double()
        a[:, j] += h
        b[:, j] -= h
        f = [sum(u * O.readout(z, labels, 0, 0.8)[k] for u, k in zip(up, ("logprob", "entropy"))) for z in (a, b)]
        _, bound = O.readout_grad(x, labels, 0, 0.8, *up)
        _close(grad[:, j], (f[0] - f[1]) / (2 * h), bound[:, j] + O.U * 4 + 1e-8, "difference")


def _list(rows, classes, k, seed, tail, dtype=torch.float32, ragged=True):
    gen = torch.Generator().manual_seed(seed)
    index = torch.stack([torch.randperm(classes, generator=gen)[:k] for _ in range(rows)])
    value = torch.randn(rows, k, generator=gen) * 1.5
    if tail:
        rest = torch.cat([value, torch.randn(rows, 1, generator=gen) + 1], 1)
        value = (value - torch.logsumexp(rest, 1, keepdim=True))
    if ragged:
        index[torch.arange(k)[None, :] >= torch.randint(1, k + 1, (rows, 1), generator=gen)] = -1
    return index, value.to(dtype)


LISTS = [(1, 1, 1), (3, 7, 7), (5, 64, 20), (9, 101, 5), (33, 174, 10), (6, 400, 64), (3, 513, 256), (2, 2049, 64), (3, 4097, 17), (1, 16385, 64),
         (2, 32003, 20), (1, 131075, 100)]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,k", LISTS)
def test_distillation(rows, classes, k, dtype, tail):
    from vitta_amd import ops
    for pad, start, temperature in ((0, 0, 1.0), (5, 1, 2.0)):
        dx, x = _scores(rows, classes, dtype, classes, pad, start)
        index, value = _list(rows, classes, k, rows + k, tail)
        up = torch.randn(rows, generator=torch.Generator().manual_seed(4))
        leaf = dx.detach().requires_grad_()
        loss = ops.top_distill(leaf, index.to(DEV), value.to(DEV), temperature=temperature, tail=tail)
        want, grad_want, b_loss, b_grad = O.distill(x, index, value, temperature, tail)
        _close(loss, want, b_loss, "loss")
        assert torch.equal(ops.top_distill(dx, index.to(DEV), value.to(DEV), temperature=temperature, tail=tail), loss)
        (grad,) = torch.autograd.grad(loss, leaf, up.to(DEV))
        u = up.double()[:, None]
        _check_grad(grad, grad_want * u, b_grad * u.abs() + 2 * O.U * (grad_want * u).abs(), dtype)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("value_dtype", TYPES)
def test_distillation_types_of_the_list(value_dtype, tail):
    from vitta_amd import ops
    dx, x = _scores(6, 222, torch.bfloat16, 8)
    index, value = _list(6, 222, 12, 3, tail, value_dtype)
    got = ops.top_distill(dx, index.int().to(DEV), value.to(DEV), tail=tail)
    want, _, b, _ = O.distill(x, index, value, 1.0, tail)
    _close(got, want, b, "loss")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("classes", [16, 101, 5000, 20001])
def test_distillation_odd_lists(classes, tail):
    """Padding only, one class, a class twice, numbers that are no class, a list of every class, a class of probability 0."""
    from vitta_amd import ops
    k = 16
    dx, x = _scores(8, classes, torch.float32, 12)
    index, value = _list(8, classes, k, 5, tail, ragged=False)
    index[0] = -1
    index[1, 1:] = -1
    index[2] = index[2, :1]
    index[3, ::2] = index[3, 1::2]
    index[4, :4] = torch.tensor([classes, -7, 2 ** 40, -2 ** 62])
    value[5, 3] = -math.inf
    value[2] -= 3.0 if tail else 0.0
    index[6] = torch.arange(k)
    value[7] = value[7, 0] if not tail else math.log(1 / 64)
    leaf = dx.detach().requires_grad_()
    loss = ops.top_distill(leaf, index.to(DEV), value.to(DEV), tail=tail)
    want, grad_want, b_loss, b_grad = O.distill(x, index, value.nan_to_num(neginf=-1e30), 1.0, tail)
    _close(loss, want, b_loss, "loss")
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    _check_grad(grad, grad_want, b_grad, torch.float32)
    assert loss[0] == 0 and (grad[0] == 0).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("classes", [101, 4097, 20001])
def test_distillation_of_odd_rows(classes, tail):
    from vitta_amd import ops
    x = _odd_rows(classes, torch.float32)
    index, value = _list(len(ROWS), classes - 1, 8, 6, tail, ragged=False)
    index += 1  # (not the class that "huge" holds at its lowest: its loss is beyond 32 bits)
    leaf = x.to(DEV).requires_grad_()
    loss = ops.top_distill(leaf, index.to(DEV), value.to(DEV), tail=tail)
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    want, grad_want, b_loss, b_grad = O.distill(x, index, value, 1.0, tail)
    keep = [r for r, k in enumerate(ROWS) if k in ("lowest", "some lowest", "equal", "zeros", "rising", "falling", "huge")]
    # a class at the type's lowest value has a log probability of that size, rounded like any other
    _close(loss[keep], want[keep], b_loss[keep], "loss")
    _check_grad(grad[keep], grad_want[keep], b_grad[keep], torch.float32)
    for k in ("nan", "nan last", "inf"):
        assert torch.isnan(loss[ROWS.index(k)]) and torch.isnan(grad[ROWS.index(k)]).all()
    for k in ("-inf", "one", "two"):
        assert loss[ROWS.index(k)] == math.inf and not torch.isnan(grad[ROWS.index(k)]).any()
    padded = ops.top_distill(leaf, torch.full_like(index, -1).to(DEV), value.to(DEV), tail=tail)
    assert (padded == 0).all() and (torch.autograd.grad(padded.sum(), leaf)[0] == 0).all()


@pytest.mark.parametrize("classes", [101, 5000])
@pytest.mark.parametrize("gap", [60.0, 90.0, 140.0, 1000.0])
def test_distillation_of_a_certain_student(classes, gap):
    """A student that gives the classes outside the list next to nothing (their sum underflows 32 bits): their share of the rest holds."""
    from vitta_amd import ops
    dx, x = _scores(3, classes, torch.float32, 13)
    index, value = _list(3, classes, 6, 7, True, ragged=False)
    x.scatter_add_(1, index, torch.full((3, 6), gap))
    leaf = x.to(DEV).requires_grad_()
    loss = ops.top_distill(leaf, index.to(DEV), value.to(DEV), tail=True)
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    z = x.double()
    listed = torch.zeros_like(z, dtype=torch.bool).scatter_(1, index, True)
    rest = 1 - torch.exp(value.double()).sum(1)
    lse = torch.logsumexp(z, 1)
    lse_out = torch.logsumexp(torch.where(listed, -math.inf, z), 1)
    want = (torch.exp(value.double()) * (value.double() - (z - lse[:, None]).gather(1, index))).sum(1) + rest * (torch.log(rest) - lse_out + lse)
    # 8 u on each logarithm and on the differences of scores, (depth + 40) u on the sums, 8 u on the list's mass
    scale = lse.abs() + lse_out.abs() + gap + value.double().abs().amax(1) + 2
    _close(loss, want, O.U * (O.depth(classes) + 100) * scale, "loss")
    share = torch.exp(torch.where(listed, -math.inf, z) - lse_out[:, None])
    grad_want = torch.exp(z - lse[:, None]) - torch.zeros_like(z).scatter_(1, index, torch.exp(value.double())) - rest[:, None] * share
    spread = (z.amax(1, keepdim=True) - z).abs()
    bound = O.U * (O.depth(classes) + 60 + 8 * torch.where(listed, spread, spread - gap).abs()) * (torch.exp(z - lse[:, None]) + share) \
        + 40 * O.U * (listed * 1.0 + share)
    _check_grad(grad, grad_want, bound, torch.float32)


def test_teacher_list_from_the_readout_trains_a_student():
    """The operators as they are used together: a teacher's readout gives the list, the student's loss and gradient follow, and the
    gradient points to the teacher (its step lowers the loss by the first order term)."""
    from vitta_amd import ops
    teacher, _ = _scores(24, 400, torch.bfloat16, 20)
    masked = teacher.clone()
    masked[:, 7:] = torch.where(torch.arange(393, device=DEV) % 50 == 0, masked[:, 7:], torch.tensor(-math.inf, dtype=torch.bfloat16, device=DEV))
    for t, tail in ((teacher, True), (teacher, False), (masked, True)):
        best = ops.label_logprobs(t, top=20, entropy=False, temperature=1.5)
        student, x = _scores(24, 400, torch.float32, 21)
        leaf = student.detach().requires_grad_()
        value = best.top_logprob if tail else best.top_logprob * 1.5
        loss = ops.top_distill(leaf, best.top_index, value, temperature=1.5, tail=tail)
        want, grad_want, b_loss, b_grad = O.distill(x, best.top_index.cpu(), value.cpu(), 1.5, tail)
        _close(loss, want, b_loss, "loss")
        (grad,) = torch.autograd.grad(loss.sum(), leaf)
        _check_grad(grad, grad_want, b_grad, torch.float32)
        if t is masked:
            assert (best.top_index[:, 15:] == -1).all()


@pytest.mark.parametrize("rows,classes,dtype", [(2, 600001, torch.float32), (520, 300001, torch.bfloat16), (1, 2 ** 24, torch.float16)])
def test_very_long_rows(rows, classes, dtype):
    """More classes than one workgroup's membership bits hold, few rows and more than have tickets; the largest vocabulary."""
    from vitta_amd import _lib, ops
    gen = torch.Generator(device=DEV).manual_seed(classes)
    dx = torch.empty(rows, classes, dtype=dtype, device=DEV).normal_(0, 2, generator=gen)
    index, value = _list(1, classes, 33, 5, True)
    index, value = (index + torch.arange(rows)[:, None]) % classes, value.expand(rows, 33).contiguous()
    index[0, -2:] = torch.tensor([0, classes - 1])
    labels = torch.arange(rows) * 7
    leaf = dx.requires_grad_()
    o = ops.label_logprobs(leaf, labels.to(DEV), top=64, lse=True)
    loss = ops.top_distill(leaf, index.to(DEV), value.to(DEV), tail=True)
    (g1,) = torch.autograd.grad(o.entropy, leaf, torch.ones(rows, device=DEV))
    (g2,) = torch.autograd.grad(loss, leaf, torch.ones(rows, device=DEV))
    for r in {0, rows // 2, rows - 1}:
        x = dx[r:r + 1].detach().cpu()
        _check_readout(ops.LabelLogprobs(*[t[r:r + 1].detach() for t in o]), x, labels[r:r + 1], 64, 1.0)
        want, bound = O.readout_grad(x, labels[r:r + 1], 64, 1.0, None, torch.ones(1))
        _check_grad(g1[r:r + 1], want, bound, dtype)
        want, grad_want, b_loss, b_grad = O.distill(x, index[r:r + 1], value[r:r + 1], 1.0, True)
        _close(loss[r:r + 1], want, b_loss, "loss")
        _check_grad(g2[r:r + 1], grad_want, b_grad, dtype)
    if classes == 2 ** 24:
        with pytest.raises(_lib.VittaHipError, match="unsupported|nsupported"):
            ops.label_logprobs(torch.zeros(1, classes + 1, dtype=dtype, device=DEV))


def test_gradients_of_no_rows():
    from vitta_amd import ops
    leaf = torch.zeros(0, 3, 9, device=DEV, requires_grad=True)
    o = ops.label_logprobs(leaf, torch.zeros(0, 3, dtype=torch.long, device=DEV), top=2)
    loss = ops.top_distill(leaf, torch.zeros(0, 3, 4, dtype=torch.long, device=DEV), torch.zeros(0, 3, 4, device=DEV))
    assert o.top_index.shape == (0, 3, 2) and loss.shape == (0, 3)
    (grad,) = torch.autograd.grad((o.logprob.sum() + o.entropy.sum() + loss.sum()), leaf)
    assert grad.shape == leaf.shape


def test_modified_scores_are_noticed():
    """The backward reads the scores again: changed in place in between, they are an error and not a wrong gradient."""
    from vitta_amd import ops
    x = torch.randn(3, 20, device=DEV)
    leaf = x.clone().requires_grad_()
    y = leaf * 1.0
    o = ops.label_logprobs(y)
    y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.entropy.sum().backward()


def test_far_offsets():
    """Rows that begin beyond 2^31 elements."""
    from vitta_amd import ops
    step = 2 ** 30 + 24
    whole = torch.zeros(3 * step, dtype=torch.bfloat16, device=DEV)
    dx = whole.as_strided((3, 5001), (step, 1))
    x = _scores(3, 5001, torch.bfloat16, 30)[1]
    dx.copy_(x.to(DEV))
    labels = torch.tensor([1, 5000, 77])
    leaf = dx.detach().requires_grad_()
    o = ops.label_logprobs(leaf, labels.to(DEV), top=8, lse=True)
    _check_readout(o, x, labels, 8, 1.0)
    (grad,) = torch.autograd.grad(o.logprob, leaf, torch.ones(3, device=DEV))
    want, bound = O.readout_grad(x, labels, 0, 1.0, torch.ones(3))
    _check_grad(grad, want, bound, torch.bfloat16)
    del whole, dx, leaf, o, grad
    rows = 70001
    big = torch.empty(rows, 32771, dtype=torch.bfloat16, device=DEV).normal_()
    leaf = big.requires_grad_()
    o = ops.label_logprobs(leaf, top=2, lse=True)
    (grad,) = torch.autograd.grad(o.entropy, leaf, torch.ones(rows, device=DEV))
    for r in (0, 40000, 65535, 65536, rows - 1):
        x = big[r:r + 1].detach().cpu()
        _check_readout(ops.LabelLogprobs(None, o.entropy[r:r + 1].detach(), o.lse[r:r + 1].detach(), o.top_logprob[r:r + 1].detach(), o.top_index[r:r + 1]), x, None, 2, 1.0)
        want, bound = O.readout_grad(x, None, 0, 1.0, None, torch.ones(1))
        _check_grad(grad[r:r + 1], want, bound, torch.bfloat16)


def test_more_rows_than_one_launch_takes():
    """Millions of rows (of stride 0, so that they need no memory): launches of 2^31 threads at most follow one another."""
    from vitta_amd import ops
    for rows, classes, top in ((4_200_000, 5000, 0), (8_400_005, 4500, 2)):
        x = _scores(1, classes, torch.bfloat16, classes)[1]
        got = ops.label_logprobs(x.to(DEV).expand(rows, classes), top=top)
        assert torch.equal(got.entropy, got.entropy[:1].expand(rows))
        if top:
            assert torch.equal(got.top_index, got.top_index[:1].expand(rows, top))
        _check_readout(ops.LabelLogprobs(*[None if t is None else t[-1:] for t in got]), x, None, top, 1.0)
    rows, classes = 8_400_005, 2049
    x = _scores(1, classes, torch.bfloat16, 3)[1]
    wide = x.to(DEV).expand(rows, classes).requires_grad_()
    (grad,) = torch.autograd.grad(ops.label_logprobs(wide).entropy.sum(), wide)
    want, bound = O.readout_grad(x, None, 0, 1.0, None, torch.ones(1))
    for r in (0, 8_388_604, 8_388_608, rows - 1):
        _check_grad(grad[r:r + 1], want, bound, torch.bfloat16)
    assert torch.equal(grad[-1], grad[0]) and bool((grad[::1000] == grad[0]).all())


@pytest.mark.parametrize("rows,classes", [(1, 131072), (40, 101), (300, 9001)])
def test_repeats_streams_and_graphs(rows, classes):
    """Equal bits on a second call, on another stream, and on every replay of a captured graph with other work in between."""
    from vitta_amd import ops
    dx, _ = _scores(rows, classes, torch.bfloat16, 40)
    labels = torch.arange(rows, device=DEV) % classes
    index, value = _list(rows, classes, 12, 41, True)
    index, value, up = index.to(DEV), value.to(DEV), torch.rand(rows, device=DEV)

    def step(x):
        x = x.detach().requires_grad_()
        o = ops.label_logprobs(x, labels, top=12, lse=True)
        g = torch.autograd.grad((o.logprob, o.entropy, o.top_logprob), x, (up, up, up[:, None].expand(rows, 12)))
        loss = ops.top_distill(x, index, value, tail=True)
        return [t.detach() for t in o] + [g[0], loss.detach(), torch.autograd.grad(loss, x, up)[0]]

    first = step(dx)
    for a, b in zip(first, step(dx)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(dx)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    static = dx.clone()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph in graphs:  # (two graphs of the same inputs, each with workspaces of its own)
        with torch.cuda.graph(graph):
            outs.append(step(static))
    for turn in range(4):
        x, _ = _scores(rows, classes, torch.bfloat16, 50 + turn)
        static.copy_(x)
        want = step(x)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for graph, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for got in outs:
            for a, b in zip(want, got):
                assert torch.equal(a, b)
        torch.rand(1000, device=DEV).sum().item()


@pytest.mark.parametrize("rows,classes,top", [(1, 131072, 20), (3, 50001, 64), (200, 40001, 0), (511, 17000, 3)])
def test_segments_join_in_one_launch_or_two(rows, classes, top, monkeypatch):
    """Equal bits whether the last segment joins a row or a second launch does, many times over, on streams side by side; and the tickets
    are zero afterwards."""
    from vitta_amd import _lib, ops
    x = [_scores(rows, classes, torch.bfloat16, 70 + i)[0] for i in range(3)]
    labels = torch.arange(rows, device=DEV)
    index, value = _list(rows, classes, 9, 71, True)
    index, value = index.to(DEV), value.to(DEV)
    assert _lib.lib().vitta_scores_workspace_bytes(rows, classes, 1, top) > 0

    def step(x):
        o = ops.label_logprobs(x, labels, top=top, lse=True)
        return [t for t in o if t is not None] + [ops.top_distill(x, index, value, tail=True)]

    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        want = [step(a) for a in x]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for turn in range(20):
        got = []
        for a, s in zip(x, streams):
            with torch.cuda.stream(s):
                got.append(step(a))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            for u, v in zip(a, b):
                assert torch.equal(u, v)
    assert len(ops._score_tickets) >= 3 and all(int(t.abs().sum()) == 0 for t in ops._score_tickets.values())


def test_refusals():
    from vitta_amd import _lib, ops
    dx, _ = _scores(4, 50, torch.float32, 60)
    labels = torch.zeros(4, dtype=torch.long, device=DEV)
    for bad in (-1, 51, 65):
        with pytest.raises(ValueError, match="top"):
            ops.label_logprobs(dx, labels, top=bad)
    for bad in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="temperature"):
            ops.label_logprobs(dx, labels, temperature=bad)
        with pytest.raises(ValueError, match="temperature"):
            ops.top_distill(dx, labels[:, None], dx[:, :1], temperature=bad)
    with pytest.raises(ValueError, match="nothing"):
        ops.label_logprobs(dx, entropy=False)
    with pytest.raises(ValueError, match="labels"):
        ops.label_logprobs(dx, labels[:3])
    with pytest.raises(_lib.VittaHipError, match="labels"):
        ops.label_logprobs(dx, labels.float())
    with pytest.raises(_lib.VittaHipError, match="labels"):
        ops.label_logprobs(dx, labels.cpu())
    with pytest.raises(_lib.VittaHipError, match="float32"):
        ops.label_logprobs(dx.double(), labels)
    with pytest.raises(ValueError, match="classes"):
        ops.label_logprobs(dx[:, :0], labels)
    with pytest.raises(ValueError, match="teacher_index"):
        ops.top_distill(dx, torch.zeros(4, 257, dtype=torch.long, device=DEV), torch.zeros(4, 257, device=DEV))
    with pytest.raises(ValueError, match="teacher_index"):
        ops.top_distill(dx, torch.zeros(4, 0, dtype=torch.long, device=DEV), torch.zeros(4, 0, device=DEV))
    with pytest.raises(ValueError, match="teacher_value"):
        ops.top_distill(dx, labels[:, None], torch.zeros(4, 2, device=DEV))
    with pytest.raises(ValueError, match="gradient"):
        ops.top_distill(dx, labels[:, None], torch.zeros(4, 1, device=DEV, requires_grad=True))
    with pytest.raises(_lib.VittaHipError, match="teacher_index"):
        ops.top_distill(dx, labels[:, None].float(), torch.zeros(4, 1, device=DEV))
    leaf = dx.detach().requires_grad_()
    (grad,) = torch.autograd.grad(ops.label_logprobs(leaf, labels).logprob.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):  # a second derivative does not exist
        grad.sum().backward()
