"""What the score operators' backward passes tell the kernels where saved-tensor hooks give back other tensors than were saved (the same
values, laid out in another way), with the launches replaced by a recorder: no GPU is needed, and no memory is read."""
import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
from vitta_amd import _lib, ops


@pytest.fixture
def launches(monkeypatch):
    """Host tensors pass for GPU tensors, and a launch is a line (name, arguments) in the list."""
    made = []
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: -1 if t.is_meta else 0)
    monkeypatch.setattr(ops, "_call", lambda name, index, *args: made.append((name, args)))
    return made


def _scores(kind):
    """Scores (rows, 20) in the layouts that are read in place."""
    whole = torch.randn(6, 5, 32, generator=torch.Generator().manual_seed(1))
    return {"dense": lambda: whole[0, :, :20].contiguous(), "padded": lambda: whole[0, :, 3:23], "cut": lambda: whole[:, :-1, :20],
            "turned": lambda: whole[:, 1:, 12:].transpose(0, 1), "one row": lambda: whole[:1, 0, :20].expand(7, 20),
            "spread": lambda: whole[:, :1, :20].expand(-1, 5, -1), "row": lambda: whole[0, 0, :20]}[kind]()


LAYOUTS = ["dense", "padded", "cut", "turned", "one row", "spread", "row"]
HOOKS = {"none": None, "dense": lambda t: t.contiguous().clone(),
         "wider": lambda t: torch.cat([t, torch.zeros_like(t[..., :1])], -1)[..., :-1] if t.dim() and t.is_floating_point() else t.clone(),
         "classes outside": lambda t: t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t.clone(),
         "groups outside": lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() > 2 else t.clone()}


def _reads(made, given):
    """The score rows that the last launch reads, from the tensors that the hook gave back (anything outside of them is an error)."""
    address, _, rows, classes, stride, inner, outer = made[-1][1][:7]
    for t in given:
        first = t.untyped_storage().data_ptr()
        if first <= address < first + t.untyped_storage().nbytes() and t.dtype == torch.float32:
            flat = torch.empty(0).set_(t.untyped_storage())
            at = (address - first) // 4 + torch.tensor([(r // inner) * outer + (r % inner) * stride for r in range(rows)])
            if at.max() + classes <= flat.numel():
                return flat[at[:, None] + torch.arange(classes)]
    return None  # (a copy that the backward made for itself, or memory that is no tensor's)


def _backward(call, x, hook):
    given = []

    def pack(t):
        return t

    def unpack(t):
        given.append(t if hook is None else hook(t))
        return given[-1]
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        out = call(x)
    (grad,) = torch.autograd.grad(out.sum(), x)
    assert grad.shape == x.shape
    return given


def _calls(lead):
    labels = torch.zeros(lead, dtype=torch.long)
    index = torch.zeros((*lead, 3), dtype=torch.long)
    value = torch.zeros((*lead, 3))
    return {"vitta_label_logprobs_bwd": lambda x: ops.label_logprobs(x, labels, top=2).logprob,
            "vitta_top_distill_bwd": lambda x: ops.top_distill(x, index, value, tail=True)}


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("name", ["vitta_label_logprobs_bwd", "vitta_top_distill_bwd"])
def test_backward_reads_the_scores_that_it_was_given(launches, name, layout, hook):
    x = _scores(layout).detach().requires_grad_()
    copies = []
    given = _backward(_calls(x.shape[:-1])[name], x, HOOKS[hook] and (lambda t: copies.append(HOOKS[hook](t)) or copies[-1]))
    assert launches[-1][0] == name
    assert launches[-1][1][2:4] == (x.numel() // 20, 20)
    read = _reads(launches, given)
    if read is None:  # only where no two strides describe the rows: the backward's own dense copy
        assert hook == "classes outside" and x.dim() > 1 or hook == "groups outside" and x.dim() > 2, "reads outside of the saved scores"
        assert launches[-1][1][4:7] == (20, x.numel() // 20, 0)
    else:
        assert torch.equal(read, x.detach().reshape(-1, 20))


@pytest.mark.parametrize("name", ["vitta_label_logprobs_bwd", "vitta_top_distill_bwd"])
def test_lists_and_statistics_are_read_dense(launches, name):
    """Labels, lists and statistics that come back with gaps between their rows are made dense before the kernel reads them."""
    x = _scores("padded").detach().requires_grad_()

    def gaps(t):
        return torch.stack([t, t], -1)[..., 0]
    given = _backward(_calls(x.shape[:-1])[name], x, gaps)
    args = launches[-1][1]
    for address in args[8:]:
        if isinstance(address, int) and address > 1 << 20:
            assert not any(t.untyped_storage().data_ptr() <= address < t.untyped_storage().data_ptr() + t.untyped_storage().nbytes()
                           for t in given if not t.is_contiguous()), "a tensor with gaps is read as a dense one"


@pytest.mark.parametrize("change", [lambda t: t.half() if t.is_floating_point() else t, lambda t: t.int() if not t.is_floating_point() else t,
                                    lambda t: t[:-1], lambda t: t.to("meta")])
@pytest.mark.parametrize("name", ["vitta_label_logprobs_bwd", "vitta_top_distill_bwd"])
def test_hooks_that_give_back_something_else_are_an_error(launches, name, change):
    x = _scores("padded").detach().requires_grad_()
    with pytest.raises((_lib.VittaHipError, ValueError), match="saved"):
        _backward(_calls(x.shape[:-1])[name], x, change)
    assert launches[-1][0] != name
