"""The score operators' gradients where saved-tensor hooks give back the scores, labels and lists in another layout: equal bits, for the
kernels read the same values wherever they lie (the layout decides only how they are loaded)."""
import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)
from test_scores_saved_cpu import HOOKS, LAYOUTS

pytestmark = pytest.mark.gpu


def _scores(kind, classes, dtype):
    whole = (torch.randn(6, 5, classes + 12, generator=torch.Generator().manual_seed(classes)) * 2).to(dtype).cuda()
    return {"dense": lambda: whole[0, :, :classes].contiguous(), "padded": lambda: whole[0, :, 3:classes + 3], "cut": lambda: whole[:, :-1, :classes],
            "turned": lambda: whole[:, 1:, 12:].transpose(0, 1), "one row": lambda: whole[:1, 0, :classes].expand(7, classes),
            "spread": lambda: whole[:, :1, :classes].expand(-1, 5, -1), "row": lambda: whole[0, 0, :classes]}[kind]()


@pytest.mark.parametrize("how", ["save_on_cpu", "save_on_cpu, pinned", *HOOKS])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("classes,dtype", [(20, torch.float32), (3001, torch.bfloat16), (40001, torch.float16)])
def test_gradients_with_saved_tensor_hooks(classes, dtype, layout, how):
    from vitta_amd import ops
    x = _scores(layout, classes, dtype).detach().requires_grad_()
    lead = x.shape[:-1]
    gen = torch.Generator().manual_seed(3)
    labels = torch.randint(classes, lead, generator=gen).cuda()
    index = torch.randint(-1, classes, (*lead, 5), generator=gen).cuda()
    value = (torch.randn((*lead, 5), generator=gen) - 3).cuda()
    up = torch.randn(lead, generator=gen).cuda()

    def grads():
        o = ops.label_logprobs(x, labels, top=4, lse=True)
        loss = ops.top_distill(x, index, value, tail=True)
        return [(o.logprob, up), (o.entropy, up), (o.top_logprob, up[..., None].expand(*lead, 4)), (loss, up)]
    want = [torch.autograd.grad(out, x, u, retain_graph=True)[0] for out, u in grads()]
    if how.startswith("save_on_cpu"):
        hooks = torch.autograd.graph.save_on_cpu(pin_memory="pinned" in how)
    else:
        hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t, HOOKS[how] or (lambda t: t))
    with hooks:
        outs = grads()
    for w, (out, u) in zip(want, outs):
        (g,) = torch.autograd.grad(out, x, u, retain_graph=True)
        assert torch.equal(g, w)


@pytest.mark.parametrize("reentrant", [False, True])
def test_gradients_of_recomputed_scores(reentrant):
    from torch.utils.checkpoint import checkpoint
    from vitta_amd import ops
    x = _scores("cut", 500, torch.float32).detach().requires_grad_()
    labels = torch.randint(500, x.shape[:-1], generator=torch.Generator().manual_seed(5)).cuda()

    def loss(y):
        o = ops.label_logprobs(y[..., 1:] * 1.5, labels % 499, top=3)
        return o.entropy - o.logprob + ops.top_distill(y[..., :499], o.top_index, o.top_logprob.detach(), tail=True)
    (want,) = torch.autograd.grad(loss(x).sum(), x)
    (got,) = torch.autograd.grad(checkpoint(loss, x, use_reentrant=False).sum(), x) if not reentrant else (None,)
    if reentrant:
        leaf = x.detach().clone().requires_grad_()
        checkpoint(loss, leaf, use_reentrant=True).sum().backward()
        got = leaf.grad
    assert torch.equal(got, want)


def test_what_a_backward_has_read_is_freed():
    """A loss that is kept with its graph holds neither scores nor statistics after its backward."""
    from vitta_amd import ops
    x = torch.randn(4096, 300, device="cuda", requires_grad=True)
    index = torch.arange(64, device="cuda").expand(4096, 64).contiguous()
    value = torch.zeros(4096, 64, device="cuda")
    held = []
    for turn in range(3):
        loss = ops.top_distill(x, index, value)
        logprob = ops.label_logprobs(x, index[:, 0].contiguous(), entropy=False).logprob
        torch.autograd.grad(loss.sum() - logprob.sum(), x)
        if turn == 0:  # (after the first turn: what the allocator rounds, and the library's own first use)
            before = torch.cuda.memory_allocated()
        held.append((loss, logprob))
    assert torch.cuda.memory_allocated() - before <= 2 * 2 * 4096 * 4 + 4 * 512
