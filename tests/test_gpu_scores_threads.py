"""The score operators called from several threads at once: two on the default stream, which they share with its tickets, two on streams of
their own.  Every answer has the bits of a call by itself."""
import threading

import pytest
import torch

import helpers as H  # noqa: F401  (puts the repo root on sys.path)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,classes", [(1, 131072), (3, 50001), (64, 400)])
def test_threads(rows, classes):
    from vitta_amd import ops
    gen = torch.Generator().manual_seed(rows)
    xs = [(torch.randn(rows, classes, generator=gen) * 2).bfloat16().cuda() for _ in range(4)]
    labels = torch.arange(rows).cuda()
    index = torch.randint(-1, classes, (rows, 9), generator=gen).cuda()
    value = (torch.randn(rows, 9, generator=gen) - 4).cuda()
    up = torch.rand(rows, generator=gen).cuda()

    def step(x):
        x = x.detach().requires_grad_()
        o = ops.label_logprobs(x, labels, top=7, lse=True)
        loss = ops.top_distill(x, index, value, tail=True)
        grads = torch.autograd.grad((o.logprob, o.entropy, loss), x, (up, up, up))
        return [t.detach() for t in o] + [loss.detach(), grads[0]]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.default_stream(), torch.cuda.default_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    wrong, start = [], threading.Barrier(4)

    def work(i):
        try:
            with torch.cuda.stream(streams[i]):
                start.wait(30)
                for turn in range(25):
                    got = step(xs[i])
                    streams[i].synchronize()
                    wrong.extend((i, turn, k) for k, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
        except Exception as e:  # (an exception of a thread would go unnoticed)
            wrong.append((i, repr(e)))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []
