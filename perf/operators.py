"""Measured cases of the score operators: `ops.label_logprobs` (log probability of given labels, entropy and best alternatives of rows of class
scores, forward and gradient) and `ops.top_distill` (distillation from a teacher's top list, forward and gradient).

`run` with `own` false computes a case in elementary torch operations, in 32 bits (the teacher's remaining mass in 64), rounded once at the
end; with `own` true it makes the calls a user of the framework makes.  `exact` restates the definitions in 64 bits."""
import math

import torch

own = False

IGNORED = -100
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
#: rows x classes of the largest listed cases; drawn cases stay below
MOST = 4096 * 131072


def _case(name, op, rows, classes, dtype, top, temperature=1.0, pad=0, masked=False, wants="both", tail=False):
    return {"name": name, "op": op, "rows": rows, "classes": classes, "dtype": dtype, "top": top, "temperature": temperature, "pad": pad,
            "masked": masked, "wants": wants, "tail": tail}


def listed():
    return [
        # the scores of one test batch of clips: label, confidence and top five of UCF101's classes -- launch latency
        _case("readout 8x101 f32", "readout", 8, 101, "float32", 5),
        # one token of a generating model: no label, entropy and 20 alternatives of a long row
        _case("readout 1x131072 bf16", "readout", 1, 131072, "bfloat16", 20, temperature=0.7),
        # scoring a text or a set of clips against a mid-sized vocabulary, rows of odd length
        _case("readout 2048x32003 f16", "readout", 2048, 32003, "float16", 5),
        # the largest: scoring a long batch, with the alternatives that a student is trained on later
        _case("readout 4096x131072 bf16", "readout", 4096, 131072, "bfloat16", 64),
        # entropy minimisation at test time on Kinetics' 400 classes
        _case("entropy grad 64x400 f32", "readout_grad", 64, 400, "float32", 0, wants="entropy"),
        # a fine-tuning step: log probabilities of the labels and their gradient; scores cut from a padded matrix
        _case("logprob grad 1024x50021 f32", "readout_grad", 1024, 50021, "float32", 0, pad=27, wants="logprob"),
        # a policy step: advantages on the log probabilities, a bonus on the entropy
        _case("policy grad 4096x131072 bf16", "readout_grad", 4096, 131072, "bfloat16", 0, wants="both"),
        # a teacher's ten best of Something-Something's 174 classes
        _case("distil grad 16x174 f32", "distill_grad", 16, 174, "float32", 10, temperature=2.0),
        # validation of a student: the loss alone, the teacher's log probabilities with the rest as one class
        _case("distil 512x65537 f32", "distill", 512, 65537, "float32", 20, tail=True),
        # a distillation step over an odd vocabulary, list renormalised
        _case("distil grad 2048x32003 bf16", "distill_grad", 2048, 32003, "bfloat16", 32, temperature=2.0),
        # the largest distillation step, with the rest as one class
        _case("distil grad 4096x131072 bf16", "distill_grad", 4096, 131072, "bfloat16", 64, tail=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["readout", "readout", "readout_grad", "distill", "distill_grad"])
    classes = _spread(rng, 48, 131072)
    if rng.random() < 0.5:
        classes |= 1
    # single rows are a generating model's long ones; class scores come by the batch
    rows = _spread(rng, 1 if classes > 4096 else 4, min(8192, MOST // classes))
    lists = op != "readout_grad"
    top = min(_spread(rng, 1, 64), classes // 2) if lists else 0
    return {"op": op, "rows": rows, "classes": classes, "dtype": rng.choice(["float32", "bfloat16", "bfloat16", "float16"]), "top": top,
            "temperature": rng.choice([1.0, 1.0, 0.7, 2.0, round(rng.uniform(0.7, 4.0), 3)]), "pad": rng.choice([0, 0, 8, rng.randint(1, 40)]),
            "masked": op in ("readout", "readout_grad") and rng.random() < 0.3, "wants": rng.choice(["both", "logprob", "entropy"]),
            "tail": op.startswith("distill") and rng.random() < 0.5}


def _scores(case, gen, dev):
    """Rows of scores as a model gives them: a broad bulk, and a matrix wider than the classes where a case has a pad."""
    rows, width = case["rows"], case["classes"] + case["pad"]
    whole = torch.empty(rows, width, dtype=TYPES[case["dtype"]], device=dev)
    for at in range(0, rows, 1024):  # (in parts: the 32-bit scores of the largest cases need not be there at once)
        part = torch.randn(min(1024, rows - at), width, generator=gen, device=dev)
        whole[at:at + 1024] = part * 2
    return whole[:, :case["classes"]]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, classes = case["rows"], case["classes"]
    x = _scores(case, gen, dev)
    r = torch.arange(rows, device=dev)
    state = {"case": case, "x": x}
    if case["op"].startswith("readout"):
        labels = torch.randint(classes, (rows,), generator=gen, device=dev)
        # a trained model gives most labels a high score
        x[r, labels] = (x[r, labels].float() + 6 * torch.rand(rows, generator=gen, device=dev)).to(x.dtype)
        if case["masked"]:  # classes that are ruled out, and now and then a whole row
            x.masked_fill_(torch.rand(rows, 1, generator=gen, device=dev) * 0.9 > torch.rand(1, classes, generator=gen, device=dev), -math.inf)
            x.masked_fill_((r % 17 == 5)[:, None], -math.inf)
        labels[torch.rand(rows, generator=gen, device=dev) < 0.05] = IGNORED  # padding
        state["labels"] = labels
        state["up_logprob"] = torch.randn(rows, generator=gen, device=dev)
        state["up_entropy"] = 0.5 + torch.rand(rows, generator=gen, device=dev)
    else:
        k = case["top"]
        step = torch.randint(1, max(2, classes // k + 1), (rows, 1), generator=gen, device=dev)
        index = (torch.randint(classes, (rows, 1), generator=gen, device=dev) + step * torch.arange(k, device=dev)) % classes
        value = 9 - torch.cumsum(-torch.log(torch.rand(rows, k, generator=gen, device=dev)) * (4.0 / k), 1)
        x[r[:, None], index] = (value + torch.randn(rows, k, generator=gen, device=dev)).to(x.dtype)
        if case["tail"]:  # log probabilities that leave some mass to the classes outside the list
            rest = value.new_zeros(rows, 1) + 3 + 4 * torch.rand(rows, 1, generator=gen, device=dev)
            both = torch.cat([value, rest], 1)
            value = (both - both.logsumexp(1, keepdim=True))[:, :k].contiguous()
        length = torch.randint(max(1, k // 2), k + 1, (rows, 1), generator=gen, device=dev)
        length[r % 16 == 11] = 0  # padded rows
        state["index"] = torch.where(torch.arange(k, device=dev) < length, index, -1)
        state["value"] = value
        state["up"] = 0.5 + torch.rand(rows, generator=gen, device=dev)
    return state


def run(state):
    case, x = state["case"], state["x"]
    if own:
        return _own(state)
    if case["op"] == "readout":
        return _readout(x, state["labels"], case["top"], case["temperature"])
    if case["op"] == "readout_grad":
        return _readout_grad(x, state["labels"], case["wants"], state["up_logprob"], state["up_entropy"], case["temperature"])
    return _distill(x, state["index"], state["value"], case["temperature"], case["tail"], state["up"] if case["op"] == "distill_grad" else None)


def _own(state):
    from vitta_amd import ops
    case, x = state["case"], state["x"]
    if case["op"] == "readout":
        out = ops.label_logprobs(x, state["labels"], top=case["top"], temperature=case["temperature"], ignore_index=IGNORED)
        return {"logprob": out.logprob, "entropy": out.entropy, "top_logprob": out.top_logprob, "top_index": out.top_index}
    if case["op"] == "readout_grad":
        x = x.detach().requires_grad_()
        wants = case["wants"]
        out = ops.label_logprobs(x, state["labels"] if wants != "entropy" else None, entropy=wants != "logprob", temperature=case["temperature"],
                                 ignore_index=IGNORED)
        outs = ([out.logprob] if wants != "entropy" else []) + ([out.entropy] if wants != "logprob" else [])
        ups = ([state["up_logprob"]] if wants != "entropy" else []) + ([state["up_entropy"]] if wants != "logprob" else [])
        (grad,) = torch.autograd.grad(outs, x, ups)
        return {"outs": [o.detach() for o in outs], "grad": grad}
    if case["op"] == "distill":
        return {"loss": ops.top_distill(x, state["index"], state["value"], temperature=case["temperature"], tail=case["tail"])}
    x = x.detach().requires_grad_()
    loss = ops.top_distill(x, state["index"], state["value"], temperature=case["temperature"], tail=case["tail"])
    (grad,) = torch.autograd.grad(loss, x, state["up"])
    return {"loss": loss.detach(), "grad": grad}


# ---- the plain forms ----------------------------------------------------------------------------------------------------------
def _softmax(x, temperature):
    """z - m, exp(z - m), its sum and m; m is 0 for a row without any finite score, whose sum is 0."""
    z = x.float() / temperature
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    d = z - m
    e = torch.exp(d)
    return d, e, e.sum(-1, keepdim=True), m


def _label_and_entropy(d, e, s, labels):
    known = (labels != IGNORED)[:, None]
    at = torch.where(known, labels[:, None], 0)
    logprob = torch.where(known, torch.where(s == 0, -math.inf, d.gather(1, at) - torch.log(s)), 0.0)
    entropy = torch.where(s == 0, 0.0, torch.log(s) - torch.where(e > 0, e * d, 0.0 * s).sum(-1, keepdim=True) / s)
    return logprob[:, 0], entropy[:, 0], known, at


def _readout(x, labels, top, temperature):
    d, e, s, m = _softmax(x, temperature)
    logprob, entropy, _, _ = _label_and_entropy(d, e, s, labels)
    # one whole number per score that orders by value, then by lowest index
    bits = (x.float() + 0.0).view(torch.int32)
    key = ((bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32) + (0x7FFFFFFF - torch.arange(x.shape[1], device=x.device))
    best = torch.topk(key, top, dim=1, sorted=True).values
    index = 0x7FFFFFFF - (best & 0x7FFFFFFF)
    value = d.gather(1, index)
    return {"logprob": logprob, "entropy": entropy, "top_logprob": torch.where(s == 0, -math.inf, value - torch.log(s)),
            "top_index": torch.where((value > -math.inf) & (s > 0), index, -1)}


def _readout_grad(x, labels, wants, up_logprob, up_entropy, temperature):
    d, e, s, m = _softmax(x, temperature)
    logprob, entropy, known, at = _label_and_entropy(d, e, s, labels)
    p = torch.where(s == 0, 0.0, e / s)
    grad = torch.zeros_like(p)
    outs = []
    if wants != "entropy":
        g = torch.where(known, up_logprob[:, None], 0.0)
        grad = -g * p
        grad.scatter_add_(1, at, torch.where(s == 0, 0.0, g) + torch.zeros_like(g))
        outs.append(logprob)
    if wants != "logprob":
        grad = grad - up_entropy[:, None] * torch.where(p > 0, p * (d - torch.log(s) + entropy[:, None]), 0.0 * s)
        outs.append(entropy)
    return {"outs": outs, "grad": (grad / temperature).to(x.dtype)}


def _distill(x, index, value, temperature, tail, up):
    rows, classes = x.shape
    d, e, s, m = _softmax(x, temperature)
    inside = index >= 0
    some = inside.any(1)
    at = torch.where(inside, index, classes)  # (one more column takes what is not in the list)
    if tail:
        log_q = torch.where(inside, value.double(), -math.inf)
        q = torch.exp(log_q)
        rest = (1 - q.sum(1)).clamp(min=0)
    else:
        log_q = torch.where(inside, value.double() / temperature, -math.inf)
        log_q = torch.where(some[:, None], log_q - torch.logsumexp(torch.where(some[:, None], log_q, 0.0), 1, keepdim=True), -math.inf)
        q = torch.exp(log_q)
    log_p = d.gather(1, torch.where(inside, index, 0)) - torch.log(s)
    loss = torch.where(q > 0, q * (log_q - log_p), 0.0).sum(1)
    p = e / s
    q_all = q.sum(1)
    pull = torch.zeros(rows, classes + 1, device=x.device).scatter_add_(1, at, q.float())[:, :classes]
    if tail:
        listed_ = torch.zeros(rows, classes + 1, dtype=torch.bool, device=x.device).scatter_(1, at, True)[:, :classes]
        p_rest = torch.where(listed_, 0.0, e).sum(1) / s[:, 0]
        counts = some & (rest > 0) & (p_rest > 0)
        loss = loss + torch.where(counts, rest * (torch.log(rest) - torch.log(p_rest)), 0.0)
        rest = torch.where(counts, rest, 0.0)
        every = (q_all + rest).float()
        factor = torch.where(listed_, every[:, None], (every - torch.where(counts, rest / p_rest, 0.0).float())[:, None])
    else:
        factor = q_all.float()[:, None]
    out = {"loss": torch.where(some, loss, 0.0).float()}
    if up is not None:
        grad = torch.where(some[:, None], p * factor - pull, 0.0) * (up / temperature)[:, None]
        out["grad"] = grad.to(x.dtype)
    return out


# ---- 64 bits, from the definitions ----------------------------------------------------------------------------------------------
def _parts(rows, classes):
    size = max(1, (1 << 26) // classes)
    return [slice(a, min(rows, a + size)) for a in range(0, rows, size)]


def _join(parts):
    if isinstance(parts[0], dict):
        return {k: _join([p[k] for p in parts]) for k in parts[0]}
    if isinstance(parts[0], list):
        return [_join([p[i] for p in parts]) for i in range(len(parts[0]))]
    return torch.cat(parts)


def exact(case, seed):
    state = prepare(case, seed)
    make = {"readout": _exact_readout, "readout_grad": _exact_readout}.get(case["op"], _exact_distill)
    return _join([make(case, state, part) for part in _parts(case["rows"], case["classes"])])


def _log_probabilities(z):
    """log softmax of rows in 64 bits; minus infinity throughout where nothing is finite."""
    log_p = z - torch.logsumexp(z, 1, keepdim=True)
    return torch.where((z == -math.inf).all(1, keepdim=True), -math.inf, log_p)


def _exact_readout(case, state, part):
    z = state["x"][part].double() / case["temperature"]
    labels = state["labels"][part]
    log_p = _log_probabilities(z)
    p = torch.exp(log_p)
    surprise = torch.where(p > 0, -log_p, 0.0)
    entropy = (p * surprise).sum(1)
    rows = torch.arange(len(labels), device=z.device)
    given = labels != IGNORED
    logprob = torch.zeros_like(entropy)
    logprob[given] = log_p[rows[given], labels[given]]
    if case["op"] == "readout":
        order = torch.sort(state["x"][part].double(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
        best = log_p.gather(1, order)
        return {"logprob": logprob, "entropy": entropy, "top_logprob": best, "top_index": torch.where(best > -math.inf, order, -1)}
    grad, outs = torch.zeros_like(p), []
    alive = p.sum(1) > 0
    if case["wants"] != "entropy":
        g = state["up_logprob"][part].double() * given * alive
        grad -= g[:, None] * p
        grad[rows[given], labels[given]] += g[given]
        outs.append(logprob)
    if case["wants"] != "logprob":
        grad += state["up_entropy"][part].double()[:, None] * p * (surprise - entropy[:, None])
        outs.append(entropy)
    return {"outs": outs, "grad": grad / case["temperature"]}


def _exact_distill(case, state, part):
    z = state["x"][part].double() / case["temperature"]
    index, value = state["index"][part], state["value"][part].double()
    rows, classes = z.shape
    log_p = _log_probabilities(z)
    row, col = torch.nonzero(index >= 0, as_tuple=True)
    target = torch.full((rows, classes), -math.inf, dtype=torch.float64, device=z.device)
    target[row, index[row, col]] = value[row, col] if case["tail"] else value[row, col] / case["temperature"]
    some = (target > -math.inf).any(1)
    if not case["tail"]:
        target = torch.where(some[:, None], _log_probabilities(target), -math.inf)
    q = torch.exp(target)
    loss = torch.where(q > 0, q * (target - log_p), 0.0).sum(1)
    p = torch.exp(log_p)
    grad = p * q.sum(1, keepdim=True) - q
    if case["tail"]:
        outside = target == -math.inf
        q_rest = (1 - q.sum(1)).clamp(min=0)
        p_rest = torch.where(outside, p, 0.0).sum(1)
        use = (q_rest > 0) & (p_rest > 0)
        loss = loss + torch.where(use, q_rest * torch.log(q_rest / p_rest), 0.0)
        grad = grad + torch.where(use, q_rest, 0.0)[:, None] * (p - torch.where(outside, p, 0.0) / torch.where(use, p_rest, 1.0)[:, None])
    out = {"loss": torch.where(some, loss, 0.0)}
    if case["op"] == "distill_grad":
        out["grad"] = torch.where(some[:, None], grad, 0.0) * (state["up"][part].double() / case["temperature"])[:, None]
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def work(case):
    rows, classes, k = case["rows"], case["classes"], case["top"]
    scores = rows * classes * SIZE[case["dtype"]]
    if case["op"] == "readout":
        return {"bytes": scores + rows * (8 + 4 + 4) + rows * k * (4 + 8), "flops": 5 * rows * classes}
    if case["op"] == "readout_grad":
        outs = 2 if case["wants"] == "both" else 1
        return {"bytes": 2 * scores + rows * 8 * outs + (rows * 8 if case["wants"] != "entropy" else 0), "flops": 9 * rows * classes}
    lists = rows * k * (8 + 4) + rows * 4
    if case["op"] == "distill":
        return {"bytes": scores + lists, "flops": 4 * rows * classes}
    return {"bytes": 2 * scores + lists + rows * 4, "flops": 7 * rows * classes}
