"""64-bit restatement of the score operators (log probabilities of labels, entropy, best alternatives; distillation from a teacher's top
list), row by row from the definitions, and the error bounds its tests use.

Bounds.  u = 2^-24 is half a step of float32.  A kernel computes a_j = (x_j - m) c with c = log2(e) / T: three roundings (difference,
constant, product), so a_j is off by 4u |a_j| and e_j = 2^a_j (one step, 2u) by (4 ln2 |a_j| + 2) u relative.  Every term of s is
positive: s is off by the e-weighted mean of that, and by u per addition on a term's way.  A thread adds at most `depth` terms
(rows beyond 4096 classes are dealt to 256 threads or more, shorter ones to 64) and some 20 partial sums are joined."""
import math

import torch

U = 2.0 ** -24


def depth(classes):
    return math.ceil(classes / 256) if classes > 4096 else math.ceil(classes / 64)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def log_softmax64(x, temperature):
    """x (rows, V) -> log probabilities in 64 bits, -inf throughout for a row of -inf, NaN throughout for a row with NaN or +inf."""
    z = x.double() / temperature
    m = z.amax(1, keepdim=True)
    d = z - torch.where(m == -math.inf, torch.zeros_like(m), m)
    s = torch.exp(d).sum(1, keepdim=True)
    lp = torch.where(s == 0, torch.full_like(d, -math.inf), d - torch.log(s))
    return torch.where(torch.isnan(s), torch.full_like(d, math.nan), lp)


def readout(x, labels=None, top=0, temperature=1.0, ignore_index=-100):
    """dict of 64-bit results of label_logprobs for x (rows, V)."""
    lp = log_softmax64(x, temperature)
    p = torch.exp(lp)
    rows, classes = x.shape
    bad = torch.isnan(lp).any(1)
    out = {"entropy": torch.where(bad, math.nan, -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)),
           "lse": torch.where(bad, math.nan, torch.logsumexp(x.double() / temperature, 1)), "lp": lp, "p": p}
    if labels is not None:
        want = []
        for r in range(rows):
            y = int(labels[r])
            want.append(0.0 if y == ignore_index else math.nan if not 0 <= y < classes else float(lp[r, y]))
        out["logprob"] = torch.tensor(want, dtype=torch.float64)
    if top:
        order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :top]
        best = lp.gather(1, order)
        out["top_index"] = torch.where((best > -math.inf) & ~bad[:, None], order, torch.full_like(order, -1))
        out["top_logprob"] = best
    return out


def readout_grad(x, labels, top, temperature, g_logprob=None, g_entropy=None, g_lse=None, g_top=None, ignore_index=-100):
    """(gradient, bound of a 32-bit one before its rounding to the scores' type) in 64 bits."""
    o = readout(x, labels, top, temperature, ignore_index)
    lp, p = o["lp"], o["p"]
    rows, classes = x.shape
    safe = torch.where(p > 0, lp, torch.zeros_like(lp))
    spread = torch.where(p > 0, (x.double() - x.double().amax(1, keepdim=True)).abs() / temperature, torch.zeros_like(p))
    grad, bound = torch.zeros_like(p), torch.zeros_like(p)
    rel = U * (depth(classes) + 40 + 8 * spread)

    def add(rows_, cols, value):
        grad[rows_, cols] += value
        bound[rows_, cols] += 4 * U * abs(value)

    all_ = torch.zeros(rows, dtype=torch.float64)
    for r in range(rows):
        dead = bool((lp[r] == -math.inf).all())
        if g_logprob is not None:
            y = int(labels[r])
            if y != ignore_index:
                all_[r] -= float(g_logprob[r])
                if not dead:
                    add(r, y, float(g_logprob[r]))
        if g_lse is not None:
            all_[r] += float(g_lse[r])
        if g_top is not None:
            for k in range(top):
                j = int(o["top_index"][r, k])
                if j >= 0:
                    all_[r] -= float(g_top[r, k])
                    add(r, j, float(g_top[r, k]))
    grad += all_[:, None] * p
    # (the 70 upstream gradients that `all_` may add up are rounded too)
    up = (g_top.abs().double().sum(1) if g_top is not None else 0) + all_.abs() + (g_logprob.abs().double() if g_logprob is not None else 0)
    bound += (all_.abs()[:, None] * rel + 70 * U * up[:, None]) * p
    if g_entropy is not None:
        h = o["entropy"][:, None]
        grad -= g_entropy.double()[:, None] * p * (safe + h)
        bound += g_entropy.double().abs()[:, None] * p * (safe.abs() + h + spread + 1) * 2 * rel
    return grad / temperature, bound / temperature + 4 * U * grad.abs() / temperature


def distill(x, index, value, temperature=1.0, tail=False):
    """(loss, gradient for an upstream 1, bound of the loss, bound of the gradient), 64 bits, row by row."""
    lp = log_softmax64(x, temperature)
    rows, classes = x.shape
    loss, grad = torch.zeros(rows, dtype=torch.float64), torch.zeros_like(lp)
    e_loss, e_grad = torch.zeros(rows, dtype=torch.float64), torch.zeros_like(lp)
    for r in range(rows):
        entries = [(int(i), float(v)) for i, v in zip(index[r], value[r].double()) if 0 <= int(i) < classes]
        if not entries:
            continue
        scale = 1.0 if tail else temperature
        if tail:
            q = [math.exp(v) for _, v in entries]
        else:
            vm = max(v for _, v in entries)
            norm = sum(math.exp((v - vm) / scale) for _, v in entries)
            q = [math.exp((v - vm) / scale) / norm for _, v in entries]
        p = torch.exp(lp[r])
        spread = torch.where(p > 0, (x[r].double() - x[r].double().max()).abs() / temperature, torch.zeros_like(p))
        rel = U * (depth(classes) + len(entries) + 60)
        by, size = {}, {}  # a class listed more than once is one class with the sum of its probabilities
        for (i, v), qk in zip(entries, q):
            by[i] = by.get(i, 0.0) + qk
            size[i] = max(size.get(i, 0.0), abs(v) if qk > 0 else 0.0)
        for i, qk in by.items():
            if qk > 0:
                log_q = math.log(qk)
                far = abs(log_q) + abs(float(lp[r, i])) + size[i] / scale + float(spread[i])
                loss[r] += qk * (log_q - float(lp[r, i]))
                # (q itself is off by (8 |v| + len) u, its logarithm by that much, the student's by rel + 8 u spread)
                e_loss[r] += qk * (rel * (1 + far) + 8 * U * far * (1 + far))
        every = sum(q)
        e_every = every * U * (len(entries) + 16 + 8 * max(abs(v) for _, v in entries) / scale)
        inside = outside = every
        e_out = e_every
        if tail:
            listed = torch.zeros(classes, dtype=torch.bool)
            listed[list(by)] = True
            q_rest = max(0.0, 1 - every)
            p_rest = float(p[~listed].sum())
            if q_rest > 0 and p_rest > 0:
                loss[r] += q_rest * (math.log(q_rest) - math.log(p_rest))
                inside = every + q_rest
                outside = inside - q_rest / p_rest
                # 1 - sum q loses what sum q is off by, and the logarithm of the small rest grows with it
                e_rest = e_every + 2 * U
                e_loss[r] += e_rest * (abs(math.log(q_rest)) + abs(math.log(p_rest)) + 1) + q_rest * 2 * rel * (2 + abs(math.log(p_rest)))
                e_out = e_every + (e_rest + q_rest * 3 * rel) / p_rest + 4 * U * (inside + q_rest / p_rest)
            else:
                e_out = e_every + 2 * U
        listed = torch.zeros(classes, dtype=torch.bool)
        listed[list(by)] = True
        factor = torch.where(listed, torch.tensor(inside, dtype=torch.float64), torch.tensor(outside, dtype=torch.float64))
        grad[r] = p * factor
        e_grad[r] = p * (factor.abs() * (rel + 8 * U * spread) + torch.where(listed, e_every + 4 * U, e_out))
        for i, qk in by.items():
            grad[r, i] -= qk
            e_grad[r, i] += qk * U * (len(entries) + 16) + 8 * U * qk * max(abs(v) for _, v in entries) / scale
        grad[r] /= temperature
        e_grad[r] = e_grad[r] / temperature + 4 * U * grad[r].abs()
    return loss, grad, e_loss + 4 * U * loss.abs(), e_grad
