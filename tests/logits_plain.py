"""The operators of ``lattice_based_tagger_amd.logits`` written plainly in 64
bits on the CPU, and how far a float32 kernel may be from them.

Error bounds, relative to a row's softmax sum S over V logits:

* a term exp((x - m) / T): the difference and its product with log2(e)/T round
  once each and that constant once, together 3 * 2^-24 of the exponent, whose
  mean under the softmax is at most ln V (<= 12.3 here) and whose value
  weighs little beyond; the exponential is off by an ulp, 2^-23;
* a thread adds at most V / 64 terms one after another (2^-24 of the sum
  each), then at most 64 partial sums are joined.

So S is off by at most ``delta(V) = (V / 64 + 64 + 3 * 12.3 + 2) * 2^-24``, a
logarithm of it by as much absolutely.
"""

import math

import torch

INF = math.inf
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def delta(vocab):
    return (vocab / 64 + 64 + 3 * 12.3 + 2) * 2.0 ** -24


def top_logits(x, k, temperature=1.0):
    x = x.double().cpu()
    order = torch.where(x.isnan(), torch.tensor(-INF, dtype=torch.float64), x)
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :k]
    lse = torch.logsumexp(x / temperature, -1)
    lse = torch.where((x == INF).any(-1), torch.tensor(INF, dtype=torch.float64), lse)   # (beside a NaN too)
    return x.gather(-1, ids), ids, lse


def lse_tolerance(lse, vocab):
    return delta(vocab) + lse.abs() * 2.0 ** -24


def distill(z, ids, top, lse, temperature, weight):
    """(loss, grad, tolerance of the loss, tolerance of the gradient) of rows
    [R, V], entry by entry."""
    z, top = z.double().cpu(), top.double().cpu()
    ids = ids.long().cpu()
    weight = weight.double().cpu()
    lse = None if lse is None else lse.double().cpu()
    rows, vocab = z.shape
    d = delta(vocab)
    loss = torch.zeros(rows, dtype=torch.float64)
    grad = torch.zeros_like(z)
    loss_tol = torch.zeros(rows, dtype=torch.float64)
    grad_tol = torch.zeros_like(z)
    for r in range(rows):
        at = ids[r]
        there = (at >= 0) & (at < vocab)
        at, t = at[there], top[r][there] / temperature
        y = z[r] / temperature
        logq = y - torch.logsumexp(y, -1)
        q = logq.exp()
        if lse is None:
            logp = t - torch.logsumexp(t, -1) if len(t) and t.max() > -INF else torch.full_like(t, -INF)
            rest = 0.0
        else:
            logp = t - lse[r]
            rest = max(0.0, 1.0 - float(logp.exp().sum()))
        p = logp.exp()
        inside = torch.zeros(vocab, dtype=torch.bool)
        inside[at] = True
        qrest = float(q[~inside].sum())
        if not qrest > 0:
            rest = 0.0
        use = p > 0
        total = float((p[use] * (logp[use] - logq[at][use])).sum())
        if rest > 0:
            total += rest * (math.log(rest) - math.log(qrest))
        whole = float(p.sum()) + rest
        other = rest / qrest if rest > 0 else 0.0
        g = torch.where(inside, whole * q, (whole - other) * q)
        mass = torch.zeros(vocab, dtype=torch.float64).index_add_(0, at, p)
        g = g - mass
        loss[r] = total
        grad[r] = g * weight[r] / temperature
        # two logarithms of sums enter; the loss is rounded once
        loss_tol[r] = 2 * d * whole + abs(total) * 2.0 ** -24 + 1e-12
        # q_v: its own exponent (3 * 2^-24 of it), the sum; p_v: a product or two
        a = (y.max() - y).clamp(max=200)
        dq = d + (3 * a + 4) * 2.0 ** -24
        grad_tol[r] = (weight[r].abs() / temperature) * (q * (whole + 2 * other) * 2 * dq + mass * 2.0 ** -22)
    return loss, grad, loss_tol, grad_tol


def type_tolerance(value, dtype):
    """Half a step of the type at a value, and at the foot of its range."""
    foot = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -125
    return value.abs() * HALF_STEP[dtype] * 1.001 + foot


def verify(target, ids, accept_u, sample_u, draft=None, lengths=None, temperature=1.0):
    target = target.double().cpu()
    draft = None if draft is None else draft.double().cpu()
    batch, places, vocab = target.shape
    tokens = torch.full((batch, places), -1, dtype=torch.int64)
    accepted = torch.zeros(batch, dtype=torch.int64)

    def soft(row):
        return torch.softmax(row / temperature, -1) if row.max() > -INF else torch.zeros_like(row)

    for b in range(batch):
        n = places - 1 if lengths is None else int(lengths[b])
        a, w = 0, None
        while a < n:
            x = int(ids[b, a])
            p = soft(target[b, a])
            q = None if draft is None else soft(draft[b, a])
            known = 0 <= x < vocab
            qx = (1.0 if q is None else float(q[x])) if known else 0.0
            if known and float(accept_u[b, a]) * qx < float(p[x]):
                tokens[b, a] = x
                a += 1
                continue
            if q is None:
                q = torch.zeros_like(p)
                if known:
                    q[x] = 1.0
            w = (p - q).clamp_min(0)
            if not float(w.sum()) > 0:
                w = p
            break
        if w is None:
            w = soft(target[b, a])
        accepted[b] = a
        cum = w.cumsum(0)
        hit = (cum > float(sample_u[b]) * float(cum[-1])) & (w > 0)
        if hit.any():
            tokens[b, a] = int(hit.int().argmax())
        elif (w > 0).any():
            tokens[b, a] = int((w > 0).nonzero()[-1])
    return tokens, accepted
