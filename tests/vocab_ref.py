"""Plain 64-bit implementations (CPU) of the vocabulary-end operators, written from their
formulas: token log probabilities, distillation from top logits, embedding lookup and its
gradient."""

import math

import torch


def score(logits, targets, top, temperature):
    """Row by row over ``logits (R, V)``: dict of logprob, entropy, lse, top_logprob, top_ids."""
    out = {k: [] for k in ("logprob", "entropy", "lse", "top_logprob", "top_ids")}
    for r in range(logits.shape[0]):
        x = logits[r].double().cpu()
        y = x / temperature
        m = y.max() if not torch.isnan(y).any() else torch.tensor(math.nan, dtype=torch.float64)
        ok = bool(torch.isfinite(m))
        # against the maximum: at 1e38 the logarithm of the sum is lost in y - lse even in 64 bits
        ln_z = torch.log(torch.exp(y - m).sum()) if ok else torch.tensor(math.nan, dtype=torch.float64)
        lse = m + ln_z
        lp = y - m - ln_z
        p = torch.exp(lp)
        out["lse"].append(lse)
        out["entropy"].append(-(p * lp)[p > 0].sum() if ok else lse)
        t = None if targets is None else int(targets[r])
        if t is not None:
            out["logprob"].append(torch.tensor(0.0).double() if t < 0 else
                                  lp[t] if t < x.numel() else torch.tensor(math.nan).double())
        # descending, NaN first, the lower index first among equals
        xs = [math.inf if math.isnan(v) else v for v in x.tolist()]
        nan = torch.isnan(x).tolist()
        order = sorted(range(len(xs)), key=lambda i: (not nan[i], -xs[i], i))[:top]
        out["top_ids"].append(torch.tensor(order, dtype=torch.int64))
        out["top_logprob"].append(lp[order])
    return {k: torch.stack(v) if v else None for k, v in out.items()}


def distill_rows(x, ids, teacher, labels, weights, temperature, hard_weight):
    """The rows' losses for f64 ``x (R, V)``, differentiable in it."""
    losses = []
    for r in range(x.shape[0]):
        w = 1.0 if weights is None else float(weights[r])
        there = [j for j in range(ids.shape[1]) if int(ids[r, j]) >= 0]
        label = -1 if labels is None else int(labels[r])
        soft, hard = bool(there) and hard_weight < 1, label >= 0 and hard_weight > 0
        loss = torch.zeros((), dtype=torch.float64)
        if w != 0 and (soft or hard):
            if soft:
                t = teacher[r, there].double() / temperature
                logp = torch.log_softmax(t, 0)
                logq = torch.log_softmax(x[r] / temperature, 0)[ids[r, there]]
                p = torch.exp(logp)
                keep = p > 0
                kl = (p[keep] * (logp[keep] - logq[keep])).sum()
                loss = loss + (1 - hard_weight) * temperature ** 2 * kl
            if hard:
                loss = loss - hard_weight * torch.log_softmax(x[r], 0)[label]
        losses.append(w * loss)
    return torch.stack(losses)


def reduce(rows, weights, reduction):
    if reduction == "none":
        return rows
    total = rows.sum()
    if reduction == "mean":
        total = total / (rows.shape[0] if weights is None else weights.double().sum())
    return total


def embed(table, tokens, scale):
    t = tokens.reshape(-1)
    out = torch.zeros(t.numel(), table.shape[1], dtype=torch.float64)
    for i, v in enumerate(t.tolist()):
        if v >= table.shape[0]:
            out[i] = math.nan
        elif v >= 0:
            out[i] = table[v].double() * scale
    return out.view(*tokens.shape, -1)


def embed_grad(dy, tokens, vocab, scale):
    t = tokens.reshape(-1)
    g = torch.zeros(vocab, dy.shape[-1], dtype=torch.float64)
    keep = (t >= 0) & (t < vocab)
    g.index_put_((t[keep],), dy.reshape(-1, dy.shape[-1])[keep].double(), accumulate=True)
    return g * scale
