"""Cases of the operators at the vocabulary end of the language model.

  score    log probability of given tokens, entropy and the top alternatives of each logits row
  distill  loss against a teacher's top logits (optionally mixed with hard labels) and its gradient
  embed    embedding lookup with scaling, and the table's gradient

``own`` chooses between the plain torch form (32 bits, rounded once at the end) and the package's operators.
"""

import functools
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba3-siso-tpu_b200")
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}
_MOST = 4096 * 128256  # logits of the largest listed case


@functools.lru_cache(None)
def _ops():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from mamba3_b200 import distill, embedding, scoring

    return scoring, distill, embedding


def listed():
    return [
        # one sequence being generated, with the alternatives of a completion API
        _score("score-token", 1, 1, 128256, "bf16", 20, 1.0),
        # one decode step of the 256-sequence decode batch, scored at the sampling temperature
        _score("score-batch", 1, 256, 128256, "bf16", 5, 0.7),
        # perplexity of prompts: logits[:, :-1] against tokens[:, 1:], fp32 logits, a head padded to 50304 columns
        _score("score-prompt", 4, 1023, 50257, "f32", 0, 1.0, pad=47, shift=True),
        # the teacher's pass over a batch of byte-level sequences
        _score("score-bytes", 16, 8192, 256, "bf16", 8, 1.0),
        # the teacher's pass over a batch of text at the large vocabulary
        _score("score-teacher", 2, 2048, 128256, "bf16", 32, 2.0),
        # distillation of a toy model: launch latency
        _distill("distill-small", 64, 512, "bf16", 8, 1.0, 0.0, "step", False),
        # a byte-level student's step, padding weighted out
        _distill("distill-bytes", 131072, 256, "bf16", 16, 1.0, 0.0, "step", True),
        # a student's step at the large vocabulary
        _distill("distill-large", 4096, 128256, "bf16", 64, 2.0, 0.0, "step", False),
        # the same through autograd: fp32 logits, an odd vocabulary, hard labels mixed in
        _distill("distill-hard", 4095, 50257, "f32", 32, 2.0, 0.3, "autograd", True),
        # the lookup of one decode step
        _embed("embed-token", 1, 256, 128256, 2048, "bf16", "bf16", 1.0, False),
        # byte-level training: every id occurs hundreds of times
        _embed("embed-bytes", 16, 8192, 256, 512, "f32", "bf16", 1.0, True),
        # training at the large vocabulary, rows scaled by sqrt(d)
        _embed("embed-large", 8, 2048, 128256, 2048, "f32", "bf16", 2048 ** 0.5, True),
    ]


def _named(name, case):
    return case if name is None else dict(case, name=name)


def _score(name, batch, length, vocab, dtype, top, temperature, pad=0, shift=False):
    return _named(name, {"op": "score", "batch": batch, "length": length, "vocab": vocab, "dtype": dtype, "top": top,
                         "temperature": temperature, "pad": pad, "shift": shift})


def _distill(name, rows, vocab, dtype, k, temperature, hard, kind, weighted):
    return _named(name, {"op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k,
                         "temperature": temperature, "hard": hard, "kind": kind, "weighted": weighted})


def _embed(name, batch, length, vocab, dim, table, out, scale, train):
    return _named(name, {"op": "embed", "batch": batch, "length": length, "vocab": vocab, "dim": dim, "table": table,
                         "out": out, "scale": scale, "train": train})


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("score", "distill", "embed"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    vocab = rng.choice((256, 512, 50000, 50257, 128256, _log_int(rng, 256, 128256), _log_int(rng, 256, 128256)))
    rows = _log_int(rng, 1, 131072)
    if op == "embed":
        dim = rng.choice((64, 512, 1024, 2048, 8 * _log_int(rng, 8, 256), _log_int(rng, 64, 2048)))
        n = max(1, min(rows, 16384 * 2048 // dim))
        batch = rng.choice((1, 2, 8))
        return _embed(None, batch, max(1, n // batch), vocab, dim, rng.choice(("f32", "bf16")), dtype,
                      rng.choice((1.0, dim ** 0.5)), rng.random() < 0.7)
    rows = max(1, min(rows, _MOST * 2 // _SIZE[dtype] // vocab))
    temperature = rng.choice((1.0, 1.0, 2.0, round(rng.uniform(0.5, 3.0), 2)))
    if op == "distill":
        kind = rng.choice(("step", "step", "autograd", "loss"))
        return _distill(None, rows, vocab, dtype, rng.choice((1, 8, 16, 32, 64, rng.randint(1, 128))), temperature,
                        rng.choice((0.0, 0.0, 0.3)), kind, rng.random() < 0.5)
    top = min(rng.choice((0, 1, 5, 8, 20, 32, rng.randint(1, 128))), vocab)
    batch = rng.choice((1, 2, 4))
    return _score(None, batch, max(1, rows // batch), vocab, dtype, top, temperature, rng.choice((0, 0, 7, 48)),
                  rng.random() < 0.3)


# ---------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"score": _prepare_score, "distill": _prepare_distill, "embed": _prepare_embed}[case["op"]](case, g)


def _randint(g, hi, shape):
    return torch.randint(0, hi, shape, generator=g, device="cuda")


def _uniform(g, shape):
    return torch.rand(shape, generator=g, device="cuda")


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=_DT[dtype])


def _prepare_score(c, g):
    b, n, v = c["batch"], c["length"] + int(c["shift"]), c["vocab"]
    buf = _normal(g, (b, n, v + c["pad"]), c["dtype"]).mul_(2.5)
    buf[..., _randint(g, v, (max(1, v // 100),))] = -math.inf  # suppressed ids
    tokens = _randint(g, v, (b, n))
    tokens[_uniform(g, (b, n)) < 0.05] = -100  # padding
    logits, targets = buf[..., :v], tokens
    if c["shift"]:
        logits, targets = logits[:, :-1], tokens[:, 1:]
    return {"case": c, "logits": logits, "targets": targets}


def _prepare_distill(c, g):
    r, v, k = c["rows"], c["vocab"], c["k"]
    logits = _normal(g, (r, v), c["dtype"]).mul_(2.0)
    step = max(1, v // k)
    ids = (_randint(g, v, (r, 1)) + torch.arange(k, device="cuda") * (1 + _randint(g, step, (r, 1)))) % v
    teacher = 6.0 - torch.cumsum(-torch.log(_uniform(g, (r, k)).clamp_min(1e-6)), 1) * 0.5
    logits.scatter_add_(1, ids, (teacher + _normal(g, (r, k), "f32")).to(logits.dtype))  # the student half knows
    if k > 1:
        ids[:, k // 2 + 1:][_uniform(g, (r, k - k // 2 - 1)) < 0.1] = -1  # shorter lists
    s = {"case": c, "logits": logits, "ids": ids, "teacher": teacher, "labels": None, "weights": None}
    if c["hard"] > 0:
        s["labels"] = torch.where(_uniform(g, (r,)) < 0.05, -100, ids[:, 0])
    if c["weighted"]:
        s["weights"] = (_uniform(g, (r,)) < 0.9).float()
        s["weights"][0] = 1.0
    return s


def _prepare_embed(c, g):
    n, v, d = c["batch"] * c["length"], c["vocab"], c["dim"]
    table = _normal(g, (v, d), c["table"]).mul_(0.02)
    rank = torch.exp(_uniform(g, (n,)) * math.log(v)).long().clamp_(max=v) - 1  # frequency ~ 1 / rank
    tokens = (rank * 7919 % v).view(c["batch"], c["length"])
    tokens[_uniform(g, tokens.shape) < 0.02] = -1  # padding
    s = {"case": c, "table": table, "tokens": tokens}
    if c["train"]:
        s["dy"] = _normal(g, (c["batch"], c["length"], d), c["out"]).mul_(1e-2)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    c = state["case"]
    if not own:
        return {"score": _plain_score, "distill": _plain_distill, "embed": _plain_embed}[c["op"]](c, state)
    scoring, distill, embedding = _ops()
    if c["op"] == "score":
        r = scoring.token_logprobs(state["logits"], state["targets"], top=c["top"], temperature=c["temperature"])
        out = {"logprob": r.logprob, "entropy": r.entropy, "lse": r.lse}
        if c["top"]:
            out["top_logprob"], out["top_ids"] = r.top_logprob, r.top_ids
        return out
    if c["op"] == "distill":
        args = dict(temperature=c["temperature"], labels=state["labels"], hard_weight=c["hard"],
                    weights=state["weights"])
        x, ids, teacher = state["logits"], state["ids"], state["teacher"]
        if c["kind"] == "loss":
            with torch.no_grad():
                return {"rows": distill.distill_loss(x, ids, teacher, reduction="none", **args)}
        if c["kind"] == "step":
            loss, grad = distill.distill_loss_and_grad(x, ids, teacher, **args)
        else:
            x = x.detach().requires_grad_(True)
            loss = distill.distill_loss(x, ids, teacher, **args)
            grad, = torch.autograd.grad(loss, x)
            loss = loss.detach()
        return {"loss": loss, "grad": grad}
    out = {"out": embedding.embed_tokens(state["table"], state["tokens"], scale=c["scale"], dtype=_DT[c["out"]])}
    if c["train"]:
        out["grad"] = embedding.embedding_grad(state["dy"], state["tokens"], c["vocab"], scale=c["scale"],
                                               dtype=_DT[c["table"]])
    return out


def _plain_score(c, s):
    x = s["logits"].float() + 0.0  # -0 and +0 are equal logits
    y = x / c["temperature"]
    lse = _lse(y)
    t = s["targets"]
    logprob = torch.where(t < 0, 0.0, y.gather(-1, t.clamp_min(0)[..., None])[..., 0] - lse)
    lp = y - lse[..., None]
    p = torch.exp(lp)
    out = {"logprob": logprob, "entropy": -torch.where(p > 0, p * lp, 0.0).sum(-1), "lse": lse}
    if c["top"]:
        bits = x.view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()  # ascends with x
        key = order * 2**32 + torch.arange(c["vocab"] - 1, -1, -1, device=x.device)  # ties: the lower index
        ids = torch.topk(key, c["top"], dim=-1).indices
        out["top_logprob"], out["top_ids"] = lp.gather(-1, ids), ids
    return out


def _lse(y):
    m = y.amax(-1, keepdim=True)
    return m[..., 0] + torch.log(torch.exp(y - m).sum(-1))


def _plain_distill(c, s):
    T, h, x = c["temperature"], c["hard"], s["logits"].float()
    w = s["weights"] if s["weights"] is not None else torch.ones(c["rows"], device=x.device)
    there = s["ids"] >= 0
    ids = s["ids"].clamp_min(0)
    t = torch.where(there, s["teacher"].float() / T, -math.inf)
    p = torch.exp(t - _lse(t)[:, None])
    y = x / T
    lse = _lse(y)
    terms = p * (torch.log(p) - (y.gather(1, ids) - lse[:, None]))
    rows = (1 - h) * T * T * torch.where(p > 0, terms, 0.0).sum(1)
    if h > 0:
        label, hard_there = s["labels"].clamp_min(0)[:, None], s["labels"] >= 0
        lse1 = _lse(x)
        rows = rows + h * torch.where(hard_there, lse1 - x.gather(1, label)[:, 0], 0.0)
    rows = rows * w
    if c["kind"] == "loss":
        return {"rows": rows}
    total = w.sum()
    grad = (1 - h) * T * torch.exp(y - lse[:, None]).scatter_add_(1, ids, -p)
    if h > 0:
        hard = torch.exp(x - lse1[:, None]).scatter_add_(1, label, -torch.ones_like(label, dtype=torch.float32))
        grad = grad + h * hard * hard_there[:, None]
    return {"loss": rows.sum() / total, "grad": (grad * (w / total)[:, None]).to(s["logits"].dtype)}


def _plain_embed(c, s):
    tokens = s["tokens"].reshape(-1)
    there = (tokens >= 0)[:, None]
    ids = tokens.clamp_min(0)
    rows = torch.where(there, s["table"][ids].float() * c["scale"], 0.0)
    out = {"out": rows.to(_DT[c["out"]]).view(*s["tokens"].shape, -1)}
    if c["train"]:
        dy = torch.where(there, s["dy"].reshape(-1, c["dim"]).float() * c["scale"], 0.0)
        grad = torch.zeros(c["vocab"], c["dim"], device=dy.device).index_add_(0, ids, dy)
        out["grad"] = grad.to(s["table"].dtype)
    return out


# ---------------------------------------------------------------------------------------------- definitions

def work(case):
    c = case
    if c["op"] == "score":
        rows = c["batch"] * c["length"]
        n = rows * c["vocab"]
        return {"bytes": n * _SIZE[c["dtype"]] + rows * (8 + 12 + 12 * c["top"]), "flops": 6 * n}
    if c["op"] == "distill":
        n = c["rows"] * c["vocab"]
        passes = 1 if c["kind"] == "loss" else 2
        side = c["rows"] * (12 * c["k"] + 8 * (c["hard"] > 0) + 4 * c["weighted"] + 4)
        return {"bytes": passes * n * _SIZE[c["dtype"]] + side, "flops": (4 if passes == 1 else 7) * n}
    n = c["batch"] * c["length"]
    seen = min(n, c["vocab"])
    size = 8 * n + c["dim"] * (seen * _SIZE[c["table"]] + n * _SIZE[c["out"]])
    if c["train"]:
        size += c["dim"] * (n * _SIZE[c["out"]] + c["vocab"] * _SIZE[c["table"]])
    return {"bytes": size, "flops": n * c["dim"] * (3 if c["train"] else 1)}


def exact(case, seed):
    """The outputs in 64 bits, from the definitions, a block of rows at a time."""
    s, c = prepare(case, seed), case
    if c["op"] == "embed":
        keep = s["tokens"] >= 0
        out = torch.zeros(*s["tokens"].shape, c["dim"], dtype=torch.float64, device="cuda")
        out[keep] = s["table"][s["tokens"][keep]].double() * c["scale"]
        if not c["train"]:
            return {"out": out}
        grad = torch.zeros(c["vocab"], c["dim"], dtype=torch.float64, device="cuda")
        grad.index_put_((s["tokens"][keep],), s["dy"][keep].double(), accumulate=True)
        return {"out": out, "grad": grad * c["scale"]}
    rows = c["batch"] * c["length"] if c["op"] == "score" else c["rows"]
    block = max(1, (1 << 26) // c["vocab"])
    parts = []
    for lo in range(0, rows, block):
        r = torch.arange(lo, min(rows, lo + block), device="cuda")
        parts.append(_exact_score(c, s, r) if c["op"] == "score" else _exact_distill(c, s, r))
    got = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    if c["op"] == "score":
        shape = (c["batch"], c["length"])
        got = {name: v.reshape(*shape, *v.shape[1:]) for name, v in got.items()}
        return dict(got, top_ids=None) if c["top"] else got
    if c["kind"] == "loss":
        return got
    total = rows if s["weights"] is None else float(s["weights"].double().sum())
    return {"loss": got["rows"].sum() / total, "grad": got["grad"] / total}


def _exact_score(c, s, r):
    x = s["logits"][r // c["length"], r % c["length"]].double() / c["temperature"]
    t = s["targets"][r // c["length"], r % c["length"]]
    logp = torch.log_softmax(x, 1)
    picked = logp[torch.arange(len(r), device="cuda"), t.clamp_min(0)]
    got = {"logprob": torch.where(t >= 0, picked, 0.0),
           "entropy": torch.special.entr(torch.softmax(x, 1)).sum(1), "lse": torch.logsumexp(x, 1)}
    if c["top"]:
        got["top_logprob"] = torch.topk(logp, c["top"], 1).values  # the values do not depend on the order of ties
    return got


def _exact_distill(c, s, r):
    T, h = c["temperature"], c["hard"]
    x, ids = s["logits"][r].double(), s["ids"][r]
    w = torch.ones(len(r), dtype=torch.float64, device="cuda") if s["weights"] is None else s["weights"][r].double()
    dense = torch.zeros_like(x)  # the teacher's distribution over the whole vocabulary
    e = torch.exp((s["teacher"][r].double() - 6.0) / T) * (ids >= 0)
    dense.scatter_add_(1, ids.clamp_min(0), e / e.sum(1, keepdim=True))
    given = e / e.sum(1, keepdim=True)
    q = torch.log_softmax(x / T, 1)
    cross = -(dense * q).sum(1)
    rows = (1 - h) * T ** 2 * (cross - torch.special.entr(given).sum(1))
    grad = (1 - h) * T * (torch.exp(q) - dense)
    if h > 0:
        label = s["labels"][r]
        hit = torch.nn.functional.one_hot(label.clamp_min(0), c["vocab"]).double()
        logq = torch.log_softmax(x, 1)
        there = (label >= 0).double()
        rows = rows - h * there * (hit * logq).sum(1)
        grad = grad + h * there[:, None] * (torch.exp(logq) - hit)
    got = {"rows": rows * w}
    if c["kind"] != "loss":
        got["grad"] = grad * w[:, None]
    return got
