"""The operators on token ids, logits and pairs of answers that stand beside the trainer's own lookups and losses: what is
measured of them. `run` computes them from elementary torch operations, or, where `own` is true, with the calls of
mlease_amd.operators that a user's program makes.

  lookup      out[t] = scale * table[ids[t]]; an id outside the table gives a row of zeros
  gradient    its gradient, dtable[v] = scale * (sum of the rows of grad_out whose id is v), written whole
  loglik      logp[t] = logits[t, target[t]] - log sum_j exp(logits[t, j]) and, in a training step, the gradient
              dlogits[t, j] = g[t] ([j == target[t]] - softmax(logits[t])[j]); a target outside the row's classes: 0
  preference  paired log ratios: a sequence's ratio is the sum (or mean) over its tokens of logp - ref_logp, a pair's margin
              h = beta (ratio_chosen - ratio_rejected) + offset, its loss (1 - eps) log(1 + e^-h) + eps log(1 + e^h), and the
              gradient of the weighted sum of the losses in every logp
  step        a training step on pairs: loglik, preference on its logp, gradient in the logits
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IDS = {"i32": torch.int32, "i64": torch.int64}
_kept = {}


def _operators():
    """The framework's operators on this device, made once as a user's program makes them."""
    if "ops" not in _kept:
        from mlease_amd.operators import HipOperators
        _kept["ops"] = HipOperators(torch.cuda.current_device())
    return _kept["ops"]


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the next token of 8 sequences that are being answered
        {"name": "lookup 8", "op": "lookup", "n": 8, "rows": 32000, "width": 4096, "type": "bf16", "ids": "i64", "absent": 0},
        # a batch of prompts, packed
        {"name": "lookup 16384", "op": "lookup", "n": 16384, "rows": 128000, "width": 4096, "type": "bf16", "ids": "i64", "absent": 0},
        # the one-hot rows of one partition of the lambda sweep (9 765 rows of 20 features, 8 models side by side), some features unknown
        {"name": "lookup sweep", "op": "lookup", "n": 195300, "rows": 100001, "width": 8, "type": "f32", "ids": "i32", "absent": 977},
        # a short batch on a small table
        {"name": "gradient 300", "op": "gradient", "n": 300, "rows": 8192, "width": 512, "type": "f16", "ids": "i64", "absent": 0},
        # a training batch: the table's gradient, padding tokens absent
        {"name": "gradient 16384", "op": "gradient", "n": 16384, "rows": 64000, "width": 4096, "type": "bf16", "ids": "i64", "absent": 1000},
        # the gradient of the sweep's lookup
        {"name": "gradient sweep", "op": "gradient", "n": 195300, "rows": 100001, "width": 8, "type": "f32", "ids": "i32", "absent": 977},
        # scoring a few tokens against a large vocabulary
        {"name": "loglik 32", "op": "loglik", "n": 32, "classes": 128000, "pad": 0, "type": "bf16", "ids": "i64", "absent": 0, "train": False},
        # a training batch, 2 of 5 tokens belong to prompts and have no target
        {"name": "loglik 8192", "op": "loglik", "n": 8192, "classes": 32000, "pad": 0, "type": "bf16", "ids": "i64", "absent": 3276, "train": True},
        # an odd number of classes in 32 bits
        {"name": "loglik odd", "op": "loglik", "n": 777, "classes": 50021, "pad": 2, "type": "f32", "ids": "i32", "absent": 33, "train": True},
        # four pairs of short answers
        {"name": "preference 4", "op": "preference", "pairs": 4, "tokens": 500, "mean": False, "reference": True, "masked": False, "smoothing": 0.0},
        # a large batch of long answers, prompts masked, mean per token
        {"name": "preference 256", "op": "preference", "pairs": 256, "tokens": 1000003, "mean": True, "reference": True, "masked": True, "smoothing": 0.1},
        # a training step on 8 pairs, from the logits to their gradient
        {"name": "step 8", "op": "step", "pairs": 8, "tokens": 4096, "classes": 64000, "type": "bf16", "ids": "i64", "smoothing": 0.0},
    ]


def _log_uniform(rng, low, high):
    return min(high, int(low * math.exp(rng.random() * math.log((high + 1) / low))))


def draw(rng):
    op = rng.choice(("lookup", "gradient", "loglik", "preference", "step"))
    kind, ids = rng.choice(("f32", "bf16", "f16")), rng.choice(("i32", "i64"))
    if op in ("lookup", "gradient"):
        width = _log_uniform(rng, 1, 8192)
        rows = _log_uniform(rng, 2, min(200000, 200_000_000 // width))
        n = _log_uniform(rng, 1, min(300000, 60_000_000 // width))
        return {"op": op, "n": n, "rows": rows, "width": width, "type": kind, "ids": ids, "absent": n // rng.choice((3, 20, 10 ** 9))}
    if op == "loglik":
        classes = _log_uniform(rng, 2, 160000)
        n = _log_uniform(rng, 1, min(100000, 120_000_000 // classes))
        return {"op": op, "n": n, "classes": classes, "pad": rng.choice((0, 0, 1, 64)), "type": kind, "ids": ids, "absent": n // rng.choice((2, 10, 10 ** 9)),
                "train": rng.random() < 0.7}
    if op == "preference":
        pairs = _log_uniform(rng, 1, 1000)
        return {"op": op, "pairs": pairs, "tokens": _log_uniform(rng, pairs, 2_000_000), "mean": rng.random() < 0.5,
                "reference": rng.random() < 0.8, "masked": rng.random() < 0.5, "smoothing": rng.choice((0.0, 0.1))}
    classes = _log_uniform(rng, 100, 130000)
    pairs = _log_uniform(rng, 1, 64)
    return {"op": op, "pairs": pairs, "tokens": _log_uniform(rng, 2, 120_000_000 // classes), "classes": classes, "type": kind, "ids": ids,
            "smoothing": rng.choice((0.0, 0.1))}


def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


def _tokens(g, n, rows, absent, kind):
    """Ids as text has them: the k-th most frequent with a probability of about 1 / k, in a shuffled numbering; `absent` of them are -1."""
    d = _device()
    rank = (torch.rand(n, generator=g, device=d, dtype=torch.float64) * math.log(rows + 1)).exp_().sub_(1).long().clamp_(0, rows - 1)
    ids = torch.randperm(rows, generator=g, device=d)[rank]
    if absent:
        ids[torch.randperm(n, generator=g, device=d)[:absent]] = -1
    return ids.to(kind)


def _sequences(g, count, tokens):
    """Where each of `count` sequences begins in a packed list of `tokens`: lengths that differ up to tenfold, some of none where tokens are few."""
    d = _device()
    ends = (torch.rand(count, generator=g, device=d, dtype=torch.float64) * 0.9 + 0.1).cumsum(0)
    return torch.nn.functional.pad((ends / ends[-1] * tokens).round().long(), (1, 0))


def _logits(g, n, classes, pad, kind, targets):
    """Logits of a model that knows something: spread 2, the target's a few units higher. Rows of a padded matrix where `pad` says so."""
    d = _device()
    x = torch.empty(n, classes + pad, device=d, dtype=TYPES[kind])
    step = max(1, (1 << 26) // (classes + pad))
    for a in range(0, n, step):
        part = torch.randn(min(step, n - a), classes + pad, generator=g, device=d).mul_(2.0)
        t = targets[a:a + step].long().clamp(0, classes - 1)
        part[torch.arange(part.shape[0], device=d), t] += 6.0
        x[a:a + step] = part
    return x[:, :classes]


def prepare(case, seed):
    d = _device()
    g = torch.Generator(device=d)
    g.manual_seed(int(seed))
    op = case["op"]
    s = {"op": op, "case": dict(case)}
    if op in ("lookup", "gradient"):
        n, rows, width, kind = case["n"], case["rows"], case["width"], TYPES[case["type"]]
        s["ids"] = _tokens(g, n, rows, case["absent"], IDS[case["ids"]])
        s["scale"] = math.sqrt(width)
        if op == "lookup":
            s["table"] = torch.randn(rows, width, generator=g, device=d).mul_(0.02).to(kind)
        else:
            s["grad_out"] = torch.randn(n, width, generator=g, device=d).mul_(0.01).to(kind)
            s["rows"] = rows
        return s
    if op == "loglik":
        n, classes = case["n"], case["classes"]
        s["target"] = _tokens(g, n, classes, case["absent"], IDS[case["ids"]])
        s["logits"] = _logits(g, n, classes, case["pad"], case["type"], s["target"])
        # the gradient that comes back to each logp; in f16 the loss is scaled, as training in that type does
        s["g"] = torch.randn(n, generator=g, device=d).mul_((4096.0 if case["type"] == "f16" else 1.0) / n)
        s["train"] = case["train"]
        return s
    pairs = case["pairs"]
    s["beta"], s["smoothing"], s["scale"] = 0.1, case["smoothing"], (4096.0 if case.get("type") == "f16" else 1.0) / pairs
    s["seq_ptr"] = _sequences(g, 2 * pairs, case["tokens"])
    n = case["tokens"]
    if op == "step":
        s["target"] = _tokens(g, n, case["classes"], n // 5, IDS[case["ids"]])     # one token in five is the prompt's
        s["logits"] = _logits(g, n, case["classes"], 0, case["type"], s["target"])
        # the reference model: the same one, some steps of training ago
        policy = torch.empty(n, device=d)
        step = max(1, (1 << 26) // case["classes"])
        for a in range(0, n, step):
            x = s["logits"][a:a + step].float()
            policy[a:a + step] = x.gather(1, s["target"][a:a + step].long().clamp(0)[:, None])[:, 0] - x.logsumexp(1)
        s["ref_logp"] = policy + 0.3 * torch.randn(n, generator=g, device=d)
        s["mean"], s["mask"] = False, (s["target"] >= 0)
        return s
    s["logp"] = torch.empty(n, device=d).exponential_(0.5, generator=g).neg_()
    s["ref_logp"] = s["logp"] + 0.1 * torch.randn(n, generator=g, device=d) if case["reference"] else None
    s["mask"] = (torch.rand(n, generator=g, device=d) < 0.7) if case["masked"] else None
    s["mean"] = case["mean"]
    s["weight"] = torch.rand(pairs, generator=g, device=d).add_(0.5) if case["masked"] else None
    s["offset"] = torch.randn(pairs, generator=g, device=d).mul_(0.5) if case["masked"] else None
    return s


# ------------------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["op"]
    if own:
        k = _operators()
        if op == "lookup":
            return k.embedding_lookup(s["table"], s["ids"], scale=s["scale"])
        if op == "gradient":
            return k.embedding_gradient(s["grad_out"], s["ids"], s["rows"], scale=s["scale"])
        if op == "loglik":
            logp, stats = k.token_loglik(s["logits"], s["target"])
            if not s["train"]:
                return {"logp": logp}
            return {"logp": logp, "dlogits": k.token_loglik_gradient(s["logits"], s["target"], stats, s["g"])}
        if op == "preference":
            r = k.preference_loss(s["logp"], s["ref_logp"], s["seq_ptr"], beta=s["beta"], smoothing=s["smoothing"], scale=s["scale"], mask=s["mask"],
                                  weight=s["weight"], offset=s["offset"], mean=s["mean"])
            return {"loss": r.loss, "pair_loss": r.pair_loss, "margin": r.margin, "ratio": r.ratio, "grad": r.grad}
        logp, stats = k.token_loglik(s["logits"], s["target"])
        r = k.preference_loss(logp, s["ref_logp"], s["seq_ptr"], beta=s["beta"], smoothing=s["smoothing"], scale=s["scale"], mask=s["mask"])
        return {"loss": r.loss, "margin": r.margin, "logp": logp, "dlogits": k.token_loglik_gradient(s["logits"], s["target"], stats, r.grad)}
    if op == "lookup":
        return _lookup(s["table"], s["ids"], s["scale"])
    if op == "gradient":
        return _gradient(s["grad_out"], s["ids"], s["rows"], s["scale"])
    if op == "loglik":
        logp, top, log_sum = _loglik(s["logits"], s["target"])
        return {"logp": logp, "dlogits": _loglik_gradient(s["logits"], s["target"], top, log_sum, s["g"])} if s["train"] else {"logp": logp}
    if op == "preference":
        return _preference(s["logp"], s["ref_logp"], s["seq_ptr"], s["beta"], s["smoothing"], s["scale"], s["mask"], s["weight"], s["offset"], s["mean"])
    logp, top, log_sum = _loglik(s["logits"], s["target"])
    r = _preference(logp, s["ref_logp"], s["seq_ptr"], s["beta"], s["smoothing"], s["scale"], s["mask"], None, None, False)
    return {"loss": r["loss"], "margin": r["margin"], "logp": logp, "dlogits": _loglik_gradient(s["logits"], s["target"], top, log_sum, r["grad"])}


def _lookup(table, ids, scale):
    here = (ids >= 0) & (ids < table.shape[0])
    rows = table[torch.where(here, ids, torch.zeros_like(ids))].float() * scale
    return torch.where(here[:, None], rows, torch.zeros_like(rows)).to(table.dtype)


def _gradient(grad_out, ids, rows, scale):
    here = (ids >= 0) & (ids < rows)
    total = torch.zeros(rows + 1, grad_out.shape[1], device=ids.device)        # the last row takes what has no place
    total.index_add_(0, torch.where(here, ids, torch.full_like(ids, rows)), grad_out.float())
    return (total[:rows] * scale).to(grad_out.dtype)


def _loglik(logits, target):
    x = logits.float()
    here = (target >= 0) & (target < x.shape[1])
    at = torch.where(here, target, torch.zeros_like(target)).long()[:, None]
    top = x.amax(1, keepdim=True)
    log_sum = (x - top).exp().sum(1, keepdim=True, dtype=torch.float64).log()      # what a pair adds up is small next to it
    logp = ((x.gather(1, at) - top) - log_sum)[:, 0].float()
    return torch.where(here, logp, torch.zeros_like(logp)), top, log_sum.float()


def _loglik_gradient(logits, target, top, log_sum, g):
    here = (target >= 0) & (target < logits.shape[1])
    p = (logits.float() - top - log_sum).exp()
    hit = torch.arange(logits.shape[1], device=target.device)[None, :] == target[:, None]
    d = g[:, None] * (hit.float() - p)
    return torch.where(here[:, None], d, torch.zeros_like(d)).to(logits.dtype)


def _softplus(h):
    return h.clamp(min=0) + (-h.abs()).exp().log1p()


def _preference(logp, ref_logp, seq_ptr, beta, smoothing, scale, mask, weight, offset, mean):
    pairs, n = (seq_ptr.numel() - 1) // 2, logp.numel()
    d = logp.double() if ref_logp is None else logp.double() - ref_logp.double()      # sums over long sequences: in 64 bits
    count = torch.ones_like(d) if mask is None else mask.double()
    d = d if mask is None else torch.where(mask, d, torch.zeros_like(d))
    both = torch.nn.functional.pad(torch.stack([d, count]).cumsum(1), (1, 0))
    both = both[:, seq_ptr[1:]] - both[:, seq_ptr[:-1]]
    part = 1.0 / both[1].clamp(min=1) if mean else torch.ones_like(both[1])
    ratio = both[0] * part
    h = beta * (ratio[:pairs] - ratio[pairs:])
    h = h if offset is None else h + offset.double()
    w = scale if weight is None else scale * weight.double()
    pair_loss = (1 - smoothing) * _softplus(-h) + smoothing * _softplus(h)
    slope = w * beta * (torch.sigmoid(h) - (1 - smoothing))
    per_token = torch.cat([slope, -slope]) * part
    of = torch.searchsorted(seq_ptr[1:], torch.arange(n, device=logp.device), right=True)
    grad = per_token[of.clamp(max=2 * pairs - 1)] * count
    return {"loss": (w * pair_loss).sum().float(), "pair_loss": pair_loss.float(), "margin": h.float(), "ratio": ratio.float(), "grad": grad.float()}


# ---------------------------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "lookup":
        table = torch.cat([s["table"].double() * s["scale"], torch.zeros(1, s["table"].shape[1], dtype=torch.float64, device=s["ids"].device)])
        ids = s["ids"].long()
        return table.index_select(0, torch.where(ids < 0, table.shape[0] - 1, ids))
    if op == "gradient":
        # sorted by id, running sums, and what they gained over each id's stretch
        ids, order = torch.sort(s["ids"].long(), stable=True)
        x = s["grad_out"].double()[order] * s["scale"]
        out = torch.zeros(s["rows"], x.shape[1], dtype=torch.float64, device=ids.device)
        runs = torch.nn.functional.pad(x.cumsum(0), (0, 0, 1, 0))
        bounds = torch.searchsorted(ids, torch.arange(s["rows"] + 1, device=ids.device))
        used = (bounds[1:] > bounds[:-1]).nonzero()[:, 0]
        out[used] = runs[bounds[1:][used]] - runs[bounds[:-1][used]]
        return out
    if op == "loglik":
        logp = _exact_logp(s["logits"], s["target"])
        return {"logp": logp, "dlogits": _exact_dlogits(s["logits"], s["target"], s["g"].double())} if s["train"] else {"logp": logp}
    logp = s["logp"].double() if op == "preference" else _exact_logp(s["logits"], s["target"])
    r = _exact_preference(s, logp)
    if op == "preference":
        return r
    return {"loss": r["loss"], "margin": r["margin"], "logp": logp, "dlogits": _exact_dlogits(s["logits"], s["target"], r["grad"])}


def _parts(n, classes):
    step = max(1, (1 << 27) // classes)
    return [slice(a, min(n, a + step)) for a in range(0, n, step)]


def _exact_logp(logits, target):
    out = torch.zeros(target.numel(), dtype=torch.float64, device=target.device)
    for p in _parts(*logits.shape):
        t = target[p].long()
        all_of = torch.log_softmax(logits[p].double(), 1)
        out[p] = torch.where(t < 0, 0.0, all_of[torch.arange(t.numel(), device=t.device), t.clamp(min=0)])
    return out


def _exact_dlogits(logits, target, g):
    out = torch.empty(logits.shape, dtype=torch.float64, device=target.device)
    for p in _parts(*logits.shape):
        t = target[p].long()
        d = torch.softmax(logits[p].double(), 1).mul_(-g[p][:, None])
        d[torch.arange(t.numel(), device=t.device), t.clamp(min=0)] += g[p]
        d[t < 0] = 0
        out[p] = d
    return out


def _exact_preference(s, logp):
    seq_ptr, n = s["seq_ptr"], logp.numel()
    count, pairs = seq_ptr.numel() - 1, (seq_ptr.numel() - 1) // 2
    of = torch.repeat_interleave(torch.arange(count, device=seq_ptr.device), seq_ptr[1:] - seq_ptr[:-1], output_size=n)
    on = torch.ones(n, dtype=torch.float64, device=of.device) if s["mask"] is None else s["mask"].double()
    gain = (logp if s["ref_logp"] is None else logp - s["ref_logp"].double()) * on
    ratio = torch.zeros(count, dtype=torch.float64, device=of.device).index_add_(0, of, gain)
    long = torch.zeros(count, dtype=torch.float64, device=of.device).index_add_(0, of, on).clamp_(min=1) if s["mean"] else torch.ones_like(ratio)
    ratio = ratio / long
    h = s["beta"] * (ratio[:pairs] - ratio[pairs:])
    weight, offset = s.get("weight"), s.get("offset")
    h = h + (0.0 if offset is None else offset.double())
    w = s["scale"] * (torch.ones_like(h) if weight is None else weight.double())
    good, bad = torch.nn.functional.logsigmoid(h), torch.nn.functional.logsigmoid(-h)
    loss = -(1 - s["smoothing"]) * good - s["smoothing"] * bad
    dh = w * (s["smoothing"] * good.exp() - (1 - s["smoothing"]) * bad.exp())
    grad = torch.cat([dh, -dh])[of] * s["beta"] / long[of] * on
    return {"loss": (w * loss).sum(), "pair_loss": loss, "margin": h, "ratio": ratio, "grad": grad}


# ---------------------------------------------------------------------------------------------------------------- the least work
def _distinct(n, rows):
    """How many different ids n of them hold, on average."""
    k = np.arange(rows + 1, dtype=np.float64)
    p = np.log((k[1:] + 1) / (k[:-1] + 1)) / math.log(rows + 1)
    return float(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2, "f16": 2}.get(case.get("type"), 4)
    id_size = 4 if case.get("ids") == "i32" else 8
    if op == "lookup":
        there = case["n"] - case["absent"]
        return {"bytes": case["n"] * (id_size + case["width"] * size) + _distinct(there, case["rows"]) * case["width"] * size, "flops": there * case["width"]}
    if op == "gradient":
        there = case["n"] - case["absent"]
        return {"bytes": case["n"] * id_size + there * case["width"] * size + case["rows"] * case["width"] * size, "flops": there * case["width"]}
    if op == "loglik":
        there, row = case["n"] - case["absent"], case["classes"] * size
        # the gradient needs the whole sum first: the logits of a batch, more than the chip keeps, are read again
        return {"bytes": case["n"] * (id_size + 4) + there * row + (case["n"] * 4 + there * row + case["n"] * row if case["train"] else 0),
                "flops": there * case["classes"] * (4 + (3 if case["train"] else 0))}
    tokens = case["tokens"]
    if op == "preference":
        return {"bytes": tokens * (8 + (4 if case["reference"] else 0) + (1 if case["masked"] else 0)) + case["pairs"] * (16 + 16 + (8 if case["masked"] else 0)),
                "flops": 3 * tokens + 20 * case["pairs"]}
    there, row = tokens - tokens // 5, case["classes"] * size
    return {"bytes": tokens * (id_size + 4 + 4 + 1) + 2 * there * row + tokens * row + case["pairs"] * 20, "flops": there * case["classes"] * 7}
