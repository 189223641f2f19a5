"""The class-logit operators as cases that can be measured: log-probabilities
of given classes with their rank, the entropy and the best alternatives, the
gradient of all of these, and distillation from a teacher's listed values
(loss and gradient together, the loss alone, or the loss and then its backward
pass).

Rows run from the 16 outputs of a labelled field to vocabularies of 2^18
classes, calls from one row to 2^18 rows. `run` computes the plain form in
32-bit torch, rounded once at the end, or, where `own` is true, calls
`tiny_metal_nn.LogitOps`; `exact` states the same definitions in 64 bits.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
own = False


def _case(name, do, rows, classes, dtype, k, temperature=1.0, masked=0.0, kind="", index="i64"):
    return {"name": name, "do": do, "rows": rows, "classes": classes, "dtype": dtype, "k": k,
            "temperature": temperature, "masked": masked, "kind": kind, "index": index}


def listed():
    return [
        # the labels of a 256 x 256 view of a field with 16 class outputs
        _case("label_query", "logprobs", 1 << 16, 16, "f32", 3, index="i32"),
        # one decoded token
        _case("decode_one", "logprobs", 1, 32768, "bf16", 5, 0.7),
        # a decoding batch under a grammar: half of the classes masked
        _case("decode_masked", "logprobs", 64, 131072, "f32", 20, masked=0.5),
        # prompts scored, an odd class count (no two rows aligned alike)
        _case("score_odd", "logprobs", 4099, 50021, "f16", 8),
        # a large scoring batch
        _case("score_large", "logprobs", 4096, 131072, "bf16", 20),
        # labels of a training batch of the field: gradients of all outputs
        _case("label_grad", "logprobs_grad", 1 << 18, 16, "f32", 3, index="i32"),
        # a policy gradient with an entropy term
        _case("policy_grad", "logprobs_grad", 4096, 32768, "bf16", 0),
        # the same for few rows of an odd class count, with alternatives
        _case("policy_grad_odd", "logprobs_grad", 515, 100003, "f32", 8, 0.7),
        # a field that learns its labels from a teacher, 2^18 points a step
        _case("field_distill", "distill", 1 << 18, 16, "f32", 4, 2.0, kind="logits", index="i32"),
        # a classifier's step on a ragged batch, the teacher's tail as a class
        _case("class_distill", "distill", 30011, 1000, "f16", 8, 2.0, kind="logprobs"),
        # few long rows: the loss first, its backward pass with the caller's weights
        _case("long_distill", "distill_two", 12, 262144, "f32", 64, kind="logits"),
        # a training step over a vocabulary
        _case("vocab_distill", "distill", 8192, 65536, "bf16", 32, kind="logprobs", index="i32"),
    ]


def draw(rng):
    do = rng.choice(["logprobs"] * 3 + ["logprobs_grad"] * 2 + ["distill"] * 3 +
                    ["distill_loss", "distill_two"])
    classes = int(round(2.0 ** rng.uniform(1, 18)))
    rows = int(round(2.0 ** rng.uniform(0, min(18.0, 28.0 - math.log2(classes)))))
    if rows > 8 and rng.random() < 0.7:
        rows |= 1
    top = min(classes, 64)
    case = _case(None, do, rows, classes, rng.choice(["f32", "f16", "bf16", "bf16"]),
                 rng.choice([1, min(3, top), min(8, top), min(20, top), top]),
                 rng.choice([0.7, 1.0, 1.0, 2.0]),
                 rng.choice([0.0, 0.0, 0.5]) if do.startswith("logprobs") and classes >= 256 else 0.0,
                 "" if do.startswith("logprobs") else rng.choice(["logits", "logprobs"]),
                 rng.choice(["i32", "i64"]))
    if do == "logprobs_grad" and rng.random() < 0.5:
        case["k"] = 0
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------


def _mean_weight(case):
    """A row's weight in the mean over the batch; 16-bit gradients with few
    exponent bits are scaled up, as training in that type scales its loss."""
    return (1024.0 if case["dtype"] == "f16" else 1.0) / case["rows"]


def _rows_at_once(case):
    return max(1, (1 << 26) // case["classes"])


def _logits(case, g, scale):
    """Logits of a trained network: a broad floor, about one class in 64
    raised, a few far above the rest."""
    n, v = case["rows"], case["classes"]
    z = torch.empty(n, v, device=DEVICE, dtype=TYPES[case["dtype"]])
    for lo in range(0, n, _rows_at_once(case)):
        part = z[lo:lo + _rows_at_once(case)]
        x = torch.randn(part.shape, device=DEVICE, generator=g)
        x *= 1.5 * scale
        u = torch.rand(part.shape, device=DEVICE, generator=g)
        x += (u < 1 / 64) * (3.0 * scale)
        if v >= 256:
            best = torch.randint(0, v, (part.shape[0], 4), device=DEVICE, generator=g)
            x.scatter_add_(1, best, torch.rand(best.shape, device=DEVICE, generator=g) * 6 * scale + 6)
        part.copy_(x)
    return z


def _best(values, k):
    """The k best classes of each row: (ids, values), by value and then by the
    lowest index; -inf is no alternative (id -1)."""
    v = values.shape[1]
    bits = (values + 0.0).view(torch.int32)
    order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    key = (order.to(torch.int64) << 32) + (v - 1 - torch.arange(v, device=values.device))
    key = torch.topk(key, min(k, v), dim=1).values
    ids = v - 1 - (key & 0xFFFFFFFF)
    got = values.gather(1, ids)
    ids = ids.masked_fill(got == -math.inf, -1)
    if k > v:
        ids = torch.nn.functional.pad(ids, (0, k - v), value=-1)
        got = torch.nn.functional.pad(got, (0, k - v), value=-math.inf)
    return ids, got


def _best_of_parts(case, z, k):
    ids = torch.empty(z.shape[0], k, dtype=torch.int64, device=DEVICE)
    got = torch.empty(z.shape[0], k, device=DEVICE)
    for lo in range(0, z.shape[0], _rows_at_once(case)):
        hi = lo + _rows_at_once(case)
        ids[lo:hi], got[lo:hi] = _best(z[lo:hi].float(), k)
    return ids, got


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    n, v, k = case["rows"], case["classes"], case["k"]
    index = torch.int32 if case["index"] == "i32" else torch.int64
    f32 = {"device": DEVICE, "dtype": torch.float32}
    s = {"case": case, "z": _logits(case, g, 1.0)}
    if case["do"].startswith("logprobs"):
        # tokens that the rows' own distribution draws; one in 16 is padding
        tokens = torch.empty(n, dtype=torch.int64, device=DEVICE)
        for lo in range(0, n, _rows_at_once(case)):
            part = s["z"][lo:lo + _rows_at_once(case)]
            u = torch.rand(part.shape, device=DEVICE, generator=g).clamp_min_(1e-20)
            tokens[lo:lo + _rows_at_once(case)] = (part.float() / case["temperature"] -
                                                   torch.log(-torch.log(u))).argmax(1)
            if case["masked"]:
                hide = torch.rand(part.shape, device=DEVICE, generator=g) < case["masked"]
                hide.scatter_(1, tokens[lo:lo + _rows_at_once(case)].unsqueeze(1), False)
                part.masked_fill_(hide, -math.inf)
        if n >= 16:
            tokens[torch.rand(n, device=DEVICE, generator=g) < 1 / 16] = -1
        s["tokens"] = tokens.to(index)
        s["out"] = {"logprob": torch.empty(n, **f32), "entropy": torch.empty(n, **f32),
                    "rank": torch.empty(n, dtype=torch.int32, device=DEVICE),
                    "stats": torch.empty(n, 2, **f32),
                    "top_ids": torch.empty(n, k, dtype=torch.int32, device=DEVICE),
                    "top_logprobs": torch.empty(n, k, **f32)}
        if case["do"] == "logprobs_grad":
            # what a forward pass left (its outputs are this pass's inputs)
            lp, h, m, total, ids = [], [], [], [], []
            for lo in range(0, n, _rows_at_once(case)):
                part = s["z"][lo:lo + _rows_at_once(case)].float()
                x = (part / case["temperature"]).double()
                top = part.amax(1)
                lse = torch.logsumexp(x, 1)
                p = torch.exp(x - lse.unsqueeze(1))
                h.append(-(p * (x - lse.unsqueeze(1)).masked_fill(p == 0, 0)).sum(1))
                m.append(top)
                total.append(torch.exp(lse - top.double() / case["temperature"]))
                if k:
                    ids.append(_best(part, k)[0])
            s["out"]["entropy"].copy_(torch.cat(h))
            s["out"]["stats"].copy_(torch.stack([torch.cat(m).double(), torch.cat(total)], 1))
            if k:
                s["out"]["top_ids"].copy_(torch.cat(ids))
            mean = _mean_weight(case)
            s["d_logprob"] = torch.randn(n, device=DEVICE, generator=g) * mean
            s["d_entropy"] = torch.full((n,), 0.01 * mean, **f32)
            s["d_top"] = torch.randn(n, k, device=DEVICE, generator=g) * (0.1 * mean) if k else None
            s["d_logits"] = torch.empty_like(s["z"])
        return s
    # the teacher sees what the student sees, with another noise
    t = _logits(case, g, 0.5)
    for lo in range(0, n, _rows_at_once(case)):
        hi = lo + _rows_at_once(case)
        t[lo:hi] += 0.7 * s["z"][lo:hi]
    s["ids"], s["teacher"] = _best_of_parts(case, t, k)
    if case["kind"] == "logprobs":
        lse = torch.cat([torch.logsumexp(t[lo:lo + _rows_at_once(case)].float() / case["temperature"], 1)
                         for lo in range(0, n, _rows_at_once(case))])
        s["teacher"] = s["teacher"] / case["temperature"] - lse.unsqueeze(1)
    if k > 1:  # some rows keep fewer values
        short = torch.rand(n, device=DEVICE, generator=g) < 1 / 8
        s["ids"][:, k - 1].masked_fill_(short, -1)
    s["ids"] = s["ids"].to(index)
    weights = torch.full((n,), _mean_weight(case), **f32)
    if n >= 16:
        weights[torch.rand(n, device=DEVICE, generator=g) < 1 / 16] = 0
    s["weights"] = weights
    s["out"] = {"loss": torch.empty(n, **f32), "stats": torch.empty(n, 4, **f32)}
    if case["do"] != "distill_loss":
        s["out"]["d_logits"] = torch.empty_like(s["z"])
    return s


# ---- the framework's operators -------------------------------------------------

_handle = None


def _ops():
    global _handle
    if _handle is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "tiny-metal-nn_amd"))
        from tiny_metal_nn import LogitOps
        _handle = LogitOps()
    return _handle


def _run_own(s):
    ops, case = _ops(), s["case"]
    t, out = case["temperature"], s["out"]
    if case["do"] == "logprobs":
        ops.token_logprobs(s["z"], s["tokens"], top_k=case["k"], temperature=t, out=out)
        return {name: out[name] for name in ("logprob", "entropy", "rank", "top_ids", "top_logprobs")}
    if case["do"] == "logprobs_grad":
        return {"d_logits": ops.token_logprobs_backward(
            s["z"], s["tokens"], out, d_logprob=s["d_logprob"], d_entropy=s["d_entropy"],
            d_top_logprobs=s["d_top"], temperature=t, out=s["d_logits"])}
    if case["do"] == "distill_two":
        ops.distill(s["z"], s["ids"], s["teacher"], kind=case["kind"], temperature=t,
                    gradient=False, out=out)
        ops.distill_backward(s["z"], s["ids"], s["teacher"], out["stats"], s["weights"],
                             kind=case["kind"], temperature=t, out=out["d_logits"])
        return {"loss": out["loss"], "d_logits": out["d_logits"]}
    ops.distill(s["z"], s["ids"], s["teacher"], kind=case["kind"], temperature=t,
                row_weights=s["weights"], gradient=case["do"] == "distill", out=out)
    return {name: out[name] for name in ("loss", "d_logits") if name in out}


# ---- the plain form: 32 bits, rounded once ---------------------------------------


def _plain_logprobs(s):
    case, z, tokens = s["case"], s["z"].float(), s["tokens"].long()
    x = z / case["temperature"]
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total[:, 0] - (e * x.masked_fill(e == 0, 0)).sum(1) / total[:, 0]
    given = tokens >= 0
    at = tokens.clamp_min(0).unsqueeze(1)
    logprob = torch.where(given, (x.gather(1, at) - log_total)[:, 0], 0.0)
    mine = z.gather(1, at)
    index = torch.arange(z.shape[1], device=z.device)
    rank = ((z > mine) | ((z == mine) & (index < at))).sum(1)
    rank = torch.where(given, rank, -1).to(torch.int32)
    ids, _ = _best(z, case["k"])
    top = torch.where(ids >= 0, x.gather(1, ids.clamp_min(0)) - log_total, -math.inf)
    return {"logprob": logprob, "entropy": entropy, "rank": rank,
            "top_ids": ids.to(torch.int32), "top_logprobs": top}


def _plain_logprobs_grad(s):
    case, z, tokens = s["case"], s["z"].float(), s["tokens"].long()
    c = 1 / case["temperature"]
    m, total = s["out"]["stats"][:, :1], s["out"]["stats"][:, 1:]
    logp = (z - m) * c - torch.log(total)
    p = torch.exp(logp)
    given = (tokens >= 0).unsqueeze(1)
    g_token = torch.where(given, s["d_logprob"].unsqueeze(1), 0.0)
    g_entropy = s["d_entropy"].unsqueeze(1)
    d = -p * (g_token + g_entropy * (logp.masked_fill(p == 0, 0) + s["out"]["entropy"].unsqueeze(1)))
    if case["k"]:
        ids = s["out"]["top_ids"].long()
        g_top = torch.where(ids >= 0, s["d_top"], 0.0)
        d -= p * g_top.sum(1, keepdim=True)
        d.scatter_add_(1, ids.clamp_min(0), g_top)
    d.scatter_add_(1, tokens.clamp_min(0).unsqueeze(1), g_token)
    return {"d_logits": (d * c).to(s["z"].dtype)}


def _plain_distill(s):
    case, ids = s["case"], s["ids"].long()
    t, w = case["temperature"], s["weights"].unsqueeze(1)
    x = s["z"].float() / t
    x = x - x.amax(1, keepdim=True)
    p = torch.exp(x)
    total = p.sum(1, keepdim=True)
    log_total = torch.log(total)
    p /= total
    used = ids >= 0
    at = ids.clamp_min(0)
    if case["kind"] == "logits":
        a = (s["teacher"] / t).masked_fill(~used, -math.inf)
        logq = a - torch.logsumexp(a, 1, keepdim=True)
    else:
        logq = s["teacher"].masked_fill(~used, -math.inf)
    q = torch.exp(logq)
    term = q * (logq - (x.gather(1, at) - log_total))
    loss = term.masked_fill(q == 0, 0).sum(1)
    mass = q.sum(1, keepdim=True)
    if case["kind"] == "logits":
        d = p * mass
    else:
        listed_ = torch.zeros(x.shape, dtype=torch.int32, device=x.device)
        listed_.scatter_add_(1, at, used.int())
        rest = x.masked_fill(listed_ > 0, -math.inf)
        top = rest.amax(1, keepdim=True)
        any_left = top > -math.inf
        top = torch.where(any_left, top, 0.0)
        rest = torch.exp(rest - top)
        rest_total = torch.where(any_left, rest.sum(1, keepdim=True), 1.0)
        q_rest = torch.where(any_left, (1 - mass).clamp_min(0), 0.0)
        logp_rest = top + torch.log(rest_total) - log_total
        more = q_rest * (torch.log(q_rest) - logp_rest)
        loss = loss + more.masked_fill(q_rest == 0, 0)[:, 0]
        d = p * (mass + q_rest) - rest * (q_rest / rest_total)
    if case["do"] == "distill_two":
        out = {"loss": loss * t * t}
    else:
        out = {"loss": torch.where(w[:, 0] == 0, 0.0, loss * t * t * w[:, 0])}
    if case["do"] != "distill_loss":
        d.scatter_add_(1, at, torch.where(used, -q, 0.0))
        out["d_logits"] = torch.where(w == 0, 0.0, d * (t * w)).to(s["z"].dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"logprobs": _plain_logprobs, "logprobs_grad": _plain_logprobs_grad}.get(
        state["case"]["do"], _plain_distill)(state)


def work(case):
    n, v, k, size = case["rows"], case["classes"], case["k"], SIZES[case["dtype"]]
    index = 4 if case["index"] == "i32" else 8
    logits = n * v
    if case["do"] == "logprobs":  # logits and tokens; log p, entropy, rank, alternatives
        return {"bytes": logits * size + n * (index + 12 + 8 * k), "flops": 8 * logits}
    if case["do"] == "logprobs_grad":  # logits, statistics, upstream gradients; the gradient
        return {"bytes": 2 * logits * size + n * (index + 20 + 8 * k), "flops": 8 * logits}
    rows = n * (k * (index + 4) + 8)
    if case["do"] == "distill_loss":
        return {"bytes": logits * size + rows, "flops": 6 * logits}
    if case["do"] == "distill":
        return {"bytes": 2 * logits * size + rows, "flops": 10 * logits}
    return {"bytes": 3 * logits * size + 2 * rows, "flops": 12 * logits}


# ---- the definitions in 64 bits ---------------------------------------------------


def _exact_rows(case, s, lo, hi):
    """The rows lo..hi, from log-probabilities over all classes."""
    z = s["z"][lo:hi].double()
    t = case["temperature"]
    logp = torch.log_softmax(z / t, 1)
    p = logp.exp()
    if case["do"] == "logprobs":
        tokens = s["tokens"][lo:hi].long()
        row = torch.arange(hi - lo, device=DEVICE)
        logprob = torch.where(tokens >= 0, logp[row, tokens.clamp_min(0)], 0.0)
        plogp = torch.where(p > 0, p * logp, 0.0)
        best = torch.topk(logp, min(case["k"], case["classes"]), dim=1).values
        return {"logprob": logprob, "entropy": -plogp.sum(1), "rank": None, "top_ids": None,
                "top_logprobs": best}
    if case["do"] == "logprobs_grad":
        tokens = s["tokens"][lo:hi].long()
        row = torch.arange(hi - lo, device=DEVICE)
        # L = sum_n g_n log p(token_n) + h_n H_n + sum_j t_nj log p(top_nj): the
        # weight of each class's log p, and of the entropy
        weight = torch.zeros_like(logp)
        weight[row, tokens.clamp_min(0)] += s["d_logprob"][lo:hi].double() * (tokens >= 0)
        if case["k"]:
            ids = s["out"]["top_ids"][lo:hi].long()
            weight.scatter_add_(1, ids.clamp_min(0), s["d_top"][lo:hi].double() * (ids >= 0))
        entropy = -torch.where(p > 0, p * logp, 0.0).sum(1, keepdim=True)
        d = weight - p * weight.sum(1, keepdim=True)
        d -= s["d_entropy"][lo:hi].double().unsqueeze(1) * torch.where(p > 0, p * (logp + entropy), 0.0)
        return {"d_logits": d / t}
    ids = s["ids"][lo:hi].long()
    used = ids >= 0
    teacher = s["teacher"][lo:hi].double()
    w = s["weights"][lo:hi].double()
    if case["kind"] == "logits":
        q = torch.softmax((teacher / t).masked_fill(~used, -math.inf), 1)
    else:
        q = teacher.exp().masked_fill(~used, 0.0)
    dense = torch.zeros_like(p).scatter_add_(1, ids.clamp_min(0), q)
    mine = torch.zeros_like(p).scatter_add_(1, ids.clamp_min(0), used.double()) > 0
    log_dense = torch.log(dense.clamp_min(1e-300))
    loss = torch.where(dense > 0, dense * (log_dense - logp), 0.0).sum(1)
    d = p * dense.sum(1, keepdim=True) - dense
    if case["kind"] == "logprobs":
        left = (~mine).any(1)
        q_rest = torch.where(left, (1 - q.sum(1)).clamp_min(0), 0.0)
        logp_rest = torch.logsumexp(logp.masked_fill(mine, -math.inf), 1)
        loss = loss + torch.where(q_rest > 0, q_rest * (torch.log(q_rest.clamp_min(1e-300)) - logp_rest), 0.0)
        share = torch.exp(logp.masked_fill(mine, -math.inf) - logp_rest.unsqueeze(1))
        share = torch.where(left.unsqueeze(1), share, 0.0)
        d += q_rest.unsqueeze(1) * (p - share)
    factor = 1.0 if case["do"] == "distill_two" else w
    out = {"loss": loss * t * t * factor}
    if case["do"] != "distill_loss":
        out["d_logits"] = d * (t * w).unsqueeze(1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    parts = []
    step = max(1, (1 << 25) // case["classes"])
    for lo in range(0, case["rows"], step):
        part = _exact_rows(case, s, lo, min(case["rows"], lo + step))
        parts.append({k: v if v is None else v.clone() for k, v in part.items()})
    return {k: None if v is None else torch.cat([q[k] for q in parts]) for k, v in parts[0].items()}
