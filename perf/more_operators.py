"""The class head as cases that can be measured: the softmax cross entropy of
features against a table of classes whose logits are never kept (the loss alone,
with its gradients, or first the loss and then its backward pass), the logits
themselves from features and a table in 8-bit floating point with a scale for each
block of 128, and the quantisation that makes both.

Features run from the 16 outputs of a labelled field to rows of 4096, tables from
two classes to 2^17, calls from one row to 2^16. `run` computes the plain form in
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
SCALES = {"f32": torch.float32, "e8m0": torch.float8_e8m0fnu}
BLOCK, LARGEST = 128, 448.0  # elements of a scale; the largest e4m3 value
own = False


def _loss(name, rows, dims, classes, dtype, gradient, temperature=1.0, two=False, index="i64"):
    return {"name": name, "do": "two" if two else "loss", "rows": rows, "dims": dims, "classes": classes,
            "dtype": dtype, "gradient": gradient, "temperature": temperature, "index": index}


def _logits(name, rows, dims, classes, dtype, scale):
    return {"name": name, "do": "logits", "rows": rows, "dims": dims, "classes": classes, "dtype": dtype,
            "scale": scale}


def _quantize(name, rows, dims, dtype, block_rows, scale):
    return {"name": name, "do": "quantize", "rows": rows, "dims": dims, "dtype": dtype,
            "block_rows": block_rows, "scale": scale}


def listed():
    return [
        # a training batch of a field whose 16 outputs are compared with 64 labels
        _loss("field_step", 4096, 16, 64, "f32", "both", index="i32"),
        # an open-vocabulary field: unit features against a fixed table of labels
        _loss("open_vocabulary", 65536, 64, 1000, "f32", "features", 0.07, index="i32"),
        # one row scored over a large table
        _loss("score_one", 1, 4096, 131072, "bf16", "none"),
        # a ragged training batch, an odd class count
        _loss("ragged_step", 515, 1000, 50021, "f16", "both"),
        # a training step over a vocabulary
        _loss("vocab_step", 4096, 2048, 131072, "bf16", "both"),
        # the loss first, its backward pass with the caller's weights
        _loss("loss_then_backward", 2048, 768, 32768, "f32", "both", two=True),
        # one row's logits over a large table in 8 bits
        _logits("f8_one", 1, 4096, 131072, "bf16", "f32"),
        # a batch of rows that are answered together
        _logits("f8_batch", 64, 2048, 65536, "f32", "e8m0"),
        # a large scoring batch
        _logits("f8_score", 4096, 4096, 65536, "bf16", "f32"),
        # odd sizes: blocks of the scales that the table ends inside of
        _logits("f8_odd", 777, 1000, 10007, "f16", "e8m0"),
        # a batch of features, a scale for 128 of a row
        _quantize("quantize_rows", 4096, 2048, "bf16", 1, "f32"),
        # a table, a scale for 128 x 128
        _quantize("quantize_table", 131072, 4096, "bf16", 128, "e8m0"),
    ]


def _between(rng, low, high):
    n = int(round(2.0 ** rng.uniform(math.log2(low), math.log2(high))))
    return n | 1 if n > 8 and rng.random() < 0.4 else n


def draw(rng):
    do = rng.choice(["loss"] * 3 + ["two"] + ["logits"] * 3 + ["quantize"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    dims = _between(rng, 8, 4096)
    if rng.random() < 0.6:
        dims = (dims + 15) // 16 * 16
    if do == "quantize":
        rows = _between(rng, 1, min(2.0 ** 17, 2.0 ** 28 / dims))
        case = _quantize(None, rows, dims, dtype, rng.choice([1, 128]), rng.choice(["f32", "e8m0"]))
    else:
        classes = _between(rng, 2, 2.0 ** 17)
        rows = _between(rng, 1, max(2.0, min(2.0 ** 16, 2.0 ** 28 / classes, 2.0 ** 39 / (classes * dims))))
        if do == "logits":
            case = _logits(None, rows, dims, classes, dtype, rng.choice(["f32", "e8m0"]))
        else:
            case = _loss(None, rows, dims, classes, dtype, rng.choice(["both", "both", "features", "table"]),
                         rng.choice([0.7, 1.0, 1.0]), do == "two", rng.choice(["i32", "i64"]))
            if do == "loss" and rng.random() < 0.3:
                case["gradient"] = "none"
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------


def _features_and_table(case, g, dtype):
    """Features of a trained network and the table that they are compared with:
    each row leans towards its label's class, three in four far enough."""
    n, d, v = case["rows"], case["dims"], case["classes"]
    unit = case.get("temperature", 1.0) < 0.5
    spread = 1.0 if unit else 1.5
    table = torch.randn(v, d, device=DEVICE, generator=g).mul_(spread / math.sqrt(d))
    labels = torch.randint(0, v, (n,), device=DEVICE, generator=g)
    lean = torch.rand(n, 1, device=DEVICE, generator=g)
    lean = torch.where(lean < 0.25, 0.0, 4.0 * lean)
    x = torch.randn(n, d, device=DEVICE, generator=g)
    if unit:
        table = torch.nn.functional.normalize(table, dim=1)
        x = torch.nn.functional.normalize(x / math.sqrt(d) + lean / 4.0 * table[labels], dim=1)
    else:
        x += lean * table[labels]
    return x.to(dtype), table.to(dtype), labels


def _scale_of(amax, scale):
    """The scale of blocks with these largest magnitudes, in fp32: a block's
    largest value becomes at most 448; blocks of zeros have scale 1."""
    s = (amax.double() / LARGEST).float().clamp_min(2.0 ** -126)  # (in 32 bits it is multiplied by 1 / 448)
    if scale == "e8m0":
        mantissa, exponent = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), torch.where(mantissa == 0.5, exponent - 1, exponent))
    return torch.where(amax == 0, 1.0, s)


def _spread_scales(s, rows, dims, block_rows):
    """A scale for each element from one for each block."""
    s = s.repeat_interleave(block_rows, 0)[:rows] if block_rows > 1 else s
    return s.repeat_interleave(BLOCK, 1)[:, :dims]


def _quantized(x, block_rows, scale):
    """(values as e4m3, scales in fp32 [row blocks][column blocks])."""
    rows, dims = x.shape
    down, across = -(-rows // block_rows), -(-dims // BLOCK)
    padded = x.new_zeros((down * block_rows, across * BLOCK), dtype=torch.float32)
    padded[:rows, :dims] = x
    amax = padded.abs().view(down, block_rows, across, BLOCK).amax((1, 3))
    s = _scale_of(amax, scale)
    # (in 64 bits: quotients in 32 can lie on a border between two values that they are beside)
    y = padded.double().view(down, block_rows, across, BLOCK) / s.double().view(down, 1, across, 1)
    y = y.view(down * block_rows, across * BLOCK)[:rows, :dims]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step).mul_(step).float().to(torch.float8_e4m3fn), s


def _rows_of_16(q):
    """8-bit values as the quantisation lays them out: rows start at multiples of 16 bytes."""
    n, d = q.shape
    place = torch.zeros(n, (d + 15) // 16 * 16, device=DEVICE, dtype=torch.uint8)
    place[:, :d] = q.view(torch.uint8)
    return place.view(torch.float8_e4m3fn)[:, :d]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    f32 = {"device": DEVICE, "dtype": torch.float32}
    s = {"case": case}
    n, d = case["rows"], case["dims"]
    dtype = TYPES[case["dtype"]]
    if case["do"] == "quantize":
        # a few columns far larger than the rest, as trained weights and features have
        wide = torch.exp(torch.randn(d, device=DEVICE, generator=g))
        s["x"] = torch.empty(n, d, device=DEVICE, dtype=dtype)
        for lo in range(0, n, 16384):
            part = s["x"][lo:lo + 16384]
            part.copy_(torch.randn(part.shape, device=DEVICE, generator=g) * wide)
        down, across = -(-n // case["block_rows"]), -(-d // BLOCK)
        s["out"] = {"values": _rows_of_16(torch.zeros(n, d, device=DEVICE, dtype=torch.float8_e4m3fn)),
                    "scales": torch.ones(down, across, **f32).to(SCALES[case["scale"]])}
        return s
    v = case["classes"]
    if case["do"] == "logits":
        x, table, _ = _features_and_table(case, g, torch.float32)
        for name, data, block_rows in (("features", x, 1), ("table", table, BLOCK)):
            q, scales = _quantized(data, block_rows, case["scale"])
            s[name], s[name + "_scales"] = _rows_of_16(q), scales.to(SCALES[case["scale"]])
        s["out"] = torch.empty(n, v, device=DEVICE, dtype=dtype)
        return s
    s["features"], s["table"], labels = _features_and_table(case, g, dtype)
    # the mean over the batch; 16-bit gradients with few exponent bits are scaled
    # up, as training in that type scales its loss; one row in 16 is padding
    mean = (4096.0 if case["dtype"] == "f16" else 1.0) / n
    weights = torch.full((n,), mean, **f32)
    if case["do"] == "two":  # upstream gradients of the caller's own
        weights *= 0.5 + torch.rand(n, device=DEVICE, generator=g)
    if n >= 16:
        labels = torch.where(torch.rand(n, device=DEVICE, generator=g) < 1 / 16, -1, labels)
    s["weights"] = weights
    s["labels"] = labels.to(torch.int32 if case["index"] == "i32" else torch.int64)
    s["out"] = {"loss": torch.empty(n, **f32), "stats": torch.empty(n, 4, **f32)}
    if case["gradient"] in ("both", "features"):
        s["out"]["d_features"] = torch.empty_like(s["features"])
    if case["gradient"] in ("both", "table"):
        s["out"]["d_table"] = torch.empty_like(s["table"])
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
    ops, case, out = _ops(), s["case"], s["out"]
    if case["do"] == "quantize":
        ops.quantize_f8(s["x"], block_rows=case["block_rows"], scale_dtype=SCALES[case["scale"]], out=out)
        return {"values": out["values"].float(), "scales": out["scales"].float()}
    if case["do"] == "logits":
        return {"logits": ops.class_logits_f8(s["features"], s["features_scales"], s["table"],
                                              s["table_scales"], out=out)}
    what = {"temperature": case["temperature"], "out": out}
    if case["do"] == "two":
        ops.class_loss(s["features"], s["table"], s["labels"], gradient="none", **what)
        ops.class_loss_backward(s["features"], s["table"], s["labels"], out["stats"], s["weights"],
                                gradient=case["gradient"], **what)
    else:
        ops.class_loss(s["features"], s["table"], s["labels"], row_weights=s["weights"],
                       gradient=case["gradient"], **what)
    return {name: out[name] for name in ("loss", "d_features", "d_table") if name in out}


# ---- the plain form: 32 bits, rounded once ---------------------------------------


def _plain_loss(s):
    case, labels = s["case"], s["labels"].long()
    x, table, weights = s["features"].float(), s["table"].float(), s["weights"]
    inv_t = 1 / case["temperature"]
    z = torch.matmul(x, table.t()) * inv_t
    z -= z.amax(1, keepdim=True)
    given = labels >= 0
    at = labels.clamp_min(0).unsqueeze(1)
    mine = z.gather(1, at)
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    loss = torch.where(given, (torch.log(total) - mine)[:, 0], 0.0)
    w = torch.where(given, weights, 0.0).unsqueeze(1)
    out = {"loss": loss if case["do"] == "two" else loss * w[:, 0]}
    if case["gradient"] == "none":
        return out
    p *= w * inv_t / total
    p.scatter_add_(1, at, -w * inv_t)
    if case["gradient"] in ("both", "features"):
        out["d_features"] = torch.matmul(p, table).to(s["features"].dtype)
    if case["gradient"] in ("both", "table"):
        out["d_table"] = torch.matmul(p.t(), x).to(s["table"].dtype)
    return out


def _plain_logits(s):
    x = s["features"].float()
    x *= _spread_scales(s["features_scales"].float(), *x.shape, 1)
    table = s["table"].float()
    table *= _spread_scales(s["table_scales"].float(), *table.shape, BLOCK)
    return {"logits": torch.matmul(x, table.t()).to(s["out"].dtype)}


def _plain_quantize(s):
    q, scales = _quantized(s["x"], s["case"]["block_rows"], s["case"]["scale"])
    return {"values": q.float(), "scales": scales}


def run(state):
    if own:
        return _run_own(state)
    return {"quantize": _plain_quantize, "logits": _plain_logits}.get(state["case"]["do"], _plain_loss)(state)


def work(case):
    n, d = case["rows"], case["dims"]
    if case["do"] == "quantize":  # the matrix; its values and scales
        blocks = -(-n // case["block_rows"]) * -(-d // BLOCK)
        return {"bytes": n * d * (SIZES[case["dtype"]] + 1) + blocks * (4 if case["scale"] == "f32" else 1),
                "flops": 2 * n * d}
    v, size = case["classes"], SIZES[case["dtype"]]
    if case["do"] == "logits":  # values and scales; the logits
        blocks = (n + -(-v // BLOCK)) * -(-d // BLOCK)
        return {"bytes": (n + v) * d + blocks * (4 if case["scale"] == "f32" else 1) + n * v * size,
                "flops": 2 * n * v * d}
    grads = {"none": 0, "both": 2}.get(case["gradient"], 1)
    read, rows = (n + v) * d * size, n * ((4 if case["index"] == "i32" else 8) + 8)
    write = (n * (case["gradient"] in ("both", "features")) + v * (case["gradient"] in ("both", "table"))) * d * size
    if case["do"] == "two":  # the backward pass begins with the logits again
        return {"bytes": 2 * read + write + 2 * rows, "flops": 2 * n * v * d * (2 + grads)}
    return {"bytes": read + write + rows, "flops": 2 * n * v * d * (1 + grads)}


# ---- the definitions in 64 bits ---------------------------------------------------


def _exact_quantize(case, s):
    """Each value is the nearest of e4m3's to x over its block's scale (the scale
    as it is stored), ties to the even one."""
    n, d = s["x"].shape
    values = torch.empty(n, d, device=DEVICE, dtype=torch.float64)
    scales = []
    grid = torch.arange(127, device=DEVICE, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double()
    middle = (grid[1:] + grid[:-1]) / 2
    for lo in range(0, n, 8192):  # (a multiple of the blocks' rows)
        x = s["x"][lo:lo + 8192].double()
        rows = x.shape[0]
        down, across = -(-rows // case["block_rows"]), -(-d // BLOCK)
        padded = torch.nn.functional.pad(x, (0, across * BLOCK - d, 0, down * case["block_rows"] - rows))
        amax = padded.view(down, case["block_rows"], across, BLOCK).abs().amax((1, 3))
        scale = amax / LARGEST
        if case["scale"] == "e8m0":
            scale = torch.exp2(torch.ceil(torch.log2(scale.clamp_min(1e-300))))
        scale = torch.where(amax == 0, 1.0, scale.clamp_min(2.0 ** -126))
        scales.append(scale)
        y = x / _spread_scales(scale.float().double(), rows, d, case["block_rows"])
        at = torch.bucketize(y.abs(), middle)  # (on a border: the lower one)
        at += (y.abs() == middle[at.clamp_max(125)]) & (at % 2 == 1)
        values[lo:lo + rows] = torch.copysign(grid[at], y)
    return {"values": values, "scales": torch.cat(scales)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["do"] == "quantize":
        return _exact_quantize(case, s)
    if case["do"] == "logits":
        x = s["features"].float().double() * _spread_scales(s["features_scales"].float().double(), *s["features"].shape, 1)
        table = s["table"].float().double()
        table *= _spread_scales(s["table_scales"].float().double(), *table.shape, BLOCK)
        out = torch.empty(x.shape[0], table.shape[0], device=DEVICE, dtype=torch.float64)
        for lo in range(0, x.shape[0], 1024):
            out[lo:lo + 1024] = x[lo:lo + 1024] @ table.t()
        return {"logits": out}
    x, table, labels = s["features"].double(), s["table"].double(), s["labels"].long()
    n = x.shape[0]
    t, weights = case["temperature"], s["weights"].double()
    loss = torch.zeros(n, device=DEVICE, dtype=torch.float64)
    d_features, d_table = torch.zeros_like(x), torch.zeros_like(table)
    step = max(1, (1 << 27) // case["classes"])
    for lo in range(0, n, step):
        part, label = x[lo:lo + step], labels[lo:lo + step]
        row = torch.arange(part.shape[0], device=DEVICE)[label >= 0]
        logp = torch.log_softmax((part @ table.t()) / t, 1)
        up = torch.zeros_like(logp)  # of the log-probabilities: the loss is -w ln p of the label
        up[row, label[row]] = -weights[lo:lo + step][row]
        loss[lo + row] = -logp[row, label[row]]
        if case["gradient"] != "none":
            d = (up - torch.exp(logp) * up.sum(1, keepdim=True)) / t
            d_features[lo:lo + step] = d @ table
            d_table += d.t() @ part
    out = {"loss": loss if case["do"] == "two" else loss * weights}
    if case["gradient"] in ("both", "features"):
        out["d_features"] = d_features
    if case["gradient"] in ("both", "table"):
        out["d_table"] = d_table
    return out
