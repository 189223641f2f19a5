"""The class head's operators in 64 bits (torch, on the inputs' device), from their
definitions, with the sums of absolute terms that error bounds are taken from."""
from __future__ import annotations

import torch

BLOCK = 128


def class_loss(features, table, labels, weights=None, t=1.0):
    """loss, stats, d_features, d_table of the weighted sum; and what bounds are relative to:
    `z` sum |h W| per logit (largest of a row), `x` sum |d| |W|, `y` sum |d| |h|."""
    h, w, labels = features.double(), table.double(), labels.long()
    n, v = h.shape[0], w.shape[0]
    weights = torch.ones(n, dtype=torch.float64, device=h.device) if weights is None else weights.double()
    used = (labels >= 0) & (weights != 0)
    h = torch.where(used.unsqueeze(1), h, 0.0)
    z = h @ w.t() / t
    logp = torch.log_softmax(z, 1)
    row = torch.arange(n, device=h.device)
    at = labels.clamp(0, v - 1)
    up = torch.where(used, weights, 0.0)
    p = logp.exp()
    d = p * (up / t).unsqueeze(1)
    # 1 - p of the label from the other classes
    others = torch.logsumexp(logp.scatter(1, at.unsqueeze(1), float("-inf")), 1).exp()
    d[row, at] = -others * up / t
    # -ln p, small ones from 1 - p too
    loss = torch.where(others < 0.5, -torch.log1p(-others), -logp[row, at])
    loss = torch.where(used, loss, 0.0) * up
    return {"loss": loss, "m": z.amax(1) * t, "missing": others, "d_features": d @ w, "d_table": d.t() @ h,
            "z": (h.abs() @ w.abs().t()).amax(1) if n else loss, "x": d.abs() @ w.abs(), "y": d.abs().t() @ h.abs(),
            "d": d}


def spread(scales, rows, dims, block_rows):
    s = scales.float().double()
    s = s.repeat_interleave(block_rows, 0)[:rows]
    return s.repeat_interleave(BLOCK, 1)[:, :dims]


def logits_f8(x, sx, w, sw):
    """(logits, sum of absolute terms)."""
    a = x.float().double() * spread(sx, *x.shape, 1)
    b = w.float().double() * spread(sw, *w.shape, BLOCK)
    return a @ b.t(), a.abs() @ b.abs().t()


GRID = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def quantize(x, block_rows, power):
    """(values as numbers, scales): the nearest e4m3 to the exact quotient, ties to even."""
    x = x.double().cpu()
    n, d = x.shape
    down, across = -(-n // block_rows), -(-d // BLOCK)
    finite = torch.where(x.isfinite(), x, 0.0).abs()
    finite = torch.nn.functional.pad(finite, (0, across * BLOCK - d, 0, down * block_rows - n))
    most = finite.view(down, block_rows, across, BLOCK).amax((1, 3))
    s = (most / 448).float()
    if power:
        m, e = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), e - (m == 0.5).int())
    s = torch.where(most == 0, 1.0, s.clamp_min(2.0 ** -126))
    y = x / spread(s, n, d, block_rows)
    mid = (GRID[1:] + GRID[:-1]) / 2
    at = torch.bucketize(y.abs(), mid)
    at += (y.abs() == mid[at.clamp_max(125)]) & (at % 2 == 1)
    values = torch.copysign(GRID[at.clamp_max(126)], y)
    return torch.where(x.isfinite(), values, float("nan")), s
