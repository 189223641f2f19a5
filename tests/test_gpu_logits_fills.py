"""Class logits with finite mask fills of any size, at temperatures down to the
smallest: every kernel against the 64-bit oracle. Marked gpu.

The tolerances are those of test_gpu_logits.py: a masked class adds a term that is 0
in 32 bits, and the classes of a row that holds the fill alone differ by nothing."""
from __future__ import annotations

import numpy as np
import pytest

import logits_oracle as ref
from test_gpu_logits import (check_forward, check_gradient, check_loss, dev, host, matrix, ops,  # noqa: F401
                             teacher_of, upstream)

pytestmark = pytest.mark.gpu

# fp16's lowest value is only huge against a small temperature
FILLS = [("f32", -1e9, 1.0), ("f32", -1e10, 1.0), ("f32", -1e10, 2.0), ("f32", -1e12, 0.7),
         ("f32", -1e20, 0.7), ("f32", -1e30, 1.0), ("f32", -1e4, 1e-6), ("bf16", -1e10, 1.0),
         ("bf16", -1e12, 2.0), ("bf16", -1e20, 2.0), ("bf16", -1e30, 0.7), ("f16", -6e4, 1e-6),
         ("f16", -1e4, 1e-5)]
# a block a row of one and of more waves, split rows; many rows of each
SHAPES = [(10, 16), (10, 900), (10, 1100), (10, 20011), (10, 140003), (600, 1100), (520, 20011)]


def filled(n, v, fill, rng):
    rows = rng.normal(size=(10, v)) * 2
    at = np.arange(v)
    rows[0] = fill                           # nothing else
    rows[1, ::2] = fill                      # every other class
    rows[2, :(v + 1) // 2] = fill            # the first half: whole threads, tiles and parts
    rows[3, v // 2:] = fill                  # the second half
    rows[4, at != v // 2] = fill             # all but one
    rows[5, :-1] = fill                      # all but the last
    rows[6, rng.random(v) < 0.9] = fill
    rows[7, at // 96 % 2 == 0] = fill        # runs
    rows[8, v // 3] = -fill                  # as far above the rest
    return np.tile(rows, ((n + 9) // 10, 1))[:n]


def params():
    for shape in SHAPES:
        for dtype, fill, t in FILLS:
            yield pytest.param(shape, dtype, fill, float(np.float32(t)),
                               id=f"{shape[0]}x{shape[1]}-{dtype}{fill:g}-{t:g}")


@pytest.mark.parametrize("shape,dtype,fill,t", params())
def test_finite_fills(ops, shape, dtype, fill, t):  # noqa: F811
    n, v = shape
    rng = np.random.default_rng(v)
    z = matrix(filled(n, v, fill, rng), dtype, pad=1)
    some = list(range(10)) + [n - 3] * (n > 10)  # (the others repeat them)
    tokens = rng.integers(0, v, n)
    tok, k = dev(tokens), 4
    got = ops.token_logprobs(z, tok, top_k=k, temperature=t)
    x = host(z[some])
    want = ref.token_logprobs(x, tokens[some], k, t)
    check_forward({name: a[some] for name, a in got.items()}, want, k)

    # (the gradient is 1 / T of what comes from above, and has to fit its type)
    g, h, gt = (np.float32(min(t, 1.0)) * a for a in upstream(rng, n, k))
    d = ops.token_logprobs_backward(z, tok, got, d_logprob=dev(g), d_entropy=dev(h),
                                    d_top_logprobs=dev(gt), temperature=t)
    want, size = ref.token_logprobs_backward(x, tokens[some], host(got["top_ids"])[some], g[some], h[some],
                                             gt[some], t)
    check_gradient(d[some], want, size, dtype)

    # A teacher of ordinary values, whose classes the student has masked in part. Relative to
    # row 8's maximum, 64 bits hold less of its other classes' shares of the rest than the
    # kernels, which take them relative to the rest's own.
    fit = np.arange(len(some)) != 8
    plain = rng.normal(size=(len(some), v)) * 2
    for kind in ("logits", "logprobs"):
        ids, val = teacher_of(rng, plain, 8, kind, t if t > 0.1 else 1.0, dup=False)
        if t < 0.1 and kind == "logits":
            val *= np.float32(t)  # its softmax at t is that of plain values
        full = np.zeros((n, 8), np.int64), np.zeros((n, 8), np.float32)
        full[0][some], full[1][some] = ids, val
        loss, dd, loss_size, size = ref.distill(x, ids, val, kind, t)
        both = ops.distill(z, dev(full[0]), dev(full[1]), kind=kind, temperature=t)
        at = dev(np.array(some)[fit])
        check_loss(both["loss"][at], loss[fit], loss_size[fit])
        check_gradient(both["d_logits"][at], dd[fit], size[fit], dtype)
        back = ops.distill_backward(z, dev(full[0]), dev(full[1]), both["stats"], dev(np.ones(n, np.float32)),
                                    kind=kind, temperature=t)
        check_gradient(back[at], dd[fit], size[fit], dtype)
        assert both["loss"].isfinite().all() and both["d_logits"].isfinite().all() and back.isfinite().all()
