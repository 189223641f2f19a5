"""Gradients of rows whose best class has almost all of the probability, against
the 64-bit oracle. Marked gpu.

The best class's gradient is g (1 - p) - h p (ln p + H) over T, both factors as
small as 1 - p. Each is a sum of the other classes' terms: relative errors of
60 u (test_gpu_logits.py), below 3e-5 with the exponents', of
|g| (1 - p) + |h| p (|ln p| + H), and the rounding of the output. The oracle's 1 - p
has 2^-53 / (1 - p) of its own, 1e-7 at the closest here."""
from __future__ import annotations

import numpy as np
import pytest

import logits_oracle as ref
from test_gpu_logits import GRAD_REL, HALF_ULP, check_gradient, dev, host, matrix, ops, upstream  # noqa: F401

pytestmark = pytest.mark.gpu

MISSING = [0.05, 1e-2, 1e-4, 2e-6, 8e-7, 1e-7, 2e-8, 2e-9]
SHAPES = [(8, 2), (8, 16), (8, 30), (8, 250), (8, 1000), (8, 1100), (8, 20011), (8, 140003), (600, 16),
          (600, 1000), (600, 1100), (520, 20011)]


def peaked(n, v, rng, t):
    """Rows of 1 - p about MISSING, the best class anywhere."""
    z = rng.normal(size=(8, v)) * (0.5 if v > 2 else 0.0)
    best = rng.integers(0, v, 8)
    for i, share in enumerate(MISSING):
        rest = np.log(np.exp(np.delete(z[i], best[i]) / t).sum()) * t
        z[i, best[i]] = rest - t * np.log(share)
    z += rng.normal(size=(8, 1))
    return np.tile(z, ((n + 7) // 8, 1))[:n], np.tile(best, (n + 7) // 8)[:n]


def check_best(d, z, tokens, best, g, h, w, t, dtype):
    """The best classes' gradients, and all others by the ordinary bounds. `w`: the sum of
    |upstream| of other classes."""
    n, v = z.shape
    none = np.zeros((n, 0), np.int32)
    want, size = ref.token_logprobs_backward(z, tokens, none, g, h, None, t)
    check_gradient(d, want, size, dtype)
    row = np.arange(n)
    x = (z - z.max(1, keepdims=True)) / t
    e = np.exp(x)
    e[row, best] = 0.0
    rest = e.sum(1)
    p = 1 / (1 + rest)
    entropy = np.log1p(rest) * p + (e * p[:, None] * (np.log1p(rest)[:, None] - x)).sum(1)
    scale = np.abs(g) * rest * p + np.abs(h) * p * (np.log1p(rest) + entropy) + w * p
    got, want = host(d)[row, best], want[row, best]
    rel, step = HALF_ULP[dtype]
    tol = GRAD_REL * scale / t + 1.01 * rel * np.abs(want) + step + 1e-37
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_best_class_of_peaked_rows(ops, shape, dtype):  # noqa: F811
    n, v = shape
    rng = np.random.default_rng(v)
    t = [0.7, 1.0, 2.0][v % 3]
    rows, best = peaked(n, v, rng, t)
    z = matrix(rows, dtype, pad=1)
    some = list(range(8)) + [n - 3]
    tokens = best.copy()
    tok = dev(tokens)
    fwd = ops.token_logprobs(z, tok, top_k=2, temperature=t)
    x = host(z[some])
    best = best[some]
    assert np.array_equal(x.argmax(1), best)
    g, h, _ = upstream(rng, n, 1)
    zero = 0 * g
    for a, b in ((g, zero), (zero, h), (g, h)):
        d = ops.token_logprobs_backward(z, tok, fwd, d_logprob=dev(a), d_entropy=dev(b), temperature=t)
        check_best(d[some], x, tokens[some], best, a[some], b[some], 0.0, t, dtype)
    # the entropy alone, without tokens
    d = ops.token_logprobs_backward(z, None, fwd, d_entropy=dev(h), temperature=t)
    check_best(d[some], x, tokens[some], best, zero[some], h[some], 0.0, t, dtype)
    # the same class as the first alternative; then with a weight of the second's
    for second in (0.0, 1e-3):
        gt = np.stack([g, np.full_like(g, second)], 1)
        d = ops.token_logprobs_backward(z, tok, fwd, d_top_logprobs=dev(gt), temperature=t)
        ids = host(fwd["top_ids"])[some]
        want, size = ref.token_logprobs_backward(x, tokens[some], ids, None, None, gt[some], t)
        check_gradient(d[some], want, size, dtype)
        if second == 0.0:
            check_best(d[some], x, tokens[some], best, g[some], zero[some], 0.0, t, dtype)
    # tokens that are not the best class
    other = dev((tokens + 1) % v)
    d = ops.token_logprobs_backward(z, other, fwd, d_logprob=dev(g), d_entropy=dev(h), temperature=t)
    check_best(d[some], x, (tokens[some] + 1) % v, best, g[some], h[some], np.abs(g[some]), t, dtype)


@pytest.mark.parametrize("shape", [(8, 16), (8, 1000), (8, 1100), (8, 20011), (8, 140003)],
                         ids=lambda s: f"{s[0]}x{s[1]}")
def test_in_place_and_repeated(ops, shape):  # noqa: F811
    """Peaked rows in the logits' own place, the same bits each time."""
    n, v = shape
    rng = np.random.default_rng(v + 1)
    rows, best = peaked(n, v, rng, 1.0)
    z, tok = matrix(rows, "f32"), dev(best)
    fwd = ops.token_logprobs(z, tok, top_k=2)
    g, h, gt = (dev(a) for a in upstream(rng, n, 2))
    apart = ops.token_logprobs_backward(z, tok, fwd, d_logprob=g, d_entropy=h, d_top_logprobs=gt)
    again = ops.token_logprobs_backward(z, tok, fwd, d_logprob=g, d_entropy=h, d_top_logprobs=gt)
    assert (apart == again).all()
    y = matrix(rows, "f32")
    ops.token_logprobs_backward(y, tok, fwd, d_logprob=g, d_entropy=h, d_top_logprobs=gt, out=y)
    assert (apart == y).all()
