"""The loss of students that are near a flat teacher, where the logarithms of the two
rests nearly cancel. Marked gpu.

loss = T^2 [sum q_j (ln q_j - ln p_j) + q_r (ln q_r - ln p_r)]. The listed terms have the
errors of test_gpu_logits.py's check_loss, 130 u of q_j (|ln q_j| + |ln p_j| + 1). The rest's
logarithms are of shares near 1, and taken from what is missing to 1, a few sums of
relative error 60 u each: 130 u of q_r (|ln q_r| + |ln p_r|) for both, with nothing
added for the 1. Logarithms of the sums themselves would be off by u ln(classes) each,
a hundred times these bounds at 90000 classes."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_logits import U, dev, host, matrix, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1.0, 2.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(9, 300), (9, 1000), (600, 5003), (9, 40000), (575, 93665), (3, 200001)],
                         ids=lambda s: f"{s[0]}x{s[1]}")
def test_flat_teachers(ops, shape, dtype, t):  # noqa: F811
    n, v = shape
    rng = np.random.default_rng(v)
    z = matrix(rng.normal(size=(9, v))[np.arange(n) % 9] * 0.1, dtype, pad=1)
    some = np.arange(min(n, 9))
    x = host(z[: some.size])
    y = x / t + rng.normal(size=x.shape) * 0.05
    logq = y - y.max(1, keepdims=True)
    logq -= np.log(np.exp(logq).sum(1, keepdims=True))
    ids = np.argsort(-y, axis=1)[:, :3]
    val = np.take_along_axis(logq, ids, 1).astype(np.float32)
    rows = np.arange(n) % 9
    got = host(ops.distill(z, dev(ids[rows]), dev(val[rows]), kind="logprobs", temperature=t)["loss"])
    for i in some:
        lp = x[i] / t - (x[i] / t).max()
        log_sum = np.log(np.exp(lp).sum())
        a = val[i].astype(np.float64)
        q, mine = np.exp(a), lp[ids[i]] - log_sum
        # the rests' logarithms from what is missing, in 64 bits
        log_qr, log_pr = np.log1p(-q.sum()), np.log1p(-np.exp(mine).sum())
        qr = 1 - q.sum()
        want = t * t * ((q * (a - mine)).sum() + qr * (log_qr - log_pr))
        size = (q * (np.abs(a) + np.abs(mine) + 1)).sum() + qr * (abs(log_qr) + abs(log_pr))
        assert abs(got[i] - want) <= 130 * U * t * t * size, (i, got[i], want, abs(got[i] - want) / size / U)
    assert np.array_equal(got, got[rows])
