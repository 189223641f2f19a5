"""Distillation of rows whose classes are all masked, whatever their teacher
brings: loss and gradient 0, in one call and in two. Marked gpu."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_logits import INF, TYPES, dev, matrix, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(9, 2), (9, 16), (9, 250), (9, 1000), (9, 1100), (9, 20011), (9, 140003),
                                   (600, 16), (600, 700), (600, 1500)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_rows_without_a_class(ops, shape, dtype, kind):  # noqa: F811
    n, v = shape
    k = 12
    rng = np.random.default_rng(v)
    rows = np.full((n, v), -INF)
    rows[4::9] = rng.normal(size=v)          # an ordinary row among them
    ids = rng.integers(0, v, (n, k))
    val = np.full((n, k), -4.0, np.float32)
    ids[0::9] = -1                           # nothing listed
    val[1::9] = -INF                         # listed, without mass
    ids[2::9, 1:] = -1
    val[2::9] = -INF
    ids[3::9, ::2] = -1                      # with mass (and 4, 5)
    ids[6::9, 0] = v                         # an id beyond the classes
    val[7::9, 0] = np.nan
    ids[8::9] = v
    z, did, dval = matrix(rows, dtype, pad=1), dev(ids), dev(val)
    masked = np.arange(n) % 9 != 4
    got = ops.distill(z, did, dval, kind=kind)
    assert not got["loss"].cpu().numpy()[masked].any()
    assert not got["d_logits"].float().cpu().numpy()[masked].any()
    alone = ops.distill(z, did, dval, kind=kind, gradient=False)
    assert not alone["loss"].cpu().numpy()[masked].any()
    for stats in (got["stats"], alone["stats"]):
        back = ops.distill_backward(z, did, dval, stats, dev(np.ones(n, np.float32)), kind=kind)
        assert not back.float().cpu().numpy()[masked].any()
    assert got["loss"][4::9].isfinite().all() and got["d_logits"][4::9].float().abs().sum() > 0
