"""How small a probability the class head's gradients hold, as include/tmnn_hip.h states it: 39 + log2 p bits, at most
11 (bf16) or 22 (fp32), and nothing below 2^-39. Marked gpu."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_class_loss import DEV, TYPES, ops  # noqa: E402,F401


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [8, 136])
def test_gradients_of_unlikely_classes(ops, d, dtype):
    """One row of features (1, 0, ..), so that a class's row of d_table is (p, 0, ..); logits of 0 and of -1 / 4 to -32
    in steps that bf16 holds."""
    z = torch.cat([torch.zeros(1), -torch.arange(1, 129) / 4.0]).double()
    h = torch.zeros(1, d, device=DEV, dtype=TYPES[dtype])
    h[0, 0] = 1.0
    w = torch.zeros(len(z), d, device=DEV, dtype=TYPES[dtype])
    w[:, 0] = z.to(DEV)
    assert torch.equal(w[:, 0].double().cpu(), z)
    got = ops.class_loss(h, w, torch.zeros(1, dtype=torch.int64, device=DEV))["d_table"].double().cpu()
    p = torch.softmax(z, 0)[1:]
    # the exponential and the sum (3e-5 as in test_gpu_class_loss.py), d's rounding: half a unit of its last place, which ends at
    # 2^-24 - 14, the table's own type
    out = 2.0 ** -24 if dtype == "f32" else 2.0 ** -8
    terms = 2.0 ** -11 if dtype == "bf16" else 2.0 ** -21
    err = p * (3e-5 + terms) + 2.0 ** -39
    err = err + out * (p + err)
    assert ((got[1:, 0] - p).abs() <= err).all(), ((got[1:, 0] - p).abs() / err).max()
    assert not got[1:, 0][p < 2.0 ** -39.1].any() and not got[:, 1:].any()
    # what the other classes leave of the label's
    assert abs(got[0, 0] + p.sum()) <= p.sum() * (3e-5 + terms + out)
