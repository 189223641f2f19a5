"""The class head's operators together, as they are used: the example runs, a step's
gradients are the formula's and go through a field's backward pass as differences of
the loss do, and 8-bit logits give the answers that 64-bit products of the same values give.
Marked gpu."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import head_oracle as ref  # noqa: E402
from test_gpu_class_loss import ops  # noqa: E402,F401

EXAMPLE = Path(__file__).resolve().parent.parent / "examples" / "open_vocabulary_field.py"


def test_the_example_runs():
    spec = importlib.util.spec_from_file_location("open_vocabulary_field", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.main(steps=5)
    assert all(np.isfinite(v) for v in got.values()), got
    assert got["in_top_3"] >= got["accuracy"] >= 0.0


def test_a_step_together(ops):
    from tiny_metal_nn import Trainer
    rng = np.random.default_rng(1)
    n, v = 256, 300
    config = {"encoding": {"n_levels": 4, "n_features_per_level": 2, "log2_hashmap_size": 10, "base_resolution": 4.0,
                           "per_level_scale": 1.5},
              "network": {"n_neurons": 32, "n_hidden_layers": 2}, "batch_size": n}
    points = rng.random((n, 3), dtype=np.float32)
    table = rng.normal(size=(v, 16)).astype(np.float32)
    labels = rng.integers(0, v, n)
    weights = np.full(n, 1.0 / n, np.float32)
    with Trainer.from_config(config, n_input=3, n_output=16) as field:
        features = field.forward_for_training(points)
        out = ops.class_loss(features, table, labels, row_weights=weights, temperature=0.5)
        want = ref.class_loss(torch.as_tensor(features), torch.as_tensor(table), torch.as_tensor(labels),
                              torch.as_tensor(weights), 0.5)
        for name in ("loss", "d_features", "d_table"):
            scale = want[name].abs().max()
            assert (torch.as_tensor(out[name]).double() - want[name]).abs().max() <= 1e-4 * scale, name  # (3e-5 p, 2^-20)
        field.zero_gradients()
        field.backward_accumulate(points, out["d_features"])
        _, grad = field.debug_gradients()
        hash_w, mlp = field.get_weights()
        # along the gradient: a difference of the loss is its squared length (to the curvature's share of the step)
        def total(w):
            field.set_initial_weights(hash_w, w.astype(np.float32))
            x = field.forward_for_training(points)
            return float(ref.class_loss(torch.as_tensor(x), torch.as_tensor(table), torch.as_tensor(labels),
                                        torch.as_tensor(weights), 0.5)["loss"].sum())
        length = float((grad.astype(np.float64) ** 2).sum())
        step = 1e-3 / np.sqrt(length)
        slope = (total(mlp + step * grad) - total(mlp - step * grad)) / (2 * step)
        # central differences of step 1e-3 along a unit direction: fp32 forward passes (1e-6 of a loss near ln 300 over
        # 2e-3) and a third derivative's 1e-6
        assert abs(slope - length) <= 2e-2 * length + 3e-3 * np.sqrt(length)
    rows, classes = ops.quantize_f8(features), ops.quantize_f8(table, block_rows=128)
    logits = ops.class_logits_f8(rows["values"], rows["scales"], classes["values"], classes["scales"])

    def f8(q):
        return torch.as_tensor(q).view(torch.float8_e4m3fn)
    exact, _ = ref.logits_f8(f8(rows["values"]), torch.as_tensor(rows["scales"]), f8(classes["values"]),
                             torch.as_tensor(classes["scales"]))
    answer = ops.token_logprobs(logits, labels, top_k=1)
    best = exact.argmax(1).numpy()
    at = np.arange(n)
    close = exact.numpy()[at, best] - exact.numpy()[at, answer["top_ids"][:, 0]]
    assert (close <= 1e-4 * np.abs(exact.numpy()).max(1)).all()
