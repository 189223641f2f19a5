"""A field that learns labels from a teacher's top logits, then answers with
probabilities: the trainer's own-loss path (forward_for_training,
backward_accumulate, adam_step) around LogitOps.distill, and
LogitOps.token_logprobs over the trained field's outputs.

The teacher labels the unit cube by 16 sites: its logits at a point fall with the
squared distance to each site, and only its best four are kept, as a label store
would. Run: python examples/semantic_field.py [steps]
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "tiny-metal-nn_amd"))

from tiny_metal_nn import LogitOps, Trainer  # noqa: E402

CLASSES, KEPT, BATCH, TEMPERATURE = 16, 4, 4096, 2.0


def teacher_top(points: np.ndarray, sites: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """The teacher's best classes at each point and their logits."""
    d = ((points[:, None, :] - sites[None, :, :]) ** 2).sum(-1)
    ids = np.argsort(d, axis=1, kind="stable")[:, :KEPT].astype(np.int32)
    return ids, (-40.0 * np.take_along_axis(d, ids, 1)).astype(np.float32)


def main(steps: int = 200, seed: int = 0) -> dict:
    rng = np.random.default_rng(seed)
    sites = rng.random((CLASSES, 3), dtype=np.float32)
    config = {"encoding": {"n_levels": 8, "n_features_per_level": 2, "log2_hashmap_size": 14,
                           "base_resolution": 4.0, "per_level_scale": 1.5},
              "network": {"n_neurons": 64, "n_hidden_layers": 2},
              "optimizer": {"otype": "Adam", "learning_rate": 1e-2}, "batch_size": BATCH}
    weights = np.full(BATCH, 1.0 / BATCH, np.float32)
    with Trainer.from_config(config, n_input=3, n_output=CLASSES) as field, LogitOps() as ops:
        losses = []
        for _ in range(steps):
            points = rng.random((BATCH, 3), dtype=np.float32)
            ids, values = teacher_top(points, sites)
            logits = field.forward_for_training(points)
            out = ops.distill(logits, ids, values, temperature=TEMPERATURE, row_weights=weights)
            field.zero_gradients()
            field.backward_accumulate(points, out["d_logits"])
            field.adam_step()
            losses.append(float(out["loss"].sum()))
        points = rng.random((BATCH, 3), dtype=np.float32)
        labels = teacher_top(points, sites)[0][:, 0].copy()
        answer = ops.token_logprobs(field.inference(points), labels, top_k=3)
    return {"first_loss": losses[0], "last_loss": losses[-1],
            "accuracy": float((answer["rank"] == 0).mean()),
            "in_top_3": float((answer["top_ids"] == labels[:, None]).any(1).mean()),
            "mean_logprob": float(answer["logprob"].mean()),
            "mean_entropy": float(answer["entropy"].mean())}


if __name__ == "__main__":
    for name, value in main(int(sys.argv[1]) if len(sys.argv) > 1 else 200).items():
        print(f"{name} {value:.4f}")
