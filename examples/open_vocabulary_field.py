"""A field whose 16 outputs are features, compared with a table of labels: it learns
the labels of a scene and the table together with LogitOps.class_loss (which needs no
tensor of logits), then answers from features and a table in 8 bits with
LogitOps.class_logits_f8 and LogitOps.token_logprobs.

The scene labels the unit cube by 500 sites, each point by its nearest. Run:
python examples/open_vocabulary_field.py [steps]
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "tiny-metal-nn_amd"))

from tiny_metal_nn import LogitOps, Trainer  # noqa: E402

LABELS, DIMS, BATCH, TEMPERATURE = 500, 16, 4096, 0.5


def labels_of(points: np.ndarray, sites: np.ndarray) -> np.ndarray:
    d = (sites * sites).sum(1) - 2.0 * points @ sites.T
    return d.argmin(1).astype(np.int32)


def main(steps: int = 200, seed: int = 0) -> dict:
    rng = np.random.default_rng(seed)
    sites = rng.random((LABELS, 3), dtype=np.float32)
    table = rng.normal(size=(LABELS, DIMS)).astype(np.float32)
    config = {"encoding": {"n_levels": 8, "n_features_per_level": 2, "log2_hashmap_size": 14,
                           "base_resolution": 4.0, "per_level_scale": 1.5},
              "network": {"n_neurons": 64, "n_hidden_layers": 2},
              "optimizer": {"otype": "Adam", "learning_rate": 1e-2}, "batch_size": BATCH}
    weights = np.full(BATCH, 1.0 / BATCH, np.float32)
    with Trainer.from_config(config, n_input=3, n_output=DIMS) as field, LogitOps() as ops:
        losses = []
        for _ in range(steps):
            points = rng.random((BATCH, 3), dtype=np.float32)
            features = field.forward_for_training(points)
            out = ops.class_loss(features, table, labels_of(points, sites), row_weights=weights,
                                 temperature=TEMPERATURE)
            field.zero_gradients()
            field.backward_accumulate(points, out["d_features"])
            field.adam_step()
            table -= 2.0 * out["d_table"]
            losses.append(float(out["loss"].sum()))
        points = rng.random((BATCH, 3), dtype=np.float32)
        labels = labels_of(points, sites)
        features = field.inference(points)
        rows = ops.quantize_f8(features)
        classes = ops.quantize_f8(table, block_rows=128)
        logits = ops.class_logits_f8(rows["values"], rows["scales"], classes["values"], classes["scales"])
        answer = ops.token_logprobs(logits, labels, top_k=3, temperature=TEMPERATURE)
    return {"first_loss": losses[0], "last_loss": losses[-1],
            "accuracy": float((answer["rank"] == 0).mean()),
            "in_top_3": float((answer["top_ids"] == labels[:, None]).any(1).mean()),
            "off_by_8_bits": float(np.abs(logits - features @ table.T).max() / np.abs(logits).max()),
            "mean_logprob": float(answer["logprob"].mean())}


if __name__ == "__main__":
    for name, value in main(int(sys.argv[1]) if len(sys.argv) > 1 else 200).items():
        print(f"{name} {value:.4f}")
