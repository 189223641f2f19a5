"""Class logits at the ends of their ranges: the most rows, the most classes, split
rows in several launches. Marked gpu."""
from __future__ import annotations

import math

import numpy as np
import pytest

import logits_oracle as ref
from test_gpu_logits import (U, check_forward, check_gradient, check_loss, dev, host, logits_of, matrix,
                             teacher_of, upstream)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_most_rows():
    """2^31 - 1 rows of two classes (8.6 GB): the grid's sum of rows passes 31 bits."""
    from tiny_metal_nn import LogitOps, _lib, logits
    n = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of free device memory")
    z = torch.zeros(n, 2, device="cuda:0", dtype=torch.float16)
    z[-1, 1] = -math.inf
    z[n // 2, 0] = -math.inf
    entropy = torch.full((n,), 7.0, device="cuda:0")
    with LogitOps() as ops:
        packed = logits._PACK_LOGPROBS.pack(
            logits._SIZE_LOGPROBS, _lib.DTYPES["float16"], 0, 0, n, 2, 2, 2, z.data_ptr(), 0, 0,
            entropy.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 1.0, 0)
        _lib.check(ops._lib.tmnn_token_logprobs_device(ops._h, packed,
                                                       torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert float(entropy[-1]) == 0.0 and float(entropy[n // 2]) == 0.0
    entropy[-1] = entropy[n // 2] = entropy[0]
    assert abs(float(entropy[0]) - math.log(2.0)) < 1e-6
    # (in pieces: torch's reductions over more than 2^31 elements are no concern of this test)
    assert all(bool((part == entropy[0]).all()) for part in entropy.split(1 << 28))
    del z, entropy
    torch.cuda.empty_cache()


def same_bits(got, groups):
    """Rows of equal contents have equal results."""
    for name, x in got.items():
        assert torch.equal(x, x[:groups].repeat((len(x) // groups,) + (1,) * (x.dim() - 1))), name


def test_split_rows_in_several_launches():
    """More split rows than the workspace holds at once: 1104 of two parts, 512 a launch, of
    eight kinds whose results must not depend on the launch."""
    from tiny_metal_nn import LogitOps
    n, v, k = 1104, 131080, 5
    rng = np.random.default_rng(1)
    rows = logits_of(rng, 8, v)
    rows[7] += np.where(np.arange(v) == 1234, 30.0, 0.0)  # a peaked one
    z = dev(rows.astype(np.float32)).repeat(n // 8, 1)
    tokens = rng.integers(0, v, 8)
    tokens[7] = 1234
    tok = dev(np.tile(tokens, n // 8))
    x = host(z[:8])
    with LogitOps() as ops:
        fwd = ops.token_logprobs(z, tok, top_k=k)
        check_forward({name: a[:8] for name, a in fwd.items()}, ref.token_logprobs(x, tokens, k, 1.0), k)
        same_bits(fwd, 8)
        g, h, gt = upstream(rng, 8, k)
        d = ops.token_logprobs_backward(z, tok, fwd, d_logprob=dev(np.tile(g, n // 8)),
                                        d_entropy=dev(np.tile(h, n // 8)),
                                        d_top_logprobs=dev(np.tile(gt, (n // 8, 1))))
        want, size = ref.token_logprobs_backward(x, tokens, host(fwd["top_ids"])[:8], g, h, gt, 1.0)
        check_gradient(d[:8], want, size, "f32")
        same_bits({"d_logits": d}, 8)
        del d
        for kind in ("logits", "logprobs"):
            ids, val = teacher_of(rng, x, 20, kind, 1.0)
            did, dval = dev(np.tile(ids, (n // 8, 1))), dev(np.tile(val, (n // 8, 1)))
            loss, dd, loss_size, size = ref.distill(x, ids, val, kind, 1.0)
            out = ops.distill(z, did, dval, kind=kind)
            check_loss(out["loss"][:8], loss, loss_size)
            check_gradient(out["d_logits"][:8], dd, size, "f32")
            same_bits(out, 8)
            alone = ops.distill(z, did, dval, kind=kind, gradient=False)
            assert torch.equal(alone["loss"], out["loss"])
            back = ops.distill_backward(z, did, dval, alone["stats"], torch.ones(n, device="cuda:0"), kind=kind)
            check_gradient(back[:8], dd, size, "f32")
            same_bits({"d_logits": back}, 8)


@pytest.mark.parametrize("shape,dtype", [((1, 2 ** 24), "f16"), ((2, 2 ** 24 - 3), "bf16"),
                                         ((1, 3000017), "f32"), ((3, 262149), "f16")],
                         ids=lambda s: s if isinstance(s, str) else f"{s[0]}x{s[1]}")
def test_most_classes(shape, dtype):
    """Up to 2^24 classes, 128 parts of a row. The entropy's bound with E|x| below 20 here."""
    from tiny_metal_nn import LogitOps
    n, v = shape
    k = 4
    rng = np.random.default_rng(v)
    z = matrix(logits_of(rng, n, v), dtype, pad=1)
    x = host(z)
    tokens = rng.integers(0, v, n)
    tokens[-1] = v - 1
    with LogitOps() as ops:
        fwd = ops.token_logprobs(z, dev(tokens), top_k=k)
        want = ref.token_logprobs(x, tokens, k, 1.0)
        np.testing.assert_allclose(host(fwd["entropy"]), want["entropy"], rtol=0, atol=60 * U * 20)
        fwd_entropy, want["entropy"] = fwd["entropy"], host(fwd["entropy"])
        check_forward(fwd, want, k)
        g, h, gt = upstream(rng, n, k)
        d = ops.token_logprobs_backward(z, dev(tokens), dict(fwd, entropy=fwd_entropy), d_logprob=dev(g),
                                        d_entropy=dev(h), d_top_logprobs=dev(gt))
        check_gradient(d, *ref.token_logprobs_backward(x, tokens, host(fwd["top_ids"]), g, h, gt, 1.0), dtype)
        del d
        ids = np.concatenate([host(fwd["top_ids"]), rng.integers(0, v, (n, 3))], 1).astype(np.int64)
        ids[:, -1] = v - 1
        val = (rng.normal(size=ids.shape) - 3).astype(np.float32)
        for kind in ("logits", "logprobs"):
            loss, dd, loss_size, size = ref.distill(x, ids, val, kind, 1.0)
            out = ops.distill(z, dev(ids), dev(val), kind=kind)
            check_loss(out["loss"], loss, loss_size)
            check_gradient(out["d_logits"], dd, size, dtype)
