"""Class logits at the ends of their ranges: the most rows, the most classes, split
rows in several launches. Marked gpu."""
from __future__ import annotations

import math

import pytest

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
