"""Gradients that would lie over logits that are still to be read are refused; rows
that only interleave with them, and the logits' own place, are not. Marked gpu."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

N, V = 6, 40


def calls(ops, z, tokens, ids, val):
    """The three calls that write d_logits, as functions of the place."""
    ones = torch.ones(N, device="cuda:0")
    fwd = ops.token_logprobs(z, tokens)
    stats = ops.distill(z, ids, val, gradient=False)["stats"]
    return [lambda d: ops.token_logprobs_backward(z, tokens, fwd, d_logprob=ones, d_entropy=ones, out=d),
            lambda d: ops.distill(z, ids, val, out={"d_logits": d})["d_logits"],
            lambda d: ops.distill_backward(z, ids, val, stats, ones, out=d)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_overlapping_gradients(dtype):
    from tiny_metal_nn import LogitOps
    g = torch.Generator(device="cuda:0").manual_seed(1)
    tokens = torch.randint(0, V, (N,), device="cuda:0", generator=g)
    ids = torch.randint(0, V, (N, 3), device="cuda:0", generator=g)
    val = torch.randn(N, 3, device="cuda:0", generator=g)
    values = torch.randn(N, V, device="cuda:0", generator=g).to(dtype)

    def view(buf, at, stride):
        return buf[at:].as_strided((N, V), (stride, 1), storage_offset=at)

    with LogitOps() as ops:
        want = [call(None) for call in calls(ops, values, tokens, ids, val)]
        buf = torch.zeros(48 * V, device="cuda:0", dtype=dtype)
        stride, at = 2 * V + 4, 16 * V
        for i, (shift, d_stride, fine) in enumerate([
                (0, stride, True),                    # the logits' place
                (1, stride, False), (-1, stride, False), (V - 1, stride, False), (1 - V, stride, False),
                (V, stride, True), (-V, stride, True), (V + 4, stride, True), (V + 5, stride, False),
                (3 * stride, stride, False), (3 * stride + V, stride, True), (-2 * stride - V, stride, True),
                (N * stride, stride, True), (-N * stride, stride, True), ((N - 1) * stride, stride, False),
                (V, 2 * stride, True), (V, stride + 3, False), (-V, V, False), (-N * V, V, True),
                ((N - 1) * stride + V, V, True), ((N - 1) * stride + V - 1, V, False)]):
            for k in range(3):
                buf.zero_()
                z = view(buf, at, stride)
                z.copy_(values)
                call = calls(ops, z, tokens, ids, val)[k]
                d = view(buf, at + shift, d_stride)
                if fine:
                    assert torch.equal(call(d), want[k]), (i, k)
                    assert shift == 0 or torch.equal(z, values), (i, k)
                else:
                    with pytest.raises(ValueError, match="overlaps"):
                        call(d)
                    assert torch.equal(z, values), (i, k)
