"""LogitOps beside torch's autograd: results without history, and writes that
autograd knows of. Marked gpu."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

N, V, K = 5, 33, 3


def test_results_have_no_history_and_writes_are_known():
    from tiny_metal_nn import LogitOps
    g = torch.Generator(device="cuda:0").manual_seed(1)
    w = torch.randn(8, V, device="cuda:0", generator=g, requires_grad=True)
    x = torch.randn(N, 8, device="cuda:0", generator=g)
    tokens = torch.randint(0, V, (N,), device="cuda:0", generator=g)
    ids = torch.randint(0, V, (N, K), device="cuda:0", generator=g)
    val = torch.randn(N, K, device="cuda:0", generator=g)
    ones = torch.ones(N, device="cuda:0")
    f32 = {"device": "cuda:0", "dtype": torch.float32}
    i32 = {"device": "cuda:0", "dtype": torch.int32}
    with LogitOps() as ops:
        logits = x @ w
        out = {"logprob": torch.empty(N, **f32), "entropy": torch.empty(N, **f32),
               "rank": torch.empty(N, **i32), "stats": torch.empty(N, 2, **f32),
               "top_ids": torch.empty(N, K, **i32), "top_logprobs": torch.empty(N, K, **f32)}
        before = {name: t._version for name, t in out.items()}
        fwd = ops.token_logprobs(logits, tokens, top_k=K, out=out)
        assert not any(t.requires_grad for t in fwd.values())
        assert all(t._version > before[name] for name, t in out.items())
        version = logits._version
        d = ops.token_logprobs_backward(logits, tokens, fwd, d_logprob=ones, d_entropy=ones)
        assert logits._version == version and not d.requires_grad  # only read
        # the gradient goes on by logits.backward, also from the logits' own place
        logits.backward(d)
        apart, w.grad = w.grad, None
        logits = x @ w
        same = ops.token_logprobs_backward(logits, tokens, fwd, d_logprob=ones, d_entropy=ones,
                                           out=logits.detach())
        logits.backward(same)
        assert torch.equal(w.grad, apart)
        w.grad = None
        # an operation that saved the logits finds them changed
        for write in (
                lambda z: ops.token_logprobs_backward(z, tokens, fwd, d_logprob=ones, out=z),
                lambda z: ops.distill(z, ids, val, out={"d_logits": z}),
                lambda z: ops.distill_backward(z, ids, val, torch.zeros(N, 4, **f32), ones, out=z)):
            logits = x @ w
            squares = (logits * logits).sum()
            write(logits.detach())
            with pytest.raises(RuntimeError, match="inplace"):
                squares.backward()
        o = {"loss": torch.empty(N, **f32), "stats": torch.empty(N, 4, **f32)}
        before = {name: t._version for name, t in o.items()}
        ops.distill(x @ w, ids, val, gradient=False, out=o)
        assert all(t._version > before[name] for name, t in o.items())
        # in inference mode, and tensors of it
        with torch.inference_mode():
            z = x @ w
            got = ops.token_logprobs(z, tokens, top_k=K)
            ops.token_logprobs(z, tokens, top_k=K, out=got)
        ops.token_logprobs(z, tokens, top_k=K, out=got)
        assert torch.equal(got["top_ids"], fwd["top_ids"])
