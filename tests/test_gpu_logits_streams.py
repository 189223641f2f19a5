"""A logits handle whose workspace moves between streams that are captured or
destroyed meanwhile. Marked gpu."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import logits_oracle as ref
from test_gpu_logits import check_forward, dev, host, logits_of, matrix

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

N, V, K = 3, 60000, 6  # few long rows: split, so that they share the workspace


def test_calls_while_the_last_stream_is_captured():
    """Warmed up on a stream that another handle's graph then captures: a call on a third stream,
    which would have to wait for the captured one, is refused and does not become part of
    the graph. Afterwards the handle goes on."""
    from tiny_metal_nn import LogitOps
    from tiny_metal_nn._lib import TmnnError
    rng = np.random.default_rng(1)
    z, y = (matrix(logits_of(rng, N, V), "f32") for _ in range(2))
    want = ref.token_logprobs(host(y), None, K, 1.0)
    ones = dev(np.ones(N, np.float32))
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    with LogitOps() as warm, LogitOps() as mine:
        out, other, d = {}, {}, torch.empty_like(y)
        with torch.cuda.stream(t):
            fwd = warm.token_logprobs(y, None, top_k=K)
            warm.token_logprobs(y, None, top_k=K, out=other)
        with torch.cuda.stream(s):
            mine.token_logprobs(z, None, top_k=K, out=out)
            warm.token_logprobs(z, None, top_k=K, out=out)  # `warm` was last on s
        torch.cuda.synchronize()
        for x in (*other.values(), d):
            x.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            mine.token_logprobs(z, None, top_k=K, out=out)
            with pytest.raises(TmnnError, match="captured"):
                warm.token_logprobs(y, None, top_k=K, out=other, stream=t)
            with pytest.raises(TmnnError, match="captured"):
                warm.token_logprobs_backward(y, None, fwd, d_entropy=ones, out=d, stream=t)
        torch.cuda.synchronize()
        for _ in range(3):
            for x in out.values():
                x.zero_()
            z.copy_(torch.as_tensor(logits_of(rng, N, V)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            check_forward(out, ref.token_logprobs(host(z), None, K, 1.0), K)
            assert not any(x.any() for x in other.values()) and not d.any()
            # eager calls between the replays, on both streams
            with torch.cuda.stream(t):
                got = warm.token_logprobs(y, None, top_k=K)
            with torch.cuda.stream(s):
                again = warm.token_logprobs(y, None, top_k=K)
            torch.cuda.synchronize()
            check_forward(got, want, K)
            assert all(torch.equal(got[key], again[key]) for key in got)


def test_the_last_stream_is_destroyed():
    """Neither the next call nor the end of the handle needs the stream of the last one."""
    from tiny_metal_nn import LogitOps
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    hip = ctypes.CDLL(path)
    rng = np.random.default_rng(2)
    z = matrix(logits_of(rng, N, V), "bf16")
    want = ref.token_logprobs(host(z), None, K, 1.0)
    torch.cuda.synchronize()
    ops = LogitOps()
    out = {}
    ops.token_logprobs(z, None, top_k=K, out=out)
    torch.cuda.synchronize()
    for _ in range(3):
        s = ctypes.c_void_p()
        assert hip.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0  # (non-blocking)
        for x in out.values():
            x.zero_()
        torch.cuda.synchronize()
        ops.token_logprobs(z, None, top_k=K, out=out, stream=s.value)
        assert hip.hipStreamSynchronize(s) == 0
        assert hip.hipStreamDestroy(s) == 0
        check_forward(out, want, K)
    check_forward(ops.token_logprobs(z, None, top_k=K), want, K)
    s = ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0
    ops.token_logprobs(z, None, top_k=K, out=out, stream=s.value)
    assert hip.hipStreamSynchronize(s) == 0
    assert hip.hipStreamDestroy(s) == 0
    ops.close()
    check_forward(out, want, K)
