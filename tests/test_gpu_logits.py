"""The class-logit operators on the GPU against the 64-bit oracle
(logits_oracle.py). Marked gpu.

Tolerances, with u = 2^-24 (half an ulp of fp32). A log-probability is
c (z - m) ln 2 - ln S: four roundings of the first term (4 u |ln p|), and a
relative error of S, which holds that of each exponent (its terms weigh
e^-|x| (2 u |x| + 2 u) < 3 u), of the sums (at most about 30 additions in
sequence on these sizes) and of the logarithm: below 60 u together. The entropy
adds E[|x|] (< 13 here) of the same relative error; a probability in a gradient has
e^(4 u |x| + 60 u) of it, |x| < 60 where it is not far below the type's
smallest number: 3e-5, relative to the sum of the absolute terms. 16-bit
gradients round once: half an ulp of their type."""
from __future__ import annotations

import numpy as np
import pytest

import logits_oracle as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
LOGP_ABS, LOGP_REL, ENTROPY_ABS, SUM_REL = 60 * U, 8 * U, 60 * U * 13, 60 * U
GRAD_REL = 3e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half an ulp, and half of the smallest step between numbers, of each type
HALF_ULP = {"f32": (2.0 ** -24, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}
INF = float("inf")


@pytest.fixture(scope="module")
def ops():
    from tiny_metal_nn import LogitOps
    with LogitOps() as o:
        yield o


def matrix(values, dtype, pad=0, offset=0):
    """A device matrix with `pad` elements between rows, its data `offset`
    elements into the allocation."""
    n, v = values.shape
    buf = torch.full((offset + n * (v + pad) + 8,), 7.0, device="cuda:0", dtype=TYPES[dtype])
    z = buf[offset:offset + n * (v + pad)].view(n, v + pad)[:, :v]
    z.copy_(torch.as_tensor(values))
    return z


def host(x):
    return x.detach().double().cpu().numpy() if x.is_floating_point() else x.cpu().numpy()


def logits_of(rng, n, v, scale=2.0):
    z = rng.normal(size=(n, v)) * scale
    if v >= 8:  # a few far above, and ties
        z[np.arange(n), rng.integers(0, v, n)] += 4 * scale
        z = np.where(rng.random((n, v)) < 0.25, np.round(z), z)
    return z


def check_forward(got, want, k):
    lp = want["logprob"]
    np.testing.assert_allclose(host(got["logprob"]), lp, rtol=LOGP_REL, atol=LOGP_ABS)
    np.testing.assert_allclose(host(got["entropy"]), want["entropy"], rtol=0, atol=ENTROPY_ABS)
    assert np.array_equal(host(got["rank"]), want["rank"])
    s = want["stats"]
    bad = np.isnan(s[:, 1])
    np.testing.assert_allclose(host(got["stats"])[~bad], s[~bad], rtol=SUM_REL, atol=0)
    assert np.isnan(host(got["stats"])[bad, 1]).all()
    if k:
        assert np.array_equal(host(got["top_ids"]), want["top_ids"])
        np.testing.assert_allclose(host(got["top_logprobs"]), want["top_logprobs"], rtol=LOGP_REL,
                                   atol=LOGP_ABS)


# one lane to 64 lanes a row, one block, several blocks; odd counts beside each bound
SHAPES = [(1, 1), (3, 2), (5, 3), (70, 4), (64, 16), (9, 17), (6, 64), (5, 129), (3, 256), (3, 257),
          (2, 512), (3, 513), (2, 1000), (600, 1031), (3, 4096), (2, 5003), (513, 2049), (1, 32768),
          (2, 50021), (1, 131072), (1, 262147)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_forward(ops, shape, dtype):
    n, v = shape
    rng = np.random.default_rng(n * 1000003 + v)
    t = float(rng.choice([0.7, 1.0, 2.0]))
    k = int(rng.choice([1, 3, 8, 20]))
    z = matrix(logits_of(rng, n, v), dtype, pad=int(rng.integers(0, 4)), offset=int(rng.integers(0, 3)))
    tokens = rng.integers(0, v, n)
    if n > 2:
        tokens[1] = -1
    index = torch.int32 if v % 2 else torch.int64
    got = ops.token_logprobs(z, torch.as_tensor(tokens, device="cuda:0").to(index), top_k=k,
                             temperature=t)
    check_forward(got, ref.token_logprobs(host(z), tokens, k, t), k)


@pytest.mark.parametrize("k", [2, 64, 65, 128])
@pytest.mark.parametrize("shape", [(2, 100), (2, 300), (2, 700), (520, 3000), (3, 40000)],
                         ids=lambda s: f"{s[0]}x{s[1]}")
def test_many_alternatives(ops, shape, k):
    n, v = shape
    rng = np.random.default_rng(v + k)
    z = matrix(logits_of(rng, n, v), "bf16")
    got = ops.token_logprobs(z, None, top_k=k)
    check_forward(got, ref.token_logprobs(host(z), None, k, 1.0), k)


# the order of equal logits, and rows whose best classes sit where one thread reads
@pytest.mark.parametrize("v", [16, 300, 1030, 9000, 70001])
@pytest.mark.parametrize("rows", ["few", "many"])
def test_alternatives_of_unusual_orders(ops, v, rows):
    base = np.arange(v, dtype=np.float64)
    rng = np.random.default_rng(v)
    z = [np.zeros(v), base / v, -base / v, np.where(base % 2 == 0, 1.0, 0.0),
         np.where(rng.random(v) < 0.5, -0.0, 0.0)]
    for stride in (1024, 2048, 4096, 8192):  # the best ones a block's tile apart
        z.append(np.where(base % stride < 4, 8.0 - (base % 4) / 4, 0.0))
    z.append(np.where(base % 8192 < 64, 5.0, rng.normal(size=v)))
    z = np.array(z)
    if rows == "many":
        if v > 9000:
            pytest.skip("few rows cover it")
        z = np.tile(z, (53, 1))
    x = matrix(z, "f32")
    for k in (5, 128):
        got = ops.token_logprobs(x, None, top_k=k)
        want = ref.token_logprobs(host(x)[:10], None, k, 1.0)
        assert np.array_equal(host(got["top_ids"])[:10], want["top_ids"])
        assert np.array_equal(host(got["top_ids"])[-10:], want["top_ids"])
        np.testing.assert_allclose(host(got["top_logprobs"])[:10], want["top_logprobs"],
                                   rtol=LOGP_REL, atol=LOGP_ABS)


def edge_rows(v, dtype, rng):
    low = float(torch.finfo(TYPES[dtype]).min)
    rows = np.tile(rng.normal(size=v), (12, 1))
    rows[0] = -INF                         # nothing left
    rows[1] = low                          # the type's lowest value everywhere
    rows[2, ::2] = low                     # and as a mask
    rows[3] = -INF
    rows[3, v // 2] = -3.0                 # one class left
    rows[4, rng.random(v) < 0.9] = -INF
    rows[5, v // 3] = np.nan
    rows[6, v // 3] = INF
    rows[7] = -INF
    rows[7, v // 2] = low                  # one class left, of the lowest value
    rows[8] = -INF
    rows[8, 0] = np.nan
    rows[9, v // 2] = -low                 # the largest finite value
    rows[10] = np.where(np.arange(v) % 2, low, -INF)
    rows[11, : (v + 1) // 2] = -INF
    return rows


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("v", [2, 16, 250, 1500, 20011])
@pytest.mark.parametrize("many", [False, True])
def test_edge_rows_forward(ops, v, dtype, many):
    rng = np.random.default_rng(v)
    rows = edge_rows(v, dtype, rng)
    if many:
        if v > 1500:
            pytest.skip("few rows cover it")
        rows = np.tile(rows, (44, 1))
    z = matrix(rows, dtype, pad=1)
    tokens = rng.integers(0, v, len(rows))
    tokens[0::24] = v // 2
    tokens[4] = v  # beyond the classes
    got = ops.token_logprobs(z, torch.as_tensor(tokens, device="cuda:0"), top_k=4)
    check_forward(got, ref.token_logprobs(host(z), tokens, 4, 1.0), 4)


def check_gradient(got, want, size, dtype):
    got = host(got)
    rel, step = HALF_ULP[dtype]
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad)
    tol = GRAD_REL * size + 1.01 * rel * np.abs(want) + step + 1e-37
    worst = (np.abs(got - want) / tol)[~bad]
    assert worst.size == 0 or worst.max() <= 1.0, worst.max()


def upstream(rng, n, k):
    g = rng.normal(size=n).astype(np.float32)
    h = (rng.normal(size=n) * 0.3).astype(np.float32)
    gt = (rng.normal(size=(n, k)) * 0.5).astype(np.float32)
    return g, h, gt


def dev(x, dtype=None):
    t = torch.as_tensor(x, device="cuda:0")
    return t if dtype is None else t.to(dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_logprob_gradient(ops, shape, dtype):
    n, v = shape
    rng = np.random.default_rng(n * 999983 + v)
    t = float(rng.choice([0.7, 1.0, 2.0]))
    k = int(min(v, rng.choice([1, 3, 8, 20])))
    z = matrix(logits_of(rng, n, v), dtype, pad=int(rng.integers(0, 4)), offset=int(rng.integers(0, 3)))
    tokens = rng.integers(0, v, n)
    if n > 2:
        tokens[1] = -1
    tok = dev(tokens, torch.int32 if v % 2 else torch.int64)
    fwd = ops.token_logprobs(z, tok, top_k=k, temperature=t)
    g, h, gt = upstream(rng, n, k)
    ids = host(fwd["top_ids"])
    for parts in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
        a, b, c = (x if use else None for x, use in zip((g, h, gt), parts))
        got = ops.token_logprobs_backward(
            z, tok, fwd, d_logprob=None if a is None else dev(a),
            d_entropy=None if b is None else dev(b), d_top_logprobs=None if c is None else dev(c),
            temperature=t, out=matrix(np.zeros((n, v)), dtype, pad=2, offset=1))
        want, size = ref.token_logprobs_backward(host(z), tokens, ids, a, b, c, t)
        check_gradient(got, want, size, dtype)
        if n > 600:
            break


@pytest.mark.parametrize("v", [16, 250, 1500, 20011])
def test_edge_rows_logprob_gradient(ops, v):
    rng = np.random.default_rng(v)
    z = matrix(edge_rows(v, "f32", rng), "f32", pad=1)
    n = z.shape[0]
    tokens = rng.integers(0, v, n)
    tokens[4] = v
    tok = dev(tokens)
    fwd = ops.token_logprobs(z, tok, top_k=4)
    g, h, gt = upstream(rng, n, 4)
    # a class listed twice counts by its first entry, ids outside the classes do not
    ids = host(fwd["top_ids"]).copy()
    ids[2] = [1, v + 5, 1, -7]
    fwd = dict(fwd, top_ids=dev(ids))
    got = ops.token_logprobs_backward(z, tok, fwd, d_logprob=dev(g), d_entropy=dev(h),
                                      d_top_logprobs=dev(gt))
    # differences of numbers near the type's largest are not differences of reals
    fine = [i for i in range(n) if i != 9]
    want, size = ref.token_logprobs_backward(host(z), tokens, ids, g, h, gt, 1.0)
    check_gradient(got[fine], want[fine], size[fine], "f32")
    # no upstream gradient: 0, whatever the row holds
    zero = ops.token_logprobs_backward(z, tok, fwd, d_logprob=dev(0 * g), d_entropy=dev(0 * h),
                                       d_top_logprobs=dev(0 * gt))
    assert not zero.any()


@pytest.mark.parametrize("v", [16, 300, 3000])
def test_logprob_gradient_against_differences(ops, v):
    """Central differences of the forward kernel, step 2^-5 in fp32: h^2 / 6 of a
    third derivative of a few times the gradient's size (2e-4), and 60 u 13 / h of
    rounding (3e-4 of a unit upstream gradient)."""
    rng = np.random.default_rng(v)
    step = 2.0 ** -5
    z = logits_of(rng, 1, v).astype(np.float32)
    at = np.concatenate([np.argsort(-z[0])[:3], rng.integers(0, v, 3)])
    tokens = np.array([int(at[1])])
    g, h, _ = upstream(rng, 1, 1)
    rows = np.repeat(z, 2 * at.size, 0)
    for i, c in enumerate(at):
        rows[2 * i, c] += step
        rows[2 * i + 1, c] -= step
    up = rows[np.arange(0, 2 * at.size, 2), at].astype(np.float64)
    down = rows[np.arange(1, 2 * at.size, 2), at].astype(np.float64)
    o = ops.token_logprobs(dev(rows), dev(np.repeat(tokens, 2 * at.size)))
    f = g[0] * host(o["logprob"]) + h[0] * host(o["entropy"])
    diff = (f[0::2] - f[1::2]) / (up - down)
    fwd = ops.token_logprobs(dev(z), dev(tokens))
    d = host(ops.token_logprobs_backward(dev(z), dev(tokens), fwd, d_logprob=dev(g), d_entropy=dev(h)))
    assert np.abs(d[0, at] - diff).max() < 2e-3 * (abs(g[0]) + abs(h[0]) + 1)


def teacher_of(rng, z, k, kind, t, dup=True):
    """The best classes of a noisy copy, some entries unused, one listed twice."""
    n, v = z.shape
    y = z + rng.normal(size=z.shape)
    m = min(k, v)
    ids = np.full((n, k), -1, np.int64)
    ids[:, :m] = np.argsort(-y, axis=1)[:, :m]
    y = np.where(np.isfinite(y), y, -30.0)
    val = np.take_along_axis(y, np.maximum(ids, 0), 1)
    if kind == "logprobs":
        x = y / t
        val = val / t - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)) - x.max(1, keepdims=True)
    if k > 2 and n > 1:
        ids[n // 2, 1] = -1
        if dup:
            ids[n - 1, 2] = ids[n - 1, 0]
    return ids, val.astype(np.float32)


def check_loss(got, want, size):
    got = host(got)
    bad = ~np.isfinite(want)
    assert np.array_equal(got[bad], want[bad], equal_nan=True)
    # every term has the error of its log p (60 u + 8 u |ln p|) or of its q (the same)
    assert (np.abs(got - want) <= 130 * U * size + 1e-30)[~bad].all(), (np.abs(got - want) / size)[~bad].max()


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_distill(ops, shape, dtype, kind):
    n, v = shape
    rng = np.random.default_rng(n * 7919 + v)
    t = float(rng.choice([0.7, 1.0, 2.0]))
    k = int(rng.choice([1, 3, 8, 20, 64]))
    z = matrix(logits_of(rng, n, v), dtype, pad=int(rng.integers(0, 4)), offset=int(rng.integers(0, 3)))
    ids, val = teacher_of(rng, host(z), k, kind, t)
    w = rng.uniform(0.5, 2.0, n).astype(np.float32)
    if n > 2:
        w[1] = 0.0
    did = dev(ids, torch.int32 if v % 2 else torch.int64)
    loss, d, loss_size, size = ref.distill(host(z), ids, val, kind, t, w)
    out = {"d_logits": matrix(np.zeros((n, v)), dtype, pad=1, offset=1)}
    got = ops.distill(z, did, dev(val), kind=kind, temperature=t, row_weights=dev(w), out=out)
    check_loss(got["loss"], loss, loss_size)
    check_gradient(got["d_logits"], d, size, dtype)
    # the loss alone, then its backward pass
    alone = ops.distill(z, did, dev(val), kind=kind, temperature=t, gradient=False)
    assert "d_logits" not in alone
    loss1, _, size1, _ = ref.distill(host(z), ids, val, kind, t)
    check_loss(alone["loss"], loss1, size1)
    back = ops.distill_backward(z, did, dev(val), alone["stats"], dev(w), kind=kind, temperature=t)
    check_gradient(back, d, size, dtype)


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("shape", [(2, 200), (3, 1000), (520, 1500), (2, 40001)],
                         ids=lambda s: f"{s[0]}x{s[1]}")
def test_distill_256_entries(ops, shape, kind):
    n, v = shape
    rng = np.random.default_rng(v)
    z = matrix(logits_of(rng, n, v), "f32")
    ids, val = teacher_of(rng, host(z), 256, kind, 1.0)
    loss, d, loss_size, size = ref.distill(host(z), ids, val, kind, 1.0)
    got = ops.distill(z, dev(ids), dev(val), kind=kind)
    check_loss(got["loss"], loss, loss_size)
    check_gradient(got["d_logits"], d, size, "f32")


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("v", [2, 16, 250, 1500, 20011])
@pytest.mark.parametrize("many", [False, True])
def test_edge_rows_distill(ops, v, kind, many):
    rng = np.random.default_rng(v)
    rows = edge_rows(v, "f32", rng)
    rows[9] = rng.normal(size=v) * 30      # a peaked row, nothing left for the rest
    rows = np.concatenate([rows, rng.normal(size=(6, v))])
    if many:
        if v > 1500:
            pytest.skip("few rows cover it")
        rows = np.tile(rows, (30, 1))
    z = matrix(rows, "f32", pad=3)
    n = z.shape[0]
    # (np.where: a teacher of a plain row everywhere)
    plain = np.where(np.isfinite(rows) & (np.abs(rows) < 1e30), rows, -2.0)
    ids, val = teacher_of(rng, plain, 5, kind, 1.0)
    ids[12] = -1                            # nothing listed
    ids[13, 0] = v                          # an id beyond the classes
    val[14, 0] = np.nan
    val[15] = -INF                          # listed, without mass
    if v >= 5:
        ids[16, :5] = np.arange(5)
        val[16] = -0.5                      # more mass than 1 (logprobs)
    loss, d, loss_size, size = ref.distill(host(z), ids, val, kind, 1.0)
    got = ops.distill(z, dev(ids), dev(val), kind=kind)
    check_loss(got["loss"], loss, loss_size)
    check_gradient(got["d_logits"], d, size, "f32")


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("v", [12, 64, 300, 1500])
def test_distill_all_classes_listed(ops, v, kind):
    """Every class listed: the tail is empty and drops out."""
    rng = np.random.default_rng(v)
    k = min(v, 256)
    z = matrix(logits_of(rng, 4, v)[:, :k], "f32")
    ids, val = teacher_of(rng, host(z), k, kind, 1.0, dup=False)
    loss, d, loss_size, size = ref.distill(host(z), ids, val, kind, 1.0)
    got = ops.distill(z, dev(ids), dev(val), kind=kind)
    check_loss(got["loss"], loss, loss_size)
    check_gradient(got["d_logits"], d, size, "f32")


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("v", [16, 300, 3000])
def test_distill_gradient_against_differences(ops, v, kind):
    """Central differences of the loss kernel; the bounds of the log-probabilities'."""
    rng = np.random.default_rng(v)
    step = 2.0 ** -5
    z = logits_of(rng, 1, v, 1.0).astype(np.float32)
    ids, val = teacher_of(rng, z.astype(np.float64), 4, kind, 2.0)
    at = np.concatenate([ids[0], rng.integers(0, v, 4)])
    rows = np.repeat(z, 2 * at.size, 0)
    for i, c in enumerate(at):
        rows[2 * i, c] += step
        rows[2 * i + 1, c] -= step
    up = rows[np.arange(0, 2 * at.size, 2), at].astype(np.float64)
    down = rows[np.arange(1, 2 * at.size, 2), at].astype(np.float64)
    m = 2 * at.size
    o = ops.distill(dev(rows), dev(np.repeat(ids, m, 0)), dev(np.repeat(val, m, 0)), kind=kind,
                    temperature=2.0, gradient=False)
    f = host(o["loss"])
    diff = (f[0::2] - f[1::2]) / (up - down)
    d = host(ops.distill(dev(z), dev(ids), dev(val), kind=kind, temperature=2.0)["d_logits"])
    assert np.abs(d[0, at] - diff).max() < 2e-3 * 4


@pytest.mark.parametrize("shape", [(40, 16), (5, 300), (600, 1500), (2, 40000)],
                         ids=lambda s: f"{s[0]}x{s[1]}")
def test_gradient_in_place_of_the_logits(ops, shape):
    n, v = shape
    rng = np.random.default_rng(v)
    z = matrix(logits_of(rng, n, v), "bf16", pad=3, offset=1)
    ids, val = teacher_of(rng, host(z), 8, "logprobs", 1.0)
    tokens = dev(rng.integers(0, v, n))
    fwd = ops.token_logprobs(z, tokens, top_k=3)
    g, h, gt = (dev(x) for x in upstream(rng, n, 3))
    apart = ops.token_logprobs_backward(z, tokens, fwd, d_logprob=g, d_entropy=h, d_top_logprobs=gt)
    x = z.as_strided(z.shape, z.stride()).clone()
    y = matrix(host(z), "bf16", pad=3, offset=1)
    same = ops.token_logprobs_backward(y, tokens, fwd, d_logprob=g, d_entropy=h, d_top_logprobs=gt, out=y)
    assert same is y and torch.equal(y, apart)
    for kind in ("logits", "logprobs"):
        want = ops.distill(x, dev(ids), dev(val), kind=kind)
        y = matrix(host(z), "bf16", pad=3, offset=1)
        got = ops.distill(y, dev(ids), dev(val), kind=kind, out={"d_logits": y})
        assert torch.equal(got["loss"], want["loss"]) and torch.equal(y, want["d_logits"])


def test_what_lies_between_rows_stays(ops):
    rng = np.random.default_rng(1)
    for v in (13, 301, 5001):
        buf = torch.full((6, v + 5), 7.0, device="cuda:0", dtype=torch.float16)
        z = matrix(logits_of(rng, 6, v), "f16")
        ids, val = teacher_of(rng, host(z), 4, "logits", 1.0)
        ops.distill(z, dev(ids), dev(val), out={"d_logits": buf[:, 2:v + 2]})
        assert (buf[:, :2] == 7).all() and (buf[:, v + 2:] == 7).all()


def test_results_repeat_bit_for_bit(ops):
    rng = np.random.default_rng(2)
    for n, v in ((2, 60000), (530, 2000), (3, 40)):
        z = matrix(logits_of(rng, n, v), "bf16")
        tokens = dev(rng.integers(0, v, n))
        ids, val = teacher_of(rng, host(z), 16, "logprobs", 1.0)
        a = ops.token_logprobs(z, tokens, top_k=20)
        d = ops.distill(z, dev(ids), dev(val), kind="logprobs")
        for _ in range(3):
            b = ops.token_logprobs(z, tokens, top_k=20)
            assert all(torch.equal(a[key], b[key]) for key in a)
            e = ops.distill(z, dev(ids), dev(val), kind="logprobs")
            assert all(torch.equal(d[key], e[key]) for key in d)


def test_offsets_beyond_32_bits(ops):
    """Rows that begin beyond 2^31 elements and beyond 2^32 bytes."""
    n, v = 36000, 65600
    z = torch.zeros(n, v, device="cuda:0", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda:0").manual_seed(1)
    at = [0, 17, n // 2, n - 2, n - 1]
    for i in at:
        z[i].copy_(torch.randn(v, device="cuda:0", generator=g) * 3)
    tokens = np.full(n, v - 1)
    tok = dev(tokens)
    got = ops.token_logprobs(z, tok, top_k=3)
    want = ref.token_logprobs(host(z[at]), tokens[at], 3, 1.0)
    check_forward({key: x[at] for key, x in got.items()}, want, 3)
    ones = torch.ones(n, device="cuda:0")
    d = ops.token_logprobs_backward(z, tok, got, d_logprob=ones, out=z)  # in place
    del got
    full, size = ref.token_logprobs_backward(
        np.zeros((1, v)), tokens[:1], np.zeros((1, 0), np.int32), np.ones(1), None, None, 1.0)
    check_gradient(d[n - 3:n - 2], full, size, "bf16")


def test_streams_and_a_shared_handle(ops):
    """Calls on several streams, each ordered after the stream's own writes; few
    long rows share the handle's workspace."""
    rng = np.random.default_rng(5)
    n, v, k = 2, 60000, 8
    data = [matrix(logits_of(rng, n, v), "f32") for _ in range(4)]
    want = [ref.token_logprobs(host(z), None, k, 1.0) for z in data]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got, keep = [], []
    for i in range(12):
        s = streams[i % 3]
        with torch.cuda.stream(s):
            z = torch.zeros_like(data[i % 4])
            z.copy_(data[i % 4], non_blocking=True)
            got.append(ops.token_logprobs(z, None, top_k=k))  # on the current stream
            keep.append(z)
    for i in range(4):  # and by an argument
        got.append(ops.token_logprobs(data[i], None, top_k=k, stream=streams[i % 3]))
    torch.cuda.synchronize()
    for i in range(12):
        check_forward(got[i], want[i % 4], k)
    for i in range(4):
        check_forward(got[12 + i], want[i], k)


@pytest.mark.parametrize("raw", [False, True])
def test_new_arrays_belong_to_the_calls_stream(ops, raw):
    """Memory of the current stream that is free to it may still be in use there: what a
    call makes for another stream comes from that stream's memory."""
    rng = np.random.default_rng(15)
    n, v = 3, 5000
    z = matrix(logits_of(rng, n, v), "f32")
    want = ref.token_logprobs(host(z), None, 4, 1.0)
    ids, val = teacher_of(rng, host(z), 4, "logits", 1.0)
    did, dval, ones = dev(ids), dev(val), dev(np.ones(n, np.float32))
    s = torch.cuda.Stream()
    on = s.cuda_stream if raw else s
    torch.cuda.synchronize()
    a = ops.token_logprobs(z, None, top_k=4, stream=on)
    b = ops.distill(z, did, dval, stream=on)
    made = [*a.values(), *b.values(),
            ops.token_logprobs_backward(z, None, a, d_entropy=ones, stream=on),
            ops.distill_backward(z, did, dval, b["stats"], ones, stream=on)]
    here = ops.token_logprobs(z, None)["stats"]
    torch.cuda.synchronize()

    def owner(x):
        at = x.data_ptr()
        return [q["stream"] for q in torch.cuda.memory_snapshot()
                if q["address"] <= at < q["address"] + q["total_size"]]

    assert all(owner(x) == [s.cuda_stream] for x in made)
    assert owner(here) == [torch.cuda.current_stream().cuda_stream]
    check_forward(a, want, 4)


def test_graph_capture():
    """A captured step, replayed on new contents, with eager calls between."""
    from tiny_metal_nn import LogitOps
    rng = np.random.default_rng(6)
    n, v, k = 3, 30000, 6
    z = matrix(logits_of(rng, n, v), "bf16")
    tokens = dev(rng.integers(0, v, n))
    ids, val = teacher_of(rng, host(z), 8, "logprobs", 1.0)
    did, dval = dev(ids), dev(val)
    with LogitOps() as mine, LogitOps() as eager:
        out, dout = {}, {}
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            mine.token_logprobs(z, tokens, top_k=k, out=out)
            mine.distill(z, did, dval, kind="logprobs", out=dout)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            mine.token_logprobs(z, tokens, top_k=k, out=out)
            mine.distill(z, did, dval, kind="logprobs", out=dout)
        for i in range(4):
            z.copy_(torch.as_tensor(logits_of(rng, n, v)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            a = eager.token_logprobs(z, tokens, top_k=k)
            b = eager.distill(z, did, dval, kind="logprobs")
            torch.cuda.synchronize()
            assert all(torch.equal(a[key], out[key]) for key in a), i
            assert all(torch.equal(b[key], dout[key]) for key in b), i


def test_host_arrays(ops):
    rng = np.random.default_rng(7)
    for n, v, dtype in ((9, 16, np.float32), (4, 700, np.float16), (2, 20001, np.float32), (0, 5, np.float32)):
        whole = (logits_of(rng, max(n, 1), v + 3)[:n]).astype(dtype)
        z = whole[:, 1:v + 1]
        tokens = rng.integers(0, v, n).astype(np.int32)
        got = ops.token_logprobs(z, tokens, top_k=3, temperature=2.0)
        want = ref.token_logprobs(z, tokens, 3, 2.0)
        check_forward({key: torch.as_tensor(x) for key, x in got.items()}, want, 3)
        g, h, gt = upstream(rng, n, 3)
        d = ops.token_logprobs_backward(z, tokens, got, d_logprob=g, d_entropy=h, d_top_logprobs=gt,
                                        temperature=2.0)
        ref_d, size = ref.token_logprobs_backward(z, tokens, got["top_ids"], g, h, gt, 2.0)
        kind = "f32" if dtype == np.float32 else "f16"
        check_gradient(torch.as_tensor(d), ref_d, size, kind)
        if n == 0:
            continue
        ids, val = teacher_of(rng, z.astype(np.float64), 3, "logprobs", 2.0)
        place = np.full((n, v + 2), 7, dtype)
        o = ops.distill(z, ids, val, kind="logprobs", temperature=2.0, out={"d_logits": place[:, 1:v + 1]})
        loss, dd, loss_size, dsize = ref.distill(z, ids, val, "logprobs", 2.0)
        check_loss(torch.as_tensor(o["loss"]), loss, loss_size)
        check_gradient(torch.as_tensor(np.ascontiguousarray(o["d_logits"])), dd, dsize, kind)
        assert (place[:, 0] == 7).all() and (place[:, -1] == 7).all()
        back = ops.distill_backward(z, ids, val, o["stats"], np.ones(n, np.float32), kind="logprobs",
                                    temperature=2.0)
        check_gradient(torch.as_tensor(back), dd, dsize, kind)


def test_no_rows(ops):
    z = torch.empty(0, 9, device="cuda:0")
    out = ops.token_logprobs(z, torch.empty(0, dtype=torch.int64, device="cuda:0"), top_k=2)
    assert out["logprob"].shape == (0,) and out["top_ids"].shape == (0, 2)
    d = ops.distill(z, torch.empty(0, 2, dtype=torch.int64, device="cuda:0"), torch.empty(0, 2, device="cuda:0"))
    assert d["d_logits"].shape == (0, 9)


def test_refusals(ops):
    from tiny_metal_nn import ClosedError, DTypeError, LogitOps
    z = torch.zeros(4, 10, device="cuda:0")
    tok = torch.zeros(4, dtype=torch.int64, device="cuda:0")
    ids = torch.zeros(4, 2, dtype=torch.int64, device="cuda:0")
    val = torch.zeros(4, 2, device="cuda:0")
    fwd = ops.token_logprobs(z, tok, top_k=2)
    with pytest.raises(DTypeError, match="logits"):
        ops.token_logprobs(z.double(), tok)
    with pytest.raises(DTypeError, match="tokens"):
        ops.token_logprobs(z, tok.float())
    with pytest.raises(ValueError, match="2D"):
        ops.token_logprobs(z[0], tok)
    with pytest.raises(ValueError, match="unit stride"):
        ops.token_logprobs(z.t().contiguous().t(), tok)
    with pytest.raises(ValueError, match="overlap"):
        ops.token_logprobs(z[:1].expand(4, 10), tok)
    with pytest.raises(ValueError, match="shape"):
        ops.token_logprobs(z, tok[:3])
    with pytest.raises(TypeError, match="tokens"):
        ops.token_logprobs(z, np.zeros(4, np.int64))
    with pytest.raises(TypeError, match="tokens"):
        ops.token_logprobs(np.zeros((4, 10), np.float32), tok)
    with pytest.raises(ValueError, match="device"):
        ops.token_logprobs(z.cpu(), tok)
    with pytest.raises(ValueError, match="at least one class"):
        ops.token_logprobs(z[:, :0], tok)
    for k in (-1, 129):
        with pytest.raises(ValueError):
            ops.token_logprobs(z, tok, top_k=k)
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-9):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_logprobs(z, tok, temperature=t)
    with pytest.raises(ValueError, match="top_ids"):
        ops.token_logprobs(z, tok, top_k=2, out={"top_ids": fwd["top_ids"][:, :1]})
    with pytest.raises(DTypeError, match="rank"):
        ops.token_logprobs(z, tok, out={"rank": torch.zeros(4, device="cuda:0")})
    with pytest.raises(ValueError, match="tokens"):
        ops.token_logprobs_backward(z, None, fwd, d_logprob=val[:, 0].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        ops.token_logprobs_backward(z, tok, fwd, d_logprob=val[:, 0])
    with pytest.raises(DTypeError, match="d_logits"):
        ops.token_logprobs_backward(z, tok, fwd, d_logprob=fwd["logprob"], out=z.half())
    with pytest.raises(ValueError, match="kind"):
        ops.distill(z, ids, val, kind="probs")
    with pytest.raises(ValueError, match="teacher"):
        ops.distill(z, ids, val[:, :1].contiguous())
    with pytest.raises(ValueError, match="teacher_k"):
        ops.distill(z, ids[:, :0].contiguous(), val[:, :0].contiguous())
    with pytest.raises(ValueError, match="teacher_k"):
        ops.distill(z, torch.zeros(4, 257, dtype=torch.int64, device="cuda:0"), torch.zeros(4, 257, device="cuda:0"))
    with pytest.raises(DTypeError, match="teacher"):
        ops.distill(z, ids, val.half())
    with pytest.raises(ValueError, match="aligned"):
        ops.distill(z, ids, val, out={"stats": torch.zeros(17, device="cuda:0")[1:].view(4, 4)})
    with pytest.raises(ValueError, match="row_weights"):
        ops.distill(z, ids, val, row_weights=val)
    with pytest.raises(ValueError, match="stream"):
        ops.token_logprobs(np.zeros((4, 10), np.float32), stream=torch.cuda.current_stream())
    other = LogitOps()
    other.close()
    assert other.closed
    with pytest.raises(ClosedError):
        other.token_logprobs(z, tok)


def test_gradients_in_place_need_the_logits_layout(ops):
    """From one address with another row stride, a row's gradient would lie over the
    logits of the next."""
    buf = torch.zeros(4 * 20, device="cuda:0")
    z, d = buf.view(4, 20)[:, :10], buf[:40].view(4, 10)
    ids = torch.zeros(4, 2, dtype=torch.int64, device="cuda:0")
    val, ones = torch.zeros(4, 2, device="cuda:0"), torch.ones(4, device="cuda:0")
    fwd = ops.token_logprobs(z, None)
    with pytest.raises(ValueError, match="row_stride"):
        ops.token_logprobs_backward(z, None, fwd, d_entropy=ones, out=d)
    with pytest.raises(ValueError, match="row_stride"):
        ops.distill(z, ids, val, out={"d_logits": d})
    with pytest.raises(ValueError, match="row_stride"):
        ops.distill_backward(z, ids, val, torch.zeros(4, 4, device="cuda:0"), ones, out=d)
    assert not buf.any()
    # one row has no stride
    assert ops.distill(z[:1], ids[:1], val[:1], out={"d_logits": d[:1]})["d_logits"] is not None


def test_a_captured_stream_needs_its_own_handle():
    """A capture cannot wait for another stream's work: the call says so."""
    from tiny_metal_nn import LogitOps
    from tiny_metal_nn._lib import TmnnError
    z = torch.zeros(1, 60000, device="cuda:0")
    out = {}
    with LogitOps() as o:
        o.token_logprobs(z, None, out=out)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            with pytest.raises(TmnnError, match="own"):
                o.token_logprobs(z, None, out=out)
            z.add_(0.0)
        torch.cuda.synchronize()
