"""The class head on the GPU where it can go wrong: rows that do not count, labels out of
range, values that are not finite, confident rows, weights and inputs of any size, far offsets, streams,
captured graphs, host arrays and refusals. Marked gpu.

Tolerances are those of test_gpu_class_loss.py."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import head_oracle as ref  # noqa: E402
from test_gpu_class_loss import (DEV, HALF_ULP, TYPES, U, check_all, check_gradient, check_loss, inputs, matrix,  # noqa: E402,F401
                                 ops)
from test_gpu_head_f8 import laid, operands  # noqa: E402

# the walks of few dims, and tiles
DIMS = [16, 100, 200]
NAMES = ("loss", "d_features", "d_table")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", DIMS)
def test_rows_that_do_not_count_may_hold_anything(ops, d, dtype):
    n, v = 150, 70
    h, w, labels, weights = inputs(n, d, v, 3)
    labels[10], weights[20] = -5, 0.0
    clean = matrix(h, dtype)
    dirty = clean.clone()
    for row in (10, 20):
        dirty[row] = float("nan")
        dirty[row, ::3] = float("inf")
    w = matrix(w, dtype)
    got = ops.class_loss(dirty, w, labels, row_weights=weights)
    for name in ("loss", "d_features"):
        assert not got[name][10].any() and not got[name][20].any()
    check_all(got, ref.class_loss(clean, w, labels, weights), clean, w, weights, dtype, 1.0)
    # a table that holds NaN leaves them at 0 too
    w[5] = float("nan")
    got = ops.class_loss(clean, w, labels, row_weights=weights)
    for name in ("loss", "d_features"):
        assert not got[name][10].any() and not got[name][20].any() and got[name][30].isnan().all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", DIMS)
def test_no_row_counts(ops, d, dtype):
    h, w, labels, weights = inputs(40, d, 30, 3)
    h, w = matrix(h, dtype), matrix(w, dtype)
    got = ops.class_loss(h, w, torch.full_like(labels, -1), row_weights=weights)
    assert not any(got[name].any() for name in NAMES)
    got = ops.class_loss(h, w, labels, row_weights=torch.zeros_like(weights))
    assert not any(got[name].any() for name in NAMES)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", DIMS)
def test_labels_out_of_range_and_values_that_are_not_finite(ops, d, dtype):
    n, v = 150, 70
    h, w, labels, weights = inputs(n, d, v, 3)
    labels = labels.clamp_min(0)
    weights = weights.abs() + 0.5
    h, w = matrix(h, dtype), matrix(w, dtype)
    want = ops.class_loss(h, w, labels, row_weights=weights)
    for kind in ("label", "large label", "nan", "inf"):
        x, l = h.clone(), labels.clone()
        if kind == "label":
            l[7] = v
        elif kind == "large label":
            l[7] = 2 ** 40
        else:
            x[7, 1] = float(kind)
        got = ops.class_loss(x, w, l, row_weights=weights)
        assert got["loss"][7].isnan() and got["d_features"][7].isnan().all() and got["d_table"].isnan().all(), kind
        rest = torch.arange(n, device=DEV) != 7
        assert torch.equal(got["loss"][rest], want["loss"][rest])
        assert torch.equal(got["d_features"][rest], want["d_features"][rest])


@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("v", [1, 2, 300])
def test_confident_rows_keep_their_bits(ops, d, v):
    """Small losses and gradients are relative to 1 - p, not to 1."""
    n = 40
    g = torch.Generator(device=DEV).manual_seed(5)
    w = torch.randint(-8, 9, (v, d), device=DEV, generator=g) / 8.0
    labels = torch.randint(0, v, (n,), device=DEV, generator=g)
    w[:, 0] = 0.0
    w[:, 1:5] = torch.tensor([[(i >> b) % 2 for b in range(4)] for i in range(v)], device=DEV).float()
    h = w[labels] * 2.0
    h[:, 0] = 0.0
    for i in range(n):  # the label's class above the others by up to 40
        h[i] *= 1 + i % 8
    got = ops.class_loss(h, w, labels)
    want = ref.class_loss(h, w, labels)
    # logits are exact here: 60 u of the sums, 3e-5 of the others' probabilities; what is below fp32's
    # smallest normal number, 2^-126, may be 0 (rows here pass e^-800)
    assert ((got["loss"].double() - want["loss"]).abs() <= (64 * U + 3e-5) * want["loss"] + 2.0 ** -126).all()
    assert ((got["stats"][:, 2].double() - want["missing"]).abs() <= 4e-5 * want["missing"] + 2.0 ** -126).all()
    check_all(got, want, h, w, None, "f32", 1.0, exact=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", DIMS)
def test_weights_of_any_size(ops, d, dtype):
    n, v = 60, 50
    h, w, labels, _ = inputs(n, d, v, 3)
    labels = labels.clamp_min(0)
    # (16-bit results of other sizes would lose theirs)
    weights = torch.ldexp(torch.randn(n, device=DEV), torch.randint(-30, 30, (n,), device=DEV) if dtype != "f16" else
                          torch.randint(-3, 4, (n,), device=DEV))
    h, w = matrix(h, dtype), matrix(w, dtype)
    got = ops.class_loss(h, w, labels, row_weights=weights)
    want = ref.class_loss(h, w, labels, weights)
    check_all(got, want, h, w, weights, dtype, 1.0, names=("d_features",))
    # rows far below the largest weight are small against the table's gradient: bounded as a whole
    off = (got["d_table"].double() - want["d_table"]).norm() / want["d_table"].norm()
    assert off < {"f32": 1e-5, "f16": 2e-3, "bf16": 1e-2}[dtype]  # (the largest terms' 3e-5 p, 2^-11, 2^-8)


@pytest.mark.parametrize("size", [1e-15, 1e-6, 1e6])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", DIMS)
def test_inputs_of_any_size(ops, d, dtype, size):
    """Features and table of far sizes whose products are ordinary."""
    h, w, labels, weights = inputs(70, d, 90, 3)
    h, w = matrix(h * size, dtype), matrix(w / size, dtype)
    got = ops.class_loss(h, w, labels, row_weights=weights)
    check_all(got, ref.class_loss(h, w, labels, weights), h, w, weights, dtype, 1.0)


@pytest.mark.parametrize("t", [1e-3, 0.05, 20.0])
@pytest.mark.parametrize("d", DIMS)
def test_temperatures(ops, d, t):
    n, v = 70, 90
    h, w, labels, weights = inputs(n, d, v, 3, exact=True)  # (logits that fp32 holds: t divides their errors too)
    got = ops.class_loss(h, w, labels, row_weights=weights, temperature=t)
    want = ref.class_loss(h, w, labels, weights, t)
    # an exponent of x is 3 u |x| off
    span = (want["z"] / t).max()
    up = weights.double().abs()
    err = (60 * U + 8 * U * span) * (up * (span + 1)) + 1e-30
    assert ((got["loss"].double() - want["loss"]).abs() <= err).all()
    prob = 3e-5 + 8 * U * span
    floor = 2.0 ** -39 / t * (up.unsqueeze(1) * w.double().abs().sum(0) + 1)
    check_gradient(got["d_features"], want["d_features"], want["x"], prob, v, floor, "f32")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", DIMS)
def test_gradients_one_at_a_time_and_again(ops, d, dtype):
    h, w, labels, weights = inputs(150, d, 700, 3)
    h, w = matrix(h, dtype), matrix(w, dtype)
    both = ops.class_loss(h, w, labels, row_weights=weights)
    again = ops.class_loss(h, w, labels, row_weights=weights)
    for name in NAMES:
        assert torch.equal(both[name], again[name])
    for name in ("features", "table"):
        one = ops.class_loss(h, w, labels, row_weights=weights, gradient=name)
        assert set(one) == {"loss", "stats", "d_" + name}
        assert torch.equal(one["d_" + name], both["d_" + name]) and torch.equal(one["loss"], both["loss"])
        back = ops.class_loss_backward(h, w, labels, both["stats"], weights, gradient=name)
        assert set(back) == {"d_" + name}
        assert torch.equal(back["d_" + name], both["d_" + name])


@pytest.mark.parametrize("d", DIMS)
def test_few_rows_over_many_classes_and_the_reverse(ops, d):
    for n, v in ((2, 40000), (40000, 2)):
        for dtype in TYPES:
            h, w, labels, weights = inputs(n, d, v, 11)
            h, w = matrix(h, dtype), matrix(w, dtype)
            got = ops.class_loss(h, w, labels, row_weights=weights)
            check_all(got, ref.class_loss(h, w, labels, weights), h, w, weights, dtype, 1.0)


def test_without_rows(ops):
    h = torch.zeros(0, 40, device=DEV)
    w = torch.ones(6, 40, device=DEV)
    labels = torch.zeros(0, dtype=torch.int64, device=DEV)
    got = ops.class_loss(h, w, labels)
    assert got["loss"].shape == (0,) and got["stats"].shape == (0, 4) and got["d_features"].shape == (0, 40)
    assert got["d_table"].shape == (6, 40) and not got["d_table"].any()
    assert ops.class_loss(h, w, labels, gradient="none")["loss"].shape == (0,)
    x = torch.zeros(0, 40, device=DEV, dtype=torch.float8_e4m3fn)
    q = ops.quantize_f8(w, block_rows=128)
    s = ops.quantize_f8(h)
    assert s["values"].shape == (0, 40) and s["scales"].shape == (0, 1)
    assert ops.class_logits_f8(x, s["scales"], q["values"], q["scales"]).shape == (0, 6)


@pytest.mark.parametrize("d", [64, 136])
def test_offsets_past_32_bits(ops, d):
    """Rows that lie gigabytes apart, and a stride that no tile takes in place."""
    n, v, stride = 70, 70001, 32768
    h, w, labels, weights = inputs(n, d, v, 3)
    h = matrix(h, "f16")
    far = torch.empty(v, stride, device=DEV, dtype=torch.float16)[:, :d]
    far.copy_(w)
    near = far.contiguous()
    out = {"d_table": torch.empty(v, stride, device=DEV, dtype=torch.float16)[:, :d]}
    got = ops.class_loss(h, far, labels, row_weights=weights, out=out)
    want = ops.class_loss(h, near, labels, row_weights=weights)
    for name in NAMES:
        assert torch.equal(got[name], want[name])
    del far, out, got
    apart = torch.empty(3, 5_000_000, device=DEV, dtype=torch.float16)[:, :d]
    apart.copy_(h[:3])
    got = ops.class_loss(apart, near, labels[:3], row_weights=weights[:3])
    want = ops.class_loss(h[:3], near, labels[:3], row_weights=weights[:3])
    for name in NAMES:
        assert torch.equal(got[name], want[name])


def test_f8_offsets_past_32_bits(ops):
    x, sx, w, sw = operands(40, 200, 70001, "f32", 5)
    far = torch.empty(70001, 65536, device=DEV, dtype=torch.uint8)
    far[:, :200] = w.view(torch.uint8)
    far = far.view(torch.float8_e4m3fn)[:, :200]
    want = ops.class_logits_f8(laid(x), sx, laid(w), sw)
    assert torch.equal(ops.class_logits_f8(laid(x), sx, far, sw), want)
    out = torch.full((40, 40_000_000), 3.0, device=DEV, dtype=torch.float16)  # 3.2 GB of rows
    got = ops.class_logits_f8(laid(x), sx, far, sw, out=out[:, :70001])
    assert torch.equal(got, want.half()) and (out[:, 70001] == 3.0).all()


def test_what_lies_beside_stays(ops):
    """Nothing is written between rows or behind the last one."""
    for d in DIMS:
        h, w, labels, weights = inputs(37, d, 41, 3)
        for dtype in TYPES:
            x, y = matrix(h, dtype), matrix(w, dtype)
            px = torch.full((40, d + 5), 9.0, device=DEV, dtype=TYPES[dtype])
            py = torch.full((44, d + 3), 9.0, device=DEV, dtype=TYPES[dtype])
            ops.class_loss(x, y, labels, row_weights=weights,
                           out={"d_features": px[1:38, 2:d + 2], "d_table": py[1:42, 1:d + 1]})
            for p, rows, at in ((px, 37, 2), (py, 41, 1)):
                assert (p[0] == 9).all() and (p[rows + 1:] == 9).all() and (p[:, :at] == 9).all()
                assert (p[:, at + d:] == 9).all()
    x = torch.randn(37, 130, device=DEV)
    place = torch.full((40, 160), 77, device=DEV, dtype=torch.uint8)
    for block_rows in (1, 128):
        ops.quantize_f8(x, block_rows=block_rows, out={"values": place.view(torch.float8_e4m3fn)[1:38, 3:133]})
        assert (place[0] == 77).all() and (place[38:] == 77).all() and (place[:, :3] == 77).all() and (place[:, 133:] == 77).all()


@pytest.mark.parametrize("d", DIMS)
def test_side_streams(ops, d):
    """Calls on several streams at once, through one handle: nothing is shared between them."""
    cases = []
    for i in range(4):
        h, w, labels, weights = inputs(300, d, 900, 20 + i)
        cases.append((h, w, labels, weights, ops.class_loss(h, w, labels, row_weights=weights)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        got = []
        for s, (h, w, labels, weights, _) in zip(streams, cases):
            got.append(ops.class_loss(h, w, labels, row_weights=weights, stream=s))
    torch.cuda.synchronize()
    for g, c in zip(got, cases):
        for name in NAMES:
            assert torch.equal(g[name], c[4][name])


def test_the_context_stream_needs_a_workspace(ops):
    h, w, labels, weights = inputs(30, 40, 50, 3)
    with pytest.raises(ValueError, match="workspace"):
        ops.class_loss(h, w, labels, stream=-1)
    want = ops.class_loss(h, w, labels)
    out = {name: torch.zeros_like(t) for name, t in want.items()}
    room = torch.empty(1 << 22, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    ops.class_loss(h, w, labels, out=out, workspace=room, stream=-1)
    torch.cuda.synchronize()
    for name in NAMES:
        assert torch.equal(out[name], want[name])
    with pytest.raises(ValueError, match="workspace must be"):
        ops.class_loss(h, w, labels, workspace=room[:256])
    with pytest.raises(ValueError, match="aligned"):
        ops.class_loss(h, w, labels, workspace=room[1:])
    with pytest.raises(TypeError, match="uint8"):
        ops.class_loss(h, w, labels, workspace=room.view(torch.int32))


@pytest.mark.parametrize("d", DIMS)
def test_captured_graphs(ops, d):
    """Two graphs of calls with workspaces of their own, replayed in turn with eager work between."""
    n, v = 200, 500
    graphs = []
    for i in range(2):
        h, w, labels, weights = inputs(n, d, v, 30 + i)
        q = ops.quantize_f8(w, block_rows=128)
        ops.class_loss(h, w, labels, row_weights=weights)  # (before the capture: modules are loaded)
        p = ops.quantize_f8(h)
        ops.class_logits_f8(p["values"], p["scales"], q["values"], q["scales"])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.class_loss(h, w, labels, row_weights=weights)
            back = ops.class_loss_backward(h, w, labels, out["stats"], weights)
            p = ops.quantize_f8(h)
            z = ops.class_logits_f8(p["values"], p["scales"], q["values"], q["scales"])
            top = None
        graphs.append((graph, h, w, labels, weights, q, out, back, z, top))
    for turn in range(4):
        for graph, h, w, labels, weights, q, out, back, z, _ in graphs:
            h.copy_(torch.randn(n, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(turn)))
            graph.replay()
        torch.cuda.synchronize()
        for graph, h, w, labels, weights, q, out, back, z, _ in graphs:
            want = ops.class_loss(h, w, labels, row_weights=weights)
            for name in NAMES:
                assert torch.equal(out[name], want[name])
            assert torch.equal(back["d_table"], want["d_table"]) and torch.equal(back["d_features"], want["d_features"])
            p = ops.quantize_f8(h)
            assert torch.equal(z, ops.class_logits_f8(p["values"], p["scales"], q["values"], q["scales"]))


@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_host_arrays(ops, d, kind):
    """numpy arrays, rows apart, give the device's bits."""
    h, w, labels, weights = inputs(33, d, 70, 3)
    h, w = matrix(h, kind), matrix(w, kind)
    want = ops.class_loss(h, w, labels, row_weights=weights, temperature=0.7)
    x = np.zeros((33, d + 3), h.cpu().numpy().dtype)
    x[:, 1:d + 1] = h.cpu().numpy()
    y, place = w.cpu().numpy(), np.full((70, d + 2), 5, x.dtype)
    got = ops.class_loss(x[:, 1:d + 1], y, labels.cpu().numpy(), row_weights=weights.cpu().numpy(), temperature=0.7,
                         out={"d_table": place[:, 1:d + 1]})
    for name in NAMES + ("stats",):
        assert np.array_equal(got[name], want[name].cpu().numpy()), name
    assert (place[:, 0] == 5).all() and (place[:, d + 1] == 5).all()
    back = ops.class_loss_backward(x[:, 1:d + 1], y, labels.cpu().numpy(), got["stats"], weights.cpu().numpy(),
                                   temperature=0.7)
    assert np.array_equal(back["d_features"], got["d_features"]) and np.array_equal(back["d_table"], got["d_table"])
    for power in ("float32", "float8_e8m0fnu"):
        q = ops.quantize_f8(y, block_rows=128, scale_dtype=power)
        p = ops.quantize_f8(x[:, 1:d + 1], scale_dtype=power)
        dq, dp = ops.quantize_f8(w, block_rows=128, scale_dtype=power), ops.quantize_f8(h, scale_dtype=power)
        assert np.array_equal(q["values"], dq["values"].view(torch.uint8).cpu().numpy())
        assert np.array_equal(p["values"], dp["values"].view(torch.uint8).cpu().numpy())
        z = ops.class_logits_f8(p["values"], p["scales"], q["values"], q["scales"], dtype="float16")
        dz = ops.class_logits_f8(dp["values"], dp["scales"], dq["values"], dq["scales"], dtype=torch.float16)
        assert np.array_equal(z, dz.cpu().numpy())


def test_refusals(ops):
    from tiny_metal_nn import DTypeError, LogitOps
    from tiny_metal_nn.trainer import ClosedError
    h, w, labels, weights = inputs(30, 40, 50, 3)
    bad = [
        (dict(labels=labels[:-1]), ValueError, "labels"), (dict(labels=labels.float()), DTypeError, "labels"),
        (dict(table=w[:, :-1]), ValueError, "values in a row"), (dict(table=w.half()), DTypeError, "table"),
        (dict(table=w.t().contiguous().t()), ValueError, "unit stride"), (dict(table=w.cpu()), ValueError, "device"),
        (dict(features=h.double()), DTypeError, "features"), (dict(features=h[0]), ValueError, "2D"),
        (dict(row_weights=weights[:-1]), ValueError, "row_weights"),
        (dict(row_weights=weights.double()), DTypeError, "row_weights"), (dict(temperature=0.0), ValueError, "temperature"),
        (dict(gradient="all"), ValueError, "gradient"),
        (dict(out={"d_table": torch.empty_like(w).half()}), DTypeError, "d_table"),
        (dict(out={"d_features": torch.empty(30, 39, device=DEV)}), ValueError, "d_features"),
        (dict(out={"loss": torch.empty(29, device=DEV)}), ValueError, "loss"),
        (dict(out={"d_features": h}), ValueError, "d_features overlaps features"),
        (dict(out={"d_table": w}), ValueError, "d_table overlaps the table"),
    ]
    for more, error, frag in bad:
        args = dict(features=h, table=w, labels=labels, row_weights=weights) | more
        x, y, l = args.pop("features"), args.pop("table"), args.pop("labels")
        with pytest.raises(error, match=frag):
            ops.class_loss(x, y, l, **args)
    with pytest.raises(ValueError, match="gradient must be"):
        ops.class_loss_backward(h, w, labels, torch.empty(30, 4, device=DEV), weights, gradient="none")
    # gradients that lie over each other; rows that interleave are fine
    place = torch.empty(60, 100, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        ops.class_loss(h, w, labels, out={"d_features": place[:30, :40], "d_table": place[:50, 20:60]})
    want = ops.class_loss(h, w, labels)
    got = ops.class_loss(h, w, labels, out={"d_features": place[:30, :40], "d_table": place[:50, 50:90]})
    assert torch.equal(got["d_features"], want["d_features"]) and torch.equal(got["d_table"], want["d_table"])

    x, sx, y, sy = operands(30, 200, 50, "f32", 3)
    power = operands(30, 200, 50, "e8m0", 3)
    for args, error, frag in (
            ((x.float(), sx, y, sy), DTypeError, "features"), ((x, sx[:, :1], y, sy), ValueError, "feature_scales"),
            ((x, sx, y[:, :100], sy), ValueError, "values in a row"), ((x, sx, y, sy.expand(2, 2)), ValueError, "table_scales"),
            ((x, sx, y, power[3]), DTypeError, "table_scales"), ((x, sx.double(), y, sy), DTypeError, "feature_scales")):
        with pytest.raises(error, match=frag):
            ops.class_logits_f8(*args)
    with pytest.raises(DTypeError, match="dtype"):
        ops.class_logits_f8(x, sx, y, sy, dtype="float64")
    with pytest.raises(ValueError, match="out must have shape"):
        ops.class_logits_f8(x, sx, y, sy, out=torch.empty(30, 49, device=DEV))
    for more, error, frag in ((dict(block_rows=2), ValueError, "block_rows"), (dict(scale_dtype="int8"), DTypeError, "scale_dtype"),
                              (dict(out={"values": torch.empty(30, 40, device=DEV)}), DTypeError, "values"),
                              (dict(out={"values": h.view(torch.float8_e4m3fn)[:, :40]}), ValueError, "overlaps")):
        with pytest.raises(error, match=frag):
            ops.quantize_f8(h, **more)
    closed = LogitOps()
    closed.close()
    with pytest.raises(ClosedError):
        closed.class_loss(h, w, labels)


def test_outputs_are_marked_as_changed(ops):
    h, w, labels, _ = inputs(30, 40, 50, 3)
    out = ops.class_loss(h, w, labels)
    before = {name: t._version for name, t in out.items()}
    ops.class_loss(h, w, labels, out=out)
    assert all(t._version > before[name] for name, t in out.items())
    q = ops.quantize_f8(w, block_rows=128)
    before = {name: t._version for name, t in q.items()}
    ops.quantize_f8(w, block_rows=128, out=q)
    assert all(t._version > before[name] for name, t in q.items())


# many rows of few classes: the table's gradient comes in hundreds of parts; few rows of wide features in a
# few; many classes of many rows go 32 a wave
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n, d, v", [(60001, 16, 5), (30000, 40, 70), (9, 136, 3), (2000, 200, 3), (600, 8, 131200)])
def test_parts_of_few_sums(ops, n, d, v, dtype):
    h, w, labels, weights = inputs(n, d, v, 5)
    h, w = matrix(h, dtype), matrix(w, dtype)
    got = ops.class_loss(h, w, labels, row_weights=weights)
    check_all(got, ref.class_loss(h, w, labels, weights), h, w, weights, dtype, 1.0)
    again = ops.class_loss(h, w, labels, row_weights=weights)
    for name in NAMES:  # sums are added in one order
        assert torch.equal(got[name], again[name])


# more classes than one piece of the logits' gradient holds, the last piece a short one; and as many as are kept
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n, v", [(1100, 130001), (1100, 60000)])
def test_pieces_of_classes(ops, n, v, dtype):
    d = 136
    h, w, labels, weights = inputs(n, d, v, 5)
    labels[:3] = torch.tensor([v - 1, 0, v // 2])
    h, w = matrix(h, dtype), matrix(w, dtype)
    got = ops.class_loss(h, w, labels, row_weights=weights)
    want = ref.class_loss(h, w, labels, weights)
    check_all(got, want, h, w, weights, dtype, 1.0)
    # the backward call computes the logits again
    plain = ops.class_loss(h, w, labels, gradient="none")
    again = ops.class_loss_backward(h, w, labels, plain["stats"], weights)
    check_all({"loss": got["loss"], **again}, want, h, w, weights, dtype, 1.0)


@pytest.mark.parametrize("d", DIMS)
def test_calls_of_several_threads(ops, d):
    import threading

    cases, got = [], [None] * 4
    for i in range(4):
        h, w, labels, weights = inputs(70 + 30 * i, d, 200 + 100 * i, i)
        cases.append((matrix(h, "bf16"), matrix(w, "bf16"), labels, weights))
    want = [ops.class_loss(h, w, labels, row_weights=weights) for h, w, labels, weights in cases]
    torch.cuda.synchronize()

    def work(i):
        h, w, labels, weights = cases[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = ops.class_loss(h, w, labels, row_weights=weights)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        for name in NAMES:
            assert torch.equal(a[name], b[name])


@pytest.mark.parametrize("d", DIMS)
def test_one_matrix_as_features_and_table(ops, d):
    h, _, labels, weights = inputs(90, d, 90, 3)
    h = matrix(h, "f32")
    got = ops.class_loss(h, h, labels, row_weights=weights)
    check_all(got, ref.class_loss(h, h, labels, weights), h, h, weights, "f32", 1.0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", DIMS)
def test_large_values_in_rows_that_do_not_count(ops, d, dtype):
    """What such rows hold does not cost the others their bits."""
    n, v = 150, 70
    h, w, labels, weights = inputs(n, d, v, 3)
    labels[10], labels[149], weights[20] = -5, -1, 0.0
    clean, w = matrix(h, dtype), matrix(w, dtype)
    want = ref.class_loss(clean, w, labels, weights)
    dirty = clean.clone()
    for row in (10, 20, 149):
        dirty[row] = 6e4 if dtype == "f16" else 1e38
    got = ops.class_loss(dirty, w, labels, row_weights=weights)
    check_all(got, want, clean, w, weights, dtype, 1.0)
    plain = ops.class_loss(clean, w, labels, gradient="none")
    back = ops.class_loss_backward(dirty, w, labels, plain["stats"], weights)
    check_all({"loss": got["loss"], **back}, want, clean, w, weights, dtype, 1.0)


# a walk over the table in a few parts and in many
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n, d, v", [(20001, 32, 700), (9000, 100, 3001), (4097, 50, 5000), (70, 64, 5000)])
def test_parts_of_rows(ops, n, d, v, dtype):
    h, w, labels, weights = inputs(n, d, v, 5)
    h, w = matrix(h, dtype), matrix(w, dtype)
    want = ref.class_loss(h, w, labels, weights)
    for gradient in ("both", "features", "none"):
        got = ops.class_loss(h, w, labels, row_weights=weights, gradient=gradient)
        check_all(got, want, h, w, weights, dtype, 1.0, names=[name for name in NAMES[1:] if name in got])
