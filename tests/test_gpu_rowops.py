"""The operators on rows of typed tensors against plain implementations in 64 bits on the host.

Bars.  u = 2^-24 is the relative error of one fp32 operation and h(t) that of the rounding to the result's type: half a step,
2^-24, 2^-11 or 2^-8.  A result of s fp32 operations on terms of magnitudes a_i is off by at most s * u * sum(a_i) before it is
rounded, and by h(t) of the value more after; a value below the type's smallest normal number is rounded to a multiple of its
smallest step.  Copies, whole numbers and 8-bit steps have to be equal.
"""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
KINDS = ["float32", "float16", "bfloat16"]
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SMALLEST = {"float32": 2.0 ** -149, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}  # smallest step
RAW = {"bfloat16": np.uint16}


def encode(x, kind):
    """Numbers as the bits of a type, rounded to nearest even."""
    if kind != "bfloat16":
        with np.errstate(all="ignore"):
            return np.asarray(x).astype(kind)
    bits = np.asarray(x, np.float32).view(np.uint32)
    with np.errstate(over="ignore"):
        up = (bits + np.uint32(0x7FFF) + ((bits >> 16) & 1)) >> 16
    return np.where((bits & 0x7FFFFFFF) > 0x7F800000, 0x7FC0, up).astype(np.uint16)


def decode(raw, kind):
    if kind != "bfloat16":
        return raw.astype(np.float64)
    return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def typed(x, kind):
    """The numbers that a type has for x."""
    return decode(encode(x, kind), kind)


class Device:
    """A typed, possibly strided tensor in device memory, as a caller's tensor library would hand it over."""

    def __init__(self, ctx, x, kind, pad=0, fill=77):
        x = np.asarray(x)
        self.kind, self.dtype, self.shape, self.pad = kind, kind, x.shape, pad
        width = (x.shape[-1] if x.ndim else 1) + pad
        block = encode(np.full(x.shape[:-1] + (width,), fill), kind)
        block[..., : width - pad] = encode(x, kind)
        self.memory = ctx.array(block)
        steps, step = [], 1
        for size in reversed(block.shape):
            steps.insert(0, step)
            step *= size
        self._stride = tuple(steps)

    def stride(self):
        return self._stride

    def data_ptr(self):
        return self.memory.ptr

    def raw(self):
        return self.memory.download()[..., : self.shape[-1]] if self.memory.nbytes else np.zeros(self.shape)

    def host(self):
        return decode(self.raw(), self.kind)

    def set(self, x):
        assert self.pad == 0
        self.memory.upload(encode(x, self.kind))

    def margin_untouched(self):
        return self.pad == 0 or bool(np.all(decode(self.memory.download(), self.kind)[..., self.shape[-1]:] == 77))


@pytest.fixture
def dev(ctx):
    """Makes device tensors that are released at the end of the test."""
    made = []

    def make(x, kind, pad=0):
        made.append(Device(ctx, x, kind, pad))
        return made[-1]

    yield make
    for d in made:
        d.memory.free()


@pytest.fixture(scope="module")
def ops(ctx):
    from superkmeans_amd.rowops import RowOperators

    return RowOperators(ctx=ctx)


def close(out, want, terms, ops, rows=None):
    """|out - want| <= ops * u * terms + h(type) * |value|, values in 64 bits; terms: the sum of the magnitudes added up."""
    got = out.host() if rows is None else out.host()[rows]
    off = ops * U * terms
    bar = off + HALF_STEP[out.kind] * (np.abs(want) + off) + SMALLEST[out.kind] / 2
    wrong = np.abs(got - want) - bar
    assert not np.any(np.isnan(wrong)) and np.all(wrong <= 0), f"off by {np.nanmax(wrong)} more than the bar"

# ---------------------------------------------------------------------------------------------------------------------
# lookup
# ---------------------------------------------------------------------------------------------------------------------

WIDTHS = [1, 2, 3, 8, 17, 64, 100, 257, 1000, 1024, 4104]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", WIDTHS)
def test_lookup(dev, ops, kind, d):
    g = np.random.default_rng(d)
    for n, rows, ids_kind, pad in [(1, 1, "int64", 0), (7, 5, "int32", 3), (130, 1000, "int64", 8), (1000, 33, "int32", 0)]:
        table = typed(g.standard_normal((rows, d)), kind)
        ids = g.integers(-2, rows + 2, n)
        there = (ids >= 0) & (ids < rows)
        want = np.where(there[:, None], table[ids.clip(0, rows - 1)], 0.0)
        on_device, where, out = dev(table, kind, pad), dev(ids, ids_kind), dev(np.full((n, d), 5), kind, pad)
        assert ops.lookup(on_device, where, out) is out
        assert np.array_equal(out.host(), want) and out.margin_untouched()
        ops.lookup(on_device, where, out, scale=0.37)
        want = want * float(np.float32(0.37))
        close(out, want, np.abs(want), 1)


def test_lookup_of_nothing_and_from_nothing(dev, ops):
    ops.lookup(dev(np.ones((4, 8)), "float32"), dev(np.zeros(0), "int64"), dev(np.zeros((0, 8)), "float32"))
    out = dev(np.full((3, 8), 9), "float32")
    ops.lookup(dev(np.zeros((0, 8)), "float32"), dev([0, -1, 5], "int64"), out)
    assert np.all(out.host() == 0)


def test_lookup_carries_infinities_and_nan(dev, ops):
    inf, nan = np.inf, np.nan
    for kind in KINDS:
        table = dev([[inf, 1.0], [nan, -2.0], [3.0, -inf]], kind)
        out = dev(np.zeros((5, 2)), kind)
        for scale in (1.0, 0.5):
            ops.lookup(table, dev([2, -1, 1, 0, 3], "int64"), out, scale=scale)
            want = np.array([[3.0, -inf], [0, 0], [nan, -2.0], [inf, 1.0], [0, 0]]) * scale
            assert np.array_equal(out.host(), want, equal_nan=True)


def test_lookup_past_32_bits_of_elements(ctx, capi, dev, ops):
    """Rows 2^20 elements apart: the last ones lie 10 GB and 5 * 10^9 elements behind the first."""
    rows, d, stride = 5000, 64, 1 << 20
    memory = ctx.empty(rows * stride, np.uint16)
    ids = np.array([4999, 0, 4096, 4998, 2047, 2048])
    want = np.arange(d) + (ids % 100)[:, None]
    for i, row in zip(ids, want):
        block = encode(row, "bfloat16")
        capi.check(ctx.lib.skm_upload(ctx.handle, memory.offset(int(i) * stride), block.ctypes.data, block.nbytes))
    table = dev(np.zeros((1, 1)), "bfloat16")
    table.shape, table._stride, table.data_ptr = (rows, d), (stride, 1), lambda: memory.ptr
    out = dev(np.zeros((6, d)), "bfloat16")
    ops.lookup(table, dev(ids, "int64"), out)
    assert np.array_equal(out.host(), want)
    memory.free()


# ---------------------------------------------------------------------------------------------------------------------
# gradient of the lookup
# ---------------------------------------------------------------------------------------------------------------------


def summed(grad, ids, rows, scale):
    """(sums, sums of magnitudes, most terms of a row) in 64 bits."""
    there = (ids >= 0) & (ids < rows)
    ids, g = ids[there], grad[there]
    sums, sizes = np.zeros((rows, grad.shape[1])), np.zeros((rows, grad.shape[1]))
    np.add.at(sums, ids, g * scale)
    np.add.at(sizes, ids, np.abs(g * scale))
    return sums, sizes, int(np.bincount(ids, minlength=1).max())


def spread_ids(g, n, rows, how):
    if how == "even":
        return g.integers(-1, rows + 1, n)
    if how == "one":
        return np.full(n, rows // 2)
    if how == "none":
        return np.full(n, -1)
    if how == "two runs":  # two long rows next to each other, their border inside a chunk
        return np.where(np.arange(n) % 3 == 0, rows - 1, max(rows - 2, 0))
    return (np.exp(g.random(n) * np.log(rows + 1)) - 1).astype(np.int64).clip(0, rows - 1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("how", ["even", "one", "none", "two runs", "text"])
@pytest.mark.parametrize("n,rows,d", [(1, 1, 1), (5, 3, 7), (63, 40, 8), (64, 1, 100), (257, 300, 130), (2048, 1000, 24),
                                      (2049, 1000, 24), (2049, 3, 257), (5000, 70001, 8), (40000, 2049, 20),
                                      (3000, 1100000, 3), (140000, 500, 5)])
def test_lookup_grad(dev, ops, kind, how, n, rows, d):
    g = np.random.default_rng(n + d)
    grad = typed(g.standard_normal((n, d)), kind)
    ids = spread_ids(g, n, rows, how)
    scale = float(np.float32(0.3))
    want, sizes, most = summed(grad, ids, rows, scale)
    pad = d % 3 * 8
    on_device = dev(grad, kind, pad)
    before = g.standard_normal((rows, d))
    touched = np.zeros(rows, bool)
    touched[ids[(ids >= 0) & (ids < rows)]] = True
    for out_kind in sorted({"float32", kind}):
        for ids_kind in ("int64", "int32"):
            where = dev(ids, ids_kind)
            out = dev(np.full((rows, d), 5), out_kind, pad)
            ops.lookup_grad(on_device, where, out, scale=scale)
            close(out, want, sizes, most + 2)
            assert out.margin_untouched()
            held = typed(before, out_kind)
            out = dev(held, out_kind, pad)
            ops.lookup_grad(on_device, where, out, scale=scale, accumulate=True)
            close(out, want + held, sizes + np.abs(held), most + 3)
            assert np.array_equal(out.host()[~touched], held[~touched])


def test_lookup_grad_of_a_million_tokens(dev, ops):
    """More tiles of the sort than one workgroup adds up, the longest chunks, and rows that thousands of chunks belong to."""
    g = np.random.default_rng(0)
    n, rows, d = 1100000, 40, 2
    grad, ids = typed(g.standard_normal((n, d)), "float16"), spread_ids(g, n, rows, "text")
    out = dev(np.full((rows, d), 5), "float32")
    ops.lookup_grad(dev(grad, "float16"), dev(ids, "int32"), out)
    want, sizes, most = summed(grad, ids, rows, 1.0)
    close(out, want, sizes, most + 2)


def test_lookup_grad_of_nothing(dev, ops):
    out = dev(np.full((5, 4), 3), "float32")
    ops.lookup_grad(dev(np.zeros((0, 4)), "float32"), dev(np.zeros(0), "int32"), out, accumulate=True)
    assert np.all(out.host() == 3)
    ops.lookup_grad(dev(np.zeros((0, 4)), "float32"), dev(np.zeros(0), "int32"), out)
    assert np.all(out.host() == 0)
    ops.lookup_grad(dev(np.ones((3, 4)), "float32"), dev(np.zeros(3), "int32"), dev(np.zeros((0, 4)), "float32"))


def test_lookup_grad_gives_the_same_bits_again(dev, ops):
    g = np.random.default_rng(1)
    grad = dev(g.standard_normal((30000, 96)), "bfloat16")
    ids = dev(spread_ids(g, 30000, 4000, "text"), "int64")
    a, b = dev(np.zeros((4000, 96)), "float32"), dev(np.ones((4000, 96)), "float32")
    ops.lookup_grad(grad, ids, a)
    scratch = dev(np.full(ops.lookup_grad_scratch(30000, 4000, 96), -1), "int8")
    ops.lookup_grad(grad, ids, b, scratch=scratch)
    assert np.array_equal(a.raw(), b.raw())


def test_lookup_grad_is_the_slope_of_the_lookup(dev, ops):
    """<g, lookup(T + D / 2) - lookup(T - D / 2)> == <grad, D>: the lookup is linear, so only fp32 rounding is between them."""
    g = np.random.default_rng(2)
    n, rows, d = 300, 50, 36
    table, way, weight = (typed(g.standard_normal(s), "float32") for s in ((rows, d), (rows, d), (n, d)))
    ids = dev(g.integers(0, rows, n), "int64")
    grad = dev(np.zeros((rows, d)), "float32")
    ops.lookup_grad(dev(weight, "float32"), ids, grad, scale=2.5)
    ends = []
    for h in (0.5, -0.5):
        out = dev(np.zeros((n, d)), "float32")
        ops.lookup(dev(table + h * way, "float32"), ids, out, scale=2.5)
        ends.append((out.host() * weight).sum())
    # n * d products of magnitudes below 5 * 5 * 2.5, each off by a few u
    assert abs(ends[0] - ends[1] - (grad.host() * way).sum()) <= 8 * U * 62.5 * n * d


# ---------------------------------------------------------------------------------------------------------------------
# rows sorted by group and back
# ---------------------------------------------------------------------------------------------------------------------


def routed(choices, groups):
    """(slots, order, offsets) by a stable sort on the host."""
    flat = choices.reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < groups), flat, groups)
    order = np.argsort(key, kind="stable")
    kept = int((key < groups).sum())
    slots = np.full(flat.size, -1, np.int32)
    slots[order[:kept]] = np.arange(kept)
    order = order.astype(np.int32)
    order[kept:] = -1
    offsets = np.searchsorted(np.sort(key), np.arange(groups + 1)).astype(np.int32)
    return slots.reshape(choices.shape), order, offsets


SHAPES = [(1, 1, 1), (1, 8, 64), (3, 2, 5), (64, 8, 64), (171, 6, 1000), (512, 2, 1022), (512, 2, 1023), (1024, 8, 8), (1025, 8, 8),
          (2000, 4, 1024), (5000, 3, 2047), (5000, 3, 2048), (4096, 2, 100000), (70000, 4, 33), (300000, 4, 7),
          (3000, 1, 1048576)]


@pytest.mark.parametrize("n,choices,groups", SHAPES)
def test_route(dev, ops, n, choices, groups):
    g = np.random.default_rng(n + groups)
    for how in ("even", "one", "dropped"):
        c = g.integers(-1, groups + 2, (n, choices))
        if how == "one":
            c[:] = groups - 1
        elif how == "dropped":
            c[:] = -1
        want_slots, want_order, want_offsets = routed(c, groups)
        on_device = dev(c, "int32")
        for with_order in (True, False):
            slots, offsets = dev(np.full((n, choices), 9), "int32"), dev(np.full(groups + 1, 9), "int32")
            order = dev(np.full(n * choices, 9), "int32") if with_order else None
            ops.route(on_device, groups, slots, offsets, order=order)
            assert np.array_equal(slots.raw(), want_slots)
            assert np.array_equal(offsets.raw(), want_offsets)
            if with_order:
                assert np.array_equal(order.raw(), want_order)


def test_route_of_nothing(dev, ops):
    offsets = dev(np.full(5, 9), "int32")
    ops.route(dev(np.zeros((0, 2)), "int32"), 4, dev(np.zeros((0, 2)), "int32"), offsets)
    assert np.all(offsets.raw() == 0)


def test_route_takes_what_knn_answers(capi, ctx, ops):
    """The stage that finds the nearest centroids is the router: k beyond their number leaves slots that are no group."""
    g = np.random.default_rng(3)
    n, groups, d, k = 500, 6, 32, 8
    X, C = g.standard_normal((n, d)).astype(np.float32), g.standard_normal((groups, d)).astype(np.float32)
    dX, dC = ctx.array(X), ctx.array(C)
    xn, cn = ctx.empty(n), ctx.empty(groups)
    idx, dist = ctx.empty((n, k), np.uint32), ctx.empty((n, k))
    slots, offsets = ctx.empty((n, k), np.uint32), ctx.empty(groups + 1, np.uint32)
    rows, back = ctx.array(np.zeros((n * k, d), np.float32)), ctx.empty((n, d))
    capi.check(ctx.lib.skm_norms(ctx.handle, dX.ptr, n, d, d, xn.ptr))
    capi.check(ctx.lib.skm_norms(ctx.handle, dC.ptr, groups, d, d, cn.ptr))
    capi.check(ctx.lib.skm_knn(ctx.handle, dX.ptr, n, dC.ptr, groups, d, xn.ptr, cn.ptr, k, idx.ptr, dist.ptr))
    ops.route(idx, groups, slots, offsets)
    ops.dispatch(dX, slots, rows)
    ops.combine(rows, slots, back)
    assert np.array_equal(offsets.download(), np.arange(groups + 1) * n)  # every row goes to all six centroids
    assert np.array_equal(slots.download() == 0xFFFFFFFF, np.broadcast_to(np.arange(k) >= groups, (n, k)))
    sums = np.zeros((n, d), np.float32)
    for _ in range(groups):
        sums += X
    assert np.array_equal(back.download(), sums)
    for a in (dX, dC, xn, cn, idx, dist, slots, offsets, rows, back):
        a.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [1, 3, 8, 100, 257, 1024, 2056])
@pytest.mark.parametrize("n,choices,groups", [(1, 1, 1), (9, 2, 4), (130, 6, 17), (400, 9, 64)])
def test_rows_to_groups_and_back(dev, ops, kind, d, n, choices, groups):
    g = np.random.default_rng(n + d)
    chosen = g.integers(-1, groups + 1, (n, choices))
    slots, order, offsets = routed(chosen, groups)
    places, kept = n * choices, int(offsets[-1])
    pad = d % 3 * 4
    x = typed(g.standard_normal((n, d)), kind)
    dx, ds, sorted_rows = dev(x, kind, pad), dev(slots, "int32"), dev(np.full((places, d), 5), kind, pad)
    ops.dispatch(dx, ds, sorted_rows)
    want = np.full((places, d), 5.0)
    want[:kept] = x[order[:kept] // choices]
    assert np.array_equal(sorted_rows.host(), want) and sorted_rows.margin_untouched()

    there = slots >= 0
    rows = typed(g.standard_normal((places, d)), kind)
    rows[kept:] = np.nan  # behind the last place: nobody's
    drows = dev(rows, kind, pad)
    picked = np.where(there[..., None], rows[slots.clip(0)], 0.0)
    grad = typed(g.standard_normal((n, d)), kind)
    dgrad = dev(grad, kind, pad)
    for weights_kind in sorted({"float32", kind}):
        weights = typed(g.random((n, choices)), weights_kind)
        weights[~there] = np.nan  # of a dropped choice: not looked at
        dweights = dev(weights, weights_kind)
        w = np.where(there, weights, 0.0)
        out = dev(np.full((n, d), 5), kind, pad)
        ops.combine(drows, ds, out, weights=dweights)
        parts = picked * w[..., None]
        close(out, parts.sum(1), np.abs(parts).sum(1), choices + 1)
        assert out.margin_untouched()

        grad_rows, grad_weights = dev(np.full((places, d), 5), kind, pad), dev(np.full((n, choices), 5), weights_kind)
        ops.combine_grad(dgrad, drows, ds, dweights, grad_rows, grad_weights)
        source = order[:kept]
        value = grad[source // choices] * w.reshape(-1)[source][:, None]
        close(grad_rows, value, np.abs(value), 1, rows=slice(0, kept))
        assert np.all(grad_rows.host()[kept:] == 5) and grad_rows.margin_untouched()
        products = picked * grad[:, None, :]
        close(grad_weights, products.sum(-1), np.abs(products).sum(-1), d + 1)
        # one output at a time gives the same
        alone = dev(np.full((places, d), 5), kind)
        ops.combine_grad(dgrad, None, ds, dweights, alone, None)
        assert np.array_equal(alone.raw(), grad_rows.raw())
        alone = dev(np.zeros((n, choices)), weights_kind)
        ops.combine_grad(dgrad, drows, ds, dweights, None, alone)
        assert np.array_equal(alone.raw(), grad_weights.raw())
    out = dev(np.full((n, d), 5), kind)
    ops.combine(drows, ds, out)
    close(out, picked.sum(1), np.abs(picked).sum(1), choices)


def test_slots_outside_the_rows_are_not_followed(dev, ops):
    """Slots are data: places past the last row given count as no place."""
    slots = dev([[0, 7], [-2, 3], [2 ** 31 - 1, 1]], "int32")
    x = np.arange(12.0).reshape(3, 4)
    dx, out, back, dots, rows = (dev(v, "float32") for v in (x, np.full((3, 4), -1), np.zeros((3, 4)), np.zeros((3, 2)), np.full((3, 4), -1)))
    ops.dispatch(dx, slots, out)
    assert np.array_equal(out.host(), np.stack([x[0], x[2], np.full(4, -1.0)]))
    ops.combine(dx, slots, back)
    assert np.array_equal(back.host(), np.stack([x[0], np.zeros(4), x[1]]))
    ops.combine_grad(dx, dx, slots, dev(np.ones((3, 2)), "float32"), rows, dots)
    assert np.array_equal(rows.host(), out.host())
    assert np.array_equal(dots.host(), [[14.0, 0], [0, 0], [0, 8 * 4 + 9 * 5 + 10 * 6 + 11 * 7]])


def test_combine_gradients_are_its_slopes(dev, ops):
    """combine is linear in the rows and in the weights: differences over a long step show only fp32 rounding."""
    g = np.random.default_rng(5)
    n, k, groups, d = 60, 3, 7, 44
    slots = dev(routed(g.integers(-1, groups, (n, k)), groups)[0], "int32")
    rows, way, grad = (typed(g.standard_normal(s), "float32") for s in ((n * k, d), (n * k, d), (n, d)))
    weights, weights_way = typed(g.random((n, k)), "float32"), typed(g.random((n, k)), "float32")
    grad_rows, grad_weights = dev(np.zeros((n * k, d)), "float32"), dev(np.zeros((n, k)), "float32")
    ops.combine_grad(dev(grad, "float32"), dev(rows, "float32"), slots, dev(weights, "float32"), grad_rows, grad_weights)

    def value(r, w):
        out = dev(np.zeros((n, d)), "float32")
        ops.combine(dev(r, "float32"), slots, out, weights=dev(w, "float32"))
        return (out.host() * grad).sum()

    bar = 16 * U * 25 * n * k * d  # products of magnitudes below 5 * 5, a few operations each
    slope = value(rows + 0.5 * way, weights) - value(rows - 0.5 * way, weights)
    assert abs(slope - (grad_rows.host() * way).sum()) <= bar
    slope = value(rows, weights + 0.5 * weights_way) - value(rows, weights - 0.5 * weights_way)
    assert abs(slope - (grad_weights.host() * weights_way).sum()) <= bar


# ---------------------------------------------------------------------------------------------------------------------
# 8-bit rows
# ---------------------------------------------------------------------------------------------------------------------


def steps(x):
    """(q, scales) of rows in 64 bits, by the definition."""
    most = np.abs(x).max(1)
    with np.errstate(all="ignore"):
        q = np.rint(127 * x / most[:, None])
        usable = np.isfinite(most) & (most > 0)
        return np.where(usable[:, None], q, 0), np.where(np.isfinite(most), most / 127, np.nan)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [1, 3, 8, 64, 100, 1000, 2049, 4096, 20000])
def test_quantize(dev, ops, kind, d):
    g = np.random.default_rng(d)
    x = g.standard_normal((37, d))
    x[0] = 0
    x[1] *= 1e-3
    x[2, d // 2] = 100.0
    x[3] = np.arange(d) % 64 - 31.5
    x[4, 0], x[4, d - 1] = 2.0, 1.0  # 63.5: a tie, where d > 1
    x[5, d // 3] = np.inf
    x[6, d - 1] = np.nan
    x[7] = SMALLEST[kind] * g.integers(-9, 10, d)
    x = typed(x, kind)
    want_q, want_scales = steps(x)
    pad = d % 3 * 16
    q, scales = dev(np.full((37, d), 5), "int8", pad), dev(np.zeros(37), "float32")
    ops.quantize(dev(x, kind, pad), q, scales)
    assert np.array_equal(q.raw(), want_q) and q.margin_untouched()
    got = scales.host()
    assert np.array_equal(np.isnan(got), np.isnan(want_scales))
    fine = ~np.isnan(got)
    assert np.all(np.abs(got[fine] - want_scales[fine]) <= U * want_scales[fine] + 2.0 ** -150)


def test_quantize_decides_at_the_borders_like_64_bits(dev, ops):
    """Rows made of the fp32 numbers around the borders between two steps, where a quotient in fp32 goes either way."""
    g = np.random.default_rng(0)
    d = 2048
    most = g.uniform(0.5, 2, 64).astype(np.float32)
    border = ((g.integers(-126, 126, (64, d)) + 0.5) / 127 * most[:, None].astype(np.float64)).astype(np.float32)
    aside = np.nextafter(border, np.where(g.random((64, d)) < 0.5, np.float32(9), np.float32(-9)))
    x = np.where(g.random((64, d)) < 0.5, border, aside)
    x[:, 0] = most
    q = dev(np.zeros((64, d)), "int8")
    ops.quantize(dev(x, "float32"), q, dev(np.zeros(64), "float32"))
    assert np.array_equal(q.raw(), steps(x.astype(np.float64))[0])


PRODUCTS = [(1, 1, 1), (1, 5, 3), (2, 64, 64), (3, 17, 100), (16, 256, 128), (17, 130, 1000), (33, 1000, 272), (64, 64, 2048),
            (100, 300, 516), (129, 257, 1040), (300, 520, 64), (1, 1024, 4096), (8, 2000, 1024), (512, 512, 512), (257, 1023, 769),
            (300, 64, 15), (5, 6, 16), (300, 300, 31), (70, 33, 129), (250, 2048, 80), (100, 2048, 144), (40, 1000, 96), (1000, 1000, 100), (1000, 2048, 160),
            (2048, 2040, 176)]


def product_of(a, a_scales, b, b_scales, bias):
    """(value, magnitude) in 64 bits."""
    value = (a.astype(np.float64) @ b.astype(np.float64).T) * a_scales[:, None] * b_scales
    shift = 0 if bias is None else bias
    return value + shift, np.abs(value) + np.abs(shift)


@pytest.mark.parametrize("out_kind", KINDS)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(dev, ops, out_kind, m, n, k):
    g = np.random.default_rng(m + n + k)
    for pad, with_bias in ((0, False), (k % 5 + 1, True)):
        a, b = g.integers(-128, 128, (m, k)), g.integers(-128, 128, (n, k))
        a_scales, b_scales = typed(g.random(m) * 0.01, "float32"), typed((g.random(n) - 0.5) * 0.01, "float32")
        bias = typed(g.standard_normal(n), "float32") if with_bias else None
        out = dev(np.full((m, n), 5), out_kind, pad)
        ops.product(dev(a, "int8", pad), dev(a_scales, "float32"), dev(b, "int8", pad), dev(b_scales, "float32"), out,
                    bias=None if bias is None else dev(bias, "float32"))
        want, size = product_of(a, a_scales, b, b_scales, bias)
        close(out, want, size, 4)  # the sum's rounding to fp32, two products, the bias
        assert out.margin_untouched()


@pytest.mark.parametrize("out_kind", ["float32", "bfloat16"])
def test_product_of_a_long_prompt(dev, ops, out_kind):
    """Whole and partial tiles of the largest shape, with columns that end inside a stage."""
    g = np.random.default_rng(9)
    m, n, k = 4093, 4090, 1000
    a, b = g.integers(-128, 128, (m, k)), g.integers(-128, 128, (n, k))
    a_scales, b_scales = typed(g.random(m) * 0.01, "float32"), typed(g.random(n) * 0.01, "float32")
    out = dev(np.full((m, n), 5), out_kind)
    ops.product(dev(a, "int8"), dev(a_scales, "float32"), dev(b, "int8"), dev(b_scales, "float32"), out)
    want, size = product_of(a, a_scales, b, b_scales, None)
    close(out, want, size, 4)


def test_product_with_rows_far_apart(capi, ctx, dev, ops):
    """Rows of a 2^24 bytes apart: past the 32-bit offsets that the tiles' loads use."""
    m, n, k, stride = 300, 300, 64, 1 << 24
    g = np.random.default_rng(1)
    a, b = g.integers(-128, 128, (m, k)).astype(np.int8), g.integers(-128, 128, (n, k))
    memory = ctx.empty(m * stride, np.int8)
    for i in range(m):
        capi.check(ctx.lib.skm_upload(ctx.handle, memory.offset(i * stride), a[i].ctypes.data, k))
    da = dev(np.zeros((1, 1)), "int8")
    da.shape, da._stride, da.data_ptr = (m, k), (stride, 1), lambda: memory.ptr
    ones, out = dev(np.ones(300), "float32"), dev(np.zeros((m, n)), "float32")
    ops.product(da, ones, dev(b, "int8"), ones, out)
    assert np.array_equal(out.host(), a.astype(np.float64) @ b.T)
    memory.free()


def test_product_of_the_largest_values(dev, ops):
    """131,071 products of -128 and -128 are 2^31 - 2^14: the sum does not wrap."""
    k = 131071
    a, one, out = dev(np.full((3, k), -128), "int8"), dev(np.ones(3), "float32"), dev(np.zeros((3, 3)), "float32")
    ops.product(a, one, dev(np.full((3, k), -128), "int8"), one, out)
    assert np.all(out.host() == float(np.float32(128.0 * 128 * k)))


@pytest.mark.parametrize("out_kind", KINDS)
@pytest.mark.parametrize("m,n,k,sizes", [
    (1, 8, 16, [1]), (5, 17, 100, [0, 5, 0]), (60, 300, 64, [1, 0, 20, 3, 16, 17]), (500, 130, 256, [0, 129, 128, 1, 0, 200]),
    (64, 1024, 512, [1] * 64), (700, 257, 528, [350, 0, 350]), (3, 40, 33, [0, 0, 0]), (200, 96, 144, [2] * 100), (90, 64, 64, [33, 32, 25]),
    (1500, 520, 320, [700, 0, 513, 256]), (300, 64, 32, [0] * 70 + [1] * 100 + [0] * 5000 + [100, 0, 64]), (2100, 2048, 64, [600, 500, 0, 1000]),
    (1000, 600, 80, [9, 11, 0, 30] * 20),
])
def test_product_of_groups(dev, ops, out_kind, m, n, k, sizes):
    g = np.random.default_rng(m + n)
    groups = len(sizes)
    offsets = np.concatenate([[0], np.cumsum(sizes)])
    for pad in (0, 3, 16):
        a, b = g.integers(-128, 128, (m, k)), g.integers(-128, 128, (groups, n, k))
        a_scales, b_scales = typed(g.random(m) * 0.01, "float32"), typed(g.random((groups, n)) * 0.01, "float32")
        bias = typed(g.standard_normal((groups, n)), "float32") if pad else None
        out = dev(np.full((m, n), 5), out_kind, pad)
        ops.product(dev(a, "int8", pad), dev(a_scales, "float32"), dev(b, "int8", pad), dev(b_scales, "float32"), out,
                    bias=None if bias is None else dev(bias, "float32"), offsets=dev(offsets, "int32"))
        for e in range(groups):
            i, j = offsets[e], offsets[e + 1]
            if i < j:
                want, size = product_of(a[i:j], a_scales[i:j], b[e], b_scales[e], None if bias is None else bias[e])
                close(out, want, size, 4, rows=slice(i, j))
        assert np.all(out.host()[offsets[-1]:] == 5) and out.margin_untouched()


def test_offsets_past_the_rows_are_clamped(dev, ops):
    """Offsets are data: rows beyond those given are not touched, a group that ends before it begins is empty."""
    a = dev(np.ones((4, 32)), "int8")
    b = dev(np.arange(1, 4)[:, None, None] * np.ones((3, 16, 32)), "int8")
    ones, scales = dev(np.ones(4), "float32"), dev(np.ones((3, 16)), "float32")
    for offsets, want in (([0, 2, 1, 900], {0: 1, 2: 3, 3: 3}), ([-1, 2, 3, 4], {0: 0, 1: 0, 2: 2, 3: 3})):
        out = dev(np.zeros((4, 16)), "float32")
        ops.product(a, ones, b, scales, out, offsets=dev(offsets, "int32"))
        # a malformed table may name a row twice (row 1 of the first): either product is an answer
        for row, value in want.items():
            assert np.all(out.host()[row] == value * 32)


def test_groups_that_begin_behind_the_first_row(dev, ops):
    """A part of a larger table of offsets: rows before its first group and behind its last one are nobody's."""
    g = np.random.default_rng(4)
    m, n, k, offsets = 700, 300, 64, [5, 5, 90, 91, 600]
    a, b = g.integers(-128, 128, (m, k)), g.integers(-128, 128, (4, n, k))
    ones, out = dev(np.ones(m), "float32"), dev(np.full((m, n), 5), "float32")
    ops.product(dev(a, "int8"), ones, dev(b, "int8"), dev(np.ones((4, n)), "float32"), out, offsets=dev(offsets, "int32"))
    want = np.full((m, n), 5.0)
    for e in range(4):
        rows = slice(offsets[e], offsets[e + 1])
        want[rows] = a[rows].astype(np.float64) @ b[e].T
    assert np.array_equal(out.host(), want)


def test_products_of_rows_that_hold_nan_are_nan(dev, ops):
    x = np.ones((3, 64))
    x[1, 5], x[2, 0] = np.nan, -np.inf
    q, s, out = dev(np.zeros((3, 64)), "int8"), dev(np.zeros(3), "float32"), dev(np.zeros((3, 8)), "float32")
    ops.quantize(dev(x, "float32"), q, s)
    ops.product(q, s, dev(np.ones((8, 64)), "int8"), dev(np.ones(8), "float32"), out)
    assert np.allclose(out.host()[0], 64, rtol=4 * U) and np.all(np.isnan(out.host()[1:]))


@pytest.mark.parametrize("d", [1048573, 131072])
def test_the_longest_rows(dev, ops, d):
    g = np.random.default_rng(d)
    table = typed(g.standard_normal((3, d)), "bfloat16")
    ids, slots = np.array([2, -1, 0, 2]), np.array([[1, 2], [-1, 0], [3, -1], [-1, -1]])
    x, rows, out = dev(np.zeros((4, d)), "bfloat16"), dev(np.zeros((4, d)), "bfloat16"), dev(np.zeros((4, d)), "bfloat16")
    ops.lookup(dev(table, "bfloat16"), dev(ids, "int64"), x)
    want = np.where((ids >= 0)[:, None], table[ids.clip(0)], 0)
    assert np.array_equal(x.host(), want)
    ds, weights = dev(slots, "int32"), typed(g.random((4, 2)), "float32")
    ops.dispatch(x, ds, rows)
    places = want[[1, 0, 0, 2]]
    assert np.array_equal(rows.host(), places)
    ops.combine(rows, ds, out, weights=dev(weights, "float32"))
    picked = np.where((slots >= 0)[..., None], places[slots.clip(0)], 0)
    parts = picked * weights[..., None]
    close(out, parts.sum(1), np.abs(parts).sum(1), 3)
    dots = dev(np.zeros((4, 2)), "float32")
    ops.combine_grad(x, rows, ds, dev(weights, "float32"), None, dots)
    products = picked * want[:, None]
    close(dots, products.sum(-1), np.abs(products).sum(-1), d)
    grad = dev(np.zeros((3, d)), "float32")
    ops.lookup_grad(x, dev(ids, "int64"), grad)
    sums, sizes, most = summed(want, ids, 3, 1.0)
    close(grad, sums, sizes, most + 2)
    q, scales = dev(np.zeros((4, d)), "int8"), dev(np.zeros(4), "float32")
    ops.quantize(x, q, scales)
    assert np.array_equal(q.raw(), steps(want)[0])


# ---------------------------------------------------------------------------------------------------------------------
# together, on streams, in graphs
# ---------------------------------------------------------------------------------------------------------------------


class Layer:
    """Tokens looked up, sent to k of the experts, through their 8-bit matrices, and back; buffers and scratch kept."""

    def __init__(self, dev, g, n, vocabulary, d, f, experts, k, with_scratch_of=None):
        self.n, self.vocabulary, self.d, self.f, self.experts, self.k = n, vocabulary, d, f, experts, k
        self.table = typed(g.standard_normal((vocabulary, d)), "bfloat16")
        self.w = g.integers(-127, 128, (experts, f, d))
        self.w_scales = typed(g.random((experts, f)) * 1e-3, "float32")
        self.t = {name: dev(np.zeros(shape), kind) for name, shape, kind in [
            ("ids", (n,), "int64"), ("choices", (n, k), "int32"), ("shares", (n, k), "float32"), ("grad", (n, f), "bfloat16"),
            ("x", (n, d), "bfloat16"), ("rows", (n * k, d), "bfloat16"), ("q", (n * k, d), "int8"), ("q_scales", (n * k,), "float32"),
            ("y", (n * k, f), "bfloat16"), ("out", (n, f), "bfloat16"), ("slots", (n, k), "int32"), ("offsets", (experts + 1,), "int32"),
            ("grad_y", (n * k, f), "bfloat16"), ("grad_shares", (n, k), "float32"), ("grad_table", (vocabulary, d), "float32")]}
        self.t |= {"table": dev(self.table, "bfloat16"), "w": dev(self.w, "int8"), "w_scales": dev(self.w_scales, "float32")}
        self.scratch = None
        if with_scratch_of is not None:
            o = with_scratch_of
            self.scratch = dev(np.zeros(max(16, o.route_scratch(n, k, experts), o.lookup_grad_scratch(n, vocabulary, d))), "int8")

    def set(self, g):
        self.ids = g.integers(-1, self.vocabulary, self.n)
        self.choices = np.argsort(g.random((self.n, self.experts)), axis=1)[:, : self.k]
        self.shares = typed(g.random((self.n, self.k)), "float32")
        self.grad = typed(g.standard_normal((self.n, self.f)), "bfloat16")
        for name in ("ids", "choices", "shares", "grad"):
            self.t[name].set(getattr(self, name))
        for name in ("out", "grad_shares", "grad_table"):
            self.t[name].set(np.full(self.t[name].shape, np.nan))

    def run(self, ops):
        t = self.t
        ops.lookup(t["table"], t["ids"], t["x"], scale=0.5)
        ops.route(t["choices"], self.experts, t["slots"], t["offsets"], scratch=self.scratch)
        ops.dispatch(t["x"], t["slots"], t["rows"])
        ops.quantize(t["rows"], t["q"], t["q_scales"])
        ops.product(t["q"], t["q_scales"], t["w"], t["w_scales"], t["y"], offsets=t["offsets"])
        ops.combine(t["y"], t["slots"], t["out"], weights=t["shares"])
        ops.combine_grad(t["grad"], t["y"], t["slots"], t["shares"], t["grad_y"], t["grad_shares"])
        ops.lookup_grad(t["x"], t["ids"], t["grad_table"], scratch=self.scratch)

    def check(self):
        x = np.where((self.ids >= 0)[:, None], self.table[self.ids.clip(0)] * 0.5, 0.0)  # halves: exact
        q, s = steps(x)
        w = self.w * self.w_scales[..., None]
        h = HALF_STEP["bfloat16"]
        out, size, dots, sizes = 0, 0, [], []
        for j in range(self.k):
            y = np.zeros((self.n, self.f))
            for e in range(self.experts):
                at = self.choices[:, j] == e
                y[at] = (q[at] @ w[e].T) * s[at, None]
            out, size = out + y * self.shares[:, j, None], size + np.abs(y) * self.shares[:, j, None]
            dots.append((y * self.grad).sum(1))
            sizes.append(np.abs(y * self.grad).sum(1))
        # y is rounded to bfloat16 once (h), the sums add k + 6 roundings of fp32, the result is rounded once more
        bar = size * (h + (self.k + 6) * U) * (1 + h) + h * np.abs(out) + 1e-30
        assert np.all(np.abs(self.t["out"].host() - out) <= bar)
        bar = np.stack(sizes, 1) * (h + (self.f + 6) * U) * (1 + U) + 1e-30
        assert np.all(np.abs(self.t["grad_shares"].host() - np.stack(dots, 1)) <= bar)
        sums, sizes, most = summed(x, self.ids, self.vocabulary, 1.0)
        close(self.t["grad_table"], sums, sizes, most + 2)


@pytest.mark.parametrize("n,experts,k,d,f", [(1, 4, 2, 64, 48), (50, 16, 4, 128, 96), (3000, 8, 2, 72, 40), (6000, 8, 3, 64, 64)])
def test_a_layer_of_experts(dev, ops, n, experts, k, d, f):
    g = np.random.default_rng(n)
    layer = Layer(dev, g, n, 200, d, f, experts, k)
    for _ in range(2):
        layer.set(g)
        layer.run(ops)
        layer.check()


class Hip:
    """The stream and graph calls of the HIP runtime that the library is linked with."""

    def __init__(self):
        self.lib = ctypes.CDLL("libamdhip64.so.7")

    def __getattr__(self, name):
        fn = getattr(self.lib, name)

        def call(*args):
            rc = fn(*args)
            assert rc == 0, f"{name} gave {rc}"

        return call

    def stream(self):
        s = ctypes.c_void_p()
        self.hipStreamCreate(ctypes.byref(s))
        return s

    def capture(self, stream, work):
        """An executable graph of what `work` queues on the stream."""
        graph, executable = ctypes.c_void_p(), ctypes.c_void_p()
        self.hipStreamBeginCapture(stream, 0)  # global mode
        try:
            work()
        finally:
            self.hipStreamEndCapture(stream, ctypes.byref(graph))
        self.hipGraphInstantiate(ctypes.byref(executable), graph, None, None, ctypes.c_size_t(0))
        self.hipGraphDestroy(graph)
        return executable


@pytest.fixture(scope="module")
def hip(ctx):
    return Hip()


def test_a_stream_of_the_caller_s(hip, dev):
    """Calls on the caller's stream; the object leaves the stream behind in working order."""
    from superkmeans_amd.rowops import RowOperators

    stream = hip.stream()
    g = np.random.default_rng(0)
    for _ in range(2):
        with RowOperators(device=0, stream=stream.value) as ops:
            layer = Layer(dev, g, 400, 100, 64, 64, 8, 2)
            layer.set(g)
            layer.run(ops)
            hip.hipStreamSynchronize(stream)  # the caller's own wait
            layer.check()
    with RowOperators(device=0, stream=0) as ops:  # the default stream
        layer.set(g)
        layer.run(ops)
        ops.sync()
        layer.check()
    hip.hipStreamDestroy(stream)


def test_two_graphs_and_eager_calls_between(hip, ctx, dev):
    """Two captured layers with scratch of their own, replayed in turn with new inputs and eager work between the replays."""
    from superkmeans_amd.rowops import RowOperators

    g = np.random.default_rng(1)
    stream = hip.stream()
    with RowOperators(device=0, stream=stream.value) as ops:
        layers = [Layer(dev, g, n, 150, 64, 96, 8, 2, with_scratch_of=ops) for n in (40, 9000)]
        graphs = []
        for layer in layers:
            layer.set(g)
            layer.run(ops)
            ops.sync()
            layer.check()
            graphs.append(hip.capture(stream, lambda: layer.run(ops)))
        eager = Layer(dev, g, 5000, 150, 64, 96, 8, 2)
        for _ in range(4):
            for layer, graph in zip(layers, graphs):
                layer.set(g)
                hip.hipGraphLaunch(graph, stream)
                ops.sync()
                layer.check()
                eager.set(g)
                eager.run(ops)
                ops.sync()
                eager.check()
        # both queued before either is waited for
        for layer in layers:
            layer.set(g)
        for graph in graphs:
            hip.hipGraphLaunch(graph, stream)
        ops.sync()
        for layer in layers:
            layer.check()
        for graph in graphs:
            hip.hipGraphExecDestroy(graph)
    hip.hipStreamDestroy(stream)


def test_a_captured_call_brings_its_scratch(hip, dev):
    from superkmeans_amd.rowops import RowOperators

    stream = hip.stream()
    with RowOperators(device=0, stream=stream.value) as ops:
        n = 20000
        choices, slots, offsets = dev(np.zeros((n, 2)), "int32"), dev(np.zeros((n, 2)), "int32"), dev(np.zeros(9), "int32")
        few = dev(np.zeros((4, 2)), "int32")

        def work():
            with pytest.raises(ValueError, match="scratch"):
                ops.route(choices, 8, slots, offsets)
            ops.route(few, 8, dev_few, offsets)  # few choices need no scratch

        dev_few = dev(np.zeros((4, 2)), "int32")
        graph = hip.capture(stream, work)
        hip.hipGraphLaunch(graph, stream)
        ops.sync()
        assert np.array_equal(offsets.raw(), [0] + [8] * 8)
        hip.hipGraphExecDestroy(graph)
    hip.hipStreamDestroy(stream)


WITH_TORCH = """
import torch
from superkmeans_amd.rowops import RowOperators
assert torch.cuda.is_available()
torch.manual_seed(0)
n, k, groups, d = 3000, 2, 8, 96
x = torch.randn((n, d), device="cuda").to(torch.bfloat16)
side = torch.cuda.Stream()
for stream in (torch.cuda.current_stream(), side):
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), RowOperators(device=0, stream=stream.cuda_stream) as ops:
        # queued behind torch's own work on the stream, and before more of it, without a wait
        choices = torch.rand((n, groups), device="cuda").topk(k, 1).indices.to(torch.int32)
        slots, offsets = torch.empty_like(choices), torch.empty(groups + 1, dtype=torch.int32, device="cuda")
        rows, out = torch.empty((n * k, d), dtype=x.dtype, device="cuda"), torch.empty_like(x)
        scratch = torch.empty(ops.route_scratch(n, k, groups) + 16, dtype=torch.uint8, device="cuda")
        def work():
            ops.route(choices, groups, slots, offsets, scratch=scratch)
            ops.dispatch(x, slots, rows)
            rows.mul_(2)
            ops.combine(rows, slots, out, weights=shares)
        shares = torch.full((n, k), 0.25, device="cuda")
        work()
        ok = torch.equal(out, x) & torch.equal(offsets[1:] - offsets[:-1], torch.bincount(choices.reshape(-1), minlength=groups).int())
        assert ok
        if stream is side:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                work()
            for _ in range(3):
                choices.copy_(torch.rand((n, groups), device="cuda").topk(k, 1).indices)
                out.zero_()
                graph.replay()
                assert torch.equal(out, x)
        torch.cuda.synchronize()
for bad in (lambda o: o.dispatch(x.cpu(), slots, rows), lambda o: o.dispatch(x.t(), slots, rows), lambda o: o.dispatch(x.double(), slots, rows)):
    with RowOperators() as ops:
        try:
            bad(ops)
        except (TypeError, ValueError):
            continue
        raise AssertionError("not refused")
print("with torch: ok")
"""


def test_torch_tensors_streams_and_graphs():
    """In a process of its own: torch brings a HIP runtime, which has to be the first one that a process loads."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", WITH_TORCH], cwd=root, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "with torch: ok" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


def test_refusals_of_the_library(dev, ops, capi):
    """What the C entries refuse on their own, each with SKM_ERR_INVALID and before anything is queued."""
    lib, h = ops.ctx.lib, ops.ctx.handle
    x = dev(np.zeros(4096), "float32")
    p = x.data_ptr()
    far = p + 8192
    bad = {
        "type": lambda: lib.skm_lookup_rows(h, p, 9, 4, 4, 4, p, 3, 2, 1.0, far, 4),
        "ids type": lambda: lib.skm_lookup_rows(h, p, 0, 4, 4, 4, p, 0, 2, 1.0, far, 4),
        "stride": lambda: lib.skm_lookup_rows(h, p, 0, 4, 4, 3, p, 3, 2, 1.0, far, 4),
        "null table": lambda: lib.skm_lookup_rows(h, None, 0, 4, 4, 4, p, 3, 2, 1.0, far, 4),
        "unaligned": lambda: lib.skm_lookup_rows(h, p + 2, 0, 4, 4, 4, p, 3, 2, 1.0, far, 4),
        "no columns": lambda: lib.skm_lookup_rows(h, p, 0, 4, 0, 4, p, 3, 2, 1.0, far, 4),
        "in place": lambda: lib.skm_lookup_rows(h, p, 0, 4, 4, 4, far, 3, 2, 1.0, p + 16, 4),
        "gradient's type": lambda: lib.skm_lookup_rows_grad(h, p, 1, 4, p, 3, 2, 4, 4, 1.0, far, 2, 4, 0, None, 0),
        "little scratch": lambda: lib.skm_lookup_rows_grad(h, p, 1, 1, p, 3, 4000, 4, 1, 1.0, far + 128, 1, 1, 0, far, 64),
        "unaligned scratch": lambda: lib.skm_route(h, p, 2000, 1, 2000, far, None, far, p + 4, 1 << 40),
        "no groups": lambda: lib.skm_route(h, p, 2, 2, 0, far, None, far, None, 0),
        "no choices": lambda: lib.skm_route(h, p, 2, 0, 4, far, None, far, None, 0),
        "route in place": lambda: lib.skm_route(h, p, 2, 2, 4, p, None, far, None, 0),
        "dispatch in place": lambda: lib.skm_dispatch_rows(h, p, 0, 4, 4, 4, far, 1, p, 4, 4),
        "combine in place": lambda: lib.skm_combine_rows(h, p, 0, 4, 4, 4, far, 4, 1, None, 0, p, 4),
        "weights' type": lambda: lib.skm_combine_rows(h, p, 0, 4, 4, 4, far, 4, 1, p, 7, far + 256, 4),
        "no gradient asked": lambda: lib.skm_combine_rows_grad(h, p, 0, 4, 4, 4, p, 4, 4, far, 1, p, 0, None, 4, None),
        "quantize stride": lambda: lib.skm_quantize_rows(h, p, 0, 4, 8, 8, far, 4, far + 64),
        "product k": lambda: lib.skm_product_i8(h, p, 1, 1 << 20, p, p, 1, 1 << 20, 1 << 20, p, None, 0, 0, None, far, 0, 1),
        "product groups": lambda: lib.skm_product_i8(h, p, 2, 8, p, p, 2, 8, 8, p, None, 0, 16, p, far, 0, 2),
        "product overlapping groups": lambda: lib.skm_product_i8(h, p, 2, 8, p, p, 2, 8, 8, p, None, 2, 8, p, far, 0, 2),
        "product in place": lambda: lib.skm_product_i8(h, p, 2, 8, p, far, 2, 8, 8, far, None, 0, 0, None, p, 0, 2),
        "product over its scales": lambda: lib.skm_product_i8(h, p, 2, 8, far + 64, p, 2, 8, 8, p, None, 0, 0, None, far, 0, 32),
        "route over its slots": lambda: lib.skm_route(h, p, 2, 2, 4, far, far, far + 64, None, 0),
        "weights in place": lambda: lib.skm_combine_rows_grad(h, p, 0, 4, 4, 4, p, 4, 4, far, 1, far + 256, 0, None, 4, far + 256),
        "product out unaligned": lambda: lib.skm_product_i8(h, p, 2, 8, p, p, 2, 8, 8, p, None, 0, 0, None, far + 2, 0, 2),
    }
    for what, call in bad.items():
        assert call() == capi.SKM_ERR_INVALID, what
        assert lib.skm_last_error(), what
    ops.sync()
    assert np.all(x.host() == 0)


# ---------------------------------------------------------------------------------------------------------------------
# sizes past one launch
# ---------------------------------------------------------------------------------------------------------------------


class Block:
    """A contiguous tensor too large to keep on the host, filled with one 32-bit word; parts of it can be read and set."""

    def __init__(self, capi, ctx, shape, kind, word):
        self.capi, self.ctx, self.shape, self.dtype, self.kind = capi, ctx, shape, kind, kind
        size = int(np.prod(shape, dtype=np.int64))
        self.raw_type = np.dtype(RAW.get(kind, kind))
        self.memory = ctx.empty((size + 7) // 4 * 4, self.raw_type)  # whole words, some behind the last element
        capi.check(ctx.lib.skm_fill_u32(ctx.handle, self.memory.ptr, word, self.memory.nbytes // 4))

    def stride(self):
        steps, step = [], 1
        for size in reversed(self.shape):
            steps.insert(0, step)
            step *= size
        return tuple(steps)

    def data_ptr(self):
        return self.memory.ptr

    def part(self, first, count):
        """`count` elements from the given one on."""
        out = np.empty(count, self.raw_type)
        self.capi.check(self.ctx.lib.skm_download(self.ctx.handle, out.ctypes.data, self.memory.offset(first), out.nbytes))
        return decode(out, self.kind)

    def put(self, first, x):
        block = np.ascontiguousarray(encode(x, self.kind))
        self.capi.check(self.ctx.lib.skm_upload(self.ctx.handle, self.memory.offset(first), block.ctypes.data, block.nbytes))


@pytest.fixture
def block(capi, ctx):
    made = []

    def make(shape, kind, word=0):
        made.append(Block(capi, ctx, shape, kind, word))
        return made[-1]

    yield make
    for b in made:
        b.memory.free()
    ctx.lib.skm_device_cache_trim(0)


@pytest.mark.parametrize("n", [5, 3000])
@pytest.mark.parametrize("rows", [2 ** 29 + 195, 2 ** 30 + 100, 2 ** 32 - 2])
def test_lookup_grad_of_more_rows_than_a_launch_has_threads(dev, block, ops, n, rows):
    """A launch has fewer than 2^32 threads: 2^24 workgroups of 256, each for 64 rows, or 2^23 of 512."""
    g = np.random.default_rng(n)
    places = np.unique(np.concatenate([[0, 1, rows // 2, rows - 2, rows - 1], g.integers(0, rows, 20)]))
    ids = np.resize(places, n)
    grad = g.integers(-2, 3, (n, 1))  # sums of up to 600 of them are whole numbers that every type has
    out = block((rows, 1), "float16", 0x3C003C00)  # ones
    ops.lookup_grad(dev(grad, "float16"), dev(ids, "int64"), out)
    window = 1 << 20
    for at in sorted({0, rows - window, *(int(v) for v in (np.clip(places - window // 2, 0, rows - window)))}):
        want = np.zeros(window)
        inside = (ids >= at) & (ids < at + window)
        np.add.at(want, ids[inside] - at, grad[inside, 0])
        assert np.array_equal(out.part(at, window), want)


def test_product_of_more_rows_than_a_launch_has_threads(dev, block, ops):
    """Rows too short for the tiles' loads: 2^23 workgroups of 512 threads and one more."""
    m, n, k = 2 ** 28 + 5, 8, 8
    g = np.random.default_rng(0)
    a, a_scales, out = block((m, k), "int8", 0x01010101), block((m,), "float32", 0x3F800000), block((m, n), "bfloat16", 0)
    b = g.integers(-3, 4, (n, k))
    windows = [0, m // 2 - 50, 2 ** 27, m - 100]
    for at in windows:
        a.put(at * k, np.full((100, k), at % 5 + 1) * (np.arange(100) % 3 - 1)[:, None])
    ops.product(a, a_scales, dev(b, "int8"), dev(np.ones(n), "float32"), out)
    for at in windows:
        rows = a.part(at * k, 100 * k).reshape(100, k)  # as they are now: two of the windows share rows
        assert np.array_equal(out.part(at * n, 100 * n).reshape(100, n), rows @ b.T)
    assert np.array_equal(out.part((m // 4) * n, 100 * n).reshape(100, n), np.tile(b.sum(1), (100, 1)))


def test_product_of_more_tiles_than_a_launch_has_threads(dev, block, ops):
    """65,536 groups of nine rows: 17 million tiles of 64 x 64, 256 threads each."""
    groups, each, n, k = 65536, 9, 14400, 16
    m = groups * each
    g = np.random.default_rng(0)
    a = g.integers(-4, 5, (m, k))
    b, b_scales, out = block((groups, n, k), "int8", 0x01010101), block((groups, n), "float32", 0x3F800000), block((m, n), "bfloat16", 0)
    ops.product(dev(a, "int8"), dev(np.ones(m), "float32"), b, b_scales, out, offsets=dev(np.arange(groups + 1) * each, "int32"))
    for at in (0, m // 3, m // 2 + 7, m - 20):
        assert np.array_equal(out.part(at * n, 20 * n).reshape(20, n), np.tile(a[at: at + 20].sum(1)[:, None], (1, n)))


class Columns:
    """Some columns of a tensor in device memory."""

    def __init__(self, whole, first, count):
        self.whole, self.first, self.count = whole, first, count
        self.shape, self.dtype, self.kind = (whole.shape[0], count), whole.dtype, whole.kind

    def stride(self):
        return self.whole.stride()

    def data_ptr(self):
        return self.whole.memory.offset(self.first)

    def host(self):
        return self.whole.host()[:, self.first: self.first + self.count]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [1, 7, 64, 515])
def test_inputs_and_outputs_in_columns_of_one_buffer(dev, ops, kind, d):
    """Results between the rows of their inputs: nothing else of the buffer changes."""
    g = np.random.default_rng(d)
    n, k = 60, 3
    start = typed(g.standard_normal((n * k, 3 * d + 5)), kind)
    whole = dev(start, kind)
    left, middle, right = (Columns(whole, at, d) for at in (1, d + 2, 2 * d + 3))
    want = start.copy()

    def check(columns, values):
        want[:, columns.first: columns.first + d] = values
        assert np.array_equal(whole.host(), want)

    ids = g.integers(0, n * k, n * k)
    ops.lookup(left, dev(ids, "int32"), middle)
    check(middle, start[ids, 1: 1 + d])
    slots = g.permutation(n * k).reshape(n * k, 1)
    ops.dispatch(middle, dev(slots, "int32"), right)
    there = np.empty((n * k, d))
    there[slots[:, 0]] = middle.host()
    check(right, there)
    ops.combine(right, dev(slots, "int32"), left)
    check(left, there[slots[:, 0]])
    ops.combine_grad(left, right, dev(slots, "int32"), None, middle, None)
    scattered = np.empty((n * k, d))
    scattered[slots[:, 0]] = left.host()
    check(middle, scattered)
    ops.lookup_grad(middle, dev(slots[:, 0], "int64"), right)
    again = np.empty((n * k, d))
    again[slots[:, 0]] = scattered
    check(right, again)


def test_arrays_know_their_device(capi, ctx, ops):
    assert ctx.device == ops.device == 0
    a = ctx.array(np.ones((2, 4), np.float32))
    assert a.get_device() == 0
    km = capi.KMeans(4, 8)
    assert km.ctx.device == 0
    km.close()
    a.free()


@pytest.mark.parametrize("scale", [-1.0, np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("n", [5, 3000])
def test_rows_without_a_token_are_zeros_whatever_the_scale(dev, ops, n, scale):
    """Zeros are stored, not a product of zero and the scale: neither NaN nor -0."""
    rows, d = 40, 12
    ids = np.arange(n) % 3 * 11 + 2
    for kind in KINDS:
        out = dev(np.full((rows, d), 5), kind)
        ops.lookup_grad(dev(np.ones((n, d)), kind), dev(ids, "int64"), out, scale=scale)
        named = np.zeros(rows, bool)
        named[ids] = True
        assert np.all(out.raw()[~named].view(np.uint8) == 0)
        got = out.host()[named]
        assert np.all(np.isnan(got)) if np.isnan(scale) else np.all(np.sign(got) == np.sign(scale))


def test_device_timers_leave_captured_calls_out(hip, dev):
    """With the timers on, calls are captured and replayed as without; the timers count the eager calls only."""
    from superkmeans_amd.rowops import RowOperators

    g = np.random.default_rng(2)
    stream = hip.stream()
    with RowOperators(device=0, stream=stream.value) as ops:
        layer = Layer(dev, g, 300, 150, 64, 96, 8, 2, with_scratch_of=ops)
        ops.ctx.prof_enable()
        ops.ctx.prof_reset()
        layer.set(g)
        layer.run(ops)
        graph = hip.capture(stream, lambda: layer.run(ops))
        for _ in range(3):
            layer.set(g)
            hip.hipGraphLaunch(graph, stream)
            ops.sync()
            layer.check()
            assert ops.ctx.prof()["rows/route"][1] == 1
        layer.set(g)
        layer.run(ops)
        ops.sync()
        layer.check()
        timers = ops.ctx.prof()
        assert {name: calls for name, (_, calls) in timers.items()} == {
            f"rows/{name}": 2 for name in ("lookup", "route", "dispatch", "quantize", "product", "combine", "combine_grad", "lookup_grad")}
        assert all(ms > 0 for ms, _ in timers.values())
        ops.ctx.prof_enable(False)
        hip.hipGraphExecDestroy(graph)
    hip.hipStreamDestroy(stream)


# ---------------------------------------------------------------------------------------------------------------------
# long rows of a gradient, exactly
# ---------------------------------------------------------------------------------------------------------------------

# Gradients of whole numbers from 1 to 8, sums below 2^24: fp32 adds them exactly in any order, so results have to be equal, and as
# every token adds something to every column, none can be lost unseen.
WHOLE = [(2100, 3, 257, "one"), (2500, 7, 600, "text"), (40000, 2049, 20, "one"), (40000, 2049, 20, "two runs"), (40000, 2049, 20, "even"),
         (131072, 11, 9, "two runs"), (140000, 500, 5, "one"), (140000, 500, 5, "text"), (500000, 4, 33, "even"), (1048577, 1, 3, "one"),
         (1100000, 40, 2, "text"), (1100000, 40, 2, "two runs"), (1100000, 70001, 3, "even"), (1100000, 70001, 3, "one")]


def whole_case(n, rows, d, how):
    """(grad, ids, sums) in whole numbers."""
    g = np.random.default_rng(n + rows + d)
    grad, ids = g.integers(1, 9, (n, d)), spread_ids(g, n, rows, how)
    there = (ids >= 0) & (ids < rows)
    sums = np.stack([np.bincount(ids[there], weights=column[there], minlength=rows) for column in grad.T], 1)
    assert sums.max() < 1 << 24
    return grad, ids, sums


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,rows,d,how", WHOLE)
def test_lookup_grad_of_whole_numbers(dev, ops, kind, n, rows, d, how):
    grad, ids, sums = whole_case(n, rows, d, how)
    on_device, held = dev(grad, kind), np.arange(rows * d).reshape(rows, d) % 100
    for ids_kind, scale in (("int64", 1.0), ("int32", -0.5)):
        where = dev(ids, ids_kind)
        out = dev(np.full((rows, d), 5), "float32")
        ops.lookup_grad(on_device, where, out, scale=scale)
        assert np.array_equal(out.host(), sums * scale)
        out = dev(held, "float32")
        ops.lookup_grad(on_device, where, out, scale=scale, accumulate=True)
        assert np.array_equal(out.host(), sums * scale + held)
        if kind != "float32":
            out = dev(np.full((rows, d), 5), kind)
            ops.lookup_grad(on_device, where, out, scale=scale)
            assert np.array_equal(out.host(), typed(sums * scale, kind))  # one rounding of the exact sum


# ---------------------------------------------------------------------------------------------------------------------
# variants that only some sizes choose
# ---------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind,d", [("float16", 24), ("float32", 100), ("bfloat16", 257), ("float32", 7), ("bfloat16", 2056), ("float32", 1024)])
@pytest.mark.parametrize("rest", [0, 1, 2, 3])
def test_lookup_of_so_many_rows_that_wavefronts_take_four(dev, block, ops, kind, d, rest):
    """From 32,768 wavefronts of work on each takes four times its rows: those of a last, partly filled one among them."""
    elements = min(16 // (4 if kind == "float32" else 2), d)
    elements = 1 << (elements.bit_length() - 1)
    vectors, lanes = -(-d // elements), 1
    while lanes < 64 and lanes * 4 < vectors:
        lanes *= 2
    pieces = -(-vectors // (4 * lanes))
    n = 32768 // pieces * (64 // lanes) + 4 * (64 // lanes) * 5 + rest * (64 // lanes) + rest
    g = np.random.default_rng(n)
    rows = 1000
    table, ids = typed(g.standard_normal((rows, d)), kind), g.integers(-1, rows + 1, n)
    on_device, where, out = dev(table, kind, 3), dev(ids, "int32"), block((n, d), kind, 0x01010101)
    there = (ids >= 0) & (ids < rows)
    for scale in (1.0, -0.5):
        ops.lookup(on_device, where, out, scale=scale)
        want = encode(np.concatenate([table * scale, np.zeros((1, d))]), kind)[np.where(there, ids, rows)]
        got = out.memory.download()
        assert np.array_equal(got[: n * d].reshape(n, d).view(np.uint8), want.view(np.uint8))
        assert np.all(got[n * d:].view(np.uint8) == 1)  # nothing behind the last row


@pytest.mark.parametrize("kind,out_kind", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("d", [300, 301, 500, 512, 516, 768, 900, 1100, 2047])
def test_lookup_grad_of_few_tokens_on_wide_rows(dev, ops, kind, out_kind, d):
    """Rows of up to 64, 128, 192 and more vectors, alone and with more than eight tokens, stored and accumulated, exactly."""
    g = np.random.default_rng(d)
    for n, rows in ((1021, 200), (2048, 64), (250, 3)):
        grad, ids = g.integers(1, 9, (n, d)), spread_ids(g, n, rows, "text")
        held = g.integers(-50, 50, (rows, d))
        there = (ids >= 0) & (ids < rows)
        sums = np.zeros((rows, d))
        np.add.at(sums, ids[there], grad[there])
        counts = np.bincount(ids[there], minlength=rows)
        assert counts.max() > 8 and (rows < 10 or counts.min() <= 8)
        on_device, where = dev(grad, kind, 5), dev(ids, "int64")
        out = dev(np.full((rows, d), 5), out_kind, 1)
        ops.lookup_grad(on_device, where, out)
        assert np.array_equal(out.host(), typed(sums, out_kind)) and out.margin_untouched()
        out = dev(held, out_kind, 1)
        ops.lookup_grad(on_device, where, out, accumulate=True)
        assert np.array_equal(out.host(), typed(sums + held, out_kind)) and out.margin_untouched()


@pytest.mark.parametrize("out_kind", KINDS)
@pytest.mark.parametrize("m,n,k,sizes", [(2047, 4095, 272, None), (2048, 4096, 128, None), (2000, 4095, 144, [700, 0, 513, 780]),
                                         (2047, 4096, 272, [1, 1023, 900, 123])])
def test_product_of_tiles_of_128_by_256(dev, ops, out_kind, m, n, k, sizes):
    """Sizes that give 256 workgroups a tile of 128 x 256, and too few of them one of 256 x 256."""
    groups = 1 if sizes is None else len(sizes)
    rows = -(-m // groups)
    tiles = lambda tm, tn: groups * -(-rows // tm) * -(-n // tn)
    assert rows > 64 and tiles(256, 256) < 192 and tiles(128, 256) >= 256
    g = np.random.default_rng(m + k)
    for pad in (0, 3):
        a, b = g.integers(-128, 128, (m, k)), g.integers(-128, 128, (groups, n, k))
        a_scales, b_scales = typed(g.random(m) * 0.01, "float32"), typed(g.random((groups, n)) * 0.01, "float32")
        bias = typed(g.standard_normal((groups, n)), "float32") if pad else None
        out = dev(np.full((m, n), 5), out_kind, pad)
        if sizes is None:
            ops.product(dev(a, "int8", pad), dev(a_scales, "float32"), dev(b[0], "int8", pad), dev(b_scales[0], "float32"), out,
                        bias=None if bias is None else dev(bias[0], "float32"))
            offsets = [0, m]
        else:
            offsets = np.concatenate([[0], np.cumsum(sizes)])
            ops.product(dev(a, "int8", pad), dev(a_scales, "float32"), dev(b, "int8", pad), dev(b_scales, "float32"), out,
                        bias=None if bias is None else dev(bias, "float32"), offsets=dev(offsets, "int32"))
        for e in range(groups):
            i, j = offsets[e], offsets[e + 1]
            if i < j:
                want, size = product_of(a[i:j], a_scales[i:j], b[e], b_scales[e], None if bias is None else bias[e])
                close(out, want, size, 4, rows=slice(i, j))
        assert np.all(out.host()[offsets[-1]:] == 5) and out.margin_untouched()


def test_lookup_of_what_assign_answers(capi, ctx, ops):
    """The framework's own use: every point replaced by its centroid, and the sums of the points by centroid as the gradient."""
    g = np.random.default_rng(6)
    n, k, d = 3001, 37, 48
    X, C = g.integers(-9, 10, (n, d)).astype(np.float32), g.integers(-9, 10, (k, d)).astype(np.float32)
    dX, dC = ctx.array(X), ctx.array(C)
    xn, cn, idx, dist = ctx.empty(n), ctx.empty(k), ctx.empty(n, np.uint32), ctx.empty(n)
    out, sums, update, sizes = ctx.empty((n, d)), ctx.empty((k, d)), ctx.empty((k, d)), ctx.empty(k, np.uint32)
    capi.check(ctx.lib.skm_norms(ctx.handle, dX.ptr, n, d, d, xn.ptr))
    capi.check(ctx.lib.skm_norms(ctx.handle, dC.ptr, k, d, d, cn.ptr))
    capi.check(ctx.lib.skm_assign_full(ctx.handle, dX.ptr, n, dC.ptr, k, d, xn.ptr, cn.ptr, idx.ptr, dist.ptr))
    ops.lookup(dC, idx, out)
    ops.lookup_grad(dX, idx, sums)
    capi.check(ctx.lib.skm_update(ctx.handle, dX.ptr, n, d, idx.ptr, k, update.ptr, sizes.ptr))
    assert np.array_equal(out.download(), C[idx.download()])
    assert np.array_equal(((X - out.download()) ** 2).sum(1), dist.download())  # whole numbers: exact
    assert np.array_equal(sums.download(), update.download())
    for a in (dX, dC, xn, cn, idx, dist, out, sums, update, sizes):
        a.free()


def test_no_context_is_made_on_a_capturing_stream(hip, dev, capi):
    """The refusal leaves the capture in working order."""
    from superkmeans_amd.rowops import RowOperators

    stream = hip.stream()
    few, slots, offsets = dev(np.ones((4, 2)), "int32"), dev(np.zeros((4, 2)), "int32"), dev(np.zeros(9), "int32")
    with RowOperators(device=0, stream=stream.value) as ops:
        def work():
            with pytest.raises(capi.SkmError, match="captured"):
                RowOperators(device=0, stream=stream.value)
            ops.route(few, 8, slots, offsets)

        graph = hip.capture(stream, work)
        hip.hipGraphLaunch(graph, stream)
        ops.sync()
        assert np.array_equal(offsets.raw(), [0, 0] + [8] * 7)
        hip.hipGraphExecDestroy(graph)
    hip.hipStreamDestroy(stream)


def test_two_threads_with_an_object_each(hip, ctx):
    """Calls at the same time on two streams, with workspaces that grow meanwhile."""
    import threading

    from superkmeans_amd import _capi
    from superkmeans_amd.rowops import RowOperators

    failures = []

    def work(seed):
        try:
            stream = hip.stream()
            mine = _capi.Context(0)
            made = []

            def make(x, kind, pad=0):
                made.append(Device(mine, x, kind, pad))
                return made[-1]

            g = np.random.default_rng(seed)
            with RowOperators(device=0, stream=stream.value) as ops:
                for n in (40, 3000, 9000, 500, 12000):
                    layer = Layer(make, g, n, 150, 64, 96, 8, 2)
                    for _ in range(2):
                        layer.set(g)
                        layer.run(ops)
                        ops.sync()
                        layer.check()
            mine.close()
            hip.hipStreamDestroy(stream)
        except BaseException as e:
            failures.append(e)

    threads = [threading.Thread(target=work, args=(seed,)) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(100)
    assert not failures, failures


FIRST_CALLS = """
import sys
sys.path.insert(0, "tests")
import numpy as np
from superkmeans_amd import _capi
from superkmeans_amd.rowops import RowOperators
from test_gpu_rowops import Device, Hip, Layer
ctx, hip = _capi.Context(0), Hip()
made = []
def dev(x, kind, pad=0):
    made.append(Device(ctx, x, kind, pad))
    return made[-1]
g = np.random.default_rng(0)
stream = hip.stream()
with RowOperators(device=0, stream=stream.value) as ops:
    layer = Layer(dev, g, 9000, 150, 64, 96, 8, 2, with_scratch_of=ops)
    graph = hip.capture(stream, lambda: layer.run(ops))
    for _ in range(3):
        layer.set(g)
        hip.hipGraphLaunch(graph, stream)
        ops.sync()
        layer.check()
    layer.set(g)
    layer.run(ops)
    ops.sync()
    layer.check()
print("first calls: ok")
"""


def test_the_first_calls_of_a_process_may_be_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "first calls: ok" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
