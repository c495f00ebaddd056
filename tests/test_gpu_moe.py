"""The ops of a mixture-of-experts layer against the same in 64 bits (moe_model.py)."""

from __future__ import annotations

import numpy as np
import pytest

import moe_model as mm

pytestmark = pytest.mark.gpu

EPS = 1e-6


def up(backend, dev, a):
    return backend.HipBuffer.from_host(dev, np.ascontiguousarray(a))


def bits(a):
    return np.ascontiguousarray(a, np.float32).view(np.uint32)


# ---- residual and norm -----------------------------------------------------------

def norm_inputs(rng, batch, dim):
    t = (rng.standard_normal((batch, dim)) * rng.uniform(0.1, 30, (batch, 1))).astype(np.float32)
    t[:, ::31] *= 40
    h = (rng.standard_normal((batch, dim)) * 5).astype(np.float32)
    w = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2)]
    return t, h, w


@pytest.mark.parametrize("norm_t", [False, True])
@pytest.mark.parametrize("dim,batch", [(32, 1), (64, 5), (96, 130), (704, 3), (1024, 2), (1056, 2), (2304, 9), (2816, 1),
                                       (2816, 77), (4096, 2), (5120, 3), (8192, 2), (12288, 3)])
def test_residual_norm(backend, dev, orc, synth, dim, batch, norm_t):
    rng = synth.rng_for(dim * 31 + batch + norm_t)
    t, h, (wp, wn) = norm_inputs(rng, batch, dim)
    if batch > 2:
        t[1], h[1] = 0, 0  # a row of zeros: scale 1 / sqrt(eps), everything stays 0
    want_h, want_xn = mm.residual_norm(t, wp, h, wn, EPS, norm_t)
    tb, hb, wpb, wnb = (up(backend, dev, a) for a in (t, h, wp, wn))
    hob, xnb = backend.HipBuffer.alloc(dev, batch * dim), backend.HipBuffer.alloc(dev, batch * dim)
    pb = backend.HipBuffer.alloc(dev, batch * dim // 32 * 40, np.uint8)
    dev.residual_rms_norm_batch(tb, wpb, hb, hob, wnb, xnb, dim, batch, EPS, pack=pb, norm_t=norm_t)
    dev.sync()
    xn = xnb.numpy().reshape(batch, dim)
    # the sums in 64 bits fix every later rounding
    assert np.array_equal(bits(hob.numpy().reshape(batch, dim)), bits(want_h))
    assert np.array_equal(bits(xn), bits(want_xn))
    q, d, s = mm.pack_parts(pb.numpy(), batch * dim)
    want_q, want_d = mm.q8_0_parts(orc, xn)
    assert np.array_equal(q, want_q) and np.array_equal(d, want_d.astype(np.float32))
    assert np.array_equal(s, want_q.astype(np.int32).sum(1))
    # the single-row op has the sequential sum: dim roundings of it, halved by the root, and four steps more
    row = backend.HipBuffer.from_host(dev, h[-1])
    one = backend.HipBuffer.alloc(dev, dim)
    if norm_t:
        last = up(backend, dev, t[-1])
        dev.residual_rms_norm(last, wpb, row, wnb, one, dim, EPS)
        dev.sync()
        assert np.abs(one.numpy() - xn[-1]).max() <= (dim + 8) * mm.U * 3 * np.abs(xn[-1]).max()


@pytest.mark.parametrize("norm_t", [False, True])
@pytest.mark.parametrize("dim,batch", [(96, 300), (1024, 257), (1056, 258), (2304, 300), (2848, 257), (4096, 290), (8192, 260),
                                       (8224, 257), (12288, 259)])
def test_residual_norm_of_many_rows(backend, dev, orc, synth, dim, batch, norm_t):
    """More than 256 rows: 256 threads a row, of one to twelve chunks."""
    test_residual_norm(backend, dev, orc, synth, dim, batch, norm_t)


def test_residual_norm_in_place_and_without_parts(backend, dev, synth):
    """h_out = h and xn = t, no weights, no outputs but h: each the bits of the call with everything apart."""
    batch, dim = 6, 352
    rng = synth.rng_for(11)
    t, h, _ = norm_inputs(rng, batch, dim)
    for norm_t in (False, True):
        want_h, want_xn = mm.residual_norm(t, None, h, None, EPS, norm_t)
        tb, hb = up(backend, dev, t), up(backend, dev, h)
        dev.residual_rms_norm_batch(tb, None, hb, hb, None, tb, dim, batch, EPS, norm_t=norm_t)
        dev.sync()
        assert np.array_equal(bits(hb.numpy()), bits(want_h)) and np.array_equal(bits(tb.numpy()), bits(want_xn))
        tb, hb, ob = up(backend, dev, t), up(backend, dev, h), backend.HipBuffer.alloc(dev, batch * dim)
        dev.residual_rms_norm_batch(tb, None, hb, ob, None, None, dim, batch, EPS, norm_t=norm_t)
        dev.sync()
        assert np.array_equal(bits(ob.numpy().reshape(batch, dim)), bits(want_h)) and np.array_equal(hb.numpy(), h)


def test_residual_norm_values_that_are_not_finite(backend, dev, synth):
    """A row with an infinity or NaN spoils itself alone."""
    batch, dim = 4, 64
    t, h, (wp, wn) = norm_inputs(synth.rng_for(3), batch, dim)
    t[1, 5], h[2, 7] = np.inf, np.nan
    with np.errstate(invalid="ignore"):
        want_h, want_xn = mm.residual_norm(t, wp, h, wn, EPS, False)
    tb, hb, wnb = (up(backend, dev, a) for a in (t, h, wn))
    ob, xb = (backend.HipBuffer.alloc(dev, batch * dim) for _ in "ab")
    dev.residual_rms_norm_batch(tb, None, hb, ob, wnb, xb, dim, batch, EPS, norm_t=False)
    dev.sync()
    assert np.array_equal(ob.numpy().reshape(batch, dim), want_h, equal_nan=True)
    assert np.array_equal(xb.numpy().reshape(batch, dim), want_xn, equal_nan=True)


# ---- the router's product -----------------------------------------------------------

@pytest.mark.parametrize("batch,experts,cols", [(1, 1, 32), (1, 128, 2816), (3, 5, 64), (5, 128, 2816), (17, 60, 2048),
                                                (40, 8, 96), (41, 8, 96), (41, 1, 32), (90, 33, 288), (1537, 100, 64),
                                                (33, 31, 160), (64, 64, 96), (65, 130, 352), (130, 128, 704),
                                                (257, 512, 64), (300, 3, 4096), (1000, 128, 2816)])
def test_logits(backend, dev, synth, batch, experts, cols):
    rng = synth.rng_for(batch * 7 + experts + cols)
    x = (rng.standard_normal((batch, cols)) * 10.0 ** rng.uniform(-4, 4, (batch, 1))).astype(np.float32)
    w = (rng.standard_normal((experts, cols)) * 10.0 ** rng.uniform(-3, 1, (experts, 1))).astype(np.float32)
    xb, wb, out = up(backend, dev, x), up(backend, dev, w), backend.HipBuffer.alloc(dev, batch * experts)
    dev.moe_logits(xb, wb, out, experts, cols, batch)
    dev.sync()
    want = x.astype(np.float64) @ w.astype(np.float64).T
    bound = (cols + 2) * mm.U * (np.abs(x).astype(np.float64) @ np.abs(w).astype(np.float64).T)
    assert (np.abs(out.numpy().reshape(batch, experts) - want) <= bound).all()


def test_logits_rows_that_are_not_finite(backend, dev, synth):
    rng = synth.rng_for(2)
    x, w = rng.standard_normal((20, 64)).astype(np.float32), rng.standard_normal((9, 64)).astype(np.float32)
    x[3, 1], x[4, 2], w[8, 9] = np.nan, np.inf, np.inf
    xb, wb, out = up(backend, dev, x), up(backend, dev, w), backend.HipBuffer.alloc(dev, 180)
    dev.moe_logits(xb, wb, out, 9, 64, 20)
    dev.sync()
    got = out.numpy().reshape(20, 9)
    ok = np.isfinite(got)
    assert not ok[3:5].any() and not ok[:, 8].any()
    assert ok[np.r_[0:3, 5:20]][:, :8].all()


# ---- the route -------------------------------------------------------------------------

class Route:
    def __init__(self, backend, dev, logits, bias, k, **how):
        self.dev, self.n, self.e, self.k, self.how = dev, *logits.shape, k, how
        self.logits, self.bias = up(backend, dev, logits), None if bias is None else up(backend, dev, bias)
        self.ids, self.weights = backend.HipBuffer.alloc(dev, self.n * k, np.int32), backend.HipBuffer.alloc(dev, self.n * k)
        self.starts, self.order = (backend.HipBuffer.alloc(dev, c, np.int32) for c in (self.e + 1, self.n * k))

    def call(self):
        self.dev.moe_route(self.logits, self.bias, self.ids, self.weights, self.starts, self.order, self.e, self.n, self.k,
                           **self.how)

    def got(self):
        self.dev.sync()
        return (self.ids.numpy().reshape(self.n, self.k), self.weights.numpy().reshape(self.n, self.k),
                self.starts.numpy(), self.order.numpy())


def check_route(backend, dev, logits, bias, k, **how):
    r = Route(backend, dev, logits, bias, k, **how)
    r.call()
    ids, w, starts, order = r.got()
    want_ids, want_w = mm.route(logits, bias, k, **how)
    assert np.array_equal(ids, want_ids)
    # one rounding to f32, and the 64-bit steps before it
    assert (np.abs(w - want_w) <= 1.01 * mm.U * np.abs(want_w) + 2.0 ** -149).all()
    want_starts, want_order = mm.plan(want_ids, logits.shape[1])
    assert np.array_equal(starts, want_starts) and np.array_equal(order, want_order)


@pytest.mark.parametrize("scoring", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("n,e,k,groups,top,best", [
    (1, 1, 1, 1, 1, 1), (1, 128, 8, 1, 1, 1), (3, 4, 4, 1, 1, 1), (5, 7, 3, 1, 1, 1), (9, 60, 4, 1, 1, 1),
    (65, 64, 1, 1, 1, 1), (130, 65, 6, 5, 2, 1), (33, 128, 8, 8, 4, 2), (200, 256, 8, 8, 4, 2), (17, 512, 32, 64, 9, 2),
    (16, 40, 5, 1, 1, 1), (17, 40, 5, 1, 1, 1), (16, 512, 32, 1, 1, 1), (15, 512, 32, 2, 1, 2), (7, 130, 32, 13, 5, 2),
    (300, 192, 8, 64, 16, 2), (40, 12, 3, 6, 2, 2), (40, 12, 2, 12, 2, 2), (2, 96, 8, 3, 3, 1), (1030, 16, 2, 1, 1, 1)])
def test_route(backend, dev, synth, n, e, k, groups, top, best, with_bias, scoring):
    rng = synth.rng_for(n + 13 * e + k + 2 * scoring + with_bias)
    logits = (rng.standard_normal((n, e)) * 2).astype(np.float32)
    bias = (rng.standard_normal(e) * 0.2).astype(np.float32) if with_bias else None
    check_route(backend, dev, logits, bias, k, scoring=scoring, n_groups=groups, top_groups=top, group_best=best,
                renormalise=bool((n + k) % 2), scale=1.0 if n % 2 else 2.5)


@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups,top,best", [(1, 1, 1), (4, 2, 1), (4, 3, 2)])
def test_route_ties(backend, dev, synth, groups, top, best, with_bias):
    """Few distinct values: equal ones go to the lower id, equal groups to the lower group."""
    rng = synth.rng_for(groups + best)
    logits = rng.integers(-1, 2, (50, 64)).astype(np.float32)
    logits[0] = 0
    bias = (rng.integers(0, 2, 64) * 0.25).astype(np.float32) if with_bias else None
    for scoring in (0, 1):
        check_route(backend, dev, logits, bias, 8, scoring=scoring, n_groups=groups, top_groups=top, group_best=best)


@pytest.mark.parametrize("step", [1e-7, 1e-9])
def test_route_near_ties(backend, dev, synth, step):
    """Values nearer to each other than f32 can tell apart once a score is formed."""
    rng = synth.rng_for(8)
    base = rng.standard_normal((40, 1)) * 0.01
    logits = (base + rng.integers(0, 40, (40, 96)) * step).astype(np.float32)
    bias = (0.5 + rng.integers(0, 9, 96) * 2.0 ** -24).astype(np.float32)
    for scoring in (0, 1):
        check_route(backend, dev, logits, bias, 6, scoring=scoring)
        check_route(backend, dev, logits, None, 6, scoring=scoring, n_groups=8, top_groups=3, group_best=2)


@pytest.mark.parametrize("groups,top,best", [(1, 1, 1), (4, 2, 1), (4, 2, 2)])
@pytest.mark.parametrize("scoring", [0, 1])
def test_route_masks_and_extremes(backend, dev, synth, scoring, groups, top, best):
    """Experts switched off (all of a token's among them), the type's lowest value, infinities, NaN, far logits."""
    rng = synth.rng_for(4 + groups)
    n, e, k = 24, 32, 6
    x = (rng.standard_normal((n, e)) * 3).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 1:] = -np.inf
    x[3, 4:] = -np.inf
    x[4] = np.finfo(np.float32).min
    x[5, ::2] = np.finfo(np.float32).min
    x[6, 3] = x[6, 20] = np.inf
    x[7] = np.finfo(np.float32).max
    x[8, ::3] = np.nan
    x[9] = -800
    x[10, 0:8] = -np.inf
    x[11] *= 1e30
    x[12] *= 100
    x[13:, rng.integers(0, e, 5)] = -np.inf
    bias = (rng.standard_normal(e) * 0.1).astype(np.float32)
    for b in (None, bias):
        check_route(backend, dev, x, b, k, scoring=scoring, n_groups=groups, top_groups=top, group_best=best)
        check_route(backend, dev, x, b, k, scoring=scoring, n_groups=groups, top_groups=top, group_best=best,
                    renormalise=False, scale=-3.0)
    bias[3], bias[5], bias[7] = np.nan, -np.inf, np.inf
    check_route(backend, dev, x, bias, k, scoring=scoring, n_groups=groups, top_groups=top, group_best=best)


def test_route_without_a_plan(backend, dev, synth):
    logits = synth.rng_for(1).standard_normal((70, 40)).astype(np.float32)
    r = Route(backend, dev, logits, None, 5)
    dev.moe_route(r.logits, None, r.ids, r.weights, None, None, 40, 70, 5)
    ids, w, _, _ = r.got()
    assert np.array_equal(ids, mm.route(logits, None, 5, mm.SOFTMAX)[0])


@pytest.mark.parametrize("n,e,k", [(4099, 128, 8), (131072, 64, 8), (700, 512, 32)])
def test_route_large(backend, dev, synth, n, e, k):
    logits = synth.rng_for(n).standard_normal((n, e)).astype(np.float32)
    r = Route(backend, dev, logits, None, k)
    r.call()
    ids, w, starts, order = r.got()
    want = np.argsort(-logits, 1, kind="stable")[:, :k]
    assert np.array_equal(ids, want)
    flat = want.reshape(-1)
    assert np.array_equal(order, np.argsort(flat, kind="stable"))
    assert np.array_equal(starts, np.searchsorted(np.sort(flat), np.arange(e + 1)))
    assert np.abs(w.sum(1) - 1).max() <= (k + 1) * mm.U


# ---- the experts' products ----------------------------------------------------------------

class Experts:
    """Weights of e experts: matrices on the device and their 64-bit values."""

    def __init__(self, backend, dev, synth, seed, e, rows, cols, n=1):
        rng = synth.rng_for(seed)
        self.e, self.rows, self.cols = e, rows, cols
        raw = [synth.q4_0_matrix(rng, e * rows, cols) for _ in range(n)]
        self.values = [mm.q4_0_values(r, e * rows, cols).reshape(e, rows, cols) for r in raw]
        self.dev = [backend.HipBuffer.from_gguf(dev, r, backend.Q4_0, e * rows, cols) for r in raw]


def some_ids(rng, n, e, k, how):
    if how == "even":
        return np.stack([rng.permutation(e)[:k] for _ in range(n)]).astype(np.int32)
    if how == "skew":  # most tokens ask for the same experts
        p = 1.0 / (1 + np.arange(e)) ** 1.5
        return np.stack([rng.choice(e, k, False, p / p.sum()) for _ in range(n)]).astype(np.int32)
    if how == "one":  # the last expert alone, in every slot
        return np.full((n, k), e - 1, np.int32)
    ids = some_ids(rng, n, e, k, "even")  # holes: some slots, and whole tokens, without an expert
    ids[rng.random((n, k)) < 0.3] = -1
    ids[:: 5] = -1
    return ids


def planned(backend, dev, ids, e):
    return [up(backend, dev, a) for a in (ids.reshape(-1), *mm.plan(ids, e))]


SHAPES = [(1, 1, 1, 1, 32, "even"), (4, 2, 1, 17, 64, "even"), (3, 3, 2, 5, 96, "holes"), (8, 8, 1, 100, 704, "even"),
          (128, 8, 1, 33, 352, "even"), (60, 4, 3, 47, 288, "even"), (16, 4, 5, 64, 2816, "even"),
          (5, 2, 16, 31, 160, "one"), (5, 2, 17, 32, 160, "skew"), (6, 2, 40, 70, 416, "holes"),
          (3, 1, 65, 48, 128, "one"), (4, 2, 130, 16, 224, "skew"), (40, 6, 64, 129, 64, "even"),
          (2, 2, 200, 15, 32, "even"), (7, 3, 90, 257, 192, "holes"), (128, 8, 50, 12, 96, "even"),
          (9, 1, 300, 80, 480, "skew"), (2, 1, 9, 4, 4128, "even"), (2, 1, 70, 20, 4128, "skew"),
          (40, 32, 3, 20, 64, "even"), (33, 32, 60, 18, 96, "even"), (8, 2, 110, 65, 1056, "holes"),
          (4, 2, 14, 33, 4096, "even"), (3, 2, 130, 33, 4096, "even"), (512, 8, 40, 5, 64, "even"),
          (4, 4, 4, 30, 4064, "holes"), (2, 1, 400, 9, 32, "even"), (16, 2, 20, 40, 704, "even"),
          (16, 2, 20, 88, 992, "holes"), (6, 3, 30, 8, 32, "skew"), (6, 3, 30, 24, 224, "even"), (20, 4, 9, 200, 160, "even"),
          (1, 1, 130, 70, 96, "even"), (1, 1, 130, 33, 64, "even"), (1, 1, 101, 40, 704, "even"), (1, 1, 180, 150, 160, "even"),
          (4, 2, 260, 129, 352, "skew"), (4, 2, 300, 47, 416, "holes"), (3, 2, 250, 257, 192, "one"), (2, 1, 40, 20, 4160, "even"),
          (2, 1, 33, 130, 4224, "skew"), (8, 4, 210, 31, 128, "even"), (30, 4, 140, 1100, 32, "skew")]


@pytest.mark.parametrize("activation", [0, 1])
@pytest.mark.parametrize("e,k,n,rows,cols,how", SHAPES)
def test_gate_up(backend, dev, orc, synth, e, k, n, rows, cols, how, activation):
    rng = synth.rng_for(e + n * 3 + rows)
    w = Experts(backend, dev, synth, rows * 5 + cols, e, rows, cols, 2)
    x = (rng.standard_normal((n, cols)) * rng.uniform(0.2, 3, (n, 1))).astype(np.float32)
    ids = some_ids(rng, n, e, k, how)
    want, bound = mm.gate_up(*w.values, mm.q8_0_values(orc, x), ids, k, activation)
    xb, plan = up(backend, dev, x), planned(backend, dev, ids, e)
    for packed in (False, True):
        out = up(backend, dev, np.full(n * k * rows, 7.0, np.float32))
        if packed:
            pack = backend.HipBuffer.alloc(dev, n * cols // 32 * 40, np.uint8)
            dev.quantize_q8_0(xb, pack=pack, n=n * cols)
            dev.moe_gate_up_q4_0_q8(*w.dev, pack, *plan, out, e, rows, cols, n, k, activation)
        else:
            dev.moe_gate_up_q4_0(*w.dev, xb, *plan, out, e, rows, cols, n, k, activation)
        dev.sync()
        got = out.numpy().reshape(n * k, rows)
        none = ids.reshape(-1) < 0
        assert (got[none] == 7.0).all(), "rows without an expert were written"
        off = np.abs(got[~none] - want[~none]) / bound[~none]
        assert (off <= 1).all(), off.max()


@pytest.mark.parametrize("e,k,n,rows,cols,how", SHAPES)
def test_down(backend, dev, orc, synth, e, k, n, rows, cols, how):
    rng = synth.rng_for(e + n * 3 + rows + 1)
    w = Experts(backend, dev, synth, rows * 5 + cols + 1, e, rows, cols)
    act = (rng.standard_normal((n * k, cols)) * rng.uniform(0.01, 3, (n * k, 1))).astype(np.float32)
    ids = some_ids(rng, n, e, k, how)
    weights = rng.uniform(-0.2, 1, (n, k)).astype(np.float32)
    weights[ids < 0] = np.nan  # of no meaning there
    want, bound = mm.down(w.values[0], mm.q8_0_values(orc, act), ids, weights, k)
    bid, starts, order = planned(backend, dev, ids, e)
    act[ids.reshape(-1) < 0] = np.nan  # nor the rows
    out = up(backend, dev, np.full(n * rows, 7.0, np.float32))
    dev.moe_down_q4_0(w.dev[0], up(backend, dev, act), bid, up(backend, dev, weights), starts, order, out, e, rows, cols,
                      n, k)
    dev.sync()
    got = out.numpy().reshape(n, rows)
    off = np.abs(got - want) / bound
    assert (off <= 1).all(), off.max()
    assert (got[(ids < 0).all(1)] == 0).all()


# Forms that the sizes above leave out: streams whose scales come four at once (rows of 36, 44 blocks; odd numbers of rows of
# 12), down's streams of more than four tokens an expert in each of their forms, rows of 1025 to 4096 values in tiles.
MORE_SHAPES = [(8, 2, 20, 33, 1152, "even"), (16, 2, 40, 31, 384, "holes"), (16, 2, 20, 17, 1408, "even"),
               (10, 5, 11, 40, 96, "even"), (10, 5, 11, 31, 96, "even"), (10, 5, 11, 31, 96, "one"),
               (10, 5, 11, 33, 192, "skew"), (10, 5, 11, 48, 256, "one"), (10, 5, 11, 150, 704, "skew"),
               (10, 5, 11, 270, 1152, "skew"), (2, 2, 220, 24, 2816, "even"), (2, 2, 220, 24, 2848, "holes")]


@pytest.mark.parametrize("activation", [0, 1])
@pytest.mark.parametrize("e,k,n,rows,cols,how", MORE_SHAPES)
def test_gate_up_in_more_forms(backend, dev, orc, synth, e, k, n, rows, cols, how, activation):
    test_gate_up(backend, dev, orc, synth, e, k, n, rows, cols, how, activation)


@pytest.mark.parametrize("e,k,n,rows,cols,how", MORE_SHAPES)
def test_down_in_more_forms(backend, dev, orc, synth, e, k, n, rows, cols, how):
    test_down(backend, dev, orc, synth, e, k, n, rows, cols, how)


def padded(backend, dev, raw, rows, cols, to):
    """A Q4_0 matrix with blocks of zeros behind every row."""
    b = np.frombuffer(np.ascontiguousarray(raw).tobytes(), np.uint8).reshape(rows, cols // 32, 18)
    return backend.HipBuffer.from_gguf(dev, np.pad(b, ((0, 0), (0, (to - cols) // 32), (0, 0))).reshape(-1), backend.Q4_0,
                                       rows, to)


@pytest.mark.parametrize("nb,to", [(5, 6), (5, 8), (7, 8), (9, 10), (13, 16), (15, 16), (129, 130), (131, 132)])
def test_tiles_of_odd_rows(backend, dev, synth, nb, to):
    """Tiles of one to six token groups over rows with an odd number of blocks: to the bit what the same rows give with
    zeros up to an even one, whose scales and weights are read by other loads."""
    rows, cols, wide = 77, nb * 32, to * 32
    rng = synth.rng_for(nb + to)
    counts = [16, 32, 48, 64, 80, 96, 700]  # of the experts; so many that they are not streamed
    e, n = len(counts), sum(counts)
    ids = rng.permutation(np.repeat(np.arange(e), counts)).astype(np.int32)[:, None]
    plan = planned(backend, dev, ids, e)
    raw = [synth.q4_0_matrix(rng, e * rows, cols) for _ in range(3)]
    x = rng.standard_normal((n, cols)).astype(np.float32)
    weights = up(backend, dev, rng.uniform(-1, 1, (n, 1)).astype(np.float32))
    got = []
    for c in (cols, wide):
        w = [padded(backend, dev, r, e * rows, cols, c) for r in raw]
        xb = up(backend, dev, np.pad(x, ((0, 0), (0, c - cols))))
        act, y = (up(backend, dev, np.full(n * rows, 7.0, np.float32)) for _ in range(2))
        dev.moe_gate_up_q4_0(w[0], w[1], xb, *plan, act, e, rows, c, n, 1)
        dev.moe_down_q4_0(w[2], xb, plan[0], weights, plan[1], plan[2], y, e, rows, c, n, 1)
        dev.sync()
        got.append((act.numpy(), y.numpy()))
    for a, b in zip(*got):
        assert np.isfinite(a).all() and np.array_equal(bits(a), bits(b))


@pytest.mark.parametrize("n", [1, 3, 40, 150, 250])
def test_products_of_very_uneven_activations(backend, dev, orc, synth, n):
    """Blocks from 1e-9 to 1e6 in one row, rows of zeros, weights with zero scales: exact where Q8_0 is."""
    e, k, rows, cols = 4, 2, 40, 512
    rng = synth.rng_for(n)
    w = Experts(backend, dev, synth, 77, e, rows, cols, 2)
    x = (rng.standard_normal((n, cols // 32, 32)) * 10.0 ** rng.uniform(-9, 6, (n, cols // 32, 1))).astype(np.float32)
    x = x.reshape(n, cols)
    x[n // 2, : cols // 2] = 0
    if n > 2:
        x[1] = 0
    ids = some_ids(rng, n, e, k, "even")
    want, bound = mm.gate_up(*w.values, mm.q8_0_values(orc, x), ids, k, mm.SWIGLU)
    out = backend.HipBuffer.alloc(dev, n * k * rows)
    dev.moe_gate_up_q4_0(*w.dev, up(backend, dev, x), *planned(backend, dev, ids, e), out, e, rows, cols, n, k, mm.SWIGLU)
    dev.sync()
    off = np.abs(out.numpy().reshape(n * k, rows) - want) / bound
    assert (off <= 1).all(), off.max()


@pytest.mark.parametrize("n", [12, 24, 300])
def test_products_of_blocks_far_below_the_largest(backend, dev, orc, synth, n):
    """Rows whose largest block the weights leave out (q - 8 = 0), so that only blocks with scales 2^-27 of its remain.  In
    whole numbers nothing is lost; in tiles (n = 300) each value is off by at most 2^-32 of the row's largest scale."""
    e, rows, cols = 4, 40, 96
    rng = synth.rng_for(n)
    raw = synth.q4_0_matrix(rng, e * rows, cols).reshape(-1, 3, 18)
    raw[:, 0, 2:] = 0x88
    w = backend.HipBuffer.from_gguf(dev, raw.reshape(-1), backend.Q4_0, e * rows, cols)
    values = mm.q4_0_values(raw, e * rows, cols).reshape(e, rows, cols)
    x = rng.standard_normal((n, cols)).astype(np.float32)
    x[:, :32] *= 127 * 2.0 ** 14 / np.abs(x[:, :32]).max(1, keepdims=True)
    x[:, 32:] *= 127 * 2.0 ** -13 / np.abs(x[:, 32:]).max(1, keepdims=True)
    ids, weights = some_ids(rng, n, e, 1, "even"), np.ones((n, 1), np.float32)
    want, bound = mm.down(values, mm.q8_0_values(orc, x), ids, weights, 1)
    if n == 300:
        bound += np.abs(values[ids[:, 0], :, 32:]).sum(2) * 2.0 ** -32 * 2.0 ** 14
    else:
        assert bound.max() < 1e-6  # the largest block counts nothing here: its weights are zeros
    y = backend.HipBuffer.alloc(dev, n * rows)
    bid, starts, order = planned(backend, dev, ids, e)
    dev.moe_down_q4_0(w, up(backend, dev, x), bid, up(backend, dev, weights), starts, order, y, e, rows, cols, n, 1)
    dev.sync()
    off = np.abs(y.numpy().reshape(n, rows) - want) / bound
    assert (off <= 1).all(), off.max()


@pytest.mark.parametrize("n", [1, 20, 100, 200])
def test_products_keep_rows_that_are_not_finite_apart(backend, dev, synth, n):
    """Blocks whose scale passes f16, infinities among them, give values that are not finite in their token's rows
    alone."""
    e, k, rows, cols = 3, 2, 20, 128
    rng = synth.rng_for(6)
    w = Experts(backend, dev, synth, 5, e, rows, cols, 2)
    x = rng.standard_normal((n, cols)).astype(np.float32)
    ids = some_ids(rng, n, e, k, "even")
    plan = planned(backend, dev, ids, e)
    out = [backend.HipBuffer.alloc(dev, n * k * rows) for _ in range(3)]
    dev.moe_gate_up_q4_0(*w.dev, up(backend, dev, x), *plan, out[0], e, rows, cols, n, k)
    bad = n // 2
    for i, value in ((1, np.inf), (2, 3e9)):
        y = x.copy()
        y[bad, 40] = value
        dev.moe_gate_up_q4_0(*w.dev, up(backend, dev, y), *plan, out[i], e, rows, cols, n, k)
    dev.sync()
    a, b, c = (o.numpy().reshape(n, k * rows) for o in out)
    for got in (b, c):
        assert not np.isfinite(got[bad]).any()
        rest = np.arange(n) != bad
        assert np.array_equal(got[rest], a[rest])


@pytest.mark.parametrize("n", [8, 30, 130, 250])
def test_bad_ids_and_orders_are_left_out_and_reported(backend, dev, synth, n):
    e, k, rows, cols = 4, 2, 24, 64
    rng = synth.rng_for(9)
    gu, dn = Experts(backend, dev, synth, 1, e, rows, cols, 2), Experts(backend, dev, synth, 2, e, cols, 32)
    x = up(backend, dev, rng.standard_normal((n, cols)).astype(np.float32))
    act32 = up(backend, dev, rng.standard_normal((n * k, 32)).astype(np.float32))
    weights = up(backend, dev, np.ones((n, k), np.float32))
    ids = some_ids(rng, n, e, k, "even")
    out, y = backend.HipBuffer.alloc(dev, n * k * rows), backend.HipBuffer.alloc(dev, n * cols)

    def both(ids, starts, order):
        b = [up(backend, dev, np.asarray(a, np.int32).reshape(-1)) for a in (ids, starts, order)]
        dev.moe_gate_up_q4_0(*gu.dev, x, *b, out, e, rows, cols, n, k)
        dev.moe_down_q4_0(dn.dev[0], act32, b[0], weights, b[1], b[2], y, e, cols, 32, n, k)

    starts, order = mm.plan(ids, e)
    both(ids, starts, order)
    dev.sync()
    wrong = ids.copy()
    wrong[3, 1], wrong[7, 0] = e, -2
    for bad in ((wrong, starts, order), (ids, starts, np.where(np.arange(n * k) == 5, n * k, order)),
                (ids, starts, np.where(np.arange(n * k) == 6, -7, order)),
                (ids, np.where(np.arange(e + 1) == 2, 1 << 30, starts), order),
                (ids, np.where(np.arange(e + 1) == 1, -5, starts), order), (ids, starts[::-1], order),
                (ids[::-1], starts, order)):
        both(*bad)
        with pytest.raises(backend.HipError, match="expert ops"):
            dev.sync()
        dev.sync()
    both(ids, starts, order)
    dev.sync()


@pytest.mark.parametrize("n,off", [(n, off) for n in (1, 3, 7, 40, 300, 2500) for off in ("none", "some", "all")])
def test_plans_of_the_route_agree(backend, dev, synth, n, off):
    """What the route writes for tokens with few experts or none left is a plan that the products take without a word."""
    e, k, rows, cols = 16, 4, 24, 64
    rng = synth.rng_for(n)
    gu, dn = Experts(backend, dev, synth, 5, e, rows, cols, 2), Experts(backend, dev, synth, 6, e, cols, 32)
    logits = rng.standard_normal((n, e)).astype(np.float32)
    if off == "all":
        logits[:] = -np.inf
    elif off == "some":
        logits[rng.random((n, e)) < 0.5] = -np.inf
        logits[::3] = np.nan
        logits[1::4, 2:] = -np.inf
    r = Route(backend, dev, logits, None, k)
    r.call()
    x, act32 = (up(backend, dev, rng.standard_normal(s).astype(np.float32)) for s in ((n, cols), (n * k, 32)))
    out, y = (up(backend, dev, np.full(c, 7.0, np.float32)) for c in (n * k * rows, n * cols))
    dev.moe_gate_up_q4_0(*gu.dev, x, r.ids, r.starts, r.order, out, e, rows, cols, n, k)
    dev.moe_down_q4_0(dn.dev[0], act32, r.ids, r.weights, r.starts, r.order, y, e, cols, 32, n, k)
    ids = r.got()[0]  # (syncs)
    out, y = out.numpy().reshape(n * k, rows), y.numpy().reshape(n, cols)
    assert ((out == 7.0).all(1) == (ids.reshape(-1) < 0)).all()
    assert ((y == 0).all(1) == (ids < 0).all(1)).all() and np.isfinite(y).all()
    assert off != "all" or (ids == -1).all()


def plans_that_do_not_agree(ids, e):
    """(what, starts, order, whether the starts ascend) for valid ids."""
    starts, order = mm.plan(ids, e)
    end = starts[-1]
    run = int(np.argmax(np.diff(starts)))  # the longest
    at = starts[run]
    assert starts[run + 1] - at >= 3

    def changed(**places):
        o = order.copy()
        for place, value in places.items():
            o[int(place[1:])] = value
        return o

    yield "one twice, one nowhere", starts, changed(**{f"p{at + 1}": order[at]}), True
    yield "nothing named", np.zeros_like(starts), np.full_like(order, -1), True
    short = starts.copy()
    short[np.flatnonzero(starts == end)] = end - 1
    yield "the last one missing", short, changed(**{f"p{end - 1}": -1}), True
    yield "a hole in a run", starts, changed(**{f"p{at + 1}": -1}), True
    other = starts[run + 1] % end  # a place of another run
    yield "two in each other's run", starts, changed(**{f"p{at}": order[other], f"p{other}": order[at]}), True
    moved = starts.copy()
    moved[run + 1] = moved[run]
    yield "a run in the next one's", moved, order, True
    moved = starts.copy()
    moved[1], moved[2] = end, 0
    yield "starts that fall", moved, order, False
    moved = starts.copy()
    moved[0] = 1
    yield "not from 0 on", moved, order, False


@pytest.mark.parametrize("n", [8, 11, 30, 130, 250])
def test_what_a_plan_does_not_name_is_left_out(backend, dev, synth, n):
    """Assignments that are nowhere, twice, or in another expert's run: reported, the others as they should be, and what
    earlier calls left in the workspace (NaN here) in no output."""
    e, k, rows, cols = 4, 2, 40, 96
    rng = synth.rng_for(n + 1)
    gu, dn = Experts(backend, dev, synth, 3, e, rows, cols, 2), Experts(backend, dev, synth, 4, e, cols, 64)
    x = up(backend, dev, rng.standard_normal((n, cols)).astype(np.float32))
    act64 = up(backend, dev, rng.standard_normal((n * k, 64)).astype(np.float32))
    weights, nans = (up(backend, dev, a) for a in (rng.uniform(0.1, 1, (n, k)).astype(np.float32),
                                                   np.full((n, k), np.nan, np.float32)))
    ids = some_ids(rng, n, e, k, "even")

    def both(ids, starts, order):
        good = planned(backend, dev, some_ids(rng, n, e, k, "even"), e)
        out, y = (up(backend, dev, np.full(c, 7.0, np.float32)) for c in (n * k * rows, n * cols))
        dev.moe_down_q4_0(dn.dev[0], act64, good[0], nans, good[1], good[2], y, e, cols, 64, n, k)
        dev.sync()
        assert np.isnan(y.numpy()).all()
        b = [up(backend, dev, np.asarray(a, np.int32).reshape(-1)) for a in (ids, starts, order)]
        dev.moe_gate_up_q4_0(*gu.dev, x, *b, out, e, rows, cols, n, k)
        yield out
        dev.moe_down_q4_0(dn.dev[0], act64, b[0], weights, b[1], b[2], y, e, cols, 64, n, k)
        yield y

    def right(ids):
        out, y = both(ids, *mm.plan(ids, e))
        dev.sync()
        return out.numpy().reshape(n * k, rows), y.numpy().reshape(n, cols)

    whole = right(ids)
    slots = [right(np.where(np.arange(k) == s, ids, -1).astype(np.int32))[1] for s in range(k)]
    for what, starts, order, ascend in plans_that_do_not_agree(ids, e):
        got = []
        for b in both(ids, starts, order):
            with pytest.raises(backend.HipError, match="expert ops"):
                dev.sync()
            got.append(b.numpy())
        runs = [order[max(starts[j], 0):max(starts[j + 1], 0)] for j in range(e)]
        flat = ids.reshape(-1)
        named = np.array([i in runs[j] for i, j in enumerate(flat)])
        sure = named & ascend & np.array([(np.diff(runs[j]) > 0).all() for j in flat])
        # gate and up: what is named, or (starts that fall) nothing of it
        act = bits(got[0].reshape(n * k, rows))
        done, left = (act == bits(whole[0])).all(1), (act == bits(np.full(rows, 7.0))).all(1)
        assert (done | left).all() and not done[~named].any() and (not ascend or done[named].all()), what
        # down: the sum of each token's sure slots, with or without the named ones
        y, named, sure = got[1].reshape(n, cols), named.reshape(n, k), sure.reshape(n, k)
        for t in range(n):
            some = [np.zeros(cols, np.float32), slots[0][t], slots[1][t], whole[1][t]]  # of no slot, 0, 1, both
            may = [u for u in range(4) if all(sure[t, s] <= (u >> s & 1) <= named[t, s] for s in range(k))]
            assert any(np.array_equal(y[t], some[u]) for u in may), (what, t, may)


# ---- refusals --------------------------------------------------------------------------------

def test_refusals(backend, dev):
    b = [backend.HipBuffer.alloc(dev, 1 << 14) for _ in range(9)]
    p = [x.ptr for x in b]

    def refused(fn, *a, **kw):
        with pytest.raises(backend.HipError) as err:
            fn(*a, **kw)
        assert err.value.status == -1, str(err.value)

    norm = dev.residual_rms_norm_batch
    for dim, batch in ((0, 1), (48, 1), (12320, 1), (32, 0), (32, -1), (32, (1 << 20) + 1)):
        refused(norm, p[0], None, p[1], p[2], None, p[3], dim, batch, EPS)
    refused(norm, None, None, p[1], p[2], None, p[3], 32, 1, EPS)
    refused(norm, p[0], None, p[1], None, None, p[3], 32, 1, EPS)
    refused(norm, p[0] + 4, None, p[1], p[2], None, p[3], 32, 1, EPS)
    refused(norm, p[0], None, p[1], p[2], None, p[2], 32, 1, EPS)            # xn over h_out
    refused(norm, p[0], None, p[1], p[1] + 64, None, p[3], 32, 2, EPS)       # h_out half over h
    refused(norm, p[0], None, p[1], p[2], None, p[0] + 64, 32, 2, EPS)       # xn half over t
    refused(norm, p[0], None, p[1], p[0], None, p[3], 32, 2, EPS)            # h_out is t
    refused(norm, p[0], None, p[1], p[2], None, p[3], 32, 2, EPS, pack=p[3])
    refused(norm, p[0], p[2], p[1], p[2], None, p[3], 32, 2, EPS)            # w_post in h_out
    lg = dev.moe_logits
    for e, cols, batch in ((0, 32, 1), (513, 32, 1), (4, 16, 1), (4, 0, 1), (4, 32800, 1), (4, 32, 0)):
        refused(lg, p[0], p[1], p[2], e, cols, batch)
    refused(lg, p[0] + 4, p[1], p[2], 4, 32, 1)
    refused(lg, p[0], p[1], p[1] + 64, 4, 32, 1)
    rt = dev.moe_route
    for e, batch, k in ((0, 1, 1), (4, 0, 1), (4, 1, 0), (4, 1, 5), (64, 1, 33), (64, 1 << 18, 8)):
        refused(rt, p[0], None, p[1], p[2], p[3], p[4], e, batch, k)
    for kw in (dict(scoring=2), dict(n_groups=3), dict(n_groups=0), dict(n_groups=4, top_groups=5), dict(group_best=0),
               dict(n_groups=4, top_groups=0), dict(group_best=3), dict(scale=float("nan"))):
        refused(rt, p[0], None, p[1], p[2], p[3], p[4], 8, 2, 2, **kw)
    refused(rt, p[0], None, p[1], p[2], p[3], None, 8, 2, 2)
    refused(rt, p[0], None, p[1], p[1], p[3], p[4], 8, 2, 2)
    refused(rt, p[0], None, p[0], p[2], p[3], p[4], 8, 2, 2)
    gu, dn = dev.moe_gate_up_q4_0, dev.moe_down_q4_0
    for e, rows, cols, batch, k in ((0, 8, 32, 1, 1), (513, 8, 32, 1, 1), (4, 0, 32, 1, 1), (4, 8, 48, 1, 1),
                                    (4, 8, 32800, 1, 1), (4, 8, 32, 0, 1), (4, 8, 32, 1, 5), (4, 8, 32, 1, 0),
                                    (4, (1 << 20) + 1, 32, 1, 1), (4, 8, 32, (1 << 20) + 1, 1)):
        refused(gu, p[0], p[1], p[2], p[3], p[4], p[5], p[6], e, rows, cols, batch, k)
        refused(dn, p[0], p[2], p[3], p[1], p[4], p[5], p[6], e, rows, cols, batch, k)
    refused(gu, p[0], p[1], p[2], p[3], p[4], p[5], p[6], 4, 8, 32, 1, 1, 2)
    refused(gu, p[0], p[1], p[2], p[3], p[4], p[5], p[2], 4, 8, 32, 1, 1)
    refused(gu, p[0], None, p[2], p[3], p[4], p[5], p[6], 4, 8, 32, 1, 1)
    refused(gu, p[0], p[1], p[2] + 4, p[3], p[4], p[5], p[6], 4, 8, 32, 1, 1)
    refused(dn, p[0], p[2], p[3], None, p[4], p[5], p[6], 4, 8, 32, 1, 1)
    refused(dn, p[0], p[2], p[3], p[1], p[4], p[5], p[1], 4, 8, 32, 1, 1)
    dev.sync()


def test_more_tiles_than_a_launch_holds_are_refused(backend, dev):
    """Before anything is launched or allocated: of such outputs, of terabytes, only the place is looked at."""
    b = [backend.HipBuffer.alloc(dev, 1 << 8) for _ in range(6)]
    p, out, before = [x.ptr for x in b], 1 << 50, dev.workspace_bytes()
    for e in (1, 512):
        sizes = (e, 1 << 20, 32, 1 << 19, 1)
        for fn in (lambda: dev.moe_gate_up_q4_0(*p, out, *sizes), lambda: dev.moe_down_q4_0(*p, out, *sizes)):
            with pytest.raises(backend.HipError, match="too many for one call") as err:
                fn()
            assert err.value.status == -1
    assert dev.workspace_bytes() == before
    dev.sync()


def test_stream_of_more_threads_than_32_bits_count(backend, dev, orc, synth):
    """600 assignments, 512 experts of 2^20 rows: 9.6 million workgroups of 256 threads, an output past 2 GiB."""
    e, rows, cols, n = 512, 1 << 20, 32, 600
    rng = synth.rng_for(31)
    quants, base = rng.integers(0, 256, rows * 16, np.uint8), rng.uniform(0.01, 0.02, rows).astype(np.float16)
    w, first = backend.HipBuffer.alloc(dev, e * rows * 18, np.uint8), up(backend, dev, quants)
    lib, ctx = dev.lib, dev.ctx
    for i in range(e):  # the same quants, scales of their own
        assert lib.mrml_hip_memcpy_d2d_async(ctx, w.ptr + i * rows * 16, first.ptr, rows * 16) == 0
        scales = base * np.float16(1 << i % 5)
        assert lib.mrml_hip_memcpy_h2d(ctx, w.ptr + e * rows * 16 + i * rows * 2, scales.ctypes.data, rows * 2) == 0
    x = rng.standard_normal((n, cols)).astype(np.float32)
    ids = rng.integers(0, e, (n, 1)).astype(np.int32)
    act = backend.HipBuffer.alloc(dev, n * rows)
    dev.moe_gate_up_q4_0(w, w, up(backend, dev, x), *planned(backend, dev, ids, e), act, e, rows, cols, n, 1)
    dev.sync()
    some = np.r_[0:40, rows // 2:rows // 2 + 40, rows - 40:rows]
    q = quants.reshape(rows, 16)[some]
    q = np.concatenate([q & 15, q >> 4], 1).astype(np.float64) - 8.0
    xq, got = mm.q8_0_values(orc, x), np.empty(rows, np.float32)
    for a in (0, 1, 299, 511, 512, 598, 599):
        assert lib.mrml_hip_memcpy_d2h(ctx, got.ctypes.data, act.ptr + a * rows * 4, rows * 4) == 0
        wa = (q * base[some].astype(np.float64)[:, None] * (1 << ids[a, 0] % 5))[None]
        want, bound = mm.gate_up(wa, wa, xq[a:a + 1], np.zeros((1, 1), np.int32), 1, mm.GEGLU)
        assert (np.abs(got[some] - want[0]) <= bound[0]).all(), a


# ---- the layer -----------------------------------------------------------------------------------

class Layer:
    """Norm, logits, route, gate and up, down, and the next residual's norm, as a server's step calls them."""

    def __init__(self, backend, dev, synth, n, e=16, k=4, dim=256, ffn=96, seed=0):
        rng = synth.rng_for(100 + seed)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.dev, self.n, self.e, self.k, self.dim, self.ffn = dev, n, e, k, dim, ffn
        self.gu, self.dn = Experts(backend, dev, synth, seed + 1, e, ffn, dim, 2), Experts(backend, dev, synth, seed + 2, e, dim, ffn)
        self.router = f(e, dim) / 16
        self.w = {name: 1 + 0.1 * f(dim) for name in ("post", "next", "post2", "next2")}
        self.b = {name: up(backend, dev, a) for name, a in self.w.items()}
        self.b["router"] = up(backend, dev, self.router)
        sizes = dict(t=n * dim, h=n * dim, h1=n * dim, xn=n * dim, logits=n * e, weights=n * k, act=n * k * ffn, y=n * dim,
                     h2=n * dim, xn2=n * dim)
        self.b |= {name: backend.HipBuffer.alloc(dev, c) for name, c in sizes.items()}
        self.b |= {name: backend.HipBuffer.alloc(dev, c, np.int32) for name, c in
                   dict(ids=n * k, starts=e + 1, order=n * k).items()}
        self.b["pack"] = backend.HipBuffer.alloc(dev, n * dim // 32 * 40, np.uint8)

    def feed(self, rng):
        for name in ("t", "h"):
            self.b[name].copy_from_host((rng.standard_normal(self.n * self.dim) * 3).astype(np.float32))

    def call(self):
        b, d, n, e, k = self.b, self.dev, self.n, self.e, self.k
        d.residual_rms_norm_batch(b["t"], b["post"], b["h"], b["h1"], b["next"], b["xn"], self.dim, n, EPS, pack=b["pack"])
        d.moe_logits(b["xn"], b["router"], b["logits"], e, self.dim, n)
        d.moe_route(b["logits"], None, b["ids"], b["weights"], b["starts"], b["order"], e, n, k)
        d.moe_gate_up_q4_0_q8(*self.gu.dev, b["pack"], b["ids"], b["starts"], b["order"], b["act"], e, self.ffn, self.dim, n, k)
        d.moe_down_q4_0(self.dn.dev[0], b["act"], b["ids"], b["weights"], b["starts"], b["order"], b["y"], e, self.dim,
                        self.ffn, n, k)
        d.residual_rms_norm_batch(b["y"], b["post2"], b["h1"], b["h2"], b["next2"], b["xn2"], self.dim, n, EPS)

    def got(self, *names):
        self.dev.sync()
        return [self.b[name].numpy() for name in names]


@pytest.mark.parametrize("n", [1, 2, 19, 150, 450])
def test_layer(backend, dev, orc, synth, n):
    """Each step of the layer against 64 bits on the values that it was given."""
    L = Layer(backend, dev, synth, n, seed=n)
    L.feed(synth.rng_for(n))
    L.call()
    t, h, h1, xn, y, h2, xn2 = (a.reshape(n, -1) for a in L.got("t", "h", "h1", "xn", "y", "h2", "xn2"))
    logits, ids, weights, act = L.got("logits", "ids", "weights", "act")
    want_h1, want_xn = mm.residual_norm(t, L.w["post"], h, L.w["next"], EPS, True)
    assert np.array_equal(bits(h1), bits(want_h1)) and np.array_equal(bits(xn), bits(want_xn))
    logits, ids, weights = logits.reshape(n, -1), ids.reshape(n, -1), weights.reshape(n, -1)
    assert np.abs(logits - xn.astype(np.float64) @ L.router.astype(np.float64).T).max() <= 1e-5 * np.abs(logits).max()
    want_ids, want_w = mm.route(logits, None, L.k, mm.SOFTMAX)
    assert np.array_equal(ids, want_ids) and np.abs(weights - want_w).max() <= 2 * mm.U
    want, bound = mm.gate_up(*L.gu.values, mm.q8_0_values(orc, xn), ids, L.k, mm.GEGLU)
    assert (np.abs(act.reshape(n * L.k, -1) - want) <= bound).all()
    want, bound = mm.down(L.dn.values[0], mm.q8_0_values(orc, act.reshape(n * L.k, -1)), ids, weights, L.k)
    assert (np.abs(y - want) <= bound).all()
    want_h2, want_xn2 = mm.residual_norm(y, L.w["post2"], h1, L.w["next2"], EPS, True)
    assert np.array_equal(bits(h2), bits(want_h2)) and np.array_equal(bits(xn2), bits(want_xn2))


@pytest.mark.parametrize("n", [1, 30, 140, 450])
def test_layer_captured(backend, dev, synth, n):
    """A graph of the layer replayed over new inputs, with eager work of another size between: the eager bits each time."""
    a, b = Layer(backend, dev, synth, n, seed=50 + n), Layer(backend, dev, synth, 2 * n + 1, seed=60)
    rng = synth.rng_for(n + 7)
    a.feed(rng), b.feed(rng)
    b.call()
    a.call()
    dev.sync()
    graph = dev.capture(a.call)
    try:
        for _ in range(4):
            a.feed(rng)
            graph.launch()
            b.call()
            replayed = a.got("h1", "ids", "weights", "starts", "order", "act", "y", "h2", "xn2")
            a.call()
            for x, y in zip(replayed, a.got("h1", "ids", "weights", "starts", "order", "act", "y", "h2", "xn2")):
                assert np.array_equal(x, y)
    finally:
        graph.close()


def test_two_contexts_at_once(backend, dev, synth):
    """Layers on two contexts' streams at the same time give what each gives alone."""
    other = backend.HipDevice.new(0)
    try:
        layers = [Layer(backend, d, synth, n, seed=n) for d, n in ((dev, 60), (other, 90))]
        alone = []
        for L in layers:
            L.feed(synth.rng_for(1))
            L.call()
            alone.append(L.got("act", "y", "xn2"))
        for _ in range(5):
            for L in layers:
                L.call()
        for L, want in zip(layers, alone):
            for x, y in zip(L.got("act", "y", "xn2"), want):
                assert np.array_equal(x, y)
        del layers, L
    finally:
        other.close()
