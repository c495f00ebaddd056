"""A batch of requests over one paged KV cache: page tables and slots
(mrml_hip_block_tables), the K/V append (mrml_hip_rope_kv_append_paged) and
attention with a shared prefix (mrml_hip_attention_paged), each against a plain
implementation, and a run of the three together.
"""

from __future__ import annotations

import numpy as np
import pytest

import paged_model as pm

pytestmark = pytest.mark.gpu


def up(backend, dev, a):
    return backend.HipBuffer.from_host(dev, np.ascontiguousarray(a))


# ------------------------------------------------------------ page tables
class Tables:
    """The arguments of block_tables on the device, in place or not."""

    def __init__(self, backend, dev, lens, want, table, free, n_free, page_size, max_rows, pos0=0, in_place=False):
        self.dev, self.page_size, self.max_rows, self.pos0 = dev, page_size, max_rows, pos0
        i32 = lambda v: up(backend, dev, np.array(v, np.int32))  # noqa: E731
        n = len(lens)
        self.n, self.stride, self.n_pages = n, table.shape[1], len(free)
        self.lens, self.want, self.table, self.free, self.n_free = i32(lens), i32(want), i32(table), i32(free), i32([n_free])
        self.table.shape = table.shape
        self.lens_out = self.lens if in_place else i32([-7] * n)
        self.n_free_out = self.n_free if in_place else i32([-7])
        self.row_start, self.slots, self.pos, self.status = i32([-7] * (n + 1)), i32([-7] * max_rows), i32([-7] * max_rows), i32([-7] * n)

    def call(self):
        self.dev.block_tables(self.lens, self.want, self.n, self.table, self.stride, self.page_size, self.free,
                              self.n_free, self.n_pages, self.lens_out, self.n_free_out, self.row_start, self.slots,
                              self.pos, self.max_rows, self.status, self.pos0)

    def check(self, ref, table, free, what=""):
        got = dict(lens=self.lens_out.numpy(), row_start=self.row_start.numpy(), slots=self.slots.numpy(),
                   pos=self.pos.numpy(), status=self.status.numpy())
        for k, v in got.items():
            assert np.array_equal(v, ref[k]), f"{what} {k}: {v} is not {ref[k]}"
        assert int(self.n_free_out.numpy()[0]) == ref["n_free"], what
        assert np.array_equal(self.table.numpy(), table), f"{what} table"
        assert np.array_equal(self.free.numpy()[:ref["n_free"]], free[:ref["n_free"]]), f"{what} free list"


def random_tables(rng, n, page_size, longest, stride, spare, finished=0.1, idle=0.1, most=40):
    lens = rng.integers(0, longest + 1, n)
    want = np.where(rng.random(n) < 0.5, 1, rng.integers(1, most + 1, n))
    want = np.where(rng.random(n) < idle, 0, want)
    want = np.where(rng.random(n) < finished, -1, want)
    held = [pm.pages(int(m), page_size) for m in lens]
    n_pages = max(1, sum(held) + spare)  # a cache has a page at least
    perm = rng.permutation(n_pages)
    table = np.full((n, stride), -1, np.int32)
    at = 0
    for r, k in enumerate(held):
        table[r, :k] = perm[at:at + k]
        at += k
    free = np.full(n_pages, -1, np.int32)
    free[:n_pages - at] = perm[at:]
    return lens, want, table, free, n_pages - at


@pytest.mark.parametrize("n,page_size,longest,max_rows", [
    (1, 16, 0, 1), (1, 1, 5, 64), (3, 16, 40, 7), (7, 24, 100, 200), (63, 8, 300, 1000), (64, 16, 64, 64),
    (65, 32, 500, 3000), (1000, 16, 700, 9000), (1025, 100, 300, 20000), (4096, 16, 50, 70000)])
def test_block_tables(backend, dev, n, page_size, longest, max_rows):
    rng = np.random.default_rng(n * 1000 + page_size)
    stride = pm.pages(longest + 20, page_size)
    for spare in (0, 3, n, 5 * n):  # from no free page to enough for all
        lens, want, table, free, n_free = random_tables(rng, n, page_size, longest, stride, spare)
        t = Tables(backend, dev, lens, want, table, free, n_free, page_size, max_rows, pos0=spare * 3)
        ref = pm.block_tables(lens, want, table, free, n_free, page_size, len(free), max_rows, spare * 3)
        for again in range(2):  # not in place: the same call gives the same answer
            t.call()
            dev.sync()
            t.check(ref, table, free, f"spare {spare}, call {again}")


def test_block_tables_refused_requests(backend, dev):
    """Each status: bad numbers, a table row too short, no row left, no page left; and nobody overtakes."""
    ps, stride = 4, 3
    lens = np.array([-1, 13, 5, 2, 12, 0, 4, 3, 8, 0], np.int32)
    want = np.array([1, 1, -2, 11, 0, 9, 4, 1, 1, -1], np.int32)
    table = np.arange(30, dtype=np.int32).reshape(10, 3) % 9
    for max_rows, n_free in ((100, 6), (13, 6), (14, 4), (9, 3), (8, 6), (100, 0)):
        free = np.array([20, 21, 22, 23, 24, 25] + [-1] * 24, np.int32)
        tab = table.copy()
        t = Tables(backend, dev, lens, want, tab, free, n_free, ps, max_rows)
        ref = pm.block_tables(lens, want, tab, free, n_free, ps, len(free), max_rows, 0)
        t.call()
        dev.sync()
        t.check(ref, tab, free, f"max_rows {max_rows}, {n_free} free")
        assert list(ref["status"][:3]) == [4, 4, 4] and ref["status"][3] == 2


def test_block_tables_in_place_and_captured(backend, dev):
    """A captured step replayed: lengths and free list advance in place; requests end and return their pages."""
    rng = np.random.default_rng(77)
    n, ps, stride, max_rows = 37, 16, 9, 60
    lens, want, table, free, n_free = random_tables(rng, n, ps, 100, stride, 40, finished=0.0)
    want = np.ones(n, np.int32)
    t = Tables(backend, dev, lens, want, table, free, n_free, ps, max_rows, pos0=11, in_place=True)
    graph = dev.capture(t.call)
    held_lens, held_free = np.array(lens, np.int32), n_free
    for step in range(40):
        if step % 9 == 8:
            want = np.where(rng.random(n) < 0.3, -1, 1).astype(np.int32)
        else:
            want = rng.integers(0, 2, n).astype(np.int32)
        t.want.copy_from_host(want)
        ref = pm.block_tables(held_lens, want, table, free, held_free, ps, len(free), max_rows, 11)
        graph.launch()
        dev.sync()
        t.check(ref, table, free, f"step {step}")
        held_lens, held_free = ref["lens"], ref["n_free"]
        own = [int(table[r, j]) for r in range(n) for j in range(pm.pages(int(held_lens[r]), ps))]
        assert len(set(own)) == len(own) and not set(own) & set(int(x) for x in free[:held_free])
    graph.close()


def test_block_tables_page_ids_outside(backend, dev):
    """Ids outside the cache in the table or the free list: slot -1, and the next sync says so, once."""
    table = np.array([[7, -1], [99, -1], [3, -1]], np.int32)
    free = np.array([1, 2, 400, -3, 5, 6, 8, 9], np.int32)
    t = Tables(backend, dev, [2, 2, 4], [1, 1, 1], table, free, 4, 4, 8)
    t.call()
    with pytest.raises(backend.HipError, match="outside the cache"):
        dev.sync()
    dev.sync()
    assert list(t.slots.numpy()) == [7 * 4 + 2, -1, -1] + [-1] * 5


def test_block_tables_refusals(backend, dev):
    ok = dict(lens=[1], want=[1], table=np.zeros((1, 2), np.int32), free=np.zeros(4, np.int32), n_free=2, page_size=4,
              max_rows=4)
    for change in (dict(page_size=0), dict(page_size=2049), dict(max_rows=0), dict(pos0=-1), dict(pos0=(1 << 21) + 1)):
        t = Tables(backend, dev, **{**ok, "max_rows": 4})
        for k, v in change.items():
            setattr(t, k, v)
        with pytest.raises(backend.HipError):
            t.call()
    for attr in ("n", "stride", "n_pages"):
        for v in (0, -1, 1 << 30):
            t = Tables(backend, dev, **ok)
            setattr(t, attr, v)
            with pytest.raises(backend.HipError):
                t.call()
    for attr in ("lens", "want", "table", "free", "n_free", "lens_out", "n_free_out", "row_start", "slots", "pos", "status"):
        t = Tables(backend, dev, **ok)
        setattr(t, attr, None)
        with pytest.raises(backend.HipError):
            t.call()
    dev.sync()


# ------------------------------------------------------------ append
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 4, 256), (1, 1, 32), (6, 2, 96), (16, 1, 64), (3, 3, 512), (4, 2, 160)])
@pytest.mark.parametrize("k_format,v_format", [(0, 0), (1, 2), (2, 1), (0, 1), (1, 0), (2, 2)])
def test_append_bit_exact(backend, dev, heads, kv_heads, head_dim, k_format, v_format):
    """Every row as the ring append stores it (one call a row, the slot as the cache row); slots of -1 and rows of the
    cache without a slot stay as they were."""
    rng = np.random.default_rng(heads * 100 + head_dim + k_format * 7 + v_format)
    n, ps, n_pages, base = 9, 3, 11, 10000.0
    width, qd, slots_n = (heads + 2 * kv_heads) * head_dim, heads * head_dim, ps * n_pages
    qkv = (rng.standard_normal((n, width)) * rng.choice([1e-3, 1.0, 300.0], (n, 1))).astype(np.float32)
    qkv[2, :40] = 0.0
    slots = rng.permutation(slots_n)[:n].astype(np.int32)
    slots[4] = -1
    pos = np.array([0, 5, 31, 32, 7, 40, 100000, 2, 63], np.int32)  # past the table too
    n_table = 41
    table = backend.HipBuffer.alloc(dev, n_table * head_dim)
    dev.rope_table(table, n_table, head_dim, base)
    kb, vb = (pm.ROW_BYTES[f](kv_heads * head_dim) for f in (k_format, v_format))
    k0, v0 = rng.integers(0, 256, (slots_n, kb)).astype(np.uint8), rng.integers(0, 256, (slots_n, vb)).astype(np.uint8)
    k, v, kr, vr = up(backend, dev, k0), up(backend, dev, v0), up(backend, dev, k0), up(backend, dev, v0)
    x, q = up(backend, dev, qkv), up(backend, dev, np.full((n, qd), 7.0, np.float32))
    want_q = np.full((n, qd), 7.0, np.float32)
    for i in range(n):
        if slots[i] < 0:
            continue
        row = up(backend, dev, qkv[i])
        dev.qkv_postprocess_batch(row, kr, vr, int(pos[i]), int(slots[i]), heads, kv_heads, head_dim, base, 1, slots_n,
                                  k_format, v_format, table=table, n_table=n_table)
        want_q[i] = row.numpy()[:qd]
    dev.qkv_postprocess_paged(x, q, k, v, up(backend, dev, slots), up(backend, dev, pos), n, n_pages, ps, heads,
                              kv_heads, head_dim, base, k_format, v_format, table=table, n_table=n_table)
    dev.sync()
    assert np.array_equal(q.numpy().view(np.uint32), want_q.view(np.uint32)), "q"
    assert np.array_equal(k.numpy(), kr.numpy()), "k"
    assert np.array_equal(v.numpy(), vr.numpy()), "v"
    assert np.array_equal(x.numpy(), qkv), "the stacked rows stay"


def test_append_slots_outside(backend, dev):
    """A slot past the cache stores nothing and the next sync fails."""
    n, heads, kv, hd = 3, 2, 1, 64
    k = up(backend, dev, np.zeros((8, kv * hd), np.float16))
    v = up(backend, dev, np.zeros((8, kv * hd), np.float16))
    x, q = up(backend, dev, np.ones((n, (heads + 2 * kv) * hd), np.float32)), up(backend, dev, np.zeros((n, heads * hd), np.float32))
    slots, pos = up(backend, dev, np.array([8, 2, 1 << 30], np.int32)), up(backend, dev, np.zeros(n, np.int32))
    dev.qkv_postprocess_paged(x, q, k, v, slots, pos, n, 2, 4, heads, kv, hd, 10000.0)
    with pytest.raises(backend.HipError, match="outside the cache"):
        dev.sync()
    dev.sync()
    got = v.numpy()
    assert (got[2] == 1).all() and np.count_nonzero(got) == hd and np.count_nonzero(q.numpy()[[0, 2]]) == 0


# ------------------------------------------------------------ attention
class Batch:
    """Requests over a paged cache, on the host and the device; rows outside every request's positions hold NaN."""

    def __init__(self, backend, dev, seed, before, new, prefix_len, page_size, heads, kv_heads, head_dim, k_format=0,
                 v_format=0, window=0, pad=2, q_stride=None, scale=None, spread=1.0):
        rng = np.random.default_rng(seed)
        self.dev, self.backend = dev, backend
        self.heads, self.kv_heads, self.hd, self.ps = heads, kv_heads, head_dim, page_size
        self.k_format, self.v_format, self.window, self.prefix_len = k_format, v_format, window, prefix_len
        self.scale = scale if scale is not None else 1.0 / np.sqrt(head_dim)
        lens = [b + n for b, n in zip(before, new)]
        self.lens, self.row_start = np.array(lens, np.int32), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.row_start[-1])
        self.max_rows = self.rows + pad
        pp, held = pm.pages(prefix_len, page_size), [pm.pages(m, page_size) for m in lens]
        self.stride = max(held) + 1
        self.n_pages = pp + sum(held) + 2
        perm = rng.permutation(self.n_pages).astype(np.int32)
        self.prefix = perm[:pp]
        self.table = np.full((len(lens), self.stride), -1, np.int32)
        at = pp
        for r, k in enumerate(held):
            self.table[r, :k] = perm[at:at + k]
            at += k
        t = np.arange(prefix_len)
        kept = [self.prefix[t // page_size].astype(np.int64) * page_size + t % page_size] if prefix_len else []
        for r, m in enumerate(lens):
            u = np.arange(m)
            kept.append(self.table[r, u // page_size].astype(np.int64) * page_size + u % page_size)
        kept = np.concatenate(kept) if kept else np.zeros(0, np.int64)
        n = self.n_pages * page_size
        self.k = pm.poison(pm.random_cache(rng, k_format, n, kv_heads, head_dim), k_format, kept)
        self.v = pm.poison(pm.random_cache(rng, v_format, n, kv_heads, head_dim), v_format, kept)
        self.q_stride = q_stride or heads * head_dim
        self.q = (rng.standard_normal((self.max_rows, self.q_stride)) * spread).astype(np.float32)

    def upload(self):
        b, d = self.backend, self.dev
        self.d = dict(q=up(b, d, self.q), k=up(b, d, self.k), v=up(b, d, self.v),
                      out=up(b, d, np.full((self.max_rows, self.heads * self.hd), 5.0, np.float32)),
                      prefix=up(b, d, self.prefix) if self.prefix_len else None, table=up(b, d, self.table),
                      lens=up(b, d, self.lens), row_start=up(b, d, self.row_start))
        return self

    def call(self):
        d = self.d
        self.dev.attention_paged(d["q"], d["k"], d["v"], d["out"], self.n_pages, self.ps, d["prefix"], self.prefix_len,
                                 d["table"], self.stride, d["lens"], d["row_start"], len(self.lens), self.max_rows,
                                 self.heads, self.kv_heads, self.hd, self.scale, self.window or None, self.k_format,
                                 self.v_format, self.q_stride)

    def reference(self, total=None):
        q = self.q[:, :self.heads * self.hd].reshape(self.max_rows, self.heads, self.hd)
        k, v = (pm.values(c, f, self.kv_heads, self.hd) for c, f in ((self.k, self.k_format), (self.v, self.v_format)))
        return pm.attention(q, k, v, self.k_format, self.prefix, self.prefix_len, self.table, self.lens, self.row_start,
                            self.ps, self.heads // self.kv_heads, self.scale, self.window, self.max_rows, total)

    def check(self, what=""):
        """Within 1e-5 of the largest value (the documented bound), and within what 32-bit arithmetic can do
        elementwise: a score is off by at most (hd + 8) half-steps of its terms' sizes (a half-step for each of hd
        products' sums and the splits of q), which shifts each weight by that much twice over (its own and the sum's),
        and the weights, their products and n sums by 64 half-steps more.  A weight is held as two f16 terms of its
        2^14-fold, relative to the largest one, rounded towards zero: in steps of 2^-24, so off by up to 2^-38 of the
        largest weight however small it is, which counts where the largest weight meets a v of 0 (quantised caches
        have many) and adds 2^-38 * sum_t |v_t|."""
        got = self.d["out"].numpy().reshape(self.max_rows, self.heads, self.hd).astype(np.float64)
        total = np.zeros((self.max_rows, self.heads, self.hd))
        ref, mag, unit = self.reference(total)
        assert (got[self.rows:] == 5.0).all(), f"{what}: rows behind the last request changed"
        got, ref, mag, unit = got[:self.rows], ref[:self.rows], mag[:self.rows], unit[:self.rows]
        assert np.isfinite(got).all(), what
        tol = mag * (2 * (self.hd + 8) * unit[..., None] + 64) * 2.0 ** -24 + total[:self.rows] * 2.0 ** -38
        off = np.abs(got - ref)
        worst = float((off / np.maximum(tol, 1e-300)).max())
        assert (off <= tol).all(), f"{what}: {worst:.3g} of the elementwise bound"
        top = np.abs(ref).max()
        assert off.max() <= 1e-5 * top, f"{what}: {off.max() / top:.3g} of the largest value"

    def run(self, what=""):
        self.upload()
        self.call()
        self.dev.sync()
        self.check(what)


SHAPES = [(8, 4, 256), (1, 1, 32), (3, 1, 64), (6, 2, 96), (8, 8, 128), (16, 1, 128), (4, 2, 512), (32, 2, 160)]


@pytest.mark.parametrize("heads,kv_heads,head_dim", SHAPES)
@pytest.mark.parametrize("k_format,v_format", [(0, 0), (1, 1), (2, 2), (1, 2), (0, 1), (2, 0)])
def test_attention_shapes_and_formats(backend, dev, heads, kv_heads, head_dim, k_format, v_format):
    Batch(backend, dev, 1, [0, 3, 40, 131], [1, 1, 1, 1], 75, 16, heads, kv_heads, head_dim, k_format, v_format).run()
    Batch(backend, dev, 2, [0, 30, 7], [3, 1, 19], 33, 7, heads, kv_heads, head_dim, k_format, v_format).run("several rows")


@pytest.mark.parametrize("before,new,prefix_len,page_size", [
    ([0], [1], 0, 16),            # one position at all
    ([0], [1], 1, 16),
    ([0], [200], 0, 16),          # a prompt from nothing
    ([5], [0], 10, 16),           # no rows
    ([0, 0, 9], [0, 1, 0], 64, 16),
    ([63, 64, 65], [1, 1, 1], 63, 64),
    ([127], [1], 128, 1),         # a page a position
    ([500], [1], 1000, 2048),     # a page larger than everything
    ([3000], [2], 5, 24),
    ([31] * 70, [1] * 70, 257, 16),   # more rows than a tile
    ([1, 900, 2], [130, 1, 65], 100, 32),
    ([17] * 33, [5] * 33, 511, 100)])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_attention_lengths(backend, dev, before, new, prefix_len, page_size, window):
    b = Batch(backend, dev, 3, before, new, prefix_len, page_size, 4, 2, 128, window=window).upload()
    b.call()
    dev.sync()
    if b.rows:
        b.check()
    else:
        assert (b.d["out"].numpy() == 5.0).all()


@pytest.mark.parametrize("k_format,v_format", [(0, 0), (1, 2)])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 4, 256), (12, 4, 64), (8, 1, 512)])
def test_attention_long(backend, dev, heads, kv_heads, head_dim, k_format, v_format):
    """Long enough that positions are split over workgroups; uneven requests; a window that cuts the prefix."""
    for window in (0, 2500):
        Batch(backend, dev, 5, [0, 2900, 10, 1111, 333], [1, 1, 4, 1, 1], 3001, 16, heads, kv_heads, head_dim, k_format,
              v_format, window=window).run(f"window {window}")


def test_attention_query_stride_and_idle_requests(backend, dev):
    """q inside stacked rows; requests without rows in between, first and last."""
    Batch(backend, dev, 6, [4, 9, 0, 70, 2], [0, 2, 0, 1, 0], 20, 8, 4, 2, 64, q_stride=4 * 64 + 2 * 2 * 64).run()


def test_attention_large_and_small_scores(backend, dev):
    """Scores of some hundreds (weights that vanish) and near zero; q beyond f16's range and far below it."""
    for spread, scale in ((3e5, 1e-5), (1e-6, 1e4), (40.0, 0.4)):
        b = Batch(backend, dev, 8, [20, 300], [1, 3], 90, 16, 4, 2, 128, spread=spread, scale=scale).upload()
        b.call()
        dev.sync()
        got = b.d["out"].numpy().reshape(b.max_rows, b.heads, b.hd)[:b.rows].astype(np.float64)
        ref, mag, unit = (x[:b.rows] for x in b.reference())
        tol = mag * (2 * (b.hd + 8) * unit[..., None] + 64) * 2.0 ** -24  # Batch.check's; errors grow with the scores
        assert (np.abs(got - ref) <= tol).all(), (spread, scale)


def test_attention_same_prefix_for_all_is_each_alone(backend, dev):
    """The batch's rows are the rows that each request gets in a call of its own."""
    b = Batch(backend, dev, 9, [10, 500, 3, 77], [1, 2, 1, 1], 700, 16, 8, 4, 256).upload()
    b.call()
    dev.sync()
    both = b.d["out"].numpy()[:b.rows].astype(np.float64)
    for r in range(4):
        lo, hi = b.row_start[r], b.row_start[r + 1]
        d, out = b.d, backend.HipBuffer.alloc(dev, int(hi - lo) * 8 * 256)
        dev.attention_paged(up(backend, dev, b.q[lo:hi]), d["k"], d["v"], out, b.n_pages, b.ps, d["prefix"], b.prefix_len,
                            up(backend, dev, b.table[r]), b.stride, up(backend, dev, b.lens[r:r + 1]),
                            up(backend, dev, np.array([0, hi - lo], np.int32)), 1, int(hi - lo), 8, 4, 256, b.scale)
        dev.sync()
        off = np.abs(out.numpy().reshape(hi - lo, -1) - both[lo:hi]).max()
        assert off <= 2e-5 * np.abs(both).max(), f"request {r}: {off}"  # 1e-5 each


def test_attention_equals_ring_attention(backend, dev):
    """A ring cache taken as a paged one gives mrml_hip_attention_causal's values (1e-5 of the largest)."""
    rng = np.random.default_rng(10)
    heads, kv, hd, cap, n_past = 8, 4, 256, 512, 400
    for kf, vf in ((0, 0), (1, 1), (2, 2), (1, 2)):
        k, v = (up(backend, dev, pm.random_cache(rng, f, cap, kv, hd)) for f in (kf, vf))
        q = up(backend, dev, rng.standard_normal(heads * hd).astype(np.float32))
        ring, out = backend.HipBuffer.alloc(dev, heads * hd), backend.HipBuffer.alloc(dev, heads * hd)
        for window in (None, 100):
            dev.attention_causal_ref(q, k, v, ring, n_past, heads, kv, hd, 1 / 16, window, cap, kf, vf)
            ids = up(backend, dev, np.arange(cap // 16, dtype=np.int32))
            i32 = lambda *a: up(backend, dev, np.array(a, np.int32))  # noqa: E731
            for prefix_len in (0, 300, 400):  # the first pages as the prefix, the rest as the request's own
                pages = prefix_len // 16
                own = ids.ptr + 4 * pages
                dev.attention_paged(q, k, v, out, cap // 16, 16, ids, pages * 16, own, cap // 16 - pages,
                                    i32(n_past + 1 - pages * 16), i32(0, 1), 1, 1, heads, kv, hd, 1 / 16, window, kf, vf)
                dev.sync()
                off = np.abs(out.numpy().astype(np.float64) - ring.numpy()).max()
                assert off <= 1e-5 * np.abs(ring.numpy()).max(), (kf, vf, window, prefix_len, off)


@pytest.mark.parametrize("bad", [-1, 1 << 20])
def test_attention_page_ids_outside(backend, dev, bad):
    """Positions of a page outside the cache are left out, as is what a length has past the table; sync says so."""
    b = Batch(backend, dev, 11, [40, 9], [1, 1], 48, 16, 4, 2, 128).upload()
    want = b.reference()[0]
    t = b.table.copy()
    t[0, 1] = bad
    b.d["table"].copy_from_host(t)
    b.call()
    with pytest.raises(backend.HipError, match="outside the cache"):
        dev.sync()
    dev.sync()
    got = b.d["out"].numpy().reshape(b.max_rows, 4, 128)
    # request 0 without its positions 16..31
    q = b.q.reshape(b.max_rows, 4, 128).astype(np.float64)
    k, v = pm.values(b.k, 0, 2, 128), pm.values(b.v, 0, 2, 128)
    slots = [int(p) * 16 + o for p in b.prefix for o in range(16)] + \
            [int(b.table[0, u // 16]) * 16 + u % 16 for u in range(41) if u // 16 != 1]
    for h in range(4):
        s = k[slots, h // 2] @ q[0, h] * b.scale
        p = np.exp(s - s.max())
        ref = p @ v[slots, h // 2] / p.sum()
        assert np.abs(got[0, h] - ref).max() <= 1e-5 * np.abs(want[:2]).max()
    assert np.abs(got[1] - want[1]).max() <= 1e-5 * np.abs(want[:2]).max()


def test_attention_infinite_values(backend, dev):
    """An infinite or NaN value reaches the rows that see its position, and only those."""
    for value in (np.inf, np.nan):
        b = Batch(backend, dev, 12, [0], [40], 0, 16, 2, 1, 128, pad=0)
        slot = int(b.table[0, 1]) * 16 + 4  # own position 20
        b.v.view(np.float16)[slot, 3] = value
        b.upload()
        b.call()
        dev.sync()
        got = b.d["out"].numpy().reshape(40, 2, 128)
        bad = np.zeros(got.shape, bool)
        bad[20:, :, 3] = True
        assert np.isfinite(got[~bad]).all(), value
        assert (np.isnan(got[bad]) if np.isnan(value) else got[bad] == value).all(), value


def test_attention_row_starts_outside(backend, dev):
    """Row starts and lengths that make no sense touch nothing outside the buffers; rows of no request stay."""
    b = Batch(backend, dev, 13, [10, 20, 30], [1, 1, 1], 16, 16, 4, 2, 64).upload()
    for starts, lens in (([0, 1 << 30, 2, 3], [5, 5, 5]), ([-5, -1, 1, 900], [1 << 30, -9, 31]), ([3, 2, 1, 0], [1, 1, 1])):
        b.d["row_start"].copy_from_host(np.array(starts, np.int32))
        b.d["lens"].copy_from_host(np.array(lens, np.int32))
        b.call()
        try:
            dev.sync()
        except backend.HipError as e:
            assert "outside the cache" in str(e)
    dev.sync()


def test_attention_refusals(backend, dev):
    def call(**change):
        b = Batch(backend, dev, 14, [3], [1], 4, 4, 4, 2, 64).upload()
        for k, v in change.items():
            if k in b.d:
                b.d[k] = v
            else:
                setattr(b, k, v)
        b.call()
        dev.sync()
    call()
    for k in ("q", "k", "v", "out", "table", "lens", "row_start", "prefix"):
        with pytest.raises(backend.HipError):
            call(**{k: None})
    for change in (dict(ps=0), dict(ps=4096), dict(n_pages=0), dict(n_pages=1 << 30), dict(stride=0), dict(stride=1 << 22),
                   dict(prefix_len=-1), dict(prefix_len=(1 << 21) + 1), dict(max_rows=0), dict(max_rows=(1 << 20) + 1),
                   dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(heads=64), dict(hd=48), dict(hd=544), dict(hd=0),
                   dict(q_stride=252), dict(q_stride=257), dict(k_format=3), dict(v_format=-1)):
        with pytest.raises(backend.HipError):
            call(**change)
    b = Batch(backend, dev, 14, [3], [1], 4, 4, 4, 2, 64).upload()
    b.d["q"] = b.d["q"].ptr + 4
    with pytest.raises(backend.HipError):
        b.call()


def test_attention_two_graphs_and_eager(backend, dev):
    """Two captured calls of different sizes and eager ones in between share the context's scratch: each replay gives
    the eager result, also after a larger eager call has made the scratch grow."""
    small = Batch(backend, dev, 15, [100, 7], [1, 1], 500, 16, 8, 4, 256).upload()
    wide = Batch(backend, dev, 16, [60] * 40, [1] * 40, 900, 16, 8, 4, 256).upload()
    one = backend.HipDevice.new(0)
    try:
        batches = []
        for b in (small, wide):
            b.dev = one
            b.upload()
            b.call()
            one.sync()
            batches.append((b, b.d["out"].numpy().copy(), one.capture(b.call)))
        grown = Batch(backend, one, 17, [0] * 9, [200] * 9, 64, 16, 8, 4, 256).upload()
        for turn in range(3):
            for b, want, graph in batches:
                b.d["out"].copy_from_host(np.zeros_like(want))
                graph.launch()
                one.sync()
                got = b.d["out"].numpy()
                assert np.array_equal(got[:b.rows], want[:b.rows]), f"replay {turn}"
            grown.call()
            one.sync()
            grown.check(f"eager {turn}")
        for _, _, graph in batches:
            graph.close()
        for b in (small, wide, grown):
            for x in b.d.values():
                if x is not None:
                    x.close()
    finally:
        one.close()


@pytest.mark.parametrize("n,heads,kv_heads,head_dim,k_format,v_format", [
    (700, 4, 2, 64, 0, 0), (513, 8, 1, 128, 0, 0), (600, 2, 1, 256, 1, 2), (300, 2, 1, 512, 0, 1), (4096, 2, 1, 32, 0, 0)])
def test_attention_many_requests(backend, dev, n, heads, kv_heads, head_dim, k_format, v_format):
    """More requests than a workgroup has threads: threads stand for several, some without rows, some with many."""
    rng = np.random.default_rng(n)
    before = rng.integers(0, 12, n)
    new = np.where(rng.random(n) < 0.2, 0, 1)
    new[[0, n // 2, n - 1]] = (3, 70, 0)
    before[[1, n // 2 + 1]] = (900, 333)
    for window in (0, 20):
        Batch(backend, dev, 30, list(before), list(new), 37, 16, heads, kv_heads, head_dim, k_format, v_format,
              window=window).run(f"window {window}")


@pytest.mark.parametrize("head_dim,k_format", [(64, 0), (256, 0), (128, 1)])
@pytest.mark.parametrize("window", [0, 7, 90])
def test_attention_rows_before_the_first_position(backend, dev, head_dim, k_format, window):
    """Rows of a request shorter than its rows stand inside the prefix, or before everything and see nothing (0)."""
    for prefix_len in (0, 5, 160):
        Batch(backend, dev, 31, [-3, 5, -150, -20], [5, 2, 160, 20], prefix_len, 16, 4, 2, head_dim, k_format, k_format,
              window=window).run(f"prefix {prefix_len}")


@pytest.mark.parametrize("k_format", [0, 1, 2])
def test_attention_scale_of_any_sign(backend, dev, k_format):
    for scale in (-0.2, 0.0, -3.0):
        Batch(backend, dev, 32, [20, 300, 0], [1, 3, 40], 90, 16, 4, 2, 128, k_format, k_format, scale=scale).run(f"{scale}")


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 4, 256), (4, 1, 128), (3, 3, 64), (2, 1, 512)])
@pytest.mark.parametrize("window", [1, 33, 400])
def test_attention_windows_over_many_rows(backend, dev, heads, kv_heads, head_dim, window):
    """Prompts' chunks whose windows begin in the prefix, in the chunk, and in a tile's middle."""
    Batch(backend, dev, 33, [0, 500, 77], [150, 300, 131], 290, 24, heads, kv_heads, head_dim, window=window).run()


@pytest.mark.parametrize("k_format,v_format", [(0, 0), (1, 1), (2, 2)])
@pytest.mark.parametrize("heads,kv_heads,rows", [(2, 1, 1), (32, 4, 140)])
def test_attention_not_finite_in_quantised_and_wide_calls(backend, dev, k_format, v_format, heads, kv_heads, rows):
    """A NaN in V's row or K's reaches every dim, or the block's dims, of the rows that see it and of its kv head."""
    at = 20
    for which in ("v", "k"):
        b = Batch(backend, dev, 34, [60, 0], [1, rows], 0, 16, heads, kv_heads, 64, k_format, v_format, pad=1)
        slot = int(b.table[0, at // 16]) * 16 + at % 16 if rows == 1 else int(b.table[1, at // 16]) * 16 + at % 16
        fmt = k_format if which == "k" else v_format
        cache = b.k if which == "k" else b.v
        cache[slot, :2] = (0x00, 0x7E)  # f16: dim 0 of kv head 0; else the scale of its first block
        b.upload()
        b.call()
        dev.sync()
        got = b.d["out"].numpy().reshape(b.max_rows, heads, 64)[:b.rows]
        bad = np.zeros(got.shape, bool)
        seen = slice(0, 1) if rows == 1 else slice(1 + at, None)
        bad[seen, :heads // kv_heads, slice(None) if which == "k" else slice(0, 1 if fmt == 0 else 32)] = True
        assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all(), which
        if rows > 1:
            assert heads * b.max_rows > 4096


def test_attention_not_finite_k_alone_among_many(backend, dev):
    """One NaN and one -inf among the scores of 64 positions: NaN, and no weight."""
    for value in (np.nan, np.inf, -np.inf):
        b = Batch(backend, dev, 35, [63], [1], 0, 16, 2, 1, 128, pad=0)
        b.q[:] = np.abs(b.q)
        slot = int(b.table[0, 1]) * 16 + 5
        b.k.view(np.float16)[slot, 7] = value
        b.upload()
        b.call()
        dev.sync()
        got = b.d["out"].numpy().reshape(2, 128)
        if value == -np.inf:
            with np.errstate(invalid="ignore"):
                ref = b.reference()[0][0]
            assert np.abs(got - ref).max() <= 1e-5 * np.abs(ref).max()
        else:
            assert np.isnan(got).all(), value


def test_attention_not_finite_q(backend, dev):
    """A row of q that is not finite gives NaN in its own head and row alone."""
    for k_format in (0, 1):
        for value in (np.nan, np.inf):
            b = Batch(backend, dev, 36, [70, 9], [1, 2], 40, 16, 4, 2, 64, k_format, k_format, pad=0)
            b.q[1, 64 + 3] = value
            b.upload()
            b.call()
            dev.sync()
            got = b.d["out"].numpy().reshape(3, 4, 64)
            ok = np.ones(got.shape, bool)
            ok[1, 1] = False
            assert np.isfinite(got[ok]).all(), (k_format, value)
            if k_format == 0:
                assert np.isnan(got[~ok]).all(), value


@pytest.mark.parametrize("k_format,v_format", [(0, 0), (1, 2)])
def test_places_past_four_gib(backend, dev, k_format, v_format):
    """Append and attention at places whose bytes lie past 32 bits give what they give at the first places."""
    heads, kv, hd, ps, m = 8, 8, 256, 16, 90
    rb = min(pm.ROW_BYTES[f](kv * hd) for f in (k_format, v_format))
    n_pages = (1 << 32) // (rb * ps) + 100
    rng = np.random.default_rng(37)
    width = (heads + 2 * kv) * hd
    x = up(backend, dev, rng.standard_normal((m, width)).astype(np.float32))
    k, v = (backend.HipBuffer.alloc(dev, n_pages * ps * pm.ROW_BYTES[f](kv * hd), np.uint8) for f in (k_format, v_format))
    i32 = lambda a: up(backend, dev, np.array(a, np.int32))  # noqa: E731
    pos, lens, starts = i32(np.arange(m)), i32([m - 40]), i32([0, 5])
    outs = []
    for pages in (rng.permutation(6), n_pages - 1 - rng.permutation(6)):
        t = np.arange(m)
        slots = i32(pages[t // ps] * ps + t % ps)
        q, out = backend.HipBuffer.alloc(dev, m * heads * hd), up(backend, dev, np.zeros((5, heads * hd), np.float32))
        dev.qkv_postprocess_paged(x, q, k, v, slots, pos, m, n_pages, ps, heads, kv, hd, 10000.0, k_format, v_format)
        prefix, own = i32(pages[:2]), i32(pages[2:])  # the first 32 positions as the prefix, the others the request's
        dev.attention_paged(q, k, v, out, n_pages, ps, prefix, 32, own, 4, lens, starts, 1, 5, heads,
                            kv, hd, hd ** -0.5, None, k_format, v_format)
        dev.sync()
        outs.append(out.numpy())
    assert np.isfinite(outs[0]).all() and np.array_equal(outs[0], outs[1])
    for y in (k, v):
        y.close()


def test_attention_uncountable_work_is_refused(backend, dev):
    """4096 requests over table rows of 2^21 positions could have more units of work than 32 bits count."""
    b = Batch(backend, dev, 38, [3], [1], 4, 16, 8, 8, 64).upload()
    d = b.d
    with pytest.raises(backend.HipError, match="too many"):
        dev.attention_paged(d["q"], d["k"], d["v"], d["out"], b.n_pages, 16, d["prefix"], 4, d["table"], 1 << 17,
                            d["lens"], d["row_start"], 4096, 4096, 8, 8, 64, 0.1)


def test_attention_largest_window_and_scales_refused(backend, dev):
    """A window past every position is none, also for rows before the first position; a scale that is no number is
    refused."""
    for before, new in ([40, 0], [1, 9]), ([-3, -150], [5, 160]):
        b = Batch(backend, dev, 40, before, new, 70, 16, 4, 2, 64, window=2 ** 31 - 1)
        b.run()
        wide = b.d["out"].numpy()
        b.window = 0
        b.run()
        assert np.array_equal(wide[:b.rows], b.d["out"].numpy()[:b.rows])
    for scale in (np.nan, np.inf, -np.inf):
        b.scale = scale
        with pytest.raises(backend.HipError, match="scale"):
            b.call()


def test_attention_two_contexts_at_once(backend, dev):
    """Calls of two contexts in flight together, each with its own stream and scratch."""
    one = backend.HipDevice.new(0)
    try:
        a = Batch(backend, dev, 41, [900, 30, 7], [1, 1, 1], 1500, 16, 8, 4, 256).upload()
        b = Batch(backend, one, 42, [3, 800], [60, 1], 700, 32, 16, 2, 128, 1, 2).upload()
        for _ in range(20):
            a.call()
            b.call()
        dev.sync()
        one.sync()
        a.check("first")
        b.check("second")
        for x in b.d.values():
            if x is not None:
                x.close()
    finally:
        one.close()


def test_append_captured(backend, dev):
    """A captured append replayed with other rows, slots and positions in between other work."""
    heads, kv, hd, ps, n_pages, n = 4, 2, 64, 4, 6, 5
    rng = np.random.default_rng(39)
    width = (heads + 2 * kv) * hd
    k, v = (up(backend, dev, np.zeros((n_pages * ps, kv * hd), np.float16)) for _ in range(2))
    x, q = backend.HipBuffer.alloc(dev, n * width), backend.HipBuffer.alloc(dev, n * heads * hd)
    slots, pos = up(backend, dev, np.zeros(n, np.int32)), up(backend, dev, np.zeros(n, np.int32))
    call = lambda: dev.qkv_postprocess_paged(x, q, k, v, slots, pos, n, n_pages, ps, heads, kv, hd, 10000.0)  # noqa: E731
    x.copy_from_host(np.zeros(n * width, np.float32))
    call()
    dev.sync()
    graph = dev.capture(call)
    for turn in range(4):
        rows, at, place = rng.standard_normal(n * width).astype(np.float32), rng.integers(0, 500, n), rng.permutation(n_pages * ps)[:n]
        got = []
        for run in (graph.launch, call):
            for c in (k, v):
                c.copy_from_host(np.zeros((n_pages * ps, kv * hd), np.float16))
            x.copy_from_host(rows)
            pos.copy_from_host(at.astype(np.int32))
            slots.copy_from_host(place.astype(np.int32))
            run()
            dev.sync()
            got.append([y.numpy().copy() for y in (q, k, v)])
        assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*got)), f"turn {turn}"
        assert np.count_nonzero(got[0][1].reshape(n_pages * ps, -1).any(1)) == n
    graph.close()


# ------------------------------------------------------------ the three together
@pytest.mark.parametrize("k_format,v_format", [(0, 0), (1, 1)])
def test_decode_loop(backend, dev, k_format, v_format):
    """Requests behind a shared prefix: a prompt step, then a captured decode step replayed, against a cache kept on
    the host (each request's rows as they were appended)."""
    rng = np.random.default_rng(20)
    heads, kv, hd, ps, n, prefix_len, base = 4, 2, 128, 16, 5, 100, 10000.0
    width, n_pages, stride, max_rows = (heads + 2 * kv) * hd, 60, 6, 64
    kb, vb = (pm.ROW_BYTES[f](kv * hd) for f in (k_format, v_format))
    k, v = (up(backend, dev, np.full((n_pages * ps, x), 0x7E, np.uint8)) for x in (kb, vb))
    table_rope = backend.HipBuffer.alloc(dev, 256 * hd)
    dev.rope_table(table_rope, 256, hd, base)
    i32 = lambda a: up(backend, dev, np.array(a, np.int32))  # noqa: E731
    # the prefix: appended as one request's rows, whose pages then stay as they are
    perm = rng.permutation(n_pages)
    prefix = i32(perm[:pm.pages(prefix_len, ps)])
    t = np.arange(prefix_len)
    x = up(backend, dev, rng.standard_normal((prefix_len, width)).astype(np.float32))
    q = backend.HipBuffer.alloc(dev, max(max_rows, prefix_len) * heads * hd)
    slots0 = (perm[t // ps] * ps + t % ps).astype(np.int32)
    dev.qkv_postprocess_paged(x, q, k, v, i32(slots0), i32(t), prefix_len, n_pages, ps, heads, kv, hd, base, k_format,
                              v_format, table=table_rope, n_table=256)
    free = np.full(n_pages, -1, np.int32)
    rest = perm[pm.pages(prefix_len, ps):]
    free[:len(rest)] = rest
    b = Tables(backend, dev, [0] * n, [1] * n, np.full((n, stride), -1, np.int32), free, len(rest), ps, max_rows,
               prefix_len, in_place=True)
    qkv = backend.HipBuffer.alloc(dev, max_rows * width)
    out = backend.HipBuffer.alloc(dev, max_rows * heads * hd)

    def step():
        b.call()
        dev.qkv_postprocess_paged(qkv, q, k, v, b.slots, b.pos, max_rows, n_pages, ps, heads, kv, hd, base, k_format,
                                  v_format, table=table_rope, n_table=256)
        dev.attention_paged(q, k, v, out, n_pages, ps, prefix, prefix_len, b.table, stride, b.lens, b.row_start, n,
                            max_rows, heads, kv, hd, hd ** -0.5, None, k_format, v_format)

    lens = np.zeros(n, np.int64)
    graph = None
    for turn in range(6):
        want = np.array([7, 1, 20, 3, 12]) if turn == 0 else np.array([1, 1, 0, 1, 1]) if turn != 4 else np.array([1, -1, 1, 1, 0])
        b.want.copy_from_host(want.astype(np.int32))
        qkv.copy_from_host(rng.standard_normal(max_rows * width).astype(np.float32))
        out.copy_from_host(np.full(max_rows * heads * hd, 5.0, np.float32))
        if turn < 2:
            step()
        else:
            graph = graph or dev.capture(step)
            graph.launch()
        dev.sync()
        lens = np.where(want < 0, 0, lens + want)
        starts = b.row_start.numpy()
        assert np.array_equal(b.lens.numpy(), lens) and np.array_equal(np.diff(starts), np.maximum(want, 0))
        ref, _, _ = pm.attention(q.numpy()[:max_rows * heads * hd].reshape(max_rows, heads, hd),
                                 pm.values(k.numpy().reshape(-1, kb), k_format, kv, hd),
                                 pm.values(v.numpy().reshape(-1, vb), v_format, kv, hd), k_format, prefix.numpy(),
                                 prefix_len, b.table.numpy(), lens, starts, ps, heads // kv, hd ** -0.5, 0, max_rows)
        got = out.numpy().reshape(max_rows, heads, hd)
        rows = int(starts[-1])
        assert (got[rows:] == 5.0).all()
        assert np.abs(got[:rows] - ref[:rows]).max() <= 1e-5 * np.abs(ref[:rows]).max(), f"turn {turn}"
    graph.close()
