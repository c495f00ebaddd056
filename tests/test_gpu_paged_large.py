"""The paged ops at sizes past what one launch, one workgroup's pass or a small batch takes, and steps whose first
request does not begin at row 0."""

from __future__ import annotations

import numpy as np
import pytest

import paged_model as pm
import paged_rules
from test_gpu_paged import Batch, Tables, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k_format,v_format", [(0, 0), (2, 1)])
def test_append_more_rows_than_a_launch_takes(backend, dev, k_format, v_format):
    """140001 rows (more than two grids of 65535) in one call and in calls of 50000: the same bits, -1 slots among them."""
    heads, kv, hd, ps, n = 2, 1, 32, 16, 140001
    rng = np.random.default_rng(150)
    n_pages, width = n // ps + 2, (heads + 2 * kv) * hd
    kb, vb = (pm.ROW_BYTES[f](kv * hd) for f in (k_format, v_format))
    x = up(backend, dev, rng.standard_normal((n, width), dtype=np.float32))
    slots_h = rng.permutation(n_pages * ps)[:n].astype(np.int32)
    slots_h[rng.integers(0, n, 500)] = -1
    slots, pos = up(backend, dev, slots_h), up(backend, dev, rng.integers(0, 3000, n).astype(np.int32))
    got = []
    for step in (n, 50000):
        k, v = (up(backend, dev, np.full(n_pages * ps * b, 0x5A, np.uint8)) for b in (kb, vb))
        q = up(backend, dev, np.full(n * heads * hd, 7.0, np.float32))
        for at in range(0, n, step):
            m = min(step, n - at)
            dev.qkv_postprocess_paged(x.ptr + 4 * at * width, q.ptr + 4 * at * heads * hd, k, v, slots.ptr + 4 * at,
                                      pos.ptr + 4 * at, m, n_pages, ps, heads, kv, hd, 10000.0, k_format, v_format)
        dev.sync()
        got.append([q.numpy(), k.numpy(), v.numpy()])
        for b in (k, v, q):
            b.close()
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*got))
    q = got[0][0].reshape(n, -1)
    assert (q[slots_h < 0] == 7.0).all() and not (q[slots_h >= 0] == 7.0).all(1).any()
    rows = got[0][1].reshape(n_pages * ps, kb)
    assert (rows == 0x5A).all(1).sum() == n_pages * ps - (slots_h >= 0).sum()


def test_block_tables_largest_steps(backend, dev):
    """2^20 rows a step: four requests that add 100000 to 300000 tokens each; and 4096 requests of 256."""
    for n, ps, add in ((4, 2048, [100000, 300000, 262143, 300000]), (4096, 64, [256] * 4096)):
        stride, lens = (1 << 21) // ps // (1 if n == 4 else 256), np.arange(n, dtype=np.int32) % 7
        held = [pm.pages(int(m), ps) for m in lens]
        n_pages = sum(pm.pages(int(m) + a, ps) for m, a in zip(lens, add)) + 3
        perm = np.random.default_rng(n).permutation(n_pages)
        table, at = np.full((n, stride), -1, np.int32), 0
        for r, k in enumerate(held):
            table[r, :k] = perm[at:at + k]
            at += k
        free = np.concatenate([perm[at:], np.full(at, -1)]).astype(np.int32)
        t = Tables(backend, dev, lens, add, table, free, n_pages - at, ps, 1 << 20, pos0=1 << 21)
        ref = paged_rules.block_tables(lens, add, table, free, n_pages - at, ps, n_pages, 1 << 20, 1 << 21)
        t.call()
        dev.sync()
        t.check(ref, table, free)
        assert ref["row_start"][-1] > 900000


@pytest.mark.parametrize("heads,kv_heads,head_dim,k_format,window", [(2, 1, 64, 0, 0), (2, 1, 256, 0, 3000), (4, 1, 32, 1, 0), (1, 1, 512, 0, 0)])
def test_attention_long_prompt(backend, dev, heads, kv_heads, head_dim, k_format, window):
    """A prompt of 20011 rows from nothing, behind 100 shared positions: some of its rows against 64 bits."""
    b = Batch(backend, dev, 151, [0, 5], [20011, 1], 100, 32, heads, kv_heads, head_dim, k_format, k_format, window=window).upload()
    b.call()
    dev.sync()
    got = b.d["out"].numpy().reshape(b.max_rows, heads, head_dim)
    assert np.isfinite(got[:b.rows]).all() and (got[b.rows:] == 5.0).all()
    kv, vv = (pm.values(c, k_format, kv_heads, head_dim) for c in (b.k, b.v))
    q = b.q.reshape(b.max_rows, heads, head_dim)
    q = q.astype(np.float64) if k_format == 0 else pm.q8_values(q)
    slots = [b.prefix[t // 32] * 32 + t % 32 for t in range(100)] + [b.table[0, u // 32] * 32 + u % 32 for u in range(20011)]
    top, off = 0.0, 0.0
    for row in (0, 1, 15, 16, 127, 128, 129, 4095, 9999, 16384, 19999, 20010):
        see = np.array(slots[max(0, 101 + row - window) if window else 0:101 + row])
        for h in range(heads):
            s = kv[see, 0] @ q[row, h] * b.scale
            p = np.exp(s - s.max())
            want = p @ vv[see, 0] / p.sum()
            top, off = max(top, np.abs(want).max()), max(off, np.abs(got[row, h] - want).max())
    assert off <= 1e-5 * top, off / top


@pytest.mark.parametrize("heads,kv_heads,head_dim,k_format", [(8, 4, 256, 0), (4, 2, 64, 1)])
@pytest.mark.parametrize("requests,new", [(3, 1), (70, 1), (4, 50)])
def test_attention_first_request_behind_row_0(backend, dev, heads, kv_heads, head_dim, k_format, requests, new):
    """Rows before the first request's belong to none: they stay, and the others are what they are at row 0."""
    for window in (0, 60):
        b = Batch(backend, dev, 152, [40] * requests, [new] * requests, 75, 16, heads, kv_heads, head_dim, k_format, k_format,
                  window=window, pad=9).upload()
        b.row_start = b.row_start + 7
        b.d["row_start"].copy_from_host(b.row_start)
        b.call()
        dev.sync()
        got = b.d["out"].numpy().reshape(b.max_rows, heads, head_dim)
        ref = b.reference()[0]
        assert (got[:7] == 5.0).all() and (got[b.rows + 7:] == 5.0).all()
        own = slice(7, b.rows + 7)
        assert np.abs(got[own] - ref[own]).max() <= 1e-5 * np.abs(ref[own]).max()
