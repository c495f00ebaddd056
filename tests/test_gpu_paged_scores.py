"""Attention over a paged cache where its scores are very large or all minus infinity, against the formula in 64
bits."""

from __future__ import annotations

import numpy as np
import pytest

import paged_model as pm
from test_gpu_paged import Batch

pytestmark = pytest.mark.gpu


def scores(b, row, r):
    """[heads][seen positions]: a row's scores in 64 bits, |scale| * sum_d |q_d k_td|, and v of those positions."""
    heads, kv, hd, ps = b.heads, b.kv_heads, b.hd, b.ps
    q = b.q[row, :heads * hd].reshape(heads, hd)
    q = q.astype(np.float64) if b.k_format == 0 else pm.q8_values(q)
    t, u = np.arange(b.prefix_len), np.arange(b.lens[r])
    slots = [b.table[r, u // ps].astype(np.int64) * ps + u % ps]
    if b.prefix_len:
        slots.insert(0, b.prefix[t // ps].astype(np.int64) * ps + t % ps)
    at = b.prefix_len + int(b.lens[r]) - (int(b.row_start[r + 1]) - row)
    see = np.concatenate(slots)[max(0, at - b.window + 1) if b.window else 0:at + 1]
    k, v = (pm.values(c, f, kv, hd)[see] for c, f in ((b.k, b.k_format), (b.v, b.v_format)))
    group = np.arange(heads) // (heads // kv)
    s = np.einsum("hd,thd->ht", q, k[:, group]) * b.scale
    size = np.einsum("hd,thd->ht", np.abs(q), np.abs(k[:, group])) * abs(b.scale)
    return s, size, v[:, group]


@pytest.mark.parametrize("spread", [1e3, 3e5, 1e7, 1e9, 1e12, 1e20, -1e9])
@pytest.mark.parametrize("heads,kv_heads,head_dim,k_format,v_format", [
    (4, 2, 128, 0, 0), (8, 4, 256, 0, 0), (2, 1, 64, 0, 1), (3, 1, 512, 0, 0), (4, 2, 128, 1, 2), (2, 1, 512, 2, 0)])
def test_large_scores_leave_one_position(backend, dev, heads, kv_heads, head_dim, k_format, v_format, spread):
    """Scores up to 10^20 apart from each other: where the largest one leads by more than 32-bit scores can be off, the
    row's output is that position's v.  A score is off by at most (hd + 8) half-steps of its terms' sizes, and a lead
    of 40 beyond that of both leaves the others at most n e^-40 < 2^-44 of the weight, for n < 2^13.  The weight itself
    is held in two f16 terms rounded towards zero (2^-21 of it) and its sum, product and quotient take a few half-steps
    of 2^-24: 2^-20 in all.  The quantised path rounds q to d * quants with d in f16, so its q stays within f16 and
    the scale carries the size."""
    far = abs(spread)
    q_size = far if k_format == 0 else min(far, 1e3)
    scale = (1.0 if k_format == 0 else far / q_size) * np.sign(spread)
    for seed, before, new, prefix_len, window in ((50, [0], [1], 0, 0), (51, [0, 300, 12], [1, 3, 40], 90, 0), (52, [700, 5], [1, 30], 130, 60)):
        b = Batch(backend, dev, seed, before, new, prefix_len, 16, heads, kv_heads, head_dim, k_format, v_format,
                  window=window, spread=q_size, scale=scale).upload()
        b.call()
        dev.sync()
        got = b.d["out"].numpy().reshape(b.max_rows, heads, head_dim).astype(np.float64)
        led = all_rows = 0
        for r in range(len(before)):
            for row in range(b.row_start[r], b.row_start[r + 1]):
                s, size, v = scores(b, row, r)
                for h in range(heads):
                    all_rows += 1
                    order = np.argsort(s[h])
                    top = order[-1]
                    off = (head_dim + 8) * size[h] * 2.0 ** -24
                    if len(order) > 1 and (s[h, top] - off[top] - (s[h] + off))[order[:-1]].min() < 40:
                        continue
                    led += 1
                    want = v[top, h]
                    others = np.abs(v[:, h]).max(0) * 2.0 ** -44
                    assert (np.abs(got[row, h] - want) <= np.abs(want) * 2.0 ** -20 + others).all(), \
                        (seed, row, h, s[h, top], got[row, h][:4], want[:4])
        assert led == all_rows if before == [0] else spread == 1e3 or led > all_rows // 2


@pytest.mark.parametrize("k_format,v_format", [(0, 0), (0, 1)])
@pytest.mark.parametrize("n", [1, 40, 900])
def test_scores_of_minus_infinity_only(backend, dev, k_format, v_format, n):
    """0 / 0 where every score that a row sees is minus infinity: NaN, as mrml_hip_attention_causal gives; a finite one
    among them takes the whole weight."""
    heads, kv, hd = 2, 1, 64
    for finite in (False, True):
        b = Batch(backend, dev, 60 + n, [n - 1, 3], [1, 1], 0, 16, heads, kv, hd, k_format, v_format, pad=0)
        b.q[:] = np.abs(b.q) + np.float32(0.5)
        u = np.arange(n)
        slots = b.table[0, u // 16].astype(np.int64) * 16 + u % 16
        b.k.view(np.float16)[slots, 9] = -np.inf
        if finite:
            b.k.view(np.float16)[slots[n // 2], 9] = 1.0
        b.upload()
        b.call()
        dev.sync()
        got = b.d["out"].numpy().reshape(2, heads, hd)
        if finite:
            v = pm.values(b.v, v_format, kv, hd)[slots[n // 2], 0]
            assert (np.abs(got[0] - v) <= np.abs(v) * 2.0 ** -20).all()
        else:
            assert np.isnan(got[0]).all()
        assert np.isfinite(got[1]).all()
        ring = backend.HipBuffer.alloc(dev, heads * hd)
        if not finite and (k_format, v_format) == (0, 0):
            d = {x: backend.HipBuffer.from_host(dev, np.ascontiguousarray(getattr(b, x)[slots])) for x in ("k", "v")}
            dev.attention_causal_ref(backend.HipBuffer.from_host(dev, b.q[0]), d["k"], d["v"], ring, n - 1, heads, kv, hd,
                                     b.scale, None, n, 0, 0)
            dev.sync()
            assert np.isnan(ring.numpy()).all()


def test_products_past_f32_give_what_the_formula_in_f32_gives(backend, dev):
    """q and K so large that the scores themselves leave f32: +inf or -inf only; 0 / 0 either way."""
    for sign in (1.0, -1.0):
        b = Batch(backend, dev, 70, [40], [1], 20, 16, 2, 1, 64, pad=0)
        b.k.view(np.float16)[np.isfinite(b.k.view(np.float16))] = 6e4
        b.q[:] = np.float32(sign * 3e38)
        b.scale = 1.0
        b.upload()
        b.call()
        dev.sync()
        assert np.isnan(b.d["out"].numpy()).all(), sign


def test_rows_that_see_nothing_stay_zero(backend, dev):
    """Beside rows whose scores are all minus infinity, rows before the first position still give 0."""
    b = Batch(backend, dev, 71, [-3, 20], [5, 2], 0, 16, 2, 1, 64)
    b.q[:] = np.abs(b.q) + np.float32(0.5)
    b.k.view(np.float16)[:, 9] = -np.inf
    b.upload()
    b.call()
    dev.sync()
    got = b.d["out"].numpy().reshape(b.max_rows, -1)
    assert (got[:3] == 0.0).all() and np.isnan(got[3:7]).all() and (got[7:] == 5.0).all()
