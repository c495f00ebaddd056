"""Outputs that share memory with the rows they are formed from: refused, but for attention in place."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_paged import Batch, up

pytestmark = pytest.mark.gpu


def test_append_refuses_overlap(backend, dev):
    heads, kv, hd, n = 4, 2, 64, 3
    width, qd = (heads + 2 * kv) * hd, heads * hd
    k, v = (up(backend, dev, np.zeros((8, kv * hd), np.float16)) for _ in range(2))
    x = up(backend, dev, np.ones(qd * n + width * n + qd * n, np.float32))
    i32 = lambda a: up(backend, dev, np.array(a, np.int32))  # noqa: E731
    slots, pos = i32([0, 1, 2]), i32([0, 1, 2])
    qkv = x.ptr + 4 * qd * n
    for q, ok in ((qkv, False), (qkv + 16, False), (qkv + 4 * width, False), (qkv + 4 * width * n - 16, False),
                  (qkv - 4 * qd * n + 16, False), (qkv - 4 * qd * n, True), (qkv + 4 * width * n, True)):
        call = lambda: dev.qkv_postprocess_paged(qkv, q, k, v, slots, pos, n, 2, 4, heads, kv, hd, 1e4)  # noqa: B023, E731
        if ok:
            call()
            dev.sync()
        else:
            with pytest.raises(backend.HipError, match="share memory"):
                call()


def test_attention_refuses_overlap(backend, dev):
    for stride, shift, ok in ((256, 0, True), (256, 16, False), (512, 0, False), (512, 256 * 4, False), (256, 256 * 4, False)):
        b = Batch(backend, dev, 130, [3, 9], [1, 2], 20, 16, 4, 2, 64, pad=1, q_stride=stride).upload()
        b.d["out"] = b.d["q"].ptr + shift
        if ok:
            b.call()
            dev.sync()
        else:
            with pytest.raises(backend.HipError, match="shares memory"):
                b.call()
    rows = 4 * 256 * 4  # right behind, and right before
    b = Batch(backend, dev, 130, [3, 9], [1, 2], 20, 16, 4, 2, 64, pad=1).upload()
    both = up(backend, dev, np.concatenate([b.q.reshape(-1)] * 2))
    for q, out in ((both.ptr, both.ptr + rows), (both.ptr + rows, both.ptr)):
        b.d["q"], b.d["out"] = q, out
        both.copy_from_host(np.concatenate([b.q.reshape(-1)] * 2))
        b.call()
        dev.sync()


@pytest.mark.parametrize("requests", [3, 40, 300])  # each of the join's forms
@pytest.mark.parametrize("k_format", [0, 1])
def test_attention_in_place(backend, dev, requests, k_format):
    """out = q: the bits of a call with an output of its own, among them rows that the join forms again."""
    b = Batch(backend, dev, 131, [40] * requests, [1] * requests, 70, 16, 8, 2, 64, k_format, k_format).upload()
    b.q[1] = np.float32(3e7) * np.sign(b.q[1])  # scores past 2^20
    b.v[int(b.table[2, 0]) * 16 + 3, :2] = (0x00, 0x7E)  # a NaN that request 2 sees
    for name in ("q", "v"):
        b.d[name].copy_from_host(np.ascontiguousarray(getattr(b, name)))
    b.call()
    dev.sync()
    want = b.d["out"].numpy().reshape(b.max_rows, -1)[:b.rows]
    assert np.isnan(want[2]).any() and np.isfinite(want[0]).all()
    assert np.isfinite(want[1]).all() == (k_format == 0)  # q's block scales, 3e7 / 127, leave f16
    b.d["out"] = b.d["q"]
    b.call()
    dev.sync()
    got = b.d["q"].numpy().reshape(b.max_rows, -1)
    assert np.array_equal(got[:b.rows].view(np.uint32), want.view(np.uint32))
    assert np.array_equal(got[b.rows:], b.q[b.rows:])
