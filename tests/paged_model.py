"""Paged KV caches in numpy for the tests: the step's bookkeeping as a plain
loop over the requests, cache rows in their formats, and attention in 64 bits.
"""

from __future__ import annotations

import numpy as np

ROW_BYTES = {0: lambda n: 2 * n, 1: lambda n: n // 32 * 34, 2: lambda n: n // 32 * 18}


def pages(n: int, ps: int) -> int:
    return -(-n // ps)


def block_tables(lens, want, table, free, n_free, page_size, n_pages, max_rows, pos0):
    """The rules of mrml_hip_block_tables, one request after the other.  table and free are changed in place; the
    rest is returned."""
    n, stride = table.shape
    free_list = [int(x) for x in free[:max(0, min(n_free, n_pages))]]
    for r in range(n):
        if want[r] == -1 and 0 <= lens[r] <= stride * page_size:
            free_list += [int(x) for x in table[r, :pages(int(lens[r]), page_size)]]
    free_list = free_list[:n_pages]
    free[:len(free_list)] = free_list
    total, rows_asked, pages_asked, taken = len(free_list), 0, 0, 0
    out, status, starts, slots, pos = [], [], [0], [], []
    for r in range(n):
        have, add = int(lens[r]), int(want[r])
        code, rows = 0, 0
        if have < 0 or have > stride * page_size or add < -1:
            code = 4
        elif add > stride * page_size - have:
            code = 2
        elif add == -1:
            have = 0
        elif add > 0:
            need = pages(have + add, page_size) - pages(have, page_size)
            rows_asked += add
            pages_asked += need
            if rows_asked > max_rows:
                code = 3
            elif need and pages_asked > total:
                code = 1
            else:
                for j in range(pages(have, page_size), pages(have + add, page_size)):
                    table[r, j] = free_list[total - 1 - taken]
                    taken += 1
                rows = add
        for i in range(rows):
            p = have + i
            slots.append(int(table[r, p // page_size]) * page_size + p % page_size)
            pos.append(pos0 + p)
        out.append(have + rows)
        status.append(code)
        starts.append(starts[-1] + rows)
    fill = max_rows - len(slots)
    i32 = lambda v: np.array(v, np.int32)  # noqa: E731
    return dict(lens=i32(out), n_free=total - taken, row_start=i32(starts), slots=i32(slots + [-1] * fill),
                pos=i32(pos + [0] * fill), status=i32(status))


def random_cache(rng, fmt: int, slots: int, kv_heads: int, head_dim: int) -> np.ndarray:
    """Cache bytes [slots][row bytes], values of about unit size."""
    if fmt == 0:
        return rng.standard_normal((slots, kv_heads * head_dim)).astype(np.float16).view(np.uint8).reshape(slots, -1)
    nb = kv_heads * head_dim // 32
    d = (rng.uniform(0.5, 1.5, (slots, nb, 1)) * (1.7 / 127 if fmt == 1 else 0.22)).astype(np.float16).view(np.uint8)
    q = rng.integers(0, 256, (slots, nb, 32 if fmt == 1 else 16)).astype(np.uint8)
    return np.concatenate([d, q], -1).reshape(slots, -1)


def poison(cache: np.ndarray, fmt: int, kept: np.ndarray) -> np.ndarray:
    """NaN (f16 values, or block scales) in every row but the kept ones."""
    c = cache.copy()
    hole = np.ones(len(c), bool)
    hole[kept] = False
    if fmt == 0:
        c.view(np.uint16)[hole] = 0x7E00
    else:
        b = c.reshape(len(c), -1, 34 if fmt == 1 else 18)
        b[hole, :, 0] = 0x00
        b[hole, :, 1] = 0x7E
    return c


def values(cache: np.ndarray, fmt: int, kv_heads: int, head_dim: int) -> np.ndarray:
    """[slots][kv_heads][head_dim] in 64 bits."""
    n = len(cache)
    if fmt == 0:
        return cache.view(np.float16).reshape(n, kv_heads, head_dim).astype(np.float64)
    b = cache.reshape(n, -1, 34 if fmt == 1 else 18)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    if fmt == 1:
        q = np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64)
    else:
        q = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8
    return (d * q).reshape(n, kv_heads, head_dim)


def q8_values(q: np.ndarray) -> np.ndarray:
    """q after quantize_f32_to_q8_0 (quant.rs:193-228), in 64 bits."""
    x = q.astype(np.float32).reshape(-1, 32)
    scale = (np.abs(x).max(1, keepdims=True) / np.float32(127)).astype(np.float32)
    d = (scale.view(np.uint32) & np.uint32(0xFFFFE000)).view(np.float32).astype(np.float64)
    d[scale < 2.0 ** -14] = 0.0
    inv = np.where(scale > 0, np.float32(1) / np.where(scale > 0, scale, np.float32(1)), np.float32(0)).astype(np.float32)
    t = (x * inv).astype(np.float64)
    return (d * np.clip(np.sign(t) * np.floor(np.abs(t) + 0.5), -128, 127)).reshape(q.shape)


def attention(q, k, v, k_fmt, prefix, prefix_len, table, lens, row_start, page_size, group, scale, window, max_rows, total=None):
    """(out, weight of |v|, largest score error unit) in 64 bits: rows [max_rows][heads][head_dim], NaN where a row
    belongs to no request; the second is sum_t p_t |v_t|, the third max_t |scale| * sum_d |q_d k_td| a row and head.
    total, if given, gets sum_t |v_t|."""
    heads, hd = q.shape[1:]
    out = np.full((max_rows, heads, hd), np.nan)
    mag, unit = np.zeros((max_rows, heads, hd)), np.zeros((max_rows, heads))
    qv = q.astype(np.float64) if k_fmt == 0 else q8_values(q)
    t = np.arange(prefix_len)
    shared = (np.asarray(prefix, np.int64)[t // page_size] * page_size + t % page_size) if prefix_len else t
    for r in range(len(lens)):
        rows = range(row_start[r], row_start[r + 1])
        u = np.arange(lens[r])
        mine = np.asarray(table[r], np.int64)[u // page_size] * page_size + u % page_size
        slots = np.concatenate([shared, mine]).astype(np.int64)
        for row in rows:
            at = prefix_len + int(lens[r]) - (int(row_start[r + 1]) - row)
            lo = max(0, at - window + 1) if window else 0
            see = slots[lo:at + 1]
            if at < 0 or not len(see):
                out[row] = 0.0
                continue
            for h in range(heads):
                kk, vv = k[see, h // group], v[see, h // group]
                s = kk @ qv[row, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[row, h] = p @ vv
                mag[row, h] = p @ np.abs(vv)
                if total is not None:
                    total[row, h] = np.abs(vv).sum(0)
                unit[row, h] = abs(scale) * (np.abs(kk) @ np.abs(qv[row, h])).max()
    return out, mag, unit
