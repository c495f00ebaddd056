"""Which requests of a step are served (mrml_hip_block_tables), as a plain loop: pages are counted over all requests
so far that lack some, rows over all so far that want some and have their pages."""

from __future__ import annotations

import numpy as np

import paged_model as pm


def block_tables(lens, want, table, free, n_free, page_size, n_pages, max_rows, pos0):
    """table and free are changed in place; the rest is returned."""
    n, stride = table.shape
    stack = [int(x) for x in free[:n_free]]
    for r in range(n):
        if want[r] == -1 and 0 <= lens[r] <= stride * page_size:
            stack += [int(x) for x in table[r, :pm.pages(int(lens[r]), page_size)]]
    assert len(stack) <= n_pages
    free[:len(stack)] = stack
    there, lacked, wanted = len(stack), 0, 0
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
        elif add:
            first, last = pm.pages(have, page_size), pm.pages(have + add, page_size)
            lacked += last - first
            waits = last > first and lacked > there
            code = 3 if wanted + add > max_rows else 1 if waits else 0
            if not waits:
                wanted += add
            if code == 0:
                for j in range(first, last):
                    table[r, j] = stack.pop()
                rows = add
        for p in range(have, have + rows):
            slots.append(int(table[r, p // page_size]) * page_size + p % page_size)
            pos.append(pos0 + p)
        out.append(have + rows)
        status.append(code)
        starts.append(starts[-1] + rows)
    fill = max_rows - len(slots)
    i32 = lambda v: np.array(v, np.int32)  # noqa: E731
    return dict(lens=i32(out), n_free=len(stack), row_start=i32(starts), slots=i32(slots + [-1] * fill),
                pos=i32(pos + [0] * fill), status=i32(status))


def starved_chunk():
    """A prompt's chunk of 62 tokens that no page is there for, ahead of four decoders that have room in their
    pages of 16; 64 rows a step.  (lens, table, free, n_free, page_size, n_pages, max_rows)."""
    lens = np.array([0, 17, 20, 33, 3], np.int32)
    table = np.full((5, 6), -1, np.int32)
    at = 0
    for r, m in enumerate(lens):
        k = pm.pages(int(m), 16)
        table[r, :k] = range(at, at + k)
        at += k
    return lens, table, np.full(at, -1, np.int32), 0, 16, at, 64


def serve(step, lens, ends):
    """Steps until the chunk is in: step(want) gives (lens, status) after it; each decoder ends at its length of
    `ends`.  The statuses of every step."""
    history = []
    for _ in range(40):
        want = np.array([62] + [0 if m == 0 else -1 if m >= e else 1 for m, e in zip(lens[1:], ends)], np.int32)
        lens, status = step(want)
        history.append(status)
        if lens[0]:
            return lens, history
    raise AssertionError("the chunk was never served")
