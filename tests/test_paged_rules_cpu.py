"""Who is served in a step of a batch of requests, without a GPU: what waits, and that waiting ends."""

from __future__ import annotations

import numpy as np
import pytest

import paged_model as pm
import paged_rules


def test_decoders_go_on_beside_a_chunk_that_waits_for_pages():
    lens, table, free, n_free, ps, n_pages, max_rows = paged_rules.starved_chunk()
    state = dict(lens=lens, n_free=n_free)

    def step(want):
        state.update(paged_rules.block_tables(state["lens"], want, table, free, state["n_free"], ps, n_pages, max_rows, 0))
        return state["lens"], state["status"]

    end, history = paged_rules.serve(step, lens, [25, 24, 40, 10])
    assert end[0] == 62 and len(history) > 6
    for status in history[:-1]:
        assert list(status) == [1, 0, 0, 0, 0]


@pytest.mark.parametrize("seed", range(5))
def test_nobody_takes_what_another_waits_for(seed):
    """After a request that waits for pages none behind it takes one; after one that waits for rows none gets any."""
    rng = np.random.default_rng(seed)
    n, ps, stride, n_pages = 30, 4, 8, 60
    for _ in range(100):
        lens = rng.integers(0, 5, n).astype(np.int32)
        table = np.full((n, stride), -1, np.int32)
        perm, at = rng.permutation(n_pages), 0
        for r, m in enumerate(lens):
            if m:
                table[r, 0], at = perm[at], at + 1
        free = np.concatenate([perm[at:], np.full(at, -1)]).astype(np.int32)
        want, n_free = rng.choice([0, 1, 1, 2, 9], n), int(rng.integers(0, n_pages - at + 1))
        got = paged_rules.block_tables(lens, want, table, free, n_free, ps, n_pages, int(rng.integers(1, 60)), 0)
        lacked, waits_page, waits_row = 0, False, False
        for r in range(n):
            rows = got["row_start"][r + 1] - got["row_start"][r]
            need = pm.pages(int(lens[r] + want[r]), ps) - pm.pages(int(lens[r]), ps)
            lacked += need
            assert not rows or not (waits_row or need and waits_page)
            assert (got["status"][r] == 0) == (rows == want[r])
            waits_page |= got["status"][r] == 1
            waits_row |= got["status"][r] == 3 and not (need and lacked > n_free)  # its pages were there
