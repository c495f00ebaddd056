"""Which requests of a step are served where pages or rows are short (mrml_hip_block_tables)."""

from __future__ import annotations

import numpy as np
import pytest

import paged_model as pm
import paged_rules
from test_gpu_paged import Tables, random_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,page_size,longest,max_rows", [
    (2, 16, 20, 9), (64, 16, 64, 300), (65, 8, 30, 300), (700, 16, 500, 5000), (1025, 32, 200, 7000), (4096, 4, 30, 6000)])
def test_short_of_pages_and_rows(backend, dev, n, page_size, longest, max_rows):
    rng = np.random.default_rng(n * 7 + page_size)
    seen = set()
    for spare in (0, 1, n // 9, n // 2, 2 * n):
        for most in (1, 3, 40):
            lens, want, table, free, n_free = random_tables(rng, n, page_size, longest, 64, spare, most=most,
                                                               finished=0.02)
            t = Tables(backend, dev, lens, want, table, free, n_free, page_size, max_rows, pos0=5)
            ref = paged_rules.block_tables(lens, want, table, free, n_free, page_size, len(free), max_rows, 5)
            t.call()
            dev.sync()
            t.check(ref, table, free, f"spare {spare}, most {most}")
            seen |= set(ref["status"])
    assert n == 2 or seen == {0, 1, 3}  # both kinds of waiting are there


def test_decoders_go_on_beside_a_chunk_that_waits_for_pages(backend, dev):
    """The chunk's rows are not kept from the decoders behind it; they end, return their pages, and it is served."""
    lens, table, free, n_free, ps, _, max_rows = paged_rules.starved_chunk()
    t = Tables(backend, dev, lens, np.zeros(5, np.int32), table, free, n_free, ps, max_rows, in_place=True)

    def step(want):
        t.want.copy_from_host(want)
        t.call()
        dev.sync()
        return t.lens.numpy(), t.status.numpy()

    end, history = paged_rules.serve(step, lens, [25, 24, 40, 10])
    assert end[0] == 62
    for status in history[:-1]:
        assert list(status) == [1, 0, 0, 0, 0]
    assert int(t.n_free.numpy()[0]) + sum(pm.pages(int(m), ps) for m in end) == len(free)
