"""The context's scratch while captured graphs live: what is kept for them, and for how long."""

from __future__ import annotations

import gc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
MIB = 1 << 20


def used(dev):
    free, total = dev.memory_info()
    return total - free


def test_growing_scratch_beside_a_graph_stays_bounded(backend):
    """Scratch that grows in many small steps while a graph lives keeps less than its own size of outgrown scratch, and
    frees that when it grows after the last graph has gone; the graph replays throughout."""
    gc.collect()
    dev = backend.HipDevice.new(0)
    try:
        dev.reserve_workspace(64 * MIB)
        x = backend.HipBuffer.from_host(dev, np.arange(8, dtype=np.float32))
        y = backend.HipBuffer.alloc(dev, 8)
        graphs = [dev.capture(lambda: dev.add(x, x, y, 8)) for _ in range(2)]
        start = used(dev)
        for step in range(65, 201):  # 136 sizes, 18 GiB in all
            dev.reserve_workspace(step * MIB)
            assert dev.workspace_bytes() >= step * MIB
        kept = used(dev) + 64 * MIB - start
        assert kept <= 2 * dev.workspace_bytes() + 8 * MIB, kept / MIB
        graphs[0].close()
        size = dev.workspace_bytes()
        dev.reserve_workspace(size + 1)  # one graph is left: nothing is freed
        assert used(dev) + 64 * MIB - start >= size + dev.workspace_bytes()
        y.copy_from_host(np.zeros(8, np.float32))
        graphs[1].launch()
        dev.sync()
        assert np.array_equal(y.numpy(), 2 * np.arange(8, dtype=np.float32))
        graphs[1].close()
        last = dev.workspace_bytes() + MIB
        dev.reserve_workspace(last)
        assert dev.workspace_bytes() == last  # no graph: no more than asked for
        assert used(dev) + 64 * MIB - start <= last + 8 * MIB
        x.close(), y.close()
    finally:
        dev.close()
