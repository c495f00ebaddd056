"""What can be checked of the paged cache without a GPU: page arithmetic (the
kernels' own header compiled for the host), the refusals of a null context, and
the tests' own model of the step's bookkeeping."""

from __future__ import annotations

import subprocess
from pathlib import Path

import numpy as np
import pytest

import paged_model as pm

ROOT = Path(__file__).resolve().parents[1]


def test_page_arithmetic(tmp_path):
    exe = tmp_path / "page_map_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", str(exe), str(ROOT / "tests/native/page_map_check.cpp")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout


def test_null_context_is_refused(backend):
    lib = backend.load_library()
    p = [None] * 3
    assert lib.mrml_hip_block_tables(None, *p[:2], 1, None, 1, 16, None, None, 1, *p, None, None, 1, None, 0) == -1
    assert lib.mrml_hip_rope_kv_append_paged(None, *p, None, None, None, 1, 1, 16, 1, 1, 64, 1e4, 1.0, 0, 0, None, 0) == -1
    assert lib.mrml_hip_attention_paged(None, None, 64, *p, 1, 16, None, 0, None, 1, None, None, 1, 1, 1, 1, 64, 1.0, -1,
                                        0, 0) == -1


@pytest.mark.parametrize("page_size", [1, 4, 16])
def test_model_keeps_every_page_once(page_size):
    """Over random steps no page has two owners, none is lost, and refused requests stay as they were."""
    rng = np.random.default_rng(page_size)
    n, stride, n_pages = 12, 9, 40
    lens, n_free = np.zeros(n, np.int32), n_pages
    table, free = np.full((n, stride), -1, np.int32), rng.permutation(n_pages).astype(np.int32)
    for _ in range(300):
        want = rng.choice([-1, 0, 1, 1, 1, 7], n)
        got = pm.block_tables(lens, want, table, free, n_free, page_size, n_pages, 20, 0)
        for r in range(n):
            if got["status"][r]:
                assert got["lens"][r] == lens[r] and got["row_start"][r] == got["row_start"][r + 1]
        lens, n_free = got["lens"], got["n_free"]
        held = [int(table[r, j]) for r in range(n) for j in range(pm.pages(int(lens[r]), page_size))]
        assert sorted(held + [int(x) for x in free[:n_free]]) == list(range(n_pages))
