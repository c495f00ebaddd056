"""What can be checked of the expert ops without a GPU: the refusals of a null context, and the tests' own model."""

from __future__ import annotations

from pathlib import Path

import numpy as np
import pytest

import moe_model as mm


def test_null_context_is_refused(backend):
    lib = backend.load_library()
    assert lib.mrml_hip_residual_rms_norm_batch(None, None, None, None, None, None, None, None, 32, 1, 1e-6, 1) == -1
    assert lib.mrml_hip_moe_logits(None, None, None, None, 4, 32, 1) == -1
    assert lib.mrml_hip_moe_route(None, None, None, None, None, None, None, 4, 1, 1, 0, 1, 1, 1, 1, 1.0) == -1
    for fn in (lib.mrml_hip_moe_gate_up_q4_0, lib.mrml_hip_moe_gate_up_q4_0_q8):
        assert fn(None, None, None, None, None, None, None, None, 4, 8, 32, 1, 1, 0) == -1
    assert lib.mrml_hip_moe_down_q4_0(None, None, None, None, None, None, None, None, 4, 8, 32, 1, 1) == -1


def test_lds_words_may_name_any_object():
    """moe_ffn.hip writes quants and scales to LDS in words of one width and reads them in another: through any_bytes.h's
    types, so that the compiler keeps their order.  Plain 16, 32 and 64 bit words are of global memory alone."""
    s = (Path(__file__).resolve().parents[1] / "qt_llama.cpp_amd/csrc/moe_ffn.hip").read_text()
    for line in s[s.index("// ---- few tokens an expert"):s.index("// y = the sum of a token's weighted")].splitlines():
        if any(plain in line for plain in ("uint16_t *", "uint32_t *", "long *", "int64_t *")):
            assert "*>(at(i))" in line or "*>(ws)" in line, line


def test_model_route_ties_and_masks():
    x = np.array([[1, 3, 3, -np.inf, 2, 3], [-np.inf] * 6, [np.nan, 0, np.inf, np.inf, 5, -1]], np.float32)
    ids, w = mm.route(x, None, 4, mm.SOFTMAX)
    assert ids.tolist() == [[1, 2, 5, 4], [-1] * 4, [2, 3, 4, 1]]
    assert np.allclose(w.sum(1), [1, 0, 1]) and w[2].tolist() == [0.5, 0.5, 0, 0]
    starts, order = mm.plan(ids, 6)
    assert starts.tolist() == [0, 0, 2, 4, 5, 7, 8] and order.tolist() == [0, 11, 1, 8, 9, 3, 10, 2] + [-1] * 4


def test_model_groups():
    x = np.array([[9, 0, 1, 2, 5, 5, -3, 4]], np.float32)
    assert mm.route(x, None, 3, mm.SIGMOID, 4, 2, 1)[0].tolist() == [[0, 4, 5]]
    # by the sum of two sigmoids (1.50, 1.61, 1.99, 1.03) the groups rank 2, 1, 0, 3
    assert mm.route(x, None, 4, mm.SIGMOID, 4, 2, 2)[0].tolist() == [[4, 5, 3, 2]]


@pytest.mark.parametrize("activation", [mm.GEGLU, mm.SWIGLU])
def test_model_products_against_f32(orc, synth, activation):
    """The bounds of the model hold for plain f32 sums of the same values."""
    rng = synth.rng_for(5)
    e, k, n, rows, cols = 3, 2, 4, 9, 96
    wg, wu = (mm.q4_0_values(synth.q4_0_matrix(rng, e * rows, cols), e * rows, cols).reshape(e, rows, cols) for _ in "gu")
    xq = mm.q8_0_values(orc, rng.standard_normal((n, cols)).astype(np.float32))
    ids = np.array([[0, 2], [1, -1], [2, 1], [0, 1]])
    act, bound = mm.gate_up(wg, wu, xq, ids, k, activation)
    assert np.isnan(act[3]).all()
    for a, i in enumerate(ids.reshape(-1)):
        if i >= 0:
            x = xq[a // k].astype(np.float32)
            g, u = (np.array([np.cumsum((w[i][r].astype(np.float32) * x), dtype=np.float32)[-1] for r in range(rows)])
                    for w in (wg, wu))
            assert (np.abs(mm.gated(g.astype(np.float64), u.astype(np.float64), activation) - act[a]) <= bound[a]).all()
