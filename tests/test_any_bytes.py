"""csrc/any_bytes.h compiled for the host with the optimiser on: stores and loads of different widths keep their
order."""

from __future__ import annotations

import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def test_words_of_other_types(tmp_path):
    exe = tmp_path / "any_bytes_check"
    subprocess.run(["g++", "-O3", "-std=c++17", "-o", str(exe), str(ROOT / "tests/native/any_bytes_check.cpp")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_quantised_tiles_use_them():
    """attn_paged.hip reads and writes its LDS tiles through those types alone: no pointer to a plain 16 or 32 bit
    word, or to _Float16, is formed where the tiles are used."""
    s = (ROOT / "qt_llama.cpp_amd/csrc/attn_paged.hip").read_text()
    tiles = s[s.index("struct QuantTile {"):s.index("// ---- block items")]
    for plain in ("uint16_t *>", "uint32_t *>", "_Float16 *>", "))) uint32_t *", "))) uint16_t *"):
        at = [line for line in tiles.splitlines() if plain in line]
        assert not at, at
