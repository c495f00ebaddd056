"""The experts' tiles wait by count for the loads that go straight to LDS (csrc/moe_ffn.hip, loads_barrier): on every path
through the compiled kernels those loads are complete where a barrier lets their readers go on."""

from __future__ import annotations

import re
import shlex
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "qt_llama.cpp_amd" / "csrc"
DONE = 99  # more than a wait can leave out


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """name -> lines, of the unit's tile kernels as the Makefile builds them."""
    out = tmp_path_factory.mktemp("asm") / "moe_ffn.s"
    lines = subprocess.run(["make", "-n", "-B", "--no-print-directory", "../_build/moe_ffn.o"], cwd=CSRC, check=True,
                           capture_output=True, text=True).stdout.replace("\\\n", " ").splitlines()
    cmd = shlex.split(next(line for line in lines if "moe_ffn.hip" in line))
    at = cmd.index("-c")
    subprocess.run([*cmd[:at], "--cuda-device-only", "-S", cmd[at + 1], "-o", str(out)], cwd=CSRC, check=True)
    found, name = {}, None
    for line in out.read_text().splitlines():
        m = re.match(r"(_Z\w*moe_tile_kernel\w*):", line)
        if m:
            name = m.group(1)
            found[name] = []
        elif line.startswith(".Lfunc_end"):
            name = None
        elif name:
            found[name].append(line.split(";")[0].strip())
    return found


def behind_lds_loads(lines):
    """Before each line the fewest loads that any path issued behind its last load to LDS; DONE where each such load has
    been waited for on every path."""
    lines = [line for line in lines if line]
    label = {line[:-1]: i for i, line in enumerate(lines) if line.endswith(":")}
    state, todo = {0: DONE}, [0]
    while todo:
        i = todo.pop()
        n, line = state[i], lines[i]
        op = line.split()[0]
        if op.startswith("global_load_lds"):
            n = 0
        elif re.match(r"(global|flat|buffer|scratch)_(load|store|atomic)", op):
            n = min(n + 1, DONE) if n < DONE else n
        elif op == "s_waitcnt":
            m = re.search(r"vmcnt\((\d+)\)", line)
            # a wait that leaves no more than were issued behind the loads to LDS has waited for those
            if m and int(m.group(1)) <= n:
                n = DONE
        target = line.split()[-1] if op.startswith(("s_cbranch", "s_branch")) else None
        to = [label[target]] if target else []
        if op not in ("s_branch", "s_endpgm"):
            to.append(i + 1)
        for j in to:
            if j < len(lines) and n < state.get(j, DONE + 1):
                state[j] = n
                todo.append(j)
    return lines, state


def test_the_walk_itself():
    """A load that a branch may leave out does not count towards a wait."""
    def at_barrier(text):
        lines, state = behind_lds_loads(text.replace("|", "\n").split("\n"))
        return [state[i] for i, line in enumerate(lines) if line == "s_barrier"]

    load, lds = "global_load_dword v0, v1, s[0:1]", "global_load_lds_dwordx4 v[0:1], off"
    assert at_barrier(f"{lds}|{load}|{load}|s_waitcnt vmcnt(2)|s_barrier|s_endpgm") == [DONE]
    assert at_barrier(f"{lds}|{load}|s_waitcnt vmcnt(2)|s_barrier|s_endpgm") == [1]
    assert at_barrier(f"{lds}|{load}|s_cbranch_scc1 a|{load}|a:|s_waitcnt vmcnt(2)|s_barrier|s_endpgm") == [1]
    assert at_barrier(f"{lds}|s_cbranch_scc1 a|{load}|a:|{load}|{load}|s_waitcnt vmcnt(2)|s_barrier|s_endpgm") == [DONE]


def test_loads_to_lds_are_waited_for(kernels):
    assert len(kernels) == 6, sorted(kernels)  # gate and up, down; scales of a row by four, by two, by one
    for name, code in kernels.items():
        lines, state = behind_lds_loads(code)
        assert sum(line.startswith("global_load_lds") for line in lines) >= 6 * 3, name
        early = [i for i, line in enumerate(lines) if line == "s_barrier" and state.get(i, DONE) < DONE]
        assert not early, f"{name}: {len(early)} barriers before a load to LDS is complete, the first with " \
                          f"{state[early[0]]} loads behind it: {lines[early[0] - 1]}"
