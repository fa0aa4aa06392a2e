"""Properties of the serving kernels' generated gfx950 code that no result test can pin reliably (CPU
only: hipcc cross-compiles the device code to assembly).

- The prefill kernel waits for a step's keys and values by the count of loads that every wave issues
  a step, so between two barriers of its pipeline each wave must issue exactly that many, whatever
  the step's page.
- No serving kernel spills registers to memory, and none holds a packed 32-bit float form.
"""
from __future__ import annotations

import re

import pytest

from test_codegen import _device_asm, _functions

UNITS = ("kv_append.hip", "kv_attention.hip", "pages.hip", "logprobs.hip")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    return {u: _device_asm(u, tmp_path_factory.mktemp("asm")) for u in UNITS}


def test_prefill_steps_issue_their_loads(asm):
    found = 0
    for name, body in _functions(asm["kv_attention.hip"], r"_ZN12_GLOBAL__N_121bsg_kv_prefill_kernel"):
        loads = 2 * int(re.search(r"Li(\d+)E", name).group(1)) // 64
        at = [i for i, line in enumerate(body) if line.strip().startswith("s_barrier")]
        steps = [body[a:b] for a, b in zip(at, at[1:]) if any("mfma" in line for line in body[a:b])]
        assert len(steps) == 3, (name, len(steps))
        for step in steps:
            assert sum(line.rstrip().endswith(" lds") or " lds" in line for line in step) == loads, name
        # none of the loads lies behind a branch of its own: they come in one run of instructions
        for step in steps:
            lines = [i for i, line in enumerate(step) if " lds" in line]
            between = step[lines[0]:lines[-1]]
            assert not any(re.match(r"\s*(s_cbranch|\.LBB)", line) for line in between), name
        found += 1
    assert found == 4  # two types x two head sizes


def test_no_spills_and_no_packed_floats(asm):
    for unit, text in asm.items():
        assert not re.search(r"\bscratch_(load|store)", text), unit
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32", text), unit
