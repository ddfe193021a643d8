"""The hand-placed matrix instructions of the 4-bit product as the compiler emits them: the wait
states its hazard checks do not see, no accumulator moves, no scratch access (see
tests/check_mx_loops.py).  Needs hipcc but no GPU; about a minute."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT


def test_compiler_leaves_the_hand_placed_instructions_alone():
    from fastmoe_amd import build as lib_build

    if not os.path.exists(lib_build.HIPCC):
        pytest.skip("no hipcc on this machine")
    res = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "check_mx_loops.py")],
                         capture_output=True, text=True, timeout=900)
    assert res.returncode == 0, (res.stdout + res.stderr)[-3000:]
    assert " 0 flagged" in res.stdout
