"""The hand-placed matrix instructions of the 8-bit product as the compiler emits them, by the same
rules as the 4-bit ones (tests/check_mx_loops.py).  Needs hipcc but no GPU; about a minute."""
import importlib.util
import os
import re
import subprocess
import tempfile

import pytest

from conftest import ROOT


def _module(name, *path):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, *path))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_compiler_leaves_the_hand_placed_instructions_alone():
    build = _module("i8_build", "fastmoe_amd", "build.py")
    loops = _module("mx_loops", "tests", "check_mx_loops.py")
    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc on this machine")
    with tempfile.TemporaryDirectory() as tmp:
        out = os.path.join(tmp, "i8_gemm.s")
        flags = [f for f in build.FLAGS if f != "-fPIC"]
        subprocess.run([build.HIPCC, *flags, "-S", "--cuda-device-only",
                        os.path.join(build.CSRC, "i8_gemm.hip"), "-o", out],
                       check=True, capture_output=True)
        text = open(out).read()
    kernels = re.findall(r"^(_ZN4fmoe14i8_tile_kernel\S*):(.*?)^\.Lfunc_end", text, re.M | re.S)
    assert len(kernels) == 18          # 3 types, 3 tiles, packed rows and any
    assert sum(loops.check(name, body) for name, body in kernels) == 0
