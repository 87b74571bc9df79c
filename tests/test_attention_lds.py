"""What an attention block asks for of a compute unit's 160 KB of LDS is checked
when the kernels are compiled (csrc/attention_plan.hpp)."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import PKG_DIR

PROGRAM = """
#include "attention_plan.hpp"
int main() { return mhc::att_fits<%s>() > 0 ? 0 : 1; }
"""


@pytest.fixture(scope="module")
def compiles(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("lds")

    def run(bytes_):
        (d / "a.cpp").write_text(PROGRAM % bytes_)
        p = subprocess.run([cxx, "-std=c++17", "-fsyntax-only", "-I", os.path.join(PKG_DIR, "csrc"), str(d / "a.cpp")],
                           capture_output=True, text=True)
        assert p.returncode == 0 or "exceeds a compute unit's" in p.stderr, p.stderr
        return p.returncode == 0

    return run


# es, blocks of 32 columns, waves, rows a stage, own rows of v: the widest of each type, and the 256 keys of heads of 128
@pytest.mark.parametrize("args,size", [("2, 8, 4, 32, true", 131584), ("2, 4, 8, 32, true", 98816), ("4, 4, 4, 32, true", 131584),
                                       ("2, 2, 4, 64, false", 33792)])
def test_what_runs_fits(compiles, args, size):
    assert compiles(f"mhc::att_dkv_lds({args})")
    assert compiles(f"mhc::att_dkv_lds({args}) == {size} ? 1 : mhc::kCuLds")


def test_what_does_not_fit_is_not_compiled(compiles):
    # fp32 heads of 256 columns, which are refused: 262656 bytes
    assert not compiles("mhc::att_dkv_lds(4, 8, 4, 32, true)")
    assert compiles("mhc::att_dkv_lds(4, 8, 4, 32, true) == 262656 ? 1 : mhc::kCuLds")
    assert compiles("mhc::kCuLds - mhc::kOwnLds") and not compiles("mhc::kCuLds - mhc::kOwnLds + 1")

