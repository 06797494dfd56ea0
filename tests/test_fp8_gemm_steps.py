"""CPU tests of the steps by which the FP8 product's warps wait for one another
(wohper_b200/csrc/mm_steps.cuh), compiled for the host: every order of the warps is run
through on a model of the barriers (tests/mm_steps.cpp)."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def compiled(source: str, folder) -> Path:
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    out = folder / Path(source).stem
    subprocess.run([cxx, "-std=c++17", "-O2", "-pthread", "-o", str(out), str(HERE / source)], check=True)
    return out


@pytest.fixture(scope="module")
def steps(tmp_path_factory):
    program = compiled("mm_steps.cpp", tmp_path_factory.mktemp("steps"))

    def run(*args):
        return subprocess.run([str(program), *map(str, args)], check=True, capture_output=True, text=True, timeout=120).stdout.strip()

    return run


@pytest.mark.parametrize("fold", [8, 256])  # K tiles of a sum: f32 and 16-bit outputs
@pytest.mark.parametrize("tiles", [1, 4, 5, 8, 9, 10, 12, 13, 16, 17, 18, 24, 25, 26, 34])
def test_every_order_of_the_warps_ends(steps, tiles, fold):
    assert steps("kernel", tiles, fold) == "ok"


@pytest.mark.parametrize("tiles", [9, 17, 24])
def test_the_model_finds_waits_that_miss_their_phase(steps, tiles):
    # a barrier a stage: the phase of the fill before the last may be two back, that of the last may not have begun
    assert steps("both", tiles, 8) == "stuck"
    assert steps("last", tiles, 8) == "overwritten"
    assert steps("both", 8, 8) == steps("last", 8, 8) == "ok"
