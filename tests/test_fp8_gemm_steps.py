"""CPU tests of the steps by which the FP8 product's warps wait for one another
(wohper_b200/csrc/mm_steps.cuh), compiled for the host: every order of the warps is run
through on a model of the barriers (tests/mm_steps.cpp), and an epilogue in which a wait
runs out on threads (tests/mm_tile.cpp)."""
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


def runner(source: str, folder):
    program = compiled(source, folder)

    def run(*args):
        return subprocess.run([str(program), *map(str, args)], check=True, capture_output=True, text=True, timeout=120).stdout.strip()

    return run


@pytest.fixture(scope="module")
def steps(tmp_path_factory):
    return runner("mm_steps.cpp", tmp_path_factory.mktemp("steps"))


@pytest.fixture(scope="module")
def tile(tmp_path_factory):
    return runner("mm_tile.cpp", tmp_path_factory.mktemp("tile"))


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


@pytest.mark.parametrize("agree,bad,warp,want", [
    ("kernel", 5, 0, "left after 5"),  # no wait runs out
    *(("kernel", bad, warp, f"left after {bad}") for bad in (0, 1, 4) for warp in range(4)),
    ("alone", 5, 0, "left after 5"), ("alone", 0, 0, "waits"), ("alone", 3, 2, "waits")])
def test_a_wait_that_runs_out_ends_the_epilogue(tile, agree, bad, warp, want):
    # four threads as the four warps of a column half, one of which gives up at tile `bad`
    assert tile(agree, bad, warp) == want
