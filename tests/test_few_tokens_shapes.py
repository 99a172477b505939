"""Shapes of the few-token NVFP4 kernels' blocks (csrc/gplk_nvfp4_shape.cuh), for
every number of tokens, tiles and stages. Blocks of a cluster wait for one
another, and tcgen05.alloc waits without a limit for columns that are free and
adjacent. So no block may ever wait there: a block that an SM's shared memory
has room for must find its TMEM, whatever other blocks are resident."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent
CSRC = REPO / "gpu-power-lab_b200" / "csrc"
SM_SMEM, BLOCK_SMEM, RESERVED, TMEM = 228 * 1024, 227 * 1024, 1024, 512

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    exe = tmp_path_factory.mktemp("shapes") / "shapes"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wno-unused-function", f"-I{CSRC}", "-o", str(exe),
                    str(REPO / "tests/csrc/few_token_shapes.cpp")], check=True)
    return [line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()]


@pytest.fixture(scope="module")
def shapes(lines):
    names = ("kind", "planes", "tokens", "tiles", "stages", "tmem", "smem", "per_sm", "ring", "w", "b", "cols", "ring_used",
             "image", "nb")
    out = [dict(zip(names, [r[0], *map(int, r[1:])])) for r in lines if r[0] != "map"]
    assert {s["kind"] for s in out} == {"convert", "image", "gateup", "item"}
    return out


def test_blocks_take_halves_of_an_sm(shapes):
    """With TMEM taken in halves or whole, and at least that share of the
    shared memory, at most two halves or one whole are resident: a half is free
    at column 0 or 256 whenever the shared memory of one is. Smaller parts could
    leave free columns apart from one another (128 + 128 beside two blocks of
    128 have no room for 256), and would fit beside a GEMM that takes all 512
    columns but leaves shared memory."""
    for s in shapes:
        assert s["tmem"] in (TMEM // 2, TMEM), s
        assert s["smem"] <= BLOCK_SMEM, s
        assert (s["smem"] + RESERVED) * TMEM >= SM_SMEM * s["tmem"], s
        assert s["per_sm"] == TMEM // s["tmem"], s


def test_rings_and_columns_fit(shapes):
    for s in shapes:
        assert s["cols"] <= s["tmem"] and s["ring_used"] <= s["ring"] < s["smem"], s
        assert s["ring"] >= s["tiles"] * s["tokens"] * 128 * 4, s  # the slices' sums lie over it
        assert s["image"] % 16 == 0 and s["nb"] % 8 == 0 and s["nb"] <= 256, s
        assert s["w"] >= s["tiles"] and s["b"] >= 1, s
        if s["tiles"] == 2:  # pairs: a stage's slot is free once both its tiles' slots are
            assert 2 * s["b"] >= s["w"], s


def test_boxes_of_a_matrix_stay_in_it(lines):
    """An expert's weights are read to their end and no other expert's are:
    those may be on their way in or out of memory while a layer runs."""
    maps = [tuple(map(int, r[1:])) for r in lines if r[0] == "map"]
    assert len(maps) == 15
    for rows, matrices, k, outside, covered in maps:
        assert outside == 0, (rows, k, outside)
        assert covered == matrices * rows * k // 2
