"""How the lanes of a warp share a row of the normed rotary positions, for every head size, turned part, type and order of
pairs: the host's plan, compiled by itself.  A row lies within one warp, or the kernel would never get to the next."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r"""
#include "normed_plan.cuh"
#include <cstdio>
int main() {
    for (int bytes = 2; bytes <= 4; bytes += 2)
        for (int D = 2; D <= 256; ++D)
            for (int half = 1; 2 * half <= D; ++half)
                for (int interleaved = 0; interleaved < 2; ++interleaved)
                    for (int whole = 0; whole < (D % (16 / bytes) == 0 ? 2 : 1); ++whole) {
                        const rfdetr::NormPlan p = rfdetr::plan_normed(bytes, D, half, interleaved, whole);
                        std::printf("%d %d %d %d %d %d %d %d %d %d\n", bytes, D, half, interleaved, whole, p.mode, p.vec,
                                    p.pieces, p.each, p.lanes);
                    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("needs g++")
    folder = tmp_path_factory.mktemp("plan")
    source, program = folder / "plan.cc", folder / "plan"
    source.write_text(PROGRAM)
    made = subprocess.run([compiler, "-std=c++17", "-o", str(program), str(source),
                           f"-I{os.path.join(ROOT, 'rf-detr-jax_b200', 'csrc')}"], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    out = subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout
    return [tuple(map(int, line.split())) for line in out.splitlines()]


def test_a_row_lies_within_a_warp(plans):
    assert len(plans) > 50_000
    assert [p for p in plans if not 1 <= p[9] <= 32] == []


def test_pieces_hold_every_channel(plans):
    """Paired pieces are two vectors where they turn and one behind; lanes hold all of a row's pieces."""
    for plan in plans:
        bytes_, dim, half, interleaved, whole, mode, vec, pieces, each, lanes = plan
        vectors = pieces + (half // vec if mode == 0 else 0)
        assert vectors * vec == dim and lanes * each >= pieces > (lanes - 1) * each, plan
        assert vec == (16 // bytes_ if whole else 1) and (mode == 0) == (whole and not interleaved and half % vec == 0), plan


def test_float32_rows_that_turn_in_part_take_two_pieces_a_lane(plans):
    """Those that one piece to a lane would spread over more than a warp; no others change."""
    wide = [p for p in plans if p[5] == 0 and p[7] > 32]
    assert wide and all(p[0] == 4 and p[8] == 2 and p[1] - p[2] > 128 for p in wide)
    assert all(p[8] == 1 for p in plans if p[5] == 0 and p[7] <= 32)
