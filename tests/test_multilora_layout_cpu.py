"""Where the projection's kernels read their operands (csrc/multilora_layout.h), compiled for the host: no
piece that they read without a guard reaches past the numbers that are there."""

import os
import shutil
import subprocess

import pytest

from tests.conftest import ROOT

SRC = r"""
#include <cstdio>
#include <initializer_list>
#include "multilora_layout.h"
using namespace bsml;
// The thin kernels read a row of ranks of the transposed operand in pieces of 8 numbers (from rank
// 8 i on) or of 2 (up to the last pair of the row's stride), wherever the stride covers them.
int main() {
    int checked = 0, bad = 0;
    for (int at : {4096, 4098, 4104})
        for (long long rows : {1ll, 2ll, 3ll, 7ll, 64ll})
            for (int rank = 1; rank <= 128; ++rank)
                for (bool f32 : {false, true}) {
                    const Operand o = operand((const void*)(size_t)at, rank, rows, rank, f32, true);
                    const long long there = o.moved ? rows * o.ld : rows * rank;
                    const long long pieces = (rank + 7) / 8 * 8;
                    if (o.moved && (o.ld < pieces || o.bytes < o.planes * o.rows * o.ld * 2)) ++bad;
                    if (o.ld >= pieces && (rows - 1) * o.ld + pieces > there) ++bad;
                    if ((rows - 1) * o.ld + o.ld > there) ++bad;
                    if (!o.moved && (o.ld % 8 != 0 || at % 16 != 0)) ++bad;
                    ++checked;
                }
    // operands behind guards stay where they are: one row of any length, on 16 bytes
    for (int cols = 1; cols < 100; ++cols) bad += operand((const void*)4096, cols, 1, cols, false, false).moved;
    std::printf("%d checked, %d bad\n", checked, bad);
    return bad != 0;
}
"""


def test_no_piece_reaches_past_an_operand(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "layout.cpp", tmp_path / "layout"
    src.write_text(SRC)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "brosoundml_b200", "csrc"),
                    str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.endswith(" checked, 0 bad\n"), out.stdout
