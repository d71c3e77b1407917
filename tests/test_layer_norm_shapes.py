"""How wide rows of the layer norm's forward pass lie over a block's threads (layer_norm_shapes.hh), compiled for the host: every place of
a row belongs to one thread, and the quads that are loaded without a look lie in the row."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include "layer_norm_shapes.hh"
#include <cstdio>
#include <vector>
using namespace cb200;
int main() {
    for (int columns = kWarpColumns + 1; columns <= kRowColumns; ++columns) {
        const int threads = row_threads_of(columns), quads = row_quads_of(columns);
        bool right = threads % 32 == 0 && threads >= 32 && threads <= kRowThreads && row_fits(columns);
        // the places of the first and the last thread's quads, as the kernel has them
        for (int thread : {0, threads - 1})
            for (int i = 0; i + 1 < quads; ++i) right = right && (i * threads + thread) * 4 + 4 <= columns;
        std::vector<char> held((columns + 3) / 4, 0);
        for (int i = 0; i < quads; ++i)
            for (int thread = 0; thread < threads; ++thread)
                if (i * threads + thread < (int)held.size()) ++held[i * threads + thread];
        for (char h : held) right = right && h == 1;
        if (!right) { std::printf("%d\n", columns); return 1; }
    }
    // the check itself says no where it has to
    return rows_fit(kWarpColumns + 1, kRowColumns) && !rows_fit(1, kWarpColumns) && !row_fits(kRowColumns + 1) ? 0 : 2;
}
"""


def test_inner_quads_lie_in_the_row(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    source, binary = tmp_path / "shapes.cc", tmp_path / "shapes"
    source.write_text(PROGRAM)
    subprocess.run([cxx, "-O1", "-std=c++17", "-I", os.path.join(ROOT, "cellerator_b200", "csrc"), "-o", str(binary), str(source)], check=True)
    done = subprocess.run([str(binary)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
