"""The division of the shared-prefix decode's work (prefix.cuh), compiled for the host: no GPU needed."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG, ROOT

PROGRAM = r"""
#include <cstdio>
#include "prefix.cuh"
using namespace attn::prefix;
int main() {
    // a part that a call does not have (no own rows, or no prefixes): nothing set, and nothing to divide by
    const Part none = {};
    const Line nothing = {};
    for (int row = 0; row < 3; row++)
        for (int hk = 0; hk < 5; hk++)
            if (segment_begin(none, nothing, row, hk, 0) < 0) return 1;
    // 5 key heads in blocks of 2, blocks of 4 query rows, lines of 7 steps
    Part w = {};
    w.lines = 1; w.head_block = 2; w.n_blocks = 3; w.log_rows = 2;
    Line l = {};
    l.steps = 7;
    for (int row = 0; row < 12; row++)
        for (int hk = 0; hk < 5; hk++)
            if (segment_begin(w, l, row, hk, 100) != 100 + (row / 4 * 3 + hk / 2) * (7 + kBegin) + kBegin) return 2;
    puts("ok");
}
"""


def test_segment_begin(tmp_path):
    if shutil.which("nvcc") is None:
        pytest.skip("nvcc not present")
    (tmp_path / "t.cu").write_text(PROGRAM)
    build = subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr",
                            "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(PKG, "csrc"), "-o", "t", "t.cu", "-lcudart"],
                           cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stderr
    run = subprocess.run(["./t"], cwd=tmp_path, capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout == "ok\n", run.returncode
