"""What a block that gives up waits for before it leaves: the last copy into each buffer of its ring.  The count behind it runs
on the host too; here it is held against walks that write down every fill."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include <cstdio>
#include "umma.cuh"
// The layer norm's walk: all buffers at first, then from its second batch on the buffer before the current one; the last batch may be
// short and is no fill.  It breaks after `until` batches.
int main()
{
    int bad = 0, walks = 0;
    for (int depth = 2; depth <= 4; ++depth)
        for (int batches = 1; batches <= 14; ++batches)
            for (int tail = 0; tail < 2; ++tail)
                for (int until = 1; until <= batches; ++until, ++walks) {
                    const int full = batches - tail;
                    unsigned fills[4] = {}, used = 0;
                    const auto fill = [&](int s, int batch) {
                        if (batch < full) ++fills[s], ++used;
                    };
                    for (int s = 0; s < depth && s < batches; ++s) fill(s, s);
                    for (int b = 0, s = 0; b < until; ++b, s = s + 1 == depth ? 0 : s + 1) {
                        if (b + 1 == until) break;  // gives up here
                        const int next = b + depth - 1;
                        if (b != 0 && next < batches) fill(s == 0 ? depth - 1 : s - 1, next);
                    }
                    for (int s = 0; s < depth; ++s) bad += sgnn::ring_fills(used, s, depth) != fills[s];
                }
    // a plain ring, any number of fills
    for (unsigned buffers = 1; buffers <= 6; ++buffers) {
        unsigned fills[6] = {};
        for (unsigned used = 0; used < 40; ++used) {
            for (unsigned s = 0; s < buffers; ++s) bad += sgnn::ring_fills(used, s, buffers) != fills[s];
            ++fills[used % buffers];
        }
    }
    std::printf("%d walks, %d wrong\n", walks, bad);
    return bad != 0;
}
"""


def test_fills_of_the_buffers_of_a_ring(tmp_path):
    nvcc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    nvcc = nvcc if os.path.exists(nvcc) else shutil.which("nvcc")
    if not nvcc:
        pytest.skip("no nvcc")
    src, exe = tmp_path / "ring.cu", tmp_path / "ring"
    src.write_text(SOURCE)
    subprocess.check_call([nvcc, "-std=c++17", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a",
                           "-I", os.path.join(ROOT, "super_gnn_b200", "csrc"), "-I", os.path.join(ROOT, "include"),
                           str(src), "-o", str(exe)])
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout + done.stderr
