"""Shared memory of the row kernels, width by width, from the host code that sizes it: compiled into a small program,
no GPU needed."""

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STUBS = r"""
namespace gmm_sm100 {
int set_error(int code, const char*) noexcept { return code; }
int current_sm_count(int* sms) { *sms = 148; return 0; }
}
"""

GATE = r"""
#include "norm_sm100.cuh"
using namespace gmm_sm100;
// The words an fp32 gate's row is read in beside 16-bit rows that start `shift` elements into their first unit of
// eight: from the word the row starts in to the end of the last unit.
int main() {
  for (int dim = 1; dim <= kMaxNormDim; ++dim) {
    const RowLayout l = row_layout(dim, 2, true);
    if (l.layout != kShifted) continue;
    NormParams p = {};
    p.y = &p;  // a post-norm
    p.dim = dim;
    p.gate_mode = GMM_GATE_MODE_FULL;
    p.gate_f32 = 1;
    const size_t room = slot_bytes(p, 2, kShifted, 2) - 2 * row_pitch(2 * dim, false);
    for (int b = 0; b < l.period; ++b) {
      const int shift = static_cast<long long>(b) * dim % 8, units = (shift + dim + 7) / 8;
      const size_t read = 32 * units - shift / 4 * 16;
      if (read > room) return std::printf("dim %d shift %d: reads %zu of %zu bytes\n", dim, shift, read, room), 1;
    }
  }
  return 0;
}
"""


def run(tmp_path, source):
    nvcc = "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    src, exe = str(tmp_path / "shapes.cu"), str(tmp_path / "shapes")
    with open(src, "w") as f:
        f.write(source + STUBS)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-w", "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "gmm_b200", "csrc"), "-o", exe, src], check=True)
    got = subprocess.run([exe], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout


def test_a_slot_holds_the_words_its_gate_is_read_in(tmp_path):
    run(tmp_path, GATE)
