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
#include <cstdio>
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

QUANT = r"""
#include <cstdio>
#include "quant_sm100.cu"
using namespace gmm_sm100;
// Every width and type of the quantiser's ring asks for no more than a block may have, and its blocks for no more than
// an SM has (228 KB, with 1 KB of the system's and under 512 bytes of static scratch a block).
int main() {
  for (int es : {2, 4})
    for (bool vec : {false, true})
      for (int dim = 1; dim <= kMaxRingDim; ++dim) {
        if (vec && dim % 8) continue;
        const QuantShape r = quant_shape(dim, (dim + 15) / 16 * 16, es, vec);
        if (r.smem > kRingBlockBytes || r.slots < 2 || r.resident * (r.smem + 1024 + 512) > 228 * 1024)
          return std::printf("dim %d es %d vec %d: %d blocks of %d bytes\n", dim, es, vec, r.resident, r.smem), 1;
      }
  return 0;
}
"""

NORM = r"""
#include <cstdio>
#include "norm_sm100.cuh"
using namespace gmm_sm100;
// The same of the norms: rows of one to five inputs, the last an fp32 gate's where there is one.
int main() {
  for (int es : {2, 4})
    for (int dim = 1; dim <= kMaxNormDim; ++dim)
      for (bool words : {false, true})
        for (int inputs = 1; inputs <= 4; ++inputs)
          for (int gate = 0; gate <= 1; ++gate)
            for (bool backward : {false, true}) {
              const RowLayout l = row_layout(dim, es, words);
              if (l.span > (backward ? 8192 : kMaxNormDim) || (!backward && inputs > 2)) continue;
              NormParams p = {};
              p.y = &p;
              p.dim = dim;
              p.gate_mode = gate ? GMM_GATE_MODE_FULL : GMM_GATE_MODE_NONE;
              p.gate_f32 = gate;
              const int per = l.span <= 4096 && !backward ? 8 : 16;
              const int threads = backward ? kBwdThreadsSm : l.span <= 4096 ? 1024 : l.span <= 8192 ? kFwdThreadsSm : 1024;
              const RingShape r = ring_shape(l.span, per, threads, slot_bytes(p, es, l.layout, inputs));
              if (r.slots < 1 || r.smem > kRingBlockBytes || r.resident * (r.smem + 1024 + 1024) > 228 * 1024)
                return std::printf("dim %d es %d layout %d inputs %d: %d blocks of %d bytes\n", dim, es, l.layout, inputs,
                                   r.resident, r.smem), 1;
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


def test_the_quantisers_ring_fits_at_every_width(tmp_path):
    run(tmp_path, QUANT)


def test_the_norms_ring_fits_at_every_width(tmp_path):
    run(tmp_path, NORM)
