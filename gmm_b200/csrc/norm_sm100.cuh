// norm_sm100.cuh -- the norms around a block, fused with its gate, its residual
// scale and the next block's norm, forward and backward.  No reference
// counterpart (the reference stops at the grouped GEMM).
//
// For each row, with r(z) = (mean(z^2) + eps)^-1/2 and o the weight offset:
//   n  = (w + o) * y * r(y)            post-norm of the block's output y
//   x' = x + s * act(g) * n            gate g, residual scale s
//   h  = (v + o) * x' * r(x')          pre-norm of the next block (optional)
// Without y the kernel is the pre-norm alone (x' = x).  The gate is one value
// a channel, one a token, or one an element; act is none, tanh or sigmoid.
//
// Backward, from dx' and dh (either may be absent):
//   u  = dh * (v + o)
//   dx = dx' + r(x') (u - xh mean(u xh)),      xh = x' r(x')
//   t  = s act(g) dx (w + o)
//   dy = r(y) (t - yh mean(t yh)),             yh = y r(y)
//   dw = sum_rows s act(g) dx yh,  dv = sum_rows dh xh,  dg = s act'(g) n dx
// x' is computed again from y and x in fp32 (the same bytes as reading it
// back, and without its rounding).  mean(t yh) needs dx, which needs
// mean(u xh); it is linear in it, so four sums of one pass give both.  With
// Q = s act(g) (w + o) y:
//   C = sum u x',  A1 = sum Q dx',  A2 = sum Q u,  B = sum Q x'
//   c = r(x')^2 C / D,   sum t yh = r(y) (A1 + r(x') A2 - c r(x') B).
// Without dh: dx = dx', sum t yh = r(y) A1, and x is not read.
// Everything is held in fp32 and rounded once, on store.  Rows are walked by
// blocks in a fixed order and parameter gradients added up per block, then
// over blocks in order, so results do not change from run to run.
//
// Bound by HBM: a row is read once and written once.  The kernels stream
// rows into shared memory with bulk copies (no registers and no threads held
// by loads in flight), several rows ahead of the two block-wide sums a row
// waits for; parameters stay in registers over all rows of a block.  Next to
// HBM comes the issue rate: two neighbouring elements share an instruction
// (f32x2), and the sums of a row take half the shuffles of separate ones.

#pragma once

#include <algorithm>
#include <cstdio>
#include <type_traits>

#include "gmm_sm100.h"
#include "row_ring.cuh"
#include "row_vec.cuh"
#include "status.h"

namespace gmm_sm100 {
namespace {

constexpr int kMaxNormDim = 16384;
constexpr int kBwdThreadsSm = 512;  // backward: threads of all blocks of an SM, 128 registers each (and of a block, at most)
constexpr int kFwdThreadsSm = 768;  // forward with 16 elements a thread: 80 registers each

enum GateMode { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };

struct NormParams {
  const void* y;      // block output (null: pre-norm only)
  const void* x;      // residual
  const void* w;      // post-norm weight [D]
  const void* v;      // next pre-norm weight [D] (null: no h)
  const void* gate;
  const void* dxn;    // backward: gradient of x' (may be null)
  const void* dh;     // backward: gradient of h (may be null)
  void* xn;           // x' (null when y is)
  void* h;
  void* dy;
  void* dx;
  void* dgate_row;    // token / full gate gradient
  float* rstd_y;      // [rows], null: not kept
  float* rstd_x;
  float* partial;     // backward: [2][blocks][D], the blocks' sums of act(g) dx yh (1 for a channel gate) and dh xh
  float4* sums;       // backward in column windows: [windows][rows], a window's C, A1, A2, B
  long long rows;
  int dim;
  int pitch;          // elements from a row to the next (= dim but in column windows)
  int windows, window;
  int phase;          // in column windows: 1 the sums, 2 the gradients
  int w_f32, gate_f32;  // parameters in fp32 (else the rows' type)
  int gate_mode, act;
  float scale, eps, offset;
};

// g[j] = act(g[j]) and, with kSlope, slope[j] = act'(g[j]); one branch for all
// N, so that their exponentials overlap.  With e = exp(-|g|), r = 1 / (1 + e):
//   sigmoid  r or e r by the sign of g, slope e r^2  (kFast without kSlope: from exp(-g) alone)
//   tanh     slope 4 e r^2 with e = exp(-2 |g|)
// Slopes from a (1 - a) or 1 - a^2 would lose a saturated gate's to the
// rounding of a.
//
// kFast: a 16-bit gate per element beside 16-bit rows.  There exponential and
// reciprocal are the fast ones, within 2 + 1.173 |x| and 2 ulp (an ulp is up to
// 2^-23 of a value): the sigmoid (10 + 2.35 |g|) * 2^-24 and the slopes, twice
// the reciprocal and twice the argument for tanh, below (20 + 4.7 |g|) * 2^-24,
// less than a half step of 16 bits (results below 2^-126 may be 0).  expf
// and a division made such a gate cost more than its rows' bytes (8191 x 6144
// fp16 forward: 111 us against 70); fp32 rows have twice the
// bytes to hide them, and gates shared by rows or elements are few.
template <bool kFast, bool kSlope, int N>
__device__ __forceinline__ void act_of(float* g, int act, float* slope = nullptr) {
  // e = exp(x) and 1 / (1 + e); kFast for any x, else for x <= 0: 1 + e is in
  // [1, 2] then, and one step of Newton and Raphson on the fast reciprocal leaves
  // its last rounding, without the division's path for numbers out of range.
  auto ratio = [](float x, float& e) {
    e = kFast ? __expf(x) : expf(x);
    const float d = 1.f + e, r = __fdividef(1.f, d);
    return kFast ? r : fmaf(r, fmaf(-d, r, 1.f), r);
  };
  if (act == GMM_GATE_TANH) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (kSlope) {
        float e;
        const float r = ratio(-2.f * fabsf(g[j]), e);
        slope[j] = 4.f * (e * r) * r;
      }
      g[j] = tanhf(g[j]);
    }
  } else if (act == GMM_GATE_SIGMOID) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float e;
      if constexpr (kFast && !kSlope) {
        g[j] = ratio(-g[j], e);
      } else {
        const float r = ratio(-fabsf(g[j]), e), er = e * r;
        if constexpr (kSlope) slope[j] = er * r;
        g[j] = g[j] >= 0.f ? r : er;
      }
    }
  } else if constexpr (kSlope) {
#pragma unroll
    for (int j = 0; j < N; ++j) slope[j] = 1.f;
  }
}

constexpr int kMaxWarps = 32;

// Sum over the block; every thread gets it.  `scratch` holds kMaxWarps floats,
// zero where there is no warp; two calls in a row need different scratch.
__device__ __forceinline__ float block_sum(float s, float* scratch) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (blockDim.x == 32) return s;
  const int lane = threadIdx.x & 31;
  if (lane == 0) scratch[threadIdx.x >> 5] = s;
  __syncthreads();
  s = scratch[lane & 7] + scratch[8 + (lane & 7)];
  if (blockDim.x > 16 * 32) s += scratch[16 + (lane & 7)] + scratch[24 + (lane & 7)];
#pragma unroll
  for (int o = 4; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// Four sums over at most 16 warps.  Halves of a warp trade sums until each
// group of eight lanes works on one: 9 shuffles in a warp instead of 20.
// `scratch` holds 4 * 16 floats, zero where there is no warp.
__device__ __forceinline__ void block_sum4(float (&s)[4], float* scratch) {
  const int lane = threadIdx.x & 31;
  const bool up = lane & 16, odd = lane & 8;
  float a = up ? s[2] : s[0], b = up ? s[3] : s[1];
  a += __shfl_xor_sync(0xffffffffu, up ? s[0] : s[2], 16);
  b += __shfl_xor_sync(0xffffffffu, up ? s[1] : s[3], 16);
  float t = odd ? b : a;
  t += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
  for (int o = 4; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (blockDim.x > 32) {  // lanes 8 j .. 8 j + 7 hold sum j of the warp
    if ((lane & 7) == 0) scratch[(lane >> 3) * 16 + (threadIdx.x >> 5)] = t;
    __syncthreads();
    t = scratch[(lane >> 3) * 16 + (lane & 7)] + scratch[(lane >> 3) * 16 + 8 + (lane & 7)];
#pragma unroll
    for (int o = 4; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j] = __shfl_sync(0xffffffffu, t, 8 * j);
}

// A token gate's row, and act(g) of it (1 for the other gates).
template <typename T>
__device__ __forceinline__ float token_value(const NormParams& p, long long row) {
  return p.gate_f32 ? static_cast<const float*>(p.gate)[row] : as_float(static_cast<const T*>(p.gate)[row]);
}
template <typename T>
__device__ __forceinline__ float token_gate(const NormParams& p, long long row) {
  if (p.gate_mode != kGateToken) return 1.f;
  float g = token_value<T>(p, row);
  act_of<false, false, 1>(&g, p.act);
  return g;
}

// ------------------------------------------------------------------ ring kernels
// A thread owns kE elements of every row, in units of V neighbouring elements:
// the units threadIdx.x + i * blockDim.x.  Three layouts:
//   kWhole    V is 16 bytes and rows are whole words;
//   kShifted  V is 16 bytes and tensors start on a word but rows (dim not a
//             multiple of V) do not.  Units are the words of memory, so that
//             loads and stores stay whole; a row's first and last unit are
//             partly its neighbours' and masked.  A row starts `shift` elements
//             into its first unit; the grid is a multiple of the shift's
//             period, so a block's rows all have the same one and its
//             parameters and sums stay in registers;
//   kSingle   V is 1 (tensors off the 16-byte grid): neighbouring threads read
//             neighbouring elements.
// 16384 x 4001 bf16, channel gate, forward, and forward and backward: kSingle
// 160 and 600 us, kShifted 104 and 332; 4000 columns (kWhole) 88 and 231.
enum Layout { kWhole = 0, kShifted = 1, kSingle = 2 };
// no y | gate none, channel, token | gate per element of the rows' type | of fp32 beside 16-bit rows
enum RingMode { kPreNorm = 0, kSharedGate = 1, kFullGate = 2, kFullGateF32 = 3 };
__host__ __device__ constexpr bool is_full(int mode) { return mode >= kFullGate; }
template <typename T, int kMode>
using GateOf = typename std::conditional<kMode == kFullGateF32, float, T>::type;

template <typename T, int kLayout>
constexpr int kUnit = kLayout == kSingle ? 1 : 16 / static_cast<int>(sizeof(T));

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& r, float* f) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = unpack2(w[i], static_cast<const T*>(nullptr));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  } else {
    f[0] = __uint_as_float(r.x);
    f[1] = __uint_as_float(r.y);
    f[2] = __uint_as_float(r.z);
    f[3] = __uint_as_float(r.w);
  }
}

// Unit c of a row of T (shared or global memory), as it lies there and as fp32.
template <typename T, int V>
using RawUnit = typename std::conditional<V == 1, T, uint4>::type;

template <typename T, int V>
__device__ __forceinline__ void unpack_unit(const RawUnit<T, V>& r, float* f) {
  if constexpr (V == 1) f[0] = as_float(r);
  else unpack16<T>(r, f);
}

template <typename T, int V>
__device__ __forceinline__ void read_unit(const void* row, int c, float* f) {
  unpack_unit<T, V>(static_cast<const RawUnit<T, V>*>(row)[c], f);
}

// The same, 0 where the unit is past the row's end (`in` false), and through `mask`.
template <typename T, int V, typename Mask>
__device__ __forceinline__ void read_unit_or_0(const void* row, int c, bool in, const Mask& mask, float* f) {
  RawUnit<T, V> r = {};
  if (in) r = static_cast<const RawUnit<T, V>*>(row)[c];
  unpack_unit<T, V>(mask(r), f);
}

// Unit c (V elements) of a row of G: a gate's, or a parameter's.
template <typename G, int V>
__device__ __forceinline__ void read_param(const void* row, int c, float* f) {
  if constexpr (V == 1) {
    f[0] = as_float(static_cast<const G*>(row)[c]);
  } else {
    constexpr int kPer = 16 / static_cast<int>(sizeof(G));
#pragma unroll
    for (int q = 0; q < V / kPer; ++q) unpack16<G>(static_cast<const uint4*>(row)[c * (V / kPer) + q], f + kPer * q);
  }
}
template <typename T, int V>
__device__ __forceinline__ void read_param(const void* row, bool f32, int c, float* f) {
  if (f32 && sizeof(T) == 2) read_param<float, V>(row, c, f);
  else read_param<T, V>(row, c, f);
}

template <typename T, int V>
__device__ __forceinline__ void write_unit(T* row, int c, const float* f) {
  if constexpr (V == 1) {
    row[c] = from_float<T>(f[0]);
  } else if constexpr (sizeof(T) == 2) {
    const T* t = nullptr;
    reinterpret_cast<uint4*>(row)[c] = make_uint4(pack_pair(f[0], f[1], t), pack_pair(f[2], f[3], t),
                                                  pack_pair(f[4], f[5], t), pack_pair(f[6], f[7], t));
  } else {
    reinterpret_cast<float4*>(row)[c] = make_float4(f[0], f[1], f[2], f[3]);
  }
}

// Elements [col, col + V) of a row that lie in it.  A call, so that the other
// units' path stays free of it.
template <typename T>
__device__ __noinline__ void write_partial_raw(T* row, int col, int dim, uint4 raw) {
  constexpr int kN = 16 / static_cast<int>(sizeof(T));
  const T* f = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int j = 0; j < kN; ++j)
    if (col + j >= 0 && col + j < dim) row[col + j] = f[j];
}
template <typename T, int V>
__device__ __forceinline__ void write_partial(T* row, int col, int dim, const float* f) {
  if constexpr (V > 1) {
    uint4 raw;
    write_unit<T, V>(reinterpret_cast<T*>(&raw), 0, f);
    write_partial_raw<T>(row, col, dim, raw);
  }
}

// Which of the row's elements a unit holds.
template <int V, int kLayout>
struct Span {
  int dim, units, shift;
  __device__ __forceinline__ Span(int d, int pitch) : dim(d) {
    shift = kLayout == kShifted ? static_cast<int>(static_cast<long long>(blockIdx.x) * pitch % V) : 0;
    units = (shift + d + V - 1) / V;
  }
  __device__ __forceinline__ bool partial(int c) const { return kLayout == kShifted && (c == 0 || c == units - 1); }
  __device__ __forceinline__ int col(int c, int j) const { return c * V + j - shift; }
  __device__ __forceinline__ bool has(int c, int j) const { return col(c, j) >= 0 && col(c, j) < dim; }
  // A partial unit's elements that are not the row's become 0.
  __device__ __forceinline__ void mask(int c, float* f) const {
    if (partial(c))
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = has(c, j) ? f[j] : 0.f;
  }
  // The same unit of a row in global memory: rows of one block start at the same place in a word.
  template <typename T>
  __device__ __forceinline__ void write(T* row, int c, const float* f) const {
    if (partial(c)) write_partial<T, V>(row, col(c, 0), dim, f);
    else write_unit<T, V>(row - shift, c, f);
  }
};

// Bits of a unit that are the row's: all ones but in a shifted row's first and
// last unit, whose other elements are its neighbours' and read as 0.  (Masked
// after unpacking, element by element, a forward pass of 16384 x 4001 bf16
// took 126 us; cleared in the ring by the units' owners, 150 us.)
template <typename T, int V, int kLayout>
struct UnitMask {
  __device__ __forceinline__ void set(const Span<V, kLayout>&, int) {}
  __device__ __forceinline__ RawUnit<T, V> operator()(const RawUnit<T, V>& r) const { return r; }
};
template <typename T, int V>
struct UnitMask<T, V, kShifted> {
  uint32_t m[4];
  __device__ __forceinline__ void set(const Span<V, kShifted>& span, int c) {
    constexpr int kPer = 4 / static_cast<int>(sizeof(T));  // elements of a 32-bit word
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      m[w] = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (span.has(c, w * kPer + j)) m[w] |= (kPer == 1 ? 0xffffffffu : 0xffffu) << (16 * j);
    }
  }
  __device__ __forceinline__ uint4 operator()(const uint4& r) const {
    return make_uint4(r.x & m[0], r.y & m[1], r.z & m[2], r.w & m[3]);
  }
};

// s (w + o), times act(g) of a channel gate; v + o.  Zero past the row's end.
// All loads first: they come from DRAM, one latency for all of them.
template <typename T, int V, int kLayout, int kE, int kMode>
__device__ __forceinline__ void row_params(const NormParams& p, const Span<V, kLayout>& span, bool with_v,
                                           float (&pw)[kE], float (&vo)[kE]) {
  const bool channel = kMode == kSharedGate && p.gate_mode == kGateChannel;
  float g[kMode == kSharedGate ? kE : 1];
  auto load = [&](const void* row, int f32, int c, float* f) {
    if constexpr (kLayout == kShifted) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (span.has(c, j)) read_param<T, 1>(row, f32, span.col(c, j), f + j);
    } else {
      if (c < span.units) read_param<T, V>(row, f32, c, f);
    }
  };
#pragma unroll
  for (int j = 0; j < kE; ++j) pw[j] = vo[j] = 0.f;
#pragma unroll
  for (int i = 0; i < kE / V; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (kMode != kPreNorm) load(p.w, p.w_f32, c, pw + i * V);
    if (with_v) load(p.v, p.w_f32, c, vo + i * V);
    if constexpr (kMode == kSharedGate) {
#pragma unroll
      for (int j = 0; j < V; ++j) g[i * V + j] = 0.f;
      if (channel) load(p.gate, p.gate_f32, c, g + i * V);
    }
  }
#pragma unroll
  for (int i = 0; i < kE / V; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool in = span.has(c, j);
      const int e = i * V + j;
      if (kMode != kPreNorm) {
        pw[e] = in ? (pw[e] + p.offset) * p.scale : 0.f;
        if constexpr (kMode == kSharedGate) {
          if (channel) {
            act_of<false, false, 1>(g + e, p.act);
            pw[e] *= g[e];
          }
        }
      }
      vo[e] = in && with_v ? vo[e] + p.offset : 0.f;
    }
  }
}

// ------------------------------------------------------------------ launches
constexpr int kMaxSlots = 8;

// Blocks of a ring kernel on one SM, and how many row slots each has.
struct RingShape {
  int threads, resident, slots, smem;
};
RingShape ring_shape(int dim, int per_thread, int max_threads_sm, size_t slot_bytes) {
  RingShape r;
  r.threads = threads_for((dim + per_thread - 1) / per_thread);
  r.resident = std::max(1, std::min(16, max_threads_sm / r.threads));
  const size_t share = kRingBytes / r.resident - 1024 - 1024;  // static scratch and the system's own part
  r.slots = static_cast<int>(std::min<size_t>(kMaxSlots, share / (slot_bytes + 8)));
  r.smem = r.slots * static_cast<int>(slot_bytes + 8);
  return r;
}

// The layout of a call's rows, the elements a row's units span, and the number
// of blocks after which rows start at the same place in a word again.
struct RowLayout {
  int layout, span, period;
};
RowLayout row_layout(int dim, int es, bool words) {
  const int v = 16 / es;
  if (!words) return {kSingle, dim, 1};
  if (dim % v == 0) return {kWhole, dim, 1};
  int period = v;
  for (int d = dim; d % 2 == 0; d /= 2) period /= 2;
  return {kShifted, dim + 2 * (v - 1), period};
}

// Blocks for `rows`: at most `most`, and with several rows a block a multiple of the period.
int blocks_for(int64_t rows, int64_t most, int period) {
  if (rows <= most) return static_cast<int>(rows);
  return static_cast<int>(std::max<int64_t>(period, most / period * period));
}

int mode_of(const NormParams& p, int es) {
  if (!p.y) return kPreNorm;
  if (p.gate_mode != GMM_GATE_MODE_FULL) return kSharedGate;
  return es == 2 && p.gate_f32 ? kFullGateF32 : kFullGate;
}

// Bytes of a slot behind an fp32 gate's row beside 16-bit rows off the word:
// the kernels read it in units of two words, the last of which may end one
// word past the row's last.
__host__ __device__ constexpr uint32_t gate_pad(int layout, int mode) {
  return layout == kShifted && mode == kFullGateF32 ? 16 : 0;
}

// Bytes of a slot that holds `inputs` rows of the data type and, with a gate
// per element, one of the gate's.
size_t slot_bytes(const NormParams& p, int es, int layout, int inputs) {
  const bool whole = layout == kWhole;
  const uint32_t gate = p.gate_mode == GMM_GATE_MODE_FULL ? p.dim * (p.gate_f32 ? 4 : es) : 0;
  return static_cast<size_t>(row_pitch(p.dim * es, whole)) * inputs + (gate ? row_pitch(gate, whole) : 0) +
         gate_pad(layout, mode_of(p, es));
}

bool on(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_common(int64_t rows, int64_t dim, int dtype, int weight_dtype, int gate_dtype, int gate_mode, int gate_act,
                 float eps) {
  if (rows < 0 || dim < 0) return set_error(GMM_ERR_INVALID_ARGUMENT, "negative size");
  if (dtype != GMM_DTYPE_F32 && dtype != GMM_DTYPE_BF16 && dtype != GMM_DTYPE_F16)
    return set_error(GMM_ERR_DTYPE, "rows must be fp32, bf16 or fp16");
  if ((weight_dtype != dtype && weight_dtype != GMM_DTYPE_F32) || (gate_dtype != dtype && gate_dtype != GMM_DTYPE_F32))
    return set_error(GMM_ERR_DTYPE, "weights and gate must have the rows' type or be fp32");
  if (gate_mode < GMM_GATE_MODE_NONE || gate_mode > GMM_GATE_MODE_FULL || gate_act < GMM_GATE_IDENTITY ||
      gate_act > GMM_GATE_SIGMOID)
    return set_error(GMM_ERR_INVALID_ARGUMENT, "unknown gate mode or gate activation");
  if (!(eps >= 0.f)) return set_error(GMM_ERR_INVALID_ARGUMENT, "eps must be >= 0");
  if (dim > kMaxNormDim || rows > INT32_MAX)
    return set_error(GMM_ERR_TOO_LARGE, "the norms take dim <= 16384 and fewer than 2^31 rows");
  return GMM_OK;
}

}  // namespace
}  // namespace gmm_sm100
