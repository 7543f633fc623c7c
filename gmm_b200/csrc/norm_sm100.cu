// norm_sm100.cu -- the norms around a block, fused with its gate, its residual
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
constexpr int kMaxThreads = 512;

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
  long long rows;
  int dim;
  int w_f32, gate_f32;  // parameters in fp32 (else the rows' type)
  int gate_mode, act;
  float scale, eps, offset;
};

__device__ __forceinline__ float act_of(float g, int act) {
  // The sigmoid's fast exponential is within (2 |g| + 4) * 2^-24 of e^-g and
  // its fast reciprocal within 2 * 2^-24; expf and a full division made a
  // gate per element cost more than its rows' bytes (8191 x 6144 fp16: 111 us).
  return act == GMM_GATE_TANH ? tanhf(g) : act == GMM_GATE_SIGMOID ? __fdividef(1.f, 1.f + __expf(-g)) : g;
}
// act'(g) from a = act(g)
__device__ __forceinline__ float act_slope(float a, int act) {
  return act == GMM_GATE_TANH ? 1.f - a * a : act == GMM_GATE_SIGMOID ? a * (1.f - a) : 1.f;
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

// act(g) of a token gate's row, 1 for the others.
template <typename T>
__device__ __forceinline__ float token_gate(const NormParams& p, long long row) {
  if (p.gate_mode != kGateToken) return 1.f;
  const float g = p.gate_f32 ? static_cast<const float*>(p.gate)[row] : as_float(static_cast<const T*>(p.gate)[row]);
  return act_of(g, p.act);
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
enum RingMode { kPreNorm = 0, kSharedGate = 1, kFullGate = 2 };  // no y | gate none, channel, token | gate per element

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

// Unit c of a parameter or gate row that is T or fp32.
template <typename T, int V>
__device__ __forceinline__ void read_param(const void* row, bool f32, int c, float* f) {
  if (f32 && sizeof(T) == 2) {
    if constexpr (V == 1) {
      f[0] = static_cast<const float*>(row)[c];
    } else {
#pragma unroll
      for (int q = 0; q < V / 4; ++q) unpack16<float>(static_cast<const uint4*>(row)[c * (V / 4) + q], f + 4 * q);
    }
  } else {
    read_unit<T, V>(row, c, f);
  }
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
  __device__ __forceinline__ Span(int d) : dim(d) {
    shift = kLayout == kShifted ? static_cast<int>(static_cast<long long>(blockIdx.x) * d % V) : 0;
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
        if (kMode == kSharedGate && channel) pw[e] *= act_of(g[e], p.act);
      }
      vo[e] = in && with_v ? vo[e] + p.offset : 0.f;
    }
  }
}

template <typename T, int kLayout, int kE, int kMode, int kThreads, int kBlocks>
__global__ void __launch_bounds__(kThreads, kBlocks) norm_fwd_ring_kernel(const NormParams p, int slots) {
  constexpr int V = kUnit<T, kLayout>, kUnits = kE / V;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float scratch[2][2][kMaxWarps];  // by sum and by parity of the row
  const int D = p.dim;
  RowRing<3, kLayout == kWhole> ring;
  ring.src[0] = static_cast<const char*>(p.x);
  ring.src[1] = static_cast<const char*>(p.y);
  ring.src[2] = static_cast<const char*>(p.gate);
  ring.bytes[0] = D * sizeof(T);
  ring.bytes[1] = kMode == kPreNorm ? 0 : D * sizeof(T);
  ring.bytes[2] = kMode == kFullGate ? D * (p.gate_f32 ? 4 : static_cast<int>(sizeof(T))) : 0;
  ring.start(smem, slots, p.rows);
  if (threadIdx.x < 32)
#pragma unroll
    for (int i = 0; i < 4; ++i) scratch[i >> 1][i & 1][threadIdx.x] = 0.f;

  const Span<V, kLayout> span(D);
  const int units = span.units;
  float pw[kE], vo[kE];
  row_params<T, V, kLayout, kE, kMode>(p, span, p.h != nullptr, pw, vo);
  auto input = [&](int i, int slot, long long row) {
    return smem + (kLayout == kShifted ? ring.word_at(slot, i) : ring.at(slot, i, row));
  };
  // An fp32 gate beside 16-bit rows: a unit is two words, and the row may start in the second.
  const bool wide_gate = kLayout == kShifted && kMode == kFullGate && sizeof(T) == 2 && p.gate_f32;
  const int gate_words = wide_gate ? span.shift / 4 * 16 : 0;
  UnitMask<T, V, kLayout> mask[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) mask[i].set(span, threadIdx.x + i * blockDim.x);
  __syncthreads();  // barriers initialised
  const float inv_d = 1.f / static_cast<float>(D);

  int slot = 0;
  uint32_t phase = 0;
  int odd = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float tok = kMode == kSharedGate ? token_gate<T>(p, row) : 1.f;
    ring.wait(slot, phase, row);
    const auto* xs = reinterpret_cast<const RawUnit<T, V>*>(input(0, slot, row));
    float x[kE];
    float sq[2] = {0.f, 0.f};
    if constexpr (kMode == kPreNorm) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        read_unit_or_0<T, V>(xs, c, c < units, mask[i], x + i * V);
      }
    } else {
      const auto* ys = input(1, slot, row);
      float y[kE];
      RawUnit<T, V> xr[kUnits];
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        read_unit_or_0<T, V>(ys, c, c < units, mask[i], y + i * V);
        xr[i] = RawUnit<T, V>{};
        if (c < units) xr[i] = mask[i](xs[c]);
      }
#pragma unroll
      for (int j = 0; j < kE; j += 2) fma2(sq, y + j, y + j, sq);
      if constexpr (kMode == kFullGate) {  // y * act(g): the gate is not needed again
        const auto* gs = input(2, slot, row) - gate_words;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int c = threadIdx.x + i * blockDim.x;
          float g[V];
#pragma unroll
          for (int j = 0; j < V; ++j) g[j] = 0.f;
          if (c < units) read_param<T, V>(gs, p.gate_f32, c, g);
          if (kLayout == kShifted) span.mask(c, g);
#pragma unroll
          for (int j = 0; j < V; ++j) y[i * V + j] *= act_of(g[j], p.act);
        }
      }
      const float ry = rsqrtf(block_sum(sq[0] + sq[1], scratch[0][odd]) * inv_d + p.eps);
      if (p.rstd_y && threadIdx.x == 0) p.rstd_y[row] = ry;
      const Both c0(ry * tok);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) unpack_unit<T, V>(xr[i], x + i * V);
#pragma unroll
      for (int j = 0; j < kE; j += 2) {
        mul2(y + j, y + j, c0);
        fma2(x + j, y + j, pw + j, x + j);
      }
      T* xn = static_cast<T*>(p.xn) + row * D;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        if (c < units) span.write(xn, c, x + i * V);
      }
    }
    if (p.h) {
      sq[0] = sq[1] = 0.f;
#pragma unroll
      for (int j = 0; j < kE; j += 2) fma2(sq, x + j, x + j, sq);
      const float rx = rsqrtf(block_sum(sq[0] + sq[1], scratch[1][odd]) * inv_d + p.eps);
      if (p.rstd_x && threadIdx.x == 0) p.rstd_x[row] = rx;
      const Both r2(rx);
#pragma unroll
      for (int j = 0; j < kE; j += 2) {
        mul2(x + j, x + j, r2);
        mul2(x + j, x + j, vo + j);
      }
      T* h = static_cast<T*>(p.h) + row * D;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        if (c < units) span.write(h, c, x + i * V);
      }
    }
    // Every thread has read the slot before the (first or only) sum's barrier.
    if (blockDim.x == 32) __syncwarp();
    if (threadIdx.x == 0 && !ring.dead) {
      const long long next = row + static_cast<long long>(slots) * gridDim.x;
      if (next < p.rows) ring.fetch(slot, next);
    }
    if (++slot == slots) {
      slot = 0;
      phase ^= 1;
    }
    odd ^= 1;  // the next row's sums use the other scratch: its barriers free this one
  }
}

// Backward.  The rows stay in the ring between the sums and the results
// (re-reading shared memory costs less than holding four rows in registers),
// so a slot is refilled one row later, past the next row's barrier -- or, with
// a single slot, behind a barrier of its own.
template <typename T, int kLayout, int kE, int kMode, int kThreads, int kBlocks>
__global__ void __launch_bounds__(kThreads, kBlocks) norm_bwd_ring_kernel(const NormParams p, int slots) {
  constexpr int V = kUnit<T, kLayout>;
  // A thread works on groups of kG elements: one unit, or two of one element.
  constexpr int kU = V == 1 ? 2 : 1, kG = V * kU, kGroups = kE / kG;
  static_assert(kThreads <= 16 * 32, "block_sum4");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float scratch[2][4 * 16];
  const int D = p.dim;
  RowRing<5, kLayout == kWhole> ring;
  ring.src[0] = static_cast<const char*>(p.x);
  ring.src[1] = static_cast<const char*>(p.y);
  ring.src[2] = static_cast<const char*>(p.dxn);
  ring.src[3] = static_cast<const char*>(p.dh);
  ring.src[4] = static_cast<const char*>(p.gate);
  ring.bytes[0] = D * sizeof(T);
  ring.bytes[1] = kMode == kPreNorm ? 0 : D * sizeof(T);
  ring.bytes[2] = p.dxn ? D * sizeof(T) : 0;
  ring.bytes[3] = p.dh ? D * sizeof(T) : 0;
  ring.bytes[4] = kMode == kFullGate ? D * (p.gate_f32 ? 4 : static_cast<int>(sizeof(T))) : 0;
  ring.start(smem, slots, p.rows);
  if (threadIdx.x < 32)
#pragma unroll
    for (int i = 0; i < 4; ++i) scratch[i >> 1][(i & 1) * 32 + threadIdx.x] = 0.f;

  const Span<V, kLayout> span(D);
  const int units = span.units;
  float pw[kE], vo[kE], acc[kE], dv[kE];
  row_params<T, V, kLayout, kE, kMode>(p, span, p.dh != nullptr, pw, vo);
  auto input = [&](int i, int slot, long long row) {
    return smem + (kLayout == kShifted ? ring.word_at(slot, i) : ring.at(slot, i, row));
  };
  // An fp32 gate beside 16-bit rows: a unit is two words, and the row may start in the second.
  const bool wide_gate = kLayout == kShifted && kMode == kFullGate && sizeof(T) == 2 && p.gate_f32;
  const int gate_words = wide_gate ? span.shift / 4 * 16 : 0;
  UnitMask<T, V, kLayout> mask[kE / V];
#pragma unroll
  for (int i = 0; i < kE / V; ++i) mask[i].set(span, threadIdx.x + i * blockDim.x);
#pragma unroll
  for (int j = 0; j < kE; ++j) acc[j] = dv[j] = 0.f;
  __syncthreads();  // barriers initialised
  const float inv_d = 1.f / static_cast<float>(D);

  int slot = 0;
  uint32_t phase = 0;
  int odd = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float ry = kMode == kPreNorm ? 0.f : p.rstd_y[row];
    const float rx = p.dh ? p.rstd_x[row] : 0.f;
    const float tok = kMode == kSharedGate ? token_gate<T>(p, row) : 1.f;
    ring.wait(slot, phase, row);
    const uint8_t *in_x = input(0, slot, row), *in_y = input(1, slot, row), *in_dx = input(2, slot, row),
                  *in_dh = input(3, slot, row), *in_g = input(4, slot, row) - gate_words;
    auto unit = [&](int g, int u) { return static_cast<int>(threadIdx.x + (g * kU + u) * blockDim.x); };
    const Both to_x(kMode == kFullGate ? ry : ry * tok);
    // Of a group's elements: y, Q (times act(g) with a gate per element, which
    // `a` returns), x', u = dh (v + o), dh.  Zeros past the row's end.
    auto read = [&](int g, float (&y)[kG], float (&q)[kG], float (&a)[kG], float (&x)[kG], float (&u)[kG],
                    float (&dh)[kG]) {
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        const int c = unit(g, k);
        const bool in = V > 1 || c < units;
        const auto& own = mask[g * kU + k];
        read_unit_or_0<T, V>(in_x, c, in, own, x + k * V);
        if constexpr (kMode != kPreNorm) read_unit_or_0<T, V>(in_y, c, in, own, y + k * V);
        if (p.dh) {
          read_unit_or_0<T, V>(in_dh, c, in, own, dh + k * V);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) dh[k * V + j] = 0.f;
        }
        if constexpr (kMode == kFullGate) {
#pragma unroll
          for (int j = 0; j < V; ++j) a[k * V + j] = 0.f;
          if (in) read_param<T, V>(in_g, p.gate_f32, c, a + k * V);
          if (kLayout == kShifted) span.mask(c, a + k * V);
#pragma unroll
          for (int j = 0; j < V; ++j) a[k * V + j] = act_of(a[k * V + j], p.act);
        }
      }
#pragma unroll
      for (int j = 0; j < kG; j += 2) {
        if constexpr (kMode != kPreNorm) {
          mul2(q + j, y + j, pw + g * kG + j);
          if constexpr (kMode == kFullGate) mul2(q + j, q + j, a + j);
          fma2(x + j, q + j, to_x, x + j);
        }
        mul2(u + j, dh + j, vo + g * kG + j);
      }
    };
    auto read_dx = [&](int g, float (&d)[kG]) {
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        const int c = unit(g, k);
        if (p.dxn) {
          read_unit_or_0<T, V>(in_dx, c, V > 1 || c < units, mask[g * kU + k], d + k * V);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) d[k * V + j] = 0.f;
        }
      }
    };
    float s2[4][2] = {};  // C, A1, A2, B: even and odd elements
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (V > 1 && unit(g, 0) >= units) continue;
      float y[kG], q[kG], a[kG], x[kG], u[kG], dh[kG], d[kG];
      read(g, y, q, a, x, u, dh);
      if constexpr (kMode != kPreNorm) read_dx(g, d);
#pragma unroll
      for (int j = 0; j < kG; j += 2) {
        fma2(s2[0], u + j, x + j, s2[0]);
        if constexpr (kMode != kPreNorm) {
          fma2(s2[1], q + j, d + j, s2[1]);
          fma2(s2[2], q + j, u + j, s2[2]);
          fma2(s2[3], q + j, x + j, s2[3]);
        }
      }
    }
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = s2[j][0] + s2[j][1];
    block_sum4(s, scratch[odd]);
    // Every thread is past the previous row's last read of its slot.
    if (threadIdx.x == 0 && slots > 1 && !ring.dead && row >= gridDim.x) {
      const long long next = row + static_cast<long long>(slots - 1) * gridDim.x;
      if (next < p.rows) ring.fetch(slot == 0 ? slots - 1 : slot - 1, next);
    }
    const float cx = rx * rx * (s[0] * inv_d) * rx;       // dx = dx' + r(x') u - cx x'
    const float qdx = ry * (s[1] + rx * s[2] - cx * s[3]);  // sum of s (w + o) yh [act(g)] dx
    const float m = qdx * inv_d * tok;                    // mean(t yh)
    if (kMode == kSharedGate && p.gate_mode == kGateToken && threadIdx.x == 0) {
      const float d = qdx * act_slope(tok, p.act);
      if (p.gate_f32) static_cast<float*>(p.dgate_row)[row] = d;
      else static_cast<T*>(p.dgate_row)[row] = from_float<T>(d);
    }
    const Both r2(rx), neg_cx(-cx), neg_m(-ry * ry * m), ry2(ry);
    T* dx_out = static_cast<T*>(p.dx) + row * D;
    T* dy_out = static_cast<T*>(p.dy) + row * D;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (V > 1 && unit(g, 0) >= units) continue;
      float y[kG], q[kG], a[kG], x[kG], u[kG], dh[kG], d[kG];
      read(g, y, q, a, x, u, dh);
      read_dx(g, d);
#pragma unroll
      for (int j = 0; j < kG; j += 2) {
        const int e = g * kG + j;
        fma2(d + j, u + j, r2, d + j);
        fma2(d + j, x + j, neg_cx, d + j);  // dx
        mul2(x + j, x + j, r2);
        fma2(dv + e, dh + j, x + j, dv + e);
      }
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        const int c = unit(g, k);
        if (V > 1 || c < units) span.write(dx_out, c, d + k * V);
      }
      if constexpr (kMode != kPreNorm) {
        float dg[kG];
#pragma unroll
        for (int j = 0; j < kG; j += 2) {
          const int e = g * kG + j;
          if constexpr (kMode == kFullGate) {
            float yh[2];
            mul2(yh, y + j, ry2);
#pragma unroll
            for (int i = 0; i < 2; ++i) dg[j + i] = pw[e + i] * yh[i] * d[j + i] * act_slope(a[j + i], p.act);
            mul2(d + j, d + j, a + j);
            fma2(acc + e, d + j, yh, acc + e);
            mul2(d + j, d + j, ry2);
          } else {
            mul2(d + j, d + j, to_x);
            fma2(acc + e, d + j, y + j, acc + e);
          }
          mul2(y + j, y + j, neg_m);
          fma2(y + j, d + j, pw + e, y + j);  // dy
        }
#pragma unroll
        for (int k = 0; k < kU; ++k) {
          const int c = unit(g, k);
          if (V == 1 && c >= units) continue;
          span.write(dy_out, c, y + k * V);
          if constexpr (kMode == kFullGate) {
            if (p.gate_f32 && sizeof(T) == 2) {
              float* out = static_cast<float*>(p.dgate_row) + row * D;
              if (V == 1 || span.partial(c)) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                  if (span.has(c, j)) out[span.col(c, j)] = dg[k * V + j];
              } else {
#pragma unroll
                for (int i = 0; i < V / 4; ++i)
                  write_unit<float, 4>(out - span.shift, c * (V / 4) + i, dg + 4 * i);
              }
            } else {
              span.write(static_cast<T*>(p.dgate_row) + row * D, c, dg + k * V);
            }
          }
        }
      }
    }
    if (slots == 1) {
      __syncthreads();
      const long long next = row + gridDim.x;
      if (threadIdx.x == 0 && !ring.dead && next < p.rows) ring.fetch(0, next);
    } else if (blockDim.x == 32) {
      __syncwarp();
    }
    if (++slot == slots) {
      slot = 0;
      phase ^= 1;
    }
    odd ^= 1;
  }
  float* part = p.partial + static_cast<long long>(blockIdx.x) * D;
  const long long slice = static_cast<long long>(gridDim.x) * D;
#pragma unroll
  for (int i = 0; i < kE / V; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (kLayout == kWhole && D % 4 == 0) {
      if (c >= units) continue;
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        if (kMode != kPreNorm) write_unit<float, 4>(part, c * (V / 4) + q, acc + i * V + 4 * q);
        if (p.dh) write_unit<float, 4>(part + slice, c * (V / 4) + q, dv + i * V + 4 * q);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (!span.has(c, j)) continue;
        if (kMode != kPreNorm) part[span.col(c, j)] = acc[i * V + j];
        if (p.dh) part[slice + span.col(c, j)] = dv[i * V + j];
      }
    }
  }
}

// ------------------------------------------------------------------ wide rows
template <typename T>
__device__ __forceinline__ float param1(const void* p, int f32, long long at) {
  return f32 ? __ldg(static_cast<const float*>(p) + at) : as_float(static_cast<const T*>(p)[at]);
}

template <typename T>
__device__ __forceinline__ float gate1(const NormParams& p, long long row, int col, float tok) {
  if (p.gate_mode != kGateChannel && p.gate_mode != kGateFull) return tok;
  return act_of(param1<T>(p.gate, p.gate_f32, p.gate_mode == kGateFull ? row * p.dim + col : col), p.act);
}

// Backward of rows wider than the ring's registers hold (dim > 8192): a thread
// owns elements threadIdx.x + i * blockDim.x, read from global memory.
template <typename T, int kE>
__global__ void __launch_bounds__(kMaxThreads) norm_bwd_kernel(const NormParams p) {
  __shared__ float scratch[4 * 16];
  if (threadIdx.x < 64) scratch[threadIdx.x] = 0.f;
  __syncthreads();
  const int D = p.dim;
  const float inv_d = 1.f / static_cast<float>(D);
  float acc[kE], dv[kE];
#pragma unroll
  for (int i = 0; i < kE; ++i) acc[i] = dv[i] = 0.f;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const long long at = row * D;
    const float ry = p.y ? p.rstd_y[row] : 0.f;
    const float rx = p.dh ? p.rstd_x[row] : 0.f;
    const float tok = token_gate<T>(p, row);
    float yh[kE], e[kE], xh[kE];
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const int col = threadIdx.x + i * blockDim.x;
      const bool in_row = col < D;
      xh[i] = in_row ? as_float(static_cast<const T*>(p.x)[at + col]) : 0.f;
      yh[i] = in_row && p.y ? as_float(static_cast<const T*>(p.y)[at + col]) * ry : 0.f;
      e[i] = in_row && p.dxn ? as_float(static_cast<const T*>(p.dxn)[at + col]) : 0.f;
    }
    // sum u xh, sum P e, sum P xh with P = s (w + o) yh [act(g)]; e = dx' + r(x') u
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const int col = threadIdx.x + i * blockDim.x;
      if (col >= D) continue;
      float q = 0.f;
      if (p.y) {
        const float a = gate1<T>(p, row, col, tok);
        q = (param1<T>(p.w, p.w_f32, col) + p.offset) * p.scale * yh[i];
        xh[i] = fmaf(a, q, xh[i]);
        if (p.gate_mode != kGateToken) q *= a;
      }
      if (p.dh) {
        const float u = as_float(static_cast<const T*>(p.dh)[at + col]) * (param1<T>(p.v, p.w_f32, col) + p.offset);
        xh[i] *= rx;
        e[i] = fmaf(rx, u, e[i]);
        sums[0] = fmaf(u, xh[i], sums[0]);
      } else {
        xh[i] = 0.f;
      }
      sums[1] = fmaf(q, e[i], sums[1]);
      sums[2] = fmaf(q, xh[i], sums[2]);
    }
    block_sum4(sums, scratch);
    const float c1 = rx * (sums[0] * inv_d);
    const float qdx = sums[1] - c1 * sums[2];
    const float m = qdx * inv_d * tok;
    if (p.gate_mode == kGateToken && threadIdx.x == 0) {
      const float d = qdx * act_slope(tok, p.act);
      if (p.gate_f32) static_cast<float*>(p.dgate_row)[row] = d;
      else static_cast<T*>(p.dgate_row)[row] = from_float<T>(d);
    }
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const int col = threadIdx.x + i * blockDim.x;
      if (col >= D) continue;
      const float dx = fmaf(-c1, xh[i], e[i]);
      if (p.dh) dv[i] = fmaf(as_float(static_cast<const T*>(p.dh)[at + col]), xh[i], dv[i]);
      static_cast<T*>(p.dx)[at + col] = from_float<T>(dx);
      if (p.y) {
        const float a = gate1<T>(p, row, col, tok);
        const float w = (param1<T>(p.w, p.w_f32, col) + p.offset) * p.scale;
        // a channel gate's act is a factor of the whole sum (norm_reduce_kernel)
        acc[i] = fmaf(p.gate_mode == kGateChannel ? dx : a * dx, yh[i], acc[i]);
        static_cast<T*>(p.dy)[at + col] = from_float<T>(ry * fmaf(a * dx, w, -yh[i] * m));
        if (p.gate_mode == kGateFull) {
          const float d = w * yh[i] * dx * act_slope(a, p.act);
          if (p.gate_f32) static_cast<float*>(p.dgate_row)[at + col] = d;
          else static_cast<T*>(p.dgate_row)[at + col] = from_float<T>(d);
        }
      }
    }
    __syncthreads();  // scratch is reused by the next row
  }
  const long long slice = static_cast<long long>(gridDim.x) * D;
  float* part = p.partial + static_cast<long long>(blockIdx.x) * D;
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    const int col = threadIdx.x + i * blockDim.x;
    if (col >= D) continue;
    if (p.y) part[col] = acc[i];
    if (p.dh) part[slice + col] = dv[i];
  }
}

// Column sums of the blocks' partial sums, and the gradients they stand for:
// with S = sum act(g) dx yh (act(g) left out for a channel gate),
//   dw = s S  (s act(g) S for a channel gate),  dgate = s (w + o) act'(g) S.
// 32 columns a block, 32 warps over the partials, in order (8 warps a block
// took 11 us for 296 partials of 4096 columns: a chain of 37 reads each).
struct ReduceParams {
  const float* partial;
  const void *w, *gate;
  void *dw, *dv, *dgate;  // null: not wanted
  int w_f32, gate_f32, act;
  float scale, offset;
  int blocks, dim;
};

template <typename T>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const ReduceParams p) {
  __shared__ float sums[32][33];
  const bool second = blockIdx.y == 1;
  if (second ? !p.dv : !p.dw) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  const float* src = p.partial + (second ? static_cast<long long>(p.blocks) * p.dim : 0) + col;
  float s = 0.f;
  if (col < p.dim)
#pragma unroll 8
    for (int b = warp; b < p.blocks; b += 32) s += src[static_cast<long long>(b) * p.dim];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || col >= p.dim) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) s += sums[w][lane];
  auto store = [&](void* out, int f32, float v) {
    if (f32) static_cast<float*>(out)[col] = v;
    else static_cast<T*>(out)[col] = from_float<T>(v);
  };
  if (second) {
    store(p.dv, p.w_f32, s);
    return;
  }
  s *= p.scale;
  if (p.dgate) {
    const float a = act_of(param1<T>(p.gate, p.gate_f32, col), p.act);
    store(p.dgate, p.gate_f32, s * (param1<T>(p.w, p.w_f32, col) + p.offset) * act_slope(a, p.act));
    s *= a;
  }
  store(p.dw, p.w_f32, s);
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

template <typename T, int kLayout, int kE, int kMode, int kThreads, int kBlocks>
cudaError_t launch_fwd_ring(const NormParams& p, const RingShape& r, int period, int sms, cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  auto kernel = norm_fwd_ring_kernel<T, kLayout, kE, kMode, kThreads, kBlocks>;
  const cudaError_t e = allow_smem(kernel, done);
  if (e != cudaSuccess) return e;
  const int grid = blocks_for(p.rows, static_cast<int64_t>(sms) * r.resident, period);
  kernel<<<grid, r.threads, r.smem, s>>>(p, r.slots);
  return cudaSuccess;
}

template <typename T, int kLayout, int kMode, int kThreads, int kBlocks>
cudaError_t launch_bwd_ring(const NormParams& p, const RingShape& r, int blocks, cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  auto kernel = norm_bwd_ring_kernel<T, kLayout, 16, kMode, kThreads, kBlocks>;
  const cudaError_t e = allow_smem(kernel, done);
  if (e != cudaSuccess) return e;
  kernel<<<blocks, r.threads, r.smem, s>>>(p, r.slots);
  return cudaSuccess;
}

int mode_of(const NormParams& p) {
  return !p.y ? kPreNorm : (p.gate_mode == GMM_GATE_MODE_FULL ? kFullGate : kSharedGate);
}

// Bytes of a slot that holds `inputs` rows of the data type and, with a gate
// per element, one of the gate's.
size_t slot_bytes(const NormParams& p, int es, int layout, int inputs) {
  const bool whole = layout == kWhole;
  const uint32_t gate = p.gate_mode == GMM_GATE_MODE_FULL ? p.dim * (p.gate_f32 ? 4 : es) : 0;
  return static_cast<size_t>(row_pitch(p.dim * es, whole)) * inputs + (gate ? row_pitch(gate, whole) : 0);
}

template <typename T, int kLayout, int kE, int kMode, int kThreads, int kBlocks>
cudaError_t fwd_ring(const NormParams& p, const RowLayout& l, int sms, cudaStream_t s) {
  const RingShape r = ring_shape(l.span, kE, kThreads * kBlocks, slot_bytes(p, sizeof(T), kLayout, p.y ? 2 : 1));
  return launch_fwd_ring<T, kLayout, kE, kMode, kThreads, kBlocks>(p, r, l.period, sms, s);
}

// Elements a thread and blocks an SM.  More elements a thread share the cost
// of a row's sums, fewer leave registers for more warps: one B200, bf16, a
// channel gate unless said,
//                                8 a thread      16 a thread
//   16384 x 4096 (whole words)      88 us           100 us
//   16384 x 4000, gate per element  124             118
//   16384 x 4001 (shifted)          137             104
//   10240 x 6144                    96              92
//   10240 x 6144, gate per element  138             111
//   8192 x 7168                     87              75
template <typename T, int kLayout, int kMode>
cudaError_t fwd_ring_width(const NormParams& p, const RowLayout& l, int sms, cudaStream_t s) {
  constexpr int kNarrow = kLayout == kShifted ? 288 : 256;  // a shifted row of 4096 spans at most one warp more
  if (l.span <= 16 * kNarrow) {
    if constexpr (kLayout != kShifted && kMode != kFullGate)
      return fwd_ring<T, kLayout, 8, kMode, 512, 2>(p, l, sms, s);
    else
      return fwd_ring<T, kLayout, 16, kMode, kNarrow, 3 * 256 / kNarrow>(p, l, sms, s);
  }
  if (l.span <= 6144) return fwd_ring<T, kLayout, 16, kMode, 384, 2>(p, l, sms, s);
  if (l.span <= 8192) return fwd_ring<T, kLayout, 16, kMode, 512, 1>(p, l, sms, s);
  return fwd_ring<T, kLayout, 16, kMode, 1024, 1>(p, l, sms, s);
}

template <typename T, int kLayout>
cudaError_t fwd_ring_mode(const NormParams& p, const RowLayout& l, int sms, cudaStream_t s) {
  switch (mode_of(p)) {
    case kPreNorm: return fwd_ring_width<T, kLayout, kPreNorm>(p, l, sms, s);
    case kSharedGate: return fwd_ring_width<T, kLayout, kSharedGate>(p, l, sms, s);
    default: return fwd_ring_width<T, kLayout, kFullGate>(p, l, sms, s);
  }
}

constexpr int kMaxRingFwdSpan = 16384;

template <typename T>
cudaError_t launch_fwd(const NormParams& p, bool words, int sms, cudaStream_t s) {
  RowLayout l = row_layout(p.dim, sizeof(T), words);
  if (l.span > kMaxRingFwdSpan) l = row_layout(p.dim, sizeof(T), false);
  switch (l.layout) {
    case kWhole: return fwd_ring_mode<T, kWhole>(p, l, sms, s);
    case kShifted: return fwd_ring_mode<T, kShifted>(p, l, sms, s);
    default: return fwd_ring_mode<T, kSingle>(p, l, sms, s);
  }
}

// The ring's backward kernels keep 16 elements a thread (their parameters and
// sums over rows in registers) in at most 512 threads.
constexpr int kMaxRingBwdSpan = 8192;

RowLayout bwd_layout(int dim, int es, bool words) {
  const RowLayout l = row_layout(dim, es, words);
  return l.span > kMaxRingBwdSpan ? row_layout(dim, es, false) : l;
}

constexpr int kBwdThreadsSm = 512;  // threads of all blocks of an SM (128 registers each)

// Blocks of the backward pass: what is resident at once, so that every block
// adds up as many rows as possible before it leaves its partial sums.
int64_t bwd_most_blocks(int span, int sms) {
  const int threads = threads_for((span + 15) / 16);  // one block an SM past kMaxRingBwdSpan
  return static_cast<int64_t>(sms) * std::max(1, std::min(16, kBwdThreadsSm / threads));
}

template <typename T, int kLayout, int kThreads, int kBlocks>
cudaError_t bwd_ring_mode(const NormParams& p, const RowLayout& l, int blocks, cudaStream_t s) {
  const int inputs = 1 + (p.y ? 1 : 0) + (p.dxn ? 1 : 0) + (p.dh ? 1 : 0);
  const RingShape r = ring_shape(l.span, 16, kThreads * kBlocks, slot_bytes(p, sizeof(T), kLayout, inputs));
  switch (mode_of(p)) {
    case kPreNorm: return launch_bwd_ring<T, kLayout, kPreNorm, kThreads, kBlocks>(p, r, blocks, s);
    case kSharedGate: return launch_bwd_ring<T, kLayout, kSharedGate, kThreads, kBlocks>(p, r, blocks, s);
    default: return launch_bwd_ring<T, kLayout, kFullGate, kThreads, kBlocks>(p, r, blocks, s);
  }
}

template <typename T, int kLayout>
cudaError_t bwd_ring_width(const NormParams& p, const RowLayout& l, int blocks, cudaStream_t s) {
  return l.span <= 4096 ? bwd_ring_mode<T, kLayout, 256, 2>(p, l, blocks, s)
                        : bwd_ring_mode<T, kLayout, 512, 1>(p, l, blocks, s);
}

template <typename T>
cudaError_t launch_bwd(const NormParams& p, const RowLayout& l, int blocks, cudaStream_t s) {
  if (l.span > kMaxRingBwdSpan) {
    norm_bwd_kernel<T, kMaxNormDim / kMaxThreads><<<blocks, kMaxThreads, 0, s>>>(p);
    return cudaSuccess;
  }
  switch (l.layout) {
    case kWhole: return bwd_ring_width<T, kWhole>(p, l, blocks, s);
    case kShifted: return bwd_ring_width<T, kShifted>(p, l, blocks, s);
    default: return bwd_ring_width<T, kSingle>(p, l, blocks, s);
  }
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

int norm_device_error(int* status, bool clear) { return read_row_error(status, clear); }

}  // namespace gmm_sm100

extern "C" {

int gmm_sm100_post_norm(const void* y, const void* x, const void* weight, const void* gate, const void* next_weight,
                        int64_t rows, int64_t dim, int dtype, int weight_dtype, int gate_dtype, int gate_mode,
                        int gate_act, float residual_scale, float eps, float weight_offset, void* x_new, void* h,
                        float* rstd_y, float* rstd_x, void* stream) {
  using namespace gmm_sm100;
  if (int rc = check_common(rows, dim, dtype, weight_dtype, gate_dtype, gate_mode, gate_act, eps)) return rc;
  if (rows == 0 || dim == 0) return GMM_OK;
  if (!x || (y && (!weight || !x_new)) || (!y && !h) || (h && !next_weight) ||
      (gate_mode != GMM_GATE_MODE_NONE && (!y || !gate)))
    return set_error(GMM_ERR_INVALID_ARGUMENT, "null pointer");
  const uintptr_t es = dtype == GMM_DTYPE_F32 ? 4 : 2, ws = weight_dtype == GMM_DTYPE_F32 ? 4 : 2,
                  gs = gate_dtype == GMM_DTYPE_F32 ? 4 : 2;
  if (!on(y, es) || !on(x, es) || !on(x_new, es) || !on(h, es) || !on(weight, ws) || !on(next_weight, ws) ||
      !on(gate, gs) || !on(rstd_y, 4) || !on(rstd_x, 4))
    return set_error(GMM_ERR_ALIGNMENT, "a pointer is not aligned to its element size");
  int sms = 0;
  if (int rc = current_sm_count(&sms)) return rc;
  NormParams p = {};
  p.y = y; p.x = x; p.w = weight; p.v = next_weight; p.gate = gate;
  p.xn = x_new; p.h = h; p.rstd_y = rstd_y; p.rstd_x = rstd_x;
  p.rows = rows; p.dim = static_cast<int>(dim);
  p.w_f32 = weight_dtype == GMM_DTYPE_F32; p.gate_f32 = gate_dtype == GMM_DTYPE_F32;
  p.gate_mode = gate_mode; p.act = gate_act;
  p.scale = residual_scale; p.eps = eps; p.offset = weight_offset;
  const bool words = on(y, 16) && on(x, 16) && on(x_new, 16) && on(h, 16) && on(weight, 16) && on(next_weight, 16) &&
                     (gate_mode == GMM_GATE_MODE_TOKEN || on(gate, 16));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = dtype == GMM_DTYPE_F32    ? launch_fwd<float>(p, words, sms, s)
                  : dtype == GMM_DTYPE_BF16 ? launch_fwd<__nv_bfloat16>(p, words, sms, s)
                                            : launch_fwd<__half>(p, words, sms, s);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GMM_OK : set_error(GMM_ERR_CUDA, cudaGetErrorString(e));
}

size_t gmm_sm100_post_norm_backward_workspace_size(int64_t rows, int64_t dim) {
  using namespace gmm_sm100;
  if (rows <= 0 || dim <= 0 || dim > kMaxNormDim) return 0;
  int sms = 0;
  if (current_sm_count(&sms)) return 0;
  // the largest count of any layout (a narrower span never has fewer blocks)
  const int64_t most = std::min<int64_t>(rows, bwd_most_blocks(static_cast<int>(dim), sms));
  return 2 * sizeof(float) * static_cast<size_t>(most) * dim;
}

int gmm_sm100_post_norm_backward(const void* y, const void* x, const void* weight, const void* gate,
                                 const void* next_weight, const float* rstd_y, const float* rstd_x,
                                 const void* dx_new, const void* dh, int64_t rows, int64_t dim, int dtype,
                                 int weight_dtype, int gate_dtype, int gate_mode, int gate_act, float residual_scale,
                                 float weight_offset, void* dy, void* dx, void* dweight, void* dgate,
                                 void* dnext_weight, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gmm_sm100;
  if (int rc = check_common(rows, dim, dtype, weight_dtype, gate_dtype, gate_mode, gate_act, 0.f)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t ws = weight_dtype == GMM_DTYPE_F32 ? 4 : 2, gs = gate_dtype == GMM_DTYPE_F32 ? 4 : 2,
               es = dtype == GMM_DTYPE_F32 ? 4 : 2;
  if (dim == 0) return GMM_OK;
  if (rows == 0) {  // sums over no row
    cudaError_t e = cudaSuccess;
    if (dweight) e = cudaMemsetAsync(dweight, 0, ws * dim, s);
    if (e == cudaSuccess && dnext_weight) e = cudaMemsetAsync(dnext_weight, 0, ws * dim, s);
    if (e == cudaSuccess && dgate && gate_mode == GMM_GATE_MODE_CHANNEL) e = cudaMemsetAsync(dgate, 0, gs * dim, s);
    return e == cudaSuccess ? GMM_OK : set_error(GMM_ERR_CUDA, cudaGetErrorString(e));
  }
  if (!x || (!dx_new && !dh) || (y && (!weight || !rstd_y || !dy || !dweight)) || (!y && !dh) ||
      (dh && (!next_weight || !rstd_x || !dnext_weight)) || !dx ||
      (gate_mode != GMM_GATE_MODE_NONE && (!y || !gate || !dgate)))
    return set_error(GMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (!on(y, es) || !on(x, es) || !on(dx_new, es) || !on(dh, es) || !on(dy, es) || !on(dx, es) || !on(weight, ws) ||
      !on(next_weight, ws) || !on(dweight, ws) || !on(dnext_weight, ws) || !on(gate, gs) || !on(dgate, gs) ||
      !on(rstd_y, 4) || !on(rstd_x, 4))
    return set_error(GMM_ERR_ALIGNMENT, "a pointer is not aligned to its element size");
  int sms = 0;
  if (int rc = current_sm_count(&sms)) return rc;
  const size_t need = gmm_sm100_post_norm_backward_workspace_size(rows, dim);
  if (!workspace || workspace_bytes < need || !on(workspace, 16)) {
    char msg[96];
    std::snprintf(msg, sizeof msg, "workspace needs %zu bytes (16-byte aligned), got %zu", need, workspace_bytes);
    return set_error(GMM_ERR_WORKSPACE, msg);
  }
  NormParams p = {};
  p.y = y; p.x = x; p.w = weight; p.v = next_weight; p.gate = gate; p.dxn = dx_new; p.dh = dh;
  p.dy = dy; p.dx = dx; p.dgate_row = dgate;
  p.rstd_y = const_cast<float*>(rstd_y); p.rstd_x = const_cast<float*>(rstd_x);
  p.partial = static_cast<float*>(workspace);
  p.rows = rows; p.dim = static_cast<int>(dim);
  p.w_f32 = weight_dtype == GMM_DTYPE_F32; p.gate_f32 = gate_dtype == GMM_DTYPE_F32;
  p.gate_mode = gate_mode; p.act = gate_act;
  p.scale = residual_scale; p.offset = weight_offset;
  const bool words = on(y, 16) && on(x, 16) && on(dx_new, 16) && on(dh, 16) && on(dy, 16) && on(dx, 16) &&
                     on(weight, 16) && on(next_weight, 16) &&
                     (gate_mode == GMM_GATE_MODE_TOKEN || (on(gate, 16) && on(dgate, 16)));
  const RowLayout layout = bwd_layout(p.dim, static_cast<int>(es), words);
  const int blocks = blocks_for(rows, bwd_most_blocks(layout.span, sms), layout.period);
  ReduceParams r = {};
  r.partial = p.partial;
  r.w = weight;
  r.gate = gate;
  r.dw = y ? dweight : nullptr;
  r.dv = dh ? dnext_weight : nullptr;
  r.dgate = gate_mode == GMM_GATE_MODE_CHANNEL ? dgate : nullptr;
  r.w_f32 = p.w_f32;
  r.gate_f32 = p.gate_f32;
  r.act = gate_act;
  r.scale = residual_scale;
  r.offset = weight_offset;
  r.blocks = blocks;
  r.dim = p.dim;
  const dim3 rgrid((p.dim + 31) / 32, 2);
  auto go = [&](auto t) {
    using T = decltype(t);
    const cudaError_t e = launch_bwd<T>(p, layout, blocks, s);
    if (e != cudaSuccess) return e;
    norm_reduce_kernel<T><<<rgrid, 1024, 0, s>>>(r);
    return cudaGetLastError();
  };
  const cudaError_t e = dtype == GMM_DTYPE_F32    ? go(float{})
                        : dtype == GMM_DTYPE_BF16 ? go(__nv_bfloat16{})
                                                  : go(__half{});
  return e == cudaSuccess ? GMM_OK : set_error(GMM_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
