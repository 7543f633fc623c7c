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
// mean(u xh); it is linear in it, so three sums of one pass give both:
//   C = sum u xh,  A = sum P e,  B = sum P r(x') xh   with e = dx' + r(x') u and
//   P = s act(g) n:   sum t yh = A - (C / D) B.
// Everything is held in fp32 and rounded once, on store.  Rows are walked by
// blocks in a fixed order and parameter gradients added up per block, then
// over blocks in order, so results do not change from run to run.

#include <algorithm>
#include <cstdio>

#include "gmm_sm100.h"
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
  float* partial;     // backward: [3][blocks][D] sums of dw, dv, dgate (channel)
  long long rows;
  int dim;
  int w_f32, gate_f32;  // parameters in fp32 (else the rows' type)
  int gate_mode, act;
  float scale, eps, offset;
};

template <typename T, bool kVec>
__device__ __forceinline__ void load_param(const void* p, int f32, long long at, int col, int dim, float (&f)[8]) {
  if (f32 || sizeof(T) == 4) {
    const Raw8<float> r = load8<float, kVec>(static_cast<const float*>(p) + at, col, dim);
    unpack(r, f);
  } else {
    const Raw8<T> r = load8<T, kVec>(static_cast<const T*>(p) + at, col, dim);
    unpack(r, f);
  }
}

__device__ __forceinline__ float act_of(float g, int act) {
  return act == GMM_GATE_TANH ? tanhf(g) : act == GMM_GATE_SIGMOID ? 1.f / (1.f + expf(-g)) : g;
}
// act'(g) from a = act(g)
__device__ __forceinline__ float act_slope(float a, int act) {
  return act == GMM_GATE_TANH ? 1.f - a * a : act == GMM_GATE_SIGMOID ? a * (1.f - a) : 1.f;
}

// Sums of n values over the block; every thread gets them.  `scratch` holds
// 32 * n floats; two calls in a row need different scratch.
template <int n>
__device__ __forceinline__ void block_sum(float (&s)[n], float* scratch) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int j = 0; j < n; ++j) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
  if (blockDim.x > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0)
#pragma unroll
      for (int j = 0; j < n; ++j) scratch[j * 32 + warp] = s[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < n; ++j) s[j] = lane < warps ? scratch[j * 32 + lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
      for (int j = 0; j < n; ++j) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
  }
}

// The gate of a chunk: act(g) (ones without a gate); `token` is the row's
// value of a token gate, already through act.
template <typename T, bool kVec>
__device__ __forceinline__ void load_gate(const NormParams& p, long long row, int col, float token, float (&a)[8]) {
  if (p.gate_mode == kGateChannel || p.gate_mode == kGateFull) {
    load_param<T, kVec>(p.gate, p.gate_f32, p.gate_mode == kGateFull ? row * p.dim : 0, col, p.dim, a);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = act_of(a[j], p.act);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = token;
  }
}

template <typename T>
__device__ __forceinline__ float token_gate(const NormParams& p, long long row) {
  if (p.gate_mode != kGateToken) return 1.f;
  const float g = p.gate_f32 ? static_cast<const float*>(p.gate)[row] : as_float(static_cast<const T*>(p.gate)[row]);
  return act_of(g, p.act);
}

// One block per row (grid-stride); a thread holds the 8-element chunks
// threadIdx.x + i * blockDim.x of the row in registers.
template <typename T, int kChunks, bool kVec>
__global__ void __launch_bounds__(kMaxThreads) norm_fwd_kernel(const NormParams p) {
  __shared__ float scratch[2][32];
  const int D = p.dim;
  const float inv_d = 1.f / static_cast<float>(D);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * D;
    float xs[kChunks][8];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) unpack(load8<T, kVec>(x, (threadIdx.x + i * blockDim.x) * 8, D), xs[i]);
    if (p.y) {
      const T* y = static_cast<const T*>(p.y) + row * D;
      float ys[kChunks][8];
      float sq[1] = {0.f};
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        unpack(load8<T, kVec>(y, (threadIdx.x + i * blockDim.x) * 8, D), ys[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) sq[0] = fmaf(ys[i][j], ys[i][j], sq[0]);
      }
      block_sum(sq, scratch[0]);
      const float ry = rsqrtf(sq[0] * inv_d + p.eps);
      if (p.rstd_y && threadIdx.x == 0) p.rstd_y[row] = ry;
      const float tok = token_gate<T>(p, row);
      T* xn = static_cast<T*>(p.xn) + row * D;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = (threadIdx.x + i * blockDim.x) * 8;
        float w[8], a[8];
        load_param<T, kVec>(p.w, p.w_f32, 0, col, D, w);
        load_gate<T, kVec>(p, row, col, tok, a);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          xs[i][j] = col + j < D ? fmaf(p.scale * a[j], (w[j] + p.offset) * (ys[i][j] * ry), xs[i][j]) : 0.f;
        store8<T, kVec>(xn, col, D, xs[i]);
      }
    }
    if (p.h) {
      float sq[1] = {0.f};
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sq[0] = fmaf(xs[i][j], xs[i][j], sq[0]);
      block_sum(sq, scratch[1]);
      const float rx = rsqrtf(sq[0] * inv_d + p.eps);
      if (p.rstd_x && threadIdx.x == 0) p.rstd_x[row] = rx;
      T* h = static_cast<T*>(p.h) + row * D;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = (threadIdx.x + i * blockDim.x) * 8;
        float v[8], o[8];
        load_param<T, kVec>(p.v, p.w_f32, 0, col, D, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (v[j] + p.offset) * (xs[i][j] * rx);
        store8<T, kVec>(h, col, D, o);
      }
    }
    __syncthreads();  // scratch is reused by the next row
  }
}

// Backward of the same rows; a block adds up its rows' parameter gradients in
// registers (a thread owns its columns) and leaves them in `partial`.
template <typename T, int kChunks, bool kVec>
__global__ void __launch_bounds__(kMaxThreads) norm_bwd_kernel(const NormParams p) {
  __shared__ float scratch[4 * 32];
  const int D = p.dim;
  const float inv_d = 1.f / static_cast<float>(D);
  float dw[kChunks][8], dv[kChunks][8], dg[kChunks][8];
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = dv[i][j] = dg[i][j] = 0.f;

  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const long long at = row * D;
    Raw8<T> rx_[kChunks], ry_[kChunks], rdx[kChunks], rdh[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      rx_[i] = load8<T, kVec>(static_cast<const T*>(p.x) + at, col, D);
      if (p.y) ry_[i] = load8<T, kVec>(static_cast<const T*>(p.y) + at, col, D);
      if (p.dxn) rdx[i] = load8<T, kVec>(static_cast<const T*>(p.dxn) + at, col, D);
      if (p.dh) rdh[i] = load8<T, kVec>(static_cast<const T*>(p.dh) + at, col, D);
    }
    const float ry = p.y ? p.rstd_y[row] : 0.f;
    const float rx = p.dh ? p.rstd_x[row] : 0.f;
    const float tok = token_gate<T>(p, row);
    // Q = s n (the gate left out when it is the row's own), e = dx' + r(x') u, xh
    auto chunk = [&](int i, float (&yh)[8], float (&w)[8], float (&a)[8], float (&e)[8], float (&xh)[8],
                     float (&dhv)[8], float (&v)[8]) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      float xs[8];
      unpack(rx_[i], xs);
      if (p.y) {
        unpack(ry_[i], yh);
        load_param<T, kVec>(p.w, p.w_f32, 0, col, D, w);
        load_gate<T, kVec>(p, row, col, tok, a);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          yh[j] *= ry;
          w[j] = (w[j] + p.offset) * p.scale;
          xs[j] = fmaf(a[j], w[j] * yh[j], xs[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) yh[j] = w[j] = a[j] = 0.f;
      }
      if (p.dxn) unpack(rdx[i], e);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = 0.f;
      if (p.dh) {
        unpack(rdh[i], dhv);
        load_param<T, kVec>(p.v, p.w_f32, 0, col, D, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          xh[j] = xs[j] * rx;
          e[j] = fmaf(rx * dhv[j], v[j] + p.offset, e[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) xh[j] = dhv[j] = v[j] = 0.f;
      }
    };
    const bool own_gate = p.gate_mode == kGateToken;  // act(g) is one number of the row
    float sums[3] = {0.f, 0.f, 0.f};                  // C, A, B
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float yh[8], w[8], a[8], e[8], xh[8], dhv[8], v[8];
      chunk(i, yh, w, a, e, xh, dhv, v);
      const int col = (threadIdx.x + i * blockDim.x) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float q = w[j] * yh[j] * (own_gate ? 1.f : a[j]);
        if (col + j < D) {
          sums[0] = fmaf(dhv[j] * (v[j] + p.offset), xh[j], sums[0]);
          sums[1] = fmaf(q, e[j], sums[1]);
          sums[2] = fmaf(q, rx * xh[j], sums[2]);
        }
      }
    }
    block_sum(sums, scratch);
    const float c = sums[0] * inv_d;
    const float qdx = sums[1] - c * sums[2];  // sum of Q dx
    const float m = qdx * inv_d * (own_gate ? tok : 1.f);  // mean(t yh)
    if (own_gate && threadIdx.x == 0) {
      const float d = qdx * act_slope(tok, p.act);
      if (p.gate_f32) static_cast<float*>(p.dgate_row)[row] = d;
      else static_cast<T*>(p.dgate_row)[row] = from_float<T>(d);
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      float yh[8], w[8], a[8], e[8], xh[8], dhv[8], v[8];
      chunk(i, yh, w, a, e, xh, dhv, v);
      float dx[8], dy[8], dgr[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dx[j] = fmaf(-rx * c, xh[j], e[j]);
        const float t = a[j] * dx[j];  // without s (w + o)
        dy[j] = ry * (t * w[j] - yh[j] * m);
        dw[i][j] = fmaf(p.scale * t, yh[j], dw[i][j]);
        dv[i][j] = fmaf(dhv[j], xh[j], dv[i][j]);
        dgr[j] = w[j] * yh[j] * dx[j] * act_slope(a[j], p.act);
        dg[i][j] += dgr[j];
      }
      if (p.dx) store8<T, kVec>(static_cast<T*>(p.dx) + at, col, D, dx);
      if (p.y) store8<T, kVec>(static_cast<T*>(p.dy) + at, col, D, dy);
      if (p.gate_mode == kGateFull) {
        if (p.gate_f32) store8<float, kVec>(static_cast<float*>(p.dgate_row) + at, col, D, dgr);
        else store8<T, kVec>(static_cast<T*>(p.dgate_row) + at, col, D, dgr);
      }
    }
    __syncthreads();  // scratch is reused by the next row
  }
  const long long slice = static_cast<long long>(gridDim.x) * D;
  float* part = p.partial + static_cast<long long>(blockIdx.x) * D;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int col = (threadIdx.x + i * blockDim.x) * 8;
    if (p.y) store8<float, kVec>(part, col, D, dw[i]);
    if (p.dh) store8<float, kVec>(part + slice, col, D, dv[i]);
    if (p.gate_mode == kGateChannel) store8<float, kVec>(part + 2 * slice, col, D, dg[i]);
  }
}

struct ReduceParams {
  const float* partial;  // [3][blocks][D]
  void* out[3];          // null: not wanted
  int f32[3];
  int blocks, dim;
};

// Column sums of the blocks' partial sums: 32 columns a block, 8 warps over
// the partials, in order.
template <typename T>
__global__ void __launch_bounds__(256) norm_reduce_kernel(const ReduceParams p) {
  __shared__ float sums[8][33];
  const int which = blockIdx.y;
  if (!p.out[which]) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  const float* src = p.partial + static_cast<long long>(which) * p.blocks * p.dim;
  float s = 0.f;
  if (col < p.dim)
    for (int b = warp; b < p.blocks; b += 8) s += src[static_cast<long long>(b) * p.dim + col];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < p.dim) {
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][lane];
    if (p.f32[which]) static_cast<float*>(p.out[which])[col] = s;
    else static_cast<T*>(p.out[which])[col] = from_float<T>(s);
  }
}

int chunks_of(int dim) { return (dim + 7) / 8; }
int threads_of(int dim, int per) { return std::max(32, (chunks_of(dim) + 32 * per - 1) / (32 * per) * 32); }

// Blocks of the backward pass: what is resident at once, so that every block
// adds up as many rows as possible before it leaves its partial sums.
int bwd_blocks(int64_t rows, int dim, int sms) {
  const int per = dim <= 8 * kMaxThreads ? 1 : (dim <= 16 * kMaxThreads ? 2 : 4);
  const int resident = std::max(1, std::min(16, 512 / threads_of(dim, per)));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, static_cast<int64_t>(sms) * resident)));
}

template <typename T, bool kVec>
void launch_fwd(const NormParams& p, int sms, cudaStream_t s) {
  const int grid = static_cast<int>(std::min<long long>(p.rows, 64LL * sms));
  if (p.dim <= 8 * kMaxThreads) norm_fwd_kernel<T, 1, kVec><<<grid, threads_of(p.dim, 1), 0, s>>>(p);
  else if (p.dim <= 16 * kMaxThreads) norm_fwd_kernel<T, 2, kVec><<<grid, threads_of(p.dim, 2), 0, s>>>(p);
  else norm_fwd_kernel<T, 4, kVec><<<grid, threads_of(p.dim, 4), 0, s>>>(p);
}

template <typename T, bool kVec>
void launch_bwd(const NormParams& p, int blocks, cudaStream_t s) {
  if (p.dim <= 8 * kMaxThreads) norm_bwd_kernel<T, 1, kVec><<<blocks, threads_of(p.dim, 1), 0, s>>>(p);
  else if (p.dim <= 16 * kMaxThreads) norm_bwd_kernel<T, 2, kVec><<<blocks, threads_of(p.dim, 2), 0, s>>>(p);
  else norm_bwd_kernel<T, 4, kVec><<<blocks, threads_of(p.dim, 4), 0, s>>>(p);
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
  const bool vec = dim % 8 == 0 && on(y, 16) && on(x, 16) && on(x_new, 16) && on(h, 16) && on(weight, 16) &&
                   on(next_weight, 16) && (gate_mode == GMM_GATE_MODE_TOKEN || on(gate, 16));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    vec ? launch_fwd<T, true>(p, sms, s) : launch_fwd<T, false>(p, sms, s);
  };
  if (dtype == GMM_DTYPE_F32) go(float{});
  else if (dtype == GMM_DTYPE_BF16) go(__nv_bfloat16{});
  else go(__half{});
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GMM_OK : set_error(GMM_ERR_CUDA, cudaGetErrorString(e));
}

size_t gmm_sm100_post_norm_backward_workspace_size(int64_t rows, int64_t dim) {
  using namespace gmm_sm100;
  if (rows <= 0 || dim <= 0 || dim > kMaxNormDim) return 0;
  int sms = 0;
  if (current_sm_count(&sms)) return 0;
  return 3 * sizeof(float) * static_cast<size_t>(bwd_blocks(rows, static_cast<int>(dim), sms)) * dim;
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
  const int blocks = bwd_blocks(rows, static_cast<int>(dim), sms);
  const size_t need = 3 * sizeof(float) * static_cast<size_t>(blocks) * dim;
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
  const bool vec = dim % 8 == 0 && on(y, 16) && on(x, 16) && on(dx_new, 16) && on(dh, 16) && on(dy, 16) && on(dx, 16) &&
                   on(weight, 16) && on(next_weight, 16) &&
                   (gate_mode == GMM_GATE_MODE_TOKEN || (on(gate, 16) && on(dgate, 16)));
  ReduceParams r = {};
  r.partial = p.partial;
  r.out[0] = y ? dweight : nullptr;
  r.out[1] = dh ? dnext_weight : nullptr;
  r.out[2] = gate_mode == GMM_GATE_MODE_CHANNEL ? dgate : nullptr;
  r.f32[0] = r.f32[1] = p.w_f32;
  r.f32[2] = p.gate_f32;
  r.blocks = blocks;
  r.dim = p.dim;
  const dim3 rgrid((p.dim + 31) / 32, 3);
  auto go = [&](auto t) {
    using T = decltype(t);
    vec ? launch_bwd<T, true>(p, blocks, s) : launch_bwd<T, false>(p, blocks, s);
    norm_reduce_kernel<T><<<rgrid, 256, 0, s>>>(r);
  };
  if (dtype == GMM_DTYPE_F32) go(float{});
  else if (dtype == GMM_DTYPE_BF16) go(__nv_bfloat16{});
  else go(__half{});
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GMM_OK : set_error(GMM_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
