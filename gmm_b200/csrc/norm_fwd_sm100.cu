// norm_fwd_sm100.cu -- forward of the norms around a block (norm_sm100.cuh).

#include "norm_sm100.cuh"

namespace gmm_sm100 {
namespace {

template <typename T, int kLayout, int kE, int kMode, int kThreads, int kBlocks>
__global__ void __launch_bounds__(kThreads, kBlocks) norm_fwd_ring_kernel(const NormParams p, int slots) {
  constexpr int V = kUnit<T, kLayout>, kUnits = kE / V;
  using G = GateOf<T, kMode>;  // of a gate per element
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float scratch[2][2][kMaxWarps];  // by sum and by parity of the row
  const int D = p.dim;
  RowRing<3, kLayout == kWhole> ring;
  ring.input(0, p.x, sizeof(T), D, D);
  ring.input(1, p.y, sizeof(T), kMode == kPreNorm ? 0 : D, D);
  // The element size from the call: as a constant it lets the compiler merge the
  // inputs' addressing, at the price of spills (8192 x 6144 bf16, 89 -> 104 us).
  ring.input(2, p.gate, p.gate_f32 ? 4 : sizeof(T), is_full(kMode) ? D : 0, D);
  ring.start(smem, slots, p.rows, gate_pad(kLayout, kMode));
  if (threadIdx.x < 32)
#pragma unroll
    for (int i = 0; i < 4; ++i) scratch[i >> 1][i & 1][threadIdx.x] = 0.f;

  const Span<V, kLayout> span(D, D);
  const int units = span.units;
  float pw[kE], vo[kE];
  row_params<T, V, kLayout, kE, kMode>(p, span, p.h != nullptr, pw, vo);
  auto input = [&](int i, int slot, long long row) {
    return smem + (kLayout == kShifted ? ring.word_at(slot, i) : ring.at(slot, i, row));
  };
  // An fp32 gate beside 16-bit rows: a unit is two words, and the row may start in the second.
  const int gate_words = kLayout == kShifted && kMode == kFullGateF32 ? span.shift / 4 * 16 : 0;
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
      if constexpr (is_full(kMode)) {  // y * act(g): the gate is not needed again
        const auto* gs = input(2, slot, row) - gate_words;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int c = threadIdx.x + i * blockDim.x;
          float g[V];
#pragma unroll
          for (int j = 0; j < V; ++j) g[j] = 0.f;
          if (c < units) read_param<G, V>(gs, c, g);
          if (kLayout == kShifted) span.mask(c, g);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            act_of<sizeof(G) == 2, false, 1>(g + j, p.act);
            y[i * V + j] *= g[j];
          }
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
  if constexpr (kLayout != kShifted && !is_full(kMode))
    if (l.span <= 4096) return fwd_ring<T, kLayout, 8, kMode, 512, 2>(p, l, sms, s);
  if (l.span <= 8192) return fwd_ring<T, kLayout, 16, kMode, kFwdThreadsSm, 1>(p, l, sms, s);
  return fwd_ring<T, kLayout, 16, kMode, 1024, 1>(p, l, sms, s);
}

template <typename T, int kLayout>
cudaError_t fwd_ring_mode(const NormParams& p, const RowLayout& l, int sms, cudaStream_t s) {
  switch (mode_of(p, sizeof(T))) {
    case kPreNorm: return fwd_ring_width<T, kLayout, kPreNorm>(p, l, sms, s);
    case kSharedGate: return fwd_ring_width<T, kLayout, kSharedGate>(p, l, sms, s);
    case kFullGateF32:
      if constexpr (sizeof(T) == 2) return fwd_ring_width<T, kLayout, kFullGateF32>(p, l, sms, s);
      [[fallthrough]];
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

}  // namespace

int norm_fwd_device_error(int* status, bool clear) { return read_row_error(status, clear); }

}  // namespace gmm_sm100

extern "C" int gmm_sm100_post_norm(const void* y, const void* x, const void* weight, const void* gate, const void* next_weight,
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
