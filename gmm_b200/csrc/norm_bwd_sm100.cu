// norm_bwd_sm100.cu -- backward of the norms around a block (norm_sm100.cuh).

#include "norm_sm100.cuh"

namespace gmm_sm100 {
namespace {

// Backward.  The rows stay in the ring between the sums and the results
// (re-reading shared memory costs less than holding four rows in registers),
// so a slot is refilled one row later, past the next row's barrier -- or, with
// a single slot, behind a barrier of its own.
//
// kWide: rows wider than the registers hold, in column windows of D elements
// of rows `pitch` apart, each by a launch of its own: first every window's part
// of the four sums, then its gradients from all windows' sums.
//
// kNext: h has a gradient.  Without one the residual has no part in any
// gradient (dx = dx', and of the four sums only A1 is left), and it is not
// read: zeros times an infinity in it would be NaN.
template <typename T, int kLayout, int kE, int kMode, bool kWide, bool kNext>
__global__ void __launch_bounds__(kBwdThreadsSm) norm_bwd_ring_kernel(const NormParams p, int slots) {
  constexpr int V = kUnit<T, kLayout>;
  using G = GateOf<T, kMode>;  // of a gate per element
  // A thread works on groups of kG elements: one unit, or two of one element.
  constexpr int kU = V == 1 ? 2 : 1, kG = V * kU, kGroups = kE / kG;
  static_assert(kBwdThreadsSm <= 16 * 32, "block_sum4");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float scratch[2][4 * 16];
  const int D = p.dim;
  RowRing<5, kLayout == kWhole> ring;
  const int pitch = kWide ? p.pitch : D;
  ring.input(0, p.x, sizeof(T), kNext ? D : 0, pitch);
  ring.input(1, p.y, sizeof(T), kMode == kPreNorm ? 0 : D, pitch);
  ring.input(2, p.dxn, sizeof(T), p.dxn ? D : 0, pitch);
  ring.input(3, p.dh, sizeof(T), kNext ? D : 0, pitch);
  ring.input(4, p.gate, sizeof(G), is_full(kMode) ? D : 0, pitch);
  ring.start(smem, slots, p.rows, gate_pad(kLayout, kMode));
  if (threadIdx.x < 32)
#pragma unroll
    for (int i = 0; i < 4; ++i) scratch[i >> 1][(i & 1) * 32 + threadIdx.x] = 0.f;

  const Span<V, kLayout> span(D, pitch);
  const int units = span.units;
  float pw[kE], vo[kE], acc[kE], dv[kE];
  row_params<T, V, kLayout, kE, kMode>(p, span, kNext, pw, vo);
  auto input = [&](int i, int slot, long long row) {
    return smem + (kLayout == kShifted ? ring.word_at(slot, i) : ring.at(slot, i, row));
  };
  // An fp32 gate beside 16-bit rows: a unit is two words, and the row may start in the second.
  const int gate_words = kLayout == kShifted && kMode == kFullGateF32 ? span.shift / 4 * 16 : 0;
  UnitMask<T, V, kLayout> mask[kE / V];
#pragma unroll
  for (int i = 0; i < kE / V; ++i) mask[i].set(span, threadIdx.x + i * blockDim.x);
#pragma unroll
  for (int j = 0; j < kE; ++j) acc[j] = dv[j] = 0.f;
  __syncthreads();  // barriers initialised
  const float inv_d = 1.f / static_cast<float>(pitch);

  int slot = 0;
  uint32_t phase = 0;
  int odd = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float ry = kMode == kPreNorm ? 0.f : p.rstd_y[row];
    const float rx = kNext ? p.rstd_x[row] : 0.f;
    const float tok = kMode == kSharedGate ? token_gate<T>(p, row) : 1.f;
    ring.wait(slot, phase, row);
    const uint8_t *in_x = input(0, slot, row), *in_y = input(1, slot, row), *in_dx = input(2, slot, row),
                  *in_dh = input(3, slot, row), *in_g = input(4, slot, row) - gate_words;
    auto unit = [&](int g, int u) { return static_cast<int>(threadIdx.x + (g * kU + u) * blockDim.x); };
    const Both to_x(is_full(kMode) ? ry : ry * tok);
    // Of a group's elements: y, Q (times act(g) with a gate per element, which
    // `a` returns), x', u = dh (v + o), dh.  Zeros past the row's end; x', u
    // and dh only with kNext.  `slope` returns act'(g) if it is there.
    auto read = [&](int g, float (&y)[kG], float (&q)[kG], float (&a)[kG], float (&x)[kG], float (&u)[kG],
                    float (&dh)[kG], float* slope) {
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        const int c = unit(g, k);
        const bool in = V > 1 || c < units;
        const auto& own = mask[g * kU + k];
        if constexpr (kNext) read_unit_or_0<T, V>(in_x, c, in, own, x + k * V);
        if constexpr (kMode != kPreNorm) read_unit_or_0<T, V>(in_y, c, in, own, y + k * V);
        if constexpr (kNext) read_unit_or_0<T, V>(in_dh, c, in, own, dh + k * V);
        if constexpr (is_full(kMode)) {
#pragma unroll
          for (int j = 0; j < V; ++j) a[k * V + j] = 0.f;
          if (in) read_param<G, V>(in_g, c, a + k * V);
          if (kLayout == kShifted) span.mask(c, a + k * V);
          if (slope) act_of<sizeof(G) == 2, true, V>(a + k * V, p.act, slope + k * V);
          else act_of<sizeof(G) == 2, false, V>(a + k * V, p.act);
        }
      }
#pragma unroll
      for (int j = 0; j < kG; j += 2) {
        if constexpr (kMode != kPreNorm) {
          mul2(q + j, y + j, pw + g * kG + j);
          if constexpr (is_full(kMode)) mul2(q + j, q + j, a + j);
          if constexpr (kNext) fma2(x + j, q + j, to_x, x + j);
        }
        if constexpr (kNext) mul2(u + j, dh + j, vo + g * kG + j);
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
    float s[4];
    if (!kWide || p.phase == 1) {
      float s2[4][2] = {};  // C, A1, A2, B: even and odd elements
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (V > 1 && unit(g, 0) >= units) continue;
        float y[kG], q[kG], a[kG], x[kG], u[kG], dh[kG], d[kG];
        read(g, y, q, a, x, u, dh, nullptr);
        if constexpr (kMode != kPreNorm) read_dx(g, d);
#pragma unroll
        for (int j = 0; j < kG; j += 2) {
          if constexpr (kNext) fma2(s2[0], u + j, x + j, s2[0]);
          if constexpr (kMode != kPreNorm) {
            fma2(s2[1], q + j, d + j, s2[1]);
            if constexpr (kNext) {
              fma2(s2[2], q + j, u + j, s2[2]);
              fma2(s2[3], q + j, x + j, s2[3]);
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = s2[j][0] + s2[j][1];
      block_sum4(s, scratch[odd]);
    } else {
      s[0] = s[1] = s[2] = s[3] = 0.f;
      for (int w = 0; w < p.windows; ++w) {
        const float4 q = p.sums[w * p.rows + row];
        s[0] += q.x;
        s[1] += q.y;
        s[2] += q.z;
        s[3] += q.w;
      }
      __syncthreads();
    }
    // Every thread is past the previous row's last read of its slot.
    if (threadIdx.x == 0 && slots > 1 && !ring.dead && row >= gridDim.x) {
      const long long next = row + static_cast<long long>(slots - 1) * gridDim.x;
      if (next < p.rows) ring.fetch(slot == 0 ? slots - 1 : slot - 1, next);
    }
    const bool results = !kWide || p.phase == 2;
    if (kWide && !results && threadIdx.x == 0) p.sums[p.window * p.rows + row] = make_float4(s[0], s[1], s[2], s[3]);
    const float cx = kNext ? rx * rx * (s[0] * inv_d) * rx : 0.f;                   // dx = dx' + r(x') u - cx x'
    const float qdx = kNext ? ry * (s[1] + rx * s[2] - cx * s[3]) : ry * s[1];  // sum of s (w + o) yh [act(g)] dx
    const float m = qdx * inv_d * tok;                    // mean(t yh)
    if (results && (!kWide || p.window == 0) && kMode == kSharedGate && p.gate_mode == kGateToken && threadIdx.x == 0) {
      float g = token_value<T>(p, row), slope;
      act_of<false, true, 1>(&g, p.act, &slope);
      const float d = qdx * slope;
      if (p.gate_f32) static_cast<float*>(p.dgate_row)[row] = d;
      else static_cast<T*>(p.dgate_row)[row] = from_float<T>(d);
    }
    const Both r2(rx), neg_cx(-cx), neg_m(-ry * ry * m), ry2(ry);
    T* dx_out = static_cast<T*>(p.dx) + row * pitch;
    T* dy_out = static_cast<T*>(p.dy) + row * pitch;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (!results || (V > 1 && unit(g, 0) >= units)) continue;
      float y[kG], q[kG], a[kG], x[kG], u[kG], dh[kG], d[kG], dg[kG];  // dg: act'(g) first
      read(g, y, q, a, x, u, dh, dg);
      read_dx(g, d);
      if constexpr (kNext) {
#pragma unroll
        for (int j = 0; j < kG; j += 2) {
          const int e = g * kG + j;
          fma2(d + j, u + j, r2, d + j);
          fma2(d + j, x + j, neg_cx, d + j);  // dx
          mul2(x + j, x + j, r2);
          fma2(dv + e, dh + j, x + j, dv + e);
        }
      }
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        const int c = unit(g, k);
        if (V > 1 || c < units) span.write(dx_out, c, d + k * V);
      }
      if constexpr (kMode != kPreNorm) {
#pragma unroll
        for (int j = 0; j < kG; j += 2) {
          const int e = g * kG + j;
          if constexpr (is_full(kMode)) {
            float yh[2];
            mul2(yh, y + j, ry2);
#pragma unroll
            for (int i = 0; i < 2; ++i) dg[j + i] *= pw[e + i] * yh[i] * d[j + i];
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
          if constexpr (is_full(kMode)) {
            if constexpr (kMode == kFullGateF32) {
              float* out = static_cast<float*>(p.dgate_row) + row * pitch;
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
              span.write(static_cast<T*>(p.dgate_row) + row * pitch, c, dg + k * V);
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
  if (kWide && p.phase == 1) return;
  float* part = p.partial + static_cast<long long>(blockIdx.x) * pitch;
  const long long slice = static_cast<long long>(gridDim.x) * pitch;
#pragma unroll
  for (int i = 0; i < kE / V; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (kLayout == kWhole) {
      if (c >= units) continue;
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        if (kMode != kPreNorm) write_unit<float, 4>(part, c * (V / 4) + q, acc + i * V + 4 * q);
        if (kNext) write_unit<float, 4>(part + slice, c * (V / 4) + q, dv + i * V + 4 * q);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (!span.has(c, j)) continue;
        if (kMode != kPreNorm) part[span.col(c, j)] = acc[i * V + j];
        if (kNext) part[slice + span.col(c, j)] = dv[i * V + j];
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ float param1(const void* p, int f32, long long at) {
  return f32 ? __ldg(static_cast<const float*>(p) + at) : as_float(static_cast<const T*>(p)[at]);
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
    float a = param1<T>(p.gate, p.gate_f32, col), slope;
    act_of<false, true, 1>(&a, p.act, &slope);
    store(p.dgate, p.gate_f32, s * (param1<T>(p.w, p.w_f32, col) + p.offset) * slope);
    s *= a;
  }
  store(p.dw, p.w_f32, s);
}

template <typename T, int kLayout, int kMode, bool kWide, bool kNext>
cudaError_t launch_bwd_ring(const NormParams& p, const RingShape& r, int blocks, cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  auto kernel = norm_bwd_ring_kernel<T, kLayout, 16, kMode, kWide, kNext>;
  const cudaError_t e = allow_smem(kernel, done);
  if (e != cudaSuccess) return e;
  kernel<<<blocks, r.threads, r.smem, s>>>(p, r.slots);
  return cudaSuccess;
}

// The ring's backward kernels keep 16 elements a thread (their parameters and
// sums over rows in registers) in at most 512 threads.
constexpr int kMaxRingBwdSpan = 8192;

// The backward pass's layout; rows wider than kMaxRingBwdSpan go in column
// windows (a multiple of 8 wide, so that windows of whole words are whole too).
struct BwdShape {
  RowLayout layout;  // of a window
  int windows, width;
};
BwdShape bwd_shape(int dim, int es, bool words) {
  const RowLayout l = row_layout(dim, es, words);
  if (l.span <= kMaxRingBwdSpan) return {l, 1, dim};
  const int windows = (dim + kMaxRingBwdSpan - 1) / kMaxRingBwdSpan;
  if (windows == 1) return {row_layout(dim, es, false), 1, dim};
  const int width = ((dim + windows - 1) / windows + 7) / 8 * 8;
  return {{l.layout == kWhole ? kWhole : kSingle, width, 1}, windows, width};
}

// Blocks of the backward pass: what is resident at once, so that every block
// adds up as many rows as possible before it leaves its partial sums.
int64_t bwd_most_blocks(int span, int sms) {
  const int threads = threads_for((span + 15) / 16);
  return static_cast<int64_t>(sms) * std::max(1, std::min(16, kBwdThreadsSm / threads));
}

// The workspace: the blocks' partial sums, then the windows' sums of each row.
// Sized for any layout (a narrower span never has fewer blocks).
struct BwdSpace {
  size_t partial, sums;
};
BwdSpace bwd_space(int64_t rows, int dim, int sms) {
  const int windows = bwd_shape(dim, 2, false).windows;
  const int64_t most = std::min<int64_t>(rows, bwd_most_blocks(windows > 1 ? kMaxRingBwdSpan / 2 : dim, sms));
  const size_t partial = (2 * sizeof(float) * static_cast<size_t>(most) * dim + 15) / 16 * 16;
  return {partial, windows > 1 ? sizeof(float4) * static_cast<size_t>(windows) * rows : 0};
}

template <typename T, int kLayout, bool kWide>
cudaError_t bwd_ring_mode(const NormParams& p, const RowLayout& l, int blocks, cudaStream_t s) {
  const int inputs = (p.y ? 1 : 0) + (p.dxn ? 1 : 0) + (p.dh ? 2 : 0);  // x is read where dh is
  const RingShape r = ring_shape(l.span, 16, kBwdThreadsSm, slot_bytes(p, sizeof(T), kLayout, inputs));
  auto go = [&](auto mode) {
    constexpr int kMode = decltype(mode)::value;
    return p.dh ? launch_bwd_ring<T, kLayout, kMode, kWide, true>(p, r, blocks, s)
                : launch_bwd_ring<T, kLayout, kMode, kWide, false>(p, r, blocks, s);
  };
  switch (mode_of(p, sizeof(T))) {
    case kPreNorm: return launch_bwd_ring<T, kLayout, kPreNorm, kWide, true>(p, r, blocks, s);
    case kSharedGate: return go(std::integral_constant<int, kSharedGate>{});
    case kFullGateF32:
      if constexpr (sizeof(T) == 2) return go(std::integral_constant<int, kFullGateF32>{});
      [[fallthrough]];
    default: return go(std::integral_constant<int, kFullGate>{});
  }
}

const void* columns(const void* p, int first, int elem) {
  return p ? static_cast<const char*>(p) + static_cast<int64_t>(first) * elem : nullptr;
}
void* columns(void* p, int first, int elem) { return const_cast<void*>(columns(static_cast<const void*>(p), first, elem)); }

// Every window's sums, then every window's gradients.
template <typename T, int kLayout>
cudaError_t bwd_windows(const NormParams& p, const BwdShape& shape, int blocks, cudaStream_t s) {
  const int es = sizeof(T), ws = p.w_f32 ? 4 : es, gs = p.gate_f32 ? 4 : es;
  for (int phase = 1; phase <= 2; ++phase)
    for (int w = 0; w < shape.windows; ++w) {
      const int first = w * shape.width;
      NormParams q = p;
      q.dim = std::min(shape.width, p.dim - first);
      q.windows = shape.windows;
      q.window = w;
      q.phase = phase;
      q.y = columns(p.y, first, es);
      q.x = columns(p.x, first, es);
      q.dxn = columns(p.dxn, first, es);
      q.dh = columns(p.dh, first, es);
      q.dy = columns(p.dy, first, es);
      q.dx = columns(p.dx, first, es);
      q.w = columns(p.w, first, ws);
      q.v = columns(p.v, first, ws);
      if (p.gate_mode == GMM_GATE_MODE_CHANNEL || p.gate_mode == GMM_GATE_MODE_FULL) q.gate = columns(p.gate, first, gs);
      if (p.gate_mode == GMM_GATE_MODE_FULL) q.dgate_row = columns(p.dgate_row, first, gs);
      q.partial = p.partial + first;
      const cudaError_t e = bwd_ring_mode<T, kLayout, true>(q, shape.layout, blocks, s);
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

template <typename T, int kLayout>
cudaError_t bwd_ring_width(const NormParams& p, const BwdShape& shape, int blocks, cudaStream_t s) {
  if constexpr (kLayout != kShifted)
    if (shape.windows > 1) return bwd_windows<T, kLayout>(p, shape, blocks, s);
  return bwd_ring_mode<T, kLayout, false>(p, shape.layout, blocks, s);
}

template <typename T>
cudaError_t launch_bwd(const NormParams& p, const BwdShape& shape, int blocks, cudaStream_t s) {
  switch (shape.layout.layout) {
    case kWhole: return bwd_ring_width<T, kWhole>(p, shape, blocks, s);
    case kShifted: return bwd_ring_width<T, kShifted>(p, shape, blocks, s);
    default: return bwd_ring_width<T, kSingle>(p, shape, blocks, s);
  }
}

}  // namespace

int norm_bwd_device_error(int* status, bool clear) { return read_row_error(status, clear); }

}  // namespace gmm_sm100

extern "C" {

size_t gmm_sm100_post_norm_backward_workspace_size(int64_t rows, int64_t dim) {
  using namespace gmm_sm100;
  if (rows <= 0 || dim <= 0 || dim > kMaxNormDim) return 0;
  int sms = 0;
  if (current_sm_count(&sms)) return 0;
  const BwdSpace space = bwd_space(rows, static_cast<int>(dim), sms);
  return space.partial + space.sums;
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
  p.pitch = p.dim;
  p.sums = reinterpret_cast<float4*>(static_cast<char*>(workspace) + bwd_space(rows, p.dim, sms).partial);
  const BwdShape shape = bwd_shape(p.dim, static_cast<int>(es), words);
  const int blocks = blocks_for(rows, bwd_most_blocks(shape.layout.span, sms), shape.layout.period);
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
    const cudaError_t e = launch_bwd<T>(p, shape, blocks, s);
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
