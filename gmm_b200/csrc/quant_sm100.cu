// quant_sm100.cu -- rows to signed 8-bit codes with one scale each, written to
// every place a row is wanted: the activations of the 8-bit grouped product,
// quantised straight into expert order.  No reference counterpart (the
// reference's grouped GEMM has no 8-bit form).
//
//   scale = max|x| / 127,   code = rint(x / scale) in [-127, 127]
//
// both divisions correctly rounded in fp32.  A row of zeros (or one so small
// that its scale rounds to 0) has scale 0 and codes 0; a row that holds an
// infinity or a NaN has scale NaN and codes 0, so that everything computed
// from it is NaN.
//
// Bound by HBM: a row is read once (one block holds it in registers between
// its maximum and its codes) and written k times, where a quantiser followed
// by a gather would read and write the codes once more.  Rows come through a
// shared-memory ring and leave as one bulk store a place.

#include <algorithm>

#include "gmm_sm100.h"
#include "row_ring.cuh"
#include "row_vec.cuh"
#include "status.h"

namespace gmm_sm100 {
namespace {

constexpr int kMaxDim = 65536;
constexpr int kMaxRingDim = 16384;  // wider rows go through quantize_rows_kernel

// Largest |x| of eight elements, as its fp32 bits: ordered like the values,
// with NaN above infinity.  16-bit types compare two at a time.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Raw8<T>& r) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t m = __vmaxu2(__vmaxu2(r.q[0].x & 0x7fff7fffu, r.q[0].y & 0x7fff7fffu),
                                __vmaxu2(r.q[0].z & 0x7fff7fffu, r.q[0].w & 0x7fff7fffu));
    const float2 f = unpack2(m, static_cast<const T*>(nullptr));
    return max(__float_as_uint(f.x), __float_as_uint(f.y));
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      m = max(max(max(m, r.q[i].x & 0x7fffffffu), r.q[i].y & 0x7fffffffu),
              max(r.q[i].z & 0x7fffffffu, r.q[i].w & 0x7fffffffu));
    return m;
  }
}

// rint(x / scale) of eight elements, two's complement bytes.
//
// x * inv, inv = 1 / scale rounded, lies within 2^-24 of x / scale (relative,
// and one more 2^-24 for the division that defines the code), so both round
// to the same integer unless the product comes within 3 * 2^-24 * 127.5 <
// 2^-15 of a half.  Adding 1.5 * 2^23 rounds the exact product to an integer
// and leaves it in the low bits; only chunks with a product that near to a
// half (1 in 2000) divide.  16384 x 4096 bf16 into two places on one B200: 77 us
// with a division per element, 49 now (5.45 TB/s, 0.84 of the copy bandwidth).
// `divide`: 1 / scale may not be finite.
__device__ __forceinline__ uint2 quantize8(const float (&f)[8], float scale, float inv, bool divide) {
  const Both magic(12582912.f), inv2(inv), minus(-1.f);
  uint32_t u[8];
  float half = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    float r[2], n[2];
    fma2(r, f + j, inv2, magic);
    u[j] = __float_as_uint(r[0]);
    u[j + 1] = __float_as_uint(r[1]);
    fma2(n, r, minus, magic);  // minus the integer
    fma2(n, f + j, inv2, n);
    half = fmaxf(half, fmaxf(fabsf(n[0]), fabsf(n[1])));
  }
  if (divide || half > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = max(-127, min(127, __float2int_rn(__fdiv_rn(f[j], scale))));
  }
  return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}

struct QuantParams {
  const void* x;
  const int32_t* dst;
  int8_t* q;
  float* scales;
  long long rows, out_rows;
  int dim, dim_padded, k;
};

// Place `s` of a row for lane s of a warp; -1: none, or outside the result.
__device__ __forceinline__ long long place_of(const QuantParams& p, long long row, int lane) {
  if (lane >= p.k || row >= p.rows) return -1;
  const long long place = p.dst ? p.dst[row * p.k + lane] : row;
  return place < p.out_rows ? place : -1;
}

// What a row's codes are made with, from the largest |x| of each thread.
struct RowScale {
  float scale, inv;
  bool codes, divide;
};
__device__ __forceinline__ RowScale row_scale(uint32_t top, uint32_t* warp_max) {
  const int lane = threadIdx.x & 31;
  top = __reduce_max_sync(0xffffffffu, top);
  if (blockDim.x > 32) {
    if (lane == 0) warp_max[threadIdx.x >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < (blockDim.x >> 5) ? warp_max[lane] : 0u);
  }
  RowScale r;
  const bool finite = top < 0x7f800000u;
  r.scale = finite ? __fdiv_rn(__uint_as_float(top), 127.f) : __uint_as_float(0x7fffffffu);
  r.inv = __frcp_rn(r.scale);
  r.divide = r.scale < 0x1p-126f;  // the reciprocal may not be finite
  r.codes = finite && r.scale > 0.f;
  return r;
}

// Eight elements of a row in the ring; kVec: on 16-byte boundaries.
template <typename T, bool kVec>
__device__ __forceinline__ Raw8<T> ring8(const uint8_t* row, int col, int dim) {
  return load8<T, kVec>(reinterpret_cast<const T*>(row), col, dim);
}

// Persistent blocks over the ring.  A row's codes are staged in shared memory
// (two buffers) and lane s of warp 0 stores them to place s.
constexpr int kRingChunks = 4;  // 8-element chunks of a row a thread holds

template <typename T, bool kVec>
__global__ void __launch_bounds__(512, 2) quantize_ring_kernel(const QuantParams p, int slots) {
  constexpr int kChunks = kRingChunks;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t warp_max[2][32];
  uint8_t* staged = smem;  // 2 rows of codes
  RowRing<1, kVec> ring;
  ring.input(0, p.x, sizeof(T), p.dim, p.dim);
  ring.start(smem + 2 * p.dim_padded, slots, p.rows);
  __syncthreads();
  const int lane = threadIdx.x & 31;
  long long place = threadIdx.x < 32 ? place_of(p, blockIdx.x, lane) : -1;
  int slot = 0, odd = 0;
  uint32_t phase = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    ring.wait(slot, phase, row);
    const uint8_t* in = smem + 2 * p.dim_padded + ring.at(slot, 0, row);
    Raw8<T> raw[kChunks];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      raw[i] = ring8<T, kVec>(in, (threadIdx.x + i * blockDim.x) * 8, p.dim);
      top = max(top, top_bits(raw[i]));
    }
    // the stores that read this staging buffer two rows ago are done with it
    if (threadIdx.x < 32) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    const RowScale rs = row_scale(top, warp_max[odd]);
    if (blockDim.x == 32) __syncwarp();
    if (threadIdx.x == 0 && !ring.dead) {  // every thread holds its part of the row
      const long long next = row + static_cast<long long>(slots) * gridDim.x;
      if (next < p.rows) ring.fetch(slot, next);
    }
    uint8_t* codes = staged + odd * p.dim_padded;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      uint2 w = make_uint2(0, 0);
      if (rs.codes) {
        float f[8];
        unpack(raw[i], f);
        w = quantize8(f, rs.scale, rs.inv, rs.divide);
      }
      if (col < p.dim_padded) *reinterpret_cast<uint2*>(codes + col) = w;
    }
    fence_proxy_async_smem();
    __syncthreads();
    if (threadIdx.x < 32) {
      if (place >= 0) {
        p.scales[place] = rs.scale;
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p.q + place * p.dim_padded),
                     "r"(smem_u32(codes)), "r"(p.dim_padded)
                     : "memory");
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      place = place_of(p, row + gridDim.x, lane);
    }
    if (++slot == slots) {
      slot = 0;
      phase ^= 1;
    }
    odd ^= 1;
  }
  if (threadIdx.x < 32) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// Rows too wide for the ring, one block each; thread t holds the 8-element
// chunks t, t + blockDim.x, ...
template <typename T, int kChunks, bool kVec>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const QuantParams p) {
  __shared__ uint32_t warp_max[32];
  const long long row = blockIdx.x;
  const T* src = static_cast<const T*>(p.x) + row * p.dim;
  const long long place = place_of(p, row, threadIdx.x & 31);
  Raw8<T> raw[kChunks];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) raw[i] = load8<T, kVec>(src, (threadIdx.x + i * blockDim.x) * 8, p.dim);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) top = max(top, top_bits(raw[i]));
  const RowScale rs = row_scale(top, warp_max);
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int col = (threadIdx.x + i * blockDim.x) * 8;
    uint2 w = make_uint2(0, 0);
    if (rs.codes) {
      float f[8];
      unpack(raw[i], f);
      w = quantize8(f, rs.scale, rs.inv, rs.divide);
    }
    for (int s = 0; s < p.k; ++s) {
      const long long pos = __shfl_sync(0xffffffffu, place, s);
      if (pos >= 0 && col < p.dim_padded) *reinterpret_cast<uint2*>(p.q + pos * p.dim_padded + col) = w;
    }
  }
  if (threadIdx.x < p.k && place >= 0) p.scales[place] = rs.scale;
}

// Blocks of the ring kernel on one SM, their row slots and dynamic shared
// memory: as many blocks as threads and memory allow with two slots each, and
// up to four slots in what is left, within what one block may have (two fit at
// every width).  Besides its dynamic part a block takes its static scratch and
// the system's, 1536 bytes.
struct QuantShape {
  int threads, resident, slots, smem;
};
QuantShape quant_shape(int dim, int dim_padded, int es, bool vec) {
  QuantShape r;
  r.threads = threads_for((dim_padded / 8 + kRingChunks - 1) / kRingChunks);
  const int slot = static_cast<int>(row_pitch(dim * es, vec)) + 8, staged = 2 * dim_padded, extra = 1536;
  r.resident = std::max(1, std::min({16, 1024 / r.threads, kRingBytes / (staged + extra + 2 * slot)}));
  const int most = std::min(kRingBytes / r.resident - extra, kRingBlockBytes);
  r.slots = std::max(2, std::min(4, (most - staged) / slot));
  r.smem = staged + r.slots * slot;
  return r;
}

template <typename T, bool kVec>
cudaError_t launch(const QuantParams& p, int sms, cudaStream_t s) {
  const int chunks = p.dim_padded / 8;
  if (p.dim <= kMaxRingDim && p.dim > 0) {
    const QuantShape r = quant_shape(p.dim, p.dim_padded, sizeof(T), kVec);
    static std::atomic<unsigned long long> done{0};
    auto kernel = quantize_ring_kernel<T, kVec>;
    const cudaError_t e = allow_smem(kernel, done);
    if (e != cudaSuccess) return e;
    const int grid = static_cast<int>(std::min<long long>(p.rows, static_cast<long long>(sms) * r.resident));
    kernel<<<grid, r.threads, r.smem, s>>>(p, r.slots);
    return cudaSuccess;
  }
  const unsigned grid = static_cast<unsigned>(p.rows);
  quantize_rows_kernel<T, 8, kVec><<<grid, threads_for((chunks + 7) / 8), 0, s>>>(p);
  return cudaSuccess;
}

}  // namespace

int quant_device_error(int* status, bool clear) { return read_row_error(status, clear); }

}  // namespace gmm_sm100

extern "C" int gmm_sm100_quantize_rows(const void* x, int dtype, int64_t num_rows, int64_t dim,
                                       const int32_t* dst_pos, int k, int64_t out_rows, int8_t* q, float* scale,
                                       void* stream) {
  using namespace gmm_sm100;
  if (num_rows < 0 || dim < 0 || out_rows < 0) return set_error(GMM_ERR_INVALID_ARGUMENT, "negative size");
  if (k < 1 || k > 32 || (!dst_pos && k != 1 && num_rows > 0))
    return set_error(GMM_ERR_INVALID_ARGUMENT, "need 1 <= k <= 32, and k = 1 without dst_pos");
  if (dtype != GMM_DTYPE_F32 && dtype != GMM_DTYPE_BF16 && dtype != GMM_DTYPE_F16)
    return set_error(GMM_ERR_DTYPE, "rows must be fp32, bf16 or fp16");
  if (!dst_pos && out_rows < num_rows)
    return set_error(GMM_ERR_INVALID_ARGUMENT, "without dst_pos the output holds at least num_rows rows");
  if (dim > kMaxDim || num_rows > INT32_MAX || out_rows > INT32_MAX)
    return set_error(GMM_ERR_TOO_LARGE, "quantize_rows takes dim <= 65536 and fewer than 2^31 rows");
  if (num_rows == 0 || out_rows == 0) return GMM_OK;
  if ((!x && dim > 0) || (!q && dim > 0) || !scale) return set_error(GMM_ERR_INVALID_ARGUMENT, "null pointer");
  const int es = dtype == GMM_DTYPE_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) % es) || (reinterpret_cast<uintptr_t>(q) & 15u) ||
      (reinterpret_cast<uintptr_t>(scale) & 3u) || (reinterpret_cast<uintptr_t>(dst_pos) & 3u))
    return set_error(GMM_ERR_ALIGNMENT, "x, scale or dst_pos is misaligned, or q not 16-byte aligned");
  int sms = 0;
  if (int rc = current_sm_count(&sms)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int D = static_cast<int>(dim), P = (D + 15) / 16 * 16;
  const QuantParams p{x, dst_pos, q, scale, num_rows, out_rows, D, P, k};
  const bool vec = D % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
  auto go = [&](auto t) {
    using T = decltype(t);
    const cudaError_t e = vec ? launch<T, true>(p, sms, s) : launch<T, false>(p, sms, s);
    return e == cudaSuccess ? cudaGetLastError() : e;
  };
  const cudaError_t e = dtype == GMM_DTYPE_F32    ? go(float{})
                        : dtype == GMM_DTYPE_BF16 ? go(__nv_bfloat16{})
                                                  : go(__half{});
  return e == cudaSuccess ? GMM_OK : set_error(GMM_ERR_CUDA, cudaGetErrorString(e));
}
