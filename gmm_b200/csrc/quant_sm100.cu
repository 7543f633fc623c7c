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
// by a gather would read and write the codes once more.

#include <algorithm>
#include <cstdio>

#include "gmm_sm100.h"
#include "row_vec.cuh"
#include "status.h"

namespace gmm_sm100 {
namespace {

constexpr int kMaxDim = 65536;

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
// half (1 in 2000) divide.  A division per element made the kernel issue-bound
// (77 us for 16384 x 4096 bf16 into two places).
// `divide`: 1 / scale may not be finite.
__device__ __forceinline__ uint2 quantize8(const float (&f)[8], float scale, float inv, bool divide) {
  constexpr float kMagic = 12582912.f;
  uint32_t u[8];
  float half = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float r = fmaf(f[j], inv, kMagic);
    u[j] = __float_as_uint(r);
    half = fmaxf(half, fabsf(fmaf(f[j], inv, kMagic - r)));
  }
  if (divide || half > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = max(-127, min(127, __float2int_rn(__fdiv_rn(f[j], scale))));
  }
  return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}

// One block per row; thread t holds the 8-element chunks t, t + blockDim.x, ...
template <typename T, int kChunks, bool kVec>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const T* __restrict__ x, int dim, int dim_padded,
                                                             const int32_t* __restrict__ dst, int k,
                                                             long long out_rows, int8_t* __restrict__ q,
                                                             float* __restrict__ scales) {
  __shared__ uint32_t warp_max[32];
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 31;
  const T* src = x + row * dim;
  // lane s knows place s; a place outside the result is -1
  long long place = -1;
  if (lane < k) {
    place = dst ? dst[row * k + lane] : row;
    if (place >= out_rows) place = -1;
  }
  Raw8<T> raw[kChunks];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) raw[i] = load8<T, kVec>(src, (threadIdx.x + i * blockDim.x) * 8, dim);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) top = max(top, top_bits(raw[i]));
  top = __reduce_max_sync(0xffffffffu, top);
  if (blockDim.x > 32) {
    if (lane == 0) warp_max[threadIdx.x >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < (blockDim.x >> 5) ? warp_max[lane] : 0u);
  }
  const bool finite = top < 0x7f800000u;
  const float scale = finite ? __fdiv_rn(__uint_as_float(top), 127.f) : __uint_as_float(0x7fffffffu);
  const bool tiny = scale < 0x1p-126f;
  const float inv = __frcp_rn(scale);
  const bool codes = finite && scale > 0.f;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int col = (threadIdx.x + i * blockDim.x) * 8;
    uint2 w = make_uint2(0, 0);
    if (codes) {
      float f[8];
      unpack(raw[i], f);
      w = quantize8(f, scale, inv, tiny);
    }
    for (int s = 0; s < k; ++s) {
      const long long pos = __shfl_sync(0xffffffffu, place, s);
      if (pos >= 0 && col < dim_padded) *reinterpret_cast<uint2*>(q + pos * dim_padded + col) = w;
    }
  }
  if (threadIdx.x < k && place >= 0) scales[place] = scale;
}

template <typename T, bool kVec>
void launch(const void* x, long long rows, int dim, int dim_padded, const int32_t* dst, int k, long long out_rows,
            int8_t* q, float* scales, cudaStream_t s) {
  const int chunks = dim_padded / 8;
  const T* xt = static_cast<const T*>(x);
  const unsigned grid = static_cast<unsigned>(rows);
  auto threads = [&](int per) { return std::max(32, (chunks + 32 * per - 1) / (32 * per) * 32); };
  if (chunks <= 256)
    quantize_rows_kernel<T, 1, kVec><<<grid, threads(1), 0, s>>>(xt, dim, dim_padded, dst, k, out_rows, q, scales);
  else if (chunks <= 2048)
    quantize_rows_kernel<T, 2, kVec><<<grid, threads(2), 0, s>>>(xt, dim, dim_padded, dst, k, out_rows, q, scales);
  else
    quantize_rows_kernel<T, 8, kVec><<<grid, threads(8), 0, s>>>(xt, dim, dim_padded, dst, k, out_rows, q, scales);
}

}  // namespace
}  // namespace gmm_sm100

extern "C" int gmm_sm100_quantize_rows(const void* x, int dtype, int64_t num_rows, int64_t dim,
                                       const int32_t* dst_pos, int k, int64_t out_rows, int8_t* q, float* scale,
                                       void* stream) {
  using namespace gmm_sm100;
  if (num_rows < 0 || dim < 0 || out_rows < 0) return set_error(GMM_ERR_INVALID_ARGUMENT, "negative size");
  if (k < 1 || k > 32 || (!dst_pos && k != 1))
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
  const bool vec = D % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
  auto go = [&](auto t) {
    using T = decltype(t);
    vec ? launch<T, true>(x, num_rows, D, P, dst_pos, k, out_rows, q, scale, s)
        : launch<T, false>(x, num_rows, D, P, dst_pos, k, out_rows, q, scale, s);
  };
  if (dtype == GMM_DTYPE_F32) go(float{});
  else if (dtype == GMM_DTYPE_BF16) go(__nv_bfloat16{});
  else go(__half{});
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(GMM_ERR_CUDA, cudaGetErrorString(e));
  return GMM_OK;
}
