// row_vec.cuh -- eight consecutive elements of a row as fp32, for the row
// kernels (quantisation, norms): 16-byte accesses where rows allow them,
// element by element where they do not.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace gmm_sm100 {

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Two fp32 operations in one instruction, each rounded like its own.
__device__ __forceinline__ void fma2(float* d, const float* a, const float* b, const float* c) {
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d[0]), "=f"(d[1])
      : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]), "f"(c[0]), "f"(c[1]));
}
__device__ __forceinline__ void mul2(float* d, const float* a, const float* b) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d[0]), "=f"(d[1])
      : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
}
// A number for both halves.
struct Both {
  float v[2];
  __device__ __forceinline__ explicit Both(float f) : v{f, f} {}
  __device__ __forceinline__ operator const float*() const { return v; }
};

// Eight elements as they lie in memory.
template <typename T>
struct Raw8 {
  uint4 q[sizeof(T) / 2];  // one 16-byte word for 16-bit types, two for fp32
};

__device__ __forceinline__ float2 unpack2(uint32_t u, const __nv_bfloat16*) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
}
__device__ __forceinline__ float2 unpack2(uint32_t u, const __half*) {
  return __half22float2(*reinterpret_cast<__half2*>(&u));
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, const __nv_bfloat16*) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, const __half*) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ void unpack(const Raw8<T>& r, float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = unpack2(w[i], static_cast<const T*>(nullptr));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i] = __uint_as_float(r.q[i].x);
      f[4 * i + 1] = __uint_as_float(r.q[i].y);
      f[4 * i + 2] = __uint_as_float(r.q[i].z);
      f[4 * i + 3] = __uint_as_float(r.q[i].w);
    }
  }
}

template <typename T>
__device__ __forceinline__ Raw8<T> pack(const float (&f)[8]) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 2) {
    const T* t = nullptr;
    r.q[0] = make_uint4(pack_pair(f[0], f[1], t), pack_pair(f[2], f[3], t), pack_pair(f[4], f[5], t),
                        pack_pair(f[6], f[7], t));
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      r.q[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                          __float_as_uint(f[4 * i + 3]));
  }
  return r;
}

// Elements [col, col + 8) of a row of `dim`; those past the end read as 0.
template <typename T, bool kVec>
__device__ __forceinline__ Raw8<T> load8(const T* row, int col, int dim) {
  if constexpr (kVec) {  // dim is a multiple of 8 and every row 16-byte aligned
    Raw8<T> r;
    const uint4* p = reinterpret_cast<const uint4*>(row + col);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.q[i] = col < dim ? p[i] : make_uint4(0, 0, 0, 0);
    return r;
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = col + i < dim ? as_float(row[col + i]) : 0.f;
    return pack<T>(f);  // exact: the values came from T
  }
}

}  // namespace gmm_sm100
