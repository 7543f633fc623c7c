// gmm_stream_kernel.cuh -- 8-bit grouped products of a few rows an expert
// (decode): the weights pass once from HBM through registers into mma.sync.
//
// With m <= 16 rows an expert the product is bound by reading B[e] (each byte
// meets m MACs), and for a single token by latency: a tcgen05 tile needs its
// operands staged in shared memory, an accumulator in tensor memory and a
// 256-column tile an SM, which leaves most SMs without work.  Here a task is 16
// output columns (16 gate and the 16 matching up columns for SwiGLU) of one
// block of up to 16 rows, small enough to spread over every warp of the GPU,
// and further over the contraction:
//
//   * mma.sync m16n8k32: its 16 rows are output columns (rows of B[e]), its 8
//     columns token rows; two of them cover 16 tokens.  The contraction's order
//     is free as long as both operands agree, so a lane takes 16 neighbouring
//     bytes of its row (four lanes 64 bytes) and feeds them to two MMAs as they
//     are: no shared memory, no transposition, on either side.
//   * a warp issues the loads of four 64-byte steps before it uses the first;
//     the token rows come from L1 / L2.
//   * if there are fewer tasks than warps, 2, 4 or 8 warps of a block share a
//     task, each a part of the contraction, and add their 32-bit sums (exact
//     in any order) in shared memory.
//   * persistent blocks walk the task list in order, so concurrent warps read
//     neighbouring rows of B.
#pragma once

constexpr int kStreamRows = 16;     // token rows of a task
constexpr int kStreamCols = 16;     // output columns of a task
constexpr int kStreamWarps = 8;
constexpr int kStreamBlocksSm = 2;  // resident blocks an SM
constexpr int kStreamStep = 64;     // bytes of a row per step: 16 a lane

// Two 16 x 8 x 32 products.  a: 16 bytes of rows lane / 4 and lane / 4 + 8 of the
// column operand, b: 16 bytes of token row lane / 4.
__device__ __forceinline__ void stream_mma(int (&c)[4], const uint4& a0, const uint4& a8, const uint4& b) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0.x), "r"(a8.x), "r"(a0.y), "r"(a8.y), "r"(b.x), "r"(b.y));
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0.z), "r"(a8.z), "r"(a0.w), "r"(a8.w), "r"(b.z), "r"(b.w));
}

// Weights are read once: they do not displace the token rows from L1.
__device__ __forceinline__ uint4 stream_load(const int8_t* p, bool in) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (in)
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}

template <int kTableInts>
struct StreamParams : GmmParamsT<kTableInts> {
  const int8_t* a;
  const int8_t* b;
  long long k;       // bytes of a row of A and B
  long long b_cols;  // rows of B[e] (2 * dim_out for SwiGLU)
};

// One block of 16 output columns (kParts = 1), or of gate and of up columns (2).
template <int kParts, typename OutT, int kTableInts>
__global__ void __launch_bounds__(kStreamWarps * 32, kStreamBlocksSm)
    gmm_stream_kernel(const __grid_constant__ StreamParams<kTableInts> p) {
  constexpr int kAhead = 4 / kParts;  // steps whose weights are loaded together
  __shared__ __align__(16) uint8_t table_area[kDevTableBytes];
  __shared__ int sums[kStreamWarps][kParts * 8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g8 = lane >> 2, quad = lane & 3;

  int num_groups = p.num_groups;
  const int32_t* tab = p.ext_table ? p.ext_table : p.inline_table;
  if (p.dev_bs) {
    int32_t* dtab = reinterpret_cast<int32_t*>(table_area);
    int32_t* meta = dtab + 3 * kMaxDevExperts + 2;
    build_device_table(p, dtab, meta, reinterpret_cast<long long*>(meta + 4));
    num_groups = meta[0];
    if (threadIdx.x == 0 && meta[2] != 0) atomicCAS(&g_device_error, 0, meta[2]);
    tab = dtab;
  }
  const TableView tv = make_table_view(p, tab, num_groups);
  const long long tasks = static_cast<long long>(tv.tile_off[num_groups]) * p.n_tiles;

  // Warps that share a task: as many as keep every warp of the grid busy once.
  const long long warps = static_cast<long long>(gridDim.x) * kStreamWarps;
  const int steps = static_cast<int>((p.k + kStreamStep - 1) / kStreamStep);
  int split = 1;
  while (split < kStreamWarps && tasks * split * 2 <= warps && steps >= split * 4) split *= 2;
  const int part = warp & (split - 1);
  const int first = static_cast<int>(static_cast<long long>(steps) * part / split);
  const int last = static_cast<int>(static_cast<long long>(steps) * (part + 1) / split);

  int g = 0;
  for (long long task = blockIdx.x * static_cast<long long>(kStreamWarps / split) + warp / split; task < tasks;
       task += gridDim.x * static_cast<long long>(kStreamWarps / split)) {
    while (task >= static_cast<long long>(tv.tile_off[g + 1]) * p.n_tiles) ++g;
    const long long local = task - static_cast<long long>(tv.tile_off[g]) * p.n_tiles;
    const int m = static_cast<int>(local / p.n_tiles), col0 = static_cast<int>(local % p.n_tiles) * kStreamCols;
    const int row0 = tv.row_off[g] + m * kStreamRows;
    const int rows = min(kStreamRows, tv.row_off[g + 1] - row0);
    const long long expert = tv.expert[g];
    // rows of B past the last column and token rows past the block are read
    // from the last one: their sums are not stored
    const int8_t *w0[kParts], *w8[kParts];
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      const long long base = expert * p.b_cols + (j ? p.act_cols : 0);
      w0[j] = p.b + (base + min(col0 + g8, p.dim_out - 1)) * p.k + quad * 16;
      w8[j] = p.b + (base + min(col0 + 8 + g8, p.dim_out - 1)) * p.k + quad * 16;
    }
    const int8_t* t0 = p.a + static_cast<long long>(row0 + min(g8, rows - 1)) * p.k + quad * 16;
    const int8_t* t8 = p.a + static_cast<long long>(row0 + min(g8 + 8, rows - 1)) * p.k + quad * 16;
    const bool two = rows > 8;

    int c[kParts][2][4] = {};
    for (int s0 = first; s0 < last; s0 += kAhead) {
      uint4 a0[kAhead][kParts], a8[kAhead][kParts];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const long long at = static_cast<long long>(s0 + i) * kStreamStep;
        const bool in = s0 + i < last && at + quad * 16 < p.k;
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          a0[i][j] = stream_load(w0[j] + at, in);
          a8[i][j] = stream_load(w8[j] + at, in);
        }
      }
      uint4 b0[kAhead], b8[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const long long at = static_cast<long long>(s0 + i) * kStreamStep;
        const bool in = s0 + i < last && at + quad * 16 < p.k;
        b0[i] = b8[i] = make_uint4(0, 0, 0, 0);
        if (in) b0[i] = __ldg(reinterpret_cast<const uint4*>(t0 + at));
        if (in && two) b8[i] = __ldg(reinterpret_cast<const uint4*>(t8 + at));
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          stream_mma(c[j][0], a0[i][j], a8[i][j], b0[i]);
          if (two) stream_mma(c[j][1], a0[i][j], a8[i][j], b8[i]);
        }
    }

    if (split > 1) {  // the task's first warp adds the others' sums
      const int id = 1 + warp / split;
      if (part != 0) {
#pragma unroll
        for (int j = 0; j < kParts; ++j)
#pragma unroll
          for (int q = 0; q < 8; ++q) sums[warp][j * 8 + q][lane] = c[j][q >> 2][q & 3];
      }
      asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(split * 32) : "memory");
      if (part == 0)
        for (int w = 1; w < split; ++w)
#pragma unroll
          for (int j = 0; j < kParts; ++j)
#pragma unroll
            for (int q = 0; q < 8; ++q) c[j][q >> 2][q & 3] += sums[warp + w][j * 8 + q][lane];
      asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(split * 32) : "memory");  // before the next task's sums
      if (part != 0) continue;
    }

    // lane: columns col0 + g8 (+ 8), token rows 2 quad, 2 quad + 1 (+ 8)
    float sb[kParts][2];
#pragma unroll
    for (int j = 0; j < kParts; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        sb[j][h] = __ldg(p.scale_b + expert * p.scale_cols + (j ? p.act_cols : 0) + min(col0 + g8 + 8 * h, p.dim_out - 1));
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = 2 * quad + (t & 1) + 8 * (t >> 1);
      if (row >= rows) continue;
      const float sa = __ldg(p.scale_a + row0 + row);
      OutT* out = static_cast<OutT*>(p.d) + static_cast<long long>(row0 + row) * p.ldd + col0 + g8;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (col0 + g8 + 8 * h >= p.dim_out) continue;
        const int q = (t & 1) + 2 * h;
        // the same operations, in the same order, as the tiled kernels' epilogue
        float v = __int2float_rn(c[0][t >> 1][q]) * sa * sb[0][h];
        if constexpr (kParts == 2) v = silu_mul_fast(v, __int2float_rn(c[1][t >> 1][q]) * sa * sb[1][h]);
        if constexpr (std::is_same<OutT, float>::value) out[8 * h] = v;
        else out[8 * h] = to_out<OutT>(v);
      }
    }
  }
}
