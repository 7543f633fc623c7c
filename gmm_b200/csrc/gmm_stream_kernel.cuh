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
//   * every lane copies the bytes it will use itself into its own part of
//     shared memory (cp.async), steps of 128 bytes ahead and on into the next
//     task: more bytes in flight than registers could hold, and nothing to
//     synchronise.  The token rows come the same way, through L1.
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
constexpr int kStreamStep = 128;    // bytes of a row per step: twice 16 a lane

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

// 16 bytes from global to this lane's part of shared memory; zeros where `in`
// is false.  Weights are read once and pass L1 by; token rows are shared by
// the warps of a block.
__device__ __forceinline__ void stream_copy(uint32_t to, const int8_t* from, bool in, bool keep) {
  const int bytes = in ? 16 : 0;
  if (keep)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

template <int kTableInts>
struct StreamParams : GmmParamsT<kTableInts> {
  const int8_t* a;
  const int8_t* b;
  long long k;       // bytes of a row of A and B
  long long b_cols;  // rows of B[e] (2 * dim_out for SwiGLU)
};

// Where a task's operands start, for this lane.
template <int kParts>
struct StreamTask {
  const int8_t *w0[kParts], *w8[kParts];  // rows lane / 4 and lane / 4 + 8 of the column block(s)
  const int8_t *t0, *t8;                  // token rows lane / 4 and lane / 4 + 8
  long long expert;
  int col0, row0, rows;                   // tasks are below 2^31 (checked on the host)

  template <typename P>
  __device__ __forceinline__ void find(const P& p, const TableView& tv, int task, int& g) {
    const int g8 = (threadIdx.x & 31) >> 2, quad = threadIdx.x & 3;
    while (task >= tv.tile_off[g + 1] * p.n_tiles) ++g;
    const unsigned local = task - tv.tile_off[g] * p.n_tiles, n = p.n_tiles;
    const int m = local < n ? 0 : static_cast<int>(local / n);
    col0 = (static_cast<int>(local) - m * p.n_tiles) * kStreamCols;
    row0 = tv.row_off[g] + m * kStreamRows;
    rows = min(kStreamRows, tv.row_off[g + 1] - row0);
    expert = tv.expert[g];
    // rows of B past the last column and token rows past the block are read
    // from the last one: their sums are not stored
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      const long long base = expert * p.b_cols + (j ? p.act_cols : 0);
      w0[j] = p.b + (base + min(col0 + g8, p.dim_out - 1)) * p.k + quad * 16;
      w8[j] = p.b + (base + min(col0 + 8 + g8, p.dim_out - 1)) * p.k + quad * 16;
    }
    t0 = p.a + static_cast<long long>(row0 + min(g8, rows - 1)) * p.k + quad * 16;
    t8 = p.a + static_cast<long long>(row0 + min(g8 + 8, rows - 1)) * p.k + quad * 16;
  }
};

template <int kParts>
struct StreamCfg {
  static constexpr int kLoads = 2 * (2 * kParts + 2);     // 16-byte words a lane takes per step
  static constexpr int kDepth = kParts == 1 ? 3 : 2;      // steps a warp's ring holds
  static constexpr int kRingBytes = kStreamWarps * kDepth * kLoads * 32 * 16;
  static constexpr int kSmemBytes = kRingBytes + kDevTableBytes;
  static_assert(kParts * 8 * 4 <= kDepth * kLoads * 16, "a lane's sums fit into its ring");
  static_assert(kStreamBlocksSm * (kSmemBytes + 1024) <= 228 * 1024, "shared memory budget");
};

// One block of 16 output columns (kParts = 1), or of gate and of up columns (2).
template <int kParts, typename OutT, int kTableInts>
__global__ void __launch_bounds__(kStreamWarps * 32, kStreamBlocksSm)
    gmm_stream_kernel(const __grid_constant__ StreamParams<kTableInts> p) {
  using C = StreamCfg<kParts>;
  extern __shared__ __align__(128) uint8_t stream_smem[];
  uint8_t* table_area = stream_smem + C::kRingBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g8 = lane >> 2, quad = lane & 3;
  // this lane's words: [step of the ring][load][lane]
  uint8_t* ring = stream_smem + warp * (C::kDepth * C::kLoads * 512) + lane * 16;
  const uint32_t ring_at = smem_u32(ring);

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
  const int tasks = tv.tile_off[num_groups] * p.n_tiles;

  // Warps that share a task: as many as keep every warp of the grid busy once.
  const int warps = gridDim.x * kStreamWarps;
  const int steps = static_cast<int>((p.k + kStreamStep - 1) / kStreamStep);
  int split = 1;
  while (split < kStreamWarps && tasks * 2 <= warps / split && steps >= split * 2) split *= 2;
  const int part = warp & (split - 1);
  const int first = steps * part / split;
  const int last = steps * (part + 1) / split;
  const int stride = gridDim.x * (kStreamWarps / split);
  const int task0 = blockIdx.x * (kStreamWarps / split) + warp / split;

  // The copying side runs ahead of the multiplying side, on into later tasks.
  // Its pointers move along the rows; `left` counts the bytes from the lane's
  // first word of the step to the rows' end.
  StreamTask<kParts> from;
  int from_g = 0, from_step = first, from_slot = 0, from_task = task0;
  int left = 0;
  auto start_task = [&]() {
    if (from_task >= tasks) return;
    from.find(p, tv, from_task, from_g);
    const int at = first * kStreamStep;
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      from.w0[j] += at;
      from.w8[j] += at;
    }
    from.t0 += at;
    from.t8 += at;
    left = static_cast<int>(p.k) - at - quad * 16;
  };
  start_task();
  auto copy_step = [&]() {
    if (from_task < tasks) {
      const uint32_t to = ring_at + from_slot * (C::kLoads * 512);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = left > 64 * h;
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          stream_copy(to + (h * (C::kLoads / 2) + 2 * j) * 512, from.w0[j] + 64 * h, in, false);
          stream_copy(to + (h * (C::kLoads / 2) + 2 * j + 1) * 512, from.w8[j] + 64 * h, in, false);
        }
        stream_copy(to + (h * (C::kLoads / 2) + 2 * kParts) * 512, from.t0 + 64 * h, in, true);
        if (from.rows > 8) stream_copy(to + (h * (C::kLoads / 2) + 2 * kParts + 1) * 512, from.t8 + 64 * h, in, true);
      }
      if (++from_step == last) {
        from_step = first;
        from_task += stride;
        start_task();
      } else {
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          from.w0[j] += kStreamStep;
          from.w8[j] += kStreamStep;
        }
        from.t0 += kStreamStep;
        from.t8 += kStreamStep;
        left -= kStreamStep;
      }
    }
    if (++from_slot == C::kDepth) from_slot = 0;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < C::kDepth - 1; ++i) copy_step();

  int g = 0, slot = 0;
  for (int task = task0; task < tasks; task += stride) {
    StreamTask<kParts> t;
    t.find(p, tv, task, g);
    // lane: columns col0 + g8 (+ 8), token rows 2 quad, 2 quad + 1 (+ 8)
    float sb[kParts][2], sa[4];
#pragma unroll
    for (int j = 0; j < kParts; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        sb[j][h] = __ldg(p.scale_b + t.expert * p.scale_cols + (j ? p.act_cols : 0) +
                         min(t.col0 + g8 + 8 * h, p.dim_out - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sa[i] = __ldg(p.scale_a + t.row0 + min(2 * quad + (i & 1) + 8 * (i >> 1), t.rows - 1));
    const bool two = t.rows > 8;

    int c[kParts][2][4] = {};
    for (int s = first; s < last; ++s) {
      copy_step();
      asm volatile("cp.async.wait_group %0;" ::"n"(C::kDepth - 1) : "memory");
      const uint4* words = reinterpret_cast<const uint4*>(ring + slot * (C::kLoads * 512));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4* half = words + h * (C::kLoads / 2) * 32;
        const uint4 b0 = half[(2 * kParts) * 32], b8 = half[(2 * kParts + 1) * 32];
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          const uint4 a0 = half[(2 * j) * 32], a8 = half[(2 * j + 1) * 32];
          stream_mma(c[j][0], a0, a8, b0);
          if (two) stream_mma(c[j][1], a0, a8, b8);
        }
      }
      if (++slot == C::kDepth) slot = 0;
    }

    // The task's first warp adds the others' sums.  Warps share tasks only where
    // each has a single one, so their rings are free now.
    if (split > 1) {
      int4* mine = reinterpret_cast<int4*>(ring);
      if (part != 0) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int j = 0; j < kParts; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            mine[(2 * j + q) * 32] = make_int4(c[j][q][0], c[j][q][1], c[j][q][2], c[j][q][3]);
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / split), "r"(split * 32) : "memory");
      if (part != 0) break;
      for (int w = 1; w < split; ++w)
#pragma unroll
        for (int j = 0; j < kParts; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int4 o = mine[w * (C::kDepth * C::kLoads * 32) + (2 * j + q) * 32];
            c[j][q][0] += o.x;
            c[j][q][1] += o.y;
            c[j][q][2] += o.z;
            c[j][q][3] += o.w;
          }
    }

#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 2 * quad + (i & 1) + 8 * (i >> 1);
      if (row >= t.rows) continue;
      OutT* out = static_cast<OutT*>(p.d) + static_cast<long long>(t.row0 + row) * p.ldd + t.col0 + g8;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (t.col0 + g8 + 8 * h >= p.dim_out) continue;
        const int q = (i & 1) + 2 * h;
        // the same operations, in the same order, as the tiled kernels' epilogue
        float v = __int2float_rn(c[0][i >> 1][q]) * sa[i] * sb[0][h];
        if constexpr (kParts == 2) v = silu_mul_fast(v, __int2float_rn(c[1][i >> 1][q]) * sa[i] * sb[1][h]);
        if constexpr (std::is_same<OutT, float>::value) out[8 * h] = v;
        else out[8 * h] = to_out<OutT>(v);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}
