// row_ring.cuh -- rows of one or several [rows, dim] inputs streamed into
// shared memory by bulk copies, several rows ahead of the block that works on
// them: no registers and no threads held by loads in flight.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "gmm_sm100.h"
#include "sm100_ptx.cuh"
#include "status.h"

namespace gmm_sm100 {
namespace {

// Set when a wait for a copy ran out (gmm_sm100_device_error reads it); one
// per source file.
__device__ int g_row_error = 0;

int read_row_error(int* status, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_row_error, sizeof(int));
  const int zero = 0;
  if (e == cudaSuccess && clear && *status) e = cudaMemcpyToSymbol(g_row_error, &zero, sizeof(int));
  return e == cudaSuccess ? GMM_OK : set_error(GMM_ERR_CUDA, cudaGetErrorString(e));
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Bytes a row takes in a slot: it keeps its offset within 16 bytes there.
__host__ __device__ constexpr uint32_t row_pitch(uint32_t row_bytes, bool aligned) {
  return aligned ? row_bytes : (row_bytes + 15 + 15) / 16 * 16;
}

// A ring of row slots in shared memory, filled by bulk copies, which take
// whole 16-byte words.  A slot holds one row of each input that is there.
// kAligned: every row starts and ends on a word; otherwise a row is fetched
// with the words it shares with its neighbours, except at a tensor's two
// ends, where those words may reach beyond it: there only whole words come by
// the copy, and the block's threads bring the bytes around them.
template <int kInputs, bool kAligned>
struct RowRing {
  const char* src[kInputs];
  uint32_t bytes[kInputs];  // of a row (or of the part of it that is wanted); 0: input not there
  long long pitch_bytes[kInputs];  // from a row to the next
  long long rows;
  uint8_t* smem;            // slot 0
  uint32_t slot_bytes;
  uint32_t bars;            // shared address of the slots' barriers
  int slots;
  int edge_rows;            // rows at either end of a tensor within 15 bytes of it
  bool dead;                // a wait ran out: no more waiting or loading, the error word says so

  __device__ __forceinline__ uint32_t pitch(int i) const { return bytes[i] ? row_pitch(bytes[i], kAligned) : 0; }

  // One thread: fetch `row` into `slot`.
  __device__ __forceinline__ void fetch(int slot, long long row) const {
    const uint32_t bar = bars + 8 * slot;
    const bool inner = edge(row);  // only the words that lie wholly inside the row
    const char* from[kInputs];
    uint32_t len[kInputs], to[kInputs], total = 0, at = smem_u32(smem) + slot * slot_bytes;
#pragma unroll
    for (int i = 0; i < kInputs; ++i) {
      from[i] = src[i] + row * pitch_bytes[i];
      len[i] = bytes[i];
      to[i] = at;
      if (!kAligned && bytes[i]) {
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from[i]) & 15u);
        const uint32_t lo = inner ? (off + 15u) & ~15u : 0u;  // from the first word's start
        const uint32_t hi = inner ? (off + bytes[i]) & ~15u : (off + bytes[i] + 15u) & ~15u;
        len[i] = hi > lo ? hi - lo : 0u;
        from[i] += static_cast<int>(lo) - static_cast<int>(off);
        to[i] += lo;
      }
      total += len[i];
      at += pitch(i);
    }
    mbar_arrive_expect_tx(bar, total);
#pragma unroll
    for (int i = 0; i < kInputs; ++i)
      if (len[i]) bulk_load(to[i], from[i], len[i], bar);
  }

  // Whether the words of `row` may reach beyond an input's first or last byte
  // (they reach at most 15 bytes past the row on either side).
  __device__ __forceinline__ bool edge(long long row) const {
    return !kAligned && (row < edge_rows || row >= rows - edge_rows);
  }

  // All threads: wait for the row in `slot`.
  __device__ __forceinline__ void wait(int slot, uint32_t parity, long long row) {
    if (!dead) {
      const uint32_t bar = bars + 8 * slot;
      if (!mbar_try_wait(bar, parity)) {
        const unsigned long long t0 = global_timer_ns();
        while (!mbar_try_wait(bar, parity))
          if (global_timer_ns() - t0 > kWaitTimeoutNs) {
            dead = true;
            atomicCAS(&g_row_error, 0, GMM_ERR_DEVICE_TIMEOUT);
            break;
          }
      }
    }
    if (!edge(row)) return;
    // the row's bytes before its first and after its last whole word, at most
    // 15 on each side (rows are a multiple of 2 bytes)
    uint8_t* base = smem + slot * slot_bytes;
#pragma unroll
    for (int i = 0; i < kInputs; ++i) {
      const char* from = src[i] + row * pitch_bytes[i];
      const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from) & 15u);
      const uint32_t lo = (off + 15u) & ~15u, hi = (off + bytes[i]) & ~15u, end = off + bytes[i];
      for (uint32_t k = off + 2 * threadIdx.x; k < end; k += 2 * blockDim.x)
        if (k < lo || k >= hi)
          *reinterpret_cast<uint16_t*>(base + k) = *reinterpret_cast<const uint16_t*>(from + (k - off));
      base += pitch(i);
    }
    fence_proxy_async_smem();  // the slot's next contents come by a bulk copy
    __syncthreads();
  }

  // Where the first word of input i of `slot` lies, from slot 0's start, and
  // where the row in it starts.
  __device__ __forceinline__ uint32_t word_at(int slot, int i) const {
    uint32_t off = slot * slot_bytes;
#pragma unroll
    for (int j = 0; j < i; ++j) off += pitch(j);
    return off;
  }
  __device__ __forceinline__ uint32_t at(int slot, int i, long long row) const {
    return word_at(slot, i) +
           (kAligned ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src[i] + row * pitch_bytes[i]) & 15u));
  }

  // Input i: `n` elements of every row, `pitch` elements apart.
  __device__ __forceinline__ void input(int i, const void* first, int elem, int n, int pitch) {
    src[i] = static_cast<const char*>(first);
    bytes[i] = n * elem;
    pitch_bytes[i] = static_cast<long long>(pitch) * elem;
  }

  // Shared memory: slots * slot_bytes of rows, then one barrier a slot.  `pad`:
  // bytes of a slot behind its last input's row.  The caller synchronises the
  // block before the first wait.
  __device__ __forceinline__ void start(uint8_t* mem, int n, long long num_rows, uint32_t pad = 0) {
    smem = mem;
    slots = n;
    rows = num_rows;
    dead = false;
    slot_bytes = pad;
    uint32_t least = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kInputs; ++i) {
      slot_bytes += pitch(i);
      if (bytes[i]) least = min(least, bytes[i]);
    }
    edge_rows = (15 + least - 1) / least;
    bars = smem_u32(mem) + slots * slot_bytes;
    if (threadIdx.x == 0) {
      for (int s = 0; s < slots; ++s) mbar_init(bars + 8 * s, 1);
      fence_mbarrier_init();
      for (int s = 0; s < slots; ++s) {
        const long long row = blockIdx.x + static_cast<long long>(s) * gridDim.x;
        if (row < rows) fetch(s, row);
      }
    }
  }
};

// ------------------------------------------------------------------ host side
constexpr int kRingBytes = 224 * 1024;  // shared memory of an SM the rings may take, over its resident blocks
constexpr int kRingBlockBytes = kRingBytes - 2048;  // dynamic shared memory of one block, at most (allow_smem)

inline int threads_for(int items) { return std::max(32, (items + 31) / 32 * 32); }

// Opts a kernel into its dynamic shared memory, once a device.
template <typename K>
cudaError_t allow_smem(K kernel, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBlockBytes);
  if (e == cudaSuccess) done.fetch_or(bit);
  return e;
}

}  // namespace
}  // namespace gmm_sm100
