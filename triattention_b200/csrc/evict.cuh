// Eviction by accumulated attention weight: per (layer, request, KV head) row the keep_counts[b] tokens with the
// largest sums survive; the last `window` tokens and the first prefill_lens[b] are ranked above all others.  The
// sums live beside the cache, [num_blocks, Hkv, block_size] fp32 per layer, and are compacted with it.
//
// One CTA per row.  A row's sums are read once through the block table into shared memory (runs of block_size values);
// the radix passes and the output pass run from there, and the surviving sums go from there to their new slots.  Rows of more than
// kEvictCap tokens are read from the cache in every pass; their sums move in the output pass, run by run: rank r <= index
// i, and a run's values are in registers before any slot of it is written.
// Bound by the row's dependent look-ups and the latency of the passes, not by bytes: 128 rows of 31000 tokens 40 us (one CTA of 1024
// threads per SM), 256 rows of 2176 tokens 14 us (two CTAs of 512 per SM: with 1024 threads the second half of the rows had to
// wait, 20 us).  The compaction behind it moves its bytes at 5.7 TB/s.
#pragma once

#include "common.cuh"
#include "topk_row.cuh"

namespace triattn {

constexpr int kEvictLongRow = 8192;  // rows that may be longer run 1024 threads, one CTA per SM; others 512, two per SM
constexpr int kEvictCap = 49152;  // keys of a row kept in shared memory (192 KB); below 65536, see topk_row

struct EvictParams {
  float* sums;  // [L, num_blocks, Hkv, bs]
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* keep_counts;
  const int32_t* prefill_lens;  // or null
  int32_t* keep;                // [L, B, Hkv, pitch]
  int pitch, window;
  int B, Hkv, bs, num_blocks, max_blocks, cap;
  uint32_t* status;
};

// inverse of float_to_ordered
__device__ __forceinline__ float ordered_to_float(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) unsigned char evict_smem[];
  __shared__ TopkShared<THREADS> sh;
  grid_dependency_wait();
  trigger_dependents();
  const int h = blockIdx.x, b = blockIdx.y, l = blockIdx.z;
  unsigned err = 0u;
  int n = p.seq_lens[b];
  if (n > (long long)p.max_blocks * p.bs) {
    err |= TRIATTN_DEV_BAD_LENGTH;
    n = p.max_blocks * p.bs;
  }
  n = max(n, 0);
  const int k = max(0, min(p.keep_counts[b], min(n, p.pitch)));
  if (p.keep_counts[b] > p.pitch && n > p.pitch) err |= TRIATTN_DEV_BAD_LENGTH;  // the row holds no more
  const int guard = p.prefill_lens != nullptr ? p.prefill_lens[b] : 0;
  const int recent = n - p.window;
  const int32_t* bt = p.block_table + (long long)b * p.max_blocks;
  int32_t* out = p.keep + (((long long)l * p.B + b) * p.Hkv + h) * p.pitch;
  float* sums = p.sums + (long long)l * p.num_blocks * p.Hkv * p.bs;
  auto slot = [&](int t) -> long long {
    const int lb = t / p.bs;
    const int blk = bt[lb];
    if ((unsigned)blk >= (unsigned)p.num_blocks) {
      err |= TRIATTN_DEV_BAD_BLOCK_ID;
      return -1;
    }
    return ((long long)blk * p.Hkv + h) * p.bs + (t - lb * p.bs);
  };
  for (int i = k + threadIdx.x; i < p.pitch; i += THREADS) out[i] = -1;
  const bool cached = n <= p.cap;
  constexpr unsigned kInf = 0xff800000u;  // float_to_ordered(+inf); guarded tokens rank above it
  topk_row<THREADS>(
      n, k, reinterpret_cast<unsigned*>(evict_smem), p.cap, sh,
      slot,
      [&](long long at) -> unsigned {  // (kept invertible: the sum itself goes to its new slot)
        const float w = sums[max(at, 0ll)];
        return float_to_ordered(at < 0 ? -INFINITY : w);
      },
      [&](unsigned bits, int i) -> unsigned {
        if (i >= recent || i < guard) return kInf + 1u;
        if (bits == 0x7fffffffu) return 0x80000000u;  // -0 ranks as 0
        return bits > kInf ? 0u : bits;               // NaN last
      },
      [&](int rank, int i) { out[rank] = i; },
      [&](const bool(&sel)[4], const int(&rank)[4], const int(&at)[4], const unsigned(&bits)[4]) {
        __syncthreads();  // the run's sums are in registers before any of its destinations is written
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (!sel[j]) continue;
          out[rank[j]] = at[j];
          if (rank[j] != at[j]) {
            const long long to = slot(rank[j]);
            if (to >= 0) sums[to] = ordered_to_float(bits[j]);
          }
        }
      });
  if (cached) {
    __syncthreads();  // the CTA's keep list and the row's sums are there for all threads
    const unsigned* bits = reinterpret_cast<const unsigned*>(evict_smem);
    for (int r0 = threadIdx.x; r0 < k; r0 += THREADS * 4) {
      int from[4];
      long long to[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) from[j] = out[min(r0 + j * THREADS, k - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j) to[j] = slot(min(r0 + j * THREADS, k - 1));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + j * THREADS;
        if (r < k && from[j] != r && to[j] >= 0) sums[to[j]] = ordered_to_float(bits[from[j]]);
      }
    }
  }
  if (err) flag_status(p.status, err);
}

}  // namespace triattn
