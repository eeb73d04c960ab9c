// Block-sparse attention: per-block key bounds, and the choice of the blocks a step reads.
//
// bounds[block, h, 0/1, d] = min / max over the block's tokens of k[d].  For a query q,
//   q . k <= sum_d max(q_d min_d, q_d max_d) = q+ . max + q- . min,   q+ = max(q, 0), q- = min(q, 0),
// and the bound is linear in (q+, q-): summed over the query tokens and heads that share a KV head it is one dot product
// of 2 D terms per block.  The blocks with the largest sums are read.
#pragma once

#include "common.cuh"
#include "attend.cuh"
#include "topk_row.cuh"

namespace triattn {

constexpr int kBoundsThreads = 256;

struct BoundsParams {
  const void* const* k_ptrs;  // [L]
  uint16_t* bounds;           // [L, num_blocks, Hkv, 2, D]
  const int32_t* block_table;
  const int32_t* first;     // [B] first token that changed
  const int32_t* seq_lens;
  int B, Hkv, D, bs, num_blocks, max_blocks;
  long long block_stride, token_stride, head_stride;
  uint32_t* status;
};

__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// One warp per (block, KV head): D / 8 lanes hold 8 channels each, the other lanes take further tokens.  The warps
// of a CTA take the heads of a block in turn, so that token-major caches are read in whole blocks.
__global__ void __launch_bounds__(kBoundsThreads) block_bounds_kernel(const __grid_constant__ BoundsParams p) {
  grid_dependency_wait();
  const int b = blockIdx.y, l = blockIdx.z;
  unsigned err = 0u;
  int T = p.seq_lens[b];
  if (T > (long long)p.max_blocks * p.bs) {
    err |= TRIATTN_DEV_BAD_LENGTH;
    T = p.max_blocks * p.bs;
  }
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int lpr = p.D / 8, rpw = 32 / lpr;  // lanes per row, rows per step
  const int sub = lane / lpr, piece = lane - sub * lpr;
  const int blk0 = max(p.first[b], 0) / p.bs, blk1 = (T + p.bs - 1) / p.bs;
  const long long items = (long long)max(blk1 - blk0, 0) * p.Hkv;
  const unsigned char* kbase = static_cast<const unsigned char*>(p.k_ptrs[l]);
  for (long long it = (long long)blockIdx.x * (kBoundsThreads / 32) + wid; it < items; it += (long long)gridDim.x * (kBoundsThreads / 32)) {
    const int lb = blk0 + (int)(it / p.Hkv), h = (int)(it % p.Hkv);
    const int blk = p.block_table[(long long)b * p.max_blocks + lb];
    if ((unsigned)blk >= (unsigned)p.num_blocks) {
      err |= TRIATTN_DEV_BAD_BLOCK_ID;
      continue;
    }
    const int n = min(p.bs, T - lb * p.bs);
    const unsigned char* src = kbase + ((long long)blk * p.block_stride + (long long)h * p.head_stride) * 2 + piece * 16;
    uint32_t lo[4] = {0x7f807f80u, 0x7f807f80u, 0x7f807f80u, 0x7f807f80u};
    uint32_t hi[4] = {0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
#pragma unroll 8
    for (int t = sub; t < n; t += rpw) {
      const uint4 w = *reinterpret_cast<const uint4*>(src + (long long)t * p.token_stride * 2);
      lo[0] = min2_nan(lo[0], w.x);
      lo[1] = min2_nan(lo[1], w.y);
      lo[2] = min2_nan(lo[2], w.z);
      lo[3] = min2_nan(lo[3], w.w);
      hi[0] = max2_nan(hi[0], w.x);
      hi[1] = max2_nan(hi[1], w.y);
      hi[2] = max2_nan(hi[2], w.z);
      hi[3] = max2_nan(hi[3], w.w);
    }
    for (int s = 16; s >= lpr; s >>= 1) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        lo[x] = min2_nan(lo[x], __shfl_xor_sync(0xffffffffu, lo[x], s));
        hi[x] = max2_nan(hi[x], __shfl_xor_sync(0xffffffffu, hi[x], s));
      }
    }
    uint16_t* dst = p.bounds + ((((long long)l * p.num_blocks + blk) * p.Hkv + h) * 2) * p.D + piece * 8;
    if (sub == 0) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      *reinterpret_cast<uint4*>(dst + p.D) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    }
  }
  if (err) flag_status(p.status, err);
}

// ------------------------------------------------------------------------------------------ block scores
// The order of the scores decides which blocks are read, so they are formed in 64 bits and rounded to 32 once: equal scores
// stay equal whatever the order of the sum.  A bf16 word shifted into the high half of a double is the value times
// 2^-896, exactly (subnormal bf16 values land on subnormal doubles): no conversion instructions.
constexpr int kScoreThreads = 256;

struct SelectBlocksParams {
  const uint16_t* q;
  long long q_ts, q_hs;
  const int32_t* qsl;
  const uint16_t* bounds;  // [num_blocks, Hkv, 2, D]
  const int32_t* block_table;
  const int32_t* seq_lens;
  int B, Hkv, g, bs, num_blocks, max_blocks, N, max_q;
  int num_selected, sink, recent;
  float* scores;      // [B, Hkv, max_blocks]
  int32_t* block_list;  // [B, Hkv, num_selected]
  uint32_t* status;
};

struct BlocksReq {
  int T, n, q0, blocks, forced_from;
};
__device__ __forceinline__ BlocksReq blocks_req(const SelectBlocksParams& p, int b, unsigned& err) {
  BlocksReq r;
  r.T = p.seq_lens[b];
  r.q0 = p.qsl[b];
  r.n = p.qsl[b + 1] - r.q0;
  r.blocks = r.forced_from = 0;
  if (r.n == 0) return r;
  if (r.n < 0 || r.n > p.max_q || r.q0 < 0 || r.q0 > p.N - r.n || r.T < r.n || r.T > (long long)p.max_blocks * p.bs) {
    err |= TRIATTN_DEV_BAD_LENGTH;
    r.n = 0;
    return r;
  }
  r.blocks = (r.T + p.bs - 1) / p.bs;
  r.forced_from = min(r.blocks - p.recent, (r.T - r.n) / p.bs);  // the query's own tokens are always read
  return r;
}

template <int D>
__global__ void __launch_bounds__(kScoreThreads) block_scores_kernel(const __grid_constant__ SelectBlocksParams p) {
  __shared__ double qsum[2][D];
  grid_dependency_wait();
  unsigned err = 0u;
  const int h = blockIdx.y, b = blockIdx.z;
  const BlocksReq r = blocks_req(p, b, err);
  if (err && blockIdx.x == 0 && h == 0 && threadIdx.x == 0) flag_status(p.status, err);
  err = 0u;
  if (r.blocks <= (int)blockIdx.x * (kScoreThreads / 32)) return;
  for (int d = threadIdx.x; d < D; d += kScoreThreads) {
    double up = 0.0, down = 0.0;
    for (int x = 0; x < r.n * p.g; ++x) {
      const int i = x / p.g, j = x - i * p.g;
      const float v = bf16_to_float(p.q[(long long)(r.q0 + i) * p.q_ts + (long long)(h * p.g + j) * p.q_hs + d]);
      up += v > 0.f ? (double)v : 0.0;
      down += v < 0.f ? (double)v : 0.0;
    }
    qsum[0][d] = down;
    qsum[1][d] = up;
  }
  __syncthreads();
  constexpr int PER = 2 * D / 32;  // values per lane: 4 at D = 64, 8 at 128, 16 at 256
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  double q[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) q[x] = (&qsum[0][0])[lane * PER + x];
  const double unscale = __hiloint2double((1023 + 896) << 20, 0);
  float* out = p.scores + ((long long)b * p.Hkv + h) * p.max_blocks;
  for (int lb = blockIdx.x * (kScoreThreads / 32) + wid; lb < r.blocks; lb += gridDim.x * (kScoreThreads / 32)) {
    float score;
    if (lb < p.sink || lb >= r.forced_from) {
      score = INFINITY;
    } else {
      const int blk = p.block_table[(long long)b * p.max_blocks + lb];
      if ((unsigned)blk >= (unsigned)p.num_blocks) {
        err |= TRIATTN_DEV_BAD_BLOCK_ID;
        score = -INFINITY;
      } else {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(p.bounds + ((long long)blk * p.Hkv + h) * 2 * D) + lane * (PER / 2);
        uint32_t w[PER / 2];
#pragma unroll
        for (int x = 0; x < PER / 2; x += 2) {
          const uint2 u = *reinterpret_cast<const uint2*>(src + x);
          w[x] = u.x;
          w[x + 1] = u.y;
        }
        double s = 0.0;
#pragma unroll
        for (int x = 0; x < PER / 2; ++x) {
          const uint32_t a = w[x] << 16, c = w[x] & 0xffff0000u;
          s = fma(__hiloint2double((int)((a & 0x80000000u) | ((a & 0x7fffffffu) >> 3)), 0), q[2 * x], s);
          s = fma(__hiloint2double((int)((c & 0x80000000u) | ((c & 0x7fffffffu) >> 3)), 0), q[2 * x + 1], s);
        }
#pragma unroll
        for (int k = 16; k; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
        score = (float)(s * unscale);
      }
    }
    if (lane == 0) out[lb] = score;
  }
  if (err) flag_status(p.status, err);
}

constexpr int kPickThreads = 256;
__global__ void __launch_bounds__(kPickThreads) pick_blocks_kernel(const __grid_constant__ SelectBlocksParams p, const int cap) {
  extern __shared__ __align__(16) unsigned char pick_smem[];
  __shared__ TopkShared<kPickThreads> sh;
  grid_dependency_wait();
  const int h = blockIdx.x, b = blockIdx.y;
  unsigned err = 0u;
  const BlocksReq r = blocks_req(p, b, err);
  const int k = min(p.num_selected, r.blocks);
  const float* x = p.scores + ((long long)b * p.Hkv + h) * p.max_blocks;
  int32_t* out = p.block_list + ((long long)b * p.Hkv + h) * p.num_selected;
  for (int i = k + threadIdx.x; i < p.num_selected; i += kPickThreads) out[i] = -1;
  topk_row<kPickThreads>(
      r.blocks, k, reinterpret_cast<unsigned*>(pick_smem), cap, sh,
      [&](int i) -> unsigned {
        const float w = x[i];
        return float_to_ordered(w == w ? w + 0.f : -INFINITY);
      },
      [&](bool sel, int rank, int i) {
        if (sel) out[rank] = i;
      });
}

}  // namespace triattn
