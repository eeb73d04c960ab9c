// Block-sparse attention: per-block key bounds, and the choice of the blocks a step reads.
//
// bounds[block, h, 0/1, d] = min / max over the block's tokens of k[d].  For a query q,
//   q . k <= sum_d max(q_d min_d, q_d max_d) = q+ . max + q- . min,   q+ = max(q, 0), q- = min(q, 0),
// and the bound is linear in (q+, q-): summed over the query tokens and heads that share a KV head it is one dot product
// of 2 D terms per block.  The blocks with the largest sums are read.
#pragma once

#include <cfloat>

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

// Bound by HBM: K read once (bounds of 4 x 26400 tokens x 2 layers, 486 MB, in 74 us: the copy bandwidth).
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
  const unsigned char* kbase = static_cast<const unsigned char*>(p.k_ptrs[l]);
  // (block, head) pairs, the head fastest; the warps of the grid's row stride over them
  const int stride = (int)gridDim.x * (kBoundsThreads / 32), start = (int)blockIdx.x * (kBoundsThreads / 32) + wid;
  const int d_blk = stride / p.Hkv, d_head = stride - d_blk * p.Hkv;
  int lb = blk0 + start / p.Hkv, h = start % p.Hkv;
  for (; lb < blk1; lb += d_blk, h += d_head, lb += h >= p.Hkv ? 1 : 0, h -= h >= p.Hkv ? p.Hkv : 0) {
    const int blk = p.block_table[(long long)b * p.max_blocks + lb];
    if ((unsigned)blk >= (unsigned)p.num_blocks) {
      err |= TRIATTN_DEV_BAD_BLOCK_ID;
      continue;
    }
    const int n = min(p.bs, T - lb * p.bs);
    const unsigned char* src = kbase + ((long long)blk * p.block_stride + (long long)h * p.head_stride) * 2 + piece * 16;
    const long long step = (long long)rpw * p.token_stride * 2;
    src += (long long)sub * p.token_stride * 2;
    uint32_t lo[4] = {0x7f807f80u, 0x7f807f80u, 0x7f807f80u, 0x7f807f80u};
    uint32_t hi[4] = {0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
    for (int t = sub; t < n; t += 8 * rpw, src += 8 * step) {
      uint4 w[8];  // eight loads in flight; tokens that are not there repeat the first
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const uint4*>(src + (t + j * rpw < n ? j * step : 0));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[0] = min2_nan(lo[0], w[j].x);
        lo[1] = min2_nan(lo[1], w[j].y);
        lo[2] = min2_nan(lo[2], w[j].z);
        lo[3] = min2_nan(lo[3], w[j].w);
        hi[0] = max2_nan(hi[0], w[j].x);
        hi[1] = max2_nan(hi[1], w[j].y);
        hi[2] = max2_nan(hi[2], w[j].z);
        hi[3] = max2_nan(hi[3], w[j].w);
      }
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
// 2^-896, exactly: no conversion instructions.  Infinite bounds count as 2^128, so that 0 times them is 0; a block whose bounds
// hold NaN (a NaN among its keys) gets some score of that size.
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

//
// A warp takes `per_warp` consecutive blocks of one (request, KV head): its lanes fetch the block ids together, the bounds come
// in through a ring of eight rows per warp (cp.async: in registers the loads in flight cost occupancy, and with either too few
// loads or too few warps the kernel took half as long again), and four blocks' sums are reduced together; a lane holds the same
// 2 D / 32 channels' weights throughout.  Bound by the bounds' bytes (4 D per block and KV head), read once: 128 MB in 33 us,
// of which 8 are the queries' sums at the start of every CTA.
constexpr int kScoreRing = 8;  // rows
template <int D>
constexpr size_t score_smem_bytes() { return (size_t)(kScoreThreads / 32) * kScoreRing * D * 4 + 2 * (kScoreThreads / 32) * D * sizeof(double); }
template <int D>
__global__ void __launch_bounds__(kScoreThreads) block_scores_kernel(const __grid_constant__ SelectBlocksParams p, const int per_warp) {
  constexpr int WARPS = kScoreThreads / 32, PCS = D / 8, GROUPS = kScoreThreads / PCS;  // 16-byte pieces of a row, rows at a time
  constexpr int PER = 2 * D / 32;  // values per lane: 4 at D = 64, 8 at 128, 16 at 256
  extern __shared__ __align__(16) unsigned char score_smem[];
  __shared__ double qsum[2 * D];
  unsigned char* ring = score_smem + (threadIdx.x >> 5) * (kScoreRing * D * 4);
  double(*part)[WARPS][D] = reinterpret_cast<double(*)[WARPS][D]>(score_smem + WARPS * kScoreRing * D * 4);  // by sign and warp
  grid_dependency_wait();
  trigger_dependents();
  unsigned err = 0u;
  const int h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const BlocksReq r = blocks_req(p, b, err);
  if (err && blockIdx.x == 0 && h == 0 && tid == 0) flag_status(p.status, err);
  err = 0u;
  const int lb0 = ((int)blockIdx.x * WARPS + wid) * per_warp, lb1 = min(lb0 + per_warp, r.blocks);
  if ((int)blockIdx.x * WARPS * per_warp >= r.blocks) return;
  // ---- block ids of this warp's blocks; -1: always read, or not there
  int my_blk = -1;
  if (lb0 + lane < lb1 && lb0 + lane >= p.sink && lb0 + lane < r.forced_from) {
    my_blk = p.block_table[(long long)b * p.max_blocks + lb0 + lane];
    if ((unsigned)my_blk >= (unsigned)p.num_blocks) {
      err |= TRIATTN_DEV_BAD_BLOCK_ID;
      my_blk = -2;
    }
  }
  const int count = lb1 - lb0;
  auto fetch = [&](int j) {  // bounds of the warp's block j
    const int blk = __shfl_sync(0xffffffffu, my_blk, j & 31);
    if (j < count && blk >= 0) {
      const unsigned char* src = reinterpret_cast<const unsigned char*>(p.bounds + ((long long)blk * p.Hkv + h) * 2 * D);
      const uint32_t dst = smem_u32(ring + (j % kScoreRing) * (D * 4));
#pragma unroll
      for (int x = lane; x < D / 4; x += 32) cp_async16(dst + x * 16, src + x * 16, true);
    }
  };
#pragma unroll
  for (int j = 0; j < kScoreRing; ++j) {
    fetch(j);
    if (j % 4 == 3) cp_async_commit();
  }
  // ---- the query rows' sums, eight channels per thread
  {
    const int pc = tid % PCS, gr = tid / PCS;
    double up[8], down[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) up[x] = down[x] = 0.0;
    for (int row = gr; row < r.n * p.g; row += GROUPS) {
      const int i = row / p.g, j = row - i * p.g;
      const uint4 w = *reinterpret_cast<const uint4*>(p.q + (long long)(r.q0 + i) * p.q_ts + (long long)(h * p.g + j) * p.q_hs + pc * 8);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 e = bf16x2_to_float2(u[x]);
        up[2 * x] += (double)fmaxf(e.x, 0.f);
        down[2 * x] += (double)fminf(e.x, 0.f);
        up[2 * x + 1] += (double)fmaxf(e.y, 0.f);
        down[2 * x + 1] += (double)fminf(e.y, 0.f);
      }
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) {
#pragma unroll
      for (int k = PCS; k < 32; k <<= 1) {
        up[x] += __shfl_xor_sync(0xffffffffu, up[x], k);
        down[x] += __shfl_xor_sync(0xffffffffu, down[x], k);
      }
      if (lane < PCS) {
        part[0][wid][pc * 8 + x] = down[x];
        part[1][wid][pc * 8 + x] = up[x];
      }
    }
  }
  __syncthreads();
  for (int e = tid; e < 2 * D; e += kScoreThreads) {
    double s = 0.0;
    for (int w = 0; w < WARPS; ++w) s += part[e / D][w][e % D];
    qsum[e] = s;
  }
  __syncthreads();
  double q[PER];
#pragma unroll
  for (int x = 0; x < PER; ++x) q[x] = qsum[lane * PER + x];
  const double unscale = __hiloint2double((1023 + 896) << 20, 0);
  float* out = p.scores + ((long long)b * p.Hkv + h) * p.max_blocks;
  for (int j0 = 0; j0 < count; j0 += 4) {
    cp_async_wait<kScoreRing / 4 - 1>();
    __syncwarp();
    uint32_t w[4][PER / 2];
#pragma unroll
    for (int y = 0; y < 4; ++y) {  // (rows that were not fetched hold anything: their sums are not used)
#pragma unroll
      for (int x = 0; x < PER / 2; x += 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(ring + ((j0 + y) % kScoreRing) * (D * 4) + (lane * (PER / 2) + x) * 4);
        w[y][x] = u.x;
        w[y][x + 1] = u.y;
      }
    }
    __syncwarp();
#pragma unroll
    for (int y = 0; y < 4; ++y) fetch(j0 + kScoreRing + y);
    cp_async_commit();
    double s[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      s[y] = 0.0;
#pragma unroll
      for (int x = 0; x < PER / 2; ++x) {
        const uint32_t a = w[y][x] << 16, c = w[y][x] & 0xffff0000u;
        s[y] = fma(__hiloint2double((int)((a & 0x80000000u) | ((a & 0x7fffffffu) >> 3)), 0), q[2 * x], s[y]);
        s[y] = fma(__hiloint2double((int)((c & 0x80000000u) | ((c & 0x7fffffffu) >> 3)), 0), q[2 * x + 1], s[y]);
      }
    }
    // lanes 0-15 go on with blocks 0 and 1, 16-31 with 2 and 3; then a quarter of the warp has one block
    const bool upper = (lane & 16) != 0, odd = (lane & 8) != 0;
#pragma unroll
    for (int y = 0; y < 2; ++y) s[y] = (upper ? s[y + 2] : s[y]) + __shfl_xor_sync(0xffffffffu, upper ? s[y] : s[y + 2], 16);
    s[0] = (odd ? s[1] : s[0]) + __shfl_xor_sync(0xffffffffu, odd ? s[0] : s[1], 8);
#pragma unroll
    for (int k = 4; k; k >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], k);
    const int j = j0 + (upper ? 2 : 0) + (odd ? 1 : 0);
    const int blk = __shfl_sync(0xffffffffu, my_blk, j & 31);
    if ((lane & 7) == 0 && j < count) {
      float v = (float)(s[0] * unscale);
      if (v == INFINITY) v = FLT_MAX;  // only the blocks that are always read are above every number
      out[lb0 + j] = blk >= 0 ? v : blk == -1 ? INFINITY : -INFINITY;
    }
  }
  if (err) flag_status(p.status, err);
}

constexpr int kPickThreads = 1024;
__global__ void __launch_bounds__(kPickThreads) pick_blocks_kernel(const __grid_constant__ SelectBlocksParams p, const int cap) {
  extern __shared__ __align__(16) unsigned char pick_smem[];
  __shared__ TopkShared<kPickThreads> sh;
  grid_dependency_wait();
  trigger_dependents();
  const int h = blockIdx.x, b = blockIdx.y;
  unsigned err = 0u;
  const BlocksReq r = blocks_req(p, b, err);
  const int k = min(p.num_selected, r.blocks);
  const float* x = p.scores + ((long long)b * p.Hkv + h) * p.max_blocks;
  int32_t* out = p.block_list + ((long long)b * p.Hkv + h) * p.num_selected;
  for (int i = k + threadIdx.x; i < p.num_selected; i += kPickThreads) out[i] = -1;
  topk_row<kPickThreads>(
      r.blocks, k, reinterpret_cast<unsigned*>(pick_smem), cap, sh, [](int i) -> long long { return i; },
      [&](long long i) -> unsigned { return __float_as_uint(x[i]); },
      [&](unsigned bits, int i) -> unsigned {
        const float w = __uint_as_float(bits);
        return float_to_ordered(w == w ? w + 0.f : -INFINITY);  // -0 ranks as 0, NaN last
      },
      [&](int rank, int i) { out[rank] = i; },
      [&](const bool(&sel)[4], const int(&rank)[4], const int(&at)[4], const unsigned(&)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (sel[j]) out[rank[j]] = at[j];
      });
}

}  // namespace triattn
