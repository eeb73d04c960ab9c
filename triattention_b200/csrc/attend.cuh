// Attention of a few query tokens per request over the paged bf16 cache (decode steps and trees of drafted tokens).
//
//   s[r, t] = scale * q_r . k_t          r: query row = (query token i, head of the KV head's group), t: cached token
//   o_r     = sum_t exp(s[r, t] - lse_r) v_t,   lse_r = log sum_t exp(s[r, t])
//
// over the tokens a row sees: every token before the request's query tokens, and of these (their keys are the last
// slots of the sequence) the ones whose bit is set in the row's 64-bit word.  The softmax runs in one pass with a
// running maximum and sum in fp32, in the base-2 domain.  Exponentials are taken against a reference that lies the base-2
// logarithm of the segment's tokens (rounded up) above the maximum: a row's exponentials then add up to at most 1, and the
// unnormalised o is finite for all finite values (against the maximum itself, 700 values of 2^126 and equal weights gave infinities).
// What that costs lies at the other end: of 2^n tokens, weights below 2^(n - 126) of the largest vanish, and outputs below
// that size lose bits of fp32.
//
// Bound: K and V are read once, 4 D bytes per (KV head, token), for 4 D R operations with R rows; up to about 32 rows the cache
// stream is the limit, so what counts is that all SMs stream all the time.  The work of a KV head - the sequence of
// token tiles of all (request, row tile) segments - is therefore cut into J equal runs of tiles, wherever the cut falls:
// lengths may be as ragged as they like, and a single long request fills the device.  CTA j * Hkv + h takes run j of
// head h, so that neighbouring CTAs read the heads of the same tokens at the same time: a token's heads lie side by side
// in memory, and runs over all (head, token) tiles, in which the heads of a token are read far apart in time, streamed a fifth slower.
// A CTA that owns a whole segment writes its output; the others leave (m, l, unnormalised o) in a workspace slot, at most two
// per CTA, and attend_combine_kernel joins them in a fixed order (no atomics: results repeat bit for bit).
#pragma once

#include "common.cuh"

namespace triattn {

constexpr int kAttendMaxQuery = 64;  // query tokens per request: bits of a mask word
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttendParams {
  const uint16_t* q;  // [N, Hq, D] bf16
  long long q_ts, q_hs;
  const unsigned char* k;
  const unsigned char* v;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* qsl;        // [B + 1]
  const int64_t* tree;       // [N] or null (chain)
  const int32_t* block_list; // [B, Hkv, num_listed] or null
  int num_listed;
  int B, Hkv, g, bs, num_blocks, max_blocks;
  long long block_stride, token_stride, head_stride;  // elements
  int N, max_q;
  int box;        // tokens per TMA box: the tile's tokens, halved until they divide the block size (tiled kernels)
  int slots_per_block;  // head slots per block: block_stride / head_stride (tiled kernels)
  int min_tiles;  // tiles a CTA should have before another one is started
  float scale_log2;
  uint16_t* out;
  long long o_ts, o_hs;
  float* lse;  // [N, Hq]
  float* part_o;   // [2 * G][rows][D]
  float* part_ml;  // [2 * G][rows][2]
  float* sums;     // [num_blocks, Hkv, bs] or null
  int reset_sums;
  uint32_t* status;
};

// One request as the kernels see it; tiles == 0: nothing to do (no query tokens, or bad metadata, which is flagged).
struct AttendReq {
  int T, n, q0, vlen, tiles, row_tiles;
};

__device__ __forceinline__ AttendReq attend_req(const AttendParams& p, int b, int tile, int rows_per_tile, unsigned& err) {
  AttendReq r;
  r.T = p.seq_lens[b];
  r.q0 = p.qsl[b];
  r.n = p.qsl[b + 1] - r.q0;
  r.tiles = r.row_tiles = r.vlen = 0;
  if (r.n == 0) return r;
  if (r.n < 0 || r.n > p.max_q || r.q0 < 0 || r.q0 > p.N - r.n || r.T < r.n || r.T > (long long)p.max_blocks * p.bs) {
    err |= TRIATTN_DEV_BAD_LENGTH;
    r.n = 0;
    return r;
  }
  r.vlen = r.T;
  if (p.block_list != nullptr) r.vlen = min(p.num_listed, (r.T + p.bs - 1) / p.bs) * p.bs;
  r.tiles = (r.vlen + tile - 1) / tile;
  r.row_tiles = (r.n * p.g + rows_per_tile - 1) / rows_per_tile;
  return r;
}

// ceil(log2(n)) of n >= 1
__device__ __forceinline__ int ceil_log2(int n) { return 32 - __clz(n - 1); }

// sum of `v` over the CTA; `red` holds one value per warp
template <int THREADS>
__device__ __forceinline__ long long block_sum_ll(long long v, long long* red) {
#pragma unroll
  for (int s = 16; s; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  long long t = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) t += red[w];
  __syncthreads();
  return t;
}

// tiles of requests [0, upto) per KV head
template <int THREADS>
__device__ __forceinline__ long long attend_work_before(const AttendParams& p, int upto, int tile, int rows_per_tile,
                                                        unsigned& err, long long* red) {
  long long w = 0;
  for (int b = threadIdx.x; b < upto; b += THREADS) {
    const AttendReq r = attend_req(p, b, tile, rows_per_tile, err);
    w += (long long)r.tiles * r.row_tiles;
  }
  return block_sum_ll<THREADS>(w, red);
}

// runs that W tiles are cut into, of at most `runs`
__device__ __forceinline__ int attend_runs(int runs, long long W, int min_tiles) {
  return (int)min((long long)runs, (W + min_tiles - 1) / min_tiles);
}
// first tile of run j of J over W >= J tiles, floor(W j / J) (every run has one at least), and the run that owns a tile
__device__ __forceinline__ long long attend_first_tile(long long W, int J, int j) {
  if (W < (1ll << 31)) {  // 32-bit divisions
    const unsigned w = (unsigned)W, q = w / (unsigned)J, r = w - q * (unsigned)J;
    return (long long)q * j + (r * (unsigned)j) / (unsigned)J;  // r j < J^2
  }
  return W * j / J;
}
__device__ __forceinline__ int attend_owner(long long W, int J, long long tile) {
  return (int)(((tile + 1) * J - 1) / W);
}

// A position in a KV head's sequence of tiles: segment (request b, row tile rt), tile t of it.
struct AttendCursor {
  AttendReq r;
  int b, h, rt, t;
};

// Shared memory of attend_plan_run.
template <int THREADS>
struct AttendPlanShared {
  long long warp_sum[THREADS / 32], at;
  AttendReq req;
  int b;
};

// The tiles of up to 32 requests, one per lane: this lane's request, the tiles before it, the tiles of all.
__device__ __forceinline__ long long attend_scan32(const AttendParams& p, int tile, int rows_per_tile, AttendReq& mine,
                                                   long long& before, unsigned& err) {
  const int lane = threadIdx.x & 31;
  mine.tiles = mine.row_tiles = 0;
  long long w = 0;
  if (lane < p.B) {
    mine = attend_req(p, lane, tile, rows_per_tile, err);
    w = (long long)mine.tiles * mine.row_tiles;
  }
  long long incl = w;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, incl, s);
    if (lane >= s) incl += u;
  }
  before = incl - w;
  return __shfl_sync(0xffffffffu, incl, 31);
}

// Where run `run` (at most `runs`) of the call starts, and how many tiles it has; false: there is no such run.  All threads
// call it; bad metadata is reported by run 0 of head 0.  Up to 32 requests every warp finds out for itself, without a
// barrier (with one, planning took three times as long); more take a request per thread and pass.
template <int THREADS>
__device__ __forceinline__ bool attend_plan_run(const AttendParams& p, int runs, int min_tiles, int run, int tile,
                                                int rows_per_tile, AttendPlanShared<THREADS>& sh, AttendCursor& c, int& count) {
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  unsigned err = 0u;
  AttendReq mine{};
  long long before = 0, W = 0;  // tiles before this thread's request of the pass, tiles of all passes
  if (p.B <= 32) {
    W = attend_scan32(p, tile, rows_per_tile, mine, before, err);
    if (blockIdx.x == 0 && wid == 0 && err) flag_status(p.status, err);
    const int J = attend_runs(runs, W, min_tiles);
    if (run >= J) return false;
    const long long first = attend_first_tile(W, J, run);
    count = (int)(attend_first_tile(W, J, run + 1) - first);
    const bool here = first >= before && first < before + (long long)mine.tiles * mine.row_tiles;
    const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    const long long at = __shfl_sync(0xffffffffu, first - before, from);
    c.b = from;
    c.r.T = __shfl_sync(0xffffffffu, mine.T, from);
    c.r.n = __shfl_sync(0xffffffffu, mine.n, from);
    c.r.q0 = __shfl_sync(0xffffffffu, mine.q0, from);
    c.r.vlen = __shfl_sync(0xffffffffu, mine.vlen, from);
    c.r.tiles = __shfl_sync(0xffffffffu, mine.tiles, from);
    c.r.row_tiles = __shfl_sync(0xffffffffu, mine.row_tiles, from);
    c.rt = at < (1ll << 31) ? (int)((unsigned)at / (unsigned)c.r.tiles) : (int)(at / c.r.tiles);
    c.t = (int)(at - (long long)c.rt * c.r.tiles);
    __syncthreads();  // what the CTA has set up meanwhile
    return true;
  }
  auto pass = [&](int b0) {
    long long w = 0;
    mine.tiles = mine.row_tiles = 0;
    if (b0 + tid < p.B) {
      mine = attend_req(p, b0 + tid, tile, rows_per_tile, err);
      w = (long long)mine.tiles * mine.row_tiles;
    }
    long long incl = w;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, incl, s);
      if (lane >= s) incl += u;
    }
    if (lane == 31) sh.warp_sum[wid] = incl;
    __syncthreads();
    before = incl - w;
    long long total = 0;
#pragma unroll
    for (int x = 0; x < THREADS / 32; ++x) {
      const long long u = sh.warp_sum[x];
      if (x < wid) before += u;
      total += u;
    }
    return total;
  };
  for (int b0 = 0; b0 < p.B; b0 += THREADS) {
    if (b0 > 0) __syncthreads();
    W += pass(b0);
  }
  if (blockIdx.x == 0 && err) flag_status(p.status, err);
  const int J = attend_runs(runs, W, min_tiles);
  if (run >= J) return false;
  const long long first = attend_first_tile(W, J, run);
  count = (int)(attend_first_tile(W, J, run + 1) - first);
  long long base = 0;
  for (int b0 = 0; b0 < p.B; b0 += THREADS) {
    if (p.B > THREADS) {
      __syncthreads();
      const long long total = pass(b0);
      before += base;
      base += total;
    }
    if (first >= before && first < before + (long long)mine.tiles * mine.row_tiles) {
      sh.at = first - before;
      sh.req = mine;
      sh.b = b0 + tid;
    }
  }
  __syncthreads();
  c.r = sh.req;
  c.b = sh.b;
  c.rt = (int)((unsigned long long)sh.at / (unsigned)c.r.tiles);
  c.t = (int)(sh.at - (long long)c.rt * c.r.tiles);
  return true;
}

__device__ __forceinline__ void attend_advance(const AttendParams& p, AttendCursor& c, int tile, int rows_per_tile) {
  if (++c.t < c.r.tiles) return;
  c.t = 0;
  if (++c.rt < c.r.row_tiles) return;
  c.rt = 0;
  unsigned err = 0u;
  do {
    if (++c.b >= p.B) return;  // behind the last tile: never used again
    c.r = attend_req(p, c.b, tile, rows_per_tile, err);
  } while (c.r.tiles == 0);
}

// ------------------------------------------------------------------------------------------ mma.sync building blocks
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 16 bytes global -> shared; ok == false writes zeros and reads nothing
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// bf16 pairs: exponent all ones in either half
__device__ __forceinline__ bool nonfinite2(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ bool has_nonfinite(const uint4& w) {
  return nonfinite2(w.x) || nonfinite2(w.y) || nonfinite2(w.z) || nonfinite2(w.w);
}
__device__ __forceinline__ uint32_t zero_nonfinite2(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
  return w;
}
__device__ __forceinline__ uint4 zero_nonfinite(const uint4& w) {
  return make_uint4(zero_nonfinite2(w.x), zero_nonfinite2(w.y), zero_nonfinite2(w.z), zero_nonfinite2(w.w));
}

constexpr int kAttendThreads = 128;
constexpr int kAttendTile = 64;  // tokens per tile
template <int D>
constexpr int kAttendStages = D > 128 ? 2 : 3;

// byte offset of 16-byte piece `piece` of row `row` in a [rows][D] bf16 tile: pieces are permuted inside a row so that
// eight rows' equal pieces fall into different banks (ldmatrix and cp.async without conflicts, no padding)
template <int D>
__device__ __forceinline__ uint32_t tile_off(int row, int piece) {
  return (uint32_t)(row * (D * 2) + ((piece ^ (row & 7)) << 4));
}

template <int D>
constexpr int kAttendStageBytes = kAttendTile * D * 2;

template <int D, int MT>
constexpr size_t attend_smem_bytes() {
  // stages of K and V, then Q (bf16) and the join scratch (fp32, when several warps share the rows) in the same place
  const size_t q = (size_t)16 * MT * D * 2, join = MT == 4 ? 0 : (size_t)16 * MT * D * 4;
  return (size_t)kAttendStages<D> * 2 * kAttendStageBytes<D> + (D > 128 ? q + join : (q > join ? q : join));
}

// Where token `vp` of the segment's token sequence lives: byte offset of its row, logical position (-1: masked).
struct TokenAt {
  long long off;
  int pos;
};
__device__ __forceinline__ TokenAt attend_token(const AttendParams& p, const AttendCursor& c, int vp, unsigned& err) {
  TokenAt a{0, -1};
  if (vp >= c.r.vlen) return a;
  int lb = vp / p.bs;
  const int in = vp - lb * p.bs;
  if (p.block_list != nullptr) {
    lb = p.block_list[((long long)c.b * p.Hkv + c.h) * p.num_listed + lb];
    if (lb < 0) return a;  // an unused entry of the list
    if (lb >= (c.r.T + p.bs - 1) / p.bs) {
      err |= TRIATTN_DEV_BAD_KEEP_INDEX;
      return a;
    }
  }
  const int pos = lb * p.bs + in;
  if (pos >= c.r.T) return a;
  const int blk = p.block_table[(long long)c.b * p.max_blocks + lb];
  if ((unsigned)blk >= (unsigned)p.num_blocks) {
    err |= TRIATTN_DEV_BAD_BLOCK_ID;
    return a;
  }
  a.off = ((long long)blk * p.block_stride + (long long)in * p.token_stride + (long long)c.h * p.head_stride) * 2;
  a.pos = pos;
  return a;
}

// Rows of a segment and the words of what they see
__device__ __forceinline__ unsigned long long attend_word(const AttendParams& p, const AttendReq& r, int i) {
  if (i >= r.n) return 0ull;
  if (p.tree != nullptr) return (unsigned long long)p.tree[r.q0 + i];
  return i >= 63 ? ~0ull : ((2ull << i) - 1ull);
}

// P V of the rounded probabilities and of their remainders.  Where an infinite value makes the first infinite the second says nothing:
// remainders have either sign, or are 0, and would turn it into NaN.
__device__ __forceinline__ float add_remainder(float o, float rest) { return isfinite(o) ? o + rest : o; }

// The general kernel, for caches the TMA kernels do not take (block sizes that are no multiple of 8, odd strides, more than 16 rows at
// head dimension 256): cp.async, token by token, 16 bytes a piece.  Bound by the address arithmetic and the waits of its
// loads: 2.8 TB/s on the case the TMA kernel streams at 5.7.
// MT x 16 query rows per CTA: MT warps side by side over the rows, 4 / MT over the tokens of a tile.
// SPLIT_P (at most 8 rows): the probabilities are carried as bf16 + bf16 remainder; the remainders ride in the
// eight rows of the operand that would otherwise be padding, so their products cost nothing.
template <int D, int MT, bool SPLIT_P>
__global__ void __launch_bounds__(kAttendThreads) attend_paged_kernel(const __grid_constant__ AttendParams p, const int runs) {
  static_assert(!SPLIT_P || MT == 1, "");
  constexpr int WK = 4 / MT;                // warps over the tokens
  constexpr int KW = kAttendTile / WK;      // tokens per warp and tile
  constexpr int ROWS = SPLIT_P ? 8 : 16 * MT;
  constexpr int PPR = D / 8;                // 16-byte pieces per row
  constexpr int RPI = kAttendThreads / PPR; // rows per copy step of the CTA
  constexpr int STEPS = kAttendTile / RPI;
  constexpr bool QREG = D <= 128;
  constexpr int kStages = kAttendStages<D>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int kpos[kStages][kAttendTile];
  __shared__ int bad_tile[kStages];
  __shared__ AttendPlanShared<kAttendThreads> plan;
  __shared__ float join_ml[4][16][2];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int wr = wid % MT, wk = wid / MT;

  grid_dependency_wait();
  trigger_dependents();
  unsigned err = 0u;
  const int run = (int)blockIdx.x / p.Hkv;
  AttendCursor lc;  // loads
  int count;
  if (tid < kStages) bad_tile[tid] = -1;
  if (!attend_plan_run<kAttendThreads>(p, runs, p.min_tiles, run, kAttendTile, ROWS, plan, lc, count)) return;
  lc.h = (int)blockIdx.x - run * p.Hkv;
  AttendCursor c = lc;  // arithmetic

  const uint32_t stage0 = smem_u32(smem);
  constexpr uint32_t kStage = kAttendStageBytes<D>;
  unsigned char* q_smem = smem + kStages * 2 * kStage;
  float* join = reinterpret_cast<float*>(q_smem + (QREG ? 0 : (size_t)16 * MT * D * 2));
  const uint32_t q_base = smem_u32(q_smem);

  auto load_tile = [&](int it) {
    const int s = it % kStages;
    const uint32_t kb = stage0 + s * 2 * kStage, vb = kb + kStage;
    const int piece = tid % PPR, row0 = tid / PPR;
    TokenAt a[STEPS];
#pragma unroll
    for (int j = 0; j < STEPS; ++j) a[j] = attend_token(p, lc, lc.t * kAttendTile + row0 + j * RPI, err);
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const int row = row0 + j * RPI;
      const bool ok = a[j].pos >= 0;
      const uint32_t d = tile_off<D>(row, piece);
      cp_async16(kb + d, p.k + a[j].off + piece * 16, ok);
      cp_async16(vb + d, p.v + a[j].off + piece * 16, ok);
      if (piece == 0) {
        kpos[s][row] = a[j].pos;
        if (!ok) bad_tile[s] = it;  // some token of this tile is masked for everybody
      }
    }
    attend_advance(p, lc, kAttendTile, ROWS);
  };

  for (int it = 0; it < kStages - 1; ++it) {
    if (it < count) load_tile(it);
    cp_async_commit();
  }

  uint32_t qf[QREG ? D / 16 : 1][4];
  float o[D / 8][4];
  float m[2], l[2];
  unsigned long long word[2];
  bool fresh = true;
  int t_begin = 0;

  for (int it = 0; it < count; ++it) {
    if (fresh) {
      // ---- a new segment: its query rows to shared memory and registers
      fresh = false;
      t_begin = c.t;
      __syncthreads();  // the join scratch shares the place
      const int R = c.r.n * p.g;
      for (int x = tid; x < 16 * MT * PPR; x += kAttendThreads) {
        const int row = x / PPR, piece = x % PPR;
        const int r = c.rt * ROWS + row;
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (row < ROWS && r < R) {
          const int i = r / p.g, j = r - i * p.g;
          w = *reinterpret_cast<const uint4*>(p.q + (long long)(c.r.q0 + i) * p.q_ts + (long long)(c.h * p.g + j) * p.q_hs + piece * 8);
        }
        *reinterpret_cast<uint4*>(q_smem + tile_off<D>(row, piece)) = w;
      }
      __syncthreads();
      if constexpr (QREG) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          ldsm_x4(qf[k], q_base + tile_off<D>(wr * 16 + (lane & 15), k * 2 + (lane >> 4)));
        // the join scratch overwrites Q only after the barrier at the end of the segment
      }
#pragma unroll
      for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m[x] = -INFINITY;
        l[x] = 0.f;
        const int row = wr * 16 + (lane >> 2) + 8 * x;
        word[x] = row < ROWS ? attend_word(p, c.r, (c.rt * ROWS + row) / p.g) : 0ull;
      }
    }
    cp_async_wait<kStages - 2>();
    __syncthreads();
    if (it + kStages - 1 < count) load_tile(it + kStages - 1);
    cp_async_commit();

    const int s = it % kStages;
    const uint32_t kb = stage0 + s * 2 * kStage, vb = kb + kStage;
    const int key0 = wk * KW;
    // ---- S = Q K^T
    float sc[KW / 8][4];
#pragma unroll
    for (int j = 0; j < KW / 8; ++j) {
      sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        uint32_t kf[4];
        ldsm_x4(kf, kb + tile_off<D>(key0 + j * 8 + (lane & 7), k * 4 + (lane >> 3)));
        if constexpr (QREG) {
          mma_bf16(sc[j], qf[2 * k], kf[0], kf[1]);
          mma_bf16(sc[j], qf[2 * k + 1], kf[2], kf[3]);
        } else {
          uint32_t a0[4], a1[4];
          ldsm_x4(a0, q_base + tile_off<D>(wr * 16 + (lane & 15), k * 4 + (lane >> 4)));
          ldsm_x4(a1, q_base + tile_off<D>(wr * 16 + (lane & 15), k * 4 + 2 + (lane >> 4)));
          mma_bf16(sc[j], a0, kf[0], kf[1]);
          mma_bf16(sc[j], a1, kf[2], kf[3]);
        }
      }
    }
    // ---- masks: only tiles that reach the drafted tokens, the end, or an unusable block
    const int ctx = c.r.T - c.r.n;
    if (p.block_list != nullptr || c.t * kAttendTile + kAttendTile > ctx || bad_tile[s] == it) {
#pragma unroll
      for (int j = 0; j < KW / 8; ++j) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int pos = kpos[s][key0 + j * 8 + (lane & 3) * 2 + (x & 1)];
          const int d = pos - ctx;
          const bool sees = pos >= 0 && (d < 0 || ((word[x >> 1] >> d) & 1ull));
          if (!sees) sc[j][x] = -INFINITY;
        }
      }
    }
    // ---- running maximum and sum
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < KW / 8; ++j) {
      mx[0] = fmaxf(mx[0], fmaxf(sc[j][0], sc[j][1]));
      mx[1] = fmaxf(mx[1], fmaxf(sc[j][2], sc[j][3]));
    }
    float base[2];
    bool grew = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
      mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
      const float mn = fmaxf(m[x], fmaf(mx[x], p.scale_log2, (float)ceil_log2(c.r.vlen)));
      grew = grew || mn > m[x];
      base[x] = mn == -INFINITY ? 0.f : mn;
      mx[x] = mn;
    }
    if (__any_sync(0xffffffffu, grew)) {
      const float a0 = ex2(m[0] - base[0]);
      const float a1 = SPLIT_P ? a0 : ex2(m[1] - base[1]);
      l[0] *= a0;
      l[1] *= a1;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] *= a0;
        o[j][1] *= a0;
        o[j][2] *= a1;
        o[j][3] *= a1;
      }
      m[0] = mx[0];
      m[1] = mx[1];
    }
    // ---- a hidden token's value must not reach a row through 0 * inf: infinities and NaN of the query's own tokens
    // go to the rows that see them here, and are zero in the product
    if ((p.tree != nullptr || c.r.n > 1) && (p.block_list != nullptr || c.t * kAttendTile + kAttendTile > ctx)) {
      const int piece = tid % PPR, row0 = tid / PPR;
      const uint4* vrow = reinterpret_cast<const uint4*>(smem + (vb - stage0));
      bool odd = false;
#pragma unroll 1
      for (int j = 0; j < STEPS; ++j)
        if (kpos[s][row0 + j * RPI] >= ctx) odd = odd || has_nonfinite(vrow[tile_off<D>(row0 + j * RPI, piece) >> 4]);
      if (__syncthreads_or(odd)) {
#pragma unroll 1
        for (int key = key0; key < key0 + KW; ++key) {
          const int d = kpos[s][key] - ctx;
          if (d < 0) continue;
#pragma unroll
          for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
            if (!((word[x] >> d) & 1ull)) continue;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(smem + (vb - stage0) + tile_off<D>(key, j) + (lane & 3) * 4);
              const float2 e = bf16x2_to_float2(w);
              if (!isfinite(e.x)) o[j][2 * x] += e.x;
              if (!isfinite(e.y)) o[j][2 * x + 1] += e.y;
            }
          }
        }
        __syncthreads();
#pragma unroll 1
        for (int j = 0; j < STEPS; ++j) {
          if (kpos[s][row0 + j * RPI] < ctx) continue;
          uint4* w = reinterpret_cast<uint4*>(smem + (vb - stage0) + tile_off<D>(row0 + j * RPI, piece));
          *w = zero_nonfinite(*w);
        }
        __syncthreads();
      }
    }
    // ---- P, and O += P V
#pragma unroll
    for (int kk = 0; kk < KW / 16; ++kk) {
      uint32_t pf[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* e = sc[kk * 2 + h];
        const float p0 = ex2(fmaf(e[0], p.scale_log2, -base[0])), p1 = ex2(fmaf(e[1], p.scale_log2, -base[0]));
        l[0] += p0 + p1;
        pf[h * 2] = pack_bf16(p0, p1);
        if constexpr (SPLIT_P) {
          const float2 hi = bf16x2_to_float2(pf[h * 2]);
          pf[h * 2 + 1] = pack_bf16(p0 - hi.x, p1 - hi.y);
        } else {
          const float p2 = ex2(fmaf(e[2], p.scale_log2, -base[1])), p3 = ex2(fmaf(e[3], p.scale_log2, -base[1]));
          l[1] += p2 + p3;
          pf[h * 2 + 1] = pack_bf16(p2, p3);
        }
      }
      const uint32_t a[4] = {pf[0], pf[1], pf[2], pf[3]};
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t vf[4];
        ldsm_x4_t(vf, vb + tile_off<D>(key0 + kk * 16 + (lane & 15), j * 2 + (lane >> 4)));
        mma_bf16(o[2 * j], a, vf[0], vf[1]);
        mma_bf16(o[2 * j + 1], a, vf[2], vf[3]);
      }
    }

    // ---- end of the segment, or of this CTA's run
    const bool seg_end = c.t + 1 == c.r.tiles;
    if (seg_end || it + 1 == count) {
      const bool whole = seg_end && t_begin == 0;
      if constexpr (SPLIT_P) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[j][0] = add_remainder(o[j][0], o[j][2]);
          o[j][1] = add_remainder(o[j][1], o[j][3]);
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      }
      if constexpr (WK > 1) {
        // the warps that share rows agree on the maximum, then add their parts up in turn
        if ((lane & 3) == 0) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            join_ml[wid][(lane >> 2) + 8 * x][0] = m[x];
            join_ml[wid][(lane >> 2) + 8 * x][1] = l[x];
          }
        }
        __syncthreads();
        float f[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = (lane >> 2) + 8 * x;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < WK; ++w) top = fmaxf(top, join_ml[w * MT + wr][row][0]);
          const float b0 = top == -INFINITY ? 0.f : top;
          f[x] = ex2(m[x] - b0);
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < WK; ++w) sum += join_ml[w * MT + wr][row][1] * ex2(join_ml[w * MT + wr][row][0] - b0);
          m[x] = top;
          l[x] = sum;
        }
        for (int w = 1; w < WK; ++w) {
          if (wk == w) {
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
#pragma unroll
              for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
                float2* d = reinterpret_cast<float2*>(join + (wr * 16 + (lane >> 2) + 8 * x) * D + j * 8 + (lane & 3) * 2);
                float2 v = make_float2(o[j][2 * x] * f[x], o[j][2 * x + 1] * f[x]);
                if (w > 1) {
                  const float2 u = *d;
                  v.x += u.x;
                  v.y += u.y;
                }
                *d = v;
              }
            }
          }
          __syncthreads();
        }
        if (wk == 0) {
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
#pragma unroll
            for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
              const float2 u = *reinterpret_cast<const float2*>(join + (wr * 16 + (lane >> 2) + 8 * x) * D + j * 8 + (lane & 3) * 2);
              o[j][2 * x] = fmaf(o[j][2 * x], f[x], u.x);
              o[j][2 * x + 1] = fmaf(o[j][2 * x + 1], f[x], u.y);
            }
          }
        }
      }
      if (wk == 0) {
        const int slot = 2 * (int)blockIdx.x + (t_begin > 0 ? 0 : 1);
#pragma unroll
        for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
          const int row = wr * 16 + (lane >> 2) + 8 * x;
          const int r = c.rt * ROWS + row;
          if (r >= c.r.n * p.g) continue;
          if (whole) {
            const int i = r / p.g, hq = c.h * p.g + (r - i * p.g);
            const float inv = l[x] > 0.f ? 1.f / l[x] : l[x];  // a NaN sum stays one
            uint16_t* dst = p.out + (long long)(c.r.q0 + i) * p.o_ts + (long long)hq * p.o_hs;
#pragma unroll
            for (int j = 0; j < D / 8; ++j)
              *reinterpret_cast<uint32_t*>(dst + j * 8 + (lane & 3) * 2) = pack_bf16(o[j][2 * x] * inv, o[j][2 * x + 1] * inv);
            if ((lane & 3) == 0) p.lse[(long long)(c.r.q0 + i) * (p.Hkv * p.g) + hq] = (m[x] + log2f(l[x])) * kLn2;
          } else {
            float* dst = p.part_o + ((long long)slot * ROWS + row) * D;
#pragma unroll
            for (int j = 0; j < D / 8; ++j)
              *reinterpret_cast<float2*>(dst + j * 8 + (lane & 3) * 2) = make_float2(o[j][2 * x], o[j][2 * x + 1]);
            if ((lane & 3) == 0)
              *reinterpret_cast<float2*>(p.part_ml + ((long long)slot * ROWS + row) * 2) = make_float2(m[x], l[x]);
          }
        }
      }
      fresh = true;
    }
    attend_advance(p, c, kAttendTile, ROWS);
  }
  if (err) flag_status(p.status, err);
}

// Joins the parts of segments that several CTAs worked on.  One CTA per (request, KV head, 8 rows); a warp takes a row, or -
// fewer rows than warps - a share of a row's parts, visited in the order of the tokens and joined in a fixed one.
// Everything that depends on lengths alone runs before the wait for the attention kernel, which releases this one
// early: by then its own predecessors are complete.
constexpr int kCombineThreads = 256;
template <int D>
__global__ void __launch_bounds__(kCombineThreads) attend_combine_kernel(const __grid_constant__ AttendParams p,
                                                                         const int runs, const int tile, const int rows) {
  constexpr int V = D / 32;  // columns per lane
  constexpr int WARPS = kCombineThreads / 32;
  __shared__ long long red[WARPS];
  __shared__ float part[WARPS][D];
  __shared__ float part_ml[WARPS][2];
  unsigned err = 0u;
  const int chunks = (rows + WARPS - 1) / WARPS;  // CTAs per row tile
  const int b = blockIdx.z, h = blockIdx.y, rt = (int)blockIdx.x / chunks;
  const int first_row = ((int)blockIdx.x - rt * chunks) * WARPS;
  const AttendReq r = attend_req(p, b, tile, rows, err);
  int i0 = 0, i1 = 0;
  if (rt < r.row_tiles) {
    long long before, W;
    if (p.B <= 32) {
      AttendReq mine{};
      W = attend_scan32(p, tile, rows, mine, before, err);
      before = __shfl_sync(0xffffffffu, before, b);
    } else {
      before = attend_work_before<kCombineThreads>(p, b, tile, rows, err, red);
      W = attend_work_before<kCombineThreads>(p, p.B, tile, rows, err, red);
    }
    const long long s0 = before + (long long)rt * r.tiles;
    const int J = attend_runs(runs, W, p.min_tiles);
    i0 = attend_owner(W, J, s0);
    i1 = attend_owner(W, J, s0 + r.tiles - 1);
  }
  grid_dependency_wait();
  trigger_dependents();
  const int live = min(min(WARPS, rows - first_row), r.n * p.g - rt * rows - first_row);
  if (i0 == i1 || live <= 0) return;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int share = WARPS / live;  // warps per row
  const int mine = wid / share, turn = wid - mine * share;
  const int parts = i1 - i0 + 1;
  const int from = i0 + (int)((long long)parts * turn / share), to = i0 + (int)((long long)parts * (turn + 1) / share);
  const int row = first_row + mine;
  const bool on = mine < live;
  float acc[V], l = 0.f, top = -INFINITY;
#pragma unroll
  for (int x = 0; x < V; ++x) acc[x] = 0.f;
  if (on) {
    for (int i = from + lane; i < to; i += 32) top = fmaxf(top, p.part_ml[((long long)(2 * (i * p.Hkv + h) + (i == i0)) * rows + row) * 2]);
#pragma unroll
    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
    for (int i = from; i < to; ++i) {
      const long long at = (long long)(2 * (i * p.Hkv + h) + (i == i0)) * rows + row;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
      const float f = ex2(ml.x - base);
      l = fmaf(ml.y, f, l);
      const float* src = p.part_o + at * D + lane * V;
      if constexpr (V % 4 == 0) {
#pragma unroll
        for (int x = 0; x < V; x += 4) {
          const float4 u = *reinterpret_cast<const float4*>(src + x);
          acc[x] = fmaf(u.x, f, acc[x]);
          acc[x + 1] = fmaf(u.y, f, acc[x + 1]);
          acc[x + 2] = fmaf(u.z, f, acc[x + 2]);
          acc[x + 3] = fmaf(u.w, f, acc[x + 3]);
        }
      } else {
        const float2 u = *reinterpret_cast<const float2*>(src);
        acc[0] = fmaf(u.x, f, acc[0]);
        acc[1] = fmaf(u.y, f, acc[1]);
      }
    }
  }
  if (share > 1) {
#pragma unroll
    for (int x = 0; x < V; ++x) part[wid][lane * V + x] = acc[x];
    if (lane == 0) {
      part_ml[wid][0] = top;
      part_ml[wid][1] = l;
    }
    __syncthreads();
    if (turn == 0 && on) {
      const float mine_top = top;
      for (int w = 1; w < share; ++w) top = fmaxf(top, part_ml[wid + w][0]);
      const float base = top == -INFINITY ? 0.f : top;
      const float f0 = ex2(mine_top - base);
      l *= f0;
#pragma unroll
      for (int x = 0; x < V; ++x) acc[x] *= f0;
      for (int w = 1; w < share; ++w) {
        const float f = ex2(part_ml[wid + w][0] - base);
        l = fmaf(part_ml[wid + w][1], f, l);
#pragma unroll
        for (int x = 0; x < V; ++x) acc[x] = fmaf(part[wid + w][lane * V + x], f, acc[x]);
      }
    }
  }
  if (on && turn == 0) {
    const int rr = rt * rows + row, i = rr / p.g, hq = h * p.g + (rr - i * p.g);
    const float inv = l > 0.f ? 1.f / l : l;
    uint16_t* dst = p.out + (long long)(r.q0 + i) * p.o_ts + (long long)hq * p.o_hs + lane * V;
#pragma unroll
    for (int x = 0; x < V; x += 2) *reinterpret_cast<uint32_t*>(dst + x) = pack_bf16(acc[x] * inv, acc[x + 1] * inv);
    if (lane == 0) p.lse[(long long)(r.q0 + i) * (p.Hkv * p.g) + hq] = (top + log2f(l)) * kLn2;
  }
}

// ------------------------------------------------------------------------------------------ weight sums
// sums[t] (+)= sum over the rows of the KV head's group of exp(s[r, t] - lse_r).  The output's softmax statistics are
// complete only after the last tile, so the weights are formed in a second pass over K (not V): S^T = K Q^T with the
// tokens as the rows of the product, so that a token's sum over query rows stays inside four lanes.  Every (token, KV head)
// belongs to one CTA: no atomics, results repeat bit for bit.  A token of the query itself starts at 0 (its slot
// may hold an earlier owner's sum), an older one keeps its sum unless the call starts the sums anew.  This kernel serves the
// caches that no tensor map describes; the others take attend_observe_mma_kernel.
constexpr int kObserveRows = 128;  // query rows in shared memory at a time
template <int D>
constexpr size_t observe_smem_bytes() { return (size_t)kAttendStages<D> * kAttendStageBytes<D> + (size_t)kObserveRows * D * 2; }

template <int D>
__global__ void __launch_bounds__(kAttendThreads) attend_observe_kernel(const __grid_constant__ AttendParams p, const int runs) {
  constexpr int PPR = D / 8, RPI = kAttendThreads / PPR, STEPS = kAttendTile / RPI;
  constexpr int kStages = kAttendStages<D>;
  constexpr int kAll = 1 << 24;  // one row tile per segment: all rows of a (request, KV head)
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int kpos[kStages][kAttendTile];
  __shared__ long long kadr[kStages][kAttendTile];  // index of the token's sum
  __shared__ AttendPlanShared<kAttendThreads> plan;
  __shared__ float lse2[kObserveRows];
  __shared__ unsigned long long words[kObserveRows];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  grid_dependency_wait();
  unsigned err = 0u;
  const int run = (int)blockIdx.x / p.Hkv;
  AttendCursor lc;
  int count;
  if (!attend_plan_run<kAttendThreads>(p, runs, 1, run, kAttendTile, kAll, plan, lc, count)) return;
  lc.h = (int)blockIdx.x - run * p.Hkv;
  AttendCursor c = lc;
  const uint32_t stage0 = smem_u32(smem);
  constexpr uint32_t kStage = kAttendStageBytes<D>;
  unsigned char* q_smem = smem + kStages * kStage;
  const uint32_t q_base = smem_u32(q_smem);

  auto load_tile = [&](int it) {
    const int s = it % kStages;
    const uint32_t kb = stage0 + s * kStage;
    const int piece = tid % PPR, row0 = tid / PPR;
    TokenAt a[STEPS];
#pragma unroll
    for (int j = 0; j < STEPS; ++j) a[j] = attend_token(p, lc, lc.t * kAttendTile + row0 + j * RPI, err);
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const int row = row0 + j * RPI;
      cp_async16(kb + tile_off<D>(row, piece), p.k + a[j].off + piece * 16, a[j].pos >= 0);
      if (piece == 0) {
        kpos[s][row] = a[j].pos;
        long long at = 0;
        if (a[j].pos >= 0) {
          const int lb = a[j].pos / p.bs;
          at = ((long long)p.block_table[(long long)lc.b * p.max_blocks + lb] * p.Hkv + lc.h) * p.bs + (a[j].pos - lb * p.bs);
        }
        kadr[s][row] = at;
      }
    }
    attend_advance(p, lc, kAttendTile, kAll);
  };
  auto load_rows = [&](int r0) {
    const int R = c.r.n * p.g;
    for (int x = tid; x < kObserveRows * PPR; x += kAttendThreads) {
      // (rows up to a multiple of 8 repeat the last one: a zero row times an infinite key would be NaN, and stay it)
      const int row = x / PPR, piece = x % PPR, r = min(r0 + row, R - 1);
      if (row >= ((min(R - r0, kObserveRows) + 7) & ~7)) break;
      const int i = r / p.g, j = r - i * p.g;
      const uint4 w = *reinterpret_cast<const uint4*>(p.q + (long long)(c.r.q0 + i) * p.q_ts + (long long)(c.h * p.g + j) * p.q_hs + piece * 8);
      *reinterpret_cast<uint4*>(q_smem + tile_off<D>(row, piece)) = w;
    }
    for (int row = tid; row < kObserveRows; row += kAttendThreads) {
      const int r = r0 + row;
      float z = INFINITY;  // rows that do not exist, or see nothing, add exp2(-inf) = 0
      unsigned long long w = 0ull;
      if (r < R) {
        const int i = r / p.g, j = r - i * p.g;
        const float e = p.lse[(long long)(c.r.q0 + i) * (p.Hkv * p.g) + c.h * p.g + j];
        if (e != -INFINITY) z = e * kLog2e;
        w = attend_word(p, c.r, i);
      }
      lse2[row] = z;
      words[row] = w;
    }
  };

  for (int it = 0; it < kStages - 1; ++it) {
    if (it < count) load_tile(it);
    cp_async_commit();
  }
  bool fresh = true;
  for (int it = 0; it < count; ++it) {
    const int R = c.r.n * p.g;
    if (fresh) {
      __syncthreads();
      load_rows(0);
      fresh = false;
    }
    cp_async_wait<kStages - 2>();
    __syncthreads();
    if (it + kStages - 1 < count) load_tile(it + kStages - 1);
    cp_async_commit();
    const int s = it % kStages;
    const uint32_t kb = stage0 + s * kStage;
    uint32_t kf[D / 16][4];
#pragma unroll
    for (int k = 0; k < D / 16; ++k) ldsm_x4(kf[k], kb + tile_off<D>(wid * 16 + (lane & 15), k * 2 + (lane >> 4)));
    const int ctx = c.r.T - c.r.n;
    const int d0 = kpos[s][wid * 16 + (lane >> 2)] - ctx, d1 = kpos[s][wid * 16 + (lane >> 2) + 8] - ctx;
    float w0 = 0.f, w1 = 0.f;
    for (int r0 = 0; r0 < R; r0 += kObserveRows) {
      if (R > kObserveRows && (r0 > 0 || it > 0)) {
        __syncthreads();
        load_rows(r0);
        __syncthreads();
      }
      const int nt = (min(R - r0, kObserveRows) + 7) >> 3;
      for (int j = 0; j < nt; ++j) {
        float e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          uint32_t qf[4];
          ldsm_x4(qf, q_base + tile_off<D>(j * 8 + (lane & 7), k * 4 + (lane >> 3)));
          mma_bf16(e, kf[2 * k], qf[0], qf[1]);
          mma_bf16(e, kf[2 * k + 1], qf[2], qf[3]);
        }
        const int row = j * 8 + (lane & 3) * 2;
        const float z0 = lse2[row], z1 = lse2[row + 1];
        float p0 = ex2(fmaf(e[0], p.scale_log2, -z0)), p1 = ex2(fmaf(e[1], p.scale_log2, -z1));
        float p2 = ex2(fmaf(e[2], p.scale_log2, -z0)), p3 = ex2(fmaf(e[3], p.scale_log2, -z1));
        if (d0 >= 0 || d1 >= 0) {
          const unsigned long long u0 = words[row], u1 = words[row + 1];
          if (d0 >= 0) {
            p0 = (u0 >> d0) & 1ull ? p0 : 0.f;
            p1 = (u1 >> d0) & 1ull ? p1 : 0.f;
          }
          if (d1 >= 0) {
            p2 = (u0 >> d1) & 1ull ? p2 : 0.f;
            p3 = (u1 >> d1) & 1ull ? p3 : 0.f;
          }
        }
        w0 += p0 + p1;
        w1 += p2 + p3;
      }
    }
    w0 += __shfl_xor_sync(0xffffffffu, w0, 1);
    w0 += __shfl_xor_sync(0xffffffffu, w0, 2);
    w1 += __shfl_xor_sync(0xffffffffu, w1, 1);
    w1 += __shfl_xor_sync(0xffffffffu, w1, 2);
    if ((lane & 3) == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = wid * 16 + (lane >> 2) + 8 * x;
        if (kpos[s][row] < 0) continue;
        const bool old = p.reset_sums == 0 && (x ? d1 : d0) < 0;
        float* d = p.sums + kadr[s][row];
        *d = (x ? w1 : w0) + (old ? *d : 0.f);
      }
    }
    fresh = c.t + 1 == c.r.tiles;
    attend_advance(p, c, kAttendTile, kAll);
  }
  if (err) flag_status(p.status, err);
}

}  // namespace triattn
