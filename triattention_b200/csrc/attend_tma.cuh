// Attention over the paged cache, cache tiles brought in by tiled TMA: the ring of tiles, and the kernel for few query
// rows (at most 16 per KV head: decode steps and small trees).
//
// The layer's K and V are rank-5 tensor maps (64 channels, token mod 8, 64-channel part, token / 8 in the block, head slot)
// with the 128-byte swizzle, a head slot being one (block, KV head) pair; one box is up to TILE tokens of one head of one
// block, all channels, and a tile arrives as [8-token group][D / 64][8 tokens][128 B]: ldmatrix reads it without
// bank conflicts and tcgen05.mma takes it as an operand.  (Boxes of 64 channels, half the size, streamed at 60 % of the
// bandwidth: the loads are bound by their number.)  One producer warp walks the CTA's run of
// tiles (see attend.cuh for how the runs are cut), looks block ids up a batch ahead, and refills a stage as soon as its
// readers have left it.  Block sizes that are multiples of 8 only: others take the kernel in attend.cuh.
#pragma once

#include <cuda.h>  // CUtensorMap

#include "attend.cuh"

namespace triattn {

__device__ __forceinline__ void tma_load_tokens(uint32_t dst, const CUtensorMap* map, uint32_t bar, int group, int slot, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %3, %3, %4, %5}], "
      "[%2], %6;"
      ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(group), "r"(slot), "l"(policy)
      : "memory");
}

// What the call does not read again leaves the L2 first, so that parts, sums and keys that it does read again stay: a tree of 26
// on 4 x 6600 tokens 60 -> 56 us on the device, the end of a prompt with weight sums (K read twice) 71 -> 65, decode of 64 x 2112 tokens
// 100 -> 97, a tree of 64 on 8 x 32768 tokens 303 -> 300.
__device__ __forceinline__ uint64_t l2_policy(bool read_again) {
  uint64_t once, keep;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(keep));
  return read_again ? keep : once;
}

// the descriptor of a kernel parameter into the descriptor cache, ahead of the first load
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// byte offset of 16-byte piece `piece` (0 .. D / 8 - 1) of token row `row` in a [tokens / 8][D / 64][8][128 B] swizzled tile
template <int D>
__device__ __forceinline__ uint32_t swz_off(int row, int piece) {
  return (uint32_t)((row >> 3) * (D * 16) + (piece >> 3) * 1024 + (row & 7) * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

// A ring of K/V tiles in shared memory.  pos[tile % kPosRing][i]: logical position of the first token of the tile's i-th run of
// 8 tokens, -1 where there is none (behind the sequence, an unused list entry, a block outside the cache): such runs
// are not loaded.  The positions are written a batch of up to kBatch tiles at a time, so their ring is deeper: at most
// STAGES + kBatch + 1 tiles are between the last one read and the last one written.
template <int TILE>
constexpr int kPosRing = TILE == 128 ? 16 : 64;
template <int TILE>
constexpr int kBatch = kPosRing<TILE> / 2;
template <int TILE, int STAGES, bool BLOCKS = false>
struct AttendRing {
  static constexpr bool kBlocks = BLOCKS;
  static_assert(STAGES + kBatch<TILE> + 2 <= kPosRing<TILE>, "positions of tiles still being read would be overwritten");
  uint64_t full[2][STAGES], empty[2][STAGES];  // K and V; the kernel for few rows has one pair for both
  int pos[kPosRing<TILE>][TILE / 8];
  int blk[BLOCKS ? kPosRing<TILE> : 1][TILE / 8];  // the cache block each run lies in, for who asks
  int gaps;  // not 0: a block outside the cache was met (its tokens are not there)
  int err;
};

// A wait of the whole warp; on a timeout the CTA's error flag is raised, and every later wait returns at once.
__device__ __forceinline__ bool ring_wait(uint64_t& bar, uint32_t parity, int* err, uint32_t* status) {
  const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&bar), parity, err));
  if (!ok && (threadIdx.x & 31) == 0) {
    if (*(volatile int*)err == 0) flag_status(status, TRIATTN_DEV_WAIT_TIMEOUT);
    *(volatile int*)err = 1;
  }
  return ok;
}

// The same for a single thread.
__device__ __forceinline__ bool thread_wait(uint64_t& bar, uint32_t parity, int* err, uint32_t* status) {
  const bool ok = mbar_try_wait(smem_u32(&bar), parity) || mbar_wait_bounded(smem_u32(&bar), parity, err);
  if (!ok) {
    if (*(volatile int*)err == 0) flag_status(status, TRIATTN_DEV_WAIT_TIMEOUT);
    *(volatile int*)err = 1;
  }
  return ok;
}

// A producer warp: K (which = 0) or V (1) of tiles 0 .. count - 1 of the run that starts at `c`; stage s is at
// dst + s * stride, its barriers are full[s] and empty[s].  Of `turns` warps that share the work, warp `turn` loads every
// turns-th tile.
// Two warps, because a warp spends some 400 cycles on a tile - waiting for the stage, arming its barrier and above all
// issuing the loads - while the SM's share of the bandwidth moves a 16 KB tile in 700.
template <int D, int TILE, int STAGES, class Ring>
__device__ __forceinline__ void attend_produce(const AttendParams& p, const CUtensorMap* map, int which, AttendCursor c,
                                               int count, int rows_per_tile, uint32_t dst, uint32_t stride,
                                               uint64_t* full, uint64_t* empty, Ring& ring, bool read_again,
                                               int turn = 0, int turns = 1) {
  const int lane = threadIdx.x & 31;
  const int boxes = TILE / p.box;
  const int my_tile = lane / boxes, my_box = lane - my_tile * boxes;
  const uint32_t box_bytes = (uint32_t)p.box * D * 2;
  const uint64_t policy = l2_policy(read_again);
  unsigned err = 0u;
  // The warp looks 32 boxes up at a time, one per lane (the next 32 / boxes tiles of the segment), a batch ahead of the
  // loads: a look-up is one or two dependent global loads, as long as a tile's transfer.
  struct Batch {
    int blk, in, pos, head, tiles;
  };
  auto look_up = [&](int left) {
    Batch u{0, 0, -1, c.h, min(min(min(32 / boxes, kBatch<TILE>), c.r.tiles - c.t), left)};
    const int vp = (c.t + my_tile) * TILE + my_box * p.box;
    if (my_tile < u.tiles && vp < c.r.vlen) {
      int lb = vp / p.bs;
      u.in = vp - lb * p.bs;
      bool ok = true;
      if (p.block_list != nullptr) {
        lb = p.block_list[((long long)c.b * p.Hkv + c.h) * p.num_listed + lb];
        ok = lb >= 0;
        if (lb >= (c.r.T + p.bs - 1) / p.bs) {
          err |= TRIATTN_DEV_BAD_KEEP_INDEX;
          ok = false;
        }
      }
      if (ok && lb * p.bs + u.in < c.r.T) {
        u.blk = p.block_table[(long long)c.b * p.max_blocks + lb];
        u.pos = lb * p.bs + u.in;
      }
    }
    c.t += u.tiles - 1;
    if (left > u.tiles) attend_advance(p, c, TILE, rows_per_tile);
    return u;
  };
  Batch next = look_up(count);
  int it = 0, seen = next.tiles;  // tiles issued, tiles looked up
  int s = 0;
  uint32_t phase = 1u;  // of the stage's previous release (the first round passes at once)
  bool stop = false;
  while (it < count && !stop) {
    Batch u = next;
    if (seen < count) {
      next = look_up(count - seen);
      seen += next.tiles;
    }
    if (u.pos >= 0 && (unsigned)u.blk >= (unsigned)p.num_blocks) {
      err |= TRIATTN_DEV_BAD_BLOCK_ID;
      u.pos = -1;
      *(volatile int*)&ring.gaps = 1;
    }
    if (which == 0 && my_tile < u.tiles && (it + my_tile) % turns == turn)
      for (int i = 0; i < p.box; i += 8) {
        ring.pos[(it + my_tile) % kPosRing<TILE>][(my_box * p.box + i) >> 3] = u.pos < 0 ? -1 : u.pos + i;
        if constexpr (Ring::kBlocks) ring.blk[(it + my_tile) % kPosRing<TILE>][(my_box * p.box + i) >> 3] = u.blk;
      }
    __syncwarp();  // before lane 0 arrives for the batch's tiles
    const unsigned live = __ballot_sync(0xffffffffu, u.pos >= 0);
    const int slot = u.blk * p.slots_per_block + u.head, group = u.in >> 3;
    const uint32_t at = dst + (uint32_t)my_box * box_bytes;
    for (int j = 0; j < u.tiles; ++j, ++it) {
      if (turns == 1 || it % turns == turn) {
        if (it >= STAGES && !ring_wait(empty[s], phase, &ring.err, p.status)) {
          stop = true;
          break;
        }
        fence_proxy_async();  // the readers' accesses (acquired above) before the refill
        const uint32_t bar = smem_u32(&full[s]);
        if (lane == 0)
          mbar_arrive_expect_tx(bar, (uint32_t)__popc((live >> (j * boxes)) & ((1u << boxes) - 1u)) * box_bytes + kTestExtraTxBytes);
        __syncwarp();
        if (my_tile == j && u.pos >= 0) tma_load_tokens(at + (uint32_t)s * stride, map, bar, group, slot, policy);
      }
      if (++s == STAGES) {
        s = 0;
        phase ^= 1u;
      }
    }
  }
  if (err) flag_status(p.status, err);
  // after a timeout: nothing may still be landing when the CTA retires
  if (*(volatile int*)&ring.err != 0)
    for (int j = max(0, it - STAGES); j < it; ++j)
      if (j % turns == turn) mbar_wait_bounded(smem_u32(&full[j % STAGES]), (uint32_t)(j / STAGES) & 1u);
}

// ------------------------------------------------------------------------------------------ few query rows
constexpr int kDecodeWarps = 6;   // consumer warps; a stage always belongs to the same warp (STAGES is a multiple)
constexpr int kDecodeThreads = (kDecodeWarps + 2) * 32;
template <int D>
constexpr int kDecodeTile = D == 64 ? 64 : 32;  // 16 KB (D = 256: 32 KB) of K and V
template <int D>
constexpr int kDecodeStages = D == 256 ? 6 : 12;  // 192 KB
template <int D, bool SPLIT_P>
constexpr size_t decode_smem_bytes() {
  return 1024 + (size_t)kDecodeStages<D> * 2 * kDecodeTile<D> * D * 2 + (size_t)(SPLIT_P && D <= 128 ? kDecodeWarps : 1) * (SPLIT_P ? 8 : 16) * D * 4;
}

// Rows are padded to the 16 of mma.sync; a tile is one warp's business from arrival to release, so tiles of different
// warps overlap without any barrier, and the warps meet only where a segment (or the CTA's run) ends.  mma.sync, not
// tcgen05: with at most 16 live rows a tile's products take a fifth of the time its bytes need.  Bound by HBM: 64 requests of 2112
// tokens, 8 KV heads, head dimension 128, in 96 us, 5.8 TB/s (88 % of the measured copy).
// SPLIT_P (at most 8 rows): P goes into the product with V as bf16 and bf16 remainder, the remainders in the operand's rows that would be
// padding.  With 9 to 16 rows there is no padding left and P is one bf16: the output's error against 64 bits is then 2.3e-3 instead of 1.7e-3
// (its own rounding), inside the 2^-8 that a bf16 output allows; remainders would take every product with V twice.  16 rows: 124 us on
// the same tokens.
template <int D, bool SPLIT_P>
__global__ void __launch_bounds__(kDecodeThreads, 1)
    attend_decode_kernel(const __grid_constant__ AttendParams p, const __grid_constant__ CUtensorMap kmap,
                         const __grid_constant__ CUtensorMap vmap, const int runs) {
  constexpr int TILE = kDecodeTile<D>, STAGES = kDecodeStages<D>, WARPS = kDecodeWarps;
  static_assert(D / 8 <= 32, "a lane per 16-byte piece of a row");
  static_assert(STAGES % WARPS == 0, "a stage belongs to one warp: its barriers are never more than a phase ahead");
  constexpr int ROWS = SPLIT_P ? 8 : 16;
  constexpr uint32_t kTileBytes = TILE * D * 2;
  constexpr bool kAllAtOnce = SPLIT_P && D <= 128;  // join scratch for every warp, or one shared and taken in turn
  extern __shared__ unsigned char smem_raw[];
  __shared__ AttendRing<TILE, STAGES> ring;
  __shared__ AttendPlanShared<kDecodeThreads> plan;
  __shared__ float join_ml[WARPS][16][2];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&ring.full[0][s]), 2);  // the K and the V producer
      mbar_init(smem_u32(&ring.empty[0][s]), 1);
    }
    mbar_fence_init();
    ring.err = ring.gaps = 0;
    prefetch_map(&kmap);
    prefetch_map(&vmap);
  }
  grid_dependency_wait();
  trigger_dependents();
  const int run = (int)blockIdx.x / p.Hkv;
  AttendCursor c;
  int count;
  if (!attend_plan_run<kDecodeThreads>(p, runs, p.min_tiles, run, TILE, ROWS, plan, c, count)) return;
  c.h = (int)blockIdx.x - run * p.Hkv;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* const base_ptr = smem_raw + (base - smem_u32(smem_raw));
  float* const join = reinterpret_cast<float*>(base_ptr + STAGES * 2 * kTileBytes);

  if (wid >= WARPS) {
    attend_produce<D, TILE, STAGES>(p, wid == WARPS ? &kmap : &vmap, wid - WARPS, c, count, ROWS,
                                    base + (wid - WARPS) * kTileBytes, 2 * kTileBytes, ring.full[0], ring.empty[0], ring,
                                    wid == WARPS && p.sums != nullptr);
    return;
  }

  auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); };
  bool dead = false;  // a wait ran out: no more waits, no more arithmetic, but every barrier is kept
  for (int it = 0; it < count;) {
    const int t_begin = c.t;
    const int piece = min(c.r.tiles - c.t, count - it);
    const int R = c.r.n * p.g, ctx = c.r.T - c.r.n;
    // ---- this segment's query rows as the A operand: row lane / 4 (and + 8), columns 2 (lane % 4) + {0, 1, 8, 9}
    uint32_t qf[D / 16][SPLIT_P ? 2 : 4];
    unsigned long long word[2];
#pragma unroll
    for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
      const int r = c.rt * ROWS + (lane >> 2) + 8 * x;
      const bool ok = r < R;
      const int i = ok ? r / p.g : 0, j = ok ? r - i * p.g : 0;
      const uint16_t* src = p.q + (long long)(c.r.q0 + i) * p.q_ts + (long long)(c.h * p.g + j) * p.q_hs + (lane & 3) * 2;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t lo = ok ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
        const uint32_t hi = ok ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
        if constexpr (SPLIT_P) {
          qf[k][0] = lo;
          qf[k][1] = hi;
        } else {
          qf[k][x] = lo;
          qf[k][2 + x] = hi;
        }
      }
      word[x] = ok ? attend_word(p, c.r, i) : 0ull;
    }
    float o[D / 8][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    for (int x0 = (wid + WARPS - it % WARPS) % WARPS; x0 < piece; x0 += WARPS) {
      const int n = it + x0, s = n % STAGES;
      if (dead || !ring_wait(ring.full[0][s], (uint32_t)(n / STAGES) & 1u, &ring.err, p.status)) {
        dead = true;
        break;
      }
      const uint32_t kb = base + (uint32_t)s * 2 * kTileBytes, vb = kb + kTileBytes;
      // ---- S = Q K^T
      float sc[TILE / 8][4];
#pragma unroll
      for (int j = 0; j < TILE / 8; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
#pragma unroll
        for (int j = 0; j < TILE / 8; ++j) {
          uint32_t kf[4];
          ldsm_x4(kf, kb + swz_off<D>(j * 8 + (lane & 7), k * 4 + (lane >> 3)));
          if constexpr (SPLIT_P) {
            const uint32_t a0[4] = {qf[2 * k][0], 0u, qf[2 * k][1], 0u}, a1[4] = {qf[2 * k + 1][0], 0u, qf[2 * k + 1][1], 0u};
            mma_bf16(sc[j], a0, kf[0], kf[1]);
            mma_bf16(sc[j], a1, kf[2], kf[3]);
          } else {
            mma_bf16(sc[j], qf[2 * k], kf[0], kf[1]);
            mma_bf16(sc[j], qf[2 * k + 1], kf[2], kf[3]);
          }
        }
      }
      // ---- masks: tiles that reach the query's own tokens, the end, or a run of tokens that is not there
      int top_pos = -1, low_pos = 1;
#pragma unroll
      for (int j = 0; j < TILE / 8; ++j) {
        const int q8 = ring.pos[n % kPosRing<TILE>][j];
        top_pos = max(top_pos, q8);
        low_pos = min(low_pos, q8);
      }
      const bool edge = low_pos < 0 || top_pos + 8 > ctx;
      if (edge) {
#pragma unroll
        for (int j = 0; j < TILE / 8; ++j) {
          const int q8 = ring.pos[n % kPosRing<TILE>][j];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int pos = q8 + (lane & 3) * 2 + (x & 1), d = pos - ctx;
            const bool sees = q8 >= 0 && pos < c.r.T && (d < 0 || ((word[x >> 1] >> d) & 1ull));
            if (!sees) sc[j][x] = -INFINITY;
          }
        }
      }
      // ---- running maximum and sum
      float mx[2] = {-INFINITY, -INFINITY}, mbase[2];
#pragma unroll
      for (int j = 0; j < TILE / 8; ++j) {
        mx[0] = fmaxf(mx[0], fmaxf(sc[j][0], sc[j][1]));
        if constexpr (!SPLIT_P) mx[1] = fmaxf(mx[1], fmaxf(sc[j][2], sc[j][3]));
      }
      bool grew = false;
#pragma unroll
      for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
        mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
        mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
        const float mn = fmaxf(m[x], fmaf(mx[x], p.scale_log2, (float)ceil_log2(c.r.vlen)));
        grew = grew || mn > m[x];
        mbase[x] = mn == -INFINITY ? 0.f : mn;
        mx[x] = mn;
      }
      if (__any_sync(0xffffffffu, grew)) {
        const float a0 = ex2(m[0] - mbase[0]);
        const float a1 = SPLIT_P ? a0 : ex2(m[1] - mbase[1]);
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
        if constexpr (!SPLIT_P) m[1] = mx[1];
      }
      // ---- edge tiles: values of tokens that are not there are zero; infinities and NaN in values of the query's own
      // tokens go to the rows that see them, and are zero in the product (a hidden one would reach a row as 0 * inf)
      if (edge) {
#pragma unroll 1
        for (int row = 0; row < TILE; ++row) {
          const int q8 = ring.pos[n % kPosRing<TILE>][row >> 3], pos = q8 + (row & 7);
          uint4* v = reinterpret_cast<uint4*>(base_ptr + (vb - base) + swz_off<D>(row, lane % (D / 8)));
          if (q8 < 0 || pos >= c.r.T) {
            if (lane < D / 8) *v = make_uint4(0u, 0u, 0u, 0u);
          } else if (pos >= ctx) {
            const bool odd = lane < D / 8 && has_nonfinite(*v);
            if (!__any_sync(0xffffffffu, odd)) continue;
#pragma unroll
            for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
              if (!((word[x] >> (pos - ctx)) & 1ull)) continue;
#pragma unroll
              for (int j = 0; j < D / 8; ++j) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(base_ptr + (vb - base) + swz_off<D>(row, j) + (lane & 3) * 4);
                const float2 e = bf16x2_to_float2(w);
                if (!isfinite(e.x)) o[j][2 * x] += e.x;
                if (!isfinite(e.y)) o[j][2 * x + 1] += e.y;
              }
            }
            __syncwarp();
            if (odd) *v = zero_nonfinite(*v);
          }
        }
        __syncwarp();
      }
      // ---- P, and O += P V
#pragma unroll
      for (int kk = 0; kk < TILE / 16; ++kk) {
        uint32_t a[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* e = sc[kk * 2 + h];
          const float p0 = ex2(fmaf(e[0], p.scale_log2, -mbase[0])), p1 = ex2(fmaf(e[1], p.scale_log2, -mbase[0]));
          l[0] += p0 + p1;
          a[h * 2] = pack_bf16(p0, p1);
          if constexpr (SPLIT_P) {
            const float2 hi = bf16x2_to_float2(a[h * 2]);
            a[h * 2 + 1] = pack_bf16(p0 - hi.x, p1 - hi.y);
          } else {
            const float p2 = ex2(fmaf(e[2], p.scale_log2, -mbase[1])), p3 = ex2(fmaf(e[3], p.scale_log2, -mbase[1]));
            l[1] += p2 + p3;
            a[h * 2 + 1] = pack_bf16(p2, p3);
          }
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t vf[4];
          ldsm_x4_t(vf, vb + swz_off<D>(kk * 16 + (lane & 15), j * 2 + (lane >> 4)));
          mma_bf16(o[2 * j], a, vf[0], vf[1]);
          mma_bf16(o[2 * j + 1], a, vf[2], vf[3]);
        }
      }
      if (edge) fence_proxy_async();  // what this warp wrote to the tile, before the refill
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ring.empty[0][s]));
    }

    // ---- the end of the segment or of this CTA's run: the warps' parts together
    const bool whole = t_begin == 0 && piece == c.r.tiles;
    const int slot = 2 * (int)blockIdx.x + (t_begin > 0 ? 0 : 1);
    const int rows = min(ROWS, R - c.rt * ROWS);
    if constexpr (SPLIT_P) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] = add_remainder(o[j][0], o[j][2]);
        o[j][1] = add_remainder(o[j][1], o[j][3]);
      }
    }
#pragma unroll
    for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if ((lane & 3) == 0) {
        join_ml[wid][(lane >> 2) + 8 * x][0] = m[x];
        join_ml[wid][(lane >> 2) + 8 * x][1] = l[x];
      }
    }
    if constexpr (kAllAtOnce) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2*>(join + (wid * 8 + (lane >> 2)) * D + j * 8 + (lane & 3) * 2) = make_float2(o[j][0], o[j][1]);
      meet();
    } else {
      // (16 rows, or a wide head: one scratch, taken in turn)
      meet();
#pragma unroll
      for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, join_ml[w][(lane >> 2) + 8 * x][0]);
        const float f = ex2(m[x] - (top == -INFINITY ? 0.f : top));
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[j][2 * x] *= f;
          o[j][2 * x + 1] *= f;
        }
      }
      for (int w = 0; w < WARPS; ++w) {
        if (wid == w) {
#pragma unroll
          for (int x = 0; x < (SPLIT_P ? 1 : 2); ++x) {
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
              float2* d = reinterpret_cast<float2*>(join + ((lane >> 2) + 8 * x) * D + j * 8 + (lane & 3) * 2);
              float2 v = make_float2(o[j][2 * x], o[j][2 * x + 1]);
              if (w > 0) {
                v.x += d->x;
                v.y += d->y;
              }
              *d = v;
            }
          }
        }
        meet();
      }
    }
    // two columns per thread
    for (int e = tid; e < rows * (D / 2); e += WARPS * 32) {
      const int row = e / (D / 2), col = (e - row * (D / 2)) * 2;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, join_ml[w][row][0]);
      const float b0 = top == -INFINITY ? 0.f : top;
      float2 v = make_float2(0.f, 0.f);
      if constexpr (!kAllAtOnce) v = *reinterpret_cast<const float2*>(join + row * D + col);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = ex2(join_ml[w][row][0] - b0);
        sum = fmaf(join_ml[w][row][1], f, sum);
        if constexpr (kAllAtOnce) {
          const float2 u = *reinterpret_cast<const float2*>(join + (w * 8 + row) * D + col);
          v.x = fmaf(u.x, f, v.x);
          v.y = fmaf(u.y, f, v.y);
        }
      }
      const int r = c.rt * ROWS + row, i = r / p.g, hq = c.h * p.g + (r - i * p.g);
      if (whole) {
        const float inv = sum > 0.f ? 1.f / sum : sum;  // a NaN sum stays one
        *reinterpret_cast<uint32_t*>(p.out + (long long)(c.r.q0 + i) * p.o_ts + (long long)hq * p.o_hs + col) = pack_bf16(v.x * inv, v.y * inv);
        if (col == 0) p.lse[(long long)(c.r.q0 + i) * (p.Hkv * p.g) + hq] = (top + log2f(sum)) * kLn2;
      } else {
        *reinterpret_cast<float2*>(p.part_o + ((long long)slot * ROWS + row) * D + col) = v;
        if (col == 0) *reinterpret_cast<float2*>(p.part_ml + ((long long)slot * ROWS + row) * 2) = make_float2(top, sum);
      }
    }
    meet();  // the scratch is free again
    it += piece;
    c.t += piece - 1;
    if (it < count) attend_advance(p, c, TILE, ROWS);
  }
}

}  // namespace triattn
