// Attention over the paged cache for many query rows (trees of drafted tokens, prompt ends): the 5th-generation tensor cores.
//
// A row tile is NT x 128 query rows of one KV head; token tiles of 64 come in through the ring of attend_tma.cuh.  Per
// token tile and 128 rows:
//   S = Q K^T      tcgen05.mma M 128, N 64, both operands K-major in shared memory, S in tensor memory (two buffers),
//   softmax        one thread per row: 64 logits from tensor memory, running maximum and sum, P = exp2(..) as bf16
//                  back into the columns of S,
//   O += P V       A operand P from tensor memory, B operand V as it lies in the cache (channels contiguous), O in
//                  tensor memory for the whole segment.
// One warp issues S of tile i before P V of tile i - 1, so the tensor cores work while the softmax threads do; with
// NT = 2 two groups of softmax threads share every K/V tile.  The maximum a row's exponentials are taken against is only
// raised when it has grown by more than 2^8 (P stays far inside bf16's and fp32's range, whose precision is relative): the
// accumulator in tensor memory is then rescaled by the row's own thread, which happens a few times per segment.
#pragma once

#include "attend_tma.cuh"
#include "umma.cuh"

namespace triattn {

constexpr int kTreeTile = 64;
constexpr int kTreeStages = 5;
constexpr float kTreeSlack = 8.f;  // log2 of how far a row's logits may exceed its reference maximum

template <int NT>
constexpr int kTreeThreads = NT * 128 + 96;  // softmax groups, MMA warp, K and V producers
template <int D, int NT>
constexpr size_t tree_smem_bytes() {
  return 1024 + (size_t)kTreeStages * 2 * kTreeTile * D * 2 + (size_t)NT * 128 * D * 2;
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D (tensor memory) += A (tensor memory) B (shared memory)
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b),
      "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
// shared-memory matrix descriptor, 128-byte swizzle.  K-major: sbo = stride of 8-row groups.  MN-major: lbo = stride of
// 64-element groups along M / N, sbo = stride of 8-row groups along K.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}

template <int D, int NT>
__global__ void __launch_bounds__(kTreeThreads<NT>, 1)
    attend_tree_kernel(const __grid_constant__ AttendParams p, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const int runs) {
  constexpr int TILE = kTreeTile, STAGES = kTreeStages, THREADS = kTreeThreads<NT>, ROWS = 128 * NT;
  constexpr int MMA_WARP = NT * 4;
  constexpr uint32_t kTileBytes = TILE * D * 2;
  constexpr uint32_t kGroup = D * 16;            // bytes of 8 tokens
  constexpr uint32_t kQBytes = 128 * D * 2;      // 128 query rows: [D / 64][128 rows][128 B]
  constexpr uint32_t kCols = NT == 1 ? 256 : 512;
  extern __shared__ unsigned char smem_raw[];
  __shared__ AttendRing<TILE, STAGES> ring;
  __shared__ uint64_t s_full[NT][2], p_ready[NT][2], o_done[NT][2], q_ready[NT], drained;
  __shared__ long long red[THREADS / 32];
  __shared__ long long found[2];
  __shared__ uint32_t s_tmem;
  __shared__ int odd_piece;  // the last piece in which a query token's value held an infinity or NaN
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&ring.full[s]), 2);   // the K and the V producer
      mbar_init(smem_u32(&ring.empty[s]), 1);  // the tensor core's commit
    }
    for (int g = 0; g < NT; ++g) {
      for (int x = 0; x < 2; ++x) {
        mbar_init(smem_u32(&s_full[g][x]), 1);
        mbar_init(smem_u32(&p_ready[g][x]), 4);
        mbar_init(smem_u32(&o_done[g][x]), 1);
      }
      mbar_init(smem_u32(&q_ready[g]), 4);
    }
    mbar_init(smem_u32(&drained), 1);
    mbar_fence_init();
    ring.err = ring.gaps = 0;
    odd_piece = -1;
  }
  grid_dependency_wait();
  trigger_dependents();
  unsigned err = 0u;
  const long long W = attend_work_before<THREADS>(p, p.B, TILE, ROWS, err, red);
  if (blockIdx.x == 0 && err) flag_status(p.status, err);
  const int J = attend_runs(runs, W, p.min_tiles), run = (int)blockIdx.x / p.Hkv;
  if (run >= J) return;  // nothing allocated yet
  const long long first = attend_first_tile(W, J, run), last = attend_first_tile(W, J, run + 1);
  AttendCursor c;
  if (wid == MMA_WARP) {
    tmem_alloc(smem_u32(&s_tmem), kCols);
    tmem_relinquish();
  }
  attend_seek<THREADS>(p, first, TILE, ROWS, red, found, c);
  c.h = (int)blockIdx.x - run * p.Hkv;
  const int count = (int)(last - first);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* const base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_base = base + STAGES * 2 * kTileBytes;
  const uint32_t o_col = NT * 128;  // S buffers first, 64 columns each, then O

  if (wid > MMA_WARP) {
    attend_produce<D, TILE, STAGES>(p, wid == MMA_WARP + 1 ? &kmap : &vmap, wid - MMA_WARP - 1, c, count, ROWS, base, ring);
  } else if (wid == MMA_WARP) {
    // ------------------------------------------------------------------------------------------ MMA issue
    constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);  // fp32 += bf16 bf16, M = 128
    constexpr uint32_t kIdescS = kIdesc | ((uint32_t)(TILE >> 3) << 17);
    constexpr uint32_t kIdescO = kIdesc | ((uint32_t)(D >> 3) << 17) | (1u << 16);         // B: channels contiguous
    bool ok = true;
    int t_in_piece = 0, piece_no = 0;  // of tile i; of tile i - 1: prev_in_piece
    int prev_in_piece = 0;
    int left = min(c.r.tiles - c.t, count);  // tiles of the piece from tile i on
    auto pv = [&](int i, int in_piece) {
      const int s = i % STAGES;
      const uint32_t vb = base + (uint32_t)s * 2 * kTileBytes + kTileBytes;
      const uint64_t dv = umma_desc(vb, 1024u, kGroup);
#pragma unroll
      for (int g = 0; g < NT; ++g) {
        if (!ring_wait(p_ready[g][i & 1], (uint32_t)(i >> 1) & 1u, &ring.err, p.status)) return false;
        tc_fence_after();
        const uint32_t pa = tmem + (uint32_t)(g * 2 + (i & 1)) * 64u;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < TILE / 16; ++k)
            umma_bf16_ts(tmem + o_col + g * D, pa + k * 8, dv + (uint64_t)(k * 2 * kGroup >> 4), kIdescO, in_piece > 0 || k > 0 ? 1u : 0u);
          umma_commit(smem_u32(&o_done[g][i & 1]));
          if (g == NT - 1) umma_commit(smem_u32(&ring.empty[s]));
        }
        __syncwarp();
      }
      return true;
    };
    int i = 0;
    for (; i < count && ok; ++i) {
      const int s = i % STAGES;
      ok = ring_wait(ring.full[s], (uint32_t)(i / STAGES) & 1u, &ring.err, p.status);
      if (!ok) break;
      fence_proxy_async();
      tc_fence_after();
      // a new segment's query rows are written after the last P V of the one before
      const bool turn = t_in_piece == 0 && i > 0;
      if (turn && !(ok = pv(i - 1, prev_in_piece))) break;
      const uint32_t kb = base + (uint32_t)s * 2 * kTileBytes;
      const uint64_t dk = umma_desc(kb, 16u, kGroup);
#pragma unroll
      for (int g = 0; g < NT; ++g) {
        if (t_in_piece == 0 && ok) {
          ok = ring_wait(q_ready[g], (uint32_t)piece_no & 1u, &ring.err, p.status);
          tc_fence_after();
        }
        if (!ok) break;
        const uint64_t dq = umma_desc(q_base + g * kQBytes, 16u, 1024u);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_bf16(tmem + (uint32_t)(g * 2 + (i & 1)) * 64u, dq + (uint64_t)((k & 3) * 2 + (k >> 2) * (16384 >> 4)),
                      dk + (uint64_t)((k & 3) * 2 + (k >> 2) * (1024 >> 4)), kIdescS, k ? 1u : 0u);
          umma_commit(smem_u32(&s_full[g][i & 1]));
        }
        __syncwarp();
      }
      if (ok && i > 0 && !turn) ok = pv(i - 1, prev_in_piece);
      prev_in_piece = t_in_piece++;
      if (--left == 0 && i + 1 < count) {
        c.t = c.r.tiles - 1;
        attend_advance(p, c, TILE, ROWS);
        t_in_piece = 0;
        ++piece_no;
        left = min(c.r.tiles, count - i - 1);
      }
    }
    if (ok) ok = pv(count - 1, prev_in_piece);
    if (!ok) {  // a wait ran out: the operands must outlive what has been issued
      if (elect_one()) umma_commit(smem_u32(&drained));
      __syncwarp();
      mbar_wait_bounded(smem_u32(&drained), 0u);
    }
  } else {
    // ------------------------------------------------------------------------------------------ softmax
    const int g = wid >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((wid & 3) * 32) << 16;
    const uint32_t t_o = tmem + lanes + o_col + g * D;
    bool ok = true;
    auto load_q = [&](const AttendCursor& at) {  // this thread's row of the operand
      const int r = at.rt * ROWS + g * 128 + row;
      const bool there = r < at.r.n * p.g;
      const int i = there ? r / p.g : 0, j = there ? r - i * p.g : 0;
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (long long)(at.r.q0 + i) * p.q_ts + (long long)(at.h * p.g + j) * p.q_hs);
      unsigned char* dst = base_ptr + STAGES * 2 * kTileBytes + g * kQBytes + row * 128;
#pragma unroll
      for (int x = 0; x < D / 8; ++x) {
        const uint4 w = there ? src[x] : make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(dst + (x >> 3) * 16384 + (((x & 7) ^ (row & 7)) << 4)) = w;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&q_ready[g]));
    };
    // P V of tile k is over.  Asked for k = n - 1 while tile n is in work, and at the end of a piece for its last tile: the
    // barrier's phase of tile k - 2 is over by then (S of tile n came after that product), and its phase of tile k + 2
    // needs this thread's P.
    auto wait_o = [&](int k) { return ring_wait(o_done[g][k & 1], (uint32_t)(k >> 1) & 1u, &ring.err, p.status); };
    load_q(c);
    int piece_no = 0;
    for (int it = 0; it < count && ok; ++piece_no) {
      const int t_begin = c.t, piece = min(c.r.tiles - c.t, count - it);
      const int R = c.r.n * p.g, ctx = c.r.T - c.r.n;
      const int r = c.rt * ROWS + g * 128 + row;
      const bool there = r < R;
      const unsigned long long word = there ? attend_word(p, c.r, r / p.g) : 0ull;
      const bool idle = c.rt * ROWS + g * 128 + (wid & 3) * 32 >= R;  // none of the warp's rows exists
      float m = -INFINITY, l = 0.f;
      for (int x = 0; x < piece; ++x) {
        const int n = it + x, s = n % STAGES;
        const uint32_t t_s = tmem + lanes + (uint32_t)(g * 2 + (n & 1)) * 64u;
        ok = ring_wait(s_full[g][n & 1], (uint32_t)(n >> 1) & 1u, &ring.err, p.status);
        if (!ok) break;
        tc_fence_after();
        // tiles that reach the query's own tokens, the end, or a run of tokens that is not there
        bool edge = false;
        if (p.block_list != nullptr || (t_begin + x + 1) * TILE > ctx || *(volatile int*)&ring.gaps != 0) {
          // positions and values are read here: wait for the tile itself (it stays until this thread's P has been used)
          ok = ring_wait(ring.full[s], (uint32_t)(n / STAGES) & 1u, &ring.err, p.status);
          if (!ok) break;
          int top_pos = -1, low_pos = 1;
#pragma unroll
          for (int j = 0; j < TILE / 8; ++j) {
            const int q8 = ring.pos[n % kPosRing<TILE>][j];
            top_pos = max(top_pos, q8);
            low_pos = min(low_pos, q8);
          }
          edge = low_pos < 0 || top_pos + 8 > ctx;
        }
        if (!idle) {
          uint32_t sv[2][32];
          tmem_ld32(t_s, sv[0]);
          tmem_ld32(t_s + 32, sv[1]);
          tmem_ld_wait();
          if (edge) {
#pragma unroll
            for (int j = 0; j < TILE; ++j) {
              const int q8 = ring.pos[n % kPosRing<TILE>][j >> 3], pos = q8 + (j & 7), d = pos - ctx;
              const bool sees = q8 >= 0 && pos < c.r.T && (d < 0 || ((word >> d) & 1ull));
              if (!sees) sv[j >> 5][j & 31] = 0xff800000u;  // -inf
            }
          }
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < TILE; ++j) mx4[j & 3] = fmaxf(mx4[j & 3], __uint_as_float(sv[j >> 5][j & 31]));
          float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          mx *= p.scale_log2;
          const bool raise = mx > m + kTreeSlack || (m == -INFINITY && mx > m);
          if (__any_sync(0xffffffffu, raise)) {
            const float mn = raise ? mx : m;
            const float a = raise ? ex2(m - mn) : 1.f;
            l *= a;
            m = mn;
            if (x > 0) {  // the accumulator exists: wait for P V of the tile before, then rescale this row
              if (!wait_o(n - 1)) ok = false;
              tc_fence_after();
#pragma unroll
              for (int q = 0; q < D / 32; ++q) {
                uint32_t ov[32];
                tmem_ld32(t_o + q * 32, ov);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * a);
                tmem_st32(t_o + q * 32, ov);
              }
              tmem_st_wait();
            }
          }
          const float mbase = m == -INFINITY ? 0.f : m;
          uint32_t pv[32];
          const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), mb2 = make_float2(-mbase, -mbase);
          float2 la = make_float2(0.f, 0.f), lb = make_float2(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < TILE / 2; ++j) {
            float2 e = ffma2(make_float2(__uint_as_float(sv[j >> 4][(2 * j) & 31]), __uint_as_float(sv[j >> 4][(2 * j + 1) & 31])), sc2, mb2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            if (j & 1) lb = fadd2(lb, e);
            else la = fadd2(la, e);
            pv[j] = pack_bf16(e.x, e.y);
          }
          la = fadd2(la, lb);
          l += la.x + la.y;
          tmem_st32(t_s, pv);
          tmem_st_wait();
        }
        if (edge && g == 0) {
          // values of tokens that are not there are zero; infinities and NaN in values of the query's own tokens are zero in the
          // product and reach the rows that see them when the piece is written (a hidden one would reach a row as 0 * inf)
          const int key = row >> 1, q8 = ring.pos[n % kPosRing<TILE>][key >> 3], pos = q8 + (key & 7);
          const bool out = q8 < 0 || pos >= c.r.T;
          if (out || pos >= ctx) {
#pragma unroll
            for (int q = 0; q < D / 16; ++q) {
              uint4* v = reinterpret_cast<uint4*>(base_ptr + (uint32_t)s * 2 * kTileBytes + kTileBytes + swz_off<D>(key, (row & 1) * (D / 16) + q));
              if (out) {
                *v = make_uint4(0u, 0u, 0u, 0u);
              } else {
                const uint4 w = *v;
                if (has_nonfinite(w)) {
                  *(volatile int*)&odd_piece = piece_no;
                  *v = zero_nonfinite(w);
                }
              }
            }
          }
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_ready[g][n & 1]));
      }
      if (!ok) break;
      ok = wait_o(it + piece - 1);
      if (!ok) break;
      tc_fence_after();
      // the next segment's query rows first: S of its first tile does not wait for what follows
      const AttendCursor done = c;
      it += piece;
      c.t += piece - 1;
      if (it < count) {
        attend_advance(p, c, TILE, ROWS);
        load_q(c);
      }
      if (idle) continue;
      const bool whole = t_begin == 0 && piece == done.r.tiles;
      const int slot = 2 * (int)blockIdx.x + (t_begin > 0 ? 0 : 1);
      const int i = there ? r / p.g : 0, hq = done.h * p.g + (there ? r - i * p.g : 0);
      const float inv = l > 0.f ? 1.f / l : l;  // a NaN sum stays one
      const bool odd = *(volatile int*)&odd_piece == piece_no;
      uint16_t* dst = p.out + (long long)(done.r.q0 + i) * p.o_ts + (long long)hq * p.o_hs;
      float* part = p.part_o + ((long long)slot * ROWS + g * 128 + row) * D;
#pragma unroll
      for (int q = 0; q < D / 32; ++q) {
        uint32_t ov[32];
        tmem_ld32(t_o + q * 32, ov);
        tmem_ld_wait();
        if (odd && there) {
          const int lo = t_begin * TILE, hi = min((t_begin + piece) * TILE, done.r.vlen);
          for (int vp = p.block_list == nullptr ? max(lo, ctx) : lo; vp < hi; ++vp) {
            const TokenAt at = attend_token(p, done, vp, err);
            if (at.pos < ctx || !((word >> (at.pos - ctx)) & 1ull)) continue;
            const uint16_t* v = reinterpret_cast<const uint16_t*>(p.v + at.off) + q * 32;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float e = bf16_to_float(v[j]);
              if (!isfinite(e)) ov[j] = __float_as_uint(__uint_as_float(ov[j]) + e);
            }
          }
        }
        if (there && whole) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 w;
            w.x = pack_bf16(__uint_as_float(ov[j]) * inv, __uint_as_float(ov[j + 1]) * inv);
            w.y = pack_bf16(__uint_as_float(ov[j + 2]) * inv, __uint_as_float(ov[j + 3]) * inv);
            w.z = pack_bf16(__uint_as_float(ov[j + 4]) * inv, __uint_as_float(ov[j + 5]) * inv);
            w.w = pack_bf16(__uint_as_float(ov[j + 6]) * inv, __uint_as_float(ov[j + 7]) * inv);
            *reinterpret_cast<uint4*>(dst + q * 32 + j) = w;
          }
        } else if (there) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(part + q * 32 + j) = make_uint4(ov[j], ov[j + 1], ov[j + 2], ov[j + 3]);
        }
      }
      if (there && whole) p.lse[(long long)(done.r.q0 + i) * (p.Hkv * p.g) + hq] = (m + log2f(l)) * kLn2;
      if (there && !whole)
        *reinterpret_cast<float2*>(p.part_ml + ((long long)slot * ROWS + g * 128 + row) * 2) = make_float2(m, l);
      tc_fence_before();  // the accumulator has been read: the next piece's first P V (after this warp's next arrival) may overwrite it
    }
  }
  // all roles are done (or gave up): free the tensor memory
  tc_fence_before();
  __syncthreads();
  if (wid == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
}

}  // namespace triattn
