// Attention over the paged cache for many query rows (trees of drafted tokens, prompt ends): the 5th-generation tensor cores.
//
// A row tile is NT x 128 query rows of one KV head; token tiles of 128 come in through the producers of attend_tma.cuh, K and
// V in rings of their own (K is left earlier).  Per token tile and 128 rows:
//   S = Q K^T      tcgen05.mma M 128, N 128, both operands K-major in shared memory, S in tensor memory,
//   softmax        two threads per row, 64 logits each from tensor memory; P = exp2(..) as bf16 back into the columns of S
//                  (each thread the first half of its own).  One bf16, not two parts as the kernel for few rows takes: remainders would
//                  double the products with V, half of the tensor cores' time.  The output's error against 64 bits is
//                  2.3e-3, of which 1.7e-3 are its own rounding to bf16; l adds the probabilities before they are rounded,
//   O += P V       A operand P from tensor memory, B operand V as it lies in the cache (channels contiguous), O in
//                  tensor memory for the whole segment.
// N = 128 because the A operand is read again for every product: at N = 64 the reads of Q, 4 KB per product, take longer than the
// product (measured: the issuing warp spent 65 cycles on each of 16 products a tile).
// NT = 2 (more than 128 rows): two groups of softmax threads share every K/V tile and take turns with the tensor cores,
// P V and the next S of one group running while the other group is at its exponentials.  (One thread per row: a group took 2500
// cycles for a tile's softmax, two and a half times what its exponentials cost, and the turns did not overlap.)  NT = 1: S has two buffers, and S of tile i
// is issued before P V of tile i - 1.
// Measured: 256 rows over 8 x 32768 tokens, 8 KV heads, in 294 us (825 TFLOP/s in bursts, 680 under the power cap), where the bytes take 165;
// what bounds it is the alternation of the two groups: per tile and group 1500 cycles for its products and 2000 for its softmax, the
// tensor cores' own time for both groups being 2050.
// A row's exponentials are taken against a reference above the maximum of the first tile it saw, which is raised only when the
// 64 exponentials of a later tile's thread add up to 2^8 of that maximum.  The reference lies so far above it that even then the
// exponentials of all tiles add up to 1 at most, and O is finite for all finite values (see attend.cuh; with the reference at the
// maximum and a slack of 2^64, values of 2^70 gave infinities).  Where the logits spread, later tiles exceed the first by more (of
// normal ones by 1.6 standard deviations in 32768): the reference is set ahead by twice the distance between the maxima of a thread's
// quarters (1.1 standard deviations), 2^40 at most.  Without that, 256 rows of logits with a standard deviation of 6 (12) on
// 8 x 32768 tokens raised in most tiles: 427 (431) us where those of deviation 1 take 297; with it 303 (319).  Precision is relative: a stale reference costs no
// accuracy, and no tile's maximum is needed; of 2^n tokens (n at least 7), weights below 2^(n - 124), of a row whose logits spread
// 2^(n - 84), of the first tile's largest vanish.  P goes to tensor memory, over
// the logits, only when it is known to be in range; the rare raise starts from the logits again and rescales what the row has
// accumulated, in its own threads.
#pragma once

#include "attend_tma.cuh"
#include "umma.cuh"

namespace triattn {

constexpr int kTreeTile = 128;
template <int D, int NT>
constexpr int kTreeStages = 2 * (128 / D);  // of K and of V: 64 KB each
constexpr int kTreeSlack = 8;  // base 2: what a thread's 64 exponentials of a tile may add up to, above the maximum of the reference
constexpr float kTreeAhead = 40.f;  // base 2: what a reference is set ahead at most, for logits that spread

template <int NT>
constexpr int kTreeThreads = NT * 256 + 96;  // softmax groups, MMA warp, K and V producers
template <int D, int NT>
constexpr size_t tree_smem_bytes() {
  return 1024 + (size_t)kTreeStages<D, NT> * 2 * kTreeTile * D * 2 + (size_t)NT * 128 * D * 2;
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
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// waits for the loads in flight; the values are not to be used before
__device__ __forceinline__ void tmem_ld_wait32(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]),
                 "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]),
                 "+r"(v[25]), "+r"(v[26]), "+r"(v[27])
               :
               : "memory");
  asm volatile("" : "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]) : : "memory");
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
  constexpr int TILE = kTreeTile, STAGES = kTreeStages<D, NT>, THREADS = kTreeThreads<NT>, ROWS = 128 * NT;
  constexpr int MMA_WARP = NT * 8;
  constexpr int SB = NT == 1 ? 2 : 1;            // S buffers per group
  constexpr uint32_t kTileBytes = TILE * D * 2;
  constexpr uint32_t kGroup = D * 16;            // bytes of 8 tokens
  constexpr uint32_t kQBytes = 128 * D * 2;      // 128 query rows: [D / 64][128 rows][128 B]
  constexpr uint32_t kCols = 512;                // tensor memory: S buffers (128 columns each, 256 in all), then O
  extern __shared__ unsigned char smem_raw[];
  __shared__ AttendRing<TILE, STAGES> ring;
  // per group and S buffer: S is there, P is there, P V is over
  __shared__ uint64_t s_full[NT][SB], p_ready[NT][SB], o_done[NT][SB];
  __shared__ uint64_t q_ready[NT], drained;
  __shared__ AttendPlanShared<THREADS> plan;
  __shared__ uint32_t s_tmem;
  __shared__ float pair_val[2][NT][2][128];  // what the two threads of a row tell each other (tiles in turn)
  __shared__ bool pair_over[2][NT][2][4], row_over[2][NT][2][128];
  // The last even and the last odd piece in which a query token's value held an infinity or NaN.  Group 0 writes, both groups read
  // when they write their piece out.  Two words, because group 0 may be a piece ahead: S of the next piece's first tile goes
  // to it before P V of this piece's last tile to group 1.  It is never two ahead: S of that next tile for group 1, which the same
  // thread issues before anything of the piece after, waits for queries that group 1 loads after it has read its word.
  __shared__ int odd_piece[2];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s)
      for (int w = 0; w < 2; ++w) {
        mbar_init(smem_u32(&ring.full[w][s]), 1);
        mbar_init(smem_u32(&ring.empty[w][s]), 1);  // the tensor core's commit
      }
    for (int g = 0; g < NT; ++g) {
      for (int x = 0; x < SB; ++x) {
        mbar_init(smem_u32(&s_full[g][x]), 1);
        mbar_init(smem_u32(&p_ready[g][x]), 8);
        mbar_init(smem_u32(&o_done[g][x]), 1);
      }
      mbar_init(smem_u32(&q_ready[g]), 8);
    }
    mbar_init(smem_u32(&drained), 1);
    mbar_fence_init();
    ring.err = ring.gaps = 0;
    prefetch_map(&kmap);
    prefetch_map(&vmap);
    odd_piece[0] = odd_piece[1] = -1;
  }
  grid_dependency_wait();
  trigger_dependents();
  const int run = (int)blockIdx.x / p.Hkv;
  AttendCursor c;
  int count;
  if (!attend_plan_run<THREADS>(p, runs, p.min_tiles, run, TILE, ROWS, plan, c, count)) return;  // nothing allocated yet
  c.h = (int)blockIdx.x - run * p.Hkv;
  if (wid == MMA_WARP) {
    tmem_alloc(smem_u32(&s_tmem), kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* const base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t v_base = base + STAGES * kTileBytes, q_base = v_base + STAGES * kTileBytes;
  constexpr uint32_t o_col = 256;

  if (wid > MMA_WARP) {
    const int w = wid - MMA_WARP - 1;
    attend_produce<D, TILE, STAGES>(p, w == 0 ? &kmap : &vmap, w, c, count, ROWS, w == 0 ? base : v_base, kTileBytes,
                                    ring.full[w], ring.empty[w], ring, (w == 0 && p.sums != nullptr) || p.max_q * p.g > ROWS);
  } else if (wid == MMA_WARP) {
    // ------------------------------------------------------------------------------------------ MMA issue: one thread
    if (elect_one()) {
    constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);  // fp32 += bf16 bf16, M = 128
    constexpr uint32_t kIdescS = kIdesc | ((uint32_t)(TILE >> 3) << 17);
    constexpr uint32_t kIdescO = kIdesc | ((uint32_t)(D >> 3) << 17) | (1u << 16);         // B: channels contiguous
    bool ok = true;
    int t_in_piece = 0, prev_in_piece = 0, piece_no = 0;  // tile i's place in its piece, tile i - 1's
    int left = min(c.r.tiles - c.t, count);               // tiles of the piece from tile i on
    auto issue_s = [&](int i, int g) {
      const int s = i % STAGES;
      if (g == 0 && !thread_wait(ring.full[0][s], (uint32_t)(i / STAGES) & 1u, &ring.err, p.status)) return false;
      if (t_in_piece == 0 && !thread_wait(q_ready[g], (uint32_t)piece_no & 1u, &ring.err, p.status)) return false;
      tc_fence_after();
      const uint64_t dk = umma_desc(base + (uint32_t)s * kTileBytes, 16u, kGroup), dq = umma_desc(q_base + g * kQBytes, 16u, 1024u);
      {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_bf16(tmem + (uint32_t)(g * SB + i % SB) * 128u, dq + (uint64_t)((k & 3) * 2 + (k >> 2) * (16384 >> 4)),
                    dk + (uint64_t)((k & 3) * 2 + (k >> 2) * (1024 >> 4)), kIdescS, k ? 1u : 0u);
        umma_commit(smem_u32(&s_full[g][i % SB]));
        if (g == NT - 1) umma_commit(smem_u32(&ring.empty[0][s]));
      }
      return true;
    };
    auto issue_pv = [&](int i, int g, int in_piece) {
      const int s = i % STAGES;
      if (g == 0 && !thread_wait(ring.full[1][s], (uint32_t)(i / STAGES) & 1u, &ring.err, p.status)) return false;
      if (!thread_wait(p_ready[g][i % SB], (uint32_t)(i / SB) & 1u, &ring.err, p.status)) return false;
      tc_fence_after();
      const uint32_t pa = tmem + (uint32_t)(g * SB + i % SB) * 128u;
      const uint64_t dv = umma_desc(v_base + (uint32_t)s * kTileBytes, 1024u, kGroup);
      {
#pragma unroll
        for (int k = 0; k < TILE / 16; ++k)
          umma_bf16_ts(tmem + o_col + g * D, pa + (k & 3) * 8 + (k >> 2) * 64, dv + (uint64_t)((k * 2 * kGroup) >> 4), kIdescO, in_piece > 0 || k > 0 ? 1u : 0u);
        umma_commit(smem_u32(&o_done[g][i % SB]));
        if (g == NT - 1) umma_commit(smem_u32(&ring.empty[1][s]));
      }
      return true;
    };
    // (one place in the code for each of the two: the kernel's loops share the instruction cache)
#pragma unroll 1
    for (int i = 0; i <= count && ok; ++i) {
      // a new segment's query rows are written after the last P V of the one before; with one S buffer P V comes first anyway
      const bool pv_first = SB == 1 || t_in_piece == 0 || i == count;
#pragma unroll 1
      for (int step = 0; step < 2 * NT && ok; ++step) {
        const int g = step >> 1;
        if (((step & 1) == 0) == pv_first) {
          if (i > 0) ok = issue_pv(i - 1, g, prev_in_piece);
        } else if (i < count) {
          ok = issue_s(i, g);
        }
      }
      prev_in_piece = t_in_piece++;
      if (--left == 0 && i + 1 < count) {
        c.t = c.r.tiles - 1;
        attend_advance(p, c, TILE, ROWS);
        t_in_piece = 0;
        ++piece_no;
        left = min(c.r.tiles, count - i - 1);
      }
    }
    if (!ok) {  // a wait ran out: the operands must outlive what has been issued
      umma_commit(smem_u32(&drained));
      mbar_wait_bounded(smem_u32(&drained), 0u);
    }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------------------------------ softmax
    const int g = wid >> 3, half = (wid >> 2) & 1, row = tid & 127;
    const uint32_t lanes = (uint32_t)((wid & 3) * 32) << 16;
    const uint32_t t_o = tmem + lanes + o_col + g * D;
    // the two warps that share these 32 rows
    auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(2 + g * 4 + (wid & 3)) : "memory"); };
    // A wait that runs out ends the work but not the control flow: a warp that left would strand its partner at a barrier.
    bool dead = false;
    auto load_q = [&](const AttendCursor& at) {  // the pair's 32 rows of the operand, half of them per warp; D / 8 lanes to a row
      const int pc = lane % (D / 8), rr0 = (wid & 3) * 32 + half * 16 + lane / (D / 8);
      constexpr int STEP = 256 / D;  // rows at a time
      unsigned char* dst = base_ptr + (q_base - base) + g * kQBytes;
      int r = at.rt * ROWS + g * 128 + rr0, i = r / p.g, j = r - i * p.g;
      uint4 w[D / 16];  // all loads in flight
#pragma unroll
      for (int y = 0; y < D / 16; ++y) {
        w[y] = make_uint4(0u, 0u, 0u, 0u);
        if (i < at.r.n)
          w[y] = *reinterpret_cast<const uint4*>(p.q + (long long)(at.r.q0 + i) * p.q_ts + (long long)(at.h * p.g + j) * p.q_hs + pc * 8);
        for (j += STEP; j >= p.g; j -= p.g) ++i;
      }
#pragma unroll
      for (int y = 0; y < D / 16; ++y) {
        const int rr = rr0 + y * STEP;
        *reinterpret_cast<uint4*>(dst + rr * 128 + (pc >> 3) * 16384 + (((pc & 7) ^ (rr & 7)) << 4)) = w[y];
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&q_ready[g]));
    };
    // P V of tile k is over.  Asked for k = n - 1 while tile n is in work (two S buffers; with one, S of tile n came after it) and
    // for a piece's last tile: the barrier's phase before is over by then, since S of a later tile came after that
    // product, and its next phase needs this thread's P.
    auto wait_o = [&](int k) { return ring_wait(o_done[g][k % SB], (uint32_t)(k / SB) & 1u, &ring.err, p.status); };
    load_q(c);
    int piece_no = 0;
    for (int it = 0; it < count; ++piece_no) {
      const int t_begin = c.t, piece = min(c.r.tiles - c.t, count - it);
      const int R = c.r.n * p.g, ctx = c.r.T - c.r.n;
      const int r = c.rt * ROWS + g * 128 + row;
      const bool there = r < R;
      const unsigned long long word = there ? attend_word(p, c.r, r / p.g) : 0ull;
      const bool idle = c.rt * ROWS + g * 128 + (wid & 3) * 32 >= R;  // none of the warp's rows exists
      // 2^-share: what a thread's exponentials of a tile may add up to, a row's over its 2 x tiles of them to 1
      const int share = ceil_log2(2 * c.r.tiles);
      float m = -INFINITY, l = 0.f;
      for (int x = 0; x < piece; ++x) {
        const int n = it + x, s = n % STAGES;
        const uint32_t t_s = tmem + lanes + (uint32_t)(g * SB + n % SB) * 128u;
        dead = dead || !ring_wait(s_full[g][n % SB], (uint32_t)(n / SB) & 1u, &ring.err, p.status);
        tc_fence_after();
        // tiles that reach the query's own tokens, the end, or a run of tokens that is not there
        const int* pos8 = ring.pos[n % kPosRing<TILE>];
        bool edge = false;
        if (!dead && (p.block_list != nullptr || (t_begin + x + 1) * TILE > ctx || *(volatile int*)&ring.gaps != 0)) {
          // positions and values are read here: wait for the tile itself (V stays until this thread's P has been used)
          dead = !ring_wait(ring.full[1][s], (uint32_t)(n / STAGES) & 1u, &ring.err, p.status);
          int top_pos = -1, low_pos = 1;
#pragma unroll
          for (int j = 0; j < TILE / 8; ++j) {
            const int q8 = pos8[j];
            top_pos = max(top_pos, q8);
            low_pos = min(low_pos, q8);
          }
          edge = low_pos < 0 || top_pos + 8 > ctx;
        }
        if (dead) {  // as many barriers as a partner that is not (yet) dead passes
          if (!idle) {
            if (x > 0 && lane == 0) pair_over[n & 1][g][half][wid & 3] = false;
            pair_sync();
            if (x > 0 && pair_over[n & 1][g][half ^ 1][wid & 3]) pair_sync();
          }
          continue;
        }
        if (!idle) {
          // which of this thread's 64 tokens its row sees (the code of the loop is kept small: with the tests spelled out per logit
          // the instruction cache missed, and a tile took a tenth longer)
          uint32_t sees[2] = {0xffffffffu, 0xffffffffu};
          if (edge) {
#pragma unroll 1
            for (int j = 0; j < 8; ++j) {
              const int q8 = pos8[half * 8 + j];
              uint32_t bits = 0u;  // of a run of 8 tokens
              if (q8 >= 0) {
                const int d = q8 - ctx;  // its first token's place among the query's own
                const unsigned long long own = d >= 0 ? word >> d : (word << -max(d, -8)) | ((1ull << -max(d, -8)) - 1ull);
                bits = (uint32_t)own & (q8 + 8 <= c.r.T ? 0xffu : (1u << (c.r.T - q8 > 0 ? c.r.T - q8 : 0)) - 1u);
              }
              const uint32_t at = (uint32_t)(j & 3) * 8u;
              if (j < 4) sees[0] = (sees[0] & ~(0xffu << at)) | (bits & 0xffu) << at;
              else sees[1] = (sees[1] & ~(0xffu << at)) | (bits & 0xffu) << at;
            }
          }
          // 32 of the logits; hidden tokens are -inf
          auto logits = [&](int q, uint32_t (&sv)[32]) {
            tmem_ld32(t_s + half * 64 + q * 32, sv);
            tmem_ld_wait32(sv);
            if (edge) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!((sees[q] >> j) & 1u)) sv[j] = 0xff800000u;
            }
          };
          uint32_t pv[2][16];  // P, kept until it is known to be in range: the logits stay where they are until then
          float sum = 0.f;
          bool over = true;  // this thread's half of the row asks for a new reference
          for (bool raise = x == 0;;) {
            if (raise) {
              // the reference of a row that asks for it becomes the maximum so far (of both threads), and what the row has
              // accumulated is rescaled; the warp's other rows stay as they are
              float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
              for (int q = 0; q < 2; ++q) {
                uint32_t sv[32];
                logits(q, sv);
#pragma unroll
                for (int j = 0; j < 32; ++j) m4[j & 3] = fmaxf(m4[j & 3], __uint_as_float(sv[j]));
              }
              float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
              const float low = fminf(fminf(m4[0], m4[1]), fminf(m4[2], m4[3]));
              mx = fmaf(mx, p.scale_log2, fminf(2.f * p.scale_log2 * (mx - low), kTreeAhead));  // (no logit at all: -inf)
              pair_val[n & 1][g][half][row] = mx;
              row_over[n & 1][g][half][row] = over;
              pair_sync();
              mx = over || row_over[n & 1][g][half ^ 1][row] ? fmaxf(m, fmaxf(mx, pair_val[n & 1][g][half ^ 1][row]) + (float)(share + kTreeSlack)) : m;
              const float f = mx > m ? ex2(m - mx) : 1.f;
              l *= f;
              m = mx;
              if (x > 0) {  // the accumulator, after P V of the tile before; each thread half of the channels
                if (SB > 1) dead = !wait_o(n - 1);
                tc_fence_after();
#pragma unroll 1
                for (int y = 0; y < D / 32; ++y) {
                  uint32_t ov[16];
                  tmem_ld16(t_o + half * (D / 2) + y * 16, ov);
                  tmem_ld_wait();
#pragma unroll
                  for (int j = 0; j < 16; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * f);
                  tmem_st16(t_o + half * (D / 2) + y * 16, ov);
                }
                tmem_st_wait();
              }
            }
            const float mbase = m == -INFINITY ? 0.f : m;
            const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), mb2 = make_float2(-mbase, -mbase);
            float2 la = make_float2(0.f, 0.f), lb = make_float2(0.f, 0.f);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t sv[32];
              logits(q, sv);
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                float2 e = ffma2(make_float2(__uint_as_float(sv[2 * j]), __uint_as_float(sv[2 * j + 1])), sc2, mb2);
                e.x = ex2(e.x);
                e.y = ex2(e.y);
                if (j & 1) lb = fadd2(lb, e);
                else la = fadd2(la, e);
                pv[q][j] = pack_bf16(e.x, e.y);
              }
            }
            la = fadd2(la, lb);
            sum = la.x + la.y;
            if (raise) break;  // nothing exceeds 2^-(share + kTreeSlack)
            over = !(sum < __int_as_float((127 - share) << 23)) || m == -INFINITY;
            const bool any = __any_sync(0xffffffffu, over);
            if (lane == 0) pair_over[n & 1][g][half][wid & 3] = any;
            pair_sync();
            if (!any && !pair_over[n & 1][g][half ^ 1][wid & 3]) break;
            raise = true;
          }
          l += sum;
#pragma unroll
          for (int q = 0; q < 2; ++q) tmem_st16(t_s + half * 64 + q * 16, pv[q]);  // columns of its own logits
          tmem_st_wait();
        }
        if (edge && g == 0) {
          // values of tokens that are not there are zero; infinities and NaN in values of the query's own tokens are zero in the
          // product and reach the rows that see them when the piece is written (a hidden one would reach a row as 0 * inf)
          const int q8 = pos8[row >> 3], pos = q8 + (row & 7);  // half a token per thread
          const bool out = q8 < 0 || pos >= c.r.T;
          if (out || pos >= ctx) {
#pragma unroll 1
            for (int q = half * (D / 16); q < (half + 1) * (D / 16); ++q) {
              uint4* v = reinterpret_cast<uint4*>(base_ptr + (v_base - base) + (uint32_t)s * kTileBytes + swz_off<D>(row, q));
              if (out) {
                *v = make_uint4(0u, 0u, 0u, 0u);
              } else {
                const uint4 w = *v;
                if (has_nonfinite(w)) {
                  *(volatile int*)&odd_piece[piece_no & 1] = piece_no;
                  *v = zero_nonfinite(w);
                }
              }
            }
          }
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_ready[g][n % SB]));
      }
      dead = dead || !wait_o(it + piece - 1);
      tc_fence_after();
      // ---- the piece is written; each thread holds half of the channels of its row.  A warp's 32 rows x 32 channels pass through
      // the place of the (used) query operand, so that eight lanes write 128 consecutive bytes of a row
      const bool whole = t_begin == 0 && piece == c.r.tiles;
      if (!idle) {
        pair_sync();  // the last exchange has been read
        pair_val[0][g][half][row] = l;
        pair_sync();
        l += pair_val[0][g][half ^ 1][row];
        pair_sync();  // read before the next one
        const int slot = 2 * (int)blockIdx.x + (t_begin > 0 ? 0 : 1);
        const float inv = !whole ? 1.f : l > 0.f ? 1.f / l : l;  // a NaN sum stays one
        const bool odd = *(volatile int*)&odd_piece[piece_no & 1] == piece_no;
        // the four rows this lane writes pieces of: where they go (null: they do not exist)
        unsigned char* to[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int at = c.rt * ROWS + g * 128 + (wid & 3) * 32 + k * 8 + (lane >> 2);
          const int i = at / p.g, hq = c.h * p.g + (at - i * p.g);
          to[k] = at >= R ? nullptr
                          : whole ? reinterpret_cast<unsigned char*>(p.out + (long long)(c.r.q0 + i) * p.o_ts + (long long)hq * p.o_hs)
                                  : reinterpret_cast<unsigned char*>(p.part_o + ((long long)slot * ROWS + at - c.rt * ROWS) * D);
        }
        unsigned char* stage = base_ptr + (q_base - base) + wid * (16 * D * 2);  // 16 rows of the operand: 4 KB (D = 128)
#pragma unroll 1
        for (int y = 0; y < (dead ? 0 : D / 64); ++y) {
          const int q = half * (D / 64) + y;
          uint32_t ov[32];
          tmem_ld32(t_o + q * 32, ov);
          tmem_ld_wait32(ov);
          if (odd && there) {
            unsigned err = 0u;  // (the producers have reported it)
            const int lo = t_begin * TILE, hi = min((t_begin + piece) * TILE, c.r.vlen);
            for (int vp = p.block_list == nullptr ? max(lo, ctx) : lo; vp < hi; ++vp) {
              const TokenAt at = attend_token(p, c, vp, err);
              if (at.pos < ctx || !((word >> (at.pos - ctx)) & 1ull)) continue;
              const uint16_t* v = reinterpret_cast<const uint16_t*>(p.v + at.off) + q * 32;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float e = bf16_to_float(v[j]);
                ov[j] = __float_as_uint(__uint_as_float(ov[j]) + (isfinite(e) ? 0.f : e));
              }
            }
          }
          // 2 KB at a time (16 channels per row): both head dimensions have room for that
#pragma unroll
          for (int z = 0; z < 2; ++z) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float4*>(stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                  make_float4(__uint_as_float(ov[z * 16 + 4 * j]) * inv, __uint_as_float(ov[z * 16 + 4 * j + 1]) * inv,
                              __uint_as_float(ov[z * 16 + 4 * j + 2]) * inv, __uint_as_float(ov[z * 16 + 4 * j + 3]) * inv);
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // eight rows at a time, four lanes to a row
              const int rr = k * 8 + (lane >> 2);
              const float4 e = *reinterpret_cast<const float4*>(stage + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
              const int col = q * 32 + z * 16 + (lane & 3) * 4;
              if (to[k] == nullptr) continue;
              if (whole) *reinterpret_cast<uint2*>(to[k] + col * 2) = make_uint2(pack_bf16(e.x, e.y), pack_bf16(e.z, e.w));
              else *reinterpret_cast<float4*>(to[k] + col * 4) = e;
            }
            __syncwarp();
          }
        }
        if (there && half == 0 && !dead) {
          const int i = r / p.g, hq = c.h * p.g + (r - i * p.g);
          if (whole) p.lse[(long long)(c.r.q0 + i) * (p.Hkv * p.g) + hq] = (m + log2f(l)) * kLn2;
          else *reinterpret_cast<float2*>(p.part_ml + ((long long)slot * ROWS + g * 128 + row) * 2) = make_float2(m, l);
        }
      }
      it += piece;
      c.t += piece - 1;
      if (it < count) {
        attend_advance(p, c, TILE, ROWS);
        // the group's warps share the operand's place: all of them are done staging
        asm volatile("bar.sync %0, 256;" ::"r"(10 + g) : "memory");
        load_q(c);
      }
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

// ------------------------------------------------------------------------------------------ weight sums
// The second pass over K (see attend.cuh for the formula): S^T = K Q^T with 128 tokens as the rows of the product (M) and up to
// 256 query rows as its columns (N), so that a thread has one token and adds up its row of tensor memory: no exchange between
// threads.  K tiles come in through the ring (two loading warps: a warp issues a load every 80 cycles or so), one thread issues
// the products into two accumulators, two groups of four warps empty them in turn.  Bound by the keys' bytes and, from about 128 rows,
// by the exponentials, N per token.  (With the products on mma.sync and a token's sum spread over four lanes, 128 rows took 43
// instead of 27 us for 2 x 14300 tokens and 8 heads, and a decode step of 16 x 4600 tokens 6 us longer.)  More rows than N: one launch per N
// (row0), the first sets or adds, the others add.
template <int D>
constexpr int kObserveRowsMax = D == 256 ? 128 : 256;
template <int D>
constexpr int kObserveMmaStages = D == 64 ? 6 : D == 128 ? 4 : 2;
constexpr int kObserveMmaThreads = (8 + 1 + 2) * 32;
template <int D>
constexpr size_t observe_mma_smem_bytes() {
  return 1024 + (size_t)kObserveMmaStages<D> * 128 * D * 2 + (size_t)kObserveRowsMax<D> * D * 2;
}

template <int D>
__global__ void __launch_bounds__(kObserveMmaThreads, 1)
    attend_observe_mma_kernel(const __grid_constant__ AttendParams p, const __grid_constant__ CUtensorMap kmap, const int runs,
                              const int row0) {
  constexpr int TILE = 128, STAGES = kObserveMmaStages<D>, THREADS = kObserveMmaThreads, RMAX = kObserveRowsMax<D>;
  constexpr int kAll = 1 << 24;  // all rows of a (request, KV head) in one segment
  constexpr uint32_t kTileBytes = TILE * D * 2, kGroup = D * 16;
  extern __shared__ unsigned char smem_raw[];
  __shared__ AttendRing<TILE, STAGES, true> ring;
  __shared__ AttendPlanShared<THREADS> plan;
  __shared__ uint64_t acc_full[2], acc_empty[2], q_ready, drained;
  __shared__ __align__(16) float lse2[RMAX];
  __shared__ unsigned long long words[RMAX];
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&ring.full[0][s]), 1);
      mbar_init(smem_u32(&ring.empty[0][s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&acc_full[a]), 1);
      mbar_init(smem_u32(&acc_empty[a]), 4);
    }
    mbar_init(smem_u32(&q_ready), 8);
    mbar_init(smem_u32(&drained), 1);
    mbar_fence_init();
    ring.err = ring.gaps = 0;
    prefetch_map(&kmap);
  }
  grid_dependency_wait();
  trigger_dependents();
  const int run = (int)blockIdx.x / p.Hkv;
  AttendCursor c;
  int count;
  if (!attend_plan_run<THREADS>(p, runs, 2, run, TILE, kAll, plan, c, count)) return;  // nothing allocated yet
  c.h = (int)blockIdx.x - run * p.Hkv;
  if (wid == 8) {
    tmem_alloc(smem_u32(&s_tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, q_base = base + STAGES * kTileBytes;
  unsigned char* const q_smem = smem_raw + (q_base - smem_u32(smem_raw));
  // columns of the product for a request's rows of this pass: a multiple of 32 (what the threads read at a time)
  auto columns = [&](const AttendReq& r) { return (min(max(r.n * p.g - row0, 1), RMAX) + 31) & ~31; };

  if (wid > 8) {
    attend_produce<D, TILE, STAGES>(p, &kmap, 0, c, count, kAll, base, kTileBytes, ring.full[0], ring.empty[0], ring,
                                p.max_q * p.g > row0 + RMAX, wid - 9, 2);
  } else if (wid == 8) {
    if (elect_one()) {
      bool ok = true;
      int piece_no = 0;
      for (int it = 0; it < count && ok; ++piece_no) {
        const int piece = min(c.r.tiles - c.t, count - it);
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(columns(c.r) >> 3) << 17) | ((128u >> 4) << 24);
        ok = thread_wait(q_ready, (uint32_t)piece_no & 1u, &ring.err, p.status);
        for (int x = 0; x < piece && ok; ++x) {
          const int n = it + x, s = n % STAGES, a = n & 1;
          ok = thread_wait(ring.full[0][s], (uint32_t)(n / STAGES) & 1u, &ring.err, p.status) &&
               (n < 2 || thread_wait(acc_empty[a], (uint32_t)((n >> 1) - 1) & 1u, &ring.err, p.status));
          if (!ok) break;
          tc_fence_after();
          const uint64_t dk = umma_desc(base + (uint32_t)s * kTileBytes, 16u, kGroup), dq = umma_desc(q_base, 16u, 1024u);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_bf16(tmem + (uint32_t)a * 256u, dk + (uint64_t)((k & 3) * 2 + (k >> 2) * (1024 >> 4)),
                      dq + (uint64_t)((k & 3) * 2 + (k >> 2) * ((RMAX * 128) >> 4)), idesc, k ? 1u : 0u);
          umma_commit(smem_u32(&acc_full[a]));
          umma_commit(smem_u32(&ring.empty[0][s]));
        }
        it += piece;
        c.t += piece - 1;
        if (it < count) attend_advance(p, c, TILE, kAll);
      }
      if (!ok) {  // a wait ran out: the operands must outlive what has been issued
        umma_commit(smem_u32(&drained));
        mbar_wait_bounded(smem_u32(&drained), 0u);
      }
    }
    __syncwarp();
  } else {
    const int group = wid >> 2, token = (wid & 3) * 32 + lane;
    const uint32_t t_acc = tmem + ((uint32_t)((wid & 3) * 32) << 16) + (uint32_t)group * 256u;
    auto meet = [&]() { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    bool dead = false;
    for (int it = 0; it < count;) {
      const int piece = min(c.r.tiles - c.t, count - it);
      const int R = c.r.n * p.g, ctx = c.r.T - c.r.n, cols = columns(c.r);
      meet();  // the tiles of the piece before have been emptied: its rows are not needed any more
      for (int x = tid; x < cols * (D / 8); x += 256) {
        // (columns without a row repeat the last one: a zero row times an infinite key would be NaN, and stay it)
        const int row = x / (D / 8), pc = x % (D / 8), r = min(row0 + row, R - 1);
        const int i = r / p.g, j = r - i * p.g;
        const uint4 w = *reinterpret_cast<const uint4*>(p.q + (long long)(c.r.q0 + i) * p.q_ts + (long long)(c.h * p.g + j) * p.q_hs + pc * 8);
        *reinterpret_cast<uint4*>(q_smem + (pc >> 3) * (RMAX * 128) + row * 128 + (((pc & 7) ^ (row & 7)) << 4)) = w;
      }
      if (tid < cols) {
        const int r = row0 + tid;
        float z = INFINITY;  // rows that do not exist, or see nothing, add exp2(-inf) = 0
        unsigned long long w = 0ull;
        if (r < R) {
          const int i = r / p.g, j = r - i * p.g;
          const float e = p.lse[(long long)(c.r.q0 + i) * (p.Hkv * p.g) + c.h * p.g + j];
          if (e != -INFINITY) z = e * kLog2e;
          w = attend_word(p, c.r, i);
        }
        lse2[tid] = z;
        words[tid] = w;
      }
      fence_proxy_async();
      meet();
      if (lane == 0) mbar_arrive(smem_u32(&q_ready));
      for (int x = (group + it) & 1; x < piece; x += 2) {  // tiles whose accumulator is this group's
        const int n = it + x;
        dead = dead || !ring_wait(acc_full[group], (uint32_t)(n >> 1) & 1u, &ring.err, p.status);
        if (dead) break;
        tc_fence_after();
        const int q8 = ring.pos[n % kPosRing<TILE>][token >> 3], pos = q8 + (token & 7);
        float* at = nullptr;
        float old = 0.f;
        if (q8 >= 0 && pos < c.r.T) {
          at = p.sums + ((long long)ring.blk[n % kPosRing<TILE>][token >> 3] * p.Hkv + c.h) * p.bs + pos % p.bs;
          // a query's own token, or sums that start anew: whatever the slot holds is nobody's
          if (row0 > 0 || (p.reset_sums == 0 && pos < ctx)) old = *at;
        }
        const bool own = __any_sync(0xffffffffu, at != nullptr && pos >= ctx);
        float2 wa = make_float2(0.f, 0.f), wb = make_float2(0.f, 0.f);
        const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
#pragma unroll 1
        for (int c0 = 0; c0 < cols; c0 += 32) {
          uint32_t sv[32];
          tmem_ld32(t_acc + (uint32_t)c0, sv);
          tmem_ld_wait32(sv);
          if (own && pos >= ctx) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!((words[c0 + j] >> ((pos - ctx) & 63)) & 1ull)) sv[j] = 0xff800000u;
          }
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 z = *reinterpret_cast<const float4*>(lse2 + c0 + j);
            float2 e = ffma2(make_float2(__uint_as_float(sv[j]), __uint_as_float(sv[j + 1])), sc2, make_float2(-z.x, -z.y));
            float2 f = ffma2(make_float2(__uint_as_float(sv[j + 2]), __uint_as_float(sv[j + 3])), sc2, make_float2(-z.z, -z.w));
            wa = fadd2(wa, make_float2(ex2(e.x), ex2(e.y)));
            wb = fadd2(wb, make_float2(ex2(f.x), ex2(f.y)));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&acc_empty[group]));
        wa = fadd2(wa, wb);
        if (at != nullptr) *at = old + (wa.x + wa.y);
      }
      it += piece;
      c.t += piece - 1;
      if (it < count) attend_advance(p, c, TILE, kAll);
    }
  }
  // all roles are done (or gave up): free the tensor memory
  tc_fence_before();
  __syncthreads();
  if (wid == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace triattn
