// The k largest keys of one row by one CTA: ties go to the lowest index, indices come out ascending.
// A row of up to `cap` keys is kept in shared memory after its first read; longer rows are read again per pass.
#pragma once

#include "common.cuh"

namespace triattn {

constexpr int kTopkBins = 2048;  // 11 bits per radix pass: three passes cover a 32-bit key

template <int THREADS>
struct TopkShared {
  unsigned hist[kTopkBins];
  unsigned warp_tot[THREADS / 32];
  unsigned prefix, remaining;
};

// exclusive prefix over the CTA's threads and the total; two barriers
template <int THREADS>
__device__ __forceinline__ unsigned topk_scan(unsigned v, TopkShared<THREADS>& sh, unsigned& total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  unsigned incl = v;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const unsigned u = __shfl_up_sync(0xffffffffu, incl, s);
    if (lane >= s) incl += u;
  }
  if (lane == 31) sh.warp_tot[wid] = incl;
  __syncthreads();
  const unsigned w = lane < THREADS / 32 ? sh.warp_tot[lane] : 0u;
  unsigned winc = w;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const unsigned u = __shfl_up_sync(0xffffffffu, winc, s);
    if (lane >= s) winc += u;
  }
  total = __shfl_sync(0xffffffffu, winc, 31);
  const unsigned before = __shfl_sync(0xffffffffu, winc - w, wid);
  __syncthreads();
  return before + incl - v;
}

// load(i) -> key of element i < n (called once per element when n <= cap).  emit(sel, rank, i) is called by all threads
// together, for runs of THREADS consecutive elements in ascending order: where sel holds, element i is chosen with that
// rank (0 .. k-1, ascending with i).
template <int THREADS, class Load, class Emit>
__device__ __forceinline__ void topk_row(int n, int k, unsigned* keys, int cap, TopkShared<THREADS>& sh, Load load, Emit emit) {
  const int tid = threadIdx.x;
  const bool cached = n <= cap;
  if (k <= 0) return;
  if (k >= n) {
    for (int i0 = 0; i0 < n; i0 += THREADS) emit(i0 + tid < n, i0 + tid, i0 + tid);
    return;
  }
  if (cached)
    for (int i = tid; i < n; i += THREADS) keys[i] = load(i);
  auto key_at = [&](int i) { return cached ? keys[i] : load(i); };
  if (tid == 0) {
    sh.prefix = 0u;
    sh.remaining = (unsigned)k;
  }
  unsigned himask = 0u;
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const unsigned bins = pass == 2 ? 1024u : 2048u;
    for (int i = tid; i < kTopkBins; i += THREADS) sh.hist[i] = 0u;
    __syncthreads();
    const unsigned prefix = sh.prefix, remaining = sh.remaining;
    for (int i = tid; i < n; i += THREADS) {
      const unsigned key = key_at(i);
      if (((key ^ prefix) & himask) == 0u) atomicAdd(&sh.hist[(key >> shift) & (bins - 1u)], 1u);
    }
    __syncthreads();
    // thread t owns PER consecutive bins, from the top
    constexpr int PER = kTopkBins / THREADS;
    unsigned local[PER], sum = 0u;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const unsigned bin = tid * PER + j;
      local[j] = bin < bins ? sh.hist[bins - 1u - bin] : 0u;
      sum += local[j];
    }
    unsigned total;
    unsigned above = topk_scan<THREADS>(sum, sh, total);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (above < remaining && above + local[j] >= remaining) {
        sh.prefix = prefix | ((bins - 1u - (tid * PER + j)) << shift);
        sh.remaining = remaining - above;
      }
      above += local[j];
    }
    himask |= (bins - 1u) << shift;
    __syncthreads();
  }
  const unsigned kth = sh.prefix, need_eq = sh.remaining;
  unsigned base_eq = 0u, base_out = 0u;
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + tid;
    const unsigned key = i < n ? key_at(i) : 0u;
    const bool gt = i < n && key > kth, eq = i < n && key == kth;
    // both prefixes at once: counts of a chunk fit 16 bits each
    unsigned total;
    const unsigned pre = topk_scan<THREADS>((gt ? 1u : 0u) | (eq ? 0x10000u : 0u), sh, total);
    const unsigned eq_before = base_eq + (pre >> 16), gt_before = pre & 0xffffu;
    const bool sel = gt || (eq && eq_before < need_eq);
    const unsigned rank = base_out + gt_before + (min(eq_before, need_eq) - min(base_eq, need_eq));
    emit(sel, (int)rank, i);
    const unsigned eq_after = base_eq + (total >> 16);
    base_out += (total & 0xffffu) + (min(eq_after, need_eq) - min(base_eq, need_eq));
    base_eq = eq_after;
    if (base_out >= (unsigned)k) break;
  }
}

}  // namespace triattn
