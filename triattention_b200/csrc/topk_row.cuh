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

// where(i) -> the address index of element i < n, fetch(index) -> its bits, key(bits, i) -> what it is ranked by.  put(rank, i) is called once for every chosen element
// (rank 0 .. k-1, ascending with i).  Rows of n <= cap (a multiple of 4; bits 16-byte aligned) are read once; they are
// counted and put segment by segment, a thread's segment being an odd number of consecutive elements (no bank conflicts), with a
// single scan over the threads.  Longer rows are read again in every pass, and put in runs of 4 * THREADS elements: all threads
// call run(sel, rank, i, bits) together, run by run in ascending order, before the puts of the next one.
template <int THREADS, class Where, class Fetch, class Key, class Put, class Run>
__device__ __forceinline__ void topk_row(int n, int k, unsigned* bits, int cap, TopkShared<THREADS>& sh, Where where,
                                         Fetch fetch, Key key, Put put, Run run) {
  constexpr int VEC = 4;
  const int tid = threadIdx.x;
  const bool cached = n <= cap;
  if (k <= 0) return;
  if (cached) {
    for (int i0 = tid; i0 < n; i0 += THREADS * 8) {  // eight look-ups, then eight loads in flight per thread
      long long at[8];
      unsigned v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) at[j] = where(min(i0 + j * THREADS, n - 1));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fetch(at[j]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j * THREADS < n) bits[i0 + j * THREADS] = v[j];
    }
  }
  auto bits_at = [&](int i) { return cached ? bits[i] : fetch(where(i)); };
  // four consecutive elements (those at or behind n are not used)
  auto four_at = [&](int i, unsigned(&v)[VEC]) {
    if (cached) {
      const uint4 w = *reinterpret_cast<const uint4*>(bits + i);
      v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = i + j < n ? bits_at(i + j) : 0u;
    }
  };
  if (k >= n) {  // everything stays where it is
    for (int i = tid; i < n; i += THREADS) put(i, i);
    return;
  }
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
    for (int i = tid * VEC; i < n; i += THREADS * VEC) {
      unsigned v[VEC];
      four_at(i, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const unsigned x = key(v[j], i + j);
        if (i + j < n && ((x ^ prefix) & himask) == 0u) atomicAdd(&sh.hist[(x >> shift) & (bins - 1u)], 1u);
      }
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
  if (cached) {
    const int len = ((n + THREADS - 1) / THREADS) | 1, i0 = min(tid * len, n), i1 = min(i0 + len, n);
    unsigned gt = 0u, eq = 0u;
    for (int i = i0; i < i1; ++i) {
      const unsigned x = key(bits[i], i);
      gt += x > kth ? 1u : 0u;
      eq += x == kth ? 1u : 0u;
    }
    // both prefixes in one scan where the counts fit 16 bits each (n < 65536: cap is below that)
    unsigned total;
    const unsigned before = topk_scan<THREADS>(gt | eq << 16, sh, total);
    unsigned eq_before = before >> 16, rank = (before & 0xffffu) + min(eq_before, need_eq);
    for (int i = i0; i < i1; ++i) {
      const unsigned x = key(bits[i], i);
      const bool border = x == kth;
      if (x > kth || (border && eq_before < need_eq)) put((int)rank++, i);
      eq_before += border ? 1u : 0u;
    }
    return;
  }
  unsigned base_eq = 0u, base_out = 0u;
  for (int i0 = 0; i0 < n; i0 += THREADS * VEC) {
    bool sel[VEC], eq[VEC];
    int rank[VEC], at[VEC];
    unsigned v[VEC] = {0u, 0u, 0u, 0u}, mine = 0u;  // this thread's counts: above the border, at the border (16 bits each)
    if (i0 + tid * VEC < n) four_at(i0 + tid * VEC, v);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      at[j] = i0 + tid * VEC + j;
      const unsigned x = at[j] < n ? key(v[j], at[j]) : 0u;
      sel[j] = at[j] < n && x > kth;
      eq[j] = at[j] < n && x == kth;
      mine += (sel[j] ? 1u : 0u) + (eq[j] ? 0x10000u : 0u);
    }
    unsigned total;
    unsigned before = topk_scan<THREADS>(mine, sh, total);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const unsigned eq_before = base_eq + (before >> 16);
      rank[j] = (int)(base_out + (before & 0xffffu) + (min(eq_before, need_eq) - min(base_eq, need_eq)));
      before += (sel[j] ? 1u : 0u) + (eq[j] ? 0x10000u : 0u);
      sel[j] = sel[j] || (eq[j] && eq_before < need_eq);
    }
    run(sel, rank, at, v);
    const unsigned eq_after = base_eq + (total >> 16);
    base_out += (total & 0xffffu) + (min(eq_after, need_eq) - min(base_eq, need_eq));
    base_eq = eq_after;
    if (base_out >= (unsigned)k) break;
  }
}

}  // namespace triattn
