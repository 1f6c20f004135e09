// Work items of the tensor-core prompt kernel: how CTAs find their row tiles, and the rows that belong to no sequence.
#pragma once

#include "kvbm_attention.cuh"

namespace kvbm {

// A work item: tile qt of kRows query rows of sequence b, head h.
struct Item {
  int b, h, qt;
};

// Tiles in order of falling qt (under causal the longest first), heads
// fastest: the heads of a group read the same keys at the same time.  With
// lengths on the device the CTA finds its tile by counting: cnt(q) = tiles of
// level >= q.  One warp.
template <int kRows>
__device__ __forceinline__ int tiles_of(const PromptArgs& a, int b) {
  return (seq_view(a.lens, a.cu, true, b, a.N, a.total).n + kRows - 1) / kRows;
}

template <int kRows>
__device__ __forceinline__ long long count_from(const PromptArgs& a, int q) {
  long long n = 0;
  for (int b = threadIdx.x & 31; b < a.B; b += 32) n += max(0, tiles_of<kRows>(a, b) - q);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

template <int kRows>
__device__ __forceinline__ Item find_item(const PromptArgs& a, long long L) {
  Item it;
  const int nt = (a.N + kRows - 1) / kRows;
  const long long i = L / a.Hq;
  it.h = (int)(L % a.Hq);
  if (a.lens == nullptr && a.cu == nullptr) {
    it.qt = nt - 1 - (int)(i / a.B);
    it.b = (int)(i % a.B);
    return it;
  }
  int lo = 0, hi = nt;  // cnt(lo) > i >= cnt(hi)
  long long chi = 0;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    const long long c = count_from<kRows>(a, mid);
    if (c > i)
      lo = mid;
    else {
      hi = mid;
      chi = c;
    }
  }
  it.qt = lo;
  long long left = i - chi;  // the left-th sequence with more than lo tiles
  const int lane = threadIdx.x & 31;
  it.b = 0;
  for (int base = 0; base < a.B; base += 32) {
    const int b = base + lane;
    const bool in = b < a.B && tiles_of<kRows>(a, b) > lo;
    const unsigned m = __ballot_sync(0xffffffffu, in);
    const int n = __popc(m);
    if (left < n) {
      const bool me = in && __popc(m & ((1u << lane) - 1u)) == (int)left;
      it.b = base + __ffs(__ballot_sync(0xffffffffu, me)) - 1;
      break;
    }
    left -= n;
  }
  return it;
}

// Rows of no sequence: out 0, lse -inf; thread `who` of `of`.
__device__ __forceinline__ void fill_rows(const PromptArgs& a, long long who, long long of) {
  // gap g: the rows between what sequence g - 1 covers and where sequence g starts
  const int gaps = a.cu != nullptr ? a.B + 1 : a.B;
  for (int g = 0; g < gaps; ++g) {
    long long r0, r1, bo = 0, bl = 0;
    if (a.cu != nullptr) {
      r0 = 0;
      if (g > 0) {
        const SeqView p = seq_view(nullptr, a.cu, true, g - 1, a.N, a.total);
        r0 = (long long)p.q_row + p.n;
      }
      r1 = g < a.B ? seq_view(nullptr, a.cu, true, g, a.N, a.total).q_row : a.total;
    } else {
      r0 = seq_view(a.lens, nullptr, true, g, a.N, a.total).n;
      r1 = a.N;
      bo = g * a.os[0];
      bl = g * a.ls[0];
    }
    const int vecs = a.D / 8;
    const long long n = (r1 - r0) * a.Hq;
    if (n <= 0) continue;
    for (long long e = who; e < n * vecs; e += of) {
      const int d = (int)(e % vecs);
      const long long rh = e / vecs;
      const int h = (int)(rh % a.Hq);
      const long long r = r0 + rh / a.Hq;
      uint16_t* out = static_cast<uint16_t*>(a.out) + bo + h * a.os[1] + r * a.os[2];
      *reinterpret_cast<uint4*>(out + d * 8) = make_uint4(0u, 0u, 0u, 0u);
      if (d == 0) a.lse[bl + h * a.ls[1] + r * a.ls[2]] = -INFINITY;
    }
  }
}

}  // namespace kvbm
