// The softmax of a 128 x 128 score tile, shared by the tcgen05 attention
// kernels.  Two threads own a row, 64 scores each, 32 in registers at a time;
// its weights go to TMEM as the A operand of P V, over the same scores; its
// output accumulator is in TMEM, half of the columns to each of the two.
//
// Why two threads a row: with two tiles in flight the tensor pipe waits for
// one tile's softmax while it does the other's P V and next S (1024 cycles at
// D = 128); two threads halve the chain of 128 exponentials a row, and the
// price is one exchange of the row maximum through shared memory (16k causal
// prompt, calls one after another: one thread a row 2.25 ms, two 2.17).  The
// first 32 scores are read from TMEM twice (for the maximum, and again for the
// weights): with all 64 in registers the loop spilled (2.10 ms where it now
// takes 1.89, single calls).  All exponentials are MUFU's: taking one or two
// in eight from the FMA pipe cost 2 and 5 % of the call.
#pragma once

#include "kvbm_sm100.cuh"

namespace kvbm {

// A 4-D map over a 16-bit [B, H, N, D] operand, boxes of 64 elements x `rows`
// rows with 128-byte swizzle (kvbm_tc.cu).
bool make_attention_map(CUtensorMap* map, const void* base, bool bf16, int B, int H, int N, int D, const int64_t* st,
                        int rows);

namespace sm100 {

constexpr int kAttTile = 128;
constexpr int kAttCols = 64;  // scores of a row in one thread
// Growth of a row's maximum (base 2) over the reference (and kHead) that moves
// the reference: weights stay below 2^8, fp16 ones below 2^15, which the types
// hold.  (The difference is compared: adding the growth to a large reference
// rounds it.)
constexpr float kAttGrow = 8.f;

// A NaN among the values makes the maximum NaN (and with it the row).
__device__ __forceinline__ float max32_nan(const float (&v)[32]) {
  float mx[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) mx[e] = fmax_nan(v[e], v[e + 4]);
#pragma unroll
  for (int c = 8; c < 32; c += 8)
#pragma unroll
    for (int e = 0; e < 4; ++e) mx[e] = fmax3_nan(mx[e], v[c + e], v[c + e + 4]);
  return fmax3_nan(fmax_nan(mx[0], mx[1]), mx[2], mx[3]);
}

// Multiplies kCols accumulator columns of the thread's lane at `to` by f (whole warp).
template <int kCols>
__device__ __forceinline__ void scale_output(uint32_t to, float f) {
#pragma unroll
  for (int w = 0; w < kCols / 32; ++w) {
    float o[32];
    tmem_ld32(to + 32 * w, o);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] *= f;
    tmem_st32(to + 32 * w, o);
  }
}

// Weights of 32 scores, rounded to 16 bits, to the 16 columns at `ts`; returns
// their float32 sum (of the unrounded values).  The rounding is half a step of
// every weight, of either sign, about as much as the output's own; weights in
// two parts would double P V, half of the tensor work that binds these kernels.
//   kShift false: 2^(fl(v C) + shift), shift = -(reference in base 2).  The product
//                 is rounded before the sum, as it was in the reference: in one FMA
//                 the reference's rounding stays in every exponent of the row, up
//                 to half its step, and scores past 2^24 leave the 16-bit range
//                 (16k causal prompt 2.19 ms that way, 2.21 this)
//   kShift true:  2^((v + shift) C), shift = -(reference), so that a score of
//                 float32's lowest value less itself is 0
template <bool kBf16, bool kShift>
__device__ __forceinline__ float put_weights(const float (&v)[32], float C, float shift, uint32_t ts) {
  const float2 C2 = make_float2(C, C), N2 = make_float2(shift, shift);
  float2 s0 = make_float2(0.f, 0.f), s1 = s0;
  auto arg = [&](float a, float b) {
    if constexpr (kShift) {
      const float2 d = fadd2(make_float2(a, b), N2);
      return ffma2(d, C2, make_float2(0.f, 0.f));
    } else {
      return fadd2(ffma2(make_float2(a, b), C2, make_float2(0.f, 0.f)), N2);
    }
  };
  uint32_t p16[16];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = 4 * e;
    const float2 x0 = arg(v[c], v[c + 1]), x1 = arg(v[c + 2], v[c + 3]);
    const float2 p0 = make_float2(ex2(x0.x), ex2(x0.y)), p1 = make_float2(ex2(x1.x), ex2(x1.y));
    s0 = fadd2_ftz(s0, p0);
    s1 = fadd2_ftz(s1, p1);
    p16[2 * e] = pack16<kBf16>(p0.x, p0.y);
    p16[2 * e + 1] = pack16<kBf16>(p1.x, p1.y);
  }
  tmem_st16(ts, p16);
  s0 = fadd2(s0, s1);
  return s0.x + s0.y;
}

template <bool kBf16>
__device__ __forceinline__ bool finite16(uint32_t half) {
  const uint32_t e = kBf16 ? 0x7F80u : 0x7C00u;
  return (half & e) != e;
}

// Barrier kId of kCount threads, with one answer for all of them: whether any
// came with `stop`.  (Roles whose wait gave up leave together: nobody stays
// behind at a barrier.)
template <int kCount>
__device__ __forceinline__ bool bar_any(int id, bool stop) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)stop), "r"(id), "n"(kCount)
      : "memory");
  return r != 0;
}

// Zeroes the non-finite 16-bit elements of a 16-byte piece; true if any was.
template <bool kBf16>
__device__ __forceinline__ bool drop_nonfinite(uint4* p) {
  const uint4 w = *p;
  uint32_t x[4] = {w.x, w.y, w.z, w.w};
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (!finite16<kBf16>(x[e])) {
      x[e] &= 0xFFFF0000u;
      bad = true;
    }
    if (!finite16<kBf16>(x[e] >> 16)) {
      x[e] &= 0x0000FFFFu;
      bad = true;
    }
  }
  if (bad) *p = make_uint4(x[0], x[1], x[2], x[3]);
  return bad;
}

// Whether the 32 bits hold a non-finite 16-bit element: x * 0 + acc is NaN from
// then on (one instruction a word).
template <bool kBf16>
__device__ __forceinline__ uint32_t mark_nonfinite(uint32_t x, uint32_t acc) {
  uint32_t r;
  if constexpr (kBf16)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(acc));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(acc));
  return r;
}

// Takes the non-finite elements out of 16-byte pieces first, first + step, ...
// < count of a tile; true if there were any.  (Eight pieces a test: they are rare.)
template <bool kBf16, typename Skip>
__device__ __forceinline__ bool scrub_pieces(uint8_t* tile, int first, int step, int count, Skip&& skip) {
  bool bad = false;
  for (int i0 = first; i0 < count; i0 += 8 * step) {
    uint32_t acc = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * step;
      if (i >= count) continue;
      const uint4 w = *reinterpret_cast<const uint4*>(tile + i * 16);
      acc = mark_nonfinite<kBf16>(w.x, acc);
      acc = mark_nonfinite<kBf16>(w.y, acc);
      acc = mark_nonfinite<kBf16>(w.z, acc);
      acc = mark_nonfinite<kBf16>(w.w, acc);
    }
    if ((acc & 0x7FFF7FFFu) == 0u) continue;
    for (int i = i0; i < min(count, i0 + 8 * step); i += step)
      if (!skip(i)) bad |= drop_nonfinite<kBf16>(reinterpret_cast<uint4*>(tile + i * 16));
  }
  return bad;
}

// S = Q K^T of a 128 x 128 tile, both K-major with 128-byte swizzle.  By a whole
// warp in uniform control flow (elect_one): descriptors of later K steps are
// the first one plus a constant (addresses stay below 2^18, so no carry leaves
// the address field).
template <int DP>
__device__ __forceinline__ void issue_scores(uint32_t d_tmem, uint32_t q, uint32_t k, uint32_t idesc) {
  const uint64_t qd = sw128_desc(q), kd = sw128_desc(k);
  if (elect_one()) {
#pragma unroll
    for (int i = 0; i < DP / 64; ++i)
#pragma unroll
      for (int k4 = 0; k4 < 4; ++k4) {
        const uint64_t step = (uint64_t)((i * kAttTile * 128 + k4 * 32) >> 4);
        mma_f16(d_tmem, qd + step, kd + step, idesc, (i | k4) != 0);
      }
  }
  __syncwarp();
}

// O (+)= P V: P (128 x 128, 16 bit) in TMEM, the weights of each 32 keys over
// the first 16 columns of their own scores; V [128 keys][DP] MN-major.
template <int DP>
__device__ __forceinline__ void issue_output(uint32_t d_tmem, uint32_t p_tmem, uint32_t v, uint32_t idesc, uint32_t add) {
  const uint64_t vd = sw128_mn_desc(v, kAttTile * 128);
  if (elect_one()) {
#pragma unroll
    for (int k = 0; k < 8; ++k)  // 16 keys a step
      mma_f16_ts(d_tmem, p_tmem + (k >> 1) * 32 + (k & 1) * 8, vd + (uint64_t)((k * 2048) >> 4), idesc,
                 k > 0 ? 1u : add);
  }
  __syncwarp();
}

// Arrive on `bar` when the MMAs issued so far by this warp complete.  (The same
// lane is elected every time.)
__device__ __forceinline__ void commit_warp(uint64_t* bar) {
  if (elect_one()) mma_commit(bar);
  __syncwarp();
}

}  // namespace sm100
}  // namespace kvbm
