// Attention of a few rows per kv head over a paged cache (R = G * T up to 32,
// in tiles of 16 rows: single tokens, small trees; with weights to accumulate,
// D > 128 or a scale <= 0 any R), bf16 / fp16, split over the keys.
//
// Bound by reading k and v once per 16 rows.  Every CTA gets the same number of
// 64-key tiles (kvbm_attention.cu describes the split and the joining); three
// CTAs an SM with rings of two tiles (32 sequences of 4-8k keys: 158 us, 5.2
// TB/s) hide a tile's chain of products and shuffles better than two CTAs with
// three (174 us).  A CTA of four warps has a ring of kStages tiles of k and v:
// while one is computed, kStages - 1 are in flight with 16-byte cp.async (page
// lookups one tile further ahead), rows swizzled so that ldmatrix meets no bank
// conflict; warp w takes keys 16 w .. 16 w + 15 of each tile with mma.m16n8k16:
// one A tile holds 16 rows, so every k and v element leaves shared memory once
// for them.  Each warp has a running maximum and sum of its own; the four are
// joined once per unit.  mma.sync rather than tcgen05: 16 rows
// would fill an eighth of a tcgen05 tile, and at 64 FLOP a byte at most the
// tensor work of a tile is a third of the time its bytes take.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "kvbm_attention.cuh"

namespace kvbm {
namespace {

constexpr int KT = kCachedKeyTile;  // 64 keys a tile
constexpr int kThreads = 128;
constexpr int BM = 16;
constexpr float kGrow = 5.5f;  // growth (natural log) of a row's maximum over the reference (and kHead) that moves it

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;  // 0: the 16 bytes are zero-filled, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (kBf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (kBf16) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
  } else {
    const __half2 h = *reinterpret_cast<const __half2*>(&x);
    return __half22float2(h);
  }
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool kBf16>
__device__ __forceinline__ bool finite16(uint32_t half) {
  const uint32_t e = kBf16 ? 0x7F80u : 0x7C00u;
  return (half & e) != e;
}

// Which non-finite values the v rows of slots [lo, hi), kept by every row, hold
// in each column: bit 0 +inf, bit 1 -inf, bit 2 NaN.  The whole CTA.
template <int DP, bool kBf16, typename T>
__device__ __noinline__ void find_nonfinite(const CachedArgs& a, int b, int g, int lo, int hi, uint32_t* flags) {
  constexpr int kChunks = DP / 8, kAhead = 8;
  const float* off = a.off ? a.off + b * a.ob + g * a.oh : nullptr;
  for (int i = threadIdx.x; i < DP; i += kThreads) flags[i] = 0;
  __syncthreads();
  const int ch = threadIdx.x % kChunks;
  for (int c0 = lo + threadIdx.x / kChunks; c0 < hi; c0 += kAhead * (kThreads / kChunks)) {
    uint4 w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int c = c0 + i * (kThreads / kChunks);
      w[i] = make_uint4(0u, 0u, 0u, 0u);
      if (c >= hi || ch * 8 >= a.D || (off != nullptr && off[c] == -INFINITY)) continue;
      const int page = a.pg.page(b, a.pg.page_index(c));
      if (page < 0 || page >= a.pg.num_pages) continue;
      w[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) + (long long)page * a.vs[0] +
                                             (long long)a.pg.slot(c) * a.vs[1] + g * a.vs[2] + ch * 8);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t h = (x[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
        if (finite16<kBf16>(h)) continue;
        atomicOr(&flags[ch * 8 + e], (h & (kBf16 ? 0x7Fu : 0x3FFu)) != 0 ? 4u : h >> 15 ? 2u : 1u);
      }
    }
  }
  __syncthreads();
}

template <int DP>
struct Cfg {
  static constexpr int kChunks = DP / 8;              // 16-byte chunks of a row
  static constexpr int kTileBytes = KT * DP * 2;      // k or v of one tile
  static constexpr int kStages = DP == 64 ? 4 : DP == 128 ? 2 : 3;
  static constexpr int kRowsPerPass = kThreads / kChunks;
  static constexpr int kPasses = KT / kRowsPerPass;
  static constexpr int kPitch = DP + 4;               // floats of a row of the joining buffer
  static constexpr size_t kRing = (size_t)kStages * 2 * kTileBytes;
  static constexpr size_t kSmem = kRing + (kStages + 1) * KT * 16 + BM * DP * 2 + 4 * BM * 8 + 64;
  static_assert(kRing >= sizeof(float) * 4 * BM * kPitch, "the joining buffer reuses the ring");
  static_assert((kStages + 1) * KT * 16 >= DP * 4, "the columns' flags reuse the offsets");
};

template <int DP, bool kBf16>
__global__ void __launch_bounds__(kThreads, DP <= 128 ? kMmaCtas : 1) cached_mma_kernel(const __grid_constant__ CachedArgs a) {
  using CF = Cfg<DP>;
  using T = std::conditional_t<kBf16, __nv_bfloat16, __half>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  longlong2* offs = reinterpret_cast<longlong2*>(smem + CF::kRing);     // [kStages + 1][KT] element offsets of k, v rows (-1: zeros)
  uint8_t* qs = reinterpret_cast<uint8_t*>(offs + (CF::kStages + 1) * KT);              // [BM][DP] swizzled
  float2* ml_s = reinterpret_cast<float2*>(qs + BM * DP * 2);           // [4][BM]
  long long* sched = reinterpret_cast<long long*>(ml_s + 4 * BM);       // total, first, b
  volatile int* bad_flag = reinterpret_cast<volatile int*>(sched + 3);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  cudaTriggerProgrammaticLaunchCompletion();  // the joining kernel may be set up beside this one
  if (warp == 0) {
    long long pre, total, first = 0;
    warp_tile_prefix(a, 0, &pre, &total);
    const int b = warp_find_seq(a, split_begin(blockIdx.x, total, a.C), &first);
    if (lane == 0) {
      sched[0] = total;
      sched[1] = first;
      sched[2] = b;
      *bad_flag = 0;
    }
  }
  __syncthreads();
  const long long total = sched[0];
  const long long begin = split_begin(blockIdx.x, total, a.C), end = split_begin(blockIdx.x + 1, total, a.C);
  long long bfirst = sched[1];
  int b = (int)sched[2];
  const uint32_t ring_a = smem_addr(ring), qs_a = smem_addr(qs);
  const T *kbase = static_cast<const T*>(a.k), *vbase = static_cast<const T*>(a.v);

  for (long long at = begin; at < end;) {
    int len = cached_len(a, b), nt = (len + KT - 1) / KT;
    while (at >= bfirst + (long long)nt * a.Hkv * a.RT) {
      bfirst += (long long)nt * a.Hkv * a.RT;
      ++b;
      len = cached_len(a, b);
      nt = (len + KT - 1) / KT;
    }
    const int u = (int)((at - bfirst) / nt), g = u / a.RT, rt = u % a.RT;
    const long long ufirst = bfirst + (long long)u * nt;
    const int k0 = (int)(at - ufirst), k1 = (int)min((long long)nt, end - ufirst);
    const int pre = len - a.T;
    const float* off = a.off ? a.off + b * a.ob + g * a.oh : nullptr;
    const uint8_t* tree = a.tree ? a.tree + b * a.tb : nullptr;
    const bool drafts = a.T > 1 || tree != nullptr;  // rows may drop slots from `pre` on (a single token without a mask keeps its own)

    // ---- element offsets of a tile's rows, kStages tiles ahead of their use
    auto page_of = [&](int tile, int i) -> int {  // the page id of row i of a tile (-1: none)
      const int c = tile * KT + i;
      if (tile >= k1 || c >= len) return -1;
      return a.pg.page(b, a.pg.page_index(c));
    };
    auto put_offsets = [&](int tile, int i, int page) {
      if (tile >= k1) return;
      const int c = tile * KT + i;
      longlong2 o = make_longlong2(-1, -1);
      if (c < len && !(off != nullptr && off[c] == -INFINITY)) {
        if (page >= 0 && page < a.pg.num_pages) {
          const int in = a.pg.slot(c);
          o.x = (long long)page * a.ks[0] + (long long)in * a.ks[1] + g * a.ks[2];
          o.y = (long long)page * a.vs[0] + (long long)in * a.vs[1] + g * a.vs[2];
        } else {
          atomicOr(a.page_error, 1u);
        }
      }
      offs[((tile - k0) % (CF::kStages + 1)) * KT + i] = o;
    };
    auto load_tile = [&](int tile) {
      if (tile < k1) {
        const uint32_t kd = ring_a + ((tile - k0) % CF::kStages) * 2 * CF::kTileBytes;
        const int ch = tid % CF::kChunks;
        const bool in = ch * 8 < a.D;
#pragma unroll
        for (int i = 0; i < CF::kPasses; ++i) {
          const int r = tid / CF::kChunks + i * CF::kRowsPerPass;
          const longlong2 o = offs[((tile - k0) % (CF::kStages + 1)) * KT + r];
          const bool live = in && o.x >= 0;
          const uint32_t d = r * (DP * 2) + ((ch ^ (r & 7)) << 4);
          cp16(kd + d, live ? kbase + o.x + ch * 8 : kbase, live);
          cp16(kd + CF::kTileBytes + d, live ? vbase + o.y + ch * 8 : vbase, live);
        }
      }
      cp_commit();
    };

    // the first kStages tiles at once (their table reads overlap), then the queries
    {
      constexpr int kEach = (CF::kStages * KT + kThreads - 1) / kThreads;
      int page[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) page[i] = page_of(k0 + (tid + i * kThreads) / KT, tid % KT);
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (tid + i * kThreads < CF::kStages * KT) put_offsets(k0 + (tid + i * kThreads) / KT, tid % KT, page[i]);
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < CF::kStages - 1; ++i) load_tile(k0 + i);
    for (int i = tid; i < BM * CF::kChunks; i += kThreads) {
      const int r = i / CF::kChunks, ch = i % CF::kChunks, rr = rt * BM + r;
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (rr < a.R && ch * 8 < a.D)
        w = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qs[0] +
                                            (long long)(g * a.G + rr / a.T) * a.qs[1] +
                                            (long long)(rr % a.T) * a.qs[2] + ch * 8);
      *reinterpret_cast<uint4*>(qs + r * (DP * 2) + ((ch ^ (r & 7)) << 4)) = w;
    }
    int next_page = tid < KT ? page_of(k0 + CF::kStages, tid) : -1;
    __syncthreads();

    uint32_t qf[DP <= 128 ? DP / 16 : 1][4];
    const uint32_t q_row = (lane & 7) + ((lane >> 3) & 1) * 8, q_ch = lane >> 4;
    auto q_frag = [&](int ks, uint32_t (&r)[4]) {
      ldsm4(r, qs_a + q_row * (DP * 2) + (((ks * 2 + q_ch) ^ (q_row & 7)) << 4));
    };
    if constexpr (DP <= 128) {
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) q_frag(ks, qf[ks]);
    }

    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int rq = lane >> 2, cq = (lane & 3) * 2;

#pragma unroll 1
    for (int tile = k0; tile < k1; ++tile) {
      const int c0 = tile * KT + warp * 16;  // this warp's keys
      float bias[4];
      if (off != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = c0 + (e >> 1) * 8 + cq + (e & 1);
          bias[e] = c < len ? off[c] : -INFINITY;
        }
      }
      cp_wait<CF::kStages - 2>();
      __syncthreads();
      load_tile(tile + CF::kStages - 1);
      if (tid < KT) {
        put_offsets(tile + CF::kStages, tid, next_page);
        next_page = page_of(tile + CF::kStages + 1, tid);
      }
      const uint32_t kt = ring_a + ((tile - k0) % CF::kStages) * 2 * CF::kTileBytes + warp * 16 * (DP * 2);
      const uint32_t vt = kt + CF::kTileBytes;
      if (drafts && c0 + 16 > pre && c0 < len) {
        // drafted tokens: rows differ in which they keep.  Their non-finite
        // v elements are taken out here and added to the rows that keep them
        // at the end.  (Slots before them stay as they are: every row keeps them.)
        bool bad = false;
        for (int i = lane; i < 16 * CF::kChunks; i += 32) {
          if (c0 + i / CF::kChunks < pre) continue;
          uint4* p = reinterpret_cast<uint4*>(ring + (vt - ring_a) + i * 16);
          const uint4 w = *p;
          uint32_t x[4] = {w.x, w.y, w.z, w.w};
          bool hit = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (!finite16<kBf16>(x[e])) {
              x[e] &= 0xFFFF0000u;
              hit = true;
            }
            if (!finite16<kBf16>(x[e] >> 16)) {
              x[e] &= 0x0000FFFFu;
              hit = true;
            }
          }
          if (hit) *p = make_uint4(x[0], x[1], x[2], x[3]);
          bad |= hit;
        }
        if (bad) *bad_flag = 1;
        __syncwarp();
      }
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const uint32_t krow = (lane & 7) + (lane >> 4) * 8, kch = (lane >> 3) & 1;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        uint32_t kf[4], q4[4];
        ldsm4(kf, kt + krow * (DP * 2) + (((ks * 2 + kch) ^ (krow & 7)) << 4));
        if constexpr (DP <= 128) {
#pragma unroll
          for (int e = 0; e < 4; ++e) q4[e] = qf[ks][e];
        } else {
          q_frag(ks, q4);
        }
        mma16816<kBf16>(s[0], q4, kf[0], kf[1]);
        mma16816<kBf16>(s[1], q4, kf[2], kf[3]);
      }
      // s[nt][e]: row rq + 8 (e / 2), key c0 + 8 nt + cq + (e & 1)
#pragma unroll
      for (int nt2 = 0; nt2 < 2; ++nt2)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt2][e] *= a.scale;
          if (off != nullptr) s[nt2][e] += bias[nt2 * 2 + (e & 1)];
        }
      if (off != nullptr) {
#pragma unroll
        for (int nt2 = 0; nt2 < 2; ++nt2)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (bias[nt2 * 2 + (e & 1)] == -INFINITY) s[nt2][e] = -INFINITY;
      }
      if (c0 + 16 > (drafts ? pre : len)) {
#pragma unroll
        for (int nt2 = 0; nt2 < 2; ++nt2)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = c0 + nt2 * 8 + cq + (e & 1), tok = (rt * BM + rq + (e >> 1) * 8) % a.T;
            bool keep = c < len;
            if (keep && drafts && c >= pre) keep = tree ? tree[tok * a.tr + (c - pre)] != 0 : c - pre <= tok;
            if (!keep) s[nt2][e] = -INFINITY;
          }
      }
      if (a.scores != nullptr) {  // T = 1: rows are the heads of the group
        float* sc = a.scores + ((long long)(b * a.Hkv + g) * a.G) * a.Lmax;
#pragma unroll
        for (int nt2 = 0; nt2 < 2; ++nt2)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = c0 + nt2 * 8 + cq + (e & 1), r = rt * BM + rq + (e >> 1) * 8;
            if (r < a.R && c < len) sc[(long long)r * a.Lmax + c] = s[nt2][e];
          }
      }
      float f[2] = {1.f, 1.f};
      bool grew = false;
#pragma unroll
      for (int hrow = 0; hrow < 2; ++hrow) {
        float top = max_nan(max_nan(s[0][2 * hrow], s[0][2 * hrow + 1]), max_nan(s[1][2 * hrow], s[1][2 * hrow + 1]));
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
        constexpr float head = kHead<kBf16> * kLn2F;
        if (top - m[hrow] > kGrow + head || top != top) {  // (true from -inf to anything finite, and for NaN)
          const float mn = top - head;
          f[hrow] = m[hrow] == mn ? 1.f : ex2f((m[hrow] - mn) * kLog2eF);
          m[hrow] = mn;
          grew = true;
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][0] *= f[0];
          o[i][1] *= f[0];
          o[i][2] *= f[1];
          o[i][3] *= f[1];
        }
        l[0] *= f[0];
        l[1] *= f[1];
      }
      uint32_t pf[4], pl[4];
      {
        const float b0 = m[0] == -INFINITY ? 0.f : m[0], b1 = m[1] == -INFINITY ? 0.f : m[1];
        float p[2][4];
#pragma unroll
        for (int nt2 = 0; nt2 < 2; ++nt2)
#pragma unroll
          for (int e = 0; e < 4; ++e) p[nt2][e] = ex2f((s[nt2][e] - (e < 2 ? b0 : b1)) * kLog2eF);
        l[0] += (p[0][0] + p[0][1]) + (p[1][0] + p[1][1]);
        l[1] += (p[0][2] + p[0][3]) + (p[1][2] + p[1][3]);
        // For the product with v a weight is split into two 16-bit parts, high and
        // rest: 3 % of the time (153 -> 158 us at 32 sequences), and the rounding of
        // the result is then the only one of its size (one part alone: 1.4 times its
        // error), but for fp16 weights so small that both parts are subnormal (kHead).
        pf[0] = pack2<kBf16>(p[0][0], p[0][1]);
        pf[1] = pack2<kBf16>(p[0][2], p[0][3]);
        pf[2] = pack2<kBf16>(p[1][0], p[1][1]);
        pf[3] = pack2<kBf16>(p[1][2], p[1][3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 hi = unpack2<kBf16>(pf[e]);
          pl[e] = pack2<kBf16>(p[e >> 1][2 * (e & 1)] - hi.x, p[e >> 1][2 * (e & 1) + 1] - hi.y);
        }
      }
      const uint32_t vrow = (lane & 7) + ((lane >> 3) & 1) * 8, vch = lane >> 4;
#pragma unroll
      for (int dp = 0; dp < DP / 16; ++dp) {
        uint32_t vf[4];
        ldsm4_t(vf, vt + vrow * (DP * 2) + (((dp * 2 + vch) ^ (vrow & 7)) << 4));
        mma16816<kBf16>(o[2 * dp], pf, vf[0], vf[1]);
        mma16816<kBf16>(o[2 * dp + 1], pf, vf[2], vf[3]);
        mma16816<kBf16>(o[2 * dp], pl, vf[0], vf[1]);
        mma16816<kBf16>(o[2 * dp + 1], pl, vf[2], vf[3]);
      }
    }
    // ---- join the four warps
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) {
      l[hrow] += __shfl_xor_sync(0xffffffffu, l[hrow], 1);
      l[hrow] += __shfl_xor_sync(0xffffffffu, l[hrow], 2);
      if ((lane & 3) == 0) ml_s[warp * BM + rq + 8 * hrow] = make_float2(m[hrow], l[hrow]);
    }
    // The second part of a weight is zero or of either sign, so an infinite v of a kept key makes its column NaN:
    // a unit that ends with anything non-finite looks for it (32 sequences of 8192 keys: 0.17 ms, with one 0.59).
    float zero = 0.f;  // NaN from the first non-finite value on
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) zero = fmaf(o[i][e], 0.f, zero);
    cp_wait<0>();
    const bool odd = __syncthreads_or(zero != 0.f);  // every warp is done with the ring
    uint32_t* flags = reinterpret_cast<uint32_t*>(offs);
    if (odd) find_nonfinite<DP, kBf16, T>(a, b, g, k0 * KT, min(drafts ? pre : len, k1 * KT), flags);
    float* ob = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int hrow = 0; hrow < 2; ++hrow)
        *reinterpret_cast<float2*>(ob + (warp * BM + rq + 8 * hrow) * CF::kPitch + i * 8 + cq) =
            make_float2(o[i][2 * hrow], o[i][2 * hrow + 1]);
    __syncthreads();
    const bool whole = k0 == 0 && k1 == nt, bad = *bad_flag != 0;
    const int slot = begin >= ufirst ? 0 : 1;
    const int rl = tid >> 3, r = rt * BM + rl;
    if (r < a.R) {
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml_s[w * BM + rl].x);
      const float base = mm == -INFINITY ? 0.f : mm;
      float f[4], ll = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 x = ml_s[w * BM + rl];
        f[w] = ex2f((x.x - base) * kLog2eF);
        ll = fmaf(x.y, f[w], ll);
      }
      const int h = g * a.G + r / a.T, tok = r % a.T;
      T* out = static_cast<T*>(a.out) + b * a.os[0] + h * a.os[1] + tok * a.os[2];
      const long long pr = ((long long)blockIdx.x * 2 + slot) * a.BM + rl;
      const float inv = 1.f / ll;
      for (int d = (tid & 7) * 4; d < DP; d += 32) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(ob + (w * BM + rl) * CF::kPitch + d);
          acc.x = fmaf(x.x, f[w], acc.x);
          acc.y = fmaf(x.y, f[w], acc.y);
          acc.z = fmaf(x.z, f[w], acc.z);
          acc.w = fmaf(x.w, f[w], acc.w);
        }
        if (bad && d < a.D) add_nonfinite<T>(a, b, g, tok, max(max(pre, 0), k0 * KT), min(len, k1 * KT), pre, d, acc);
        if (odd && !isnan(ll) && d < a.D) {
          // a NaN column is the sum of its non-finite values (their weights are positive)
          auto value = [&](int e) {
            const uint32_t f = flags[d + e];
            return f == 0 ? 0.f : f == 1 ? INFINITY : f == 2 ? -INFINITY : NAN;
          };
          float4 x = make_float4(value(0), value(1), value(2), value(3));
          if (bad) add_nonfinite<T>(a, b, g, tok, max(max(pre, 0), k0 * KT), min(len, k1 * KT), pre, d, x);
          if (isnan(acc.x) && x.x != 0.f) acc.x = x.x;
          if (isnan(acc.y) && x.y != 0.f) acc.y = x.y;
          if (isnan(acc.z) && x.z != 0.f) acc.z = x.z;
          if (isnan(acc.w) && x.w != 0.f) acc.w = x.w;
        }
        if (whole) {
          if (d < a.D) {
            const bool none = ll == 0.f;
            uint2 w;
            w.x = none ? 0u : pack2<kBf16>(acc.x * inv, acc.y * inv);
            w.y = none ? 0u : pack2<kBf16>(acc.z * inv, acc.w * inv);
            *reinterpret_cast<uint2*>(out + d) = w;
          }
        } else {
          *reinterpret_cast<float4*>(a.part_o + pr * a.DP + d) = acc;
        }
      }
      if ((tid & 7) == 0) {
        if (whole) {
          a.lse[b * a.ls[0] + h * a.ls[1] + tok * a.ls[2]] = ll == 0.f ? -INFINITY : mm + logf(ll);
          if (a.stats) a.stats[(long long)(b * a.Hkv + g) * a.R + r] = make_float2(mm, ll == 0.f ? 0.f : inv);
        } else {
          a.part_ml[pr] = make_float2(mm, ll);
        }
      }
    }
    __syncthreads();  // the ring and the flag are free again
    if (tid == 0) *bad_flag = 0;
    at = ufirst + k1;
  }
}

template <int DP, bool kBf16>
int launch(const CachedArgs& a, cudaStream_t s) {
  auto kern = cached_mma_kernel<DP, kBf16>;
  constexpr size_t bytes = Cfg<DP>::kSmem;
  if (allow_smem(kern, bytes) != KVBM_OK) return KVBM_ERR_CUDA;
  kern<<<(unsigned)a.C, kThreads, bytes, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
}

}  // namespace

int launch_cached_mma(const CachedArgs& a, int dtype, cudaStream_t s) {
  const bool bf16 = dtype == KVBM_BF16;
  if (a.DP == 64) return bf16 ? launch<64, true>(a, s) : launch<64, false>(a, s);
  if (a.DP == 128) return bf16 ? launch<128, true>(a, s) : launch<128, false>(a, s);
  return bf16 ? launch<256, true>(a, s) : launch<256, false>(a, s);
}

}  // namespace kvbm
