// Attention by plain FFMA tiles: prompt attention and attention over a paged
// cache for fp32 inputs, and for 16-bit inputs whose head dim, strides or
// scale the tensor-core kernels do not take; also the joining of split units
// and the accumulation of per-key weights, which every cache kernel shares.
//
//   x_rc  = scale * q_r . k_c (+ log_offset_c)        for kept (r, c)
//   lse_r = log sum_c exp(x_rc),  out_r = sum_c exp(x_rc - lse_r) v_c
//
// One pass over the keys with a running maximum m and sum l per row:
// when a key tile raises m, l and the output row are multiplied by
// exp(m_old - m_new).  A row that keeps no key has l = 0: out 0, lse -inf.
//
// Tiles: 16 x 16 threads own RPT x 4 scores each (RPT = 4: 64 rows, for
// prompts and wide trees; RPT = 1: 16 rows, for single tokens), 64 keys a
// tile, everything in fp32 registers and shared memory.  fp32 rows in 16-byte
// pieces and D <= 128 (kAsync): k and v are double-buffered with cp.async, so that
// a tile's products hide the next one's loads.  Measured (fp32, 2048-token causal
// prompt, 8 heads of 64): 157 us, 27 TFLOP/s; 32 heads of 128: 1045 us, 33.
// Bound by shared memory's reads: 8 float4 a thread feed 64 FFMAs, and a float4
// read of a warp takes 4 passes, twice the FFMAs' time.  8 x 4 scores a thread
// need 6 instead of 8, but leave half the warps to hide latencies (158 us, and
// 1219 at D = 128); 2 x 8 need 10 (180 us).
#include <cooperative_groups.h>

#include <atomic>
#include <type_traits>

#include "kvbm_attention.cuh"
#include "kvbm_sm100.cuh"

namespace kvbm {
namespace {

// Set when a block-table entry lies outside [0, num_pages); the rows it
// names count as zero vectors.
__device__ unsigned int g_attention_page_error = 0;

constexpr int kThreads = 256;
constexpr int BN = 64;
constexpr int kPad = 4;

// Sign bit set: a masked pair (its value is not to be added, whatever it holds).
__device__ __forceinline__ bool masked_p(float p) { return __float_as_int(p) < 0; }

template <int RPT, int DP>
struct Tile {
  static constexpr int BM = 16 * RPT;
  static constexpr int kStride = DP + kPad;
  static constexpr int kPs = BN + kPad;
  static constexpr size_t bytes(int buffers) {
    return sizeof(float) * ((size_t)(BM + 2 * BN * buffers) * kStride + (size_t)BM * kPs + BN * buffers);
  }
  float o[RPT][DP / 16];
  float m[RPT], l[RPT];

  __device__ void reset() {
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) o[i][d] = 0.f;
    }
  }
};

// Four consecutive elements of a row from d (zeros past D or for a null row).
template <typename T>
__device__ __forceinline__ float4 load4(const T* row, int d, int D, long long ds, bool vec) {
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (row == nullptr || d >= D) return r;
  if (vec) {  // D % 4 == 0, unit stride, aligned rows
    if constexpr (sizeof(T) == 4) {
      r = *reinterpret_cast<const float4*>(row + d);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(row + d);
      const T* e = reinterpret_cast<const T*>(&u);
      r = make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
    }
    return r;
  }
  r.x = to_f32(row[d * ds]);
  if (d + 1 < D) r.y = to_f32(row[(d + 1) * ds]);
  if (d + 2 < D) r.z = to_f32(row[(d + 2) * ds]);
  if (d + 3 < D) r.w = to_f32(row[(d + 3) * ds]);
  return r;
}

// The tiles of shared memory: Q [BM], P [BM][BN + 4], then for each buffer
// K [BN], V [BN] (fp32, rows of DP + 4), bias [BN].
template <int RPT, int DP>
struct Smem {
  using TL = Tile<RPT, DP>;
  float *q, *k, *v, *p, *bias;
  __device__ explicit Smem(float* base, int buffer = 0) {
    q = base;
    p = q + TL::BM * TL::kStride;
    k = p + TL::BM * TL::kPs + buffer * (2 * BN * TL::kStride + BN);
    v = k + BN * TL::kStride;
    bias = v + BN * TL::kStride;
  }
};

// load_rows by cp.async (fp32 rows in 16-byte pieces); `any`: a readable address.
template <int DP, class F>
__device__ __forceinline__ void copy_rows(float* dst, int rows, F&& f, int D, const float* any) {
  constexpr int kVecs = DP / 4;
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * kVecs; i += kThreads) {
    const int r = i / kVecs, d = (i % kVecs) * 4;
    const float* row = f(r);
    const bool live = row != nullptr && d < D;
    const int n = live ? 16 : 0;  // 0: zero-filled, nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(dst + r * (DP + kPad) + d)),
                 "l"(live ? row + d : any), "r"(n)
                 : "memory");
  }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// rows(r) -> const T* of row r of the tile, or null
template <typename T, int RPT, int DP, class F>
__device__ __forceinline__ void load_rows(float* dst, int rows, F&& f, int D, long long ds, bool vec) {
  constexpr int kVecs = DP / 4;
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * kVecs; i += kThreads) {
    const int r = i / kVecs, d = (i % kVecs) * 4;
    *reinterpret_cast<float4*>(dst + r * (DP + kPad) + d) = load4<T>(f(r), d, D, ds, vec);
  }
}

// One key tile: scores of the tile's 64 keys (K, V, bias already in shared
// memory), softmax update, output update.  keep(r, j): whether row r keeps
// key j of the tile.  sink(r, j, x): called for each kept-or-not score.
// select: some row may drop a key that another keeps, so products of dropped
// pairs are left out one by one (0 * NaN is not 0).
// Products go two by two (fma.rn.f32x2): half the issue slots, and the slots
// bound as much as shared memory's reads (2048-token causal prompt, 8 heads of
// 64: 165 -> 157 us; 32 heads of 128: 1218 -> 1045).
template <int RPT, int DP, class Keep, class Sink>
__device__ __forceinline__ void tile_step(Tile<RPT, DP>& t, const Smem<RPT, DP>& s, float scale, bool has_bias,
                                          bool select, Keep&& keep, Sink&& sink) {
  using TL = Tile<RPT, DP>;
  constexpr int KC = DP / 16;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float2 x2[RPT][4];  // sums over the even and the odd elements
#pragma unroll
  for (int i = 0; i < RPT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) x2[i][j] = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 qv[RPT], kv[4];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
      qv[i] = *reinterpret_cast<const float4*>(s.q + (ty * RPT + i) * TL::kStride + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(s.k + (tx + 16 * j) * TL::kStride + d);
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x2[i][j] = sm100::ffma2(make_float2(qv[i].x, qv[i].y), make_float2(kv[j].x, kv[j].y), x2[i][j]);
        x2[i][j] = sm100::ffma2(make_float2(qv[i].z, qv[i].w), make_float2(kv[j].z, kv[j].w), x2[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = ty * RPT + i;
    float x[4], top = -INFINITY;
    bool kp[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = tx + 16 * j;
      // natural-log domain: an offset of the type's lowest value stays finite
      x[j] = (x2[i][j].x + x2[i][j].y) * scale;
      if (has_bias) x[j] += s.bias[c];
      kp[j] = keep(r, c);
      if (!kp[j]) x[j] = -INFINITY;
      sink(r, c, x[j]);
      top = fmaxf(top, x[j]);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float mn = fmaxf(t.m[i], top);
    const float base = mn == -INFINITY ? 0.f : mn;  // nothing kept so far: every exponential below is 0
    const float corr = exp2f((t.m[i] - base) * kLog2eF);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float p = exp2f((x[j] - base) * kLog2eF);
      sum += p;
      s.p[r * TL::kPs + tx + 16 * j] = kp[j] ? p : -0.f;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    t.l[i] = t.l[i] * corr + sum;
    t.m[i] = mn;
#pragma unroll
    for (int d = 0; d < KC; ++d) t.o[i][d] *= corr;
  }
  __syncwarp();  // a row's 64 weights come from its own half warp
  float2 acc[RPT][KC / 2];  // this tile's share, added once: short sums lose less
#pragma unroll
  for (int i = 0; i < RPT; ++i)
#pragma unroll
    for (int d = 0; d < KC / 2; ++d) acc[i][d] = make_float2(0.f, 0.f);
  auto product = [&](auto selects) {
#pragma unroll 2
    for (int c = 0; c < BN; c += 4) {
      float4 pv[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) pv[i] = *reinterpret_cast<const float4*>(s.p + (ty * RPT + i) * TL::kPs + c);
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
#pragma unroll
        for (int dc = 0; dc < KC / 4; ++dc) {
          const float4 vv = *reinterpret_cast<const float4*>(s.v + (c + cc) * TL::kStride + dc * 64 + tx * 4);
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float p = cc == 0 ? pv[i].x : cc == 1 ? pv[i].y : cc == 2 ? pv[i].z : pv[i].w;
            if (decltype(selects)::value && masked_p(p)) continue;
            acc[i][dc * 2] = sm100::ffma2(make_float2(p, p), make_float2(vv.x, vv.y), acc[i][dc * 2]);
            acc[i][dc * 2 + 1] = sm100::ffma2(make_float2(p, p), make_float2(vv.z, vv.w), acc[i][dc * 2 + 1]);
          }
        }
      }
    }
  };
  if (select)
    product(std::true_type{});
  else
    product(std::false_type{});
#pragma unroll
  for (int i = 0; i < RPT; ++i)
#pragma unroll
    for (int d = 0; d < KC / 2; ++d) {
      t.o[i][2 * d] += acc[i][d].x;
      t.o[i][2 * d + 1] += acc[i][d].y;
    }
}

// Output column of accumulator e of a thread.
__device__ __forceinline__ int out_col(int e, int tx) { return (e / 4) * 64 + tx * 4 + (e & 3); }

// ------------------------------------------------------------ prompt
// The parts of a tile's rows in the CTAs of a cluster: CTA `part` gets the
// joined m, l and o of its share of every thread's rows.
template <int DP>
__device__ __forceinline__ void join_parts(Tile<4, DP>& t, float* smem, int split, int part) {
  constexpr int RPT = 4, kCols = DP / 16, kEach = kCols + 2;
  static_assert(sizeof(float) * RPT * kEach * kThreads <= Tile<4, DP>::bytes(1), "the parts' room");
  cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
  __syncthreads();  // everyone is done with the tiles
  float* own = smem + threadIdx.x;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    own[i * kEach * kThreads] = t.m[i];
    own[(i * kEach + 1) * kThreads] = t.l[i];
#pragma unroll
    for (int e = 0; e < kCols; ++e) own[(i * kEach + 2 + e) * kThreads] = t.o[i][e];
  }
  cl.sync();
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    if (i * split / RPT != part) continue;
    float m = -INFINITY;
    for (int p = 0; p < split; ++p) m = fmaxf(m, cl.map_shared_rank(own, p)[i * kEach * kThreads]);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, o[kCols];
#pragma unroll
    for (int e = 0; e < kCols; ++e) o[e] = 0.f;
    for (int p = 0; p < split; ++p) {
      const float* from = cl.map_shared_rank(own, p) + i * kEach * kThreads;
      const float f = exp2f((from[0] - base) * kLog2eF);
      l = fmaf(from[kThreads], f, l);
#pragma unroll
      for (int e = 0; e < kCols; ++e) o[e] = fmaf(from[(2 + e) * kThreads], f, o[e]);
    }
    t.m[i] = m;
    t.l[i] = l;
#pragma unroll
    for (int e = 0; e < kCols; ++e) t.o[i][e] = o[e];
  }
  cl.sync();  // the others have read this CTA's part
}

// A cluster of `split` CTAs per 64-row tile, (b, h) fastest, the last (under
// causal the longest) tiles first.  CTA p takes the key tiles p, p + split, ..;
// the parts of a row are joined through the cluster's shared memory, in order.
template <typename T, int DP, bool kAsync>
__global__ void __launch_bounds__(kThreads) prompt_simt_kernel(const __grid_constant__ PromptArgs a, bool vec, int split) {
  extern __shared__ __align__(16) float smem[];
  constexpr int RPT = 4, BM = 64;
  Smem<RPT, DP> s(smem);
  const unsigned items = gridDim.x / split, bhs = a.B * a.Hq;
  const unsigned L = blockIdx.x / split;
  const int part = blockIdx.x % split;
  const int b = (L % bhs) / a.Hq, h = (L % bhs) % a.Hq, g = h / a.G;
  const int r0 = (int)(items / bhs - 1 - L / bhs) * BM;
  const SeqView sv = seq_view(a.lens, a.cu, true, b, a.N, a.total);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  T* out = static_cast<T*>(a.out) + sv.q_b * a.os[0] + h * a.os[1] + (long long)sv.q_row * a.os[2];
  float* lse = a.lse + sv.q_b * a.ls[0] + h * a.ls[1] + (long long)sv.q_row * a.ls[2];
  if (r0 < sv.n) {
    const T* q = static_cast<const T*>(a.q) + sv.q_b * a.qs[0] + h * a.qs[1] + (long long)sv.q_row * a.qs[2];
    const T* k = static_cast<const T*>(a.k) + sv.k_b * a.ks[0] + g * a.ks[1] + (long long)sv.k_row * a.ks[2];
    const T* v = static_cast<const T*>(a.v) + sv.k_b * a.vs[0] + g * a.vs[1] + (long long)sv.k_row * a.vs[2];
    const uint8_t* km = a.kmask ? a.kmask + b * a.kmb : nullptr;
    Tile<RPT, DP> t;
    t.reset();
    load_rows<T, RPT, DP>(s.q, BM, [&](int r) { return r0 + r < sv.n ? q + (long long)(r0 + r) * a.qs[2] : nullptr; },
                          a.D, a.qs[3], vec);
    const int end = a.causal ? min(sv.n, r0 + BM) : sv.n;
    // keys past the end and keys the mask drops: zero rows, never products with what they hold
    auto live = [&](int c) { return c < end && (km == nullptr || km[c] != 0); };
    auto load = [&](int c0, const Smem<RPT, DP>& to) {
      auto krow = [&](int j) { return live(c0 + j) ? k + (long long)(c0 + j) * a.ks[2] : nullptr; };
      auto vrow = [&](int j) { return live(c0 + j) ? v + (long long)(c0 + j) * a.vs[2] : nullptr; };
      if constexpr (kAsync) {
        copy_rows<DP>(to.k, BN, krow, a.D, k);
        copy_rows<DP>(to.v, BN, vrow, a.D, v);
      } else {
        load_rows<T, RPT, DP>(to.k, BN, krow, a.D, a.ks[3], vec);
        load_rows<T, RPT, DP>(to.v, BN, vrow, a.D, a.vs[3], vec);
      }
      if (threadIdx.x < BN) to.bias[threadIdx.x] = live(c0 + threadIdx.x) ? 0.f : -INFINITY;
    };
    const int step = BN * split;
    if constexpr (kAsync) {
      load(part * BN, s);
      copy_commit();
    }
    for (int c0 = part * BN, turn = 0; c0 < end; c0 += step, turn ^= 1) {
      const Smem<RPT, DP> now(smem, kAsync ? turn : 0);
      if constexpr (kAsync) {
        if (c0 + step < end) load(c0 + step, Smem<RPT, DP>(smem, turn ^ 1));
        copy_commit();
        copy_wait<1>();
      } else {
        __syncthreads();
        load(c0, now);
      }
      __syncthreads();
      const bool diag = a.causal && c0 + BN - 1 > r0;
      tile_step<RPT, DP>(
          t, now, a.scale, false, diag,
          [&](int r, int j) { return now.bias[j] == 0.f && (!a.causal || c0 + j <= r0 + r); },
          [](int, int, float) {});
      if constexpr (kAsync) __syncthreads();  // the buffer is free
    }
    if (split > 1) join_parts<DP>(t, smem, split, part);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = r0 + ty * RPT + i;
      if (r >= sv.n || i * split / RPT != part) continue;
      const float inv = t.l[i] > 0.f ? 1.f / t.l[i] : (t.l[i] == 0.f ? 0.f : t.l[i]);
#pragma unroll
      for (int e = 0; e < DP / 16; ++e) {
        const int d = out_col(e, tx);
        if (d < a.D) out[r * a.os[2] + d * a.os[3]] = from_f32<T>(t.l[i] == 0.f ? 0.f : t.o[i][e] * inv);
      }
      if (tx == 0) lse[r * a.ls[2]] = t.l[i] == 0.f ? -INFINITY : t.m[i] + logf(t.l[i]);
    }
  }
  if (a.fill && a.cu == nullptr && part == 0) {
    for (int i = threadIdx.x; i < BM; i += kThreads) {
      const int r = r0 + i;
      if (r >= sv.n && r < a.N) lse[r * a.ls[2]] = -INFINITY;
    }
    for (int i = threadIdx.x; i < BM * a.D; i += kThreads) {
      const int r = r0 + i / a.D;
      if (r >= sv.n && r < a.N) out[r * a.os[2] + (i % a.D) * a.os[3]] = from_f32<T>(0.f);
    }
  }
}

// Rows of a packed output that belong to no sequence (before the first
// offset, past the last, or past a sequence's first N rows): out 0, lse -inf.
template <typename T>
__global__ void __launch_bounds__(kThreads) prompt_fill_kernel(PromptArgs a) {
  const long long row = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  if (row >= a.total) return;
  const int lane = threadIdx.x & 31;
  bool inside = false;
  for (int b0 = 0; b0 < a.B && !inside; b0 += 32) {
    const int b = b0 + lane;
    bool in = false;
    if (b < a.B) {
      const SeqView sv = seq_view(nullptr, a.cu, true, b, a.N, a.total);
      in = row >= sv.q_row && row < (long long)sv.q_row + sv.n;
    }
    inside = __any_sync(0xffffffffu, in);
  }
  if (inside) return;
  for (int h = 0; h < a.Hq; ++h) {
    T* out = static_cast<T*>(a.out) + h * a.os[1] + row * a.os[2];
    for (int d = lane; d < a.D; d += 32) out[d * a.os[3]] = from_f32<T>(0.f);
    if (lane == 0) a.lse[h * a.ls[1] + row * a.ls[2]] = -INFINITY;
  }
}

// ------------------------------------------------------------ cache
// The linear list of (sequence, kv head, row tile, key tile), key tile
// fastest, is cut into C equal ranges, one per CTA: every SM gets the same
// number of key tiles however the lengths differ.  A unit (sequence, kv head,
// row tile) inside one range is finished by its CTA; a unit that crosses a
// border leaves one partial (m, l, unnormalised output) per CTA, in slot 0
// when it is the CTA's first unit and slot 1 when a later one, which
// cached_merge_kernel joins in CTA order.
template <typename T, int RPT, int DP, bool kAsync>
__global__ void __launch_bounds__(kThreads) cached_simt_kernel(const __grid_constant__ CachedArgs a, bool vec) {
  extern __shared__ __align__(16) float smem[];
  constexpr int BM = 16 * RPT;
  Smem<RPT, DP> s(smem);
  __shared__ long long sh_first, sh_total;
  __shared__ int sh_b;
  __shared__ longlong2 offs[3][BN];  // element offsets of three tiles' k and v rows (-1: a zero row)
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  cudaTriggerProgrammaticLaunchCompletion();  // the joining kernel may be set up beside this one
  if (threadIdx.x < 32) {
    long long pre, total, first = 0;
    warp_tile_prefix(a, 0, &pre, &total);
    const int b = warp_find_seq(a, split_begin(blockIdx.x, total, a.C), &first);
    if (threadIdx.x == 0) {
      sh_total = total;
      sh_first = first;
      sh_b = b;
    }
  }
  __syncthreads();
  const long long total = sh_total;
  const long long begin = split_begin(blockIdx.x, total, a.C), end = split_begin(blockIdx.x + 1, total, a.C);
  int b = sh_b;
  long long bfirst = sh_first;
  const int per = a.Hkv * a.RT;
  for (long long at = begin; at < end;) {
    int len = cached_len(a, b), nt = (len + BN - 1) / BN;
    while (at >= bfirst + (long long)nt * per) {
      bfirst += (long long)nt * per;
      ++b;
      len = cached_len(a, b);
      nt = (len + BN - 1) / BN;
    }
    const int u = (int)((at - bfirst) / nt), g = u / a.RT, rt = u % a.RT;
    const long long ufirst = bfirst + (long long)u * nt;
    const int k0 = (int)(at - ufirst);
    const int k1 = (int)min((long long)nt, end - ufirst);
    const int pre = len - a.T;  // keys before the drafted tokens
    const T* qb = static_cast<const T*>(a.q) + b * a.qs[0];
    const float* off = a.off ? a.off + b * a.ob + g * a.oh : nullptr;
    const uint8_t* tree = a.tree ? a.tree + b * a.tb : nullptr;
    Tile<RPT, DP> t;
    t.reset();
    __syncthreads();
    load_rows<T, RPT, DP>(
        s.q, BM,
        [&](int i) -> const T* {
          const int r = rt * BM + i;
          return r < a.R ? qb + (long long)(g * a.G + r / a.T) * a.qs[1] + (long long)(r % a.T) * a.qs[2] : nullptr;
        },
        a.D, a.qs[3], vec);
    auto put_offsets = [&](int kt) {
      if (threadIdx.x >= BN || kt >= k1) return;
      const int c = kt * BN + threadIdx.x;
      longlong2 o = make_longlong2(-1, -1);
      if (c < len && !(off != nullptr && off[c] == -INFINITY)) {
        const int in = a.pg.slot(c), page = a.pg.page(b, a.pg.page_index(c));
        if (page >= 0 && page < a.pg.num_pages) {
          o.x = (long long)page * a.ks[0] + (long long)in * a.ks[1] + g * a.ks[2];
          o.y = (long long)page * a.vs[0] + (long long)in * a.vs[1] + g * a.vs[2];
        } else {
          atomicOr(&g_attention_page_error, 1u);
        }
      }
      offs[(kt - k0) % 3][threadIdx.x] = o;
    };
    auto load = [&](int kt, const Smem<RPT, DP>& to) {
      if (kt >= k1) return;
      const T *kp = static_cast<const T*>(a.k), *vp = static_cast<const T*>(a.v);
      const longlong2* of = offs[(kt - k0) % 3];
      auto krow = [&](int j) { return of[j].x >= 0 ? kp + of[j].x : nullptr; };
      auto vrow = [&](int j) { return of[j].y >= 0 ? vp + of[j].y : nullptr; };
      if constexpr (kAsync) {
        copy_rows<DP>(to.k, BN, krow, a.D, kp);
        copy_rows<DP>(to.v, BN, vrow, a.D, vp);
      } else {
        load_rows<T, RPT, DP>(to.k, BN, krow, a.D, a.ks[3], vec);
        load_rows<T, RPT, DP>(to.v, BN, vrow, a.D, a.vs[3], vec);
      }
      if (off != nullptr && threadIdx.x < BN) {
        const int c = kt * BN + threadIdx.x;
        to.bias[threadIdx.x] = c < len ? off[c] : -INFINITY;
      }
    };
    put_offsets(k0);
    if constexpr (kAsync) {
      put_offsets(k0 + 1);
      __syncthreads();
      load(k0, s);
      copy_commit();
    }
    for (int kt = k0; kt < k1; ++kt) {
      const int c0 = kt * BN;
      const Smem<RPT, DP> now(smem, kAsync ? (kt - k0) & 1 : 0);
      if constexpr (kAsync) {
        load(kt + 1, Smem<RPT, DP>(smem, (kt + 1 - k0) & 1));
        copy_commit();
        put_offsets(kt + 2);
        copy_wait<1>();
      } else {
        __syncthreads();  // the tile's offsets are there, the buffer is free
        load(kt, now);
        put_offsets(kt + 1);
      }
      __syncthreads();
      const bool drafts = c0 + BN > pre;  // some key of the tile is a drafted token or past the end
      float* sc = a.scores ? a.scores + ((long long)(b * a.Hkv + g) * a.G) * a.Lmax + c0 : nullptr;
      tile_step<RPT, DP>(
          t, now, a.scale, off != nullptr, drafts,
          [&](int i, int j) {
            const int c = c0 + j, r = rt * BM + i;
            if (c >= len || r >= a.R) return false;
            if (off != nullptr && now.bias[j] == -INFINITY) return false;
            if (c < pre) return true;
            const int tok = r % a.T;
            return tree ? tree[tok * a.tr + (c - pre)] != 0 : c - pre <= tok;
          },
          [&](int i, int j, float x) {
            if (sc != nullptr && rt * BM + i < a.R && c0 + j < len) sc[(long long)(rt * BM + i) * a.Lmax + j] = x;
          });
      if constexpr (kAsync) __syncthreads();  // the buffer is free, and the offsets two tiles ahead are there
    }
    const bool whole = k0 == 0 && k1 == nt;
    const int slot = begin >= ufirst ? 0 : 1;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int rl = ty * RPT + i, r = rt * BM + rl;
      if (whole) {
        if (r >= a.R) continue;
        const int h = g * a.G + r / a.T, tok = r % a.T;
        const float inv = 1.f / t.l[i];
        T* out = static_cast<T*>(a.out) + b * a.os[0] + h * a.os[1] + tok * a.os[2];
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) {
          const int d = out_col(e, tx);
          if (d < a.D) out[d * a.os[3]] = from_f32<T>(t.l[i] == 0.f ? 0.f : t.o[i][e] * inv);
        }
        if (tx == 0) {
          a.lse[b * a.ls[0] + h * a.ls[1] + tok * a.ls[2]] = t.l[i] == 0.f ? -INFINITY : t.m[i] + logf(t.l[i]);
          if (a.stats) a.stats[(long long)(b * a.Hkv + g) * a.R + r] = make_float2(t.m[i], t.l[i] == 0.f ? 0.f : inv);
        }
      } else {
        const long long pr = ((long long)blockIdx.x * 2 + slot) * BM + rl;
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) a.part_o[pr * DP + out_col(e, tx)] = t.o[i][e];
        if (tx == 0) a.part_ml[pr] = make_float2(t.m[i], t.l[i]);
      }
    }
    at = ufirst + k1;
  }
}

// Joins the partials of every split unit, and writes the rows of sequences
// with no keys (out 0, lse -inf).  One warp a row, grid (B * Hkv * RT, BM /
// kMergeRows); partials in CTA order: the same bits on every run.  Lanes read 32
// partials' (m, l) at once and then stream their output rows, kAhead loads in
// flight.  A row is a chain of two memory round trips, so rows go side by side:
// four rows a warp one after another took 7 us more at 13 tokens.  kCols: columns
// a lane holds (4 for D <= 128, else 8).
constexpr int kMergeRows = 8;
template <typename T, int kCols>
__global__ void __launch_bounds__(256) cached_merge_kernel(const __grid_constant__ CachedArgs a) {
  const int unit = blockIdx.x, b = unit / (a.Hkv * a.RT), u = unit % (a.Hkv * a.RT), g = u / a.RT, rt = u % a.RT;
  const int lane = threadIdx.x & 31;
  long long pre, total;
  warp_tile_prefix(a, b, &pre, &total);
  const int nt = (cached_len(a, b) + a.KT - 1) / a.KT;
  const long long t0 = pre + (long long)u * nt, t1 = t0 + nt;
  const int i0 = nt > 0 ? (int)split_owner(t0, total, a.C) : 0, i1 = nt > 0 ? (int)split_owner(t1 - 1, total, a.C) : 0;
  // the slot that holds the unit's share of CTA i (-1: a CTA without tiles)
  auto slot_of = [&](int i) -> long long {
    if (i > i1) return -1;
    const long long s0 = split_begin(i, total, a.C), s1 = split_begin(i + 1, total, a.C);
    return s0 == s1 ? -1 : (long long)i * 2 + (s0 >= t0 ? 0 : 1);
  };
  const long long first = slot_of(i0 + lane);
  // launched while the split kernel runs: what is above overlaps it, and every
  // thread waits here for its results
  cudaGridDependencySynchronize();
  if (nt > 0 && i0 == i1) return;  // finished by its CTA
  const int lanes = a.DP < 32 * kCols ? a.DP / kCols : 32;
  const int rl = blockIdx.y * kMergeRows + threadIdx.x / 32, r = rt * a.BM + rl;
  if (rl >= a.BM || r >= a.R) return;
  const int h = g * a.G + r / a.T, tok = r % a.T;
  T* out = static_cast<T*>(a.out) + b * a.os[0] + h * a.os[1] + tok * a.os[2];
  float* lse = a.lse + b * a.ls[0] + h * a.ls[1] + tok * a.ls[2];
  if (nt == 0) {
    for (int d = lane; d < a.D; d += 32) out[d * a.os[3]] = from_f32<T>(0.f);
    if (lane == 0) *lse = -INFINITY;
    return;
  }
  auto load_ml = [&](long long slot) {
    return slot < 0 ? make_float2(-INFINITY, 0.f) : a.part_ml[slot * a.BM + rl];
  };
  long long slot = first;
  float2 ml = load_ml(slot);
  float m = ml.x;
  for (int base = i0 + 32; base <= i1; base += 32) m = fmaxf(m, load_ml(slot_of(base + lane)).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, acc[kCols];
#pragma unroll
  for (int e = 0; e < kCols; ++e) acc[e] = 0.f;
  for (int base = i0; base <= i1; base += 32) {
    if (base > i0) {
      slot = slot_of(base + lane);
      ml = load_ml(slot);
    }
    // (a partial that kept nothing has l = 0; a NaN maximum gives a NaN factor)
    const float f = ml.y == 0.f ? 0.f : exp2f((ml.x - ref) * kLog2eF);
    float lp = ml.y * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) lp += __shfl_xor_sync(0xffffffffu, lp, o);
    l += lp;
    const int n = min(32, i1 - base + 1);
    constexpr int kAhead = 16 / kCols;
    for (int k0 = 0; k0 < n; k0 += kAhead) {
      float x[kAhead][kCols], fk[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        fk[i] = __shfl_sync(0xffffffffu, f, (k0 + i) & 31);
        const long long pk = __shfl_sync(0xffffffffu, slot, (k0 + i) & 31);
        // (a part whose factor is 0 counts too: its finite values add nothing, its NaN and infinities do)
        const bool in = k0 + i < n && pk >= 0 && lane < lanes;
        const float4* src = reinterpret_cast<const float4*>(a.part_o + (pk * a.BM + rl) * a.DP + lane * kCols);
#pragma unroll
        for (int q = 0; q < kCols / 4; ++q) {
          const float4 y = in ? src[q] : make_float4(0.f, 0.f, 0.f, 0.f);
          x[i][4 * q] = y.x;
          x[i][4 * q + 1] = y.y;
          x[i][4 * q + 2] = y.z;
          x[i][4 * q + 3] = y.w;
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int e = 0; e < kCols; ++e) acc[e] = fmaf(x[i][e], fk[i], acc[e]);
    }
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int e = 0; e < kCols; ++e) {
    const int d = lane * kCols + e;
    if (lane < lanes && d < a.D) out[d * a.os[3]] = from_f32<T>(l == 0.f ? 0.f : acc[e] * inv);
  }
  if (lane == 0) {
    *lse = l == 0.f ? -INFINITY : m + logf(l);
    if (a.stats) a.stats[(long long)(b * a.Hkv + g) * a.R + r] = make_float2(m, l == 0.f ? 0.f : inv);
  }
}

// weights_out[b, g, c] = weights[b, g, c] + sum over the group's heads of
// exp(x - m) / l, c < len.  From the stored scores (G * 4 bytes a key next to
// the 4 D bytes of its k and v rows) rather than from a second pass over k.
// kVec: four keys a thread (aligned rows).
template <int kVec>
__global__ void __launch_bounds__(256) cached_weights_kernel(const __grid_constant__ CachedArgs a) {
  const int b = blockIdx.y / a.Hkv, g = blockIdx.y % a.Hkv;
  const int len = cached_len(a, b);
  const int c = (blockIdx.x * 256 + threadIdx.x) * kVec;
  const float* w = a.w + b * a.wb + g * a.wh + c;
  float* wo = a.wout + b * a.wob + g * a.woh + c;
  float sum[kVec];
  alignas(16) float old[kVec];
#pragma unroll
  for (int e = 0; e < kVec; ++e) sum[e] = old[e] = 0.f;
  if (c < len) {
    if (kVec == 4 && c + 4 <= len) {
      *reinterpret_cast<float4*>(old) = *reinterpret_cast<const float4*>(w);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (c + e < len) old[e] = w[e];
    }
  }
  cudaGridDependencySynchronize();  // the weights were there before; scores and row statistics are now
  if (c >= len) return;
  const float* sc = a.scores + (long long)blockIdx.y * a.G * a.Lmax + c;
  const float2* st = a.stats + (long long)blockIdx.y * a.R;
#pragma unroll 4
  for (int hh = 0; hh < a.G; ++hh) {
    const float2 ml = st[hh];
    const float base = ml.x == -INFINITY ? 0.f : ml.x;
    float x[kVec];
    if constexpr (kVec == 4) {
      // (inside the row: Lmax % 4 == 0)
      const float4 v = *reinterpret_cast<const float4*>(sc + (long long)hh * a.Lmax);
      x[0] = v.x;
      x[1] = v.y;
      x[2] = v.z;
      x[3] = v.w;
    } else {
      x[0] = sc[(long long)hh * a.Lmax];
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum[e] = fmaf(exp2f((x[e] - base) * kLog2eF), ml.y, sum[e]);
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e)
    if (c + e < len) wo[e] = old[e] + sum[e];
}

bool rows_aligned(const void* p, const long long* st, int D, int es) {
  return st[3] == 1 && D % 4 == 0 && (uintptr_t)p % (4 * es) == 0 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
}

template <typename T, int DP, bool kAsync>
int prompt_simt_run(const PromptArgs& a, bool vec, cudaStream_t s) {
  auto kern = prompt_simt_kernel<T, DP, kAsync>;
  constexpr size_t bytes = Tile<4, DP>::bytes(kAsync ? 2 : 1);
  static_assert(bytes <= 227 * 1024, "one CTA's shared memory");
  if (allow_smem(kern, bytes) != KVBM_OK) return KVBM_ERR_CUDA;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) return KVBM_ERR_CUDA;
  const long long tiles = (a.N + 63) / 64, items = tiles * a.B * a.Hq;
  if (items > 0x7fffffffLL) return KVBM_ERR_SHAPE;
  // CTAs an item: while the items leave CTA slots empty, or barely fill them, the
  // longest item decides (2048 causal tokens, 8 heads of 64, 256 items: 1 CTA 242
  // us, 2 164, 4 178; 512 tokens, 64 items: 53, 31, 23); beyond, splitting costs
  // the joining (1024 items of D = 128: 1217, 1304, 1618 us).
  const long long slots = (long long)attention_device_sms(dev) * (Tile<4, DP>::bytes(kAsync ? 2 : 1) <= 113 * 1024 ? 2 : 1);
  int split = 1;
  while (split < 4 && items * split <= slots && 2 * split <= tiles) split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, a, vec, split) == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
}

template <typename T, int DP>
int prompt_simt(const PromptArgs& a, cudaStream_t s) {
  const bool vec = rows_aligned(a.q, a.qs, a.D, sizeof(T)) && rows_aligned(a.k, a.ks, a.D, sizeof(T)) &&
                   rows_aligned(a.v, a.vs, a.D, sizeof(T));
  if constexpr (sizeof(T) == 4 && DP <= 128)
    if (vec) return prompt_simt_run<T, DP, true>(a, vec, s);
  return prompt_simt_run<T, DP, false>(a, vec, s);
}

template <typename T>
int prompt_simt_d(const PromptArgs& a, cudaStream_t s) {
  if (a.D <= 64) return prompt_simt<T, 64>(a, s);
  if (a.D <= 128) return prompt_simt<T, 128>(a, s);
  return prompt_simt<T, 256>(a, s);
}

template <typename T, int RPT, int DP, bool kAsync>
int cached_simt_run(const CachedArgs& a, bool vec, cudaStream_t s) {
  auto kern = cached_simt_kernel<T, RPT, DP, kAsync>;
  constexpr size_t bytes = Tile<RPT, DP>::bytes(kAsync ? 2 : 1);
  static_assert(bytes <= 227 * 1024, "one CTA's shared memory");
  if (allow_smem(kern, bytes) != KVBM_OK) return KVBM_ERR_CUDA;
  kern<<<(unsigned)a.C, kThreads, bytes, s>>>(a, vec);
  return cudaGetLastError() == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
}

template <typename T, int RPT, int DP>
int cached_simt(const CachedArgs& a, cudaStream_t s) {
  const bool vec = rows_aligned(a.q, a.qs, a.D, sizeof(T)) && rows_aligned(a.k, a.ks, a.D, sizeof(T)) &&
                   rows_aligned(a.v, a.vs, a.D, sizeof(T));
  if constexpr (sizeof(T) == 4 && DP <= 128)
    if (vec) return cached_simt_run<T, RPT, DP, true>(a, vec, s);
  return cached_simt_run<T, RPT, DP, false>(a, vec, s);
}

template <typename T>
int cached_simt_d(const CachedArgs& a, cudaStream_t s) {
  if (a.BM == 16) {
    if (a.DP == 64) return cached_simt<T, 1, 64>(a, s);
    if (a.DP == 128) return cached_simt<T, 1, 128>(a, s);
    return cached_simt<T, 1, 256>(a, s);
  }
  if (a.DP == 64) return cached_simt<T, 4, 64>(a, s);
  if (a.DP == 128) return cached_simt<T, 4, 128>(a, s);
  return cached_simt<T, 4, 256>(a, s);
}

template <typename T>
int merge(const CachedArgs& a, cudaStream_t s) {
  const int rows = a.R < a.BM ? a.R : a.BM;
  const dim3 grid((unsigned)(a.B * a.Hkv * a.RT), (unsigned)((rows + kMergeRows - 1) / kMergeRows));
  return a.DP <= 128 ? launch_dependent(cached_merge_kernel<T, 4>, grid, 256, s, a)
                     : launch_dependent(cached_merge_kernel<T, 8>, grid, 256, s, a);
}

}  // namespace

int launch_prompt_simt(const PromptArgs& a, int dtype, cudaStream_t s) {
  if (dtype == KVBM_F32) return prompt_simt_d<float>(a, s);
  if (dtype == KVBM_BF16) return prompt_simt_d<__nv_bfloat16>(a, s);
  return prompt_simt_d<__half>(a, s);
}

int launch_prompt_fill(const PromptArgs& a, int dtype, cudaStream_t s) {
  if (a.cu == nullptr || a.total == 0) return KVBM_OK;
  const unsigned grid = (unsigned)((a.total + kThreads / 32 - 1) / (kThreads / 32));
  if (dtype == KVBM_F32)
    prompt_fill_kernel<float><<<grid, kThreads, 0, s>>>(a);
  else if (dtype == KVBM_BF16)
    prompt_fill_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
  else
    prompt_fill_kernel<__half><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
}

int launch_cached_simt(const CachedArgs& a, int dtype, cudaStream_t s) {
  if (dtype == KVBM_F32) return cached_simt_d<float>(a, s);
  if (dtype == KVBM_BF16) return cached_simt_d<__nv_bfloat16>(a, s);
  return cached_simt_d<__half>(a, s);
}

int launch_cached_merge(const CachedArgs& a, int dtype, cudaStream_t s) {
  if (dtype == KVBM_F32) return merge<float>(a, s);
  if (dtype == KVBM_BF16) return merge<__nv_bfloat16>(a, s);
  return merge<__half>(a, s);
}

int launch_cached_weights(const CachedArgs& a, cudaStream_t s) {
  const bool vec = a.Lmax % 4 == 0 && (uintptr_t)a.w % 16 == 0 && a.wb % 4 == 0 && a.wh % 4 == 0;
  const int per = vec ? 1024 : 256;
  const dim3 grid((unsigned)((a.Lmax + per - 1) / per), (unsigned)(a.B * a.Hkv));
  return vec ? launch_dependent(cached_weights_kernel<4>, grid, 256, s, a)
             : launch_dependent(cached_weights_kernel<1>, grid, 256, s, a);
}

// Looked up once per device (every device has a copy of the word).
unsigned int* attention_page_error_word() {
  constexpr int kMaxDevices = 64;
  static std::atomic<unsigned int*> words[kMaxDevices] = {};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    return nullptr;
  }
  unsigned int* w = words[dev].load(std::memory_order_acquire);
  if (w != nullptr) return w;
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_attention_page_error) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  w = static_cast<unsigned int*>(p);
  words[dev].store(w, std::memory_order_release);
  return w;
}

}  // namespace kvbm
