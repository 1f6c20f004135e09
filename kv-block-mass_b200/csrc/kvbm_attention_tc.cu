// Prompt attention on the tensor cores (tcgen05), bf16 / fp16, D <= 128.
//
//   out_i = sum_c exp(x_ic - lse_i) v_c,   x_ic = scale q_i . k_c
//
// One CTA owns two tiles of 128 query rows (A and B) of one head and streams
// the key tiles of 128 keys once:
//   warps 0-7, 8-15 softmax of tile A, of tile B: two threads a row
//                   (kvbm_attention_tile.cuh); scores from TMEM, weights back
//                   to TMEM (16 bit, over the scores' columns)
//   warp 16         MMA issuer: S = Q K^T (operands in shared memory), then
//                   O += P V with P read from TMEM and V MN-major in shared
//                   memory as TMA left it
//   warp 17         TMA producer: K and V rings of two tiles each
//   warps 18-19     scrub: zero the V rows nobody keeps (masked keys, rows
//                   past the sequence) and non-finite elements of the
//                   diagonal tiles, since 0 * NaN is not 0
// Why two row tiles: while one tile's softmax runs, the tensor pipe does the
// other tile's P V and next S; per pair and key tile the four MMAs need 2048
// cycles at D = 128 and the 32768 exponentials 2048 MUFU cycles (less the
// share the FMA pipe takes), so both units are close to full.  TMEM holds S/P
// and O of both tiles: 2 * 128 + 2 * 128 columns.
//
// The running maximum is raised (and O multiplied in TMEM by its softmax
// thread) only when a row's scores grow by more than 2^8 over it: weights stay
// below 2^8, which both 16-bit types hold at full precision, sums are fp32,
// and after the first key tiles almost no tile pays for it.  S of the next
// tile is issued after P V of this one, and MMAs of a CTA complete in order,
// so a full S also means that O is up to date.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kvbm_attention.cuh"
#include "kvbm_attention_tile.cuh"

namespace kvbm {

namespace {
using namespace sm100;

constexpr int TILE = 128;
constexpr int ROWS = 2 * TILE;  // query rows of a CTA
constexpr int kThreads = 640;
constexpr int kMmaWarp = 16, kTmaWarp = 17;
constexpr int kScrubThreads = 64;
constexpr int kStages = 2;  // K ring, V ring
// Registers a thread after the split: 4 softmax warpgroups + 1 of the rest;
// the launch holds 640 x 96.
constexpr int kRegsSoftmax = 104, kRegsRest = 64;
static_assert(4 * kRegsSoftmax + kRegsRest <= 5 * 96, "the split draws on the launch's registers");

template <int DP>
struct Cfg {
  static constexpr int kBlocks = DP / 64;               // 128-byte blocks of a row
  static constexpr int kBlockBytes = TILE * 128;        // one block of a tile
  static constexpr int kTileBytes = kBlocks * kBlockBytes;
  static constexpr int kBars = 2 + 6 * kStages + 4;
  static constexpr size_t kSmem = 1024 + (size_t)kTileBytes * (2 + 2 * kStages) + 8 * kBars + 64 + 2 * 4 * TILE * 4;
};

// The work of a CTA: 256-row tile qt of sequence b, head h; or, past the last
// tile, its share of the rows that belong to no sequence.
struct Item {
  int b, h, qt;       // qt < 0: none
  long long spare;    // index among the CTAs without a tile
  long long spares;   // how many there are
};

// Tiles in order of falling qt (under causal the longest first), heads
// fastest: the heads of a group read the same keys at the same time.  With
// lengths on the device the CTA finds its tile by counting: cnt(q) = tiles of
// level >= q.  One warp.
__device__ __forceinline__ int tiles_of(const PromptArgs& a, int b) {
  return (seq_view(a.lens, a.cu, true, b, a.N, a.total).n + ROWS - 1) / ROWS;
}

__device__ __forceinline__ long long count_from(const PromptArgs& a, int q) {
  long long n = 0;
  for (int b = threadIdx.x & 31; b < a.B; b += 32) n += max(0, tiles_of(a, b) - q);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

__device__ __forceinline__ Item find_item(const PromptArgs& a) {
  Item it;
  const int nt = (a.N + ROWS - 1) / ROWS;
  const long long L = blockIdx.x, i = L / a.Hq;
  it.h = (int)(L % a.Hq);
  it.spare = 0;
  it.spares = 0;
  if (a.lens == nullptr && a.cu == nullptr) {
    it.qt = nt - 1 - (int)(i / a.B);
    it.b = (int)(i % a.B);
    return it;
  }
  const long long total = count_from(a, 0);
  if (i >= total) {
    it.qt = -1;
    it.b = 0;
    it.spare = L - total * a.Hq;
    it.spares = (long long)gridDim.x - total * a.Hq;
    return it;
  }
  int lo = 0, hi = nt;  // cnt(lo) > i >= cnt(hi)
  long long chi = 0;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    const long long c = count_from(a, mid);
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
    const bool in = b < a.B && tiles_of(a, b) > lo;
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

// Rows of no sequence: out 0, lse -inf.  `who` of `of` CTAs.
__device__ void fill_rows(const PromptArgs& a, long long who, long long of) {
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
    for (long long e = who * kThreads + threadIdx.x; e < n * vecs; e += of * kThreads) {
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

template <int DP, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, PromptArgs a, float C) {
  using CF = Cfg<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_tile = smem;                           // [2]
  uint8_t* k_ring = q_tile + 2 * CF::kTileBytes;    // [kStages]
  uint8_t* v_ring = k_ring + kStages * CF::kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_ring + kStages * CF::kTileBytes);
  uint64_t *q_full = bars, *k_full = bars + 2, *k_empty = k_full + kStages, *v_full = k_empty + kStages;
  uint64_t *v_empty = v_full + kStages, *v_raw = v_empty + kStages, *v_ready = v_raw + kStages, *s_full = v_ready + kStages, *p_ready = s_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(p_ready + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* bad_flag = abort_flag + 1;
  int* item_s = reinterpret_cast<int*>(tmem_slot + 3);  // b, h, qt
  long long* spare_s = reinterpret_cast<long long*>(p_ready + 2) + 4;
  float* max_s = reinterpret_cast<float*>(spare_s + 4);  // [2 turns][2 tiles][2 halves][TILE]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    const Item it = find_item(a);
    if (lane == 0) {
      item_s[0] = it.b;
      item_s[1] = it.h;
      item_s[2] = it.qt;
      spare_s[0] = it.spare;
      spare_s[1] = it.spares;
      *abort_flag = 0;
      *bad_flag = 0;
      for (int i = 0; i < 2; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&s_full[i], 1);
        mbar_init(&p_ready[i], 2 * TILE);
      }
      for (int s = 0; s < kStages; ++s) {
        mbar_init(&k_full[s], 1);
        mbar_init(&k_empty[s], 1);
        mbar_init(&v_full[s], 1);
        mbar_init(&v_empty[s], 1);
        mbar_init(&v_raw[s], 1);
        mbar_init(&v_ready[s], kScrubThreads);
      }
      fence_mbar_init();
    }
  }
  __syncthreads();
  if (item_s[2] < 0) {  // no tile for this CTA
    if (a.fill) fill_rows(a, spare_s[0], spare_s[1]);
    return;
  }
  const int b = item_s[0], h = item_s[1], qt = item_s[2], g = h / a.G;
  const SeqView sv = seq_view(a.lens, a.cu, true, b, a.N, a.total);
  const int n = sv.n, r0 = qt * ROWS;
  const int ntiles = (n + TILE - 1) / TILE;
  const uint8_t* km = a.kmask != nullptr ? a.kmask + b * a.kmb : nullptr;
  // key tiles of the two row tiles (B may lie past the sequence)
  const int nA = a.causal ? min(ntiles, 2 * qt + 1) : ntiles;
  const int nB = r0 + TILE < n ? (a.causal ? min(ntiles, 2 * qt + 2) : ntiles) : 0;
  const int nk = max(nA, nB);
  // V tiles from js on arrive at v_raw and go through the scrub warps to
  // v_ready; those before arrive at v_full.  Each barrier counts its own tiles.
  const int js = km != nullptr ? 0 : a.causal ? 2 * qt : (n % TILE != 0 ? n / TILE : ntiles);

  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // columns: S/P of tile t at t * 128, O of tile t at 256 + t * 128

  if (warp >= kMmaWarp) {
    reg_dec<kRegsRest>();
    if (warp == kTmaWarp) {
      if (lane == 0) {
        prefetch_tmap(&tq);
        prefetch_tmap(&tk);
        prefetch_tmap(&tv);
        auto load = [&](uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int row, int head, int batch) {
          mbar_arrive_expect_tx(bar, CF::kTileBytes);
#pragma unroll
          for (int kb = 0; kb < CF::kBlocks; ++kb)
            tma_load_4d(dst + kb * CF::kBlockBytes, m, bar, kb * 64, row, head, batch);
        };
        load(q_tile, &tq, &q_full[0], sv.q_row + r0, h, sv.q_b);
        int ki = 0, vi = 0;  // tiles issued
        for (int j = 0; j < nk; ++j) {
          const int s = j % kStages, ph = (j / kStages - 1) & 1;
          if (j >= kStages && !mbar_wait(&k_empty[s], ph, abort_flag)) break;
          load(k_ring + s * CF::kTileBytes, &tk, &k_full[s], sv.k_row + j * TILE, g, sv.k_b);
          ki = j + 1;
          if (j == 0 && nB > 0) load(q_tile + CF::kTileBytes, &tq, &q_full[1], sv.q_row + r0 + TILE, h, sv.q_b);
          if (j >= kStages && !mbar_wait(&v_empty[s], ph, abort_flag)) break;
          load(v_ring + s * CF::kTileBytes, &tv, j < js ? &v_full[s] : &v_raw[s], sv.k_row + j * TILE, g, sv.k_b);
          vi = j + 1;
        }
        // do not leave while copies are in flight
        mbar_wait(&q_full[0], 0, abort_flag);
        if (nB > 0) mbar_wait(&q_full[1], 0, abort_flag);
        for (int j = max(0, ki - kStages); j < ki; ++j) mbar_wait(&k_full[j % kStages], (j / kStages) & 1, abort_flag);
        for (int j = max(0, vi - kStages); j < vi; ++j) {
          if (j < js)
            mbar_wait(&v_full[j % kStages], (j / kStages) & 1, abort_flag);
          else
            mbar_wait(&v_raw[j % kStages], ((j - js) / kStages) & 1, abort_flag);
        }
      }
    } else if (warp == kMmaWarp) {
      if (lane == 0) {
        const uint32_t idesc_s = idesc_mma(TILE, TILE, kBf16 ? 1u : 0u);
        const uint32_t idesc_o = idesc_mma(TILE, DP, kBf16 ? 1u : 0u) | kTransposeB;
        const uint32_t qs = smem_u32(q_tile), ks = smem_u32(k_ring), vs = smem_u32(v_ring);
        auto issue_s = [&](int t, int j) {
          issue_scores<DP>(tmem + t * TILE, qs + t * CF::kTileBytes, ks + (j % kStages) * CF::kTileBytes, idesc_s);
        };
        auto issue_o = [&](int t, int j) {
          issue_output<DP>(tmem + 256 + t * TILE, tmem + t * TILE, vs + (j % kStages) * CF::kTileBytes, idesc_o, j > 0);
        };
        const int cnt[2] = {nA, nB};
        bool ok = mbar_wait(&k_full[0], 0, abort_flag);
        int pend[2] = {0, 0};  // commits made on s_full[t]
        for (int t = 0; ok && t < 2; ++t) {
          if (cnt[t] == 0) continue;
          ok = mbar_wait(&q_full[t], 0, abort_flag);
          if (!ok) break;
          tc_fence_after();
          issue_s(t, 0);
          mma_commit(&s_full[t]);
          ++pend[t];
        }
        if (ok) mma_commit(&k_empty[0]);
        for (int j = 0; ok && j < nk; ++j) {
          const int s = j % kStages;
          ok = j < js ? mbar_wait(&v_full[s], (j / kStages) & 1, abort_flag)
                      : mbar_wait(&v_ready[s], ((j - js) / kStages) & 1, abort_flag);
          if (ok && j + 1 < nk) ok = mbar_wait(&k_full[(j + 1) % kStages], ((j + 1) / kStages) & 1, abort_flag);
          for (int t = 0; ok && t < 2; ++t) {
            if (j >= cnt[t]) continue;
            ok = mbar_wait(&p_ready[t], j & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            issue_o(t, j);
            if (j + 1 < cnt[t]) issue_s(t, j + 1);
            mma_commit(&s_full[t]);  // the next S, or the finished O
            ++pend[t];
          }
          if (!ok) break;
          mma_commit(&v_empty[s]);
          if (j + 1 < nk) mma_commit(&k_empty[(j + 1) % kStages]);
        }
        // TMEM and shared memory stay until every MMA has finished
        for (int t = 0; t < 2; ++t)
          if (pend[t] > 0) mbar_wait(&s_full[t], (pend[t] - 1) & 1, abort_flag);
      }
    } else {
      const int st = threadIdx.x - (kTmaWarp + 1) * 32;
      for (int j = js; j < nk; ++j) {
        const int s = j % kStages;
        if (!mbar_wait(&v_raw[s], ((j - js) / kStages) & 1, abort_flag)) break;
        uint8_t* tile = v_ring + s * CF::kTileBytes;
        // rows that nobody keeps: zeros (a row is whole 128-byte pieces, however swizzled inside)
        for (int row = st; row < TILE; row += kScrubThreads) {
          const int c = j * TILE + row;
          if (c < n && (km == nullptr || km[c] != 0)) continue;
#pragma unroll
          for (int i = 0; i < CF::kBlocks * 8; ++i)
            *reinterpret_cast<uint4*>(tile + (i >> 3) * CF::kBlockBytes + row * 128 + (i & 7) * 16) =
                make_uint4(0u, 0u, 0u, 0u);
        }
        // diagonal tiles: rows keep different keys
        if (a.causal && j >= 2 * qt) {
          for (int i = st; i < CF::kBlocks * TILE * 8; i += kScrubThreads) {
            if (j * TILE + ((i >> 3) & (TILE - 1)) < n && drop_nonfinite<kBf16>(reinterpret_cast<uint4*>(tile + i * 16)))
              *bad_flag = 1;
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(&v_ready[s]);
      }
    }
  } else {
    reg_inc<kRegsSoftmax>();
    const int t = warp >> 3, half = (warp >> 2) & 1, sub = warp & 3;
    const int rl = sub * 32 + lane;
    const int row = r0 + t * TILE + rl;
    // this thread's scores, its weights' columns, its output columns
    constexpr int kOut = DP / 2;
    const uint32_t lanes = tmem + ((uint32_t)(sub * 32) << 16) + t * TILE;
    const uint32_t ts = lanes + half * kAttCols, tp = lanes + half * (kAttCols / 2), to = lanes + 256 + half * kOut;
    const int cnt = t == 0 ? nA : nB;
    const int rt0 = r0 + t * TILE;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < cnt; ++j) {
      const int c0 = j * TILE + half * kAttCols;
      bool kk[2];
      if (km != nullptr) {  // before the wait: the loads overlap it
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int c = c0 + w * 32 + lane;
          kk[w] = c < n && km[c] != 0;
        }
      }
      ok = mbar_wait(&s_full[t], j & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      float v[kAttCols];
      tmem_ld32(ts, *reinterpret_cast<float(*)[32]>(&v[0]));
      tmem_ld32(ts + 32, *reinterpret_cast<float(*)[32]>(&v[32]));
      tmem_ld_wait();
      if (km != nullptr) {
        uint32_t bits[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) bits[w] = __ballot_sync(0xffffffffu, kk[w]);
#pragma unroll
        for (int c = 0; c < kAttCols; ++c) v[c] = ((bits[c >> 5] >> (c & 31)) & 1u) ? v[c] : -INFINITY;
      }
      if (c0 + kAttCols > n || (a.causal && c0 + kAttCols - 1 > rt0)) {
        const int lim = min(a.causal ? row - c0 : kAttCols - 1, n - 1 - c0);
#pragma unroll
        for (int c = 0; c < kAttCols; ++c) v[c] = c <= lim ? v[c] : -INFINITY;
      }
      float mt = row_max_nan(v);
      // the row's other half (past the barrier, its scores are in registers too: the weights may overwrite them)
      float* mx = max_s + ((j & 1) * 2 + t) * 2 * TILE;
      mx[half * TILE + rl] = mt;
      if (bar_any<2 * TILE>(1 + t, !ok)) {
        ok = false;
        break;
      }
      mt = fmax_nan(mt, mx[(half ^ 1) * TILE + rl]) * C;
      const bool grow = !(mt <= m + kAttGrow);  // (true from -inf to anything finite, and for NaN)
      if (__any_sync(0xffffffffu, grow)) {
        const float mn = grow ? mt : m;
        const float f = m == mn ? 1.f : ex2(m - mn);
        l *= f;
        m = mn;
        if (j > 0) scale_output<kOut>(to, f);
      }
      l += put_weights<kBf16, false>(v, C, m == -INFINITY ? 0.f : -m, tp);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_ready[t]);
    }
    if (cnt > 0) {
      ok = ok && mbar_wait(&s_full[t], cnt & 1, abort_flag);  // O is complete
      float* ls = max_s + t * 2 * TILE;  // (the turns' slots are free: everyone has read its last maximum)
      bar_any<2 * TILE>(1 + t, !ok);
      ls[half * TILE + rl] = l;
      ok = !bar_any<2 * TILE>(1 + t, !ok);
      l += ls[(half ^ 1) * TILE + rl];
    }
    if (ok && cnt > 0) {
      tc_fence_after();
      // what the scrub warps found (their last arrivals are complete: the MMAs waited for them)
      for (int j = max(js, cnt - kStages); j < cnt; ++j)
        mbar_wait(&v_ready[j % kStages], ((j - js) / kStages) & 1, abort_flag);
      const bool bad = *bad_flag != 0;
      const bool none = l == 0.f;
      const float inv = none ? 0.f : 1.f / l;
      uint16_t* out = static_cast<uint16_t*>(a.out) + sv.q_b * a.os[0] + h * a.os[1] +
                      ((long long)sv.q_row + row) * a.os[2];
      const uint16_t* vg = static_cast<const uint16_t*>(a.v) + sv.k_b * a.vs[0] + g * a.vs[1] +
                           (long long)sv.k_row * a.vs[2];
#pragma unroll
      for (int w = 0; w < kOut / 32; ++w) {
        const int d0 = half * kOut + 32 * w;
        float o[32];
        tmem_ld32(to + 32 * w, o);
        tmem_ld_wait();
        if (row < n) {
          if (bad) {
            // the diagonal tiles' non-finite elements, which the MMAs took as zeros
#pragma unroll 1
            for (int c = 2 * qt * TILE; c <= row; ++c) {
              if (km != nullptr && km[c] == 0) continue;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                if (d0 + e >= a.D) continue;
                const uint16_t x = vg[(long long)c * a.vs[2] + d0 + e];
                if (!finite16<kBf16>(x)) {
                  float xf;
                  if constexpr (kBf16)
                    xf = __uint_as_float((uint32_t)x << 16);
                  else
                    xf = __half2float(__ushort_as_half(x));
                  o[e] += xf;
                }
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (d0 + e >= a.D) continue;  // D % 8 == 0
            uint4 r;
            r.x = none ? 0u : pack16<kBf16>(o[e] * inv, o[e + 1] * inv);
            r.y = none ? 0u : pack16<kBf16>(o[e + 2] * inv, o[e + 3] * inv);
            r.z = none ? 0u : pack16<kBf16>(o[e + 4] * inv, o[e + 5] * inv);
            r.w = none ? 0u : pack16<kBf16>(o[e + 6] * inv, o[e + 7] * inv);
            *reinterpret_cast<uint4*>(out + d0 + e) = r;
          }
        }
        __syncwarp();  // the next load is the whole warp's
      }
      if (row < n && half == 0)
        a.lse[sv.q_b * a.ls[0] + h * a.ls[1] + ((long long)sv.q_row + row) * a.ls[2]] =
            none ? -INFINITY : (m + lg2(l)) * kLn2F;
    }
    tc_fence_before();
  }

  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

bool aligned16(const void* p, const long long* st, const int* dims) {
  if ((uintptr_t)p % 16 != 0 || st[3] != 1) return false;
  for (int i = 0; i < 3; ++i) {
    if (st[i] % 8 != 0) return false;
    if (dims[i] > 1 && st[i] == 0) return false;  // an expanded dimension has no tensor map
  }
  return true;
}

template <int DP, bool kBf16>
int launch(const PromptArgs& a, cudaStream_t s) {
  CUtensorMap tq, tk, tv;
  const bool packed = a.cu != nullptr;
  const int B = packed ? 1 : a.B, N = packed ? (int)a.total : a.N;
  const int64_t qs[4] = {a.qs[0], a.qs[1], a.qs[2], 1}, ks[4] = {a.ks[0], a.ks[1], a.ks[2], 1};
  const int64_t vs[4] = {a.vs[0], a.vs[1], a.vs[2], 1};
  if (!make_attention_map(&tq, a.q, kBf16, B, a.Hq, N, a.D, qs, TILE) ||
      !make_attention_map(&tk, a.k, kBf16, B, a.Hkv, N, a.D, ks, TILE) ||
      !make_attention_map(&tv, a.v, kBf16, B, a.Hkv, N, a.D, vs, TILE))
    return KVBM_ERR_CUDA;
  auto kern = prompt_tc_kernel<DP, kBf16>;
  constexpr size_t smem = Cfg<DP>::kSmem;
  if (allow_smem(kern, smem) != KVBM_OK) return KVBM_ERR_CUDA;
  long long tiles = (long long)a.B * ((a.N + ROWS - 1) / ROWS);
  // packed rows make at most ceil(T / 256) + B tiles; one more CTA row for the rows of no sequence
  if (packed) tiles = std::min(tiles, (a.total + ROWS - 1) / ROWS + a.B) + 1;
  else if (a.lens != nullptr) tiles += 1;
  const long long grid = tiles * a.Hq;
  if (grid > 0x7fffffffLL) return KVBM_ERR_SHAPE;
  kern<<<(unsigned)grid, kThreads, smem, s>>>(tq, tk, tv, a, a.scale * kLog2eF);
  return cudaGetLastError() == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
}

}  // namespace

bool prompt_tc_supported(const PromptArgs& a, int dtype) {
  if (dtype != KVBM_BF16 && dtype != KVBM_F16) return false;
  if (a.D > 128 || a.D % 8 != 0 || !(a.scale > 0.f) || !tc_path_enabled()) return false;
  const bool packed = a.cu != nullptr;
  const int B = packed ? 1 : a.B, N = packed ? (int)a.total : a.N;
  const int qd[3] = {B, a.Hq, N}, kd[3] = {B, a.Hkv, N};
  return aligned16(a.q, a.qs, qd) && aligned16(a.k, a.ks, kd) && aligned16(a.v, a.vs, kd) &&
         aligned16(a.out, a.os, qd);
}

int launch_prompt_tc(const PromptArgs& a, int dtype, cudaStream_t s) {
  const bool bf16 = dtype == KVBM_BF16;
  if (a.D <= 64) return bf16 ? launch<64, true>(a, s) : launch<64, false>(a, s);
  return bf16 ? launch<128, true>(a, s) : launch<128, false>(a, s);
}

int read_and_clear_attention_error(cudaStream_t s, int* err) {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbolAsync(&v, g_kvbm_device_error, sizeof(v), 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
      cudaStreamSynchronize(s) != cudaSuccess)
    return KVBM_ERR_CUDA;
  *err = v != 0;
  if (v != 0) {
    const unsigned int zero = 0;
    if (cudaMemcpyToSymbolAsync(g_kvbm_device_error, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s) !=
            cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess)
      return KVBM_ERR_CUDA;
  }
  return KVBM_OK;
}

}  // namespace kvbm
