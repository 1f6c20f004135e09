// Prompt attention on the tensor cores (tcgen05), bf16 / fp16, D <= 128.
//
//   out_i = sum_c exp(x_ic - lse_i) v_c,   x_ic = scale q_i . k_c
//
// One CTA an SM takes work items of two tiles of 128 query rows (A and B) of
// one head, and streams the key tiles of 128 keys of each once:
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
// cycles at D = 128 and the 32768 exponentials 2048 MUFU cycles.  TMEM holds
// S/P and O of both tiles: 2 * 128 + 2 * 128 columns.
//
// Measured (bf16, D = 128, 32 q heads on 8, causal): one prompt of 16384 tokens
// 1.90 ms, 1.16 PFLOP/s, 70 % of cuBLAS' rate for the same work, and 2.21 ms
// called without pause (power); packed prompts of 1 to 4044 tokens, 0.22
// TFLOP, 0.28 ms.  Bound by the chain score - maximum - weights of a tile: about
// 3500 cycles, of which the other tile's tensor work fills 2048.  Of the packed
// call that chain is 187 us (102 steps of two tiles in the longest CTA); the rest
// lies between a CTA's 7 or 8 items, some 20000 cycles each.  Without any
// softmax the long prompt's loop took 1.62 ms.  A pair of CTAs on one tile of 256 rows
// (cta_group::2) took 2.66 ms: each step waits on the other CTA's softmax too.
//
// The CTAs are persistent (one per SM, items from the longest in a snake over
// the CTAs): the next item's queries, keys and first scores are under way while
// the last one's output is scaled and stored.  (A CTA per item: packed prompts
// 314 us where this took 283.)
//
// The running maximum is raised (and O multiplied in TMEM by its softmax
// thread) only when a row's scores grow by more than 2^8 over it: weights stay
// below 2^8 (fp16, whose small weights need the range: 2^15, see kHead), sums are
// fp32, and after the first key tiles almost no tile pays for it.  S of the next
// tile is issued after P V of this one, and MMAs of a CTA complete in order,
// so a full S also means that O is up to date.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kvbm_attention.cuh"
#include "kvbm_attention_items.cuh"
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
  static constexpr int kBars = 3 + 6 * kStages + 8 + 4 + 1;
  static constexpr size_t kSmem = 1024 + (size_t)kTileBytes * (2 + 2 * kStages) + 8 * kBars + 128 + 12 * TILE * 4;
};

// What the roles need of an item.
struct Work {
  int b, h, qt, g, n, r0, nA, nB, nk, js;
  int row, batch;  // where the sequence's rows start, and its batch coordinate
  const uint8_t* km;
};

__device__ __forceinline__ Work work_of(const PromptArgs& a, int b, int h, int qt, int n, int row) {
  Work w;
  w.b = b;
  w.h = h;
  w.qt = qt;
  w.g = h / a.G;
  w.n = n;
  w.row = row;
  w.batch = a.cu != nullptr ? 0 : b;
  w.r0 = qt * ROWS;
  w.km = a.kmask != nullptr ? a.kmask + b * a.kmb : nullptr;
  // key tiles of the two row tiles (B may lie past the sequence)
  const int ntiles = (w.n + TILE - 1) / TILE;
  w.nA = a.causal ? min(ntiles, 2 * qt + 1) : ntiles;
  w.nB = w.r0 + TILE < w.n ? (a.causal ? min(ntiles, 2 * qt + 2) : ntiles) : 0;
  w.nk = max(w.nA, w.nB);
  // V tiles from js on arrive at v_raw and go through the scrub warps to
  // v_ready; those before arrive at v_full.
  w.js = w.km != nullptr ? 0 : a.causal ? 2 * qt : (w.n % TILE != 0 ? w.n / TILE : ntiles);
  return w;
}

template <int DP, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const __grid_constant__ PromptArgs a, float C) {
  using CF = Cfg<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_tile = smem;                           // [2]
  uint8_t* k_ring = q_tile + 2 * CF::kTileBytes;    // [kStages]
  uint8_t* v_ring = k_ring + kStages * CF::kTileBytes;
  // barriers (each waiter keeps the parities it expects next: an item need not use all)
  uint64_t* q_full = reinterpret_cast<uint64_t*>(v_ring + kStages * CF::kTileBytes);  // [2]
  uint64_t *q_empty = q_full + 2, *k_full = q_empty + 1, *k_empty = k_full + kStages, *v_full = k_empty + kStages;
  uint64_t *v_empty = v_full + kStages, *v_raw = v_empty + kStages, *v_ready = v_raw + kStages;
  uint64_t *s_full = v_ready + kStages, *p_ready = s_full + 2, *o_full = p_ready + 2, *o_free = o_full + 2;  // [2] each
  uint64_t *item_full = o_free + 2, *item_empty = item_full + 2;                                             // [2] each
  uint64_t* drained = item_empty + 2;
  volatile int* item_s = reinterpret_cast<volatile int*>(drained + 1);  // [2][b, h, qt (-1: no more), bad, n, row]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1) + 16;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* never = abort_flag + 1;  // stays 0: the last waits run to their own limit even after an abort
  float* max_s = reinterpret_cast<float*>(drained + 1) + 24;  // [2 turns][2 tiles][2 halves][TILE]
  float* sum_s = max_s + 8 * TILE;                            // [2 tiles][2 halves][TILE]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    *never = 0;
    mbar_init(drained, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 2 * TILE / 32);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_free[i], 2 * TILE / 32);
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], kMmaWarp + 1 + kScrubThreads / 32);  // softmax warps, MMA, scrub warps
    }
    mbar_init(q_empty, 1);
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
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // columns: S/P of tile t at t * 128, O of tile t at 256 + t * 128

  // the next item of a role (whole warp): false when there is none, or after an abort
  auto next_item = [&](uint32_t k, Work* w) {
    bool ok = mbar_wait(&item_full[k & 1], (k >> 1) & 1, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) return false;
    volatile int* it = item_s + (k & 1) * 8;
    if (it[2] < 0) return false;
    *w = work_of(a, it[0], it[1], it[2], it[4], it[5]);
    return true;
  };

  if (warp >= kMmaWarp) {
    reg_dec<kRegsRest>();
    if (warp == kTmaWarp) {
      const int nt = (a.N + ROWS - 1) / ROWS;
      const long long total =
          (a.lens == nullptr && a.cu == nullptr ? (long long)a.B * nt : count_from<ROWS>(a, 0)) * a.Hq;
      if (lane == 0) {
        prefetch_tmap(&tq);
        prefetch_tmap(&tk);
        prefetch_tmap(&tv);
      }
      auto load = [&](uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int row, int head, int batch) {
        mbar_arrive_expect_tx(bar, CF::kTileBytes);
#pragma unroll
        for (int kb = 0; kb < CF::kBlocks; ++kb) tma_load_4d(dst + kb * CF::kBlockBytes, m, bar, kb * 64, row, head, batch);
      };
      uint32_t kn = 0, vn = 0;              // key tiles issued so far
      uint32_t qph[2] = {0, 0};             // loads of each Q tile so far
      uint32_t vfull_n[kStages] = {}, vraw_n[kStages] = {};  // V tiles sent to each barrier
      bool ok = true;
      for (uint32_t k = 0; ok; ++k) {
        // items in a snake over the CTAs: the long ones spread evenly
        const long long L = (long long)k * gridDim.x + ((k & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        Item it{0, 0, -1};
        SeqView sv{};
        if (L < total) {
          it = find_item<ROWS>(a, L);
          sv = seq_view(a.lens, a.cu, true, it.b, a.N, a.total);
        }
        if (k >= 2) ok = mbar_wait(&item_empty[k & 1], (k / 2 - 1) & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          volatile int* o = item_s + (k & 1) * 8;
          o[0] = it.b;
          o[1] = it.h;
          o[2] = it.qt;
          o[3] = 0;
          o[4] = sv.n;
          o[5] = sv.q_row;
          mbar_arrive(&item_full[k & 1]);
        }
        if (it.qt < 0) break;
        const Work w = work_of(a, it.b, it.h, it.qt, sv.n, sv.q_row);
        if (lane == 0) {
          if (k > 0) ok = mbar_wait(q_empty, (k - 1) & 1, abort_flag);
          if (ok) {
            load(q_tile, &tq, &q_full[0], w.row + w.r0, w.h, w.batch);
            ++qph[0];
          }
          for (int j = 0; ok && j < w.nk; ++j) {
            const int ks = kn % kStages, vs = vn % kStages;
            if (kn >= kStages) ok = mbar_wait(&k_empty[ks], (kn / kStages - 1) & 1, abort_flag);
            if (!ok) break;
            load(k_ring + ks * CF::kTileBytes, &tk, &k_full[ks], w.row + j * TILE, w.g, w.batch);
            ++kn;
            if (j == 0 && w.nB > 0) {
              load(q_tile + CF::kTileBytes, &tq, &q_full[1], w.row + w.r0 + TILE, w.h, w.batch);
              ++qph[1];
            }
            if (vn >= kStages) ok = mbar_wait(&v_empty[vs], (vn / kStages - 1) & 1, abort_flag);
            if (!ok) break;
            load(v_ring + vs * CF::kTileBytes, &tv, j < w.js ? &v_full[vs] : &v_raw[vs], w.row + j * TILE, w.g,
                 w.batch);
            if (j < w.js)
              ++vfull_n[vs];
            else
              ++vraw_n[vs];
            ++vn;
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      if (lane == 0) {
        // do not leave while copies are in flight
        for (int i = 0; i < 2; ++i)
          if (qph[i] > 0) mbar_wait(&q_full[i], (qph[i] - 1) & 1, never);
        for (int s = 0; s < kStages; ++s) {
          const uint32_t kc = (kn + kStages - 1 - s) / kStages;  // tiles that went to slot s
          if (kc > 0) mbar_wait(&k_full[s], (kc - 1) & 1, never);
          if (vfull_n[s] > 0) mbar_wait(&v_full[s], (vfull_n[s] - 1) & 1, never);
          if (vraw_n[s] > 0) mbar_wait(&v_raw[s], (vraw_n[s] - 1) & 1, never);
        }
      }
    } else if (warp == kMmaWarp) {
      // the whole warp, in uniform control flow (see elect_one)
      const uint32_t idesc_s = idesc_mma(TILE, TILE, kBf16 ? 1u : 0u);
      const uint32_t idesc_o = idesc_mma(TILE, DP, kBf16 ? 1u : 0u) | kTransposeB;
      const uint32_t qs = smem_u32(q_tile), ks = smem_u32(k_ring), vs = smem_u32(v_ring), tm = uniform(tmem);
      uint32_t kn = 0, vn = 0;                              // key tiles taken so far (K: the next to be scored)
      uint32_t qph = 0, pph = 0, fph = 0;                   // parities, one bit a barrier
      uint32_t vfull = 0, vready = 0, o_used = 0;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
      };
      auto wait_bit = [&](uint64_t* bars, uint32_t& bits, int i) {
        const bool r = wait(&bars[i], (bits >> i) & 1u);
        bits ^= 1u << i;
        return r;
      };
      auto issue_s = [&](int t, uint32_t tile) {
        issue_scores<DP>(tm + t * TILE, qs + t * CF::kTileBytes, ks + (tile % kStages) * CF::kTileBytes, idesc_s);
      };
      Work w;
      for (uint32_t k = 0; next_item(k, &w); ++k) {
        const int nA = uniform(w.nA), nB = uniform(w.nB), nk = max(nA, nB), js = uniform(w.js);
        bool ok = wait(&k_full[kn % kStages], (kn / kStages) & 1);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || (t == 0 ? nA : nB) == 0) continue;
          ok = wait_bit(q_full, qph, t);
          if (!ok) continue;
          tc_fence_after();
          issue_s(t, kn);
          commit_warp(&s_full[t]);
        }
        if (ok) {
          commit_warp(&k_empty[kn % kStages]);
          if (nk == 1) commit_warp(q_empty);
        }
        ++kn;
        for (int j = 0; ok && j < nk; ++j, ++vn) {
          const int s = vn % kStages;
          ok = j < js ? wait_bit(v_full, vfull, s) : wait_bit(v_ready, vready, s);
          if (ok && j + 1 < nk) ok = wait(&k_full[kn % kStages], (kn / kStages) & 1);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int cnt = t == 0 ? nA : nB;
            if (!ok || j >= cnt) continue;
            ok = wait_bit(p_ready, pph, t);
            if (ok && j == 0 && ((o_used >> t) & 1u)) ok = wait_bit(o_free, fph, t);  // the last item's output has been read
            if (!ok) continue;
            tc_fence_after();
            issue_output<DP>(tm + 256 + t * TILE, tm + t * TILE, vs + s * CF::kTileBytes, idesc_o, j > 0 ? 1u : 0u);
            if (j + 1 < cnt) {
              issue_s(t, kn);
              commit_warp(&s_full[t]);
            } else {
              commit_warp(&o_full[t]);
              o_used |= 1u << t;
            }
          }
          if (!ok) break;
          commit_warp(&v_empty[s]);
          if (j + 1 < nk) {
            commit_warp(&k_empty[kn % kStages]);
            ++kn;
            if (j + 2 == nk) commit_warp(q_empty);  // the item's last scores
          }
        }
        if (!ok) {
          *abort_flag = 1;
          break;
        }
        if (lane == 0) mbar_arrive(&item_empty[k & 1]);
      }
      // TMEM and shared memory stay until every MMA has finished
      __syncwarp();
      commit_warp(drained);
      mbar_wait(drained, 0, never);
      __syncwarp();
    } else {
      const int st = threadIdx.x - (kTmaWarp + 1) * 32;
      if (a.fill && (a.lens != nullptr || a.cu != nullptr))
        fill_rows(a, (long long)blockIdx.x * kScrubThreads + st, (long long)gridDim.x * kScrubThreads);
      uint32_t vn = 0, raw = 0;
      Work w;
      for (uint32_t k = 0; next_item(k, &w); ++k) {
        const int n = w.n;
        bool ok = true;
        vn += min(w.js, w.nk);
        for (int j = w.js; j < w.nk; ++j, ++vn) {
          const int s = vn % kStages;
          ok = mbar_wait(&v_raw[s], (raw >> s) & 1u, abort_flag);
          raw ^= 1u << s;
          if (!ok) break;
          uint8_t* tile = v_ring + s * CF::kTileBytes;
          // rows that nobody keeps: zeros (a row is whole 128-byte pieces, however swizzled inside;
          // a row past the end may be zeroed before or after its pieces are tested below)
          for (int row = st; row < TILE; row += kScrubThreads) {
            const int c = j * TILE + row;
            if (c < n && (w.km == nullptr || w.km[c] != 0)) continue;
#pragma unroll
            for (int i = 0; i < CF::kBlocks * 8; ++i)
              *reinterpret_cast<uint4*>(tile + (i >> 3) * CF::kBlockBytes + row * 128 + (i & 7) * 16) =
                  make_uint4(0u, 0u, 0u, 0u);
          }
          // diagonal tiles: rows keep different keys
          if (a.causal && j >= 2 * w.qt) {
            if (scrub_pieces<kBf16>(tile, st, kScrubThreads, CF::kBlocks * TILE * 8,
                                    [&](int i) { return j * TILE + ((i >> 3) & (TILE - 1)) >= n; }))
              item_s[(k & 1) * 8 + 3] = 1;
          }
          fence_proxy_async_smem();
          mbar_arrive(&v_ready[s]);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive(&item_empty[k & 1]);
      }
    }
  } else {
    reg_inc<kRegsSoftmax>();
    const int t = warp >> 3, half = (warp >> 2) & 1, sub = warp & 3;
    const int rl = sub * 32 + lane;
    // this thread's scores, its output columns
    constexpr int kOut = DP / 2;
    const uint32_t lanes = tmem + ((uint32_t)(sub * 32) << 16) + t * TILE;
    const uint32_t ts = lanes + half * kAttCols, to = lanes + 256 + half * kOut;
    uint32_t sph = 0, oph = 0, turn = 0;
    Work w;
    for (uint32_t k = 0;; ++k) {
      if (bar_any<2 * TILE>(1 + t, !next_item(k, &w))) break;  // (a row tile's warps go on or stop together)
      const int n = w.n, row = w.r0 + t * TILE + rl, rt0 = w.r0 + t * TILE;
      const int cnt = t == 0 ? w.nA : w.nB;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < cnt; ++j, turn ^= 1u) {
        const int c0 = j * TILE + half * kAttCols;
        bool kk[2];
        if (w.km != nullptr) {  // before the wait: the loads overlap it
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int c = c0 + i * 32 + lane;
            kk[i] = c < n && w.km[c] != 0;
          }
        }
        ok = mbar_wait(&s_full[t], sph, abort_flag);
        sph ^= 1u;
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        uint32_t bits[2] = {0xffffffffu, 0xffffffffu};  // the keys that the mask keeps
        if (w.km != nullptr) {
#pragma unroll
          for (int i = 0; i < 2; ++i) bits[i] = __ballot_sync(0xffffffffu, kk[i]);
        }
        const bool edge = c0 + kAttCols > n || (a.causal && c0 + kAttCols - 1 > rt0);
        const int lim = min(a.causal ? row - c0 : kAttCols - 1, n - 1 - c0);  // the last key kept, from c0
        auto scores = [&](int i, float (&v)[32]) {
          tmem_ld32(ts + 32 * i, v);
          tmem_ld_wait();
          if (edge || w.km != nullptr) {
            const int last = lim - 32 * i;
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = c <= last && ((bits[i] >> c) & 1u) ? v[c] : -INFINITY;
          }
        };
        float v[32];
        scores(0, v);
        float mt = max32_nan(v);
        scores(1, v);
        mt = fmax_nan(mt, max32_nan(v));
        // the row's other half
        float* mx = max_s + (turn * 2 + t) * 2 * TILE;
        mx[half * TILE + rl] = mt;
        if (bar_any<2 * TILE>(1 + t, !ok)) {
          ok = false;
          break;
        }
        mt = __fmul_rn(fmax_nan(mt, mx[(half ^ 1) * TILE + rl]), C);  // rounded as the weights' products are
        const bool grow = mt - m > kAttGrow + kHead<kBf16> || mt != mt;  // (true from -inf to anything finite, and for NaN)
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = grow ? mt - kHead<kBf16> : m;
          const float f = m == mn ? 1.f : ex2(m - mn);
          l *= f;
          m = mn;
          if (j > 0) scale_output<kOut>(to, f);
        }
        const float shift = m == -INFINITY ? 0.f : -m;
        l += put_weights<kBf16, false>(v, C, shift, ts + 32);
        scores(0, v);
        l += put_weights<kBf16, false>(v, C, shift, ts);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t]);  // one arrival a warp
      }
      if (cnt > 0) {
        sum_s[(t * 2 + half) * TILE + rl] = l;
        ok = ok && mbar_wait(&o_full[t], oph, abort_flag);  // the output is complete
        oph ^= 1u;
        ok = !bar_any<2 * TILE>(1 + t, !ok);
        if (!ok) break;
        l += sum_s[(t * 2 + (half ^ 1)) * TILE + rl];
        tc_fence_after();
        float o[kOut];
#pragma unroll
        for (int i = 0; i < kOut / 32; ++i) tmem_ld32(to + 32 * i, *reinterpret_cast<float(*)[32]>(&o[32 * i]));
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[t]);
        // what the scrub warps found (the MMAs that the output waited for came after them)
        const bool bad = item_s[(k & 1) * 8 + 3] != 0;
        const bool none = l == 0.f;
        const float inv = none ? 0.f : 1.f / l;
        if (row < n) {
          const long long at = (long long)w.row + row;
          uint16_t* out = static_cast<uint16_t*>(a.out) + w.batch * a.os[0] + w.h * a.os[1] + at * a.os[2];
          if (bad) {
            // the diagonal tiles' non-finite elements, which the MMAs took as zeros
            const uint16_t* vg = static_cast<const uint16_t*>(a.v) + w.batch * a.vs[0] + w.g * a.vs[1] +
                                 (long long)w.row * a.vs[2];
#pragma unroll 1
            for (int c = 2 * w.qt * TILE; c <= row; ++c) {
              if (w.km != nullptr && w.km[c] == 0) continue;
#pragma unroll
              for (int e = 0; e < kOut; ++e) {
                if (half * kOut + e >= a.D) continue;
                const uint16_t x = vg[(long long)c * a.vs[2] + half * kOut + e];
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
          for (int e = 0; e < kOut; e += 8) {
            const int d = half * kOut + e;
            if (d >= a.D) continue;  // D % 8 == 0
            uint4 r;
            r.x = none ? 0u : pack16<kBf16>(o[e] * inv, o[e + 1] * inv);
            r.y = none ? 0u : pack16<kBf16>(o[e + 2] * inv, o[e + 3] * inv);
            r.z = none ? 0u : pack16<kBf16>(o[e + 4] * inv, o[e + 5] * inv);
            r.w = none ? 0u : pack16<kBf16>(o[e + 6] * inv, o[e + 7] * inv);
            *reinterpret_cast<uint4*>(out + d) = r;
          }
          if (half == 0)
            a.lse[w.batch * a.ls[0] + w.h * a.ls[1] + at * a.ls[2]] = none ? -INFINITY : (m + lg2(l)) * kLn2F;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[k & 1]);
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
int launch(const PromptArgs& a, int sms, cudaStream_t s) {
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
  if (packed) tiles = std::min(tiles, (a.total + ROWS - 1) / ROWS + a.B);  // no more than its rows make
  const long long grid = std::min<long long>(tiles * a.Hq, sms);
  kern<<<(unsigned)grid, kThreads, smem, s>>>(tq, tk, tv, a, a.scale * kLog2eF);
  return cudaGetLastError() == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
}

}  // namespace

bool prompt_tc_supported(const PromptArgs& a, int dtype) {
  if (dtype != KVBM_BF16 && dtype != KVBM_F16) return false;
  if (a.D > 128 || a.D % 8 != 0 || !tc_scale(a.scale) || !tc_path_enabled()) return false;
  const bool packed = a.cu != nullptr;
  const int B = packed ? 1 : a.B, N = packed ? (int)a.total : a.N;
  const int qd[3] = {B, a.Hq, N}, kd[3] = {B, a.Hkv, N};
  return aligned16(a.q, a.qs, qd) && aligned16(a.k, a.ks, kd) && aligned16(a.v, a.vs, kd) &&
         aligned16(a.out, a.os, qd);
}

int launch_prompt_tc(const PromptArgs& a, int dtype, cudaStream_t s) {
  const bool bf16 = dtype == KVBM_BF16;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) return KVBM_ERR_CUDA;
  const int sms = attention_device_sms(dev);
  if (sms < 1) return KVBM_ERR_CUDA;
  if (a.D <= 64) return bf16 ? launch<64, true>(a, sms, s) : launch<64, false>(a, sms, s);
  return bf16 ? launch<128, true>(a, sms, s) : launch<128, false>(a, sms, s);
}

unsigned int* attention_error_word() { return sm100::wait_error_word(); }

}  // namespace kvbm
