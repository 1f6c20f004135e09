// Attention of many rows per kv head (drafted trees: R = G * T > 32) over a
// paged cache on the tensor cores (tcgen05), bf16 / fp16, D <= 128, split over
// the keys (kvbm_attention.cu describes the split and the joining).
//
// One CTA an SM.  warps 0-7 and 8-15: softmax of two streams, two threads a
// row (kvbm_attention_tile.cuh); warp 16: MMA issuer; warps 17-19: loaders, in one of two ways:
//   kTma:  pages of a multiple of 8 slots that tile 128 keys evenly (or are a
//          multiple of 128): warp 17 loads each page with TMA, and warps 18-19
//          zero the v rows nobody keeps in the tiles that hold any (the last
//          ones, and with log offsets all);
//   else:  any page size: all three warps read the rows with 16-byte cp.async
//          into the layout TMA would write, page ids looked up one tile ahead.
//          (32768 keys x 4 sequences, 64 tokens: 358 us this way, 219 the other.)
//   kPair (R > 128): the streams are two tiles of 128 rows that share every
//                    key tile;
//   else:            one tile of rows, the streams take the even and the odd
//                    key tiles and are joined from TMEM at the end.
// Either way the tensor pipe works for one stream while the other's softmax
// runs.  With 256 rows a key tile of 64 KB takes 2048 tensor cycles, about as
// long as its bytes take from DRAM.  Measured: 4 sequences of 32768 keys, 64
// tokens, 32 q heads on 8, D = 128: 174 us with the joining (16 us of it), 3.0
// TB/s and 0.77 PFLOP/s: 53 key tiles a CTA at about 5800 cycles.  The prompt
// kernel's loop of the same two streams takes 3500 (its softmax chain), so about
// 2300 cycles a tile are this kernel's own; which wait holds them has not been
// measured (K and V share kSlots slots, and a tile is up to 16 box loads).
//
// Log offsets are added in the natural-log domain, and subtracted from before
// the conversion to base 2, so that offsets of float32's lowest value act like
// any other.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kvbm_attention.cuh"
#include "kvbm_attention_tile.cuh"

namespace kvbm {
namespace {
using namespace sm100;

constexpr int TILE = kAttTile;
constexpr int kThreads = 640;
constexpr int kMmaWarp = 16;
constexpr int kLoaders = 96;  // warps 17-19
constexpr int kSoftmax = 4 * TILE;  // softmax threads
// barriers: 1, 2 the streams' row maxima, then
constexpr int kLoaderBarrier = 3, kSoftmaxBarrier = 4, kScrubBarrier = 5;
// Registers a thread after the split: 4 softmax warpgroups + 1 of the rest; the launch holds 640 x 96.
constexpr int kRegsSoftmax = 104, kRegsRest = 64;
static_assert(4 * kRegsSoftmax + kRegsRest <= 5 * 96, "the split draws on the launch's registers");

template <int DP, bool kPair>
struct Cfg {
  static constexpr int kChunks = DP / 8;
  static constexpr int kTileBytes = TILE * DP * 2;
  static constexpr int kQTiles = kPair ? 2 : 1;
  // k and v tiles in one ring, in the order k0 v0 k1 v1 ...  Four slots are
  // enough for the order in which the MMA warp frees them (entry i is handed
  // over when entry i + kLag is issued, and waits for entry i + kLag - kSlots,
  // which an MMA issued before the wait for entry i frees); more hide latency.
  static constexpr int kSlots = DP == 128 ? (kPair ? 4 : 5) : 6;
  static constexpr int kLag = 2;  // copies still in flight when a tile is handed over
  static constexpr int kBars = 1 + 3 * kSlots + 4;
  static constexpr size_t kRing = (size_t)kTileBytes * (kQTiles + kSlots);
  static constexpr size_t kSmem = 1024 + kRing + 2 * TILE * 16 + 16 * kAttCols * 4 + 8 * TILE * 4 + 8 * kBars + 80 + 8 * kMaxTreeTokens;
  static_assert(kSmem <= 227 * 1024, "one CTA's shared memory");
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;  // 0: zero-filled, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// A whole 32-byte sector at once.
__device__ __forceinline__ void st_global8(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
template <int kId, int kCount>
__device__ __forceinline__ void bar_sync() {
  asm volatile("bar.sync %0, %1;" ::"n"(kId), "n"(kCount) : "memory");
}

// The segments of a CTA: parts [k0, k1) of units (b, g, rt), in order.
struct Segments {
  long long at, begin, end, bfirst;
  int b;
  // the current segment
  int len, nt, g, rt, k0, k1;
  long long ufirst;
  __device__ bool next(const CachedArgs& a) {
    if (at >= end) return false;
    len = cached_len(a, b);
    nt = (len + TILE - 1) / TILE;
    while (at >= bfirst + (long long)nt * a.Hkv * a.RT) {
      bfirst += (long long)nt * a.Hkv * a.RT;
      ++b;
      len = cached_len(a, b);
      nt = (len + TILE - 1) / TILE;
    }
    const int u = (int)((at - bfirst) / nt);
    g = u / a.RT;
    rt = u % a.RT;
    ufirst = bfirst + (long long)u * nt;
    k0 = (int)(at - ufirst);
    k1 = (int)min((long long)nt, end - ufirst);
    at = ufirst + k1;
    return true;
  }
};

template <int DP, bool kBf16, bool kPair, bool kBias, bool kTma>
__global__ void __launch_bounds__(kThreads, 1)
    cached_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const __grid_constant__ CachedArgs a) {
  using CF = Cfg<DP, kPair>;
  using T = std::conditional_t<kBf16, __nv_bfloat16, __half>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_tile = smem;
  uint8_t* ring = q_tile + CF::kQTiles * CF::kTileBytes;
  longlong2* offs = reinterpret_cast<longlong2*>(smem + CF::kRing);       // [2][TILE]
  float* bias_s = reinterpret_cast<float*>(offs + 2 * TILE);              // [16 warps][kAttCols]
  float* max_s = bias_s + 16 * kAttCols;                                  // [2 turns][2 streams][2 halves][TILE]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(max_s + 8 * TILE);
  uint64_t *full = q_full + 1, *empty = full + CF::kSlots, *raw = empty + CF::kSlots, *s_full = raw + CF::kSlots;
  uint64_t* p_ready = s_full + 2;
  long long* sched = reinterpret_cast<long long*>(p_ready + 2);  // total, first
  int* sched_b = reinterpret_cast<int*>(sched + 2);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sched_b + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // [8], by segment: the loaders are at most the ring's tiles, so three segments, ahead of the softmax warps
  volatile int* bad_flag = abort_flag + 1;
  unsigned long long* tree_s = reinterpret_cast<unsigned long long*>(sched + 10);  // [64]: tokens each token keeps
  volatile int* never = bad_flag + 8;  // stays 0: the last waits run to their own limit even after an abort

  cudaTriggerProgrammaticLaunchCompletion();  // the joining kernel may be set up beside this one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    long long pre, total, first = 0;
    warp_tile_prefix(a, 0, &pre, &total);
    const int b = warp_find_seq(a, split_begin(blockIdx.x, total, a.C), &first);
    if (lane == 0) {
      sched[0] = total;
      sched[1] = first;
      *sched_b = b;
      *abort_flag = 0;
      *never = 0;
      for (int i = 0; i < 8; ++i) bad_flag[i] = 0;
      mbar_init(q_full, kSoftmax / 32);
      for (int i = 0; i < CF::kSlots; ++i) {
        mbar_init(&full[i], kTma ? 1 : kLoaders);
        mbar_init(&empty[i], 1);
        mbar_init(&raw[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_ready[i], 2 * TILE / 32);
      }
      fence_mbar_init();
    }
  } else if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // columns: S/P of stream t at t * 128, O of stream t at 256 + t * 128
  Segments sg;
  sg.begin = split_begin(blockIdx.x, sched[0], a.C);
  sg.end = split_begin(blockIdx.x + 1, sched[0], a.C);
  sg.at = sg.begin;
  sg.bfirst = sched[1];
  sg.b = *sched_b;

  if (warp >= kMmaWarp) {
    reg_dec<kRegsRest>();
    if (warp == kMmaWarp) {
      // the whole warp, in uniform control flow (see elect_one)
      const uint32_t idesc_s = idesc_mma(TILE, TILE, kBf16 ? 1u : 0u);
      const uint32_t idesc_o = idesc_mma(TILE, DP, kBf16 ? 1u : 0u) | kTransposeB;
      const uint32_t qa = smem_u32(q_tile), ra = smem_u32(ring), tm = uniform(tmem);
      uint32_t idx = 0;     // ring index of this segment's k0
      uint32_t pph = 0;     // p_ready parities
      uint32_t used = 0;    // commits on s_full[t] so far: bit t, and their parity
      uint32_t sph = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
      };
      auto wait_full = [&](uint32_t i) { return wait(&full[i % CF::kSlots], (i / CF::kSlots) & 1u); };
      auto wait_p = [&](int t) {
        const bool r = wait(&p_ready[t], (pph >> t) & 1u);
        pph ^= 1u << t;
        return r;
      };
      auto commit_s = [&](int t) {
        commit_warp(&s_full[t]);
        used |= 1u << t;
        sph ^= 1u << t;
      };
      for (uint32_t seg = 0; ok && sg.next(a); ++seg) {
        const int nk = uniform(sg.k1 - sg.k0);
        auto slot_at = [&](uint32_t i) { return ra + (i % CF::kSlots) * CF::kTileBytes; };
        auto issue_s = [&](int t, int j) {
          issue_scores<DP>(tm + t * TILE, qa + (kPair ? t : 0) * CF::kTileBytes, slot_at(idx + 2 * j), idesc_s);
        };
        ok = wait(q_full, seg & 1u);
        if constexpr (kPair) {
          ok = ok && wait_full(idx);
          if (ok) {
            tc_fence_after();
            fence_proxy_async_smem();
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              issue_s(t, 0);
              commit_s(t);
            }
            commit_warp(&empty[idx % CF::kSlots]);
          }
          for (int j = 0; ok && j < nk; ++j) {
            ok = wait_full(idx + 2 * j + 1);
            if (ok && j + 1 < nk) ok = wait_full(idx + 2 * j + 2);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              ok = ok && wait_p(t);
              if (!ok) continue;
              tc_fence_after();
              issue_output<DP>(tm + 256 + t * TILE, tm + t * TILE, slot_at(idx + 2 * j + 1), idesc_o, j > 0 ? 1u : 0u);
              if (j + 1 < nk) issue_s(t, j + 1);
              commit_s(t);  // the next S, or the finished O
            }
            if (!ok) break;
            commit_warp(&empty[(idx + 2 * j + 1) % CF::kSlots]);
            if (j + 1 < nk) commit_warp(&empty[(idx + 2 * j + 2) % CF::kSlots]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || t >= nk) continue;
            ok = wait_full(idx + 2 * t);
            if (!ok) continue;
            tc_fence_after();
            issue_s(t, t);
            commit_s(t);
            commit_warp(&empty[(idx + 2 * t) % CF::kSlots]);
          }
          for (int j = 0; ok && j < nk; ++j) {
            const int t = j & 1;
            ok = wait_full(idx + 2 * j + 1) && wait_p(t);
            if (!ok) break;
            tc_fence_after();
            issue_output<DP>(tm + 256 + t * TILE, tm + t * TILE, slot_at(idx + 2 * j + 1), idesc_o, j > 1 ? 1u : 0u);
            commit_warp(&empty[(idx + 2 * j + 1) % CF::kSlots]);
            if (j + 2 < nk) {
              ok = wait_full(idx + 2 * j + 4);
              if (!ok) break;
              tc_fence_after();
              issue_s(t, j + 2);
              commit_s(t);
              commit_warp(&empty[(idx + 2 * j + 4) % CF::kSlots]);
            } else {
              commit_s(t);  // the finished O
            }
          }
        }
        idx += 2 * (uint32_t)nk;
      }
      // TMEM and shared memory stay until every MMA has finished
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if ((used >> t) & 1u) mbar_wait(&s_full[t], ((sph >> t) & 1u) ^ 1u, never);
      __syncwarp();
    } else {
      // ---- loaders
      const int lt = threadIdx.x - (kMmaWarp + 1) * 32;
      const uint32_t ra = smem_u32(ring);
      const T *kbase = static_cast<const T*>(a.k), *vbase = static_cast<const T*>(a.v);
      const int ch = lt % CF::kChunks;
      const bool in = ch * 8 < a.D;
      uint32_t idx = 0;  // ring index of this segment's first tile (two a key tile: below 2^32 for any call)
      uint32_t raw_phase = 0;  // per slot (kTma)
      bool ok = true;
      if (kTma && lt == 0) {
        prefetch_tmap(&tk);
        prefetch_tmap(&tv);
      }
      for (uint32_t seg = 0; ok && sg.next(a); ++seg) {
        const int b = sg.b, g = sg.g, len = sg.len, pre = len - a.T;
        const float* off = kBias ? a.off + b * a.ob + g * a.oh : nullptr;
        const int nk = sg.k1 - sg.k0;
        if constexpr (kTma) {
          const int P = a.pg.page_size, rows = P < TILE ? P : TILE;
          // v tiles from js on hold rows that not every query keeps, or nobody does
          const int js = kBias ? 0 : max(0, pre / TILE - sg.k0);
          if (warp == kMmaWarp + 1) {
            // lane i: page i / kBlk of the tile, 64-column block i % kBlk
            constexpr int kBlk = DP / 64;
            const int pieces = TILE / rows;
            auto page_at = [&](int j) -> int {  // -2: past the sequence, -1: not a page
              const int c = (sg.k0 + j) * TILE + (lane / kBlk) * rows;
              if (lane / kBlk >= pieces || j >= nk || c >= len) return -2;
              const int page = a.pg.page(b, a.pg.page_index(c));
              if (page >= 0 && page < a.pg.num_pages) return page;
              atomicOr(a.page_error, 1u);
              return -1;
            };
            int next = page_at(0);
            for (int j = 0; ok && j < nk; ++j) {
              const int page = next;
              next = page_at(j + 1);
              const unsigned there = __ballot_sync(0xffffffffu, page >= 0 && lane % kBlk == 0);
              const bool gone = __any_sync(0xffffffffu, page == -1);
              const uint32_t bytes = (uint32_t)__popc(there) * rows * DP * 2;
              const int slot_c = a.pg.slot((sg.k0 + j) * TILE + (lane / kBlk) * rows);
#pragma unroll 1
              for (int kv = 0; kv < 2; ++kv) {
                const uint32_t i = idx + 2 * j + kv;
                const int slot = (int)(i % CF::kSlots);
                if (i >= CF::kSlots) ok = mbar_wait(&empty[slot], (uint32_t)(i / CF::kSlots - 1) & 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                uint8_t* tile = ring + slot * CF::kTileBytes;
                if (gone) {  // keys of a bad table entry count as zero vectors
                  for (int pc = 0; pc < pieces; ++pc) {
                    if (__shfl_sync(0xffffffffu, page, pc * kBlk) != -1) continue;
                    for (int e = lane; e < rows * 8 * kBlk; e += 32)
                      *reinterpret_cast<uint4*>(tile + (e / (rows * 8)) * (TILE * 128) + pc * rows * 128 +
                                                (e % (rows * 8)) * 16) = make_uint4(0u, 0u, 0u, 0u);
                  }
                  fence_proxy_async_smem();
                  __syncwarp();
                }
                uint64_t* bar = kv && j >= js ? &raw[slot] : &full[slot];
                if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
                __syncwarp();
                if (page >= 0)
                  tma_load_4d(tile + (lane % kBlk) * (TILE * 128) + (lane / kBlk) * rows * 128, kv ? &tv : &tk, bar,
                              (lane % kBlk) * 64, slot_c, g, page);
              }
            }
          } else {
            const int st = lt - 32;
            for (int j = js; j < nk; ++j) {
              const uint32_t i = idx + 2 * j + 1;
              const int slot = (int)(i % CF::kSlots);
              ok = mbar_wait(&raw[slot], (raw_phase >> slot) & 1u, abort_flag) && ok;
              raw_phase ^= 1u << slot;
              ok = !bar_any<kLoaders - 32>(kScrubBarrier, !ok);
              if (!ok) break;
              {
                uint8_t* tile = ring + slot * CF::kTileBytes;
                const int c0 = (sg.k0 + j) * TILE;
                for (int r = st; r < TILE; r += kLoaders - 32) {
                  const int c = c0 + r;
                  if (c < len && !(kBias && off[c] == -INFINITY)) continue;
#pragma unroll
                  for (int e = 0; e < CF::kChunks; ++e)
                    *reinterpret_cast<uint4*>(tile + (e >> 3) * (TILE * 128) + r * 128 + (e & 7) * 16) =
                        make_uint4(0u, 0u, 0u, 0u);
                }
                if (c0 + TILE > pre) {
                  // drafted tokens: rows keep different ones; non-finite elements are taken out here and
                  // added to the rows that keep them at the end
                  bar_sync<kScrubBarrier, kLoaders - 32>();
                  const bool bad =
                      scrub_pieces<kBf16>(tile, st, kLoaders - 32, TILE * CF::kChunks,
                                          [&](int e) { return c0 + ((e >> 3) & (TILE - 1)) < pre; });
                  if (bad) bad_flag[seg & 7] = 1;
                }
                fence_proxy_async_smem();
              }
              bar_sync<kScrubBarrier, kLoaders - 32>();
              if (st == 0) mbar_arrive(&full[slot]);
            }
          }
        } else {
          auto page_of = [&](int c) -> int {
            if (c >= len) return -1;
            return a.pg.page(b, a.pg.page_index(c));
          };
          auto offset_of = [&](int c, int page) {
            longlong2 o = make_longlong2(-1, -1);
            if (c >= len || (kBias && off[c] == -INFINITY)) return o;
            if (page < 0 || page >= a.pg.num_pages) {
              atomicOr(a.page_error, 1u);
              return o;
            }
            const int at = a.pg.slot(c);
            o.x = (long long)page * a.ks[0] + (long long)at * a.ks[1] + g * a.ks[2];
            o.y = (long long)page * a.vs[0] + (long long)at * a.vs[1] + g * a.vs[2];
            return o;
          };
          // hand over ring entry i (its copies have landed for this thread)
          auto hand_over = [&](uint32_t i) {
            const int j = sg.k0 + (int)((i - idx) >> 1);
            if (((i - idx) & 1) && (j + 1) * TILE > pre) {
              // v of drafted tokens: rows keep different ones; this thread's
              // own pieces are checked, non-finite elements taken out and added
              // to the rows that keep them at the end
              uint8_t* tile = ring + (int)(i % CF::kSlots) * CF::kTileBytes;
              bool bad = false;
              for (int r = lt / CF::kChunks; r < TILE; r += kLoaders / CF::kChunks)
                if (j * TILE + r >= pre)
                  bad |= drop_nonfinite<kBf16>(reinterpret_cast<uint4*>(tile + (ch >> 3) * (TILE * 128) + r * 128 +
                                                                        (((ch & 7) ^ (r & 7)) << 4)));
              if (bad) bad_flag[seg & 7] = 1;
            }
            fence_proxy_async_smem();
            mbar_arrive(&full[i % CF::kSlots]);
          };
          int page0 = page_of(sg.k0 * TILE + lt), page1 = lt < TILE - kLoaders ? page_of(sg.k0 * TILE + kLoaders + lt) : -1;
          for (int j = 0; j < nk; ++j) {
            const int c0 = (sg.k0 + j) * TILE;
            longlong2* of = offs + (j & 1) * TILE;
            of[lt] = offset_of(c0 + lt, page0);
            if (lt < TILE - kLoaders) of[kLoaders + lt] = offset_of(c0 + kLoaders + lt, page1);
            if (j + 1 < nk) {
              page0 = page_of(c0 + TILE + lt);
              if (lt < TILE - kLoaders) page1 = page_of(c0 + TILE + kLoaders + lt);
            }
            ok = !bar_any<kLoaders>(kLoaderBarrier, !ok);
            if (!ok) break;
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv) {
              const uint32_t i = idx + 2 * j + kv;
              const int slot = (int)(i % CF::kSlots);
              if (i >= CF::kSlots)
                ok = mbar_wait(&empty[slot], (uint32_t)(i / CF::kSlots - 1) & 1u, abort_flag) && ok;
              if (ok) {
                const uint32_t dst = ra + slot * CF::kTileBytes + (ch >> 3) * (TILE * 128);
                const T* base = kv ? vbase : kbase;
#pragma unroll 4
                for (int r = lt / CF::kChunks; r < TILE; r += kLoaders / CF::kChunks) {
                  const long long o = kv ? of[r].y : of[r].x;
                  const bool live = in && o >= 0;
                  cp16(dst + r * 128 + (((ch & 7) ^ (r & 7)) << 4), live ? base + o + ch * 8 : base, live);
                }
              }
              asm volatile("cp.async.commit_group;" ::: "memory");
              if (2 * j + kv >= CF::kLag) {
                cp_wait<CF::kLag>();
                hand_over(i - CF::kLag);
              }
            }
          }
          ok = !bar_any<kLoaders>(kLoaderBarrier, !ok);
          if (!ok) break;
          static_assert(CF::kLag == 2, "the tail below hands over two entries");
          cp_wait<1>();
          hand_over(idx + 2 * nk - 2);
          cp_wait<0>();
          hand_over(idx + 2 * nk - 1);
        }
        idx += 2 * (uint32_t)nk;
      }
      cp_wait<0>();
    }
  } else {
    // ---- softmax
    reg_inc<kRegsSoftmax>();
    const int t = warp >> 3, half = (warp >> 2) & 1, sub = warp & 3;
    const int rl = sub * 32 + lane;
    constexpr int kOut = DP / 2;  // output columns a thread scales
    const uint32_t row_at = tmem + ((uint32_t)(sub * 32) << 16), lanes = row_at + t * TILE;
    const uint32_t ts = lanes + half * kAttCols, to = lanes + 256 + half * kOut;
    float* wbias = bias_s + warp * kAttCols;
    const float C = kBias ? kLog2eF : a.scale * kLog2eF;
    uint32_t sn = 0;  // s_full phases used
    bool ok = true;
    for (uint32_t seg = 0; ok && sg.next(a); ++seg) {
      const int b = sg.b, g = sg.g, len = sg.len, pre = len - a.T, nk = sg.k1 - sg.k0;
      const int r = (sg.rt * CF::kQTiles + (kPair ? t : 0)) * TILE + rl;  // row of the unit
      const int tok = r % a.T, h = g * a.G + r / a.T;
      const float* off = kBias ? a.off + b * a.ob + g * a.oh : nullptr;
      {
        // the queries, by the 512 threads that have nothing else to do yet (their tile is free: every MMA of the
        // segment before has completed).  A few loader threads took 12 us of a 180 us call for it.
        const uint32_t qa = smem_u32(q_tile);
        const T* qbase = static_cast<const T*>(a.q) + b * a.qs[0];
        const int c = threadIdx.x % CF::kChunks;
        for (int row = threadIdx.x / CF::kChunks; row < CF::kQTiles * TILE; row += kSoftmax / CF::kChunks) {
          const int qr = sg.rt * CF::kQTiles * TILE + row, ql = row % TILE;
          const bool live = qr < a.R && c * 8 < a.D;
          cp16(qa + (row / TILE) * CF::kTileBytes + (c >> 3) * (TILE * 128) + ql * 128 + (((c & 7) ^ (ql & 7)) << 4),
               live ? qbase + (long long)(g * a.G + qr / a.T) * a.qs[1] + (long long)(qr % a.T) * a.qs[2] + c * 8 : qbase,
               live);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        cp_wait<0>();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      // drafted tokens this row keeps
      unsigned long long tree = 0;
      if (sg.k1 * TILE > pre) {
        if (a.tree != nullptr) {
          // a warp reads whole mask rows and packs them (a thread reading its own row byte by byte: 9 us)
          const uint8_t* tm = a.tree + b * a.tb;
          for (int x = warp; x < a.T; x += kMmaWarp) {
            const bool b0 = lane < a.T && tm[x * a.tr + lane] != 0, b1 = lane + 32 < a.T && tm[x * a.tr + lane + 32] != 0;
            const uint32_t w0 = __ballot_sync(0xffffffffu, b0), w1 = __ballot_sync(0xffffffffu, b1);
            if (lane == 0) tree_s[x] = (unsigned long long)w1 << 32 | w0;
          }
          bar_any<kSoftmax>(kSoftmaxBarrier, false);
          tree = tree_s[tok];
        } else {
          tree = ~0ull >> (63 - tok);
        }
      }
      float m = -INFINITY, l = 0.f;
      int done = 0;  // tiles of this stream
      for (int j = kPair ? 0 : t; j < nk; j += kPair ? 1 : 2, ++done) {
        const int c0 = (sg.k0 + j) * TILE + half * kAttCols;
        if constexpr (kBias) {
          __syncwarp();
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int c = c0 + 32 * w + lane;
            wbias[32 * w + lane] = c < len ? off[c] : -INFINITY;
          }
          __syncwarp();
        }
        ok = mbar_wait(&s_full[t], sn++ & 1u, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        auto scores = [&](int i, float (&v)[32]) {
          tmem_ld32(ts + 32 * i, v);
          tmem_ld_wait();
          if constexpr (kBias) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 x = *reinterpret_cast<const float4*>(wbias + 32 * i + c);
              // (a dropped key's score may be anything)
              v[c] = x.x == -INFINITY ? -INFINITY : fmaf(v[c], a.scale, x.x);
              v[c + 1] = x.y == -INFINITY ? -INFINITY : fmaf(v[c + 1], a.scale, x.y);
              v[c + 2] = x.z == -INFINITY ? -INFINITY : fmaf(v[c + 2], a.scale, x.z);
              v[c + 3] = x.w == -INFINITY ? -INFINITY : fmaf(v[c + 3], a.scale, x.w);
            }
          }
          if (c0 + kAttCols > pre) {
            const int sh = c0 + 32 * i - pre;  // drafted token of the first key
            uint32_t bits;
            if (sh <= -32)
              bits = 0xffffffffu;
            else if (sh < 0)
              bits = ((uint32_t)tree << -sh) | ((1u << -sh) - 1u);
            else
              bits = sh < 64 ? (uint32_t)(tree >> sh) : 0u;
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = ((bits >> c) & 1u) ? v[c] : -INFINITY;
          }
        };
        float v[32];
        scores(0, v);
        float mt = max32_nan(v);
        scores(1, v);
        mt = fmax_nan(mt, max32_nan(v));
        // the row's other half
        float* mx = max_s + ((done & 1) * 2 + t) * 2 * TILE;
        mx[half * TILE + rl] = mt;
        if (bar_any<2 * TILE>(1 + t, !ok)) {
          ok = false;
          break;
        }
        mt = fmax_nan(mt, mx[(half ^ 1) * TILE + rl]);
        if (!kBias) mt = __fmul_rn(mt, C);  // rounded as the weights' products are
        constexpr float kUnit = kBias ? kLn2F : 1.f;  // natural logarithms, or base 2
        const bool grow = mt - m > (kAttGrow + kHead<kBf16>) * kUnit || mt != mt;
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = grow ? mt - kHead<kBf16> * kUnit : m;
          const float f = m == mn ? 1.f : ex2(kBias ? (m - mn) * kLog2eF : m - mn);
          l *= f;
          m = mn;
          if (done > 0) scale_output<kOut>(to, f);
        }
        const float shift = m == -INFINITY ? 0.f : -m;
        l += put_weights<kBf16, kBias>(v, C, shift, ts + 32);
        scores(0, v);
        l += put_weights<kBf16, kBias>(v, C, shift, ts);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t]);  // one arrival a warp
      }
      if (ok && done > 0) ok = mbar_wait(&s_full[t], sn++ & 1u, abort_flag);  // O is complete
      // sums of the halves (and of the streams) meet in the turns' slots, which everyone has read
      if (bar_any<kSoftmax>(kSoftmaxBarrier, !ok)) break;
      float* ls = max_s;                 // [2 streams][2 halves][TILE]
      float* ms = max_s + 4 * TILE;      // [2 streams][TILE]
      ls[(t * 2 + half) * TILE + rl] = l;
      if (half == 0) ms[t * TILE + rl] = m;
      bar_any<kSoftmax>(kSoftmaxBarrier, false);
      tc_fence_after();
      l = ls[t * 2 * TILE + rl] + ls[(t * 2 + 1) * TILE + rl];
      // ---- the segment's result
      const bool whole = sg.k0 == 0 && sg.k1 == sg.nt;
      const long long pr = ((long long)blockIdx.x * 2 + (sg.begin >= sg.ufirst ? 0 : 1)) * a.BM +
                           (kPair ? t * TILE + rl : rl);
      float f0 = 1.f, f1 = 0.f;
      if constexpr (!kPair) {  // both streams hold the same rows
        const float m0 = ms[rl], m1 = ms[TILE + rl];
        m = fmaxf(m0, m1);
        const float base = m == -INFINITY ? 0.f : m;
        const float C1 = kBias ? kLog2eF : 1.f;
        f0 = ex2((m0 - base) * C1);
        f1 = ex2((m1 - base) * C1);
        l = (ls[rl] + ls[TILE + rl]) * f0 + (ls[2 * TILE + rl] + ls[3 * TILE + rl]) * f1;
      }
      const bool bad = bad_flag[seg & 7] != 0;
      const float m_nat = kBias ? m : m * kLn2F;
      const bool none = l == 0.f;
      const float inv = none ? 0.f : 1.f / l;
      // columns of the result: of the thread's own row tile half of them, of the joined streams a quarter
      constexpr int kCols = kPair ? DP / 2 : DP / 4;
      const int col0 = kPair ? half * kCols : (t * 2 + half) * kCols;
      constexpr int kStep = kCols < 32 ? 16 : 32;
      uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.os[0] + h * a.os[1] + tok * a.os[2];
#pragma unroll
      for (int w = 0; w < kCols / kStep; ++w) {
        const int d0 = col0 + kStep * w;
        float o[kStep];
        if constexpr (kPair) {
          tmem_load<kStep>(row_at + 256 + t * TILE + d0, o);
          tmem_ld_wait();
        } else {
          float o1[kStep];
          tmem_load<kStep>(row_at + 256 + d0, o);
          tmem_load<kStep>(row_at + 256 + TILE + d0, o1);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < kStep; ++e) o[e] = nk > 1 ? o[e] * f0 + o1[e] * f1 : o[e] * f0;
        }
        if (r < a.R) {
          if (bad) {
#pragma unroll
            for (int e = 0; e < kStep; e += 4) {
              float4 x = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
              if (d0 + e < a.D)
                add_nonfinite<T>(a, b, g, tok, max(max(pre, 0), sg.k0 * TILE), min(len, sg.k1 * TILE), pre, d0 + e, x);
              o[e] = x.x;
              o[e + 1] = x.y;
              o[e + 2] = x.z;
              o[e + 3] = x.w;
            }
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < kStep; e += 8) {
              if (d0 + e >= a.D) continue;  // D % 8 == 0
              uint4 x;
              x.x = none ? 0u : pack16<kBf16>(o[e] * inv, o[e + 1] * inv);
              x.y = none ? 0u : pack16<kBf16>(o[e + 2] * inv, o[e + 3] * inv);
              x.z = none ? 0u : pack16<kBf16>(o[e + 4] * inv, o[e + 5] * inv);
              x.w = none ? 0u : pack16<kBf16>(o[e + 6] * inv, o[e + 7] * inv);
              *reinterpret_cast<uint4*>(out + d0 + e) = x;
            }
          } else {
#pragma unroll
            for (int e = 0; e < kStep; e += 8) st_global8(a.part_o + pr * a.DP + d0 + e, o + e);
          }
        }
        __syncwarp();  // the next load is the whole warp's
      }
      if (r < a.R && half == 0 && (kPair || t == 0)) {
        if (whole)
          a.lse[b * a.ls[0] + h * a.ls[1] + tok * a.ls[2]] = none ? -INFINITY : m_nat + logf(l);
        else
          a.part_ml[pr] = make_float2(m_nat, l);
      }
      tc_fence_before();
      bar_any<kSoftmax>(kSoftmaxBarrier, false);  // everyone has read the flag, the sums and O
      if (threadIdx.x == 0) bad_flag[seg & 7] = 0;
    }
    tc_fence_before();
  }

  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DP, bool kBf16, bool kPair, bool kBias, bool kTma>
int launch(const CachedArgs& a, cudaStream_t s) {
  auto kern = cached_tc_kernel<DP, kBf16, kPair, kBias, kTma>;
  constexpr size_t bytes = Cfg<DP, kPair>::kSmem;
  if (allow_smem(kern, bytes) != KVBM_OK) return KVBM_ERR_CUDA;
  CUtensorMap tk = {}, tv = {};
  if constexpr (kTma) {
    const int rows = std::min(a.pg.page_size, TILE);
    const int64_t ks[4] = {a.ks[0], a.ks[2], a.ks[1], 1}, vs[4] = {a.vs[0], a.vs[2], a.vs[1], 1};
    if (!make_attention_map(&tk, a.k, kBf16, a.pg.num_pages, a.Hkv, a.pg.page_size, a.D, ks, rows) ||
        !make_attention_map(&tv, a.v, kBf16, a.pg.num_pages, a.Hkv, a.pg.page_size, a.D, vs, rows))
      return KVBM_ERR_CUDA;
  }
  kern<<<(unsigned)a.C, kThreads, bytes, s>>>(tk, tv, a);
  return cudaGetLastError() == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
}

// Pages that TMA can load as pieces of a 128-key tile: whole 8-row swizzle
// atoms, even division, no expanded dimension.
bool pages_by_tma(const CachedArgs& a) {
  const int P = a.pg.page_size;
  if (P % 8 != 0 || !(TILE % P == 0 || P % TILE == 0)) return false;
  for (const long long* st : {a.ks, a.vs})
    if ((st[0] == 0 && a.pg.num_pages > 1) || (st[1] == 0 && P > 1) || (st[2] == 0 && a.Hkv > 1)) return false;
  return true;
}

template <int DP, bool kBf16, bool kPair>
int launch_p(const CachedArgs& a, cudaStream_t s) {
  if (pages_by_tma(a))
    return a.off != nullptr ? launch<DP, kBf16, kPair, true, true>(a, s) : launch<DP, kBf16, kPair, false, true>(a, s);
  return a.off != nullptr ? launch<DP, kBf16, kPair, true, false>(a, s) : launch<DP, kBf16, kPair, false, false>(a, s);
}

template <int DP, bool kBf16>
int launch_d(const CachedArgs& a, cudaStream_t s) {
  return a.BM == 2 * TILE ? launch_p<DP, kBf16, true>(a, s) : launch_p<DP, kBf16, false>(a, s);
}

}  // namespace

int launch_cached_tc(const CachedArgs& a, int dtype, cudaStream_t s) {
  const bool bf16 = dtype == KVBM_BF16;
  if (a.DP == 64) return bf16 ? launch_d<64, true>(a, s) : launch_d<64, false>(a, s);
  return bf16 ? launch_d<128, true>(a, s) : launch_d<128, false>(a, s);
}

unsigned int* cached_error_word() { return sm100::wait_error_word(); }

}  // namespace kvbm
