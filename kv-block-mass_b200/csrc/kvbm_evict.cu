// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, weight head): the first n_sinks tokens, the last `recency`
// tokens and, of those between, the budget - n_sinks - recency with the
// highest weights stay (equal weights: the lower index; NaN counts as -inf).
// Kept tokens keep their order.
//
// Two kernels.  evict_select_kernel finds the threshold weight with a radix
// select over order-preserving 32-bit keys (three histogram passes, of the top
// 11, the next 11 and the last 10 bits) and turns the choice into slots with two
// walks over the row: 4 * len bytes of weights are all it reads from DRAM (once,
// into shared memory, where the CTAs' share of a row fits).  evict_gather_kernel
// moves the kept k and v rows, 16 bytes a thread: 4 * budget * D elements a head.
// Measured: 8 sequences of up to 16384 tokens cut to 4096 per head (8 heads of 128,
// bf16): 74 us, the choice 25 of it (the latency of three passes with three
// cluster barriers each and of the walks) and the move 49, 5.5 TB/s; one sequence
// of 32768 cut to 8192 for all heads alike: 31 us.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "kvbm_attention.cuh"

namespace kvbm {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kGatherThreads = 512;  // one element a thread at D = 256: 2 * 256 threads a slot
constexpr int kSmemKeys = 48 * 1024;
constexpr int kGatherUnroll = 8;

struct EvictArgs {
  PagedView pg;
  const char *k, *v;
  long long ks[4], vs[4];  // [num_pages, page_size, Hkv, D], in V units on the gather's 16-byte path
  char *ko, *vo;
  long long kos[4], vos[4];  // [B, capacity, Hkv, D]
  int B, Hkv, Hw, D, Lmax;
  const int32_t* lens;
  const float* w;
  long long wb, wh;
  int budget, n_sinks, recency, capacity, zero_tail;
  int32_t* lens_out;
  int32_t* kept;      // [B, Hw, budget]
  float* wout;        // [B, Hw, budget] or null
  unsigned int* page_error;
};

__device__ __forceinline__ int evict_len(const EvictArgs& a, int b) {
  const int n = a.lens[b];
  return n < 0 ? 0 : (n < a.Lmax ? n : a.Lmax);
}

// Order-preserving key: larger weight, larger key; -0 as +0, NaN as -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A cluster of kCluster CTAs per (sequence, weight head); each takes a run of
// the row and reads it once into shared memory (runs past kSmemKeys:
// re-read from L2 in every pass).  Threshold: three histogram passes of 11, 11
// and 10 bits over the candidates; in each warp the lanes that share the first
// lane's bin add once together, since many weights are alike (keys nothing
// attended to); the CTAs' histograms meet in the first CTA's shared memory.
// Slots: each warp takes a part of its CTA's run and counts its ties and kept
// tokens with ballots; sums over the warps and CTAs before it give its first
// slot, and a second walk writes.
template <int kCluster>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictArgs a, int smem_keys) {
  namespace cg = cooperative_groups;
  extern __shared__ float row_s[];
  __shared__ unsigned int hist[2048];
  __shared__ int scan_buf[kSelThreads / 32], warp_ties[kSelThreads / 32], warp_gt[kSelThreads / 32];
  __shared__ unsigned int s_prefix;
  __shared__ int s_left, cta_ties, cta_gt;
  cudaTriggerProgrammaticLaunchCompletion();
  cg::cluster_group cl = cg::this_cluster();
  const int rank = kCluster > 1 ? (int)cl.block_rank() : 0;
  auto all_ctas = [&] {
    if constexpr (kCluster > 1)
      cl.sync();
    else
      __syncthreads();
  };
  const int row = blockIdx.x / kCluster, b = row / a.Hw, hw = row % a.Hw;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int len = evict_len(a, b);
  const float* w = a.w + b * a.wb + hw * a.wh;
  int32_t* kept = a.kept + (long long)row * a.budget;
  float* wout = a.wout ? a.wout + (long long)row * a.budget : nullptr;
  const int new_len = min(len, a.budget);
  if (hw == 0 && t == 0 && rank == 0) a.lens_out[b] = new_len;
  for (int j = new_len + rank * kSelThreads + t; j < a.budget; j += kCluster * kSelThreads) {
    kept[j] = -1;
    if (wout) wout[j] = 0.f;
  }
  if (len <= a.budget) {  // the same for every CTA of the cluster
    for (int j = rank * kSelThreads + t; j < len; j += kCluster * kSelThreads) {
      kept[j] = j;
      if (wout) wout[j] = w[j];
    }
    return;
  }
  const int lo = a.n_sinks, hi = len - a.recency;  // the candidates; budget >= n_sinks + recency, so lo <= hi
  const int take = a.budget - a.n_sinks - a.recency;
  // this CTA's tokens [r_lo, r_hi), and the candidates among them
  const int cta_run = (len + kCluster * kSelThreads - 1) / (kCluster * kSelThreads) * kSelThreads;
  const int r_lo = min(len, rank * cta_run), r_hi = min(len, r_lo + cta_run);
  const int d_lo = max(lo, r_lo), d_hi = min(hi, r_hi);
  const bool cached = cta_run <= smem_keys;
  if (cached) {
#pragma unroll 8
    for (int c = r_lo + t; c < r_hi; c += kSelThreads) row_s[c - r_lo] = w[c];
  }
  auto weight_at = [&](int c) { return cached ? row_s[c - r_lo] : w[c]; };
  auto key_at = [&](int c) { return weight_key(weight_at(c)); };
  // 1. threshold key of the `take` highest candidates, and how many of its
  //    ties are taken (from the lowest index)
  uint32_t pre = 0;
  int left = take;
  if (take > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = t; i < 2048; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t high = pass == 0 ? 0u : ~0u << (shift + bits), mask = (1u << bits) - 1u;
#pragma unroll 4
      for (int c0 = d_lo + warp * 32; c0 < d_hi; c0 += kSelThreads) {
        const int c = c0 + lane;
        const uint32_t key = c < d_hi ? key_at(c) : 0u;
        const bool in = c < d_hi && ((key ^ pre) & high) == 0;
        const unsigned act = __ballot_sync(0xffffffffu, in);
        if (act == 0) continue;
        const uint32_t bin = (key >> shift) & mask;
        const int first = __ffs(act) - 1;
        const uint32_t bin0 = __shfl_sync(0xffffffffu, bin, first);
        const unsigned same = __ballot_sync(0xffffffffu, in && bin == bin0);
        if (lane == first) atomicAdd(&hist[bin0], (unsigned)__popc(same));
        if (in && bin != bin0) atomicAdd(&hist[bin], 1u);
      }
      all_ctas();
      if constexpr (kCluster > 1) {
        if (rank != 0) {
          unsigned int* root = cl.map_shared_rank(hist, 0);
          for (int i = t; i < 2048; i += kSelThreads)
            if (hist[i] != 0) atomicAdd(&root[i], hist[i]);
        }
        all_ctas();
      }
      if (rank == 0) {
        // thread t owns bins 2047 - 2t and 2046 - 2t, counted from the top (1024 threads, 2048 bins)
        const int h0 = (int)hist[2047 - 2 * t], h1 = (int)hist[2046 - 2 * t];
        int all;
        const int above = block_exclusive_scan<int, kSelThreads>(h0 + h1, scan_buf, &all);
        if (above < left && above + h0 + h1 >= left) {
          const bool second = above + h0 < left;
          s_left = left - above - (second ? h0 : 0);
          s_prefix = pre | ((uint32_t)(second ? 2046 - 2 * t : 2047 - 2 * t) << shift);
        }
      }
      all_ctas();
      if constexpr (kCluster > 1) {
        pre = *cl.map_shared_rank(&s_prefix, 0);
        left = *cl.map_shared_rank(&s_left, 0);
      } else {
        pre = s_prefix;
        left = s_left;
      }
    }
  } else {
    __syncthreads();
  }
  const uint32_t thr = pre;
  const int ties = left;
  // 2. slots in index order: warp i walks its CTA's tokens [i * run, (i + 1) * run)
  const int run = cta_run / (kSelThreads / 32);
  const int c_lo = min(r_hi, r_lo + warp * run), c_hi = min(r_hi, c_lo + run);
  int ngt = 0, ntie = 0;
#pragma unroll 4
  for (int c0 = c_lo; c0 < c_hi; c0 += 32) {
    const int c = c0 + lane;
    const bool cand = c >= lo && c < hi && take > 0 && c < c_hi;
    const uint32_t key = cand ? key_at(c) : 0u;
    ngt += __popc(__ballot_sync(0xffffffffu, c < c_hi && (c < lo || c >= hi || (cand && key > thr))));
    ntie += __popc(__ballot_sync(0xffffffffu, cand && key == thr));
  }
  if (lane == 0) {
    warp_ties[warp] = ntie;
    warp_gt[warp] = ngt;
  }
  __syncthreads();
  int seen = 0, gt = 0;  // ties and others before this warp
  for (int i = 0; i < warp; ++i) {
    gt += warp_gt[i];
    seen += warp_ties[i];
  }
  if constexpr (kCluster > 1) {
    if (t == kSelThreads - 1) {
      cta_ties = seen + ntie;
      cta_gt = gt + ngt;
    }
    all_ctas();
    for (int i = 0; i < rank; ++i) {
      gt += *cl.map_shared_rank(&cta_gt, i);
      seen += *cl.map_shared_rank(&cta_ties, i);
    }
    all_ctas();  // no CTA leaves while another reads its counts
  }
  int out = gt + min(seen, ties);
#pragma unroll 2
  for (int c0 = c_lo; c0 < c_hi; c0 += 32) {
    const int c = c0 + lane;
    const bool cand = c >= lo && c < hi && take > 0 && c < c_hi;
    const uint32_t key = cand ? key_at(c) : 0u;
    const unsigned below = (1u << lane) - 1u;
    const unsigned tie = __ballot_sync(0xffffffffu, cand && key == thr);
    const bool keep = c < c_hi && (c < lo || c >= hi ||
                                   (cand && (key > thr || (key == thr && seen + __popc(tie & below) < ties))));
    const unsigned km = __ballot_sync(0xffffffffu, keep);
    if (keep) {
      const int slot = out + __popc(km & below);
      kept[slot] = c;
      if (wout) wout[slot] = weight_at(c);
    }
    out += __popc(km);
    seen += __popc(tie);
  }
}

// Grid (slot groups, B * Hkv).  2 * dv threads move one slot: the first dv
// its k row, the others its v row, one V (16 bytes, or one element) each;
// kGatherUnroll slots a thread, all their loads before the stores.  Strides in
// V units.
template <typename V>
__global__ void __launch_bounds__(kGatherThreads) evict_gather_kernel(EvictArgs a, int dv, int rows) {
  const int spb = kGatherThreads / (2 * dv);  // slots a step
  const int t = threadIdx.x, s = t / (2 * dv), e = t % (2 * dv);
  cudaGridDependencySynchronize();  // set up beside the selection, whose slots it moves
  if (s >= spb) return;
  const bool isv = e >= dv;
  const int d = isv ? e - dv : e;
  const int b = blockIdx.y / a.Hkv, g = blockIdx.y % a.Hkv;
  const int new_len = min(evict_len(a, b), a.budget);
  const int32_t* kept = a.kept + ((long long)b * a.Hw + (a.Hw > 1 ? g : 0)) * a.budget;
  const long long* st = isv ? a.vs : a.ks;
  const long long* ot = isv ? a.vos : a.kos;
  const V* src = reinterpret_cast<const V*>(isv ? a.v : a.k) + g * st[2] + d * st[3];
  V* dst = reinterpret_cast<V*>(isv ? a.vo : a.ko) + b * ot[0] + g * ot[2] + d * ot[3];
  const int j0 = blockIdx.x * spb * kGatherUnroll + s;
  int c[kGatherUnroll], page[kGatherUnroll];
#pragma unroll
  for (int i = 0; i < kGatherUnroll; ++i) {
    const int j = j0 + i * spb;
    c[i] = j < new_len ? kept[j] : -1;
  }
#pragma unroll
  for (int i = 0; i < kGatherUnroll; ++i) {
    page[i] = c[i] < 0 ? -1 : a.pg.page(b, a.pg.page_index(c[i]));
  }
  V v[kGatherUnroll];
#pragma unroll
  for (int i = 0; i < kGatherUnroll; ++i) {
    v[i] = V{};
    if (c[i] < 0) continue;
    if (page[i] >= 0 && page[i] < a.pg.num_pages)
      v[i] = src[page[i] * st[0] + (long long)a.pg.slot(c[i]) * st[1]];
    else if (d == 0)
      atomicOr(a.page_error, 1u);
  }
#pragma unroll
  for (int i = 0; i < kGatherUnroll; ++i) {
    const int j = j0 + i * spb;
    if (j < new_len || (a.zero_tail && j < rows)) dst[j * ot[1]] = v[i];
  }
}

int esize(int dtype) { return dtype == KVBM_F64 ? 8 : dtype == KVBM_F32 ? 4 : 2; }

template <int kCluster>
int launch_select(const EvictArgs& a, cudaStream_t s) {
  auto kern = evict_select_kernel<kCluster>;
  const long long per = ((long long)a.Lmax + kCluster * kSelThreads - 1) / (kCluster * kSelThreads) * kSelThreads;
  const int keys = (int)(per < kSmemKeys ? per : kSmemKeys);
  if (allow_smem(kern, kSmemKeys * sizeof(float)) != KVBM_OK) return KVBM_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * a.Hw * kCluster));
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = keys * sizeof(float);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kCluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, a, keys) == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
}

template <typename V>
int launch_gather(EvictArgs a, int es, cudaStream_t s) {
  const int per = (int)sizeof(V) / es;
  if (per > 1)
    for (int i = 0; i < 4; ++i) {
      a.ks[i] = i == 3 ? 1 : a.ks[i] / per;
      a.vs[i] = i == 3 ? 1 : a.vs[i] / per;
      a.kos[i] = i == 3 ? 1 : a.kos[i] / per;
      a.vos[i] = i == 3 ? 1 : a.vos[i] / per;
    }
  const int dv = a.D / per;
  const int rows = a.zero_tail ? a.capacity : a.budget;
  const int per_block = kGatherThreads / (2 * dv) * kGatherUnroll;
  const long long blocks = ((long long)rows + per_block - 1) / per_block;
  return launch_dependent(evict_gather_kernel<V>, dim3((unsigned)blocks, (unsigned)(a.B * a.Hkv)), kGatherThreads, s, a,
                          dv, rows);
}

bool vec16(const void* p, const int64_t* st, int es) {
  return st[3] == 1 && (uintptr_t)p % 16 == 0 && st[0] * es % 16 == 0 && st[1] * es % 16 == 0 && st[2] * es % 16 == 0;
}

int check(const kvbm_evict_args* e) {
  if (e == nullptr) return KVBM_ERR_NULL;
  if (e->dtype < KVBM_F32 || e->dtype > KVBM_F64) return KVBM_ERR_DTYPE;
  if (e->B < 1 || e->Hkv < 1 || e->D < 1 || e->num_pages < 1 || e->page_size < 1 || e->max_pages < 1)
    return KVBM_ERR_SHAPE;
  if (e->D > 256) return KVBM_ERR_HEAD_DIM;
  if ((long long)e->B * e->Hkv > 65535) return KVBM_ERR_SHAPE;
  if ((long long)e->max_pages * e->page_size > kMaxN) return KVBM_ERR_SHAPE;
  if (e->weight_heads != 1 && e->weight_heads != e->Hkv) return KVBM_ERR_SHAPE;
  if (e->block_table == nullptr && (long long)e->B * e->max_pages > e->num_pages) return KVBM_ERR_SHAPE;
  if (e->n_sinks < 0 || e->recency < 0 || e->budget < 1 || (long long)e->n_sinks + e->recency > e->budget)
    return KVBM_ERR_SHAPE;
  if (e->capacity < e->budget || e->capacity > kMaxN) return KVBM_ERR_SHAPE;
  for (int i = 0; i < 4; ++i)
    if (e->k_stride[i] < 0 || e->v_stride[i] < 0 || e->k_out_stride[i] < 0 || e->v_out_stride[i] < 0)
      return KVBM_ERR_SHAPE;
  if (!e->k_cache || !e->v_cache || !e->seq_lens || !e->weights || !e->k_out || !e->v_out || !e->seq_lens_out ||
      !e->kept_out)
    return KVBM_ERR_NULL;
  return KVBM_OK;
}

}  // namespace
}  // namespace kvbm

using namespace kvbm;

extern "C" int kvbm_validate_evict(const kvbm_evict_args* e) { return check(e); }

extern "C" int kvbm_evict_cache(const kvbm_evict_args* e, void* stream) {
  const int st = check(e);
  if (st != KVBM_OK) return st;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return KVBM_ERR_CUDA;
  }
  if (attention_device_kind(dev) != 1) return KVBM_ERR_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  EvictArgs a;
  a.pg = paged_view(e->block_table, e->block_table_stride, e->num_pages, e->page_size, e->max_pages);
  a.k = static_cast<const char*>(e->k_cache);
  a.v = static_cast<const char*>(e->v_cache);
  a.ko = static_cast<char*>(e->k_out);
  a.vo = static_cast<char*>(e->v_out);
  for (int i = 0; i < 4; ++i) {
    a.ks[i] = e->k_stride[i];
    a.vs[i] = e->v_stride[i];
    a.kos[i] = e->k_out_stride[i];
    a.vos[i] = e->v_out_stride[i];
  }
  a.B = e->B;
  a.Hkv = e->Hkv;
  a.Hw = e->weight_heads;
  a.D = e->D;
  a.Lmax = e->max_pages * e->page_size;
  a.lens = e->seq_lens;
  a.w = e->weights;
  a.wb = e->weights_bstride;
  a.wh = e->weights_hstride;
  a.budget = e->budget;
  a.n_sinks = e->n_sinks;
  a.recency = e->recency;
  a.capacity = e->capacity;
  a.zero_tail = e->zero_tail;
  a.lens_out = e->seq_lens_out;
  a.kept = e->kept_out;
  a.wout = e->weights_out;
  a.page_error = attention_page_error_word();
  if (a.page_error == nullptr) return KVBM_ERR_CUDA;
  // CTAs per row: as many as fill the SMs, while each has a few thousand keys
  const int rows = a.B * a.Hw, sms = attention_device_sms(dev);
  int cluster = 1;
  while (cluster < 8 && rows * cluster * 2 <= sms && a.Lmax >= cluster * 4096) cluster *= 2;
  const int st2 = cluster == 1   ? launch_select<1>(a, s)
                  : cluster == 2 ? launch_select<2>(a, s)
                  : cluster == 4 ? launch_select<4>(a, s)
                                 : launch_select<8>(a, s);
  if (st2 != KVBM_OK) return st2;
  const int es = esize(e->dtype);
  if ((a.D * es) % 16 == 0 && vec16(e->k_cache, e->k_stride, es) && vec16(e->v_cache, e->v_stride, es) &&
      vec16(e->k_out, e->k_out_stride, es) && vec16(e->v_out, e->v_out_stride, es))
    return launch_gather<uint4>(a, es, s);
  if (es == 8) return launch_gather<unsigned long long>(a, es, s);
  if (es == 4) return launch_gather<unsigned int>(a, es, s);
  return launch_gather<unsigned short>(a, es, s);
}
