// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, weight head): the first n_sinks tokens, the last `recency`
// tokens and, of those between, the budget - n_sinks - recency with the
// highest weights stay (equal weights: the lower index; NaN counts as -inf).
// Kept tokens keep their order.
//
// Two kernels.  evict_select_kernel finds the threshold weight with a radix
// select (most significant byte first) over order-preserving 32-bit keys and
// turns the choice into slots with one scan: 4 * len bytes of weights are all
// it reads from DRAM.  evict_gather_kernel moves the kept k and v rows, 16
// bytes a thread: 4 * budget * D elements a head, bound by DRAM.
#include <cuda_runtime.h>

#include "kvbm_attention.cuh"

namespace kvbm {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kGatherThreads = 256;
constexpr int kGatherUnroll = 4;

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

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictArgs a) {
  __shared__ unsigned int hist[256];
  __shared__ int scan_buf[kSelThreads / 32];
  __shared__ unsigned int s_prefix;
  __shared__ int s_left;
  const int row = blockIdx.x, b = row / a.Hw, hw = row % a.Hw, t = threadIdx.x;
  const int len = evict_len(a, b);
  const float* w = a.w + b * a.wb + hw * a.wh;
  int32_t* kept = a.kept + (long long)row * a.budget;
  float* wout = a.wout ? a.wout + (long long)row * a.budget : nullptr;
  const int new_len = min(len, a.budget);
  if (hw == 0 && t == 0) a.lens_out[b] = new_len;
  for (int j = new_len + t; j < a.budget; j += kSelThreads) {
    kept[j] = -1;
    if (wout) wout[j] = 0.f;
  }
  if (len <= a.budget) {
    for (int j = t; j < len; j += kSelThreads) {
      kept[j] = j;
      if (wout) wout[j] = w[j];
    }
    return;
  }
  const int lo = a.n_sinks, hi = len - a.recency;  // the candidates; budget >= n_sinks + recency, so lo <= hi
  const int take = a.budget - a.n_sinks - a.recency;
  // 1. threshold key of the `take` highest candidates, and how many of its
  //    ties are taken (from the lowest index)
  if (t == 0) {
    s_prefix = 0;
    s_left = take;
  }
  __syncthreads();
  if (take > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = t; i < 256; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t pre = s_prefix, high = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int c = lo + t; c < hi; c += kSelThreads) {
        const uint32_t key = weight_key(w[c]);
        if (((key ^ pre) & high) == 0) atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (t < 32) {
        // lane l owns bins [248 - 8l, 256 - 8l), counted from the top
        const int left = s_left;
        int mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mine += hist[255 - 8 * t - j];
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, o);
          if (t >= o) incl += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, incl >= left);
        if (t == __ffs(hit) - 1) {
          int above = incl - mine, v = 255 - 8 * t;
          for (int j = 0; j < 7 && above + (int)hist[v] < left; ++j, --v) above += hist[v];
          s_left = left - above;
          s_prefix = pre | ((uint32_t)v << shift);
        }
      }
      __syncthreads();
    }
  }
  const uint32_t thr = s_prefix;
  const int ties = s_left;
  // 2. slots in index order
  int out = 0, seen = 0;  // kept before this chunk, ties met before it
  for (int base = 0; base < len; base += kSelThreads) {
    const int c = base + t;
    const bool cand = c >= lo && c < hi && take > 0;
    float wc = c < len ? w[c] : 0.f;
    const uint32_t key = cand ? weight_key(wc) : 0u;
    const bool tie = cand && key == thr;
    int ntie = 0, nkeep = 0;
    const int before = seen + block_exclusive_scan<int, kSelThreads>(tie ? 1 : 0, scan_buf, &ntie);
    const bool keep = c < len && (c < lo || c >= hi || (cand && (key > thr || (tie && before < ties))));
    const int slot = out + block_exclusive_scan<int, kSelThreads>(keep ? 1 : 0, scan_buf, &nkeep);
    if (keep) {
      kept[slot] = c;
      if (wout) wout[slot] = wc;
    }
    out += nkeep;
    seen += ntie;
  }
}

// One thread moves one V (16 bytes, or one element) of the k and of the v row
// of one slot; strides in V units.
template <typename V>
__global__ void __launch_bounds__(kGatherThreads) evict_gather_kernel(EvictArgs a, int dv) {
  const int rpb = kGatherThreads / dv;
  const int t = threadIdx.x;
  if (t >= rpb * dv) return;
  const int d = t % dv;
  const long long rows = (long long)a.B * a.capacity * a.Hkv, step = (long long)gridDim.x * rpb;
  const V *k = reinterpret_cast<const V*>(a.k), *v = reinterpret_cast<const V*>(a.v);
  V *ko = reinterpret_cast<V*>(a.ko), *vo = reinterpret_cast<V*>(a.vo);
  for (long long r0 = (long long)blockIdx.x * rpb + t / dv; r0 < rows; r0 += kGatherUnroll * step) {
    V kv[kGatherUnroll], vv[kGatherUnroll];
    long long dk[kGatherUnroll], dvv[kGatherUnroll];
    bool put[kGatherUnroll];
#pragma unroll
    for (int i = 0; i < kGatherUnroll; ++i) {
      const long long r = r0 + i * step;
      kv[i] = V{};
      vv[i] = V{};
      put[i] = false;
      if (r >= rows) continue;
      const int g = (int)(r % a.Hkv);
      const long long bj = r / a.Hkv;
      const int j = (int)(bj % a.capacity), b = (int)(bj / a.capacity);
      dk[i] = b * a.kos[0] + j * a.kos[1] + g * a.kos[2] + d * a.kos[3];
      dvv[i] = b * a.vos[0] + j * a.vos[1] + g * a.vos[2] + d * a.vos[3];
      if (j >= min(evict_len(a, b), a.budget)) {
        put[i] = a.zero_tail != 0;
        continue;
      }
      put[i] = true;
      const int c = a.kept[((long long)b * a.Hw + (a.Hw > 1 ? g : 0)) * a.budget + j];
      const int pi = c / a.pg.page_size;
      const int page = a.pg.table ? a.pg.table[b * a.pg.ts + pi] : b * a.pg.max_pages + pi;
      if (page >= 0 && page < a.pg.num_pages) {
        const long long in = c - pi * a.pg.page_size;
        kv[i] = k[page * a.ks[0] + in * a.ks[1] + g * a.ks[2] + d * a.ks[3]];
        vv[i] = v[page * a.vs[0] + in * a.vs[1] + g * a.vs[2] + d * a.vs[3]];
      } else if (d == 0) {
        atomicOr(a.page_error, 1u);
      }
    }
#pragma unroll
    for (int i = 0; i < kGatherUnroll; ++i) {
      if (!put[i]) continue;
      ko[dk[i]] = kv[i];
      vo[dvv[i]] = vv[i];
    }
  }
}

int esize(int dtype) { return dtype == KVBM_F64 ? 8 : dtype == KVBM_F32 ? 4 : 2; }

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
  const long long rows = (long long)a.B * (a.zero_tail ? a.capacity : a.budget) * a.Hkv;
  const int rpb = kGatherThreads / dv;
  long long blocks = (rows + rpb - 1) / rpb;
  if (blocks > 148LL * 8) blocks = 148LL * 8;
  evict_gather_kernel<V><<<(unsigned)blocks, kGatherThreads, 0, s>>>(a, dv);
  return cudaGetLastError() == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
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
  a.pg = PagedView{e->block_table, e->block_table_stride, e->num_pages, e->page_size, e->max_pages};
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
  evict_select_kernel<<<(unsigned)(a.B * a.Hw), kSelThreads, 0, s>>>(a);
  if (cudaGetLastError() != cudaSuccess) return KVBM_ERR_CUDA;
  const int es = esize(e->dtype);
  if ((a.D * es) % 16 == 0 && vec16(e->k_cache, e->k_stride, es) && vec16(e->v_cache, e->v_stride, es) &&
      vec16(e->k_out, e->k_out_stride, es) && vec16(e->v_out, e->v_out_stride, es))
    return launch_gather<uint4>(a, es, s);
  if (es == 8) return launch_gather<unsigned long long>(a, es, s);
  if (es == 4) return launch_gather<unsigned int>(a, es, s);
  return launch_gather<unsigned short>(a, es, s);
}
