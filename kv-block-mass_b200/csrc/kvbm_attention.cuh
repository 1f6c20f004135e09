// Arguments and device helpers shared by the attention kernels (prompt
// attention, attention over a paged cache) and the cache eviction.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kvbm.h"
#include "kvbm_internal.cuh"

namespace kvbm {

constexpr float kLog2eF = 1.44269504088896340736f;
constexpr float kLn2F = 0.69314718055994530942f;
// Drafted tokens of one cached call: a row of the tree mask fits a 64-bit word.
constexpr int kMaxTreeTokens = 64;

// Keys of one tile of the cache kernels.
constexpr int kCachedKeyTile = 64;
// CTAs an SM of the mma.sync cache kernel (D <= 128).
constexpr int kMmaCtas = 3;

// Prompt attention as the kernels see it (strides in elements, dims [B, H, N, D]).
struct PromptArgs {
  const void *q, *k, *v;
  long long qs[4], ks[4], vs[4];
  int B, Hq, Hkv, G, N, D;
  const uint8_t* kmask;  // [B|1, N] or null
  long long kmb;
  int causal;
  float scale;
  const int32_t* lens;  // [B] or null
  const int32_t* cu;    // [B + 1] or null
  long long total;
  int fill;             // 1: rows past a sequence's end get out 0, lse -inf
  void* out;
  long long os[4];
  float* lse;
  long long ls[3];
};

// A paged cache: row c of sequence b is slot c % page_size of page
// table[b * ts + c / page_size] (table == null: page b * max_pages + c / page_size).
struct PagedView {
  const int32_t* table;
  long long ts;
  int num_pages, page_size, max_pages;
  int shift;  // log2(page_size), or -1: integer divisions cost the page lookups more than their loads do
  // Page index and slot of row c.
  __device__ __forceinline__ int page_index(int c) const { return shift >= 0 ? c >> shift : c / page_size; }
  __device__ __forceinline__ int slot(int c) const { return shift >= 0 ? c & (page_size - 1) : c % page_size; }
  // Page id of page index pi of sequence b.
  __device__ __forceinline__ int page(int b, int pi) const { return table ? table[b * ts + pi] : b * max_pages + pi; }
};

inline PagedView paged_view(const int32_t* table, long long ts, int num_pages, int page_size, int max_pages) {
  int shift = -1;
  for (int i = 0; i < 31; ++i)
    if (page_size == 1 << i) shift = i;
  return PagedView{table, ts, num_pages, page_size, max_pages, shift};
}

// Attention over a cache: unit (b, g) has R = G * T rows, row r = hh * T + t.
struct CachedArgs {
  const void *q, *k, *v;
  long long qs[4];          // [B, Hq, T, D]
  long long ks[4], vs[4];   // [num_pages, page_size, Hkv, D]
  PagedView pg;
  int B, Hq, Hkv, G, T, D, R;
  int Lmax;                 // max_pages * page_size
  const int32_t* lens;
  const uint8_t* tree;      // [B|1, T, T] or null (u <= t)
  long long tb, tr;
  const float* off;         // [B|1, Hkv|1, Lmax] or null
  long long ob, oh;
  float scale;
  void* out;
  long long os[4];
  float* lse;
  long long ls[3];
  // weights (T == 1)
  const float* w;
  long long wb, wh;
  float* wout;
  long long wob, woh;
  // scratch
  float* scores;            // [B * Hkv, G, Lmax] or null
  float2* stats;            // [B * Hkv, R]: (max, 1 / sum) per row
  float* part_o;            // [C][2][BM][DP] unnormalised outputs of split units
  float2* part_ml;          // [C][2][BM]
  int C;                    // CTAs of the split kernel
  int BM, RT, KT, DP;       // rows per row tile, row tiles, keys per tile, padded D
  unsigned int* page_error; // set when a table entry is no page
};

// Length of sequence b, inside the table.
__device__ __forceinline__ int cached_len(const CachedArgs& a, int b) {
  const int n = a.lens[b];
  return n < 0 ? 0 : (n < a.Lmax ? n : a.Lmax);
}

// First CTA-linear tile of CTA i, and the CTA that holds tile t, when `total`
// tiles are cut into C ranges [i * total / C, (i + 1) * total / C).
// (32-bit divisions where the products fit: a 64-bit one is 100 instructions.)
__device__ __forceinline__ long long split_begin(long long i, long long total, long long C) {
  const long long p = i * total;
  return p < (1ll << 32) ? (long long)((uint32_t)p / (uint32_t)C) : p / C;
}
__device__ __forceinline__ long long split_owner(long long t, long long total, long long C) {
  const long long p = (t + 1) * C + total - 1;
  return (p < (1ll << 32) ? (long long)((uint32_t)p / (uint32_t)total) : p / total) - 1;
}

// Key tiles of sequences [0, b) (times units per sequence) by one warp:
// prefix of b, and the total over all B.
__device__ __forceinline__ void warp_tile_prefix(const CachedArgs& a, int b_end, long long* prefix, long long* total) {
  const int lane = threadIdx.x & 31;
  long long pre = 0, all = 0;
  for (int b = lane; b < a.B; b += 32) {
    const long long n = (cached_len(a, b) + a.KT - 1) / a.KT;
    all += n;
    if (b < b_end) pre += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    pre += __shfl_xor_sync(0xffffffffu, pre, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  const long long per = (long long)a.Hkv * a.RT;
  *prefix = pre * per;
  *total = all * per;
}

// The sequence that holds linear tile t: first b with prefix(b + 1) > t, and prefix(b).  One warp.
__device__ __forceinline__ int warp_find_seq(const CachedArgs& a, long long t, long long* first) {
  const int lane = threadIdx.x & 31;
  const long long per = (long long)a.Hkv * a.RT;
  long long carry = 0;
  for (int base = 0; base < a.B; base += 32) {
    const int b = base + lane;
    const long long n = b < a.B ? (long long)((cached_len(a, b) + a.KT - 1) / a.KT) * per : 0;
    long long incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, carry + incl > t);
    if (hit) {
      const int l = __ffs(hit) - 1;
      *first = carry + __shfl_sync(0xffffffffu, incl - n, l);
      return base + l;
    }
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  *first = carry;
  return a.B;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// The non-finite v elements of drafted tokens [lo, hi) that token `tok` keeps,
// added to four output columns from d (the matrix products took them as zeros).
template <typename T>
__device__ __noinline__ void add_nonfinite(const CachedArgs& a, int b, int g, int tok, int lo, int hi, int pre,
                                                 int d, float4& acc) {
  const uint8_t* tree = a.tree ? a.tree + b * a.tb : nullptr;
  const float* off = a.off ? a.off + b * a.ob + g * a.oh : nullptr;
  for (int c = lo; c < hi; ++c) {
    if (!(tree ? tree[tok * a.tr + (c - pre)] != 0 : c - pre <= tok)) continue;
    if (off != nullptr && off[c] == -INFINITY) continue;
    const int page = a.pg.page(b, a.pg.page_index(c));
    if (page < 0 || page >= a.pg.num_pages) continue;
    const T* v = static_cast<const T*>(a.v) + (long long)page * a.vs[0] + (long long)a.pg.slot(c) * a.vs[1] + g * a.vs[2];
    float* o = &acc.x;
    for (int e = 0; e < 4; ++e) {
      if (d + e >= a.D) continue;
      const float x = to_f32(v[(d + e) * a.vs[3]]);
      if (!(fabsf(x) < INFINITY)) o[e] += x;
    }
  }
}

// How far below a row's maximum (powers of two) its reference is put when the
// maximum raises it: weights of the maximum are 2^kHead.  fp16 holds 2^-14 at
// full precision, and with the growth of less than 2^8 that a reference is left
// alone for, weights of up to 2^15: the 2^7 in between goes to the small ones.
// A weight of an fp16 kernel is then rounded to 11 bits or to 2^-32 of the
// row's largest, whichever is coarser: n keys lose at most n 2^-32 of their
// values.  (Without, n 2^-25, and 131071 keys 17.5 nats below a first one lost
// the whole of their 0.3 %.)  bf16 has float32's range.
template <bool kBf16>
constexpr float kHead = kBf16 ? 0.f : 7.f;

// Scales the tcgen05 kernels take: positive (the maximum of the raw scores is
// the maximum), and finite as a factor of base-2 exponents.
inline bool tc_scale(float scale) { return scale > 0.f && scale * kLog2eF < INFINITY; }

// Launchers (kvbm_status).
int launch_prompt_simt(const PromptArgs& a, int dtype, cudaStream_t s);
int launch_prompt_fill(const PromptArgs& a, int dtype, cudaStream_t s);
bool prompt_tc_supported(const PromptArgs& a, int dtype);
int launch_prompt_tc(const PromptArgs& a, int dtype, cudaStream_t s);
int launch_cached_simt(const CachedArgs& a, int dtype, cudaStream_t s);
int launch_cached_mma(const CachedArgs& a, int dtype, cudaStream_t s);  // R <= 16 rows a tile, 16-bit types
int launch_cached_tc(const CachedArgs& a, int dtype, cudaStream_t s);   // row tiles of 128 or 256, 16-bit types, D <= 128
int launch_cached_merge(const CachedArgs& a, int dtype, cudaStream_t s);
int launch_cached_weights(const CachedArgs& a, cudaStream_t s);
// Device addresses of the error words (or null): waits that ran out in the
// prompt and the cache kernels, bad table entries (attention, eviction).
unsigned int* attention_error_word();
unsigned int* cached_error_word();
unsigned int* attention_page_error_word();

// Allows a kernel its dynamic shared memory (kvbm_attention_api.cu): set once
// per kernel and device, 4 us of a call otherwise.
int allow_smem_of(const void* kernel, size_t bytes);
template <typename K>
int allow_smem(K* kernel, size_t bytes) {
  return allow_smem_of(reinterpret_cast<const void*>(kernel), bytes);
}

// Launches a kernel that may start before the one ahead of it on the stream
// has ended (it waits for it itself, in cudaGridDependencySynchronize).
template <typename... P, typename... A>
int launch_dependent(void (*kernel)(P...), dim3 grid, unsigned threads, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? KVBM_OK : KVBM_ERR_CUDA;
}

int attention_device_kind(int dev);  // 1: sm_100
int attention_device_sms(int dev);

}  // namespace kvbm
