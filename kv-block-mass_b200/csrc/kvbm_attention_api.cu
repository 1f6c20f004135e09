// C ABI of the attention entry points (include/kvbm.h): argument checks,
// kernel choice, workspace layout and the launch sequence.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "kvbm_attention.cuh"

namespace kvbm {
namespace {

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

bool dtype_ok(int dtype) { return dtype == KVBM_F32 || dtype == KVBM_BF16 || dtype == KVBM_F16; }

// The kernels take the scale in float32 (below its smallest value: 0).
bool scale_ok(double scale) {
  const float f = (float)scale;
  return f - f == 0.f;  // neither NaN nor infinite
}

int check_prompt(const kvbm_attention_args* p) {
  if (p == nullptr) return KVBM_ERR_NULL;
  if (!dtype_ok(p->dtype)) return KVBM_ERR_DTYPE;
  if (p->B < 1 || p->Hq < 1 || p->Hkv < 1 || p->N < 1 || p->D < 1) return KVBM_ERR_SHAPE;
  if (p->Hq % p->Hkv != 0) return KVBM_ERR_GQA;
  if (p->D > 256) return KVBM_ERR_HEAD_DIM;
  if ((long long)p->B * p->Hq > 65535 || p->N > kMaxN) return KVBM_ERR_SHAPE;
  if (p->seq_lens != nullptr && p->cu_seqlens != nullptr) return KVBM_ERR_SHAPE;
  if (p->cu_seqlens != nullptr && (p->total_tokens < 0 || p->total_tokens > kMaxN)) return KVBM_ERR_SHAPE;
  for (int i = 0; i < 4; ++i)
    if (p->q_stride[i] < 0 || p->k_stride[i] < 0 || p->v_stride[i] < 0 || p->out_stride[i] < 0) return KVBM_ERR_SHAPE;
  for (int i = 0; i < 3; ++i)
    if (p->lse_stride[i] < 0) return KVBM_ERR_SHAPE;
  if (!scale_ok(p->scale)) return KVBM_ERR_SHAPE;
  const bool no_rows = p->cu_seqlens != nullptr && p->total_tokens == 0;  // an empty tensor's pointer may be NULL
  if (!no_rows && !(p->q && p->k && p->v && p->out && p->lse)) return KVBM_ERR_NULL;
  return KVBM_OK;
}

PromptArgs prompt_args(const kvbm_attention_args* p) {
  PromptArgs a;
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.out = p->out;
  a.lse = p->lse;
  for (int i = 0; i < 4; ++i) {
    a.qs[i] = p->q_stride[i];
    a.ks[i] = p->k_stride[i];
    a.vs[i] = p->v_stride[i];
    a.os[i] = p->out_stride[i];
  }
  for (int i = 0; i < 3; ++i) a.ls[i] = p->lse_stride[i];
  a.B = p->B;
  a.Hq = p->Hq;
  a.Hkv = p->Hkv;
  a.G = p->Hq / p->Hkv;
  a.N = p->N;
  a.D = p->D;
  a.kmask = p->key_mask;
  a.kmb = p->key_mask_bstride;
  a.causal = p->causal != 0;
  a.scale = (float)p->scale;
  a.lens = p->seq_lens;
  a.cu = p->cu_seqlens;
  a.total = p->total_tokens;
  a.fill = p->fill_outside != 0;
  return a;
}

int check_cached(const kvbm_cached_args* p) {
  if (p == nullptr) return KVBM_ERR_NULL;
  if (!dtype_ok(p->dtype)) return KVBM_ERR_DTYPE;
  if (p->B < 1 || p->Hq < 1 || p->Hkv < 1 || p->T < 1 || p->D < 1 || p->num_pages < 1 || p->page_size < 1 ||
      p->max_pages < 1)
    return KVBM_ERR_SHAPE;
  if (p->Hq % p->Hkv != 0) return KVBM_ERR_GQA;
  if (p->D > 256) return KVBM_ERR_HEAD_DIM;
  if (p->T > kMaxTreeTokens) return KVBM_ERR_SHAPE;
  if ((long long)p->B * p->Hq > 65535) return KVBM_ERR_SHAPE;
  if ((long long)p->max_pages * p->page_size > kMaxN) return KVBM_ERR_SHAPE;
  if (p->block_table == nullptr && (long long)p->B * p->max_pages > p->num_pages) return KVBM_ERR_SHAPE;
  for (int i = 0; i < 4; ++i)
    if (p->q_stride[i] < 0 || p->k_stride[i] < 0 || p->v_stride[i] < 0 || p->out_stride[i] < 0) return KVBM_ERR_SHAPE;
  for (int i = 0; i < 3; ++i)
    if (p->lse_stride[i] < 0) return KVBM_ERR_SHAPE;
  if (!scale_ok(p->scale)) return KVBM_ERR_SHAPE;
  if ((p->weights != nullptr) != (p->weights_out != nullptr)) return KVBM_ERR_NULL;
  if (p->weights != nullptr && p->T != 1) return KVBM_ERR_SHAPE;
  if (!p->q || !p->k_cache || !p->v_cache || !p->seq_lens || !p->out || !p->lse) return KVBM_ERR_NULL;
  return KVBM_OK;
}

// The mma.sync kernel reads rows in 16-byte pieces.
bool cached_mma_supported(const kvbm_cached_args* p) {
  if (p->dtype == KVBM_F32 || p->D % 8 != 0) return false;
  auto rows16 = [](const void* base, const int64_t* st) {
    return (uintptr_t)base % 16 == 0 && st[3] == 1 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0;
  };
  return rows16(p->q, p->q_stride) && rows16(p->k_cache, p->k_stride) && rows16(p->v_cache, p->v_stride) &&
         rows16(p->out, p->out_stride);
}

// Rows up to which the mma.sync kernel runs.
constexpr int kMmaRows = 32;

struct CachedPlan {
  CachedArgs a;
  int kernel = 0;  // 0: FFMA tiles, 1: mma.sync (16 rows a tile), 2: tcgen05 (128 or 256)
  size_t part_o = 0, part_ml = 0, stats = 0, scores = 0, total = 0;
};

// CTAs, tiles and workspace of a cached call on a device of `sms` SMs.
void plan_cached(const kvbm_cached_args* p, int sms, CachedPlan* pl) {
  CachedArgs& a = pl->a;
  a = CachedArgs{};
  a.q = p->q;
  a.k = p->k_cache;
  a.v = p->v_cache;
  a.out = p->out;
  a.lse = p->lse;
  for (int i = 0; i < 4; ++i) {
    a.qs[i] = p->q_stride[i];
    a.ks[i] = p->k_stride[i];
    a.vs[i] = p->v_stride[i];
    a.os[i] = p->out_stride[i];
  }
  for (int i = 0; i < 3; ++i) a.ls[i] = p->lse_stride[i];
  a.pg = paged_view(p->block_table, p->block_table_stride, p->num_pages, p->page_size, p->max_pages);
  a.B = p->B;
  a.Hq = p->Hq;
  a.Hkv = p->Hkv;
  a.G = p->Hq / p->Hkv;
  a.T = p->T;
  a.D = p->D;
  a.R = a.G * a.T;
  a.Lmax = p->max_pages * p->page_size;
  a.lens = p->seq_lens;
  a.tree = p->tree_mask;
  a.tb = p->tree_mask_bstride;
  a.tr = p->tree_mask_rstride;
  a.off = p->log_offsets;
  a.ob = p->log_offsets_bstride;
  a.oh = p->log_offsets_hstride;
  a.scale = (float)p->scale;
  a.w = p->weights;
  a.wb = p->weights_bstride;
  a.wh = p->weights_hstride;
  a.wout = p->weights_out;
  a.wob = p->weights_out_bstride;
  a.woh = p->weights_out_hstride;
  a.DP = a.D <= 64 ? 64 : a.D <= 128 ? 128 : 256;
  // 16-bit types: up to 32 rows, mma.sync, which reads the cache once per 16
  // rows; above, tcgen05, whose tiles of 128 rows cost a 16-row unit eight
  // times its tensor work.
  pl->kernel = !cached_mma_supported(p) ? 0 : (a.R > kMmaRows && a.D <= 128 && a.w == nullptr && tc_scale(a.scale)) ? 2 : 1;
  a.BM = pl->kernel == 2 ? (a.R > 128 ? 256 : 128) : pl->kernel == 1 || a.R <= 16 ? 16 : 64;
  a.KT = pl->kernel == 2 ? 128 : kCachedKeyTile;
  a.RT = (a.R + a.BM - 1) / a.BM;
  // no more CTAs than key tiles of full-length sequences
  const long long tiles = (long long)a.B * a.Hkv * a.RT * ((a.Lmax + a.KT - 1) / a.KT);
  const int per_sm = pl->kernel == 2 ? 1 : pl->kernel == 1 && a.DP <= 128 ? kMmaCtas : 2;
  a.C = (int)std::min<long long>(tiles, (long long)sms * per_sm);
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o = align256(o + bytes);
    return at;
  };
  pl->part_o = take((size_t)a.C * 2 * a.BM * a.DP * sizeof(float));
  pl->part_ml = take((size_t)a.C * 2 * a.BM * sizeof(float2));
  if (a.w != nullptr) {
    pl->stats = take((size_t)a.B * a.Hkv * a.R * sizeof(float2));
    pl->scores = take((size_t)a.B * a.Hq * a.Lmax * sizeof(float));
  }
  pl->total = o;
}

constexpr int kMostSms = 160;  // sizes a workspace where the device is unknown

int this_device(int* dev) {
  if (cudaGetDevice(dev) != cudaSuccess) {
    cudaGetLastError();
    *dev = -1;
    return KVBM_ERR_CUDA;
  }
  return KVBM_OK;
}

}  // namespace

int allow_smem_of(const void* kernel, size_t bytes) {
  // the last (kernel, device) pair set in each slot; two that share one only set it again
  constexpr int kSlots = 256;
  static std::atomic<uintptr_t> done[kSlots] = {};
  int dev = -1;
  if (this_device(&dev) != KVBM_OK) return KVBM_ERR_CUDA;
  const uintptr_t key = (uintptr_t)kernel * 64 + (uintptr_t)dev + 1;
  const int at = (int)((key * 0x9E3779B97F4A7C15ull) >> 56);
  if (dev < 63 && done[at].load(std::memory_order_acquire) == key) return KVBM_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) {
    cudaGetLastError();
    return KVBM_ERR_CUDA;
  }
  if (dev < 63) done[at].store(key, std::memory_order_release);
  return KVBM_OK;
}

}  // namespace kvbm

using namespace kvbm;

extern "C" int kvbm_validate_attention(const kvbm_attention_args* p) { return check_prompt(p); }

extern "C" int kvbm_attention(const kvbm_attention_args* p, void* stream) {
  const int st = check_prompt(p);
  if (st != KVBM_OK) return st;
  int dev = -1;
  if (this_device(&dev) != KVBM_OK) return KVBM_ERR_CUDA;
  if (attention_device_kind(dev) != 1) return KVBM_ERR_DEVICE;
  const PromptArgs a = prompt_args(p);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.cu != nullptr && a.total == 0) return KVBM_OK;
  if (prompt_tc_supported(a, p->dtype)) return launch_prompt_tc(a, p->dtype, s);
  if (a.fill && a.cu != nullptr) {
    const int f = launch_prompt_fill(a, p->dtype, s);
    if (f != KVBM_OK) return f;
  }
  return launch_prompt_simt(a, p->dtype, s);
}

extern "C" int kvbm_validate_cached_attention(const kvbm_cached_args* p) { return check_cached(p); }

extern "C" size_t kvbm_cached_attention_workspace_bytes(const kvbm_cached_args* p) {
  if (check_cached(p) != KVBM_OK) return 0;
  int dev = -1;
  this_device(&dev);
  const int sms = attention_device_sms(dev);
  CachedPlan pl;
  plan_cached(p, sms > 0 ? sms : kMostSms, &pl);
  return pl.total;
}

extern "C" int kvbm_cached_attention(const kvbm_cached_args* p, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  int st = check_cached(p);
  if (st != KVBM_OK) return st;
  int dev = -1;
  if (this_device(&dev) != KVBM_OK) return KVBM_ERR_CUDA;
  if (attention_device_kind(dev) != 1) return KVBM_ERR_DEVICE;
  CachedPlan pl;
  plan_cached(p, attention_device_sms(dev), &pl);
  if (workspace == nullptr || workspace_bytes < pl.total || (uintptr_t)workspace % 256 != 0) return KVBM_ERR_WORKSPACE;
  char* w = static_cast<char*>(workspace);
  CachedArgs& a = pl.a;
  a.part_o = reinterpret_cast<float*>(w + pl.part_o);
  a.part_ml = reinterpret_cast<float2*>(w + pl.part_ml);
  if (a.w != nullptr) {
    a.stats = reinterpret_cast<float2*>(w + pl.stats);
    a.scores = reinterpret_cast<float*>(w + pl.scores);
  }
  a.page_error = attention_page_error_word();
  if (a.page_error == nullptr) return KVBM_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = pl.kernel == 2   ? launch_cached_tc(a, p->dtype, s)
       : pl.kernel == 1 ? launch_cached_mma(a, p->dtype, s)
                        : launch_cached_simt(a, p->dtype, s);
  if (st != KVBM_OK) return st;
  st = launch_cached_merge(a, p->dtype, s);
  if (st != KVBM_OK) return st;
  return a.w != nullptr ? launch_cached_weights(a, s) : KVBM_OK;
}
