// Attention of the newest tokens over a quantised KV cache, and decode routing over its keys
// (semantics: include/bb_b200.h, bb_qkv_decode and bb_qkv_route).
//
//   qkv_partial_kernel  one query row (head, token) and one split of its key list: running max, sum and
//                       P.V of the split, in fp32
//   qkv_combine_kernel  merges the splits of a row
//   qkv_scores_kernel   log2 scores of every key for one query head, and per-split softmax statistics
//   qkv_pool_kernel     merged statistics, probabilities averaged over the query heads of a KV head
#include <algorithm>

#include "qkv.cuh"

namespace bb {

int topk_sorted(const float* vals, int64_t rows, int64_t n, int64_t k, void* out, bool out64, int64_t so_h,
                void* scratch, size_t scratch_bytes, cudaStream_t stream);
size_t topk_scratch_bytes(int64_t rows, int64_t n, int64_t k);

namespace {

using qkv::K_RUN;
using qkv::V_RUN;

constexpr int WARPS = 4;
constexpr float LOG2E = 1.4426950408889634f;

struct AttnParams {
  const unsigned char* kc; const uint32_t* km;
  const unsigned char* vc; const uint32_t* vm;
  int64_t kc_h, km_h, vc_h, vm_h;
  const void* q; int64_t sq_h, sq_t;
  const void* idx; int64_t si_r;
  int64_t route_k;
  int idx64, per_head;
  const int64_t* n_dev;
  int64_t n, cap, front, window;
  int d, bits, group, pairs, row_bytes, heads, kv_heads, groups, t, splits, dtype;
  float scale_log2;
  float2* part_ml;  // [heads * t][splits] (max in log2 units, sum)
  float* part_acc;  // [heads * t][splits][d]
  void* out; int64_t so_h, so_t;
  float* scores;    // [heads][cap] log2 units
  float* probs;     // [kv_heads][cap]
};

__device__ __forceinline__ int64_t cache_len(const AttnParams& p) {
  if (!p.n_dev) return p.n;
  const int64_t n = *p.n_dev;
  return n < 0 ? 0 : (n > p.cap ? p.cap : n);
}

__device__ __forceinline__ float load_elem(const void* p, int64_t i, int dtype) {
  return dtype == BB_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                          : __half2float(static_cast<const __half*>(p)[i]);
}

// The value of dimension 32 i + lane of a row.
__device__ __forceinline__ float dequant(const unsigned char* row, const uint32_t* meta, int i, int lane, int run,
                                         const AttnParams& p) {
  const int place = ((lane / run) * (p.d / 32) + i) * run + lane % run;
  const uint32_t c = p.bits == 8 ? row[place] : ((row[place >> 1] >> ((place & 1) * 4)) & 15u);
  const uint32_t m = meta[(32 * i + lane) / p.group];
  return fmaf(__uint_as_float(m << 16), (float)c, __uint_as_float(m & 0xFFFF0000u));
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// Log2 score of the key at `pos`.
__device__ __forceinline__ float key_score(const AttnParams& p, int64_t kv, int64_t pos, const float (&q)[4], int lane) {
  const unsigned char* row = p.kc + kv * p.kc_h + pos * p.row_bytes;
  const uint32_t* meta = p.km + kv * p.km_h + pos * p.pairs;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (32 * i < p.d) s = fmaf(q[i], dequant(row, meta, i, lane, K_RUN, p), s);
  return warp_sum(s) * p.scale_log2;
}

// Grid (splits, heads * t); a warp takes one key at a time, a lane every 32nd dimension.
__global__ void __launch_bounds__(32 * WARPS) qkv_partial_kernel(AttnParams p) {
  __shared__ float sm[WARPS], sl[WARPS], sacc[WARPS][128];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t row = blockIdx.y, h = row / p.t, ti = row % p.t, kv = h / p.groups;
  const int64_t n = cache_len(p);
  const int64_t seen = n - p.t + 1 + ti;  // keys up to this token's own
  float q[4], acc[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q[i] = 32 * i < p.d ? load_elem(p.q, h * p.sq_h + ti * p.sq_t + 32 * i + lane, p.dtype) : 0.f;
  float m = -INFINITY, l = 0.f;
  if (seen > 0) {
    const int64_t f = p.front < seen ? p.front : seen;
    const int64_t w0 = max(f, seen - p.window);  // window keys [w0, seen)
    const int64_t total = f + (seen - w0) + p.route_k;
    for (int64_t j = (int64_t)blockIdx.x * WARPS + warp; j < total; j += (int64_t)p.splits * WARPS) {
      int64_t pos = j < f ? j : w0 + (j - f);
      if (j >= f + (seen - w0)) {
        const int64_t o = (p.per_head ? h : kv) * p.si_r + (j - f - (seen - w0));
        pos = p.idx64 ? static_cast<const int64_t*>(p.idx)[o] : (int64_t) static_cast<const int32_t*>(p.idx)[o];
        if (pos < f || pos >= w0) continue;
      }
      const float s = key_score(p, kv, pos, q, lane);
      const float mn = fmaxf(m, s);
      const float keep = exp2f(m - mn), e = exp2f(s - mn);
      const unsigned char* vr = p.vc + kv * p.vc_h + pos * p.row_bytes;
      const uint32_t* vm = p.vm + kv * p.vm_h + pos * p.pairs;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (32 * i < p.d) acc[i] = fmaf(e, dequant(vr, vm, i, lane, V_RUN, p), acc[i] * keep);
      l = l * keep + e;
      m = mn;
    }
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sacc[warp][32 * i + lane] = acc[i];
  __syncthreads();
  float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm[w]);
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const float e = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - M);
    L = fmaf(e, sl[w], L);
    A = fmaf(e, sacc[w][threadIdx.x], A);
  }
  const int64_t at = row * p.splits + blockIdx.x;
  if (threadIdx.x == 0) p.part_ml[at] = make_float2(M, L);
  if (threadIdx.x < p.d) p.part_acc[at * p.d + threadIdx.x] = A;
}

// Grid heads * t, d threads' worth of work in 128.
__global__ void __launch_bounds__(128) qkv_combine_kernel(AttnParams p) {
  const int64_t row = blockIdx.x;
  const float2* ml = p.part_ml + row * p.splits;
  float M = -INFINITY;
  for (int s = 0; s < p.splits; ++s) M = fmaxf(M, ml[s].x);
  float L = 0.f, A = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    if (ml[s].x == -INFINITY) continue;
    const float e = exp2f(ml[s].x - M);
    L = fmaf(e, ml[s].y, L);
    if (threadIdx.x < p.d) A = fmaf(e, p.part_acc[(row * p.splits + s) * p.d + threadIdx.x], A);
  }
  if (threadIdx.x >= p.d) return;
  const float o = M == -INFINITY ? 0.f : A / L;  // a row that sees no key gives zeros
  const int64_t at = (row / p.t) * p.so_h + (row % p.t) * p.so_t + threadIdx.x;
  if (p.dtype == BB_BF16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(o);
  else static_cast<__half*>(p.out)[at] = __float2half_rn(o);
}

// Grid (splits, heads).
__global__ void __launch_bounds__(32 * WARPS) qkv_scores_kernel(AttnParams p) {
  __shared__ float sm[WARPS], sl[WARPS];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t h = blockIdx.y, kv = h / p.groups;
  const int64_t n = cache_len(p);
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = 32 * i < p.d ? load_elem(p.q, h * p.sq_h + 32 * i + lane, p.dtype) : 0.f;
  float m = -INFINITY, l = 0.f;
  for (int64_t j = (int64_t)blockIdx.x * WARPS + warp; j < n; j += (int64_t)p.splits * WARPS) {
    const float s = key_score(p, kv, j, q, lane);
    if (lane == 0) p.scores[h * p.cap + j] = s;
    const float mn = fmaxf(m, s);
    l = l * exp2f(m - mn) + exp2f(s - mn);
    m = mn;
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm[w]);
    for (int w = 0; w < WARPS; ++w) L += sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - M) * sl[w];
    p.part_ml[h * p.splits + blockIdx.x] = make_float2(M, L);
  }
}

// Grid (cdiv(cap, 1024), kv_heads); four positions a thread.
__global__ void __launch_bounds__(256) qkv_pool_kernel(AttnParams p) {
  const int64_t kv = blockIdx.y, n = cache_len(p);
  float sum[4] = {};
  for (int64_t h = kv * p.groups; h < (kv + 1) * p.groups; ++h) {
    const float2* ml = p.part_ml + h * p.splits;
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < p.splits; ++s) M = fmaxf(M, ml[s].x);
    for (int s = 0; s < p.splits; ++s) L += ml[s].x == -INFINITY ? 0.f : exp2f(ml[s].x - M) * ml[s].y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t pos = (int64_t)blockIdx.x * 1024 + i * 256 + threadIdx.x;
      if (pos < n) sum[i] += exp2f(p.scores[h * p.cap + pos] - M) / L;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t pos = (int64_t)blockIdx.x * 1024 + i * 256 + threadIdx.x;
    if (pos < p.cap)
      p.probs[kv * p.cap + pos] = (pos >= p.front && pos < n - p.window) ? sum[i] / (float)p.groups : -1.f;
  }
}

struct AttnPlan {
  int64_t splits;
  size_t ml_bytes, acc_bytes, scores_bytes, probs_bytes, topk_bytes, total;
};

int check_attn(const bb_qkv_attn_args* a, const char* what, bool need_v) {
  if (!a) return fail(BB_ERR_ARG, "%s: null args", what);
  int st = qkv::check_cache(a->cache, what, true, need_v);
  if (st) return st;
  if (a->dtype != BB_F16 && a->dtype != BB_BF16) return fail(BB_ERR_DTYPE, "%s requires fp16 or bf16 queries", what);
  if (a->heads <= 0 || a->heads % a->cache.kv_heads || a->heads > 65535)
    return fail(BB_ERR_SHAPE, "%s: heads must be a positive multiple of kv_heads (at most 65535)", what);
  if (a->t <= 0 || a->t > 65535 || a->t * a->heads > (int64_t)65535)
    return fail(BB_ERR_SHAPE, "%s: heads * tokens must lie in [1, 65535]", what);
  if (a->n < 0 || a->n > a->cache.cap) return fail(BB_ERR_ARG, "%s: n must lie in [0, capacity]", what);
  if (a->front < 0 || a->window < 0) return fail(BB_ERR_ARG, "%s: front and window must be >= 0", what);
  if (a->route_k < 0) return fail(BB_ERR_ARG, "%s: bad route count", what);
  if (a->splits < 0) return fail(BB_ERR_ARG, "%s: splits must be >= 0", what);
  return BB_OK;
}

int64_t pick_splits(int64_t asked, int64_t keys, int64_t rows) {
  int64_t s = asked > 0 ? asked : std::max<int64_t>(1, (int64_t)num_sms() * 16 / rows);
  return std::max<int64_t>(1, std::min<int64_t>({s, cdiv(std::max<int64_t>(keys, 1), (int64_t)16), (int64_t)1024}));
}

int plan_decode(const bb_qkv_attn_args* a, AttnPlan* pl) {
  int st = check_attn(a, "qkv_decode", true);
  if (st) return st;
  if (a->route_k > 0 && a->route_rows != a->cache.kv_heads && a->route_rows != a->heads)
    return fail(BB_ERR_SHAPE, "qkv_decode: indices must be [Hkv, R] (pooled) or [H, R] (per head)");
  const int64_t rows = a->heads * a->t;
  const int64_t keys = std::min(a->cache.cap, std::min(a->front, a->cache.cap) + std::min(a->window, a->cache.cap)) + a->route_k;
  *pl = {};
  pl->splits = pick_splits(a->splits, keys, rows);
  pl->ml_bytes = align_up((size_t)(rows * pl->splits) * 8, 256);
  pl->acc_bytes = align_up((size_t)(rows * pl->splits * a->cache.d) * 4, 256);
  pl->total = pl->ml_bytes + pl->acc_bytes;
  return BB_OK;
}

int plan_route(const bb_qkv_attn_args* a, AttnPlan* pl) {
  int st = check_attn(a, "qkv_route", false);
  if (st) return st;
  if (a->t != 1) return fail(BB_ERR_SHAPE, "qkv_route: one token at a time");
  if (a->route_k > a->cache.cap) return fail(BB_ERR_ARG, "qkv_route: route_k must lie in [0, capacity]");
  *pl = {};
  pl->splits = pick_splits(a->splits, a->cache.cap, a->heads);
  pl->ml_bytes = align_up((size_t)(a->heads * pl->splits) * 8, 256);
  pl->scores_bytes = align_up((size_t)(a->heads * a->cache.cap) * 4, 256);
  pl->probs_bytes = a->out_probs ? 0 : align_up((size_t)(a->cache.kv_heads * a->cache.cap) * 4, 256);
  pl->topk_bytes = align_up(topk_scratch_bytes(a->cache.kv_heads, a->cache.cap, a->route_k), 256);
  pl->total = pl->ml_bytes + pl->scores_bytes + pl->probs_bytes + pl->topk_bytes;
  return BB_OK;
}

AttnParams make_params(const bb_qkv_attn_args* a, const AttnPlan& pl, char* ws) {
  const bb_qkv_cache& c = a->cache;
  AttnParams p{};
  p.kc = static_cast<const unsigned char*>(c.k_codes); p.km = static_cast<const uint32_t*>(c.k_meta);
  p.vc = static_cast<const unsigned char*>(c.v_codes); p.vm = static_cast<const uint32_t*>(c.v_meta);
  p.kc_h = c.k_codes_h; p.km_h = c.k_meta_h; p.vc_h = c.v_codes_h; p.vm_h = c.v_meta_h;
  p.q = a->q; p.sq_h = a->sq_h; p.sq_t = a->sq_t;
  p.idx = a->idx; p.si_r = a->si_r;
  p.route_k = a->route_k;
  p.idx64 = a->idx_i64 != 0;
  p.per_head = a->route_rows != c.kv_heads;
  p.n_dev = a->n_dev;
  p.n = a->n; p.cap = c.cap; p.front = a->front; p.window = a->window;
  p.d = (int)c.d; p.bits = c.bits; p.group = c.group; p.pairs = (int)(c.d / c.group);
  p.row_bytes = (int)(c.d * c.bits / 8);
  p.heads = (int)a->heads; p.kv_heads = (int)c.kv_heads; p.groups = (int)(a->heads / c.kv_heads);
  p.t = (int)a->t; p.splits = (int)pl.splits; p.dtype = a->dtype;
  p.scale_log2 = a->scale * LOG2E;
  p.part_ml = reinterpret_cast<float2*>(ws);
  p.part_acc = reinterpret_cast<float*>(ws + pl.ml_bytes);
  p.scores = reinterpret_cast<float*>(ws + pl.ml_bytes);
  p.probs = a->out_probs ? a->out_probs : reinterpret_cast<float*>(ws + pl.ml_bytes + pl.scores_bytes);
  p.out = a->out; p.so_h = a->so_h; p.so_t = a->so_t;
  return p;
}

}  // namespace

int qkv_decode_workspace_size(const bb_qkv_attn_args* a, size_t* bytes) {
  AttnPlan pl;
  int st = plan_decode(a, &pl);
  if (st) return st;
  *bytes = pl.total;
  return BB_OK;
}

int qkv_decode(const bb_qkv_attn_args* a, void* ws, size_t ws_bytes, cudaStream_t stream) {
  AttnPlan pl;
  int st = plan_decode(a, &pl);
  if (st) return st;
  if (!ws || ws_bytes < pl.total)
    return fail(BB_ERR_WORKSPACE, "qkv_decode: workspace too small (%zu < %zu)", ws_bytes, pl.total);
  if (!a->q || !a->out || (a->route_k > 0 && !a->idx)) return fail(BB_ERR_ARG, "qkv_decode: null pointer");
  AttnParams p = make_params(a, pl, static_cast<char*>(ws));
  const unsigned rows = (unsigned)(a->heads * a->t);
  qkv_partial_kernel<<<dim3((unsigned)pl.splits, rows), 32 * WARPS, 0, stream>>>(p);
  BB_CHECK_LAUNCH("qkv_partial_kernel");
  qkv_combine_kernel<<<rows, 128, 0, stream>>>(p);
  BB_CHECK_LAUNCH("qkv_combine_kernel");
  return BB_OK;
}

int qkv_route_workspace_size(const bb_qkv_attn_args* a, size_t* bytes) {
  AttnPlan pl;
  int st = plan_route(a, &pl);
  if (st) return st;
  *bytes = pl.total;
  return BB_OK;
}

int qkv_route(const bb_qkv_attn_args* a, void* ws, size_t ws_bytes, cudaStream_t stream) {
  AttnPlan pl;
  int st = plan_route(a, &pl);
  if (st) return st;
  if (!ws || ws_bytes < pl.total)
    return fail(BB_ERR_WORKSPACE, "qkv_route: workspace too small (%zu < %zu)", ws_bytes, pl.total);
  if (!a->q || (!a->out_probs && !a->out_idx)) return fail(BB_ERR_ARG, "qkv_route: null pointer");
  char* w = static_cast<char*>(ws);
  AttnParams p = make_params(a, pl, w);
  qkv_scores_kernel<<<dim3((unsigned)pl.splits, (unsigned)a->heads), 32 * WARPS, 0, stream>>>(p);
  BB_CHECK_LAUNCH("qkv_scores_kernel");
  qkv_pool_kernel<<<dim3((unsigned)cdiv(a->cache.cap, (int64_t)1024), (unsigned)a->cache.kv_heads), 256, 0, stream>>>(p);
  BB_CHECK_LAUNCH("qkv_pool_kernel");
  if (a->route_k > 0 && a->out_idx)
    return topk_sorted(p.probs, a->cache.kv_heads, a->cache.cap, a->route_k, a->out_idx, a->out_idx_i64 != 0, a->so_i,
                       w + pl.ml_bytes + pl.scores_bytes + pl.probs_bytes, pl.topk_bytes, stream);
  return BB_OK;
}

}  // namespace bb
