// Attention of the newest tokens over a quantised KV cache, and decode routing over its keys
// (semantics: include/bb_b200.h, bb_qkv_decode and bb_qkv_route).
//
//   qkv_partial_kernel  up to 4, 8 or 16 query rows of one KV head over one split of its key list: running max,
//                       sum and P.V of the split, in fp32; the last CTA of a tile to arrive merges its splits
//   qkv_combine_kernel  merges them where the caller gave no tickets
//   qkv_scores_kernel   log2 scores of every key for the query heads of a KV head, and per-split softmax
//                       statistics; then, where its CTAs can wait for each other, the pooled probabilities
//   qkv_pool_kernel     merged statistics, probabilities averaged over the query heads of a KV head
//
// The mathematics. With codes c, a step s and a low value l for every group g of a row,
//   q . k_j   = sum_g s_jg (q_g . c_jg) + l_jg sum(q_g)
//   sum_j p_j v_j = sum_j (p_j s_jg) c_jg + sum_j p_j l_jg          (dimensions of group g)
// so both products run on the tensor cores (mma.sync m16n8k16, fp32 accumulators) with the bare codes as
// one operand: no code is multiplied by its step or moved by its low value. The codes need no conversion
// either: the bits of a code at bit 0 (or a 4-bit code at bit 4) of a 16-bit word are the fp16 number
// code 2^-24 (code 2^-20), a subnormal that the tensor cores take as it is, so a masked word is a pair of
// operands. The powers of two are undone in fp32. Keys (rows of K) and dimensions (rows of V transposed)
// are the 16 rows of a product and the query rows its 8 columns (Layout, Accum).
//   q: fp16 after a power of two that brings the row's largest element to [2^14, 2^15), against 4-bit codes that
// carry 2^-20 to [2^10, 2^11) (exact for bf16 and fp16 queries, except elements below 2^-28, there 2^-24, of the
// largest, which lose relative precision only).
//   P = p s: rounded to fp16 once, in units in which p = 1 and s = the group's bound make 2^11. The bound is a power of
// two, at most twice the largest step of the group that the warp has met; p refers to the running maximum, which may lag
// by 2^4. So P <= 2^15; it keeps all 11 bits while p s is at least 2^-24 of the group's largest step, and is off by at most
// 2^-36 of the bound below that.
// Scores, exponentials, sums and accumulators are fp32.
//
// What bounds it: bytes, 2 (d bits / 8 + 4 d / group) a key and KV head, and close behind them the issue slots that unpack
// codes (about 590 warp instructions a step of 32 keys; HBM gives a SM a step every 220 cycles, so at 4 a cycle they
// take 150). Measured on 8 KV heads x 4 query heads, d = 128, 4 bits, groups of 32: dense decode 37.7 us at 128K keys
// (168 MB, 4.5 TB/s) and 50 us more for each 256K keys beyond (the rate of a copy); the rest, about 12 us, is the first
// keys' latency and the merge of the splits. More than 4 query rows of a KV head (several tokens) are bound by instructions:
// every 8 rows unpack all codes anew, 89 us for 64 rows on 32K keys.
#include <algorithm>
#include <atomic>

#include "qkv.cuh"
#include "tc_common.cuh"

namespace bb {

int topk_sorted(const float* vals, int64_t rows, int64_t n, int64_t k, void* out, bool out64, int64_t so_h,
                void* scratch, size_t scratch_bytes, cudaStream_t stream);
size_t topk_scratch_bytes(int64_t rows, int64_t n, int64_t k);

namespace {

constexpr int SCORE_WARPS = 16, SCORE_STAGES = 3;  // one CTA a SM
constexpr float LOG2E = 1.4426950408889634f;
constexpr float M_NONE = -1.7e38f;   // running maximum before any key (finite: exp2(-inf - M_NONE) is 0)
constexpr float LAZY = 4.f;          // the running maximum moves only when a score exceeds it by 2^4
constexpr float P_SCALE = 2048.f;    // 2^(15 - LAZY)

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
  int d, heads, groups, t, cols, splits, ztiles, dtype;
  int q16;          // query rows on 16-byte boundaries
  float scale_log2;
  float2* part_ml;  // (max in log2 units, sum): [kv_heads * ztiles][splits][columns]; routing: [heads][splits]
  float* part_acc;  // [kv_heads * ztiles][splits][columns][d]
  int32_t* tickets; // [kv_heads * ztiles] arrivals, zero between calls; or null
  void* out; int64_t so_h, so_t;
  float4* scores;   // routing: log2 units, [kv_heads][steps][ztiles][score tiles][32 threads]
  int64_t steps;    // of 32 keys in the whole cache
  float* probs;     // [kv_heads][cap]
};

__device__ __forceinline__ int64_t cache_len(const AttnParams& p) {
  if (!p.n_dev) return p.n;
  const int64_t n = *p.n_dev;
  return n < 0 ? 0 : (n > p.cap ? p.cap : n);
}

// The key list of one KV head in steps of 32 keys (two tiles of 16): front keys [0, fa), keys [b0, n) in the
// window of any of the tokens, and lists (one, or one for each query head). First come the whole steps from
// `bf` on, of consecutive keys that all count for every token; then the rest: the front, the ends of the
// window and the lists. Where front and window meet, all of it is one range.
struct Steps {
  int n, fa;
  int bf, whole;
  int lo[3], hi[3], cut[3];  // the rest of the ranges, and the step after the last of each
  int nc, total;
  // every_key: the first n keys, whatever front, window and lists say.
  __device__ __forceinline__ Steps(const AttnParams& p, bool every_key) {
    const int64_t len = cache_len(p);
    n = (int)len;
    const int64_t f = p.front < len ? p.front : len;
    const bool all = every_key || len - p.window <= f;
    fa = all ? 0 : (int)f;
    const int b0 = all ? 0 : (int)min(max(f, len - p.t + 1 - p.window), len);  // first token's window
    bf = all ? 0 : (int)min(len - p.window, len);                              // every token's window
    const int last = max(0, n - p.t + 1);                                      // keys that every token sees: [0, last)
    whole = max(0, last - bf) / 32;
    lo[0] = 0;               hi[0] = fa;
    lo[1] = b0;              hi[1] = bf;
    lo[2] = bf + whole * 32; hi[2] = n;
    int u = whole;
#pragma unroll
    for (int i = 0; i < 3; ++i) cut[i] = u += (hi[i] - lo[i] + 31) / 32;
    nc = every_key ? 0 : (int)((p.route_k + 31) / 32);
    total = u + nc * (p.per_head ? p.groups : 1);
  }
  __device__ __forceinline__ bool listed(int u) const { return u >= cut[2]; }
  // Keys [from, to) of a step of the rest that is not listed.
  __device__ __forceinline__ void range(int u, int& from, int& to) const {
    const int i = u < cut[0] ? 0 : (u < cut[1] ? 1 : 2);
    from = (i == 0 ? lo[0] + (u - whole) * 32 : (i == 1 ? lo[1] + (u - cut[0]) * 32 : lo[2] + (u - cut[1]) * 32));
    to = i == 0 ? hi[0] : (i == 1 ? hi[1] : hi[2]);
  }
};

template <int BITS, int G, int NG, bool WITH_V> struct Stage {
  static constexpr int ROW = G * 4 * BITS;                // bytes of codes a row
  static constexpr int META = NG * 4;                     // bytes of (step, low) pairs a row
  static constexpr int SIDES = WITH_V ? 2 : 1;
  static constexpr int V = 32 * ROW, KM = SIDES * 32 * ROW;  // K codes at 0
  static constexpr int VM = KM + (SIDES - 1) * 32 * META;
  static constexpr int POS = VM + 32 * META;
  static constexpr int BYTES = POS + (WITH_V ? 128 : 0);
  static_assert(BYTES % 16 == 0 && V <= KM && VM < BYTES, "stages start on 16-byte boundaries");
};

// Key j of a tile feeds row slot(j) of the K product, so that the keys of a thread's V operands
// (slots 2c, 2c + 1, 2c + 8, 2c + 9) are the tile's rows c, c + 4, c + 8, c + 12, whose reads from shared
// memory fall into different banks.
__device__ __forceinline__ int slot_of(int j) { return (j & 24) | ((j & 3) << 1) | ((j >> 2) & 1); }
__device__ __forceinline__ int key_of(int r) { return ((r & 1) << 2) | (r >> 1); }  // r < 8

// 16-byte chunks of a staged row are stored at chunk ^ swizzle(row), against bank conflicts: K reads take a
// quarter row a thread, V reads an eighth of rows c.
template <int ROW> __host__ __device__ __forceinline__ constexpr int k_swizzle(int slot) { return ROW == 128 ? (slot & 1) : 0; }
template <int ROW> __device__ __forceinline__ int v_swizzle(int row) {
  return ROW == 128 ? (row & 3) << 1 : (ROW == 64 ? row & 2 : 0);
}

template <int N> __device__ __forceinline__ void cp_async_n(uint32_t dst, const void* src, bool valid) {
  if constexpr (N == 16)
    cp_async_16(dst, src, valid);
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(dst), "l"(src), "n"(N), "r"(valid ? N : 0));
}

// A warp's copies into its stages.
template <int BITS, int G, int NG, bool WITH_V> struct Source {
  using S = Stage<BITS, G, NG, WITH_V>;
  static constexpr int CH = S::ROW / 16;       // 16-byte chunks a row
  static constexpr bool FLAT = 32 % CH == 0;   // a thread's chunks lie 512 bytes apart at one place in their rows
  const unsigned char *kc, *vc;                // of this KV head, + lane * 16
  const uint32_t *km, *vm;                     // + lane * NG
  const unsigned char *k_at, *v_at;            // the next whole step
  const uint32_t *km_at, *vm_at;
  int64_t ahead;                               // rows between this warp's whole steps
  uint32_t kdst, vdst, mdst;

  __device__ __forceinline__ Source(const AttnParams& p, int64_t kv, int lane, int64_t row, int64_t rows_ahead) {
    kc = p.kc + kv * p.kc_h + lane * 16;
    km = p.km + kv * p.km_h + lane * NG;
    k_at = kc + row * S::ROW;
    km_at = km + row * NG;
    if constexpr (WITH_V) {
      vc = p.vc + kv * p.vc_h + lane * 16;
      vm = p.vm + kv * p.vm_h + lane * NG;
      v_at = vc + row * S::ROW;
      vm_at = vm + row * NG;
    }
    ahead = rows_ahead;
    const int j = lane / CH, ch = lane % CH;
    kdst = slot_of(j) * S::ROW + ((ch ^ k_swizzle<S::ROW>(slot_of(j))) << 4);
    vdst = S::V + j * S::ROW + ((ch ^ v_swizzle<S::ROW>(j)) << 4);
    mdst = S::KM + slot_of(lane) * S::META;
  }

  __device__ __forceinline__ void meta(uint32_t st, const uint32_t* k, const uint32_t* v, bool ok) const {
    constexpr int N = NG == 3 ? 4 : S::META;
#pragma unroll
    for (int i = 0; i < S::META / N; ++i) {
      cp_async_n<N>(st + mdst + i * N, k + i, ok);
      if constexpr (WITH_V) cp_async_n<N>(st + mdst + (S::VM - S::KM) + i * N, v + i, ok);
    }
  }

  // The next whole step: one address a buffer, constant offsets.
  __device__ __forceinline__ void whole(uint32_t st) {
    if constexpr (FLAT) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        // rows 32 / CH * i further on: 8 i or 16 i slots, or (CH = 8) 4 i rows: slots 8 (i / 2) + i % 2
        const uint32_t at = CH == 8 ? (kdst ^ (i & 1 ? 16u : 0u)) + (i >> 1) * 8 * S::ROW + (i & 1) * S::ROW : kdst + i * 512;
        cp_async_16(st + at, k_at + i * 512, true);
        if constexpr (WITH_V) cp_async_16(st + vdst + i * 512, v_at + i * 512, true);
      }
    } else {
      const int lane = threadIdx.x % 32;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int x = lane + 32 * i, j = x / CH, ch = x % CH, sl = slot_of(j);
        cp_async_16(st + sl * S::ROW + ((ch ^ k_swizzle<S::ROW>(sl)) << 4), k_at + i * 512, true);
        if constexpr (WITH_V) cp_async_16(st + S::V + j * S::ROW + ((ch ^ v_swizzle<S::ROW>(j)) << 4), v_at + i * 512, true);
      }
    }
    meta(st, km_at, vm_at, true);
    k_at += ahead * S::ROW;
    km_at += ahead * NG;
    if constexpr (WITH_V) {
      v_at += ahead * S::ROW;
      vm_at += ahead * NG;
    }
  }

  // Rows at `mine` (a position a lane, -1: none, filled with zeros).
  __device__ __forceinline__ void rows(uint32_t st, int mine, int lane) const {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int x = lane + 32 * i, j = x / CH, ch = x % CH, sl = slot_of(j);
      const int pos = __shfl_sync(0xffffffffu, mine, j);
      const int64_t off = (int64_t)(pos < 0 ? 0 : pos) * S::ROW + (ch - lane) * 16;
      cp_async_16(st + sl * S::ROW + ((ch ^ k_swizzle<S::ROW>(sl)) << 4), kc + off, pos >= 0);
      if constexpr (WITH_V) cp_async_16(st + S::V + j * S::ROW + ((ch ^ v_swizzle<S::ROW>(j)) << 4), vc + off, pos >= 0);
    }
    const int64_t off = (int64_t)((mine < 0 ? 0 : mine) - lane) * NG;
    meta(st, km + off, WITH_V ? vm + off : nullptr, mine >= 0);
  }

  // Step u >= whole.
  __device__ __forceinline__ void rest(const AttnParams& p, const Steps& sp, int u, uint32_t st, int64_t kv, int lane) const {
    if (!WITH_V || !sp.listed(u)) {
      int from, to;
      sp.range(u, from, to);
      rows(st, from + lane < to ? from + lane : -1, lane);
      return;
    }
    const int w = u - sp.cut[2], list = w / sp.nc;
    const int64_t j = (int64_t)(w - list * sp.nc) * 32 + lane;
    int64_t pos = -1;
    if (j < p.route_k) {
      const int64_t o = (p.per_head ? kv * p.groups + list : kv) * p.si_r + j;
      pos = p.idx64 ? static_cast<const int64_t*>(p.idx)[o] : (int64_t) static_cast<const int32_t*>(p.idx)[o];
    }
    const int mine = (pos >= sp.fa && pos < sp.n) ? (int)pos : -1;
    asm volatile("st.shared.s32 [%0], %1;" ::"r"(st + S::POS + slot_of(lane) * 4), "r"(mine) : "memory");
    rows(st, mine, lane);
  }

  __device__ __forceinline__ void fetch(const AttnParams& p, const Steps& sp, int u, uint32_t st, int64_t kv, int lane) {
    if (u < sp.whole) whole(st);
    else if (u < sp.total) rest(p, sp, u, st, kv, lane);
    cp_async_commit();
  }
};

// Runs a warp's steps first, first + stride, ... through its ring of NS stages: inner(stage) for whole steps, edge(u, stage)
// for the rest. No barrier: a warp only ever waits for its own copies.
template <int NS, typename Src, typename Inner, typename Edge>
__device__ __forceinline__ void run_steps(const AttnParams& p, const Steps& sp, Src& src, uint32_t ring, int first, int stride,
                                          int64_t kv, int lane, Inner inner, Edge edge) {
  constexpr int BYTES = Src::S::BYTES;
  int u = first;
  int left = u < sp.whole ? (sp.whole - u + stride - 1) / stride : 0;
  int next = u + (NS - 1) * stride;
  int at = 0;
  while (left > 0) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if (left > 0) {
        cp_async_wait<NS - 2>();
        __syncwarp();
        src.fetch(p, sp, next, ring + (i + NS - 1) % NS * BYTES, kv, lane);
        next += stride;
        inner(ring + i * BYTES);
        --left;
        u += stride;
        at = (i + 1) % NS;
      }
    }
  }
  for (; u < sp.total; u += stride) {
    cp_async_wait<NS - 2>();
    __syncwarp();
    src.fetch(p, sp, next, ring + (at == 0 ? NS - 1 : at - 1) * BYTES, kv, lane);
    next += stride;
    edge(u, ring + at * BYTES);
    at = at == NS - 1 ? 0 : at + 1;
  }
  cp_async_wait<0>();
}

template <int N> __device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t at) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(at + i * 4));
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[i]), "=r"(w[i + 1]) : "r"(at + i * 4));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(at + i * 4));
  }
}
__device__ __forceinline__ uint32_t lds_word(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}

// A quarter of a staged K row: the codes of dimensions 8c .. 8c + 7 of every 32.
template <int BITS, int G> __device__ __forceinline__ void k_words(uint32_t (&w)[G * BITS / 4], uint32_t rows, int slot, int c) {
  constexpr int ROW = G * 4 * BITS;
  if constexpr (ROW == 128) {
    uint32_t a[4], b[4];
    const uint32_t at = rows + slot * ROW + c * 32, x = (uint32_t)k_swizzle<ROW>(slot) << 4;
    lds_words(a, at + x);
    lds_words(b, at + (x ^ 16u));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = a[i];
      w[4 + i] = b[i];
    }
  } else {
    lds_words(w, rows + slot * ROW + c * (ROW / 4));
  }
}

// An eighth of a staged V row: the codes of dimensions 4r .. 4r + 3 of every 32; 4 bits: two blocks of 32
// dimensions a word, 8 bits: one.
template <int BITS, int G>
__device__ __forceinline__ void v_words(uint32_t (&w)[(G * BITS + 7) / 8], uint32_t rows, int row, int r) {
  constexpr int ROW = G * 4 * BITS, BYTES = ROW / 8;
  if constexpr (BYTES % 4) {
    const uint32_t at = rows + row * ROW + r * BYTES;
#pragma unroll
    for (int i = 0; i < (G + 1) / 2; ++i) {
      w[i] = lds_u16(at + i * 4);
      if (2 * i + 1 < G) w[i] |= lds_u16(at + i * 4 + 2) << 16;
    }
  } else {
    // r * BYTES with its chunk number swizzled (v_swizzle is 0 unless a thread's part lies in one chunk)
    lds_words(w, rows + row * ROW + ((r * BYTES) ^ (v_swizzle<ROW>(row) << 4)));
  }
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// Rows 8 x 8 of 16-bit elements, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float step_of(uint32_t m) { return __uint_as_float(m << 16); }
__device__ __forceinline__ float low_of(uint32_t m) { return __uint_as_float(m & 0xFFFF0000u); }

// C += A B; A 16 x 16 codes or probabilities, fp16; and the same from C = 0.
__device__ __forceinline__ void mma_h(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_h0(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
}

// C += ones B over 8 of k: rows 0-7 (half 0) or 8-15 (half 1) of C take the column sums of B. The other half's rows are
// multiplied by zero, so where two groups share C, a group's B is NaN only if the key's p is (for every group: see no_nan).
__device__ __forceinline__ void mma_sum(float (&d)[4], int half, uint32_t b) {
  constexpr uint32_t ONES = 0x3C003C00u;  // fp16 1, 1
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(half ? 0u : ONES), "r"(half ? ONES : 0u), "r"(b));
}

// How a step's 32 keys and the query rows fill a product's 16 rows and 8 columns.
//   SPLIT (at most 4 query rows): each k-slice of 16 holds 8 dimensions of both tiles, and the query rows
//     stand in columns 0-3 against the first tile's dimensions and in columns 4-7 against the second's
//     (zeros elsewhere). One product gives the scores of 32 keys, and every thread's four scores are
//     distinct (key, query) pairs, so the softmax costs half as much as with four idle columns.
//   else: 8 query rows in the columns, the two key tiles one after the other.
template <bool SPLIT> struct Layout {
  static constexpr int COLS = SPLIT ? 4 : 8;        // query rows of a warp
  static constexpr int TILES = SPLIT ? 1 : 2;       // score tiles a step
  // Query row of column 2c + k, and the key tile (of a split step) that it belongs to.
  static __device__ __forceinline__ int col(int c, int k) { return SPLIT ? (2 * c + k) & 3 : 2 * c + k; }
  static __device__ __forceinline__ int tile(int x, int c) { return SPLIT ? c >> 1 : x; }
};

// The query side of a warp: operands for its columns (query row = token * groups + head within the KV head's
// query heads), and, for this thread's columns, the sums of each group's elements and the factor that
// turns (codes . operand) into a log2 score.
template <int BITS, int G, int NG, bool SPLIT> struct Query {
  using Y = Layout<SPLIT>;
  // four sets of dimensions a block of 32, as they come out of a word of codes: SPLIT: a product each; else two
  // products of two sets
  uint32_t f[G][SPLIT ? 4 : 2][2];
  float sum[NG][2], mul[2];

  // The rows as stored: issued before the first keys are asked for, waited for after.
  struct Raw {
    uint4 v[G];
  };
  static __device__ __forceinline__ void load(Raw& raw, const AttnParams& p, int64_t kv, int col0, int lane) {
    const int r = lane / 4, c = lane % 4;
    const int col = col0 + (SPLIT ? r & 3 : r);
    const bool live = col < p.cols;
    const int token = p.t == 1 ? 0 : col / p.groups, head = col - token * p.groups;
    const uint16_t* src = static_cast<const uint16_t*>(p.q) + (live ? (kv * p.groups + head) * p.sq_h + token * p.sq_t : 0) + c * 8;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      raw.v[g] = make_uint4(0u, 0u, 0u, 0u);
      if (live && p.q16) {
        raw.v[g] = *reinterpret_cast<const uint4*>(src + g * 32);
      } else if (live) {
        uint16_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = src[g * 32 + i];
        raw.v[g] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                                  e[6] | (uint32_t)e[7] << 16);
      }
    }
  }

  __device__ __forceinline__ void take(const Raw& rows, const AttnParams& p, int lane) {
    const int r = lane / 4, c = lane % 4;
    float x[G][8];
    float top = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint4 raw = rows.v[g];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = i < 2 ? raw.x : (i < 4 ? raw.y : (i < 6 ? raw.z : raw.w));
        const uint16_t h = (uint16_t)(i % 2 ? w >> 16 : w);
        x[g][i] = p.dtype == BB_BF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
        top = fmaxf(top, fabsf(x[g][i]));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^e with top 2^e in [2^10, 2^11)
    int e = 10 - ((int)((__float_as_uint(top) >> 23) & 255) - 127);
    e = top == 0.f ? 0 : max(-118, min(118, e));
    const float up = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
    float s[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) s[i] = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[g / (G / NG)] += x[g][i];
      // Sets of dimensions in the order in which codes come out of a word. 4 bits: (0,4) (1,5) (2,6) (3,7), the
      // even sets at 2^-24 and the odd ones at 2^-20; 8 bits: (0,2) (1,3) (4,6) (5,7), all at 2^-24.
      uint32_t h[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i0 = BITS == 4 ? k : (k / 2) * 4 + k % 2, i1 = BITS == 4 ? k + 4 : i0 + 2;
        const float w = BITS == 4 && k % 2 ? up : up * 16.f;
        h[k] = pack2<__half>(x[g][i0] * w, x[g][i1] * w);
      }
      if constexpr (SPLIT) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f[g][k][0] = r < 4 ? h[k] : 0u;
          f[g][k][1] = r < 4 ? 0u : h[k];
        }
      } else if constexpr (BITS == 4) {
        f[g][0][0] = h[0]; f[g][0][1] = h[2];
        f[g][1][0] = h[1]; f[g][1][1] = h[3];
      } else {
        f[g][0][0] = h[0]; f[g][0][1] = h[1];
        f[g][1][0] = h[2]; f[g][1][1] = h[3];
      }
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      s[i] += __shfl_xor_sync(0xffffffffu, s[i], 1);
      s[i] += __shfl_xor_sync(0xffffffffu, s[i], 2);
      s[i] *= up * 9.5367431640625e-07f;  // 2^-20: in units of the codes' products
#pragma unroll
      for (int k = 0; k < 2; ++k) sum[i][k] = __shfl_sync(0xffffffffu, s[i], (2 * c + k) * 4);
    }
    const float m = p.scale_log2 * 1048576.f * down;
#pragma unroll
    for (int k = 0; k < 2; ++k) mul[k] = __shfl_sync(0xffffffffu, m, (2 * c + k) * 4);
  }
};

// The four sets of a block's codes in a thread's K words.
template <int BITS, int N> __device__ __forceinline__ uint32_t code_set(const uint32_t (&w)[N], int g, int k) {
  if constexpr (BITS == 4) {
    const uint32_t x = k < 2 ? w[g] : w[g] >> 8;
    return x & (k % 2 ? 0x00F000F0u : 0x000F000Fu);
  } else {
    const uint32_t x = w[2 * g + k / 2];
    return (k % 2 ? x >> 8 : x) & 0x00FF00FFu;
  }
}

// Scores of a staged step before the columns' factors: s[x] = (slot r, columns 2c, 2c + 1),
// (slot r + 8, ...) of key tile Layout::tile(x, c).
template <int BITS, int G, int NG, bool SPLIT>
__device__ __forceinline__ void step_scores(const Query<BITS, G, NG, SPLIT>& q, uint32_t rows, uint32_t meta, int lane,
                                            float (&s)[Layout<SPLIT>::TILES][4]) {
  using Y = Layout<SPLIT>;
  const int r = lane / 4, c = lane % 4;
#pragma unroll
  for (int x = 0; x < Y::TILES; ++x) {
    uint32_t w[SPLIT ? 4 : 2][G * BITS / 4], m0[NG], m1[NG];
#pragma unroll
    for (int i = 0; i < (SPLIT ? 4 : 2); ++i) k_words<BITS, G>(w[i], rows, x * 16 + i * 8 + r, c);
    lds_words(m0, meta + (Y::tile(x, c) * 16 + r) * NG * 4);
    lds_words(m1, meta + (Y::tile(x, c) * 16 + r + 8) * NG * 4);
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) {
      float acc[4];
#pragma unroll
      for (int b = 0; b < G / NG; ++b) {
        const int g = gi * (G / NG) + b;
#pragma unroll
        for (int k = 0; k < (SPLIT ? 4 : 2); ++k) {
          // SPLIT: set k of both tiles. Else: 4 bits: sets k and k + 2 (one power of two); 8 bits: 2k and 2k + 1.
          const int k0 = SPLIT ? k : (BITS == 4 ? k : 2 * k), k1 = SPLIT ? k : (BITS == 4 ? k + 2 : 2 * k + 1);
          uint32_t a[4];
          a[0] = code_set<BITS>(w[0], g, k0);
          a[1] = code_set<BITS>(w[1], g, k0);
          a[2] = code_set<BITS>(w[SPLIT ? 2 : 0], g, k1);
          a[3] = code_set<BITS>(w[SPLIT ? 3 : 1], g, k1);
          if (b == 0 && k == 0) mma_h0(acc, a, q.f[g][k]);
          else mma_h(acc, a, q.f[g][k]);
        }
      }
      const float s0 = step_of(m0[gi]), l0 = low_of(m0[gi]), s1 = step_of(m1[gi]), l1 = low_of(m1[gi]);
      float(&o)[4] = s[x];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        o[k] = gi == 0 ? l0 * q.sum[gi][k] : fmaf(l0, q.sum[gi][k], o[k]);
        o[2 + k] = gi == 0 ? l1 * q.sum[gi][k] : fmaf(l1, q.sum[gi][k], o[2 + k]);
        o[k] = fmaf(s0, acc[k], o[k]);
        o[2 + k] = fmaf(s1, acc[2 + k], o[2 + k]);
      }
    }
  }
}

// Whether this thread's (key, column) pair i of score tile x counts.
template <bool SPLIT> struct Mask {
  using Y = Layout<SPLIT>;
  bool ok[Y::TILES][4];
  __device__ __forceinline__ void set(const AttnParams& p, const Steps& sp, int u, uint32_t positions, int col0, int lane) {
    const int r = lane / 4, c = lane % 4;
    const bool listed = sp.listed(u);
    const int list = listed ? (u - sp.cut[2]) / sp.nc : 0;
    int from = 0, to = 0;
    if (!listed) sp.range(u, from, to);
#pragma unroll
    for (int x = 0; x < Y::TILES; ++x)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = Y::tile(x, c) * 16 + half * 8;
        int pos;
        if (listed) {
          asm volatile("ld.shared.s32 %0, [%1];" : "=r"(pos) : "r"(positions + (row + r) * 4));
        } else {
          pos = from + row + key_of(r);
          if (pos >= to) pos = -1;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int col = col0 + Y::col(c, k);
          const int own = sp.n - p.t + col / p.groups;  // the token's own position
          const bool in_window = pos > own - p.window;
          const bool list_ok = pos >= p.front && !in_window && (!p.per_head || col % p.groups == list);
          ok[x][half * 2 + k] = pos >= 0 && pos <= own && (listed ? list_ok : (pos < p.front || in_window));
        }
      }
  }
};

// Warps a CTA and stages a warp: one CTA a SM (so that few partial results are left to merge), with 128 registers a
// thread for 4 query rows in 4 bits, 168 for 8 rows and for 8 bits (whose stages are twice as large). Measured for 64
// query rows on 32K keys (8 rows at a time): 12 warps 84.6 us, 10: 100, 14: 111, 16: 88; 16 rows at a time with 8 warps
// of 255 registers: 95 (all of them before each group had its own bound of the steps: 12 warps take 89 with it).
template <int BITS, bool SPLIT> constexpr int warps() { return SPLIT && BITS == 4 ? 16 : 12; }
constexpr int stages(int warps, int bytes) {
  const int fit = 225 * 1024 / (warps * bytes);
  return fit < 2 ? 2 : (fit > 4 ? 4 : fit);
}
// Floats of shared memory that combine() uses.
template <int COLS, int THREADS> constexpr size_t combine_floats(int64_t splits) {
  return THREADS * 4 + (size_t)splits * COLS;
}
template <int BITS, int G, int NG, bool SPLIT> size_t partial_smem(int splits) {
  using S = Stage<BITS, G, NG, true>;
  const size_t ring = (size_t)warps<BITS, SPLIT>() * stages(warps<BITS, SPLIT>(), S::BYTES) * S::BYTES;
  const size_t merge = (size_t)warps<BITS, SPLIT>() * Layout<SPLIT>::COLS * (G * 32 + 2) * 4;
  const size_t last = combine_floats<Layout<SPLIT>::COLS, 32 * warps<BITS, SPLIT>()>(splits) * 4;
  return std::max({ring, merge, last});
}

// A (step, low) pair with a step of zero where it is NaN: its P is zero, and the dimensions of its group become NaN by the low
// value, in `mid`, which is per group.
__device__ __forceinline__ uint32_t no_nan(uint32_t m) { return step_of(m) == step_of(m) ? m : m & 0xFFFF0000u; }

// The steps of a group in four staged rows 8 apart, the first pair at `at`: the largest, NaN where one is.
template <int META> __device__ __forceinline__ float largest_step(uint32_t at) {
  float top = step_of(lds_word(at));
#pragma unroll
  for (int i = 1; i < 4; ++i) top = qkv::max_nan(top, step_of(lds_word(at + i * 8 * META)));
  return top;
}
// The largest of all rows' steps of the group (`top`: largest_step of this thread's rows), after NaN has been taken out of the
// staged pairs. Threads whose lanes differ in bits 2-4 watch one group's rows between them.
template <int META> __device__ __forceinline__ float clean_largest_step(uint32_t at, float top) {
  if (__any_sync(0xffffffffu, top != top)) {
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t pair = at + i * 8 * META, m = no_nan(lds_word(pair));
      top = fmaxf(top, step_of(m));
      __syncwarp();  // threads that share the pair have read it
      asm volatile("st.shared.u32 [%0], %1;" ::"r"(pair), "r"(m) : "memory");
    }
    __syncwarp();
  }
#pragma unroll
  for (int off = 4; off < 32; off *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  return top;
}

// The softmax of a warp's columns: reference points that move only when a score exceeds them by 2^LAZY or a step
// exceeds its group's bound (or is NaN), and the sum of p over this thread's keys. NB: groups that this thread's columns meet.
template <bool SPLIT, int NB> struct Running {
  using Y = Layout<SPLIT>;
  float m[2], l[2];
  float pscale[NB];  // P_SCALE over a power of two above every step of the group so far (2^-100: none)

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      m[k] = M_NONE;
      l[k] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) pscale[j] = P_SCALE * 1.2676506002282294e+30f;
  }
  // Powers of two: their quotients by their exponents. P_SCALE = 2^11.
  static __device__ __forceinline__ int field(float x) { return (int)(__float_as_uint(x) >> 23); }  // x >= 0
  static __device__ __forceinline__ float power(int field) { return __uint_as_float((uint32_t)field << 23); }
  __device__ __forceinline__ float bound(int j) const { return power(127 + 11 + 127 - field(pscale[j])); }
  // Raises group j's bound above `top`, where it is not yet. What the sums of P are to be multiplied by.
  __device__ __forceinline__ float raise(int j, float top) {
    if (!(top * pscale[j] > P_SCALE)) return 1.f;
    const int next = 127 + 11 + 127 - (field(top) + 1), before = field(pscale[j]);
    pscale[j] = power(next);
    return power(max(0, 127 + next - before));
  }

  // Scores s (before their factors) -> p in e. `move`: a step of this thread's rows exceeds its group's bound or is NaN; steps()
  // then raises the bounds. Returns whether the references moved: everything kept in units of p is then to be multiplied by
  // f, and P.V by its group's shrink as well.
  template <bool EDGE, typename Raise>
  __device__ __forceinline__ bool update(float (&e)[Y::TILES][4], const float (&s)[Y::TILES][4],
                                         const float (&mul)[2], const Mask<SPLIT>& mask, bool move, Raise steps,
                                         float (&f)[2]) {
    constexpr int X = Y::TILES;
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[x][i] = fmaf(s[x][i], mul[i & 1], -m[i & 1]);
        if (EDGE && !mask.ok[x][i]) e[x][i] = -INFINITY;
      }
#pragma unroll
    for (int x = 0; x < X; ++x) move |= fmaxf(fmax3(e[x][0], e[x][1], e[x][2]), e[x][3]) > LAZY;
    const bool moved = __any_sync(0xffffffffu, move);
    if (moved) {
      steps();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float v = -INFINITY;
#pragma unroll
        for (int x = 0; x < X; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int i = 2 * h + k;
            e[x][i] = s[x][i] * mul[k];
            if (EDGE && !mask.ok[x][i]) e[x][i] = -INFINITY;
            v = fmaxf(v, e[x][i]);
          }
#pragma unroll
        for (int off = SPLIT ? 2 : 4; off < 32; off *= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
        const float next = fmaxf(m[k], v);
        f[k] = fast_exp2(m[k] - next);
        m[k] = next;
        l[k] *= f[k];
#pragma unroll
        for (int x = 0; x < X; ++x) {
          e[x][k] -= next;
          e[x][2 + k] -= next;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < X; ++x) {
#pragma unroll
      for (int i = 0; i < 4; ++i) e[x][i] = fast_exp2(e[x][i]);
#pragma unroll
      for (int k = 0; k < 2; ++k) l[k] += e[x][k] + e[x][2 + k];
    }
    return moved;
  }
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int off = SPLIT ? 2 : 4; off < 32; off *= 2) l[k] += __shfl_xor_sync(0xffffffffu, l[k], off);
  }
};

// P.V. Written about the middle code C,
//   sum_j p_j v_j = sum_j P_j (c_j - C) + sum_j p_j (low_j + C step_j),   P = p step rounded to fp16,
// so that P's rounding, and the accumulators', act on numbers as small as the values are about their middle.
// Products with the bare codes give sum P c, products with ones sum P; every few steps C sum P is taken off.
template <int BITS> constexpr float CENTRE = BITS == 4 ? 8.f : 128.f;
constexpr int SETTLE = 4;               // steps between two subtractions

// What a power of two the codes of accumulator tile t carry: 2^-24, with 4 bits 2^-20 in the second tile.
template <int BITS> __device__ __forceinline__ constexpr float code_unit(int t) {
  return BITS == 4 && t == 1 ? 9.5367431640625e-07f : 5.9604644775390625e-08f;
}

// Up to 8 query rows in columns; a product covers 16 keys and 16 dimensions.
template <int BITS, int G, int NG, bool SPLIT> struct Accum {
  using Y = Layout<SPLIT>;
  using S = Stage<BITS, G, NG, true>;
  static constexpr int VW = (G * BITS + 7) / 8;
  float o[G][2][4];            // block of 32 dimensions, tile of 16
  float ps[(NG + 1) / 2][4];   // sum P of groups 2i (rows 0-7) and 2i + 1 (rows 8-15)
  float mid[NG][2];            // sum p (low + C step) of this thread's keys
  Running<SPLIT, NG> run;

  __device__ __forceinline__ void clear(int) {
    run.clear();
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) o[g][i / 4][i % 4] = 0.f;
#pragma unroll
    for (int i = 0; i < (NG + 1) / 2 * 4; ++i) ps[i / 4][i % 4] = 0.f;
#pragma unroll
    for (int i = 0; i < NG * 2; ++i) mid[i / 2][i % 2] = 0.f;
  }

  template <bool EDGE>
  __device__ __forceinline__ void step(const Query<BITS, G, NG, SPLIT>& q, uint32_t st, int lane,
                                       const Mask<SPLIT>& mask) {
    const int r = lane / 4, c = lane % 4;
    float s[2][4], e[2][4], f[2], shrink[NG];
    step_scores<BITS, G, NG, SPLIT>(q, st, st + S::KM, lane, s);
    // The four threads that share rows r watch a group each (all of them the only one).
    const uint32_t watch = st + S::VM + r * S::META + min(c, NG - 1) * 4;
    const float top = largest_step<S::META>(watch);
    float mine = run.pscale[0];  // of the group that this thread watches
#pragma unroll
    for (int gi = 1; gi < NG; ++gi) mine = c >= gi ? run.pscale[gi] : mine;
    const auto steps = [&] {
      const float all = clean_largest_step<S::META>(watch, top);
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) shrink[gi] = run.raise(gi, __shfl_sync(0xffffffffu, all, gi));
    };
    if (run.template update<EDGE>(e, s, q.mul, mask, !(top * mine <= P_SCALE), steps, f)) {
#pragma unroll
      for (int i = 0; i < NG * 2; ++i) mid[i / 2][i % 2] *= f[i % 2];
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[g][i / 4][i % 4] *= f[i & 1] * shrink[g / (G / NG)];
#pragma unroll
      for (int gi = 0; gi < NG; ++gi)
#pragma unroll
        for (int k = 0; k < 2; ++k) ps[gi / 2][gi % 2 * 2 + k] *= f[k] * shrink[gi];
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t m0[NG], m1[NG], b[NG][2];
      lds_words(m0, st + S::VM + (x * 16 + r) * S::META);
      lds_words(m1, st + S::VM + (x * 16 + r + 8) * S::META);
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        const float s0 = step_of(m0[gi]), s1 = step_of(m1[gi]);
        const float h0 = fmaf(CENTRE<BITS>, s0, low_of(m0[gi])), h1 = fmaf(CENTRE<BITS>, s1, low_of(m1[gi]));
        const float t0 = s0 * run.pscale[gi], t1 = s1 * run.pscale[gi];
        float u[4] = {e[x][0] * t0, e[x][1] * t0, e[x][2] * t1, e[x][3] * t1};
        if constexpr (EDGE) {  // rows that do not count may hold NaN
          float z[4] = {e[x][0] * h0, e[x][1] * h0, e[x][2] * h1, e[x][3] * h1};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[i] = mask.ok[x][i] ? u[i] : 0.f;
            z[i] = mask.ok[x][i] ? z[i] : 0.f;
          }
          mid[gi][0] += z[0] + z[2];
          mid[gi][1] += z[1] + z[3];
        } else {
          mid[gi][0] = fmaf(e[x][0], h0, fmaf(e[x][2], h1, mid[gi][0]));
          mid[gi][1] = fmaf(e[x][1], h0, fmaf(e[x][3], h1, mid[gi][1]));
        }
        b[gi][0] = transpose8(pack2<__half>(u[0], u[1]));
        b[gi][1] = transpose8(pack2<__half>(u[2], u[3]));
        mma_sum(ps[gi / 2], gi % 2, b[gi][0]);
        mma_sum(ps[gi / 2], gi % 2, b[gi][1]);
      }
      uint32_t w[4][VW];  // rows c, c + 4 (slots 2c, 2c + 1) and c + 8, c + 12 (slots 2c + 8, 2c + 9)
#pragma unroll
      for (int i = 0; i < 4; ++i) v_words<BITS, G>(w[i], st + S::V, x * 16 + c + 4 * i, r);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t a[2][4];
        operands(a, w, g);
        mma_h(o[g][0], a[0], b[g / (G / NG)]);
        mma_h(o[g][1], a[1], b[g / (G / NG)]);
      }
    }
  }

  // Operands of block g: the codes of a dimension of two keys side by side.
  static __device__ __forceinline__ void operands(uint32_t (&a)[2][4], const uint32_t (&w)[4][VW], int g) {
    if constexpr (BITS == 4) {
      const uint32_t sel = g % 2 ? 0x7632u : 0x5410u;
      const uint32_t x0 = prmt(w[0][g / 2], w[1][g / 2], sel), x1 = prmt(w[2][g / 2], w[3][g / 2], sel);
      const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
      a[0][0] = x0 & 0x000F000Fu; a[0][1] = y0 & 0x000F000Fu; a[0][2] = x1 & 0x000F000Fu; a[0][3] = y1 & 0x000F000Fu;
      a[1][0] = x0 & 0x00F000F0u; a[1][1] = y0 & 0x00F000F0u; a[1][2] = x1 & 0x00F000F0u; a[1][3] = y1 & 0x00F000F0u;
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t sel = h ? 0x7632u : 0x5410u;
        const uint32_t x0 = prmt(w[0][g], w[1][g], sel), x1 = prmt(w[2][g], w[3][g], sel);
        a[h][0] = x0 & 0x00FF00FFu; a[h][1] = (x0 >> 8) & 0x00FF00FFu;
        a[h][2] = x1 & 0x00FF00FFu; a[h][3] = (x1 >> 8) & 0x00FF00FFu;
      }
    }
  }

  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int gi = g / (G / NG);
        o[g][i / 4][i % 4] = fmaf(-CENTRE<BITS> * code_unit<BITS>(i / 4), ps[gi / 2][gi % 2 * 2 + i % 2], o[g][i / 4][i % 4]);
      }
#pragma unroll
    for (int i = 0; i < (NG + 1) / 2 * 4; ++i) ps[i / 4][i % 4] = 0.f;
  }

  // Adds up over the threads that share a column, and hands every sum of this thread to put(query row, dimension).
  template <typename F> __device__ __forceinline__ void finish(int lane, F put) {
    settle();
    run.finish();
    const int r = lane / 4, c = lane % 4;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int gi = 0; gi < NG; ++gi)
#pragma unroll
        for (int off = 4; off < 32; off *= 2) mid[gi][k] += __shfl_xor_sync(0xffffffffu, mid[gi][k], off);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h)  // 4 bits: tile t holds dimensions 4r + t, 4r + t + 2; 8 bits: 4r + 2t, + 1
            put(Y::col(c, k), g * 32 + 4 * r + (BITS == 4 ? t + 2 * h : 2 * t + h),
                fmaf(o[g][t][2 * h + k] * (1.f / (P_SCALE * code_unit<BITS>(t))), run.bound(g / (G / NG)), mid[g / (G / NG)][k]));
    }
  }
};

// At most 4 query rows (SPLIT), d = 64 or 128. A product covers 8 keys and 16 dimensions of two blocks: the pair of
// 16-bit operands that comes out of a word of codes holds a dimension of block 2i and one of block 2i + 1 (of
// one key), the query rows stand in columns 0-3 for the first and in columns 4-7 for the second (zeros
// elsewhere). All eight columns carry results, half as many accumulators as with idle ones.
template <int BITS, int G, int NG> struct Accum<BITS, G, NG, true> {
  using Y = Layout<true>;
  using S = Stage<BITS, G, NG, true>;
  static constexpr int VW = (G * BITS + 7) / 8, PAIRS = G / 2;
  static constexpr int NU = NG < PAIRS ? NG : PAIRS;  // groups that this thread's columns meet
  static_assert(G % 2 == 0 && NU <= 2, "blocks come in pairs");
  float o[PAIRS][2][4];
  float ps[4];                     // sum P of this thread's groups 0 (rows 0-7) and 1 (rows 8-15)
  float mid[NU][2];
  Running<true, NU> run;
  uint32_t sel0, sel1;             // place the first / second 16 bits of a word in this column's half

  __device__ __forceinline__ void clear(int lane) {
    run.clear();
    sel0 = lane < 16 ? 0x4410u : 0x1044u;
    sel1 = lane < 16 ? 0x4432u : 0x3244u;
#pragma unroll
    for (int i = 0; i < PAIRS * 8; ++i) o[i / 8][i / 4 % 2][i % 4] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) ps[i] = 0.f;
#pragma unroll
    for (int i = 0; i < NU * 2; ++i) mid[i / 2][i % 2] = 0.f;
  }

  template <bool EDGE>
  __device__ __forceinline__ void step(const Query<BITS, G, NG, true>& q, uint32_t st, int lane, const Mask<true>& mask) {
    const int r = lane / 4, c = lane % 4;
    float s[1][4], e[1][4], f[2], shrink[NU];
    step_scores<BITS, G, NG, true>(q, st, st + S::KM, lane, s);
    // (step, low) of this thread's group j in row r: pairs + j * PAIR; rows lie 8 apart.
    constexpr int PAIR = NG == G ? 8 : 4;
    const uint32_t pairs = st + S::VM + r * S::META + (NG == G ? (c >> 1) * 4 : 0);
    // Threads c and c ^ 1, whose pairs are the same, watch a group each (both the only one).
    const uint32_t watch = pairs + (NU > 1 ? (c & 1) * PAIR : 0);
    const float top = largest_step<S::META>(watch);
    const float mine = NU > 1 && (c & 1) ? run.pscale[NU - 1] : run.pscale[0];
    const auto steps = [&] {
      const float all = clean_largest_step<S::META>(watch, top);
#pragma unroll
      for (int j = 0; j < NU; ++j) shrink[j] = run.raise(j, __shfl_sync(0xffffffffu, all, NU > 1 ? (c & 2) | j : c));
    };
    if (run.template update<EDGE>(e, s, q.mul, mask, !(top * mine <= P_SCALE), steps, f)) {
#pragma unroll
      for (int i = 0; i < NU * 2; ++i) mid[i / 2][i % 2] *= f[i % 2];
#pragma unroll
      for (int i = 0; i < PAIRS * 8; ++i) o[i / 8][i / 4 % 2][i % 4] *= f[i & 1] * shrink[NU == PAIRS ? i / 8 : 0];
#pragma unroll
      for (int i = 0; i < NU * 2; ++i) ps[i] *= f[i & 1] * shrink[i / 2];
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      // p of key tile x from the lanes that scored it (columns 0-3: tile 0, 4-7: tile 1)
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = __shfl_sync(0xffffffffu, e[0][i], x == 0 ? lane & ~2 : lane | 2);
      bool live[4];
      if constexpr (EDGE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) live[i] = __shfl_sync(0xffffffffu, (int)mask.ok[0][i], x == 0 ? lane & ~2 : lane | 2) != 0;
      }
      uint32_t w[4][VW];  // rows c, c + 4 (slots 2c, 2c + 1) and c + 8, c + 12 (slots 2c + 8, 2c + 9)
#pragma unroll
      for (int i = 0; i < 4; ++i) v_words<BITS, G>(w[i], st + S::V, x * 16 + c + 4 * i, r);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t b[NU][2];
#pragma unroll
        for (int j = 0; j < NU; ++j) {
          const uint32_t mm = lds_word(pairs + (2 * x + half) * 8 * S::META + j * PAIR);
          const float sj = step_of(mm), hj = fmaf(CENTRE<BITS>, sj, low_of(mm)), tj = sj * run.pscale[j];
          float u[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            u[k] = t[2 * half + k] * tj;
            if (EDGE) {  // rows that do not count may hold NaN
              u[k] = live[2 * half + k] ? u[k] : 0.f;
              mid[j][k] += live[2 * half + k] ? t[2 * half + k] * hj : 0.f;
            } else {
              mid[j][k] = fmaf(t[2 * half + k], hj, mid[j][k]);
            }
          }
          const uint32_t both = transpose8(pack2<__half>(u[0], u[1]));  // keys 2c, 2c + 1 of this column
          b[j][0] = prmt(both, 0u, sel0);
          b[j][1] = prmt(both, 0u, sel1);
          mma_sum(ps, j, both);
        }
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          uint32_t a[2][4];
          operands(a, w[2 * half], w[2 * half + 1], i);
          mma_h(o[i][0], a[0], b[NU == PAIRS ? i : 0]);
          mma_h(o[i][1], a[1], b[NU == PAIRS ? i : 0]);
        }
      }
    }
  }

  // Operands of blocks 2i, 2i + 1 from the words of two keys.
  static __device__ __forceinline__ void operands(uint32_t (&a)[2][4], const uint32_t (&w0)[VW], const uint32_t (&w1)[VW], int i) {
    if constexpr (BITS == 4) {
      const uint32_t x0 = w0[i], x1 = w1[i], y0 = x0 >> 8, y1 = x1 >> 8;
      a[0][0] = x0 & 0x000F000Fu; a[0][1] = y0 & 0x000F000Fu; a[0][2] = x1 & 0x000F000Fu; a[0][3] = y1 & 0x000F000Fu;
      a[1][0] = x0 & 0x00F000F0u; a[1][1] = y0 & 0x00F000F0u; a[1][2] = x1 & 0x00F000F0u; a[1][3] = y1 & 0x00F000F0u;
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t sel = h ? 0x7632u : 0x5410u;
        const uint32_t x0 = prmt(w0[2 * i], w0[2 * i + 1], sel), x1 = prmt(w1[2 * i], w1[2 * i + 1], sel);
        a[h][0] = x0 & 0x00FF00FFu; a[h][1] = (x0 >> 8) & 0x00FF00FFu;
        a[h][2] = x1 & 0x00FF00FFu; a[h][3] = (x1 >> 8) & 0x00FF00FFu;
      }
    }
  }

  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int i = 0; i < PAIRS * 8; ++i) {
      float& x = o[i / 8][i / 4 % 2][i % 4];
      x = fmaf(-CENTRE<BITS> * code_unit<BITS>(i / 4 % 2), ps[(NU == PAIRS ? i / 8 : 0) * 2 + i % 2], x);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) ps[i] = 0.f;
  }

  template <typename F> __device__ __forceinline__ void finish(int lane, F put) {
    settle();
    run.finish();
    const int r = lane / 4, c = lane % 4;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int j = 0; j < NU; ++j)
#pragma unroll
        for (int off = 4; off < 32; off *= 2) mid[j][k] += __shfl_xor_sync(0xffffffffu, mid[j][k], off);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            put(Y::col(c, k), (2 * i + (c >> 1)) * 32 + 4 * r + (BITS == 4 ? t + 2 * h : 2 * t + h),
                fmaf(o[i][t][2 * h + k] * (1.f / (P_SCALE * code_unit<BITS>(t))), run.bound(NU == PAIRS ? i : 0),
                     mid[NU == PAIRS ? i : 0][k]));
    }
  }
};

__device__ __forceinline__ void put_out(const AttnParams& p, int64_t kv, int col, int dim, float x) {
  const int64_t at = (kv * p.groups + col % p.groups) * p.so_h + (int64_t)(col / p.groups) * p.so_t + dim;
  if (p.dtype == BB_BF16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p.out)[at] = __float2half_rn(x);
}

// Merges the splits of one tile of query rows: weights first (a warp a row), then four dimensions of a row a thread,
// the splits dealt to several threads where there are more threads than that. A row that sees no key (a sum
// of 0) gives zeros.
template <int COLS, int D, int THREADS>
__device__ __forceinline__ void combine(const AttnParams& p, int64_t tile, int64_t kv, int col0, float* smem) {
  float4* red = reinterpret_cast<float4*>(smem);  // [THREADS]
  float* wt = smem + THREADS * 4;                 // [splits][COLS] weights of the splits in the result
  constexpr int ITEMS = COLS * D / 4, PARTS = ITEMS < THREADS ? THREADS / ITEMS : 1, EARLY = 8;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, splits = p.splits;
  const float2* ml = p.part_ml + tile * splits * COLS;
  const float4* acc = reinterpret_cast<const float4*>(p.part_acc + tile * splits * COLS * D);
  const int cols = min(COLS, p.cols - col0);
  const int item0 = threadIdx.x % (PARTS > 1 ? ITEMS : THREADS), part = PARTS > 1 ? threadIdx.x / ITEMS : 0;
  // this thread's first partial results, asked for before the weights are known
  float4 early[EARLY];
#pragma unroll
  for (int k = 0; k < EARLY; ++k) {
    const int s = part + k * PARTS;
    early[k] = part < PARTS && s < splits && item0 / (D / 4) < cols ? __ldcg(acc + (int64_t)s * ITEMS + item0) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int col = warp; col < cols; col += THREADS / 32) {
    float M = M_NONE, L = 0.f;
    for (int s0 = 0; s0 < splits; s0 += 64) {  // two splits a lane at a time, kept for their weights
      float2 v[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int s = s0 + k * 32 + lane;
        v[k] = s < splits ? __ldcg(ml + s * COLS + col) : make_float2(M_NONE, 0.f);
      }
      float top = fmax3(M, v[0].x, v[1].x);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      L *= fast_exp2(M - top);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int s = s0 + k * 32 + lane;
        if (s < splits) wt[s * COLS + col] = v[k].x;
        L = fmaf(fast_exp2(v[k].x - top), v[k].y, L);  // M_NONE: 0, or 1 with a sum of 0 where no split has a key
      }
      M = top;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    const float scale = L == 0.f ? 0.f : 1.f / L;
    for (int s = lane; s < splits; s += 32) wt[s * COLS + col] = fast_exp2(wt[s * COLS + col] - M) * scale;
  }
  __syncthreads();
  for (int i0 = 0; i0 < ITEMS; i0 += THREADS) {
    const int item = i0 + item0, col = item / (D / 4);
    const bool mine = part < PARTS && item < ITEMS && col < cols;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int s, const float4& v) {
      const float w = wt[s * COLS + col];
      a.x = fmaf(w, v.x, a.x);
      a.y = fmaf(w, v.y, a.y);
      a.z = fmaf(w, v.z, a.z);
      a.w = fmaf(w, v.w, a.w);
    };
    if (mine) {
      int s = part;
      if (i0 == 0) {
#pragma unroll
        for (int k = 0; k < EARLY; ++k, s += PARTS)
          if (s < splits) add(s, early[k]);
      }
#pragma unroll 8
      for (; s < splits; s += PARTS) add(s, __ldcg(acc + (int64_t)s * ITEMS + item));
    }
    if (PARTS > 1) {
      red[threadIdx.x] = a;
      __syncthreads();
      if (mine && part == 0)
        for (int k = 1; k < PARTS; ++k) {
          const float4 v = red[k * ITEMS + item];
          a.x += v.x;
          a.y += v.y;
          a.z += v.z;
          a.w += v.w;
        }
    }
    if (mine && part == 0) {
      const int dim = item % (D / 4) * 4;
      put_out(p, kv, col0 + col, dim, a.x);
      put_out(p, kv, col0 + col, dim + 1, a.y);
      put_out(p, kv, col0 + col, dim + 2, a.z);
      put_out(p, kv, col0 + col, dim + 3, a.w);
    }
  }
}

// Grid (splits * ztiles, kv_heads). A warp owns its ring of stages and takes steps split * W + warp, then every
// (splits * W)-th: no barrier until the warps' results are merged at the end. Adjacent warps take adjacent steps, so the
// lists and ends, which come last, spread over the warps that have one step less to do. (Sparse step, 64 + 16384 + 512 of
// 128K keys: 15.8 us; 8 query rows instead of 4 cost 21.0 instead of 16.9 us at 32K keys.)
template <int BITS, int G, int NG, bool SPLIT>
__global__ void __launch_bounds__(32 * warps<BITS, SPLIT>(), 1) qkv_partial_kernel(const AttnParams p) {
  using S = Stage<BITS, G, NG, true>;
  using Y = Layout<SPLIT>;
  constexpr int NS = stages(warps<BITS, SPLIT>(), S::BYTES), D = G * 32, W = warps<BITS, SPLIT>();
  extern __shared__ __align__(128) unsigned char smem[];
  const int lane = threadIdx.x % 32;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);  // known to be the same in all lanes
  const int64_t kv = blockIdx.y;
  const int split = blockIdx.x / p.ztiles, col0 = (blockIdx.x % p.ztiles) * Y::COLS;
  const uint32_t ring = smem_u32(smem) + warp * NS * S::BYTES;
  const Steps sp(p, false);
  const int first = split * W + warp, stride = p.splits * W;
  typename Query<BITS, G, NG, SPLIT>::Raw raw;
  Query<BITS, G, NG, SPLIT>::load(raw, p, kv, col0, lane);
  Source<BITS, G, NG, true> src(p, kv, lane, sp.bf + (int64_t)first * 32, (int64_t)stride * 32);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) src.fetch(p, sp, first + i * stride, ring + i * S::BYTES, kv, lane);
  Query<BITS, G, NG, SPLIT> q;
  q.take(raw, p, lane);
  Accum<BITS, G, NG, SPLIT> acc;
  acc.clear(lane);
  int since = 0;
  run_steps<NS>(
      p, sp, src, ring, first, stride, kv, lane,
      [&](uint32_t st) {
        acc.template step<false>(q, st, lane, Mask<SPLIT>());
        if (++since == SETTLE) {
          acc.settle();
          since = 0;
        }
      },
      [&](int u, uint32_t st) {
        Mask<SPLIT> mask;
        mask.set(p, sp, u, st + S::POS, col0, lane);
        acc.template step<true>(q, st, lane, mask);
        acc.settle();
      });
  __syncthreads();  // every warp is done with its ring

  float* sm = reinterpret_cast<float*>(smem);       // [W][COLS] maxima, sums, then [W][COLS][D]
  float* sl = sm + W * Y::COLS;
  float* so = sl + W * Y::COLS;
  acc.finish(lane, [&](int row, int dim, float x) { so[(warp * Y::COLS + row) * D + dim] = x; });
  if (lane < (SPLIT ? 2 : 4)) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      sm[warp * Y::COLS + Y::col(lane, k)] = acc.run.m[k];
      sl[warp * Y::COLS + Y::col(lane, k)] = acc.run.l[k];
    }
  }
  __syncthreads();
  const int64_t tile = kv * p.ztiles + blockIdx.x % p.ztiles;
  // Each warp's weight in each query row, and the row's maximum and sum; the maxima become the weights.
  __shared__ float2 row_ml[Y::COLS];
  for (int col = warp; col < Y::COLS; col += W) {
    const float m = lane < W ? sm[lane * Y::COLS + col] : M_NONE;
    float M = m;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    const float e = fast_exp2(m - M);
    float L = lane < W ? e * sl[lane * Y::COLS + col] : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    if (lane < W) sm[lane * Y::COLS + col] = e;
    if (lane == 0) row_ml[col] = make_float2(M, L);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < Y::COLS * D; i += 32 * W) {
    const int col = i / D, dim = i % D;
    if (col0 + col >= p.cols) break;
    float A = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) A = fmaf(sm[w * Y::COLS + col], so[(w * Y::COLS + col) * D + dim], A);
    const float2 ml = row_ml[col];
    if (p.splits == 1) {
      put_out(p, kv, col0 + col, dim, ml.y == 0.f ? 0.f : A / ml.y);
    } else {
      const int64_t at = (tile * p.splits + split) * Y::COLS + col;
      if (dim == 0) p.part_ml[at] = ml;
      p.part_acc[at * D + dim] = A;
    }
  }
  if (p.splits == 1 || !p.tickets) return;
  // The last CTA of the tile to arrive merges its splits, always in the same order.
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();  // the barrier's writes before it, of all threads, and the counter's after
    last = atomicAdd(p.tickets + tile, 1) == p.splits - 1;
    if (last) p.tickets[tile] = 0;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  combine<Y::COLS, D, 32 * W>(p, tile, kv, col0, reinterpret_cast<float*>(smem));
}

// The same merge as a kernel of its own, for calls without tickets: grid (ztiles, kv_heads).
template <int COLS, int D> __global__ void __launch_bounds__(256) qkv_combine_kernel(const AttnParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  const int64_t kv = blockIdx.y;
  combine<COLS, D, 256>(p, kv * p.ztiles + blockIdx.x, kv, blockIdx.x * COLS, reinterpret_cast<float*>(smem));
}

// p of four scores (two keys, two query rows) over the rows' sums: what they add to the two keys' pooled probabilities.
__device__ __forceinline__ void add_pooled(float (&part)[2], const float4& v, const float2& a, const float2& b) {
  part[0] = fmaf(fast_exp2(v.x - a.x), a.y, fmaf(fast_exp2(v.y - b.x), b.y, part[0]));
  part[1] = fmaf(fast_exp2(v.z - a.x), a.y, fmaf(fast_exp2(v.w - b.x), b.y, part[1]));
}
// The sums over the threads that share a key; thread c of four with one r ends up with key r (c even) or r + 8 (c odd) of
// tile c / 2, that is row pooled_key() of the step.
template <bool SPLIT> __device__ __forceinline__ float pooled(float (&part)[Layout<SPLIT>::TILES][2], int c) {
#pragma unroll
  for (int x = 0; x < Layout<SPLIT>::TILES; ++x)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      part[x][h] += __shfl_xor_sync(0xffffffffu, part[x][h], 1);
      if (!SPLIT) part[x][h] += __shfl_xor_sync(0xffffffffu, part[x][h], 2);
    }
  const int x = SPLIT ? 0 : c >> 1;
  return c & 1 ? part[x][1] : part[x][0];
}
__device__ __forceinline__ int pooled_key(int r, int c) { return (c >> 1) * 16 + (c & 1) * 8 + key_of(r); }

// (maximum, 1 / (sum * groups)) of query row h over its splits, by a warp.
__device__ __forceinline__ float2 merged_stats(const AttnParams& p, int64_t kv, int h, int lane) {
  float M = M_NONE, L = 0.f;
  const float2* ml = p.part_ml + (kv * p.groups + h) * p.splits;
  for (int s0 = 0; s0 < p.splits; s0 += 64) {
    float2 v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int s = s0 + k * 32 + lane;
      v[k] = s < p.splits ? __ldcg(ml + s) : make_float2(M_NONE, 0.f);
    }
    float top = fmax3(M, v[0].x, v[1].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    L *= fast_exp2(M - top);
#pragma unroll
    for (int k = 0; k < 2; ++k) L = fmaf(fast_exp2(v[k].x - top), v[k].y, L);
    M = top;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
  return make_float2(M, 1.f / (L * (float)p.groups));
}

// Waits until `want` arrivals are counted; false if the wait limit runs out (the fault code is then recorded).
__device__ __forceinline__ bool wait_arrivals(const int32_t* count, int want) {
  unsigned long long t0 = 0;
  for (uint32_t i = 1;; ++i) {
    int32_t seen;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(seen) : "l"(count) : "memory");
    if (seen >= want) return true;
    if (i % 64 == 0) {
      const unsigned long long now = tc::gtimer();
      if (t0 == 0) t0 = now;
      if (now - t0 > *(volatile unsigned long long*)&tc::g_tc_wait_ns) {
        atomicCAS(&tc::g_tc_fault, 0, 48);
        return false;
      }
    }
  }
}

// Shared memory of the scores' kernels: the ring, and (FUSED) scores of as many steps a warp as fit.
template <int BITS, int G, int NG, bool SPLIT> struct ScoreSmem {
  static constexpr int RING = SCORE_WARPS * SCORE_STAGES * Stage<BITS, G, NG, false>::BYTES;
  static constexpr int STEP = Layout<SPLIT>::TILES * 512;
  static constexpr int KEPT = (224 * 1024 - RING) / (SCORE_WARPS * STEP);
  static constexpr int FUSED_BYTES = RING + SCORE_WARPS * KEPT * STEP;
};

// Grid (splits * ztiles, kv_heads): the K half of qkv_partial_kernel, and the statistics of this CTA's scores.
//   FUSED (one ztile, tickets, all CTAs resident by a cooperative launch): scores stay in shared memory as far as they fit
//     (the rest goes to memory and comes back from L2); the CTAs of a KV head wait for each other's statistics, then
//     every warp pools the steps that it scored.
//   else: scores go to memory for qkv_pool_kernel, as the threads hold them: [kv][step][ztile][score tile][lane].
template <int BITS, int G, int NG, bool SPLIT, bool FUSED>
__global__ void __launch_bounds__(32 * SCORE_WARPS, 1) qkv_scores_kernel(const AttnParams p) {
  using S = Stage<BITS, G, NG, false>;
  using Y = Layout<SPLIT>;
  using M = ScoreSmem<BITS, G, NG, SPLIT>;
  constexpr int NS = SCORE_STAGES, W = SCORE_WARPS, SETS = Y::TILES;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float sm[W][Y::COLS], sl[W][Y::COLS];
  const int lane = threadIdx.x % 32;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);  // known to be the same in all lanes
  const int r = lane / 4, c = lane % 4;
  const int64_t kv = blockIdx.y;
  if (!FUSED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int split = blockIdx.x / p.ztiles, col0 = (blockIdx.x % p.ztiles) * Y::COLS;
  const uint32_t ring = smem_u32(smem) + warp * NS * S::BYTES;
  const Steps sp(p, true);
  const int first = split * W + warp, stride = p.splits * W;
  typename Query<BITS, G, NG, SPLIT>::Raw raw;
  Query<BITS, G, NG, SPLIT>::load(raw, p, kv, col0, lane);
  Source<BITS, G, NG, false> src(p, kv, lane, (int64_t)first * 32, (int64_t)stride * 32);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) src.fetch(p, sp, first + i * stride, ring + i * S::BYTES, kv, lane);
  Query<BITS, G, NG, SPLIT> q;
  q.take(raw, p, lane);
  float m[2], l[2];  // of this thread's keys
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    m[k] = M_NONE;
    l[k] = 0.f;
  }
  const int64_t per_step = (int64_t)p.ztiles * SETS * 32, jump = stride * per_step;
  float4* const out0 = p.scores + (kv * p.steps + first) * per_step + blockIdx.x % p.ztiles * SETS * 32 + lane;
  float4* const kept0 = reinterpret_cast<float4*>(smem + M::RING + warp * (M::KEPT * M::STEP)) + lane;
  float4 *out = out0, *kept = kept0, *const kept_end = kept0 + M::KEPT * SETS * 32;
  auto take = [&](uint32_t st, bool whole, int keys) {  // keys: those of the step from this thread's first on
    float s[SETS][4];
    step_scores<BITS, G, NG, SPLIT>(q, st, st + S::KM, lane, s);
    bool move = false;
#pragma unroll
    for (int x = 0; x < SETS; ++x) {
      float(&v)[4] = s[x];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] *= q.mul[i & 1];
        if (!whole && Y::tile(x, c) * 16 + i / 2 * 8 >= keys) v[i] = -INFINITY;
      }
      const float4 four = make_float4(v[0], v[1], v[2], v[3]);
      if (FUSED && kept < kept_end) kept[x * 32] = four;
      else out[x * 32] = four;
#pragma unroll
      for (int k = 0; k < 2; ++k) move |= fmaxf(v[k], v[2 + k]) > m[k] + LAZY;
    }
    if (FUSED) kept += SETS * 32;
    out += jump;
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float next = m[k];
#pragma unroll
        for (int x = 0; x < SETS; ++x) next = fmax3(next, s[x][k], s[x][2 + k]);
        l[k] *= fast_exp2(m[k] - next);
        m[k] = next;
      }
    }
#pragma unroll
    for (int x = 0; x < SETS; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) l[i & 1] += fast_exp2(s[x][i] - m[i & 1]);
  };
  run_steps<NS>(p, sp, src, ring, first, stride, kv, lane, [&](uint32_t st) { take(st, true, 32); },
                [&](int u, uint32_t st) { take(st, false, sp.n - u * 32 - key_of(r)); });
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float top = m[k];
#pragma unroll
    for (int off = SPLIT ? 2 : 4; off < 32; off *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    float sum = l[k] * fast_exp2(m[k] - top);
#pragma unroll
    for (int off = SPLIT ? 2 : 4; off < 32; off *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (r == 0 && (!SPLIT || c < 2)) {
      sm[warp][Y::col(c, k)] = top;
      sl[warp][Y::col(c, k)] = sum;
    }
  }
  __syncthreads();
  const int col = threadIdx.x;
  if (col < Y::COLS && col0 + col < p.cols) {
    float top = M_NONE, sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, sm[w][col]);
#pragma unroll
    for (int w = 0; w < W; ++w) sum = fmaf(fast_exp2(sm[w][col] - top), sl[w][col], sum);
    p.part_ml[(kv * p.groups + col0 + col) * p.splits + split] = make_float2(top, sum);
  }
  if constexpr (FUSED) {
    __shared__ float2 stats[Y::COLS];
    __shared__ bool all;
    int32_t* arrived = p.tickets + 2 * kv;  // and [1]: those that have left the wait
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();  // the barrier's writes before it, of all threads
      atomicAdd(arrived, 1);
      all = wait_arrivals(arrived, p.splits);
      // Every CTA arrives once and then leaves once, whether or not its wait ran out, so the last to leave comes after all
      // arrivals: the counters are zero again after every launch.
      if (atomicAdd(arrived + 1, 1) == p.splits - 1) arrived[0] = arrived[1] = 0;
      __threadfence();
    }
    __syncthreads();
    if (warp < Y::COLS) {
      float2 v = make_float2(0.f, 0.f);
      if (!all) v = make_float2(NAN, NAN);  // the wait ran out: NaN in the place of this CTA's probabilities
      else if (warp < p.groups) v = merged_stats(p, kv, warp, lane);
      if (lane == 0) stats[warp] = v;
    }
    __syncthreads();
    const float2 a = stats[Y::col(c, 0)], b = stats[Y::col(c, 1)];
    const int64_t from = p.front, to = sp.n - p.window;  // pooled keys: [from, to)
    float* probs = p.probs + kv * p.cap;
    kept = kept0;
    out = out0;
    for (int u = first; u < sp.total; u += stride, kept += SETS * 32, out += jump) {
      const int64_t key = (int64_t)u * 32, pos = key + pooled_key(r, c);
      float sum = -1.f;
      if (key < to && key + 32 > from) {
        float part[SETS][2] = {};
#pragma unroll
        for (int x = 0; x < SETS; ++x) add_pooled(part[x], kept < kept_end ? kept[x * 32] : out[x * 32], a, b);
        sum = pooled<SPLIT>(part, c);
      }
      if (pos < p.cap) probs[pos] = pos >= from && pos < to ? sum : -1.f;
    }
    for (int64_t pos = (int64_t)sp.total * 32 + split * (32 * W) + threadIdx.x; pos < p.cap; pos += (int64_t)p.splits * 32 * W)
      probs[pos] = -1.f;
  }
}

// Grid (blocks of 8 POOL_STEPS steps, kv_heads): a warp pools steps of 32 keys, whose scores it asks for before the
// statistics are merged. Starts while qkv_scores_kernel runs and waits for its end.
constexpr int POOL_STEPS = 4;
template <bool SPLIT> __global__ void __launch_bounds__(256) qkv_pool_kernel(const AttnParams p) {
  using Y = Layout<SPLIT>;
  constexpr int SETS = Y::TILES;
  extern __shared__ float2 row_stats[];  // [ztiles * COLS]
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = lane / 4, c = lane % 4;
  const int64_t kv = blockIdx.y;
  const int u0 = (blockIdx.x * 8 + warp) * POOL_STEPS;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t n = cache_len(p), from = p.front, to = n - p.window;  // pooled keys: [from, to)
  const float4* in = p.scores + kv * p.steps * p.ztiles * SETS * 32 + lane;
  const int64_t per_step = (int64_t)p.ztiles * SETS * 32;
  float4 early[POOL_STEPS][SETS];
#pragma unroll
  for (int i = 0; i < POOL_STEPS; ++i) {
    const int64_t key = (int64_t)(u0 + i) * 32;
#pragma unroll
    for (int x = 0; x < SETS; ++x)
      if (key < to && key + 32 > from) early[i][x] = in[(u0 + i) * per_step + x * 32];
  }
  for (int h = warp; h < p.ztiles * Y::COLS; h += 8) {
    const float2 v = h < p.groups ? merged_stats(p, kv, h, lane) : make_float2(0.f, 0.f);
    if (lane == 0) row_stats[h] = v;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < POOL_STEPS; ++i) {
    const int64_t key = (int64_t)(u0 + i) * 32, pos = key + pooled_key(r, c);
    if (key >= p.cap) return;
    float sum = -1.f;
    if (key < to && key + 32 > from) {
      float part[SETS][2] = {};
      for (int z = 0; z < p.ztiles; ++z)
#pragma unroll
        for (int x = 0; x < SETS; ++x)
          add_pooled(part[x], z == 0 ? early[i][x] : in[(u0 + i) * per_step + (z * SETS + x) * 32],
                     row_stats[z * Y::COLS + Y::col(c, 0)], row_stats[z * Y::COLS + Y::col(c, 1)]);
      sum = pooled<SPLIT>(part, c);
    }
    if (pos < p.cap) p.probs[kv * p.cap + pos] = pos >= from && pos < to ? sum : -1.f;
  }
}

struct AttnPlan {
  int64_t splits, ztiles, cols;
  int columns;  // 4 (SPLIT) or 8 query rows a warp
  size_t ml_bytes, acc_bytes, scores_bytes, probs_bytes, topk_bytes, total;
};

int check_attn(const bb_qkv_attn_args* a, const char* what, bool need_v) {
  if (!a) return fail(BB_ERR_ARG, "%s: null args", what);
  int st = qkv::check_cache(a->cache, what, true, need_v);
  if (st) return st;
  if (a->dtype != BB_F16 && a->dtype != BB_BF16) return fail(BB_ERR_DTYPE, "%s requires fp16 or bf16 queries", what);
  if (a->heads <= 0 || a->heads % a->cache.kv_heads || a->heads > 65535)
    return fail(BB_ERR_SHAPE, "%s: heads must be a positive multiple of kv_heads (at most 65535)", what);
  if (a->heads / a->cache.kv_heads > 1024) return fail(BB_ERR_UNSUPPORTED, "%s: at most 1024 query heads a KV head", what);
  if (a->t <= 0 || a->t > ((int64_t)1 << 30) / a->heads)  // query rows are counted in 32 bits
    return fail(BB_ERR_SHAPE, "%s: heads * tokens must lie in [1, 2^30]", what);
  if (a->n < 0 || a->n > a->cache.cap) return fail(BB_ERR_ARG, "%s: n must lie in [0, capacity]", what);
  if (a->front < 0 || a->window < 0) return fail(BB_ERR_ARG, "%s: front and window must be >= 0", what);
  if (a->route_k < 0) return fail(BB_ERR_ARG, "%s: bad route count", what);
  if (a->splits < 0) return fail(BB_ERR_ARG, "%s: splits must be >= 0", what);
  return BB_OK;
}

// The splits of the key list: one wave of CTAs, one a SM, and no more than one step of 32 keys a warp. Up to 4
// query rows share products (SPLIT, d = 64 or 128), more go 8 at a time.
void plan_grid(const bb_qkv_attn_args* a, int64_t steps, bool decode, AttnPlan* pl) {
  pl->cols = a->heads / a->cache.kv_heads * a->t;
  pl->columns = pl->cols <= 4 && a->cache.d % 64 == 0 ? 4 : 8;
  pl->ztiles = cdiv(pl->cols, (int64_t)pl->columns);
  const int64_t w = !decode ? SCORE_WARPS : (pl->columns == 8 || a->cache.bits == 8 ? warps<8, true>() : warps<4, true>());
  const int64_t s = a->splits > 0 ? a->splits : std::max<int64_t>(1, (int64_t)num_sms() / (a->cache.kv_heads * pl->ztiles));
  pl->splits = std::max<int64_t>(1, std::min<int64_t>({s, cdiv(steps, w), (int64_t)1024, INT32_MAX / pl->ztiles}));
}

int plan_decode(const bb_qkv_attn_args* a, AttnPlan* pl) {
  int st = check_attn(a, "qkv_decode", true);
  if (st) return st;
  if (a->route_k > 0 && a->route_rows != a->cache.kv_heads && a->route_rows != a->heads)
    return fail(BB_ERR_SHAPE, "qkv_decode: indices must be [Hkv, R] (pooled) or [H, R] (per head)");
  *pl = {};
  // with a length on the device the grid is planned for a full cache
  const int64_t n = a->n_dev ? a->cache.cap : a->n;
  const int64_t f = std::min(a->front, n), w = std::min(n - f, std::min(a->window, n) + a->t - 1);
  const int64_t lists = a->route_k > 0 && a->route_rows != a->cache.kv_heads ? a->heads / a->cache.kv_heads : 1;
  if (a->route_k > ((int64_t)1 << 27) / lists) return fail(BB_ERR_UNSUPPORTED, "qkv_decode: too many routed keys");
  plan_grid(a, cdiv(f, (int64_t)32) + cdiv(w, (int64_t)32) + lists * cdiv(a->route_k, (int64_t)32), true, pl);
  // partial results, of which a single split has none
  const int64_t rows = pl->splits == 1 ? 0 : a->cache.kv_heads * pl->ztiles * pl->columns * pl->splits;
  pl->ml_bytes = align_up((size_t)rows * 8, 256);
  pl->acc_bytes = align_up((size_t)(rows * a->cache.d) * 4, 256);
  pl->total = std::max<size_t>(pl->ml_bytes + pl->acc_bytes, 256);
  return BB_OK;
}

int plan_route(const bb_qkv_attn_args* a, AttnPlan* pl) {
  int st = check_attn(a, "qkv_route", false);
  if (st) return st;
  if (a->t != 1) return fail(BB_ERR_SHAPE, "qkv_route: one token at a time");
  if (a->route_k > a->cache.cap) return fail(BB_ERR_ARG, "qkv_route: route_k must lie in [0, capacity]");
  *pl = {};
  plan_grid(a, cdiv(a->n_dev ? a->cache.cap : a->n, (int64_t)32), false, pl);
  pl->ml_bytes = align_up((size_t)(a->heads * pl->splits) * 8, 256);
  // a step of 32 keys: 4 (SPLIT) or 8 scores a key and ztile
  pl->scores_bytes = (size_t)(a->cache.kv_heads * cdiv(a->cache.cap, (int64_t)32) * pl->ztiles * pl->columns) * 128;
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
  p.q16 = qkv::al16(a->q) && a->sq_h % 8 == 0 && (a->t == 1 || a->sq_t % 8 == 0);
  p.idx = a->idx; p.si_r = a->si_r;
  p.route_k = a->route_k;
  p.idx64 = a->idx_i64 != 0;
  p.per_head = a->route_k > 0 && a->route_rows != c.kv_heads;
  p.n_dev = a->n_dev;
  p.n = a->n; p.cap = c.cap;
  p.front = a->front; p.window = a->window;
  p.d = (int)c.d;
  p.heads = (int)a->heads; p.groups = (int)(a->heads / c.kv_heads);
  p.t = (int)a->t; p.cols = (int)pl.cols;
  p.splits = (int)pl.splits; p.ztiles = (int)pl.ztiles; p.dtype = a->dtype;
  p.scale_log2 = a->scale * LOG2E;
  p.part_ml = reinterpret_cast<float2*>(ws);
  p.part_acc = reinterpret_cast<float*>(ws + pl.ml_bytes);
  p.scores = reinterpret_cast<float4*>(ws + pl.ml_bytes);
  p.steps = cdiv(c.cap, (int64_t)32);
  p.probs = a->out_probs ? a->out_probs : reinterpret_cast<float*>(ws + pl.ml_bytes + pl.scores_bytes);
  p.out = a->out; p.so_h = a->so_h; p.so_t = a->so_t;
  return p;
}

// Lets a kernel use all of a SM's shared memory: once a device and kernel (the attribute call costs as much host time as
// a third of a launch).
template <typename K> int allow_smem(K* kernel, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) dev = -1;
  if (dev >= 0 && (done.load(std::memory_order_acquire) >> dev & 1)) return BB_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024);
  if (e != cudaSuccess) return fail(BB_ERR_LAUNCH, "qkv attention: %s", cudaGetErrorString(e));
  if (dev >= 0) done.fetch_or(uint64_t{1} << dev, std::memory_order_release);
  return BB_OK;
}

template <bool DECODE, int BITS, int G, int NG, bool SPLIT>
int launch(const AttnParams& p, int64_t kv_heads, cudaStream_t stream) {
  const dim3 grid((unsigned)(p.splits * p.ztiles), (unsigned)kv_heads);
  if constexpr (DECODE) {
    const size_t smem = partial_smem<BITS, G, NG, SPLIT>(p.splits);
    auto* kernel = qkv_partial_kernel<BITS, G, NG, SPLIT>;
    static std::atomic<uint64_t> done{0};
    const int st = allow_smem(kernel, done);
    if (st) return st;
    kernel<<<grid, 32 * warps<BITS, SPLIT>(), smem, stream>>>(p);
    BB_CHECK_LAUNCH("qkv_partial_kernel");
    if (p.splits > 1 && !p.tickets) {
      constexpr int COLS = Layout<SPLIT>::COLS;
      const size_t merge = combine_floats<COLS, 256>(p.splits) * 4;  // at most 36 KB (1024 splits)
      qkv_combine_kernel<COLS, G * 32><<<dim3((unsigned)p.ztiles, (unsigned)kv_heads), 256, merge, stream>>>(p);
      BB_CHECK_LAUNCH("qkv_combine_kernel");
    }
  } else {
    using M = ScoreSmem<BITS, G, NG, SPLIT>;
    static std::atomic<uint64_t> done[2]{};
    if (p.tickets) {  // see plan_route
      auto* kernel = qkv_scores_kernel<BITS, G, NG, SPLIT, true>;
      const int st = allow_smem(kernel, done[0]);
      if (st) return st;
      cudaLaunchAttribute together{};
      together.id = cudaLaunchAttributeCooperative;
      together.val.cooperative = 1;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = grid;
      cfg.blockDim = dim3(32 * SCORE_WARPS);
      cfg.dynamicSmemBytes = M::FUSED_BYTES;
      cfg.stream = stream;
      cfg.attrs = &together;
      cfg.numAttrs = 1;
      const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
      if (e != cudaSuccess) return fail(BB_ERR_LAUNCH, "qkv_scores_kernel: %s", cudaGetErrorString(e));
    } else {
      auto* kernel = qkv_scores_kernel<BITS, G, NG, SPLIT, false>;
      const int st = allow_smem(kernel, done[1]);
      if (st) return st;
      kernel<<<grid, 32 * SCORE_WARPS, M::RING, stream>>>(p);
    }
    BB_CHECK_LAUNCH("qkv_scores_kernel");
  }
  return BB_OK;
}

template <bool SPLIT> int launch_pool(const AttnParams& p, int64_t kv_heads, cudaStream_t stream) {
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)cdiv(p.steps, (int64_t)8 * POOL_STEPS), (unsigned)kv_heads);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = (size_t)p.ztiles * Layout<SPLIT>::COLS * 8;
  cfg.stream = stream;
  cfg.attrs = &overlap;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, qkv_pool_kernel<SPLIT>, p);
  if (e != cudaSuccess) return fail(BB_ERR_LAUNCH, "qkv_pool_kernel: %s", cudaGetErrorString(e));
  BB_CHECK_LAUNCH("qkv_pool_kernel");
  return BB_OK;
}

template <bool DECODE, int BITS, int G, int NG>
int launch_columns(const AttnParams& p, int columns, int64_t kv_heads, cudaStream_t stream) {
  if constexpr (G % 2 == 0)
    if (columns == 4) return launch<DECODE, BITS, G, NG, true>(p, kv_heads, stream);
  return launch<DECODE, BITS, G, NG, false>(p, kv_heads, stream);
}

template <bool DECODE, int BITS>
int launch_shape(const AttnParams& p, int pairs, int columns, int64_t kv_heads, cudaStream_t stream) {
  switch (p.d / 32 * 8 + pairs) {
    case 1 * 8 + 1: return launch_columns<DECODE, BITS, 1, 1>(p, columns, kv_heads, stream);
    case 2 * 8 + 1: return launch_columns<DECODE, BITS, 2, 1>(p, columns, kv_heads, stream);
    case 2 * 8 + 2: return launch_columns<DECODE, BITS, 2, 2>(p, columns, kv_heads, stream);
    case 3 * 8 + 1: return launch_columns<DECODE, BITS, 3, 1>(p, columns, kv_heads, stream);
    case 3 * 8 + 3: return launch_columns<DECODE, BITS, 3, 3>(p, columns, kv_heads, stream);
    case 4 * 8 + 1: return launch_columns<DECODE, BITS, 4, 1>(p, columns, kv_heads, stream);
    case 4 * 8 + 2: return launch_columns<DECODE, BITS, 4, 2>(p, columns, kv_heads, stream);
    case 4 * 8 + 4: return launch_columns<DECODE, BITS, 4, 4>(p, columns, kv_heads, stream);
    default: return fail(BB_ERR_UNSUPPORTED, "qkv attention: head_dim %d with %d groups", p.d, pairs);
  }
}

template <bool DECODE>
int launch_attn(const bb_qkv_attn_args* a, const AttnParams& p, int columns, cudaStream_t stream) {
  const int pairs = (int)(a->cache.d / a->cache.group);
  return a->cache.bits == 4 ? launch_shape<DECODE, 4>(p, pairs, columns, a->cache.kv_heads, stream)
                            : launch_shape<DECODE, 8>(p, pairs, columns, a->cache.kv_heads, stream);
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
  if (a->tickets && a->n_tickets >= a->cache.kv_heads * pl.ztiles) p.tickets = a->tickets;
  return launch_attn<true>(a, p, pl.columns, stream);
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
  // One launch, where the CTAs can wait for each other: all of them resident (one a SM), all query rows of a KV head in
  // one ztile. Measured at 128K keys, 8 x 4 heads, 4 bits: 24.9 us, with two launches 29.7.
  if (a->tickets && a->n_tickets >= 2 * a->cache.kv_heads && pl.ztiles == 1 && pl.splits * a->cache.kv_heads <= num_sms())
    p.tickets = a->tickets;
  st = launch_attn<false>(a, p, pl.columns, stream);
  if (st) return st;
  if (!p.tickets)
    st = pl.columns == 4 ? launch_pool<true>(p, a->cache.kv_heads, stream)
                         : launch_pool<false>(p, a->cache.kv_heads, stream);
  if (st) return st;
  if (a->route_k > 0 && a->out_idx)
    return topk_sorted(p.probs, a->cache.kv_heads, a->cache.cap, a->route_k, a->out_idx, a->out_idx_i64 != 0, a->so_i,
                       w + pl.ml_bytes + pl.scores_bytes + pl.probs_bytes, pl.topk_bytes, stream);
  return BB_OK;
}

int qkv_set_wait_limit(unsigned long long ns) { return tc::unit_set_wait_limit(ns); }

int qkv_fault_take(int* code) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, tc::g_tc_fault, sizeof(int));
  if (e != cudaSuccess) return fail(BB_ERR_LAUNCH, "device_fault: %s", cudaGetErrorString(e));
  if (v) {
    const int zero = 0;
    cudaMemcpyToSymbol(tc::g_tc_fault, &zero, sizeof(int));
  }
  *code = v;
  return BB_OK;
}

}  // namespace bb
