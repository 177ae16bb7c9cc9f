// Attention of the newest tokens over a quantised KV cache, and decode routing over its keys
// (semantics: include/bb_b200.h, bb_qkv_decode and bb_qkv_route).
//
//   qkv_partial_kernel  up to 8 NT query rows of one KV head over one split of its key list: running max,
//                       sum and P.V of the split, in fp32
//   qkv_combine_kernel  merges the splits of a row
//   qkv_scores_kernel   log2 scores of every key for the query heads of a KV head, and per-split softmax
//                       statistics
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
// are the 16 rows of a product and the query rows its 8 columns, so four query heads of a KV head waste
// half a column tile rather than three quarters of a row tile.
//   q: fp16 after a power of two that brings the row's largest element to [2^14, 2^15) (exact for bf16
// and fp16 queries, except elements below 2^-28 of the largest, which lose relative precision only).
//   p s: rounded to fp16 once, scaled by powers of two (a running bound of the steps, the running
// maximum of the scores) to at most 2^15, so that p down to 2^-29 of the largest keeps all 11 bits.
// Scores, exponentials, sums and accumulators are fp32.
#include <algorithm>

#include "qkv.cuh"

namespace bb {

int topk_sorted(const float* vals, int64_t rows, int64_t n, int64_t k, void* out, bool out64, int64_t so_h,
                void* scratch, size_t scratch_bytes, cudaStream_t stream);
size_t topk_scratch_bytes(int64_t rows, int64_t n, int64_t k);

namespace {

constexpr int WARPS = 8;
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
  int d, heads, groups, t, cols, gp, splits, ztiles, dtype;
  float scale_log2;
  float2* part_ml;  // [heads * t][splits] (max in log2 units, sum); routing: [heads][splits]
  float* part_acc;  // [heads * t][splits][d]
  void* out; int64_t so_h, so_t;
  float* scores;    // routing: [kv_heads][cap][gp] log2 units
  float* probs;     // [kv_heads][cap]
};

__device__ __forceinline__ int64_t cache_len(const AttnParams& p) {
  if (!p.n_dev) return p.n;
  const int64_t n = *p.n_dev;
  return n < 0 ? 0 : (n > p.cap ? p.cap : n);
}

// The key list of one KV head, as tiles of 16: front keys [0, fa), window keys [b0, n) of any of the
// tokens, and lists (one, or one for each query head).
struct Tiles {
  int n, fa, b0, na, nb, nc, total;
  __device__ __forceinline__ Tiles(const AttnParams& p, bool all) {
    const int64_t len = cache_len(p);
    n = (int)len;
    const int64_t f = all ? 0 : (p.front < len ? p.front : len);
    const int64_t w = all ? 0 : max(f, len - p.t + 1 - p.window);
    fa = (int)f;
    b0 = (int)min(w, len);
    na = (fa + 15) / 16;
    nb = (n - b0 + 15) / 16;
    nc = all ? 0 : (int)((p.route_k + 15) / 16);
    total = na + nb + nc * (p.per_head ? p.groups : 1);
  }
};

template <int BITS, int G, int NG, bool WITH_V> struct Stage {
  static constexpr int ROW = G * 4 * BITS;                // bytes of codes a row
  static constexpr int META = NG * 4;                     // bytes of (step, low) pairs a row
  static constexpr int K = 0, V = 16 * ROW;
  static constexpr int KM = (WITH_V ? 2 : 1) * 16 * ROW, VM = KM + 16 * META;
  static constexpr int POS = KM + (WITH_V ? 2 : 1) * 16 * META;
  static constexpr int BYTES = POS + (WITH_V ? 64 : 0);
  static_assert(BYTES % 16 == 0, "stages start on 16-byte boundaries");
};

// Key j of a tile feeds row slot(j) of the K product, so that the keys of a thread's V operands
// (slots 2c, 2c + 1, 2c + 8, 2c + 9) are the tile's rows c, c + 4, c + 8, c + 12, whose reads from shared
// memory fall into different banks.
__device__ __forceinline__ int slot_of(int j) { return (j & 8) | ((j & 3) << 1) | ((j >> 2) & 1); }
__device__ __forceinline__ int key_of(int r) { return ((r & 1) << 2) | (r >> 1); }  // r < 8

// 16-byte chunks of a staged row are stored at chunk ^ swizzle(row), against bank conflicts: K reads take a
// quarter row a thread, V reads an eighth of rows c.
template <int ROW> __device__ __forceinline__ int k_swizzle(int slot) { return ROW == 128 ? (slot & 1) : 0; }
template <int ROW> __device__ __forceinline__ int v_swizzle(int row) {
  return ROW == 128 ? (row & 3) << 1 : (ROW == 64 ? row & 2 : 0);
}

template <int N> __device__ __forceinline__ void cp_async_n(uint32_t dst, const void* src, bool valid) {
  if constexpr (N == 16)
    cp_async_16(dst, src, valid);
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(dst), "l"(src), "n"(N), "r"(valid ? N : 0));
}

// Copies tile `tau` of the key list into a stage (asynchronous; rows that are no keys become zeros).
template <int BITS, int G, int NG, bool WITH_V>
__device__ __forceinline__ void fetch(const AttnParams& p, const Tiles& tl, int tau, uint32_t st, int64_t kv, int lane) {
  using S = Stage<BITS, G, NG, WITH_V>;
  constexpr int CH = S::ROW / 16;  // chunks a row
  const unsigned char* kc = p.kc + kv * p.kc_h;
  const unsigned char* vc = WITH_V ? p.vc + kv * p.vc_h : nullptr;
  int mine;   // position of row lane % 16, or -1
  int base = 0;
  const bool listed = WITH_V && tau >= tl.na + tl.nb;
  if (!listed) {
    const bool a = tau < tl.na;
    base = a ? tau * 16 : tl.b0 + (tau - tl.na) * 16;
    mine = base + lane % 16;
    if (mine >= (a ? tl.fa : tl.n)) mine = -1;
  } else {
    const int u = tau - tl.na - tl.nb;
    const int list = u / tl.nc;
    const int64_t j = (int64_t)(u - list * tl.nc) * 16 + lane % 16;
    int64_t pos = -1;
    if (j < p.route_k) {
      const int64_t o = (p.per_head ? kv * p.groups + list : kv) * p.si_r + j;
      pos = p.idx64 ? static_cast<const int64_t*>(p.idx)[o] : (int64_t) static_cast<const int32_t*>(p.idx)[o];
    }
    mine = (pos >= tl.fa && pos < tl.n) ? (int)pos : -1;
    if (lane < 16) asm volatile("st.shared.s32 [%0], %1;" ::"r"(st + S::POS + slot_of(lane) * 4), "r"(mine) : "memory");
  }
#pragma unroll
  for (int i = 0; i < (16 * CH + 31) / 32; ++i) {
    const int x = lane + 32 * i;
    const int j = x / CH, ch = x % CH;
    const int pos = __shfl_sync(0xffffffffu, mine, j & 15);
    if (16 * CH % 32 == 0 || x < 16 * CH) {
      const int64_t off = (int64_t)(pos < 0 ? 0 : pos) * S::ROW + ch * 16;
      const int sl = slot_of(j);
      cp_async_16(st + S::K + sl * S::ROW + ((ch ^ k_swizzle<S::ROW>(sl)) << 4), kc + off, pos >= 0);
      if constexpr (WITH_V)
        cp_async_16(st + S::V + j * S::ROW + ((ch ^ v_swizzle<S::ROW>(j)) << 4), vc + off, pos >= 0);
    }
  }
  if (WITH_V || lane < 16) {
    const bool second = lane >= 16;
    const uint32_t* meta = (second ? p.vm + kv * p.vm_h : p.km + kv * p.km_h) + (int64_t)(mine < 0 ? 0 : mine) * NG;
    const uint32_t dst = st + (second ? S::VM : S::KM) + slot_of(lane % 16) * S::META;
    constexpr int N = NG == 3 ? 4 : S::META;
#pragma unroll
    for (int i = 0; i < S::META / N; ++i) cp_async_n<N>(dst + i * N, meta + i, mine >= 0);
  }
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
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float step_of(uint32_t m) { return __uint_as_float(m << 16); }
__device__ __forceinline__ float low_of(uint32_t m) { return __uint_as_float(m & 0xFFFF0000u); }

// The query side of a warp: operands for 8 NT columns (column = token * groups + head within the KV head's
// query heads), and, for this thread's columns 8 nt + 2c and + 1, the sums of each group's elements and
// the factor that turns (codes . operand) into a log2 score.
template <int BITS, int G, int NG, int NT> struct Query {
  uint32_t f[NT][G][2][2];
  float sum[NT][NG][2], mul[NT][2];

  __device__ __forceinline__ void load(const AttnParams& p, int64_t kv, int col0, int lane) {
    const int r = lane / 4, c = lane % 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = col0 + nt * 8 + r;
      float x[G][8];
      float top = 0.f;
      const int64_t at = col < p.cols ? (kv * p.groups + col % p.groups) * p.sq_h + (int64_t)(col / p.groups) * p.sq_t : 0;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t e = at + g * 32 + c * 8 + i;
          float v = 0.f;
          if (col < p.cols)
            v = p.dtype == BB_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[e])
                                   : __half2float(static_cast<const __half*>(p.q)[e]);
          x[g][i] = v;
          top = fmaxf(top, fabsf(v));
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
        // In the order in which codes come out of a word: 4 bits: (0,4) (2,6) at 2^-24 and (1,5) (3,7) at
        // 2^-20; 8 bits: (0,2) (1,3) and (4,6) (5,7), all at 2^-24.
        if constexpr (BITS == 4) {
          const float up16 = up * 16.f;
          f[nt][g][0][0] = pack2<__half>(x[g][0] * up16, x[g][4] * up16);
          f[nt][g][0][1] = pack2<__half>(x[g][2] * up16, x[g][6] * up16);
          f[nt][g][1][0] = pack2<__half>(x[g][1] * up, x[g][5] * up);
          f[nt][g][1][1] = pack2<__half>(x[g][3] * up, x[g][7] * up);
        } else {
          const float up16 = up * 16.f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            f[nt][g][h][0] = pack2<__half>(x[g][4 * h] * up16, x[g][4 * h + 2] * up16);
            f[nt][g][h][1] = pack2<__half>(x[g][4 * h + 1] * up16, x[g][4 * h + 3] * up16);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 1);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 2);
        s[i] *= up * 9.5367431640625e-07f;  // 2^-20: in units of the codes' products
#pragma unroll
        for (int k = 0; k < 2; ++k) sum[nt][i][k] = __shfl_sync(0xffffffffu, s[i], (2 * c + k) * 4);
      }
      const float m = p.scale_log2 * 1048576.f * down;
#pragma unroll
      for (int k = 0; k < 2; ++k) mul[nt][k] = __shfl_sync(0xffffffffu, m, (2 * c + k) * 4);
    }
  }
};

// Scores of a staged tile before the columns' factors: s[nt] = (key r, columns 2c, 2c + 1), (key r + 8, ...)
// by slot.
template <int BITS, int G, int NG, int NT>
__device__ __forceinline__ void tile_scores(const Query<BITS, G, NG, NT>& q, uint32_t rows, uint32_t meta, int lane,
                                            float (&s)[NT][4]) {
  constexpr int WPB = BITS / 4;  // words a block of 32 dimensions
  const int r = lane / 4, c = lane % 4;
  uint32_t w0[G * WPB], w1[G * WPB], m0[NG], m1[NG];
  k_words<BITS, G>(w0, rows, r, c);
  k_words<BITS, G>(w1, rows, r + 8, c);
  lds_words(m0, meta + r * NG * 4);
  lds_words(m1, meta + (r + 8) * NG * 4);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[nt][i] = 0.f;
#pragma unroll
  for (int gi = 0; gi < NG; ++gi) {
    float acc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
#pragma unroll
    for (int b = 0; b < G / NG; ++b) {
      const int g = gi * (G / NG) + b;
      uint32_t a[2][4];
      if constexpr (BITS == 4) {
        const uint32_t x0 = w0[g], x1 = w1[g], y0 = x0 >> 8, y1 = x1 >> 8;
        a[0][0] = x0 & 0x000F000Fu; a[0][1] = x1 & 0x000F000Fu; a[0][2] = y0 & 0x000F000Fu; a[0][3] = y1 & 0x000F000Fu;
        a[1][0] = x0 & 0x00F000F0u; a[1][1] = x1 & 0x00F000F0u; a[1][2] = y0 & 0x00F000F0u; a[1][3] = y1 & 0x00F000F0u;
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x0 = w0[2 * g + h], x1 = w1[2 * g + h];
          a[h][0] = x0 & 0x00FF00FFu; a[h][1] = x1 & 0x00FF00FFu;
          a[h][2] = (x0 >> 8) & 0x00FF00FFu; a[h][3] = (x1 >> 8) & 0x00FF00FFu;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_16816<__half>(acc[nt], a[0], q.f[nt][g][0]);
        mma_16816<__half>(acc[nt], a[1], q.f[nt][g][1]);
      }
    }
    const float s0 = step_of(m0[gi]), l0 = low_of(m0[gi]), s1 = step_of(m1[gi]), l1 = low_of(m1[gi]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        s[nt][k] = fmaf(s0, acc[nt][k], fmaf(l0, q.sum[nt][gi][k], s[nt][k]));
        s[nt][2 + k] = fmaf(s1, acc[nt][2 + k], fmaf(l1, q.sum[nt][gi][k], s[nt][2 + k]));
      }
  }
}

// Which of this thread's (key, column) pairs of a tile count.
template <int NT> struct Mask {
  bool ok[NT][4];
  // `front`: keys of [0, front) count for every token at or after them; else keys of the token's window.
  __device__ __forceinline__ void range(const AttnParams& p, const Tiles& tl, int tau, int col0, int lane) {
    const bool front = tau < tl.na;
    const int base = front ? tau * 16 : tl.b0 + (tau - tl.na) * 16;
    const int end = front ? tl.fa : tl.n;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pos = base + key_of(lane / 4) + (i / 2) * 8;
        const int own = tl.n - p.t + (col0 + nt * 8 + 2 * (lane % 4) + (i & 1)) / p.groups;
        ok[nt][i] = pos < end && pos <= own && (front || pos > own - p.window);
      }
  }
  __device__ __forceinline__ void listed(const AttnParams& p, const Tiles& tl, int tau, uint32_t positions, int col0, int lane) {
    const int list = (tau - tl.na - tl.nb) / tl.nc;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      int pos;
      asm volatile("ld.shared.s32 %0, [%1];" : "=r"(pos) : "r"(positions + (lane / 4 + half * 8) * 4));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int col = col0 + nt * 8 + 2 * (lane % 4) + k;
          const int own = tl.n - p.t + col / p.groups;
          ok[nt][half * 2 + k] = pos >= 0 && pos >= p.front && pos <= own - p.window &&
                                 (!p.per_head || col % p.groups == list);
        }
    }
  }
};

constexpr int stages(int bytes) { return bytes > 3000 ? 3 : 4; }
template <int BITS, int G, int NG, int NT> constexpr size_t partial_smem() {
  using S = Stage<BITS, G, NG, true>;
  const size_t ring = (size_t)WARPS * stages(S::BYTES) * S::BYTES;
  const size_t merge = (size_t)WARPS * 8 * NT * (G * 32 + 2) * 4;
  return ring > merge ? ring : merge;
}

// Grid (splits * ztiles, kv_heads). A warp owns its ring of stages and takes tiles split * WARPS + warp,
// then every (splits * WARPS)-th: no barrier until the warps' results are merged at the end.
template <int BITS, int G, int NG, int NT>
__global__ void __launch_bounds__(32 * WARPS, NT == 1 ? 2 : 1) qkv_partial_kernel(const AttnParams p) {
  using S = Stage<BITS, G, NG, true>;
  constexpr int NS = stages(S::BYTES), D = G * 32;
  extern __shared__ __align__(128) unsigned char smem[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int r = lane / 4, c = lane % 4;
  const int64_t kv = blockIdx.y;
  const int split = blockIdx.x / p.ztiles, col0 = (blockIdx.x % p.ztiles) * 8 * NT;
  const uint32_t ring = smem_u32(smem) + warp * NS * S::BYTES;
  const Tiles tl(p, false);
  const int first = split * WARPS + warp, stride = p.splits * WARPS;

#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    const int tau = first + i * stride;
    if (tau < tl.total) fetch<BITS, G, NG, true>(p, tl, tau, ring + i * S::BYTES, kv, lane);
    cp_async_commit();
  }
  Query<BITS, G, NG, NT> q;
  q.load(p, kv, col0, lane);

  float o[NT][G][2][4];           // P.V: block, tile of 16 dimensions
  float lows[NT][NG][2];          // sum p low, of this thread's keys
  float m[NT][2], l[NT][2];       // running maximum (log2 units), sum p of this thread's keys
  float bound = 7.8886090522101181e-31f;  // power of two above every step so far (2^-100: none)
  float pscale = P_SCALE / bound;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) o[nt][g][i / 4][i % 4] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      m[nt][k] = M_NONE;
      l[nt][k] = 0.f;
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) lows[nt][gi][k] = 0.f;
    }
  }

  int at = 0;
  for (int tau = first; tau < tl.total; tau += stride) {
    cp_async_wait<NS - 2>();
    __syncwarp();
    const int ahead = tau + (NS - 1) * stride;
    const int to = at == 0 ? NS - 1 : at - 1;
    if (ahead < tl.total && ahead > tau) fetch<BITS, G, NG, true>(p, tl, ahead, ring + to * S::BYTES, kv, lane);
    cp_async_commit();
    const uint32_t st = ring + at * S::BYTES;
    at = at == NS - 1 ? 0 : at + 1;

    float s[NT][4];
    tile_scores<BITS, G, NG, NT>(q, st + S::K, st + S::KM, lane, s);

    // Tiles whose every key counts for every token need no mask.
    const bool listed = tau >= tl.na + tl.nb;
    bool edge = listed;
    if (!listed) {
      const bool front = tau < tl.na;
      const int base = front ? tau * 16 : tl.b0 + (tau - tl.na) * 16;
      edge = base + 15 > tl.n - p.t || (front ? base + 16 > tl.fa : base < tl.n - p.window);
    }
    Mask<NT> mask;
    if (edge) {
      if (listed) mask.listed(p, tl, tau, st + S::POS, col0, lane);
      else mask.range(p, tl, tau, col0, lane);
    }
    uint32_t vm0[NG], vm1[NG];
    lds_words(vm0, st + S::VM + r * S::META);
    lds_words(vm1, st + S::VM + (r + 8) * S::META);
    float smax = 0.f;
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) smax = fmaxf(smax, fmaxf(step_of(vm0[gi]), step_of(vm1[gi])));  // NaN ignored

    float x[NT][4];
    bool move = smax > bound;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[nt][i] = fmaf(s[nt][i], q.mul[nt][i & 1], -m[nt][i & 1]);
        if (edge && !mask.ok[nt][i]) x[nt][i] = -INFINITY;
        move |= x[nt][i] > LAZY;
      }
    if (__any_sync(0xffffffffu, move)) {
      const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(smax)));
      float shrink = 1.f;
      if (top > bound) {
        const float next = __uint_as_float((__float_as_uint(top) & 0x7F800000u) + 0x00800000u);
        shrink = bound / next;
        bound = next;
        pscale = P_SCALE / bound;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float v0 = s[nt][k] * q.mul[nt][k], v1 = s[nt][2 + k] * q.mul[nt][k];
          if (edge && !mask.ok[nt][k]) v0 = -INFINITY;
          if (edge && !mask.ok[nt][2 + k]) v1 = -INFINITY;
          float v = fmaxf(v0, v1);
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          const float next = fmaxf(m[nt][k], v);
          f[k] = fast_exp2(m[nt][k] - next);
          m[nt][k] = next;
          l[nt][k] *= f[k];
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) lows[nt][gi][k] *= f[k];
          x[nt][k] = v0 - next;
          x[nt][2 + k] = v1 - next;
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < 8; ++i) o[nt][g][i / 4][i % 4] *= f[i & 1] * shrink;
      }
    }

    float pr[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) pr[nt][i] = fast_exp2(x[nt][i]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) l[nt][k] += pr[nt][k] + pr[nt][2 + k];

    // V operands: rows c, c + 4 (slots 2c, 2c + 1) and c + 8, c + 12 (slots 2c + 8, 2c + 9).
    constexpr int VW = (G * BITS + 7) / 8;
    uint32_t va[VW], vb[VW], vc[VW], vd[VW];
    v_words<BITS, G>(va, st + S::V, c, r);
    v_words<BITS, G>(vb, st + S::V, c + 4, r);
    v_words<BITS, G>(vc, st + S::V, c + 8, r);
    v_words<BITS, G>(vd, st + S::V, c + 12, r);
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) {
      const float s0 = step_of(vm0[gi]) * pscale, l0 = low_of(vm0[gi]), s1 = step_of(vm1[gi]) * pscale, l1 = low_of(vm1[gi]);
      uint32_t b[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float u[4] = {pr[nt][0] * s0, pr[nt][1] * s0, pr[nt][2] * s1, pr[nt][3] * s1};
        float e[4] = {pr[nt][0] * l0, pr[nt][1] * l0, pr[nt][2] * l1, pr[nt][3] * l1};
        if (edge) {  // rows that do not count may hold NaN
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[i] = mask.ok[nt][i] ? u[i] : 0.f;
            e[i] = mask.ok[nt][i] ? e[i] : 0.f;
          }
        }
        lows[nt][gi][0] += e[0] + e[2];
        lows[nt][gi][1] += e[1] + e[3];
        b[nt][0] = transpose8(pack2<__half>(u[0], u[1]));
        b[nt][1] = transpose8(pack2<__half>(u[2], u[3]));
      }
#pragma unroll
      for (int bb = 0; bb < G / NG; ++bb) {
        const int g = gi * (G / NG) + bb;
        uint32_t a[2][4];
        if constexpr (BITS == 4) {
          const uint32_t sel = g % 2 ? 0x7632u : 0x5410u;
          const uint32_t x0 = prmt(va[g / 2], vb[g / 2], sel), x1 = prmt(vc[g / 2], vd[g / 2], sel);
          const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
          a[0][0] = x0 & 0x000F000Fu; a[0][1] = y0 & 0x000F000Fu; a[0][2] = x1 & 0x000F000Fu; a[0][3] = y1 & 0x000F000Fu;
          a[1][0] = x0 & 0x00F000F0u; a[1][1] = y0 & 0x00F000F0u; a[1][2] = x1 & 0x00F000F0u; a[1][3] = y1 & 0x00F000F0u;
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t sel = h ? 0x7632u : 0x5410u;
            const uint32_t x0 = prmt(va[g], vb[g], sel), x1 = prmt(vc[g], vd[g], sel);
            a[h][0] = x0 & 0x00FF00FFu; a[h][1] = (x0 >> 8) & 0x00FF00FFu;
            a[h][2] = x1 & 0x00FF00FFu; a[h][3] = (x1 >> 8) & 0x00FF00FFu;
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_16816<__half>(o[nt][g][0], a[0], b[nt]);
          mma_16816<__half>(o[nt][g][1], a[1], b[nt]);
        }
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // every warp is done with its ring

  float* sm = reinterpret_cast<float*>(smem);       // [WARPS][8 NT] maxima, sums, then [WARPS][8 NT][D]
  float* sl = sm + WARPS * 8 * NT;
  float* so = sl + WARPS * 8 * NT;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int off = 4; off < 32; off *= 2) l[nt][k] += __shfl_xor_sync(0xffffffffu, l[nt][k], off);
#pragma unroll
      for (int gi = 0; gi < NG; ++gi)
#pragma unroll
        for (int off = 4; off < 32; off *= 2) lows[nt][gi][k] += __shfl_xor_sync(0xffffffffu, lows[nt][gi][k], off);
      const int col = nt * 8 + 2 * c + k;
      if (r == 0) {
        sm[warp * 8 * NT + col] = m[nt][k];
        sl[warp * 8 * NT + col] = l[nt][k];
      }
      float* row = so + (size_t)(warp * 8 * NT + col) * D;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // 4 bits: tile 0 holds dimensions 4r, 4r + 2 at 2^-24, tile 1 4r + 1, 4r + 3 at 2^-20; 8 bits: tile t
            // holds 4r + 2t, 4r + 2t + 1 at 2^-24.
            const int dim = g * 32 + 4 * r + (BITS == 4 ? t + 2 * h : 2 * t + h);
            const float undo = (BITS == 4 && t == 1 ? 1048576.f : 16777216.f) / P_SCALE;
            row[dim] = fmaf(o[nt][g][t][2 * h + k] * undo, bound, lows[nt][g / (G / NG)][k]);
          }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * NT * D; i += 32 * WARPS) {
    const int col = i / D, dim = i % D;
    if (col0 + col >= p.cols) break;
    float M = M_NONE, L = 0.f, A = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm[w * 8 * NT + col]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float e = fast_exp2(sm[w * 8 * NT + col] - M);
      L = fmaf(e, sl[w * 8 * NT + col], L);
      A = fmaf(e, so[(size_t)(w * 8 * NT + col) * D + dim], A);
    }
    const int64_t row = (kv * p.groups + (col0 + col) % p.groups) * p.t + (col0 + col) / p.groups;
    const int64_t o_at = row * p.splits + split;
    if (dim == 0) p.part_ml[o_at] = make_float2(M, L);
    p.part_acc[o_at * D + dim] = A;
  }
}

// Grid heads * t; 256 threads: the d dimensions, and 256 / dpad parts of the splits. A row that sees no
// key (a sum of 0) gives zeros.
__global__ void __launch_bounds__(256) qkv_combine_kernel(AttnParams p) {
  __shared__ float red[256];
  __shared__ float wt[1024];
  __shared__ float sM[8], sL[8];
  const int64_t row = blockIdx.x;
  const float2* ml = p.part_ml + row * p.splits;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  float M = M_NONE;
  for (int s = threadIdx.x; s < p.splits; s += 256) M = fmaxf(M, ml[s].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  if (lane == 0) sM[warp] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) M = fmaxf(M, sM[w]);
  float L = 0.f;
  for (int s = threadIdx.x; s < p.splits; s += 256) {
    const float2 v = ml[s];
    const float e = fast_exp2(v.x - M);  // M_NONE: 0, or 1 with a sum of 0 where no split has a key
    wt[s] = e;
    L = fmaf(e, v.y, L);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
  if (lane == 0) sL[warp] = L;
  __syncthreads();
  L = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) L += sL[w];
  const int dp = p.d <= 32 ? 32 : (p.d <= 64 ? 64 : 128), parts = 256 / dp;
  const int dim = threadIdx.x % dp, part = threadIdx.x / dp;
  float A = 0.f;
  if (dim < p.d)
    for (int s = part; s < p.splits; s += parts)
      if (wt[s] != 0.f) A = fmaf(wt[s], p.part_acc[(row * p.splits + s) * p.d + dim], A);
  red[threadIdx.x] = A;
  __syncthreads();
  if (threadIdx.x >= p.d) return;
  for (int k = 1; k < parts; ++k) A += red[k * dp + threadIdx.x];
  const float o = L == 0.f ? 0.f : A / L;
  const int64_t at = (row / p.t) * p.so_h + (row % p.t) * p.so_t + threadIdx.x;
  if (p.dtype == BB_BF16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(o);
  else static_cast<__half*>(p.out)[at] = __float2half_rn(o);
}

// Grid (splits * ztiles, kv_heads): the K half of qkv_partial_kernel; scores go to [kv][key][gp].
template <int BITS, int G, int NG, int NT>
__global__ void __launch_bounds__(32 * WARPS, 2) qkv_scores_kernel(const AttnParams p) {
  using S = Stage<BITS, G, NG, false>;
  constexpr int NS = stages(S::BYTES * 2);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float sm[WARPS][8 * NT], sl[WARPS][8 * NT];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int r = lane / 4, c = lane % 4;
  const int64_t kv = blockIdx.y;
  const int split = blockIdx.x / p.ztiles, col0 = (blockIdx.x % p.ztiles) * 8 * NT;
  const uint32_t ring = smem_u32(smem) + warp * NS * S::BYTES;
  const Tiles tl(p, true);
  const int first = split * WARPS + warp, stride = p.splits * WARPS;
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    const int tau = first + i * stride;
    if (tau < tl.total) fetch<BITS, G, NG, false>(p, tl, tau, ring + i * S::BYTES, kv, lane);
    cp_async_commit();
  }
  Query<BITS, G, NG, NT> q;
  q.load(p, kv, col0, lane);
  float m[NT][2], l[NT][2];  // of this thread's keys
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      m[nt][k] = M_NONE;
      l[nt][k] = 0.f;
    }
  int at = 0;
  for (int tau = first; tau < tl.total; tau += stride) {
    cp_async_wait<NS - 2>();
    __syncwarp();
    const int ahead = tau + (NS - 1) * stride;
    const int to = at == 0 ? NS - 1 : at - 1;
    if (ahead < tl.total && ahead > tau) fetch<BITS, G, NG, false>(p, tl, ahead, ring + to * S::BYTES, kv, lane);
    cp_async_commit();
    const uint32_t st = ring + at * S::BYTES;
    at = at == NS - 1 ? 0 : at + 1;
    float s[NT][4];
    tile_scores<BITS, G, NG, NT>(q, st + S::K, st + S::KM, lane, s);
    const int pos = tau * 16 + key_of(r);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = pos + (i / 2) * 8 < tl.n ? s[nt][i] * q.mul[nt][i & 1] : -INFINITY;
      const int col = col0 + nt * 8 + 2 * c;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (col < p.gp && pos + h * 8 < tl.n)
          *reinterpret_cast<float2*>(p.scores + ((kv * p.cap + pos + h * 8) * p.gp + col)) =
              make_float2(s[nt][2 * h], s[nt][2 * h + 1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float top = fmaxf(s[nt][k], s[nt][2 + k]);
        if (top > m[nt][k] + LAZY) {
          l[nt][k] *= fast_exp2(m[nt][k] - top);
          m[nt][k] = top;
        }
        l[nt][k] += fast_exp2(s[nt][k] - m[nt][k]) + fast_exp2(s[nt][2 + k] - m[nt][k]);
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float M = m[nt][k];
#pragma unroll
      for (int off = 4; off < 32; off *= 2) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
      float L = l[nt][k] * fast_exp2(m[nt][k] - M);
#pragma unroll
      for (int off = 4; off < 32; off *= 2) L += __shfl_xor_sync(0xffffffffu, L, off);
      if (r == 0) {
        sm[warp][nt * 8 + 2 * c + k] = M;
        sl[warp][nt * 8 + 2 * c + k] = L;
      }
    }
  __syncthreads();
  const int col = threadIdx.x;
  if (col < 8 * NT && col0 + col < p.cols) {
    float M = M_NONE, L = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm[w][col]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) L = fmaf(fast_exp2(sm[w][col] - M), sl[w][col], L);
    p.part_ml[(kv * p.groups + col0 + col) * p.splits + split] = make_float2(M, L);
  }
}

// Grid (cdiv(cap, 1024), kv_heads); four positions a thread. The merged statistics of the KV head's query
// heads come first, a warp a head at a time, into shared memory ([groups] maxima, then 1 / sums).
__global__ void __launch_bounds__(256) qkv_pool_kernel(AttnParams p) {
  extern __shared__ float stats[];
  const int64_t kv = blockIdx.y, n = cache_len(p);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  for (int h = warp; h < p.groups; h += 8) {
    const float2* ml = p.part_ml + (kv * p.groups + h) * p.splits;
    float M = M_NONE, L = 0.f;
    for (int s = lane; s < p.splits; s += 32) M = fmaxf(M, ml[s].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    for (int s = lane; s < p.splits; s += 32) L = fmaf(fast_exp2(ml[s].x - M), ml[s].y, L);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    if (lane == 0) {
      stats[h] = M;
      stats[p.groups + h] = 1.f / (L * (float)p.groups);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t pos = (int64_t)blockIdx.x * 1024 + i * 256 + threadIdx.x;
    if (pos >= p.cap) return;
    float sum = -1.f;
    if (pos >= p.front && pos < n - p.window) {
      const float* row = p.scores + (kv * p.cap + pos) * p.gp;
      sum = 0.f;
      for (int h = 0; h < p.groups; ++h) sum = fmaf(fast_exp2(row[h] - stats[h]), stats[p.groups + h], sum);
    }
    p.probs[kv * p.cap + pos] = sum;
  }
}

struct AttnPlan {
  int64_t splits, ztiles, cols, gp;
  int nt;
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
  if (a->t <= 0 || a->t > 65535 || a->t * a->heads > (int64_t)65535)
    return fail(BB_ERR_SHAPE, "%s: heads * tokens must lie in [1, 65535]", what);
  if (a->n < 0 || a->n > a->cache.cap) return fail(BB_ERR_ARG, "%s: n must lie in [0, capacity]", what);
  if (a->front < 0 || a->window < 0) return fail(BB_ERR_ARG, "%s: front and window must be >= 0", what);
  if (a->route_k < 0) return fail(BB_ERR_ARG, "%s: bad route count", what);
  if (a->splits < 0) return fail(BB_ERR_ARG, "%s: splits must be >= 0", what);
  return BB_OK;
}

// Columns in tiles of 8 or 16, and the splits of the key list: enough CTAs for one wave at the kernels'
// residency (two CTAs a SM with 8 columns, one with 16), no more than one tile of 16 keys a warp.
void plan_grid(const bb_qkv_attn_args* a, int64_t tiles, AttnPlan* pl) {
  pl->cols = a->heads / a->cache.kv_heads * a->t;
  pl->nt = pl->cols <= 8 ? 1 : 2;
  pl->ztiles = cdiv(pl->cols, (int64_t)8 * pl->nt);
  const int64_t wave = (int64_t)num_sms() * (pl->nt == 1 ? 2 : 1);
  const int64_t s = a->splits > 0 ? a->splits : std::max<int64_t>(1, wave / (a->cache.kv_heads * pl->ztiles));
  pl->splits = std::max<int64_t>(1, std::min<int64_t>({s, cdiv(tiles, (int64_t)WARPS), (int64_t)1024}));
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
  plan_grid(a, cdiv(f, (int64_t)16) + cdiv(w, (int64_t)16) + lists * cdiv(a->route_k, (int64_t)16), pl);
  const int64_t rows = a->heads * a->t;
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
  plan_grid(a, cdiv(a->n_dev ? a->cache.cap : a->n, (int64_t)16), pl);
  pl->gp = align_up(pl->cols, 2);
  pl->ml_bytes = align_up((size_t)(a->heads * pl->splits) * 8, 256);
  pl->scores_bytes = align_up((size_t)(a->cache.kv_heads * pl->gp * a->cache.cap) * 4, 256);
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
  p.per_head = a->route_k > 0 && a->route_rows != c.kv_heads;
  p.n_dev = a->n_dev;
  p.n = a->n; p.cap = c.cap;
  p.front = a->front; p.window = a->window;
  p.d = (int)c.d;
  p.heads = (int)a->heads; p.groups = (int)(a->heads / c.kv_heads);
  p.t = (int)a->t; p.cols = (int)pl.cols; p.gp = (int)pl.gp;
  p.splits = (int)pl.splits; p.ztiles = (int)pl.ztiles; p.dtype = a->dtype;
  p.scale_log2 = a->scale * LOG2E;
  p.part_ml = reinterpret_cast<float2*>(ws);
  p.part_acc = reinterpret_cast<float*>(ws + pl.ml_bytes);
  p.scores = reinterpret_cast<float*>(ws + pl.ml_bytes);
  p.probs = a->out_probs ? a->out_probs : reinterpret_cast<float*>(ws + pl.ml_bytes + pl.scores_bytes);
  p.out = a->out; p.so_h = a->so_h; p.so_t = a->so_t;
  return p;
}

template <bool DECODE, int BITS, int G, int NG, int NT>
int launch(const AttnParams& p, int64_t kv_heads, cudaStream_t stream) {
  const dim3 grid((unsigned)(p.splits * p.ztiles), (unsigned)kv_heads);
  if constexpr (DECODE) {
    constexpr size_t smem = partial_smem<BITS, G, NG, NT>();
    if (smem > 48 * 1024)
      cudaFuncSetAttribute(qkv_partial_kernel<BITS, G, NG, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    qkv_partial_kernel<BITS, G, NG, NT><<<grid, 32 * WARPS, smem, stream>>>(p);
    BB_CHECK_LAUNCH("qkv_partial_kernel");
  } else {
    using S = Stage<BITS, G, NG, false>;
    constexpr size_t smem = (size_t)WARPS * stages(S::BYTES * 2) * S::BYTES;
    if (smem > 48 * 1024)
      cudaFuncSetAttribute(qkv_scores_kernel<BITS, G, NG, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    qkv_scores_kernel<BITS, G, NG, NT><<<grid, 32 * WARPS, smem, stream>>>(p);
    BB_CHECK_LAUNCH("qkv_scores_kernel");
  }
  return BB_OK;
}

template <bool DECODE, int BITS, int G, int NG>
int launch_nt(const AttnParams& p, int nt, int64_t kv_heads, cudaStream_t stream) {
  return nt == 1 ? launch<DECODE, BITS, G, NG, 1>(p, kv_heads, stream) : launch<DECODE, BITS, G, NG, 2>(p, kv_heads, stream);
}

template <bool DECODE, int BITS>
int launch_shape(const AttnParams& p, int pairs, int nt, int64_t kv_heads, cudaStream_t stream) {
  switch (p.d / 32 * 8 + pairs) {
    case 1 * 8 + 1: return launch_nt<DECODE, BITS, 1, 1>(p, nt, kv_heads, stream);
    case 2 * 8 + 1: return launch_nt<DECODE, BITS, 2, 1>(p, nt, kv_heads, stream);
    case 2 * 8 + 2: return launch_nt<DECODE, BITS, 2, 2>(p, nt, kv_heads, stream);
    case 3 * 8 + 1: return launch_nt<DECODE, BITS, 3, 1>(p, nt, kv_heads, stream);
    case 3 * 8 + 3: return launch_nt<DECODE, BITS, 3, 3>(p, nt, kv_heads, stream);
    case 4 * 8 + 1: return launch_nt<DECODE, BITS, 4, 1>(p, nt, kv_heads, stream);
    case 4 * 8 + 2: return launch_nt<DECODE, BITS, 4, 2>(p, nt, kv_heads, stream);
    case 4 * 8 + 4: return launch_nt<DECODE, BITS, 4, 4>(p, nt, kv_heads, stream);
    default: return fail(BB_ERR_UNSUPPORTED, "qkv attention: head_dim %d with %d groups", p.d, pairs);
  }
}

template <bool DECODE>
int launch_attn(const bb_qkv_attn_args* a, const AttnParams& p, int nt, cudaStream_t stream) {
  const int pairs = (int)(a->cache.d / a->cache.group);
  return a->cache.bits == 4 ? launch_shape<DECODE, 4>(p, pairs, nt, a->cache.kv_heads, stream)
                            : launch_shape<DECODE, 8>(p, pairs, nt, a->cache.kv_heads, stream);
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
  st = launch_attn<true>(a, p, pl.nt, stream);
  if (st) return st;
  qkv_combine_kernel<<<(unsigned)(a->heads * a->t), 256, 0, stream>>>(p);
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
  st = launch_attn<false>(a, p, pl.nt, stream);
  if (st) return st;
  qkv_pool_kernel<<<dim3((unsigned)cdiv(a->cache.cap, (int64_t)1024), (unsigned)a->cache.kv_heads), 256,
                    (size_t)p.groups * 8, stream>>>(p);
  BB_CHECK_LAUNCH("qkv_pool_kernel");
  if (a->route_k > 0 && a->out_idx)
    return topk_sorted(p.probs, a->cache.kv_heads, a->cache.cap, a->route_k, a->out_idx, a->out_idx_i64 != 0, a->so_i,
                       w + pl.ml_bytes + pl.scores_bytes + pl.probs_bytes, pl.topk_bytes, stream);
  return BB_OK;
}

}  // namespace bb
