// Quantised KV cache: writing rows and reading them back (format: include/bb_b200.h, bb_qkv_cache).
//
//   qkv_write_kernel  x -> low, step, codes (and optionally the values low + step * code)
//   qkv_read_kernel   codes -> low + step * code, of a range of rows or of listed rows
//
// Both are bound by HBM: a row of d 16-bit values is 2 d bytes on one side and d bits / 8 + 4 d / group
// on the other. A thread owns 8 consecutive dimensions (16 bytes of a 16-bit row); a group's
// minimum and maximum come from shuffles among the 4, 8, 12 or 16 threads that share it.
#include <algorithm>

#include "qkv.cuh"

namespace bb {
namespace {

using qkv::K_RUN;
using qkv::V_RUN;

struct RowsParams {
  // cache sides: 0 = keys, 1 = values
  unsigned char* codes[2];
  uint32_t* meta[2];        // (step, low) bf16 pairs
  int64_t codes_h[2], meta_h[2];
  int64_t cap;
  int d, group, pairs, row_bytes;
  // write
  const void* in[2];
  int64_t in_h[2], in_t[2];
  int64_t at;
  const int64_t* at_dev;
  // read
  const void* positions;
  int64_t sp_h;
  int pos64;
  // values out
  void* out[2];
  int64_t out_h[2], out_t[2];
  int64_t rows;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The bf16 numbers next to x: not above it; not below it (x >= 0). As fp32 bit patterns, whose upper
// halves are the bf16 numbers.
__device__ __forceinline__ uint32_t bf16_down(float x) {
  const uint32_t u = __float_as_uint(x), cut = u & 0xFFFF0000u;
  return ((u >> 31) && cut != u) ? cut + 0x10000u : cut;
}
__device__ __forceinline__ uint32_t bf16_up(float x) { return (__float_as_uint(x) + 0xFFFFu) & 0xFFFF0000u; }

// 8 consecutive elements.
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  uint4 v = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_f(e[i]);
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 v;
  v.x = pack2<T>(x[0], x[1]);
  v.y = pack2<T>(x[2], x[3]);
  v.z = pack2<T>(x[4], x[5]);
  v.w = pack2<T>(x[6], x[7]);
  *reinterpret_cast<uint4*>(p) = v;
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

// Where the 8 codes of chunk c (dimensions 8 c ...) stand in a row. Keys: one run of 8. Values: two
// runs of 4. In bytes from the row's start; the second value run is `G` runs further.
__device__ __forceinline__ int code_at(int c, int G, int bits, bool values) {
  const int g = c >> 2, a = c & 3;
  const int place = values ? (2 * a * G + g) * V_RUN : (a * G + g) * K_RUN;
  return place * bits / 8;
}

// The magic number 1.5 2^23: x + MAGIC has x, rounded to the nearest even integer, in its lowest bits.
constexpr float MAGIC = 12582912.f;
constexpr uint32_t MAGIC_BITS = 0x4B400000u;

// Minimum of the 8 elements and of their negatives (NaN if any is), as far as these threads share a group.
template <typename T> struct Extremes {  // 16-bit types: the pair (min, -max) in one register, exact
  uint32_t v;
  static __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b);
  static __device__ __forceinline__ uint32_t neg2(uint32_t a) { return a ^ 0x80008000u; }
  __device__ __forceinline__ void of(const uint4& x) {
    const uint32_t lo = min2(min2(x.x, x.y), min2(x.z, x.w));
    const uint32_t hi = min2(min2(neg2(x.x), neg2(x.y)), min2(neg2(x.z), neg2(x.w)));
    v = min2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
  }
  __device__ __forceinline__ void clear() { v = sizeof(T) == 2 ? pack2<T>(INFINITY, INFINITY) : 0u; }
  __device__ __forceinline__ void with(int off) { v = min2(v, __shfl_xor_sync(0xffffffffu, v, off)); }
  __device__ __forceinline__ void get(float& lo, float& hi) const {
    const T* e = reinterpret_cast<const T*>(&v);
    lo = Elem<T>::to_f(e[0]);
    hi = -Elem<T>::to_f(e[1]);
  }
};
template <> __device__ __forceinline__ uint32_t Extremes<__nv_bfloat16>::min2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> __device__ __forceinline__ uint32_t Extremes<__half>::min2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> struct Extremes<float> {
  float lo, hi;
  __device__ __forceinline__ void of(const float (&x)[8]) {
    lo = hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo = min_nan(lo, x[i]);
      hi = max_nan(hi, x[i]);
    }
  }
  __device__ __forceinline__ void clear() {
    lo = INFINITY;
    hi = -INFINITY;
  }
  __device__ __forceinline__ void with(int off) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  __device__ __forceinline__ void get(float& l, float& h) const {
    l = lo;
    h = hi;
  }
};

// 8 elements as loaded.
template <typename T> struct Chunk {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void extremes(Extremes<T>& e) const { e.of(v); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_f(e[i]);
  }
};
template <> struct Chunk<float> {
  float x[8];
  __device__ __forceinline__ void load(const float* p) { load8(p, x); }
  __device__ __forceinline__ void extremes(Extremes<float>& e) const { e.of(x); }
  __device__ __forceinline__ void get(float (&y)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
  }
};

// LPR threads a row (a power of two >= d / 8; with d = 96, 12 of 16 work), ROWS rows a thread, all of whose loads are
// issued before the first is used.
template <typename T, int LPR, int BITS, int ROWS>
__global__ void __launch_bounds__(256) qkv_write_kernel(const RowsParams p) {
  constexpr float TOP = (float)((1 << BITS) - 1), INV_TOP = 1.f / TOP;
  constexpr int PER = 256 / LPR;  // rows of a block at a time
  const int side = blockIdx.z;
  const int c = threadIdx.x % LPR;
  const int64_t r0 = (int64_t)blockIdx.x * (PER * ROWS) + threadIdx.x / LPR;
  const int64_t head = blockIdx.y;
  const bool mine = c * 8 < p.d;
  const T* in = static_cast<const T*>(p.in[side]) + head * p.in_h[side] + c * 8;
  Chunk<T> chunk[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
    if (mine && r0 + i * PER < p.rows) chunk[i].load(in + (r0 + i * PER) * p.in_t[side]);
  const int G = p.d / 32;
  const int64_t at = p.at_dev ? *p.at_dev : p.at;
  unsigned char* codes = p.codes[side] + head * p.codes_h[side] + code_at(c, G, BITS, side);
  uint32_t* meta = p.meta[side] + head * p.meta_h[side] + c * 8 / p.group;
  T* out = static_cast<T*>(p.out[side]);
  if (out) out += head * p.out_h[side] + c * 8;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t r = r0 + i * PER;
    const bool live = mine && r < p.rows;
    Extremes<T> ext;
    ext.clear();  // neutral where nothing is loaded
    if (live) chunk[i].extremes(ext);
    // 32 dimensions are 4 threads; 64: 8; 96 and 128: 16 (with d = 96 the last four are neutral).
#pragma unroll
    for (int off = 1; off < LPR; off *= 2)
      if (off * 8 < p.group) ext.with(off);
    if (!live) continue;
    float lo, hi;
    ext.get(lo, hi);
    uint32_t low_b = bf16_down(lo);
    // Quotients rounded as IEEE division rounds them (Markstein's theorem: with y the correctly rounded reciprocal of b
    // and q within an ulp of a / b, q + (a - q b) y by fused operations is a / b correctly rounded).
    const float range = hi - __uint_as_float(low_b), q0 = range * INV_TOP;
    const float exact_step = __fmaf_rn(__fmaf_rn(-q0, TOP, range), INV_TOP, q0);
    uint32_t step_b = bf16_up(exact_step);
    const float step0 = __uint_as_float(step_b);
    const bool bad = !(exact_step < INFINITY) || !(step0 < INFINITY);  // a NaN, an infinity, a range beyond fp32
    if (bad) step_b = low_b = 0x7FC00000u;
    else if (step0 < 7.8886090522101181e-31f) step_b = 0u;  // 2^-100
    const float low = __uint_as_float(low_b), step = __uint_as_float(step_b);
    const float inv = step > 0.f ? __frcp_rn(step) : 0.f;
    float x[8];
    chunk[i].get(x);
    const uint64_t low2 = f2_pack(low, low), inv2 = f2_pack(inv, inv), step2 = f2_pack(step, step),
                   minus2 = f2_pack(-step, -step), zero2 = f2_pack(-0.f, -0.f), magic2 = f2_pack(MAGIC, MAGIC);
    uint64_t t[4];
    uint32_t w[BITS / 4] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t a = f2_sub(f2_pack(x[2 * k], x[2 * k + 1]), low2);
      const uint64_t q = f2_fma(a, inv2, zero2);
      t[k] = f2_add(f2_fma(f2_fma(q, minus2, a), inv2, q), magic2);  // 0 <= quotient <= TOP: no clamp needed
      const uint32_t c0 = (uint32_t)t[k], c1 = (uint32_t)(t[k] >> 32);
      const int b0 = 2 * k * BITS, b1 = b0 + BITS;
      // codes side by side modulo 2^32, each with MAGIC_BITS below it, which the constants take off
      w[b0 / 32] += (c0 - MAGIC_BITS) * (1u << (b0 % 32)) + (c1 - MAGIC_BITS) * (1u << (b1 % 32));
    }
    if (bad) {
#pragma unroll
      for (int k = 0; k < BITS / 4; ++k) w[k] = 0u;
    }
    const int64_t slot = at + r;
    if (slot >= 0 && slot < p.cap) {
      unsigned char* row = codes + slot * p.row_bytes;
      if constexpr (BITS == 4) {
        if (side == 0) {
          *reinterpret_cast<uint32_t*>(row) = w[0];
        } else {
          *reinterpret_cast<uint16_t*>(row) = (uint16_t)w[0];
          *reinterpret_cast<uint16_t*>(row + G * 2) = (uint16_t)(w[0] >> 16);
        }
      } else {
        if (side == 0) {
          *reinterpret_cast<uint2*>(row) = make_uint2(w[0], w[1]);
        } else {
          *reinterpret_cast<uint32_t*>(row) = w[0];
          *reinterpret_cast<uint32_t*>(row + G * 4) = w[1];
        }
      }
      if (c * 8 % p.group == 0) meta[slot * p.pairs] = (step_b >> 16) | low_b;
    }
    if (out) {
#pragma unroll
      for (int k = 0; k < 4; ++k)  // step * code is exact in fp32
        f2_unpack(f2_fma(f2_sub(t[k], magic2), step2, low2), x[2 * k], x[2 * k + 1]);
      store8(out + r * p.out_t[side], x);
    }
  }
}

template <typename T, int LPR, int BITS, int ROWS>
__global__ void __launch_bounds__(256) qkv_read_kernel(const RowsParams p) {
  constexpr int PER = 256 / LPR;
  const int side = blockIdx.z;
  const int c = threadIdx.x % LPR;
  const int64_t r0 = (int64_t)blockIdx.x * (PER * ROWS) + threadIdx.x / LPR;
  const int64_t head = blockIdx.y;
  if (c * 8 >= p.d) return;
  const int G = p.d / 32;
  const unsigned char* codes = p.codes[side] + head * p.codes_h[side] + code_at(c, G, BITS, side);
  const uint32_t* meta = p.meta[side] + head * p.meta_h[side] + c * 8 / p.group;
  uint32_t w[ROWS][BITS / 4], m[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t r = r0 + i * PER;
    int64_t slot = p.at + r;
    if (p.positions && r < p.rows) {
      const int64_t o = head * p.sp_h + r;
      slot = p.pos64 ? static_cast<const int64_t*>(p.positions)[o] : (int64_t) static_cast<const int32_t*>(p.positions)[o];
    }
    m[i] = 0u;  // zeros outside the cache
#pragma unroll
    for (int k = 0; k < BITS / 4; ++k) w[i][k] = 0u;
    if (r < p.rows && slot >= 0 && slot < p.cap) {
      const unsigned char* row = codes + slot * p.row_bytes;
      if constexpr (BITS == 4) {
        if (side == 0)
          w[i][0] = *reinterpret_cast<const uint32_t*>(row);
        else
          w[i][0] = *reinterpret_cast<const uint16_t*>(row) | ((uint32_t) * reinterpret_cast<const uint16_t*>(row + G * 2) << 16);
      } else {
        w[i][0] = *reinterpret_cast<const uint32_t*>(row);
        w[i][1] = *reinterpret_cast<const uint32_t*>(row + (side == 0 ? 4 : G * 4));
      }
      m[i] = meta[slot * p.pairs];
    }
  }
  T* out = static_cast<T*>(p.out[side]) + head * p.out_h[side] + c * 8;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t r = r0 + i * PER;
    if (r >= p.rows) return;
    const float step = __uint_as_float(m[i] << 16), low = __uint_as_float(m[i] & 0xFFFF0000u);
    const uint64_t step2 = f2_pack(step, step), low2 = f2_pack(low, low), base2 = f2_pack(8388608.f, 8388608.f);
    float x[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t c0, c1;  // codes in bytes 2 k % 4 and + 1 of b (8 bits), or in byte k of w and of w >> 4 (4 bits)
      if constexpr (BITS == 4) {
        c0 = __byte_perm(w[i][0] & 0x0F0F0F0Fu, 0x4B000000u, 0x7540 | k);  // 2^23 + code
        c1 = __byte_perm((w[i][0] >> 4) & 0x0F0F0F0Fu, 0x4B000000u, 0x7540 | k);
      } else {
        c0 = __byte_perm(w[i][k / 2], 0x4B000000u, 0x7540 | (2 * k % 4));
        c1 = __byte_perm(w[i][k / 2], 0x4B000000u, 0x7540 | (2 * k % 4 + 1));
      }
      f2_unpack(f2_fma(f2_sub(f2_pack(__uint_as_float(c0), __uint_as_float(c1)), base2), step2, low2), x[2 * k], x[2 * k + 1]);
    }
    store8(out + r * p.out_t[side], x);
  }
}

RowsParams cache_params(const bb_qkv_cache& c) {
  RowsParams p{};
  p.codes[0] = static_cast<unsigned char*>(c.k_codes);
  p.codes[1] = static_cast<unsigned char*>(c.v_codes);
  p.meta[0] = static_cast<uint32_t*>(c.k_meta);
  p.meta[1] = static_cast<uint32_t*>(c.v_meta);
  p.codes_h[0] = c.k_codes_h; p.codes_h[1] = c.v_codes_h;
  p.meta_h[0] = c.k_meta_h; p.meta_h[1] = c.v_meta_h;
  p.cap = c.cap;
  p.d = (int)c.d;
  p.group = c.group;
  p.pairs = (int)(c.d / c.group);
  p.row_bytes = (int)(c.d * c.bits / 8);
  return p;
}

// Few rows: one a thread, for latency; from two waves of blocks on, four, whose loads overlap.
template <bool WRITE, typename T, int BITS, int LPR>
int launch_lanes(const RowsParams& p, int64_t heads, cudaStream_t stream) {
  constexpr int PER = 256 / LPR;
  const bool many = p.rows * heads * 2 >= (int64_t)num_sms() * 16 * PER * 4;
  const dim3 grid((unsigned)cdiv(p.rows, (int64_t)PER * (many ? 4 : 1)), (unsigned)heads, 2);
  if constexpr (WRITE) {
    if (many) qkv_write_kernel<T, LPR, BITS, 4><<<grid, 256, 0, stream>>>(p);
    else qkv_write_kernel<T, LPR, BITS, 1><<<grid, 256, 0, stream>>>(p);
    BB_CHECK_LAUNCH("qkv_write_kernel");
  } else {
    if (many) qkv_read_kernel<T, LPR, BITS, 4><<<grid, 256, 0, stream>>>(p);
    else qkv_read_kernel<T, LPR, BITS, 1><<<grid, 256, 0, stream>>>(p);
    BB_CHECK_LAUNCH("qkv_read_kernel");
  }
  return BB_OK;
}
template <bool WRITE, typename T, int BITS>
int launch_rows(const RowsParams& p, int64_t heads, cudaStream_t stream) {
  if (p.d <= 32) return launch_lanes<WRITE, T, BITS, 4>(p, heads, stream);
  return p.d <= 64 ? launch_lanes<WRITE, T, BITS, 8>(p, heads, stream) : launch_lanes<WRITE, T, BITS, 16>(p, heads, stream);
}

template <bool WRITE, typename T>
int launch_bits(const RowsParams& p, int bits, int64_t heads, cudaStream_t stream) {
  return bits == 4 ? launch_rows<WRITE, T, 4>(p, heads, stream) : launch_rows<WRITE, T, 8>(p, heads, stream);
}
template <bool WRITE>
int launch_dtype(const RowsParams& p, int dtype, int bits, int64_t heads, cudaStream_t stream) {
  if (dtype == BB_BF16) return launch_bits<WRITE, __nv_bfloat16>(p, bits, heads, stream);
  if (dtype == BB_F16) return launch_bits<WRITE, __half>(p, bits, heads, stream);
  return launch_bits<WRITE, float>(p, bits, heads, stream);
}

// Every row of a [heads, rows, d] tensor on a 16-byte boundary.
bool rows16(const void* p, int64_t sh, int64_t st, int64_t es) {
  return qkv::al16(p) && (sh * es) % 16 == 0 && (st * es) % 16 == 0;
}

int check_dtype(int dtype, const char* what) {
  if (dtype != BB_F16 && dtype != BB_BF16 && dtype != BB_F32)
    return fail(BB_ERR_DTYPE, "%s: dtype must be fp16, bf16 or fp32", what);
  return BB_OK;
}

constexpr int64_t MAX_ROWS = (int64_t)INT32_MAX;  // keeps the block count within the grid's limit

}  // namespace

int qkv_write(const bb_qkv_write_args* a, cudaStream_t stream) {
  if (!a) return fail(BB_ERR_ARG, "qkv_write: null args");
  int st = qkv::check_cache(a->cache, "qkv_write", true, true);
  if (!st) st = check_dtype(a->dtype, "qkv_write");
  if (st) return st;
  if (a->t < 0 || a->t > MAX_ROWS) return fail(BB_ERR_SHAPE, "qkv_write: bad row count");
  if (!a->at_dev && (a->at < 0 || a->at > a->cache.cap - a->t))
    return fail(BB_ERR_ARG, "qkv_write: rows [at, at + t) must lie in the cache");
  if (a->t == 0) return BB_OK;
  if (!a->k || !a->v || (!a->out_k) != (!a->out_v)) return fail(BB_ERR_ARG, "qkv_write: null pointer");
  const int64_t es = a->dtype == BB_F32 ? 4 : 2;
  if (!rows16(a->k, a->sk_h, a->sk_t, es) || !rows16(a->v, a->sv_h, a->sv_t, es) ||
      (a->out_k && (!rows16(a->out_k, a->sok_h, a->sok_t, es) || !rows16(a->out_v, a->sov_h, a->sov_t, es))))
    return fail(BB_ERR_STRIDE, "qkv_write: rows must start on 16-byte boundaries");
  RowsParams p = cache_params(a->cache);
  p.in[0] = a->k; p.in_h[0] = a->sk_h; p.in_t[0] = a->sk_t;
  p.in[1] = a->v; p.in_h[1] = a->sv_h; p.in_t[1] = a->sv_t;
  p.out[0] = a->out_k; p.out_h[0] = a->sok_h; p.out_t[0] = a->sok_t;
  p.out[1] = a->out_v; p.out_h[1] = a->sov_h; p.out_t[1] = a->sov_t;
  p.at = a->at;
  p.at_dev = a->at_dev;
  p.rows = a->t;
  return launch_dtype<true>(p, a->dtype, a->cache.bits, a->cache.kv_heads, stream);
}

int qkv_read(const bb_qkv_read_args* a, cudaStream_t stream) {
  if (!a) return fail(BB_ERR_ARG, "qkv_read: null args");
  int st = qkv::check_cache(a->cache, "qkv_read", true, true);
  if (!st) st = check_dtype(a->dtype, "qkv_read");
  if (st) return st;
  if (a->rows < 0 || a->rows > MAX_ROWS) return fail(BB_ERR_SHAPE, "qkv_read: bad row count");
  if (!a->positions && (a->start < 0 || a->start > a->cache.cap - a->rows))
    return fail(BB_ERR_ARG, "qkv_read: rows [start, start + rows) must lie in the cache");
  if (a->rows == 0) return BB_OK;
  if (!a->out_k || !a->out_v) return fail(BB_ERR_ARG, "qkv_read: null pointer");
  const int64_t es = a->dtype == BB_F32 ? 4 : 2;
  if (!rows16(a->out_k, a->sok_h, a->sok_t, es) || !rows16(a->out_v, a->sov_h, a->sov_t, es))
    return fail(BB_ERR_STRIDE, "qkv_read: rows must start on 16-byte boundaries");
  RowsParams p = cache_params(a->cache);
  p.out[0] = a->out_k; p.out_h[0] = a->sok_h; p.out_t[0] = a->sok_t;
  p.out[1] = a->out_v; p.out_h[1] = a->sov_h; p.out_t[1] = a->sov_t;
  p.at = a->start;
  p.positions = a->positions;
  p.sp_h = a->sp_h;
  p.pos64 = a->pos_i64 != 0;
  p.rows = a->rows;
  return launch_dtype<false>(p, a->dtype, a->cache.bits, a->cache.kv_heads, stream);
}

}  // namespace bb
