// Quantised KV cache: writing rows and reading them back (format: include/bb_b200.h, bb_qkv_cache).
//
//   qkv_write_kernel  x -> low, step, codes (and optionally the values low + step * code)
//   qkv_read_kernel   codes -> low + step * code, of a range of rows or of listed rows
//
// Both are bound by HBM: a row of d 16-bit values is 2 d bytes on one side and d bits / 8 + 4 d / group
// on the other. A thread owns 16 consecutive dimensions (32 bytes of a 16-bit row); a group's
// minimum and maximum come from shuffles among the 2, 4, 6 or 8 threads that share it.
// Measured, 128K rows of 8 heads, d = 128, 4 bits, groups of 32, bf16: writing with the values returned (1.24 GB) 221 us,
// reading (705 MB) 112 us, 86 % and 97 % of a copy's rate. On the way: 8 dimensions and 4 rows a thread 299 and 131 us
// (group and address work is shared by fewer dimensions); 16 dimensions in 16-byte accesses 232 and 145 us (each access
// touches half a sector); scalar fp32 arithmetic with library division 369 and 196 us.
#include <algorithm>

#include "qkv.cuh"

namespace bb {
namespace {

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
  int wide;                 // input and output rows start on 32-byte boundaries
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
using qkv::max_nan;

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
// The magic number 1.5 2^23: x + MAGIC has x, rounded to the nearest even integer, in its lowest bits.
constexpr float MAGIC = 12582912.f;
constexpr uint32_t MAGIC_BITS = 0x4B400000u;

// Minimum of the 8 elements and of their negatives (NaN if any is), as far as these threads share a group.
template <typename T> struct Extremes {  // 16-bit types: the pair (min, -max) in one register, exact
  uint32_t v;
  static __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b);
  static __device__ __forceinline__ uint32_t neg2(uint32_t a) { return a ^ 0x80008000u; }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);
  __device__ __forceinline__ void of(const uint4& x) {
    const uint32_t lo = min2(min2(x.x, x.y), min2(x.z, x.w));
    const uint32_t hi = neg2(max2(max2(x.x, x.y), max2(x.z, x.w)));
    v = min2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
  }
  __device__ __forceinline__ void join(const Extremes& e) { v = min2(v, e.v); }
  __device__ __forceinline__ void clear() { v = sizeof(T) == 2 ? pack2<T>(INFINITY, INFINITY) : 0u; }
  __device__ __forceinline__ void with(int off) { v = min2(v, __shfl_xor_sync(0xffffffffu, v, off)); }
  __device__ __forceinline__ void get(float& lo, float& hi) const {
    const T* e = reinterpret_cast<const T*>(&v);
    lo = Elem<T>::to_f(e[0]);
    hi = -Elem<T>::to_f(e[1]);
  }
};
template <> __device__ __forceinline__ uint32_t Extremes<__nv_bfloat16>::max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> __device__ __forceinline__ uint32_t Extremes<__nv_bfloat16>::min2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> __device__ __forceinline__ uint32_t Extremes<__half>::max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
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
  __device__ __forceinline__ void join(const Extremes& e) {
    lo = min_nan(lo, e.lo);
    hi = max_nan(hi, e.hi);
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

__device__ __forceinline__ void ld32(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p));
}
__device__ __forceinline__ void st32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
               "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
}
// 16 consecutive elements. In accesses of 32 bytes where rows allow it: a warp's 16-byte accesses at steps of 32 would
// touch every sector twice.
template <typename T> __device__ __forceinline__ void load16(const T* p, Chunk<T> (&x)[2], bool wide) {
  if (sizeof(T) == 2 && wide) {
    ld32(p, reinterpret_cast<uint4&>(x[0]), reinterpret_cast<uint4&>(x[1]));
  } else {
    x[0].load(p);
    x[1].load(p + 8);
  }
}
template <typename T> __device__ __forceinline__ void store16(T* p, const float (&x)[16], bool wide) {
  uint4 v[sizeof(T)];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) {
    if constexpr (sizeof(T) == 2)
      v[i] = make_uint4(pack2<T>(x[8 * i], x[8 * i + 1]), pack2<T>(x[8 * i + 2], x[8 * i + 3]),
                        pack2<T>(x[8 * i + 4], x[8 * i + 5]), pack2<T>(x[8 * i + 6], x[8 * i + 7]));
    else
      v[i] = make_uint4(__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]), __float_as_uint(x[4 * i + 2]),
                        __float_as_uint(x[4 * i + 3]));
  }
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); i += 2) {
    if (wide) {
      st32(reinterpret_cast<uint4*>(p) + i, v[i], v[i + 1]);
    } else {
      reinterpret_cast<uint4*>(p)[i] = v[i];
      reinterpret_cast<uint4*>(p)[i + 1] = v[i + 1];
    }
  }
}

// 1 / s, correctly rounded, for s with at most 8 significant bits: one Newton step from an approximation within an ulp
// has a relative error of 2^-46, and the exact quotient 2^m / k, k < 256, is at least 1 / 510 ulp from a tie.
__device__ __forceinline__ float reciprocal8(float s) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
  return __fmaf_rn(__fmaf_rn(-s, y, 1.f), y, y);
}

// One side's buffers as a thread of a kernel sees them.
template <typename T, int BITS, int SIDE> struct Side {
  static constexpr int RUNS = SIDE == 0 ? 2 : 4;            // runs of consecutive codes in 16 dimensions
  static constexpr int RUN_BYTES = 16 / RUNS * BITS / 8;
  unsigned char* codes;   // this thread's first run in row 0; runs lie `jump` bytes apart
  uint32_t* meta;         // its group's (step, low) in row 0
  T* out;                 // its 16 dimensions of row 0 of the values
  int64_t out_t;
  int jump, row_bytes, pairs;

  // Thread c of a row owns dimensions 16 c .. 16 c + 15: block g = c / 2, runs from (c % 2) * RUNS on.
  __device__ __forceinline__ Side(const RowsParams& p, int64_t head, int c) {
    const int G = p.d / 32;
    row_bytes = p.row_bytes;
    pairs = p.pairs;
    jump = G * RUN_BYTES;
    codes = p.codes[SIDE] + head * p.codes_h[SIDE] + (c % 2 * RUNS * G + c / 2) * RUN_BYTES;
    meta = p.meta[SIDE] + head * p.meta_h[SIDE] + c * 16 / p.group;
    out = static_cast<T*>(p.out[SIDE]);
    if (out) out += head * p.out_h[SIDE] + c * 16;
    out_t = p.out_t[SIDE];
  }
  // 16 codes as a word a run of 8 (4 bits) or of 4 (8 bits).
  static constexpr int WORDS = BITS / 2;
  __device__ __forceinline__ void put(int64_t slot, const uint32_t (&w)[WORDS]) const {
    unsigned char* row = codes + slot * row_bytes;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      if constexpr (RUN_BYTES == 2) *reinterpret_cast<uint16_t*>(row + i * jump) = (uint16_t)(w[i / 2] >> (i % 2 * 16));
      else if constexpr (RUN_BYTES == 4) *reinterpret_cast<uint32_t*>(row + i * jump) = w[i];
      else *reinterpret_cast<uint2*>(row + i * jump) = make_uint2(w[2 * i], w[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void get(int64_t slot, uint32_t (&w)[WORDS]) const {
    const unsigned char* row = codes + slot * row_bytes;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      if constexpr (RUN_BYTES == 2) {
        const uint32_t h = *reinterpret_cast<const uint16_t*>(row + i * jump);
        w[i / 2] = i % 2 ? w[i / 2] | (h << 16) : h;
      } else if constexpr (RUN_BYTES == 4) {
        w[i] = *reinterpret_cast<const uint32_t*>(row + i * jump);
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(row + i * jump);
        w[2 * i] = v.x;
        w[2 * i + 1] = v.y;
      }
    }
  }
};

// LPR threads a row (a power of two >= d / 16; with d = 96, 6 of 8 work), ROWS rows a thread, all of whose loads are
// issued before the first is used.
template <typename T, int LPR, int BITS, int ROWS, int SIDE>
__device__ __forceinline__ void write_rows(const RowsParams& p) {
  constexpr float TOP = (float)((1 << BITS) - 1), INV_TOP = 1.f / TOP;
  constexpr int PER = 256 / LPR;  // rows of a block at a time
  const int c = threadIdx.x % LPR;
  const int64_t r0 = (int64_t)blockIdx.x * (PER * ROWS) + threadIdx.x / LPR;
  const int64_t head = blockIdx.y;
  const int rows = (int)min((int64_t)(PER * ROWS), p.rows - r0);  // those from r0 on (rows < 2^31)
  const bool mine = c * 16 < p.d, wide = p.wide != 0;
  Chunk<T> chunk[ROWS][2];
  {
    const T* in = static_cast<const T*>(p.in[SIDE]) + head * p.in_h[SIDE] + r0 * p.in_t[SIDE] + c * 16;
    const int64_t step_rows = PER * p.in_t[SIDE];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (mine && i * PER < rows) load16(in + i * step_rows, chunk[i], wide);
  }
  const Side<T, BITS, SIDE> to(p, head, c);
  const bool first = c * 16 % p.group == 0;
  const int64_t cap = p.cap, at = (p.at_dev ? *p.at_dev : p.at) + r0;
  const int group = p.group;
  const uint64_t zero2 = f2_pack(-0.f, -0.f), magic2 = f2_pack(MAGIC, MAGIC);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const bool live = mine && i * PER < rows;
    Extremes<T> ext;
    ext.clear();  // neutral where nothing is loaded
    if (live) {
      Extremes<T> other;
      chunk[i][0].extremes(ext);
      chunk[i][1].extremes(other);
      ext.join(other);
    }
    // 32 dimensions are 2 threads; 64: 4; 96 and 128: 8 (with d = 96 the last two are neutral).
#pragma unroll
    for (int off = 1; off < LPR; off *= 2)
      if (off * 16 < group) ext.with(off);
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
    const bool flat = !bad && step0 < 7.8886090522101181e-31f;         // below 2^-100
    if (bad) step_b = low_b = 0x7FC00000u;
    if (flat) step_b = 0u;
    const float low = __uint_as_float(low_b), step = __uint_as_float(step_b);
    const float inv = bad || flat ? 0.f : reciprocal8(step);
    const uint64_t low2 = f2_pack(low, low), inv2 = f2_pack(inv, inv), step2 = f2_pack(step, step),
                   minus2 = f2_pack(-step, -step);
    const int64_t slot = at + i * PER;
    uint64_t t[8];
    uint32_t w[BITS / 2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[8];
      chunk[i][h].get(x);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t a = f2_sub(f2_pack(x[2 * k], x[2 * k + 1]), low2);
        const uint64_t q = f2_fma(a, inv2, zero2);
        t[4 * h + k] = f2_add(f2_fma(f2_fma(q, minus2, a), inv2, q), magic2);  // 0 <= quotient <= TOP: no clamp needed
      }
    }
    // Codes side by side modulo 2^32, then the MAGIC_BITS below each of them off.
    constexpr int PACK = 32 / BITS;
    constexpr uint32_t UNIT = BITS == 4 ? 0x11111111u : 0x01010101u;
#pragma unroll
    for (int k = 0; k < 16; ++k) w[k / PACK] += (uint32_t)(k % 2 ? t[k / 2] >> 32 : t[k / 2]) << (k % PACK * BITS);
#pragma unroll
    for (int k = 0; k < BITS / 2; ++k) w[k] = bad ? 0u : w[k] - UNIT * MAGIC_BITS;
    if (slot >= 0 && slot < cap) {
      to.put(slot, w);
      if (first) to.meta[slot * to.pairs] = (step_b >> 16) | low_b;
    }
    if (to.out) {
      float x[16];
#pragma unroll
      for (int k = 0; k < 8; ++k)  // step * code is exact in fp32
        f2_unpack(f2_fma(f2_sub(t[k], magic2), step2, low2), x[2 * k], x[2 * k + 1]);
      store16(to.out + (r0 + i * PER) * to.out_t, x, wide);
    }
  }
}

template <typename T, int LPR, int BITS, int ROWS>
__global__ void __launch_bounds__(256) qkv_write_kernel(const RowsParams p) {
  if (blockIdx.z == 0) write_rows<T, LPR, BITS, ROWS, 0>(p);
  else write_rows<T, LPR, BITS, ROWS, 1>(p);
}

template <typename T, int LPR, int BITS, int ROWS, int SIDE>
__device__ __forceinline__ void read_rows(const RowsParams& p) {
  constexpr int PER = 256 / LPR;
  const int c = threadIdx.x % LPR;
  const int64_t r0 = (int64_t)blockIdx.x * (PER * ROWS) + threadIdx.x / LPR;
  const int64_t head = blockIdx.y;
  if (c * 16 >= p.d || r0 >= p.rows) return;
  const int rows = (int)min((int64_t)(PER * ROWS), p.rows - r0);
  const Side<T, BITS, SIDE> from(p, head, c);
  const int64_t cap = p.cap;
  const bool wide = p.wide != 0;
  uint32_t w[ROWS][BITS / 2], m[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    int64_t slot = p.at + r0 + i * PER;
    if (p.positions && i * PER < rows) {
      const int64_t o = head * p.sp_h + r0 + i * PER;
      slot = p.pos64 ? static_cast<const int64_t*>(p.positions)[o] : (int64_t) static_cast<const int32_t*>(p.positions)[o];
    }
    m[i] = 0u;  // zeros outside the cache
#pragma unroll
    for (int k = 0; k < BITS / 2; ++k) w[i][k] = 0u;
    if (i * PER < rows && slot >= 0 && slot < cap) {
      from.get(slot, w[i]);
      m[i] = from.meta[slot * from.pairs];
    }
  }
  const uint64_t base2 = f2_pack(8388608.f, 8388608.f);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (i * PER >= rows) return;
    const float step = __uint_as_float(m[i] << 16), low = __uint_as_float(m[i] & 0xFFFF0000u);
    const uint64_t step2 = f2_pack(step, step), low2 = f2_pack(low, low);
    float x[16];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t c0, c1;  // 2^23 + code as fp32: the codes are bytes of the word, or of its low and high halves of bytes
      if constexpr (BITS == 4) {
        c0 = __byte_perm(w[i][k / 4] & 0x0F0F0F0Fu, 0x4B000000u, 0x7540 | (k % 4));
        c1 = __byte_perm((w[i][k / 4] >> 4) & 0x0F0F0F0Fu, 0x4B000000u, 0x7540 | (k % 4));
      } else {
        c0 = __byte_perm(w[i][k / 2], 0x4B000000u, 0x7540 | (2 * k % 4));
        c1 = __byte_perm(w[i][k / 2], 0x4B000000u, 0x7540 | (2 * k % 4 + 1));
      }
      f2_unpack(f2_fma(f2_sub(f2_pack(__uint_as_float(c0), __uint_as_float(c1)), base2), step2, low2), x[2 * k], x[2 * k + 1]);
    }
    store16(from.out + (r0 + i * PER) * from.out_t, x, wide);
  }
}

template <typename T, int LPR, int BITS, int ROWS>
__global__ void __launch_bounds__(256) qkv_read_kernel(const RowsParams p) {
  if (blockIdx.z == 0) read_rows<T, LPR, BITS, ROWS, 0>(p);
  else read_rows<T, LPR, BITS, ROWS, 1>(p);
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

// Few rows: one a thread, for latency; from two waves of blocks on, two, whose loads overlap.
template <bool WRITE, typename T, int BITS, int LPR>
int launch_lanes(const RowsParams& p, int64_t heads, cudaStream_t stream) {
  constexpr int PER = 256 / LPR;
  const bool many = p.rows * heads * 2 >= (int64_t)num_sms() * 16 * PER * 2;
  const dim3 grid((unsigned)cdiv(p.rows, (int64_t)PER * (many ? 2 : 1)), (unsigned)heads, 2);
  if constexpr (WRITE) {
    if (many) qkv_write_kernel<T, LPR, BITS, 2><<<grid, 256, 0, stream>>>(p);
    else qkv_write_kernel<T, LPR, BITS, 1><<<grid, 256, 0, stream>>>(p);
    BB_CHECK_LAUNCH("qkv_write_kernel");
  } else {
    if (many) qkv_read_kernel<T, LPR, BITS, 2><<<grid, 256, 0, stream>>>(p);
    else qkv_read_kernel<T, LPR, BITS, 1><<<grid, 256, 0, stream>>>(p);
    BB_CHECK_LAUNCH("qkv_read_kernel");
  }
  return BB_OK;
}
template <bool WRITE, typename T, int BITS>
int launch_rows(const RowsParams& p, int64_t heads, cudaStream_t stream) {
  if (p.d <= 32) return launch_lanes<WRITE, T, BITS, 2>(p, heads, stream);
  return p.d <= 64 ? launch_lanes<WRITE, T, BITS, 4>(p, heads, stream) : launch_lanes<WRITE, T, BITS, 8>(p, heads, stream);
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

// Every row of a [heads, rows, d] tensor on a boundary of `to` bytes (16 or 32).
bool rows_on(int64_t to, const void* p, int64_t sh, int64_t st, int64_t es) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && (sh * es) % to == 0 && (st * es) % to == 0;
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
  if (!rows_on(16, a->k, a->sk_h, a->sk_t, es) || !rows_on(16, a->v, a->sv_h, a->sv_t, es) ||
      (a->out_k && (!rows_on(16, a->out_k, a->sok_h, a->sok_t, es) || !rows_on(16, a->out_v, a->sov_h, a->sov_t, es))))
    return fail(BB_ERR_STRIDE, "qkv_write: rows must start on 16-byte boundaries");
  RowsParams p = cache_params(a->cache);
  p.in[0] = a->k; p.in_h[0] = a->sk_h; p.in_t[0] = a->sk_t;
  p.in[1] = a->v; p.in_h[1] = a->sv_h; p.in_t[1] = a->sv_t;
  p.out[0] = a->out_k; p.out_h[0] = a->sok_h; p.out_t[0] = a->sok_t;
  p.out[1] = a->out_v; p.out_h[1] = a->sov_h; p.out_t[1] = a->sov_t;
  p.at = a->at;
  p.at_dev = a->at_dev;
  p.rows = a->t;
  p.wide = rows_on(32, a->k, a->sk_h, a->sk_t, es) && rows_on(32, a->v, a->sv_h, a->sv_t, es) &&
           rows_on(32, a->out_k, a->sok_h, a->sok_t, es) && rows_on(32, a->out_v, a->sov_h, a->sov_t, es);
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
  if (!rows_on(16, a->out_k, a->sok_h, a->sok_t, es) || !rows_on(16, a->out_v, a->sov_h, a->sov_t, es))
    return fail(BB_ERR_STRIDE, "qkv_read: rows must start on 16-byte boundaries");
  RowsParams p = cache_params(a->cache);
  p.out[0] = a->out_k; p.out_h[0] = a->sok_h; p.out_t[0] = a->sok_t;
  p.out[1] = a->out_v; p.out_h[1] = a->sov_h; p.out_t[1] = a->sov_t;
  p.at = a->start;
  p.positions = a->positions;
  p.sp_h = a->sp_h;
  p.pos64 = a->pos_i64 != 0;
  p.rows = a->rows;
  p.wide = rows_on(32, a->out_k, a->sok_h, a->sok_t, es) && rows_on(32, a->out_v, a->sov_h, a->sov_t, es);
  return launch_dtype<false>(p, a->dtype, a->cache.bits, a->cache.kv_heads, stream);
}

}  // namespace bb
