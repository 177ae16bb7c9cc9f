// Quantised KV cache: host checks and the device view shared by its write / read kernels (qkv.cu)
// and its attention kernels (qkv_attn.cu). Format: include/bb_b200.h, bb_qkv_cache.
#pragma once

#include "bb_common.cuh"

namespace bb {
namespace qkv {

constexpr int K_RUN = 8, V_RUN = 4;  // consecutive dimensions that stay together in a row's order

// NaN if either is (fmaxf returns the other).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Checks of the cache's description; `what` opens the message.
inline int check_cache(const bb_qkv_cache& c, const char* what, bool need_k, bool need_v) {
  if (c.bits != 4 && c.bits != 8) return fail(BB_ERR_UNSUPPORTED, "%s: bits must be 4 or 8", what);
  if (c.d <= 0 || c.d > 128 || c.d % 32)
    return fail(BB_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 32 up to 128", what);
  if (c.group <= 0 || c.group % 32 || c.d % c.group)
    return fail(BB_ERR_SHAPE, "%s: group must be a multiple of 32 that divides head_dim", what);
  if (c.kv_heads <= 0 || c.kv_heads > 65535) return fail(BB_ERR_SHAPE, "%s: kv_heads must lie in [1, 65535]", what);
  if (c.cap <= 0 || c.cap > INT32_MAX - 64)  // positions rounded up to a step of 32 stay below 2^31
    return fail(BB_ERR_SHAPE, "%s: capacity must lie in [1, 2^31 - 65]", what);
  const int64_t row = c.d * c.bits / 8, pairs = c.d / c.group;
  if ((need_k && (!c.k_codes || !c.k_meta)) || (need_v && (!c.v_codes || !c.v_meta)))
    return fail(BB_ERR_ARG, "%s: null cache buffer", what);
  if ((need_k && (!al16(c.k_codes) || !al16(c.k_meta))) || (need_v && (!al16(c.v_codes) || !al16(c.v_meta))))
    return fail(BB_ERR_STRIDE, "%s: cache buffers must start on 16-byte boundaries", what);
  const int64_t ch[2] = {c.k_codes_h, c.v_codes_h}, mh[2] = {c.k_meta_h, c.v_meta_h};
  const bool need[2] = {need_k, need_v};
  for (int i = 0; i < 2; ++i) {
    if (!need[i] || c.kv_heads == 1) continue;
    if (ch[i] < c.cap * row || ch[i] % row || mh[i] < c.cap * pairs || mh[i] % pairs)
      return fail(BB_ERR_STRIDE, "%s: cache heads must not overlap and must be whole rows apart", what);
  }
  return BB_OK;
}

}  // namespace qkv
}  // namespace bb
