// The KV cache of gdn_kv_store / gdn_kv_load / gdn_attn_cached: layout and quantisation.
//
// A cache row holds, for each kv head, T tokens in blocks of 64; a block's 64 * HD values lie in the order in which
// the attention kernel's lanes take them, so that each of its loads reads 1 KB contiguous:
//   K: 16-byte pieces of E values of one token (E = 16 in e4m3, 8 in bf16).  Token 16 a + 4 i + r, piece p:
//      [p / 4][i][p % 4][4 a + r] -- lane (4 a + r, p % 4) of the scores' i-th 16-token tile.
//   V: 16 dims at a time.  e4m3: [dim][64 tokens]; bf16: token 16 a + 8 u + x at [u][dim][a][x].
// e4m3 rows (one token of one kv head) have one scale 2^e each, stored as the byte e + 127.  A power of two costs e4m3
// nothing (a format with an exponent keeps its relative precision at any scale) and is exact: codes and scales do not
// depend on how a division rounds, code * 2^e is a bf16 value, and scaling commutes with every later rounding.
#pragma once
#include "gdn_device.h"

namespace gdn {
namespace kv {
constexpr int BT = 64;  // tokens per block

template <bool F8> __device__ __forceinline__ int64_t k_at(int64_t t, int d, int hd) {
  constexpr int E = F8 ? 16 : 8;
  const int p = d / E, x = (int)(t % BT), a = x / 16, i = x / 4 % 4, r = x % 4;
  return t / BT * (BT * (int64_t)hd) + ((((p / 4) * 4 + i) * 4 + p % 4) * 16 + 4 * a + r) * E + d % E;
}
template <bool F8> __device__ __forceinline__ int64_t v_at(int64_t t, int d, int hd) {
  const int x = (int)(t % BT), m = d % 16;
  const int64_t b = t / BT * (BT * (int64_t)hd) + d / 16 * 1024;
  return F8 ? b + m * 64 + x : b + ((x / 8 % 2 * 16 + m) * 4 + x / 16) * 8 + x % 8;
}

// The scale exponent of a row whose largest finite |value| is top: the smallest e >= -126 with top <= 448 * 2^e
// (448 = 1.75 * 2^8, e4m3's largest value); 0 for a row of zeros.
__device__ __forceinline__ int scale_exp(float top) {
  const uint32_t b = __float_as_uint(top);
  const int e = (int)(b >> 23) - 135 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b == 0 ? 0 : e < -126 ? -126 : e;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127
// |x| for the row's maximum: what is not finite does not count.
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }
// Two values times 2^-e (inv) as e4m3 codes (low byte first), rounded to nearest even; not finite: NaN (0x7f).
__device__ __forceinline__ uint32_t quant2(float a, float b, float inv) {
  uint32_t c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false) & 0xffffu;
  if (!(fabsf(a) < INFINITY)) c = (c & 0xff00u) | 0x7fu;
  if (!(fabsf(b) < INFINITY)) c = (c & 0x00ffu) | 0x7f00u;
  return c;
}
}  // namespace kv
}  // namespace gdn
