// The decode attention kernels' view of the fused q|gate|k|v projection.
#pragma once
#include "gdn_device.h"

namespace gdn {
namespace attn {
// The fused projection's row n, column col: a bf16 matrix, or bf16(sum of fp32 split-K partials
// [splits][N][width] in split order) -- the same value the reduced projection holds.
struct Src {
  const uint16_t* bf;
  int64_t stride;
  const float* part;
  int splits, N;
  int64_t width;
  __device__ __forceinline__ float operator()(int n, int64_t col) const {
    if (!part) return bf2f(bf[n * stride + col]);
    float s = 0.f;
#pragma unroll 8
    for (int sp = 0; sp < splits; ++sp) s += part[((int64_t)sp * N + n) * width + col];
    return rbf(s);
  }
  // columns col + 64 e, the loads of several splits in flight
  template <int E>
  __device__ __forceinline__ void row(float (&x)[E], int n, int64_t col) const {
    if (!part) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = bf2f(bf[n * stride + col + 64 * e]);
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
#pragma unroll 4
    for (int sp = 0; sp < splits; ++sp)
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] += part[((int64_t)sp * N + n) * width + col + 64 * e];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = rbf(x[e]);
  }
};
}  // namespace attn
}  // namespace gdn
