// kv_cache_store / kv_cache_load: packed prompts' K and V rows into the slots' cache rows (quantised as they are
// written) and back.  Layout and quantisation: gdn_kv.h.
//
// Both are copies: bound by HBM, each value read once and written once.  One workgroup per (64-token cache block,
// kv head, K or V): a block is what lies together in the cache.  K's 16-byte pieces are one token's and go out as they are;
// V's lie along the tokens and turn in LDS.  16 prompts of 200 to 1500 tokens (13.6 thousand, 4 heads of 256, bf16 to e4m3
// and back, 84 MB each way): store 19.6 us (4.3 TB/s), load 17.5 us (4.8 TB/s), where a large copy runs at 4.97 TB/s; the
// same over a bf16 cache (111 MB each way): 28.6 and 25.2 us (3.9 and 4.4 TB/s: V turns 2 bytes at a time).  517 tokens
// stored and 1541 loaded, e4m3 (3.2 and 9.5 MB): 7.5 and 6.5 us, bf16: 8.2 and 7.9 us; a launch and a block's latency.
#include "gdn_internal.h"
#include "gdn_kv.h"

namespace gdn {
namespace kv {
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 16 consecutive values of a row, 16-byte aligned, as fp32.
template <typename T> __device__ __forceinline__ void load16(const T* p, float (&x)[16]);
template <> __device__ __forceinline__ void load16(const float* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = reinterpret_cast<const float4*>(p)[i];
    x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
  }
}
template <> __device__ __forceinline__ void load16(const uint16_t* p, float (&x)[16]) {  // bf16
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4 v = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[8 * i + 2 * j] = __uint_as_float(v[j] << 16);
      x[8 * i + 2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
    }
  }
}
template <> __device__ __forceinline__ void load16(const _Float16* p, float (&x)[16]) {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const h8 v = reinterpret_cast<const h8*>(p)[i];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[8 * i + j] = (float)v[j];
  }
}

// Bytes of 4 words transposed: word i's byte j becomes word j's byte i.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u), w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u), w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// A batch of sequences: sequence s is the packed tokens [lo, hi), which lie at positions start + 0, 1, .. of cache row
// `row`.  Nothing here is trusted: token ranges are cut to [0, total), a row outside [0, n_rows) is -1.
struct Batch {
  const int32_t *rows, *cu, *start;  // cu NULL: equal lengths; start NULL: 0
  int nseq, n_rows;
  int64_t total;
};
struct Seq {
  int64_t lo, hi, start;
  int row;
};
__device__ __forceinline__ Seq seq_of(const Batch& b, int s) {
  Seq q;
  const int64_t each = b.total / b.nseq;
  q.lo = b.cu ? b.cu[s] : s * each;
  q.hi = b.cu ? b.cu[s + 1] : (s + 1) * each;
  q.lo = q.lo < 0 ? 0 : q.lo > b.total ? b.total : q.lo;
  q.hi = q.hi < q.lo ? q.lo : q.hi > b.total ? b.total : q.hi;
  q.start = b.start ? b.start[s] : 0;
  q.row = state_row(b.rows, b.n_rows, s);
  return q;
}
// The 64-token blocks (by position) that sequence q touches.
__device__ __forceinline__ int64_t blocks_of(const Seq& q) {
  return q.hi > q.lo ? ((q.start + (q.hi - q.lo) - 1) >> 6) - (q.start >> 6) + 1 : 0;
}
// The `tile`-th block of the batch: its sequence and position block; false if there is none.  A wave looks at 64
// sequences at a time (every wave of the workgroup does the same).
__device__ __forceinline__ bool find_tile(const Batch& b, int64_t tile, Seq& q, int64_t& blk) {
  const int lane = threadIdx.x & 63;
  for (int s0 = 0; s0 < b.nseq; s0 += 64) {
    const int s = s0 + lane;
    int64_t n = 0;
    if (s < b.nseq) n = blocks_of(seq_of(b, s));
    int64_t sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t v = __shfl_up(sum, o, kWave);
      if (lane >= o) sum += v;
    }
    const uint64_t past = __ballot(sum > tile);
    if (past) {
      const int f = __builtin_ctzll(past);
      tile -= __shfl(sum - n, f, kWave);
      q = seq_of(b, s0 + f);
      blk = (q.start >> 6) + tile;
      return true;
    }
    tile -= __shfl(sum, 63, kWave);
  }
  return false;
}
// More tiles than any batch has: a sequence of n tokens touches at most (n + 126) / 64 blocks.
inline int64_t most_tiles(int64_t total, int nseq) { return (total + 126ll * nseq) / BT; }
}  // namespace kv

// grid (tiles, kv heads, 2: K and V), 256 threads.  A lane takes 16 dims of one token: HD / 16 lanes a token, which
// share the row's maximum.
template <int HD, bool F8, typename T>
__global__ __launch_bounds__(256) void kv_store_kernel(const T* __restrict__ xk, int64_t ks, int64_t kh,
                                                       const T* __restrict__ xv, int64_t vs, int64_t vh,
                                                       uint8_t* __restrict__ kc, uint8_t* __restrict__ vc,
                                                       uint8_t* __restrict__ ke, uint8_t* __restrict__ ve, int nkv,
                                                       int64_t len, kv::Batch batch) {
  using namespace kv;
  constexpr int S = F8 ? 1 : 2;        // bytes per value
  constexpr int LT = HD / 16;          // lanes per token
  constexpr int PITCH = HD * S + 16;   // bytes of a token's row in LDS
  __shared__ alignas(16) uint8_t tile[BT * PITCH];
  Seq q;
  int64_t blk;
  if (!find_tile(batch, blockIdx.x, q, blk)) return;
  const int64_t t0 = blk * BT;
  if (q.row < 0 || t0 < 0 || t0 >= len) return;  // no such row, or positions outside the cache
  const int head = blockIdx.y, tid = threadIdx.x;
  const bool is_v = blockIdx.z;
  const T* x = is_v ? xv + head * vh : xk + head * kh;
  const int64_t stride = is_v ? vs : ks;
  const int64_t row = (int64_t)q.row * nkv + head;
  uint8_t* out = (is_v ? vc : kc) + (row * len + t0) * HD * S;
  const int piece = tid % LT;
  for (int r0 = 0; r0 < BT; r0 += 256 / LT) {
    const int t = r0 + tid / LT;
    const int64_t i = q.lo + (t0 + t - q.start);  // the packed token at this position
    const bool in = i >= q.lo && i < q.hi;
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = 0.f;
    if (in) load16<T>(x + i * stride + 16 * piece, v);
    u32x4 w[S];
    if constexpr (F8) {
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, finite_abs(v[e]));
#pragma unroll
      for (int o = 1; o < LT; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
      const int e = scale_exp(top);
      const float inv = pow2(-e);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[0][j] = quant2(v[4 * j], v[4 * j + 1], inv) | quant2(v[4 * j + 2], v[4 * j + 3], inv) << 16;
      if (in && piece == 0) (is_v ? ve : ke)[row * len + t0 + t] = (uint8_t)(e + 127);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j / 4][j % 4] = f2bf2(v[2 * j], v[2 * j + 1]);
    }
    if (is_v) {
#pragma unroll
      for (int s = 0; s < S; ++s) *reinterpret_cast<u32x4*>(&tile[t * PITCH + (piece * S + s) * 16]) = w[s];
    } else if (in) {
#pragma unroll
      for (int s = 0; s < S; ++s)
        *reinterpret_cast<u32x4*>(out + k_at<F8>(t, (piece * S + s) * (16 / S), HD) * S) = w[s];
    }
  }
  if (!is_v) return;
  __syncthreads();
  constexpr int TK = 16 / S;  // tokens of 16 bytes of V
  auto put = [&](uint8_t* at, const uint32_t (&w)[4], int t) {  // tokens t .. t + TK - 1 of one dim
    const int64_t first = q.lo + (t0 + t - q.start);
    if (first >= q.lo && first + TK <= q.hi) {
      *reinterpret_cast<u32x4*>(at) = u32x4{w[0], w[1], w[2], w[3]};
      return;
    }
#pragma unroll
    for (int e = 0; e < TK; ++e)  // tokens outside the sequence stay as they are
      if (first + e >= q.lo && first + e < q.hi) {
        if constexpr (F8) at[e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
        else reinterpret_cast<uint16_t*>(at)[e] = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
      }
  };
  if constexpr (F8) {  // 4 dims of 16 tokens a thread: 16 words from LDS (byte by byte: 64), 4 x 4 bytes transposed in registers
    for (int o = tid; o < HD; o += 256) {
      const int a = o % 4, d = o / 4 * 4;
      uint32_t w[4][4];  // [dim][4 tokens]
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const uint32_t*>(&tile[(16 * a + 4 * j + i) * PITCH + d]);
        transpose4(x);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i][j] = x[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) put(out + (int64_t)(d + i) * 64 + 16 * a, w[i], 16 * a);
    }
  } else {  // 8 tokens of one dim at a time, in the order in which they lie in the cache: 16 dims, then [2][16 dims][4]
    for (int o = tid; o < HD * 8; o += 256) {
      const int u = o / 64 % 2, m = o / 4 % 16, a = o % 4, d = o / 128 * 16 + m, t = 16 * a + 8 * u;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = *reinterpret_cast<const uint16_t*>(&tile[(t + 2 * j) * PITCH + 2 * d]) |
               (uint32_t) * reinterpret_cast<const uint16_t*>(&tile[(t + 2 * j + 1) * PITCH + 2 * d]) << 16;
      put(out + (int64_t)o * 16, w, t);
    }
  }
}

// grid (tiles, kv heads, 2: K and V), 256 threads: cache blocks to bf16 rows [total, nkv, HD]; positions outside the
// cache and rows that do not exist give zeros.
template <int HD, bool F8>
__global__ __launch_bounds__(256) void kv_load_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                      const uint8_t* __restrict__ ke, const uint8_t* __restrict__ ve,
                                                      uint16_t* __restrict__ ok, uint16_t* __restrict__ ov, int nkv,
                                                      int64_t len, kv::Batch batch) {
  using namespace kv;
  constexpr int S = F8 ? 1 : 2;
  constexpr int LT = HD / 16;
  constexpr int PITCH = HD * S + 16;
  __shared__ alignas(16) uint8_t tile[BT * PITCH];
  Seq q;
  int64_t blk;
  if (!find_tile(batch, blockIdx.x, q, blk)) return;
  const int64_t t0 = blk * BT;
  const bool there = q.row >= 0 && t0 >= 0 && t0 < len;
  const int head = blockIdx.y, tid = threadIdx.x;
  const bool is_v = blockIdx.z;
  const int64_t row = (int64_t)q.row * nkv + head;
  const uint8_t* in = (is_v ? vc : kc) + (row * len + t0) * HD * S;
  if (is_v && there) {
    if constexpr (F8) {
      for (int o = tid; o < HD; o += 256) {
        const int a = o % 4, d = o / 4 * 4;
        u32x4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const u32x4*>(in + (int64_t)(d + i) * 64 + 16 * a);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t x[4] = {w[0][j], w[1][j], w[2][j], w[3][j]};
          transpose4(x);
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(&tile[(16 * a + 4 * j + i) * PITCH + d]) = x[i];
        }
      }
    } else {
      for (int o = tid; o < HD * 8; o += 256) {
        const int u = o / 64 % 2, m = o / 4 % 16, a = o % 4, d = o / 128 * 16 + m, t = 16 * a + 8 * u;
        const u32x4 w = *reinterpret_cast<const u32x4*>(in + (int64_t)o * 16);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint16_t*>(&tile[(t + e) * PITCH + 2 * d]) = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
      }
    }
  }
  __syncthreads();
  const int piece = tid % LT;
  for (int r0 = 0; r0 < BT; r0 += 256 / LT) {
    const int t = r0 + tid / LT;
    const int64_t i = q.lo + (t0 + t - q.start);
    if (i < q.lo || i >= q.hi) continue;
    u32x4 y[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (there) {
      u32x4 w[S];
#pragma unroll
      for (int s = 0; s < S; ++s)
        w[s] = is_v ? *reinterpret_cast<const u32x4*>(&tile[t * PITCH + (piece * S + s) * 16])
                    : *reinterpret_cast<const u32x4*>(in + k_at<F8>(t, (piece * S + s) * (16 / S), HD) * S);
      if constexpr (F8) {
        // the codes' values times the scale, rounded once to bf16 (exact but where that is subnormal)
        const float sc = __uint_as_float((uint32_t)(is_v ? ve : ke)[row * len + t0 + t] << 23);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = __builtin_amdgcn_cvt_f32_fp8((int)w[0][j], 0), b = __builtin_amdgcn_cvt_f32_fp8((int)w[0][j], 1);
          const float c = __builtin_amdgcn_cvt_f32_fp8((int)w[0][j], 2), d = __builtin_amdgcn_cvt_f32_fp8((int)w[0][j], 3);
          y[j / 2][2 * (j % 2)] = f2bf2(a * sc, b * sc);
          y[j / 2][2 * (j % 2) + 1] = f2bf2(c * sc, d * sc);
        }
      } else {
        y[0] = w[0], y[1] = w[S - 1];
      }
    }
    u32x4* o = reinterpret_cast<u32x4*>((is_v ? ov : ok) + (i * nkv + head) * HD + 16 * piece);
    o[0] = y[0], o[1] = y[1];
  }
}

}  // namespace gdn

using namespace gdn;

namespace {
// What both entry points ask of a cache and a batch.
int check_cache(const char* name, const void* k, const void* v, const void* ke, const void* ve, int dtype, int n_rows,
                int nkv, int hd, int64_t T, const int32_t* rows, int nseq, int64_t total) {
  GDN_REQUIRE(dtype == GDN_BF16 || dtype == GDN_F8E4M3, "%s: the cache's dtype must be bf16 or e4m3", name);
  GDN_SUPPORT(hd == 64 || hd == 128 || hd == 256, "%s: head_dim must be 64, 128 or 256", name);
  GDN_REQUIRE(n_rows >= 1 && nkv >= 1 && nkv <= 65535 && nseq >= 0 && total >= 0, "%s: bad sizes", name);
  GDN_REQUIRE(T >= kv::BT && T % kv::BT == 0 && T <= INT32_MAX, "%s: cache length must be a positive multiple of 64", name);
  if (nseq == 0 || total == 0) return GDN_OK;
  GDN_REQUIRE(k && v && rows && (dtype == GDN_BF16 || (ke && ve)), "%s: null pointer", name);
  GDN_REQUIRE(aligned(k, 16) && aligned(v, 16), "%s: caches must be 16-byte aligned", name);
  GDN_REQUIRE(kv::most_tiles(total, nseq) <= INT32_MAX, "%s: too many tokens", name);
  return GDN_OK;
}
template <int HD, bool F8, typename T>
void launch_store(dim3 g, hipStream_t st, const void* xk, int64_t ks, int64_t kh, const void* xv, int64_t vs, int64_t vh,
                  void* kc, void* vc, uint8_t* ke, uint8_t* ve, int nkv, int64_t len, const kv::Batch& b) {
  kv_store_kernel<HD, F8, T><<<g, 256, 0, st>>>(static_cast<const T*>(xk), ks, kh, static_cast<const T*>(xv), vs, vh,
                                                static_cast<uint8_t*>(kc), static_cast<uint8_t*>(vc), ke, ve, nkv, len, b);
}
}  // namespace

extern "C" int gdn_kv_store(const void* xk, int64_t k_stride, int64_t k_head, const void* xv, int64_t v_stride,
                            int64_t v_head, int in_dtype, void* k_cache, void* v_cache, uint8_t* k_exp, uint8_t* v_exp,
                            int cache_dtype, int n_rows, int nkv, int hd, int64_t T, const int32_t* rows,
                            const int32_t* cu_seqlens, const int32_t* start, int nseq, int64_t total_tokens, void* stream) {
  clear_error();
  const char* name = "gdn_kv_store";
  if (const int rc = check_cache(name, k_cache, v_cache, k_exp, v_exp, cache_dtype, n_rows, nkv, hd, T, rows, nseq, total_tokens))
    return rc;
  GDN_REQUIRE(in_dtype == GDN_F32 || in_dtype == GDN_BF16 || in_dtype == GDN_F16, "%s: bad input dtype", name);
  if (nseq == 0 || total_tokens == 0) return GDN_OK;
  GDN_REQUIRE(xk && xv, "%s: null pointer", name);
  GDN_REQUIRE(cu_seqlens || total_tokens % nseq == 0, "%s: without cu_seqlens the tokens must divide into nseq sequences", name);
  const int per = in_dtype == GDN_F32 ? 4 : 8;  // elements of 16 bytes
  GDN_REQUIRE(aligned(xk, 16) && aligned(xv, 16) && k_stride % per == 0 && k_head % per == 0 && v_stride % per == 0 &&
                  v_head % per == 0, "%s: rows must be 16-byte aligned", name);
  const kv::Batch b{rows, cu_seqlens, start, nseq, n_rows, total_tokens};
  const dim3 g((unsigned)kv::most_tiles(total_tokens, nseq), nkv, 2);
  const hipStream_t st = (hipStream_t)stream;
#define GDN_STORE(HD, F8, T) \
  launch_store<HD, F8, T>(g, st, xk, k_stride, k_head, xv, v_stride, v_head, k_cache, v_cache, k_exp, v_exp, nkv, T_, b)
  const int64_t T_ = T;
#define GDN_STORE_T(HD, F8)                                          \
  switch (in_dtype) {                                                \
    case GDN_F32: GDN_STORE(HD, F8, float); break;                   \
    case GDN_BF16: GDN_STORE(HD, F8, uint16_t); break;               \
    default: GDN_STORE(HD, F8, _Float16); break;                     \
  }
  const bool f8 = cache_dtype == GDN_F8E4M3;
  switch (hd) {
    case 64: if (f8) { GDN_STORE_T(64, true) } else { GDN_STORE_T(64, false) } break;
    case 128: if (f8) { GDN_STORE_T(128, true) } else { GDN_STORE_T(128, false) } break;
    default: if (f8) { GDN_STORE_T(256, true) } else { GDN_STORE_T(256, false) } break;
  }
#undef GDN_STORE_T
#undef GDN_STORE
  return check_launch(name);
}

extern "C" int gdn_kv_load(const void* k_cache, const void* v_cache, const uint8_t* k_exp, const uint8_t* v_exp,
                           int cache_dtype, int n_rows, int nkv, int hd, int64_t T, const int32_t* rows,
                           const int32_t* cu_seqlens, const int32_t* start, int nseq, int64_t total_tokens, void* out_k,
                           void* out_v, void* stream) {
  clear_error();
  const char* name = "gdn_kv_load";
  if (const int rc = check_cache(name, k_cache, v_cache, k_exp, v_exp, cache_dtype, n_rows, nkv, hd, T, rows, nseq, total_tokens))
    return rc;
  if (nseq == 0 || total_tokens == 0) return GDN_OK;
  GDN_REQUIRE(out_k && out_v, "%s: null pointer", name);
  GDN_REQUIRE(aligned(out_k, 16) && aligned(out_v, 16), "%s: outputs must be 16-byte aligned", name);
  GDN_REQUIRE(cu_seqlens || total_tokens % nseq == 0, "%s: without cu_seqlens the tokens must divide into nseq sequences", name);
  const kv::Batch b{rows, cu_seqlens, start, nseq, n_rows, total_tokens};
  const dim3 g((unsigned)kv::most_tiles(total_tokens, nseq), nkv, 2);
  const hipStream_t st = (hipStream_t)stream;
  const auto *kc = static_cast<const uint8_t*>(k_cache), *vc = static_cast<const uint8_t*>(v_cache);
  auto *ok = static_cast<uint16_t*>(out_k), *ov = static_cast<uint16_t*>(out_v);
#define GDN_LOAD(HD, F8) kv_load_kernel<HD, F8><<<g, 256, 0, st>>>(kc, vc, k_exp, v_exp, ok, ov, nkv, T, b)
  const bool f8 = cache_dtype == GDN_F8E4M3;
  switch (hd) {
    case 64: if (f8) GDN_LOAD(64, true); else GDN_LOAD(64, false); break;
    case 128: if (f8) GDN_LOAD(128, true); else GDN_LOAD(128, false); break;
    default: if (f8) GDN_LOAD(256, true); else GDN_LOAD(256, false); break;
  }
#undef GDN_LOAD
  return check_launch(name);
}
