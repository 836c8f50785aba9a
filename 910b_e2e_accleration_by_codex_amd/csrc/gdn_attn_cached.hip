// Decode attention over the KV cache of gdn_kv.h (bf16 or e4m3), one new token for each of N slots, which may continue
// prefixes that several slots share (rows of another such cache, read once for all of a prefix's slots).
//
// For query head h of slot n, kv head j = h / G (G = nh / nkv):
//   q = rope(rmsnorm(proj_q) (1 + wq)), k, v: the new token's, written into the slot's cache row first;
//   o = sum_t p_t v_t / sum_t p_t, p_t = exp(q . k_t / sqrt(hd)), over the slot's prefix and its own tokens;
//   out = o sigmoid(gate).
// Launches:
//   1. cached_prep_kernel: a wave per (slot, head row).  Norm, rotary (angles in double), q to the workspace, k and
//      v quantised into the cache.  One more workgroup sorts the slots by prefix into tiles of 32 query rows.
//   2. cached_split_kernel: partial softmax sums of a range of tokens for 16 query rows (the G heads of one slot's kv
//      head) or 32 (a tile of a prefix's slots).
//   3. cached_combine_kernel: per (slot, head) the partials merged by their maxima, and the gate.
// Rounding: K and V enter as the cache holds them (e4m3 codes are bf16 values, their scales multiply scores and
// probabilities in fp32).  The query and the probabilities are fp32 values that enter the bf16 products as a high and a low
// part, two products each: one rounding of each to bf16 would nearly double the error of the rounded output (0.0031
// against 0.0017 relative), and these products are not what bounds the kernel.  The output is rounded once, to bf16.
#include "gdn_attn.h"
#include "gdn_device.h"
#include "gdn_internal.h"
#include "gdn_kv.h"

namespace gdn {
namespace cached {
using kv::BT;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// 8 e4m3 codes -> 8 bf16 values (exact).
__device__ __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
}
// A value as the sum of two bf16: the upper half of it, cut off (two values paired), and what is left.  Both parts have the
// value's sign, and against a bf16 cache, which may hold infinities, a low part of a value is never 0: times an infinity
// the parts' products are that infinity twice, as the value's is.
__device__ __forceinline__ uint32_t high2(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
template <bool F8> __device__ __forceinline__ float low(float x) {  // x >= 0
  const float r = x - __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  return F8 ? r : fmaxf(r, x > 0.f ? 0x1p-126f : 0.f);
}
// The registers' values are not needed any more: without this, a load that only one branch does keeps the other branch's old
// values alive.
template <int N> __device__ __forceinline__ void drop(u32x4 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "=v"(x[i]));
}
constexpr int WAVES = 4;       // per split workgroup; a wave takes every 4th block of the range
constexpr int PROWS = 32;      // query rows of a prefix tile

// Ranges that a row of up to T tokens is cut into (parts at most), of `least` blocks at least: a block per wave where a
// workgroup for each such range finds room on the chip at once (one fits a CU), else two, and about 4 workgroups a CU
// where rows are long.
struct Cut {
  int parts, least;
};
inline Cut cut_of(int64_t T, int64_t items) {
  const int64_t n = (T + BT - 1) / BT, four = (n + WAVES - 1) / WAVES;
  const int least = four * items <= 256 ? WAVES : 2 * WAVES;
  const int64_t most = (n + least - 1) / least, want = (1024 + items - 1) / items;
  return Cut{(int)(most < want ? most : want), least};
}
struct Side {  // one cache: its tensors and its length (tokens, a multiple of 64)
  uint8_t *k, *v, *ke, *ve;
  int64_t T;
};
struct Args {
  attn::Src proj;
  const int64_t* pos;
  const uint16_t *q_w, *k_w;
  const float* inv_freq;
  Side own, pre;
  const int32_t *plen, *pof;  // NULL: no prefixes
  int N, nh, nkv, rd, P, tiles;
  Cut S, SP;  // partials per head: of the slot's own tokens, of its prefix
  float eps;
  uint16_t* out;
  int64_t out_stride;
};
// workspace: q (fp32 [N, nh, hd]) | m, l (fp32 [N, nh, S + SP, 2]) | o (fp32 [N, nh, S + SP, hd]) | order (int32 [N]) |
// tiles (int32 [tiles, 4]: prefix, its first place in order, first row, rows)
struct Work {
  float *q, *ml, *o;
  int32_t* order;
  int4* tiles;
};
inline int most_tiles(int N, int G, int P) {  // a prefix of m slots has ceil(m G / 32) tiles
  const int64_t rows = (int64_t)N * G;
  const int64_t t = rows / PROWS + (P < N ? P : N);
  return (int)t;
}
__host__ __device__ inline int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }
inline int64_t work_of(Work& w, char* p, int N, int nh, int nkv, int hd, int parts, int P) {
  char* const base = p;
  w.q = reinterpret_cast<float*>(p);
  p += round256((int64_t)N * nh * hd * 4);
  w.ml = reinterpret_cast<float*>(p);
  p += round256((int64_t)N * nh * parts * 8);
  w.o = reinterpret_cast<float*>(p);
  p += round256((int64_t)N * nh * parts * hd * 4);
  w.order = reinterpret_cast<int32_t*>(p);
  p += P ? round256((int64_t)N * 4) : 0;
  w.tiles = reinterpret_cast<int4*>(p);
  p += P ? round256((int64_t)most_tiles(N, nh / nkv, P) * 16) : 0;
  return p - base;
}
// What a slot attends to.
struct Slot {
  int64_t own;  // tokens of its own, the new one included (0: position below 0, or inside the prefix)
  int64_t at;   // where the new token goes in its cache row, -1: nowhere
  int prefix;   // -1: none
};
__device__ __forceinline__ int64_t prefix_len(const Args& A, int r) {
  const int64_t n = A.plen[r];
  return n < 0 ? 0 : n > A.pre.T ? A.pre.T : n;
}
__device__ __forceinline__ Slot slot_of(const Args& A, int n) {
  Slot s;
  const int64_t p = A.pos[n];
  s.prefix = A.pof ? A.pof[n] : -1;
  if (s.prefix < 0 || s.prefix >= A.P || p < 0) s.prefix = -1;
  int64_t at = p - (s.prefix >= 0 ? prefix_len(A, s.prefix) : 0);
  if (p < 0 || at < 0) at = -1;
  s.own = at < A.own.T ? at + 1 : A.own.T;
  s.at = at < A.own.T ? at : -1;
  return s;
}
// Blocks per range of n blocks.
__device__ __forceinline__ int64_t range_blocks(int64_t n, const Cut& c) {
  const int64_t b = (n + c.parts - 1) / c.parts;
  return b < c.least ? c.least : b;
}
__device__ __forceinline__ int ranges(int64_t tokens, const Cut& c) {
  const int64_t n = (tokens + BT - 1) / BT;
  const int64_t b = range_blocks(n, c);
  return (int)((n + b - 1) / b);
}
}  // namespace cached

// Workgroup 0..: a wave per (slot, row), rows: nh query heads, nkv keys, nkv values; lane l holds dims l + 64 e.  The last
// workgroup (with prefixes): the slots in the order of their prefixes, and the tiles.
template <int HD, bool F8>
__global__ __launch_bounds__(256) void cached_prep_kernel(cached::Args A, cached::Work wk) {
  using namespace cached;
  constexpr int E = HD / 64;
  __shared__ float tmp[4][HD];
  const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (A.pof && blockIdx.x == gridDim.x - 1) {
    if (wid) return;
    const int G = A.nh / A.nkv;
    int at = 0, tile = 0;
    for (int r = 0; r < A.P; ++r) {
      const int first = at;
      for (int n0 = 0; n0 < A.N; n0 += 64) {
        const int n = n0 + lane;
        const bool mine = n < A.N && slot_of(A, n).prefix == r;
        const uint64_t b = __ballot(mine);
        if (mine) wk.order[at + __popcll(b & ((1ull << lane) - 1))] = n;
        at += __popcll(b);
      }
      const int rows = (at - first) * G;
      for (int t = 0; t * PROWS < rows; ++t, ++tile)
        if (lane == 0) wk.tiles[tile] = int4{r, first, t * PROWS, rows - t * PROWS < PROWS ? rows - t * PROWS : PROWS};
    }
    for (; tile < A.tiles; ++tile)
      if (lane == 0) wk.tiles[tile] = int4{0, 0, 0, 0};
    return;
  }
  const int per = A.nh + 2 * A.nkv;
  const int64_t w = (int64_t)blockIdx.x * 4 + wid;
  if (w >= (int64_t)A.N * per) return;  // whole waves: no barrier below
  const int n = (int)(w / per), r = (int)(w % per);
  const bool is_q = r < A.nh, is_v = r >= A.nh + A.nkv;
  const int j = is_q ? r : is_v ? r - A.nh - A.nkv : r - A.nh;
  const Slot s = slot_of(A, n);
  if (!is_q && s.at < 0) return;
  float x[E];
  A.proj.row<E>(x, n, is_q ? (int64_t)r * 2 * HD + lane : (int64_t)2 * A.nh * HD + (int64_t)(r - A.nh) * HD + lane);
  if (!is_v) {
    const uint16_t* nw = is_q ? A.q_w : A.k_w;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) ss += x[e] * x[e];
    const float inv = rsqrt_f(wave_sum_fast(ss) / (float)HD + A.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] = (x[e] * inv) * (1.0f + bf2f(nw[lane + 64 * e]));
      tmp[wid][lane + 64 * e] = x[e];
    }
    // one wave's LDS accesses complete in program order: the partner reads below see the writes
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int half = A.rd / 2;
    const double p = (double)A.pos[n];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + 64 * e;
      if (d < A.rd) {
        // a far position's angle is many turns: the turns come off in double
        const double ang = p * (double)A.inv_freq[d < half ? d : d - half];
        const double turns = rint(ang * 0.15915494309189535);
        const float a = (float)fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, ang));
        const float partner = d < half ? -tmp[wid][d + half] : tmp[wid][d - half];
        x[e] = x[e] * cosf(a) + partner * sinf(a);
      }
    }
  }
  if (is_q) {
#pragma unroll
    for (int e = 0; e < E; ++e) wk.q[((int64_t)n * A.nh + r) * HD + lane + 64 * e] = x[e];
    return;
  }
  const int64_t row = ((int64_t)n * A.nkv + j) * A.own.T;
  uint8_t* c = (is_v ? A.own.v : A.own.k) + row * HD * (F8 ? 1 : 2);
  float inv = 1.f;
  if constexpr (F8) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, kv::finite_abs(x[e]));
    const int ex = kv::scale_exp(wave_max_fast(top));
    inv = kv::pow2(-ex);
    if (lane == 0) (is_v ? A.own.ve : A.own.ke)[row + s.at] = (uint8_t)(ex + 127);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 64 * e;
    const int64_t i = is_v ? kv::v_at<F8>(s.at, d, HD) : kv::k_at<F8>(s.at, d, HD);
    if constexpr (F8) c[i] = (uint8_t)kv::quant2(x[e], 0.f, inv);
    else reinterpret_cast<uint16_t*>(c)[i] = f2bf(x[e]);
  }
}

// Query rows against a range of tokens.  RT = 1: grid (S, nkv, N), 16 rows, of which G are the slot's heads.  RT = 2: grid
// (SP, nkv, tiles), 32 rows of a prefix's slots.
//
// Wave w takes blocks w, w + 4, .. of the range; the waves' sums meet in LDS at the end.  Of a block of 64 tokens (lane =
// (c, g) = (l % 16, l / 16)):
//   scores: tile i < 4 is K (16 tokens x 32 dims, A) times q^T (32 dims x 16 rows, B).  Its row 4 a + r stands for token
//      16 a + 4 i + r, so that lane (c, g) ends with row c's scores of tokens 16 g .. 16 g + 15 (D_i, r: 16 g + 4 i + r);
//   P V: V^T (16 dims x 32 tokens, A) times P^T (32 tokens x 16 rows, B), the reduction's slot (g, e) of step u < 2 standing
//      for token 16 g + 8 u + e: the lane's own scores are its operand.  O's lane (c, g) has row c, dims 16 x + 4 g + r, so
//      the running maximum's corrections are a number per lane.
template <int HD, bool F8, int RT>
__global__ __launch_bounds__(256, RT == 1 && HD < 256 ? 2 : 1) void cached_split_kernel(cached::Args A, cached::Work wk, float scale2) {
  using namespace cached;
  constexpr int R = 16 * RT, LQ = HD + 8;
  constexpr int KS = HD / 32, X = HD / 16;  // 32-dim steps of the scores, 16-dim tiles of the output
  constexpr int DS = 64;                    // dims per round of the merge
  __shared__ alignas(16) uint16_t qs[2][R * LQ];
  __shared__ alignas(16) float so[WAVES][R][DS + 4];
  __shared__ float sm[WAVES][R], sl[WAVES][R];
  __shared__ int rown[R], rowh[R];  // each row's slot (-1: none) and head
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = blockIdx.x, j = blockIdx.y, G = A.nh / A.nkv;
  int64_t tokens, row;  // of the cache row
  const Side& side = RT == 1 ? A.own : A.pre;
  const Cut& cut = RT == 1 ? A.S : A.SP;
  if (RT == 1) {
    const int n = blockIdx.z;
    tokens = slot_of(A, n).own;
    row = n;
    if (tid < R) {
      rown[tid] = tid < G ? n : -1;
      rowh[tid] = j * G + tid;
    }
  } else {
    const int4 tile = wk.tiles[blockIdx.z];
    if (!tile.w) return;  // fewer tiles than there could be
    tokens = prefix_len(A, tile.x);
    row = tile.x;
    if (tid < R) {
      const int q = tile.z + tid;
      rown[tid] = tid < tile.w ? wk.order[tile.y + q / G] : -1;
      rowh[tid] = j * G + q % G;
    }
  }
  const int64_t nblk = (tokens + BT - 1) / BT, per = range_blocks(nblk, cut);
  const int64_t b0 = part * per, b1 = b0 + per < nblk ? b0 + per : nblk;
  if (b0 >= b1) return;
  lds_barrier();
  constexpr int S1 = F8 ? 1 : 2;
  constexpr int KL = HD / 16 * S1, VL = X * S1;  // 16-byte loads of a block's K and V, per lane
  // Loads ahead: the next block's K goes out when this one's scores are done, its V when this one's is used up.
  const int64_t hrow = (row * A.nkv + j) * side.T;
  const uint8_t* kp = side.k + hrow * HD * S1;
  const uint8_t* vp = side.v + hrow * HD * S1;
  const int kat = lane * 16, vat = c * 64 + g * 16;
  u32x4 kr[KL], vr[VL], kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
  // (buffer loads: the block's address is scalar, a lane's offset one register for all of them)
  auto load_k = [&](int64_t b) {
    if constexpr (F8) kx = *reinterpret_cast<const u32x4*>(side.ke + hrow + b * BT + 16 * g);
    const auto block = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(kp) + b * (BT * HD * S1), 0, BT * HD * S1, 0x00027000);
#pragma unroll
    for (int i = 0; i < KL; ++i) kr[i] = __builtin_amdgcn_raw_buffer_load_b128(block, kat, i * 1024, 0);
  };
  auto load_v = [&](int64_t b) {
    if constexpr (F8) vx = *reinterpret_cast<const u32x4*>(side.ve + hrow + b * BT + 16 * g);
    const auto block = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(vp) + b * (BT * HD * S1), 0, BT * HD * S1, 0x00027000);
#pragma unroll
    for (int i = 0; i < VL; ++i) vr[i] = __builtin_amdgcn_raw_buffer_load_b128(block, vat, i * 1024, 0);
  };
  float m[RT], l[RT];
  f32x4 O[RT][X];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int x = 0; x < X; ++x) O[t][x] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int64_t b = b0 + wid;
  if (b < b1) {
    load_k(b);
    load_v(b);
  }
  __builtin_amdgcn_sched_barrier(0);
  // ---- q into LDS, as a high and a low bf16 part
  for (int i = tid; i < R * (HD / 8); i += 64 * WAVES) {
    const int q = i / (HD / 8), d = 8 * (i % (HD / 8));
    f32x4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (rown[q] >= 0) {
      const f32x4* p = reinterpret_cast<const f32x4*>(&wk.q[((int64_t)rown[q] * A.nh + rowh[q]) * HD + d]);
      v[0] = p[0], v[1] = p[1];
    }
    u32x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = v[e / 2][2 * (e % 2)], b2 = v[e / 2][2 * (e % 2) + 1];
      hi[e] = high2(a, b2);
      lo[e] = f2bf2(copysignf(low<F8>(fabsf(a)), a), copysignf(low<F8>(fabsf(b2)), b2));
    }
    *reinterpret_cast<u32x4*>(&qs[0][q * LQ + d]) = hi;
    *reinterpret_cast<u32x4*>(&qs[1][q * LQ + d]) = lo;
  }
  lds_barrier();
  for (; b < b1; b += WAVES) {
    asm volatile("" ::: "memory");  // q is read again for each block: held in registers it would push others out
    // ---- scores
    f32x4 D[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) D[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 q[2][RT][2];  // of this step and the next
    auto load_q = [&](int s) {
      const int d = F8 ? 16 * (4 * (s / 2) + g) + 8 * (s % 2) : 8 * (4 * s + g);
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) q[s % 2][t][h] = *reinterpret_cast<const u32x4*>(&qs[h][(16 * t + c) * LQ + d]);
    };
    load_q(0);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (s + 1 < KS) load_q(s + 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4& k = kr[F8 ? s / 2 * 4 + i : s * 4 + i];
        const u32x4 a = F8 ? widen(k[s % 2 * 2], k[s % 2 * 2 + 1]) : k;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          D[t][i] = mma(a, q[s % 2][t][1], D[t][i]);
          D[t][i] = mma(a, q[s % 2][t][0], D[t][i]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const u32x4 kx1 = kx;
    __builtin_amdgcn_sched_barrier(0);
    if (b + WAVES < b1) load_k(b + WAVES);
    else drop(kr);
    __builtin_amdgcn_sched_barrier(0);
    const int left = (int)(tokens - b * BT < BT ? tokens - b * BT : BT);  // tokens of this block in range
    // ---- softmax of row c over the lane's 16 tokens and the other g's
    u32x4 pr[RT][2][2];  // [high and low part][step]
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float mx = m[t];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float f = scale2;
          if constexpr (F8) f *= __uint_as_float((kx1[i] >> (8 * r) & 0xffu) << 23);
          D[t][i][r] = 16 * g + 4 * i + r < left ? D[t][i][r] * f : -INFINITY;
          mx = fmaxf(mx, D[t][i][r]);
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
      mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
      const float m0 = mx == -INFINITY ? 0.f : mx;
      const float fix = __builtin_amdgcn_exp2f(m[t] - m0);
      m[t] = mx;
      l[t] *= fix;
#pragma unroll
      for (int x = 0; x < X; ++x) O[t][x] *= fix;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          float p0 = __builtin_amdgcn_exp2f(D[t][i][r] - m0), p1 = __builtin_amdgcn_exp2f(D[t][i][r + 1] - m0);
          l[t] += p0 + p1;
          if constexpr (F8) {  // V's scales, by a select where nothing is in range: a stray scale may be anything
            const int t0 = 16 * g + 4 * i + r;
            p0 = t0 < left ? p0 * __uint_as_float((vx[i] >> (8 * r) & 0xffu) << 23) : 0.f;
            p1 = t0 + 1 < left ? p1 * __uint_as_float((vx[i] >> (8 * r + 8) & 0xffu) << 23) : 0.f;
          }
          pr[t][0][i / 2][2 * (i % 2) + r / 2] = high2(p0, p1);
          pr[t][1][i / 2][2 * (i % 2) + r / 2] = f2bf2(low<F8>(p0), low<F8>(p1));
        }
    }
    // ---- P V
    if (left < BT) {  // what lies behind the last token may be anything, and 0 times an infinity is NaN
#pragma unroll
      for (int i = 0; i < VL; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          constexpr int TW = 4 / S1;  // tokens per word
          const int k = left - (16 * g + 8 * (i % S1) + TW * w);
          vr[i][w] &= k >= TW ? 0xffffffffu : k <= 0 ? 0u : (1u << (32 / TW * k)) - 1u;
        }
    }
#pragma unroll
    for (int x = 0; x < X; ++x) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 a = F8 ? widen(vr[x][2 * u], vr[x][2 * u + 1]) : vr[x * S1 + u * (S1 - 1)];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          O[t][x] = mma(a, pr[t][1][u], O[t][x]);
          O[t][x] = mma(a, pr[t][0][u], O[t][x]);
        }
      }
      if (x % 2) __builtin_amdgcn_sched_barrier(0);  // (or every V is widened before the first product)
    }
    __builtin_amdgcn_sched_barrier(0);
    if (b + WAVES < b1) load_v(b + WAVES);
    else drop(vr);
    __builtin_amdgcn_sched_barrier(0);
  }
  // ---- the waves' sums: one maximum, then DS dims at a time through LDS
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    l[t] = xor32_sum(xor16_sum(l[t]));
    if (g == 0) {
      sm[wid][16 * t + c] = m[t];
      sl[wid][16 * t + c] = l[t];
    }
  }
  __syncthreads();
  float fix[RT], M[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    M[t] = sm[0][16 * t + c];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) M[t] = fmaxf(M[t], sm[w][16 * t + c]);
    fix[t] = M[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[t] - M[t]);
  }
  const int at0 = RT == 1 ? part : A.S.parts + part, all = A.S.parts + A.SP.parts;
  if (wid == 0 && g == 0) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int q = 16 * t + c;
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
        L += M[t] == -INFINITY ? 0.f : sl[w][q] * __builtin_amdgcn_exp2f(sm[w][q] - M[t]);
      if (rown[q] >= 0) {
        float* ml = wk.ml + (((int64_t)rown[q] * A.nh + rowh[q]) * all + at0) * 2;
        ml[0] = M[t];
        ml[1] = L;
      }
    }
  }
#pragma unroll
  for (int d0 = 0; d0 < HD; d0 += DS) {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int x = 0; x < DS / 16; ++x)
        *reinterpret_cast<f32x4*>(&so[wid][16 * t + c][16 * x + 4 * g]) = O[t][d0 / 16 + x] * fix[t];
    __syncthreads();
    for (int i = tid; i < R * (DS / 4); i += 64 * WAVES) {
      const int q = i / (DS / 4), d = 4 * (i % (DS / 4));
      f32x4 o = *reinterpret_cast<const f32x4*>(&so[0][q][d]);
#pragma unroll
      for (int w = 1; w < WAVES; ++w) o += *reinterpret_cast<const f32x4*>(&so[w][q][d]);
      if (rown[q] >= 0)
        *reinterpret_cast<f32x4*>(&wk.o[(((int64_t)rown[q] * A.nh + rowh[q]) * all + at0) * HD + d0 + d]) = o;
    }
    __syncthreads();
  }
}

// grid (N * nh), 256 threads: HD / 4 lanes of 4 dims times groups of partials; the groups meet in LDS.
template <int HD>
__global__ __launch_bounds__(256) void cached_combine_kernel(cached::Args A, cached::Work wk) {
  using namespace cached;
  constexpr int LN = HD / 4, GR = 256 / LN;
  __shared__ alignas(16) float so[GR][HD];
  __shared__ float sl[GR];
  const int n = blockIdx.x / A.nh, h = blockIdx.x % A.nh, t = threadIdx.x, d4 = t % LN, gr = t / LN;
  const Slot s = slot_of(A, n);
  const int ns = ranges(s.own, A.S), np = s.prefix >= 0 ? ranges(prefix_len(A, s.prefix), A.SP) : 0, all = A.S.parts + A.SP.parts;
  const float* ml = wk.ml + ((int64_t)n * A.nh + h) * all * 2;
  const float* op = wk.o + ((int64_t)n * A.nh + h) * all * HD + 4 * d4;
  const float gate = t < HD ? A.proj(n, (int64_t)h * 2 * HD + HD + t) : 0.f;
  float M = -INFINITY;
  for (int i = t & 63; i < ns + np; i += 64) M = fmaxf(M, ml[2 * (i < ns ? i : A.S.parts + i - ns)]);
  M = wave_max_fast(M);
  const float m0 = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = gr; i < ns + np; i += GR) {
    const int at = i < ns ? i : A.S.parts + i - ns;
    const float f = __builtin_amdgcn_exp2f(ml[2 * at] - m0);
    L += ml[2 * at + 1] * f;
    o += *reinterpret_cast<const f32x4*>(op + (int64_t)at * HD) * f;
  }
  *reinterpret_cast<f32x4*>(&so[gr][4 * d4]) = o;
  if (d4 == 0) sl[gr] = L;
  __syncthreads();
  if (t >= HD) return;
  float a = 0.f;
  L = 0.f;
#pragma unroll
  for (int x = 0; x < GR; ++x) {
    a += so[x][t];
    L += sl[x];
  }
  // a slot that attends to nothing: zero output
  A.out[n * A.out_stride + (int64_t)h * HD + t] = f2bf(ns + np > 0 ? a / L / (1.0f + expf(-gate)) : 0.f);
}

template <int HD, bool F8>
static int launch_cached(const cached::Args& A, const cached::Work& wk, hipStream_t st) {
  const int64_t waves = (int64_t)A.N * (A.nh + 2 * A.nkv);
  const float scale2 = 1.4426950408889634f / sqrtf((float)HD);  // scores in powers of two
  cached_prep_kernel<HD, F8><<<(unsigned)((waves + 3) / 4 + (A.pof ? 1 : 0)), 256, 0, st>>>(A, wk);
  cached_split_kernel<HD, F8, 1><<<dim3(A.S.parts, A.nkv, A.N), 256, 0, st>>>(A, wk, scale2);
  if (A.pof)
    cached_split_kernel<HD, F8, 2>
        <<<dim3(A.SP.parts, A.nkv, A.tiles), 256, 0, st>>>(A, wk, scale2);
  cached_combine_kernel<HD><<<A.N * A.nh, 256, 0, st>>>(A, wk);
  return check_launch("gdn_attn_cached");
}

}  // namespace gdn

using namespace gdn;

namespace {
// Partials per head of the own tokens and of the prefix.
void cached_cuts(int N, int nh, int nkv, int64_t T, int P, int64_t Tp, cached::Cut& S, cached::Cut& SP) {
  S = cached::cut_of(T, (int64_t)N * nkv);
  SP = P ? cached::cut_of(Tp, (int64_t)cached::most_tiles(N, nh / nkv, P) * nkv) : cached::Cut{0, 1};
}
bool cached_sizes(int N, int nh, int nkv, int64_t T, int P, int64_t Tp) {
  return N >= 0 && nh >= 1 && nkv >= 1 && nh % nkv == 0 && nkv <= 65535 && N <= 65535 && P >= 0 && T >= kv::BT &&
         T % kv::BT == 0 && T <= INT32_MAX && (P == 0 || (Tp >= kv::BT && Tp % kv::BT == 0 && Tp <= INT32_MAX)) &&
         (int64_t)N * nh <= INT32_MAX && P <= 65535;
}
}  // namespace

extern "C" int64_t gdn_attn_cached_workspace_bytes(int N, int nh, int nkv, int hd, int64_t T, int P, int64_t Tp) {
  if (!cached_sizes(N, nh, nkv, T, P, Tp) || hd < 1) return -1;
  cached::Cut S, SP;
  cached_cuts(N < 1 ? 1 : N, nh, nkv, T, P, Tp, S, SP);
  cached::Work w;
  return cached::work_of(w, nullptr, N, nh, nkv, hd, S.parts + SP.parts, P);
}

extern "C" int gdn_attn_cached(const void* proj, int64_t proj_stride, const float* part, int splits, const int64_t* pos,
                               const void* q_norm_w, const void* k_norm_w, const float* inv_freq, void* k_cache,
                               void* v_cache, uint8_t* k_exp, uint8_t* v_exp, int cache_dtype, int64_t T,
                               const void* pre_k, const void* pre_v, const uint8_t* pre_k_exp, const uint8_t* pre_v_exp,
                               const int32_t* prefix_len, const int32_t* prefix_of, int P, int64_t Tp, void* out,
                               int64_t out_stride, void* work, int64_t work_bytes, int N, int nh, int nkv, int hd, int rd,
                               float eps, void* stream) {
  clear_error();
  const char* name = "gdn_attn_cached";
  GDN_REQUIRE(cached_sizes(N, nh, nkv, T, P, Tp), "%s: bad head counts, sizes, or a cache length that is no positive multiple of 64", name);
  GDN_REQUIRE(cache_dtype == GDN_BF16 || cache_dtype == GDN_F8E4M3, "%s: the cache's dtype must be bf16 or e4m3", name);
  GDN_SUPPORT(hd == 64 || hd == 128 || hd == 256, "%s: head_dim must be 64, 128 or 256", name);
  GDN_SUPPORT(nh / nkv <= 16, "%s: at most 16 query heads per kv head", name);
  GDN_REQUIRE(rd >= 0 && rd <= hd && rd % 2 == 0, "%s: rotary dims must be even and <= head_dim", name);
  if (N == 0) return GDN_OK;
  const bool f8 = cache_dtype == GDN_F8E4M3;
  GDN_REQUIRE((proj || part) && pos && q_norm_w && k_norm_w && (inv_freq || rd == 0) && k_cache && v_cache && out && work &&
                  (!f8 || (k_exp && v_exp)), "%s: null pointer", name);
  GDN_REQUIRE(!P || (pre_k && pre_v && prefix_len && prefix_of && (!f8 || (pre_k_exp && pre_v_exp))), "%s: null prefix pointer", name);
  GDN_REQUIRE(part ? splits >= 1 : proj_stride >= (int64_t)(2 * nh + 2 * nkv) * hd, "%s: bad projection", name);
  GDN_REQUIRE(out_stride >= (int64_t)nh * hd, "%s: output row stride too small", name);
  GDN_REQUIRE(aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(k_exp, 16) && aligned(v_exp, 16) && aligned(pre_k, 16) &&
                  aligned(pre_v, 16) && aligned(pre_k_exp, 16) && aligned(pre_v_exp, 16) && aligned(work, 256) && aligned(pos, 8),
              "%s: caches and exponents must be 16-byte, the workspace 256-byte aligned", name);
  cached::Args A{};
  A.proj = part ? attn::Src{nullptr, 0, part, splits, N, (int64_t)(2 * nh + 2 * nkv) * hd}
                : attn::Src{static_cast<const uint16_t*>(proj), proj_stride, nullptr, 0, N, 0};
  A.pos = pos;
  A.q_w = static_cast<const uint16_t*>(q_norm_w);
  A.k_w = static_cast<const uint16_t*>(k_norm_w);
  A.inv_freq = inv_freq;
  A.own = {static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), k_exp, v_exp, T};
  A.pre = {static_cast<uint8_t*>(const_cast<void*>(pre_k)), static_cast<uint8_t*>(const_cast<void*>(pre_v)),
           const_cast<uint8_t*>(pre_k_exp), const_cast<uint8_t*>(pre_v_exp), Tp};
  A.plen = P ? prefix_len : nullptr;
  A.pof = P ? prefix_of : nullptr;
  A.N = N, A.nh = nh, A.nkv = nkv, A.rd = rd, A.P = P, A.tiles = P ? cached::most_tiles(N, nh / nkv, P) : 0;
  A.eps = eps;
  A.out = static_cast<uint16_t*>(out);
  A.out_stride = out_stride;
  cached_cuts(N, nh, nkv, T, P, Tp, A.S, A.SP);
  cached::Work wk;
  const int64_t need = cached::work_of(wk, static_cast<char*>(work), N, nh, nkv, hd, A.S.parts + A.SP.parts, P);
  GDN_REQUIRE(work_bytes >= need, "%s: workspace too small (%lld bytes needed)", name, (long long)need);
  const hipStream_t st = (hipStream_t)stream;
  switch (hd) {
    case 64: return f8 ? launch_cached<64, true>(A, wk, st) : launch_cached<64, false>(A, wk, st);
    case 128: return f8 ? launch_cached<128, true>(A, wk, st) : launch_cached<128, false>(A, wk, st);
    default: return f8 ? launch_cached<256, true>(A, wk, st) : launch_cached<256, false>(A, wk, st);
  }
}
