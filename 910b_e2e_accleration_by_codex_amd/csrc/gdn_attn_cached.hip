// Decode attention over the KV cache of gdn_kv.h (bf16 or e4m3), one new token for each of N slots, which may continue
// prefixes that several slots share (rows of another such cache, read once for all of a prefix's slots).
//
// For query head h of slot n, kv head j = h / G (G = nh / nkv):
//   q = rope(rmsnorm(proj_q) (1 + wq)), k, v: the new token's, written into the slot's cache row first;
//   o = sum_t p_t v_t / sum_t p_t, p_t = exp(q . k_t / sqrt(hd)), over the slot's prefix and its own tokens;
//   out = o sigmoid(gate).
// Launches:
//   1. cached_prep_kernel: a wave per (slot, head row).  Norm, rotary (angles in double), q to the workspace, k and v
//      quantised into the cache.  A few more workgroups plan: they sort the slots by prefix into tiles of 32 query rows, and cut
//      every slot's own tokens and every tile's prefix into ranges of like cost, a workgroup each.
//   2. cached_split_kernel: partial softmax sums of a range of tokens for 16 query rows (the G heads of one slot's kv
//      head) or 32 (a tile of a prefix's slots).
//   3. cached_combine_kernel: per (slot, head) the partials merged by their maxima, and the gate.
// Rounding: K and V enter as the cache holds them (e4m3 codes are fp16 and bf16 values, their scales multiply scores and
// probabilities in fp32).  The query and the probabilities enter the products as a high and a low part, two products each:
// one rounding of each to bf16 would nearly double the error of the rounded output (0.0031 against 0.0017 relative).  The
// query's parts are fp16 against e4m3 keys, in units of its row's largest value (22 bits and more), bf16 against bf16 keys,
// and the probabilities' bf16 (16 bits).  A query of 11 bits would do at scores of a few units, but its error grows with
// them: at scores of 400 the output would be off by 2 to 4 %.  The output is rounded once, to bf16.
//
// Measured, 24 query and 4 kv heads of 256 (a large read runs at 6.07 TB/s, a large bf16 product at 1374 TFLOP/s), the
// kernels' medians in us:
//                                               bytes    prep  split  combine  split's rate
//   16 slots of 512 to 4096 tokens, e4m3       76 MB     4.3   18.6    4.0     4.1 TB/s
//   the same, bf16                            152 MB     4.2   27.7    4.2     5.5 TB/s
//   16 slots of 16384 to 32768 tokens, e4m3   809 MB     5.9  157      6.2     5.2 TB/s
//   16 slots behind 8192 shared tokens, e4m3   35 MB     5.9   21.4    4.8     160 TFLOP/s
//   64 slots behind 2 x 16384, e4m3           108 MB     7.4   84      5.5     312 TFLOP/s
// Slots' own tokens are bound by HBM, and where few, by the latency of a workgroup's start and merge (6 us of the 18.6: 76 MB
// read are 12.5).
// A prefix's tiles are bound by the vector instructions around the products (codes widened, the softmax, probabilities
// split and scaled) at one wave a SIMD: about 6 us a block of 64 tokens, of which the last case's waves take 13 each.
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
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// 8 e4m3 codes -> 8 fp16 values (exact), and 8 bf16 values (exact).
__device__ __forceinline__ u32x4 widen16(uint32_t lo, uint32_t hi) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true))};
}
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
// The scheduler is asked for N products, each followed by an arithmetic instruction.
template <int N> __device__ __forceinline__ void mix() {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x2, 1, 0);
  }
}
// The registers' values are not needed any more: without this, a load that only one branch does keeps the other branch's old
// values alive.
template <int N> __device__ __forceinline__ void drop(u32x4 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "=v"(x[i]));
}
constexpr int WAVES = 4;       // per split workgroup; a wave takes every 4th block of the range
constexpr int PROWS = 32;      // query rows of a prefix tile

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
  int N, nh, nkv, rd, P;
  int items, tiles, own_parts, pre_parts;  // at most so many of each
  float eps;
  uint16_t* out;
  int64_t out_stride;
};
// The plan.  A workgroup's part of the work; a slot's partials; a tile of a prefix's query rows.
struct Item {
  int tile;      // -1: a slot's own tokens
  int row, j;    // cache row (the slot, or the prefix), kv head
  int b0, b1;    // blocks (b0 = b1: nothing)
  int tokens;    // of the row
  int part;      // where its partials go
  int pad;
};
struct SlotPlan {
  int first, count;  // its own partials
  int tile, rank;    // its prefix's first tile (-1: none), and its place among that prefix's slots
};
struct TilePlan {
  int prefix, order, row, rows;  // query rows row .. row + rows - 1 of the prefix's slots, which begin at `order`
  int first, count;              // its partials
  int pad[2];
};
// workspace: q's parts ([N, nh, 2, hd], fp16 for an e4m3 cache, bf16 for a bf16 one), its rows' scales (fp32 [N, nh]) |
// partials: m, l (fp32 [parts, 2]) and o (fp32 [parts, hd]), parts = own_parts * nkv * G of slots, then
// pre_parts * nkv * 32 of tiles | the plan
struct Work {
  uint16_t* q;
  float *scale, *ml, *o;
  Item* items;
  SlotPlan* slots;
  TilePlan* tiles;
  int32_t* order;  // the slots, prefix after prefix
};
constexpr int WGS = 256;   // workgroups planned for where ranges are short: one a CU
constexpr int LONG = 12;   // blocks of a range when four are planned for each CU
constexpr int MAXN = 1024, MAXP = 1024;  // slots and prefixes (the plan is made in LDS)
inline int most_tiles(int N, int G, int P) {  // a prefix of m slots has ceil(m G / 32) tiles
  return P ? (int)((int64_t)N * G / PROWS + (P < N ? P : N)) : 0;
}
__host__ __device__ inline int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }
// The plan's bounds: ranges of like cost are at most WGS / nkv + 1 in all (of slots' own tokens 4 times that, if caches of
// T and prefixes of Tp tokens can hold so many), and one more for each slot and tile (rounding up).
inline void bound(Args& A, int G, int64_t T, int64_t Tp) {
  A.tiles = most_tiles(A.N, G, A.P);
  const int most = WGS / A.nkv + 1;
  const bool many = (A.N * (T / BT) + 2 * A.tiles * (Tp / BT)) / most + 1 >= 4 * LONG;
  A.own_parts = (many ? 4 : 1) * most + A.N;
  A.pre_parts = A.P ? most + A.tiles : 0;
  A.items = (A.own_parts + A.pre_parts) * A.nkv;
}
inline int64_t work_of(Work& w, char* p, const Args& A, int hd) {
  char* const base = p;
  auto take = [&p](int64_t bytes) {
    char* q = p;
    p += round256(bytes);
    return q;
  };
  const int64_t parts = (int64_t)A.own_parts * A.nh + (int64_t)A.pre_parts * A.nkv * PROWS;
  w.q = reinterpret_cast<uint16_t*>(take((int64_t)A.N * A.nh * hd * 4));
  w.scale = reinterpret_cast<float*>(take((int64_t)A.N * A.nh * 4));
  w.ml = reinterpret_cast<float*>(take(parts * 8));
  w.o = reinterpret_cast<float*>(take(parts * hd * 4));
  w.items = reinterpret_cast<Item*>(take((int64_t)A.items * sizeof(Item)));
  w.slots = reinterpret_cast<SlotPlan*>(take((int64_t)A.N * sizeof(SlotPlan)));
  w.tiles = reinterpret_cast<TilePlan*>(take((int64_t)A.tiles * sizeof(TilePlan)));
  w.order = reinterpret_cast<int32_t*>(take(A.P ? (int64_t)A.N * 4 : 0));
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
template <typename Len> __device__ __forceinline__ Slot slot_of(const Args& A, int n, Len len) {  // len(r): prefix r's tokens
  Slot s;
  const int64_t p = A.pos[n];
  s.prefix = A.pof ? A.pof[n] : -1;
  if (s.prefix < 0 || s.prefix >= A.P || p < 0) s.prefix = -1;
  int64_t at = p - (s.prefix >= 0 ? len(s.prefix) : 0);
  if (p < 0 || at < 0) at = -1;
  s.own = at < A.own.T ? at + 1 : A.own.T;
  s.at = at < A.own.T ? at : -1;
  return s;
}
__device__ __forceinline__ int blocks(int64_t tokens) { return (int)((tokens + BT - 1) / BT); }
struct PlanLds {
  alignas(16) int prefix[MAXN];
  int tokens[MAXN], first[MAXN + 1];
  // a prefix's slots, tokens, first tile, place in order, first range of all its tiles
  int count[MAXP], len[MAXP], tile[MAXP + 1], order[MAXP + 1], part[MAXP + 1];
  uint64_t cost[4];  // each wave's slots' and prefixes'
  int own, pre, wave[4];
};
// The sum of x over the threads before this one (256 threads; s.wave is free before and after).
__device__ __forceinline__ int before(int x, PlanLds& s) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int up = scan_up(x);
  if (lane == 63) s.wave[wid] = up;
  __syncthreads();
  int at = up - x;
  for (int w = 0; w < wid; ++w) at += s.wave[w];
  __syncthreads();
  return at;
}
// The last entry that is at most f, of n ascending ones that begin with 0 (where several are alike, all but the last are of
// something empty).
__device__ __forceinline__ int entry_of(const int* first, int n, int f) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (first[mid] <= f) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// Workgroups of 256 threads, each of which finds the ranges and writes its share of the plan.  Ranges cost the same: a block of a tile, with twice the query rows, counts as two of a
// slot's own.  Ranges are whole turns of a workgroup's waves.
__device__ __forceinline__ void make_plan(const Args& A, const Work& wk, int planner, int planners, PlanLds& s) {
  const int tid = threadIdx.x, G = A.nh / A.nkv;
  const int i0 = planner * 256 + tid, step = planners * 256;  // of what is written
  for (int r = tid; r < A.P; r += 256) {
    s.count[r] = 0;
    s.len[r] = (int)prefix_len(A, r);
  }
  __syncthreads();
  uint64_t cost = 0;
  for (int n = tid; n < A.N; n += 256) {
    const Slot x = slot_of(A, n, [&](int r) { return (int64_t)s.len[r]; });
    s.tokens[n] = (int)x.own;
    s.prefix[n] = x.prefix;
    cost += blocks(x.own);
    if (x.prefix >= 0) atomicAdd(&s.count[x.prefix], 1);
  }
  __syncthreads();
  // thread t's prefixes are r0 .. r1 - 1, its slots n0 .. n1 - 1
  const int rp = (A.P + 255) / 256, r0 = tid * rp, r1 = r0 + rp < A.P ? r0 + rp : A.P;
  const int np = (A.N + 255) / 256, n0 = tid * np, n1 = n0 + np < A.N ? n0 + np : A.N;
  auto tiles_of = [&](int r) { return (s.count[r] * G + PROWS - 1) / PROWS; };
  if (A.P) {
    int sum = 0;  // tiles, at most 1536, times 65536, and slots
    for (int r = r0; r < r1; ++r) {
      sum += tiles_of(r) << 16 | s.count[r];
      cost += 2ull * tiles_of(r) * blocks(s.len[r]);
    }
    sum = before(sum, s);
    for (int r = r0; r < r1; ++r) {
      s.tile[r] = sum >> 16, s.order[r] = sum & 0xffff;
      sum += tiles_of(r) << 16 | s.count[r];
    }
    if (r0 < r1 && r1 == A.P) s.tile[A.P] = sum >> 16;
  }
  cost = wave_total(cost);
  if ((tid & 63) == 0) s.cost[tid >> 6] = cost;
  __syncthreads();
  if (tid == 0) {
    // a workgroup a CU; of slots' own tokens, which HBM bounds, 4 that even out where there are many blocks (16 slots of
    // 16384 to 32768 tokens: 199 us with one, 154 with four; 64 slots behind 16384 shared tokens: 105 us with four, 91)
    uint64_t each = (s.cost[0] + s.cost[1] + s.cost[2] + s.cost[3] + WGS / A.nkv) / (WGS / A.nkv + 1);
    if (each > 1 << 28) each = 1 << 28;
    s.pre = (int)((each + 2 * WAVES - 1) / (2 * WAVES)) * WAVES;
    if (each >= 4 * LONG) each = (each + 3) / 4;
    s.own = (int)((each + WAVES - 1) / WAVES) * WAVES;
  }
  __syncthreads();
  // ranges of a slot, and of one tile of a prefix
  auto own_of = [&](int n) { return s.own ? (blocks(s.tokens[n]) + s.own - 1) / s.own : 0; };
  auto pre_of = [&](int r) { return s.pre && s.count[r] ? (blocks(s.len[r]) + s.pre - 1) / s.pre : 0; };
  int sum = 0;  // ranges of slots, at most 5 WGS + MAXN, times 65536, and of tiles
  for (int n = n0; n < n1; ++n) sum += own_of(n) << 16;
  for (int r = r0; r < r1; ++r) sum += pre_of(r) * tiles_of(r);
  sum = before(sum, s);
  int at = sum >> 16, part = sum & 0xffff;
  for (int n = n0; n < n1; ++n) {
    s.first[n] = at;
    at += own_of(n);
  }
  if (n0 < n1 && n1 == A.N) s.first[A.N] = at;
  for (int r = r0; r < r1; ++r) {
    s.part[r] = part;
    part += pre_of(r) * tiles_of(r);
  }
  if (r0 < r1 && r1 == A.P) s.part[A.P] = part;
  __syncthreads();
  for (int n = i0; n < A.N; n += step) {
    SlotPlan p{s.first[n], s.first[n + 1] - s.first[n], -1, 0};
    const int r = s.prefix[n];
    if (r >= 0) {
      p.tile = s.tile[r];
#pragma unroll 4
      for (int m = 0; m < A.N; m += 4) {  // (as far for every slot: the reads are the same, and go out together)
        const int4 x = *reinterpret_cast<const int4*>(&s.prefix[m]);
        p.rank += (m < n && x.x == r) + (m + 1 < n && x.y == r) + (m + 2 < n && x.z == r) + (m + 3 < n && x.w == r);
      }
      wk.order[s.order[r] + p.rank] = n;
    }
    wk.slots[n] = p;
  }
  // ---- prefixes first, as they are the longest.  A range's tiles lie 8 workgroups apart: on one XCD, whose L2 then
  // has the range's keys and values for all of them
  int item = 0;
  if (A.P) {
    for (int t = i0; t < s.tile[A.P]; t += step) {
      const int r = entry_of(s.tile, A.P, t), in = t - s.tile[r], left = s.count[r] * G - in * PROWS, parts = pre_of(r);
      wk.tiles[t] = TilePlan{r, s.order[r], in * PROWS, left < PROWS ? left : PROWS, s.part[r] + in * parts, parts, {0, 0}};
    }
    item = s.part[A.P] * A.nkv;
    for (int i = i0; i < item; i += step) {
      const int r = entry_of(s.part, A.P, i / A.nkv), nt = tiles_of(r), parts = pre_of(r), units = parts * A.nkv;
      const int x = i - s.part[r] * A.nkv, group = x / (8 * nt), in = x % (8 * nt);
      const int left = units - 8 * group, w = left < 8 ? left : 8;
      const int t = in / w, u = 8 * group + in % w, p = u / A.nkv, end = (p + 1) * s.pre;
      const int nb = blocks(s.len[r]);
      wk.items[i] = Item{s.tile[r] + t, r, u % A.nkv, p * s.pre, end < nb ? end : nb, s.len[r], s.part[r] + t * parts + p, 0};
    }
  }
  // ---- the slots' own tokens
  const int own = s.first[A.N] * A.nkv;
  for (int i = i0; item + i < A.items; i += step) {
    Item x{-1, 0, 0, 0, 0, 0, 0, 0};
    if (i < own) {
      const int f = i / A.nkv, n = entry_of(s.first, A.N, f);
      const int nb = blocks(s.tokens[n]), parts = s.first[n + 1] - s.first[n], in = i - s.first[n] * A.nkv;
      const int p = in % parts, end = (p + 1) * s.own;
      x = Item{-1, n, in / parts, p * s.own, end < nb ? end : nb, s.tokens[n], s.first[n] + p, 0};
    }
    wk.items[item + i] = x;
  }
}
template <int HD, int RT> struct SplitLds {
  static constexpr int R = 16 * RT, LQ = HD + 8;  // query rows, and their pitch
  static constexpr int DS = 64;                   // dims per round of the merge
  alignas(16) uint16_t qs[2][R * LQ];  // q's high and low parts
  alignas(16) float so[WAVES][R][DS + 4];
  float sm[WAVES][R], sl[WAVES][R];
  int rown[R], rowh[R];  // each row's slot (-1: none) and head
};
}  // namespace cached

// A wave per (slot, row), rows: nh query heads, nkv keys, nkv values; lane l holds dims l + 64 e.  The first workgroups plan.
template <int HD, bool F8>
__global__ __launch_bounds__(256) void cached_prep_kernel(cached::Args A, cached::Work wk, int planners) {
  using namespace cached;
  constexpr int E = HD / 64;
  __shared__ union {
    float tmp[4][HD];
    PlanLds plan;
  } lds;
  auto& tmp = lds.tmp;
  const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if ((int)blockIdx.x < planners) {
    make_plan(A, wk, blockIdx.x, planners, lds.plan);
    return;
  }
  const int per = A.nh + 2 * A.nkv;
  const int64_t w = (int64_t)(blockIdx.x - planners) * 4 + wid;
  if (w >= (int64_t)A.N * per) return;  // whole waves: no barrier below
  const int n = (int)(w / per), r = (int)(w % per);
  const bool is_q = r < A.nh, is_v = r >= A.nh + A.nkv;
  const int j = is_q ? r : is_v ? r - A.nh - A.nkv : r - A.nh;
  const Slot s = slot_of(A, n, [&](int p) { return prefix_len(A, p); });
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
    const int64_t at = (int64_t)n * A.nh + r;
    if constexpr (F8) {  // fp16, the row's largest value between 2^14 and 2^15
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) top = fmaxf(top, kv::finite_abs(x[e]));
      const int e0 = (int)(__float_as_uint(wave_max_fast(top)) >> 23) - 141, ex = e0 < -100 ? -100 : e0;  // (or below, or zeros)
      const float inv = kv::pow2(-ex);
      if (lane == 0) wk.scale[at] = kv::pow2(ex);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const _Float16 hi = (_Float16)(x[e] * inv), lo = (_Float16)(x[e] * inv - (float)hi);  // (not finite: hi alone)
        wk.q[2 * at * HD + lane + 64 * e] = __builtin_bit_cast(uint16_t, hi);
        wk.q[(2 * at + 1) * HD + lane + 64 * e] = fabsf(x[e]) < INFINITY ? __builtin_bit_cast(uint16_t, lo) : 0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        wk.q[(2 * at) * HD + lane + 64 * e] = (uint16_t)(__float_as_uint(x[e]) >> 16);
        wk.q[(2 * at + 1) * HD + lane + 64 * e] = f2bf(copysignf(low<false>(fabsf(x[e])), x[e]));
      }
    }
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

// Query rows against a range of tokens: RT = 1: 16 rows, of which G are the slot's heads; RT = 2: 32 rows of a prefix's slots.
//
// Wave w takes blocks w, w + 4, .. of the range; the waves' sums meet in LDS at the end.  Of a block of 64 tokens (lane =
// (c, g) = (l % 16, l / 16)):
//   scores: tile i < 4 is K (16 tokens x 32 dims, A) times q^T (32 dims x 16 rows, B).  Its row 4 a + r stands for token
//      16 a + 4 i + r, so that lane (c, g) ends with row c's scores of tokens 16 g .. 16 g + 15 (D_i, r: 16 g + 4 i + r);
//   P V: V^T (16 dims x 32 tokens, A) times P^T (32 tokens x 16 rows, B), the reduction's slot (g, e) of step u < 2 standing
//      for token 16 g + 8 u + e: the lane's own scores are its operand.  O's lane (c, g) has row c, dims 16 x + 4 g + r, so
//      the running maximum's corrections are a number per lane.
template <int HD, bool F8, int RT>
__device__ __forceinline__ void split(const cached::Args& A, const cached::Work& wk, const cached::Item& it, cached::SplitLds<HD, RT>& lds,
                                      float scale2) {
  using namespace cached;
  typedef SplitLds<HD, RT> Lds;
  constexpr int R = Lds::R, LQ = Lds::LQ, DS = Lds::DS;
  constexpr int KS = HD / 32, X = HD / 16;  // 32-dim steps of the scores, 16-dim tiles of the output
  auto& qs = lds.qs;
  auto& so = lds.so;
  auto& sm = lds.sm;
  auto& sl = lds.sl;
  auto& rown = lds.rown;
  auto& rowh = lds.rowh;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = it.j, G = A.nh / A.nkv, tokens = it.tokens;
  const Side& side = RT == 1 ? A.own : A.pre;
  if (RT == 1) {
    if (tid < R) {
      rown[tid] = tid < G ? it.row : -1;
      rowh[tid] = j * G + tid;
    }
  } else {
    const TilePlan tile = wk.tiles[it.tile];
    if (tid < R) {
      const int q = tile.row + tid;
      rown[tid] = tid < tile.rows ? wk.order[tile.order + q / G] : -1;
      rowh[tid] = j * G + q % G;
    }
  }
  lds_barrier();
  constexpr int S1 = F8 ? 1 : 2;
  constexpr int KL = HD / 16 * S1, VL = X * S1;  // 16-byte loads of a block's K and V, per lane
  // Loads ahead: the next block's K goes out when this one's scores are done, its V when this one's is used up.
  const int64_t hrow = ((int64_t)it.row * A.nkv + j) * side.T;
  const uint8_t* kp = side.k + hrow * HD * S1;
  const uint8_t* vp = side.v + hrow * HD * S1;
  const int kat = lane * 16, vat = c * 64 + g * 16;
  u32x4 kr[KL], vr[VL], kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
  // (buffer loads: the block's address is scalar, a lane's offset one register for all of them)
  auto load_k = [&](int b) {
    if constexpr (F8) kx = *reinterpret_cast<const u32x4*>(side.ke + hrow + (int64_t)b * BT + 16 * g);
    const auto block = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(kp) + (int64_t)b * (BT * HD * S1), 0, BT * HD * S1, 0x00027000);
#pragma unroll
    for (int i = 0; i < KL; ++i) kr[i] = __builtin_amdgcn_raw_buffer_load_b128(block, kat, i * 1024, 0);
  };
  auto load_v = [&](int b) {
    if constexpr (F8) vx = *reinterpret_cast<const u32x4*>(side.ve + hrow + (int64_t)b * BT + 16 * g);
    const auto block = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(vp) + (int64_t)b * (BT * HD * S1), 0, BT * HD * S1, 0x00027000);
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
  const int b1 = it.b1;
  int b = it.b0 + wid;
  if (b < b1) {
    load_k(b);
    load_v(b);
  }
  __builtin_amdgcn_sched_barrier(0);
  // ---- q into LDS
#pragma unroll 4
  for (int i = tid; i < 2 * R * (HD / 8); i += 64 * WAVES) {
    const int q = i / (HD / 8) / 2, h = i / (HD / 8) % 2, d = 8 * (i % (HD / 8));
    u32x4 v = {0, 0, 0, 0};
    if (rown[q] >= 0) v = *reinterpret_cast<const u32x4*>(&wk.q[(((int64_t)rown[q] * A.nh + rowh[q]) * 2 + h) * HD + d]);
    *reinterpret_cast<u32x4*>(&qs[h][q * LQ + d]) = v;
  }
  float sc[RT];  // row c's scores in powers of two
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int q = 16 * t + c;
    sc[t] = scale2;
    if (F8 && rown[q] >= 0) sc[t] *= wk.scale[(int64_t)rown[q] * A.nh + rowh[q]];
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
    // Operands of a step: q, and K of its 4 tiles.  With 32 query rows, one wave a SIMD, the next step's e4m3 codes are
    // widened among this one's products; with 16, two waves a SIMD fill each other's gaps, and 256 registers are all there
    // are: two tiles at a time (6 registers too many, in scratch: 158 -> 186 us for 16 slots of 16384 to 32768 tokens).
    constexpr int AHEAD = RT == 2 && F8 ? 1 : 0, W = AHEAD ? 4 : 2;
    u32x4 a[AHEAD + 1][W], q[AHEAD + 1][RT][2];
    auto query = [&](int s) {
      const int d = F8 ? 16 * (4 * (s / 2) + g) + 8 * (s % 2) : 8 * (4 * s + g);
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          q[s % (AHEAD + 1)][t][h] = *reinterpret_cast<const u32x4*>(&qs[h][(16 * t + c) * LQ + d]);
    };
    auto keys = [&](int s, int i0) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const u32x4& k = kr[F8 ? s / 2 * 4 + i0 + i : s * 4 + i0 + i];
        a[s % (AHEAD + 1)][i] = F8 ? widen16(k[s % 2 * 2], k[s % 2 * 2 + 1]) : k;
      }
    };
    if (AHEAD) query(0), keys(0, 0);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (!AHEAD) query(s);
      else if (s + 1 < KS) query(s + 1), keys(s + 1, 0);
#pragma unroll
      for (int i0 = 0; i0 < 4; i0 += W) {
        if (!AHEAD) keys(s, i0);
#pragma unroll
        for (int h = 1; h >= 0; --h)
#pragma unroll
          for (int i = 0; i < W; ++i)
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              const u32x4 &x = a[s % (AHEAD + 1)][i], &y = q[s % (AHEAD + 1)][t][h];
              D[t][i0 + i] = F8 ? mma16(x, y, D[t][i0 + i]) : mma(x, y, D[t][i0 + i]);
            }
        if (AHEAD) mix<16>();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const u32x4 kx1 = kx;
    __builtin_amdgcn_sched_barrier(0);
    if (b + WAVES < b1) load_k(b + WAVES);
    else drop(kr);
    __builtin_amdgcn_sched_barrier(0);
    const int left = tokens - b * BT < BT ? tokens - b * BT : BT;  // tokens of this block in range
    // ---- softmax of row c over the lane's 16 tokens and the other g's
    if constexpr (F8) {  // K's scales
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) D[t][i][r] *= __uint_as_float((kx1[i] >> (8 * r) & 0xffu) << 23);
    }
    if (left < BT) {  // the last block: what lies behind the last token may be anything, and 0 times an infinity is NaN
      int k = left - 16 * g;  // this lane's tokens in range
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int t = 0; t < RT; ++t) D[t][i / 4][i % 4] = i < k ? D[t][i / 4][i % 4] : -INFINITY;
#pragma unroll
      for (int w = 0; w < 4 * S1; ++w) {  // words of 4 / S1 tokens
        constexpr int TW = 4 / S1;
        const int n = k - TW * w;
        const uint32_t mask = n >= TW ? 0xffffffffu : n <= 0 ? 0u : (1u << (32 / TW * n)) - 1u;
        if (F8) vx[w % 4] &= mask;
#pragma unroll
        for (int x = 0; x < X; ++x) vr[x * S1 + w / 4][w % 4] &= mask;
      }
    }
    u32x4 pr[RT][2][2];  // [high and low part][step]
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, D[t][i][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
      mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
      const float to2 = F8 ? sc[t] : scale2;
      mx = fmaxf(m[t], mx * to2);
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
          float p0 = __builtin_amdgcn_exp2f(fmaf(D[t][i][r], to2, -m0)), p1 = __builtin_amdgcn_exp2f(fmaf(D[t][i][r + 1], to2, -m0));
          l[t] += p0 + p1;
          if constexpr (F8) {  // V's scales
            p0 *= __uint_as_float((vx[i] >> (8 * r) & 0xffu) << 23);
            p1 *= __uint_as_float((vx[i] >> (8 * r + 8) & 0xffu) << 23);
          }
          pr[t][0][i / 2][2 * (i % 2) + r / 2] = high2(p0, p1);
          pr[t][1][i / 2][2 * (i % 2) + r / 2] = f2bf2(low<F8>(p0), low<F8>(p1));
        }
    }
    // ---- P V
    constexpr int WV = AHEAD ? 2 : 1;  // 16-dim tiles at a time
    u32x4 v[2 * AHEAD + 1][WV];
    auto values = [&](int y, int u) {
#pragma unroll
      for (int x = 0; x < WV; ++x) {
        const int at = WV * y + x;
        v[(2 * y + u) % (2 * AHEAD + 1)][x] = F8 ? widen(vr[at][2 * u], vr[at][2 * u + 1]) : vr[at * S1 + u * (S1 - 1)];
      }
    };
    if (AHEAD) values(0, 0), values(0, 1);
#pragma unroll
    for (int y = 0; y < X / WV; ++y) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (!AHEAD) values(y, u);
        else if (y + 1 < X / WV) values(y + 1, u);
#pragma unroll
        for (int h = 1; h >= 0; --h)
#pragma unroll
          for (int x = 0; x < WV; ++x)
#pragma unroll
            for (int t = 0; t < RT; ++t)
              O[t][WV * y + x] = mma(v[(2 * y + u) % (2 * AHEAD + 1)][x], pr[t][h][u], O[t][WV * y + x]);
      }
      if (AHEAD) mix<16>();
      if (AHEAD || y % 2) __builtin_amdgcn_sched_barrier(0);  // (or every V is widened before the first product)
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
  // partials: G rows of a slot's, or all of a tile's
  const int NR = RT == 1 ? G : R;
  const int64_t p0 = RT == 1 ? ((int64_t)it.part * A.nkv + j) * G
                             : (int64_t)A.own_parts * A.nh + ((int64_t)it.part * A.nkv + j) * R;
  if (wid == 0 && g == 0) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int q = 16 * t + c;
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
        L += M[t] == -INFINITY ? 0.f : sl[w][q] * __builtin_amdgcn_exp2f(sm[w][q] - M[t]);
      if (rown[q] >= 0) *reinterpret_cast<float2*>(wk.ml + (p0 + q) * 2) = float2{M[t], L};
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
    for (int i = tid; i < NR * (DS / 4); i += 64 * WAVES) {
      const int q = i / (DS / 4), d = 4 * (i % (DS / 4));
      f32x4 o = *reinterpret_cast<const f32x4*>(&so[0][q][d]);
#pragma unroll
      for (int w = 1; w < WAVES; ++w) o += *reinterpret_cast<const f32x4*>(&so[w][q][d]);
      if (rown[q] >= 0)
        *reinterpret_cast<f32x4*>(&wk.o[(p0 + q) * HD + d0 + d]) = o;
    }
    __syncthreads();
  }
}

// grid (items): a workgroup per item of the plan.  kPre: there may be prefixes.
template <int HD, bool F8, bool kPre>
__global__ __launch_bounds__(256, !kPre && (HD < 256 || F8) ? 2 : 1) void cached_split_kernel(cached::Args A, cached::Work wk, float scale2) {
  using namespace cached;
  __shared__ alignas(16) char raw[kPre ? sizeof(SplitLds<HD, 2>) : sizeof(SplitLds<HD, 1>)];
  Item it = wk.items[blockIdx.x];
  it.tile = __builtin_amdgcn_readfirstlane(it.tile);
  it.row = __builtin_amdgcn_readfirstlane(it.row);
  it.j = __builtin_amdgcn_readfirstlane(it.j);
  it.b0 = __builtin_amdgcn_readfirstlane(it.b0);
  it.b1 = __builtin_amdgcn_readfirstlane(it.b1);
  it.tokens = __builtin_amdgcn_readfirstlane(it.tokens);
  it.part = __builtin_amdgcn_readfirstlane(it.part);
  if (it.b0 >= it.b1) return;
  if (kPre && it.tile >= 0) split<HD, F8, 2>(A, wk, it, *reinterpret_cast<SplitLds<HD, 2>*>(raw), scale2);
  else split<HD, F8, 1>(A, wk, it, *reinterpret_cast<SplitLds<HD, 1>*>(raw), scale2);
}

// grid (N * nh), 256 threads: HD / 4 lanes of 4 dims times groups of partials; the groups meet in LDS.
template <int HD>
__global__ __launch_bounds__(256) void cached_combine_kernel(cached::Args A, cached::Work wk) {
  using namespace cached;
  constexpr int LN = HD / 4, GR = 256 / LN;
  __shared__ alignas(16) float so[GR][HD];
  __shared__ float sl[GR];
  const int n = blockIdx.x / A.nh, h = blockIdx.x % A.nh, t = threadIdx.x, d4 = t % LN, gr = t / LN;
  const int G = A.nh / A.nkv, j = h / G, g = h % G;
  const SlotPlan s = wk.slots[n];
  const int ns = s.count;
  int np = 0;
  // partial i of this head: own ones G * nkv apart, a tile's 32 * nkv
  int64_t first = 0;
  if (s.tile >= 0) {
    const int q = s.rank * G + g;
    const TilePlan tile = wk.tiles[s.tile + q / PROWS];
    np = tile.count;
    first = (int64_t)A.own_parts * A.nh + ((int64_t)tile.first * A.nkv + j) * PROWS + q % PROWS;
  }
  auto at = [&](int i) {
    return i < ns ? ((int64_t)(s.first + i) * A.nkv + j) * G + g : first + (int64_t)(i - ns) * A.nkv * PROWS;
  };
  const float gate = t < HD ? A.proj(n, (int64_t)h * 2 * HD + HD + t) : 0.f;
  float M = -INFINITY;
  for (int i = t & 63; i < ns + np; i += 64) M = fmaxf(M, wk.ml[2 * at(i)]);
  M = wave_max_fast(M);
  const float m0 = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = gr; i < ns + np; i += GR) {
    const int64_t p = at(i);
    const float2 ml = *reinterpret_cast<const float2*>(wk.ml + 2 * p);
    const float f = __builtin_amdgcn_exp2f(ml.x - m0);
    L += ml.y * f;
    o += *reinterpret_cast<const f32x4*>(wk.o + p * HD + 4 * d4) * f;
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
  const int planners = A.items < 8 * 256 ? (A.items + 255) / 256 : 8;
  cached_prep_kernel<HD, F8><<<(unsigned)((waves + 3) / 4 + planners), 256, 0, st>>>(A, wk, planners);
  if (A.pof) cached_split_kernel<HD, F8, true><<<A.items, 256, 0, st>>>(A, wk, scale2);
  else cached_split_kernel<HD, F8, false><<<A.items, 256, 0, st>>>(A, wk, scale2);
  cached_combine_kernel<HD><<<A.N * A.nh, 256, 0, st>>>(A, wk);
  return check_launch("gdn_attn_cached");
}

}  // namespace gdn

using namespace gdn;

namespace {
bool cached_sizes(int N, int nh, int nkv, int64_t T, int P, int64_t Tp) {
  return N >= 0 && nh >= 1 && nkv >= 1 && nh % nkv == 0 && nkv <= 65535 && N <= cached::MAXN && P >= 0 && T >= kv::BT &&
         T % kv::BT == 0 && T <= INT32_MAX && (P == 0 || (Tp >= kv::BT && Tp % kv::BT == 0 && Tp <= INT32_MAX)) &&
         (int64_t)N * nh <= INT32_MAX / 16 && P <= cached::MAXP;
}
}  // namespace

extern "C" int64_t gdn_attn_cached_workspace_bytes(int N, int nh, int nkv, int hd, int64_t T, int P, int64_t Tp) {
  if (!cached_sizes(N, nh, nkv, T, P, Tp) || hd < 1) return -1;
  cached::Args A{};
  A.N = N, A.nh = nh, A.nkv = nkv, A.P = P;
  cached::bound(A, nh / nkv, T, P ? Tp : 0);
  cached::Work w;
  return cached::work_of(w, nullptr, A, hd);
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
  GDN_REQUIRE(cached_sizes(N, nh, nkv, T, P, Tp), "%s: bad head counts, more than 1024 slots or prefixes, or a cache length that is no positive multiple of 64", name);
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
  A.N = N, A.nh = nh, A.nkv = nkv, A.rd = rd, A.P = P;
  A.eps = eps;
  A.out = static_cast<uint16_t*>(out);
  A.out_stride = out_stride;
  cached::bound(A, nh / nkv, T, P ? Tp : 0);
  cached::Work wk;
  const int64_t need = cached::work_of(wk, static_cast<char*>(work), A, hd);
  GDN_REQUIRE(work_bytes >= need, "%s: workspace too small (%lld bytes needed)", name, (long long)need);
  const hipStream_t st = (hipStream_t)stream;
  switch (hd) {
    case 64: return f8 ? launch_cached<64, true>(A, wk, st) : launch_cached<64, false>(A, wk, st);
    case 128: return f8 ? launch_cached<128, true>(A, wk, st) : launch_cached<128, false>(A, wk, st);
    default: return f8 ? launch_cached<256, true>(A, wk, st) : launch_cached<256, false>(A, wk, st);
  }
}
