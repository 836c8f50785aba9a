// One token per row of logits: temperature, top-k, top-p, min-p and a given random number.
//
// For row l of V logits (a NaN counts as -inf) with maximum M: w_i = exp((l_i - M) / T).  Kept are the top_k largest
// (ties: the lowest index), of these the fewest of the most likely whose mass reaches top_p of the top_k's mass, of these
// those with w >= min_p.  The token is the first index i with sum_{j <= i, kept} w_j > u sum_{kept} w_j.
//
// All of it is a cut in the order of (value, index), found by radix descent on the values' order-preserving keys, 8 bits a
// pass: a pass counts and weighs, per chunk of a row, the elements of each of 256 bins below the digits found so far, and
// the next pass's workgroups each merge their row's chunks and choose the bin (the same numbers in the same order: no
// atomics between workgroups, nothing to clear, the same result every time).  top_k's cut has to be known before top_p's
// target is, so a row with both descends twice.  bf16 has 2 digits, fp16 3 (as fp32 values), fp32 4; a bin of the last
// digit is one value, so that pass only counts.  The last pass also sums each chunk's mass above the bin, and the draw
// resolves the last digit, finds the chunk and walks it.
// Weights are computed in double and summed in 64-bit fixed point within a chunk (2^-50 of the largest), so that sums do
// not depend on an order, and the draw itself is exact integer arithmetic on weights rounded to 2^-sh of the largest.
#include <cmath>

#include "gdn_device.h"
#include "gdn_internal.h"

namespace gdn {
namespace sample {
constexpr int TH = 1024;  // threads
constexpr int BINS = 256; // of a digit
constexpr int COLS = 32;  // a bin's counters in LDS
typedef unsigned long long u64;

struct Params {  // per row (device), or NULL and one value for all
  const float *t, *p, *m;
  const int32_t* k;
  double t1, p1, m1;
  int32_t k1;
};
struct Row {
  double t, p, m;
  int64_t k;
  bool greedy;
};
__device__ __forceinline__ Row row_of(const Params& P, int n) {
  Row r;
  r.t = P.t ? (double)P.t[n] : P.t1;
  r.p = P.p ? (double)P.p[n] : P.p1;
  r.m = P.m ? (double)P.m[n] : P.m1;
  r.k = P.k ? P.k[n] : P.k1;
  r.greedy = !(r.t > 0.0);  // NaN too
  return r;
}
// Where a row's descent stands.
struct State {
  float M;          // the row's maximum
  int kind;         // what is being looked for: 0 nothing, 1 top_k's cut, 2 top_p's
  int level;        // digits found
  uint32_t prefix;  // those digits
  int64_t left;     // top_k: the rank still to find in the bin
  double above;     // mass above the bin
  double target;    // top_p: the mass to reach
  uint32_t thr;     // the cut so far: keys above thr are kept, and the first `quota` elements with key thr
  int64_t quota;    // -1: no cut
};
struct Hist {  // [N][S][BINS]
  uint32_t* count;
  u64* mass;
};
struct Work {
  float* lmax;      // [N][S]: the chunks' maxima and their first indexes
  int32_t* larg;
  State* state;     // [2][N]
  Hist first, step[2];
  int64_t* kept;    // [N][S][TH / 64]: mass above the cut and elements at it, of each wave's elements
  int32_t* ties;
  int64_t* cmass;   // [N][S]: of the chunks
  int32_t* cties;
};
struct Job {
  const void* logits;
  int64_t stride;
  const float* u;
  const double* u64_;
  int64_t* out;
  Params par;
  int N, V, S, levels;
  double one;  // the draw's weights: whole numbers of 1 / one
};

// Order-preserving key of a value: -0 and 0 are equal, NaN is -inf.
__device__ __forceinline__ float cleaned(float f) { return f != f ? -INFINITY : f + 0.f; }
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// The value of a key of which the first `levels` digits are given (the types' remaining bits are 0).
__device__ __forceinline__ float value_of(uint32_t digits, int levels) {
  const int sh = 32 - 8 * levels;
  uint32_t k = sh ? digits << sh : digits;
  if (!(k & 0x80000000u)) k |= sh ? (1u << sh) - 1u : 0u;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// exp((l - M) / T) for l <= M: 2^x with x = (l - M) log2(e) / T (inv2) = n + f, and the Taylor series of e^(f ln 2),
// whose first term left out is below 0.347^12 / 12! = 7e-15.  l = M gives 1 also where both are infinite, and what is
// not a number (-inf times 0) gives 0.
__device__ __forceinline__ double weight(float l, float M, double inv2) {
  const double x = fmax(((double)l - (double)M) * inv2, -1100.0);
  const double n = rint(x), f = (x - n) * 0.69314718055994530942;
  double y = 1.0 / 39916800.0;
  y = fma(y, f, 1.0 / 3628800.0);
  y = fma(y, f, 1.0 / 362880.0);
  y = fma(y, f, 1.0 / 40320.0);
  y = fma(y, f, 1.0 / 5040.0);
  y = fma(y, f, 1.0 / 720.0);
  y = fma(y, f, 1.0 / 120.0);
  y = fma(y, f, 1.0 / 24.0);
  y = fma(y, f, 1.0 / 6.0);
  y = fma(y, f, 0.5);
  y = fma(y, f, 1.0);
  y = fma(y, f, 1.0);
  y = __builtin_amdgcn_ldexp(y, (int)n);
  return l == M ? 1.0 : y;
}
__device__ __forceinline__ double inv2_of(double t) { return 1.4426950408889634074 / t; }
// w * 2^sh as a whole number (sh <= 51): added to 2^52 it lies in the sum's mantissa, rounded to nearest.
__device__ __forceinline__ u64 fixed(double w, double scale) {
  return __builtin_bit_cast(u64, fma(w, scale, 0x1p52)) - 0x4330000000000000ull;
}

template <typename T> __device__ __forceinline__ float as_float(T x);
template <> __device__ __forceinline__ float as_float(float x) { return x; }
template <> __device__ __forceinline__ float as_float(uint16_t x) { return bf2f(x); }
template <> __device__ __forceinline__ float as_float(_Float16 x) { return (float)x; }
template <typename T> __device__ __forceinline__ T lowest();
template <> __device__ __forceinline__ float lowest() { return -INFINITY; }
template <> __device__ __forceinline__ uint16_t lowest() { return 0xff80; }
template <> __device__ __forceinline__ _Float16 lowest() { return (_Float16)-INFINITY; }
// A chunk's elements of this thread, as they are stored: 16 bytes at a time, lane after lane; a wave's are contiguous.  What
// lies past the row's end is -inf.  index(e): element e's place in the chunk.
template <typename T, int EPT> struct Chunk {
  static constexpr int VEC = 16 / sizeof(T);
  alignas(16) T x[EPT];
  __device__ static __forceinline__ int index(int e) {
    return (int)(threadIdx.x >> 6) * 64 * EPT + (e / VEC * 64 + (int)(threadIdx.x & 63)) * VEC + e % VEC;
  }
  __device__ __forceinline__ void load(const T* row, int64_t c0, int V) {
    if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && c0 + TH * EPT <= V) {  // uniform
#pragma unroll
      for (int g = 0; g < EPT / VEC; ++g)
        reinterpret_cast<uint4*>(x)[g] = *reinterpret_cast<const uint4*>(row + c0 + index(g * VEC));
    } else {
#pragma unroll
      for (int e = 0; e < EPT; ++e) x[e] = c0 + index(e) < V ? row[c0 + index(e)] : lowest<T>();
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return cleaned(as_float<T>(x[e])); }
};

struct Scratch {
  int64_t ti[TH / 64];
  // choose: the chunks' bins, merged by 4 groups of threads; then [0]: the sums, and a value's weight
  int64_t count[TH / BINS][BINS];
  double mass[TH / BINS][BINS];
  double scale[BINS];
  int pick;
  int64_t pick_i;
  double pick_d, pick_w, target;
};
// Inclusive sum over the wave's lanes.
template <typename T> __device__ __forceinline__ T wave_scan(T x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o, kWave);
    if ((int)(threadIdx.x & 63) >= o) x += y;
  }
  return x;
}
// Inclusive sum over the workgroup's threads in their order (barriers in front and inside; tmp: a value per wave).
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* tmp, int64_t& total) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  x = wave_scan(x);
  __syncthreads();
  if (lane == 63) tmp[wid] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < TH / 64; ++w) {
    const int64_t t = tmp[w];
    if (w < wid) before += t;
    total += t;
  }
  return x + before;
}
// The row's maximum over its chunks, in every thread.
__device__ __forceinline__ float row_max(const Work& wk, int n, int S) {
  float m = -INFINITY;
  for (int s = threadIdx.x & 63; s < S; s += 64) m = fmaxf(m, wk.lmax[(int64_t)n * S + s]);
  return wave_max_fast(m);
}
// One digit: the row's chunks merged and the bin in which the cut lies; w: the weight of that bin's value (last digit).
// root: the descent's first digit, whose masses are relative to the chunks' own maxima (top_p: of W, its target's base; W <
// 0: the row's whole mass).
__device__ __forceinline__ void choose(State& st, const Hist& h, bool root, const Work& wk, const Row& r, int n, int S,
                                       int levels, Scratch& sc, double W, double& w) {
  const int tid = threadIdx.x, bin = tid % BINS, grp = tid / BINS;
  const double inv2 = inv2_of(r.t);
  const bool values = st.level == levels - 1;  // a bin is one value: its mass is its count times its weight
  const bool weigh = r.p < 1.0;
  int64_t cnt = 0;
  double mass = 0;
  for (int s0 = 0; s0 < S; s0 += BINS) {
    __syncthreads();
    if (tid < BINS) sc.scale[tid] = !root ? 0x1p-50 : s0 + tid < S ? weight(wk.lmax[(int64_t)n * S + s0 + tid], st.M, inv2) * 0x1p-50 : 0.0;
    __syncthreads();
    const int end = S < s0 + BINS ? S : s0 + BINS;
    const int64_t at = (int64_t)n * S * BINS + bin;
#pragma unroll 4
    for (int s = s0 + grp; s < end; s += TH / BINS) {
      cnt += h.count[at + (int64_t)s * BINS];
      if (weigh && !values) mass += (double)h.mass[at + (int64_t)s * BINS] * sc.scale[s - s0];
    }
  }
  sc.count[grp][bin] = cnt;
  sc.mass[grp][bin] = mass;
  __syncthreads();
  if (tid < BINS) {
#pragma unroll
    for (int g = 1; g < TH / BINS; ++g) cnt += sc.count[g][bin], mass += sc.mass[g][bin];
    if (values) {
      const double v = weight(value_of(st.prefix << 8 | (uint32_t)bin, levels), st.M, inv2);
      sc.scale[bin] = v;
      mass = cnt ? (double)cnt * v : 0.0;
    }
    sc.count[0][bin] = cnt;
    sc.mass[0][bin] = mass;
  }
  __syncthreads();
  if (tid < 64) {  // lane l has bins 255 - 4 l .. 252 - 4 l, from the highest
    int64_t c[4], cs[4];
    double m[4], ms[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int b = BINS - 1 - 4 * tid - e;
      c[e] = sc.count[0][b];
      m[e] = sc.mass[0][b];
      cs[e] = c[e] + (e ? cs[e - 1] : 0);
      ms[e] = m[e] + (e ? ms[e - 1] : 0);
    }
    const int64_t cb = wave_scan(cs[3]) - cs[3];
    const double mb = wave_scan(ms[3]) - ms[3];
    const double target = root && st.kind == 2 ? r.p * (W < 0 ? __shfl(mb + ms[3], 63, kWave) : W) : st.target;
    // the first bin that reaches what is looked for; none, by rounding: the last one with any mass
    int hit = 4, last = -1;
#pragma unroll
    for (int e = 3; e >= 0; --e) {
      const bool reached = st.kind == 1 ? cb + cs[e] >= st.left : st.above + (mb + ms[e]) >= target;
      if (c[e] && reached) hit = e;
      if (c[e] && m[e] > 0 && last < 0) last = e;
    }
    const uint64_t hits = __ballot(hit < 4), lasts = __ballot(last >= 0);
    const int lane = hits ? __builtin_ctzll(hits) : lasts ? 63 - __builtin_clzll(lasts) : 63;
    if (tid == lane) {
      const int e = hits ? hit : lasts ? last : 3;
      sc.pick = BINS - 1 - 4 * tid - e;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (x == e) sc.pick_i = cb + cs[x] - c[x], sc.pick_d = mb + (x ? ms[x ? x - 1 : 0] : 0.0);
      sc.pick_w = sc.scale[sc.pick];
      sc.target = target;
    }
  }
  __syncthreads();
  st.left -= sc.pick_i;
  st.above += sc.pick_d;
  st.target = sc.target;
  st.prefix = st.prefix << 8 | (uint32_t)sc.pick;
  ++st.level;
  w = sc.pick_w;
}
// The row's state at the beginning of pass i >= 1 (or of the draw, i = the passes' number), from the state at the beginning
// of pass i - 1 and that pass's histogram.
__device__ __forceinline__ State advance(const Job& J, const Work& wk, const Row& r, int n, int i, Scratch& sc) {
  State st{};
  bool root = i == 1;
  if (root) {
    st.M = row_max(wk, n, J.S);
    st.quota = -1;
    if (!r.greedy && st.M != -INFINITY) st.kind = r.k > 0 && r.k < J.V ? 1 : r.p < 1.0 ? 2 : 0;
    st.left = r.k;
  } else {
    st = wk.state[(int64_t)((i - 1) & 1) * J.N + n];
  }
  if (!st.kind) return st;
  double W = -1.0, w;
  for (;;) {
    choose(st, root ? wk.first : wk.step[(i - 1) & 1], root, wk, r, n, J.S, J.levels, sc, W, w);
    if (st.level < J.levels) return st;
    if (st.kind == 1) {
      st.thr = st.prefix;
      st.quota = st.left;
      st.kind = 0;
      if (!(r.p < 1.0)) return st;
      W = st.above + (double)st.quota * w;
      st.kind = 2;
      st.level = 0;
      st.prefix = 0;
      st.above = 0;
      root = true;
      continue;
    }
    double m = ceil((st.target - st.above) / w);
    if (!(m >= 1.0)) m = 1.0;
    const int64_t q = m < 9e15 ? (int64_t)m : INT64_MAX;
    st.quota = st.quota >= 0 && st.thr == st.prefix && st.quota < q ? st.quota : q;
    st.thr = st.prefix;
    st.kind = 0;
    return st;
  }
}
}  // namespace sample

// Pass i of `passes`, grid (S, N): the histogram of the next digit of the elements whose earlier digits are the prefix (pass
// 0: of all), and in the last pass each wave's mass above the prefix, or above the cut and the elements at it where that is
// known.
//
// A wave's values crowd a few bins, and a counter in LDS takes one lane's addition at a time: each bin has COLS counters,
// lane l adding to the (l % COLS)-th.  (One counter a bin and wave: 30 us for 61 workgroups of 4096 logits.)
template <typename T, int EPT>
__global__ __launch_bounds__(sample::TH) void sample_pass_kernel(sample::Job J, sample::Work wk, int i, int passes, bool hist) {
  using namespace sample;
  __shared__ union {
    Scratch sc;
    struct {
      u64 mass[BINS * COLS];
      uint32_t count[BINS * COLS];
    } h;
  } lds;
  __shared__ float tf[TH / 64];
  __shared__ int first;
  constexpr int CHUNK = TH * EPT;
  const int n = blockIdx.y, s = blockIdx.x, tid = threadIdx.x, wid = tid >> 6;
  const Row r = row_of(J.par, n);
  const int64_t at = (int64_t)n * J.S + s;
  Chunk<T, EPT> c;
  c.load(static_cast<const T*>(J.logits) + n * J.stride, (int64_t)s * CHUNK, J.V);
  State st{};
  float M = -INFINITY;
  if (i == 0) {
    int arg = 0;
#pragma unroll
    for (int e = 0; e < EPT; ++e)
      if (c[e] > M) M = c[e], arg = Chunk<T, EPT>::index(e);  // a thread's indexes ascend
    const float mine = M;
    M = wave_max_fast(M);
    if ((tid & 63) == 0) tf[wid] = M;
    if (tid == 0) first = CHUNK;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TH / 64; ++w) M = fmaxf(M, tf[w]);
    if (mine == M) atomicMin(&first, arg);
    __syncthreads();
    if (tid == 0) {
      wk.lmax[at] = M;
      wk.larg[at] = s * CHUNK + first;
    }
    if (!hist || r.greedy) return;
    if (!(r.k > 0 && r.k < J.V) && !(r.p < 1.0)) return;
  } else {
    st = advance(J, wk, r, n, i, lds.sc);
    if (s == 0 && tid == 0) wk.state[(int64_t)(i & 1) * J.N + n] = st;
    if (r.greedy || st.M == -INFINITY || (!st.kind && i < passes - 1)) return;
    M = st.M;
  }
  const bool last = i && i == passes - 1, count = i == 0 || st.kind;
  const bool weigh = count && r.p < 1.0 && M != -INFINITY && st.level < J.levels - 1;
  if (count) {
    __syncthreads();
    for (int x = tid; x < (int)sizeof(lds.h) / 16; x += TH) reinterpret_cast<uint4*>(&lds.h)[x] = uint4{0, 0, 0, 0};
    __syncthreads();
  }
  // keys are compared up to the digits known: the prefix, or the whole cut (no cut: every key of a number is above 0)
  const double inv2 = inv2_of(r.t);
  const int dsh = 24 - 8 * st.level, sh = count ? dsh + 8 : 32 - 8 * J.levels;
  const uint32_t ref = count ? st.prefix : st.quota >= 0 ? st.thr : 0;
  int64_t mass = 0;
  int ties = 0;
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    const float v = c[e];
    const uint32_t k = key_of(v);
    const uint32_t k1 = sh < 32 ? k >> sh : 0;
    const bool in = k1 == ref, above = last && k1 > ref && v != -INFINITY;
    u64 w = 0;
    if (above || (in && weigh)) {
      const double x = weight(v, M, inv2);
      w = fixed(x, above ? J.one : 0x1p50);
      if (above && (x >= r.m || v == M)) mass += (int64_t)w;
    }
    if (in && count) {
      const int b = (k >> dsh & 255u) * COLS + tid % COLS;
      atomicAdd(&lds.h.count[b], 1u);
      if (weigh) atomicAdd(&lds.h.mass[b], w);
    }
    ties += in;
  }
  if (last) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) mass += __shfl_xor(mass, o, kWave), ties += __shfl_xor(ties, o, kWave);
    if ((tid & 63) == 0) {
      wk.kept[at * (TH / 64) + wid] = mass;
      wk.ties[at * (TH / 64) + wid] = ties;
    }
  }
  if (!count) return;
  __syncthreads();
  // 4 threads a bin; they begin at different counters, so that a wave's reads spread over the banks
  const Hist& h = i == 0 ? wk.first : wk.step[i & 1];
  const int bin = tid / 4;
  uint32_t a = 0;
  u64 m = 0;
#pragma unroll
  for (int x = 0; x < COLS / 4; ++x) {
    const int col = bin * COLS + tid % 4 * (COLS / 4) + (x + bin) % (COLS / 4);
    a += lds.h.count[col];
    if (weigh) m += lds.h.mass[col];
  }
  a += __shfl_xor(a, 1, kWave);
  a += __shfl_xor(a, 2, kWave);
  m += __shfl_xor(m, 1, kWave);
  m += __shfl_xor(m, 2, kWave);
  if (tid % 4 == 0) {
    h.count[at * BINS + bin] = a;
    h.mass[at * BINS + bin] = m;
  }
}

// grid (N): the draw.  Sums of weights are whole numbers here: first over chunks, then over the found chunk's waves, then
// over the found wave's elements.
template <typename T, int EPT>
__global__ __launch_bounds__(sample::TH) void sample_draw_kernel(sample::Job J, sample::Work wk, int passes) {
  using namespace sample;
  __shared__ Scratch sc;
  __shared__ int64_t bin_mass[BINS], wmass[TH / 64], found_before, found_ties;
  __shared__ int found, wties[TH / 64];
  constexpr int NW = TH / 64, CHUNK = TH * EPT;
  const int n = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const Row r = row_of(J.par, n);
  const State was = wk.state[(int64_t)((passes - 1) & 1) * J.N + n];
  const int64_t base = (int64_t)n * J.S;
  if (r.greedy || was.M == -INFINITY) {
    if (tid == 0) found = INT32_MAX;
    __syncthreads();
    for (int s = tid; s < J.S; s += TH)
      if (wk.lmax[base + s] == was.M) atomicMin(&found, wk.larg[base + s]);
    __syncthreads();
    if (tid == 0) J.out[n] = was.M == -INFINITY ? -1 : found;
    return;
  }
  const State st = advance(J, wk, r, n, passes, sc);
  const double inv2 = inv2_of(r.t);
  const int sh = 32 - 8 * J.levels;
  const bool cut = st.quota >= 0, open = was.kind;  // open: the waves' masses lack the bins of the last digit above the cut
  const uint32_t digit = st.thr & 255u;
  const int64_t quota = cut ? st.quota : 0;
  __syncthreads();
  if (tid < BINS) {  // an element's mass by its last digit (0: min_p drops it), at the cut and above it
    const float v = value_of((cut ? st.thr & ~255u : 0u) | (uint32_t)tid, J.levels);
    const double w = weight(v, st.M, inv2);
    bin_mass[tid] = cut && (uint32_t)tid >= digit && v <= st.M && (w >= r.m || v == st.M) ? (int64_t)fixed(w, J.one) : 0;
  }
  __syncthreads();
  const int64_t wt = cut ? bin_mass[digit] : 0;
  const uint32_t* count = wk.step[(passes - 1) & 1].count;
  for (int s = wid; s < J.S; s += NW) {
    int64_t m = lane < NW ? wk.kept[(base + s) * NW + lane] : 0;
    int t = lane < NW && !open ? wk.ties[(base + s) * NW + lane] : 0;
    if (open) {
#pragma unroll
      for (int e = 0; e < BINS / 64; ++e) {
        const uint32_t b = lane + 64 * e, cnt = count[(base + s) * BINS + b];
        if (b > digit) m += bin_mass[b] * (int64_t)cnt;
        if (b == digit) t = (int)cnt;
      }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m += __shfl_xor(m, o, kWave), t += __shfl_xor(t, o, kWave);
    if (lane == 0) {
      wk.cmass[base + s] = m;
      wk.cties[base + s] = cut ? t : 0;
    }
  }
  __syncthreads();
  // chunk after chunk (TH at a time): the mass with the ties that are within the quota; first the sum, then the chunk
  int64_t total = 0, target = 0;
  for (int turn = 0; turn < 2; ++turn) {
    if (turn) {
      double u = J.u64_ ? J.u64_[n] : (double)J.u[n];
      u = u > 0.0 ? u < 1.0 ? u : 0x1.fffffffffffffp-1 : 0.0;
      const u64 U = (u64)(u * 0x1p53);
      target = (int64_t)(__umul64hi((u64)total, U) << 11 | (u64)total * U >> 53);
      if (tid == 0) found = -1;
    }
    int64_t sum = 0, ties = 0;
    for (int s0 = 0; s0 < J.S; s0 += TH) {
      const int s = s0 + tid;
      const int64_t a = s < J.S ? wk.cmass[base + s] : 0, t = s < J.S ? wk.cties[base + s] : 0;
      int64_t tt, mt;
      const int64_t before = block_scan(t, sc.ti, tt) - t + ties;
      const int64_t room = quota - before, in = room <= 0 ? 0 : t < room ? t : room;
      const int64_t m = a + in * wt;
      const int64_t upto = block_scan(m, sc.ti, mt) + sum;
      if (turn && m && upto > target && upto - m <= target) {
        found = s;
        found_before = upto - m;
        found_ties = before;
      }
      sum += mt;
      ties += tt;
    }
    total = sum;
  }
  __syncthreads();
  if (found < 0) return;  // no mass: a row has its maximum at least, so this does not happen
  // ---- the chunk's waves
  const T* row = static_cast<const T*>(J.logits) + n * J.stride;
  const int64_t c0 = (int64_t)found * CHUNK, at = (base + found) * NW + wid;
  int64_t m = 0;
  int t = 0;
  if (open) {
    Chunk<T, EPT> c;
    c.load(row, c0, J.V);
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const uint32_t k = key_of(c[e]) >> sh;
      if (k >> 8 == st.thr >> 8) {
        t += (k & 255u) == digit;
        if ((k & 255u) > digit) m += bin_mass[k & 255u];
      }
    }
  } else if (lane == 0) {
    t = cut ? wk.ties[at] : 0;
  }
  if (lane == 0) m += wk.kept[at];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m += __shfl_xor(m, o, kWave), t += __shfl_xor(t, o, kWave);
  if (lane == 0) wmass[wid] = m, wties[wid] = t;
  __syncthreads();
  int64_t upto = found_before, before = found_ties;
  int w0 = 0;
  for (; w0 < NW; ++w0) {
    const int64_t x = wties[w0], room = quota - before, in = room <= 0 ? 0 : x < room ? x : room;
    const int64_t y = wmass[w0] + in * wt;
    if (upto + y > target) break;
    upto += y;
    before += x;
  }
  // ---- the wave's elements, one a thread
  const int64_t i = c0 + (int64_t)w0 * (64 * EPT) + tid;
  const float v = tid < 64 * EPT && i < J.V ? cleaned(as_float<T>(row[i])) : -INFINITY;
  const uint32_t k = key_of(v) >> sh;
  const bool tie = cut && v != -INFINITY && k == st.thr;
  int64_t tt, mt;
  const int64_t rank = block_scan((int64_t)tie, sc.ti, tt) - tie + before;
  m = 0;
  if (tie) {
    m = rank < quota ? wt : 0;
  } else if (v != -INFINITY && (!cut || k > st.thr)) {
    const double x = weight(v, st.M, inv2);
    if (x >= r.m || v == st.M) m = (int64_t)fixed(x, J.one);
  }
  upto += block_scan(m, sc.ti, mt);
  if (m && upto > target && upto - m <= target) J.out[n] = i;
}

template <typename T, int EPT>
static int launch_sample(sample::Job J, const sample::Work& wk, bool by_k, bool by_p, hipStream_t st) {
  const dim3 g(J.S, J.N);
  const int open = ((int)by_k + (int)by_p) * (J.levels - 1), passes = 1 + (open ? open : 1);
  for (int i = 0; i < passes; ++i) sample_pass_kernel<T, EPT><<<g, sample::TH, 0, st>>>(J, wk, i, passes, by_k || by_p);
  sample_draw_kernel<T, EPT><<<J.N, sample::TH, 0, st>>>(J, wk, passes);
  return check_launch("gdn_sample");
}
}  // namespace gdn

using namespace gdn;

namespace {
// Elements of a row per workgroup: 16 a thread where that gives every CU a workgroup, else 8 (a single row of 248320
// logits has 31 workgroups then).
int sample_chunk(int N, int V) { return (int64_t)N * V >= 256ll * sample::TH * 16 ? sample::TH * 16 : sample::TH * 8; }
int64_t sample_work(sample::Work& w, char* p, int N, int V) {
  char* const base = p;
  const int chunk = sample_chunk(N, V);
  const int64_t S = ((int64_t)V + chunk - 1) / chunk, items = (int64_t)N * S;
  auto take = [&p](int64_t bytes) {
    char* q = p;
    p += (bytes + 255) / 256 * 256;
    return q;
  };
  w.lmax = reinterpret_cast<float*>(take(items * 4));
  w.larg = reinterpret_cast<int32_t*>(take(items * 4));
  w.state = reinterpret_cast<sample::State*>(take(2ll * N * sizeof(sample::State)));
  w.kept = reinterpret_cast<int64_t*>(take(items * (sample::TH / 64) * 8));
  w.ties = reinterpret_cast<int32_t*>(take(items * (sample::TH / 64) * 4));
  w.cmass = reinterpret_cast<int64_t*>(take(items * 8));
  w.cties = reinterpret_cast<int32_t*>(take(items * 4));
  for (sample::Hist* h : {&w.first, &w.step[0], &w.step[1]}) {
    h->mass = reinterpret_cast<sample::u64*>(take(items * sample::BINS * 8));
    h->count = reinterpret_cast<uint32_t*>(take(items * sample::BINS * 4));
  }
  return p - base;
}
}  // namespace

extern "C" int64_t gdn_sample_workspace_bytes(int N, int V) {
  if (N < 0 || N > 65535 || V < 1) return -1;
  sample::Work w;
  return sample_work(w, nullptr, N, V);
}

extern "C" int gdn_sample(const void* logits, int64_t stride, int dtype, const void* u, int u_is_f64, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, double temperature1, int top_k1,
                          double top_p1, double min_p1, int64_t* out, int N, int V, void* work, int64_t work_bytes,
                          void* stream) {
  clear_error();
  const char* name = "gdn_sample";
  GDN_REQUIRE(N >= 0 && N <= 65535 && V >= 1, "%s: bad sizes", name);
  GDN_REQUIRE(dtype == GDN_F32 || dtype == GDN_BF16 || dtype == GDN_F16, "%s: logits must be fp32, bf16 or fp16", name);
  if (N == 0) return GDN_OK;
  GDN_REQUIRE(logits && u && out && work, "%s: null pointer", name);
  GDN_REQUIRE(N == 1 || stride >= V, "%s: row stride too small", name);
  GDN_REQUIRE(aligned(logits, dtype == GDN_F32 ? 4 : 2) && aligned(work, 256) && aligned(out, 8) && aligned(u, u_is_f64 ? 8 : 4),
              "%s: misaligned pointer (the workspace: 256 bytes)", name);
  GDN_REQUIRE(temperature || std::isfinite(temperature1), "%s: the temperature must be finite", name);
  GDN_REQUIRE((top_p || (top_p1 >= 0.0 && top_p1 <= 1.0)) && (min_p || (min_p1 >= 0.0 && min_p1 <= 1.0)),
              "%s: top_p and min_p must be in [0, 1]", name);
  sample::Work wk;
  const int64_t need = sample_work(wk, static_cast<char*>(work), N, V);
  GDN_REQUIRE(work_bytes >= need, "%s: workspace too small (%lld bytes needed)", name, (long long)need);
  sample::Job J{};
  J.logits = logits;
  J.stride = stride;
  J.u = u_is_f64 ? nullptr : static_cast<const float*>(u);
  J.u64_ = u_is_f64 ? static_cast<const double*>(u) : nullptr;
  J.out = out;
  J.par = {temperature, top_p, min_p, top_k, temperature1, top_p1, min_p1, top_k1};
  const int chunk = sample_chunk(N, V);
  J.N = N, J.V = V, J.S = (int)(((int64_t)V + chunk - 1) / chunk);
  J.levels = dtype == GDN_BF16 ? 2 : dtype == GDN_F16 ? 3 : 4;
  J.one = 0x1p50;  // V weights of at most `one` stay below 2^62
  while (J.one > 1.0 && J.one * V > 0x1p62) J.one *= 0.5;
  const bool by_k = top_k || (top_k1 > 0 && top_k1 < V), by_p = top_p || top_p1 < 1.0;
  const hipStream_t st = (hipStream_t)stream;
#define GDN_SAMPLE(T) \
  return chunk == sample::TH * 16 ? launch_sample<T, 16>(J, wk, by_k, by_p, st) : launch_sample<T, 8>(J, wk, by_k, by_p, st)
  switch (dtype) {
    case GDN_F32: GDN_SAMPLE(float);
    case GDN_BF16: GDN_SAMPLE(uint16_t);
    default: GDN_SAMPLE(_Float16);
  }
#undef GDN_SAMPLE
}
