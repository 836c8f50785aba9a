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
// target is, so a row with both descends twice.  bf16 has 2 digits, fp16 3 (as fp32 values), fp32 4.
// Weights are computed in double and summed in 64-bit fixed point within a chunk (2^-50 of the largest), so that sums do
// not depend on an order, and the draw itself is exact integer arithmetic on weights rounded to 2^-sh of the largest.
#include <cmath>

#include "gdn_device.h"
#include "gdn_internal.h"

namespace gdn {
namespace sample {
constexpr int TH = 256;     // threads; also bins of a pass
constexpr int CHUNK = 4096; // elements of a row per workgroup
constexpr int EPT = CHUNK / TH;
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
struct Hist {  // [N][S][256]
  uint32_t* count;
  u64* mass;
};
struct Work {
  float* lmax;      // [N][S]: the chunks' maxima and their first indexes
  int32_t* larg;
  State* state;     // [2][N]
  Hist first, step[2];
  u64* kept;        // [N][S]: mass above the cut
  int32_t* ties;    // [N][S]: elements at it
};
struct Job {
  const void* logits;
  int64_t stride;
  const float* u;
  const double* u64_;
  int64_t* out;
  Params par;
  int N, V, S, levels, sh;
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
// whose first term left out is below 0.347^12 / 12! = 7e-15.
__device__ __forceinline__ double weight(float l, float M, double inv2) {
  if (l == M) return 1.0;
  const double x = ((double)l - (double)M) * inv2;
  if (!(x > -1000.0)) return 0.0;
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
  return ldexp(y, (int)n);
}
__device__ __forceinline__ double inv2_of(double t) { return 1.4426950408889634074 / t; }
__device__ __forceinline__ u64 fixed(double w, int sh) { return (u64)(ldexp(w, sh) + 0.5); }

template <typename T> __device__ __forceinline__ float as_float(T x);
template <> __device__ __forceinline__ float as_float(float x) { return x; }
template <> __device__ __forceinline__ float as_float(uint16_t x) { return bf2f(x); }
template <> __device__ __forceinline__ float as_float(_Float16 x) { return (float)x; }
// A chunk's elements of this thread: 16 bytes at a time, thread after thread; what lies past the row's end is -inf.
// index(e): element e's place in the chunk.
template <typename T> struct Chunk {
  static constexpr int VEC = 16 / sizeof(T);
  float v[EPT];
  __device__ static __forceinline__ int index(int e) { return (e / VEC * TH + (int)threadIdx.x) * VEC + e % VEC; }
  __device__ __forceinline__ void load(const T* row, int64_t c0, int V) {
    const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
#pragma unroll
    for (int g = 0; g < EPT / VEC; ++g) {
      const int64_t i = c0 + index(g * VEC);
      alignas(16) T x[VEC];
      if (vec && i + VEC <= V) {
        *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(row + i);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[g * VEC + e] = cleaned(as_float<T>(x[e]));
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[g * VEC + e] = i + e < V ? cleaned(as_float<T>(row[i + e])) : -INFINITY;
      }
    }
  }
};

// Inclusive sum over the workgroup's threads in their order (a barrier in front and inside; tmp: 4 values).
template <typename T> __device__ __forceinline__ T block_scan(T x, T* tmp, T& total) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o, kWave);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) tmp[wid] = x;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < TH / 64; ++w) {
    if (w < wid) before += tmp[w];
    total += tmp[w];
  }
  return x + before;
}
struct Scratch {
  int64_t ti[4];
  double td[4];
  u64 tu[4];
  float tf[4];
  int pick;
  int64_t pick_i;
  double pick_d;
};
// The row's maximum over its chunks, in every thread.
__device__ __forceinline__ float row_max(const Work& wk, int n, int S, Scratch& sc) {
  float m = -INFINITY;
  for (int s = threadIdx.x; s < S; s += TH) m = fmaxf(m, wk.lmax[(int64_t)n * S + s]);
  m = wave_max_fast(m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sc.tf[threadIdx.x >> 6] = m;
  __syncthreads();
  return fmaxf(fmaxf(sc.tf[0], sc.tf[1]), fmaxf(sc.tf[2], sc.tf[3]));
}
// One digit: the row's chunks merged (thread t: bin 255 - t) and the bin in which the cut lies.  local: the masses are
// relative to the chunks' own maxima (the first pass).  start: the descent's first digit (top_p: of W, its target's base;
// W < 0: the row's whole mass).
__device__ __forceinline__ void choose(State& st, const Hist& h, bool local, const Work& wk, const Row& r, int n, int S,
                                       Scratch& sc, bool start, double W) {
  const int bin = TH - 1 - threadIdx.x;
  const double inv2 = inv2_of(r.t);
  int64_t cnt = 0;
  double mass = 0;
  for (int s = 0; s < S; ++s) {
    const int64_t at = ((int64_t)n * S + s) * TH + bin;
    cnt += h.count[at];
    const double scale = local ? weight(wk.lmax[(int64_t)n * S + s], st.M, inv2) : 1.0;
    mass += (double)h.mass[at] * 0x1p-50 * scale;
  }
  int64_t ctotal;
  double mtotal;
  const int64_t cs = block_scan<int64_t>(cnt, sc.ti, ctotal);
  const double ms = block_scan<double>(mass, sc.td, mtotal);
  if (start && st.kind == 2) st.target = r.p * (W < 0 ? mtotal : W);
  // the first bin (from the highest) that reaches what is looked for; none, by rounding: the last one with any mass
  const bool hit = cnt > 0 && (st.kind == 1 ? cs >= st.left : st.above + ms >= st.target);
  const bool last = cnt > 0 && mass > 0;
  const uint64_t hits = __ballot(hit), lasts = __ballot(last);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    sc.ti[threadIdx.x >> 6] = hits ? (int64_t)threadIdx.x + __builtin_ctzll(hits) : -1;
    sc.td[threadIdx.x >> 6] = lasts ? (double)(threadIdx.x + 63 - __builtin_clzll(lasts)) : -1.0;
  }
  __syncthreads();
  int pick = -1;
#pragma unroll
  for (int w = TH / 64 - 1; w >= 0; --w)
    if (sc.ti[w] >= 0) pick = (int)sc.ti[w];
  if (pick < 0) {
#pragma unroll
    for (int w = 0; w < TH / 64; ++w)
      if (sc.td[w] >= 0) pick = (int)sc.td[w];
  }
  if (pick < 0) pick = TH - 1;
  if ((int)threadIdx.x == pick) {
    sc.pick_i = cs - cnt;
    sc.pick_d = ms - mass;
  }
  __syncthreads();
  st.left -= sc.pick_i;
  st.above += sc.pick_d;
  st.prefix = st.prefix << 8 | (uint32_t)(TH - 1 - pick);
  ++st.level;
}
// The row's state at the beginning of pass i >= 1 (i = passes: behind the last one), from the state at the beginning of
// pass i - 1 and that pass's histogram.
__device__ __forceinline__ State advance(const Job& J, const Work& wk, int n, int i, Scratch& sc) {
  const Row r = row_of(J.par, n);
  State st;
  if (i == 1) {
    st = State{};
    st.M = row_max(wk, n, J.S, sc);
    st.quota = -1;
    if (r.greedy || st.M == -INFINITY) return st;
    st.kind = r.k > 0 && r.k < J.V ? 1 : r.p < 1.0 ? 2 : 0;
    if (!st.kind) return st;
    st.left = r.k;
    choose(st, wk.first, true, wk, r, n, J.S, sc, true, -1.0);
  } else {
    st = wk.state[(int64_t)((i - 1) & 1) * J.N + n];
    if (!st.kind) return st;
    choose(st, wk.step[(i - 1) & 1], false, wk, r, n, J.S, sc, false, 0.0);
  }
  if (st.level < J.levels) return st;
  const double w = weight(value_of(st.prefix, J.levels), st.M, inv2_of(r.t));
  if (st.kind == 1) {
    st.thr = st.prefix;
    st.quota = st.left;
    st.kind = 0;
    if (r.p < 1.0) {
      const double W = st.above + (double)st.quota * w;
      st.kind = 2;
      st.level = 0;
      st.prefix = 0;
      st.above = 0;
      choose(st, wk.first, true, wk, r, n, J.S, sc, true, W);
    }
  } else {
    double m = ceil((st.target - st.above) / w);
    if (!(m >= 1.0)) m = 1.0;
    const int64_t q = m < 9e15 ? (int64_t)m : INT64_MAX;
    st.quota = st.quota >= 0 && st.thr == st.prefix && st.quota < q ? st.quota : q;
    st.thr = st.prefix;
    st.kind = 0;
  }
  return st;
}
}  // namespace sample

// Pass i, grid (S, N): the histogram of digit `level` of the elements whose earlier digits are the prefix (pass 0: all).
template <typename T>
__global__ __launch_bounds__(sample::TH) void sample_pass_kernel(sample::Job J, sample::Work wk, int i, bool hist) {
  using namespace sample;
  __shared__ Scratch sc;
  __shared__ uint32_t cnt[TH / 64][TH];
  __shared__ u64 mass[TH / 64][TH];
  const int n = blockIdx.y, s = blockIdx.x, tid = threadIdx.x, wid = tid >> 6;
  const Row r = row_of(J.par, n);
  Chunk<T> c;
  c.load(static_cast<const T*>(J.logits) + n * J.stride, (int64_t)s * CHUNK, J.V);
  State st{};
  float M = -INFINITY;
  if (i == 0) {
    int at = 0;
#pragma unroll
    for (int e = 0; e < EPT; ++e)
      if (c.v[e] > M) M = c.v[e], at = Chunk<T>::index(e);  // a thread's indexes ascend
    const float mine = M;
    M = wave_max_fast(M);
    if ((tid & 63) == 0) sc.tf[wid] = M;
    __syncthreads();
    M = fmaxf(fmaxf(sc.tf[0], sc.tf[1]), fmaxf(sc.tf[2], sc.tf[3]));
    if (tid == 0) sc.pick = CHUNK;
    __syncthreads();
    if (mine == M) atomicMin(&sc.pick, at);
    __syncthreads();
    if (tid == 0) {
      wk.lmax[(int64_t)n * J.S + s] = M;
      wk.larg[(int64_t)n * J.S + s] = s * CHUNK + sc.pick;
    }
    if (!hist || r.greedy) return;
    if (!(r.k > 0 && r.k < J.V) && !(r.p < 1.0)) return;
  } else {
    st = advance(J, wk, n, i, sc);
    if (s == 0 && tid == 0) wk.state[(int64_t)(i & 1) * J.N + n] = st;
    if (!st.kind) return;
    M = st.M;
  }
#pragma unroll
  for (int w = 0; w < TH / 64; ++w) cnt[w][tid] = 0, mass[w][tid] = 0;
  __syncthreads();
  const double inv2 = inv2_of(r.t);
  const int sh = 24 - 8 * st.level;
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    const uint32_t k = key_of(c.v[e]);
    if (st.level && k >> (sh + 8) != st.prefix) continue;
    const int b = k >> sh & 255u;
    atomicAdd(&cnt[wid][b], 1u);
    const u64 w = M == -INFINITY ? 0 : fixed(weight(c.v[e], M, inv2), 50);
    if (w) atomicAdd(&mass[wid][b], w);
  }
  __syncthreads();
  const Hist& h = i == 0 ? wk.first : wk.step[i & 1];
  const int64_t at = ((int64_t)n * J.S + s) * TH + tid;
  uint32_t a = 0;
  u64 m = 0;
#pragma unroll
  for (int w = 0; w < TH / 64; ++w) a += cnt[w][tid], m += mass[w][tid];
  h.count[at] = a;
  h.mass[at] = m;
}

// Behind the last pass, grid (S, N): the chunks' mass above the cut and elements at it.
template <typename T>
__global__ __launch_bounds__(sample::TH) void sample_kept_kernel(sample::Job J, sample::Work wk, int passes) {
  using namespace sample;
  __shared__ Scratch sc;
  const int n = blockIdx.y, s = blockIdx.x, tid = threadIdx.x;
  const Row r = row_of(J.par, n);
  Chunk<T> c;
  c.load(static_cast<const T*>(J.logits) + n * J.stride, (int64_t)s * CHUNK, J.V);
  const State st = advance(J, wk, n, passes, sc);
  if (s == 0 && tid == 0) wk.state[(int64_t)(passes & 1) * J.N + n] = st;
  if (r.greedy || st.M == -INFINITY) return;
  const double inv2 = inv2_of(r.t);
  const int sh = 32 - 8 * J.levels;
  u64 mass = 0;
  int64_t ties = 0;
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    if (c.v[e] == -INFINITY) continue;
    const uint32_t k = key_of(c.v[e]) >> sh;
    if (st.quota >= 0 && k < st.thr) continue;
    const double w = weight(c.v[e], st.M, inv2);
    if (!(w >= r.m) && c.v[e] != st.M) continue;
    if (st.quota >= 0 && k == st.thr) ++ties;
    else mass += fixed(w, J.sh);
  }
  u64 mt;
  int64_t tt;
  block_scan<u64>(mass, sc.tu, mt);
  block_scan<int64_t>(ties, sc.ti, tt);
  if (tid == 0) {
    wk.kept[(int64_t)n * J.S + s] = mt;
    wk.ties[(int64_t)n * J.S + s] = (int32_t)tt;
  }
}

// grid (N): the draw.  Everything here is integer.
template <typename T>
__global__ __launch_bounds__(sample::TH) void sample_draw_kernel(sample::Job J, sample::Work wk, int passes) {
  using namespace sample;
  __shared__ Scratch sc;
  __shared__ u64 found_before;
  __shared__ int found;
  __shared__ int64_t found_ties;
  const int n = blockIdx.x, tid = threadIdx.x;
  const Row r = row_of(J.par, n);
  const State st = wk.state[(int64_t)(passes & 1) * J.N + n];
  const float* lmax = wk.lmax + (int64_t)n * J.S;
  if (r.greedy || st.M == -INFINITY) {
    if (tid == 0) found = INT32_MAX;
    __syncthreads();
    for (int s = tid; s < J.S; s += TH)
      if (lmax[s] == st.M) atomicMin(&found, wk.larg[(int64_t)n * J.S + s]);
    __syncthreads();
    if (tid == 0) J.out[n] = st.M == -INFINITY ? -1 : found;
    return;
  }
  const double inv2 = inv2_of(r.t);
  const int sh = 32 - 8 * J.levels;
  const u64 wt = st.quota >= 0 ? fixed(weight(value_of(st.thr, J.levels), st.M, inv2), J.sh) : 0;
  const int64_t quota = st.quota >= 0 ? st.quota : 0;
  // chunk after chunk (TH at a time): mass with the ties that are within the quota
  u64 total = 0;
  for (int turn = 0; turn < 2; ++turn) {
    u64 target = 0;
    if (turn) {
      double u = J.u64_ ? J.u64_[n] : (double)J.u[n];
      u = u > 0.0 ? u < 1.0 ? u : 0x1.fffffffffffffp-1 : 0.0;
      const u64 U = (u64)(u * 0x1p53);
      target = __umul64hi(total, U) << 11 | total * U >> 53;
      if (tid == 0) found = -1;
    }
    u64 sum = 0;
    int64_t ties = 0;
    for (int s0 = 0; s0 < J.S; s0 += TH) {
      const int s = s0 + tid;
      const u64 a = s < J.S ? wk.kept[(int64_t)n * J.S + s] : 0;
      const int64_t t = s < J.S ? wk.ties[(int64_t)n * J.S + s] : 0;
      int64_t tt;
      const int64_t before = block_scan<int64_t>(t, sc.ti, tt) - t + ties;
      const int64_t room = quota - before, in = room <= 0 ? 0 : t < room ? t : room;
      const u64 m = a + (u64)in * wt;
      u64 mt;
      const u64 upto = block_scan<u64>(m, sc.tu, mt) + sum;
      if (turn && m && upto > target && upto - m <= target) {
        found = s;
        found_before = upto - m;
        found_ties = before;
      }
      sum += mt;
      ties += tt;
    }
    total = sum;
    if (turn) {
      __syncthreads();
      if (found < 0) return;  // no mass: a row has its maximum at least, so this does not happen
      // ---- inside the chunk: a thread takes EPT elements in their order
      const T* row = static_cast<const T*>(J.logits) + n * J.stride;
      const int64_t i0 = (int64_t)found * CHUNK + tid * EPT;
      u64 w[EPT];
      int64_t t = 0;
      u64 m = 0;
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        const float v = i0 + e < J.V ? cleaned(as_float<T>(row[i0 + e])) : -INFINITY;
        const uint32_t k = key_of(v) >> sh;
        const double x = weight(v, st.M, inv2);
        const bool out = v == -INFINITY || (st.quota >= 0 && k < st.thr) || (!(x >= r.m) && v != st.M);
        const bool tie = !out && st.quota >= 0 && k == st.thr;
        w[e] = tie ? ~0ull : out ? 0 : fixed(x, J.sh);
        t += tie;
      }
      int64_t tt;
      int64_t rank = block_scan<int64_t>(t, sc.ti, tt) - t + found_ties;
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        if (w[e] == ~0ull) w[e] = rank++ < quota ? wt : 0;
        m += w[e];
      }
      u64 mt;
      u64 upto = block_scan<u64>(m, sc.tu, mt) + found_before - m;
      if (upto <= target && upto + m > target) {
        for (int e = 0; e < EPT; ++e) {
          upto += w[e];
          if (upto > target) {
            J.out[n] = i0 + e;
            break;
          }
        }
      }
    }
  }
}

template <typename T>
static int launch_sample(const sample::Job& J, const sample::Work& wk, bool by_k, bool by_p, hipStream_t st) {
  const dim3 g(J.S, J.N);
  const int passes = 1 + ((int)by_k + (int)by_p) * (J.levels - 1);
  for (int i = 0; i < passes; ++i) sample_pass_kernel<T><<<g, sample::TH, 0, st>>>(J, wk, i, by_k || by_p);
  sample_kept_kernel<T><<<g, sample::TH, 0, st>>>(J, wk, passes);
  sample_draw_kernel<T><<<J.N, sample::TH, 0, st>>>(J, wk, passes);
  return check_launch("gdn_sample");
}
}  // namespace gdn

using namespace gdn;

namespace {
int64_t sample_work(sample::Work& w, char* p, int N, int V) {
  char* const base = p;
  const int64_t S = (V + sample::CHUNK - 1) / sample::CHUNK, items = (int64_t)N * S;
  auto take = [&p](int64_t bytes) {
    char* q = p;
    p += (bytes + 255) / 256 * 256;
    return q;
  };
  w.lmax = reinterpret_cast<float*>(take(items * 4));
  w.larg = reinterpret_cast<int32_t*>(take(items * 4));
  w.state = reinterpret_cast<sample::State*>(take(2ll * N * sizeof(sample::State)));
  w.kept = reinterpret_cast<sample::u64*>(take(items * 8));
  w.ties = reinterpret_cast<int32_t*>(take(items * 4));
  for (sample::Hist* h : {&w.first, &w.step[0], &w.step[1]}) {
    h->mass = reinterpret_cast<sample::u64*>(take(items * sample::TH * 8));
    h->count = reinterpret_cast<uint32_t*>(take(items * sample::TH * 4));
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
  J.N = N, J.V = V, J.S = (V + sample::CHUNK - 1) / sample::CHUNK;
  J.levels = dtype == GDN_BF16 ? 2 : dtype == GDN_F16 ? 3 : 4;
  J.sh = 62;  // V weights of at most 2^sh stay below 2^63
  while (J.sh > 0 && ((int64_t)V >> (62 - J.sh)) > 0) --J.sh;
  const bool by_k = top_k || (top_k1 > 0 && top_k1 < V), by_p = top_p || top_p1 < 1.0;
  const hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case GDN_F32: return launch_sample<float>(J, wk, by_k, by_p, st);
    case GDN_BF16: return launch_sample<uint16_t>(J, wk, by_k, by_p, st);
    default: return launch_sample<_Float16>(J, wk, by_k, by_p, st);
  }
}
