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
// Weights (within 4e-10 of their value: 2^n times a double from a table times a series in fp32) are summed in 64-bit fixed
// point within a workgroup, so that sums do not depend on an order: in units of 2^-50 of the largest, behind the first pass
// of that times its turns (rounded up to a power of two), so that the 65536 weights of 1 of 8 turns are 2^63.  The draw
// itself is exact integer arithmetic on weights rounded to 2^-50 of the largest (fewer bits from 4097 logits a row on, so
// that a row's sum stays below 2^62).
//
// Measured (all filters on; the launches' medians in us: first pass, passes, last pass, draw):
//    1 x 248320 bf16: 6.5, 8.7, 13.5, 7.5      16 x 248320 bf16: 10.3, 10.2, 15.8, 13.4
//   64 x 151936 fp32: 16.0, 22.3, 16.5, 15.1, 9.8, 5.9, 18.0, 10.2 (39 MB: a read of it at 6.07 TB/s is 6.4)
// A pass over few rows is a chain of latencies: the histograms' merge and the choice of a bin (3 to 4), the row's load, the
// LDS counters.  Over many rows the vector instructions bind: 50 to 75 an element, 20 of them its weight.
#include "gdn_device.h"
#include "gdn_internal.h"

namespace gdn {
namespace sample {
constexpr int TH = 512;           // threads of a pass
constexpr int EPT = 16;           // a thread's elements
constexpr int CHUNK = TH * EPT;   // a row's elements per workgroup and turn
constexpr int NW = TH / 64, WAVE = 64 * EPT;  // its waves, and their elements
constexpr int BINS = 256;         // of a digit
constexpr int COLS = 16;          // a bin's counters in LDS
constexpr int DT = 512;           // threads of the draw
constexpr int MOST = 1024 * CHUNK;  // logits of a row (the draw keeps its workgroups' sums in LDS)
constexpr int TURNS = 8;          // at most
typedef unsigned long long u64;

struct Params {  // per row (device; fp32, or fp64 where `f64` has the bit), or NULL and one value for all
  const void *t, *p, *m;
  int f64;
  const int32_t* k;
  double t1, p1, m1;
  int32_t k1;
};
struct Row {
  double t, p, m;
  int32_t k;
  bool greedy, by_k, by_p;
};
__device__ __forceinline__ double param(const void* x, bool f64, int n) {
  return f64 ? static_cast<const double*>(x)[n] : (double)static_cast<const float*>(x)[n];
}
__device__ __forceinline__ Row row_of(const Params& P, int n, int V) {
  Row r;
  r.t = P.t ? param(P.t, P.f64 & GDN_SAMPLE_F64_TEMPERATURE, n) : P.t1;
  r.p = P.p ? param(P.p, P.f64 & GDN_SAMPLE_F64_TOP_P, n) : P.p1;
  r.m = P.m ? param(P.m, P.f64 & GDN_SAMPLE_F64_MIN_P, n) : P.m1;
  r.k = P.k ? P.k[n] : P.k1;
  r.greedy = !(r.t > 0.0);  // NaN too
  // at 1e-60 two different fp32 values (2^-149 apart at least) are 1e15 in the exponent apart: nothing below it differs, and
  // 1 / T times a logit stays a double
  if (!r.greedy && r.t < 1e-60) r.t = 1e-60;
  if (r.p <= 0.0) r.p = 1e-300;  // the largest alone
  r.by_k = r.k > 0 && r.k < V;
  r.by_p = r.p < 1.0;
  return r;
}
// Where a row's descent stands.
struct State {
  float M;          // the row's maximum
  int kind;         // what is being looked for: 0 nothing, 1 top_k's cut, 2 top_p's
  int level;        // digits found
  uint32_t prefix;  // those digits
  double above;     // mass above the bin
  double target;    // top_p: the mass to reach
  int32_t left;     // top_k: the rank still to find in the bin
  int32_t quota;    // -1: no cut
  int k_level;      // top_p's descent, behind top_k's, which found so many digits (0: there was none)
  uint32_t k_path;  // ... these
  int cut_level;    // the cut's digits: all of them, or as many as set a bin apart that is kept whole
  uint32_t thr;     // the cut so far: keys above thr are kept, and the first `quota` elements with key thr
};
struct Hist {  // [N][S][BINS], of the first pass [N][S0][BINS]
  uint32_t* count;
  u64* mass;
};
struct Work {
  float* lmax;      // [N][S0]: the chunks' maxima and their first indexes
  int32_t* larg;
  State* state;     // [2][N]
  Hist step[7];     // pass i's
  int64_t* kept;    // [N][S0 or more][NW]: mass above the cut and elements at it, of each wave's elements
  int32_t* ties;
};
struct Job {
  const void* logits;
  int64_t stride;
  const float* u;
  const double* u64_;
  int64_t* out;
  Params par;
  // a row's chunks; turns of a workgroup in the passes behind the first, and workgroups a row has in them
  int N, V, S0, turns, S, levels;
  double one;  // the draw's weights: whole numbers of 1 / one
  double unit, per;  // the masses of the passes behind the first: whole numbers of per = 1 / unit
};

// The first element of workgroup s's turn, in the passes behind the first.
__device__ __forceinline__ int64_t at_turn(const Job& J, int s, int turn) { return ((int64_t)s * J.turns + turn) * CHUNK; }

// Order-preserving key of a value: -0 and 0 are equal, NaN is -inf.
__device__ __forceinline__ float cleaned(float f) { return fmaxf(f, -INFINITY) + 0.f; }
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// The value of a key of which the first `levels` digits are given (the types' remaining bits are 0).
__device__ __forceinline__ float value_of(uint32_t digits, int levels) {
  const int sh = 32 - 8 * levels;
  uint32_t k = digits << sh;
  if (!(k & 0x80000000u)) k |= (1u << sh) - 1u;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 2^(j / 64)
__device__ const double kPow[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0
};
// Weights exp((l - M) / T), l <= M, of a row: 2^(y / 64) with y = (l - M) 64 log2(e) / T = 64 n + j + f, |f| <= 1/2, as
// 2^n, a table of 2^(j / 64) and the Taylor series of 2^(f / 64) - 1 (below 0.0055) in fp32: within 4e-10, in 20
// instructions (a Taylor series of 2^f in double: 45).
struct Weights {
  double a, c;
  float M;
  const double* table;  // kPow in LDS
  __device__ __forceinline__ Weights(double t, float M_, const double* table_) : M(M_), table(table_) {
    a = 92.332482616893656877 / t;  // 64 log2(e) / T
    c = -(double)M * a;
  }
  __device__ __forceinline__ double operator()(float l) const {
    const double y = fmax(fma((double)l, a, c), -70400.0);  // (NaN, -inf times 0: the lowest)
    const double t = y + 0x1.8p52;  // the nearest whole number, in the low bits
    const int j = (int)(uint32_t)__builtin_bit_cast(u64, t);
    const float z = (float)(y - (t - 0x1.8p52)) * 0.010830424696249145f;
    const float q = z * fmaf(z, fmaf(z, fmaf(z, 1.f / 24, 1.f / 6), 0.5f), 1.f);
    const double b = table[j & 63];
    const double w = __builtin_amdgcn_ldexp(fma(b, (double)q, b), j >> 6);
    return l == M ? 1.0 : w;  // exactly, as equal logits share a mass; where both are infinite too
  }
};
// w * scale (at most 2^50) as a whole number: added to 2^52 it lies in the sum's mantissa, rounded to nearest.
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
// E elements of a wave's E * 64 contiguous ones from i0 on, as they are stored: 16 bytes at a time, lane after lane.  What
// lies past the row's end is -inf.  index(e): element e's place behind i0.
template <typename T, int E> struct Chunk {
  static constexpr int VEC = 16 / sizeof(T);
  alignas(16) T x[E];
  __device__ static __forceinline__ int index(int e) { return (e / VEC * 64 + (int)(threadIdx.x & 63)) * VEC + e % VEC; }
  __device__ __forceinline__ void load(const T* row, int64_t i0, int V) {
    if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && i0 + 64 * E <= V) {  // uniform
#pragma unroll
      for (int g = 0; g < E / VEC; ++g)
        reinterpret_cast<uint4*>(x)[g] = *reinterpret_cast<const uint4*>(row + i0 + index(g * VEC));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = i0 + index(e) < V ? row[i0 + index(e)] : lowest<T>();
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return cleaned(as_float<T>(x[e])); }
};

// A workgroup's scratch for choosing bins (W waves).
template <int W> struct Scratch {
  uint32_t count[W][BINS];  // each wave's share of the chunks
  double mass[W][BINS];
  State st;
  double w;            // of the chosen bin: its value's weight (last digit), its mass, its elements
  double bin_mass;
  uint32_t bin_count;
};
// One digit: the row's chunks merged, and by the first wave the bin in which the cut lies (sc.st).  root: the descent's
// first digit, whose masses are relative to the chunks' own maxima (first: the weights of the first 64 of these, a lane
// each), with top_p's target p times `base` (below 0: times the row's whole mass); the other digits' masses are whole
// numbers of `per`.  Before anything but the first descent's root the caller has a barrier.
template <int W>
__device__ __forceinline__ void choose(const Hist& h, bool root, const Work& wk, const Row& r, const Weights& wt, int n, int S,
                                       int levels, Scratch<W>& sc, double first, double per, double base, double& w) {
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), bin = 4 * (63 - lane);  // this lane's 4 bins
  const int level = root ? 0 : sc.st.level;
  const bool values = level == levels - 1;  // a bin is one value: its mass is its count times its weight
  const bool weigh = r.by_p && !values;
  uint32_t c[4] = {0, 0, 0, 0};
  double m[4] = {0, 0, 0, 0};
  const uint32_t* hc = h.count + (int64_t)n * S * BINS + bin;
  const u64* hm = h.mass + (int64_t)n * S * BINS + bin;
  if (weigh) {
    constexpr int U = 2;  // chunks at a time, their loads ahead of their sums
    for (int s0 = wid; s0 < S; s0 += U * W) {
      uint4 c1[U];
      ulonglong2 m0[U], m1[U];
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int64_t s = s0 + x * W < S ? s0 + x * W : s0;
        c1[x] = *reinterpret_cast<const uint4*>(hc + s * BINS);
        m0[x] = *reinterpret_cast<const ulonglong2*>(hm + s * BINS);
        m1[x] = *reinterpret_cast<const ulonglong2*>(hm + s * BINS + 2);
      }
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int s = s0 + x * W;
        if (s >= S) break;
        const double f = !root ? per : (s < 64 ? of_lane(first, s) : wt(wk.lmax[(int64_t)n * S + s])) * 0x1p-50;
        c[0] += c1[x].x, c[1] += c1[x].y, c[2] += c1[x].z, c[3] += c1[x].w;
        m[0] = fma((double)m0[x].x, f, m[0]), m[1] = fma((double)m0[x].y, f, m[1]);
        m[2] = fma((double)m1[x].x, f, m[2]), m[3] = fma((double)m1[x].y, f, m[3]);
      }
    }
  } else {
#pragma unroll 4
    for (int s = wid; s < S; s += W) {
      const uint4 c1 = *reinterpret_cast<const uint4*>(hc + (int64_t)s * BINS);
      c[0] += c1.x, c[1] += c1.y, c[2] += c1.z, c[3] += c1.w;
    }
  }
  *reinterpret_cast<uint4*>(&sc.count[wid][bin]) = uint4{c[0], c[1], c[2], c[3]};
  *reinterpret_cast<double2*>(&sc.mass[wid][bin]) = double2{m[0], m[1]};
  *reinterpret_cast<double2*>(&sc.mass[wid][bin + 2]) = double2{m[2], m[3]};
  __syncthreads();
  if (wid == 0) {
    State st = sc.st;
#pragma unroll
    for (int g = 1; g < W; ++g) {
      const uint4 c1 = *reinterpret_cast<const uint4*>(&sc.count[g][bin]);
      c[0] += c1.x, c[1] += c1.y, c[2] += c1.z, c[3] += c1.w;
      if (weigh) {
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] += sc.mass[g][bin + e];
      }
    }
    double v[4] = {0, 0, 0, 0};
    if (values) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = wt(value_of(st.prefix << 8 | (uint32_t)(bin + e), levels));
        m[e] = c[e] ? (double)c[e] * v[e] : 0.0;
      }
    }
    // running sums from the highest bin; cs[e], ms[e]: of the bins above this lane's e-th
    uint32_t cs[4];
    double ms[4];
    cs[3] = 0, ms[3] = 0;
#pragma unroll
    for (int e = 2; e >= 0; --e) cs[e] = cs[e + 1] + c[e + 1], ms[e] = ms[e + 1] + m[e + 1];
    const uint32_t csum = cs[0] + c[0];
    const double msum = ms[0] + m[0], mscan = scan_up(msum);
    const uint32_t cb = scan_up(csum) - csum;
    double mb = __shfl_up(mscan, 1, kWave);
    if (lane == 0) mb = 0;
    const double total = last_lane(mscan);
    if (root && st.kind == 2) st.target = r.p * (base < 0 ? total : base);
    // the highest bin that reaches what is looked for
    int hit = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cs[e] += cb, ms[e] += mb;
      const bool reached = st.kind == 1 ? (int)(cs[e] + c[e]) >= st.left : st.above + (ms[e] + m[e]) >= st.target;
      if (reached && (c[e] || m[e] > 0)) hit = e;
    }
    uint64_t hits = __ballot(hit >= 0);
    if (!hits) {  // none, by rounding: the lowest bin with any mass, or else with anything
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (m[e] > 0) hit = e;
      hits = __ballot(hit >= 0);
      if (!hits) {
#pragma unroll
        for (int e = 3; e >= 0; --e)
          if (c[e]) hit = e;
        hits = __ballot(hit >= 0);
      }
      if (hits) hits = 1ull << (63 - __builtin_clzll(hits));
    }
    if (hits && lane == __builtin_ctzll(hits)) {
      st.left -= (int)(hit == 0 ? cs[0] : hit == 1 ? cs[1] : hit == 2 ? cs[2] : cs[3]);
      st.above += hit == 0 ? ms[0] : hit == 1 ? ms[1] : hit == 2 ? ms[2] : ms[3];
      st.prefix = st.prefix << 8 | (uint32_t)(bin + hit);
      ++st.level;
      sc.st = st;
      sc.bin_mass = hit == 0 ? m[0] : hit == 1 ? m[1] : hit == 2 ? m[2] : m[3];
      sc.bin_count = hit == 0 ? c[0] : hit == 1 ? c[1] : hit == 2 ? c[2] : c[3];
      sc.w = hit == 0 ? v[0] : hit == 1 ? v[1] : hit == 2 ? v[2] : v[3];
    }
  }
  __syncthreads();
  w = sc.w;
}
// The row's state (sc.st) at the beginning of pass i >= 1 (or of the draw, i = the passes' number), from the state at the
// beginning of pass i - 1 and that pass's histogram.  top_k's descent has had the passes 0 .. levels - 1 in turn; top_p's,
// which follows it, takes the same histograms as long as its digits are the same.  Barriers in it; one at its end.
template <int W>
__device__ __forceinline__ void advance(const Job& J, const Work& wk, const Row& r, int n, int i, const double* table,
                                        Scratch<W>& sc) {
  const int lane = threadIdx.x & 63;
  const float mine = lane < J.S0 ? wk.lmax[(int64_t)n * J.S0 + lane] : -INFINITY;
  float M;
  if (i > 1) {
    // (a word a lane)
    const uint32_t* from = reinterpret_cast<const uint32_t*>(wk.state + (int64_t)((i - 1) & 1) * J.N + n);
    if (threadIdx.x < sizeof(State) / 4) reinterpret_cast<uint32_t*>(&sc.st)[threadIdx.x] = from[threadIdx.x];
    __syncthreads();
    if (!sc.st.kind) return;
    M = sc.st.M;
  } else {  // every wave by itself: the histograms' loads need not wait for a barrier
    M = mine;
    for (int s = 64 + lane; s < J.S0; s += 64) M = fmaxf(M, wk.lmax[(int64_t)n * J.S0 + s]);
    M = wave_max_fast(M);
    const int kind = r.greedy || M == -INFINITY ? 0 : r.by_k ? 1 : r.by_p ? 2 : 0;
    if (threadIdx.x == 0) {
      sc.st.M = M;
      sc.st.kind = kind;
      sc.st.level = 0;
      sc.st.prefix = 0;
      sc.st.above = 0;
      sc.st.target = 0;
      sc.st.left = r.k;
      sc.st.quota = -1;
      sc.st.k_level = 0;
      sc.st.k_path = 0;
      sc.st.cut_level = J.levels;
      sc.st.thr = 0;
    }
    if (!kind) {
      __syncthreads();
      return;
    }
  }
  const Weights wt(r.t, M, table);
  double base = -1.0, w;
  for (int h = i - 1;;) {
    choose(wk.step[h], h == 0, wk, r, wt, n, h ? J.S : J.S0, J.levels, sc, h ? 0.0 : wt(mine), J.per, base, w);
    State st = sc.st;
    const bool full = st.level == J.levels;
    // below top_k's cut (its whole mass, summed in another order, was a unit in the last place short of the target): all that
    // top_k left is kept, and its cut stands
    const bool beyond = st.kind == 2 && st.level <= st.k_level && st.prefix < st.k_path >> 8 * (st.k_level - st.level);
    // a bin that is kept whole (all of it is wanted, or its only element) needs no further digits: the cut lies below it
    const bool whole = !full && st.prefix && (st.kind == 1 ? st.left == (int)sc.bin_count : h > 0 && sc.bin_count == 1);
    if (!full && !whole && !beyond) {
      if (st.level >= st.k_level || st.k_path >> 8 * (st.k_level - st.level) != st.prefix) return;
      h = st.level;  // top_p's descent along top_k's
      continue;
    }
    if (st.kind == 1) {
      st.k_level = st.level;
      st.k_path = st.prefix;
      base = whole ? st.above + sc.bin_mass : st.above + (double)st.left * w;
    }
    if (beyond) {
      st.level = st.cut_level;
    } else if (whole) {
      st.thr = st.prefix - 1;
      st.quota = 0;
    } else if (st.kind == 1) {
      st.thr = st.prefix;
      st.quota = st.left;
    } else {
      const double m = ceil((st.target - st.above) / w);
      const int32_t q = m >= 1.0 ? m < 2e9 ? (int32_t)m : INT32_MAX : 1;
      const bool same = st.quota >= 0 && st.cut_level == J.levels && st.thr == st.prefix;  // as top_k's cut
      st.quota = same && st.quota < q ? st.quota : q;
      st.thr = st.prefix;
    }
    st.cut_level = st.level;
    st.kind = st.kind == 1 && r.by_p ? 2 : 0;
    if (st.kind) {
      st.level = 0;
      st.prefix = 0;
      st.above = 0;
      h = 0;
    }
    __syncthreads();
    if (threadIdx.x == 0) sc.st = st;
    __syncthreads();
    if (!st.kind) return;
  }
}
}  // namespace sample

// Elements into a histogram, in LDS.  A wave's values crowd a few bins, and a counter takes one lane's addition at a time:
// each bin has COLS counters, lane l adding to the (l % COLS)-th.  (One counter a bin and wave: 30 us for 61 workgroups of
// 4096 logits.)
namespace sample {
struct Counters {
  u64 mass[BINS * COLS];
  uint32_t count[BINS * COLS];
  __device__ __forceinline__ void clear() {  // (and a barrier)
    for (int x = threadIdx.x; x < (int)sizeof(Counters) / 16; x += TH) reinterpret_cast<uint4*>(this)[x] = uint4{0, 0, 0, 0};
  }
  // TH / BINS threads a bin; they begin at different counters, so that a wave's reads spread over the banks
  __device__ __forceinline__ void write(const Hist& h, int64_t at, bool weigh) const {
    constexpr int PER = TH / BINS;
    const int tid = threadIdx.x, bin = tid / PER;
    uint32_t a = 0;
    u64 m = 0;
#pragma unroll
    for (int x = 0; x < COLS / PER; ++x) {
      const int col = bin * COLS + tid % PER * (COLS / PER) + (x + bin) % (COLS / PER);
      a += count[col];
      if (weigh) m += mass[col];
    }
#pragma unroll
    for (int o = 1; o < PER; o <<= 1) a += __shfl_xor(a, o, kWave), m += __shfl_xor(m, o, kWave);
    if (tid % PER == 0) {
      h.count[at * BINS + bin] = a;
      h.mass[at * BINS + bin] = m;
    }
  }
};
}  // namespace sample

// Pass 0, grid (S0, N): the chunks' maxima, and the histogram of the first digit.
template <typename T>
__global__ __launch_bounds__(sample::TH, 4) void sample_first_kernel(sample::Job J, sample::Work wk) {
  using namespace sample;
  __shared__ Counters lds;
  __shared__ double table[64];
  __shared__ float tf[NW];
  __shared__ int first;
  const int n = blockIdx.y, s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int64_t at = (int64_t)n * J.S0 + s;
  Chunk<T, EPT> c;
  c.load(static_cast<const T*>(J.logits) + n * J.stride, (int64_t)s * CHUNK + wid * WAVE, J.V);
  const Row r = row_of(J.par, n, J.V);
  const bool count = !r.greedy && (r.by_k || r.by_p);
  if (tid < 64) table[tid] = kPow[tid];
  if (tid == 0) first = CHUNK;
  if (count) lds.clear();
  float M = -INFINITY;
  int arg = 0;
#pragma unroll
  for (int e = 0; e < EPT; ++e)
    if (c[e] > M) M = c[e], arg = wid * WAVE + Chunk<T, EPT>::index(e);  // a thread's indexes ascend
  const float mine = M;
  M = wave_max_fast(M);
  if (lane == 0) tf[wid] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) M = fmaxf(M, tf[w]);
  if (mine == M) atomicMin(&first, arg);
  if (count) {
    const Weights wt(r.t, M, table);
    const bool weigh = r.by_p && M != -INFINITY;
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const float v = c[e];
      const int b = (key_of(v) >> 24) * COLS + tid % COLS;
      if (r.by_k) atomicAdd(&lds.count[b], 1u);  // (top_p's first digit goes by mass alone)
      if (weigh) atomicAdd(&lds.mass[b], fixed(wt(v), 0x1p50));
    }
  }
  __syncthreads();
  if (tid == 0) {
    wk.lmax[at] = M;
    wk.larg[at] = s * CHUNK + first;
  }
  if (count) lds.write(wk.step[0], at, r.by_p);
}

// Pass i >= 1, grid (S, N): the histogram of the next digit of the elements whose earlier digits are the prefix, and in the
// last pass (kLast) each wave's mass above the prefix, or above the cut and the elements at it where that is known.
template <typename T, bool kLast>
__global__ __launch_bounds__(sample::TH, 4) void sample_pass_kernel(sample::Job J, sample::Work wk, int i) {
  using namespace sample;
  __shared__ union {
    Scratch<NW> sc;
    Counters h;
  } lds;
  __shared__ double table[64];
  const int n = blockIdx.y, s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int64_t at = (int64_t)n * J.S + s;
  const T* row = static_cast<const T*>(J.logits) + n * J.stride;
  Chunk<T, EPT> c;
  c.load(row, at_turn(J, s, 0) + wid * WAVE, J.V);
  const Row r = row_of(J.par, n, J.V);
  table[lane] = kPow[lane];  // (each wave, the same values: it may read them without a barrier)
  advance(J, wk, r, n, i, table, lds.sc);
  const State st = lds.sc.st;
  if (s == 0 && tid < (int)sizeof(State) / 4)
    reinterpret_cast<uint32_t*>(wk.state + (int64_t)(i & 1) * J.N + n)[tid] = reinterpret_cast<const uint32_t*>(&lds.sc.st)[tid];
  const bool count = st.kind;
  if (r.greedy || st.M == -INFINITY || !(count || kLast)) return;
  __syncthreads();
  // (in the last pass the digit, if any, is the last one: a bin is one value, and needs no mass)
  const bool weigh = !kLast && r.by_p && st.level < J.levels - 1;
  if (count) {
    lds.h.clear();
    __syncthreads();
  }
  // keys are compared up to the digits known: the prefix, or the whole cut (no cut: every key of a number is above 0)
  const Weights wt(r.t, st.M, table);
  const int dsh = 24 - 8 * st.level, sh = count ? dsh + 8 : 32 - 8 * st.cut_level;
  const uint32_t ref = count ? st.prefix : st.quota >= 0 ? st.thr : 0;
  for (int turn = 0; turn < J.turns; ++turn) {
    if (turn) c.load(row, at_turn(J, s, turn) + wid * WAVE, J.V);
    int64_t mass = 0;
    int ties = 0;
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const float v = c[e];
      const uint32_t k = key_of(v), k1 = k >> sh;
      if (kLast && k1 > ref && v != -INFINITY) {
        const double x = wt(v);
        if (x >= r.m || v == st.M) mass += (int64_t)fixed(x, J.one);
      }
      if (k1 == ref) {
        ++ties;
        if (count) {
          const int b = (k >> dsh & 255u) * COLS + tid % COLS;
          atomicAdd(&lds.h.count[b], 1u);
          if (weigh) atomicAdd(&lds.h.mass[b], fixed(wt(v), J.unit));
        }
      }
    }
    if (kLast) {
      mass = wave_total(mass);
      ties = wave_total(ties);
      if (lane == 0) {
        wk.kept[(at * J.turns + turn) * NW + wid] = mass;
        wk.ties[(at * J.turns + turn) * NW + wid] = ties;
      }
    }
  }
  if (!count) return;
  __syncthreads();
  lds.h.write(wk.step[i], at, weigh);
}

// grid (N): the draw.  Sums of weights are whole numbers here: first over the passes' workgroups, then over the found one's
// waves and turns, then over the found wave's elements.
template <typename T>
__global__ __launch_bounds__(sample::DT) void sample_draw_kernel(sample::Job J, sample::Work wk, int passes) {
  using namespace sample;
  constexpr int W = DT / 64, MC = MOST / CHUNK, EW = WAVE / DT;
  __shared__ Scratch<W> sc;
  __shared__ double table[64];
  __shared__ int64_t bin_mass[BINS], cmass[MC], wmass[TURNS * NW], part[W], found_before, target_;
  __shared__ int found, found_ties, cties[MC], wties[TURNS * NW], tpart[W];
  const int n = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int64_t base = (int64_t)n * J.S;
  const int nw = J.turns * NW;  // waves' sums of a workgroup
  const Row r = row_of(J.par, n, J.V);
  const int was_kind = wk.state[(int64_t)((passes - 1) & 1) * J.N + n].kind;
  double u = J.u64_ ? J.u64_[n] : (double)J.u[n];
  table[lane] = kPow[lane];  // (each wave, the same values: it may read them without a barrier)
  if (tid == 0) found = r.greedy ? INT32_MAX : -1;
  advance(J, wk, r, n, passes, table, sc);
  const State st = sc.st;
  if (r.greedy || st.M == -INFINITY) {
    if (tid == 0) found = INT32_MAX;
    __syncthreads();
    for (int s = tid; s < J.S0; s += DT)
      if (wk.lmax[(int64_t)n * J.S0 + s] == st.M) atomicMin(&found, wk.larg[(int64_t)n * J.S0 + s]);
    __syncthreads();
    if (tid == 0) J.out[n] = st.M == -INFINITY ? -1 : found;
    return;
  }
  const Weights weight(r.t, st.M, table);
  const int sh = 32 - 8 * st.cut_level;
  const bool cut = st.quota >= 0, open = was_kind;  // open: the waves' masses lack the bins of the last digit above the cut
  const uint32_t digit = st.thr & 255u;
  const int64_t quota = cut ? st.quota : 0;
  // an element's mass by its last digit (0: min_p drops it), at the cut and above it
  if (tid < BINS) {
    const float v = value_of((cut ? st.thr & ~255u : 0u) | (uint32_t)tid, J.levels);
    const double w = weight(v);
    bin_mass[tid] = cut && (uint32_t)tid >= digit && v <= st.M && (w >= r.m || v == st.M) ? (int64_t)fixed(w, J.one) : 0;
  }
  __syncthreads();
  const int64_t wt = cut ? bin_mass[digit] : 0;
  const uint32_t* count = wk.step[passes - 1].count;
  for (int s = wid; s < J.S; s += W) {
    int64_t m = lane < nw ? wk.kept[(base + s) * nw + lane] : 0;
    int t = lane < nw && !open ? wk.ties[(base + s) * nw + lane] : 0;
    if (open) {
      const uint4 c4 = *reinterpret_cast<const uint4*>(count + (base + s) * BINS + 4 * lane);
      const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t b = 4 * lane + e;
        if (b > digit) m += bin_mass[b] * (int64_t)c[e];
        if (b == digit) t = (int)c[e];
      }
    }
    m = wave_total(m);
    t = wave_total(t);
    if (lane == 0) cmass[s] = m, cties[s] = cut ? t : 0;
  }
  __syncthreads();
  // the first wave walks the chunks, 64 at a time: the whole mass (with the ties within the quota), then the chunk
  if (wid == 0) {
    int64_t target = 0;
    for (int turn = 0; turn < 2; ++turn) {
      int64_t sum = 0;
      int ties = 0;
      for (int s0 = 0; s0 < J.S; s0 += 64) {
        const int s = s0 + lane, t = s < J.S ? cties[s] : 0;
        const int upto_t = scan_up(t) + ties, before = upto_t - t;
        const int64_t room = quota - before, in = room <= 0 ? 0 : t < room ? t : room;
        const int64_t m = (s < J.S ? cmass[s] : 0) + in * wt;
        const int64_t upto = scan_up(m) + sum;
        if (turn && m && upto > target && upto - m <= target) {
          found = s;
          found_before = upto - m;
          found_ties = before;
        }
        sum = last_lane(upto);
        ties = last_lane(upto_t);
      }
      u = u > 0.0 ? u < 1.0 ? u : 0x1.fffffffffffffp-1 : 0.0;
      const u64 U = (u64)(u * 0x1p53);
      if (!turn) target = (int64_t)(__umul64hi((u64)sum, U) << 11 | (u64)sum * U >> 53);
    }
    if (lane == 0) target_ = target;
  }
  __syncthreads();
  const int64_t target = target_;
  if (found < 0) return;  // no mass: a row has its maximum at least, so this does not happen
  // ---- the chunk's waves
  const T* row = static_cast<const T*>(J.logits) + n * J.stride;
  const int64_t c0 = at_turn(J, found, 0);
  for (int x = wid; x < nw; x += W) {
    const int64_t at = (base + found) * nw + x;
    int64_t m = 0;
    int t = 0;
    if (open) {
      Chunk<T, EPT> c;
      c.load(row, c0 + x * WAVE, J.V);
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
    m = wave_total(m);
    t = wave_total(t);
    if (lane == 0) wmass[x] = m, wties[x] = t;
  }
  __syncthreads();
  int64_t upto = found_before;
  int before = found_ties, w0 = 0;
  for (; w0 < nw - 1; ++w0) {
    const int64_t x = wties[w0], room = quota - before, in = room <= 0 ? 0 : x < room ? x : room;
    const int64_t y = wmass[w0] + in * wt;
    if (upto + y > target) break;
    upto += y;
    before += (int)x;
  }
  // ---- that wave's elements, EW a thread in their order
  const int64_t i0 = c0 + (int64_t)w0 * WAVE + tid * EW;
  float v[EW];
  int t = 0;
#pragma unroll
  for (int e = 0; e < EW; ++e) {
    v[e] = i0 + e < J.V ? cleaned(as_float<T>(row[i0 + e])) : -INFINITY;
    t += cut && v[e] != -INFINITY && key_of(v[e]) >> sh == st.thr;
  }
  const int ts = scan_up(t);
  if (lane == 63) tpart[wid] = ts;
  __syncthreads();
  int rank = before + ts - t;
  for (int x = 0; x < wid; ++x) rank += tpart[x];
  int64_t m[EW], all = 0;
#pragma unroll
  for (int e = 0; e < EW; ++e) {
    const uint32_t k = key_of(v[e]) >> sh;
    m[e] = 0;
    if (v[e] != -INFINITY && (!cut || k > st.thr)) {
      const double x = weight(v[e]);
      if (x >= r.m || v[e] == st.M) m[e] = (int64_t)fixed(x, J.one);
    } else if (v[e] != -INFINITY && k == st.thr) {
      m[e] = rank++ < quota ? wt : 0;
    }
    all += m[e];
  }
  const int64_t as = scan_up(all);
  if (lane == 63) part[wid] = as;
  __syncthreads();
  upto += as - all;
  for (int x = 0; x < wid; ++x) upto += part[x];
#pragma unroll
  for (int e = 0; e < EW; ++e) {
    if (upto <= target && upto + m[e] > target) J.out[n] = i0 + e;
    upto += m[e];
  }
}

template <typename T>
static int launch_sample(sample::Job J, const sample::Work& wk, bool by_k, bool by_p, hipStream_t st) {
  const int open = ((int)by_k + (int)by_p) * (J.levels - 1), passes = 1 + (open ? open : 1);
  sample_first_kernel<T><<<dim3(J.S0, J.N), sample::TH, 0, st>>>(J, wk);
  const dim3 g(J.S, J.N);
  for (int i = 1; i < passes - 1; ++i) sample_pass_kernel<T, false><<<g, sample::TH, 0, st>>>(J, wk, i);
  sample_pass_kernel<T, true><<<g, sample::TH, 0, st>>>(J, wk, passes - 1);
  sample_draw_kernel<T><<<J.N, sample::DT, 0, st>>>(J, wk, passes);
  return check_launch("gdn_sample");
}
}  // namespace gdn

using namespace gdn;

namespace {
// A row's chunks, and the turns its workgroups take in the passes behind the first: as few as let all of them be on the
// chip at once (2 a CU), since each of them begins by merging its row's histograms.
void sample_cut(sample::Job& J) {
  J.S0 = (int)(((int64_t)J.V + sample::CHUNK - 1) / sample::CHUNK);
  const int64_t t = ((int64_t)J.N * J.S0 + 511) / 512;
  const int most = J.S0 < sample::TURNS ? J.S0 : sample::TURNS;
  J.turns = t > most ? most : t < 1 ? 1 : (int)t;
  J.S = (J.S0 + J.turns - 1) / J.turns;
}
int64_t sample_work(sample::Work& w, char* p, const sample::Job& J) {
  char* const base = p;
  const int N = J.N;
  // (J.S * J.turns may be less for more rows; a workspace for many rows has to hold fewer)
  const int64_t items = (int64_t)N * J.S0, turns = (int64_t)N * (J.S0 + sample::TURNS - 1);
  auto take = [&p](int64_t bytes) {
    char* q = p;
    p += (bytes + 255) / 256 * 256;
    return q;
  };
  w.lmax = reinterpret_cast<float*>(take(items * 4));
  w.larg = reinterpret_cast<int32_t*>(take(items * 4));
  w.state = reinterpret_cast<sample::State*>(take(2ll * N * sizeof(sample::State)));
  w.kept = reinterpret_cast<int64_t*>(take(turns * sample::NW * 8));
  w.ties = reinterpret_cast<int32_t*>(take(turns * sample::NW * 4));
  for (sample::Hist& h : w.step) {
    h.mass = reinterpret_cast<sample::u64*>(take(items * sample::BINS * 8));
    h.count = reinterpret_cast<uint32_t*>(take(items * sample::BINS * 4));
  }
  return p - base;
}
}  // namespace

extern "C" int64_t gdn_sample_workspace_bytes(int N, int V) {
  if (N < 0 || N > 65535 || V < 1 || V > sample::MOST) return -1;
  sample::Job J{};
  J.N = N, J.V = V;
  sample_cut(J);
  sample::Work w;
  return sample_work(w, nullptr, J);
}

extern "C" int gdn_sample(const void* logits, int64_t stride, int dtype, const void* u, int f64, const void* temperature,
                          const int32_t* top_k, const void* top_p, const void* min_p, double temperature1, int top_k1,
                          double top_p1, double min_p1, int64_t* out, int N, int V, void* work, int64_t work_bytes,
                          void* stream) {
  clear_error();
  const char* name = "gdn_sample";
  GDN_REQUIRE(N >= 0 && N <= 65535 && V >= 1, "%s: bad sizes", name);
  GDN_SUPPORT(V <= sample::MOST, "%s: at most %d logits a row", name, sample::MOST);
  GDN_REQUIRE(dtype == GDN_F32 || dtype == GDN_BF16 || dtype == GDN_F16, "%s: logits must be fp32, bf16 or fp16", name);
  if (N == 0) return GDN_OK;
  GDN_REQUIRE(logits && u && out && work, "%s: null pointer", name);
  GDN_REQUIRE(N == 1 || stride >= V, "%s: row stride too small", name);
  GDN_REQUIRE(f64 >= 0 && f64 < 16, "%s: bad fp64 flags", name);
  const bool u_is_f64 = f64 & GDN_SAMPLE_F64_U;
  GDN_REQUIRE(aligned(logits, dtype == GDN_F32 ? 4 : 2) && aligned(work, 256) && aligned(out, 8) && aligned(u, u_is_f64 ? 8 : 4) &&
                  aligned(temperature, f64 & GDN_SAMPLE_F64_TEMPERATURE ? 8 : 4) && aligned(top_k, 4) &&
                  aligned(top_p, f64 & GDN_SAMPLE_F64_TOP_P ? 8 : 4) && aligned(min_p, f64 & GDN_SAMPLE_F64_MIN_P ? 8 : 4),
              "%s: misaligned pointer (the workspace: 256 bytes)", name);
  GDN_REQUIRE(temperature || (temperature1 >= -1e300 && temperature1 <= 1e300), "%s: the temperature must be finite", name);
  GDN_REQUIRE((top_p || (top_p1 >= 0.0 && top_p1 <= 1.0)) && (min_p || (min_p1 >= 0.0 && min_p1 <= 1.0)),
              "%s: top_p and min_p must be in [0, 1]", name);
  sample::Job J{};
  J.N = N, J.V = V;
  sample_cut(J);
  sample::Work wk;
  const int64_t need = sample_work(wk, static_cast<char*>(work), J);
  GDN_REQUIRE(work_bytes >= need, "%s: workspace too small (%lld bytes needed)", name, (long long)need);
  J.logits = logits;
  J.stride = stride;
  J.u = u_is_f64 ? nullptr : static_cast<const float*>(u);
  J.u64_ = u_is_f64 ? static_cast<const double*>(u) : nullptr;
  J.out = out;
  J.par = {temperature, top_p, min_p, f64, top_k, temperature1, top_p1, min_p1, top_k1};
  J.levels = dtype == GDN_BF16 ? 2 : dtype == GDN_F16 ? 3 : 4;
  J.one = 0x1p50;  // V weights of at most `one` stay below 2^62
  while (J.one > 1.0 && J.one * V > 0x1p62) J.one *= 0.5;
  J.unit = 0x1p50;  // J.turns * CHUNK weights of at most `unit` stay at or below 2^63
  for (int t = 1; t < J.turns; t *= 2) J.unit *= 0.5;
  J.per = 1.0 / J.unit;
  const bool by_k = top_k || (top_k1 > 0 && top_k1 < V), by_p = top_p || top_p1 < 1.0;
  const hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case GDN_F32: return launch_sample<float>(J, wk, by_k, by_p, st);
    case GDN_BF16: return launch_sample<uint16_t>(J, wk, by_k, by_p, st);
    default: return launch_sample<_Float16>(J, wk, by_k, by_p, st);
  }
}
