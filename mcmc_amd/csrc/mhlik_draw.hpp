// mhlik_draw.hpp -- one column of each row of log weights, from a given random
// number.
//
// Row z_0 .. z_{n-1}, temperature T, top-k, top-p, min-p, and u in [0, 1):
//   w_j = exp((z_j - max) / T)                       an empty weight (-inf) is 0 at any T
//   order by z, largest first, equal ones by column; of that order keep
//     the first k                                    (k <= 0: all)
//     those before which less than p of the mass of these lies   (p >= 1: all; the first always)
//     those with w_j >= min(m, 1)                    (m <= 0: all)
//   the answer is the first column, in the COLUMNS' order, at which the kept mass exceeds u times all of it,
//   and log(w_j / kept mass).
// Every one of the three leaves a prefix of the same order, so what is kept is described by one pair (key, column): all
// larger values, and of those equal to the key the columns up to it.
//
// u is compared with sums of up to n weights, so weights and sums are double: with float sums a draw among 1e5 weights
// would land in a neighbouring column once in a few hundred draws.  Sums that pick a border are taken in 64-bit whole
// numbers (weights to 2^-51, or 2^-62 of what bounds their sum if that is more: n 2^-51 of the mass at most in all), so that
// the order of atomic additions does not matter; the sums u is compared with have a fixed shape.
#pragma once

#include "mhlik_predict.hpp"
#include "mhlik_softplus.h"

namespace mhlik {

struct DrawArgs {
  const void *z;
  int64_t rows, n, stride;
  const void *u;
  int32_t u_is_double;
  const float *temperature; // per row, or NULL: the value for all rows
  const int32_t *top_k;
  const float *top_p, *min_p;
  double temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int64_t *index;
  float *logp; // may be NULL
};

// Larger value, larger key; +0 and -0 are equal.
__device__ __forceinline__ uint32_t draw_key(float z)
{
  const uint32_t b = __float_as_uint(z + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ float draw_value(uint32_t key)
{
  return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

// A log weight as the kernels see it: +inf counts as the largest float, so that differences exist.
__device__ __forceinline__ float draw_finite(float z) { return fminf(z, 0x1.fffffep127f); }

// 2^((z - max) s), s = log2(e) / T: 1 at z = max, within 5e-16 relative where it matters ((z - max) s is rounded: another
// 1e-16 times itself), 0 below 2^-1020 and for z = -inf.  Whole part by adding 1.5 * 2^52, whose low bits then hold it;
// the rest goes through the degree-10 polynomial of mhlik_exp_fast with the powers of ln 2 multiplied in: 17 double
// instructions, of which none is slower than an addition.  EXACT_ZERO false, for sums only: 2^-1020 in place of 0.
template <bool EXACT_ZERO = true> __device__ __forceinline__ double draw_weight(float z, float max, double s)
{
  MHLIK_SP_COEF(c10, 0x1.e364ae3ebe671p-28);
  MHLIK_SP_COEF(c9, 0x1.b660a93518429p-24);
  MHLIK_SP_COEF(c8, 0x1.62c1651329726p-20);
  MHLIK_SP_COEF(c7, 0x1.ffcb6d52a8ae3p-17);
  MHLIK_SP_COEF(c6, 0x1.4309126702394p-13);
  MHLIK_SP_COEF(c5, 0x1.5d87fe93109eep-10);
  MHLIK_SP_COEF(c4, 0x1.3b2ab6fbd4a75p-7);
  MHLIK_SP_COEF(c3, 0x1.c6b08d704396dp-5);
  MHLIK_SP_COEF(c2, 0x1.ebfbdff82c46cp-3);
  MHLIK_SP_COEF(c1, 0x1.62e42fefa39efp-1);
  const double y = fmax(((double)z - (double)max) * s, EXACT_ZERO ? -1100.0 : -1020.0); // NaN (-inf * 0) too
  const double m = y + 0x1.8p52, f = y - (m - 0x1.8p52);
  double p = fma(c10, f, c9);
  p = fma(p, f, c8);
  p = fma(p, f, c7);
  p = fma(p, f, c6);
  p = fma(p, f, c5);
  p = fma(p, f, c4);
  p = fma(p, f, c3);
  p = fma(p, f, c2);
  p = fma(p, f, c1);
  p = fma(p, f, 1.0);
  const double w = __hiloint2double(__double2hiint(p) + (int)((uint32_t)__double2loint(m) << 20), __double2loint(p));
  return EXACT_ZERO && y < -1020.0 ? 0.0 : w;
}

// The choices of one row.
struct DrawChoice {
  double temp, rate, share, least, u; // rate: log2(e) / temp; least: at most 1
  int k;                               // 0: no top-k
  bool bad, greedy;                    // a choice that is not a number; temperature 0
};

__device__ inline DrawChoice draw_choice(const DrawArgs &a, int64_t row)
{
  DrawChoice c;
  c.temp = a.temperature ? (double)a.temperature[row] : a.temperature_all;
  c.share = a.top_p ? (double)a.top_p[row] : a.top_p_all;
  c.least = a.min_p ? (double)a.min_p[row] : a.min_p_all;
  c.u = a.u_is_double ? ((const double *)a.u)[row] : (double)((const float *)a.u)[row];
  c.k = a.top_k ? a.top_k[row] : a.top_k_all;
  if (c.k <= 0 || c.k >= a.n) c.k = 0;
  c.bad = !(c.temp >= 0.0) || c.share != c.share || c.least != c.least || c.u != c.u;
  c.greedy = c.temp == 0.0;
  c.rate = c.greedy ? 1.0 : 1.4426950408889634074 / c.temp;
  c.share = c.share > 0.0 ? c.share : 0.0;
  if (c.least > 1.0) c.least = 1.0;
  return c;
}

__device__ inline void draw_answer(const DrawArgs &a, int64_t row, int64_t column, double logp)
{
  a.index[row] = column;
  if (a.logp) a.logp[row] = (float)logp;
}

__device__ inline void draw_nothing(const DrawArgs &a, int64_t row)
{
  a.index[row] = -1;
  if (a.logp) a.logp[row] = __uint_as_float(0x7fc00000u);
}

// Values by distance from the largest: bin 0 holds the largest.  Distances beyond `range` share the last bin.
template <int BINS> struct DrawBin {
  float max, scale;
  __device__ DrawBin(float max_, float min_, double temp) : max(max_)
  {
    // Weights e^-40 below the largest matter to no sum here, while a row may hold a lowest-of-its-type mask: the range
    // is the nearer of the two.  All equal: one bin.
    const float range = fminf((float)(40.0 * temp), max_ - min_);
    scale = range > 0.f ? (float)BINS / range : 0.f;
    if (!(scale < __uint_as_float(0x7f800000u))) scale = 0x1p127f; // a range below the smallest normal float
  }
  __device__ __forceinline__ int of(float z) const
  {
    return (int)fminf((max - z) * scale, (float)(BINS - 1));
  }
};

// rint(w 2^shift) of a weight, shift <= 51: added to 2^(52 - shift), its whole multiples of 2^-shift are the low bits of
// the sum.  Two instructions, where scaling and converting takes twelve.
__device__ __forceinline__ unsigned long long draw_fixed(double w, int shift)
{
  const int one = (1023 + 52 - shift) << 20;
  const double v = w + __hiloint2double(one, 0);
  return (unsigned long long)(uint32_t)(__double2hiint(v) - one) << 32 | (uint32_t)__double2loint(v);
}

// A weight to within 2e-5 relative (or 2^-126), for bounds: float's own instruction.
__device__ __forceinline__ float draw_rough(float z, float max, double rate)
{
  const float y = fmaxf((z - max) * (float)fmin(rate, 0x1p127), -126.f); // NaN (-inf * 0) too
  return __builtin_amdgcn_exp2f(y);
}

// The finest shift, up to 51, at which sums of up to `bound` (at least 1) stay below 2^63.
__device__ __forceinline__ int draw_shift(float bound)
{
  const int e = (int)(__float_as_uint(bound) >> 23) - 127; // bound < 2^(e + 1)
  return __builtin_amdgcn_readfirstlane(e > 11 ? 62 - e : 51); // all lanes have the same
}

// Position in the order: smaller is earlier (larger value, lower column).
__device__ __forceinline__ unsigned long long draw_place(float z, int j)
{
  return (unsigned long long)~draw_key(z) << 32 | (uint32_t)j;
}

// The same value, of which the compiler does not know that it is: what was worked out from it before is worked out again,
// and need not wait in a register.
template <typename V> __device__ __forceinline__ V draw_again(V v)
{
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(v));
#endif
  return v;
}

// The kept prefix ends with this place.
struct DrawEnd {
  unsigned long long place;
  __device__ __forceinline__ bool kept(float z, int j) const { return draw_place(z, j) <= place; }
};

// The first column whose running sum exceeds `aim`, over weights w[i] at places base + i * 64 + lane of a wave's run;
// base: the wave's first place, waves in order.  IS_SHARE: aim is a share of the whole sum, which comes back in *total.
// On return place >= 0 in the one lane that has it, with its *weight and what is left of the aim where it begins (*rest).
template <int THREADS, int VPT, bool IS_SHARE>
__device__ int draw_pick(const double (&w)[VPT], double aim, double *total, double *weight, double *rest, double *lds /* [THREADS / 64] */)
{
  constexpr int kWaves = THREADS / kWave;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  double m = 0.0;
#pragma unroll
  for (int i = 0; i < VPT; i++) m += w[i];
  m = wave_sum(m);
  __syncthreads();
  if (lane == 0) lds[wave] = m;
  __syncthreads();
  // the first wave that exceeds the aim; if rounding leaves none, the last with any mass
  const double of = lane < kWaves ? lds[lane] : 0.0, upto = wave_running(of);
  if (IS_SHARE) {
    *total = wave_last(upto);
    aim *= *total;
  }
  const unsigned long long passed = __ballot(of > 0.0 && upto > aim), any = __ballot(of > 0.0);
  const int pick = passed ? __ffsll(passed) - 1 : 63 - __clzll((long long)any);
  const double before = pick > 0 ? wave_lane(upto, pick - 1) : 0.0;
  int place = -1;
  if (wave == pick) {
    aim -= before;
    int at = 0;
    double mine = w[0];
    if (VPT > 1) { // the same for the runs of 64: lane i has the sum of run i
      const double each = wave_sums<VPT>(w), to = wave_running(each);
      const unsigned long long runs = (1ull << VPT) - 1, over = __ballot(each > 0.0 && to > aim) & runs, some = __ballot(each > 0.0) & runs;
      at = over ? __ffsll(over) - 1 : 63 - __clzll((long long)some);
      if (at > 0) aim -= wave_lane(to, at - 1);
#pragma unroll
      for (int i = 1; i < VPT; i++)
        if (i == at) mine = w[i];
    }
    const double run = wave_running(mine);
    const unsigned long long over = __ballot(mine > 0.0 && run > aim), some = __ballot(mine > 0.0);
    const int who = over ? __ffsll(over) - 1 : 63 - __clzll((long long)some);
    if (lane == who) {
      place = (wave * VPT + at) * kWave + lane;
      *weight = mine;
      *rest = aim - (run - mine);
    }
  }
  return place;
}

// The sum before this thread's bins, from its own `mine`; *all: of all bins.  One barrier; lds is free after the next.
template <int THREADS, typename V> __device__ __forceinline__ V draw_before(V mine, V *all, V *lds)
{
  constexpr int kWaves = THREADS / kWave;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const V in = wave_running(mine);
  if (lane == kWave - 1) lds[wave] = in;
  __syncthreads();
  const V upto = wave_running(lane < kWaves ? lds[lane] : (V)0);
  *all = wave_last(upto);
  return in - mine + (wave > 0 ? wave_lane(upto, wave - 1) : (V)0);
}

// ---------------------------------------------------- whole rows, any data
//
// The key of the border is found eight bits at a time, each time from a histogram over the whole row.  It needs nothing
// of the data and serves the rows that the quick ways below hand back: more equal (or nearly equal) values at a border
// than they have places for, a top-k of thousands.

constexpr int kDrawBins = 256;

// What a workgroup shares.
struct DrawShared {
  unsigned long long mass[kDrawBins];
  uint32_t count[kDrawBins];
  double d[32];
  unsigned long long q[32];
  float f[32];
  uint32_t i[32];
};

template <typename T> struct DrawRow {
  const T *z;
  int n;
  float max;
  double rate;
  uint32_t key; // kept: larger keys, and equal ones up to column `last`
  int last;
  __device__ __forceinline__ float at(int j) const { return draw_finite((float)z[j]); }
  __device__ __forceinline__ bool kept(uint32_t k, int j) const { return k > key || (k == key && j <= last); }
};

// The prefix of the kept order that is needed for `k` values (BY_MASS false) or for `share` of the kept mass (true):
// key and column are narrowed.  The key is found eight bits at a time from a histogram of the values that share the bits
// found so far.
template <typename T, int THREADS, bool BY_MASS>
__device__ void draw_narrow(DrawRow<T> &r, DrawShared &s, int shift, uint32_t k, double share)
{
  const int tid = threadIdx.x;
  const double unit = ldexp(1.0, -shift);
  uint32_t prefix = 0, above_n = 0;
  unsigned long long above_m = 0;
  double target = 0.0;
  uint32_t equal = 0;
  for (int level = 0; level < 4; level++) {
    const int low = 24 - 8 * level, high = low + 8;
    for (int b = tid; b < kDrawBins; b += THREADS) {
      s.count[b] = 0;
      if (BY_MASS) s.mass[b] = 0;
    }
    __syncthreads();
    for (int j = tid; j < r.n; j += THREADS) {
      const float z = r.at(j);
      const uint32_t key = draw_key(z);
      if (level && key >> high != prefix) continue;
      if (!r.kept(key, j)) continue;
      const uint32_t bin = (key >> low) & 255u;
      atomicAdd(&s.count[bin], 1u);
      if (BY_MASS) {
        const unsigned long long m = draw_fixed(draw_weight(z, r.max, r.rate), shift);
        if (m) atomicAdd(&s.mass[bin], m);
      }
    }
    __syncthreads();
    // sums from the top bin down; a thread has kRun bins, or none
    constexpr int kRun = THREADS >= kDrawBins ? 1 : kDrawBins / THREADS;
    const bool has = tid * kRun < kDrawBins;
    uint32_t cn[kRun], n = 0, some;
    unsigned long long cm[kRun], m = 0, all;
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      n += cn[i] = has ? s.count[kDrawBins - 1 - tid * kRun - i] : 0;
      m += cm[i] = has && BY_MASS ? s.mass[kDrawBins - 1 - tid * kRun - i] : 0;
    }
    n = above_n + draw_before<THREADS>(n, &some, s.i);
    m = above_m + draw_before<THREADS>(m, &all, s.q);
    if (BY_MASS && level == 0) target = share * ((double)all * unit);
    if (tid == 0) {
      s.i[31] = 0;
      s.i[30] = 0;
    }
    __syncthreads();
    // the first bin, from the top, that reaches the aim; the mass may miss it by rounding: then the lowest bin in use
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      if (cn[i]) {
        const uint32_t bin = kDrawBins - 1 - tid * kRun - i;
        atomicMax(&s.i[30], kDrawBins - bin);
        const bool reach = BY_MASS ? (double)(m + cm[i]) * unit >= target : n + cn[i] >= k;
        const bool before = BY_MASS ? (double)m * unit >= target && n > 0 : n >= k;
        if (reach && !before) s.i[31] = kDrawBins - bin;
      }
      n += cn[i];
      m += cm[i];
    }
    __syncthreads();
    const uint32_t bin = kDrawBins - (s.i[31] ? s.i[31] : s.i[30]);
    // what lies above that bin
#pragma unroll
    for (int i = kRun - 1; i >= 0; i--) {
      n -= cn[i];
      m -= cm[i];
      if (has && kDrawBins - 1 - tid * kRun - i == (int)bin) {
        s.i[29] = n;
        s.q[29] = m;
        s.i[28] = cn[i];
      }
    }
    __syncthreads();
    above_n = s.i[29];
    above_m = s.q[29];
    equal = s.i[28];
    prefix = prefix << 8 | bin;
    __syncthreads();
  }
  // `prefix` is the key now; of its `equal` columns the first `take` are needed
  uint32_t take;
  if (BY_MASS) {
    const double w = draw_weight(draw_value(prefix), r.max, r.rate), a = (double)above_m * unit;
    const double c = w > 0.0 ? ceil((target - a) / w) : 1.0;
    take = c < 1.0 ? 1u : c > (double)equal ? equal : (uint32_t)c;
    if (take > 1 && a + (take - 1) * w >= target) take--;
    if (take < equal && a + take * w < target) take++;
  } else {
    take = k - above_n;
  }
  int last = prefix == r.key ? r.last : r.n; // a border among the same values stands: none of those behind it comes back
  if (take < equal) { // find the column: waves count in runs of columns, then one wave looks through the right run
    constexpr int kWaves = THREADS / kWave;
    const int run = ((r.n + kWaves - 1) / kWaves + kWave - 1) / kWave * kWave;
    const int lane = tid % kWave, wave = tid / kWave;
    const int from = wave * run < r.n ? wave * run : r.n, to = from + run < r.n ? from + run : r.n;
    uint32_t c = 0;
    for (int j = from; j < to; j += kWave) {
      const bool is = j + lane < to && draw_key(r.at(j + lane)) == prefix && r.kept(prefix, j + lane);
      c += __popcll(__ballot(is));
    }
    if (lane == 0) s.i[wave] = c;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; w++) before += s.i[w];
    __syncthreads();
    if (before < take && before + c >= take) {
      for (int j = from; j < to; j += kWave) {
        const bool is = j + lane < to && draw_key(r.at(j + lane)) == prefix && r.kept(prefix, j + lane);
        const unsigned long long b = __ballot(is);
        const uint32_t here = __popcll(b);
        if (before + here >= take) {
          const uint32_t rank = __popcll(b & ((1ull << lane) - 1));
          if (is && before + rank + 1 == take) s.i[27] = (uint32_t)(j + lane);
          break;
        }
        before += here;
      }
    }
    __syncthreads();
    last = (int)s.i[27];
    __syncthreads();
  }
  r.key = prefix;
  r.last = last;
}


// ------------------------------------------------ rows that fit a workgroup
//
// The values stay in registers, 64 consecutive columns to a wave's register.  A histogram by distance from the largest
// gives the bin in which the border falls; the few values of that bin go to LDS and each finds its rank, and the mass
// before it, by comparing with all others.  Top-k first, over counts (32-bit atomics: of all values), then top-p, over
// masses (64-bit ones: only of what top-k left).

template <int THREADS> struct ShortShared {
  static constexpr int kBins = THREADS < 256 ? 256 : THREADS;          // one a thread, or four
  static constexpr int kCap = THREADS < 256 ? 128 : THREADS;           // values of a border's bin
  unsigned long long mass[kBins];
  uint32_t count[kBins];               // later the columns of what top-k left
  float value[THREADS];                // ... and their values
  unsigned long long place[kCap];
  unsigned long long cmass[kCap];
  double d[32];
  unsigned long long q[32];
  float f[32], g[32];
  uint32_t i[32];
};

// The place of the k-th of the values above -inf; unchanged if there are no more than k.  False: no room.
template <int THREADS, int VPT, typename AT>
__device__ bool draw_by_count(const float (&z)[VPT], const int (&bin)[VPT], AT at, uint32_t k, ShortShared<THREADS> &s, DrawEnd *end)
{
  constexpr int kRun = ShortShared<THREADS>::kBins / THREADS;
  const int tid = threadIdx.x;
#pragma unroll
  for (int i = 0; i < kRun; i++) s.count[tid + i * THREADS] = 0;
  if (tid == 0) s.i[30] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < VPT; i++)
    if (z[i] > -HUGE_VALF) atomicAdd(&s.count[bin[i]], 1u);
  __syncthreads();
  uint32_t here[kRun], mine = 0, all;
#pragma unroll
  for (int i = 0; i < kRun; i++) mine += here[i] = s.count[tid * kRun + i];
  uint32_t n = draw_before<THREADS>(mine, &all, s.i);
  if (all <= k) return true;
#pragma unroll
  for (int i = 0; i < kRun; i++) {
    if (n < k && n + here[i] >= k) {
      s.i[31] = tid * kRun + i;
      s.i[29] = n;
    }
    n += here[i];
  }
  __syncthreads();
  const int border = (int)s.i[31];
#pragma unroll
  for (int i = 0; i < VPT; i++)
    if (z[i] > -HUGE_VALF && bin[i] == border) {
      const uint32_t q = atomicAdd(&s.i[30], 1u);
      if (q < ShortShared<THREADS>::kCap) s.place[q] = draw_place(draw_again(z[i]), at(i));
    }
  __syncthreads();
  const int m = (int)s.i[30];
  if (m > ShortShared<THREADS>::kCap) return false;
  for (int c = tid; c < m; c += THREADS) {
    const unsigned long long own = s.place[c];
    uint32_t rank = s.i[29];
    for (int q = 0; q < m; q++) rank += s.place[q] < own;
    if (rank == k - 1) s.q[31] = own;
  }
  __syncthreads();
  end->place = s.q[31];
  return true;
}

// Of the values with a weight, the place of the last before which (with `base` before them all) less than the target
// lies; share: the target is this share of their mass.  False: no room.
template <int THREADS, int VPT, typename AT>
__device__ bool draw_by_mass(const float (&z)[VPT], const double (&weight)[VPT], const int (&bin)[VPT], AT at, unsigned long long base,
                             double share, double target, int shift, ShortShared<THREADS> &s, DrawEnd *end)
{
  constexpr int kBins = ShortShared<THREADS>::kBins, kRun = kBins / THREADS;
  const int tid = threadIdx.x;
  const double unit = ldexp(1.0, -shift);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRun; i++) s.mass[tid + i * THREADS] = 0;
  if (tid == 0) {
    s.i[30] = 0;
    s.i[31] = kBins;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const unsigned long long m = draw_fixed(weight[i], shift);
    if (m) atomicAdd(&s.mass[bin[i]], m);
  }
  __syncthreads();
  unsigned long long here[kRun], mine = 0, all;
#pragma unroll
  for (int i = 0; i < kRun; i++) mine += here[i] = s.mass[tid * kRun + i];
  unsigned long long before = base + draw_before<THREADS>(mine, &all, s.q);
  if (share >= 0.0) target = share * ((double)all * unit);
#pragma unroll
  for (int i = 0; i < kRun; i++) {
    if (here[i] && ((double)before * unit < target || before == 0) && (double)(before + here[i]) * unit >= target) {
      s.i[31] = tid * kRun + i; // one bin at most: the sums grow
      s.q[29] = before;
    }
    before += here[i];
  }
  if (tid == 0) s.q[31] = 0;
  __syncthreads();
  const int border = (int)s.i[31];
  if (border == kBins) return true; // what is here ends before the target: all of it
#pragma unroll
  for (int i = 0; i < VPT; i++)
    if (weight[i] > 0.0 && bin[i] == border) {
      const uint32_t q = atomicAdd(&s.i[30], 1u);
      if (q < ShortShared<THREADS>::kCap) {
        s.place[q] = draw_place(draw_again(z[i]), at(i));
        s.cmass[q] = draw_fixed(draw_again(weight[i]), shift);
      }
    }
  __syncthreads();
  const int m = (int)s.i[30];
  if (m > ShortShared<THREADS>::kCap) return false;
  for (int c = tid; c < m; c += THREADS) {
    const unsigned long long own = s.place[c];
    unsigned long long b = s.q[29];
    uint32_t rank = 0;
    for (int q = 0; q < m; q++) {
      const bool earlier = s.place[q] < own;
      b += earlier ? s.cmass[q] : 0;
      rank += earlier;
    }
    if ((double)b * unit < target || (s.q[29] == 0 && rank == 0)) atomicMax(&s.q[31], own);
  }
  __syncthreads();
  end->place = s.q[31];
  return true;
}

// Weights behind the end of the kept prefix become 0.
template <int VPT, typename AT> __device__ __forceinline__ void draw_cut(const float (&z)[VPT], double (&weight)[VPT], AT at, const DrawEnd &end)
{
#pragma unroll
  for (int i = 0; i < VPT; i++)
    if (!end.kept(draw_again(z[i]), at(i))) weight[i] = 0.0;
}

// Cuts the row's top-k and top-p.  z: -inf where there is nothing; column j of z[i] from at(i); weight: of z[i].  False if
// a border's bin holds more values than there is room for.
template <int THREADS, int VPT, typename AT>
__device__ bool draw_short_narrow(const float (&z)[VPT], double (&weight)[VPT], AT at, float max, float min, const DrawChoice &c,
                                  int shift, ShortShared<THREADS> &s)
{
  const DrawBin<ShortShared<THREADS>::kBins> bin(max, min, c.temp);
  int bins[VPT];
#pragma unroll
  for (int i = 0; i < VPT; i++) bins[i] = bin.of(z[i]);
  DrawEnd end{~0ull};
  if (c.k) {
    if (!draw_by_count<THREADS, VPT>(z, bins, at, (uint32_t)c.k, s, &end)) return false;
    draw_cut<VPT>(z, weight, at, end);
  }
  if (c.share < 1.0) {
    if (!draw_by_mass<THREADS, VPT>(z, weight, bins, at, 0, c.share, 0.0, shift, s, &end)) return false;
    draw_cut<VPT>(z, weight, at, end);
  }
  return true;
}

// A row with a top-k of at most as many values as there are threads: what it leaves goes to LDS in the order of the columns,
// one value a thread, so that weights, top-p, min-p and the draw are the work of one value a thread and not of VPT (4096
// rows of 2000, top-k 40 and top-p: 28 us, with VPT 34).  The row's answer.  False if the border's bin holds more values
// than there is room for.
template <int THREADS, int VPT, typename AT>
__device__ bool draw_short_top(const DrawArgs &a, int64_t row, const float (&z)[VPT], AT at, float max, float min, const DrawChoice &c,
                               int shift, ShortShared<THREADS> &s)
{
  const DrawBin<ShortShared<THREADS>::kBins> bin(max, min, c.temp);
  int bins[VPT];
#pragma unroll
  for (int i = 0; i < VPT; i++) bins[i] = bin.of(z[i]);
  DrawEnd end{~0ull};
  if (!draw_by_count<THREADS, VPT>(z, bins, at, (uint32_t)c.k, s, &end)) return false;
  constexpr int kWaves = THREADS / kWave;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  bool keep[VPT];
  unsigned long long kept[VPT]; // the same of all lanes
  uint32_t n = 0;
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    keep[i] = z[i] > -HUGE_VALF && end.kept(draw_again(z[i]), at(i));
    kept[i] = __ballot(keep[i]);
    n += __popcll(kept[i]);
  }
  __syncthreads(); // the counts and sums of before have been read
  if (lane == 0) s.i[wave] = n;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    const uint32_t there = s.i[w];
    if (w < wave) before += there;
    all += there;
  }
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const uint32_t to = __builtin_amdgcn_mbcnt_hi((uint32_t)(kept[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)kept[i], before));
    if (keep[i]) {
      s.value[to] = z[i];
      s.count[to] = (uint32_t)at(i);
    }
    before += __popcll(kept[i]);
  }
  __syncthreads();
  const bool mine = (uint32_t)tid < all;
  const float own[1] = {mine ? s.value[tid] : -HUGE_VALF};
  const int column = mine ? (int)s.count[tid] : 0;
  double w[1] = {draw_weight(own[0], max, c.rate)};
  if (c.share < 1.0) {
    const int b[1] = {bin.of(own[0])};
    auto here = [&](int) { return column; };
    draw_by_mass<THREADS, 1>(own, w, b, here, 0, c.share, 0.0, shift, s, &end); // (there is room for every thread's)
    draw_cut<1>(own, w, here, end);
  }
  if (w[0] < c.least) w[0] = 0.0;
  double total, weight, rest;
  __syncthreads();
  if (draw_pick<THREADS, 1, true>(w, c.u, &total, &weight, &rest, s.d) >= 0) draw_answer(a, row, column, log(weight / total));
  return true;
}

// What the kernels that finish a row keep in LDS: one of the two at a time.
template <int THREADS> union RowShared {
  ShortShared<THREADS> quick;
  DrawShared whole;
};

// The whole-row way to the end of the kept prefix.
template <typename T, int THREADS>
__device__ DrawEnd draw_whole(const DrawArgs &a, int64_t row, const DrawChoice &c, float max, int shift, DrawShared &s)
{
  DrawRow<T> r;
  r.z = (const T *)a.z + row * a.stride;
  r.n = (int)a.n;
  r.max = max;
  r.rate = c.rate;
  r.key = 0;
  r.last = r.n;
  __syncthreads();
  if (c.k) draw_narrow<T, THREADS, false>(r, s, shift, (uint32_t)c.k, 0.0);
  if (c.share < 1.0) draw_narrow<T, THREADS, true>(r, s, shift, 0u, c.share);
  __syncthreads();
  return DrawEnd{(unsigned long long)~r.key << 32 | (uint32_t)r.last};
}

// Rows of up to THREADS * VPT values.  Bound by instructions (17 double ones a weight, the scans, the borders) and some 20
// barriers: 4096 rows of 2000, every choice: 36 us; no choice: 20 us; one row of 1000: 6 us.
template <typename T, int THREADS, int VPT> __global__ __launch_bounds__(THREADS) void draw_short_kernel(DrawArgs a, int shift)
{
  __shared__ RowShared<THREADS> s;
  constexpr int kWaves = THREADS / kWave;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, n = (int)a.n;
  const T *zp = (const T *)a.z + row * a.stride;
  float z[VPT];
  auto at = [&](int i) { return (wave * VPT + i) * kWave + lane; };
  float max = -HUGE_VALF, min = HUGE_VALF;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const float v = at(i) < n ? (float)zp[at(i)] : -HUGE_VALF;
    nan |= v != v;
    z[i] = draw_finite(v);
    max = fmaxf(max, z[i]);
    min = fminf(min, z[i] > -HUGE_VALF ? z[i] : HUGE_VALF);
  }
  const DrawChoice c = draw_choice(a, row);
  max = wave_max(max);
  min = wave_min(min);
  const bool any = __any(nan);
  if (lane == 0) {
    s.quick.f[wave] = max;
    s.quick.g[wave] = min;
    s.quick.i[wave] = any;
  }
  __syncthreads();
  bool bad = c.bad;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    max = fmaxf(max, s.quick.f[w]);
    min = fminf(min, s.quick.g[w]);
    bad |= s.quick.i[w] != 0;
  }
  __syncthreads();
  if (bad || max == -HUGE_VALF) {
    if (tid == 0) draw_nothing(a, row);
    return;
  }
  if (c.greedy) {
    if (tid == 0) s.quick.i[0] = 0xffffffffu;
    __syncthreads();
    int first = n;
#pragma unroll
    for (int i = VPT - 1; i >= 0; i--)
      if (z[i] == max) first = at(i);
    if (first < n) atomicMin(&s.quick.i[0], (uint32_t)first);
    __syncthreads();
    if (tid == 0) draw_answer(a, row, s.quick.i[0], 0.0);
    return;
  }
  const bool few = c.k && c.k <= THREADS;
  if (few && draw_short_top<THREADS, VPT>(a, row, z, at, max, min, c, shift, s.quick)) return;
  double w[VPT];
  auto weights = [&]() {
#pragma unroll
    for (int i = 0; i < VPT; i++) w[i] = draw_weight(draw_again(z[i]), max, c.rate);
  };
  if (!few) weights();
  if (few || ((c.k || c.share < 1.0) && !draw_short_narrow<THREADS, VPT>(z, w, at, max, min, c, shift, s.quick))) {
    const DrawEnd end = draw_whole<T, THREADS>(a, row, c, max, shift, s.whole);
    weights(); // again, so that they take no registers in there
    draw_cut<VPT>(z, w, at, end);
  }
#pragma unroll
  for (int i = 0; i < VPT; i++)
    if (w[i] < c.least) w[i] = 0.0;
  double total, weight, rest;
  __syncthreads();
  const int place = draw_pick<THREADS, VPT, true>(w, c.u, &total, &weight, &rest, s.quick.d);
  if (place >= 0) draw_answer(a, row, place, log(weight / total));
}

// --------------------------------------------------------------- long rows
//
// A row is cut into units of 64 * VPT columns, one a wave, so that a few long rows fill the chip too.  Up to four kernels,
// of which the host leaves out those that no row needs:
//   top      each unit's largest value; for plain rows (no top-k, top-p, min-p) its mass too, relative to that value
//   histo    top-k: how many values lie in each bin of distance from the row's largest; top-p: their masses
//   collect  from the histogram the border's bin.  top-k: every value down to that bin goes to the unit's list (with
//            their place in order); top-p: the bin's own values go there, the mass of what lies above is summed; min-p
//            alone: the sum
//   finish   one workgroup a row: the border among the listed values, the unit in which the kept mass exceeds u of the
//            whole, the column in it.  A row whose lists are too long goes the whole-row way.
// Few rows are bound by the four kernels' latencies (one row of 131072, top-k and top-p: 3 + 4 + 6 + 9 us); many by double
// instructions beside the reading (256 rows of 131072 without a choice: 34 us for `top`, 3.9 TB/s; with top-p 142 in all).  What the
// whole-row way takes is one workgroup's work: 64 rows of 50001 whose top-p ends in a crowded bin 142 us, others 37.

constexpr int kLongBins = 512;
constexpr int kLongList = 2048;  // listed values of a row
constexpr int kLongUnits = 1024; // units of a row: one a thread of the finishing workgroup

struct LongPart {
  float max, min; // min: of the values above -inf
  int first;      // column of max
  int nan;
  double mass;    // of exp((z - max) / T), plain rows
};

enum { kRowNothing = 0, kRowGreedy, kRowPlain, kRowSums, kRowList, kRowNucleus };

struct LongCell { // one row's border bin
  int bin;
  int too_long;
  unsigned long long above;
  double target;
  int shift;
};

struct LongCand {
  float z;
  int j;
};

struct LongSpace {
  LongPart *part;           // [rows][units]
  double *kept;             // [rows][units]
  int *listed;              // [rows][units]
  LongCand *list;           // [rows][units][unit / 2]
  unsigned long long *histo; // [rows][kLongBins]
  LongCell *cell;           // [rows]
  int *shift;               // [rows]
  int units, groups;        // per row: waves, workgroups of four
};

// What a row needs.
__device__ inline int draw_kind(const DrawChoice &c, bool bad, float max)
{
  const int kind = bad || c.bad || max == -HUGE_VALF ? kRowNothing
                   : c.greedy                        ? kRowGreedy
                   : c.k                             ? kRowList
                   : c.share < 1.0                   ? kRowNucleus
                   : c.least > 0.0                   ? kRowSums
                                                     : kRowPlain;
  return __builtin_amdgcn_readfirstlane(kind); // all lanes have the same
}

// The row's largest and smallest value from its units'; every wave does it for itself.  *own: the largest of this lane's units.
__device__ inline void draw_row_range(const LongPart *part, int units, float *max, float *min, bool *nan, float *own)
{
  float a = -HUGE_VALF, b = HUGE_VALF;
  int bad = 0;
  for (int q = threadIdx.x % kWave; q < units; q += kWave) {
    a = fmaxf(a, part[q].max);
    b = fminf(b, part[q].min);
    bad |= part[q].nan;
  }
  *own = a;
  *max = wave_max(a);
  *min = wave_min(b);
  *nan = __any(bad) != 0;
}

// The shift of a row's masses, from what its units can weigh at most: n alone as the bound would lose weights that are
// faint but many (of 2^21 columns, 2^-44 each beside one of 1: 2^-23 of the mass, and none would count).  The units'
// largest values weigh a unit-th of the bound at least, so that all roundings together stay below n 2^-51 of the mass.
__device__ inline int draw_row_shift(const LongPart *part, int units, int unit, float max, float own, double rate)
{
  float b = draw_rough(own, max, rate);
  if (units > kWave) { // a lane has several
    b = 0.f;
    for (int q = threadIdx.x % kWave; q < units; q += kWave) b += draw_rough(part[q].max, max, rate);
  }
  return draw_shift(1.001f * unit * wave_sum(b));
}

// A unit's values: register v * VEC + e of lane l holds column base + (v * 64 + l) * VEC + e; -inf past the end.  True if
// one of them is NaN.
template <typename T, int VEC, int VPT> __device__ __forceinline__ bool draw_load(const T *row, int n, int base, float (&z)[VPT])
{
  bool nan = false;
  struct __attribute__((packed, aligned(sizeof(T)))) Pack { T e[VEC]; }; // gfx950 takes unaligned accesses
  const int lane = threadIdx.x % kWave;
  if (base + VPT * kWave <= n) {
    Pack p[VPT / VEC];
#pragma unroll
    for (int v = 0; v < VPT / VEC; v++) p[v] = *(const Pack *)(row + base + (v * kWave + lane) * VEC);
#pragma unroll
    for (int v = 0; v < VPT / VEC; v++)
#pragma unroll
      for (int e = 0; e < VEC; e++) z[v * VEC + e] = (float)p[v].e[e];
  } else {
#pragma unroll
    for (int v = 0; v < VPT / VEC; v++)
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        const int j = base + (v * kWave + lane) * VEC + e;
        z[v * VEC + e] = j < n ? (float)row[j] : -HUGE_VALF;
      }
  }
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    nan |= z[i] != z[i];
    z[i] = draw_finite(z[i]);
  }
  return nan;
}
template <int VEC> __device__ __forceinline__ int draw_column(int base, int i)
{
  return base + (i / VEC * kWave + (int)threadIdx.x % kWave) * VEC + i % VEC;
}

template <typename T, int VEC, int VPT>
__global__ __launch_bounds__(kBlock) void draw_top_kernel(DrawArgs a, LongSpace g, int with_histo)
{
  const int64_t row = blockIdx.x / g.groups;
  const int group = blockIdx.x % g.groups, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  if (with_histo)
    for (int b = group * kBlock + threadIdx.x; b < kLongBins; b += g.groups * kBlock) g.histo[row * kLongBins + b] = 0;
  const int unit = group * 4 + wave;
  if (unit >= g.units) return;
  const int base = unit * VPT * kWave;
  float z[VPT];
  const bool nan = draw_load<T, VEC, VPT>((const T *)a.z + row * a.stride, (int)a.n, base, z);
  float max = -HUGE_VALF, min = HUGE_VALF;
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    max = fmaxf(max, z[i]);
    if (z[i] > -HUGE_VALF) min = fminf(min, z[i]);
  }
  max = wave_max(max);
  min = wave_min(min);
  const DrawChoice c = draw_choice(a, row);
  int first = INT32_MAX;
  double mass = 0.0;
  if (c.greedy) {
#pragma unroll
    for (int i = VPT - 1; i >= 0; i--)
      if (z[i] == max) first = draw_column<VEC>(base, i);
    first = (int)wave_min((uint32_t)first);
  } else if (draw_kind(c, false, max) == kRowPlain) {
#pragma unroll
    for (int i = 0; i < VPT; i++) mass += draw_weight<false>(z[i], max, c.rate);
    mass = wave_sum(mass);
  }
  const bool any = __any(nan);
  if (lane == 0) g.part[row * g.units + unit] = LongPart{max, min, first, any, mass};
}

// Weights that are worked out together, not each in a branch of its own: one is a chain of 17 steps.
constexpr int kAtOnce = 8;

template <typename T, int VEC, int VPT>
__global__ __launch_bounds__(kBlock) void draw_histo_kernel(DrawArgs a, LongSpace g, int groups)
{
  __shared__ unsigned long long bins[kLongBins];
  const int64_t row = blockIdx.x / groups;
  const int group = blockIdx.x % groups, wave = threadIdx.x / kWave;
  const T *zp = (const T *)a.z + row * a.stride;
  int unit = group * 4 + wave;
  float z[VPT]; // on their way before it is known what the row needs
  if (unit < g.units) draw_load<T, VEC, VPT>(zp, (int)a.n, unit * VPT * kWave, z);
  float max, min, own;
  bool nan;
  draw_row_range(g.part + row * g.units, g.units, &max, &min, &nan, &own);
  const DrawChoice c = draw_choice(a, row);
  const int kind = draw_kind(c, nan, max);
  if (kind != kRowList && kind != kRowNucleus) return;
  for (int b = threadIdx.x; b < kLongBins; b += kBlock) bins[b] = 0;
  __syncthreads();
  const DrawBin<kLongBins> bin(max, min, c.temp);
  const int shift = kind == kRowNucleus ? draw_row_shift(g.part + row * g.units, g.units, VPT * kWave, max, own, c.rate) : 0;
  if (kind == kRowNucleus && group == 0 && threadIdx.x == 0) g.shift[row] = shift;
  while (unit < g.units) {
    if (kind == kRowList) {
#pragma unroll
      for (int i = 0; i < VPT; i++)
        if (z[i] > -HUGE_VALF) atomicAdd(&bins[bin.of(z[i])], 1ull);
    } else {
#pragma unroll
      for (int o = 0; o < VPT; o += kAtOnce) {
        unsigned long long m[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) m[i] = draw_fixed(draw_weight(z[o + i], max, c.rate), shift);
#pragma unroll
        for (int i = 0; i < kAtOnce; i++)
          if (m[i]) atomicAdd(&bins[bin.of(z[o + i])], m[i]);
      }
    }
    unit += groups * 4;
    if (unit < g.units) draw_load<T, VEC, VPT>(zp, (int)a.n, unit * VPT * kWave, z);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kLongBins; b += kBlock)
    if (bins[b]) atomicAdd(&g.histo[row * kLongBins + b], bins[b]);
}

template <typename T, int VEC, int VPT>
__global__ __launch_bounds__(kBlock) void draw_collect_kernel(DrawArgs a, LongSpace g)
{
  __shared__ unsigned long long sums[kBlock / kWave];
  __shared__ LongCell cell;
  const int64_t row = blockIdx.x / g.groups;
  const int tid = threadIdx.x, group = blockIdx.x % g.groups, wave = tid / kWave, lane = tid % kWave;
  constexpr int kUnit = VPT * kWave;
  const int u = group * 4 + wave;
  float z[VPT];
  if (u < g.units) draw_load<T, VEC, VPT>((const T *)a.z + row * a.stride, (int)a.n, u * kUnit, z);
  const int shift = g.shift[row]; // of rows with a nucleus
  float max, min, own;
  bool nan;
  draw_row_range(g.part + row * g.units, g.units, &max, &min, &nan, &own);
  const DrawChoice c = draw_choice(a, row);
  const int kind = draw_kind(c, nan, max);
  if (kind < kRowSums) return;
  int border = kLongBins; // first bin that is listed (nucleus), or first that is not (list)
  bool too_long = false;
  if (kind != kRowSums) {
    constexpr int kRun = kLongBins / kBlock;
    unsigned long long h[kRun], mine = 0;
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      h[i] = g.histo[row * kLongBins + tid * kRun + i];
      mine += h[i];
    }
    unsigned long long in = wave_running(mine);
    if (lane == kWave - 1) sums[wave] = in;
    if (tid == 0) cell = LongCell{kLongBins - 1, 0, 0, 0.0, shift};
    __syncthreads();
    unsigned long long all = 0;
#pragma unroll
    for (int w = 0; w < kBlock / kWave; w++) {
      if (w < wave) in += sums[w];
      all += sums[w];
    }
    const double unit = ldexp(1.0, -shift), target = kind == kRowNucleus ? c.share * ((double)all * unit) : 0.0;
    unsigned long long before = in - mine;
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      const unsigned long long after = before + h[i];
      const bool here = kind == kRowList ? before < (unsigned long long)c.k && after >= (unsigned long long)c.k
                                         : h[i] && ((double)before * unit < target || before == 0) && (double)after * unit >= target;
      if (here) cell = LongCell{tid * kRun + i, kind == kRowList && after > kLongList, before, target, shift};
      before = after;
    }
    if (kind == kRowList && tid == 0 && all < (unsigned long long)c.k) cell.too_long = all > kLongList; // fewer values than k: all
    __syncthreads();
    border = __builtin_amdgcn_readfirstlane(cell.bin);
    too_long = __builtin_amdgcn_readfirstlane(cell.too_long) != 0;
    if (group == 0 && tid == 0) g.cell[row] = cell;
  }
  if (u >= g.units || too_long) return;
  const DrawBin<kLongBins> bin(max, min, c.temp);
  double kept = 0.0;
  int n = 0;
  LongCand *list = g.list + (row * g.units + u) * (kUnit / 2);
#pragma unroll
  for (int v = 0; v < VPT / VEC; v++) {
    int b[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) b[e] = bin.of(z[v * VEC + e]);
    if (kind != kRowList) { // (no branch for each: a weight is a chain of 17 steps)
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        const double w = draw_weight(z[v * VEC + e], max, c.rate);
        kept += (kind == kRowSums || b[e] < border) && w >= c.least ? w : 0.0;
      }
    }
    if (kind == kRowSums) continue;
    bool take[VEC];
    int earlier = 0, total = 0; // of the same columns in lower lanes; of all lanes
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      take[e] = z[v * VEC + e] > -HUGE_VALF && (kind == kRowList ? b[e] <= border : b[e] == border);
      const unsigned long long t = __ballot(take[e]);
      earlier = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(t >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)t, (uint32_t)earlier));
      total += __popcll(t);
    }
    if (total == 0) continue;
#pragma unroll
    for (int e = 0; e < VEC; e++)
      if (take[e]) {
        const int q = n + earlier++;
        if (q < kUnit / 2) list[q] = LongCand{z[v * VEC + e], draw_column<VEC>(u * kUnit, v * VEC + e)};
      }
    n += total;
  }
  kept = wave_sum(kept);
  if (lane == 0) {
    g.kept[row * g.units + u] = kept;
    g.listed[row * g.units + u] = n;
  }
}

// One workgroup of 1024 a row.
template <typename T, int VPT> __global__ __launch_bounds__(1024) void draw_finish_kernel(DrawArgs a, LongSpace g)
{
  constexpr int kThreads = 1024, kUnit = VPT * kWave, kIn = (kUnit + kThreads - 1) / kThreads;
  __shared__ RowShared<kThreads> s;
  __shared__ LongCand list[kLongList];
  __shared__ int from[kLongUnits]; // where a unit's list begins
  __shared__ int chosen;
  __shared__ double left;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const LongPart *part = g.part + row * g.units;
  float max, min, own;
  bool nan;
  draw_row_range(part, g.units, &max, &min, &nan, &own);
  const DrawChoice c = draw_choice(a, row);
  const int kind = draw_kind(c, nan, max);
  if (kind == kRowNothing) {
    if (tid == 0) draw_nothing(a, row);
    return;
  }
  if (kind == kRowGreedy) {
    if (wave == 0) {
      int first = INT32_MAX;
      for (int q = lane; q < g.units; q += kWave)
        if (part[q].max == max && part[q].first < first) first = part[q].first;
      first = (int)wave_min((uint32_t)first);
      if (lane == 0) draw_answer(a, row, first, 0.0);
    }
    return;
  }
  DrawEnd end{~0ull};
  bool whole = false;
  int listed = 0;
  LongCell cell{0, 0, 0, 0.0, 0};
  int shift = 51; // at which kLongList of them stay below 2^63
  if (kind >= kRowList) {
    cell = g.cell[row];
    if (kind == kRowNucleus) shift = __builtin_amdgcn_readfirstlane(cell.shift);
    whole = cell.too_long != 0;
    int mine = 0, in = 0;
    if (!whole) {
      mine = tid < g.units ? g.listed[row * g.units + tid] : 0;
      if (mine > kUnit / 2) mine = kLongList + 1; // the unit's list is too short
      in = (int)wave_running((uint32_t)mine);
      if (lane == kWave - 1) s.quick.i[wave] = (uint32_t)in;
      __syncthreads();
      for (int w = 0; w < kThreads / kWave; w++) {
        if (w < wave) in += (int)s.quick.i[w];
        listed += (int)s.quick.i[w];
      }
      if (tid < g.units) from[tid] = in - mine;
      __syncthreads();
      whole = listed > kLongList;
    }
    if (!whole) { // each thread finds the unit of its entry: the last one that begins at or before it
      for (int i = tid; i < listed; i += kThreads) {
        int lo = 0, hi = g.units - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) / 2;
          if (from[mid] <= i) lo = mid; else hi = mid - 1;
        }
        list[i] = g.list[(row * g.units + lo) * (kUnit / 2) + i - from[lo]];
      }
      __syncthreads();
    }
  }
  if (kind >= kRowList && !whole) {
    constexpr int kList = kLongList / kThreads;
    float z[kList];
    double w[kList];
    auto place_of = [&](int i) { return (wave * kList + i) * kWave + lane; };
    auto at = [&](int i) { return list[place_of(i)].j; };
#pragma unroll
    for (int i = 0; i < kList; i++) {
      z[i] = place_of(i) < listed ? list[place_of(i)].z : -HUGE_VALF;
      w[i] = draw_weight(z[i], max, c.rate);
    }
    if (kind == kRowList && draw_short_narrow<kThreads, kList>(z, w, at, max, min, c, shift, s.quick)) {
#pragma unroll
      for (int i = 0; i < kList; i++)
        if (w[i] < c.least) w[i] = 0.0;
      double total, weight, rest;
      __syncthreads();
      const int place = draw_pick<kThreads, kList, true>(w, c.u, &total, &weight, &rest, s.quick.d);
      if (place >= 0) draw_answer(a, row, list[place].j, log(weight / total));
      return;
    }
    if (kind == kRowNucleus) { // the border lies among the listed, which are one bin of the row: bins within it
      float top = -HUGE_VALF, low = HUGE_VALF;
#pragma unroll
      for (int i = 0; i < kList; i++) {
        top = fmaxf(top, z[i]);
        if (z[i] > -HUGE_VALF) low = fminf(low, z[i]);
      }
      top = wave_max(top);
      low = wave_min(low);
      if (lane == 0) {
        s.quick.f[wave] = top;
        s.quick.g[wave] = low;
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kThreads / kWave; q++) {
        top = fmaxf(top, s.quick.f[q]);
        low = fminf(low, s.quick.g[q]);
      }
      const DrawBin<ShortShared<kThreads>::kBins> bin(top, low, HUGE_VAL);
      int bins[kList];
#pragma unroll
      for (int i = 0; i < kList; i++) bins[i] = bin.of(z[i]);
      whole = !draw_by_mass<kThreads, kList>(z, w, bins, at, cell.above, -1.0, cell.target, shift, s.quick, &end);
      if (whole) end.place = ~0ull;
    } else
      whole = true;
  }
  const T *zp = (const T *)a.z + row * a.stride;
  const int n = (int)a.n;
  if (whole) {
    shift = draw_row_shift(part, g.units, kUnit, max, own, c.rate);
    end = draw_whole<T, kThreads>(a, row, c, max, shift, s.whole);
  }
  // The kept mass of each unit
  auto weight_of = [&](float z, int j) {
    const double w = z > -HUGE_VALF && end.kept(z, j) ? draw_weight(z, max, c.rate) : 0.0;
    return w >= c.least ? w : 0.0;
  };
  double m[1] = {0.0};
  if (whole) {
    for (int q = wave; q < g.units; q += kThreads / kWave) {
      double v = 0.0;
      for (int i = 0; i < VPT; i++) {
        const int j = q * kUnit + i * kWave + lane;
        if (j < n) v += weight_of(draw_finite((float)zp[j]), j);
      }
      v = wave_sum(v);
      if (lane == 0) g.kept[row * g.units + q] = v;
    }
    __threadfence_block();
    __syncthreads();
  }
  if (tid < g.units) {
    if (kind == kRowPlain)
      m[0] = part[tid].mass * draw_weight(part[tid].max, max, c.rate);
    else {
      m[0] = g.kept[row * g.units + tid];
      if (kind == kRowNucleus && !whole)
        for (int q = from[tid], to = tid + 1 < g.units ? from[tid + 1] : listed; q < to; q++) m[0] += weight_of(list[q].z, list[q].j);
    }
  }
  double total = 0.0, weight, rest;
  __syncthreads();
  const int unit = draw_pick<kThreads, 1, true>(m, c.u, &total, &weight, &rest, s.quick.d);
  if (unit >= 0) {
    chosen = unit;
    left = rest;
  }
  __syncthreads();
  // ... and the column in the unit
  const int base = chosen * kUnit;
  const double aim = left;
  double w[kIn];
#pragma unroll
  for (int i = 0; i < kIn; i++) {
    const int q = (wave * kIn + i) * kWave + lane, j = base + q;
    w[i] = q < kUnit && j < n ? weight_of(draw_finite((float)zp[j]), j) : 0.0;
  }
  double ignored;
  const int place = draw_pick<kThreads, kIn, false>(w, aim, &ignored, &weight, &rest, s.quick.d);
  if (place >= 0) draw_answer(a, row, base + place, log(weight / total));
}

// Rows too long for the units: one workgroup a row, whole-row ways only.
template <typename T> __global__ __launch_bounds__(1024) void draw_huge_kernel(DrawArgs a)
{
  constexpr int kThreads = 1024, kWaves = kThreads / kWave;
  __shared__ DrawShared s;
  __shared__ uint32_t first;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, n = (int)a.n;
  const T *zp = (const T *)a.z + row * a.stride;
  const DrawChoice c = draw_choice(a, row);
  float own = -HUGE_VALF, mass = 0.f; // the mass, relative to the largest so far: of up to 2^20 values, a sixteenth too small at worst
  bool nan = false;
  for (int j = tid; j < n; j += kThreads) {
    const float v = (float)zp[j], z = draw_finite(v);
    nan |= v != v;
    if (z > own) {
      mass *= draw_rough(own, z, c.rate);
      own = z;
    }
    mass += draw_rough(z, own, c.rate);
  }
  float max = wave_max(own);
  const bool any = __any(nan);
  if (lane == 0) {
    s.f[wave] = max;
    s.i[wave] = any;
  }
  if (tid == 0) first = 0xffffffffu;
  __syncthreads();
  bool bad = c.bad;
  for (int w = 0; w < kWaves; w++) {
    max = fmaxf(max, s.f[w]);
    bad |= s.i[w] != 0;
  }
  __syncthreads();
  mass = wave_sum(mass * draw_rough(own, max, c.rate));
  if (lane == 0) s.f[wave] = mass;
  __syncthreads();
  mass = 0.f;
  for (int w = 0; w < kWaves; w++) mass += s.f[w];
  const int shift = draw_shift(1.1f * mass);
  if (bad || max == -HUGE_VALF) {
    if (tid == 0) draw_nothing(a, row);
    return;
  }
  if (c.greedy) {
    for (int j = tid; j < n; j += kThreads)
      if (draw_finite((float)zp[j]) == max) {
        atomicMin(&first, (uint32_t)j);
        break;
      }
    __syncthreads();
    if (tid == 0) draw_answer(a, row, first, 0.0);
    return;
  }
  const DrawEnd end = draw_whole<T, kThreads>(a, row, c, max, shift, s);
  auto weight_of = [&](int j) {
    const float z = draw_finite((float)zp[j]);
    const double w = z > -HUGE_VALF && end.kept(z, j) ? draw_weight(z, max, c.rate) : 0.0;
    return w >= c.least ? w : 0.0;
  };
  // Runs of columns, one a wave; then the run in which the kept mass exceeds u of it is cut into runs again.
  int64_t from = 0, to = n;
  double total = 0.0, aim = 0.0;
  for (bool start = true; start || to - from > kWave; start = false) {
    const int64_t run = ((to - from + kWaves - 1) / kWaves + kWave - 1) / kWave * kWave;
    const int64_t lo = from + wave * run < to ? from + wave * run : to, hi = lo + run < to ? lo + run : to;
    double m = 0.0;
    for (int64_t j = lo + lane; j < hi; j += kWave) m += weight_of((int)j);
    m = wave_sum(m);
    __syncthreads();
    if (lane == 0) s.d[wave] = m;
    __syncthreads();
    if (start) {
      for (int w = 0; w < kWaves; w++) total += s.d[w];
      aim = c.u * total;
    }
    int pick = -1;
    double before = 0.0, sum = 0.0;
    for (int w = 0; w < kWaves; w++) {
      const double v = s.d[w];
      if (v > 0.0) {
        pick = w;
        before = sum;
        if (sum + v > aim) break;
      }
      sum += v;
    }
    aim -= before;
    from += pick * run;
    to = from + run < to ? from + run : to;
  }
  if (wave == 0) {
    const double w = lane < to - from ? weight_of((int)from + lane) : 0.0;
    const double m = wave_running(w);
    const unsigned long long over = __ballot(w > 0.0 && m > aim), some = __ballot(w > 0.0);
    const int pick = over ? __ffsll(over) - 1 : 63 - __clzll((long long)some);
    if (lane == pick) draw_answer(a, row, from + lane, log(w / total));
  }
}

} // namespace mhlik
