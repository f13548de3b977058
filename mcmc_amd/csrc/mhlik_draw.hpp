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
// numbers (weights to 2^-63 n), so that the order of atomic additions does not matter; the sums u is compared with have
// a fixed shape.
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

// exp((z - max) / T); z = max: 1, also for infinite max; -800 underflows to 0, and fmax takes NaN (-inf * 0) there too
__device__ __forceinline__ double draw_weight(float z, float max, double inv_t)
{
  const double d = z == max ? 0.0 : (double)z - (double)max;
  return z == -HUGE_VALF ? 0.0 : mhlik_exp_fast(fmax(d * inv_t, -800.0));
}

constexpr int kDrawBins = 2048;

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
  double inv_t;
  uint32_t key; // kept: larger keys, and equal ones up to column `last`
  int last;
  __device__ __forceinline__ float at(int j) const { return (float)z[j]; }
  __device__ __forceinline__ bool kept(uint32_t k, int j) const { return k > key || (k == key && j <= last); }
};

// The row's largest value; *bad: it holds a NaN.
template <typename T, int THREADS> __device__ float draw_row_max(const DrawRow<T> &r, DrawShared &s, bool *bad)
{
  float m = -HUGE_VALF;
  bool nan = false;
  for (int j = threadIdx.x; j < r.n; j += THREADS) {
    const float z = r.at(j);
    nan |= z != z;
    m = fmaxf(m, z);
  }
#pragma unroll
  for (int k = 1; k < kWave; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
  const bool any = __any(nan);
  if (threadIdx.x % kWave == 0) {
    s.f[threadIdx.x / kWave] = m;
    s.i[threadIdx.x / kWave] = any;
  }
  __syncthreads();
  *bad = false;
  for (int w = 0; w < THREADS / kWave; w++) {
    m = fmaxf(m, s.f[w]);
    *bad |= s.i[w] != 0;
  }
  __syncthreads();
  return m;
}

// The prefix of the kept order that is needed for `k` values (BY_MASS false) or for `share` of the kept mass (true):
// key and column are narrowed.  The key is found eleven bits at a time from a histogram of the values that share the
// bits found so far.
template <typename T, int THREADS, bool BY_MASS>
__device__ void draw_narrow(DrawRow<T> &r, DrawShared &s, int shift, uint32_t k, double share)
{
  const int tid = threadIdx.x;
  const double unit = ldexp(1.0, -shift);
  uint32_t prefix = 0, above_n = 0;
  unsigned long long above_m = 0;
  double target = 0.0;
  uint32_t equal = 0;
  for (int level = 0; level < 3; level++) {
    const int low = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11, high = low + bits;
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
      const uint32_t bin = (key >> low) & ((1u << bits) - 1);
      atomicAdd(&s.count[bin], 1u);
      if (BY_MASS) {
        const unsigned long long m = (unsigned long long)rint(ldexp(draw_weight(z, r.max, r.inv_t), shift));
        if (m) atomicAdd(&s.mass[bin], m);
      }
    }
    __syncthreads();
    // sums from the top bin down; each thread takes a run of bins
    constexpr int kRun = kDrawBins / THREADS;
    uint32_t cn = 0;
    unsigned long long cm = 0;
    const int top = kDrawBins - 1 - tid * kRun;
    for (int i = 0; i < kRun; i++) {
      cn += s.count[top - i];
      if (BY_MASS) cm += s.mass[top - i];
    }
    uint32_t in = cn;
    unsigned long long im = cm;
    const int lane = tid % kWave;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const uint32_t a = __shfl_up(in, d);
      const unsigned long long b = __shfl_up(im, d);
      if (lane >= d) {
        in += a;
        im += b;
      }
    }
    if (lane == kWave - 1) {
      s.i[tid / kWave] = in;
      s.q[tid / kWave] = im;
    }
    __syncthreads();
    uint32_t bn = above_n;
    unsigned long long bm = above_m, all = 0;
    for (int w = 0; w < THREADS / kWave; w++) {
      if (w < tid / kWave) {
        bn += s.i[w];
        bm += s.q[w];
      }
      all += s.q[w];
    }
    if (BY_MASS && level == 0) target = share * ((double)all * unit);
    // the first bin, from the top, that reaches the aim; the mass may miss it by rounding: then the lowest bin in use
    __syncthreads();
    if (tid == 0) {
      s.i[31] = 0xffffffffu;
      s.i[30] = 0xffffffffu;
    }
    __syncthreads();
    uint32_t n = bn + in - cn;
    unsigned long long m = bm + im - cm;
    for (int i = 0; i < kRun; i++) {
      const uint32_t c = s.count[top - i];
      const unsigned long long w = BY_MASS ? s.mass[top - i] : 0;
      if (c) {
        atomicMin(&s.i[30], (uint32_t)(top - i));
        const bool reach = BY_MASS ? (double)(m + w) * unit >= target : n + c >= k;
        const bool before = BY_MASS ? (double)m * unit >= target && n > 0 : n >= k;
        if (reach && !before) s.i[31] = (uint32_t)(top - i);
      }
      n += c;
      m += w;
    }
    __syncthreads();
    const uint32_t bin = s.i[31] != 0xffffffffu ? s.i[31] : s.i[30];
    // what lies above that bin
    __syncthreads();
    n = bn + in - cn;
    m = bm + im - cm;
    for (int i = 0; i < kRun; i++) {
      if ((uint32_t)(top - i) == bin) {
        s.i[29] = n;
        s.q[29] = m;
        s.i[28] = s.count[bin];
      }
      n += s.count[top - i];
      m += BY_MASS ? s.mass[top - i] : 0;
    }
    __syncthreads();
    above_n = s.i[29];
    above_m = s.q[29];
    equal = s.i[28];
    prefix = prefix << bits | bin;
    __syncthreads();
  }
  // `prefix` is the key now; of its `equal` columns the first `take` are needed
  uint32_t take;
  if (BY_MASS) {
    const double w = draw_weight(draw_value(prefix), r.max, r.inv_t), a = (double)above_m * unit;
    const double c = w > 0.0 ? ceil((target - a) / w) : 1.0;
    take = c < 1.0 ? 1u : c > (double)equal ? equal : (uint32_t)c;
    if (take > 1 && a + (take - 1) * w >= target) take--;
    if (take < equal && a + take * w < target) take++;
  } else {
    take = k - above_n;
  }
  int last = r.n;
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

// One workgroup a row.
template <typename T, int THREADS> __global__ __launch_bounds__(THREADS) void draw_row_kernel(DrawArgs a, int shift)
{
  __shared__ DrawShared s;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  constexpr int kWaves = THREADS / kWave;
  DrawRow<T> r;
  r.z = (const T *)a.z + row * a.stride;
  r.n = (int)a.n;
  const double temp = a.temperature ? (double)a.temperature[row] : a.temperature_all;
  const double share = a.top_p ? (double)a.top_p[row] : a.top_p_all;
  const double least = a.min_p ? (double)a.min_p[row] : a.min_p_all;
  const int k = a.top_k ? a.top_k[row] : a.top_k_all;
  const double u = a.u_is_double ? ((const double *)a.u)[row] : (double)((const float *)a.u)[row];
  bool bad;
  r.max = draw_row_max<T, THREADS>(r, s, &bad);
  // nothing to draw: no weight, or a number that is none
  if (bad || r.max == -HUGE_VALF || !(temp >= 0.0) || share != share || least != least || u != u) {
    if (tid == 0) {
      a.index[row] = -1;
      if (a.logp) a.logp[row] = __uint_as_float(0x7fc00000u);
    }
    return;
  }
  r.key = 0;
  r.last = r.n;
  const bool greedy = temp == 0.0;
  r.inv_t = greedy ? 1.0 : 1.0 / temp;
  if (greedy)
    draw_narrow<T, THREADS, false>(r, s, shift, 1u, 0.0);
  else {
    if (k > 0 && k < r.n) draw_narrow<T, THREADS, false>(r, s, shift, (uint32_t)k, 0.0);
    if (share < 1.0) draw_narrow<T, THREADS, true>(r, s, shift, 0u, share > 0.0 ? share : 0.0);
  }
  const double least1 = least > 1.0 ? 1.0 : least;
  auto weight = [&](int j) {
    const float z = r.at(j);
    if (!r.kept(draw_key(z), j)) return 0.0;
    const double w = draw_weight(z, r.max, r.inv_t);
    return w >= least1 ? w : 0.0;
  };

  // Runs of columns, one a wave; then the run in which the kept mass exceeds u of it is cut into runs again.
  int from = 0, to = r.n;
  double total = 0.0, aim = 0.0;
  for (bool first = true; first || to - from > kWave; first = false) {
    const int run = ((to - from + kWaves - 1) / kWaves + kWave - 1) / kWave * kWave;
    const int lo = from + wave * run < to ? from + wave * run : to, hi = lo + run < to ? lo + run : to;
    double m = 0.0;
    for (int j = lo + lane; j < hi; j += kWave) m += weight(j);
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) m += __shfl_xor(m, d);
    __syncthreads();
    if (lane == 0) s.d[wave] = m;
    __syncthreads();
    if (first) {
      for (int w = 0; w < kWaves; w++) total += s.d[w];
      aim = u * total;
    }
    // the first run that exceeds the aim; if rounding leaves none, the last one with any mass
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
    const double w = lane < to - from ? weight(from + lane) : 0.0;
    double m = w;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const double b = __shfl_up(m, d);
      if (lane >= d) m += b;
    }
    const unsigned long long over = __ballot(w > 0.0 && m > aim), some = __ballot(w > 0.0);
    const int pick = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll(some);
    if (lane == pick) {
      a.index[row] = from + lane;
      if (a.logp) a.logp[row] = greedy ? 0.f : (float)log(w / total);
    }
  }
}

} // namespace mhlik
