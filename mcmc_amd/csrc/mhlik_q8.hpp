// mhlik_q8.hpp -- rows in 8 bits with a power of two for each block of 128
// columns, and the product X.Theta^T of two matrices held that way.
//
// A row of `cols` values is cut into blocks of 128.  Block b holds
//   q_c = e4m3(x_c 2^-k),   k = least integer in [-96, 119] with max|x| <= 448 2^k   (max over the finite values; 0: k = 0)
// one byte per value, columns padded with zeros to whole blocks, and k + 127 as
// one byte per block (four blocks to an aligned word; spare bytes 127).  x 2^-k
// is exact, so a value is rounded ONCE, to nearest even in e4m3 (half a step:
// 2^-4 relative); what exceeds 448 2^119 or is not finite becomes NaN.  k stays
// above -96 so that q 2^k is a normal bfloat16, which the wide product needs.
#pragma once

#include <type_traits>

#include "mhlik_predict.hpp"

namespace mhlik {

constexpr int kQ8Block = 128;     // columns that share a scale
constexpr int kQ8Lane = 8;        // columns a lane packs in the row kernel
constexpr int kQ8MinExp = -96, kQ8MaxExp = 119;

typedef float q8_f4 __attribute__((ext_vector_type(4)));
typedef float q8_f16 __attribute__((ext_vector_type(16)));
typedef int q8_i4 __attribute__((ext_vector_type(4)));
typedef int q8_i8 __attribute__((ext_vector_type(8)));
typedef __bf16 q8_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 q8_b8 __attribute__((ext_vector_type(8)));

__host__ __device__ inline int64_t q8_blocks(int64_t cols) { return (cols + kQ8Block - 1) / kQ8Block; }
__host__ __device__ inline int64_t q8_scale_stride(int64_t cols) { return (q8_blocks(cols) + 3) / 4 * 4; }

// ------------------------------------------------------------ quantization

// The value as a float that rounds to e4m3 as the value itself does.  A double is cut to 24 bits with the last one set
// if anything was lost: comparisons against, and roundings to, fewer bits come out as for the double.
template <typename T> __device__ __forceinline__ float q8_load(T v) { return (float)v; }
template <> __device__ __forceinline__ float q8_load<double>(double v)
{
  const float f = (float)v;
  uint32_t b = __float_as_uint(f);
  b -= fabs((double)f) > fabs(v); // toward zero
  return (double)f < v || (double)f > v ? __uint_as_float(b | 1u) : f;
}

__device__ __forceinline__ float q8_finite_abs(float v)
{
  const float a = fabsf(v);
  return a < __uint_as_float(0x7f800000u) ? a : 0.f; // NaN too: 0
}

// k for the block whose largest finite magnitude is `top`; 448 = 1.75 * 2^8
__device__ __forceinline__ int q8_exponent(float top)
{
  const uint32_t b = __float_as_uint(top);
  if (b == 0) return 0;
  const int k = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return k < kQ8MinExp ? kQ8MinExp : k > kQ8MaxExp ? kQ8MaxExp : k;
}

__device__ __forceinline__ float q8_scaled(float v, float inv)
{
  const float y = v * inv;
  return fabsf(y) <= 448.f ? y : __uint_as_float(0x7fc00000u);
}

__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d)
{
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Values that go to or come from any address of their type in one access: gfx950 takes unaligned ones, an access that
// spans two lines costs one more.
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Q8Run {
  T e[N];
};

// Values of a matrix whose type the kernel learns at run time (the same numbers as MHLIK_T_*).
struct Q8Values {
  const void *x;
  int64_t rs, cs;
  int32_t type; // 1 double, 2 float, 3 bfloat16, 4 half; 0: there are none
};

// Eight values of a row, from column c0; 0 from column n on.
template <typename T> __device__ __forceinline__ void q8_eight(const Q8Values &x, int64_t row, int64_t c0, int64_t n, float (&v)[kQ8Lane])
{
  const T *p = (const T *)x.x + row * x.rs + c0 * x.cs;
  if (x.cs == 1 && c0 + kQ8Lane <= n) {
    const Q8Run<T, kQ8Lane> q = *(const Q8Run<T, kQ8Lane> *)p;
#pragma unroll
    for (int i = 0; i < kQ8Lane; i++) v[i] = q8_load<T>(q.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kQ8Lane; i++) v[i] = c0 + i < n ? q8_load<T>(p[i * x.cs]) : 0.f;
  }
}

__device__ __forceinline__ void q8_eight(const Q8Values &x, int64_t row, int64_t c0, int64_t n, float (&v)[kQ8Lane])
{
  switch (x.type) {
  case 1: return q8_eight<double>(x, row, c0, n, v);
  case 2: return q8_eight<float>(x, row, c0, n, v);
  case 3: return q8_eight<__bf16>(x, row, c0, n, v);
  default: return q8_eight<_Float16>(x, row, c0, n, v);
  }
}

// A block's share of one of 16 lanes: its eight values as bytes, and k.
__device__ __forceinline__ uint2 q8_pack_block(const float (&v)[kQ8Lane], int *k)
{
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kQ8Lane; i++) top = fmaxf(top, q8_finite_abs(v[i]));
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 16));
  *k = q8_exponent(top);
  const float inv = __uint_as_float((uint32_t)(127 - *k) << 23);
  uint2 out;
  out.x = q8_pack4(q8_scaled(v[0], inv), q8_scaled(v[1], inv), q8_scaled(v[2], inv), q8_scaled(v[3], inv));
  out.y = q8_pack4(q8_scaled(v[4], inv), q8_scaled(v[5], inv), q8_scaled(v[6], inv), q8_scaled(v[7], inv));
  return out;
}

// Rows: 16 lanes take one block, 8 consecutive columns a lane (16 bytes of a 16-bit type in one load, 64 of a double in
// four), the block's largest magnitude goes round the 16 lanes in four exchanges.
// Memory bound: cols sizeof(T) bytes read, cols written, nothing kept.
template <typename T>
__global__ __launch_bounds__(kBlock) void q8_rows_kernel(Q8Values x, int64_t units, int64_t cols, uint32_t blocks, uint32_t sstride,
                                                         uint8_t *__restrict__ data, uint8_t *__restrict__ scale)
{
  const int64_t unit = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / 16;
  const int l = threadIdx.x & 15;
  if (unit >= units) return; // whole groups of 16 lanes
  const int64_t row = blocks == 1 ? unit : unit < (int64_t)1 << 32 ? (int64_t)((uint32_t)unit / blocks) : unit / blocks;
  const int64_t blk = unit - row * blocks, c0 = blk * kQ8Block + l * kQ8Lane;
  float v[kQ8Lane];
  q8_eight<T>(x, row, c0, cols, v);
  int k;
  *(uint2 *)(data + row * blocks * kQ8Block + c0) = q8_pack_block(v, &k);
  if (l == 0) {
    uint8_t *s = scale + row * sstride + blk;
    *s = (uint8_t)(k + 127);
    if (blk == blocks - 1)
      for (uint32_t i = blocks; i < sstride; i++) s[i - blk] = 127;
  }
}

// A matrix that lies column by column (the design matrix of the samplers): a lane takes one row of a block, so that 64
// lanes read 64 consecutive values of a column; the 128 values stay in registers between the maximum and the packing.
template <typename T>
__global__ __launch_bounds__(kBlock) void q8_columns_kernel(const T *__restrict__ x, int64_t rows, int64_t cols, int64_t cs,
                                                            uint32_t blocks, uint32_t sstride, uint8_t *__restrict__ data,
                                                            uint8_t *__restrict__ scale)
{
  const int64_t row = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (row >= rows) return;
  constexpr int kAtOnce = 16; // columns whose loads are under way together
  const uint32_t blk = blockIdx.y;
  const int64_t c0 = (int64_t)blk * kQ8Block;
  const int n = cols - c0 < kQ8Block ? (int)(cols - c0) : kQ8Block;
  const T *p = x + row + c0 * cs;
  float v[kQ8Block], top = 0.f;
#pragma unroll
  for (int i = 0; i < kQ8Block; i += kAtOnce) {
    if (i + kAtOnce <= n) {
      T t[kAtOnce];
#pragma unroll
      for (int q = 0; q < kAtOnce; q++) t[q] = p[(i + q) * cs];
#pragma unroll
      for (int q = 0; q < kAtOnce; q++) v[i + q] = q8_load<T>(t[q]);
    } else {
#pragma unroll
      for (int q = 0; q < kAtOnce; q++) v[i + q] = i + q < n ? q8_load<T>(p[(i + q) * cs]) : 0.f;
    }
#pragma unroll
    for (int q = 0; q < kAtOnce; q++) top = fmaxf(top, q8_finite_abs(v[i + q]));
  }
  const int k = q8_exponent(top);
  const float inv = __uint_as_float((uint32_t)(127 - k) << 23);
  q8_i4 *d = (q8_i4 *)(data + (row * blocks + blk) * kQ8Block);
#pragma unroll
  for (int i = 0; i < kQ8Block / 16; i++) {
    q8_i4 o;
#pragma unroll
    for (int j = 0; j < 4; j++)
      o[j] = (int)q8_pack4(q8_scaled(v[i * 16 + j * 4], inv), q8_scaled(v[i * 16 + j * 4 + 1], inv),
                           q8_scaled(v[i * 16 + j * 4 + 2], inv), q8_scaled(v[i * 16 + j * 4 + 3], inv));
    d[i] = o;
  }
  uint8_t *s = scale + row * sstride + blk;
  *s = (uint8_t)(k + 127);
  if (blk == blocks - 1)
    for (uint32_t i = blocks; i < sstride; i++) s[i - blk] = 127;
}

// ----------------------------------------------------------------- product
//
//   C[i][j] = sum_b 2^(kx[i][b] + kw[j][b]) sum_{c in block b} qx[i][c] qw[j][c]
//
// Two ways to multiply, chosen by the type of C:
//   wide   (float C)     the bytes become bfloat16 WITH their scale on the way into the matrix instruction (exact: 4
//                        significant bits), products and sums are float's: 1.3e-7 of the result's norm at 8192 columns.
//   narrow (16-bit C)    the scaled 8-bit matrix instruction, which takes the block's exponents as operands and runs at
//                        twice the rate.  It aligns the products of one step before adding and keeps about 16 bits of
//                        them: 1.6e-5 of the result's norm (measured, the same at 128 and 8192 columns), a
//                        hundredth of what rounding C to bfloat16 costs and a tenth of float16's.
// All 128 columns of a step share their scales, so which column goes to which place of the instruction is free as long
// as both operands agree: a lane's 32 bytes are consecutive.

__device__ __forceinline__ float q8_scale_value(uint32_t code) { return __uint_as_float(code << 23); } // 2^(code - 127)

// bytes 8 s .. 8 s + 7 of a lane's 32, as scaled bfloat16
__device__ __forceinline__ q8_b8 q8_widen(q8_i8 v, int s, float scale)
{
  const q8_b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * s], scale, false);
  const q8_b2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * s], scale, true);
  const q8_b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * s + 1], scale, false);
  const q8_b2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * s + 1], scale, true);
  return q8_b8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <typename T> __device__ __forceinline__ T q8_round(float v) { return (T)v; }

// N (4 or 8) consecutive values of a row of C, of which the first n are there.
template <typename T, int N> __device__ __forceinline__ void q8_store(T *p, const float (&v)[N], int64_t n)
{
  constexpr int kPer = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  Q8Run<T, kPer> f[N / kPer];
#pragma unroll
  for (int i = 0; i < N; i++) f[i / kPer].e[i % kPer] = q8_round<T>(v[i]);
  if (n >= N) {
#pragma unroll
    for (int i = 0; i < N / kPer; i++) *(Q8Run<T, kPer> *)(p + i * kPer) = f[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < n) p[i] = f[i / kPer].e[i % kPer];
  }
}

struct Q8Product {
  const uint8_t *x, *xs, *w, *ws; // data and scales of rows and draws
  int64_t rows, draws;
  int64_t cols;
  int64_t kp;                     // padded columns: bytes per row
  int32_t blocks, sstride;
  void *out;
  int64_t os;                     // row stride of C
};

// Few rows (up to 16 a fragment, RF fragments): what bounds it is reading the draws once.  A wave takes 16 draws and every
// ks-th block of 128 columns; its lanes load 32 consecutive bytes of a draw straight into the instruction's operand, 4
// lanes a block, four blocks ahead of the four being multiplied.  The ks waves of a 16-draw group add up through LDS in
// wave order.  The draws are the instruction's rows, so that a lane ends with four consecutive values of one row of C.
// FROM_VALUES: the rows come as values; each workgroup quantizes all of them into LDS (they are few: up to 16 KB) while
// its first draws are on their way, which saves a kernel and its start.
constexpr int kQ8FewBytes = 16384;

template <typename T, int RF, bool FROM_VALUES>
__global__ __launch_bounds__(512) void q8_skinny_kernel(Q8Product a, Q8Values values, int ks)
{
  __shared__ __align__(16) q8_f4 part[RF == 1 ? 16 : 8 * RF][kWave]; // the rows' bytes and scales first, then the waves' sums
  static_assert(sizeof(part) >= kQ8FewBytes, "room for the rows");
  __shared__ uint8_t codes[FROM_VALUES ? kQ8FewBytes / kQ8Block : 1];
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, r = lane & 15, g = lane >> 4;
  const int kw = wave % ks, nw = blockDim.x / kWave;
  const int64_t j0 = ((int64_t)blockIdx.x * (nw / ks) + wave / ks) * 16;
  const int64_t jr = j0 + r < a.draws ? j0 + r : a.draws - 1; // past the end: the last draw again, not stored
  const uint8_t *w = a.w + jr * a.kp + g * 32, *ws = a.ws + jr * a.sstride;
  constexpr int kAhead = 4;
  q8_i8 wn[kAhead];
  uint32_t sn[kAhead];
  auto fetch = [&](int b0) {
#pragma unroll
    for (int q = 0; q < kAhead; q++) {
      const int b = b0 + q * ks < a.blocks ? b0 + q * ks : a.blocks - 1;
      wn[q] = *(const q8_i8 *)(w + (int64_t)b * kQ8Block);
      sn[q] = ws[b];
    }
  };
  fetch(kw);
  uint8_t *bytes = (uint8_t *)part;
  if (FROM_VALUES) {
    const int l = tid & 15, units = (int)a.rows * a.blocks;
    for (int unit = tid / 16; unit < units; unit += blockDim.x / 16) {
      const int row = unit / a.blocks;
      const int64_t c0 = (int64_t)(unit - row * a.blocks) * kQ8Block + l * kQ8Lane;
      float v[kQ8Lane];
      q8_eight(values, row, c0, a.cols, v);
      int k;
      *(uint2 *)(bytes + unit * kQ8Block + l * kQ8Lane) = q8_pack_block(v, &k);
      if (l == 0) codes[unit] = (uint8_t)(k + 127);
    }
    __syncthreads();
  }
  const uint8_t *x[RF], *xs[RF];
#pragma unroll
  for (int f = 0; f < RF; f++) {
    const int64_t ir = f * 16 + r < a.rows ? f * 16 + r : a.rows - 1;
    x[f] = (FROM_VALUES ? bytes : a.x) + ir * a.kp + g * 32;
    xs[f] = FROM_VALUES ? codes + ir * a.blocks : a.xs + ir * a.sstride;
  }
  q8_f4 acc[RF];
#pragma unroll
  for (int f = 0; f < RF; f++) acc[f] = q8_f4{0.f, 0.f, 0.f, 0.f};
  for (int b0 = kw; b0 < a.blocks; b0 += kAhead * ks) {
    q8_i8 wv[kAhead];
    uint32_t sv[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; q++) {
      wv[q] = wn[q];
      sv[q] = sn[q];
    }
    if (b0 + kAhead * ks < a.blocks) fetch(b0 + kAhead * ks);
#pragma unroll
    for (int q = 0; q < kAhead; q++) {
      const int b = b0 + q * ks;
      if (b >= a.blocks) break;
      q8_i8 xv[RF];
      float xsv[RF];
#pragma unroll
      for (int f = 0; f < RF; f++) {
        xv[f] = *(const q8_i8 *)(x[f] + b * kQ8Block);
        xsv[f] = q8_scale_value(xs[f][b]);
      }
#pragma unroll
      for (int s = 0; s < 4; s++) {
        const q8_b8 wb = q8_widen(wv[q], s, q8_scale_value(sv[q]));
#pragma unroll
        for (int f = 0; f < RF; f++)
          acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb, q8_widen(xv[f], s, xsv[f]), acc[f], 0, 0, 0);
      }
    }
  }
  if (ks > 1) {
    if (FROM_VALUES) __syncthreads(); // the rows have been read
#pragma unroll
    for (int f = 0; f < RF; f++) part[wave * RF + f][lane] = acc[f];
    __syncthreads();
    if (kw) return;
    for (int q = 1; q < ks; q++)
#pragma unroll
      for (int f = 0; f < RF; f++) acc[f] += part[(wave + q) * RF + f][lane];
  }
  const int64_t j = j0 + g * 4;
  if (j >= a.draws) return;
#pragma unroll
  for (int f = 0; f < RF; f++) {
    const int64_t i = f * 16 + r;
    const float v[4] = {acc[f][0], acc[f][1], acc[f][2], acc[f][3]};
    if (i < a.rows) q8_store<T, 4>((T *)a.out + i * a.os + j, v, a.draws - j);
  }
}

// Narrow matrices (one or two blocks of columns: the samplers' own widths), many rows: C's bytes are what there is to
// do.  A wave keeps 64 draws in registers and walks down the rows, 16 at a time, straight from memory into the
// instruction's operand, the next 16 on their way; the four waves of a workgroup take neighbouring draws of the same rows.
// Lane (r, g) holds bytes 16 g and 64 + 16 g of a block, so that four lanes read 64 consecutive bytes.  Fragment f of
// the draws has draw 32 (f / 2) + 8 (i / 4) + 4 (f % 2) + i % 4 as its row i: a lane ends with two runs of eight values
// of a row of C, four lanes with 64 consecutive bytes of a 16-bit type.
template <typename T, bool WIDE, int BLOCKS>
__global__ __launch_bounds__(kBlock) void q8_thin_kernel(Q8Product a, int groups_n, int walk)
{
#if defined(__HIP_DEVICE_COMPILE__)
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;
  const int64_t j0 = (int64_t)(blockIdx.x % groups_n) * 256 + wave * 64;
  const int64_t from = (int64_t)(blockIdx.x / groups_n) * walk;
  const int64_t to = from + walk < a.rows ? from + walk : a.rows;
  if (j0 >= a.draws) return;
  auto fragment = [&](const uint8_t *p) {
    const q8_i4 lo = *(const q8_i4 *)(p + g * 16), hi = *(const q8_i4 *)(p + 64 + g * 16);
    return q8_i8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  q8_i8 wv[BLOCKS][4];
  uint32_t ws[BLOCKS][4];
#pragma unroll
  for (int f = 0; f < 4; f++) {
    int64_t j = j0 + (f >> 1) * 32 + (r >> 2) * 8 + (f & 1) * 4 + (r & 3);
    j = j < a.draws ? j : a.draws - 1;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
      wv[b][f] = fragment(a.w + j * a.kp + b * kQ8Block);
      ws[b][f] = a.ws[j * a.sstride + b];
    }
  }
  constexpr int kDown = BLOCKS == 1 ? 4 : 2; // fragments of rows under way
  q8_i8 xn[kDown][BLOCKS];
  uint32_t sn[kDown][BLOCKS];
  auto fetch = [&](int64_t i0) {
#pragma unroll
    for (int d = 0; d < kDown; d++) {
      const int64_t i = i0 + d * 16 + r < to ? i0 + d * 16 + r : to - 1;
#pragma unroll
      for (int b = 0; b < BLOCKS; b++) {
        xn[d][b] = fragment(a.x + i * a.kp + b * kQ8Block);
        sn[d][b] = a.xs[i * a.sstride + b];
      }
    }
  };
  // WHOLE: the wave's 64 draws are all there.  Rows past the end are the last one again and are stored as such, so that no
  // branch lies between a fetch and its use: the wait for it would be one for the stores as well (one counter for both).
  auto walk_down = [&](auto whole) {
    fetch(from);
    for (int64_t i0 = from; i0 < to; i0 += kDown * 16) {
      q8_i8 xv[kDown][BLOCKS];
      uint32_t xs[kDown][BLOCKS];
#pragma unroll
      for (int d = 0; d < kDown; d++)
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
          xv[d][b] = xn[d][b];
          xs[d][b] = sn[d][b];
        }
      fetch(i0 + kDown * 16);
#pragma unroll
      for (int d = 0; d < kDown; d++) {
        q8_f4 acc[4];
#pragma unroll
        for (int f = 0; f < 4; f++) acc[f] = q8_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
          if (WIDE) {
#pragma unroll
            for (int s = 0; s < 4; s++) {
              const q8_b8 xb = q8_widen(xv[d][b], s, q8_scale_value(xs[d][b]));
#pragma unroll
              for (int f = 0; f < 4; f++)
                acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q8_widen(wv[b][f], s, q8_scale_value(ws[b][f])), xb, acc[f], 0, 0, 0);
            }
          } else {
#pragma unroll
            for (int f = 0; f < 4; f++)
              acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv[b][f], xv[d][b], acc[f], 0, 0, 0, (int)ws[b][f], 0, (int)xs[d][b]);
          }
        }
        const int64_t i = i0 + d * 16 + r < to ? i0 + d * 16 + r : to - 1;
#pragma unroll
        for (int f = 0; f < 4; f += 2) {
          const int64_t j = j0 + (f >> 1) * 32 + g * 8;
          const float v[8] = {acc[f][0], acc[f][1], acc[f][2], acc[f][3], acc[f + 1][0], acc[f + 1][1], acc[f + 1][2], acc[f + 1][3]};
          if (whole.value || j < a.draws) q8_store<T, 8>((T *)a.out + i * a.os + j, v, whole.value ? 8 : a.draws - j);
        }
      }
    }
  };
  if (j0 + 64 <= a.draws)
    walk_down(std::true_type{});
  else
    walk_down(std::false_type{});
#endif
}

// Many rows, many columns: a workgroup of four waves makes a B x B tile of C (256, or 128 where that would leave CUs
// without a tile), a quarter each.  A step of 128 columns of both sides comes straight from memory into LDS, a whole
// line a row (64-byte pieces: 14 TB/s out of the L2s, lines: 24), into one of two buffers.  Registers hold half a step's
// fragments twice, so that LDS is read for the next half while this one is multiplied, one read and one fetch to each
// few matrix instructions.  In the middle of a step all of it has been read: one barrier, and its buffer is fetched into
// again, a whole step before it is needed.
// A ds_read_b128 serves lanes 0-3, 12-15, 20-23, 24-27 (and the like) together: q8_key orders the 16-byte pieces of a row
// so that these 16 lanes touch 16 different places of 256 bytes (SQ_LDS_BANK_CONFLICT: 0).  Fragments are 32 x 32; a
// draws' fragment has draw 16 (a / 2) + 8 g + 4 (a % 2) + e as its row 8 a + 4 g + e, which leaves a lane with runs of
// eight values of a row of C.
// Rows past the end: the last one again, never stored.
__device__ __forceinline__ int q8_key(int row)
{
  const int q = row >> 2;
  return ((row >> 1) & 1) | ((q ^ (q >> 1)) & 3) << 1;
}

// Tiles in the order in which workgroups start, which go to the eight dies in turn: a die has a run of tiles of its own,
// four tile rows of C high, so that its L2 serves each line to several of its 32 CUs.
__device__ __forceinline__ void q8_tile_of(int id, int tiles, int tiles_n, int *tm, int *tn)
{
  const int full = tiles / 8, rest = tiles % 8, die = id % 8;
  const int t = die * full + (die < rest ? die : rest) + id / 8;
  const int run = 4 * tiles_n, first = t / run * 4, tiles_m = tiles / tiles_n;
  const int high = tiles_m - first < 4 ? tiles_m - first : 4, in = t % run;
  *tm = first + in % high;
  *tn = in / high;
}

template <typename T, bool WIDE, int B>
__global__ __launch_bounds__(kBlock, B == 256 ? 1 : 2) void q8_tile_kernel(Q8Product a, int tiles_n, int tiles)
{
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int F = B / 64;                  // fragments of 32 a wave has of either side
  constexpr int kSide = B * kQ8Block, kFetch = B / 32; // bytes; kilobytes a wave fetches of either side
  __shared__ __align__(1024) uint8_t lds[4 * kSide]; // [buffer][rows, draws][B][128]
  const int tid = threadIdx.x, lane = tid % kWave, r = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  int tm, tn;
  q8_tile_of(blockIdx.x, tiles, tiles_n, &tm, &tn);
  const int64_t i0 = (int64_t)tm * B, j0 = (int64_t)tn * B;
  const int wi = (wave >> 1) * (B / 2), wj = (wave & 1) * (B / 2), kp = (int)a.kp;
  const int xlast = (int)(a.rows - i0 < B ? a.rows - i0 : B) - 1, wlast = (int)(a.draws - j0 < B ? a.draws - j0 : B) - 1;
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc((void *)(a.x + i0 * a.kp), 0, (xlast + 1) * kp, 0x00020000);
  const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc((void *)(a.w + j0 * a.kp), 0, (wlast + 1) * kp, 0x00020000);
  const uint8_t *xsp = a.xs + i0 * a.sstride, *wsp = a.ws + j0 * a.sstride;

  int xvo[kFetch], wvo[kFetch]; // eight rows a fetch, eight lanes a row
#pragma unroll
  for (int q = 0; q < kFetch; q++) {
    const int row = (wave * kFetch + q) * 8 + (lane >> 3), piece = ((lane & 7) ^ q8_key(row)) * 16;
    xvo[q] = (row < xlast ? row : xlast) * kp + piece;
    wvo[q] = (row < wlast ? row : wlast) * kp + piece;
  }
  auto fetch = [&](int b) {
    uint8_t *to = lds + (b & 1) * 2 * kSide + wave * kFetch * 1024;
#pragma unroll
    for (int q = 0; q < kFetch; q++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (__attribute__((address_space(3))) void *)(to + q * 1024), 16, xvo[q], b * kQ8Block, 0, 0);
#pragma unroll
    for (int q = 0; q < kFetch; q++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void *)(to + kSide + q * 1024), 16, wvo[q], b * kQ8Block, 0, 0);
  };

  const int wl = (r >> 4) * 16 + ((r >> 2) & 1) * 8 + ((r >> 3) & 1) * 4 + (r & 3); // this lane's draw of a fragment
  int xo[2][2], wo[2][2]; // [half of the step][16-byte piece]
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const int piece = h * 4 + 2 * g + q;
      xo[h][q] = (wi + r) * kQ8Block + (piece ^ q8_key(r)) * 16;
      wo[h][q] = kSide + (wj + wl) * kQ8Block + (piece ^ q8_key(wl)) * 16;
    }
  q8_i8 xv[2][F], wv[2][F];
  auto read = [&](int h, int b) {
    const uint8_t *base = lds + (b & 1) * 2 * kSide;
#pragma unroll
    for (int f = 0; f < F; f++) {
      const q8_i4 lo = *(const q8_i4 *)(base + xo[h][0] + f * 32 * kQ8Block), hi = *(const q8_i4 *)(base + xo[h][1] + f * 32 * kQ8Block);
      xv[h][f] = q8_i8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
#pragma unroll
    for (int f = 0; f < F; f++) {
      const q8_i4 lo = *(const q8_i4 *)(base + wo[h][0] + f * 32 * kQ8Block), hi = *(const q8_i4 *)(base + wo[h][1] + f * 32 * kQ8Block);
      wv[h][f] = q8_i8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  };

  // Scales: one word has four blocks; the next word is loaded two steps before its first use.
  int xso[F], wso[F];
#pragma unroll
  for (int f = 0; f < F; f++) {
    const int i = wi + f * 32 + r, j = wj + f * 32 + wl;
    xso[f] = (i < xlast ? i : xlast) * a.sstride;
    wso[f] = (j < wlast ? j : wlast) * a.sstride;
  }
  uint32_t xs[F], ws[F], xsn[F], wsn[F];
  auto scales = [&](int b) {
#pragma unroll
    for (int f = 0; f < F; f++) {
      xsn[f] = *(const uint32_t *)(xsp + xso[f] + b);
      wsn[f] = *(const uint32_t *)(wsp + wso[f] + b);
    }
  };

  q8_f16 acc[F][F]; // [draws' fragment][rows' fragment]
#pragma unroll
  for (int f = 0; f < F; f++)
#pragma unroll
    for (int h = 0; h < F; h++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[f][h][e] = 0.f;
  auto multiply = [&](int k) {
    if (WIDE) {
#pragma unroll
      for (int s = 0; s < 4; s++) {
        q8_b8 xb[F];
#pragma unroll
        for (int h = 0; h < F; h++) xb[h] = q8_widen(xv[k][h], s, q8_scale_value(xs[h] & 255u));
#pragma unroll
        for (int f = 0; f < F; f++) {
          const q8_b8 wb = q8_widen(wv[k][f], s, q8_scale_value(ws[f] & 255u));
#pragma unroll
          for (int h = 0; h < F; h++) acc[f][h] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb, xb[h], acc[f][h], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int f = 0; f < F; f++)
#pragma unroll
        for (int h = 0; h < F; h++)
          acc[f][h] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[k][f], xv[k][h], acc[f][h], 0, 0, 0, (int)ws[f], 0, (int)xs[h]);
    }
  };
  // For the scheduler: of a half's 4 F reads (and 2 kFetch fetches) an equal share before each of F F groups of products
  constexpr int kGroups = F * F, kReads = 4 * F / kGroups, kFetches = 2 * kFetch / kGroups, kProducts = WIDE ? 4 : 1;

  scales(0);
  fetch(0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (a.blocks > 1) fetch(1);
  read(0, 0);
  auto step = [&](int b, auto more) {
    if ((b & 3) == 0) {
#pragma unroll
      for (int f = 0; f < F; f++) {
        xs[f] = xsn[f];
        ws[f] = wsn[f];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    read(1, b);
    multiply(0);
#pragma unroll
    for (int i = 0; i < kGroups; i++) {
      __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, kProducts, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    // this wave has read all of the step, and has its part of the next; behind the barrier, all waves
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (more.value) {
      if ((b & 3) == 2) scales(b + 2);
      fetch(b + 2);
    }
    read(0, b + 1); // past the last step: what lies there, unused
    multiply(1);
#pragma unroll
    for (int i = 0; i < kGroups; i++) {
      __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
      if (more.value) __builtin_amdgcn_sched_group_barrier(0x20, kFetches, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, kProducts, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < F; f++) {
      xs[f] >>= 8;
      ws[f] >>= 8;
    }
  };
  int b = 0;
  for (; b < a.blocks - 2; b++) step(b, std::true_type{});
  for (; b < a.blocks; b++) step(b, std::false_type{});

#pragma unroll
  for (int h = 0; h < F; h++) {
    const int64_t i = i0 + wi + h * 32 + r;
    if (i >= a.rows) continue;
#pragma unroll
    for (int f = 0; f < F; f++)
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const int64_t j = j0 + wj + f * 32 + q * 16 + g * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = acc[f][h][q * 8 + e];
        if (j < a.draws) q8_store<T, 8>((T *)a.out + i * a.os + j, v, a.draws - j);
      }
  }
#endif
}

} // namespace mhlik
