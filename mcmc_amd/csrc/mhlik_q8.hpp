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
// Memory bound: cols sizeof(T) bytes read, cols written, nothing kept: 8192 x 4096 bfloat16 19.6 us, 5.1 TB/s; 200000 x 64
// float 17.5 us, 4.4 TB/s (four blocks a group of lanes: 29 and 25 us).
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
// Memory bound: 1000003 x 64 double 134 us, 4.3 TB/s (before 16 loads were under way together: 262).
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
//                        them: 1.5e-5 to 1.6e-5 of the result's norm with random signs, without a bias (measured, 64
//                        to 8192 columns), 1e-6 with equal ones; a hundredth of what rounding C to bfloat16 costs and
//                        a tenth of float16's, of whose values one in fifteen gets another last bit.  The few-rows
//                        kernel is bound by reading the draws and multiplies the wide way whatever C's type.
// All 128 columns of a step share their scales, so which column goes to which place of the instruction is free as long
// as both operands agree.

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

// A lane's 32 bytes of a block: pieces g and 4 + g, 16 bytes each (four lanes read 64 consecutive bytes at a time).
__device__ __forceinline__ q8_i8 q8_pieces(const uint8_t *block, int g)
{
  const q8_i4 lo = *(const q8_i4 *)(block + g * 16), hi = *(const q8_i4 *)(block + 64 + g * 16);
  return q8_i8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
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

// A workgroup's units (blocks of rows, row by row) to bytes and scales in LDS, 16 lanes a unit, the loads of a few of them
// under way together.
template <typename T>
__device__ __forceinline__ void q8_pack_units(const Q8Values &x, int units, int blocks, int64_t cols, uint8_t *bytes, uint8_t *codes)
{
  constexpr int kAtOnce = 4;
  const int l = threadIdx.x & 15, step = blockDim.x / 16;
#pragma unroll 1
  for (int u0 = threadIdx.x / 16; u0 < units; u0 += step * kAtOnce) {
    float v[kAtOnce][kQ8Lane];
#pragma unroll
    for (int q = 0; q < kAtOnce; q++) {
      const int unit = u0 + q * step, row = unit / blocks;
      if (unit < units) q8_eight<T>(x, row, (int64_t)(unit - row * blocks) * kQ8Block + l * kQ8Lane, cols, v[q]);
    }
#pragma unroll
    for (int q = 0; q < kAtOnce; q++) {
      const int unit = u0 + q * step;
      if (unit < units) { // whole groups of 16 lanes
        int k;
        *(uint2 *)(bytes + unit * kQ8Block + l * kQ8Lane) = q8_pack_block(v[q], &k);
        if (l == 0) codes[unit] = (uint8_t)(k + 127);
      }
    }
  }
}

// Few rows (up to 16 a fragment, RF fragments): what bounds it is reading the draws once.  A wave takes 16 draws and every
// ks-th block of 128 columns; its lanes load a draw's bytes straight into the instruction's operand, 4 lanes a block, four
// blocks ahead, each into the registers of the one just taken up (1 row x 8192 draws x 8192 in 8 bits: 17.4 us, 3.9 TB/s;
// with registers for four more blocks, so that a SIMD has three waves and not five, 20.9).  The ks waves of a 16-draw group add up through LDS in
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
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, r = lane & 15, g = lane >> 4;
  const int kw = wave % ks, nw = blockDim.x / kWave;
  const int64_t j0 = ((int64_t)blockIdx.x * (nw / ks) + wave / ks) * 16;
  const int64_t jr = j0 + r < a.draws ? j0 + r : a.draws - 1; // past the end: the last draw again, not stored
  const uint8_t *w = a.w + jr * a.kp, *ws = a.ws + jr * a.sstride;
  constexpr int kAhead = 4;
  q8_i8 wn[kAhead];
  uint32_t sn[kAhead];
  auto fetch = [&](int q, int b) {
    wn[q] = q8_pieces(w + (int64_t)b * kQ8Block, g);
    sn[q] = ws[b];
  };
#pragma unroll
  for (int q = 0; q < kAhead; q++)
    if (kw + q * ks < a.blocks) fetch(q, kw + q * ks);
  uint8_t *bytes = (uint8_t *)part;
  if (FROM_VALUES) {
    const int units = (int)a.rows * a.blocks;
    switch (values.type) {
    case 1: q8_pack_units<double>(values, units, a.blocks, a.cols, bytes, codes); break;
    case 2: q8_pack_units<float>(values, units, a.blocks, a.cols, bytes, codes); break;
    case 3: q8_pack_units<__bf16>(values, units, a.blocks, a.cols, bytes, codes); break;
    default: q8_pack_units<_Float16>(values, units, a.blocks, a.cols, bytes, codes); break;
    }
    __syncthreads();
  }
  const uint8_t *x[RF], *xs[RF];
#pragma unroll
  for (int f = 0; f < RF; f++) {
    const int64_t ir = f * 16 + r < a.rows ? f * 16 + r : a.rows - 1;
    x[f] = (FROM_VALUES ? bytes : a.x) + ir * a.kp;
    xs[f] = FROM_VALUES ? codes + ir * a.blocks : a.xs + ir * a.sstride;
  }
  q8_f4 acc[RF];
#pragma unroll
  for (int f = 0; f < RF; f++) acc[f] = q8_f4{0.f, 0.f, 0.f, 0.f};
  for (int b0 = kw; b0 < a.blocks; b0 += kAhead * ks) {
#pragma unroll
    for (int q = 0; q < kAhead; q++) {
      const int b = b0 + q * ks;
      if (b < a.blocks) {
        const q8_i8 wv = wn[q];
        const float wsv = q8_scale_value(sn[q]);
        if (b + kAhead * ks < a.blocks) fetch(q, b + kAhead * ks);
        q8_i8 xv[RF];
        float xsv[RF];
#pragma unroll
        for (int f = 0; f < RF; f++) {
          xv[f] = q8_pieces(x[f] + (int64_t)b * kQ8Block, g);
          xsv[f] = q8_scale_value(xs[f][b]);
        }
#pragma unroll
        for (int s = 0; s < 4; s++) {
          const q8_b8 wb = q8_widen(wv, s, wsv);
#pragma unroll
          for (int f = 0; f < RF; f++)
            acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb, q8_widen(xv[f], s, xsv[f]), acc[f], 0, 0, 0);
        }
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

// Rows of C seldom start at a line of 128 bytes, and stores that end inside lines cost: 200000 rows of 1024 bfloat16 take
// 96 us, rows of 1000 (16 bytes off a line more or less) took 164, of 1025 (2 bytes) 249.  So a lane's pieces of 16 bytes
// are put together anew: brought to 16-byte words of memory (a funnel shift of a piece and the one before it, which the
// lane 16 below has), and a word that belongs to the next line is held back for a step: each pair of stores then writes
// one whole line of each row.  A step is 128 bytes of a row, eight pieces, two to each of the row's four lanes: g and
// 4 + g of a 16-bit type, 2 g and 2 g + 1 of float (as the fragments leave them).
typedef uint32_t q8_u4 __attribute__((ext_vector_type(4)));

// Sixteen bytes of C: the four values of a, or the eight of a and b.
template <typename T> __device__ __forceinline__ q8_u4 q8_word(q8_f4 a, q8_f4 b)
{
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(q8_u4, a);
  } else {
    typedef T Eight __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(q8_u4, Eight{q8_round<T>(a[0]), q8_round<T>(a[1]), q8_round<T>(a[2]), q8_round<T>(a[3]), q8_round<T>(b[0]),
                                           q8_round<T>(b[1]), q8_round<T>(b[2]), q8_round<T>(b[3])});
  }
}

template <typename T> struct Q8RowWriter {
  static constexpr int kWord = 16 / sizeof(T); // values
  typedef q8_u4 Word;
  T *word0;   // the 16-byte word in which the row begins
  int shift;  // bytes of that word before the row
  int len;    // values of the row
  int place[2];
  bool hold[2];
  Word held[2], last; // words held back; the piece before this step's first (shifted rows)

  __device__ __forceinline__ Q8RowWriter() {}
  __device__ __forceinline__ void begin(T *row, int n, int g)
  {
    shift = (int)((uintptr_t)row & 15);
    word0 = row - shift / (int)sizeof(T); // (from the row, so that the compiler still knows it for global memory)
    len = n;
    const int first = (int)((uintptr_t)row >> 4 & 7);
    place[0] = sizeof(T) == 2 ? g : 2 * g;
    place[1] = sizeof(T) == 2 ? 4 + g : 2 * g + 1;
#pragma unroll
    for (int a = 0; a < 2; a++) {
      hold[a] = first + place[a] >= 8;
      held[a] = Word{0, 0, 0, 0};
    }
    last = Word{0, 0, 0, 0};
  }
  // bytes 16 - shift .. 31 - shift of before:piece
  __device__ __forceinline__ Word shifted(Word before, Word piece) const
  {
    const int off = 16 - shift, dw = off >> 2;
    const bool two = dw & 2, one = dw & 1; // dw is 4 only without a shift
    const uint32_t w0 = two ? before[2] : before[0], w1 = two ? before[3] : before[1], w2 = two ? piece[0] : before[2],
                   w3 = two ? piece[1] : before[3], w4 = two ? piece[2] : piece[0], w5 = two ? piece[3] : piece[1];
    const uint32_t x0 = one ? w1 : w0, x1 = one ? w2 : w1, x2 = one ? w3 : w2, x3 = one ? w4 : w3, x4 = one ? w5 : w4;
    const Word o = {__builtin_amdgcn_alignbyte(x1, x0, off & 3), __builtin_amdgcn_alignbyte(x2, x1, off & 3),
                    __builtin_amdgcn_alignbyte(x3, x2, off & 3), __builtin_amdgcn_alignbyte(x4, x3, off & 3)};
    return shift ? o : piece;
  }
  // Step t's two pieces.  SHIFTED: some row does not begin at 16 bytes.  WHOLE: every word of this step lies within the row.
  template <bool WHOLE, bool SHIFTED> __device__ __forceinline__ void step(int t, Word piece0, Word piece1, int g)
  {
    Word word[2] = {piece0, piece1};
    if (SHIFTED) {
      const int from = (((int)threadIdx.x + 48) & 63) * 4;
      Word up0, up1;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        up0[i] = sizeof(T) == 2 ? (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)piece0[i]) : 0u;
        up1[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)piece1[i]);
      }
      const Word before0 = g == 0 ? last : sizeof(T) == 2 ? up0 : up1;
      const Word before1 = sizeof(T) == 2 ? (g == 0 ? up0 : up1) : piece0;
      word[0] = shifted(before0, piece0);
      word[1] = shifted(before1, piece1);
      last = up1;
    }
#pragma unroll
    for (int a = 0; a < 2; a++) {
      const Word o = hold[a] ? held[a] : word[a];
      const int w = (hold[a] ? t - 1 : t) * 8 + place[a];
      held[a] = word[a];
      if (WHOLE) {
        *(Word *)(word0 + w * kWord) = o;
      } else {
        const int e = w * kWord - (SHIFTED ? shift / (int)sizeof(T) : 0);
        if (e >= 0 && e + kWord <= len) {
          *(Word *)(word0 + w * kWord) = o;
        } else if (e > -kWord && e < len) {
          typedef T Values __attribute__((ext_vector_type(kWord)));
          const Values v = __builtin_bit_cast(Values, o);
#pragma unroll
          for (int i = 0; i < kWord; i++)
            if (e + i >= 0 && e + i < len) word0[w * kWord + i] = v[i];
        }
      }
    }
  }
};

// Narrow matrices (one or two blocks of columns: the samplers' own widths), many rows: C's bytes are what there is to
// do.  A wave keeps 64 rows (two blocks: 32) in registers and goes along the draws; a workgroup's four waves have rows
// of their own and share the draws, 128 at a time, in LDS, the next 128 on their way: few loads, since loads queue behind
// the stores (every wave fetching its own draws into registers: 154 us for 200000 x 1024 bfloat16, of which 77 for the
// stores alone, 45 the loads, 35 the products, one after the other; this way 97).
// Lane (r, g) holds pieces g and 4 + g, 16 bytes each, of a row's block.  Fragment f of 64 draws has draw 32 (f / 2) +
// 8 (i / 4) + 4 (f % 2) + i % 4 as its row i: a lane ends with two runs of eight values of a row of C, four lanes with 64
// consecutive bytes of a 16-bit type.  In LDS the pieces of draw d are ordered by a key of d, so that the lanes that a
// ds_read_b128 serves together touch different banks.
constexpr int kQ8ThinDraws = 128;

// Fragments of 16 rows a wave has: as many as leave registers for two waves a SIMD.
__host__ __device__ constexpr int q8_thin_down(int blocks, int size) { return blocks == 1 ? (size == 2 ? 4 : 2) : size == 2 ? 2 : 1; }

template <typename T, bool WIDE, int BLOCKS, bool SHIFTED>
__global__ __launch_bounds__(kBlock, 2) void q8_thin_kernel(Q8Product a, int splits, int chunks)
{
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kDown = q8_thin_down(BLOCKS, (int)sizeof(T)), kN = kQ8ThinDraws; // draws at a time
  constexpr int kSide = kN * kQ8Block;
  // A wave's stores for one chunk of draws.  It writes 16 kDown rows of kN values, a store instruction takes 16 bytes a lane
  // at most: there cannot be fewer, and more would only make the wait that counts them a longer one.
  constexpr int kStores = 16 * kDown * kN * (int)sizeof(T) / (kWave * 16);
  static_assert(kStores < 64, "what a wait can count to");
  __shared__ __align__(1024) uint8_t lds[2][BLOCKS * kSide];
  __shared__ __align__(1024) uint32_t lds_scale[2][kN];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;
  const int64_t i0 = ((int64_t)(blockIdx.x / splits) * (kBlock / kWave) + wave) * kDown * 16;
  const int64_t from = (int64_t)(blockIdx.x % splits) * chunks * kN;
  const int64_t to = from + (int64_t)chunks * kN < a.draws ? from + (int64_t)chunks * kN : a.draws;

  q8_i8 xv[kDown][BLOCKS];
  uint32_t xs[kDown][BLOCKS];
  Q8RowWriter<T> out[kDown];
#pragma unroll
  for (int d = 0; d < kDown; d++) { // rows past the end: the last one again, and stored as such
    const int64_t i = i0 + d * 16 + r < a.rows ? i0 + d * 16 + r : a.rows - 1;
    out[d].begin((T *)a.out + i * a.os + from, (int)(to - from), g);
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
      xv[d][b] = q8_pieces(a.x + i * a.kp + b * kQ8Block, g);
      xs[d][b] = a.xs[i * a.sstride + b];
    }
  }

  auto key = [](int d) { return (d & 3) | ((d >> 3) & 1) << 2; };
  auto fetch = [&](int buf, int64_t j0) { // a wave brings a quarter of the draws, eight draws of a block at once
    const int last = (int)(a.draws - j0 < kN ? a.draws - j0 : kN) - 1, kp = (int)a.kp;
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc((void *)(a.w + j0 * a.kp), 0, (last + 1) * kp, 0x00020000);
#pragma unroll
    for (int q = 0; q < kN / 32; q++) {
      const int d = (wave * (kN / 32) + q) * 8 + (lane >> 3);
      const int at = (d < last ? d : last) * kp + ((lane & 7) ^ key(d)) * 16;
#pragma unroll
      for (int b = 0; b < BLOCKS; b++)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void *)(lds[buf] + b * kSide + (wave * (kN / 32) + q) * 1024), 16, at,
                                                 b * kQ8Block, 0, 0);
    }
    if (wave < kN / kWave) { // the word that holds the scales of a draw's first four blocks
      const __amdgpu_buffer_rsrc_t sr = __builtin_amdgcn_make_buffer_rsrc((void *)(a.ws + j0 * a.sstride), 0, (last + 1) * a.sstride, 0x00020000);
      const int d = wave * kWave + lane;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sr, (__attribute__((address_space(3))) void *)(lds_scale[buf] + wave * kWave), 4, (d < last ? d : last) * a.sstride, 0, 0, 0);
    }
  };

  const int wl = (r >> 2) * 8 + (r & 3); // this lane's draw of fragment 0; the others have the same key
  typedef typename Q8RowWriter<T>::Word Word;
  auto chunk = [&](int buf, int t0, auto whole) {
#pragma unroll 1
    for (int h = 0; h < kN; h += 64) {
      q8_i8 wv[BLOCKS][4];
      uint32_t ws[4];
#pragma unroll
      for (int f = 0; f < 4; f++) {
        const int d = h + (f >> 1) * 32 + (f & 1) * 4 + wl;
        ws[f] = lds_scale[buf][d];
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
          const uint8_t *p = lds[buf] + b * kSide + d * kQ8Block;
          const q8_i4 lo = *(const q8_i4 *)(p + (g ^ key(wl)) * 16), hi = *(const q8_i4 *)(p + ((4 + g) ^ key(wl)) * 16);
          wv[b][f] = q8_i8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
      }
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
                acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q8_widen(wv[b][f], s, q8_scale_value(ws[f] >> (8 * b) & 255u)), xb, acc[f], 0, 0, 0);
            }
          } else {
#pragma unroll
            for (int f = 0; f < 4; f++)
              acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv[b][f], xv[d][b], acc[f], 0, 0, 0, (int)(ws[f] >> (8 * b)), 0, (int)xs[d][b]);
          }
        }
#pragma unroll
        for (int q = 0; q < (int)sizeof(T) / 2; q++) { // 64 values of a row are 16 sizeof(T) words over its four lanes
          const Word p0 = q8_word<T>(acc[sizeof(T) == 2 ? 0 : 2 * q], acc[1]), p1 = q8_word<T>(acc[sizeof(T) == 2 ? 2 : 2 * q + 1], acc[3]);
          const int t = t0 + h * (int)sizeof(T) / 128 + q;
          if (whole.value || (t > 0 && (t + 1) * 8 * Q8RowWriter<T>::kWord <= (int)(to - from))) // the same for all lanes
            out[d].template step<true, SHIFTED>(t, p0, p1, g);
          else
            out[d].template step<false, SHIFTED>(t, p0, p1, g);
        }
      }
    }
  };

  constexpr int kSteps = kN * (int)sizeof(T) / 128; // of the row writers, for one chunk
  fetch(0, from);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int buf = 0, t = 0;
  for (int64_t j0 = from; j0 < to; j0 += kN, buf ^= 1, t += kSteps) {
    const bool more = j0 + kN < to;
    if (more) fetch(buf ^ 1, j0 + kN);
    asm volatile("" ::: "memory"); // the fetch stays ahead of the chunk's stores
    if (t > 0 && j0 + kN <= to)
      chunk(buf, t, std::true_type{});
    else
      chunk(buf, t, std::false_type{});
    if (more) {
      // the fetch is older than this chunk's stores, which need not be waited for (the first chunk's number varies)
      if (t > 0)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kStores) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
    }
  }
#pragma unroll
  for (int d = 0; d < kDown; d++) out[d].template step<false, SHIFTED>(t, Word{0, 0, 0, 0}, Word{0, 0, 0, 0}, g); // what is held
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
// Rows past the end: the last one again, never stored.  Bound by the matrix instructions, of which a wave has one stream
// and nothing beside it when it waits: 8192 x 8192 x 8192 to bfloat16 464 us, 2.37 PFLOP/s; 4096 x 4096 x 4096 to float
// 115 us, 1.19 PFLOP/s; tiles of 128, 2048 x 2048 x 2048 to bfloat16: 16 us, 1.06 PFLOP/s (of 256: 36 us).
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
  // in scalar registers: the buffer descriptors are built from them (from vector registers each load becomes a loop)
  *tm = __builtin_amdgcn_readfirstlane(first + in % high);
  *tn = __builtin_amdgcn_readfirstlane(in / high);
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
