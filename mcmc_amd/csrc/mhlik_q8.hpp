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

#include "mhlik_predict.hpp"

namespace mhlik {

constexpr int kQ8Block = 128;     // columns that share a scale
constexpr int kQ8Lane = 8;        // columns a lane packs in the row kernel
constexpr int kQ8MinExp = -96, kQ8MaxExp = 119;

typedef float q8_f4 __attribute__((ext_vector_type(4)));
typedef int q8_i4 __attribute__((ext_vector_type(4)));
typedef int q8_i8 __attribute__((ext_vector_type(8)));
typedef __bf16 q8_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 q8_b4 __attribute__((ext_vector_type(4)));
typedef __bf16 q8_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 q8_h4 __attribute__((ext_vector_type(4)));

__host__ __device__ inline int64_t q8_blocks(int64_t cols) { return (cols + kQ8Block - 1) / kQ8Block; }
__host__ __device__ inline int64_t q8_scale_stride(int64_t cols) { return (q8_blocks(cols) + 3) / 4 * 4; }

// ------------------------------------------------------------ quantization

// The value as a float that rounds to e4m3 as the value itself does.  A double is cut to 24 bits with the last one set
// if anything was lost: comparisons against, and roundings to, fewer bits come out as for the double.
template <typename T> __device__ __forceinline__ float q8_load(T v) { return (float)v; }
template <> __device__ __forceinline__ float q8_load<double>(double v)
{
  const float f = (float)v;
  if ((double)f == v || v != v || fabs(v) == HUGE_VAL) return f;
  uint32_t b = __float_as_uint(f);
  if (fabs((double)f) > fabs(v)) b--; // toward zero
  return __uint_as_float(b | 1u);
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

// Rows: 16 lanes take one block, 8 consecutive columns a lane (16 bytes of a 16-bit type in one load, 64 of a double in
// four), the block's largest magnitude goes round the 16 lanes in four exchanges.  VEC: every lane's columns start at a
// multiple of 16 bytes and the last block is whole, or else its columns are loaded one by one.
// Memory bound: cols sizeof(T) bytes read, cols written, nothing kept.
template <typename T, bool VEC>
__global__ __launch_bounds__(kBlock) void q8_rows_kernel(const T *__restrict__ x, int64_t units, int64_t cols, int64_t rs,
                                                         int64_t cs, uint32_t blocks, uint32_t sstride,
                                                         uint8_t *__restrict__ data, uint8_t *__restrict__ scale)
{
  const int64_t unit = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / 16;
  const int l = threadIdx.x & 15;
  if (unit >= units) return; // whole groups of 16 lanes
  const int64_t row = blocks == 1 ? unit : unit < (int64_t)1 << 32 ? (int64_t)((uint32_t)unit / blocks) : unit / blocks;
  const int64_t blk = unit - row * blocks;
  const int64_t c0 = blk * kQ8Block + l * kQ8Lane;
  float v[kQ8Lane];
  const T *p = x + row * rs + c0 * (VEC ? 1 : cs);
  if (VEC && c0 + kQ8Lane <= cols) {
    struct alignas(16) Pack { T e[16 / sizeof(T)]; };
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < kQ8Lane / kPer; i++) {
      const Pack q = ((const Pack *)p)[i];
#pragma unroll
      for (int j = 0; j < kPer; j++) v[i * kPer + j] = q8_load<T>(q.e[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kQ8Lane; i++) v[i] = c0 + i < cols ? q8_load<T>(p[i * (VEC ? 1 : cs)]) : 0.f;
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kQ8Lane; i++) top = fmaxf(top, q8_finite_abs(v[i]));
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 16));
  const int k = q8_exponent(top);
  const float inv = __uint_as_float((uint32_t)(127 - k) << 23);
  uint2 out;
  out.x = q8_pack4(q8_scaled(v[0], inv), q8_scaled(v[1], inv), q8_scaled(v[2], inv), q8_scaled(v[3], inv));
  out.y = q8_pack4(q8_scaled(v[4], inv), q8_scaled(v[5], inv), q8_scaled(v[6], inv), q8_scaled(v[7], inv));
  *(uint2 *)(data + row * blocks * kQ8Block + c0) = out;
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
  const uint32_t blk = blockIdx.y;
  const int64_t c0 = (int64_t)blk * kQ8Block;
  const int n = cols - c0 < kQ8Block ? (int)(cols - c0) : kQ8Block;
  const T *p = x + row + c0 * cs;
  float v[kQ8Block];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kQ8Block; i++) {
    v[i] = i < n ? q8_load<T>(p[i * cs]) : 0.f;
    top = fmaxf(top, q8_finite_abs(v[i]));
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

// Four consecutive values of a row of C.
template <typename T> __device__ __forceinline__ void q8_store4(T *p, q8_f4 v, int n, bool aligned)
{
  struct alignas(4 * sizeof(T)) Four { T e[4]; };
  Four f;
#pragma unroll
  for (int i = 0; i < 4; i++) f.e[i] = q8_round<T>(v[i]);
  if (aligned && n >= 4)
    *(Four *)p = f;
  else
    for (int i = 0; i < 4; i++)
      if (i < n) p[i] = f.e[i];
}

struct Q8Product {
  const uint8_t *x, *xs, *w, *ws; // data and scales of rows and draws
  int64_t rows, draws;
  int64_t kp;                     // padded columns: bytes per row
  int32_t blocks, sstride;
  void *out;
  int64_t os;                     // row stride of C
  int32_t aligned;                // rows of C start at a multiple of 4 values' bytes
};

// Few rows (up to 16 a fragment): what bounds it is reading the draws once.  A wave takes 16 draws and every KS-th block
// of 128 columns; its lanes load 32 consecutive bytes of a draw straight into the instruction's operand, 4 lanes a block.
// The KS waves of a 16-draw group add up through LDS in wave order.  The draws are the instruction's rows, so that a
// lane ends with four consecutive values of one row of C.
template <typename T, int RF>
__global__ __launch_bounds__(1024) void q8_skinny_kernel(Q8Product a, int ks)
{
  __shared__ q8_f4 part[16][RF][kWave];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, r = lane & 15, g = lane >> 4;
  const int kw = wave % ks, nw = blockDim.x / kWave;
  const int64_t j0 = ((int64_t)blockIdx.x * (nw / ks) + wave / ks) * 16;
  const int64_t jr = j0 + r < a.draws ? j0 + r : a.draws - 1; // past the end: the last draw again, not stored
  const uint8_t *w = a.w + jr * a.kp + g * 32, *ws = a.ws + jr * a.sstride;
  const int64_t i0 = (int64_t)blockIdx.y * 16 * RF;
  const uint8_t *x[RF], *xs[RF];
#pragma unroll
  for (int f = 0; f < RF; f++) {
    const int64_t ir = i0 + f * 16 + r < a.rows ? i0 + f * 16 + r : a.rows - 1;
    x[f] = a.x + ir * a.kp + g * 32;
    xs[f] = a.xs + ir * a.sstride;
  }
  q8_f4 acc[RF];
#pragma unroll
  for (int f = 0; f < RF; f++) acc[f] = q8_f4{0.f, 0.f, 0.f, 0.f};
  for (int b = kw; b < a.blocks; b += ks) {
    const q8_i8 wv = *(const q8_i8 *)(w + (int64_t)b * kQ8Block);
    const float wsv = q8_scale_value(ws[b]);
    q8_i8 xv[RF];
    float xsv[RF];
#pragma unroll
    for (int f = 0; f < RF; f++) {
      xv[f] = *(const q8_i8 *)(x[f] + (int64_t)b * kQ8Block);
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
  if (ks > 1) {
#pragma unroll
    for (int f = 0; f < RF; f++) part[wave][f][lane] = acc[f];
    __syncthreads();
    if (kw) return;
    for (int q = 1; q < ks; q++)
#pragma unroll
      for (int f = 0; f < RF; f++) acc[f] += part[wave + q][f][lane];
  }
  const int64_t j = j0 + g * 4;
  if (j >= a.draws) return;
  const int n = a.draws - j < 4 ? (int)(a.draws - j) : 4;
#pragma unroll
  for (int f = 0; f < RF; f++) {
    const int64_t i = i0 + f * 16 + r;
    if (i < a.rows) q8_store4<T>((T *)a.out + i * a.os + j, acc[f], n, a.aligned);
  }
}

// Many rows: a workgroup of four waves makes a 128 x 128 tile of C, 64 x 64 a wave.  A step of 128 columns of both sides
// (16 KB each) comes straight from memory into LDS while the step before is multiplied.  A row's eight 16-byte pieces are
// stored in an order that depends on the row, so that the eight lanes that read at a time touch all banks: row r of X has
// piece c at place c ^ (r & 7).  Fragment f of a wave's draws takes the draws 16 (i / 4) + 4 f + i % 4 as its rows i, so
// that a lane ends with 16 CONSECUTIVE values of a row of C over its four fragments; the order key of the draws' rows is
// changed to fit.
constexpr int kQ8Tile = 128;

__device__ __forceinline__ int q8_draw_key(int r) { return (r & 3) | ((r >> 4) & 1) << 2; }

template <typename T, bool WIDE>
__global__ __launch_bounds__(kBlock) void q8_tile_kernel(Q8Product a, int tiles_n)
{
  __shared__ __align__(1024) uint8_t lds[2][2][kQ8Tile * kQ8Block]; // [buffer][rows, draws]
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, r = lane & 15, g = lane >> 4;
  const int64_t i0 = (int64_t)(blockIdx.x / tiles_n) * kQ8Tile, j0 = (int64_t)(blockIdx.x % tiles_n) * kQ8Tile;
  const int wi = (wave & 1) * 64, wj = (wave >> 1) * 64;
  const int64_t xrows = a.rows - i0 < kQ8Tile ? a.rows - i0 : kQ8Tile, wrows = a.draws - j0 < kQ8Tile ? a.draws - j0 : kQ8Tile;
  // rows past the end read as zeros: the descriptors end with the last row
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc((void *)(a.x + i0 * a.kp), 0, (int)(xrows * a.kp), 0x00020000);
  const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc((void *)(a.w + j0 * a.kp), 0, (int)(wrows * a.kp), 0x00020000);
  const int lr = lane >> 3, lp = lane & 7;

  auto fetch = [&](int buf, int b) {
#pragma unroll
    for (int q = 0; q < 4; q++) { // this wave's 32 rows of either side, 8 at a time
      const int row = wave * 32 + q * 8 + lr;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (__attribute__((address_space(3))) void *)(lds[buf][0] + (wave * 32 + q * 8) * kQ8Block), 16,
                                               (int)(row * a.kp) + (lp ^ (row & 7)) * 16, b * kQ8Block, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void *)(lds[buf][1] + (wave * 32 + q * 8) * kQ8Block), 16,
                                               (int)(row * a.kp) + (lp ^ q8_draw_key(row)) * 16, b * kQ8Block, 0, 0);
    }
  };

  // this lane's rows of the fragments; past the end any row's scale will do, its data are zeros
  int xrow[4], wrow[4];
  const uint8_t *xsp[4], *wsp[4];
#pragma unroll
  for (int f = 0; f < 4; f++) {
    xrow[f] = wi + f * 16 + r;
    wrow[f] = wj + (r >> 2) * 16 + f * 4 + (r & 3);
    xsp[f] = a.xs + (i0 + (xrow[f] < xrows ? xrow[f] : xrows - 1)) * a.sstride;
    wsp[f] = a.ws + (j0 + (wrow[f] < wrows ? wrow[f] : wrows - 1)) * a.sstride;
  }
  q8_f4 acc[4][4]; // [draws' fragment][rows' fragment]
#pragma unroll
  for (int f = 0; f < 4; f++)
#pragma unroll
    for (int h = 0; h < 4; h++) acc[f][h] = q8_f4{0.f, 0.f, 0.f, 0.f};

  auto piece = [&](const uint8_t *base, int row, int key) {
    const q8_i4 lo = *(const q8_i4 *)(base + row * kQ8Block + ((2 * g) ^ key) * 16);
    const q8_i4 hi = *(const q8_i4 *)(base + row * kQ8Block + ((2 * g + 1) ^ key) * 16);
    return q8_i8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };

  fetch(0, 0);
  __syncthreads();
  for (int b = 0; b < a.blocks; b++) {
    const int buf = b & 1;
    if (b + 1 < a.blocks) fetch(buf ^ 1, b + 1);
    q8_i8 xv[4], wv[4];
    uint32_t xc[4], wc[4];
#pragma unroll
    for (int f = 0; f < 4; f++) {
      xv[f] = piece(lds[buf][0], xrow[f], xrow[f] & 7);
      wv[f] = piece(lds[buf][1], wrow[f], q8_draw_key(wrow[f]));
      xc[f] = xsp[f][b];
      wc[f] = wsp[f][b];
    }
    if (WIDE) {
#pragma unroll
      for (int s = 0; s < 4; s++) {
        q8_b8 xb[4];
#pragma unroll
        for (int h = 0; h < 4; h++) xb[h] = q8_widen(xv[h], s, q8_scale_value(xc[h]));
#pragma unroll
        for (int f = 0; f < 4; f++) {
          const q8_b8 wb = q8_widen(wv[f], s, q8_scale_value(wc[f]));
#pragma unroll
          for (int h = 0; h < 4; h++) acc[f][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb, xb[h], acc[f][h], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int f = 0; f < 4; f++)
#pragma unroll
        for (int h = 0; h < 4; h++)
          acc[f][h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv[f], xv[h], acc[f][h], 0, 0, 0, (int)wc[f], 0, (int)xc[h]);
    }
    __syncthreads(); // the next step has arrived (the barrier waits for this wave's loads), this one has been read
  }

#pragma unroll
  for (int h = 0; h < 4; h++) {
    const int64_t i = i0 + xrow[h];
    if (i >= a.rows) continue;
#pragma unroll
    for (int f = 0; f < 4; f++) {
      const int64_t j = j0 + wj + g * 16 + f * 4;
      if (j < a.draws) q8_store4<T>((T *)a.out + i * a.os + j, acc[f][h], a.draws - j < 4 ? (int)(a.draws - j) : 4, a.aligned);
    }
  }
}

} // namespace mhlik
