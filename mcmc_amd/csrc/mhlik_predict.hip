// mhlik_predict.hip -- C-ABI of the predictive operators (include/mhlik.h, "answers from posterior draws"): checks,
// variant choice and launches of mhlik_q8.hpp and mhlik_draw.hpp.  All data are on the device and stay there; a call
// queues its kernels on the caller's stream, allocates nothing and waits for nothing.
#include "mhlik.h"

#include <hip/hip_runtime.h>

#include <algorithm>

#include "mhlik_draw.hpp"
#include "mhlik_internal.h"
#include "mhlik_q8.hpp"

using namespace mhlik;

namespace {

// A call answers for its own errors: it reads none that other code has left with the runtime (so no hipGetLastError after a
// launch), and takes back those that it reports, so that no later call finds them.
int report(hipError_t e, const char *what, int line)
{
  (void)hipGetLastError();
  return fail_no_ctx(e == hipErrorOutOfMemory ? MHLIK_ENOMEM : MHLIK_EHIP, "%s failed: %s (%s:%d)", what, hipGetErrorString(e), __FILE__, line);
}
#define PCHK(expr)                                                \
  do {                                                            \
    const hipError_t e_ = (expr);                                 \
    if (e_ != hipSuccess) return report(e_, #expr, __LINE__);     \
  } while (0)

template <typename V> struct Given {
  typedef V type; // arguments convert to the kernel's parameters
};
template <typename... P>
hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, typename Given<P>::type... args)
{
  void *at[] = {(void *)&args...};
  return hipLaunchKernel((const void *)kernel, grid, block, at, 0, stream);
}

// The device a call names is current until the call returns; the caller's comes back.
class OnDevice {
public:
  explicit OnDevice(int device)
  {
    err = hipGetDevice(&before);
    if (err == hipSuccess && device >= 0 && device != before) {
      err = hipSetDevice(device);
      changed = err == hipSuccess;
    }
  }
  ~OnDevice()
  {
    if (changed) (void)hipSetDevice(before);
  }
  hipError_t err;

private:
  int before = 0;
  bool changed = false;
};

size_t type_size(int32_t type)
{
  return type == MHLIK_T_F64 ? 8 : type == MHLIK_T_F32 ? 4 : type == MHLIK_T_BF16 || type == MHLIK_T_F16 ? 2 : 0;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// 256 rows of a matrix are reached with 31-bit offsets
constexpr int64_t kMaxCols = (int64_t)1 << 22;
constexpr int64_t kMaxRows = (int64_t)1 << 40;
constexpr int64_t kMaxDraws = (int64_t)1 << 29;
// A launch has fewer than 2^32 threads; larger calls go in parts, one after the other on the stream.
constexpr int64_t kPartRows = (int64_t)1 << 28;     // of a product or a quantization: 4 threads a row at most, or
constexpr int64_t kPartBlocks = (int64_t)1 << 27;   // 16 a block
constexpr int64_t kPartDrawRows = (int64_t)1 << 20; // of a draw: 1024 threads a row
constexpr int64_t kPartWeights = (int64_t)1 << 27;  // of a draw's long rows, which bounds its workspace (0.75 GB)

int check_rows8(const char *what, const void *data, const void *scale, int64_t rows)
{
  if (rows && (!data || !scale)) return fail_no_ctx(MHLIK_EINVAL, "%s: data and scale must not be NULL", what);
  if (!aligned16(data)) return fail_no_ctx(MHLIK_EINVAL, "%s: data must start at a multiple of 16 bytes", what);
  if ((uintptr_t)scale & 3) return fail_no_ctx(MHLIK_EINVAL, "%s: scale must start at a multiple of 4 bytes", what);
  return MHLIK_OK;
}

template <typename T>
int quantize_launch(const T *x, int64_t rows, int64_t cols, int64_t rs, int64_t cs, uint8_t *data, uint8_t *scale, hipStream_t stream)
{
  const int64_t blocks = q8_blocks(cols), sstride = q8_scale_stride(cols);
  // Column by column if columns are contiguous and there are rows enough for a wave's loads to be (a wave of the row
  // kernel would touch 64 lines for 64 values); a single row is both: the row kernel spreads it over more lanes.
  const bool by_column = rs == 1 && cs != 1 && rows >= 16;
  const int64_t part = by_column ? kPartRows : kPartBlocks / blocks; // at least 2^12: blocks <= 2^15
  for (int64_t first = 0; first < rows; first += part) {
    const int64_t n = std::min(part, rows - first);
    const T *from = x + first * rs;
    uint8_t *d = data + first * blocks * kQ8Block, *s = scale + first * sstride;
    if (by_column)
      PCHK(launch(q8_columns_kernel<T>, dim3((unsigned)((n + kBlock - 1) / kBlock), (unsigned)blocks), dim3(kBlock), stream, from, n, cols,
                  cs, (uint32_t)blocks, (uint32_t)sstride, d, s));
    else
      PCHK(launch(q8_rows_kernel<T>, dim3((unsigned)((n * blocks * 16 + kBlock - 1) / kBlock)), dim3(kBlock), stream,
                  Q8Values{from, rs, cs, 0}, n * blocks, cols, (uint32_t)blocks, (uint32_t)sstride, d, s));
  }
  return MHLIK_OK;
}

int quantize(const void *x, int32_t type, int64_t rows, int64_t cols, int64_t rs, int64_t cs, uint8_t *data, uint8_t *scale,
             hipStream_t stream)
{
  switch (type) {
  case MHLIK_T_F64: return quantize_launch((const double *)x, rows, cols, rs, cs, data, scale, stream);
  case MHLIK_T_F32: return quantize_launch((const float *)x, rows, cols, rs, cs, data, scale, stream);
  case MHLIK_T_BF16: return quantize_launch((const __bf16 *)x, rows, cols, rs, cs, data, scale, stream);
  default: return quantize_launch((const _Float16 *)x, rows, cols, rs, cs, data, scale, stream);
  }
}

int check_shape(int64_t rows, int64_t cols)
{
  if (rows < 0 || rows > kMaxRows || cols < 1 || cols > kMaxCols)
    return fail_no_ctx(MHLIK_EINVAL, "need 0 <= rows <= 2^40 and 1 <= cols <= 2^22 (rows=%lld cols=%lld)", (long long)rows, (long long)cols);
  return MHLIK_OK;
}

int check_workspace(const void *space, size_t bytes, size_t need)
{
  if (need && (!space || !aligned16(space) || bytes < need))
    return fail_no_ctx(MHLIK_EINVAL, "workspace: %zu bytes at a multiple of 16 are needed (%zu given)", need, bytes);
  return MHLIK_OK;
}

int check_values(const char *what, const void *x, int32_t type, int64_t rows, int64_t rs, int64_t cs)
{
  if (!type_size(type)) return fail_no_ctx(MHLIK_EINVAL, "%s: unknown element type %d", what, type);
  if (rows && !x) return fail_no_ctx(MHLIK_EINVAL, "%s must not be NULL", what);
  if ((uintptr_t)x % type_size(type)) return fail_no_ctx(MHLIK_EINVAL, "%s: not aligned to its type", what);
  if (rs < 0 || cs < 0) return fail_no_ctx(MHLIK_EINVAL, "%s: strides must not be negative (%lld, %lld)", what, (long long)rs, (long long)cs);
  return MHLIK_OK;
}

// Rows that the few-rows kernel quantizes by itself.
bool few_rows(int64_t rows, int64_t cols) { return rows <= 64 && rows * q8_blocks(cols) * kQ8Block <= kQ8FewBytes; }

size_t product_space(int64_t rows, int64_t cols)
{
  return few_rows(rows, cols) ? 0 : (size_t)rows * (size_t)(q8_blocks(cols) * kQ8Block + q8_scale_stride(cols));
}

// values.type != 0: the rows are those (few_rows says that they are few enough), not a.x
template <typename T> int product_part(const Q8Product &a, const Q8Values &values, hipStream_t stream)
{
  constexpr bool kWide = sizeof(T) == 4;
  // Up to 64 rows a wave keeps all of them beside 16 draws, so that the draws are read once for all rows; more rows go
  // to the tiles, which read the draws once per 128 rows.
  if (a.rows <= 64) {
    const int rf = a.rows <= 16 ? 1 : a.rows <= 32 ? 2 : 4;
    const int64_t groups16 = (a.draws + 15) / 16;
    int ks = 1; // waves that share 16 draws: until the chip's 1024 SIMDs have four each, or a wave's part is two steps
    while (ks < 8 && groups16 * ks < 4096 && a.blocks >= 4 * ks) ks *= 2;
    const int waves = ks < 4 ? 4 : ks;
    const int64_t groups = (groups16 + waves / ks - 1) / (waves / ks);
    const dim3 grid((unsigned)groups), block(waves * kWave);
    if (values.type && rf == 1)
      PCHK(launch((q8_skinny_kernel<T, 1, true>), grid, block, stream, a, values, ks));
    else if (values.type && rf == 2)
      PCHK(launch((q8_skinny_kernel<T, 2, true>), grid, block, stream, a, values, ks));
    else if (values.type)
      PCHK(launch((q8_skinny_kernel<T, 4, true>), grid, block, stream, a, values, ks));
    else if (rf == 1)
      PCHK(launch((q8_skinny_kernel<T, 1, false>), grid, block, stream, a, values, ks));
    else if (rf == 2)
      PCHK(launch((q8_skinny_kernel<T, 2, false>), grid, block, stream, a, values, ks));
    else
      PCHK(launch((q8_skinny_kernel<T, 4, false>), grid, block, stream, a, values, ks));
  } else if (a.blocks <= 2) {
    const int64_t high = kBlock / kWave * 16 * q8_thin_down(a.blocks, sizeof(T)), gm = (a.rows + high - 1) / high;
    const int64_t chunks = (a.draws + kQ8ThinDraws - 1) / kQ8ThinDraws;
    // Splits of the draws.  The chip takes 512 workgroups at once: no more than that if a whole number of splits comes
    // near it (16-bit C, 10000 x 10000: 39 us, with twice as many 43; 110000 x 4000, no split: 194, three: 231), else at
    // least 1024, so that the last ones do not leave half the chip idle (float C, 50000 x 5600: 227 us, 391 workgroups 281).
    const int64_t once = sizeof(T) == 2 ? 512 : 256;
    int64_t splits = std::min(chunks, gm <= once ? 512 / gm : (1023 + gm) / gm);
    const int64_t each = (chunks + splits - 1) / splits;
    splits = (chunks + each - 1) / each;
    const dim3 grid((unsigned)(gm * splits));
    const bool shifted = !aligned16(a.out) || a.os * (int64_t)sizeof(T) % 16 != 0; // rows that do not begin at 16 bytes
    if (a.blocks == 1 && !shifted)
      PCHK(launch((q8_thin_kernel<T, kWide, 1, false>), grid, dim3(kBlock), stream, a, (int)splits, (int)each));
    else if (a.blocks == 1)
      PCHK(launch((q8_thin_kernel<T, kWide, 1, true>), grid, dim3(kBlock), stream, a, (int)splits, (int)each));
    else if (!shifted)
      PCHK(launch((q8_thin_kernel<T, kWide, 2, false>), grid, dim3(kBlock), stream, a, (int)splits, (int)each));
    else
      PCHK(launch((q8_thin_kernel<T, kWide, 2, true>), grid, dim3(kBlock), stream, a, (int)splits, (int)each));
  } else {
    // Tiles of 256 do a quarter of the fetching per product that tiles of 64 would, and half of what tiles of 128 do; from
    // where they fill three quarters of the chip's 256 CUs they are the faster ones.
    const int64_t big = ((a.rows + 255) / 256) * ((a.draws + 255) / 256);
    const int64_t side = big >= 192 ? 256 : 128, tm = (a.rows + side - 1) / side, tn = (a.draws + side - 1) / side;
    if (tm * tn >= (int64_t)1 << 24) // 10^12 results
      return fail_no_ctx(MHLIK_EINVAL, "too large a product (%lld x %lld)", (long long)a.rows, (long long)a.draws);
    const dim3 grid((unsigned)(tm * tn));
    if (side == 256)
      PCHK(launch((q8_tile_kernel<T, kWide, 256>), grid, dim3(kBlock), stream, a, (int)tn, (int)(tm * tn)));
    else
      PCHK(launch((q8_tile_kernel<T, kWide, 128>), grid, dim3(kBlock), stream, a, (int)tn, (int)(tm * tn)));
  }
  return MHLIK_OK;
}

template <typename T> int product_launch(Q8Product a, const Q8Values &values, hipStream_t stream)
{
  const int64_t rows = a.rows;
  for (int64_t left = rows; left > 0; left -= kPartRows) {
    a.rows = std::min(left, kPartRows);
    if (int rc = product_part<T>(a, values, stream)) return rc;
    a.x += a.rows * a.kp; // (more than one part has 8-bit rows)
    a.xs += a.rows * a.sstride;
    a.out = (T *)a.out + a.rows * a.os;
  }
  return MHLIK_OK;
}

// How a batch of rows is drawn from.
struct DrawPlan {
  int vpt = 0;     // long rows: values a lane of a unit holds; 0: rows that fit a workgroup, or too long for units
  bool short_rows = false;
  LongSpace space;
  size_t bytes = 0;
  int64_t part = 0; // rows at a time
};

constexpr int kShortMax = 8192;  // columns that fit a workgroup's registers (1024 threads, 8 each)
constexpr int64_t kLongVpt = 32; // a unit: 2048 columns; 1024 where those would not give the 1024 SIMDs two each

DrawPlan draw_plan(int64_t rows, int64_t n, void *workspace)
{
  DrawPlan p;
  p.short_rows = n <= kShortMax;
  p.part = kPartDrawRows;
  if (p.short_rows) return p;
  if (n <= kLongVpt * kWave * kLongUnits) rows = p.part = std::min(rows, std::max<int64_t>(1, kPartWeights / n));
  p.vpt = rows * ((n + kLongVpt * kWave - 1) / (kLongVpt * kWave)) < 2048 && n <= (int64_t)16 * kWave * kLongUnits ? 16 : kLongVpt;
  const int64_t unit = p.vpt * kWave, units = (n + unit - 1) / unit;
  if (units > kLongUnits) {
    p.vpt = 0;
    return p;
  }
  LongSpace &g = p.space;
  g.units = (int)units;
  g.groups = (int)((units + 3) / 4);
  uint8_t *at = (uint8_t *)workspace;
  auto take = [&](size_t bytes) {
    uint8_t *q = at ? at + p.bytes : nullptr;
    p.bytes += (bytes + 63) / 64 * 64;
    return q;
  };
  g.part = (LongPart *)take(sizeof(LongPart) * rows * units);
  g.kept = (double *)take(sizeof(double) * rows * units);
  g.listed = (int *)take(sizeof(int) * rows * units);
  g.histo = (unsigned long long *)take(sizeof(unsigned long long) * rows * kLongBins);
  g.cell = (LongCell *)take(sizeof(LongCell) * rows);
  g.shift = (int *)take(sizeof(int) * rows);
  g.list = (LongCand *)take(sizeof(LongCand) * rows * units * (unit / 2));
  return p;
}

template <typename T, int VEC, int VPT> int draw_long(const DrawArgs &a, const LongSpace &g, bool histo, bool collect, hipStream_t stream)
{
  const dim3 grid((unsigned)(a.rows * g.groups));
  PCHK(launch((draw_top_kernel<T, VEC, VPT>), grid, dim3(kBlock), stream, a, g, (int)histo));
  if (histo) { // a workgroup's histogram is added to the row's at the end: no more workgroups than fill the chip four times
    int groups = g.groups;
    while (groups > 1 && a.rows * groups > 1024) groups = (groups + 1) / 2;
    PCHK(launch((draw_histo_kernel<T, VEC, VPT>), dim3((unsigned)(a.rows * groups)), dim3(kBlock), stream, a, g, groups));
  }
  if (collect) PCHK(launch((draw_collect_kernel<T, VEC, VPT>), grid, dim3(kBlock), stream, a, g));
  PCHK(launch((draw_finish_kernel<T, VPT>), dim3((unsigned)a.rows), dim3(1024), stream, a, g));
  return MHLIK_OK;
}

template <typename T> int draw_part(const DrawArgs &a, const DrawPlan &p, hipStream_t stream)
{
  if (p.short_rows) {
    const int shift = a.n <= 4096 ? 51 : 50; // weights in whole numbers: n of them, of 1 at most, stay below 2^63
    // Many rows: few waves a row, since a wave's own cost (scans, the border) adds up (top-k, top-p and min-p, 4096 rows:
    // of 2000, 4 waves 28 us, 8 waves 41; of 400, 1 wave 11 us, 4 waves 20; 512 rows are about even).  Few rows: as many
    // waves as there is work for, which shortens a row's chain of steps (1 row of 1000: 8 waves 7.1 us, 4 waves 8.4).
    const dim3 grid((unsigned)a.rows);
    const bool many = a.rows >= 512;
    if (many && a.n <= 128)
      PCHK(launch((draw_short_kernel<T, 64, 2>), grid, dim3(64), stream, a, shift));
    else if (many && a.n <= 512)
      PCHK(launch((draw_short_kernel<T, 64, 8>), grid, dim3(64), stream, a, shift));
    else if (a.n <= 512)
      PCHK(launch((draw_short_kernel<T, 256, 2>), grid, dim3(256), stream, a, shift));
    else if (many && a.n <= 2048)
      PCHK(launch((draw_short_kernel<T, 256, 8>), grid, dim3(256), stream, a, shift));
    else if (a.n <= 2048)
      PCHK(launch((draw_short_kernel<T, 512, 4>), grid, dim3(512), stream, a, shift));
    else if (many)
      PCHK(launch((draw_short_kernel<T, 512, 16>), grid, dim3(512), stream, a, shift));
    else
      PCHK(launch((draw_short_kernel<T, 1024, 8>), grid, dim3(1024), stream, a, shift));
  } else if (!p.vpt) {
    PCHK(launch(draw_huge_kernel<T>, dim3((unsigned)a.rows), dim3(1024), stream, a));
  } else {
    const bool histo = a.top_k || a.top_p || (a.top_k_all > 0 && a.top_k_all < a.n) || a.top_p_all < 1.0;
    const bool collect = histo || a.min_p || a.min_p_all > 0.0;
    constexpr int kVec = 16 / sizeof(T);
    return p.vpt == 16 ? draw_long<T, kVec, 16>(a, p.space, histo, collect, stream) : draw_long<T, kVec, kLongVpt>(a, p.space, histo, collect, stream);
  }
  return MHLIK_OK;
}

template <typename T> int draw_launch(DrawArgs a, const DrawPlan &p, hipStream_t stream)
{
  for (int64_t left = a.rows; left > 0; left -= p.part) {
    const int64_t rows = a.rows = std::min(left, p.part);
    if (int rc = draw_part<T>(a, p, stream)) return rc;
    a.z = (const T *)a.z + rows * a.stride;
    a.u = (const char *)a.u + rows * (a.u_is_double ? 8 : 4);
    if (a.temperature) a.temperature += rows;
    if (a.top_k) a.top_k += rows;
    if (a.top_p) a.top_p += rows;
    if (a.min_p) a.min_p += rows;
    a.index += rows;
    if (a.logp) a.logp += rows;
  }
  return MHLIK_OK;
}

int check_draw_shape(int64_t rows, int64_t n)
{
  if (rows < 0 || rows > INT32_MAX || n < 1 || n >= (int64_t)1 << 30)
    return fail_no_ctx(MHLIK_EINVAL, "need 0 <= rows < 2^31 and 1 <= n < 2^30 (rows=%lld n=%lld)", (long long)rows, (long long)n);
  return MHLIK_OK;
}

} // namespace

extern "C" {

int mhlik_q8_quantize(const void *x, int32_t type, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride, uint8_t *data,
                      uint8_t *scale, int32_t device, void *stream)
{
  if (int rc = check_shape(rows, cols)) return rc;
  if (int rc = check_values("x", x, type, rows, row_stride, col_stride)) return rc;
  if (int rc = check_rows8("output", data, scale, rows)) return rc;
  if (rows == 0) return MHLIK_OK;
  OnDevice on(device);
  PCHK(on.err);
  return quantize(x, type, rows, cols, row_stride, col_stride, data, scale, (hipStream_t)stream);
}

int mhlik_q8_product_workspace(int64_t rows, int64_t cols, size_t *bytes)
{
  if (!bytes) return fail_no_ctx(MHLIK_EINVAL, "bytes must not be NULL");
  if (int rc = check_shape(rows, cols)) return rc;
  *bytes = product_space(rows, cols);
  return MHLIK_OK;
}

int mhlik_q8_product(const mhlik_q8_operands *p, int32_t device, void *stream)
{
  if (!p) return fail_no_ctx(MHLIK_EINVAL, "operands must not be NULL");
  if (int rc = check_shape(p->rows, p->cols)) return rc;
  if (p->draws < 0 || p->draws > kMaxDraws) return fail_no_ctx(MHLIK_EINVAL, "need 0 <= rows <= 2^40 and 0 <= draws <= 2^29 (draws=%lld)", (long long)p->draws);
  if (int rc = check_rows8("w", p->w_data, p->w_scale, p->draws)) return rc;
  const bool ready = p->x_type == MHLIK_T_Q8;
  if (ready) {
    if (int rc = check_rows8("x", p->x, p->x_scale, p->rows)) return rc;
  } else {
    if (int rc = check_values("x", p->x, p->x_type, p->rows, p->x_row_stride, p->x_col_stride)) return rc;
  }
  if (p->out_type != MHLIK_T_F32 && p->out_type != MHLIK_T_BF16 && p->out_type != MHLIK_T_F16)
    return fail_no_ctx(MHLIK_EINVAL, "out: unknown element type %d", p->out_type);
  if (p->rows == 0 || p->draws == 0) return MHLIK_OK;
  if (!p->out || (uintptr_t)p->out % type_size(p->out_type)) return fail_no_ctx(MHLIK_EINVAL, "out is NULL or not aligned to its type");
  if (p->out_stride < p->draws)
    return fail_no_ctx(MHLIK_EINVAL, "out_stride=%lld is less than draws=%lld", (long long)p->out_stride, (long long)p->draws);
  if (!ready) {
    if (int rc = check_workspace(p->workspace, p->workspace_bytes, product_space(p->rows, p->cols))) return rc;
  }
  OnDevice on(device);
  PCHK(on.err);
  Q8Product a;
  a.rows = p->rows;
  a.draws = p->draws;
  a.blocks = (int32_t)q8_blocks(p->cols);
  a.cols = p->cols;
  a.kp = (int64_t)a.blocks * kQ8Block;
  a.sstride = (int32_t)q8_scale_stride(p->cols);
  a.w = p->w_data;
  a.ws = p->w_scale;
  a.out = p->out;
  a.os = p->out_stride;
  Q8Values values = {nullptr, 0, 0, MHLIK_T_Q8};
  if (ready) {
    a.x = (const uint8_t *)p->x;
    a.xs = p->x_scale;
  } else if (few_rows(p->rows, p->cols)) {
    values = Q8Values{p->x, p->x_row_stride, p->x_col_stride, p->x_type};
    a.x = a.xs = nullptr;
  } else {
    uint8_t *data = (uint8_t *)p->workspace, *scale = data + p->rows * a.kp;
    if (int rc = quantize(p->x, p->x_type, p->rows, p->cols, p->x_row_stride, p->x_col_stride, data, scale, (hipStream_t)stream)) return rc;
    a.x = data;
    a.xs = scale;
  }
  switch (p->out_type) {
  case MHLIK_T_F32: return product_launch<float>(a, values, (hipStream_t)stream);
  case MHLIK_T_BF16: return product_launch<__bf16>(a, values, (hipStream_t)stream);
  default: return product_launch<_Float16>(a, values, (hipStream_t)stream);
  }
}

int mhlik_draw_workspace(int64_t rows, int64_t n, size_t *bytes)
{
  if (!bytes) return fail_no_ctx(MHLIK_EINVAL, "bytes must not be NULL");
  if (int rc = check_draw_shape(rows, n)) return rc;
  *bytes = draw_plan(rows, n, nullptr).bytes;
  return MHLIK_OK;
}

int mhlik_draw(const mhlik_draw_rows *p, int32_t device, void *stream)
{
  if (!p) return fail_no_ctx(MHLIK_EINVAL, "rows must not be NULL");
  if (int rc = check_draw_shape(p->rows, p->n)) return rc;
  if (p->z_type != MHLIK_T_F32 && p->z_type != MHLIK_T_BF16 && p->z_type != MHLIK_T_F16)
    return fail_no_ctx(MHLIK_EINVAL, "z: unknown element type %d", p->z_type);
  if (p->u_type != MHLIK_T_F64 && p->u_type != MHLIK_T_F32) return fail_no_ctx(MHLIK_EINVAL, "u: unknown element type %d", p->u_type);
  if (int rc = check_values("z", p->z, p->z_type, p->rows, p->stride, 0)) return rc;
  if (p->rows && (!p->u || !p->index)) return fail_no_ctx(MHLIK_EINVAL, "u and index must not be NULL");
  if (!p->temperature && !(p->temperature_all == 0.0 || (p->temperature_all >= 1e-100 && p->temperature_all <= HUGE_VAL)))
    return fail_no_ctx(MHLIK_EINVAL, "the temperature is 0 (the largest weight) or at least 1e-100 (%g)", p->temperature_all);
  if (!p->top_p && p->top_p_all != p->top_p_all) return fail_no_ctx(MHLIK_EINVAL, "top_p is not a number");
  if (!p->min_p && p->min_p_all != p->min_p_all) return fail_no_ctx(MHLIK_EINVAL, "min_p is not a number");
  if (p->rows == 0) return MHLIK_OK;
  const DrawPlan plan = draw_plan(p->rows, p->n, p->workspace);
  if (int rc = check_workspace(p->workspace, p->workspace_bytes, plan.bytes)) return rc;
  OnDevice on(device);
  PCHK(on.err);
  DrawArgs a;
  a.z = p->z;
  a.rows = p->rows;
  a.n = p->n;
  a.stride = p->stride;
  a.u = p->u;
  a.u_is_double = p->u_type == MHLIK_T_F64;
  a.temperature = p->temperature;
  a.top_k = p->top_k;
  a.top_p = p->top_p;
  a.min_p = p->min_p;
  a.temperature_all = p->temperature_all;
  a.top_k_all = p->top_k_all;
  a.top_p_all = p->top_p_all;
  a.min_p_all = p->min_p_all;
  a.index = p->index;
  a.logp = p->logp;
  switch (p->z_type) {
  case MHLIK_T_F32: return draw_launch<float>(a, plan, (hipStream_t)stream);
  case MHLIK_T_BF16: return draw_launch<__bf16>(a, plan, (hipStream_t)stream);
  default: return draw_launch<_Float16>(a, plan, (hipStream_t)stream);
  }
}
}
