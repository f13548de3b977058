// mhlik_predict.hpp -- what the kernels of the predictive operators share (mhlik_q8.hpp, mhlik_draw.hpp).
#pragma once

#include <type_traits>

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace mhlik {

constexpr int kBlock = 256; // threads per workgroup (4 waves) unless a kernel says otherwise
constexpr int kWave = 64;

// ---- sums and maxima over a wave with DPP moves (no LDS, a tenth of a shuffle's latency): row_shr 1, 2, 4, 8 scan each 16
// lanes, row_bcast 15 and 31 carry the totals on.  A lane without a source reads the identity.

template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_move(uint32_t v, uint32_t identity)
{
  return (uint32_t)__builtin_amdgcn_update_dpp((int)identity, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_move(float v, float identity)
{
  return __uint_as_float(dpp_move<CTRL, ROWS>(__float_as_uint(v), __float_as_uint(identity)));
}
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned long long dpp_move(unsigned long long v, unsigned long long identity)
{
  const uint32_t lo = dpp_move<CTRL, ROWS>((uint32_t)v, (uint32_t)identity), hi = dpp_move<CTRL, ROWS>((uint32_t)(v >> 32), (uint32_t)(identity >> 32));
  return (unsigned long long)hi << 32 | lo;
}
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_move(double v, double identity)
{
  return __longlong_as_double((long long)dpp_move<CTRL, ROWS>((unsigned long long)__double_as_longlong(v), (unsigned long long)__double_as_longlong(identity)));
}

template <typename V, typename OP> __device__ __forceinline__ V wave_scan(V v, V identity, OP op)
{
  v = op(v, dpp_move<0x111, 0xf>(v, identity));
  v = op(v, dpp_move<0x112, 0xf>(v, identity));
  v = op(v, dpp_move<0x114, 0xf>(v, identity));
  v = op(v, dpp_move<0x118, 0xf>(v, identity));
  v = op(v, dpp_move<0x142, 0xa>(v, identity));
  v = op(v, dpp_move<0x143, 0xc>(v, identity));
  return v;
}

__device__ __forceinline__ uint32_t wave_last(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, kWave - 1); }
__device__ __forceinline__ float wave_last(float v) { return __uint_as_float(wave_last(__float_as_uint(v))); }
__device__ __forceinline__ unsigned long long wave_last(unsigned long long v)
{
  return (unsigned long long)wave_last((uint32_t)(v >> 32)) << 32 | wave_last((uint32_t)v);
}
__device__ __forceinline__ double wave_last(double v)
{
  return __longlong_as_double((long long)wave_last((unsigned long long)__double_as_longlong(v)));
}

// Lane `from`'s value (the same for all lanes).
__device__ __forceinline__ uint32_t wave_lane(uint32_t v, int from) { return (uint32_t)__builtin_amdgcn_readlane((int)v, from); }
__device__ __forceinline__ unsigned long long wave_lane(unsigned long long v, int from)
{
  return (unsigned long long)wave_lane((uint32_t)(v >> 32), from) << 32 | wave_lane((uint32_t)v, from);
}
__device__ __forceinline__ double wave_lane(double v, int from)
{
  return __longlong_as_double((long long)wave_lane((unsigned long long)__double_as_longlong(v), from));
}

// Running sum over the lanes up to and with this one.
template <typename V> __device__ __forceinline__ V wave_running(V v)
{
  return wave_scan(v, (V)0, [](V a, V b) { return a + b; });
}
// Sums over the wave of N values a lane has, N a power of two up to 16: lane l gets that of value l % N.  While there are
// several values, lanes give half of them to a partner and add up the other half: N - 1 exchanges and 6 - log2 N more,
// not 6 N.
template <int N> __device__ __forceinline__ double wave_sums(const double (&w)[N])
{
#if defined(__HIP_DEVICE_COMPILE__)
  const int lane = threadIdx.x % kWave;
  double v[N];
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = w[i];
  auto halve = [&](auto n, auto from) { // the partner agrees in the bits above n, and differs in n (and below, where nothing is decided)
#pragma unroll
    for (int i = 0; i < n.value; i++) {
      const bool upper = lane & n.value;
      v[i] = (upper ? v[i + n.value] : v[i]) + from(upper ? v[i] : v[i + n.value]);
    }
  };
  if constexpr (N >= 16) halve(std::integral_constant<int, 8>{}, [](double x) { return dpp_move<0x140, 0xf>(x, 0.0); }); // lane ^ 15
  if constexpr (N >= 8) halve(std::integral_constant<int, 4>{}, [](double x) { return dpp_move<0x141, 0xf>(x, 0.0); });  // lane ^ 7
  if constexpr (N >= 4) halve(std::integral_constant<int, 2>{}, [](double x) { return dpp_move<0x4e, 0xf>(x, 0.0); });   // lane ^ 2
  if constexpr (N >= 2) halve(std::integral_constant<int, 1>{}, [](double x) { return dpp_move<0xb1, 0xf>(x, 0.0); });   // lane ^ 1
  double s = v[0];
  if constexpr (N < 2) s += dpp_move<0xb1, 0xf>(s, 0.0);
  if constexpr (N < 4) s += dpp_move<0x4e, 0xf>(s, 0.0);
  if constexpr (N < 8) s += dpp_move<0x124, 0xf>(s, 0.0);  // four lanes round in the 16
  if constexpr (N < 16) s += dpp_move<0x128, 0xf>(s, 0.0); // eight
  auto swapped = [](double x, auto swap) { // what two rows of 16, or two halves, have, added up in both
    const auto lo = swap((unsigned)__double2loint(x)), hi = swap((unsigned)__double2hiint(x));
    return __hiloint2double((int)hi[0], (int)lo[0]) + __hiloint2double((int)hi[1], (int)lo[1]);
  };
  s = swapped(s, [](unsigned x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  return swapped(s, [](unsigned x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
#else
  return w[0];
#endif
}
template <typename V> __device__ __forceinline__ V wave_sum(V v) { return wave_last(wave_running(v)); }
__device__ __forceinline__ float wave_max(float v)
{
  return wave_last(wave_scan(v, -HUGE_VALF, [](float a, float b) { return fmaxf(a, b); }));
}
__device__ __forceinline__ float wave_min(float v)
{
  return wave_last(wave_scan(v, HUGE_VALF, [](float a, float b) { return fminf(a, b); }));
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v)
{
  return wave_last(wave_scan(v, 0xffffffffu, [](uint32_t a, uint32_t b) { return a < b ? a : b; }));
}

} // namespace mhlik
