// mhlik_predict.hpp -- what the kernels of the predictive operators share (mhlik_q8.hpp, mhlik_draw.hpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mhlik {

constexpr int kBlock = 256; // threads per workgroup (4 waves) unless a kernel says otherwise
constexpr int kWave = 64;

} // namespace mhlik
