// Launch shapes of the row kernels, shared by their translation units.
#pragma once

#include <climits>
#include <type_traits>

#include "host_common.h"
#include "row_kernels.cuh"

namespace b200 {

// log2 of a group's size; 0 for one scale a row
inline int group_bits(int subchannel) { return subchannel == 32 ? 5 : subchannel == 64 ? 6 : subchannel == 128 ? 7 : subchannel == 256 ? 8 : 0; }

template <int TPR>
inline unsigned row_blocks(long long rows) {
  const long long blocks = (rows + RowPlace<TPR>::kRows - 1) / RowPlace<TPR>::kRows;
  return static_cast<unsigned>(blocks < INT_MAX ? blocks : INT_MAX);
}

// Threads and values a thread for a row.  Many rows: a warp as far as MAX_V groups of eight a lane go, then as few
// threads as that leaves, since what is done once for a row is done by each of them.  Few rows (fewer than would give
// each SM four): as many threads as there are groups of eight, since the time is that of one row.
// Rows that the wide loads cannot take (their length is no multiple of eight, or a tensor does not start on 16 bytes)
// are bound by their many narrow loads whatever the shape is: they have three.
constexpr long long kFewRows = 4 * 148;

template <int MAX_V, typename Fn>
void for_row_shape(long long rows, long long cols, bool wide, Fn&& fn) {
  using std::integral_constant;
  auto shape = [&](auto tpr, auto v) { fn(tpr, v, std::true_type()); };
  if (wide) {
    if (cols <= 256) shape(integral_constant<int, 32>(), integral_constant<int, 1>());
    else if (cols > 16384) shape(integral_constant<int, 512>(), integral_constant<int, 0>());
    else if (rows < kFewRows) {
      if (cols <= 2048) shape(integral_constant<int, 256>(), integral_constant<int, 1>());
      else if (cols <= 4096) shape(integral_constant<int, 512>(), integral_constant<int, 1>());
      else if (cols <= 8192) shape(integral_constant<int, 512>(), integral_constant<int, 2>());
      else shape(integral_constant<int, 512>(), integral_constant<int, 4>());
    } else {
      if (cols <= 512) shape(integral_constant<int, 32>(), integral_constant<int, 2>());
      else if (cols <= 1024) shape(integral_constant<int, 32>(), integral_constant<int, 4>());
      else if (cols <= 2048) shape(integral_constant<int, 256 / MAX_V>(), integral_constant<int, MAX_V>());
      else if (cols <= 4096) shape(integral_constant<int, 512 / MAX_V>(), integral_constant<int, MAX_V>());
      else if (cols <= 8192) shape(integral_constant<int, 1024 / MAX_V>(), integral_constant<int, MAX_V>());
      else shape(integral_constant<int, 2048 / MAX_V>(), integral_constant<int, MAX_V>());
    }
  } else {
    if (cols <= 512) fn(integral_constant<int, 32>(), integral_constant<int, 2>(), std::false_type());
    else if (cols <= 4096) fn(integral_constant<int, 256>(), integral_constant<int, 2>(), std::false_type());
    else fn(integral_constant<int, 512>(), integral_constant<int, 0>(), std::false_type());
  }
}

template <typename Fn>
void for_bool(bool value, Fn&& fn) {
  if (value) fn(std::true_type());
  else fn(std::false_type());
}

inline int launched(const char* what) {
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? 0 : host_fail_cuda(what, err);
}

// layer_norm_quantize for one type of x (norm_quantize.cu, a unit for each)
struct NormQuantizeCall {
  const void *x, *weight, *bias;
  void *codes, *scales;
  long long rows, cols;
  bool weight_f32, wide;
  int bits, subchannel;
  double eps;
  cudaStream_t stream;
};
int launch_norm_quantize_bf16(const NormQuantizeCall& call);
int launch_norm_quantize_f32(const NormQuantizeCall& call);

}  // namespace b200
