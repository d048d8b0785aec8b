// Launch shapes of the row kernels, shared by their translation units.
#pragma once

#include <climits>
#include <type_traits>

#include "host_common.h"
#include "row_kernels.cuh"

namespace b200 {

template <int TPR>
inline unsigned row_blocks(long long rows) {
  const long long blocks = (rows + RowPlace<TPR>::kRows - 1) / RowPlace<TPR>::kRows;
  return static_cast<unsigned>(blocks < INT_MAX ? blocks : INT_MAX);
}

// Threads and values a thread for a row: a warp as far as 32 values a lane go (no barrier), then 16 a thread, so
// that two 16-byte loads of bf16 are in flight in every thread, and 32 in the longest rows (512 threads have 128
// registers each, 1024 would have 64 and spill).  Rows that the wide loads cannot take (their length
// is no multiple of eight, or a tensor does not start on 16 bytes) are bound by their many narrow loads whatever the
// shape is: they have three.
template <typename Fn>
void for_row_shape(long long cols, bool wide, Fn&& fn) {
  using std::integral_constant;
  if (wide) {
    if (cols <= 256) fn(integral_constant<int, 32>(), integral_constant<int, 1>(), std::true_type());
    else if (cols <= 512) fn(integral_constant<int, 32>(), integral_constant<int, 2>(), std::true_type());
    else if (cols <= 1024) fn(integral_constant<int, 32>(), integral_constant<int, 4>(), std::true_type());
    else if (cols <= 2048) fn(integral_constant<int, 128>(), integral_constant<int, 2>(), std::true_type());
    else if (cols <= 4096) fn(integral_constant<int, 256>(), integral_constant<int, 2>(), std::true_type());
    else if (cols <= 8192) fn(integral_constant<int, 512>(), integral_constant<int, 2>(), std::true_type());
    else if (cols <= 16384) fn(integral_constant<int, 512>(), integral_constant<int, 4>(), std::true_type());
    else fn(integral_constant<int, 512>(), integral_constant<int, 0>(), std::true_type());
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
