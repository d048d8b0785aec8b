// C entry points of the row kernels: quantize_tokens, layer_norm, layer_norm_quantize, layer_norm_bwd.
#include "../../include/b200_int4_gemms.h"
#include "host_common.h"
#include "row_launch.h"

namespace {

using namespace b200;

// x as bf16 or fp32, weight and bias as bf16 or fp32
template <typename Fn>
void for_types(int x_type, int w_type, Fn&& fn) {
  if (x_type == B200_OUT_BF16 && w_type == B200_OUT_BF16) fn(bf16(), bf16());
  else if (x_type == B200_OUT_BF16) fn(bf16(), float());
  else if (w_type == B200_OUT_BF16) fn(float(), bf16());
  else fn(float(), float());
}

int check_rows(int64_t rows, int64_t cols) {
  if (rows < 0) return host_fail("rows must be non-negative");
  if (cols <= 0) return host_fail("cols must be positive");
  if (cols > INT_MAX) return host_fail("too many columns for one launch");
  return 0;
}

int check_quantisation(int32_t bits, int32_t subchannel) {
  if (bits != 4 && bits != 8) return host_fail("bits must be 4 or 8");
  if (subchannel != 0 && subchannel != 32 && subchannel != 64 && subchannel != 128 && subchannel != 256)
    return host_fail("subchannel must be 0 (one scale a row), 32, 64, 128 or 256");
  return 0;
}

int check_types(int32_t x_type, int32_t w_type) {
  if ((x_type != B200_OUT_BF16 && x_type != B200_OUT_F32) || (w_type != B200_OUT_BF16 && w_type != B200_OUT_F32))
    return host_fail("x and weight types must be bf16 or float32");
  return 0;
}

size_t type_size(int32_t type) { return type == B200_OUT_F32 ? 4 : 2; }

// Natural alignment is a condition of every access; 16 bytes, and rows of a multiple of eight values, are what the
// wide loads need.
int check_alignment(const char* name, const void* p, size_t bytes) {
  if (!is_aligned(p, bytes)) return host_fail(std::string(name) + " is not aligned to its element size");
  return 0;
}

// Blocks of the backward kernel: as many as are resident at once (its launch bounds), one row of partial sums each.
int bwd_threads(int64_t cols) {
  return cols <= 256 ? 32 : cols <= 512 ? 64 : cols <= 1024 ? 128 : cols <= 2048 ? 256 : cols <= 4096 ? 512 : 1024;
}

long long bwd_blocks(int sm_count, long long rows, long long cols) {
  if (cols > 16384) return 0;  // no partial sums
  const int tpr = bwd_threads(cols);
  const long long resident = static_cast<long long>(sm_count) * (tpr == 32 ? 3 : tpr == 1024 ? 1 : 768 / tpr);
  const long long needed = tpr == 32 ? (rows + 7) / 8 : rows;
  return needed < resident ? needed : resident;
}

}  // namespace

extern "C" int b200_int4_gemms_quantize_tokens(int device_index, uintptr_t stream_handle, const void* src_bf16, void* codes,
                                               void* scales_bf16, int64_t rows, int64_t cols, int32_t bits, int32_t subchannel) {
  return guarded([&]() -> int {
    if (int rc = check_rows(rows, cols); rc != 0) return rc;
    if (int rc = check_quantisation(bits, subchannel); rc != 0) return rc;
    if (rows == 0) return 0;
    if (src_bf16 == nullptr || codes == nullptr || scales_bf16 == nullptr) return host_fail("src, codes and scales pointers must be non-null");
    if (int rc = check_alignment("src", src_bf16, 2); rc != 0) return rc;
    if (int rc = check_alignment("scales", scales_bf16, 2); rc != 0) return rc;
    DeviceScope device;
    int sms = 0;
    if (int rc = device.enter(device_index, &sms); rc != 0) return rc;
    const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
    const bool wide = cols % 8 == 0 && is_aligned(src_bf16, 16) && is_aligned(codes, 8);
    for_row_shape(cols, wide, [&](auto tpr, auto v, auto aligned) {
      constexpr int TPR = decltype(tpr)::value, V = decltype(v)::value;
      for_bool(bits == 4, [&](auto four) {
        quantize_tokens_kernel<TPR, V, decltype(four)::value ? 4 : 8, decltype(aligned)::value>
            <<<row_blocks<TPR>(rows), RowPlace<TPR>::kThreads, 0, stream>>>(
                static_cast<const bf16*>(src_bf16), static_cast<uint8_t*>(codes), static_cast<bf16*>(scales_bf16), rows, cols, subchannel);
      });
    });
    return launched("quantize_tokens launch");
  });
}

extern "C" int b200_int4_gemms_layer_norm(int device_index, uintptr_t stream_handle, const void* x, const void* weight, const void* bias,
                                          void* y, float* mean, float* rstd, int64_t rows, int64_t cols, int32_t x_type,
                                          int32_t weight_type, double eps) {
  return guarded([&]() -> int {
    if (int rc = check_rows(rows, cols); rc != 0) return rc;
    if (int rc = check_types(x_type, weight_type); rc != 0) return rc;
    if (!(eps >= 0.0)) return host_fail("eps must be non-negative");
    if (rows == 0) return 0;
    if (x == nullptr || weight == nullptr || y == nullptr || mean == nullptr || rstd == nullptr)
      return host_fail("x, weight, y, mean and rstd pointers must be non-null");
    if (int rc = check_alignment("x", x, type_size(x_type)); rc != 0) return rc;
    if (int rc = check_alignment("y", y, type_size(x_type)); rc != 0) return rc;
    if (int rc = check_alignment("weight", weight, type_size(weight_type)); rc != 0) return rc;
    if (int rc = check_alignment("bias", bias, type_size(weight_type)); rc != 0) return rc;
    if (int rc = check_alignment("mean", mean, 4); rc != 0) return rc;
    if (int rc = check_alignment("rstd", rstd, 4); rc != 0) return rc;
    DeviceScope device;
    int sms = 0;
    if (int rc = device.enter(device_index, &sms); rc != 0) return rc;
    const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
    const bool wide = cols % 8 == 0 && is_aligned(x, 16) && is_aligned(y, 16) && is_aligned(weight, 16) && is_aligned(bias, 16);
    for_types(x_type, weight_type, [&](auto xt, auto wt) {
      using T = decltype(xt);
      using W = decltype(wt);
      for_row_shape(cols, wide, [&](auto tpr, auto v, auto aligned) {
        constexpr int TPR = decltype(tpr)::value, V = decltype(v)::value;
        layer_norm_kernel<T, W, TPR, V, decltype(aligned)::value><<<row_blocks<TPR>(rows), RowPlace<TPR>::kThreads, 0, stream>>>(
            static_cast<const T*>(x), static_cast<const W*>(weight), static_cast<const W*>(bias), static_cast<T*>(y), mean, rstd, rows,
            cols, static_cast<float>(eps));
      });
    });
    return launched("layer_norm launch");
  });
}

extern "C" int b200_int4_gemms_layer_norm_quantize(int device_index, uintptr_t stream_handle, const void* x, const void* weight,
                                                   const void* bias, void* codes, void* scales_bf16, int64_t rows, int64_t cols,
                                                   int32_t x_type, int32_t weight_type, double eps, int32_t bits, int32_t subchannel) {
  return guarded([&]() -> int {
    if (int rc = check_rows(rows, cols); rc != 0) return rc;
    if (int rc = check_types(x_type, weight_type); rc != 0) return rc;
    if (int rc = check_quantisation(bits, subchannel); rc != 0) return rc;
    if (!(eps >= 0.0)) return host_fail("eps must be non-negative");
    if (rows == 0) return 0;
    if (x == nullptr || weight == nullptr || codes == nullptr || scales_bf16 == nullptr)
      return host_fail("x, weight, codes and scales pointers must be non-null");
    if (int rc = check_alignment("x", x, type_size(x_type)); rc != 0) return rc;
    if (int rc = check_alignment("weight", weight, type_size(weight_type)); rc != 0) return rc;
    if (int rc = check_alignment("bias", bias, type_size(weight_type)); rc != 0) return rc;
    if (int rc = check_alignment("scales", scales_bf16, 2); rc != 0) return rc;
    DeviceScope device;
    int sms = 0;
    if (int rc = device.enter(device_index, &sms); rc != 0) return rc;
    NormQuantizeCall call{x, weight, bias, codes, scales_bf16, rows, cols};
    call.weight_f32 = weight_type == B200_OUT_F32;
    call.wide = cols % 8 == 0 && is_aligned(x, 16) && is_aligned(codes, 8) && is_aligned(weight, 16) && is_aligned(bias, 16);
    call.bits = bits;
    call.subchannel = subchannel;
    call.eps = eps;
    call.stream = reinterpret_cast<cudaStream_t>(stream_handle);
    return x_type == B200_OUT_F32 ? launch_norm_quantize_f32(call) : launch_norm_quantize_bf16(call);
  });
}

extern "C" size_t b200_int4_gemms_layer_norm_bwd_workspace_bytes(int device_index, int64_t rows, int64_t cols) {
  size_t bytes = 0;
  guarded([&]() -> int {
    if (int rc = check_rows(rows, cols); rc != 0) return rc;
    DeviceScope device;
    int sms = 0;
    if (int rc = device.enter(device_index, &sms); rc != 0) return rc;
    bytes = static_cast<size_t>(bwd_blocks(sms, rows, cols)) * 2 * static_cast<size_t>(cols) * sizeof(float);
    return 0;
  });
  return bytes;
}

extern "C" int b200_int4_gemms_layer_norm_bwd(int device_index, uintptr_t stream_handle, const void* dy, const void* x,
                                              const void* weight, const float* mean, const float* rstd, void* dx, float* dweight,
                                              float* dbias, void* workspace, size_t workspace_bytes, int64_t rows, int64_t cols,
                                              int32_t x_type, int32_t weight_type) {
  return guarded([&]() -> int {
    if (int rc = check_rows(rows, cols); rc != 0) return rc;
    if (int rc = check_types(x_type, weight_type); rc != 0) return rc;
    if (dweight == nullptr || dbias == nullptr) return host_fail("dweight and dbias pointers must be non-null");
    if (rows > 0 && (dy == nullptr || x == nullptr || weight == nullptr || mean == nullptr || rstd == nullptr || dx == nullptr))
      return host_fail("dy, x, weight, mean, rstd and dx pointers must be non-null");
    if (int rc = check_alignment("dy", dy, type_size(x_type)); rc != 0) return rc;
    if (int rc = check_alignment("x", x, type_size(x_type)); rc != 0) return rc;
    if (int rc = check_alignment("dx", dx, type_size(x_type)); rc != 0) return rc;
    if (int rc = check_alignment("weight", weight, type_size(weight_type)); rc != 0) return rc;
    for (const void* p : {static_cast<const void*>(mean), static_cast<const void*>(rstd), static_cast<const void*>(dweight),
                          static_cast<const void*>(dbias), static_cast<const void*>(workspace)})
      if (int rc = check_alignment("a float32 pointer", p, 4); rc != 0) return rc;
    DeviceScope device;
    int sms = 0;
    if (int rc = device.enter(device_index, &sms); rc != 0) return rc;
    const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
    const long long blocks = bwd_blocks(sms, rows, cols);
    if (blocks > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(blocks) * 2 * cols * sizeof(float)))
      return host_fail("workspace must hold b200_int4_gemms_layer_norm_bwd_workspace_bytes bytes");
    float* partial = static_cast<float*>(workspace);
    const bool wide = cols % 8 == 0 && is_aligned(dy, 16) && is_aligned(x, 16) && is_aligned(dx, 16) && is_aligned(weight, 16);
    const dim3 column_grid(static_cast<unsigned>((cols + 31) / 32)), column_block(32, 32);
    int rc = 0;
    if (rows > 0) {
      for_types(x_type, weight_type, [&](auto xt, auto wt) {
        using T = decltype(xt);
        using W = decltype(wt);
        const T* dy_t = static_cast<const T*>(dy);
        const T* x_t = static_cast<const T*>(x);
        const W* w_t = static_cast<const W*>(weight);
        T* dx_t = static_cast<T*>(dx);
        for_bool(wide, [&](auto aligned) {
          constexpr bool A = decltype(aligned)::value;
          auto narrow = [&](auto tpr) {
            constexpr int TPR = decltype(tpr)::value;
            layer_norm_bwd_kernel<T, W, TPR, A><<<static_cast<unsigned>(blocks), RowPlace<TPR>::kThreads, 0, stream>>>(
                dy_t, x_t, w_t, mean, rstd, dx_t, partial, rows, cols);
          };
          if (cols <= 256) narrow(std::integral_constant<int, 32>());
          else if (cols <= 512) narrow(std::integral_constant<int, 64>());
          else if (cols <= 1024) narrow(std::integral_constant<int, 128>());
          else if (cols <= 2048) narrow(std::integral_constant<int, 256>());
          else if (cols <= 4096) narrow(std::integral_constant<int, 512>());
          else if (cols <= 8192) narrow(std::integral_constant<int, 1024>());
          else if (cols <= 16384) {
            constexpr int kSmem = 2 * 2 * 8 * 1024 * 4;
            const cudaError_t err = cudaFuncSetAttribute(layer_norm_bwd_wide_kernel<T, W, A>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
            if (err != cudaSuccess) {
              rc = host_fail_cuda("cudaFuncSetAttribute(max dynamic shared memory)", err);
              return;
            }
            layer_norm_bwd_wide_kernel<T, W, A><<<static_cast<unsigned>(blocks), 1024, kSmem, stream>>>(dy_t, x_t, w_t, mean, rstd, dx_t,
                                                                                                     partial, rows, cols);
          } else {
            layer_norm_bwd_long_kernel<T, W, A><<<row_blocks<1024>(rows), 1024, 0, stream>>>(dy_t, x_t, w_t, mean, rstd, dx_t, rows, cols);
          }
        });
        if (rc == 0 && cols > 16384)
          layer_norm_bwd_columns_kernel<T><<<column_grid, column_block, 0, stream>>>(dy_t, x_t, mean, rstd, rows, cols, dweight, dbias);
      });
      if (rc != 0) return rc;
      if (rc = launched("layer_norm_bwd launch"); rc != 0) return rc;
    }
    if (rows == 0 || cols <= 16384)
      column_sums_kernel<<<column_grid, column_block, 0, stream>>>(partial, static_cast<int>(blocks), cols, dweight, dbias);
    return launched("layer_norm_bwd column sums launch");
  });
}
