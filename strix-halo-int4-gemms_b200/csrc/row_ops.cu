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

// The backward kernel's shape: threads of a row (of half of it, above 8192 values) and groups of eight values a thread:
// two of bf16, one of fp32, whose registers are twice as many.
struct BwdPlan {
  int threads, vectors, cluster;
  int groups() const { return threads < 512 ? 512 / threads : 1; }
};
BwdPlan bwd_plan(long long cols, int x_type) {
  const int v = x_type == B200_OUT_BF16 ? 2 : 1;
  const int cluster = cols > 8192 ? 2 : 1;
  int threads = 32;
  while (static_cast<long long>(threads) * v * 8 * cluster < cols) threads *= 2;
  return {threads, v, cluster};
}

// As many clusters of its blocks as are resident at once, one row of partial sums each.
long long bwd_units(int sm_count, long long rows, long long cols, int x_type) {
  if (cols > 16384) return 0;  // no partial sums
  const BwdPlan plan = bwd_plan(cols, x_type);
  // 512 threads: two blocks an SM of bf16 (about 64 registers a thread would allow it), 1024: one
  const long long resident = static_cast<long long>(sm_count) / plan.cluster;
  const long long needed = (rows + plan.groups() - 1) / plan.groups();
  return needed < resident ? needed : resident;
}

template <typename T, typename W, int TPR, int V, int CLUSTER, bool kAligned>
int launch_bwd(const T* dy, const T* x, const W* weight, const float* mean, const float* rstd, T* dx, float* partial, long long units,
               long long rows, long long cols, volatile int* status, cudaStream_t stream) {
  auto kernel = layer_norm_bwd_kernel<T, W, TPR, V, CLUSTER, kAligned>;
  using Shape = BwdShape<TPR, CLUSTER>;
  constexpr int smem = Shape::kGroups > 1 ? TPR * V * 8 * 4 : 0;
  static_assert(smem <= 32 * 1024, "fits without permission");
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(units * CLUSTER));
  config.blockDim = dim3(Shape::kThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = CLUSTER;
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, dy, x, weight, mean, rstd, dx, partial, rows, cols, status);
  return err == cudaSuccess ? 0 : host_fail_cuda("layer_norm_bwd launch", err);
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
    for_row_shape<8>(rows, cols, wide, [&](auto tpr, auto v, auto aligned) {
      constexpr int TPR = decltype(tpr)::value, V = decltype(v)::value;
      for_bool(bits == 4, [&](auto four) {
        quantize_tokens_kernel<TPR, V, decltype(four)::value ? 4 : 8, decltype(aligned)::value>
            <<<row_blocks<TPR>(rows), RowPlace<TPR>::kThreads, 0, stream>>>(
                static_cast<const bf16*>(src_bf16), static_cast<uint8_t*>(codes), static_cast<bf16*>(scales_bf16), rows, cols, group_bits(subchannel));
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
      for_row_shape<sizeof(T) == 2 ? 8 : 4>(rows, cols, wide, [&](auto tpr, auto v, auto aligned) {
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
    call.sm_count = sms;
    call.eps = eps;
    call.stream = reinterpret_cast<cudaStream_t>(stream_handle);
    return x_type == B200_OUT_F32 ? launch_norm_quantize_f32(call) : launch_norm_quantize_bf16(call);
  });
}

extern "C" size_t b200_int4_gemms_layer_norm_bwd_workspace_bytes(int device_index, int64_t rows, int64_t cols, int32_t x_type) {
  size_t bytes = 0;
  guarded([&]() -> int {
    if (int rc = check_rows(rows, cols); rc != 0) return rc;
    if (int rc = check_types(x_type, x_type); rc != 0) return rc;
    DeviceScope device;
    int sms = 0;
    if (int rc = device.enter(device_index, &sms); rc != 0) return rc;
    bytes = static_cast<size_t>(bwd_units(sms, rows, cols, x_type)) * 2 * static_cast<size_t>(cols) * sizeof(float);
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
    const long long units = bwd_units(sms, rows, cols, x_type);
    if (units > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(units) * 2 * cols * sizeof(float)))
      return host_fail("workspace must hold b200_int4_gemms_layer_norm_bwd_workspace_bytes bytes");
    float* partial = static_cast<float*>(workspace);
    volatile int* status = device_status_word(device_index);
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
          constexpr int V = sizeof(T) == 2 ? 2 : 1;
          using std::integral_constant;
          auto rows_of = [&](auto tpr, auto cluster) {
            rc = launch_bwd<T, W, decltype(tpr)::value, V, decltype(cluster)::value, A>(dy_t, x_t, w_t, mean, rstd, dx_t, partial, units, rows, cols, status, stream);
          };
          const BwdPlan plan = bwd_plan(cols, x_type);
          if (cols > 16384) layer_norm_bwd_long_kernel<T, W, A><<<row_blocks<1024>(rows), 1024, 0, stream>>>(dy_t, x_t, w_t, mean, rstd, dx_t, rows, cols);
          else if (plan.cluster == 2) rows_of(integral_constant<int, 1024 / V>(), integral_constant<int, 2>());
          else if (plan.threads == 32) rows_of(integral_constant<int, 32>(), integral_constant<int, 1>());
          else if (plan.threads == 64) rows_of(integral_constant<int, 64>(), integral_constant<int, 1>());
          else if (plan.threads == 128) rows_of(integral_constant<int, 128>(), integral_constant<int, 1>());
          else if (plan.threads == 256) rows_of(integral_constant<int, 256>(), integral_constant<int, 1>());
          else if (plan.threads == 512) rows_of(integral_constant<int, 512>(), integral_constant<int, 1>());
          else rows_of(integral_constant<int, V == 1 ? 1024 : 512>(), integral_constant<int, 1>());
        });
        if (rc == 0 && cols > 16384)
          layer_norm_bwd_columns_kernel<T><<<column_grid, column_block, 0, stream>>>(dy_t, x_t, mean, rstd, rows, cols, dweight, dbias);
      });
      if (rc != 0) return rc;
      if (rc = launched("layer_norm_bwd launch"); rc != 0) return rc;
    }
    if (rows > 0 && cols > 16384) return launched("layer_norm_bwd columns launch");
    // may start while the kernel before it ends: it waits for it by itself
    cudaLaunchConfig_t config{};
    config.gridDim = column_grid;
    config.blockDim = dim3(32, kSumRows);
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = rows > 0 ? 1 : 0;
    config.attrs = attribute;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, column_sums_kernel, static_cast<const float*>(partial), static_cast<int>(units),
                                               static_cast<long long>(cols), dweight, dbias);
    return err == cudaSuccess ? 0 : host_fail_cuda("layer_norm_bwd column sums launch", err);
  });
}
