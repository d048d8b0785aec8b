// C entry points of the row kernels: quantize_tokens, layer_norm, layer_norm_quantize, layer_norm_bwd.
#include "../../include/b200_int4_gemms.h"
#include "host_common.h"
#include "row_launch.h"

#include <algorithm>
#include <atomic>
#include <cfloat>

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

// The backward pass of rows of up to kBwdHeld values: threads of a row, with two groups of eight bf16 values or one of
// fp32, whose registers are twice as many.  Wider rows: two kernels, with the rows divided into `parts`.
constexpr long long kBwdHeld = 8192;

// Columns of a thread of the strips kernel: 16 bytes of them where rows can be read that way.
template <typename T, bool kWide>
constexpr int strip_columns() { return kWide ? 16 / static_cast<int>(sizeof(T)) : 1; }

int bwd_threads(long long cols, int x_type) {
  const int v = x_type == B200_OUT_BF16 ? 2 : 1;
  int threads = 32;
  while (static_cast<long long>(threads) * v * 8 < cols) threads *= 2;
  return threads;
}

// Blocks of the strips kernel (wide rows) that an SM holds at once, by its registers: one in bf16, two in fp32, three where
// rows cannot be read 16 bytes at a time.  0 with a message if the device does not say.
template <typename T, typename W, int G>
int strip_blocks_an_sm() {
  static std::atomic<int> known{0};
  if (int blocks = known.load(std::memory_order_relaxed); blocks > 0) return blocks;
  int blocks = 0;
  const cudaError_t err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, layer_norm_bwd_strips_kernel<T, W, G>, 32 * kStripWarps, 0);
  if (err != cudaSuccess || blocks <= 0) {
    host_fail_cuda("cudaOccupancyMaxActiveBlocksPerMultiprocessor", err);
    return 0;
  }
  known.store(blocks, std::memory_order_relaxed);
  return blocks;
}

// Parts of the rows for the strips kernel: the fewest with which its blocks fill their waves to four fifths, or the best of six.
// (Measured at 8704 to 131072 columns, 128 to 4096 rows: 1 % above the best number on average.  4096 x 20000 in fp32, 157
// strips, two blocks an SM: 291 us in one part, 304 in two, 257 in five; 4096 x 40000 in bf16, 157 strips, one block an SM:
// 451 us in one part, 365 in three.)  A warp adds up at most 512 rows in one chain.
long long strip_parts(long long strips, long long at_once, long long rows) {
  const long long least = (rows + 4095) / 4096, most = std::max(least, std::min(least + 5, (rows + 31) / 32));
  long long best = least;
  double best_fill = 0.0;
  for (long long parts = least; parts <= most && best_fill < 0.8; ++parts) {
    const long long blocks = strips * parts, waves = (blocks + at_once - 1) / at_once;
    const double fill = static_cast<double>(blocks) / static_cast<double>(waves * at_once);
    if (fill > best_fill) {
      best = parts;
      best_fill = fill;
    }
  }
  return best;
}

// Rows of partial sums: one for each block that is resident at once (512 threads or more, one an SM), or, for wide rows, one
// for each part.
int bwd_partials(int sm_count, long long rows, long long cols, int x_type, int w_type, bool wide, long long* partials) {
  *partials = 0;
  if (rows == 0) return 0;
  if (cols <= kBwdHeld) {
    const int threads = bwd_threads(cols, x_type), groups = threads < 512 ? 512 / threads : 1;
    *partials = std::min<long long>((rows + groups - 1) / groups, sm_count);
    return 0;
  }
  int at_once = 0, width = 0;
  for_types(x_type, w_type, [&](auto xt, auto wt) {
    using T = decltype(xt);
    using W = decltype(wt);
    for_bool(wide, [&](auto aligned) {
      constexpr int G = strip_columns<T, decltype(aligned)::value>();
      at_once = strip_blocks_an_sm<T, W, G>() * sm_count;
      width = 32 * G;
    });
  });
  if (at_once == 0) return 1;
  *partials = strip_parts((cols + width - 1) / width, at_once, rows);
  return 0;
}

size_t bwd_sums_bytes(long long partials, long long cols) { return (static_cast<size_t>(partials) * 2 * cols * sizeof(float) + 15) / 16 * 16; }

// Enough for every type of weight, and whether rows can be read 16 bytes at a time or not.
int bwd_workspace(int sm_count, long long rows, long long cols, int x_type, size_t* bytes) {
  long long most = 0;
  for (const int w_type : {B200_OUT_BF16, B200_OUT_F32})
    for (const bool wide : {false, true}) {
      long long partials = 0;
      if (int rc = bwd_partials(sm_count, rows, cols, x_type, w_type, wide, &partials); rc != 0) return rc;
      most = std::max(most, partials);
    }
  *bytes = bwd_sums_bytes(most, cols) + (cols > kBwdHeld ? static_cast<size_t>(rows) * sizeof(RowTerms) : 0);
  return 0;
}

// A launch that may start while the kernel before it on the stream still runs (it waits for it by itself).
template <typename... Params, typename... Args>
int launch_after(void (*kernel)(Params...), dim3 grid, dim3 block, bool overlap, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = overlap ? 1 : 0;
  config.attrs = attribute;
  config.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
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
    // it is added to a float32 variance: what rounds to zero there would make rows of equal values NaN
    if (eps != 0.0 && !(eps > 0.5 * FLT_TRUE_MIN && eps <= FLT_MAX)) return host_fail("eps must be zero or within the range of float32");
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
      for_row_shape<4>(rows, cols, wide, [&](auto tpr, auto v, auto aligned) {
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

extern "C" size_t b200_int4_gemms_layer_norm_bwd_workspace_bytes(int device_index, int64_t rows, int64_t cols, int32_t x_type) {
  size_t bytes = 0;
  guarded([&]() -> int {
    if (int rc = check_rows(rows, cols); rc != 0) return rc;
    if (int rc = check_types(x_type, x_type); rc != 0) return rc;
    DeviceScope device;
    int sms = 0;
    if (int rc = device.enter(device_index, &sms); rc != 0) return rc;
    return bwd_workspace(sms, rows, cols, x_type, &bytes);
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
    const bool wide = cols % 8 == 0 && is_aligned(dy, 16) && is_aligned(x, 16) && is_aligned(dx, 16) && is_aligned(weight, 16);
    size_t need = 0;
    if (int rc = bwd_workspace(sms, rows, cols, x_type, &need); rc != 0) return rc;
    long long partials = 0;
    if (int rc = bwd_partials(sms, rows, cols, x_type, weight_type, wide, &partials); rc != 0) return rc;
    if (need > 0 && (workspace == nullptr || !is_aligned(workspace, 16) || workspace_bytes < need))
      return host_fail("workspace must be 16-byte aligned and hold b200_int4_gemms_layer_norm_bwd_workspace_bytes bytes");
    float* partial = static_cast<float*>(workspace);
    RowTerms* terms = reinterpret_cast<RowTerms*>(static_cast<char*>(workspace) + bwd_sums_bytes(partials, cols));  // wide rows only
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
          if (cols > kBwdHeld) {
            constexpr int G = strip_columns<T, A>();
            const long long blocks = std::min<long long>(rows, 4LL * sms);
            layer_norm_bwd_rows_kernel<T, W, A><<<static_cast<unsigned>(blocks), 512, 0, stream>>>(dy_t, x_t, w_t, mean, rstd, terms, rows, cols);
            if (rc = launched("layer_norm_bwd launch"); rc != 0) return;
            const dim3 grid(static_cast<unsigned>((cols + 32 * G - 1) / (32 * G)), static_cast<unsigned>(partials));
            rc = launch_after(layer_norm_bwd_strips_kernel<T, W, G>, grid, dim3(32 * kStripWarps), true, stream, dy_t, x_t, w_t, terms, dx_t, partial, rows, cols);
            return;
          }
          using std::integral_constant;
          auto rows_of = [&](auto tpr) {
            constexpr int TPR = decltype(tpr)::value, kThreads = BwdShape<TPR>::kThreads;
            constexpr int sums = BwdShape<TPR>::kGroups > 1 ? TPR * V * 8 * 4 : 0, smem = A ? std::max(sums, BwdShape<TPR>::kRingBytes) : sums;
            constexpr auto kernel = layer_norm_bwd_kernel<T, W, TPR, V, A>;
            if (rc = allow_shared_memory<kernel>(smem); rc != 0) return;
            kernel<<<static_cast<unsigned>(partials), kThreads, smem, stream>>>(dy_t, x_t, w_t, mean, rstd, dx_t, partial, rows, cols);
            rc = launched("layer_norm_bwd launch");
          };
          const int threads = bwd_threads(cols, x_type);
          if (threads == 32) rows_of(integral_constant<int, 32>());
          else if (threads == 64) rows_of(integral_constant<int, 64>());
          else if (threads == 128) rows_of(integral_constant<int, 128>());
          else if (threads == 256) rows_of(integral_constant<int, 256>());
          else if (threads == 512) rows_of(integral_constant<int, 512>());
          else rows_of(integral_constant<int, V == 1 ? 1024 : 512>());
        });
      });
      if (rc != 0) return rc;
    }
    return launch_after(column_sums_kernel, dim3(static_cast<unsigned>((cols + 31) / 32)), dim3(32, kSumRows), rows > 0, stream, partial,
                        static_cast<int>(partials), cols, dweight, dbias);
  });
}
