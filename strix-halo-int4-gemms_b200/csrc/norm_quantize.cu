// layer_norm_quantize_kernel for one type of x: compiled with B200_NORM_X_F32 0 and 1.
#include "row_launch.h"

namespace b200 {

#if B200_NORM_X_F32
using NormX = float;
int launch_norm_quantize_f32(const NormQuantizeCall& c) {
#else
using NormX = bf16;
int launch_norm_quantize_bf16(const NormQuantizeCall& c) {
#endif
  for_bool(c.weight_f32, [&](auto weight_f32) {
    using W = std::conditional_t<decltype(weight_f32)::value, float, bf16>;
    for_row_shape<4>(c.rows, c.cols, c.wide, [&](auto tpr, auto v, auto aligned) {
      constexpr int TPR = decltype(tpr)::value, V = decltype(v)::value;
      for_bool(c.bits == 4, [&](auto four) {
        layer_norm_quantize_kernel<NormX, W, TPR, V, decltype(four)::value ? 4 : 8, decltype(aligned)::value>
            <<<row_blocks<TPR>(c.rows), RowPlace<TPR>::kThreads, 0, c.stream>>>(
                static_cast<const NormX*>(c.x), static_cast<const W*>(c.weight), static_cast<const W*>(c.bias),
                static_cast<uint8_t*>(c.codes), static_cast<bf16*>(c.scales), c.rows, c.cols, group_bits(c.subchannel),
                1.0 / static_cast<double>(c.cols), c.eps);
      });
    });
  });
  return launched("layer_norm_quantize launch");
}

}  // namespace b200
