// The expert layer's kernels for one code type: compiled with B200_MOE_BITS 4 and 8.
#include "moe_launch.h"

#include <type_traits>

namespace b200 {
namespace {

constexpr int kBits = B200_MOE_BITS;

template <bool NN, bool SC, int WORDS>
void launch_products(const MoeParams& p, cudaStream_t stream) {
  const int cols = MoeShape<NN>::kCols;
  const int up_ranges = (p.inner + cols / 2 - 1) / (cols / 2);
  moe_product_kernel<kBits, NN, SC, WORDS, false><<<p.slots * up_ranges, kMoeThreads, 0, stream>>>(p);
  moe_product_kernel<kBits, NN, SC, WORDS, true><<<p.slots * p.down_ranges, kMoeThreads, 0, stream>>>(p);
}

}  // namespace

#if B200_MOE_BITS == 4
int launch_moe_int4(const MoeParams& p, bool n_major, cudaStream_t stream) {
#else
int launch_moe_int8(const MoeParams& p, bool n_major, cudaStream_t stream) {
#endif
  const int logit_blocks = p.router != nullptr ? (p.experts + 7) / 8 * ((p.tokens + 7) / 8) : 0;
  moe_route_kernel<kBits><<<p.tokens + 1 + logit_blocks, 256, 0, stream>>>(p);
  moe_select_kernel<<<1, 1024, 0, stream>>>(p);
  // K-major weights with scales for groups of K: a warp's load stays within one group (32 K a word of nibbles, 16 a
  // word of bytes)
  constexpr int kWord = kBits == 4 ? 32 : 16;
  if (n_major) {
    if (p.sub) launch_products<true, true, 4>(p, stream);
    else launch_products<true, false, 4>(p, stream);
  } else if (!p.sub) {
    launch_products<false, false, 4>(p, stream);
  } else if (p.sub >= 4 * kWord) {
    launch_products<false, true, 4>(p, stream);
  } else if (p.sub == 2 * kWord) {
    launch_products<false, true, 2>(p, stream);
#if B200_MOE_BITS == 4
  } else {
    launch_products<false, true, 1>(p, stream);
#endif
  }
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? 0 : host_fail_cuda("moe_swiglu launch", err);
}

}  // namespace b200
