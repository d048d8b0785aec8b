// The expert layer's kernels for one code type: compiled with B200_MOE_BITS 4 and 8.
#include "moe_launch.h"

namespace b200 {
namespace {

constexpr int kBits = B200_MOE_BITS;

// A launch that may start while the kernel before it on the stream still runs (it waits for it by itself).
template <typename... Args>
int launch_dependent(void (*kernel)(Args...), dim3 blocks, int threads, int smem_bytes, cudaStream_t stream, const MoeParams& p) {
  cudaLaunchConfig_t config{};
  config.gridDim = blocks;
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, p);
  return err == cudaSuccess ? 0 : host_fail_cuda("moe_swiglu launch", err);
}

template <bool NN, bool SC, int WORDS, int kMaxN, bool kChoose, bool kDown>
int launch_product(const MoeParams& p, int sm_count, cudaStream_t stream) {
  using Stage = MoeStage<kBits, NN, SC, WORDS, kMaxN>;
  constexpr int smem = Stage::kSmemBytes;
  constexpr auto kernel = moe_product_kernel<kBits, NN, SC, WORDS, kMaxN, kChoose, kDown>;
  if (int rc = allow_shared_memory<kernel>(smem); rc != 0) return rc;
  const long long units = static_cast<long long>(p.slots) * (kDown ? p.down_ranges * p.down_splits : p.up_ranges);
  const long long resident = static_cast<long long>(Stage::kResident) * sm_count, blocks = units < resident ? units : resident;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(blocks)), kMoeThreads, smem, stream, p);
}

// Rows of an expert that a pass over its weights can serve.  The fewer it has to be ready for, the more registers and
// shared memory are left for copies in flight, but a second pass reads the weights again.  As many as the average and
// two of its square roots: with tokens that choose at random, one expert in some 40 has more.  (64 tokens, two of 8
// experts of 4096 x 14336: 171 us with 24, 179 with 32.  13 tokens, 6 of 64 experts, K-group scales: 68 us with 8, 75 with 16.)
int rows_of_a_pass(const MoeParams& p) {
  const int pairs = p.tokens * p.top_k, most = p.sub ? 16 : 32;  // K-group scales: 24 rows of fp64 sums do not fit the registers
  int rows = 8;
  const int mean[] = {4, 9, 16};  // + 2 sqrt: 8, 15, 24
  for (const int m : mean)
    if (rows < most && rows < p.tokens && pairs > m * p.experts) rows += 8;
  return rows;
}

template <bool NN, bool SC, int WORDS>
int launch_for_tokens(const MoeParams& p, bool few, int sm_count, cudaStream_t stream) {
  auto products = [&](auto max_n, auto choose) -> int {
    constexpr int kMaxN = decltype(max_n)::value;
    constexpr bool kChoose = decltype(choose)::value;
    if (int rc = launch_product<NN, SC, WORDS, kMaxN, kChoose, false>(p, sm_count, stream); rc != 0) return rc;
    constexpr int kRow = kMoeQuantThreads * 2;
    auto quantize = SC || p.inner <= 4 * kRow ? moe_quantize_kernel<kBits, 4> : p.inner <= 14 * kRow ? moe_quantize_kernel<kBits, 14> : moe_quantize_kernel<kBits, 0>;
    if (int rc = launch_dependent(quantize, dim3(p.tokens * p.top_k), kMoeQuantThreads, 0, stream, p); rc != 0) return rc;
    if (int rc = launch_product<NN, SC, WORDS, kMaxN, kChoose, true>(p, sm_count, stream); rc != 0) return rc;
    const int lines = p.top_k < kCombineLines ? p.top_k : kCombineLines;
    return launch_dependent(moe_combine_kernel<SC>, dim3((p.hidden + 63) / 64, p.tokens), 32 * lines, 0, stream, p);
  };
  using std::integral_constant;
  if (few) return products(integral_constant<int, 1>(), std::true_type());
  if (p.rows_a_pass == 8) return products(integral_constant<int, 1>(), std::false_type());
  if constexpr (!SC) {
    if (p.rows_a_pass == 32) return products(integral_constant<int, 4>(), std::false_type());
    if (p.rows_a_pass == 24) return products(integral_constant<int, 3>(), std::false_type());
  }
  return products(integral_constant<int, 2>(), std::false_type());
}

}  // namespace

#if B200_MOE_BITS == 4
int launch_moe_int4(const MoeParams& params, bool n_major, int sm_count, cudaStream_t stream) {
#else
int launch_moe_int8(const MoeParams& params, bool n_major, int sm_count, cudaStream_t stream) {
#endif
  MoeParams p = params;
  const bool few = p.tokens <= kMoeFewTokens && p.experts <= kMoeFewExperts;
  p.rows_a_pass = rows_of_a_pass(p);
  const int logit_blocks = p.router != nullptr ? (p.experts + 3) / 4 * ((p.tokens + 3) / 4) : 0;
  moe_route_kernel<kBits><<<p.tokens + logit_blocks, 256, 0, stream>>>(p);
  if (const cudaError_t err = cudaGetLastError(); err != cudaSuccess) return host_fail_cuda("moe_swiglu launch", err);
  if (!few) {  // experts <= 64, 256, 1024: logits a lane keeps
    auto select = p.experts <= 64 ? moe_select_kernel<2, 1024> : p.experts <= 256 ? moe_select_kernel<8, 1024> : moe_select_kernel<32, 1024>;
    if (int rc = launch_dependent(select, dim3(1), 1024, 0, stream, p); rc != 0) return rc;
  }
  // words of token codes that a lane takes at a step: as many as keep a step within a group of K (32 K a word of
  // nibbles, 16 a word of bytes) and the ring's stages small
  constexpr int kWord = kBits == 4 ? 32 : 16, kLeast = kBits == 4 ? 1 : 2;
  const bool two_words = !p.sub || p.sub >= 2 * kWord;
  if (n_major) {
    if (!p.sub) return launch_for_tokens<true, false, 2>(p, few, sm_count, stream);
    return two_words ? launch_for_tokens<true, true, 2>(p, few, sm_count, stream) : launch_for_tokens<true, true, kLeast>(p, few, sm_count, stream);
  }
  if (!p.sub || p.sub >= 4 * kWord) return p.sub ? launch_for_tokens<false, true, 4>(p, few, sm_count, stream) : launch_for_tokens<false, false, 4>(p, few, sm_count, stream);
  return two_words ? launch_for_tokens<false, true, 2>(p, few, sm_count, stream) : launch_for_tokens<false, true, kLeast>(p, few, sm_count, stream);
}

}  // namespace b200
