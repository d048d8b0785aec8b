// C entry points of the expert layer for a few tokens: argument checks, scratch layout, launches.
#include "../../include/b200_int4_gemms.h"
#include "moe_launch.h"

namespace {

using namespace b200;

static_assert(kMoeMaxTokens == B200_MOE_MAX_TOKENS && kMoeMaxTopK == B200_MOE_MAX_TOP_K && kMoeMaxExperts == B200_MOE_MAX_EXPERTS,
              "the header states the kernels' limits");

int check_problem(const b200_moe_problem* m) {
  if (m == nullptr) return host_fail("problem must be non-null");
  if (m->dtype != B200_DTYPE_INT4 && m->dtype != B200_DTYPE_INT8) return host_fail("problem.dtype is not INT4 or INT8");
  if (m->layout != B200_LAYOUT_NN && m->layout != B200_LAYOUT_NT) return host_fail("problem.layout must be NN or NT");
  if (m->subchannel != 0 && m->subchannel != 32 && m->subchannel != 64 && m->subchannel != 128 && m->subchannel != 256)
    return host_fail("problem.subchannel must be 0 (one scale a column), 32, 64, 128 or 256");
  if (m->tokens < 0 || m->tokens > kMoeMaxTokens)
    return host_fail("tokens must be at most " + std::to_string(kMoeMaxTokens) + "; use the grouped dots for more rows");
  if (m->experts <= 0 || m->experts > kMoeMaxExperts) return host_fail("experts must be in [1, " + std::to_string(kMoeMaxExperts) + "]");
  if (m->top_k <= 0 || m->top_k > kMoeMaxTopK || m->top_k > m->experts)
    return host_fail("top_k must be in [1, " + std::to_string(kMoeMaxTopK) + "] and at most the number of experts");
  // 16 x the int4 codes on both sides: 256 * 64 * K stays below 2^31 for K < 131072 (and 127 * 128 * K for int8)
  for (const int32_t size : {m->hidden, m->inner})
    if (size <= 0 || size % 32 != 0 || size >= 131072)
      return host_fail("hidden and inner must be multiples of 32 (the K of one tensor-core instruction) below 131072");
  if (m->router_type != B200_OUT_BF16 && m->router_type != B200_OUT_F32) return host_fail("router weights must be bf16 or float32");
  if (m->ids_bits != 32 && m->ids_bits != 64) return host_fail("ids must have 32 or 64 bits");
  return 0;
}

// Lays the scratch out from `base` (null to count only) and returns its size.
size_t lay_out(const b200_moe_problem& m, char* base, MoeParams* p) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* here = base == nullptr ? nullptr : base + at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t pairs = static_cast<size_t>(m.tokens) * m.top_k;
  const size_t per_byte = m.dtype == B200_DTYPE_INT4 ? 2 : 1;
  const size_t x_groups = m.subchannel ? (m.hidden + m.subchannel - 1) / m.subchannel : 1;
  const size_t a_groups = m.subchannel ? (m.inner + m.subchannel - 1) / m.subchannel : 1;
  const int down_cols = m.layout == B200_LAYOUT_NN ? 128 : 64;  // of one block
  p->slots = static_cast<int>(pairs < static_cast<size_t>(m.experts) ? pairs : m.experts);
  p->up_ranges = (m.inner + down_cols / 2 - 1) / (down_cols / 2);
  p->down_ranges = (m.hidden + down_cols - 1) / down_cols;
  // The down product divides K between blocks where there are fewer (expert, column range) units than would keep the
  // blocks that the device holds (2 or 3 an SM) evenly busy, as long as each of a block's warps has four steps left.
  const int step = (m.dtype == B200_DTYPE_INT4 ? 64 : 32) * (m.layout == B200_LAYOUT_NN ? 1 : 2), shares = 4;
  p->down_splits = 1;
  while (p->down_splits < 8 && static_cast<long long>(p->slots) * p->down_ranges * p->down_splits < 1024 &&
         m.inner >= static_cast<long long>(step) * shares * p->down_splits * 2 * 4)
    p->down_splits *= 2;
  p->xq = reinterpret_cast<uint8_t*>(take(static_cast<size_t>(m.tokens) * m.hidden / per_byte));
  p->xs = reinterpret_cast<float*>(take(m.tokens * x_groups * 4));
  p->logits = reinterpret_cast<double*>(take(static_cast<size_t>(m.tokens) * m.experts * 8));
  p->pair_expert = reinterpret_cast<int*>(take(pairs * 4));
  p->pair_logit = reinterpret_cast<double*>(take(pairs * 8));
  p->active = reinterpret_cast<int*>(take((1 + static_cast<size_t>(p->slots)) * 16));
  p->pair_list = reinterpret_cast<int*>(take(pairs * 4));
  p->act = reinterpret_cast<double*>(take(pairs * m.inner * 8));
  p->aq = reinterpret_cast<uint8_t*>(take(pairs * m.inner / per_byte));
  p->as = reinterpret_cast<float*>(take(pairs * a_groups * 4));
  p->part = take(pairs * p->down_splits * m.hidden * (m.subchannel ? 8 : 4));
  return at;
}

}  // namespace

extern "C" size_t b200_int4_gemms_moe_swiglu_workspace_bytes(const b200_moe_problem* problem) {
  size_t bytes = 0;
  guarded([&]() -> int {
    if (int rc = check_problem(problem); rc != 0) return rc;
    MoeParams p{};
    bytes = problem->tokens > 0 ? lay_out(*problem, nullptr, &p) : 0;
    return 0;
  });
  return bytes;
}

extern "C" int b200_int4_gemms_moe_swiglu(const b200_moe_problem* problem, int device_index, uintptr_t stream_handle, const void* x_bf16,
                                          const void* router_weight, void* topk_ids, float* topk_weights, const void* w_up_gate,
                                          const void* up_gate_scale, const void* w_down, const void* down_scale, void* out_bf16,
                                          void* workspace, size_t workspace_bytes) {
  return guarded([&]() -> int {
    if (int rc = check_problem(problem); rc != 0) return rc;
    const b200_moe_problem& m = *problem;
    if (m.tokens == 0) return 0;
    if (x_bf16 == nullptr || w_up_gate == nullptr || up_gate_scale == nullptr || w_down == nullptr || down_scale == nullptr || out_bf16 == nullptr)
      return host_fail("x, weight, scale and out pointers must be non-null");
    if (router_weight == nullptr && (topk_ids == nullptr || topk_weights == nullptr))
      return host_fail("either router weights or topk_ids and topk_weights must be given");
    if (router_weight != nullptr && topk_ids != nullptr && m.ids_bits != 32) return host_fail("topk_ids are written as int32");
    for (const void* ptr : {x_bf16, router_weight, w_up_gate, w_down, up_gate_scale, down_scale})
      if (!is_aligned(ptr, 16)) return host_fail("x, weight and scale pointers must be 16-byte aligned");
    if (!is_aligned(out_bf16, 2) || !is_aligned(topk_weights, 4) || !is_aligned(topk_ids, m.ids_bits / 8))
      return host_fail("out, topk_ids and topk_weights pointers must be aligned to their element size");
    DeviceScope device;
    int sms = 0;
    if (int rc = device.enter(device_index, &sms); rc != 0) return rc;
    MoeParams p{};
    const size_t need = lay_out(m, static_cast<char*>(workspace), &p);
    if (workspace == nullptr || !is_aligned(workspace, 256) || workspace_bytes < need)
      return host_fail("workspace must be 256-byte aligned and hold b200_int4_gemms_moe_swiglu_workspace_bytes bytes");
    p.x = static_cast<const bf16*>(x_bf16);
    p.router = router_weight;
    p.ids_in = router_weight == nullptr ? topk_ids : nullptr;
    p.weights_in = router_weight == nullptr ? topk_weights : nullptr;
    p.ids_out = router_weight == nullptr ? nullptr : static_cast<int*>(topk_ids);
    p.weights_out = router_weight == nullptr ? nullptr : topk_weights;
    p.w_up_gate = static_cast<const uint8_t*>(w_up_gate);
    p.w_down = static_cast<const uint8_t*>(w_down);
    p.s_up_gate = static_cast<const bf16*>(up_gate_scale);
    p.s_down = static_cast<const bf16*>(down_scale);
    p.out = static_cast<bf16*>(out_bf16);
    p.tokens = m.tokens;
    p.hidden = m.hidden;
    p.inner = m.inner;
    p.experts = m.experts;
    p.top_k = m.top_k;
    p.sub = m.subchannel;
    while ((1 << p.sub_bits) < p.sub) ++p.sub_bits;
    p.router_f32 = m.router_type == B200_OUT_F32;
    p.ids_64 = m.ids_bits == 64;
    p.renormalize = m.renormalize;
    const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
    const bool n_major = m.layout == B200_LAYOUT_NN;
    return m.dtype == B200_DTYPE_INT4 ? launch_moe_int4(p, n_major, sms, stream) : launch_moe_int8(p, n_major, sms, stream);
  });
}
