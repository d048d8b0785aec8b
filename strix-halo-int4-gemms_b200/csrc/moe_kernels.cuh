// A whole mixture-of-experts layer for a few tokens:
//   moe_route_kernel     router logits (fp64 sums), the tokens' codes and scales
//   moe_select_kernel    top-k, and for each expert in use the list of its (token, choice) pairs (up to eight tokens: the
//                        blocks of the products do this themselves)
//   moe_product_kernel   up/gate product, SwiGLU
//   moe_quantize_kernel  the activations' codes and scales
//   moe_product_kernel   down product
//   moe_combine_kernel   softmax; the experts' shares of every token added up
// Each kernel is launched while the one before it still runs (programmatic dependent launch) and waits for it where
// it needs its results; the down product's first weights are on their way before the up/gate product has ended.
// One token, 8 of 64 experts of 2048 x 1408 in int4: 18.5 us on the device, 2 for the router, 3 until the first weights are
// on their way, 7 and 3 for the products, 1.5 for the codes, 1 for the shares, the rest between them.  The last block of an expert (of a column
// range) to finish can make the codes (add up the shares) without a launch; that was slower (26 us), since the
// counting costs each unit 1 us and what the last block does is not shared.
//
// At a few tokens each weight is used by a handful of rows, so the layer is bound by reading the weights of the
// experts in use once from HBM.  The products therefore run on mma.sync.m16n8k32 (int8, exact int32 sums) with the
// WEIGHTS as the 16-row operand and eight tokens at a time as the other.  Every warp copies its share of the weights
// into a ring of its own in shared memory (cp.async), several steps ahead: some 100 KB an SM in flight within a unit of
// work, which is what HBM's latency asks for.  At the end of a unit the ring runs empty: the first weights of the next one
// are asked for behind its last step, before its sums are finished.  tcgen05 would
// want 128-row tiles of unpacked weights in shared memory; its rate is of no use here (measured on this part:
// m16n8k32 every 2 clocks an SM, 256 weights a clock for eight tokens and 85 for 24, where HBM delivers 46).
//
// Operand order.  A lane (g = lane / 4, q = lane % 4) supplies rows g and g + 8 of the 16 x 32 operand and, for
// each, K values that a quad of lanes divides up.  Which K a lane holds does not matter as long as both operands
// agree, so a lane takes consecutive packed bytes.  A word of eight nibbles is two words of the int8 operand: even
// K (w << 4) & 0xF0F0F0F0, odd K w & 0xF0F0F0F0, each value 16 times too large; the sum is 256 times too large and
// shifted right at the end, exactly.
#pragma once

#include <type_traits>

#include "row_common.cuh"

namespace b200 {

constexpr int kMoeMaxTokens = 64;
constexpr int kMoeMaxTopK = 16;
constexpr int kMoeMaxExperts = 1024;
constexpr int kMoeMaxPairs = kMoeMaxTokens * kMoeMaxTopK;

struct MoeParams {
  const bf16* x;            // [tokens, hidden]
  const void* router;       // [experts, hidden] bf16 or fp32, or null: ids and weights are given
  const void* ids_in;       // [tokens, top_k] int32 or int64 (router == null)
  const float* weights_in;  // [tokens, top_k]
  int* ids_out;             // [tokens, top_k], may be null
  float* weights_out;
  const uint8_t* w_up_gate;
  const uint8_t* w_down;
  const bf16* s_up_gate;
  const bf16* s_down;
  bf16* out;                // [tokens, hidden]
  int tokens, hidden, inner, experts, top_k, sub, sub_bits;  // a group of K: sub = 2^sub_bits values; 0: none
  int router_f32, ids_64, renormalize, rows_a_pass;
  // scratch
  uint8_t* xq;              // [tokens, hidden bytes]
  float* xs;                // [tokens, groups of hidden]
  double* logits;           // [tokens, experts]
  int* pair_expert;         // [pairs], -1: no expert
  double* pair_logit;       // [pairs]: of the chosen experts (router != null)
  int* active;              // {experts in use, passes in all, units handed out by the two products}; then slots of
                            // {expert, first pair, pairs, passes of those before}
  int* pair_list;           // [pairs], by expert
  double* act;              // [pairs, inner]
  uint8_t* aq;              // [pairs, inner bytes]
  float* as;                // [pairs, groups of inner]
  void* part;               // [down_splits, pairs, hidden]: sums of the codes' products (int32), or scaled ones (fp64)
  int slots, up_ranges, down_ranges, down_splits;
};

// Up to eight tokens (the products' kChoose) the time is that of the kernels' starts: every block of the up/gate product
// (and then of the down product) picks the experts by itself.
constexpr int kMoeFewTokens = 8;
constexpr int kMoeFewExperts = 256;
constexpr int kMoeFewPairs = kMoeFewTokens * kMoeMaxTopK;

template <int DT>
__device__ __forceinline__ long long code_bytes(long long k) { return DT == 4 ? k / 2 : k; }

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---------------------------------------------------------------------------------------------------------------
// Logits of four experts for up to four tokens: 8 values converted to fp64 (16 a clock and SM) for 16 products (64 a
// clock); the eight warps divide K between them.
template <typename W>
__device__ __forceinline__ void route_logits(const MoeParams& p, int block) {
  __shared__ double part[8][16];
  const int expert_blocks = (p.experts + 3) / 4;
  const int e0 = (block % expert_blocks) * 4, t0 = (block / expert_blocks) * 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, last_e = p.experts - 1, last_t = p.tokens - 1;
  double acc[16];  // [expert][token]
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.0;
  for (int at = threadIdx.x * 8; at < p.hidden; at += 2048) {
    Raw8<W> w[4];
    Raw8<bf16> x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)  // beyond the last expert or token: the last one again, not stored
      w[e].template load<true>(static_cast<const W*>(p.router) + static_cast<long long>(min(e0 + e, last_e)) * p.hidden, at, p.hidden);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t0 + t <= last_t) x[t].load<true>(p.x + static_cast<long long>(t0 + t) * p.hidden, at, p.hidden);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t0 + t > last_t) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double v = static_cast<double>(x[t].get(i));
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e * 4 + t] = fma(v, static_cast<double>(w[e].get(i)), acc[e * 4 + t]);
      }
    }
  }
  // sums of 16 values over the lanes; lanes 2 i and 2 i + 1 are left with halves of value i
#pragma unroll
  for (int o = 16; o > 1; o >>= 1) {
#pragma unroll
    for (int j = 0; j < o / 2; ++j) {
      const bool upper = (lane & o) != 0;
      const double send = upper ? acc[j] : acc[j + o / 2], keep = upper ? acc[j + o / 2] : acc[j];
      acc[j] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, o);
    }
  }
  acc[0] += __shfl_xor_sync(0xFFFFFFFFu, acc[0], 1);
  if ((lane & 1) == 0) part[warp][lane >> 1] = acc[0];
  __syncthreads();
  if (threadIdx.x < 16) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += part[i][threadIdx.x];
    const int e = e0 + threadIdx.x / 4, t = t0 + threadIdx.x % 4;
    if (e <= last_e && t <= last_t) p.logits[static_cast<long long>(t) * p.experts + e] = sum;
  }
}

// The codes and scales of one token, as quantize_tokens makes them.
template <int DT>
__device__ __forceinline__ void route_quantize(const MoeParams& p, int token) {
  __shared__ uint32_t scratch[8];
  const bf16* row = p.x + static_cast<long long>(token) * p.hidden;
  uint8_t* codes = p.xq + static_cast<long long>(token) * code_bytes<DT>(p.hidden);
  const int lanes = p.sub >> 3, groups = p.sub ? (p.hidden + p.sub - 1) / p.sub : 1;
  float s = 1.f;
  if (!lanes) {
    uint32_t m = 0;
    for (int at = threadIdx.x * 8; at < p.hidden; at += 2048) {
      Raw8<bf16> raw;
      raw.load<true>(row, at, p.hidden);
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __vmaxu2(m, raw.w[i] & 0x7FFF7FFFu);
    }
    s = scale_of_bf16<DT>(row_reduce<256>(max(m & 0xFFFFu, m >> 16), MaxOp(), scratch));
    if (threadIdx.x == 0) p.xs[token] = s;
  }
  for (int base = 0; base < p.hidden; base += 2048) {
    const int at = base + threadIdx.x * 8;
    Raw8<bf16> raw;
    raw.load<true>(row, at, p.hidden);
    if (lanes) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __vmaxu2(m, raw.w[i] & 0x7FFF7FFFu);
      s = scale_of_bf16<DT>(warp_reduce(max(m & 0xFFFFu, m >> 16), MaxOp(), lanes));
      if ((threadIdx.x & (lanes - 1)) == 0 && at < p.hidden) p.xs[token * groups + (at >> p.sub_bits)] = s;
    }
    uint32_t c[8];
    if (scale_is_ordinary(s)) {
      const ExactQuotient q(s);
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = q.code(raw.get(i));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = code_by_division<DT>(raw.get(i), s);
    }
    store_codes<DT, true>(codes, at, p.hidden, c);
  }
}

// Blocks [0, tokens): a token's codes.  The others: logits of four experts for up to four tokens.  The sums are in fp64, so
// that the choice of experts does not hang on the order of a sum.  Latency: 2 us for one token and 64 experts of 2048.
template <int DT>
__global__ void __launch_bounds__(256) moe_route_kernel(const MoeParams p) {
  grid_release();
  const int b = blockIdx.x;
  if (b == 0 && threadIdx.x < 2) p.active[2 + threadIdx.x] = 0;  // few tokens; else the select kernel does it
  if (b < p.tokens) {
    route_quantize<DT>(p, b);
  } else if (p.router_f32) {
    route_logits<float>(p, b - p.tokens);
  } else {
    route_logits<bf16>(p, b - p.tokens);
  }
}

// fp64 numbers as whole numbers in the same order: 0 stands for "taken", 1 for NaN, which is below everything.
__device__ __forceinline__ unsigned long long logit_key(double v) {
  if (!(v == v)) return 1ull;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));  // -0 becomes 0
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double logit_of_key(unsigned long long k) {
  if (k == 1ull) return __longlong_as_double(0x7FF8000000000000LL);
  return __longlong_as_double(static_cast<long long>((k >> 63) ? (k & 0x7FFFFFFFFFFFFFFFull) : ~k));
}

// A warp picks a token's experts one after the other: the largest logit that is left, ties to the lowest index (a token
// whose logits are NaN gets the first experts).  A lane keeps PER logits, of experts lane, lane + 32, ...; lane j
// hands choice j on.
template <int PER, typename Take>
__device__ __forceinline__ void pick_experts(const MoeParams& p, int token, Take&& take) {
  const int lane = threadIdx.x & 31;
  unsigned long long key[PER], mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    key[i] = e < p.experts ? logit_key(__ldcg(p.logits + static_cast<long long>(token) * p.experts + e)) : 0ull;
  }
  int mine_id = -1;
#pragma unroll 1
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long best = 0;
    unsigned best_id = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] > best) {
        best = key[i];
        best_id = lane + 32 * i;
      }
    const unsigned hi = static_cast<unsigned>(best >> 32), lo = static_cast<unsigned>(best);
    const unsigned top_hi = __reduce_max_sync(0xFFFFFFFFu, hi);
    const unsigned top_lo = __reduce_max_sync(0xFFFFFFFFu, hi == top_hi ? lo : 0u);
    const unsigned id = __reduce_min_sync(0xFFFFFFFFu, hi == top_hi && lo == top_lo ? best_id : 0xFFFFFFFFu);
    if (lane == j) {
      mine = (static_cast<unsigned long long>(top_hi) << 32) | top_lo;
      mine_id = static_cast<int>(id);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (id == static_cast<unsigned>(lane + 32 * i)) key[i] = 0;
  }
  if (lane < p.top_k) take(lane, mine_id, logit_of_key(mine));
}

// The expert that the caller gives a pair; -1 for a number that is none.
__device__ __forceinline__ int given_expert(const MoeParams& p, int pair) {
  const long long id = p.ids_64 ? static_cast<const long long*>(p.ids_in)[pair] : static_cast<const int*>(p.ids_in)[pair];
  return id >= 0 && id < p.experts ? static_cast<int>(id) : -1;
}

// One block: picks the experts, and lists each one's pairs.  Latency: 3.5 us for 13 tokens and 64 experts.
template <int PER, int THREADS>
__global__ void __launch_bounds__(THREADS) moe_select_kernel(const MoeParams p) {
  __shared__ int chosen[kMoeMaxPairs];
  __shared__ int count[PER * 32];
  __shared__ int first[PER * 32];
  __shared__ int2 warp_sums[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = p.tokens * p.top_k;
  for (int e = threadIdx.x; e < PER * 32; e += THREADS) count[e] = 0;
  grid_wait();
  grid_release();
  if (p.router != nullptr) {
    for (int t = warp; t < p.tokens; t += THREADS / 32) {
      pick_experts<PER>(p, t, [&](int choice, int expert, double logit) {
        chosen[t * p.top_k + choice] = expert;
        p.pair_logit[t * p.top_k + choice] = logit;
      });
    }
  } else {
    for (int i = threadIdx.x; i < pairs; i += THREADS) {
      chosen[i] = given_expert(p, i);
    }
  }
  __syncthreads();
  constexpr int kPerThread = (kMoeMaxPairs + THREADS - 1) / THREADS;
  int place[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int i = threadIdx.x + k * THREADS;
    place[k] = i < pairs && chosen[i] >= 0 ? atomicAdd(&count[chosen[i]], 1) : 0;  // the order within an expert changes no result
  }
  __syncthreads();
  // scan over the experts, THREADS at a time: pairs (low half) and experts in use (high half) before, and their passes
  int2 carry = make_int2(0, 0);
  for (int base = 0; base < PER * 32; base += THREADS) {
    const int e = base + threadIdx.x, mine = e < PER * 32 ? count[e] : 0;
    const int2 here = make_int2(mine + (mine > 0 ? 1 << 16 : 0), (mine + p.rows_a_pass - 1) / p.rows_a_pass);
    int2 sum = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xFFFFFFFFu, sum.x, o), y = __shfl_up_sync(0xFFFFFFFFu, sum.y, o);
      if (lane >= o) {
        sum.x += x;
        sum.y += y;
      }
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    int2 total = make_int2(0, 0);
    for (int w = 0; w < THREADS / 32; ++w) {
      const int2 other = warp_sums[w];
      if (w < warp) {
        sum.x += other.x;
        sum.y += other.y;
      }
      total.x += other.x;
      total.y += other.y;
    }
    if (mine > 0) {
      const int before = carry.x + sum.x - here.x;
      first[e] = before & 0xFFFF;
      *reinterpret_cast<int4*>(p.active + 4 + 4 * (before >> 16)) = make_int4(e, before & 0xFFFF, mine, carry.y + sum.y - here.y);
    }
    carry.x += total.x;
    carry.y += total.y;
    __syncthreads();
  }
  if (threadIdx.x == 0) *reinterpret_cast<int4*>(p.active) = make_int4(carry.x >> 16, carry.y, 0, 0);
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int i = threadIdx.x + k * THREADS;
    if (i >= pairs) break;
    p.pair_expert[i] = chosen[i];
    if (chosen[i] >= 0) p.pair_list[first[chosen[i]] + place[k]] = i;
    if (p.ids_out != nullptr) p.ids_out[i] = chosen[i];
  }
}

// The same within a block of the products of few tokens.  An expert's pairs go into slots of eight, in order, so that
// every block makes the same ones.
struct MoeFewChoice {
  double logit[kMoeFewPairs];
  int expert[kMoeFewPairs];        // of a pair
  int slot_expert[kMoeFewPairs];
  alignas(4) uint8_t list[kMoeFewPairs * 8];  // the pairs of each slot
  uint8_t slot_pairs[kMoeFewPairs];
  uint8_t slot_of[kMoeFewPairs];   // of a pair that begins one
  int turn[kMoeFewPairs / 32], in_use;
};

__device__ __forceinline__ void choose_few(const MoeParams& p, MoeFewChoice& few) {
  const int pairs = p.tokens * p.top_k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.router != nullptr) {
    auto take = [&](int choice, int expert, double logit) {
      few.expert[warp * p.top_k + choice] = expert;
      few.logit[warp * p.top_k + choice] = logit;
    };
    if (warp < p.tokens) {
      if (p.experts <= 64) pick_experts<2>(p, warp, take);
      else pick_experts<kMoeFewExperts / 32>(p, warp, take);
    }
  } else if (threadIdx.x < pairs) {
    few.expert[threadIdx.x] = given_expert(p, threadIdx.x);
  }
  __syncthreads();
  const int i = threadIdx.x, mine = i < pairs ? few.expert[i] : -1;
  int all = 0, before = 0, leader = i;  // pairs of the same expert; those before this one; the first of its eight
#pragma unroll 4
  for (int j = 0; j < pairs; ++j) {
    if (few.expert[j] != mine) continue;
    if (j <= i && (all & 7) == 0) leader = j;
    before += j < i;
    ++all;
  }
  const bool leads = mine >= 0 && leader == i;
  const unsigned leaders = __ballot_sync(0xFFFFFFFFu, leads);
  if (lane == 0 && warp < kMoeFewPairs / 32) few.turn[warp] = __popc(leaders);
  __syncthreads();
  int slot = __popc(leaders & ((1u << lane) - 1u)), total = 0;
#pragma unroll
  for (int w = 0; w < kMoeFewPairs / 32; ++w) {
    if (w < warp) slot += few.turn[w];
    total += few.turn[w];
  }
  if (leads) {
    few.slot_expert[slot] = mine;
    few.slot_pairs[slot] = static_cast<uint8_t>(min(8, all - before));
    few.slot_of[i] = static_cast<uint8_t>(slot);
  }
  if (i == 0) few.in_use = total;
  __syncthreads();
  if (mine >= 0) few.list[few.slot_of[leader] * 8 + (before & 7)] = static_cast<uint8_t>(i);
}

// ---------------------------------------------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_i8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// BYTES of global memory to shared memory, or zeros.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool valid) {
  const int size = valid ? BYTES : 0;
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(size) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

template <int WORDS>
__device__ __forceinline__ void read_words(uint32_t (&w)[4], const uint8_t* p) {
  if (WORDS == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

__device__ __forceinline__ uint32_t even_codes(uint32_t w) { return (w << 4) & 0xF0F0F0F0u; }
__device__ __forceinline__ uint32_t odd_codes(uint32_t w) { return w & 0xF0F0F0F0u; }

// Two 16 x 16 byte matrices, transposed: lane (g, q) gets bytes 4 q .. 4 q + 3 of columns g and g + 8 of each.
__device__ __forceinline__ void load_transposed(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}

// Sums over K: exact integers, or (a scale for each group of K) scaled ones.
template <bool SC>
struct MoeSum {
  using type = int;
};
template <>
struct MoeSum<true> {
  using type = double;
};

constexpr int kMoeThreads = 256;
constexpr int kMoeWarps = kMoeThreads / 32;

// A block works on a range of columns at a time: 64 (K-major weights, NT) or 128 (N-major, NN), for up/gate half of
// them up columns and half the same columns of the gate.  Its eight warps divide K into four shares and the
// columns into halves; a warp has two or four fragments of 16 columns.  (NT: two, with 64 bytes of each column a step in
// 16-byte copies.  Four, with 32 bytes in 8-byte copies, kept HBM at a third of its rate.)
// A step is 4 * WORDS * (8 or 4) values of K, of which lane q of a quad has WORDS consecutive words of the token codes.
// NT: and the same words of each column.  NN: rows of 64 columns, which ldmatrix transposes; the row that a lane names
// for it puts the right values of K into each quad's words.
// One stage of a warp's ring: weights, token codes, and (SC) the scales of the step's group of K.
template <int DT, bool NN, bool SC, int WORDS, int kN>
struct MoeStage {
  static constexpr int kFrags = NN ? 4 : 2, kHalves = 2, kCols = kHalves * kFrags * 16, kShares = kMoeWarps / kHalves;
  static constexpr int kStepK = 4 * WORDS * (DT == 4 ? 8 : 4), kStepBytes = 16 * WORDS;  // of a column
  static constexpr int kWeights = kFrags * 16 * kStepBytes;                              // bytes
  static constexpr int kCodeBytes = 4 * WORDS;                                           // of a token, by a lane
  static constexpr int kScalesAt = kWeights + kN * 32 * kCodeBytes;
  static constexpr int kRowScalesAt = kScalesAt + (SC ? kFrags * 32 : 0);
  static constexpr int kBytes = kRowScalesAt + (SC ? kN * 8 * 4 : 0);
  using Sum = typename MoeSum<SC>::type;
  // integers are added in place; fp64 numbers by two shares at a time, each pair's first to one half, second to the other
  static constexpr int kSums = kFrags * kHalves * kN * 4 * 32;
  static constexpr int kSumParts = SC ? 2 : 1, kSumBytes = kSums * kSumParts * static_cast<int>(sizeof(Sum));
  // blocks an SM, by registers, and a ring that fills their part of its shared memory
  static constexpr int kResident = SC || kN >= 3 || (!NN && kN == 2) ? 2 : 3;
  static constexpr int kFit = ((kResident == 3 ? 74 : 110) * 1024 - kSumBytes) / kMoeWarps / kBytes;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static_assert(kStages >= 3, "two steps have to be on their way while one is worked on");
  static constexpr int kRingBytes = kMoeWarps * kStages * kBytes;
  static constexpr int kSmemBytes = kRingBytes + kSumBytes;
};

// int32 -> fp64 without a conversion instruction (16 a clock and SM; the subtraction runs at 64): 2^52 + 2^31 + v, bit
// by bit, minus 2^52 + 2^31.
__device__ __forceinline__ double exact_double(int v) {
  return __hiloint2double(0x43300000, v ^ 0x80000000) - 4503601774854144.0;
}

// Where the sum of fragment `frag` (of the block), token group n and result j of a lane lies: spread over the banks.
template <int kN>
__device__ __forceinline__ int sum_place(int frag, int n, int j, int lane) {
  return (((frag * kN + n) * 4 + j) << 5) + (lane ^ ((frag * 4 + j) & 31));
}

// Quantises the activations of one pair (fp64 in, as they were computed): what quantize_tokens does, with values that
// are not exactly known in fp32, so that a code is settled against them where it has to be.  The row is divided among
// all threads, V pairs of values each, held in registers (V == 0: read again); or a group of values belongs to a warp.
constexpr int kMoeQuantThreads = 512;  // 1.5 us for one token of 1408 activations, 3 for 128 pairs of 14336

template <int DT, int V>
__global__ void __launch_bounds__(kMoeQuantThreads) moe_quantize_kernel(const MoeParams p) {
  constexpr double kTop = DT == 4 ? 7.0 : 127.0;
  constexpr int kWarps = kMoeQuantThreads / 32;
  __shared__ unsigned long long warp_max[kWarps];
  grid_release();  // so that the down product's first weights are on their way while the up/gate product ends
  grid_wait();
  const int pair = blockIdx.x;
  if (p.pair_expert[pair] < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const double* row = p.act + static_cast<long long>(pair) * p.inner;
  uint8_t* codes = p.aq + static_cast<long long>(pair) * code_bytes<DT>(p.inner);
  auto largest = [](unsigned long long most, double2 v) {
    const unsigned long long a = __double_as_longlong(v.x) & 0x7FFFFFFFFFFFFFFFLL, b = __double_as_longlong(v.y) & 0x7FFFFFFFFFFFFFFFLL;
    return max(most, max(a, b));
  };
  auto scale_of = [&](unsigned long long most) { return nonzero_scale(bf16_from_double(__longlong_as_double(most) / kTop)); };
  // Codes of two values; bit `bit` of `border` is set where one of them has to be settled.  (Settling them here would
  // put a division into every step of an unrolled loop: code that runs once, and is fetched for longer than it runs.)
  auto put = [&](int c, double2 v, float inv, uint32_t& border, int bit) {
    const float delta = static_cast<float>(kTop) * 4.76837158203125e-7f;  // fp32 value, product: 3 roundings
    const float x = static_cast<float>(v.x), y = static_cast<float>(v.y);
    const uint32_t a = __float_as_uint(__fadd_rn(__fmaf_rn(x, inv, -delta), kRoundMagic)), b = __float_as_uint(__fadd_rn(__fmaf_rn(y, inv, -delta), kRoundMagic));
    if (((a ^ __float_as_uint(__fadd_rn(__fmaf_rn(x, inv, delta), kRoundMagic))) | (b ^ __float_as_uint(__fadd_rn(__fmaf_rn(y, inv, delta), kRoundMagic)))) != 0)
      border |= 1u << bit;
    if (DT == 4) codes[c / 2] = static_cast<uint8_t>((a & 0xFu) | ((b & 0xFu) << 4));
    else *reinterpret_cast<uint16_t*>(codes + c) = static_cast<uint16_t>((a & 0xFFu) | ((b & 0xFFu) << 8));
  };
  auto settle = [&](int c, float s) {
    const double2 v = *reinterpret_cast<const double2*>(row + c);
    uint32_t code[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double quotient = rint((i ? v.y : v.x) / static_cast<double>(s));
      code[i] = s < __int_as_float(0x7F800000) ? static_cast<uint32_t>(static_cast<int>(fmin(fmax(quotient, -kTop), kTop))) : 0u;
    }
    if (DT == 4) codes[c / 2] = static_cast<uint8_t>((code[0] & 0xFu) | ((code[1] & 0xFu) << 4));
    else *reinterpret_cast<uint16_t*>(codes + c) = static_cast<uint16_t>((code[0] & 0xFFu) | ((code[1] & 0xFFu) << 8));
  };
  // the settling of the values c + 2 i stride that `border` names (all of them where the scale is not ordinary)
  auto settle_all = [&](uint32_t border, int c, int step, int count, float s) {
    if (!scale_is_ordinary(s)) border = 0xFFFFFFFFu >> (32 - count);
#pragma unroll 1
    for (; border != 0; border &= border - 1) {
      const int i = __ffs(border) - 1;
      settle(c + i * step, s);
    }
  };
  if (p.sub) {
    const int groups = (p.inner + p.sub - 1) / p.sub;
    for (int group = warp; group < groups; group += kWarps) {
      const int c0 = group * p.sub + lane * 2, c1 = min((group + 1) * p.sub, p.inner);
      double2 v[4];  // up to 256 values
      unsigned long long most = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = c0 + 64 * i < c1 ? *reinterpret_cast<const double2*>(row + c0 + 64 * i) : make_double2(0.0, 0.0);
        most = largest(most, v[i]);
      }
      const float s = scale_of(warp_reduce(most, MaxOp()));
      if (lane == 0) p.as[static_cast<long long>(pair) * groups + group] = s;
      const float inv = __frcp_rn(s);
      uint32_t border = 0;
      int count = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c0 + 64 * i < c1) {
          put(c0 + 64 * i, v[i], inv, border, i);
          ++count;
        }
      if (count > 0) settle_all(border, c0, 64, count, s);
    }
    return;
  }
  const int c0 = threadIdx.x * 2, stride = kMoeQuantThreads * 2;
  double2 v[V > 0 ? V : 1];
  unsigned long long most = 0;
  if (V > 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] = c0 + i * stride < p.inner ? *reinterpret_cast<const double2*>(row + c0 + i * stride) : make_double2(0.0, 0.0);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) most = largest(most, v[i]);
  } else {
#pragma unroll 4
    for (int c = c0; c < p.inner; c += stride) most = largest(most, *reinterpret_cast<const double2*>(row + c));
  }
  most = warp_reduce(most, MaxOp());
  if (lane == 0) warp_max[warp] = most;
  __syncthreads();
  const float s = scale_of(warp_reduce(warp_max[lane % kWarps], MaxOp()));
  if (threadIdx.x == 0) p.as[pair] = s;
  const float inv = __frcp_rn(s);
  if (V > 0) {
    uint32_t border = 0;
    int count = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c0 + i * stride < p.inner) {
        put(c0 + i * stride, v[i], inv, border, i);
        ++count;
      }
    if (count > 0) settle_all(border, c0, stride, count, s);
  } else {
    for (int c = c0; c < p.inner; c += stride) {
      uint32_t border = 0;
      put(c, *reinterpret_cast<const double2*>(row + c), inv, border, 0);
      settle_all(border, c, stride, 1, s);
    }
  }
}

// A unit of work: a column range of an expert in use, for one part of K and up to 8 kMaxN of its rows.
struct MoeUnit {
  int first, here;    // its pairs: list + first, `here` of them
  int range, split;
  int expert;
  int begin, mine;    // steps of K of this warp: begin, begin + by, ...
};

// What a lane reads of the weights of a unit, at its warp's first step.
struct MoeSource {
  const uint8_t* w;
  const bf16* scale;  // of its columns in the first group of K
  bool valid, scale_valid;
};

// The grid is as large as the device holds at once.  Units are handed out in order, so that blocks that run at the same
// time read neighbouring columns (a row of N-major weights in long pieces) and light and heavy ones even out: a block's
// first two by its number, the others by a counter, two units ahead of their use.  When a warp has done the last step
// of a unit it starts the copies of its weights of the next one, before the sums are finished.
// kMaxN: groups of eight tokens that a pass over the weights can serve; more tokens of an expert take more passes.
// kChoose: the blocks pick the experts themselves.
// 64 tokens, two of 8 experts of 4096 x 14336 in int4: 470 MB of up/gate weights in 102 us (4.6 TB/s), then 235 MB in 54; the
// blocks issue in half of the cycles and wait for copies in most others: 16 warps an SM is what the sums of 24 rows leave
// room for.  With K-group scales (13 tokens, 6 of 64 experts of 2048 x 1408, groups of 128): 134 MB in 35 us, with 230
// instructions a step of eight tensor-core products where the plain sums take 145, and half as many again for what a
// warp does once a unit (eight steps).
template <int DT, bool NN, bool SC, int WORDS, int kMaxN, bool kChoose, bool kDown>
__global__ void __launch_bounds__(kMoeThreads, MoeStage<DT, NN, SC, WORDS, kMaxN>::kResident) moe_product_kernel(const MoeParams p) {
  using Stage = MoeStage<DT, NN, SC, WORDS, kMaxN>;
  using Sum = typename Stage::Sum;
  constexpr int kFrags = Stage::kFrags, kStages = Stage::kStages, kAllFrags = kFrags * Stage::kHalves, kShares = Stage::kShares;
  constexpr int kStepBytes = Stage::kStepBytes, kStepK = Stage::kStepK, kStepBits = kStepK == 128 ? 7 : kStepK == 64 ? 6 : 5, kCols = Stage::kCols, out_cols = kDown ? kCols : kCols / 2;
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kHead = kChoose ? kMoeFewPairs : 64;  // slots whose records are at hand
  __shared__ int4 head[1 + kHead];
  __shared__ __align__(4) uint8_t list[kChoose ? kMoeFewPairs * 8 : 4];
  __shared__ int rows[2][kMaxN * 8], pair_of[2][kMaxN * 8];
  __shared__ float row_scale[2][kMaxN * 8];
  __shared__ int unit_after_next;
  if (!kDown) {
    grid_wait();
    grid_release();
  }
  // The down product reads before it waits: the logits, or the select kernel's records, which were there before the up/gate
  // product let the next kernels start.
  const int4* records = reinterpret_cast<const int4*>(p.active);
  if constexpr (kChoose) {
    MoeFewChoice& few = *reinterpret_cast<MoeFewChoice*>(smem);  // in the ring, which is not in use yet
    static_assert(sizeof(MoeFewChoice) <= Stage::kRingBytes, "the choice of experts has to fit the ring");
    choose_few(p, few);
    __syncthreads();
    const int i = threadIdx.x;
    if (i == 0) head[0] = make_int4(few.in_use, few.in_use, 0, 0);
    if (i < few.in_use) head[1 + i] = make_int4(few.slot_expert[i], i * 8, few.slot_pairs[i], i);
    *reinterpret_cast<uint32_t*>(list + i * 4) = *reinterpret_cast<const uint32_t*>(few.list + i * 4);
    if (!kDown && blockIdx.x == 0 && i < p.tokens * p.top_k) {
      p.pair_expert[i] = few.expert[i];
      if (p.router != nullptr) p.pair_logit[i] = few.logit[i];
      if (p.ids_out != nullptr) p.ids_out[i] = few.expert[i];
    }
  } else if (threadIdx.x < min(1 + kHead, 1 + p.slots)) {
    head[threadIdx.x] = __ldcg(records + threadIdx.x);
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int half = warp & 1, share = warp >> 1;
  const int k = kDown ? p.inner : p.hidden, columns = kDown ? p.hidden : 2 * p.inner, gate = p.inner;  // gate columns start there
  const int out_n = kDown ? p.hidden : p.inner, ranges = kDown ? p.down_ranges : p.up_ranges, splits = kDown ? p.down_splits : 1;
  const int groups = SC ? (k + p.sub - 1) / p.sub : 1, steps = (k + kStepK - 1) / kStepK;
  const long long code_pitch = code_bytes<DT>(k);
  const uint8_t* all_codes = kDown ? p.aq : p.xq;
  const float* all_scales = kDown ? p.as : p.xs;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * kStages * Stage::kBytes;
  const uint8_t* ring = smem + warp * kStages * Stage::kBytes;
  Sum* sums = reinterpret_cast<Sum*>(smem + Stage::kRingBytes);
  if constexpr (!SC)  // integers are added to what lies here
    for (int i = threadIdx.x; i < Stage::kSums; i += kMoeThreads) sums[i] = 0;
  __syncthreads();
  const int in_use = head[0].x, units = head[0].y * splits * ranges;
  int* counter = p.active + (kDown ? 3 : 2);

  // A share's steps.  NN: consecutive ones (whole groups of K as far as it goes).  NT: a group's of every fourth group of
  // K, or every fourth step, so that the four read a row in one long piece.
  const int run_bits = SC && !NN ? p.sub_bits - kStepBits : 0;
  auto step_of = [&](const MoeUnit& unit, int i) {
    if (NN) return unit.begin + i;
    return unit.begin + ((i >> run_bits) << run_bits) * kShares + (i & ((1 << run_bits) - 1));
  };
  auto group_of = [&](int step) { return (step << kStepBits) >> p.sub_bits; };
  auto decode = [&](int u) {
    MoeUnit unit;
    const int pass = u / (splits * ranges), rest = u - pass * splits * ranges;
    unit.split = splits == 1 ? 0 : rest / ranges;
    unit.range = rest - unit.split * ranges;
    int low = 0, high = in_use;  // the last slot whose passes start at or before this one
    auto record = [&](int slot) { return slot < kHead ? head[1 + slot] : __ldcg(records + 1 + slot); };
    while (high - low > 1) {
      const int middle = (low + high) >> 1;
      if (record(middle).w <= pass) low = middle;
      else high = middle;
    }
    const int4 r = record(low);
    const int done = (pass - r.w) * kMaxN * 8;
    unit.expert = r.x;
    unit.first = r.y + done;
    unit.here = min(kMaxN * 8, r.z - done);
    const int step0 = steps * unit.split / splits, count = steps * (unit.split + 1) / splits - step0;
    if (NN) {
      const int per_share = (count + kShares - 1) / kShares;
      unit.begin = step0 + share * per_share;
      unit.mine = max(0, min(count - share * per_share, per_share));
    } else {
      const int run = 1 << run_bits, rounds = count >> run_bits, rest = count - (rounds / kShares * kShares << run_bits);
      unit.begin = step0 + (share << run_bits);
      unit.mine = (rounds / kShares << run_bits) + max(0, min(rest - (share << run_bits), run));
    }
    return unit;
  };
  // first column of a fragment of this warp in a range, and whether the matrix has it (16 columns at a time)
  auto column_of = [&](int range, int f) {
    const int frag = half * kFrags + f;
    if (kDown) return range * kCols + frag * 16;
    return frag < kAllFrags / 2 ? range * (kCols / 2) + frag * 16 : gate + range * (kCols / 2) + (frag - kAllFrags / 2) * 16;
  };
  auto column_valid = [&](int range, int f) {
    if (kDown) return column_of(range, f) < columns;
    return range * (kCols / 2) + (half * kFrags + f) % (kAllFrags / 2) * 16 < gate;
  };
  const long long w_step = static_cast<long long>(kStepBytes) * columns;                           // NN: to the next step
  const long long w_rows = NN ? 8LL * columns : 8 * code_pitch;                                    // to the next of a lane's loads
  const uint8_t* all_weights = kDown ? p.w_down : p.w_up_gate;
  const bf16* all_weight_scales = kDown ? p.s_down : p.s_up_gate;
  auto source_of = [&](const MoeUnit& unit) {
    MoeSource source;
    const uint8_t* matrix = all_weights + static_cast<long long>(unit.expert) * columns * code_pitch;
    const bf16* scales = all_weight_scales + static_cast<long long>(unit.expert) * columns * groups;
    source.valid = source.scale_valid = true;
    source.scale = scales;
    if constexpr (NN) {
      source.valid = column_valid(unit.range, lane & 3);
      source.w = matrix + (source.valid ? column_of(unit.range, lane & 3) : 0) + (static_cast<long long>(unit.begin) * kStepBytes + (lane >> 2)) * columns;
      if (SC) {
        source.scale_valid = column_valid(unit.range, lane >> 3);
        source.scale = scales + (source.scale_valid ? column_of(unit.range, lane >> 3) + (lane & 7) * 2 : 0);
      }
    } else {
      // sizes are multiples of 32: both fragments are there, or none
      source.valid = source.scale_valid = column_valid(unit.range, 0);
      source.w = matrix + (column_of(unit.range, 0) + g) * code_pitch + static_cast<long long>(unit.begin) * kStepBytes + q * 4 * WORDS;
      source.scale = scales + (source.scale_valid ? column_of(unit.range, (lane >> 3) & 1) + (lane & 7) * 2 : 0);
    }
    return source;
  };
  // step `i` of a warp's steps of a unit; for NN source.w moves on with every call.  Nothing is read where `valid` is false
  // (the copy's size is zero), whatever the address is.
  auto copy_weights = [&](const MoeUnit& unit, MoeSource& source, int i, int slot) {
    const uint32_t at = ring_at + slot * Stage::kBytes;
    const int step = step_of(unit, i);
    if constexpr (NN) {
      // 16 bytes of row r and fragment f to place r * 4 + (f ^ (r / 2 % 4)): eight rows of a fragment on eight banks
      const uint8_t* src = source.w;
      const uint32_t to = at + ((lane >> 2) * 4 + ((lane & 3) ^ ((lane >> 3) & 3))) * 16;
      // the last step may reach beyond K, which is a multiple of 32: by whole groups of eight rows
      const int rows_left = static_cast<int>(code_pitch) - step * kStepBytes;
#pragma unroll
      for (int l = 0; l < kStepBytes / 8; ++l, src += w_rows) {
        const bool valid = source.valid && l * 8 < rows_left;
        copy_async<16>(to + l * 512, src, valid);
      }
      source.w += w_step;
    } else {
      const bool in_k = step * kStepK + q * (kStepK / 4) < k;
#pragma unroll
      for (int l = 0; l < 2 * kFrags; ++l) {
        const bool valid = in_k && source.valid;  // columns g and g + 8 of fragment l / 2
        const uint8_t* src = source.w + (step - unit.begin) * kStepBytes + ((l & 1) ? w_rows : 0) + ((l & 2) ? 2 * w_rows : 0);
        copy_async<4 * WORDS>(at + (l * 32 + lane) * 4 * WORDS, src, valid);
      }
    }
    if constexpr (SC) {
      const long long group = static_cast<long long>(group_of(step)) * columns;
      if (lane < kFrags * 8) copy_async<4>(at + Stage::kScalesAt + lane * 4, source.scale + group, source.scale_valid);
    }
  };
  // the pairs of a unit: read by its first threads, written down when the buffer is free
  auto read_pair = [&](const MoeUnit& unit) {
    if (threadIdx.x >= unit.here) return 0;
    if constexpr (kChoose) return static_cast<int>(list[unit.first + threadIdx.x]);
    else return __ldcg(p.pair_list + unit.first + threadIdx.x);
  };
  auto write_pair = [&](const MoeUnit& unit, int pair, int buffer) {
    if (threadIdx.x < unit.here) {
      const int row = kDown ? pair : pair / p.top_k;
      pair_of[buffer][threadIdx.x] = pair;
      rows[buffer][threadIdx.x] = row;
    }
  };

  MoeUnit unit, next;
  MoeSource source{};
  int slot = 0;        // of the ring: the stage of the step that is worked on
  int buffer = 0;
  int number = blockIdx.x, next_number = blockIdx.x + gridDim.x;
  if (number < units) {
    unit = decode(number);
    source = source_of(unit);
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i)
      if (i < unit.mine) copy_weights(unit, source, i, i);
  }
  if (kDown) {
    grid_wait();
    grid_release();
  }
  if (number >= units) return;
  write_pair(unit, read_pair(unit), 0);
  __syncthreads();
  const int c = threadIdx.x % out_cols;  // a thread's outputs are all of one column of a range

  while (true) {
    const bool more = next_number < units;
    const int col = unit.range * out_cols + c;
    int handed_out = 0, next_pair = 0;
    float my_scale = 0.f;
    float2 scale = make_float2(0.f, 0.f);
    // what comes later, asked for while the first copies are on their way
    auto look_ahead = [&]() {
      if (threadIdx.x == 0) handed_out = atomicAdd(counter, 1) + 2 * static_cast<int>(gridDim.x);
      if (!SC && !kDown) {
        if (threadIdx.x < unit.here) my_scale = __ldcg(all_scales + rows[buffer][threadIdx.x]);
        if (col < out_n) {
          const bf16* scales = all_weight_scales + static_cast<long long>(unit.expert) * columns + col;
          scale = make_float2(to_f32(scales[0]), to_f32(scales[p.inner]));
        }
      }
      if (more) {
        next = decode(next_number);
        next_pair = read_pair(next);
      }
    };

    auto products = [&](auto n_groups) {
      constexpr int kN = decltype(n_groups)::value;
      const uint8_t* codes[kN];  // of this lane's tokens, at its first step
      bool has_token[kN];
      const float* token_scale = all_scales;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        has_token[n] = n * 8 + g < unit.here;
        codes[n] = all_codes + (has_token[n] ? rows[buffer][n * 8 + g] * code_pitch : 0) + static_cast<long long>(unit.begin) * kStepBytes + q * 4 * WORDS;
      }
      if (SC && lane < unit.here && lane < kN * 8) token_scale = all_scales + static_cast<long long>(rows[buffer][lane]) * groups;
      auto copy_codes = [&](int i, int to_slot) {
        const uint32_t at = ring_at + to_slot * Stage::kBytes;
        const int step = step_of(unit, i), offset = (step - unit.begin) * kStepBytes;
        const bool in_k = step * kStepK + q * (kStepK / 4) < k;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          const bool valid = in_k && has_token[n];
          copy_async<4 * WORDS>(at + Stage::kWeights + (n * 32 + lane) * 4 * WORDS, codes[n] + offset, valid);
        }
        if constexpr (SC) {
          if (lane < kN * 8) copy_async<4>(at + Stage::kRowScalesAt + lane * 4, token_scale + group_of(step), lane < unit.here);
        }
      };
      int ahead = slot;  // the stage that is copied to next
#pragma unroll 1
      for (int i = 0; i < kStages - 1; ++i) {
        if (i < unit.mine) copy_codes(i, ahead);
        copy_commit();
        if (++ahead == kStages) ahead = 0;
      }
      look_ahead();
      // Packed: a group's sum is below 2^22 in size (256 times 256 products of up to 56), and starts at the bits of 3, so
      // that it is an fp32 number as it stands: 3 + 2^-22 times the sum, less than 1 away from 3.
      constexpr int kAccZero = SC && DT == 4 ? 0x40400000 : 0;
      int acc[kFrags][kN][4];
      double sum[SC ? kFrags : 1][SC ? kN : 1][4];
#pragma unroll
      for (int f = 0; f < kFrags; ++f)
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[f][n][i] = kAccZero;
            if (SC) sum[f][n][i] = 0.0;
          }
      // What is worked on kStages - 1 steps later.  Before the products of a step or behind them: NT gains 2 % by the
      // first (one token 18.4 us, not 18.8), NN loses 1 % (64 tokens 173 us, not 171).
      auto copy_ahead = [&](int i) {
        if (i + kStages - 1 < unit.mine) {
          copy_weights(unit, source, i + kStages - 1, ahead);
          copy_codes(i + kStages - 1, ahead);
        }
        copy_commit();
        if (++ahead == kStages) ahead = 0;
      };
#pragma unroll 1
      for (int i = 0; i < unit.mine; ++i) {
        copy_wait<kStages - 2>();
        __syncwarp();  // what the other lanes have copied; and they have read the stage of a step ago
        if (!NN) copy_ahead(i);
        const uint8_t* stage = ring + slot * Stage::kBytes;
        uint32_t x[kN][4];
#pragma unroll
        for (int n = 0; n < kN; ++n) read_words<WORDS>(x[n], stage + Stage::kWeights + (n * 32 + lane) * 4 * WORDS);
        if constexpr (NN) {
          const uint32_t at = ring_at + slot * Stage::kBytes;
          // Row rho = 4 q' + i of a matrix holds byte i of a word of lane q' of each quad, which is row
          // q' * 4 * WORDS + (4 * word) + i of the stage.  Lanes 0 .. 15 name the rows of the first matrix, the others
          // those of the second: the same word of two fragments (packed), or two words of one (int8).
          const int rho = lane & 15, second = lane >> 4;
          const int row0 = (rho >> 2) * 4 * WORDS + (rho & 3);
          if constexpr (DT == 4) {
#pragma unroll
            for (int word = 0; word < WORDS; ++word) {
              const int r = row0 + 4 * word;
              const uint32_t line = at + r * 64;
              const int flip = (r >> 1) & 3;
              uint32_t even_x[kN], odd_x[kN];
#pragma unroll
              for (int n = 0; n < kN; ++n) {
                even_x[n] = even_codes(x[n][word]);
                odd_x[n] = odd_codes(x[n][word]);
              }
#pragma unroll
              for (int l = 0; l < kFrags / 2; ++l) {
                uint32_t m[4];
                load_transposed(m, line + (((2 * l + second) ^ flip) << 4));
#pragma unroll
                for (int n = 0; n < kN; ++n) mma_i8(acc[2 * l][n], even_codes(m[0]), even_codes(m[1]), odd_codes(m[0]), odd_codes(m[1]), even_x[n], odd_x[n]);
#pragma unroll
                for (int n = 0; n < kN; ++n) mma_i8(acc[2 * l + 1][n], even_codes(m[2]), even_codes(m[3]), odd_codes(m[2]), odd_codes(m[3]), even_x[n], odd_x[n]);
              }
            }
          } else {
#pragma unroll
            for (int word = 0; word < WORDS; word += 2) {
              const int r = row0 + 4 * (word + second);
              const uint32_t line = at + r * 64;
              const int flip = (r >> 1) & 3;
#pragma unroll
              for (int f = 0; f < kFrags; ++f) {
                uint32_t m[4];
                load_transposed(m, line + ((f ^ flip) << 4));
#pragma unroll
                for (int n = 0; n < kN; ++n) mma_i8(acc[f][n], m[0], m[1], m[2], m[3], x[n][word], x[n][word + 1]);
              }
            }
          }
        } else {
#pragma unroll
          for (int f = 0; f < kFrags; ++f) {
            uint32_t wa[4], wb[4];
            read_words<WORDS>(wa, stage + (2 * f * 32 + lane) * 4 * WORDS);
            read_words<WORDS>(wb, stage + ((2 * f + 1) * 32 + lane) * 4 * WORDS);
            if constexpr (DT == 4) {
#pragma unroll
              for (int j = 0; j < WORDS; ++j)
#pragma unroll
                for (int n = 0; n < kN; ++n)
                  mma_i8(acc[f][n], even_codes(wa[j]), even_codes(wb[j]), odd_codes(wa[j]), odd_codes(wb[j]), even_codes(x[n][j]), odd_codes(x[n][j]));
            } else {
#pragma unroll
              for (int j = 0; j < WORDS; j += 2)
#pragma unroll
                for (int n = 0; n < kN; ++n) mma_i8(acc[f][n], wa[j], wb[j], wa[j + 1], wb[j + 1], x[n][j], x[n][j + 1]);
            }
          }
        }
        if constexpr (SC) {
          // the integers of a group of K end here: scaled and added up in fp64 (a step lies in one group)
          const int next_step = step_of(unit, i) + 1;
          if (i + 1 == unit.mine || ((next_step << kStepBits) & (p.sub - 1)) == 0 || (!NN && ((i + 1) & ((1 << run_bits) - 1)) == 0)) {
            const uint16_t* w_scales = reinterpret_cast<const uint16_t*>(stage + Stage::kScalesAt);
            const float* row_scales = reinterpret_cast<const float*>(stage + Stage::kRowScalesAt);
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              const float2 st = *reinterpret_cast<const float2*>(row_scales + n * 8 + 2 * q);
              // (packed: the sums are 256 times too large, and 2^22 times too small)
              const double st0 = static_cast<double>(st.x) * (DT == 4 ? 16384.0 : 1.0), st1 = static_cast<double>(st.y) * (DT == 4 ? 16384.0 : 1.0);
#pragma unroll
              for (int f = 0; f < kFrags; ++f)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const float sw = __uint_as_float(static_cast<uint32_t>(w_scales[f * 16 + g + h * 8]) << 16);
                  int &a = acc[f][n][2 * h], &b = acc[f][n][2 * h + 1];
                  // 14 bits of the sum, 8 of the scale: exact in fp32.  For every scale: the factor, a multiple of 2^-14 below 1,
                  // makes no product larger than the scale, and of a multiple of 2^-133 (the least scale) one of 2^-147.
                  if (DT == 4) {
                    const Pair part = add2(Pair(__int_as_float(a), __int_as_float(b)), Pair(-3.f));
                    const float2 scaled = mul2(part, Pair(sw)).get();
                    sum[f][n][2 * h] = fma(static_cast<double>(scaled.x), st0, sum[f][n][2 * h]);
                    sum[f][n][2 * h + 1] = fma(static_cast<double>(scaled.y), st1, sum[f][n][2 * h + 1]);
                  } else {
                    sum[f][n][2 * h] = fma(exact_double(a), st0 * static_cast<double>(sw), sum[f][n][2 * h]);
                    sum[f][n][2 * h + 1] = fma(exact_double(b), st1 * static_cast<double>(sw), sum[f][n][2 * h + 1]);
                  }
                  a = b = kAccZero;
                }
            }
          }
        }
        if (NN) {
          __syncwarp();
          copy_ahead(i);
        }
        if (++slot == kStages) slot = 0;
      }
      // the next unit's first weights
      __syncwarp();
      if (more) {
        source = source_of(next);
        int to_slot = slot;
#pragma unroll 1
        for (int i = 0; i < kStages - 1; ++i) {
          if (i < next.mine) copy_weights(next, source, i, to_slot);
          if (++to_slot == kStages) to_slot = 0;
        }
      }
      if (!SC && !kDown && threadIdx.x < unit.here) row_scale[buffer][threadIdx.x] = my_scale;
      if (threadIdx.x == 0) unit_after_next = handed_out;
      if constexpr (!SC) {  // exact integers, in any order
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) atomicAdd(sums + sum_place<kMaxN>(half * kFrags + f, n, j, lane), DT == 4 ? acc[f][n][j] >> 8 : acc[f][n][j]);
        __syncthreads();
      } else {  // two shares after two others
        for (int turn = 0; turn < kShares / 2; ++turn) {
          if (share >> 1 == turn) {
#pragma unroll
            for (int f = 0; f < kFrags; ++f)
#pragma unroll
              for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  Sum* at = sums + (share & 1) * Stage::kSums + sum_place<kMaxN>(half * kFrags + f, n, j, lane);
                  *at = turn == 0 ? sum[f][n][j] : *at + sum[f][n][j];
                }
          }
          __syncthreads();
        }
      }
    };
    if (kMaxN == 1 || unit.here <= 8) products(std::integral_constant<int, 1>());
    else if (kMaxN == 2 || unit.here <= 16) products(std::integral_constant<int, kMaxN < 2 ? kMaxN : 2>());
    else if (unit.here <= 24) products(std::integral_constant<int, kMaxN < 3 ? kMaxN : 3>());
    else products(std::integral_constant<int, kMaxN>());

    if (col < out_n) {
      auto sum_of = [&](int t, bool gate_part) {
        const int column = c + (gate_part ? kCols / 2 : 0);
        const int place = sum_place<kMaxN>(column >> 4, t >> 3, ((column >> 3) & 1) * 2 + (t & 1), (column & 7) * 4 + ((t & 7) >> 1));
        Sum total = sums[place];
        if constexpr (SC) total += sums[Stage::kSums + place];
        else sums[place] = 0;  // for the next unit
        return total;
      };
      for (int t = threadIdx.x / out_cols; t < unit.here; t += kMoeThreads / out_cols) {
        if (kDown) {
          const long long pairs = static_cast<long long>(p.tokens) * p.top_k;
          static_cast<Sum*>(p.part)[(unit.split * pairs + rows[buffer][t]) * p.hidden + col] = sum_of(t, false);
        } else {
          double up = static_cast<double>(sum_of(t, false)), gated = static_cast<double>(sum_of(t, true));
          if (!SC) {
            const double s = static_cast<double>(row_scale[buffer][t]);
            up *= s * static_cast<double>(scale.x);  // exact; in fp32 it could be beyond the range, or below the least number
            gated *= s * static_cast<double>(scale.y);
          }
          p.act[static_cast<long long>(pair_of[buffer][t]) * p.inner + col] = up * gated / (1.0 + exp(-gated));
        }
      }
    }
    if (!more) break;
    write_pair(next, next_pair, buffer ^ 1);
    number = next_number;
    next_number = unit_after_next;
    unit = next;
    buffer ^= 1;
    __syncthreads();
  }
  copy_wait<0>();
}

// Adds up the parts of K, scales, and adds up the experts' shares of a token in the order of its choices, for 64 columns
// of one token.  A thread has two columns of one choice (two choices, beyond eight), whose share it leaves in shared memory:
// with all choices to a thread the unrolled code took longer to be fetched than to run (3.5 us behind the wait).  What
// depends on the pair alone is worked out once a block: the softmax of the chosen logits (or of all) in fp64.  What the
// choice of experts left and the scales are read before the down product has ended.
constexpr int kCombineLines = 8;

template <bool SC>
__global__ void __launch_bounds__(32 * kCombineLines) moe_combine_kernel(const MoeParams p) {
  using Sum = typename MoeSum<SC>::type;
  using Sum2 = typename std::conditional<SC, double2, int2>::type;
  constexpr int kEach = kMoeMaxTopK / kCombineLines;
  __shared__ float weight[kMoeMaxTopK];
  __shared__ bool counts[kMoeMaxTopK];  // a choice without an expert adds nothing, whatever its weight is
  __shared__ float2 share[kMoeMaxTopK][32];
  const int token = blockIdx.y, lane = threadIdx.x & 31, line = threadIdx.x >> 5, col = (blockIdx.x * 32 + lane) * 2;
  const bool inside = col < p.hidden;
  int expert[kEach];
  uint32_t w[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = line + i * kCombineLines;
    expert[i] = j < p.top_k ? __ldcg(p.pair_expert + token * p.top_k + j) : -1;
    if (lane == 0) counts[j] = expert[i] >= 0;
    w[i] = !SC && inside && expert[i] >= 0 ? *reinterpret_cast<const uint32_t*>(p.s_down + static_cast<long long>(expert[i]) * p.hidden + col) : 0u;
  }
  if (line == 0) {
    const int pair = token * p.top_k + min(lane, p.top_k - 1);
    float v;
    if (p.router != nullptr) {
      const double logit = __ldcg(p.pair_logit + pair), top = __shfl_sync(0xFFFFFFFFu, logit, 0);
      const double mine = lane < p.top_k ? exp(logit - top) : 0.0;
      double all = mine;
      if (!p.renormalize) {
        all = 0.0;
        for (int e = lane; e < p.experts; e += 32) all += exp(__ldcg(p.logits + static_cast<long long>(token) * p.experts + e) - top);
      }
      v = static_cast<float>(mine / warp_reduce(all, SumOp()));
    } else {
      v = p.weights_in[pair];
    }
    if (lane < p.top_k) {
      weight[lane] = v;
      if (p.weights_out != nullptr && blockIdx.x == 0) p.weights_out[pair] = v;
    }
  }
  grid_wait();
  const long long plane = static_cast<long long>(p.tokens) * p.top_k * p.hidden;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = line + i * kCombineLines, pair = token * p.top_k + j;
    if (!inside || expert[i] < 0) continue;
    const Sum2* at = reinterpret_cast<const Sum2*>(static_cast<const Sum*>(p.part) + static_cast<long long>(pair) * p.hidden + col);
    const float scale = SC ? 0.f : __ldcg(p.as + pair);
    Sum2 sum = __ldcg(at);
#pragma unroll 4
    for (int s = 1; s < p.down_splits; ++s) {
      const Sum2 more = __ldcg(at + s * (plane / 2));
      sum.x += more.x;
      sum.y += more.y;
    }
    double y0 = static_cast<double>(sum.x), y1 = static_cast<double>(sum.y);
    if (!SC) {
      y0 *= static_cast<double>(scale) * static_cast<double>(bf16_lo(w[i]));  // exact, as above
      y1 *= static_cast<double>(scale) * static_cast<double>(bf16_hi(w[i]));
    }
    share[j][lane] = make_float2(static_cast<float>(y0), static_cast<float>(y1));
  }
  __syncthreads();
  if (line > 0 || !inside) return;
  float x = 0.f, y = 0.f;
#pragma unroll 4
  for (int j = 0; j < p.top_k; ++j) {
    if (!counts[j]) continue;
    x = __fmaf_rn(share[j][lane].x, weight[j], x);
    y = __fmaf_rn(share[j][lane].y, weight[j], y);
  }
  bf16* out = p.out + static_cast<long long>(token) * p.hidden + col;
  out[0] = __float2bfloat16_rn(x);
  out[1] = __float2bfloat16_rn(y);
}

}  // namespace b200
