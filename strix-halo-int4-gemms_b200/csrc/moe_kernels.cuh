// A whole mixture-of-experts layer for a few tokens:
//   moe_route_kernel     router logits (fp64 sums), the tokens' codes and scales, counters set to zero
//   moe_select_kernel    top-k, softmax, and for each expert in use the list of its (token, choice) pairs
//   moe_product_kernel   up/gate product, SwiGLU; the last block of an expert quantises the activations
//   moe_product_kernel   down product; the last block of a column range adds the experts' shares for every token
//
// At a few tokens each weight is used by a handful of rows, so the layer is bound by reading the weights of the
// experts in use once from HBM.  The products therefore run on mma.sync.m16n8k32 (int8, exact int32 sums) with the
// WEIGHTS as the 16-row operand and up to eight tokens as the other: the weights go from global memory straight
// into the registers that feed the matrix instruction, with no stop in shared memory and no barrier in the loop.
// tcgen05 would want 128-row tiles of unpacked weights in shared memory; its rate is of no use here.
//
// Operand order.  A lane (g = lane / 4, q = lane % 4) supplies rows g and g + 8 of the 16 x 32 operand and, for
// each, K values that a quad of lanes divides up.  Which K a lane holds does not matter as long as both operands
// agree, so a lane takes consecutive packed bytes.  A word of eight nibbles is two words of the int8 operand: even
// K (w << 4) & 0xF0F0F0F0, odd K w & 0xF0F0F0F0, each value 16 times too large; the sum is 256 times too large and
// shifted right at the end, exactly.
#pragma once

#include <climits>

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
  int tokens, hidden, inner, experts, top_k, sub;
  int router_f32, ids_64, renormalize;
  // scratch
  uint8_t* xq;              // [tokens, hidden bytes]
  bf16* xs;                 // [tokens, groups of hidden]
  double* logits;           // [tokens, experts]
  int* pair_expert;         // [pairs], -1: no expert
  float* pair_weight;       // [pairs]
  int* active;              // [0]: experts in use; then slots of {expert, first, count}
  int* pair_list;           // [pairs], by expert
  double* act;              // [pairs, inner]
  uint8_t* aq;              // [pairs, inner bytes]
  bf16* as;                 // [pairs, groups of inner]
  float* part;              // [pairs, hidden]
  int* done_up;             // [slots]
  int* done_down;           // [column ranges]
  int slots, down_ranges;
};

template <int DT>
__device__ __forceinline__ long long code_bytes(long long k) { return DT == 4 ? k / 2 : k; }

// ---------------------------------------------------------------------------------------------------------------
template <typename W>
__device__ __forceinline__ void route_logits(const MoeParams& p, int block) {
  const int expert_blocks = (p.experts + 7) / 8;
  const int e = (block % expert_blocks) * 8 + (threadIdx.x >> 5), t0 = (block / expert_blocks) * 8;
  if (e >= p.experts) return;
  const W* row = static_cast<const W*>(p.router) + static_cast<long long>(e) * p.hidden;
  const int lane = threadIdx.x & 31, count = min(8, p.tokens - t0);
  double acc[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) acc[t] = 0.0;
  for (int at = lane * 8; at < p.hidden; at += 256) {
    Raw8<W> w;
    w.template load<true>(row, at, p.hidden);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      if (t >= count) break;
      Raw8<bf16> x;
      x.load<true>(p.x + static_cast<long long>(t0 + t) * p.hidden, at, p.hidden);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[t] = fma(static_cast<double>(x.get(i)), static_cast<double>(w.get(i)), acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    if (t >= count) break;
    const double sum = warp_reduce(acc[t], SumOp());
    if (lane == 0) p.logits[static_cast<long long>(t0 + t) * p.experts + e] = sum;
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
    if (threadIdx.x == 0) p.xs[token] = __float2bfloat16_rn(s);
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
      if ((threadIdx.x & (lanes - 1)) == 0 && at < p.hidden) p.xs[token * groups + at / p.sub] = __float2bfloat16_rn(s);
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

// Blocks [0, tokens): a token's codes.  Block `tokens`: counters.  The others: logits of eight experts for up to
// eight tokens.  The sums are in fp64, so that the choice of experts does not hang on the order of a sum.
template <int DT>
__global__ void __launch_bounds__(256) moe_route_kernel(const MoeParams p) {
  const int b = blockIdx.x;
  if (b < p.tokens) {
    route_quantize<DT>(p, b);
  } else if (b == p.tokens) {
    for (int i = threadIdx.x; i < p.slots; i += 256) p.done_up[i] = 0;
    for (int i = threadIdx.x; i < p.down_ranges; i += 256) p.done_down[i] = 0;
  } else if (p.router_f32) {
    route_logits<float>(p, b - p.tokens - 1);
  } else {
    route_logits<bf16>(p, b - p.tokens - 1);
  }
}

// One block of 1024 threads.  A warp picks a token's experts one after the other: the largest logit that is left,
// ties to the lowest index, NaN below everything (a token with such logits gets weights of NaN).
static __global__ void __launch_bounds__(1024) moe_select_kernel(const MoeParams p) {
  __shared__ int chosen[kMoeMaxPairs];
  __shared__ int count[kMoeMaxExperts];
  __shared__ int first[kMoeMaxExperts];
  __shared__ int warp_sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = p.tokens * p.top_k;
  if (p.router != nullptr) {
    for (int t = warp; t < p.tokens; t += 32) {
      const double* row = p.logits + static_cast<long long>(t) * p.experts;
      uint32_t taken = 0;  // of this lane's experts lane, lane + 32, ...
      double mine = 0.0;   // lane j: the logit of choice j
      int mine_id = -1;
      for (int j = 0; j < p.top_k; ++j) {
        double best = 0.0;
        int best_id = INT_MAX;
        for (int i = 0, e = lane; e < p.experts; ++i, e += 32) {
          if ((taken >> i) & 1u) continue;
          double v = row[e];
          if (!(v == v)) v = -__longlong_as_double(0x7FF0000000000000LL);
          if (best_id == INT_MAX || v > best) {
            best = v;
            best_id = e;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const double v = __shfl_xor_sync(0xFFFFFFFFu, best, o);
          const int id = __shfl_xor_sync(0xFFFFFFFFu, best_id, o);
          if (id != INT_MAX && (best_id == INT_MAX || v > best || (v == best && id < best_id))) {
            best = v;
            best_id = id;
          }
        }
        if ((best_id & 31) == lane) taken |= 1u << (best_id >> 5);
        if (lane == j) {
          mine = row[best_id];
          mine_id = best_id;
        }
      }
      const double top = __shfl_sync(0xFFFFFFFFu, mine, 0);
      const double e = lane < p.top_k ? exp(mine - top) : 0.0;
      double total;
      if (p.renormalize) {
        total = warp_reduce(e, SumOp());
      } else {
        total = 0.0;
        for (int i = lane; i < p.experts; i += 32) total += exp(row[i] - top);
        total = warp_reduce(total, SumOp());
      }
      if (lane < p.top_k) {
        chosen[t * p.top_k + lane] = mine_id;
        p.pair_weight[t * p.top_k + lane] = static_cast<float>(e / total);
      }
    }
  } else {
    for (int i = threadIdx.x; i < pairs; i += 1024) {
      const long long id = p.ids_64 ? static_cast<const long long*>(p.ids_in)[i] : static_cast<const int*>(p.ids_in)[i];
      chosen[i] = id >= 0 && id < p.experts ? static_cast<int>(id) : -1;  // any other number: no expert
      p.pair_weight[i] = p.weights_in[i];
    }
  }
  const int e = threadIdx.x;
  count[e] = 0;
  __syncthreads();
  int place = 0;
  const int my_choice = threadIdx.x < pairs ? chosen[threadIdx.x] : -1;  // pairs <= 1024
  if (my_choice >= 0) place = atomicAdd(&count[my_choice], 1);  // the order within an expert changes no result
  __syncthreads();
  // scan over the experts: pairs before (low half) and experts in use before (high half)
  const int here = count[e] + (count[e] > 0 ? 1 << 16 : 0);
  int sum = here;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, s, o);
      if (lane >= o) s += v;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  sum += (warp > 0 ? warp_sums[warp - 1] : 0) - here;
  first[e] = sum & 0xFFFF;
  if (count[e] > 0) {
    int* slot = p.active + 1 + 3 * (sum >> 16);
    slot[0] = e;
    slot[1] = first[e];
    slot[2] = count[e];
  }
  if (threadIdx.x == 0) p.active[0] = warp_sums[31] >> 16;
  __syncthreads();
  if (threadIdx.x < pairs) {
    p.pair_expert[threadIdx.x] = my_choice;
    if (my_choice >= 0) p.pair_list[first[my_choice] + place] = threadIdx.x;
    if (p.ids_out != nullptr) p.ids_out[threadIdx.x] = my_choice;
    if (p.weights_out != nullptr) p.weights_out[threadIdx.x] = p.pair_weight[threadIdx.x];
  }
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

// Weights: read once, kept out of L1.
template <int WORDS>
__device__ __forceinline__ void load_weight_words(uint32_t (&w)[4], const uint8_t* p, bool valid) {
#pragma unroll
  for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  if (!valid) return;
  if (WORDS == 4)
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  else if (WORDS == 2)
    asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  else
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
}

template <int WORDS>
__device__ __forceinline__ void load_code_words(uint32_t (&w)[4], const uint8_t* p, bool valid) {
#pragma unroll
  for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  if (!valid) return;
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

// 4 x 4 bytes: r[i] holds row i of four columns; the result w[c] holds column c of four rows.
__device__ __forceinline__ void transpose_bytes(uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, uint32_t (&w)[4]) {
  const uint32_t a = __byte_perm(r0, r1, 0x5140), b = __byte_perm(r0, r1, 0x7362);  // columns 0,1 and 2,3 of rows 0,1
  const uint32_t c = __byte_perm(r2, r3, 0x5140), d = __byte_perm(r2, r3, 0x7362);
  w[0] = __byte_perm(a, c, 0x5410);
  w[1] = __byte_perm(a, c, 0x7632);
  w[2] = __byte_perm(b, d, 0x5410);
  w[3] = __byte_perm(b, d, 0x7632);
}

// What a block knows of its product: rows of weight codes times the codes of `count` pairs.
struct MoeTile {
  const uint8_t* w;       // the expert's matrix
  const bf16* w_scale;    // the expert's scales: [N] or [groups, N]
  const uint8_t* codes;   // of all rows; row index given by rows_of
  const bf16* scales;
  int k, n;               // K, and N of the matrix (2 * inner for up/gate)
  int groups;
};

// Accumulators of one lane: kFrags fragments of 16 rows, kN groups of eight tokens.
template <bool SC>
struct MoeSum {
  using type = int;
};
template <>
struct MoeSum<true> {
  using type = double;
};

// `columns`: kTileCols weight columns (rows of the transposed matrix) a block works on.
// K-major weights (NT): 32 columns, warps = 2 fragments x 4 shares of K.
// N-major weights (NN): 128 columns in 8 fragments, 8 shares of K; lane group g holds columns 16 g .. 16 g + 15, of
// which fragment f takes the two at 2 f.
template <bool NN>
struct MoeShape {
  static constexpr int kCols = NN ? 128 : 32;
  static constexpr int kFrags = NN ? 8 : 1;
  static constexpr int kShares = NN ? 8 : 4;
};

constexpr int kMoeThreads = 256;

template <int DT, bool NN, bool SC, int WORDS, int TOKENS, bool kDown>
__device__ __forceinline__ void moe_product(const MoeParams& p, const MoeTile& tile, int tile_index, const int* row_of, int count,
                                            typename MoeSum<SC>::type* red) {
  using Sum = typename MoeSum<SC>::type;
  constexpr int kN = TOKENS / 8, kFrags = MoeShape<NN>::kFrags, kCols = MoeShape<NN>::kCols;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int half_n = tile.n / 2;  // up/gate: the gate columns start here
  int acc[kFrags][kN][4];
  double sum[SC ? kFrags : 1][SC ? kN : 1][4];
#pragma unroll
  for (int f = 0; f < kFrags; ++f)
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[f][n][i] = 0;
        if (SC) sum[f][n][i] = 0.0;
      }
  // rows of the token operand that this lane reads, and (for the scales) the rows its results belong to
  const long long code_pitch = code_bytes<DT>(tile.k);
  const uint8_t* codes[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n) codes[n] = n * 8 + g < count ? tile.codes + row_of[n * 8 + g] * code_pitch : nullptr;

  if constexpr (!NN) {
    // a lane takes 4 * WORDS consecutive bytes of a row, a quad 16 * WORDS: `chunk` values of K
    constexpr int kPerLane = WORDS * (DT == 4 ? 8 : 4), chunk = 4 * kPerLane;
    const int frag = warp & 1, share = warp >> 1;
    const int col0 = kDown ? tile_index * 32 + frag * 16 : frag * half_n + tile_index * 16;
    const uint8_t* row_a = tile.w + (col0 + g) * code_pitch;
    const uint8_t* row_b = row_a + 8 * code_pitch;
    const int chunks = (tile.k + chunk - 1) / chunk;
#pragma unroll 2
    for (int c = share; c < chunks; c += MoeShape<false>::kShares) {
      const int k0 = c * chunk + q * kPerLane;
      const bool valid = k0 < tile.k;
      const long long at = code_bytes<DT>(k0);
      uint32_t wa[4], wb[4], x[kN][4];
      load_weight_words<WORDS>(wa, row_a + at, valid);
      load_weight_words<WORDS>(wb, row_b + at, valid);
#pragma unroll
      for (int n = 0; n < kN; ++n) load_code_words<WORDS>(x[n], codes[n] + at, valid && codes[n] != nullptr);
      if constexpr (DT == 4) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
#pragma unroll
          for (int n = 0; n < kN; ++n)
            mma_i8(acc[0][n], even_codes(wa[i]), even_codes(wb[i]), odd_codes(wa[i]), odd_codes(wb[i]), even_codes(x[n][i]), odd_codes(x[n][i]));
      } else {
#pragma unroll
        for (int i = 0; i < WORDS; i += 2)
#pragma unroll
          for (int n = 0; n < kN; ++n) mma_i8(acc[0][n], wa[i], wb[i], wa[i + 1], wb[i + 1], x[n][i], x[n][i + 1]);
      }
      if constexpr (SC) {  // the chunk lies in one group of K
        const int kg = c * chunk / p.sub;
        const double sa = to_f32(tile.w_scale[static_cast<long long>(kg) * tile.n + col0 + g]);
        const double sb = to_f32(tile.w_scale[static_cast<long long>(kg) * tile.n + col0 + g + 8]);
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int token = n * 8 + 2 * q + (i & 1);
            const double st = token < count ? to_f32(tile.scales[row_of[token] * tile.groups + kg]) : 0.f;
            sum[0][n][i] = fma(static_cast<double>(DT == 4 ? acc[0][n][i] >> 8 : acc[0][n][i]), st * (i < 2 ? sa : sb), sum[0][n][i]);
            acc[0][n][i] = 0;
          }
      }
    }
  } else {
    // a step is 32 values of K: a lane takes 4 (packed) or 8 rows of K, 16 columns each
    const int block = kDown ? tile_index * 128 + g * 16 : (g < 4 ? tile_index * 64 + g * 16 : half_n + tile_index * 64 + (g - 4) * 16);
    const bool col_valid = kDown ? block < tile.n : (g < 4 ? block < half_n : block < tile.n);
    const int steps = tile.k / 32, share_steps = (steps + 7) / 8;
    const int begin = warp * share_steps, end = min(steps, begin + share_steps);
    constexpr int kRows = DT == 4 ? 4 : 8;
    const uint8_t* base = tile.w + block + static_cast<long long>(q * kRows) * tile.n;
    for (int s = begin; s < end; ++s) {
      uint32_t r[kRows][4], x[kN][4];
      const uint8_t* at = base + static_cast<long long>(s) * 4 * kRows * tile.n;
#pragma unroll
      for (int i = 0; i < kRows; ++i) load_weight_words<4>(r[i], at + static_cast<long long>(i) * tile.n, col_valid);
#pragma unroll
      for (int n = 0; n < kN; ++n)
        load_code_words<DT == 4 ? 1 : 2>(x[n], codes[n] + code_bytes<DT>(s * 32 + q * 8), codes[n] != nullptr);
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {  // four columns at a time: fragments 2 c4 and 2 c4 + 1
        uint32_t lo[4], hi[4];
        transpose_bytes(r[0][c4], r[1][c4], r[2][c4], r[3][c4], lo);
        if constexpr (DT == 8) transpose_bytes(r[4][c4], r[5][c4], r[6][c4], r[7][c4], hi);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            if constexpr (DT == 4)
              mma_i8(acc[2 * c4 + h][n], even_codes(lo[2 * h]), even_codes(lo[2 * h + 1]), odd_codes(lo[2 * h]), odd_codes(lo[2 * h + 1]),
                     even_codes(x[n][0]), odd_codes(x[n][0]));
            else
              mma_i8(acc[2 * c4 + h][n], lo[2 * h], lo[2 * h + 1], hi[2 * h], hi[2 * h + 1], x[n][0], x[n][1]);
          }
      }
      if constexpr (SC) {
        const bool last = s + 1 == end || ((s + 1) * 32) % p.sub == 0;
        if (last) {
          const int kg = s * 32 / p.sub;
          const bf16* ws = tile.w_scale + static_cast<long long>(kg) * tile.n + block;
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            double st[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int token = n * 8 + 2 * q + i;
              st[i] = token < count ? to_f32(tile.scales[row_of[token] * tile.groups + kg]) : 0.f;
            }
#pragma unroll
            for (int f = 0; f < kFrags; ++f)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const double sw = col_valid ? to_f32(ws[2 * f + (i >> 1)]) : 0.f;
                sum[f][n][i] = fma(static_cast<double>(DT == 4 ? acc[f][n][i] >> 8 : acc[f][n][i]), st[i & 1] * sw, sum[f][n][i]);
                acc[f][n][i] = 0;
              }
          }
        }
      }
    }
  }

  // the shares of K: exact integers in any order, or fp64 numbers one warp after the other
  for (int i = threadIdx.x; i < kCols * TOKENS; i += kMoeThreads) red[i] = 0;
  __syncthreads();
  auto column = [&](int f, int i) { return NN ? g * 16 + 2 * f + (i >> 1) : (warp & 1) * 16 + g + (i >> 1) * 8; };
  if constexpr (!SC) {
#pragma unroll
    for (int f = 0; f < kFrags; ++f)
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int token = n * 8 + 2 * q + (i & 1);
          if (token < count) atomicAdd(&red[column(f, i) * TOKENS + token], DT == 4 ? acc[f][n][i] >> 8 : acc[f][n][i]);
        }
    __syncthreads();
  } else {
    for (int turn = 0; turn < MoeShape<NN>::kShares; ++turn) {
      if ((NN ? warp : warp >> 1) == turn) {
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[column(f, i) * TOKENS + n * 8 + 2 * q + (i & 1)] += sum[f][n][i];
      }
      __syncthreads();
    }
  }
}

// Quantises the activations of one expert's pairs (fp64 in, as they were computed): what quantize_tokens does, with
// values that are not exactly known in fp32, so that each code is settled against them where it has to be.
template <int DT>
__device__ __forceinline__ void quantize_activations(const MoeParams& p, const int* list, int count) {
  constexpr double kTop = DT == 4 ? 7.0 : 127.0;
  __shared__ unsigned long long warp_max[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int length = p.sub ? p.sub : p.inner, groups = p.sub ? (p.inner + p.sub - 1) / p.sub : 1;
  // a row by all warps, by four, two or one; a group of values by one
  const int per_row = p.sub ? 1 : (count == 1 ? 8 : count == 2 ? 4 : count <= 4 ? 2 : 1);
  const int items = count * groups, step = 8 / per_row;
  for (int base = 0; base < items; base += step) {
    const int item = base + warp / per_row;
    const bool live = item < items;
    const int pair = live ? list[item / groups] : 0, c0 = live ? (item % groups) * length : 0;
    const int c1 = live ? min(c0 + length, p.inner) : 0;
    const double* row = p.act + static_cast<long long>(pair) * p.inner;
    const int begin = c0 + ((warp % per_row) * 32 + lane) * 2, stride = per_row * 64;
    unsigned long long most = 0;
    for (int c = begin; c < c1; c += stride) {
      const double2 v = __ldcg(reinterpret_cast<const double2*>(row + c));
      const unsigned long long a = __double_as_longlong(v.x) & 0x7FFFFFFFFFFFFFFFLL, b = __double_as_longlong(v.y) & 0x7FFFFFFFFFFFFFFFLL;
      most = max(most, max(a, b));
    }
    most = warp_reduce(most, MaxOp());
    if (per_row > 1) {
      if (lane == 0) warp_max[warp] = most;
      __syncthreads();
      for (int i = 0; i < per_row; ++i) most = max(most, warp_max[warp / per_row * per_row + i]);
      __syncthreads();
    }
    const float s = nonzero_scale(bf16_from_double(__longlong_as_double(most) / kTop));
    if (live && begin == c0) p.as[static_cast<long long>(pair) * groups + item % groups] = __float2bfloat16_rn(s);
    const bool ordinary = scale_is_ordinary(s);
    const float inv = __frcp_rn(s), delta = static_cast<float>(kTop) * 4.76837158203125e-7f;  // fp32 value, product: 3 roundings
    uint8_t* codes = p.aq + static_cast<long long>(pair) * code_bytes<DT>(p.inner);
    for (int c = begin; c < c1; c += stride) {
      const double2 v = __ldcg(reinterpret_cast<const double2*>(row + c));
      uint32_t code[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const double exact = i ? v.y : v.x;
        const float approx = static_cast<float>(exact);
        code[i] = __float_as_uint(__fadd_rn(__fmaf_rn(approx, inv, -delta), kRoundMagic));
        const uint32_t other = __float_as_uint(__fadd_rn(__fmaf_rn(approx, inv, delta), kRoundMagic));
        if (!ordinary || code[i] != other) {
          const double quotient = rint(exact / static_cast<double>(s));
          code[i] = s < __int_as_float(0x7F800000) ? static_cast<uint32_t>(static_cast<int>(fmin(fmax(quotient, -kTop), kTop))) : 0u;
        }
      }
      if (DT == 4) codes[c / 2] = static_cast<uint8_t>((code[0] & 0xFu) | ((code[1] & 0xFu) << 4));
      else *reinterpret_cast<uint16_t*>(codes + c) = static_cast<uint16_t>((code[0] & 0xFFu) | ((code[1] & 0xFFu) << 8));
    }
  }
}

// True in the whole block for the last of `total` blocks that count up `counter`: what the others wrote before is
// then visible to it (through L2: read with __ldcg).
__device__ __forceinline__ bool last_block(int* counter, int total) {
  __shared__ int is_last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    is_last = atomicAdd(counter, 1) == total - 1;
    __threadfence();
  }
  __syncthreads();
  return is_last != 0;
}

template <int DT, bool NN, bool SC, int WORDS, bool kDown>
__global__ void __launch_bounds__(kMoeThreads) moe_product_kernel(const MoeParams p) {
  using Sum = typename MoeSum<SC>::type;
  constexpr int kCols = MoeShape<NN>::kCols;
  constexpr int kMaxTokens = SC ? 8 : 16;  // of one pass over the weights: what the accumulators leave room for
  __shared__ Sum red[kCols * kMaxTokens];
  __shared__ int rows[kMaxTokens];
  const int out_cols = kDown ? kCols : kCols / 2;
  const int ranges = ((kDown ? p.hidden : p.inner) + out_cols - 1) / out_cols;
  const int slot = blockIdx.x / ranges, range = blockIdx.x % ranges, col0 = range * out_cols;
  const int in_use = p.active[0];
  if (slot >= in_use) {
    if (kDown && in_use == 0 && slot == 0)  // no pair has an expert: nothing is added up
      for (int i = threadIdx.x; i < p.tokens * kCols; i += kMoeThreads)
        if (col0 + i % kCols < p.hidden) p.out[static_cast<long long>(i / kCols) * p.hidden + col0 + i % kCols] = __float2bfloat16_rn(0.f);
    return;
  }
  const int expert = p.active[1 + 3 * slot], first = p.active[2 + 3 * slot], count = p.active[3 + 3 * slot];
  const int* list = p.pair_list + first;
  MoeTile tile;
  tile.k = kDown ? p.inner : p.hidden;
  tile.n = kDown ? p.hidden : 2 * p.inner;
  tile.groups = SC ? (tile.k + p.sub - 1) / p.sub : 1;
  tile.w = (kDown ? p.w_down : p.w_up_gate) + static_cast<long long>(expert) * tile.n * code_bytes<DT>(tile.k);
  tile.w_scale = (kDown ? p.s_down : p.s_up_gate) + static_cast<long long>(expert) * tile.n * tile.groups;
  tile.codes = kDown ? p.aq : p.xq;
  tile.scales = kDown ? p.as : p.xs;

  for (int done = 0; done < count; done += kMaxTokens) {
    const int here = min(kMaxTokens, count - done);
    __syncthreads();
    if (threadIdx.x < kMaxTokens) rows[threadIdx.x] = threadIdx.x < here ? (kDown ? list[done + threadIdx.x] : list[done + threadIdx.x] / p.top_k) : 0;
    __syncthreads();
    if (SC || here <= 8) moe_product<DT, NN, SC, WORDS, 8, kDown>(p, tile, range, rows, here, red);
    else moe_product<DT, NN, SC, WORDS, kMaxTokens, kDown>(p, tile, range, rows, here, red);
    const int width = SC || here <= 8 ? 8 : kMaxTokens;
    for (int i = threadIdx.x; i < here * out_cols; i += kMoeThreads) {
      const int token = i / out_cols, c = i % out_cols, col = col0 + c, pair = list[done + token];
      if (col >= (kDown ? p.hidden : p.inner)) continue;
      if (kDown) {
        double y = static_cast<double>(red[c * width + token]);
        if (!SC) y *= static_cast<double>(to_f32(tile.scales[rows[token]])) * static_cast<double>(to_f32(tile.w_scale[col]));
        p.part[static_cast<long long>(pair) * p.hidden + col] = static_cast<float>(y) * p.pair_weight[pair];
      } else {
        double up = static_cast<double>(red[c * width + token]), gate = static_cast<double>(red[(c + out_cols) * width + token]);
        if (!SC) {
          const double s = to_f32(tile.scales[rows[token]]);
          up *= s * static_cast<double>(to_f32(tile.w_scale[col]));
          gate *= s * static_cast<double>(to_f32(tile.w_scale[p.inner + col]));
        }
        p.act[static_cast<long long>(pair) * p.inner + col] = up * gate / (1.0 + exp(-gate));
      }
    }
  }
  if (!kDown) {
    if (last_block(p.done_up + slot, ranges)) quantize_activations<DT>(p, list, count);
  } else if (last_block(p.done_down + range, in_use)) {
    for (int i = threadIdx.x; i < p.tokens * kCols; i += kMoeThreads) {
      const int token = i / kCols, col = col0 + i % kCols;
      if (col >= p.hidden) continue;
      float y = 0.f;
      for (int j = 0; j < p.top_k; ++j) {
        const int pair = token * p.top_k + j;
        if (p.pair_expert[pair] >= 0) y += __ldcg(p.part + static_cast<long long>(pair) * p.hidden + col);
      }
      p.out[static_cast<long long>(token) * p.hidden + col] = __float2bfloat16_rn(y);
    }
  }
}

}  // namespace b200
