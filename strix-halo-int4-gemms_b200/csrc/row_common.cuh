// Pieces of the kernels that work on rows of values: 8-value loads and stores, reductions over the threads of a
// row, and the two quantisers (of exactly known bf16 values, and of values known to within a small error).
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

namespace b200 {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }

// Eight consecutive values of a row, kept as they were read (4 registers of bf16, 8 of fp32).  Values past the
// end of the row are zero.
template <typename T>
struct Raw8;

template <>
struct Raw8<bf16> {
  uint32_t w[4];
  __device__ __forceinline__ float get(int i) const { return (i & 1) ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]); }
  __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0u; }
  // G values (8 or 4) at place i
  template <int G>
  __device__ __forceinline__ void load_chunk(int i, const bf16* p, bool valid) {
    if constexpr (G == 8) {
      const uint4 v = valid ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
      const uint2 v = valid ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0u, 0u);
      w[i / 2] = v.x;
      w[i / 2 + 1] = v.y;
    }
  }
  // eight values in 16 bytes
  __device__ __forceinline__ void from_chunks(const uint4* at, int) {
    const uint4 v = *at;
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ __forceinline__ void set(const bf16 (&e)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = static_cast<uint32_t>(__bfloat16_as_ushort(e[2 * i])) | (static_cast<uint32_t>(__bfloat16_as_ushort(e[2 * i + 1])) << 16);
  }
  template <bool kAligned>
  __device__ __forceinline__ void load(const bf16* row, long long at, long long cols) {
    if (kAligned) {
      if (at < cols) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + at));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      } else {
        zero();
      }
    } else {
      const unsigned short* src = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = at + 2 * i < cols ? __ldg(src + at + 2 * i) : 0u;
        const uint32_t b = at + 2 * i + 1 < cols ? __ldg(src + at + 2 * i + 1) : 0u;
        w[i] = a | (b << 16);
      }
    }
  }
};

template <>
struct Raw8<float> {
  float f[8];
  __device__ __forceinline__ float get(int i) const { return f[i]; }
  template <int G>
  __device__ __forceinline__ void load_chunk(int i, const float* p, bool valid) {
#pragma unroll
    for (int k = 0; k < G; k += 4) {
      const float4 v = valid ? __ldg(reinterpret_cast<const float4*>(p + k)) : make_float4(0.f, 0.f, 0.f, 0.f);
      f[i + k] = v.x; f[i + k + 1] = v.y; f[i + k + 2] = v.z; f[i + k + 3] = v.w;
    }
  }
  // two times four values, the second `step` chunks behind the first
  __device__ __forceinline__ void from_chunks(const uint4* at, int step) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(at + k * step);
      f[4 * k] = v.x; f[4 * k + 1] = v.y; f[4 * k + 2] = v.z; f[4 * k + 3] = v.w;
    }
  }
  __device__ __forceinline__ void set(const float (&e)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = e[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
  }
  template <bool kAligned>
  __device__ __forceinline__ void load(const float* row, long long at, long long cols) {
    if (kAligned) {
      if (at < cols) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(row + at));
        const float4 b = __ldg(reinterpret_cast<const float4*>(row + at + 4));
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
      } else {
        zero();
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = at + i < cols ? __ldg(row + at + i) : 0.f;
    }
  }
};

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Which columns thread t of the TPR threads of a row has: eight values for each v, in chunks of G consecutive ones, G the
// number of values in 16 bytes (8 of bf16, 4 of fp32), so that a warp's loads are neighbours; or 1 where wide loads
// cannot be used.
template <int TPR, int G>
struct Columns {
  int thread;
  long long cols;
  __device__ __forceinline__ long long at(int v, int i) const { return (static_cast<long long>(v * (8 / G) + i / G) * TPR + thread) * G + i % G; }
  // A chunk is inside or outside.  (Rows have less than 2^31 values, and a thread's places end less than 2^31 behind them.)
  __device__ __forceinline__ bool has(int v, int i) const { return static_cast<unsigned>(at(v, i - i % G)) < static_cast<unsigned>(cols); }
  // Values behind the row: zero, or (narrow loads) `behind`.
  template <typename T>
  __device__ __forceinline__ Raw8<T> load(const T* row, int v, T behind = T(0.f)) const {
    Raw8<T> r;
    if constexpr (G == 1) {
      T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = has(v, i) ? row[at(v, i)] : behind;
      r.set(e);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += G) r.template load_chunk<G>(i, row + at(v, i), has(v, i));
    }
    return r;
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, int v, const float (&f)[8]) const {
    if constexpr (G == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (has(v, i)) row[at(v, i)] = static_cast<T>(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += G) {
        if (!has(v, i)) continue;
        static_assert(G * sizeof(T) == 16, "a chunk is one store");
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<float4*>(row + at(v, i)) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
        } else {
          *reinterpret_cast<uint4*>(row + at(v, i)) =
              make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
        }
      }
    }
  }
};

// ---------------------------------------------------------------------------------------------------------------
// reductions over the threads of a row: one warp (TPR == 32) or one block (TPR threads)
// ---------------------------------------------------------------------------------------------------------------
struct SumOp {
  template <typename V>
  __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
// NaN if one of the two is; the sizes of both.
__device__ __forceinline__ float max_size(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
// The same of three.
__device__ __forceinline__ float max_size(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The larger of m and two sizes; NaN are passed over.
__device__ __forceinline__ float max_abs(float m, float a, float b) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
  return r;
}
struct MaxSizeOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return max_size(a, b); }
};
struct MaxOp {
  template <typename V>
  __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; }
};

// Two fp32 numbers in a register pair: one instruction works on both, each rounded as on its own.
struct Pair {
  unsigned long long v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ explicit Pair(float both) : Pair(both, both) {}
  __device__ __forceinline__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

template <typename V, typename Op>
__device__ __forceinline__ V warp_reduce(V v, Op op, int width = 32) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < width) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

// Over a whole warp one instruction does it, for whole numbers and for sizes.
__device__ __forceinline__ uint32_t warp_reduce(uint32_t v, MaxOp op, int width = 32) {
  if (width == 32) return __reduce_max_sync(0xFFFFFFFFu, v);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < width) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
__device__ __forceinline__ float warp_reduce(float v, MaxSizeOp, int width = 32) {
  // bit patterns of sizes have the order of the sizes, NaN above infinity
  return __uint_as_float(warp_reduce(__float_as_uint(v) & 0x7FFFFFFFu, MaxOp(), width));
}

// Two values at once; every thread of the row gets both results.  `scratch` holds 2 * TPR / 32 values and is not
// shared by consecutive reductions, so one barrier is enough; the caller has a barrier between two uses of it.
template <int TPR, typename A, typename B, typename OpA, typename OpB>
__device__ __forceinline__ void row_reduce2(A& a, B& b, OpA op_a, OpB op_b, void* scratch) {
  a = warp_reduce(a, op_a);
  b = warp_reduce(b, op_b);
  if (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    A* sa = static_cast<A*>(scratch);
    B* sb = reinterpret_cast<B*>(sa + kWarps);
    if ((threadIdx.x & 31) == 0) {
      sa[threadIdx.x >> 5] = a;
      sb[threadIdx.x >> 5] = b;
    }
    __syncthreads();
    const int lane = threadIdx.x & (kWarps - 1);
    a = sa[lane];
    b = sb[lane];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
      a = op_a(a, __shfl_xor_sync(0xFFFFFFFFu, a, o));
      b = op_b(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
    }
  }
}

template <int TPR, typename A, typename OpA>
__device__ __forceinline__ A row_reduce(A a, OpA op_a, void* scratch) {
  a = warp_reduce(a, op_a);
  if (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    A* sa = static_cast<A*>(scratch);
    if ((threadIdx.x & 31) == 0) sa[threadIdx.x >> 5] = a;
    __syncthreads();
    a = sa[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) a = op_a(a, __shfl_xor_sync(0xFFFFFFFFu, a, o));
  }
  return a;
}

// ---------------------------------------------------------------------------------------------------------------
// quantisation
// ---------------------------------------------------------------------------------------------------------------
// float64 -> bf16 with one rounding: to odd in fp32 (16 more bits than bf16 keeps), then to nearest even.
__device__ __forceinline__ float bf16_from_double(double v) {
  float f = __double2float_rz(v);
  if (static_cast<double>(f) != v) f = __uint_as_float(__float_as_uint(f) | 1u);
  return __bfloat162float(__float2bfloat16_rn(f));
}

// A scale that rounds to zero (a row of zeros, or of numbers below the least bf16) counts as one: every code is
// then zero, and the scale stays a positive number as the rest of the library asks.
__device__ __forceinline__ float nonzero_scale(float s) { return s == 0.f ? 1.f : s; }

// bf16(amax / top) of a bf16 amax given by its bit pattern (NaN patterns are above infinity's, so that a row with
// a NaN gets a NaN scale).  A tie of two bf16 numbers is an odd multiple of 2^-9 of a power of two; 7 or 127 times
// that has more than eight significant bits, so the quotient never is one, and it is at least 2^-17 (relative) away from
// all of them: a product with the rounded 1 / top rounds to the same bf16 number.
template <int BITS>
__device__ __forceinline__ float scale_of_bf16(uint32_t amax_bits) {
  const float per_top = BITS == 4 ? 1.f / 7.f : 1.f / 127.f;
  return nonzero_scale(__bfloat162float(__float2bfloat16_rn(__uint_as_float(amax_bits << 16) * per_top)));
}

// 1 / s to within 2^-22, for ordinary scales
__device__ __forceinline__ float about_inverse(float s) { return __fdividef(1.f, s); }

constexpr float kRoundMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to the nearest even integer, left in the low bits

// A scale for which 1 / s and the products below are normal numbers.
__device__ __forceinline__ bool scale_is_ordinary(float s) { return s >= 7.9e-31f && s <= 1.3e30f; }

// round_half_even(x / s) of bf16 x and s, by multiplication.  x / s = (mx / ms) 2^j with significands below 256:
// it is a tie n + 1/2 or, |2^(j+1) mx - (2n+1) ms| being a whole number from j = -1 on and ms < 256, at least 1 / 1020 away
// from every tie, and it is at most 128.  The products with 1 / s made 2^-20 smaller and larger (1.5e-4 at 128) therefore
// round to one integer, which is the answer, or, at a tie, to its two neighbours.  Both carry kRoundMagic; their sum
// has steps of two, so that it rounds to the even neighbour, and its last bits are the code's.  Three instructions on
// the multiply-add pipe instead of a division's nine: the kernels are bound by instructions.
struct ExactQuotient {
  float low, high;
  __device__ __forceinline__ explicit ExactQuotient(float s) {
    const float inv = about_inverse(s);
    low = inv * (1.f - 9.5367431640625e-7f);
    high = inv * (1.f + 9.5367431640625e-7f);
  }
  __device__ __forceinline__ uint32_t code(float x) const {
    return __float_as_uint(__fadd_rn(__fmaf_rn(x, low, kRoundMagic), __fmaf_rn(x, high, kRoundMagic)));
  }
};

// The same by division, for scales outside the ordinary range (and codes of 0 where the scale is not finite).
template <int BITS>
__device__ __forceinline__ uint32_t code_by_division(float x, float s) {
  const float top = BITS == 4 ? 7.f : 127.f;
  const float q = rintf(__fdiv_rn(x, s));
  if (!(q == q) || !(s < __int_as_float(0x7F800000))) return 0u;
  return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(q, -top), top)));
}

// Eight codes (low bits of each word), packed: 4 bytes of nibbles or 8 bytes.
template <int BITS>
struct CodeWords {
  using type = uint2;
  __device__ __forceinline__ static uint2 pack(const uint32_t (&c)[8]) {
    return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
  }
};
template <>
struct CodeWords<4> {
  using type = uint32_t;
  __device__ __forceinline__ static uint32_t pack(const uint32_t (&c)[8]) {
    // bytes of even and of odd values, then their low nibbles side by side
    const uint32_t even = __byte_perm(__byte_perm(c[0], c[2], 0x0040), __byte_perm(c[4], c[6], 0x0040), 0x5410);
    const uint32_t odd = __byte_perm(__byte_perm(c[1], c[3], 0x0040), __byte_perm(c[5], c[7], 0x0040), 0x5410);
    return (even & 0x0F0F0F0Fu) | ((odd << 4) & 0xF0F0F0F0u);
  }
};

template <int BITS, bool kAligned>
__device__ __forceinline__ void store_packed(uint8_t* row, long long at, long long cols, typename CodeWords<BITS>::type w) {
  if (at >= cols) return;
  if (BITS == 4) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(&w);
    if (kAligned) {
      *reinterpret_cast<uint32_t*>(row + at / 2) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + 2 * i < cols) row[at / 2 + i] = static_cast<uint8_t>(v >> (8 * i));
    }
  } else {
    const uint32_t* v = reinterpret_cast<const uint32_t*>(&w);
    if (kAligned) {
      *reinterpret_cast<uint2*>(row + at) = make_uint2(v[0], v[BITS == 8 ? 1 : 0]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < cols) row[at + i] = static_cast<uint8_t>(v[BITS == 8 ? i >> 2 : 0] >> (8 * (i & 3)));
    }
  }
}

// Eight codes (low bits of each word) to memory: 4 bytes of nibbles or 8 bytes.
template <int BITS, bool kAligned>
__device__ __forceinline__ void store_codes(uint8_t* row, long long at, long long cols, const uint32_t (&c)[8]) {
  store_packed<BITS, kAligned>(row, at, cols, CodeWords<BITS>::pack(c));
}

}  // namespace b200
