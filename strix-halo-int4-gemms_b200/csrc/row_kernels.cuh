// Kernels that go over rows of values once: the quantiser with a scale for each token, layer norm, layer norm
// with the quantiser behind it, and layer norm's backward pass.  All of them are bound by HBM on large inputs.
//
// One row belongs to a warp (TPR == 32) or to a block of TPR threads; a thread holds V groups of eight values in
// registers, so that a row is read once.  V == 0 is the form for rows that no block can hold: the same code, reading
// the row again (from L2) for every pass over it.  What is done once for a row (reductions, scales, addresses) costs some
// 100 instructions a thread, as much as ten values: many values a thread (V = 8) where rows are many, few (V = 1) where
// they are too few to fill the device (quantize_tokens of 32768 x 2048 to int4: 30 us, 5.6 TB/s, with 64 values a
// thread; 48 us with 16).
#pragma once

#include <cstring>

#include "row_common.cuh"

namespace b200 {

template <int TPR>
struct RowPlace {
  static constexpr int kThreads = TPR == 32 ? 256 : TPR;
  static constexpr int kRows = kThreads / TPR;  // rows a block works on at once
  __device__ __forceinline__ static int thread() { return TPR == 32 ? (threadIdx.x & 31) : threadIdx.x; }
  __device__ __forceinline__ static long long first() {
    return static_cast<long long>(blockIdx.x) * kRows + (TPR == 32 ? (threadIdx.x >> 5) : 0);
  }
  __device__ __forceinline__ static long long step() { return static_cast<long long>(gridDim.x) * kRows; }
};

// The vectors of a thread: in registers, or read anew each time (V == 0).
template <typename T, int TPR, int V, bool kAligned>
struct RowValues {
  Raw8<T> held[V > 0 ? V : 1];
  const T* row;
  long long cols;
  __device__ __forceinline__ RowValues(const T* r, long long n) : row(r), cols(n) {
    if (V > 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) held[v].template load<kAligned>(row, at(v), cols);
    }
  }
  __device__ __forceinline__ long long at(int v) const { return (static_cast<long long>(v) * TPR + RowPlace<TPR>::thread()) * 8; }
  __device__ __forceinline__ int count() const { return V > 0 ? V : static_cast<int>((cols + TPR * 8 - 1) / (TPR * 8)); }
  __device__ __forceinline__ Raw8<T> get(int v) const {
    if (V > 0) return held[v];
    Raw8<T> r;
    r.template load<kAligned>(row, at(v), cols);
    return r;
  }
};

// ---------------------------------------------------------------------------------------------------------------
// quantize_tokens: scale = bf16(amax / top), code = round_half_even(x / scale), for every row (sub == 0) or every
// `sub` values of it (32, 64, 128 or 256: 4 to 32 lanes of one warp).
// ---------------------------------------------------------------------------------------------------------------
// The codes of eight values where the scale is not ordinary: by division, zero where it is not finite.
template <int BITS>
__device__ __noinline__ typename CodeWords<BITS>::type divided_codes(Raw8<bf16> raw, float s) {
  uint32_t c[8];
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    c[2 * i] = code_by_division<BITS>(bf16_lo(raw.w[i]), s);
    c[2 * i + 1] = code_by_division<BITS>(bf16_hi(raw.w[i]), s);
  }
  return CodeWords<BITS>::pack(c);
}

template <int TPR, int V, int BITS, bool kAligned>
__global__ void __launch_bounds__(RowPlace<TPR>::kThreads)
quantize_tokens_kernel(const bf16* __restrict__ src, uint8_t* __restrict__ codes, bf16* __restrict__ scales,
                       long long rows, long long cols, int sub_bits) {  // groups of 2^sub_bits values; 0: the row
  __shared__ uint32_t scratch[2][TPR / 32];
  const long long pitch = BITS == 4 ? (cols + 1) / 2 : cols;
  const int lanes = sub_bits ? 1 << (sub_bits - 3) : 0;  // of a group; 0: one scale a row
  const long long groups = sub_bits ? (cols + (1 << sub_bits) - 1) >> sub_bits : 1;
  auto largest = [](uint32_t m, const Raw8<bf16>& raw) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __vmaxu2(m, raw.w[i] & 0x7FFF7FFFu);
    return m;
  };
  auto put = [&](uint8_t* row, long long at, const Raw8<bf16>& raw, float s, bool ordinary, const ExactQuotient& q) {
    if (ordinary) {
      uint32_t c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = q.code(raw.get(i));
      store_codes<BITS, kAligned>(row, at, cols, c);
    } else {
      store_packed<BITS, kAligned>(row, at, cols, divided_codes<BITS>(raw, s));
    }
  };
  int turn = 0;
  for (long long r = RowPlace<TPR>::first(); r < rows; r += RowPlace<TPR>::step(), turn ^= 1) {
    const RowValues<bf16, TPR, V, kAligned> x(src + r * cols, cols);
    uint8_t* out = codes + r * pitch;
    if (!lanes) {
      uint32_t m = 0;
#pragma unroll
      for (int v = 0; v < x.count(); ++v) m = largest(m, x.get(v));
      const float s = scale_of_bf16<BITS>(row_reduce<TPR>(max(m & 0xFFFFu, m >> 16), MaxOp(), scratch[turn]));
      if (RowPlace<TPR>::thread() == 0) scales[r] = __float2bfloat16_rn(s);
      const bool ordinary = scale_is_ordinary(s);
      const ExactQuotient q(s);
#pragma unroll
      for (int v = 0; v < x.count(); ++v) put(out, x.at(v), x.get(v), s, ordinary, q);
    } else {
#pragma unroll
      for (int v = 0; v < x.count(); ++v) {
        const Raw8<bf16> raw = x.get(v);
        const uint32_t m = largest(0u, raw);
        const float s = scale_of_bf16<BITS>(warp_reduce(max(m & 0xFFFFu, m >> 16), MaxOp(), lanes));
        if ((threadIdx.x & (lanes - 1)) == 0 && x.at(v) < cols) scales[r * groups + (x.at(v) >> sub_bits)] = __float2bfloat16_rn(s);
        put(out, x.at(v), raw, s, scale_is_ordinary(s), ExactQuotient(s));
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// layer norm: y = (x - mean) rstd w + b, from registers, in fp32.  What is added up is x - s, s being the row's first value,
// and the mean is kept in two parts, hi + lo, hi = s + average.  lo corrects the variance (mean((x - hi)^2) - lo^2) and
// every value, so that the errors are the spread's and not the offset's: a row of equal values has exactly that mean, no
// variance and its bias as its norm, and the rounding of a large mean shifts no row.
// In fp32 lo is the average of x - hi, summed up beside the squares; a second sum costs nothing there.  In bf16, with twice
// the values a byte, it costs 2 us of the 46 below: lo is what the rounding of s + average loses, and x - hi is added up
// only where s turns out to be far from the others (more than eight times the spread from the mean).  And where rows are
// read 16 bytes at a time s is zero unless the row's next three values are within a quarter of the first: rows around
// zero, the usual ones, are added up as they are (1 us of 47).
// The values are kept as fp32, and as x - hi: bf16 is taken apart once, not in each pass; pairs of fp32 numbers.
// 32 values a thread, so that the registers allow 1,024 threads an SM (fp32 holds its words twice for a while: 768).
// 32768 x 2048 in bf16: 46 us, 5.9 TB/s, where a copy of the same bytes takes 44; 55 us with 64 values a thread and half
// of the threads, 54 with 16 (the work done once for a row), 56 with resident blocks that read the next row ahead.
// ---------------------------------------------------------------------------------------------------------------
// The row's first value if the next three are within a quarter of it, else zero.
template <typename T>
__device__ __forceinline__ float common_value(const T* row) {
  Raw8<T> head;
  head.template load_chunk<4>(0, row, true);
  const float first = head.get(0), apart = fmaxf(fabsf(head.get(1) - first), fmaxf(fabsf(head.get(2) - first), fabsf(head.get(3) - first)));
  return apart <= 0.25f * fabsf(first) ? first : 0.f;
}

template <typename T, typename W, int TPR, int V, bool kAligned>
__global__ void __launch_bounds__(RowPlace<TPR>::kThreads, (sizeof(T) == 2 ? 1024 : 768) / RowPlace<TPR>::kThreads)
layer_norm_kernel(const T* __restrict__ src, const W* __restrict__ weight, const W* __restrict__ bias, T* __restrict__ y,
                  float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows, long long cols, float eps) {
  __shared__ float scratch[4][TPR / 32];  // of two sums at once in fp32: the second and the third
  const float inv_cols = 1.f / static_cast<float>(cols);
  constexpr int G = kAligned ? 16 / sizeof(T) : 1;
  const Columns<TPR, G> column{RowPlace<TPR>::thread(), cols};
  const int count = V > 0 ? V : static_cast<int>((cols + TPR * 8 - 1) / (TPR * 8));
  constexpr int kHeld = V > 0 ? V : 1;
  constexpr bool kZeroToo = sizeof(T) == 2 && kAligned, kTwice = sizeof(T) == 4;
  for (long long r = RowPlace<TPR>::first(); r < rows; r += RowPlace<TPR>::step()) {
    const T* row = src + r * cols;
    const T first = row[0], behind = G == 1 && sizeof(T) == 2 ? first : T(0.f);
    const float shift = kZeroToo ? common_value(row) : to_f32(first);
    Pair held[kHeld][4];
    auto take = [&](const Raw8<T>& raw, Pair (&f)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = Pair(raw.get(2 * i), raw.get(2 * i + 1));
    };
    if (V > 0) {
      Raw8<T> raw[kHeld];
#pragma unroll
      for (int v = 0; v < kHeld; ++v) raw[v] = column.load(row, v, behind);
#pragma unroll
      for (int v = 0; v < kHeld; ++v) take(raw[v], held[v]);
    }
    const Pair minus_shift(-shift);
    // Behind the row, narrow loads of bf16 have s, which adds nothing; other values are left out.  (Loads of fp32 would wait
    // for s to arrive: 20000 x 2047 took 132 us, not 95.)
    Pair sum(0.f);
    float sum1 = 0.f;
    if (kZeroToo && shift == 0.f) {  // the same for all threads of the row; the values behind it are zero
#pragma unroll
      for (int v = 0; v < count; ++v) {
        Pair(&x)[4] = held[V > 0 ? v : 0];
        if (V == 0) take(column.load(row, v), x);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = add2(sum, x[i]);
      }
    } else {
#pragma unroll
      for (int v = 0; v < count; ++v) {
        Pair(&x)[4] = held[V > 0 ? v : 0];
        if (V == 0) take(column.load(row, v, behind), x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Pair d = add2(x[i], minus_shift);
          if constexpr (G > 1) {
            if (column.has(v, 2 * i)) sum = add2(sum, d);
          } else if constexpr (sizeof(T) == 2) {
            sum = add2(sum, d);
          } else {
            if (column.has(v, 2 * i)) sum1 += d.get().x;
            if (column.has(v, 2 * i + 1)) sum1 += d.get().y;
          }
        }
      }
    }
    const float average = row_reduce<TPR>(sum.get().x + sum.get().y + sum1, SumOp(), scratch[0]) * inv_cols;
    const float hi = shift + average, moved = hi - shift;
    float lo = (shift - (hi - moved)) + (average - moved);  // exactly
    const Pair minus_hi(-hi);
    auto read_differences = [&](int v, Pair (&x)[4]) {
      take(column.load(row, v), x);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = add2(x[i], minus_hi);
    };
    Pair square(0.f), rest(0.f);
    float square1 = 0.f, rest1 = 0.f;
#pragma unroll
    for (int v = 0; v < count; ++v) {
      Pair(&x)[4] = held[V > 0 ? v : 0];
      if (V == 0) take(column.load(row, v), x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = add2(x[i], minus_hi);
        if constexpr (G > 1) {
          if (column.has(v, 2 * i)) {
            square = fma2(x[i], x[i], square);
            if (kTwice) rest = add2(rest, x[i]);
          }
        } else {
          const float2 f = x[i].get();
          if (column.has(v, 2 * i)) {
            square1 = __fmaf_rn(f.x, f.x, square1);
            if (kTwice) rest1 += f.x;
          }
          if (column.has(v, 2 * i + 1)) {
            square1 = __fmaf_rn(f.y, f.y, square1);
            if (kTwice) rest1 += f.y;
          }
        }
      }
    }
    float squares = square.get().x + square.get().y + square1, off = rest.get().x + rest.get().y + rest1;
    if (kTwice) {
      row_reduce2<TPR>(squares, off, SumOp(), SumOp(), scratch[1]);
      lo = off * inv_cols;
    } else {
      squares = row_reduce<TPR>(squares, SumOp(), scratch[1]);
    }
    squares *= inv_cols;
    float spread = __fmaf_rn(-lo, lo, squares), base = hi;
    if (kTwice ? !(spread == spread) : !(average * average <= 64.f * spread)) {  // the same for all threads of the row; rows that are not finite too
      base = fabsf(hi) < __int_as_float(0x7F800000) ? hi : 0.f;  // (infinities have their mean)
      off = 0.f;  // read again, in a short loop: this code runs for few rows and takes no registers from the others
#pragma unroll 1
      for (long long at = RowPlace<TPR>::thread(); at < cols; at += TPR) off += to_f32(row[at]) - base;
      lo = row_reduce<TPR>(off, SumOp(), scratch[3]) * inv_cols;
      spread = __fmaf_rn(-lo, lo, squares);
    }
    const float rstd = rsqrtf((spread < 0.f ? 0.f : spread) + eps);  // NaN stays NaN
    if (RowPlace<TPR>::thread() == 0) {
      mean_out[r] = base + lo;
      rstd_out[r] = rstd;
    }
    const Pair scale(rstd), minus_lo(-(lo * rstd));
#pragma unroll
    for (int v = 0; v < count; ++v) {
      Pair(&x)[4] = held[V > 0 ? v : 0];
      if (V == 0) read_differences(v, x);
      const Raw8<W> w = column.load(weight, v);
      Raw8<W> b;
      if (bias != nullptr) b = column.load(bias, v);
      else b.zero();
      float out[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = fma2(fma2(x[i], scale, minus_lo), Pair(w.get(2 * i), w.get(2 * i + 1)), Pair(b.get(2 * i), b.get(2 * i + 1))).get();
        out[2 * i] = f.x;
        out[2 * i + 1] = f.y;
      }
      column.store(y + r * cols, v, out);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// layer norm with quantize_tokens behind it: the normalised row never leaves the registers.
//
// A code is decided by the exact value, not by fp32's rounding of it: a value next to the border of two codes
// would otherwise go to the one or the other with the order of a sum.  The statistics are sums in fp64.  The
// values are computed in fp32, where they are off by at most E = 2^-21 (|t| + |b|), t = (x - mean) rstd w: with the mean
// in two parts, hi + lo, h = (x - hi) rstd - lo rstd.  Where x - hi is rounded it is far larger than lo; where it is not,
// it is zero, or at least 2 |lo|, or of the other sign, so that each part is at most 2 |h|.  With rstd's rounding h is off by
// at most 6 steps of 2^-24 |h|, and t + b by one of its own more.  |t| <= amax + |b|, so E <= 2^-21 (amax + 2 max|b|) for a
// whole group.  A quotient that is further than E/s from every border has its code; otherwise (once in some 10^4
// values) the eight values of the thread are computed again in fp64.  The scale is settled in the same way: where
// amax / top is within its error of a tie of two bf16 numbers, or fp32 has no room for it, the group's maximum is found
// again in fp64.  Both are loops that read their values again, out of the way of the code that runs always.
//
// 4096 x 4096 in bf16 with groups of 256: 26 us, 7 of them HBM's.  33 instructions a value (two conversions and two sums in
// fp64 among them) with pairs of fp32 numbers and three-way maxima, which is 15 us of issue; 43 without those, 30 us.  The
// other ten are the chain of a row (sums and exchanges of doubles, a barrier, the scale, the codes), with six rows an SM
// at it.  More threads an SM with fewer registers change nothing (896 and 1,024).
// ---------------------------------------------------------------------------------------------------------------
struct NormExact {
  double mean, rstd;
  __device__ __forceinline__ double value(float x, float w, float b) const {
    return (static_cast<double>(x) - mean) * rstd * static_cast<double>(w) + static_cast<double>(b);
  }
};

// Whether bf16(v) could be another number for a v that is off by `error`.
__device__ __forceinline__ bool near_bf16_tie(float v, float error) {
  const float tie = __uint_as_float((__float_as_uint(v) & 0xFFFF0000u) | 0x8000u);
  return !(fabsf(v - tie) > error);
}

// The largest size of up to eight exact values from `at` on, as a bit pattern: its order is that of the sizes, with NaN
// above infinity.
template <typename T, typename W>
__device__ __noinline__ unsigned long long exact_size(const T* row, const W* weight, const W* bias, long long at, long long cols, const NormExact& exact) {
  unsigned long long most = 0;
  for (int i = 0; i < 8 && at + i < cols; ++i) {
    const double v = exact.value(to_f32(row[at + i]), to_f32(weight[at + i]), bias != nullptr ? to_f32(bias[at + i]) : 0.f);
    most = MaxOp()(most, static_cast<unsigned long long>(__double_as_longlong(fabs(v))));
  }
  return most;
}

// Eight codes from `at` on, from exact values; zero where the scale is not finite and behind the row.
template <typename T, typename W, int BITS>
__device__ __noinline__ unsigned long long exact_codes(const T* row, const W* weight, const W* bias, long long at, long long cols,
                                                       const NormExact& exact, float s) {
  const double top = BITS == 4 ? 7.0 : 127.0;
  unsigned long long packed = 0;
  if (!(s < __int_as_float(0x7F800000))) return 0;
  for (int i = 0; i < 8 && at + i < cols; ++i) {
    const double q = rint(exact.value(to_f32(row[at + i]), to_f32(weight[at + i]), bias != nullptr ? to_f32(bias[at + i]) : 0.f) / static_cast<double>(s));
    const unsigned long long code = static_cast<unsigned long long>(static_cast<int>(fmin(fmax(q, -top), top))) & (BITS == 4 ? 0xFull : 0xFFull);
    packed |= code << (BITS * i);
  }
  return packed;
}

template <typename T, typename W, int TPR, int V, int BITS, bool kAligned>
__global__ void __launch_bounds__(RowPlace<TPR>::kThreads, (sizeof(T) == 2 ? 768 : 512) / RowPlace<TPR>::kThreads)
layer_norm_quantize_kernel(const T* __restrict__ src, const W* __restrict__ weight, const W* __restrict__ bias,
                           uint8_t* __restrict__ codes, bf16* __restrict__ scales, long long rows, long long cols, int sub_bits,
                           double inv_cols, double eps) {
  __shared__ double scratch_d[2][2 * (TPR / 32)];
  __shared__ float scratch_m[2 * (TPR / 32)];
  __shared__ unsigned long long scratch_x[TPR / 32];
  constexpr int kHeld = V > 0 ? V : 1;
  constexpr float kTop = BITS == 4 ? 7.f : 127.f;
  constexpr float kError = 4.76837158203125e-7f;  // 2^-21
  const long long pitch = BITS == 4 ? (cols + 1) / 2 : cols;
  const int lanes = sub_bits ? 1 << (sub_bits - 3) : 0;
  const long long groups = sub_bits ? (cols + (1 << sub_bits) - 1) >> sub_bits : 1;
  const int count = V > 0 ? V : static_cast<int>((cols + TPR * 8 - 1) / (TPR * 8));
  auto place = [&](int v) { return (static_cast<long long>(v) * TPR + RowPlace<TPR>::thread()) * 8; };
  auto read_affine = [&](int v, Raw8<W>& w, Raw8<W>& b) {
    w.template load<kAligned>(weight, place(v), cols);
    if (bias != nullptr) b.template load<kAligned>(bias, place(v), cols);
    else b.zero();
  };
  int turn = 0;
  for (long long r = RowPlace<TPR>::first(); r < rows; r += RowPlace<TPR>::step(), turn ^= 1) {
    const T* row = src + r * cols;
    const RowValues<T, TPR, V, kAligned> x(row, cols);
    // sums of x - shift and of its square; bf16 values need no shift (8 bits of significand against fp64's 53)
    const float shift = sizeof(T) == 4 ? to_f32(row[0]) : 0.f;
    double s1 = 0.0, s2 = 0.0;
#pragma unroll
    for (int v = 0; v < count; ++v) {
      const Raw8<T> raw = x.get(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        double d = static_cast<double>(raw.get(i));
        if (sizeof(T) == 4) d = place(v) + i < cols ? d - static_cast<double>(shift) : 0.0;
        s1 += d;
        s2 = fma(d, d, s2);
      }
    }
    row_reduce2<TPR>(s1, s2, SumOp(), SumOp(), scratch_d[turn]);
    NormExact exact;
    // the mean with one step of refinement: a row of equal values has that value as its mean, and no variance
    double off = s1 * inv_cols;
    off = fma(fma(-off, static_cast<double>(cols), s1), inv_cols, off);
    exact.mean = off + static_cast<double>(shift);
    const double spread = fma(-s1, off, s2) * inv_cols;
    const double var = fmax(spread, 0.0) + eps;
    // 1 / sqrt(var): Newton's iteration from the fp32 value, which squares the relative error each time
    double root = static_cast<double>(rsqrtf(static_cast<float>(var)));
    root = root * (1.5 - 0.5 * var * root * root);
    root = root * (1.5 - 0.5 * var * root * root);
    // beyond fp32's range, and for NaN: the library's own
    const bool wild = !(var > 1e-30 && var < 1e30);
    if (wild) root = rsqrt(spread + eps);
    exact.rstd = root;
    const float mean_hi = static_cast<float>(exact.mean);
    const float mean_lo = static_cast<float>(exact.mean - static_cast<double>(mean_hi));
    const float rstd = static_cast<float>(exact.rstd);

    const Pair minus_hi(-mean_hi), scale(rstd), minus_lo(-mean_lo * rstd);
    auto norm8 = [&](int v, Pair (&out)[4], float& amax, float& bmax) {
      if (place(v) >= cols) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = Pair(0.f);
        return;
      }
      const Raw8<T> raw = x.get(v);
      Raw8<W> w, b;
      read_affine(v, w, b);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const Pair h = fma2(add2(Pair(raw.get(i), raw.get(i + 1)), minus_hi), scale, minus_lo);
        out[i / 2] = fma2(h, Pair(w.get(i), w.get(i + 1)), Pair(b.get(i), b.get(i + 1)));
        float2 f = out[i / 2].get();
        if (!kAligned) {  // behind the row w and b are zero, but h may be infinite or NaN
          if (place(v) + i + 1 >= cols) f.y = 0.f;
          out[i / 2] = Pair(f.x, f.y);
          if (place(v) + i >= cols) out[i / 2] = Pair(0.f);
          f = out[i / 2].get();
        }
        amax = max_size(amax, f.x, f.y);
        bmax = max_size(bmax, b.get(i), b.get(i + 1));
      }
    };
    float s = 1.f, error = 0.f, delta = 0.f, inv = 1.f;
    bool ordinary = true;
    auto take_scale = [&](float scale) {
      s = nonzero_scale(scale);
      ordinary = !wild && scale_is_ordinary(s);
      inv = about_inverse(s);
      delta = error * inv + kTop * kError;
    };
    // bf16(amax / top) and the half-width of the border zones in codes; true if the scale has to be found from the
    // exact maximum
    auto scale_from = [&](float amax, float bmax) {
      const float quotient = amax * (1.f / kTop);
      error = kError * (amax + 2.f * bmax);
      take_scale(__bfloat162float(__float2bfloat16_rn(quotient)));
      if (!wild && amax == 0.f && bmax == 0.f) return false;  // with a bias, zeros may be what fp32 left of other numbers
      // what fp32 has no room for, or too few digits, is settled too
      return wild || !(amax > 1e-29f && amax < __int_as_float(0x7F800000)) || near_bf16_tie(quotient, error * (2.f / kTop));
    };
    auto settled = [&](unsigned long long most) {
      take_scale(bf16_from_double(__longlong_as_double(static_cast<long long>(most)) / static_cast<double>(kTop)));
    };
    auto put = [&](int v, const Pair (&out)[4]) {
      const long long at = place(v);
      if (at >= cols) return;
      uint32_t c[8];
      float far = 0.f;  // the largest distance of a quotient from its code
      const Pair inv2(inv);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const Pair code = fma2(out[i / 2], inv2, Pair(kRoundMagic));
        const float2 word = code.get();
        c[i] = __float_as_uint(word.x);
        c[i + 1] = __float_as_uint(word.y);
        // the code less the quotient
        const Pair minus = fma2(out[i / 2], Pair(-inv), add2(code, Pair(-kRoundMagic)));
        far = max_abs(far, minus.get().x, minus.get().y);
      }
      typename CodeWords<BITS>::type packed = CodeWords<BITS>::pack(c);
      if (!(ordinary && far < 0.5f - delta)) {
        const unsigned long long exactly = exact_codes<T, W, BITS>(row, weight, bias, at, cols, exact, s);
        memcpy(&packed, &exactly, sizeof(packed));
      }
      store_packed<BITS, kAligned>(codes + r * pitch, at, cols, packed);
    };

    Pair out[kHeld][4];
    if (!lanes) {
      float amax = 0.f, bmax = 0.f;
#pragma unroll
      for (int v = 0; v < count; ++v) norm8(v, out[V > 0 ? v : 0], amax, bmax);
      row_reduce2<TPR>(amax, bmax, MaxSizeOp(), MaxSizeOp(), scratch_m);
      if (scale_from(amax, bmax)) {  // the same for all threads of the row
        unsigned long long most = 0;
        for (int v = 0; v < count; ++v) most = MaxOp()(most, exact_size<T, W>(row, weight, bias, place(v), cols, exact));
        most = row_reduce<TPR>(most, MaxOp(), scratch_x);
        settled(most);
      }
      if (RowPlace<TPR>::thread() == 0) scales[r] = __float2bfloat16_rn(s);
#pragma unroll
      for (int v = 0; v < count; ++v) {
        float again = 0.f, unused = 0.f;
        if (V == 0) norm8(v, out[0], again, unused);
        put(v, out[V > 0 ? v : 0]);
      }
    } else {
#pragma unroll
      for (int v = 0; v < count; ++v) {
        float amax = 0.f, bmax = 0.f;
        norm8(v, out[0], amax, bmax);
        amax = warp_reduce(amax, MaxSizeOp(), lanes);
        bmax = warp_reduce(bmax, MaxSizeOp(), lanes);
        const bool settle = scale_from(amax, bmax);
        if (__any_sync(0xFFFFFFFFu, settle)) {
          const unsigned long long most = warp_reduce(exact_size<T, W>(row, weight, bias, place(v), cols, exact), MaxOp(), lanes);
          if (settle) settled(most);
        }
        if ((threadIdx.x & (lanes - 1)) == 0 && place(v) < cols) scales[r * groups + (place(v) >> sub_bits)] = __float2bfloat16_rn(s);
        put(v, out[0]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// layer norm's backward pass, with h = (x - mean) rstd and g = dy w:
//   dx = rstd (g - mean(g) - h mean(g h)),   dw = sum over rows of dy h,   db = sum over rows of dy.
// A thread keeps its columns for all of its rows, so the sums over rows stay in registers and x and dy are read once.
// A block has several groups of TPR threads, each with rows of its own (and a barrier of its own); the sums of the groups
// are added up in shared memory, each block leaves one row of partial sums, and column_sums_kernel adds those in a fixed
// order: no atomics, the same bits on every run.  Four rows of a group are on their way (in shared memory: one, in
// registers, was what bounded the kernel, with 32 KB an SM in flight; two in registers spill).
// 32768 x 2048 in bf16: 66 us, 6.1 TB/s (75 us with one row ahead), and 4 us for the partial sums, whose kernel starts
// while this one ends.
// Rows of more than 8192 values are left to two kernels, below.
// ---------------------------------------------------------------------------------------------------------------
template <int TPR>
struct BwdShape {
  static constexpr int kThreads = TPR < 512 ? 512 : TPR;
  static constexpr int kGroups = kThreads / TPR;  // rows at once
  // A thread's 64 bytes of x and dy of each row to come lie in shared memory, copied there asynchronously by the thread
  // itself: four rows of a group on their way, 128 KB in all; three with 1,024 threads, 192 KB.
  static constexpr int kAhead = kThreads == 512 ? 4 : 3;
  static constexpr int kRingBytes = kAhead * kThreads * 64;
};

__device__ __forceinline__ void copy_16(void* shared, const void* global, bool valid) {
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(shared));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(global), "r"(valid ? 16 : 0) : "memory");
}

// Barrier of one group of a block.
template <int TPR>
__device__ __forceinline__ void group_barrier(int group) {
  if (TPR > 32) asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
}

template <typename T, typename W, int TPR, int V, bool kAligned>
__global__ void __launch_bounds__(BwdShape<TPR>::kThreads)
layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ src, const W* __restrict__ weight,
                      const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
                      float* __restrict__ partial, long long rows, long long cols) {
  constexpr int kWarps = TPR / 32, kGroups = BwdShape<TPR>::kGroups;
  __shared__ float2 scratch[2][kGroups][kWarps];
  // the ring of rows to come [kAhead][4][kThreads]; behind the last row [TPR * V * 8] sums, where there are groups to be added up
  extern __shared__ __align__(16) uint8_t bwd_smem[];
  float* across = reinterpret_cast<float*>(bwd_smem);
  uint4* ring = reinterpret_cast<uint4*>(bwd_smem) + threadIdx.x;
  const int group = threadIdx.x / TPR, thread = threadIdx.x % TPR;
  const long long step = static_cast<long long>(gridDim.x) * kGroups;
  constexpr int G = kAligned ? 16 / sizeof(T) : 1;
  const Columns<TPR, G> column{thread, cols};
  const float inv_cols = 1.f / static_cast<float>(cols);
  Raw8<W> w[V];
  Pair dw[V][4], db[V][4];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    w[v] = column.load(weight, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[v][i] = db[v][i] = Pair(0.f);
  }
  constexpr int kThreads = BwdShape<TPR>::kThreads, kAhead = BwdShape<TPR>::kAhead;
  float next_mean = 0.f, next_rstd = 0.f;
  auto read_terms = [&](long long row) {
    next_mean = __ldg(mean_in + row);
    next_rstd = __ldg(rstd_in + row);
  };
  Raw8<T> next_x[kAligned ? 1 : V], next_dy[kAligned ? 1 : V];  // where rows cannot be copied 16 bytes at a time: one row in registers
  auto fetch = [&](long long row, int slot) {
    if constexpr (kAligned) {
      if (row < rows) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int i = 0; i < 8; i += G) {
            const int chunk = v * (8 / G) + i / G;
            const bool has = column.has(v, i);
            const long long at = row * cols + (has ? column.at(v, i) : 0);
            copy_16(ring + (slot * 4 + chunk) * kThreads, src + at, has);
            copy_16(ring + (slot * 4 + 2 + chunk) * kThreads, dy + at, has);
          }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    } else if (row < rows) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        next_x[v] = column.load(src + row * cols, v);
        next_dy[v] = column.load(dy + row * cols, v);
      }
    }
  };
  static_assert(V * 8 / G <= 2 || !kAligned, "two chunks of x and two of dy a thread");
  long long r = static_cast<long long>(blockIdx.x) * kGroups + group;
  if (r < rows) read_terms(r);
#pragma unroll
  for (int i = 0; i < (kAligned ? kAhead : 1); ++i) fetch(r + i * step, i);
  int turn = 0, slot = 0;
  for (; r < rows; r += step, turn ^= 1) {
    Raw8<T> x[V], d[V];
    const float mean = next_mean, rstd = next_rstd;
    if (r + step < rows) read_terms(r + step);
    if constexpr (kAligned) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v].from_chunks(ring + (slot * 4 + v) * kThreads, kThreads);
        d[v].from_chunks(ring + (slot * 4 + 2 + v) * kThreads, kThreads);
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = next_x[v];
        d[v] = next_dy[v];
      }
      fetch(r + step, 0);
    }
    auto two = [](const auto& raw, int i) { return Pair(raw.get(2 * i), raw.get(2 * i + 1)); };
    const Pair minus_mean(-mean), scale(rstd);
    Pair sums(0.f), sums_h(0.f);
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Pair e = two(d[v], i), h = mul2(add2(two(x[v], i), minus_mean), scale), g = mul2(e, two(w[v], i));
        sums = add2(sums, g);
        sums_h = fma2(g, h, sums_h);
        dw[v][i] = fma2(e, h, dw[v][i]);
        db[v][i] = add2(db[v][i], e);
      }
    }
    float sg = sums.get().x + sums.get().y, sgh = sums_h.get().x + sums_h.get().y;
    sg = warp_reduce(sg, SumOp());
    sgh = warp_reduce(sgh, SumOp());
    if constexpr (kAligned) {  // the row has been read: its place is free
      __syncwarp();
      fetch(r + kAhead * step, slot);
      if (++slot == kAhead) slot = 0;
    }
    if (TPR > 32) {
      if ((thread & 31) == 0) scratch[turn][group][thread >> 5] = make_float2(sg, sgh);
      group_barrier<TPR>(group);
      const float2 mine = scratch[turn][group][thread & (kWarps - 1)];
      sg = mine.x;
      sgh = mine.y;
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) {
        sg += __shfl_xor_sync(0xFFFFFFFFu, sg, o);
        sgh += __shfl_xor_sync(0xFFFFFFFFu, sgh, o);
      }
    }
    const Pair minus_mg(-sg * inv_cols), minus_mgh(-sgh * inv_cols);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float out[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Pair h = mul2(add2(two(x[v], i), minus_mean), scale);
        const float2 f = mul2(fma2(h, minus_mgh, fma2(two(d[v], i), two(w[v], i), minus_mg)), scale).get();
        out[2 * i] = f.x;
        out[2 * i + 1] = f.y;
      }
      column.store(dx + r * cols, v, out);
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // column_sums_kernel, which waits for this one's end
  float dw1[V][8], db1[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 fw = dw[v][i / 2].get(), fb = db[v][i / 2].get();
      dw1[v][i] = i % 2 ? fw.y : fw.x;
      db1[v][i] = i % 2 ? fb.y : fb.x;
    }
  float* mine = partial + static_cast<long long>(blockIdx.x) * 2 * cols;
  if (kGroups == 1) {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (column.has(v, i)) {
          mine[column.at(v, i)] = dw1[v][i];
          mine[cols + column.at(v, i)] = db1[v][i];
        }
    return;
  }
  // groups one after the other, in place (i * TPR * V + ...: a warp's lanes on neighbouring words)
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    for (int k = 0; k < kGroups; ++k) {
      __syncthreads();
      if (group == k) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float* at = across + (v * 8 + i) * TPR + thread;
            const float sum = half ? db1[v][i] : dw1[v][i];
            *at = k == 0 ? sum : *at + sum;
          }
      }
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (column.has(v, i)) mine[half * cols + column.at(v, i)] = across[(v * 8 + i) * TPR + thread];
    }
  }
}

// Rows of more than 8192 values, whose columns do not fit the registers of one block: the means of g and g h of every
// row, and then dx and the sums over rows with a thread for each chunk of columns, which needs no reduction over the
// row.  x and dy are read twice, the second time from L2 as far as it holds them.  517 rows of 14336 values: 26 us in fp32,
// 12 to 13 of them for the means, 21 in bf16.  (A block of 1024 threads a row took 47 us in fp32, clusters of two blocks 37,
// both waiting for their reductions with one row ahead; neither has been tried with the ring of the kernel above.)
struct __align__(16) RowTerms {
  float mean, rstd, mean_g, mean_gh;
};

template <typename T, typename W, bool kAligned>
__global__ void __launch_bounds__(512)
layer_norm_bwd_rows_kernel(const T* __restrict__ dy, const T* __restrict__ src, const W* __restrict__ weight,
                           const float* __restrict__ mean_in, const float* __restrict__ rstd_in, RowTerms* __restrict__ terms,
                           long long rows, long long cols) {
  constexpr int TPR = 512, G = kAligned ? 16 / sizeof(T) : 1;
  __shared__ float scratch[2][2 * (TPR / 32)];
  const float inv_cols = 1.f / static_cast<float>(cols);
  const Columns<TPR, G> column{static_cast<int>(threadIdx.x), cols};
  const int count = static_cast<int>((cols + TPR * 8 - 1) / (TPR * 8));
  int turn = 0;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x, turn ^= 1) {
    const T* x_row = src + r * cols;
    const T* d_row = dy + r * cols;
    const float mean = __ldg(mean_in + r), rstd = __ldg(rstd_in + r);
    float sg = 0.f, sgh = 0.f;
#pragma unroll 2
    for (int v = 0; v < count; ++v) {
      const Raw8<T> x = column.load(x_row, v), d = column.load(d_row, v);
      const Raw8<W> w = column.load(weight, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float g = d.get(i) * w.get(i);
        sg += g;
        sgh = __fmaf_rn(g, (x.get(i) - mean) * rstd, sgh);
      }
    }
    row_reduce2<TPR>(sg, sgh, SumOp(), SumOp(), scratch[turn]);
    if (threadIdx.x == 0) terms[r] = RowTerms{mean, rstd, sg * inv_cols, sgh * inv_cols};
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// A block has a strip of 32 chunks of G columns and a part of the rows, which its eight warps take in turns; the sums
// of the warps are added in order and leave one row of partial sums for each part.
constexpr int kStripWarps = 8;

template <typename T, typename W, int G>
__global__ void __launch_bounds__(32 * kStripWarps)
layer_norm_bwd_strips_kernel(const T* __restrict__ dy, const T* __restrict__ src, const W* __restrict__ weight,
                             const RowTerms* terms, T* __restrict__ dx, float* __restrict__ partial, long long rows, long long cols) {
  constexpr int kAtOnce = 4;
  __shared__ float across[2][kStripWarps][32 * G];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long col = (static_cast<long long>(blockIdx.x) * 32 + lane) * G;
  const bool inside = col < cols;
  const long long row0 = rows * blockIdx.y / gridDim.y, row1 = rows * (blockIdx.y + 1) / gridDim.y;
  struct Chunk {
    T e[G];
  };
  auto read = [&](const T* p) {
    Chunk c;
    if constexpr (G * sizeof(T) == 16) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      memcpy(c.e, &v, 16);
    } else {
#pragma unroll
      for (int i = 0; i < G; ++i) c.e[i] = p[i];
    }
    return c;
  };
  float w[G], dw[G], db[G];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    w[i] = inside ? to_f32(weight[col + i]) : 0.f;
    dw[i] = db[i] = 0.f;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (inside) {
    for (long long r0 = row0 + warp; r0 < row1; r0 += kStripWarps * kAtOnce) {
      Chunk x[kAtOnce], d[kAtOnce];
      RowTerms t[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const long long r = r0 + k * kStripWarps;
        if (r >= row1) continue;
        x[k] = read(src + r * cols + col);
        d[k] = read(dy + r * cols + col);
        t[k] = terms[r];
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const long long r = r0 + k * kStripWarps;
        if (r >= row1) continue;
        float out[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
          const float e = to_f32(d[k].e[i]), h = (to_f32(x[k].e[i]) - t[k].mean) * t[k].rstd;
          dw[i] = __fmaf_rn(e, h, dw[i]);
          db[i] += e;
          out[i] = t[k].rstd * (e * w[i] - t[k].mean_g - h * t[k].mean_gh);
        }
        T* to = dx + r * cols + col;
        if constexpr (G == 8) *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3]), pack_bf16x2(out[4], out[5]), pack_bf16x2(out[6], out[7]));
        else if constexpr (G == 4) *reinterpret_cast<float4*>(to) = make_float4(out[0], out[1], out[2], out[3]);
        else to[0] = static_cast<T>(out[0]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < G; ++i) {
    across[0][warp][i * 32 + lane] = dw[i];
    across[1][warp][i * 32 + lane] = db[i];
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __syncthreads();
  for (int k = threadIdx.x; k < 2 * 32 * G; k += 32 * kStripWarps) {
    const int half = k / (32 * G), place = k % (32 * G);
    const long long c = (static_cast<long long>(blockIdx.x) * 32 + place % 32) * G + place / 32;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kStripWarps; ++j) sum += across[half][j][place];
    if (c < cols) partial[(2LL * blockIdx.y + half) * cols + c] = sum;
  }
}

// Adds up the rows of partial sums: a block for 32 columns, kSumRows rows at a time, in a fixed order.
constexpr int kSumRows = 16;

static __global__ void __launch_bounds__(32 * kSumRows)
column_sums_kernel(const float* __restrict__ partial, int parts, long long cols, float* __restrict__ dweight, float* __restrict__ dbias) {
  const long long col = static_cast<long long>(blockIdx.x) * 32 + threadIdx.x;
  float sw = 0.f, sb = 0.f;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (col < cols) {
#pragma unroll 8
    for (int p = threadIdx.y; p < parts; p += kSumRows) {
      sw += partial[(2LL * p) * cols + col];
      sb += partial[(2LL * p + 1) * cols + col];
    }
  }
  __shared__ float tile[2][kSumRows][33];
  tile[0][threadIdx.y][threadIdx.x] = sw;
  tile[1][threadIdx.y][threadIdx.x] = sb;
  __syncthreads();
  // the first warp adds up dw, the second db, a column a lane
  if (threadIdx.y < 2 && col < cols) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kSumRows; ++k) sum += tile[threadIdx.y][k][threadIdx.x];
    (threadIdx.y == 0 ? dweight : dbias)[col] = sum;
  }
}

}  // namespace b200
