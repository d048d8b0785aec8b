// Kernels that go over rows of values once: the quantiser with a scale for each token, layer norm, layer norm
// with the quantiser behind it, and layer norm's backward pass.  All of them are bound by HBM on large inputs.
//
// One row belongs to a warp (TPR == 32, up to 1024 values) or to a block of TPR threads; a thread holds V groups
// of eight consecutive values in registers, group v of thread t at (v * TPR + t) * 8, so that a row is read once
// and a warp's load covers consecutive bytes.  V == 0 is the form for rows that no block can hold: the same code,
// reading the row again (from L2) for every pass over it.
#pragma once

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
template <int TPR, int V, int BITS, bool kAligned>
__global__ void __launch_bounds__(RowPlace<TPR>::kThreads)
quantize_tokens_kernel(const bf16* __restrict__ src, uint8_t* __restrict__ codes, bf16* __restrict__ scales,
                       long long rows, long long cols, int sub) {
  __shared__ uint32_t scratch[2][TPR / 32];
  const long long pitch = BITS == 4 ? (cols + 1) / 2 : cols;
  const int lanes = sub >> 3;  // of a group; 0: one scale a row
  const long long groups = sub ? (cols + sub - 1) / sub : 1;
  int turn = 0;
  for (long long r = RowPlace<TPR>::first(); r < rows; r += RowPlace<TPR>::step(), turn ^= 1) {
    const RowValues<bf16, TPR, V, kAligned> x(src + r * cols, cols);
    float s = 1.f;
    if (!lanes) {
      uint32_t m = 0;
#pragma unroll
      for (int v = 0; v < x.count(); ++v) {
        const Raw8<bf16> raw = x.get(v);
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, raw.w[i] & 0x7FFF7FFFu);
      }
      m = max(m & 0xFFFFu, m >> 16);
      s = scale_of_bf16<BITS>(row_reduce<TPR>(m, MaxOp(), scratch[turn]));
      if (RowPlace<TPR>::thread() == 0) scales[r] = __float2bfloat16_rn(s);
    }
#pragma unroll
    for (int v = 0; v < x.count(); ++v) {
      const Raw8<bf16> raw = x.get(v);
      const long long at = x.at(v);
      if (lanes) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, raw.w[i] & 0x7FFF7FFFu);
        m = warp_reduce(max(m & 0xFFFFu, m >> 16), MaxOp(), lanes);
        s = scale_of_bf16<BITS>(m);
        if ((threadIdx.x & (lanes - 1)) == 0 && at < cols) scales[r * groups + at / sub] = __float2bfloat16_rn(s);
      }
      uint32_t c[8];
      if (scale_is_ordinary(s)) {
        const ExactQuotient q(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = q.code(raw.get(i));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = code_by_division<BITS>(raw.get(i), s);
      }
      store_codes<BITS, kAligned>(codes + r * pitch, at, cols, c);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// layer norm: y = (x - mean) rstd w + b; mean, then the mean square of the differences, both from registers, in fp32.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, typename W, int TPR, int V, bool kAligned>
__global__ void __launch_bounds__(RowPlace<TPR>::kThreads)
layer_norm_kernel(const T* __restrict__ src, const W* __restrict__ weight, const W* __restrict__ bias, T* __restrict__ y,
                  float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows, long long cols, float eps) {
  __shared__ float scratch[2][TPR / 32];
  const float inv_cols = 1.f / static_cast<float>(cols);
  for (long long r = RowPlace<TPR>::first(); r < rows; r += RowPlace<TPR>::step()) {
    const RowValues<T, TPR, V, kAligned> x(src + r * cols, cols);
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < x.count(); ++v) {
      const Raw8<T> raw = x.get(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += raw.get(i);
    }
    const float mean = row_reduce<TPR>(sum, SumOp(), scratch[0]) * inv_cols;
    float square = 0.f;
#pragma unroll
    for (int v = 0; v < x.count(); ++v) {
      const Raw8<T> raw = x.get(v);
      const long long at = x.at(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = raw.get(i) - mean;
        if (at + i < cols) square = __fmaf_rn(d, d, square);
      }
    }
    const float rstd = rsqrtf(row_reduce<TPR>(square, SumOp(), scratch[1]) * inv_cols + eps);
    if (RowPlace<TPR>::thread() == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
#pragma unroll
    for (int v = 0; v < x.count(); ++v) {
      const Raw8<T> raw = x.get(v);
      const long long at = x.at(v);
      Raw8<W> w, b;
      w.template load<kAligned>(weight, at, cols);
      if (bias != nullptr) b.template load<kAligned>(bias, at, cols);
      else b.zero();
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = __fmaf_rn((raw.get(i) - mean) * rstd, w.get(i), b.get(i));
      store8<kAligned>(y + r * cols, at, cols, out);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// layer norm with quantize_tokens behind it: the normalised row never leaves the registers.
//
// A code is decided by the exact value, not by fp32's rounding of it: a value next to the border of two codes
// would otherwise go to the one or the other with the order of a sum.  The statistics are sums in fp64.  The
// values are computed in fp32, where they are off by at most E = 2^-21 (|t| + |b|), t = (x - mean) rstd w (four
// roundings of 2^-24 each, and room); |t| <= amax + |b|, so E <= 2^-21 (amax + 2 max|b|) for a whole group.  If
// q - E/s and q + E/s round to one integer, that is the code; otherwise (once in some 10^4 values) the value is
// computed again in fp64.  The scale is settled in the same way: where amax / top is within its error of a tie of
// two bf16 numbers, the group's maximum is found again in fp64.
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

template <typename T, typename W, int TPR, int V, int BITS, bool kAligned>
__global__ void __launch_bounds__(RowPlace<TPR>::kThreads)
layer_norm_quantize_kernel(const T* __restrict__ src, const W* __restrict__ weight, const W* __restrict__ bias,
                           uint8_t* __restrict__ codes, bf16* __restrict__ scales, long long rows, long long cols, int sub,
                           double inv_cols, double eps) {
  __shared__ double scratch_d[2 * (TPR / 32)];
  __shared__ uint32_t scratch_m[2 * (TPR / 32)];
  __shared__ double scratch_x[TPR / 32];
  constexpr float kTop = BITS == 4 ? 7.f : 127.f;
  constexpr float kError = 4.76837158203125e-7f;  // 2^-21
  const long long pitch = BITS == 4 ? (cols + 1) / 2 : cols;
  const int lanes = sub >> 3;
  const long long groups = sub ? (cols + sub - 1) / sub : 1;
  for (long long r = RowPlace<TPR>::first(); r < rows; r += RowPlace<TPR>::step()) {
    const RowValues<T, TPR, V, kAligned> x(src + r * cols, cols);
    // sums of x - shift and of its square; bf16 values need no shift (8 bits of significand against fp64's 53)
    const float shift = sizeof(T) == 4 ? to_f32(src[r * cols]) : 0.f;
    double s1 = 0.0, s2 = 0.0;
#pragma unroll
    for (int v = 0; v < x.count(); ++v) {
      const Raw8<T> raw = x.get(v);
      const long long at = x.at(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        double d = static_cast<double>(raw.get(i));
        if (sizeof(T) == 4) d = at + i < cols ? d - static_cast<double>(shift) : 0.0;
        s1 += d;
        s2 = fma(d, d, s2);
      }
    }
    row_reduce2<TPR>(s1, s2, SumOp(), SumOp(), scratch_d);
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
    if (!(var > 1e-30 && var < 1e30)) root = rsqrt(spread + eps);
    exact.rstd = root;
    const float mean_hi = static_cast<float>(exact.mean);
    const float mean_lo = static_cast<float>(exact.mean - static_cast<double>(mean_hi));
    const float rstd = static_cast<float>(exact.rstd);

    // amax (as bits: NaN is above infinity) and max |b|
    uint32_t amax = 0, bmax = 0;
    float s = 1.f, delta = 0.f;
    bool ordinary = false;
    auto norm8 = [&](const Raw8<T>& raw, long long at, Raw8<W>& w, Raw8<W>& b, float (&out)[8]) {
      w.template load<kAligned>(weight, at, cols);
      if (bias != nullptr) b.template load<kAligned>(bias, at, cols);
      else b.zero();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        out[i] = __fmaf_rn(((raw.get(i) - mean_hi) - mean_lo) * rstd, w.get(i), b.get(i));
        if (!kAligned && at + i >= cols) out[i] = 0.f;
        amax = max(amax, __float_as_uint(out[i]) & 0x7FFFFFFFu);
        bmax = max(bmax, __float_as_uint(b.get(i)) & 0x7FFFFFFFu);
      }
    };
    // bf16(amax / top), and the half-width of the border zones in codes.  `settle`: the scale has to be found from
    // the exact maximum.
    auto scale_from = [&](bool& settle) {
      const float most = __uint_as_float(amax), error = kError * (most + 2.f * __uint_as_float(bmax));
      const float quotient = __fdiv_rn(most, kTop);
      s = nonzero_scale(__bfloat162float(__float2bfloat16_rn(quotient)));
      ordinary = scale_is_ordinary(s);
      delta = error * __frcp_rn(s) + kTop * kError;
      settle = most < __int_as_float(0x7F800000) && most > 0.f && near_bf16_tie(quotient, error);
    };

    if (!lanes) {
      float out[8];
      Raw8<W> w, b;
#pragma unroll
      for (int v = 0; v < x.count(); ++v)
        if (x.at(v) < cols) norm8(x.get(v), x.at(v), w, b, out);
      row_reduce2<TPR>(amax, bmax, MaxOp(), MaxOp(), scratch_m);
      bool settle;
      scale_from(settle);
      if (settle) {  // the same for all threads of the row
        double most = 0.0;
        for (int v = 0; v < x.count(); ++v) {
          const long long at = x.at(v);
          const Raw8<T> raw = x.get(v);
          if (at >= cols) continue;
          w.template load<kAligned>(weight, at, cols);
          if (bias != nullptr) b.template load<kAligned>(bias, at, cols);
          else b.zero();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (at + i < cols) most = fmax(most, fabs(exact.value(raw.get(i), w.get(i), b.get(i))));
        }
        most = row_reduce<TPR>(most, MaxOp(), scratch_x);
        s = nonzero_scale(bf16_from_double(most / static_cast<double>(kTop)));
        if (TPR > 32) __syncthreads();  // scratch_x may be used again by the next row
      }
      if (RowPlace<TPR>::thread() == 0) scales[r] = __float2bfloat16_rn(s);
    }

    const float inv = __frcp_rn(s);
#pragma unroll
    for (int v = 0; v < x.count(); ++v) {
      const long long at = x.at(v);
      const Raw8<T> raw = x.get(v);
      Raw8<W> w, b;
      float out[8];
      w.zero();
      b.zero();
      if (lanes) {
        amax = bmax = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = 0.f;
      }
      if (at < cols) norm8(raw, at, w, b, out);
      float inv_group = inv;
      if (lanes) {
        amax = warp_reduce(amax, MaxOp(), lanes);
        bmax = warp_reduce(bmax, MaxOp(), lanes);
        bool settle;
        scale_from(settle);
        if (__any_sync(0xFFFFFFFFu, settle)) {
          double most = 0.0;
          if (at < cols)
            for (int i = 0; i < 8; ++i)
              if (at + i < cols) most = fmax(most, fabs(exact.value(raw.get(i), w.get(i), b.get(i))));
          most = warp_reduce(most, MaxOp(), lanes);
          if (settle) s = nonzero_scale(bf16_from_double(most / static_cast<double>(kTop)));
        }
        inv_group = __frcp_rn(s);
        if ((threadIdx.x & (lanes - 1)) == 0 && at < cols) scales[r * groups + at / sub] = __float2bfloat16_rn(s);
      }
      if (at >= cols) continue;
      uint32_t c[8], border = ordinary ? 0u : 1u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = __float_as_uint(__fadd_rn(__fmaf_rn(out[i], inv_group, -delta), kRoundMagic));
        border |= c[i] ^ __float_as_uint(__fadd_rn(__fmaf_rn(out[i], inv_group, delta), kRoundMagic));
      }
      if (border) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (at + i >= cols || !(s < __int_as_float(0x7F800000))) {
            c[i] = 0u;  // outside the row, or a row that is not finite
          } else {
            const double q = rint(exact.value(raw.get(i), w.get(i), b.get(i)) / static_cast<double>(s));
            c[i] = static_cast<uint32_t>(static_cast<int>(fmin(fmax(q, -static_cast<double>(kTop)), static_cast<double>(kTop))));
          }
        }
      }
      store_codes<BITS, kAligned>(codes + r * pitch, at, cols, c);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// layer norm's backward pass, with h = (x - mean) rstd and g = dy w:
//   dx = rstd (g - mean(g) - h mean(g h)),   dw = sum over rows of dy h,   db = sum over rows of dy.
// A thread keeps its eight columns for all of its block's rows, so the sums over rows stay in registers (or, for
// wide rows, in shared memory) and x and dy are read once.  Each block leaves one row of partial sums;
// column_sums_kernel adds those in a fixed order: no atomics, the same bits on every run.
// The next row is read while the present one is reduced.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, typename W, int TPR, bool kAligned>
__global__ void __launch_bounds__(RowPlace<TPR>::kThreads, TPR == 1024 ? 1 : (TPR == 32 ? 3 : 768 / TPR))
layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ src, const W* __restrict__ weight,
                      const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
                      float* __restrict__ partial, long long rows, long long cols) {
  __shared__ float scratch[2][2 * (TPR / 32)];
  __shared__ float across[TPR == 32 ? 8 * 256 : 1];
  const float inv_cols = 1.f / static_cast<float>(cols);
  const long long at = RowPlace<TPR>::thread() * 8LL;
  float w[8], dw[8], db[8];
  {
    Raw8<W> raw;
    raw.template load<kAligned>(weight, at, cols);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = raw.get(i);
      dw[i] = db[i] = 0.f;
    }
  }
  Raw8<T> next_x, next_dy;
  float next_mean = 0.f, next_rstd = 0.f;
  long long r = RowPlace<TPR>::first();
  auto fetch = [&](long long row) {
    next_x.template load<kAligned>(src + row * cols, at, cols);
    next_dy.template load<kAligned>(dy + row * cols, at, cols);
    next_mean = __ldg(mean_in + row);
    next_rstd = __ldg(rstd_in + row);
  };
  if (r < rows) fetch(r);
  int turn = 0;
  for (; r < rows; r += RowPlace<TPR>::step(), turn ^= 1) {
    const Raw8<T> x = next_x, d = next_dy;
    const float mean = next_mean, rstd = next_rstd;
    if (r + RowPlace<TPR>::step() < rows) fetch(r + RowPlace<TPR>::step());
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float h = (x.get(i) - mean) * rstd, g = d.get(i) * w[i];
      sg += g;
      sgh = __fmaf_rn(g, h, sgh);
      dw[i] = __fmaf_rn(d.get(i), h, dw[i]);
      db[i] += d.get(i);
    }
    row_reduce2<TPR>(sg, sgh, SumOp(), SumOp(), scratch[turn]);
    const float mg = sg * inv_cols, mgh = sgh * inv_cols;
    float out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float h = (x.get(i) - mean) * rstd;
      out[i] = rstd * (d.get(i) * w[i] - mg - h * mgh);
    }
    store8<kAligned>(dx + r * cols, at, cols, out);
  }
  float* mine = partial + static_cast<long long>(blockIdx.x) * 2 * cols;
  if (TPR == 32) {  // eight warps with the same columns
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int warp = threadIdx.x >> 5;
#pragma unroll
      for (int i = 0; i < 8; ++i) across[warp * 256 + i * 32 + (threadIdx.x & 31)] = half ? db[i] : dw[i];
      __syncthreads();
      const int col = threadIdx.x;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += across[k * 256 + (col & 7) * 32 + (col >> 3)];
      if (col < cols) mine[half * cols + col] = sum;
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (at + i < cols) {
        mine[at + i] = dw[i];
        mine[cols + at + i] = db[i];
      }
    }
  }
}

// The same for rows of up to 16384 values: two groups of eight a thread, the sums over rows in shared memory
// (8 bytes a column), where each thread touches its own columns only.
template <typename T, typename W, bool kAligned>
__global__ void __launch_bounds__(1024)
layer_norm_bwd_wide_kernel(const T* __restrict__ dy, const T* __restrict__ src, const W* __restrict__ weight,
                           const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
                           float* __restrict__ partial, long long rows, long long cols) {
  constexpr int TPR = 1024, V = 2;
  extern __shared__ float sums[];  // [2][V][8][1024]: value i of group v of thread t at ((v * 8 + i) * 1024 + t)
  __shared__ float scratch[2][2 * (TPR / 32)];
  const float inv_cols = 1.f / static_cast<float>(cols);
  float* sum_w = sums + threadIdx.x;
  float* sum_b = sums + V * 8 * TPR + threadIdx.x;
#pragma unroll
  for (int k = 0; k < V * 8; ++k) sum_w[k * TPR] = sum_b[k * TPR] = 0.f;
  int turn = 0;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x, turn ^= 1) {
    const RowValues<T, TPR, V, kAligned> x(src + r * cols, cols);
    const RowValues<T, TPR, V, kAligned> d(dy + r * cols, cols);
    const float mean = __ldg(mean_in + r), rstd = __ldg(rstd_in + r);
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Raw8<W> w;
      w.template load<kAligned>(weight, x.at(v), cols);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = d.held[v].get(i), h = (x.held[v].get(i) - mean) * rstd, g = e * w.get(i);
        sg += g;
        sgh = __fmaf_rn(g, h, sgh);
        sum_w[(v * 8 + i) * TPR] = __fmaf_rn(e, h, sum_w[(v * 8 + i) * TPR]);
        sum_b[(v * 8 + i) * TPR] += e;
      }
    }
    row_reduce2<TPR>(sg, sgh, SumOp(), SumOp(), scratch[turn]);
    const float mg = sg * inv_cols, mgh = sgh * inv_cols;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Raw8<W> w;
      w.template load<kAligned>(weight, x.at(v), cols);
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float h = (x.held[v].get(i) - mean) * rstd;
        out[i] = rstd * (d.held[v].get(i) * w.get(i) - mg - h * mgh);
      }
      store8<kAligned>(dx + r * cols, x.at(v), cols, out);
    }
  }
  float* mine = partial + static_cast<long long>(blockIdx.x) * 2 * cols;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const long long at = (static_cast<long long>(v) * TPR + threadIdx.x) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (at + i < cols) {
        mine[at + i] = sum_w[(v * 8 + i) * TPR];
        mine[cols + at + i] = sum_b[(v * 8 + i) * TPR];
      }
    }
  }
}

// Rows of more than 16384 values: dx alone, reading the row twice, and the sums over rows column by column.
template <typename T, typename W, bool kAligned>
__global__ void __launch_bounds__(1024)
layer_norm_bwd_long_kernel(const T* __restrict__ dy, const T* __restrict__ src, const W* __restrict__ weight,
                           const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
                           long long rows, long long cols) {
  constexpr int TPR = 1024;
  __shared__ float scratch[2][2 * (TPR / 32)];
  const float inv_cols = 1.f / static_cast<float>(cols);
  int turn = 0;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x, turn ^= 1) {
    const RowValues<T, TPR, 0, kAligned> x(src + r * cols, cols);
    const RowValues<T, TPR, 0, kAligned> d(dy + r * cols, cols);
    const float mean = __ldg(mean_in + r), rstd = __ldg(rstd_in + r);
    float sg = 0.f, sgh = 0.f;
    for (int v = 0; v < x.count(); ++v) {
      const Raw8<T> xv = x.get(v), dv = d.get(v);
      Raw8<W> w;
      w.template load<kAligned>(weight, x.at(v), cols);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float g = dv.get(i) * w.get(i);
        sg += g;
        sgh = __fmaf_rn(g, (xv.get(i) - mean) * rstd, sgh);
      }
    }
    row_reduce2<TPR>(sg, sgh, SumOp(), SumOp(), scratch[turn]);
    const float mg = sg * inv_cols, mgh = sgh * inv_cols;
    for (int v = 0; v < x.count(); ++v) {
      const Raw8<T> xv = x.get(v), dv = d.get(v);
      Raw8<W> w;
      w.template load<kAligned>(weight, x.at(v), cols);
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = rstd * (dv.get(i) * w.get(i) - mg - (xv.get(i) - mean) * rstd * mgh);
      store8<kAligned>(dx + r * cols, x.at(v), cols, out);
    }
  }
}

// Block of 32 columns x 32 rows at a time; the 32 sums of a column are added in a fixed order.
__device__ __forceinline__ void column_finish(float sw, float sb, long long col, long long cols, float* dweight, float* dbias) {
  __shared__ float tile[2][32][33];
  tile[0][threadIdx.y][threadIdx.x] = sw;
  tile[1][threadIdx.y][threadIdx.x] = sb;
  __syncthreads();
  // warp y takes column y of the tile
  const float a = warp_reduce(tile[0][threadIdx.x][threadIdx.y], SumOp());
  const float b = warp_reduce(tile[1][threadIdx.x][threadIdx.y], SumOp());
  const long long mine = col - threadIdx.x + threadIdx.y;
  if (threadIdx.x == 0 && mine < cols) {
    dweight[mine] = a;
    dbias[mine] = b;
  }
}

static __global__ void __launch_bounds__(1024)
column_sums_kernel(const float* __restrict__ partial, int parts, long long cols, float* __restrict__ dweight, float* __restrict__ dbias) {
  const long long col = static_cast<long long>(blockIdx.x) * 32 + threadIdx.x;
  float sw = 0.f, sb = 0.f;
  if (col < cols) {
#pragma unroll 4
    for (int p = threadIdx.y; p < parts; p += 32) {
      sw += __ldg(partial + (2LL * p) * cols + col);
      sb += __ldg(partial + (2LL * p + 1) * cols + col);
    }
  }
  column_finish(sw, sb, col, cols, dweight, dbias);
}

template <typename T>
__global__ void __launch_bounds__(1024)
layer_norm_bwd_columns_kernel(const T* __restrict__ dy, const T* __restrict__ src, const float* __restrict__ mean_in,
                              const float* __restrict__ rstd_in, long long rows, long long cols, float* __restrict__ dweight,
                              float* __restrict__ dbias) {
  const long long col = static_cast<long long>(blockIdx.x) * 32 + threadIdx.x;
  float sw = 0.f, sb = 0.f;
  if (col < cols) {
    for (long long r = threadIdx.y; r < rows; r += 32) {
      const float d = to_f32(dy[r * cols + col]);
      sw = __fmaf_rn(d, (to_f32(src[r * cols + col]) - __ldg(mean_in + r)) * __ldg(rstd_in + r), sw);
      sb += d;
    }
  }
  column_finish(sw, sb, col, cols, dweight, dbias);
}

}  // namespace b200
