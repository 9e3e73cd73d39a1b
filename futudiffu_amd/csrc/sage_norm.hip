// The RMS norms around the attention of a transformer block, for gfx950: before
// it with the modulation's scale, after it with the gate and the residual, and
// the norm after one half of a block together with the one before the next.
//
//   xhat = x * rrms, rrms = 1 / sqrt(mean(x^2) + eps)   over the C channels of a token
//   modulate:       y = xhat * w * (1 + s)
//   gate:           y = r + g * xhat * w
//   gate, modulate: h = r + g * xhat * w,  y = norm(h) * w2 * (1 + s2)
//
// s, g and s2 have a row per batch item, or, with document ids, per document (a
// token of no document has s = g = s2 = 0).  With m = 1 + s or g, constant over the
// tokens of one row, and d the gradient of the normed output, the backward is
//
//   dx = rrms * (d*w*m - xhat * mean(d*w*m * xhat))
//   S[row] = sum over its tokens of d * xhat;  ds = dg = w * S;  dw = sum over rows of m * S
//
// so the channel sums need one fp32 accumulator a channel, whatever the documents.
// All arithmetic is fp32; each output is rounded once.  h enters the second norm
// unrounded, in the backward too, which forms it again from r and x (it reads as
// many tensors as with h, and dw2 and ds2 stay fp32-exact).
//
// Every kernel is bound by memory: a token's channels are held in registers between
// the reads and the writes, so each tensor is touched once.
#include <algorithm>
#include <type_traits>

#include "sage_common.h"
#include "sage_launch.h"
#include "sage_mx.h"

namespace sage {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kVec = 8;      // channels of one 16-byte access
constexpr int kPer = 16;     // channels a thread holds of a token

template <typename T>
struct Vec8;
template <>
struct Vec8<__bf16> {
  typedef bf16x8 type;
};
template <>
struct Vec8<_Float16> {
  typedef f16x8 type;
};

// Sum over the 64 lanes of a wave, in all of them: a fixed tree of lane distances 1,
// 2, 4, 8 (DPP within rows of 16), 16 and 32.
__device__ __forceinline__ float wave_sum(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v += dpp(v, std::integral_constant<int, 0xb1>{});   // quad_perm [1,0,3,2]
  v += dpp(v, std::integral_constant<int, 0x4e>{});   // quad_perm [2,3,0,1]
  v += dpp(v, std::integral_constant<int, 0x141>{});  // row_half_mirror: the other quad of eight lanes
  v += dpp(v, std::integral_constant<int, 0x140>{});  // row_mirror: the other eight of sixteen
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const uint32_t w = __float_as_uint(v);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Sums of K values over the TPR threads of a token, in all of them.  `red`: a slot of
// (waves of the workgroup) x K floats that no thread of an earlier sum still reads.
template <int TPR, int K>
__device__ __forceinline__ void token_sum(float (&v)[K], float* red, int wave) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave * K + k] = v[k];
    }
    __syncthreads();
    const int w0 = wave / W * W;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = red[w0 * K + k];
#pragma unroll
      for (int w = 1; w < W; ++w) s += red[(w0 + w) * K + k];
      v[k] = s;
    }
  }
}

// The channels a thread holds: with VEC two runs of eight, 16-byte accesses; without
// (odd widths, misaligned rows), every TPR-th channel, so that a wave's accesses are
// consecutive.
template <int TPR, bool VEC>
struct Cols {
  static __device__ __forceinline__ int col(int t, int j) {
    return VEC ? ((j / kVec) * TPR + t) * kVec + j % kVec : j * TPR + t;
  }
};

// Rows are read and written through a buffer resource that ends at the row's last
// channel: reads past it give zeros and writes past it are dropped, so no access is
// behind a branch.  A row is uniform over a wave.  One thread's channels of a row of T
// stay as they lie in memory until they are used.
template <typename T, int TPR, bool VEC>
struct Raw {
  using V = typename Vec8<T>::type;
  V v[kPer / kVec];
  __device__ __forceinline__ void load(const T* row, int t, int c) {
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(row, (uint32_t)c * 2);
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kPer / kVec; ++i)
        v[i] = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(rs, (i * TPR + t) * kVec * 2, 0, 0));
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        v[j / kVec][j % kVec] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(rs, (j * TPR + t) * 2, 0, 0));
    }
  }
  __device__ __forceinline__ float operator[](int j) const { return (float)v[j / kVec][j % kVec]; }
};

template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void store_row(T* row, int t, int c, const float (&f)[kPer]) {
  const __amdgpu_buffer_rsrc_t rs = raw_rsrc(row, (uint32_t)c * 2);
  if constexpr (VEC) {
    using V = typename Vec8<T>::type;
#pragma unroll
    for (int i = 0; i < kPer / kVec; ++i) {
      V o;
#pragma unroll
      for (int j = 0; j < kVec; ++j) o[j] = (T)f[i * kVec + j];
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), rs, (i * TPR + t) * kVec * 2, 0, 0);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (T)f[j]), rs, (j * TPR + t) * 2, 0, 0);
  }
}

// A thread's channels of a parameter row (T or fp32, or none: `fill`).
template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void load_param(const void* p, bool f32, int64_t off, int t, int c, float fill,
                                           float (&f)[kPer]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) f[j] = fill;
  } else if (f32) {
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(static_cast<const float*>(p) + off, (uint32_t)c * 4);
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kPer / 4; ++i) {
        const int at = Cols<TPR, VEC>::col(t, i * 4);
        const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at * 4, 0, 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) f[i * 4 + j] = v[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        f[j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, Cols<TPR, VEC>::col(t, j) * 4, 0, 0));
    }
  } else {
    Raw<T, TPR, VEC> r;
    r.load(static_cast<const T*>(p) + off, t, c);
#pragma unroll
    for (int j = 0; j < kPer; ++j) f[j] = r[j];
  }
}

__device__ __forceinline__ float rrms(float sum_sq, int c, float eps) {
  return 1.0f / sqrtf(sum_sq / (float)c + eps);
}

// w * (scale ? 1 + s : g) of conditioning row `id` of batch item b (id < 0 or >= groups: no
// document), of one thread's channels.
template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void weight_row(const NormParam& w, const NormCond& k, bool scale, int b, int id, int t,
                                           int c, float (&wm)[kPer]) {
  float m[kPer];
  load_param<T, TPR, VEC>(w.p, w.f32, 0, t, c, 1.0f, wm);
  const bool live = k.p && id >= 0 && id < k.groups;
  load_param<T, TPR, VEC>(live ? k.p : nullptr, k.f32, b * k.bs + id * k.gs, t, c, scale || k.p ? 0.0f : 1.0f, m);
#pragma unroll
  for (int j = 0; j < kPer; ++j) wm[j] *= scale ? 1.0f + m[j] : m[j];
}

template <typename T>
__device__ __forceinline__ const T* row_of(const NormRows& r, int b, int64_t n) {
  return static_cast<const T*>(r.p) + b * r.bs + n * r.rs;
}

// A token of no document behind a gate: its x is not read (whatever padding holds there
// reaches neither the output nor a gradient), xhat is 0.
__device__ __forceinline__ bool no_document(const NormArgs& a, int id) {
  return a.doc && a.cond.p && (id < 0 || id >= a.groups);
}

// Forward: TPR threads a token, one token a thread group, so a token's whole row is in flight
// at once and the many small workgroups keep the memory busy through each other's sums.  All
// loads of a token, the parameter rows included, are issued before its first sum.  Measured:
// gate of 4416 x 3840 bf16, 102 MB in 16.9 us; gate + modulate of 4 x 4352 x 3840, 535 MB in
// 109 us = 4.9 TB/s, a large copy's rate; modulate of 32 tokens, 3.1 us of latency.
template <typename T, int OP, int TPR, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_fwd_kernel(NormArgs a) {
  constexpr int NT = TPR > 256 ? TPR : 256;
  constexpr int TOK = NT / TPR;
  __shared__ float red[NT / 64], red2[NT / 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * TOK + wave / (TPR / 64), rows = (int64_t)a.b * a.n;
  const bool live = row < rows;  // a thread group past the last token takes part in the barriers alone
  const int b = live ? (int)(row / a.n) : 0;
  const int64_t n = live ? row - (int64_t)b * a.n : 0;
  const int c = live ? a.c : 0;
  Raw<T, TPR, VEC> x, r;
  const int id = a.doc && live ? load_uniform(a.doc, row) : 0;
  const bool gated = OP == kNormModulate || !no_document(a, id);
  x.load(row_of<T>(a.x, b, n), t, gated ? c : 0);
  if constexpr (OP != kNormModulate) r.load(row_of<T>(a.res, b, n), t, c);
  float wm[kPer], wm2[kPer];
  weight_row<T, TPR, VEC>(a.w, a.cond, OP == kNormModulate, b, id, t, c, wm);
  if constexpr (OP == kNormGateModulate) weight_row<T, TPR, VEC>(a.w2, a.cond2, true, b, id, t, c, wm2);
  float s[1] = {0.0f};
#pragma unroll
  for (int j = 0; j < kPer; ++j) s[0] += x[j] * x[j];
  token_sum<TPR>(s, red, wave);
  const float rr = gated ? rrms(s[0], a.c, a.eps) : 0.0f;
  float y[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    y[j] = x[j] * rr * wm[j];
    if constexpr (OP != kNormModulate) y[j] += r[j];
  }
  if constexpr (OP == kNormGateModulate) {
    if (live) store_row<T, TPR, VEC>(static_cast<T*>(a.hidden) + row * a.c, t, c, y);
    s[0] = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) s[0] += y[j] * y[j];
    token_sum<TPR>(s, red2, wave);
    const float r2 = rrms(s[0], a.c, a.eps);
#pragma unroll
    for (int j = 0; j < kPer; ++j) y[j] = y[j] * r2 * wm2[j];
  }
  if (live) store_row<T, TPR, VEC>(static_cast<T*>(a.out) + row * a.c, t, c, y);
}

// ---------------------------------------------------------------- norms into MXFP4

// A thread's channels of a row of E for the quantization: two runs of eight whatever the access, so
// that a block of 32 is four neighbouring lanes'.
template <typename E, int TPR, bool VEC>
__device__ __forceinline__ void load_runs(const E* row, int t, int c, float (&f)[kPer]) {
  const __amdgpu_buffer_rsrc_t rs = raw_rsrc(row, (uint32_t)c * (uint32_t)sizeof(E));
#pragma unroll
  for (int i = 0; i < kPer / kVec; ++i) {
    const int at = (i * TPR + t) * kVec;
    if constexpr (VEC && sizeof(E) == 2) {
      const auto v = __builtin_bit_cast(typename Vec8<E>::type, __builtin_amdgcn_raw_buffer_load_b128(rs, at * 2, 0, 0));
#pragma unroll
      for (int j = 0; j < kVec; ++j) f[i * kVec + j] = (float)v[j];
    } else if constexpr (VEC) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at * 4 + q * 16, 0, 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) f[i * kVec + q * 4 + j] = v[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if constexpr (sizeof(E) == 2)
          f[i * kVec + j] = (float)__builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b16(rs, (at + j) * 2, 0, 0));
        else
          f[i * kVec + j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, (at + j) * 4, 0, 0));
      }
    }
  }
}

template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void param_runs(const void* p, bool f32, int64_t off, int t, int c, float fill,
                                           float (&f)[kPer]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) f[j] = fill;
  } else if (f32) {
    load_runs<float, TPR, VEC>(static_cast<const float*>(p) + off, t, c, f);
  } else {
    load_runs<T, TPR, VEC>(static_cast<const T*>(p) + off, t, c, f);
  }
}

// scale or gate of conditioning row `id` (weight_row's rule).
template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void cond_runs(const NormCond& k, bool scale, int b, int id, int t, int c, float (&f)[kPer]) {
  const bool live = k.p && id >= 0 && id < k.groups;
  param_runs<T, TPR, VEC>(live ? k.p : nullptr, k.f32, b * k.bs + id * k.gs, t, c, scale || k.p ? 0.0f : 1.0f, f);
}

// wave_sum of fp64 values.
__device__ __forceinline__ double wave_sum64(double v) {
  auto moved = [](double x, auto move) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)move((uint32_t)(u >> 32)) << 32 | move((uint32_t)u));
  };
  auto dpp = [&](double x, auto ctrl) {
    return moved(x, [](uint32_t w) {
      return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, decltype(ctrl)::value, 0xf, 0xf, true);
    });
  };
  v += dpp(v, std::integral_constant<int, 0xb1>{});
  v += dpp(v, std::integral_constant<int, 0x4e>{});
  v += dpp(v, std::integral_constant<int, 0x141>{});
  v += dpp(v, std::integral_constant<int, 0x140>{});
  const bool up16 = threadIdx.x & 16, up32 = threadIdx.x & 32;
  v += moved(v, [&](uint32_t w) {
    const auto s = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return up16 ? s[0] : s[1];
  });
  v += moved(v, [&](uint32_t w) {
    const auto s = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return up32 ? s[0] : s[1];
  });
  return v;
}

// token_sum of one fp64 value.
template <int TPR>
__device__ __forceinline__ double token_sum64(double v, double* red, int wave) {
  v = wave_sum64(v);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    const int w0 = wave / W * W;
    v = red[w0];
#pragma unroll
    for (int w = 1; w < W; ++w) v += red[w0 + w];
  }
  return v;
}

// 1 / sqrt(sum_sq / c + eps) by v_rsq_f64 (2^-23 off or less) and one step of third order: a sixth of the
// instructions of the library's root and quotient.
__device__ __forceinline__ double rrms64(double sum_sq, double inv_c, double eps) {
  const double v = fma(sum_sq, inv_c, eps), r = __builtin_amdgcn_rsq(v);
  const double e = fma(-v * r, r, 1.0);
  return e == e ? fma(r * e, fma(e, 0.375, 0.5), r) : r;  // of 0 and infinity
}

// fp64 to fp32 by rounding to odd: what lies beside a border between two codes stays on its
// side when the codes are taken from the fp32 value.
__device__ __forceinline__ float to_odd(double y) {
  const float f = (float)y;
  const double d = y - (double)f;
  const bool past = fabs((double)f) > fabs(y);  // the rounding went away from zero
  uint32_t u = __float_as_uint(f);
  if (d != 0.0 && d == d) u = (u - (past ? 1u : 0u)) | 1u;  // d is NaN where y is, or infinite
  return __uint_as_float(u);
}

// A lane's eight channels (from `at` on, of c) to codes and the scale of their block.  y: the values
// in fp32, off by less than 7 of its roundings (2^-24 each); exact(j): in fp64.  Where y (1 +- 2^-21) have the same
// codes and scale, so has the exact value; where they have not (one in 10^6 values) the wave takes the
// codes from the exact ones.  So it does where fp32's range may have cost more than that: `odd`, and a block below
// 2^-30 (one of zeros, and those behind the last column) or not finite.
template <typename Exact>
__device__ __forceinline__ uint32_t mx_codes(const float (&y)[kVec], bool odd, int at, int c, Exact exact, int& e) {
  constexpr float kLow = 1.0f - 0x1p-21f, kHigh = 1.0f + 0x1p-21f;
  float top = fabsf(y[0]);  // NaN if one is
#pragma unroll
  for (int j = 1; j < kVec; ++j) top = __builtin_elementwise_maximum(top, fabsf(y[j]));
  const float t = __uint_as_float(quad_max(__float_as_uint(top)));
  e = block_exponent(__float_as_uint(t * kLow));
  odd = odd || e == 255 || e != block_exponent(__float_as_uint(t * kHigh)) || t < 0x1p-30f;
  const float sc = scale_of(e);
  uint32_t lo = 0, hi = 0;
  auto two = [&](auto q) {
    constexpr int Q = decltype(q)::value;
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, y[2 * Q] * kLow, y[2 * Q + 1] * kLow, sc, Q);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(hi, y[2 * Q] * kHigh, y[2 * Q + 1] * kHigh, sc, Q);
  };
  two(std::integral_constant<int, 0>{});
  two(std::integral_constant<int, 1>{});
  two(std::integral_constant<int, 2>{});
  two(std::integral_constant<int, 3>{});
  if (__ballot(odd || lo != hi) == 0) return lo;
  float f[kVec];
  auto take = [&](double unit) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      f[j] = at + j < c ? to_odd(exact(j) * unit) : 0.0f;
      most = max(most, __float_as_uint(f[j]) & 0x7fffffffu);
    }
    return quad_max(most);
  };
  uint32_t most = take(1.0);
  // a finite value past fp32's range became its largest: such a block's are taken 2^-16 times, and past the
  // largest scale (2^127) the code is that of 6
  int up = 0;
  if (__ballot(most == 0x7f7fffffu)) {
    up = most == 0x7f7fffffu ? 16 : 0;
    most = take(up ? 0x1p-16 : 1.0);
    const float six = up ? 6.0f * 0x1p111f : INFINITY;
#pragma unroll
    for (int j = 0; j < kVec; ++j) f[j] = fminf(fmaxf(f[j], -six), six);
  }
  e = block_exponent(most);
  e = e == 255 ? 255 : min(e, 254 - up);
  const float s = scale_of(e);
  e = e == 255 ? 255 : e + up;
  uint32_t q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0], f[1], s, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[2], f[3], s, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[4], f[5], s, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[6], f[7], s, 3);
  return e == 255 ? 0u : q;
}

// Forward of the modulated norms with y in MXFP4: norm_fwd_kernel's shares.  fp32 would put one value in
// 10^6 on the other side of a border between two codes, a whole step away: sums, and the hidden stream, are
// fp64, and the codes those of the exact values (mx_codes).  The instructions bound it (401 a wave for its 16
// channels a lane, of them 39 fp64 sums and products and 44 conversions; gated 730, 118 and 118): 25 us for 6912
// tokens of 3840 channels modulated, 35 us for 4416 gated and modulated, where the bytes take 13.5 and 22.6.  All
// of it in fp64 took 30.5 and 39.2; a wave a token with 64 channels a lane, which does the sums over lanes once
// for four times the channels, 25.7 and, for its registers, 69; several tokens a workgroup with their
// parameters kept and the next token's rows on their way, 24.6 and 33.9 at best.
template <typename T, int OP, int TPR, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_mx_kernel(NormArgs a, uint8_t* codes, uint8_t* scales) {
  constexpr int NT = TPR > 256 ? TPR : 256;
  constexpr int TOK = NT / TPR;
  constexpr bool kGate = OP == kNormGateModulate;
  __shared__ double red[NT / 64], red2[NT / 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * TOK + wave / (TPR / 64), rows = (int64_t)a.b * a.n;
  const bool live = row < rows;  // a thread group past the last token takes part in the barriers alone
  const int b = live ? (int)((uint32_t)row / (uint32_t)a.n) : 0;  // rows are fewer than 2^23
  const int64_t n = live ? row - (int64_t)b * a.n : 0;
  const int c = live ? a.c : 0;
  const int id = a.doc && live ? load_uniform(a.doc, row) : 0;
  const bool gated = OP == kNormModulate || !no_document(a, id);
  // w, k: the parameters behind the last norm; w1, g: the gated one's
  float x[kPer], r[kPer], w1[kPer], g[kPer], w[kPer], k[kPer];
  load_runs<T, TPR, VEC>(row_of<T>(a.x, b, n), t, gated ? c : 0, x);
  if constexpr (kGate) {
    load_runs<T, TPR, VEC>(row_of<T>(a.res, b, n), t, c, r);
    param_runs<T, TPR, VEC>(a.w.p, a.w.f32, 0, t, c, 1.0f, w1);
    cond_runs<T, TPR, VEC>(a.cond, false, b, id, t, c, g);
  }
  param_runs<T, TPR, VEC>(kGate ? a.w2.p : a.w.p, kGate ? a.w2.f32 : a.w.f32, 0, t, c, 1.0f, w);
  cond_runs<T, TPR, VEC>(kGate ? a.cond2 : a.cond, true, b, id, t, c, k);
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) s = fma((double)x[j], (double)x[j], s);
  s = token_sum64<TPR>(s, red, wave);
  double rr = gated ? rrms64(s, a.inv_c, a.eps64) : 0.0;
  double h[kPer];  // what the last norm takes
  if constexpr (kGate) {
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(static_cast<T*>(a.hidden) + row * a.c, (uint32_t)c * 2);
    s = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      h[j] = fma((double)x[j] * rr, (double)w1[j] * (double)g[j], (double)r[j]);
      s = fma(h[j], h[j], s);
    }
#pragma unroll
    for (int i = 0; i < kPer / kVec; ++i) {
      // rounded by way of fp32, but for what lies between two values of T there
      constexpr uint32_t kTie = std::is_same<T, __bf16>::value ? 0x7fffu : 0xfffu;
      float f[kVec];
      bool tie = false;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        f[j] = (float)h[i * kVec + j];
        tie = tie || (__float_as_uint(f[j]) & kTie) == 0;
      }
      if (__ballot(tie)) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) f[j] = to_odd(h[i * kVec + j]);
      }
      const int at = (i * TPR + t) * kVec;
      if constexpr (VEC) {
        typename Vec8<T>::type o;
#pragma unroll
        for (int j = 0; j < kVec; ++j) o[j] = (T)f[j];
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), rs, at * 2, 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (T)f[j]), rs, (at + j) * 2, 0, 0);
      }
    }
    s = token_sum64<TPR>(s, red2, wave);
    rr = rrms64(s, a.inv_c, a.eps64);
  }
  // rf * wm can leave fp32's range at the bottom only where |wm| is under 2^-66, so that the value is 0 beside
  // any block that counts
  const float rf = (float)rr;
  const bool odd = !(rf > 0x1p-60f && rf < 0x1p60f);
  const int kp = (a.c + 255) / 256 * 256;
#pragma unroll
  for (int i = 0; i < kPer / kVec; ++i) {
    const int at = (i * TPR + t) * kVec;
    float y[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int v = i * kVec + j;
      y[j] = (kGate ? (float)h[v] : x[v]) * (rf * (w[v] * (1.0f + k[v])));
    }
    int e;
    const uint32_t q = mx_codes(y, odd, at, a.c, [&](int j) {
      const int v = i * kVec + j;
      return (kGate ? h[v] : (double)x[v]) * rr * (double)w[v] * (1.0 + (double)k[v]);
    }, e);
    if (live && at < kp) {
      *reinterpret_cast<uint32_t*>(codes + row * (kp / 2) + at / 2) = q;
      if ((t & 3) == 0) scales[((int64_t)(at >> 8) * rows + row) * 8 + (at >> 5 & 7)] = (uint8_t)e;
    }
  }
}

constexpr int kBwdNT = 512;  // threads of a backward workgroup; also the most tokens of its chunk

// One token's tensors in the backward.
template <typename T, int OP, int TPR, bool VEC>
struct BwdRow {
  Raw<T, TPR, VEC> x, d, r, dh;  // r, dh: gate_modulate alone
  __device__ __forceinline__ void load(const NormArgs& a, int b, int64_t n, int t, int c, bool gated) {
    x.load(row_of<T>(a.x, b, n), t, gated ? c : 0);
    d.load(row_of<T>(a.dout, b, n), t, c);
    if constexpr (OP == kNormGateModulate) {
      r.load(row_of<T>(a.res, b, n), t, c);
      dh.load(row_of<T>(a.dhidden, b, n), t, c);
    }
  }
};

// Adds the groups' channel sums (halves of the groups at a time, a fixed tree) and stores
// them as one partial row.  `sum`: G / 2 rows of TPR * kPer floats.
template <int TPR, bool VEC>
__device__ __forceinline__ void store_partial(float* dst, float* sum, int grp, int t, int c, float (&acc)[kPer]) {
#pragma unroll
  for (int half = kBwdNT / TPR / 2; half > 0; half /= 2) {
    // a thread's value j lies at j * TPR + t: no bank conflicts
    if (grp >= half && grp < 2 * half) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) sum[((grp - half) * kPer + j) * TPR + t] = acc[j];
    }
    __syncthreads();
    if (grp < half) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) acc[j] += sum[(grp * kPer + j) * TPR + t];
    }
    __syncthreads();
  }
  if (grp == 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int at = Cols<TPR, VEC>::col(t, j);
      if (at < c) dst[at] = acc[j];
    }
  }
}

// Backward: a workgroup takes a chunk of consecutive tokens of one batch item, its
// kBwdNT / TPR thread groups one token each at a time, the next token's loads in flight
// under the present one's sums.  With document ids the chunk's tokens are taken document
// by document (ids in order, the tokens of none last), so m is constant over a run and its
// S is one partial row: part[chunk][slot][set][cp], its id in part_id.  Runs are few (a
// chunk has as many as it has documents), and the order is fixed by the ids alone.  One
// workgroup a CU, so that the partial rows are few.  Measured: modulate of 6912 x 3840 bf16
// in three documents, 159 MB in 33 us = 4.8 TB/s; gate + modulate of 3071 x 3840, 141 MB in
// 38.5 us = 3.7 TB/s: six steps a workgroup, two tokens in flight and two behind them, and the
// start and the two sets of partial rows around them (its second and third sum as one, with
// the parts of the third in which the gradient of h is linear: 39.6).
template <typename T, int OP, int TPR, bool VEC>
__global__ __launch_bounds__(kBwdNT, 2) void norm_bwd_kernel(NormArgs a) {
  constexpr int G = kBwdNT / TPR, W = kBwdNT / 64;
  constexpr int SETS = OP == kNormGateModulate ? 2 : 1;
  constexpr bool kScale = OP == kNormModulate;
  __shared__ float red[2][W * 2], red1[W], red3[W];
  __shared__ float sum[G == 1 ? 1 : G / 2 * TPR * kPer];
  __shared__ int ids_min[W], counts[W];
  __shared__ uint16_t list[kBwdNT];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int t = threadIdx.x % TPR, grp = wave / (TPR / 64);
  const int b = blockIdx.x / a.chunks;
  const int64_t n0 = (int64_t)(blockIdx.x % a.chunks) * a.chunk;
  const int len = (int)(a.n - n0 < a.chunk ? a.n - n0 : a.chunk);
  const int c = a.c;
  const bool sums = a.part != nullptr;

  int my = 0x7fffffff, prev = -1, slot = 0, done = 0;
  if (a.doc && (int)threadIdx.x < len) {
    my = a.doc[(int64_t)b * a.n + n0 + threadIdx.x];
    if (my < 0 || my >= a.groups) my = a.groups;
  }
  while (done < len) {
    // the next run: its id and its tokens
    int id = 0, run = len;  // uniform
    if (a.doc) {
      int least = my > prev ? my : 0x7fffffff;
#pragma unroll
      for (int s = 1; s < 64; s *= 2) least = min(least, __shfl_xor(least, s));
      if (lane == 0) ids_min[wave] = least;
      __syncthreads();
      id = ids_min[0];
#pragma unroll
      for (int w = 1; w < W; ++w) id = min(id, ids_min[w]);
      id = __builtin_amdgcn_readfirstlane(id);
      const uint64_t mine = __ballot(my == id);
      if (lane == 0) counts[wave] = __popcll(mine);
      __syncthreads();
      int before = 0;
      run = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        before += w < wave ? counts[w] : 0;
        run += counts[w];
      }
      run = __builtin_amdgcn_readfirstlane(run);
      if (my == id) list[before + __popcll(mine & ((1ull << lane) - 1))] = (uint16_t)threadIdx.x;
      prev = id;
      __syncthreads();
    }
    // the first tokens' loads, then the parameters', in flight together
    const bool gated = kScale || !no_document(a, id);
    BwdRow<T, OP, TPR, VEC> cur, next;
    auto token = [&](int pos) { return n0 + (a.doc ? __builtin_amdgcn_readfirstlane(list[pos]) : pos); };
    // a group past its last token loads nothing (its channels are zeros)
    cur.load(a, b, grp < run ? token(grp) : n0, t, grp < run ? c : 0, gated);
    float wm[kPer], wm2[kPer], acc[kPer] = {}, acc2[kPer] = {};
    weight_row<T, TPR, VEC>(a.w, a.cond, kScale, b, id, t, c, wm);
    if constexpr (SETS == 2) weight_row<T, TPR, VEC>(a.w2, a.cond2, true, b, id, t, c, wm2);
    const int iters = (run + G - 1) / G;
#pragma unroll 1
    for (int it = 0; it < iters; ++it) {
      const int pos = it * G + grp, npos = pos + G;
      const int64_t n = pos < run ? token(pos) : n0;
      if (it + 1 < iters) next.load(a, b, npos < run ? token(npos) : n0, t, npos < run ? c : 0, gated);
      const int64_t at = ((int64_t)b * a.n + n) * c;
      const bool has = gated && pos < run;  // zeros else, whose norm is not formed (infinite where eps is 0)
      float o[kPer];
      if constexpr (OP != kNormGateModulate) {
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          s[0] += cur.x[j] * cur.x[j];
          s[1] += cur.d[j] * wm[j] * cur.x[j];
        }
        token_sum<TPR>(s, red[it & 1], wave);
        const float r = has ? rrms(s[0], c, a.eps) : 0.0f, k = s[1] * r / (float)c;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const float xh = cur.x[j] * r;
          o[j] = r * (cur.d[j] * wm[j] - xh * k);
          acc[j] += cur.d[j] * xh;
        }
      } else {
        float s1[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < kPer; ++j) s1[0] += cur.x[j] * cur.x[j];
        token_sum<TPR>(s1, red1, wave);
        const float r1 = has ? rrms(s1[0], c, a.eps) : 0.0f;
        float s[2] = {0.0f, 0.0f};
        float h[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          h[j] = cur.r[j] + cur.x[j] * r1 * wm[j];
          s[0] += h[j] * h[j];
          s[1] += cur.d[j] * wm2[j] * h[j];
        }
        token_sum<TPR>(s, red[it & 1], wave);
        const float r2 = pos < run ? rrms(s[0], c, a.eps) : 0.0f, k2 = s[1] * r2 / (float)c;
        float s3[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const float hh = h[j] * r2;
          acc2[j] += cur.d[j] * hh;
          h[j] = cur.dh[j] + r2 * (cur.d[j] * wm2[j] - hh * k2);  // the gradient of h
          s3[0] += h[j] * wm[j] * cur.x[j];
        }
        if (pos < run) store_row<T, TPR, VEC>(static_cast<T*>(a.dres) + at, t, c, h);
        token_sum<TPR>(s3, red3, wave);
        const float k1 = s3[0] * r1 / (float)c;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const float xh = cur.x[j] * r1;
          o[j] = r1 * (h[j] * wm[j] - xh * k1);
          acc[j] += h[j] * xh;
        }
      }
      if (pos < run && a.dx) store_row<T, TPR, VEC>(static_cast<T*>(a.dx) + at, t, c, o);
      cur = next;
    }
    if (sums) {
      const int64_t p = ((int64_t)blockIdx.x * a.slots + slot) * SETS;
      store_partial<TPR, VEC>(a.part + p * a.cp, sum, grp, t, c, acc);
      if constexpr (SETS == 2) store_partial<TPR, VEC>(a.part + (p + 1) * a.cp, sum, grp, t, c, acc2);
      if (a.doc && threadIdx.x == 0) a.part_id[(int64_t)blockIdx.x * a.slots + slot] = id;
    }
    done += run;
    ++slot;
    // the sums' slots and the list are read no more when the next run writes them
    __syncthreads();
  }
  if (sums && a.doc)
    for (int s = slot + (int)threadIdx.x; s < a.slots; s += kBwdNT) a.part_id[(int64_t)blockIdx.x * a.slots + s] = -1;
}

// The parameters' gradients from the partial rows, in jobs of one workgroup: first dw = sum
// over all partials of m * S, 64 channels a job; then dcond[b][g] = w * (sum of the partials
// of its id), `cond_blocks` jobs a row, each every cond_blocks-th 64 channels.
// 16 threads of 4 channels; the workgroup's 32 thread rows take every 32nd partial and are
// added in order at the end.  All of it is latency, so the loads of kBatch partials are in
// flight together, and two workgroups a CU: with eight partials a batch (160 registers, one
// workgroup a CU) three documents of 6912 x 3840 took 8.0 us for 7.0, both sets of 3071 x 3840
// 9.8 for 7.4; with the conditioning loaded value by value 9.2 and 12.6.
//
// A chunk's ids ascend and end in -1, so a row's partials are found by a search in each
// chunk, one thread a chunk, once a job: 4000 documents in 16384 tokens of 2304 channels
// took 5.5 ms with a scan of every chunk's ids, and take 58 us.
constexpr int kParamRows = 32, kBatch = 4, kParamNT = 16 * kParamRows;

template <typename T>
__device__ __forceinline__ float param_value(const void* p, bool f32, int64_t at) {
  return f32 ? static_cast<const float*>(p)[at] : (float)static_cast<const T*>(p)[at];
}

// Stores acc * w (null: acc) at row `row` of dst.
template <typename T>
__device__ __forceinline__ void store_param(const f32x4& acc, int col, int c, NormParam w, void* dst, bool f32,
                                            int64_t row) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int at = col + j;
    if (at >= c) continue;
    const float v = w.p ? acc[j] * param_value<T>(w.p, w.f32, at) : acc[j];
    if (f32)
      static_cast<float*>(dst)[row * c + at] = v;
    else
      static_cast<T*>(dst)[row * c + at] = (T)v;
  }
}

// The thread rows' sums added in order, in the first of them; true there.
__device__ __forceinline__ bool add_rows(f32x4& acc, f32x4 (*sum)[16]) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  __syncthreads();  // an earlier block of channels has been read
  sum[ty][tx] = acc;
  __syncthreads();
  if (ty != 0) return false;
#pragma unroll
  for (int i = 1; i < kParamRows; ++i) acc += sum[i][tx];
  return true;
}

// Four consecutive values as they lie in memory, in one load (WHOLE) or up to the row's last.
template <bool WHOLE, typename U>
__device__ __forceinline__ void load_four(const U* p, int last, uint32_t (&v)[4]) {
  U u[4];
  if constexpr (WHOLE) {
    __builtin_memcpy(u, p, sizeof(u));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = p[min(j, last)];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = u[j];
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kParamNT, 4) void norm_param_kernel(NormArgs a, int sets, int modulate, int cond_blocks) {
  __shared__ f32x4 sum[kParamRows][16];
  __shared__ int list[kParamNT], counts[kParamNT / 64];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, blocks = (a.c + 63) / 64;
  const int dws = sets * blocks;
  auto partial = [&](int set, int64_t q, int s, int col) {
    return *reinterpret_cast<const f32x4*>(a.part + ((q * a.slots + s) * sets + set) * a.cp + col);
  };
  if ((int)blockIdx.x < dws) {
    const int set = blockIdx.x / blocks, col = (blockIdx.x - set * blocks) * 64 + tx * 4;
    const NormParam w = set ? a.w2 : a.w;
    const NormCond k = set ? a.cond2 : a.cond;
    void* dst = set ? a.dw2 : a.dw;
    if (!dst) return;  // uniform over the workgroup
    const bool scale = set || modulate;
    f32x4 acc = {};
    const int last = col < a.cp ? a.b * a.chunks : 0;
    for (int q0 = ty; q0 < last; q0 += kParamRows * kBatch) {
      int id[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int q = q0 + i * kParamRows;
        id[i] = q >= last ? -1 : a.doc ? a.part_id[(int64_t)q * a.slots] : 0;
      }
      // a chunk's first document, then its others
      for (int s = 0; s < a.slots; ++s) {
        // every load of the batch before the first use, none behind a branch of its own: a
        // partial of no document takes row 0 of the conditioning and a factor of its own
        f32x4 v[kBatch];
        uint32_t raw[kBatch][4] = {};
        int more[kBatch], any = -1;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int q = q0 + i * kParamRows;
          more[i] = id[i] >= 0 && s + 1 < a.slots ? a.part_id[(int64_t)q * a.slots + s + 1] : -1;
          v[i] = id[i] >= 0 ? partial(set, q, s, col) : f32x4{};
        }
        auto row = [&](int i) {
          const bool live = id[i] >= 0 && id[i] < k.groups;
          return live ? ((q0 + i * kParamRows) / a.chunks) * k.bs + id[i] * k.gs + col : (int64_t)col;
        };
        if (k.p && k.f32) {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) load_four<WHOLE>(static_cast<const uint32_t*>(k.p) + row(i), a.c - 1 - col, raw[i]);
        } else if (k.p) {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) load_four<WHOLE>(static_cast<const uint16_t*>(k.p) + row(i), a.c - 1 - col, raw[i]);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const bool live = k.p && id[i] >= 0 && id[i] < k.groups;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float given = k.f32 ? __uint_as_float(raw[i][j]) : (float)__builtin_bit_cast(T, (uint16_t)raw[i][j]);
            const float m = live ? given : scale || k.p ? 0.0f : 1.0f;
            acc[j] += (scale ? m + 1.0f : m) * v[i][j];
          }
          id[i] = more[i];
          any = max(any, id[i]);
        }
        if (any < 0) break;
      }
    }
    if (add_rows(acc, sum)) store_param<T>(acc, col, a.c, NormParam{}, dst, w.f32, 0);
    return;
  }
  const int job = blockIdx.x - dws, row = job / cond_blocks, set = row / (a.b * a.groups);
  const int at = row - set * a.b * a.groups, b = at / a.groups, g = at - b * a.groups;
  void* dst = set ? a.dcond2 : a.dcond;
  if (!dst) return;
  const int first = b * a.chunks, window = a.doc ? kParamNT : a.chunks;
  const bool f32 = set ? a.cond2.f32 : a.cond.f32;
  int count = 0;
  for (int block = job - row * cond_blocks; block < blocks; block += cond_blocks) {
    const int col = block * 64 + tx * 4;
    f32x4 acc = {};
    for (int w0 = 0; w0 < a.chunks; w0 += window) {
      // the partials of id g in this window of chunks, listed once where one window is all
      if (!a.doc) {
        count = a.chunks;
      } else if (a.chunks > window || block < cond_blocks) {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, q = w0 + (int)threadIdx.x;
        int lo = 0;
        bool found = false;
        if (q < a.chunks) {
          const int* ids = a.part_id + (int64_t)(first + q) * a.slots;
          if (a.slots <= kBatch) {  // all of them at once: one latency
#pragma unroll
            for (int s = 0; s < kBatch; ++s)
              if (s < a.slots && ids[s] == g) {
                lo = s;
                found = true;
              }
          } else {
            int hi = a.slots;  // the first id that is not below g (-1 is above all)
            while (lo < hi) {
              const int mid = (lo + hi) / 2;
              if ((uint32_t)ids[mid] < (uint32_t)g) lo = mid + 1;
              else hi = mid;
            }
            found = lo < a.slots && ids[lo] == g;
          }
        }
        const uint64_t mine = __ballot(found);
        __syncthreads();  // the last window's list has been read
        if (lane == 0) counts[wave] = __popcll(mine);
        __syncthreads();
        int before = 0;
        count = 0;
#pragma unroll
        for (int i = 0; i < kParamNT / 64; ++i) {
          before += i < wave ? counts[i] : 0;
          count += counts[i];
        }
        if (found) list[before + __popcll(mine & ((1ull << lane) - 1))] = q * a.slots + lo;
        __syncthreads();
      }
      if (a.doc && a.chunks <= window && count <= kBatch) {
        // few partials: a thread row adds them all, the rows take blocks of channels in turn
        for (int k = block + ty * cond_blocks; k < blocks; k += kParamRows * cond_blocks) {
          const int at_col = k * 64 + tx * 4;
          if (at_col >= a.cp) continue;
          f32x4 v[kBatch], s = {};
#pragma unroll
          for (int i = 0; i < kBatch; ++i) v[i] = i < count ? partial(set, first, list[i], at_col) : f32x4{};
#pragma unroll
          for (int i = 0; i < kBatch; ++i) s += v[i];
          store_param<T>(s, at_col, a.c, set ? a.w2 : a.w, dst, f32, at);
        }
        return;
      }
      if (col >= a.cp) continue;
      for (int e0 = ty; e0 < count; e0 += kParamRows * kBatch) {
        f32x4 v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int e = e0 + i * kParamRows;
          v[i] = f32x4{};
          if (e < count) v[i] = partial(set, first, a.doc ? list[e] : e, col);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) acc += v[i];
      }
    }
    if (add_rows(acc, sum)) store_param<T>(acc, col, a.c, set ? a.w2 : a.w, dst, f32, at);
  }
}

// Whether every row of the call allows 16-byte accesses.
bool all_vec(const NormArgs& a) {
  bool ok = a.c % kVec == 0;
  auto rows = [&](const NormRows& r) {
    if (r.p)
      ok = ok && (reinterpret_cast<uintptr_t>(r.p) & 15) == 0 && (a.b == 1 || r.bs % kVec == 0) &&
           (a.n == 1 || r.rs % kVec == 0);
  };
  auto cond = [&](const NormCond& k) {
    if (k.p)
      ok = ok && (reinterpret_cast<uintptr_t>(k.p) & 15) == 0 && (a.b == 1 || k.bs % kVec == 0) &&
           (k.groups == 1 || k.gs % kVec == 0);
  };
  auto ptr = [&](const void* p) { ok = ok && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  rows(a.x), rows(a.res), rows(a.dout), rows(a.dhidden);
  cond(a.cond), cond(a.cond2);
  ptr(a.w.p), ptr(a.w2.p);
  ptr(a.out), ptr(a.hidden), ptr(a.dx), ptr(a.dres);
  return ok;
}

template <typename T, int OP, int TPR, bool VEC>
hipError_t fwd(const NormArgs& a, hipStream_t st) {
  constexpr int NT = TPR > 256 ? TPR : 256, TOK = NT / TPR;
  const int64_t rows = (int64_t)a.b * a.n;
  norm_fwd_kernel<T, OP, TPR, VEC><<<(uint32_t)((rows + TOK - 1) / TOK), NT, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T, int OP, int TPR, bool VEC>
hipError_t bwd(const NormArgs& a, hipStream_t st) {
  norm_bwd_kernel<T, OP, TPR, VEC><<<(uint32_t)((int64_t)a.b * a.chunks), kBwdNT, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T, int OP, int TPR>
hipError_t fwd_mx(const NormArgs& a, uint8_t* codes, uint8_t* scales, hipStream_t st) {
  constexpr int NT = TPR > 256 ? TPR : 256, TOK = NT / TPR;
  const uint32_t grid = (uint32_t)(((int64_t)a.b * a.n + TOK - 1) / TOK);
  if (all_vec(a)) norm_mx_kernel<T, OP, TPR, true><<<grid, NT, 0, st>>>(a, codes, scales);
  else norm_mx_kernel<T, OP, TPR, false><<<grid, NT, 0, st>>>(a, codes, scales);
  return hipGetLastError();
}

template <typename T, int OP>
hipError_t mx_width(const NormArgs& a, uint8_t* codes, uint8_t* scales, hipStream_t st) {
  if (a.c <= 64 * kPer) return fwd_mx<T, OP, 64>(a, codes, scales, st);
  if (a.c <= 256 * kPer) return fwd_mx<T, OP, 256>(a, codes, scales, st);
  return fwd_mx<T, OP, 512>(a, codes, scales, st);
}

template <bool BWD, typename T, int OP, int TPR>
hipError_t pick_vec(const NormArgs& a, hipStream_t st) {
  if (all_vec(a)) return BWD ? bwd<T, OP, TPR, true>(a, st) : fwd<T, OP, TPR, true>(a, st);
  return BWD ? bwd<T, OP, TPR, false>(a, st) : fwd<T, OP, TPR, false>(a, st);
}

template <bool BWD, typename T, int OP>
hipError_t pick_width(const NormArgs& a, hipStream_t st) {
  if (a.c <= 64 * kPer) return pick_vec<BWD, T, OP, 64>(a, st);
  if (a.c <= 256 * kPer) return pick_vec<BWD, T, OP, 256>(a, st);
  return pick_vec<BWD, T, OP, 512>(a, st);
}

template <bool BWD, typename T>
hipError_t pick_op(int op, const NormArgs& a, hipStream_t st) {
  if (op == kNormModulate) return pick_width<BWD, T, kNormModulate>(a, st);
  if (op == kNormGate) return pick_width<BWD, T, kNormGate>(a, st);
  return pick_width<BWD, T, kNormGateModulate>(a, st);
}

}  // namespace

NormChunks norm_chunks(int64_t b, int64_t n, int64_t c, int64_t groups, bool doc) {
  const int64_t g = kBwdNT / (c <= 64 * kPer ? 64 : c <= 256 * kPer ? 256 : 512);
  NormChunks k{};
  // one workgroup a CU, at least two tokens a thread group, at most kBwdNT tokens
  int64_t chunks = (256 + b - 1) / b;
  if (chunks > (n + 2 * g - 1) / (2 * g)) chunks = (n + 2 * g - 1) / (2 * g);
  if (chunks < (n + kBwdNT - 1) / kBwdNT) chunks = (n + kBwdNT - 1) / kBwdNT;
  k.chunk = (n + chunks - 1) / chunks;
  k.chunks = (n + k.chunk - 1) / k.chunk;
  k.slots = !doc ? 1 : groups + 1 < k.chunk ? groups + 1 : k.chunk;
  k.cp = (c + 3) / 4 * 4;
  return k;
}

hipError_t launch_norm_fwd(int op, int f16, const NormArgs& a, hipStream_t st) {
  return f16 ? pick_op<false, _Float16>(op, a, st) : pick_op<false, __bf16>(op, a, st);
}

hipError_t launch_norm_mx(int op, int f16, const NormArgs& args, uint8_t* codes, uint8_t* scales, hipStream_t st) {
  NormArgs a = args;
  a.inv_c = 1.0 / (double)a.c;
  if (op == kNormModulate)
    return f16 ? mx_width<_Float16, kNormModulate>(a, codes, scales, st)
               : mx_width<__bf16, kNormModulate>(a, codes, scales, st);
  return f16 ? mx_width<_Float16, kNormGateModulate>(a, codes, scales, st)
             : mx_width<__bf16, kNormGateModulate>(a, codes, scales, st);
}

hipError_t launch_norm_bwd(int op, int f16, const NormArgs& a, hipStream_t st) {
  hipError_t e = f16 ? pick_op<true, _Float16>(op, a, st) : pick_op<true, __bf16>(op, a, st);
  if (e != hipSuccess || !a.part) return e;
  const int sets = op == kNormGateModulate ? 2 : 1;
  // workgroups a conditioning row: one for each 64 channels while that fills the card about
  // twice, fewer (which look for the row's partials less often) with more rows
  const int64_t blocks = (a.c + 63) / 64, rows = (int64_t)sets * a.b * a.groups;
  const int64_t most = std::max<int64_t>(1, 2048 / rows), cond_blocks = std::min(blocks, most);
  const uint32_t grid = (uint32_t)(sets * blocks + rows * cond_blocks);
  auto run = [&](auto kernel) {
    kernel<<<grid, kParamNT, 0, st>>>(a, sets, op == kNormModulate, (int)cond_blocks);
  };
  const bool whole = a.c % 4 == 0;
  if (f16) whole ? run(norm_param_kernel<_Float16, true>) : run(norm_param_kernel<_Float16, false>);
  else whole ? run(norm_param_kernel<__bf16, true>) : run(norm_param_kernel<__bf16, false>);
  return hipGetLastError();
}

}  // namespace sage
