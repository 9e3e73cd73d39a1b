// Linear layers of a transformer block for gfx950: out = act(x W^T + b) + r, and its
// gradients, bf16 or fp16 with fp32 accumulation.
//
// One product C[m][n] = sum_k A[m][k] B[n][k] in three operand layouts:
//   forward  A = x  [M][K],  B = W [N][K]          (both with the contraction contiguous)
//   dx       A = dz [M][N'], B = W as [N'][K]      (B: the output's columns contiguous)
//   dW       A = dz as [M][N'], B = x as [M][K]    (both: the contraction strided)
// and four kernels: tiles through LDS (gemm_kernel) and the sum of their pieces (join_kernel),
// few rows on one side (skinny_kernel), a contraction of one stage (thin_kernel).  Beside the
// products: copies of operands whose rows take no 16-byte accesses (pack_kernel), and the
// gradient through the activation with the bias's (dact_kernel, dbias_kernel).
#include <type_traits>

#include "sage_common.h"
#include "sage_launch.h"

namespace sage {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

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

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// ---------------------------------------------------------------- activations

constexpr float kGeluA = 0.7978845608028654f;  // sqrt(2/pi)

// 1 / (1 + exp(-z)), the quotient by v_rcp_f32 (within one step of fp32, as the exponential
// is: far below the 16-bit results' rounding); exp(-z) may overflow to infinity, which gives 0.
__device__ __forceinline__ float sigmoidf(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

__device__ __forceinline__ float act_fwd(int act, float z) {
  if (act == kActSilu || act == kActSwiglu) return z * sigmoidf(z);
  if (act == kActGelu)  // 0.5 z (1 + tanh(u)) = z sigmoid(2u), u = a (z + 0.044715 z^3)
    return z * sigmoidf(2.0f * kGeluA * (z + 0.044715f * z * z * z));
  return z;
}

__device__ __forceinline__ float act_grad(int act, float z) {
  if (act == kActSilu || act == kActSwiglu) {
    const float s = sigmoidf(z);
    return s + z * s * (1.0f - s);
  }
  if (act == kActGelu) {  // with s = sigmoid(2u): s + z s (1 - s) 2 u'
    const float s = sigmoidf(2.0f * kGeluA * (z + 0.044715f * z * z * z));
    // past |z| = 5e19 u' leaves fp32, where s (1 - s) is long 0: their product stays 0
    const float up = fminf(2.0f * kGeluA * (1.0f + 3.0f * 0.044715f * z * z), 3e38f);
    return s + z * s * (1.0f - s) * up;
  }
  return 1.0f;
}

// ---------------------------------------------------------------- epilogues

__device__ __forceinline__ float param_at(const void* p, bool f32, bool f16, int64_t i) {
  if (f32) return static_cast<const float*>(p)[i];
  return f16 ? (float)static_cast<const _Float16*>(p)[i] : (float)static_cast<const __bf16*>(p)[i];
}

// Columns 8 h .. + 7 of half p (16 columns) of a 32 x 32 accumulator of the transposed
// product, in which lane (h, r) holds row r, columns 8 J + 4 h + i: swapping J = 2 p + 1 of the
// lower lanes with J = 2 p of the upper gives each lane eight consecutive columns.
__device__ __forceinline__ void eight_of(const f32x16& c, int p, float (&z)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(c[8 * p + i]), __float_as_uint(c[8 * p + 4 + i]),
                                                    false, false);
    z[i] = __uint_as_float(s[0]);
    z[4 + i] = __uint_as_float(s[1]);
  }
}

__device__ __forceinline__ u32x4 load_16(__amdgpu_buffer_rsrc_t rs, int off) {
  return __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0);
}
__device__ __forceinline__ void store_16(u32x4 v, __amdgpu_buffer_rsrc_t rs, int off) {
  __builtin_amdgcn_raw_buffer_store_b128(v, rs, off, 0, 0);
}

__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }

// The two halves' packed columns of a 32 x 32 block (lane (h, r): row r, columns 16 p + 8 h of
// half p) to rows: x: row lane % 16, y: row 16 + lane % 16, both with columns 16 g + 8 h (g:
// lane bit 4), so that a store's four lanes of a row write 64 bytes together.  Its own inverse.
__device__ __forceinline__ void halves_to_rows(u32x4& x, u32x4& y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto s = __builtin_amdgcn_permlane16_swap(x[i], y[i], false, false);
    x[i] = s[0];
    y[i] = s[1];
  }
}

// The epilogue of a wave's MI x NI blocks from row m0 and column n0 on: z = acc + bias, kept
// when the backward wants it, out = act(z) + residual, rounded once.  Every access is 16 bytes
// through a buffer resource over the rows that exist, straight from the accumulators with no
// pass through LDS.  What a call does not have (bias, residual, z) has a resource of no
// bytes, so there is no branch.  PLAIN: out alone.
template <typename T, int ACT, bool PLAIN, int MI, int NI>
__device__ __forceinline__ void finish_wave(const GemmArgs& a, int lane, int64_t m0, int n0, f32x16 (&c)[MI][NI]) {
  using V = typename Vec8<T>::type;
  constexpr bool kGlu = ACT == kActSwiglu;
  constexpr int kStep = kGlu ? 2 : 1;
  const int64_t left = a.m - m0;
  if (left <= 0) return;
  const int rows = left < 32 * MI ? (int)left : 32 * MI, h = lane >> 5, row = lane & 15;
  const int wide = kGlu ? 2 * a.n : a.n;
  const __amdgpu_buffer_rsrc_t out = raw_rsrc(static_cast<T*>(a.out) + m0 * a.n, (uint32_t)rows * a.n * 2);
  const __amdgpu_buffer_rsrc_t res = raw_rsrc(static_cast<const T*>(a.res) + m0 * a.ldr,
                                              a.res ? (uint32_t)(((rows - 1) * a.ldr + a.n) * 2) : 0u);
  const __amdgpu_buffer_rsrc_t zs = raw_rsrc(a.z + m0 * wide, a.z ? (uint32_t)rows * wide * 4 : 0u);
  const __amdgpu_buffer_rsrc_t b16 = raw_rsrc(a.bias, a.bias && !a.bias_f32 ? (uint32_t)wide * 2 : 0u);
  const __amdgpu_buffer_rsrc_t b32 = raw_rsrc(a.bias, a.bias && a.bias_f32 ? (uint32_t)wide * 4 : 0u);
  auto bias_at = [&](int n, float (&b)[8]) {  // one of the two reads zeros
    const V v = __builtin_bit_cast(V, load_16(b16, n * 2));
    const f32x4 lo = __builtin_bit_cast(f32x4, load_16(b32, n * 4)), hi = __builtin_bit_cast(f32x4, load_16(b32, n * 4 + 16));
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = (float)v[e] + (e < 4 ? lo[e & 3] : hi[e & 3]);
  };
  // the columns of block column j that this lane loads and stores, and whether they exist
  // (else an offset past any size)
  auto column = [&](int j) { return n0 + (32 / kStep) * j + 16 * ((lane >> 4) & 1) + 8 * h; };
  auto beyond = [&](int n) { return n < a.n ? 0 : (int)0x80000000; };
  // a block column's residual is read one block column ahead; the scheduling barriers keep
  // the rest of the loads where they are, or registers run out
  u32x4 ahead[2][MI][2];
  auto residual = [&](int j, int to) {
    const int n = column(j), none = beyond(n);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q) ahead[to][i][q] = load_16(res, (int)((32 * i + 16 * q + row) * a.ldr + n) * 2 | none);
  };
  auto store = [&](int i, int n, int none, V v0, V v1) {
    u32x4 x = __builtin_bit_cast(u32x4, v0), y = __builtin_bit_cast(u32x4, v1);
    halves_to_rows(x, y);
    store_16(x, out, ((32 * i + row) * a.n + n) * 2 | none);
    store_16(y, out, ((32 * i + 16 + row) * a.n + n) * 2 | none);
  };
  auto keep = [&](int i, int n, int none, const float (&z)[8]) {
    const int at = ((32 * i + (lane & 31)) * wide + n) * 4 | none;
    store_16(__builtin_bit_cast(u32x4, f32x4{z[0], z[1], z[2], z[3]}), zs, at);
    store_16(__builtin_bit_cast(u32x4, f32x4{z[4], z[5], z[6], z[7]}), zs, at + 16);
  };
  if constexpr (!PLAIN) residual(0, 0);
#pragma unroll
  for (int j = 0; j < NI; j += kStep) {
    const int n = column(j), none = beyond(n);
    float b[2][8], b2[2][8];
    if constexpr (!PLAIN) {
      if (j + kStep < NI) residual(j + kStep, (j / kStep + 1) & 1);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        // beyond the last column a column that lies past any bias, in bytes too
        const int nb = n0 + (32 / kStep) * j + 16 * p + 8 * h, nob = nb < a.n ? 0 : 0x10000000;
        bias_at(nb | nob, b[p]);
        if constexpr (kGlu) bias_at((nb + a.n) | nob, b2[p]);
      }
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      V o[2];
      if constexpr (!PLAIN) halves_to_rows(ahead[j / kStep & 1][i][0], ahead[j / kStep & 1][i][1]);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float z[8], z2[8];
        eight_of(c[i][j], p, z);
        if constexpr (kGlu) eight_of(c[i][j + 1], p, z2);
        if constexpr (!PLAIN) {
          const V rv = __builtin_bit_cast(V, ahead[j / kStep & 1][i][p]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            z[e] += b[p][e];
            if constexpr (kGlu) z2[e] += b2[p][e];
          }
          if constexpr (ACT != kActNone) {
            const int nz = n0 + (32 / kStep) * j + 16 * p + 8 * h, noz = beyond(nz);
            keep(i, nz, noz, z);
            if constexpr (kGlu) keep(i, nz + a.n, noz, z2);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            z[e] = act_fwd(ACT, z[e]);
            if constexpr (kGlu) z[e] *= z2[e];
            z[e] += (float)rv[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) o[p][e] = (T)z[e];
      }
      store(i, n, none, o[0], o[1]);
    }
    keep_order();
  }
}

template <typename T, int MI, int NI>
__device__ __forceinline__ void finish(const GemmArgs& a, int lane, int64_t m0, int n0, f32x16 (&c)[MI][NI]) {
  if (a.act == kActSwiglu) finish_wave<T, kActSwiglu, false>(a, lane, m0, n0, c);
  else if (a.act == kActSilu) finish_wave<T, kActSilu, false>(a, lane, m0, n0, c);
  else if (a.act == kActGelu) finish_wave<T, kActGelu, false>(a, lane, m0, n0, c);
  else finish_wave<T, kActNone, false>(a, lane, m0, n0, c);
}

// The same for 32 R x 64 parts of a tile whose rows have any alignment: by way of LDS, so that
// a wave's lanes take consecutive elements of a row (of two rows for a swiglu, which has 32
// columns here), kAnyRows rows in flight.  `lds`: 32 R x kAnyPitch floats of this wave.
constexpr int kAnyPitch = 65, kAnyRows = 16;

__device__ __forceinline__ uint16_t load_2(__amdgpu_buffer_rsrc_t rs, int off) {
  return __builtin_amdgcn_raw_buffer_load_b16(rs, off, 0, 0);
}
__device__ __forceinline__ uint32_t load_4(__amdgpu_buffer_rsrc_t rs, int off) {
  return __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
}
__device__ __forceinline__ void store_2(uint16_t v, __amdgpu_buffer_rsrc_t rs, int off) {
  __builtin_amdgcn_raw_buffer_store_b16(v, rs, off, 0, 0);
}
__device__ __forceinline__ void store_4(uint32_t v, __amdgpu_buffer_rsrc_t rs, int off) {
  __builtin_amdgcn_raw_buffer_store_b32(v, rs, off, 0, 0);
}

// Puts a pair of accumulators at row block i of the wave's LDS.
__device__ __forceinline__ void stage_any(float* lds, int lane, int i, const f32x16& c0, const f32x16& c1) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int col = 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
    lds[(32 * i + (lane & 31)) * kAnyPitch + col] = c0[e];
    lds[(32 * i + (lane & 31)) * kAnyPitch + 32 + col] = c1[e];
  }
}

template <typename T, int ACT, int R>
__device__ __forceinline__ void finish_any(const GemmArgs& a, const float* lds, int lane, int64_t m0, int n0) {
  constexpr bool kGlu = ACT == kActSwiglu;
  constexpr int kCols = kGlu ? 32 : 64, kPer = 64 / kCols;  // rows a wave takes at a time
  const int64_t left = a.m - m0;
  if (left <= 0) return;
  const int rows = left < 32 * R ? (int)left : 32 * R, wide = kGlu ? 2 * a.n : a.n;
  const int col = lane % kCols, n = n0 + col, none = n < a.n ? 0 : (int)0x80000000;
  const __amdgpu_buffer_rsrc_t out = raw_rsrc(static_cast<T*>(a.out) + m0 * a.n, (uint32_t)rows * a.n * 2);
  const __amdgpu_buffer_rsrc_t res = raw_rsrc(static_cast<const T*>(a.res) + m0 * a.ldr,
                                              a.res ? (uint32_t)(((rows - 1) * a.ldr + a.n) * 2) : 0u);
  const __amdgpu_buffer_rsrc_t zs = raw_rsrc(a.z + m0 * wide, a.z ? (uint32_t)rows * wide * 4 : 0u);
  const bool f16 = std::is_same<T, _Float16>::value, bias = a.bias && !none;
  const float b = bias ? param_at(a.bias, a.bias_f32, f16, n) : 0.0f;
  const float b2 = kGlu && bias ? param_at(a.bias, a.bias_f32, f16, a.n + n) : 0.0f;
#pragma unroll 1
  for (int r0 = lane / kCols; r0 < 32 * R; r0 += kAnyRows * kPer) {
    float r[kAnyRows];
#pragma unroll
    for (int u = 0; u < kAnyRows; ++u)
      r[u] = (float)__builtin_bit_cast(T, load_2(res, (int)((r0 + u * kPer) * a.ldr + n) * 2 | none));
#pragma unroll
    for (int u = 0; u < kAnyRows; ++u) {
      const int row = r0 + u * kPer;
      const float z = lds[row * kAnyPitch + col] + b, z2 = kGlu ? lds[row * kAnyPitch + 32 + col] + b2 : 1.0f;
      if constexpr (ACT != kActNone) {
        store_4(__float_as_uint(z), zs, (row * wide + n) * 4 | none);
        if constexpr (kGlu) store_4(__float_as_uint(z2), zs, (row * wide + a.n + n) * 4 | none);
      }
      store_2(__builtin_bit_cast(uint16_t, (T)(act_fwd(ACT, z) * z2 + r[u])), out, (row * a.n + n) * 2 | none);
    }
  }
}

template <typename T, bool ACTS, int R>
__device__ __forceinline__ void finish_any_act(const GemmArgs& a, float* lds, int lane, int64_t m0, int n0) {
  // the wave's sums are written before they are read
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (ACTS && a.act == kActSwiglu) finish_any<T, kActSwiglu, R>(a, lds, lane, m0, n0);
  else if (ACTS && a.act == kActSilu) finish_any<T, kActSilu, R>(a, lds, lane, m0, n0);
  else if (ACTS && a.act == kActGelu) finish_any<T, kActGelu, R>(a, lds, lane, m0, n0);
  else finish_any<T, kActNone, R>(a, lds, lane, m0, n0);
}

// ---------------------------------------------------------------- tiles

constexpr int kBK = 64;  // contraction of one LDS stage

// A tile shape: WM x WN waves, each with MI x NI blocks of 32 x 32, `SIMD` waves a SIMD.
template <int WM_, int WN_, int MI_, int NI_, int SIMD_>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, MI = MI_, NI = NI_, SIMD = SIMD_;
  static constexpr int WAVES = WM * WN, NT = 64 * WAVES;
  static constexpr int BM = WM * MI * 32, BN = WN * NI * 32;
  static constexpr int A_BYTES = BM * kBK * 2, B_BYTES = BN * kBK * 2, B_AT = 3 * A_BYTES;
  static constexpr int LDS = 3 * A_BYTES + 2 * B_BYTES;
};

// One direct global -> LDS load of 64 chunks: lane l's 16 bytes land at lds + 16 l; an
// offset past the resource's end gives zeros.
__device__ __forceinline__ void dma_16(uint8_t* lds, __amdgpu_buffer_rsrc_t rs, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds, 16, off, 0, 0, 0);
}

// One operand's part of an LDS stage: ROWS rows (of the output's m or n) by kBK.
//
// KC (contraction contiguous in memory): 128-byte rows, row r's 16-byte chunk c at
// c ^ ((r >> 1) & 7): the 16 rows that a fragment read touches at a time lie on 16
// different 16-byte columns of the 256 bytes of banks.
// Not KC: the kBK contraction rows of ROWS * 2 bytes, 64-byte runs u at u ^ (k & 3), so
// that the 4 rows of a transposing read (ds_read_b64_tr_b16: 16 lanes read 4 rows by 16
// columns, each lane gets one column's 4 rows) lie on different banks.
// Every load is a direct global -> LDS load of 1 KiB by one wave, whose lanes choose
// their source accordingly.
template <int ROWS, bool KC, int WAVES>
struct Operand {
  static constexpr int LOADS = ROWS * kBK * 2 / 1024 / WAVES;  // of one wave
  const uint8_t* base;
  int64_t ld2;  // bytes between rows in memory
  int valid;    // rows (KC) or columns (not KC) of this tile that exist
  int off[LOADS];
  int kpos;     // KC: first contraction index of the lane's chunk (the same in every load)

  // glu: tile row j is row (j / 64) * 32 + j % 32 of half (j / 32) % 2, the halves `half`
  // rows apart.
  __device__ __forceinline__ void init(const void* p, int64_t ld, int64_t row0, int64_t rows, int wave, int lane,
                                       bool glu, int64_t half) {
    ld2 = ld * 2;
    base = static_cast<const uint8_t*>(p) + row0 * (KC ? ld2 : 2);
    const int64_t left = rows - row0;
    valid = (int)(left < ROWS ? left : ROWS);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int q = i * WAVES + wave;
      if constexpr (KC) {
        int r = q * 8 + (lane >> 3);
        const int c = (lane & 7) ^ ((r >> 1) & 7);
        kpos = c * 8;
        const bool up = glu && ((r >> 5) & 1);
        if (glu) r = (r >> 6) * 32 + (r & 31);
        off[i] = r < valid ? (int)(r * ld2 + (up ? half * ld2 : 0)) + c * 16 : (int)0x80000000;
      } else {
        const int at = q * 1024 + lane * 16, k = at / (ROWS * 2), in = at % (ROWS * 2);
        off[i] = (int)(k * ld2) + ((((in >> 6) ^ (k & 3)) << 6) | (in & 63));
      }
    }
  }
  // Issues loads FIRST .. FIRST + COUNT - 1 of contraction k0 .. k0 + kBK - 1 of K into `lds`.
  template <int FIRST, int COUNT>
  __device__ __forceinline__ void issue(uint8_t* lds, int64_t k0, int64_t K, int wave) const {
    const int left = (int)(K - k0 < kBK ? K - k0 : kBK);  // 0 or less behind the end
    // KC: rows past the last have an offset past any size, and so get chunks past K.  Not
    // KC: columns past the last read what follows in memory (they reach outputs that are not
    // stored alone), up to the end of the last row, in whole 4 bytes; rows past K read zeros.
    const __amdgpu_buffer_rsrc_t rs =
        KC ? raw_rsrc(base + k0 * 2, 0x7fffffff)
           : raw_rsrc(base + k0 * ld2, left > 0 ? (uint32_t)((left - 1) * ld2 + (valid + 1) / 2 * 4) : 0u);
#pragma unroll
    for (int i = FIRST; i < FIRST + COUNT; ++i)
      dma_16(lds + (i * WAVES + wave) * 1024, rs, !KC || kpos < left ? off[i] : (int)0x80000000);
  }
};

// Byte offset in an operand's stage of the fragment of 32 rows from `row` on: lane (h, r)
// gets row r, contraction 16 s + 8 h .. + 7.
template <int ROWS, bool KC>
struct FragAddr {
  int at[KC ? kBK / 16 : 1];
  __device__ __forceinline__ void init(int row, int lane) {
    const int h = lane >> 5, r = row + (lane & 31);
    if constexpr (KC) {
#pragma unroll
      for (int s = 0; s < kBK / 16; ++s) at[s] = r * 128 + (((2 * s + h) ^ ((r >> 1) & 7)) << 4);
    } else {
      const int l = lane & 15, g = (lane >> 4) & 1, k = 8 * h + (l >> 2);
      const int col = (row + 16 * g + 4 * (l & 3)) * 2;
      at[0] = k * (ROWS * 2) + ((((col >> 6) ^ (k & 3)) << 6) | (col & 63));
    }
  }
};

// A transposing read of 8 bytes a lane.  `p` is restrict so that the read carries alias
// information: without any, the compiler waits for the direct loads in flight before it.
__device__ __forceinline__ s16x4 read_tr(const uint8_t* __restrict__ p) {
  typedef __attribute__((address_space(3))) s16x4* LdsPtr;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(p));
}

template <typename T, int ROWS, bool KC>
__device__ __forceinline__ typename Vec8<T>::type frag(const uint8_t* __restrict__ stage, const FragAddr<ROWS, KC>& f,
                                                       int s) {
  if constexpr (KC) {
    return *reinterpret_cast<const typename Vec8<T>::type*>(stage + f.at[s]);
  } else {
    const uint8_t* p = stage + f.at[0] + s * 16 * (ROWS * 2);
    const s16x4 a = read_tr(p), b = read_tr(p + 4 * (ROWS * 2));
    return __builtin_bit_cast(typename Vec8<T>::type, s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
  }
}

// Tile t of the schedule: groups of 4 tile rows, column by column inside, so that the 32
// tiles an XCD runs together share 4 row panels and 8 column panels.
__device__ __forceinline__ void tile_at(const GemmArgs& a, int t, int& tm, int& tn) {
  constexpr int G = 4;
  const int g = t / (G * a.tn), in = t - g * G * a.tn;
  const int rows = min(G, a.tm - g * G);
  tn = in / rows;
  tm = g * G + in - tn * rows;
}

// Work unit of workgroup `b`: the hardware hands workgroup b to XCD b % 8; every XCD takes
// a contiguous range of the whole tiles, then of the cut ones' pieces.
__device__ __forceinline__ int xcd_share(int b, int total) {
  const int x = b % 8, local = b / 8, per = total / 8, rem = total % 8;
  return x * per + min(x, rem) + local;
}

// Waits for every LDS read and for all but the last LEFT direct loads.
template <int LEFT>
__device__ __forceinline__ void wait_loads();
template <>
__device__ __forceinline__ void wait_loads<0>() { __builtin_amdgcn_s_waitcnt(0x0070); }
template <>
__device__ __forceinline__ void wait_loads<4>() { __builtin_amdgcn_s_waitcnt(0x0074); }
template <>
__device__ __forceinline__ void wait_loads<6>() { __builtin_amdgcn_s_waitcnt(0x0076); }
template <>
__device__ __forceinline__ void wait_loads<8>() { __builtin_amdgcn_s_waitcnt(0x0078); }
template <>
__device__ __forceinline__ void wait_loads<12>() { __builtin_amdgcn_s_waitcnt(0x007c); }

// No memory access moves across it.
__device__ __forceinline__ void hold_memory() { asm volatile("" ::: "memory"); }

template <typename V>
__device__ __forceinline__ V operand_at(const uint8_t* __restrict__ p) {
  return *reinterpret_cast<const V*>(p);
}

// A workgroup barrier that waits for no load (__syncthreads waits for all of them); no
// memory access moves across it.
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The scheduler's next instruction of a kind.
__device__ __forceinline__ void order_mfma() { __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); }
__device__ __forceinline__ void order_read() { __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); }

__device__ __forceinline__ void order_load() { __builtin_amdgcn_sched_group_barrier(0x020, 1, 0); }

// The product by tiles.  A wave of 128 x 128 reads 256 rows of fragments for 16 products of 32
// x 32: LDS gives 128 bytes a cycle to a CU, and four such waves need 64 of them where four
// of 64 x 64 need all 128.  The large tile therefore runs at one wave a SIMD with 256
// accumulators; the small one, two workgroups a CU, is for what has too few large tiles.
// Measured, bf16: 4416 x 11520 x 3840 with the bias 346 us = 1130 TFLOP/s, its dx 332 us =
// 1177, its dW 356 us = 1097 (transposing reads on both sides); the swiglu of 4416 x 20480 x
// 3840 570 us = 1220.  Two things bound it.  The clock, which falls with the data's power: the
// forward's 549 k cycles take 343 us at 1.6 GHz, those of zeros 267 us at 2.1.  And the 27 to 34 %
// of the cycles in which the matrix cores are idle (busy: 70 %, dx 73, dW 66, swiglu 68): the
// last, partly filled round, each round's start and epilogue, and the barriers; no LDS bank
// conflict, 4 to 5 % of the waves' time waits for LDS, memory moves 1.4 to 1.5 TB/s.  A stage
// takes the same time with the loads in bursts, with LDS slots a wave and with the next tile's
// first stages loaded under the epilogue.
template <typename T, bool AK, bool BKC, typename TL>
__global__ __launch_bounds__(TL::NT, TL::SIMD) void gemm_kernel(GemmArgs a) {
  __shared__ __align__(1024) uint8_t lds[TL::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const bool glu = BKC && a.act == kActSwiglu;
  const int bid = blockIdx.x;
  int t, piece = 0;
  int kt0 = 0, kt1 = a.kt;
  const bool cut = bid >= a.whole;
  if (!cut) {
    t = xcd_share(bid, a.whole);
  } else {
    const int u = xcd_share(bid - a.whole, ((int)gridDim.x - a.whole));
    t = a.whole + u / a.parts;
    piece = u - (t - a.whole) * a.parts;
    kt0 = (int)((int64_t)a.kt * piece / a.parts);
    kt1 = (int)((int64_t)a.kt * (piece + 1) / a.parts);
  }
  int tm, tn;
  tile_at(a, t, tm, tn);
  const int64_t m0 = (int64_t)tm * TL::BM;
  const int n0 = tn * (glu ? TL::BN / 2 : TL::BN);

  Operand<TL::BM, AK, TL::WAVES> A;
  Operand<TL::BN, BKC, TL::WAVES> B;
  A.init(a.a, a.lda, m0, a.m, wave, lane, false, 0);
  B.init(a.b, a.ldb, n0, a.n, wave, lane, glu, a.n);
  const int wm = wave / TL::WN, wn = wave % TL::WN;
  FragAddr<TL::BM, AK> fa[TL::MI];
  FragAddr<TL::BN, BKC> fb[TL::NI];
#pragma unroll
  for (int i = 0; i < TL::MI; ++i) fa[i].init((wm * TL::MI + i) * 32, lane);
#pragma unroll
  for (int i = 0; i < TL::NI; ++i) fb[i].init((wn * TL::NI + i) * 32, lane);

  // A stage's four steps of 16, the next step's fragments read under this one's products.
  // Before a stage's last step the next stage has arrived and every wave has read this
  // one's last fragments: behind that barrier later loads go into its place, and the last
  // products run beside the next stage's first reads.  LDS holds three stages of A and two
  // of B.  A wave's eight loads of a stage are spread over the four steps (B's, which the
  // next barrier waits for, first): issued together behind the barrier they hold the
  // waves up, 64 loads at 16 cycles of the address unit each.  Loads past the last stage,
  // and the reads of it in the last round, give nothing that is used.
  using V = typename Vec8<T>::type;
  f32x16 acc[TL::MI][TL::NI] = {};
  V va[2][TL::MI], vb[2][TL::NI];
  // nothing is read past the piece's last stage
  const int64_t end = (int64_t)kt1 * kBK, ka = min(AK ? a.k : a.kv, end), kb = min(BKC ? a.k : a.kv, end);
  auto read = [&](const uint8_t* sa, const uint8_t* sb, int s, int to) {
#pragma unroll
    for (int i = 0; i < TL::NI; ++i) vb[to][i] = frag<T>(sb, fb[i], s);
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) va[to][i] = frag<T>(sa, fa[i], s);
  };
  auto products = [&](int from) {
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
      for (int j = 0; j < TL::NI; ++j) acc[i][j] = mfma32(vb[from][j], va[from][i], acc[i][j]);
  };
  constexpr int H = decltype(A)::LOADS / 2;
  static_assert(H * 2 == decltype(B)::LOADS, "as many loads of A as of B");
  // the order of one step: a product, then reads of the next step and loads, and so on
  auto order = [&]() {
    constexpr int M = TL::MI * TL::NI, R = TL::MI * (AK ? 1 : 2) + TL::NI * (BKC ? 1 : 2);
#pragma unroll
    for (int i = 0; i < M; ++i) {
      order_mfma();
      if constexpr (R > M) order_read();
      order_read();
      if (i % (M / H) == M / H / 2) order_load();
    }
  };
  uint8_t* const lb = lds + TL::B_AT;
  A.template issue<0, 2 * H>(lds, (int64_t)kt0 * kBK, ka, wave);
  B.template issue<0, 2 * H>(lb, (int64_t)kt0 * kBK, kb, wave);
  A.template issue<0, 2 * H>(lds + TL::A_BYTES, (int64_t)(kt0 + 1) * kBK, ka, wave);
  B.template issue<0, H>(lb + TL::B_BYTES, (int64_t)(kt0 + 1) * kBK, kb, wave);
  wait_loads<3 * H>();
  barrier();
  read(lds, lb, 0, 0);
  int a0 = 0, b0 = 0;             // the present stage's place
  int a2 = 2 * TL::A_BYTES;       // the place of the stage after next
  for (int kt = kt0; kt < kt1; ++kt) {
    uint8_t* const sa = lds + a0;
    uint8_t* const sb = lb + b0;
    read(sa, sb, 1, 1);
    products(0);
    B.template issue<H, H>(lb + (b0 ^ TL::B_BYTES), (int64_t)(kt + 1) * kBK, kb, wave);
    order();
    read(sa, sb, 2, 0);
    products(1);
    A.template issue<0, H>(lds + a2, (int64_t)(kt + 2) * kBK, ka, wave);
    order();
    read(sa, sb, 3, 1);
    products(0);
    A.template issue<H, H>(lds + a2, (int64_t)(kt + 2) * kBK, ka, wave);
    order();
    wait_loads<2 * H>();
    barrier();
    a2 = a0;
    a0 = a0 == 2 * TL::A_BYTES ? 0 : a0 + TL::A_BYTES;
    b0 ^= TL::B_BYTES;
    read(lds + a0, lb + b0, 0, 0);
    products(1);
    B.template issue<0, H>(sb, (int64_t)(kt + 2) * kBK, kb, wave);
    order();
  }
  wait_vmem();  // the loads in flight write this workgroup's LDS
  if (cut) {
    // the piece's sums, in the order the lanes hold them
    float* dst = a.part + ((int64_t)(t - a.whole) * a.parts + piece) * (TL::BM * TL::BN) +
                 wave * (TL::MI * TL::NI * 1024);
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
      for (int j = 0; j < TL::NI; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(dst + ((i * TL::NI + j) * 4 + q) * 256 + lane * 4) =
              f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    return;
  }
  const int64_t mw = m0 + wm * TL::MI * 32;
  const int nw = n0 + wn * TL::NI * (glu ? 16 : 32);
  if constexpr (TL::SIMD > 1) {
    if (!a.vec) {
      barrier();  // every wave has read its last fragments: the stages' LDS is free
      static_assert(TL::NI == 2 && TL::WAVES * TL::MI * 32 * kAnyPitch * 4 <= TL::LDS, "the sums fit");
      float* const mine = reinterpret_cast<float*>(lds) + wave * TL::MI * 32 * kAnyPitch;
#pragma unroll
      for (int i = 0; i < TL::MI; ++i) stage_any(mine, lane, i, acc[i][0], acc[i][1]);
      finish_any_act<T, AK && BKC, TL::MI>(a, mine, lane, mw, nw);
      return;
    }
  }
  if constexpr (AK && BKC)
    finish<T>(a, lane, mw, nw, acc);
  else
    finish_wave<T, kActNone, true>(a, lane, mw, nw, acc);
}

// The products of at most one stage's contraction (an adapter's second product): bound by
// the output and the residual, so one stage of LDS, several workgroups a CU, and no steps
// past the last 16 that exist.  4416 x 3840 x 16 onto a residual: 68 MB in 18.5 us.
template <typename T, typename TL>
__global__ __launch_bounds__(TL::NT, 3) void thin_kernel(GemmArgs a) {
  __shared__ __align__(1024) uint8_t lds[TL::A_BYTES + TL::B_BYTES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const bool glu = a.act == kActSwiglu;
  int tm, tn;
  tile_at(a, xcd_share(blockIdx.x, a.whole), tm, tn);
  const int64_t m0 = (int64_t)tm * TL::BM;
  const int n0 = tn * (glu ? TL::BN / 2 : TL::BN);
  Operand<TL::BM, true, TL::WAVES> A;
  Operand<TL::BN, true, TL::WAVES> B;
  A.init(a.a, a.lda, m0, a.m, wave, lane, false, 0);
  B.init(a.b, a.ldb, n0, a.n, wave, lane, glu, a.n);
  A.template issue<0, decltype(A)::LOADS>(lds, 0, a.k, wave);
  B.template issue<0, decltype(B)::LOADS>(lds + TL::A_BYTES, 0, a.k, wave);
  const int wm = wave / TL::WN, wn = wave % TL::WN;
  FragAddr<TL::BM, true> fa[TL::MI];
  FragAddr<TL::BN, true> fb[TL::NI];
#pragma unroll
  for (int i = 0; i < TL::MI; ++i) fa[i].init((wm * TL::MI + i) * 32, lane);
#pragma unroll
  for (int i = 0; i < TL::NI; ++i) fb[i].init((wn * TL::NI + i) * 32, lane);
  f32x16 acc[TL::MI][TL::NI] = {};
  wait_vmem();
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kBK / 16; ++s) {
    if (s * 16 >= a.k) break;
    typename Vec8<T>::type va[TL::MI], vb[TL::NI];
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) va[i] = frag<T>(lds, fa[i], s);
#pragma unroll
    for (int i = 0; i < TL::NI; ++i) vb[i] = frag<T>(lds + TL::A_BYTES, fb[i], s);
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
      for (int j = 0; j < TL::NI; ++j) acc[i][j] = mfma32(vb[j], va[i], acc[i][j]);
  }
  finish<T>(a, lane, m0 + wm * TL::MI * 32, n0 + wn * TL::NI * (glu ? 16 : 32), acc);
}

// Adds the pieces of the cut tiles in order and finishes them: a wave takes one 32 x 64
// block of a tile.  Large tiles whose rows take no 16-byte accesses all come through here.
// Bound by the sums' way back: 75 tiles of 256 x 256 in three pieces, 79 MB with the residual
// and the output, in 16 us = 4.9 TB/s.
template <typename T, typename TL>
__global__ __launch_bounds__(256) void join_kernel(GemmArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  constexpr int PAIRS = TL::NI / 2, BLOCKS = TL::WAVES * TL::MI * PAIRS;
  const int u = blockIdx.x * 4 + wave, t = u / BLOCKS, blk = u - t * BLOCKS;
  const float* src = a.part + (int64_t)t * a.parts * (TL::BM * TL::BN) + blk * 2048 + lane * 4;
  f32x16 c[1][2] = {};
#pragma unroll 2
  for (int p = 0; p < a.parts; ++p) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(src + (j * 4 + q) * 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) c[0][j][4 * q + e] += v[e];
      }
    src += TL::BM * TL::BN;
  }
  int tm, tn;
  tile_at(a, a.whole + t, tm, tn);
  const int w = blk / (TL::MI * PAIRS), wm = w / TL::WN, wn = w % TL::WN;
  const int i = blk / PAIRS % TL::MI, j = blk % PAIRS * 2;
  const bool glu = a.act == kActSwiglu;
  const int64_t m0 = (int64_t)tm * TL::BM + (wm * TL::MI + i) * 32;
  const int n0 = tn * (glu ? TL::BN / 2 : TL::BN) + (wn * TL::NI + j) * (glu ? 16 : 32);
  __shared__ float any[4][32 * kAnyPitch];
  if (a.vec) {
    finish<T>(a, lane, m0, n0, c);
  } else {
    stage_any(any[wave], lane, 0, c[0][0], c[0][1]);
    finish_any_act<T, true, 1>(a, any[wave], lane, m0, n0);
  }
}

// ---------------------------------------------------------------- few rows

constexpr int kSkinnyWaves = 4;

// out for at most 16 * MT rows on the short side: a workgroup takes 16 rows of the long
// side and reads them once; its waves share the contraction, chunks of 64 in turn, and their
// sums are added in order.  swap: the long side is x (m), not W (n).
//
// A wave has its own ring of D stages in LDS (a chunk of its H x 16 long rows and of the
// short ones) and waits for nobody.  Direct global -> LDS loads, eight rows of 128 bytes
// each: loaded straight to the matrix operand's registers, neighbouring lanes lie on
// different rows, and the address unit takes 64 cycles a load (16 rows by 3840 x 11520 in 22.6
// us, 32 in 32.8).  Measured so: 14.8 and 17.0 us, 88 MB at the rate of memory and the cache
// above it; 2 x 256 by 15360 x 256 4.3 us, a launch and two trips to memory.
template <typename T, int MT, bool GLU>
__global__ __launch_bounds__(64 * kSkinnyWaves, 2) void skinny_kernel(GemmArgs a, int swap) {
  using V = typename Vec8<T>::type;
  constexpr int H = GLU ? 2 : 1, TILES = H + MT, STAGE = TILES * 2048;
  constexpr int D = TILES == 2 ? 4 : TILES == 3 ? 3 : 2;  // two workgroups a CU
  __shared__ __align__(1024) uint8_t lds[kSkinnyWaves * D * STAGE];
  static_assert(sizeof(lds) <= 80 * 1024 && H * MT * 1024 <= D * STAGE, "two workgroups a CU, and the sums fit");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  uint8_t* const mine = lds + wave * D * STAGE;
  const uint8_t* lp = static_cast<const uint8_t*>(swap ? a.a : a.b);
  const int64_t lld = (swap ? a.lda : a.ldb) * 2, sld = (swap ? a.ldb : a.lda) * 2;
  const int64_t llen = swap ? a.m : a.n, slen = swap ? a.n : a.m;
  const int64_t l0 = (int64_t)blockIdx.x * 16;
  const __amdgpu_buffer_rsrc_t srs = raw_rsrc(swap ? a.b : a.a, 0x7fffffff);
  __amdgpu_buffer_rsrc_t lrs[H];
#pragma unroll
  for (int h = 0; h < H; ++h) lrs[h] = raw_rsrc(lp + (l0 + h * llen) * lld, 0x7fffffff);
  // of a load's eight rows, lane l takes row l / 8 and, as in a stage of the tiles, the
  // chunk of 16 bytes that lies at l % 8; rows past the last read the last one again (what
  // they give is not stored), the contraction past its end zeros
  int kpos[2], loff[2], soff[MT][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = 8 * i + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
    kpos[i] = c * 8;
    loff[i] = (int)((min(l0 + row, llen - 1) - l0) * lld) + c * 16;
#pragma unroll
    for (int j = 0; j < MT; ++j) soff[j][i] = (int)(min((int64_t)(16 * j + row), slen - 1) * sld) + c * 16;
  }
  auto issue = [&](uint8_t* stage, int chunk) {
    const int k0 = chunk * 64, left = (int)a.k - k0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int none = kpos[i] < left ? 0 : (int)0x80000000;
#pragma unroll
      for (int h = 0; h < H; ++h) dma_16(stage + h * 2048 + i * 1024, lrs[h], (loff[i] + k0 * 2) | none);
#pragma unroll
      for (int j = 0; j < MT; ++j) dma_16(stage + (H + j) * 2048 + i * 1024, srs, (soff[j][i] + k0 * 2) | none);
    }
  };
  const int q = lane >> 4, r = lane & 15;
  int at[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) at[s] = r * 128 + (((4 * s + q) ^ ((r >> 1) & 7)) << 4);
  f32x4 acc[H][MT] = {};
  const int chunks = (int)((a.k + 63) / 64);
  // wave i finishes short rows 16 i ..: lane (q, r) long rows 4 q .. + 3 of short row r.  Bias and
  // residual are asked for first (zeros where there are none) and waited for last.
  const int64_t mr = 16 * wave + r;
  uint32_t bias[H][4];
  uint16_t res[4];
  if (wave < MT) {
    const __amdgpu_buffer_rsrc_t brs = raw_rsrc(a.bias, a.bias ? (uint32_t)(a.n * H) * (a.bias_f32 ? 4 : 2) : 0u);
    const __amdgpu_buffer_rsrc_t rrs =
        raw_rsrc(static_cast<const T*>(a.res) + (swap ? l0 * a.ldr : 0), a.res ? 0x7fffffffu : 0u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int l = 4 * q + e, n = swap ? (int)mr : (int)l0 + l;
      const int none = l0 + l < llen && mr < slen ? 0 : (int)0x80000000;
#pragma unroll
      for (int h = 0; h < H; ++h)
        bias[h][e] = a.bias_f32 ? load_4(brs, (n + h * a.n) * 4 | none) : load_2(brs, (n + h * a.n) * 2 | none);
      res[e] = load_2(rrs, (int)((swap ? l * a.ldr + mr : mr * a.ldr + n) * 2) | none);
    }
    keep_order();
  }
#pragma unroll
  for (int d = 0; d < D - 1; ++d)
    if (wave + d * kSkinnyWaves < chunks) issue(mine + d * STAGE, wave + d * kSkinnyWaves);
  int now = 0, free = (D - 1) * STAGE;
#pragma unroll 1
  for (int c = wave; c < chunks; c += kSkinnyWaves) {
    // this stage has arrived, and the last one's reads are done: its place takes the next loads
    if (c + (D - 1) * kSkinnyWaves < chunks) {
      wait_loads<2 * TILES * (D - 2)>();
      hold_memory();
      issue(mine + free, c + (D - 1) * kSkinnyWaves);
    } else {
      wait_loads<0>();
      hold_memory();
    }
    const uint8_t* stage = mine + now;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      V l[H], x[MT];
#pragma unroll
      for (int h = 0; h < H; ++h) l[h] = operand_at<V>(stage + h * 2048 + at[s]);
#pragma unroll
      for (int j = 0; j < MT; ++j) x[j] = operand_at<V>(stage + (H + j) * 2048 + at[s]);
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[h][j] = mfma16(l[h], x[j], acc[h][j]);
    }
    free = now;
    now = now == (D - 1) * STAGE ? 0 : now + STAGE;
  }
  wait_vmem();  // the loads in flight write this wave's LDS
  hold_memory();
  // the waves' sums, in the place of the stages
  f32x4* const part = reinterpret_cast<f32x4*>(mine);
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < MT; ++i) part[(h * MT + i) * 64 + lane] = acc[h][i];
  __syncthreads();
  if (wave >= MT) return;
  f32x4 z = {}, z2 = {};
#pragma unroll
  for (int w = 0; w < kSkinnyWaves; ++w) {
    const f32x4* const p = reinterpret_cast<const f32x4*>(lds + w * D * STAGE) + threadIdx.x;
    z += p[0];
    if (GLU) z2 += p[(H - 1) * MT * 64];
  }
  if (mr >= slen) return;
  auto bias_of = [&](uint32_t v) {
    return a.bias_f32 ? __uint_as_float(v) : (float)__builtin_bit_cast(T, (uint16_t)v);
  };
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t l = l0 + 4 * q + e;
    if (l >= llen) continue;
    const int64_t m = swap ? l : mr, n = swap ? mr : l;
    const float v = z[e] + bias_of(bias[0][e]), v2 = GLU ? z2[e] + bias_of(bias[H - 1][e]) : 1.0f;
    if (a.z) {
      float* row = a.z + m * a.n * H;
      row[n] = v;
      if (GLU) row[a.n + n] = v2;
    }
    const float y = act_fwd(a.act, v) * v2 + (float)__builtin_bit_cast(T, res[e]);
    static_cast<T*>(a.out)[m * a.n + n] = (T)y;
  }
}

// ---------------------------------------------------------------- operands and gradients beside the products

// Rows [rows][cols] of 16-bit elements at any alignment into 16-byte aligned rows of `pc`
// columns (a multiple of 8), zeros behind the last column: what the products read.  Two
// operands in one launch.
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a0, PackArgs a1, int64_t units0, int64_t units) {
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < units; u += (int64_t)gridDim.x * 256) {
    const PackArgs& a = u < units0 ? a0 : a1;
    const int64_t v = u < units0 ? u : u - units0, chunks = a.pc / 8, r = v / chunks;
    const int c = (int)(v - r * chunks) * 8;
    const uint16_t* const src = static_cast<const uint16_t*>(a.src) + r * a.ld + c;
    const int last = (int)a.cols - 1 - c;
    uint16_t e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = src[min(j, last)];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = j <= last ? e[j] : (uint16_t)0;
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = e[2 * j] | (uint32_t)e[2 * j + 1] << 16;
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.dst) + r * a.pc + c) = o;
  }
}

// The gradient of z: dz = dout * act'(z) (swiglu: both halves), rounded to T as the products'
// operand, into rows of `ldz` with zeros behind the last column; with `part` the column sums
// of the unrounded values over each chunk of rows, for the bias.  The rounding is the matrix
// cores' operand type: its remainder as a second operand would double both products.  With it dx
// and dW are 1.4 times as far from the exact gradients as their own rounding alone puts them
// (bf16 2.35e-3 for 1.66e-3 of their norm, fp16 2.9e-4 for 2.1e-4); db has its own alone.
// A workgroup takes 512 columns of a chunk, a wave every fourth row, kRows of them in flight; a
// lane holds eight consecutive columns (VEC), or every 64th where rows take no 16-byte accesses.
// Reads past a row's end give zeros and writes are dropped there, so nothing is behind a branch.
// Memory bounds it: the swiglu of 4416 x 10240 reads dout and z and writes dz, 633 MB in 130 us
// = 4.9 TB/s; the sums of 4416 x 11520 alone take 102 MB in 27.2 us (four rows in flight: 28.7).
template <typename T, bool VEC>
struct Eight {
  typename Vec8<T>::type v;
  static __device__ __forceinline__ int col(int lane, int j) { return VEC ? lane * 8 + j : j * 64 + lane; }
  __device__ __forceinline__ void load(const T* row, int n, int cols, int lane) {
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(row, (uint32_t)cols * 2);
    if constexpr (VEC) {
      v = __builtin_bit_cast(typename Vec8<T>::type, load_16(rs, (n + lane * 8) * 2));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __builtin_bit_cast(T, load_2(rs, (n + j * 64 + lane) * 2));
    }
  }
  __device__ __forceinline__ void store(T* row, int n, int cols, int lane) const {
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(row, (uint32_t)cols * 2);
    if constexpr (VEC) {
      store_16(__builtin_bit_cast(u32x4, v), rs, (n + lane * 8) * 2);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) store_2(__builtin_bit_cast(uint16_t, (T)v[j]), rs, (n + j * 64 + lane) * 2);
    }
  }
};

// The same columns of a row of fp32 values.
template <bool VEC>
struct EightF32 {
  float v[8];
  __device__ __forceinline__ void load(const float* row, int n, int cols, int lane) {
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(row, (uint32_t)cols * 4);
    if constexpr (VEC) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const f32x4 x = __builtin_bit_cast(f32x4, load_16(rs, (n + lane * 8 + q * 4) * 4));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[q * 4 + j] = x[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(load_4(rs, (n + j * 64 + lane) * 4));
    }
  }
};

template <typename T, int ACT, bool VEC>
__global__ __launch_bounds__(256) void dact_kernel(DactArgs a) {
  constexpr bool kGlu = ACT == kActSwiglu;
  constexpr int kRows = ACT == kActNone ? 8 : 4;
  __shared__ float sum[kGlu ? 2 : 1][4][512];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = blockIdx.x * 512, wide = kGlu ? 2 * a.n : a.n;
  const int64_t r0 = (int64_t)blockIdx.y * a.chunk, r1 = r0 + a.chunk < a.m ? r0 + a.chunk : a.m;
  float s1[8] = {}, s2[8] = {};
  for (int64_t m0 = r0 + wave; m0 < r1; m0 += 4 * kRows) {
    Eight<T, VEC> d[kRows], up[kRows];
    EightF32<VEC> z[kRows], z2[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int64_t m = m0 + 4 * u;
      const int cols = m < r1 ? a.n : 0;  // rows past the chunk: nothing is read, zeros are added
      d[u].load(static_cast<const T*>(a.dout) + m * a.ldd, n, cols, lane);
      if constexpr (ACT != kActNone) {
        z[u].load(a.z + m * wide, n, cols, lane);
        if constexpr (kGlu) z2[u].load(a.z + m * wide + a.n, n, cols, lane);
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int64_t m = m0 + 4 * u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float g = (float)d[u].v[j];
        if constexpr (kGlu) {
          const float zz = z[u].v[j], h = g * act_fwd(ACT, zz);
          g = g * z2[u].v[j] * act_grad(ACT, zz);
          up[u].v[j] = (T)h;
          s2[j] += h;
        } else if constexpr (ACT != kActNone) {
          g *= act_grad(ACT, z[u].v[j]);
        }
        d[u].v[j] = (T)g;
        s1[j] += g;
      }
      if (a.dz && m < r1) {
        T* row = static_cast<T*>(a.dz) + m * a.ldz;
        // the last columns of a row go up to its end
        d[u].store(row, n, kGlu ? a.n : (int)a.ldz, lane);
        if constexpr (kGlu) up[u].store(row + a.n, n, (int)a.ldz - a.n, lane);
      }
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    sum[0][wave][j * 64 + lane] = s1[j];
    if constexpr (kGlu) sum[1][wave][j * 64 + lane] = s2[j];
  }
  __syncthreads();
  for (int u = threadIdx.x; u < (kGlu ? 1024 : 512); u += 256) {
    const int half = u >> 9, at = u & 511, col = n + at;
    const int v = VEC ? (at & 7) * 64 + (at >> 3) : at;
    if (col < a.n)
      a.part[(int64_t)blockIdx.y * wide + half * a.n + col] =
          sum[half][0][v] + sum[half][1][v] + sum[half][2][v] + sum[half][3][v];
  }
}

// The bias's gradient: the chunks' column sums, added in order by 16 thread rows.
template <typename T>
__global__ __launch_bounds__(256) void dbias_kernel(const float* part, int chunks, int n, void* dst, int f32) {
  __shared__ float sum[16][16];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, col = blockIdx.x * 16 + tx;
  float s = 0.0f;
  if (col < n)
    for (int q = ty; q < chunks; q += 16) s += part[(int64_t)q * n + col];
  sum[ty][tx] = s;
  __syncthreads();
  if (ty != 0 || col >= n) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += sum[i][tx];
  if (f32)
    static_cast<float*>(dst)[col] = s;
  else
    static_cast<T*>(dst)[col] = (T)s;
}

using Big = Tile<2, 2, 4, 4, 1>;    // 256 x 256, 4 waves of 128 x 128, one workgroup a CU
using Small = Tile<2, 2, 2, 2, 2>;  // 128 x 128, 4 waves of 64 x 64, two workgroups a CU

template <typename T, bool AK, bool BKC, typename TL>
hipError_t run_tiles(const GemmArgs& a, hipStream_t st) {
  const int tiles = a.tm * a.tn, rest = tiles - a.whole;
  gemm_kernel<T, AK, BKC, TL><<<a.whole + rest * a.parts, TL::NT, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || rest == 0) return e;
  join_kernel<T, TL><<<rest * (TL::WAVES * TL::MI * TL::NI / 2) / 4, 256, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T, bool AK, bool BKC>
hipError_t run_shape(const GemmArgs& a, hipStream_t st) {
  return a.big ? run_tiles<T, AK, BKC, Big>(a, st) : run_tiles<T, AK, BKC, Small>(a, st);
}

template <typename T>
hipError_t run_skinny(const GemmArgs& a, hipStream_t st) {
  const int swap = a.skinny == 2;
  const int64_t len = swap ? a.m : a.n, s = swap ? a.n : a.m;
  const uint32_t grid = (uint32_t)((len + 15) / 16);
  constexpr int NT = 64 * kSkinnyWaves;
  if (a.act == kActSwiglu) {
    if (s <= 16) skinny_kernel<T, 1, true><<<grid, NT, 0, st>>>(a, swap);
    else skinny_kernel<T, 2, true><<<grid, NT, 0, st>>>(a, swap);
  } else if (s <= 16) skinny_kernel<T, 1, false><<<grid, NT, 0, st>>>(a, swap);
  else if (s <= 32) skinny_kernel<T, 2, false><<<grid, NT, 0, st>>>(a, swap);
  else if (s <= 48) skinny_kernel<T, 3, false><<<grid, NT, 0, st>>>(a, swap);
  else skinny_kernel<T, 4, false><<<grid, NT, 0, st>>>(a, swap);
  return hipGetLastError();
}

template <typename T>
hipError_t run(const GemmArgs& a, hipStream_t st) {
  if (a.skinny) return run_skinny<T>(a, st);
  if (a.thin) {
    thin_kernel<T, Small><<<a.whole, Small::NT, 0, st>>>(a);
    return hipGetLastError();
  }
  if (a.a_kc && a.b_kc) return run_shape<T, true, true>(a, st);
  if (a.a_kc) return run_shape<T, true, false>(a, st);
  return run_shape<T, false, false>(a, st);
}

}  // namespace

void gemm_plan(GemmArgs& a) {
  const bool glu = a.act == kActSwiglu;
  a.kt = (int)((a.k + kBK - 1) / kBK);
  a.skinny = a.thin = 0;
  if (a.a_kc && a.b_kc) {
    // 49 to 64 rows only while the long side is one round of two workgroups a CU (64 by 3840 x
    // 3840: 11.4 us, tiles 16.3; by 3840 x 11520: 30.3, tiles 27.0); 48 by 3840 x 11520 25.5,
    // by 10240 x 3840 22.0, tiles 27.0 and 23.8; 32 by a swiglu of 3840 x 2 x 5760 17.2, tiles
    // 26.7, by 10240 x 2 x 1920 22.5, tiles 23.3.
    auto few = [&](int64_t rows, int64_t len) { return rows <= (glu ? 32 : len <= 512 * 16 ? 64 : 48); };
    if (few(a.m, a.n)) a.skinny = 1;
    else if (few(a.n, a.m) && !glu) a.skinny = 2;
  }
  a.part_floats = 0;
  a.parts = 1;
  a.tm = a.tn = a.whole = 0;
  if (a.skinny) return;
  a.thin = a.a_kc && a.b_kc && a.k <= kBK && a.vec;
  if (a.thin) {
    a.tm = (int)((a.m + Small::BM - 1) / Small::BM);
    a.tn = (int)((a.n + (glu ? Small::BN / 2 : Small::BN) - 1) / (glu ? Small::BN / 2 : Small::BN));
    a.whole = a.tm * a.tn;
    return;
  }
  // The tile shape and the split of the last round's tiles with the least estimated time, in
  // stages of the large tile on every CU.  Measured at 8192 x 8192 x K: large tiles 1.48 us a
  // stage and 11 us for a round's start and epilogue; small ones 0.94 us and 5 us for a round
  // of two a CU, 0.55 us a stage for one a CU; joining 4 us and the sums' way out and back at
  // 4 TB/s.  1280 x 3840 x 10240: 75 large tiles, whole 254 us, in 3 pieces 109; 300 small
  // ones 136.
  double best = 1e30;
  for (int big = 1; big >= 0; --big) {
    const int bm = big ? Big::BM : Small::BM, bn = (big ? Big::BN : Small::BN) / (glu ? 2 : 1);
    const int64_t tm = (a.m + bm - 1) / bm, tn = (a.n + bn - 1) / bn, tiles = tm * tn;
    const int slots = big ? 256 : 512;
    const double start = big ? 7.5 : 3.6;
    for (int p = 1; p <= 16; ++p) {
      // rows that take no 16-byte accesses are finished by the small tiles themselves, and
      // with large ones by the join
      const int64_t rest = !a.vec && (big || p > 1) ? tiles : p == 1 ? 0 : tiles % slots;
      if (p > 1 && (rest == 0 || a.kt / p < 4)) continue;
      const int64_t whole = tiles - rest;
      const double stage = big ? 1.0 : tiles <= 256 && rest * p <= 256 ? 0.37 : 0.63;
      double cost = (double)((whole + slots - 1) / slots) * (a.kt * stage + start);
      if (rest) {
        const double bytes = (double)rest * p * bm * (big ? Big::BN : Small::BN) * 4;
        cost += (double)((rest * p + slots - 1) / slots) * ((a.kt + p - 1) / p * stage + start) + 2.7 +
                bytes * 2 / 4e6 / 1.48;
      }
      if (cost < best) {
        best = cost;
        a.big = big;
        a.tm = (int)tm;
        a.tn = (int)tn;
        a.whole = (int)whole;
        a.parts = p;
        a.part_floats = rest * p * bm * (big ? Big::BN : Small::BN);
      }
    }
  }
}

hipError_t launch_gemm(const GemmArgs& a, int f16, hipStream_t st) {
  return f16 ? run<_Float16>(a, st) : run<__bf16>(a, st);
}

hipError_t launch_pack(const PackArgs& a, const PackArgs& b, hipStream_t st) {
  const int64_t units0 = a.src ? a.rows * (a.pc / 8) : 0, units = units0 + (b.src ? b.rows * (b.pc / 8) : 0);
  if (units == 0) return hipSuccess;
  const int64_t blocks = (units + 255) / 256;
  pack_kernel<<<(uint32_t)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(a, b, units0, units);
  return hipGetLastError();
}

namespace {

template <typename T, bool VEC>
void run_dact(const DactArgs& a, dim3 grid, hipStream_t st) {
  if (a.act == kActSwiglu) dact_kernel<T, kActSwiglu, VEC><<<grid, 256, 0, st>>>(a);
  else if (a.act == kActSilu) dact_kernel<T, kActSilu, VEC><<<grid, 256, 0, st>>>(a);
  else if (a.act == kActGelu) dact_kernel<T, kActGelu, VEC><<<grid, 256, 0, st>>>(a);
  else dact_kernel<T, kActNone, VEC><<<grid, 256, 0, st>>>(a);
}

}  // namespace

hipError_t launch_dact(int f16, const DactArgs& a, hipStream_t st) {
  const int64_t rows = a.act == kActSwiglu ? 2 * a.n : a.n;
  const int64_t cols = a.dz ? a.ldz - (rows - a.n) : a.n;  // of the (last) half, with the zeros behind it
  const dim3 grid((uint32_t)((cols + 511) / 512), (uint32_t)a.chunks);
  if (f16) a.vec ? run_dact<_Float16, true>(a, grid, st) : run_dact<_Float16, false>(a, grid, st);
  else a.vec ? run_dact<__bf16, true>(a, grid, st) : run_dact<__bf16, false>(a, grid, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.part) return e;
  if (f16)
    dbias_kernel<_Float16><<<(uint32_t)((rows + 15) / 16), 256, 0, st>>>(a.part, (int)a.chunks, (int)rows, a.dbias, a.bias_f32);
  else
    dbias_kernel<__bf16><<<(uint32_t)((rows + 15) / 16), 256, 0, st>>>(a.part, (int)a.chunks, (int)rows, a.dbias, a.bias_f32);
  return hipGetLastError();
}

}  // namespace sage
