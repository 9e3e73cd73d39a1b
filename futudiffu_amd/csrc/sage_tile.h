// Device code that the products of the linear layers share: the activations, the epilogues
// straight from the accumulators or by way of LDS, an operand's part of an LDS stage and its
// fragments, the schedule of tiles over the XCDs, and the waits between loads and products.
#pragma once
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

// Tile t of the schedule: groups of G tile rows, column by column inside, so that the 32
// tiles an XCD runs together share G row panels and 32 / G column panels.
template <int G = 4>
__device__ __forceinline__ void tile_at(const GemmArgs& a, int t, int& tm, int& tn) {
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

// A tile's sums of one piece of the contraction, in the order the lanes hold them.
template <int MI, int NI>
__device__ __forceinline__ void store_piece(float* part, int wave, int lane, const f32x16 (&acc)[MI][NI]) {
  float* const dst = part + wave * (MI * NI * 1024) + lane * 4;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(dst + ((i * NI + j) * 4 + q) * 256) =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
}

// Adds the pieces of the cut tiles in order and finishes them: a wave takes one 32 x 64
// block of a tile.  Large tiles whose rows take no 16-byte accesses all come through here.
// Bound by the sums' way back: 75 tiles of 256 x 256 in three pieces, 79 MB with the residual
// and the output, in 16 us = 4.9 TB/s.
template <typename T, typename TL, int G = 4>
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
  tile_at<G>(a, a.whole + t, tm, tn);
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

}  // namespace

}  // namespace sage
