// Microscaled 4-bit floating point (MXFP4) for gfx950: rows to codes and back, and the linear
// layer out = act(Q(x) W^T + b) + r over codes.
//
// A row's columns in blocks of 32 share a scale 2^e (E8M0: e + 127 in a byte, 255: NaN), a
// column is an e2m1 code: +-{0, .5, 1, 1.5, 2, 3, 4, 6} times the scale.  Of a block with the
// largest magnitude amax, e = max(floor(log2 amax) - 2, -127), so x / 2^e is exact and below 8;
// codes are its nearest, ties to the even one, past 6 it saturates.  A block that holds NaN or
// infinity gets the scale 255: all of it reads as NaN.
//
// In memory: codes [rows][cols / 2], the even column in a byte's low half, rows padded to 256
// columns with zeros; scales [cols / 256][rows][8].  256 columns are 128 bytes of codes and 8 of
// scales a row: one LDS stage, read as the linear layers' 16-bit operands read theirs, 4 codes for
// an element of 16 bits (the sizes in GemmArgs count those).
#include <algorithm>

#include "sage_mx.h"
#include "sage_tile.h"

namespace sage {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------- codes

// Eight columns of T (a 16-byte access) to codes; bits: the largest magnitude of the lane's.
__device__ __forceinline__ uint32_t top_of(bf16x8 v) {
  const u32x4 u = __builtin_bit_cast(u32x4, v);
  uint32_t lo = 0, hi = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo = max(lo, u[i] << 17);
    hi = max(hi, u[i] << 1 >> 17 << 17);
  }
  return max(lo, hi) >> 1;
}
__device__ __forceinline__ uint32_t top_of(f16x8 v) {
  const u32x4 u = __builtin_bit_cast(u32x4, v);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, max(u[i] & 0x7fffu, u[i] >> 16 & 0x7fffu));
  return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m));
}
__device__ __forceinline__ uint32_t codes_of(bf16x8 v, float scale) {
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, bf16x2{v[0], v[1]}, scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, bf16x2{v[2], v[3]}, scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, bf16x2{v[4], v[5]}, scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, bf16x2{v[6], v[7]}, scale, 3);
}
__device__ __forceinline__ uint32_t codes_of(f16x8 v, float scale) {
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(0u, f16x2{v[0], v[1]}, scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, f16x2{v[2], v[3]}, scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, f16x2{v[4], v[5]}, scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, f16x2{v[6], v[7]}, scale, 3);
}

// Columns n .. n + 7 of a row of `cols`, through a resource that ends with the row.
template <typename T, bool VEC>
__device__ __forceinline__ typename Vec8<T>::type load_eight(const T* row, int n, int cols) {
  using V = typename Vec8<T>::type;
  const __amdgpu_buffer_rsrc_t rs = raw_rsrc(row, (uint32_t)cols * 2);
  if constexpr (VEC) return __builtin_bit_cast(V, load_16(rs, n * 2));
  V v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = __builtin_bit_cast(T, load_2(rs, (n + j) * 2));
  return v;
}

constexpr int kQuantRows = 4;  // rows of a wave, in flight together

// A wave takes 512 columns of kQuantRows rows, a lane eight of each row: four lanes a block.  The bytes bound it:
// 17408 x 3840, 170 MB in 33 us, a large copy's rate; one row, 1.7 us of latency.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(MxQuantArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t row0 = ((int64_t)blockIdx.x * 4 + wave) * kQuantRows;
  if (row0 >= a.m) return;
  const int n = blockIdx.y * 512 + lane * 8, left = (int)min((int64_t)kQuantRows, a.m - row0);
  const bool in = n < a.kp;
  typename Vec8<T>::type v[kQuantRows];
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r)
    v[r] = load_eight<T, VEC>(static_cast<const T*>(a.x) + (row0 + r) * a.ldx, n, r < left ? a.k : 0);
  int mine = 0;
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r) {
    const int e = block_exponent(quad_max(top_of(v[r])));
    const uint32_t c = e == 255 ? 0u : codes_of(v[r], scale_of(e));
    if (r < left && in) *reinterpret_cast<uint32_t*>(a.codes + (row0 + r) * (a.kp / 2) + n / 2) = c;
    if ((lane & 3) == r) mine = e;
  }
  // lane 4 i + r has row r's scale of block i
  if ((lane & 3) < left && in)
    a.scales[((int64_t)(n >> 8) * a.m + row0 + (lane & 3)) * 8 + (n >> 5 & 7)] = (uint8_t)mine;
}

template <typename T>
struct Decode;
template <>
struct Decode<__bf16> {
  static constexpr uint16_t kNaN = 0x7fc0;
  template <int I>
  static __device__ __forceinline__ uint32_t pair(uint32_t c, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, I));
  }
};
template <>
struct Decode<_Float16> {
  static constexpr uint16_t kNaN = 0x7e00;
  template <int I>
  static __device__ __forceinline__ uint32_t pair(uint32_t c, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, I));
  }
};

// Codes to rows of T, ldo apart; the same shares.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(MxDequantArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t row0 = ((int64_t)blockIdx.x * 4 + wave) * kQuantRows;
  if (row0 >= a.m) return;
  const int n = blockIdx.y * 512 + lane * 8, left = (int)min((int64_t)kQuantRows, a.m - row0);
  if (n >= a.k) return;
  uint32_t c[kQuantRows];
  int e[kQuantRows];
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r) {
    const int64_t row = row0 + min(r, left - 1);
    c[r] = *reinterpret_cast<const uint32_t*>(a.codes + row * (a.kp / 2) + n / 2);
    e[r] = a.scales[((int64_t)(n >> 8) * a.m + row) * 8 + (n >> 5 & 7)];
  }
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r) {
    if (r >= left) break;
    const float s = scale_of(e[r]);
    using D = Decode<T>;
    u32x4 o = {D::template pair<0>(c[r], s), D::template pair<1>(c[r], s), D::template pair<2>(c[r], s),
               D::template pair<3>(c[r], s)};
    if (e[r] == 255) o = u32x4{D::kNaN * 0x10001u, D::kNaN * 0x10001u, D::kNaN * 0x10001u, D::kNaN * 0x10001u};
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(static_cast<T*>(a.out) + (row0 + r) * a.ldo, (uint32_t)a.k * 2);
    if constexpr (VEC) {
      store_16(o, rs, n * 2);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) store_2((uint16_t)(o[j / 2] >> 16 * (j & 1)), rs, (n + j) * 2);
    }
  }
}

// ---------------------------------------------------------------- tiles

__device__ __forceinline__ i32x8 wide(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

template <int S>
__device__ __forceinline__ f32x16 mx32(i32x4 a, int sa, i32x4 b, int sb, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), c, 4, 4, S, sa, S, sb);
}
template <int S>
__device__ __forceinline__ f32x4 mx16(i32x4 a, int sa, i32x4 b, int sb, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(a), wide(b), c, 4, 4, S, sa, S, sb);
}

constexpr int kMxGroup = 8;   // tile rows that the schedule takes together

// A tile shape: WM x WN waves, each with MI x NI blocks of 32 x 32, two waves a SIMD, and D stages
// of LDS.  A stage is 128 columns: 64 bytes a row.  The scales of two stages (8 bytes a row) lie behind the ring, in
// D / 2 places.
template <int WM_, int WN_, int MI_, int NI_, int D_>
struct MxTile {
  static constexpr int WM = WM_, WN = WN_, MI = MI_, NI = NI_, D = D_;
  static constexpr int WAVES = WM * WN, NT = 64 * WAVES;
  static constexpr int BM = WM * MI * 32, BN = WN * NI * 32;
  static constexpr int A_BYTES = BM * 64, STAGE = (BM + BN) * 64, RING = D * STAGE;
  static constexpr int SCALES = (BM + BN) * 8, LDS = RING + D / 2 * SCALES, SLOADS = (SCALES / 256 + WAVES - 1) / WAVES;
  static constexpr int OUT = 32 * NI * 64;  // of the epilogue: 32 rows of a wave's columns
};

using MxBig = MxTile<2, 4, 4, 2, 4>;    // 256 x 256, 8 waves of 128 x 64, one workgroup a CU
using MxTail = MxTile<4, 2, 1, 2, 4>;   // 128 x 128, 8 waves of 32 x 64, behind them
using MxMid = MxTile<4, 2, 2, 2, 4>;    // 256 x 128, 8 waves of 64 x 64, one workgroup a CU
using MxSmall = MxTile<2, 2, 2, 2, 4>;  // 128 x 128, 4 waves of 64 x 64, two workgroups a CU

// One operand's part of an LDS stage: ROWS rows of 64 bytes, row r's 16-byte chunk c at
// c ^ ((r >> 2) & 3): the 16 rows that a fragment read touches at a time lie on 16 different
// 16-byte columns of the 256 bytes of banks.  A load moves 16 rows, four lanes a row.
template <int ROWS, int WAVES>
struct MxOperand {
  static constexpr int LOADS = ROWS * 64 / 1024 / WAVES;  // of one wave
  int off[LOADS];
  // glu: tile row j is row (j / 64) * 32 + j % 32 of half (j / 32) % 2, the halves `half` rows apart
  __device__ __forceinline__ void init(int64_t pitch, int wave, int lane, bool glu, int64_t half) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int r = (i * WAVES + wave) * 16 + (lane >> 2);
      const int c = (lane & 3) ^ ((r >> 2) & 3);
      const bool up = glu && ((r >> 5) & 1);
      if (glu) r = (r >> 6) * 32 + (r & 31);
      off[i] = (int)(r * pitch + (up ? half * pitch : 0)) + c * 16;
    }
  }
  // Issues the loads of a stage that starts at `p`, `left` bytes before the operand's end: rows past
  // the last read zeros.
  __device__ __forceinline__ void issue(uint8_t* lds, const uint8_t* p, uint32_t left, int wave) const {
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(p, left);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) dma_16(lds + (i * WAVES + wave) * 1024, rs, off[i]);
  }
};

// A tile's place: rows from m0 and columns from n0 on, columns 256 g0 .. 256 g1 of the contraction, and where
// its sums go if they are a piece's.
struct MxPlace {
  int64_t m0;
  int n0, g0, g1;
  float* part;
};

// The bytes from row row0 to the end of `rows` rows, as a resource takes them.
__device__ __forceinline__ uint32_t bytes_left(int64_t rows, int64_t row0, int64_t pitch) {
  return (uint32_t)min((rows - row0) * pitch, (int64_t)0x7fffffff);
}

// Waits for every LDS read and for all but the last N loads.
template <int N>
__device__ __forceinline__ void wait_all_but() {
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
}

// The epilogue of a wave's MI x NI blocks from row m0 and column n0 on: z = acc + bias, kept when the
// backward wants it, out = act(z) + residual, rounded once.  A lane's accumulators are four
// consecutive columns of its row, again and again: 32 rows at a time go through LDS (`lds`: this
// wave's; a row's 16-byte chunks permuted so that rows lie on different banks), so that the stores
// are whole rows of the wave.
// What a call does not have (residual, z) has a resource of no bytes.  PLAIN: out alone.
template <typename T, int ACT, bool PLAIN, int MI, int NI>
__device__ __forceinline__ void mx_finish(const GemmArgs& a, uint8_t* lds, int lane, int64_t m0, int n0,
                                          f32x16 (&c)[MI][NI]) {
  constexpr bool kGlu = ACT == kActSwiglu;
  constexpr int kStep = kGlu ? 2 : 1, kCols = NI * 32 / kStep, kLanes = kCols / 8, kRows = 64 / kLanes;
  // byte offset of 16-byte chunk v of row r: 256 bytes hold 128 / kCols rows, which the permutation keeps
  auto at_of = [](int r, int v) {
    return r * (kCols * 2) + ((v ^ (kLanes == 4 ? (r >> 2) & 3 : r & (kLanes - 1))) << 4);
  };
  const int64_t left = a.m - m0;
  if (left <= 0) return;
  const int rows = left < 32 * MI ? (int)left : 32 * MI, h = lane >> 5, r = lane & 31;
  const int wide = kGlu ? 2 * a.n : a.n;
  const __amdgpu_buffer_rsrc_t out = raw_rsrc(static_cast<T*>(a.out) + m0 * a.n, (uint32_t)rows * a.n * 2);
  const __amdgpu_buffer_rsrc_t res = raw_rsrc(static_cast<const T*>(a.res) + m0 * a.ldr,
                                              a.res ? (uint32_t)(((rows - 1) * a.ldr + a.n) * 2) : 0u);
  const __amdgpu_buffer_rsrc_t zs = raw_rsrc(a.z + m0 * wide, a.z ? (uint32_t)rows * wide * 4 : 0u);
  const __amdgpu_buffer_rsrc_t bs = raw_rsrc(a.bias, a.bias ? (uint32_t)wide * (a.bias_f32 ? 4 : 2) : 0u);
  typedef T V4 __attribute__((ext_vector_type(4)));
  auto load_8 = [](__amdgpu_buffer_rsrc_t rs, int off) {
    return __builtin_bit_cast(V4, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0));
  };
  // the column of this lane's first accumulator of block j (its half for a swiglu), group q; an offset past any
  // size for one that does not exist
  auto column = [&](int j, int q) { return n0 + j / kStep * 32 + 8 * q + 4 * h; };
  auto beyond = [&](int n) { return n < a.n ? 0 : (int)0x80000000; };
  // the bias of the lane's columns, and a row block's residual: asked for together, and not at all where there is
  // none (4416 x 3840 onto 2 x 10240 197 us where the loads found nothing, 194 without them)
  f32x4 bias[NI][4] = {};
  V4 rows_of[NI / kStep][4] = {};
  auto residual = [&](int i) {
    if (!a.res) return;
#pragma unroll
    for (int j = 0; j < NI; j += kStep)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = column(j, q);
        rows_of[j / kStep][q] = load_8(res, (int)((32 * i + r) * a.ldr + n) * 2 | beyond(n));
      }
  };
  if constexpr (!PLAIN) {
    if (a.bias) {
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          // past the last column a column that lies past any bias, in bytes too
          const int n = column(j, q), at = (n < a.n ? n : 0x10000000) + (kGlu && (j & 1) ? a.n : 0);
          if (a.bias_f32) {
            bias[j][q] = __builtin_bit_cast(f32x4, load_16(bs, at * 4));
          } else {
            const V4 v = load_8(bs, at * 2);
            bias[j][q] = f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
          }
        }
    }
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    if constexpr (!PLAIN) residual(i);
#pragma unroll
    for (int j = 0; j < NI; j += kStep) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 z = {c[i][j][4 * q], c[i][j][4 * q + 1], c[i][j][4 * q + 2], c[i][j][4 * q + 3]};
        if constexpr (!PLAIN) {
          const V4 rv = rows_of[j / kStep][q];
          f32x4 z2;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            z[e] += bias[j][q][e];
            if constexpr (kGlu) z2[e] = c[i][j + 1][4 * q + e] + bias[j + 1][q][e];
          }
          if constexpr (ACT != kActNone) {
            if (a.z) {
              const int n = column(j, q), at = ((32 * i + r) * wide + n) * 4 | beyond(n);
              store_16(__builtin_bit_cast(u32x4, z), zs, at);
              if constexpr (kGlu) store_16(__builtin_bit_cast(u32x4, z2), zs, at + a.n * 4);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            z[e] = act_fwd(ACT, z[e]);
            if constexpr (kGlu) z[e] *= z2[e];
            z[e] += (float)rv[e];
          }
        }
        V4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)z[e];
        *reinterpret_cast<V4*>(lds + at_of(r, j / kStep * 4 + q) + 8 * h) = o;
      }
    }
    // the wave's values are written before they are read, and read before the next are written
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int n = n0 + lane % kLanes * 8, none = n < a.n ? 0 : (int)0x80000000;
#pragma unroll
    for (int u = 0; u < 32 / kRows; ++u) {
      const int row = u * kRows + lane / kLanes;
      const u32x4 v = *reinterpret_cast<const u32x4*>(lds + at_of(row, lane % kLanes));
      store_16(v, out, ((32 * i + row) * a.n + n) * 2 | none);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

constexpr int kPlain = 8, kAny = 9;

// One tile.  LDS holds D stages; a stage is two steps of 64 columns, the next step's fragments read under
// this one's products.  Before a stage's last step the next stage has arrived and every wave has read
// this one's last fragments: behind that barrier A's loads of the stage D further on go into its place,
// and B's under the next stage's first step.  The scales of two stages go to one of D / 2 places behind
// the ring, with A's loads, D stages ahead.  FIN: the activation (kPlain: no bias and no
// residual either), a kernel each, so that none carries the others' registers; or kAny for rows that
// take no 16-byte accesses.
template <typename T, typename TL, int FIN>
__device__ __forceinline__ void mx_tile(const MxGemmArgs& x, uint8_t* lds, int wave, int lane, const MxPlace p) {
  const GemmArgs& a = x.g;
  const bool glu = FIN == kAny ? a.act == kActSwiglu : FIN == kActSwiglu;
  const int64_t pitch = a.lda * 2, rows = glu ? 2 * (int64_t)a.n : a.n;
  MxOperand<TL::BM, TL::WAVES> A;
  MxOperand<TL::BN, TL::WAVES> B;
  constexpr int ALOADS = decltype(A)::LOADS, BLOADS = decltype(B)::LOADS, LOADS = ALOADS + BLOADS;
  A.init(pitch, wave, lane, false, 0);
  B.init(pitch, wave, lane, glu, a.n);
  const int wm = wave / TL::WN, wn = wave % TL::WN;
  const int h = lane >> 5, r = lane & 31;
  // the fragment of block i in step s: chunk 2 h + s of row r; blocks are 2 KiB apart
  int fa[2], fb[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int in = r * 64 + (((2 * h + s) ^ ((r >> 2) & 3)) << 4);
    fa[s] = wm * TL::MI * 2048 + in;
    fb[s] = TL::A_BYTES + wn * TL::NI * 2048 + in;
  }
  // the scales of 32 rows in 256 columns (two stages): a load moves them to LDS; lane (h, r) reads its row's
  // eight bytes and keeps the four that it needs, of chunks 2 h and 2 h + 1 of either stage, in the order of
  // the four steps.  (Through registers they would be waited for in order, and the stages asked for before
  // them too.)
  auto issue_scales = [&](int g) {  // zeros past the last
    uint8_t* const to = lds + TL::RING + (uint32_t)(g - p.g0) % (TL::D / 2) * TL::SCALES;
#pragma unroll
    for (int i = 0; i < TL::SLOADS; ++i) {
      // (of 12 parts and 8 waves four are loaded twice: every wave waits for the same number)
      const int u = (i * TL::WAVES + wave) % (TL::SCALES / 256), v = u - TL::BM / 32;
      const bool left = v < 0;
      const uint8_t* const from = left ? x.sa + ((int64_t)g * a.m + p.m0) * 8 : x.sb + ((int64_t)g * rows + p.n0) * 8;
      const uint32_t bytes = left ? bytes_left(a.m, p.m0, 8) : bytes_left(rows, p.n0, 8);
      const int row = left ? u * 32 : glu ? (v >> 1) * 32 + (v & 1) * a.n : v * 32;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(raw_rsrc(from, g < p.g1 ? bytes : 0u), to + u * 256, 4,
                                               row * 8 + lane * 4, 0, 0, 0);
    }
  };
  u32x2 na[TL::MI], nb[TL::NI];
  int sa[TL::MI], sb[TL::NI];
  auto read_scales = [&](int g) {
    const uint8_t* const at = lds + TL::RING + (uint32_t)(g - p.g0) % (TL::D / 2) * TL::SCALES + r * 8;
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) na[i] = operand_at<u32x2>(at + (wm * TL::MI + i) * 256);
#pragma unroll
    for (int i = 0; i < TL::NI; ++i) nb[i] = operand_at<u32x2>(at + TL::BM * 8 + (wn * TL::NI + i) * 256);
  };
  const uint32_t pick = h ? 0x07060302u : 0x05040100u;
  auto keep_scales = [&]() {
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) sa[i] = (int)__builtin_amdgcn_perm(na[i][1], na[i][0], pick);
#pragma unroll
    for (int i = 0; i < TL::NI; ++i) sb[i] = (int)__builtin_amdgcn_perm(nb[i][1], nb[i][0], pick);
  };
  const uint8_t* const pa = static_cast<const uint8_t*>(a.a) + p.m0 * pitch;
  const uint8_t* const pb = static_cast<const uint8_t*>(a.b) + p.n0 * pitch;
  const uint32_t la = bytes_left(a.m, p.m0, pitch), lb = bytes_left(rows, p.n0, pitch);
  // the loads of stage t: zeros past the last
  auto issue_a = [&](uint8_t* to, int t) { A.issue(to, pa + t * 64u, t < 2 * p.g1 ? la - t * 64u : 0, wave); };
  auto issue_b = [&](uint8_t* to, int t) {
    B.issue(to + TL::A_BYTES, pb + t * 64u, t < 2 * p.g1 ? lb - t * 64u : 0, wave);
  };

  f32x16 acc[TL::MI][TL::NI] = {};
  i32x4 va[2][TL::MI], vb[2][TL::NI];
  auto read = [&](const uint8_t* at, int s) {
#pragma unroll
    for (int i = 0; i < TL::NI; ++i) vb[s][i] = operand_at<i32x4>(at + fb[s] + i * 2048);
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) va[s][i] = operand_at<i32x4>(at + fa[s] + i * 2048);
  };
  auto products = [&](auto step) {  // step of the 256 columns
    constexpr int S = decltype(step)::value;
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
      for (int j = 0; j < TL::NI; ++j)
        acc[i][j] = mx32<S>(vb[S & 1][j], sb[j], va[S & 1][i], sa[i], acc[i][j]);
  };
  // the order of one step: the reads first, two a product, then the loads (direct ones stay behind the
  // reads)
  auto order = [&](auto reads, auto loads) {
    constexpr int M = TL::MI * TL::NI, R = decltype(reads)::value, N = decltype(loads)::value;
    constexpr int E = (R + 1) / 2 < M ? (R + 1) / 2 : M, L = M - E;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      order_mfma();
      if (i < E) order_read(), order_read();
      if constexpr (L > 0) {
        if (i >= E) {
#pragma unroll
          for (int l = (i - E) * N / L; l < (i - E + 1) * N / L; ++l) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
        }
      }
    }
    keep_order();
  };
  constexpr int R = TL::MI + TL::NI, AHEAD = (TL::D / 2 - 1) * (2 * LOADS + TL::SLOADS);
#pragma unroll
  for (int d = 0; d < TL::D; ++d) {
    issue_a(lds + d * TL::STAGE, 2 * p.g0 + d);
    if (d < TL::D - 1) issue_b(lds + d * TL::STAGE, 2 * p.g0 + d);
    if (d % 2 == 0) issue_scales(p.g0 + d / 2);
  }
  wait_all_but<AHEAD + ALOADS>();
  barrier();
  read(lds, 0);
  read_scales(p.g0);
  keep_scales();
  int now = 0, before = TL::RING - TL::STAGE;  // the present stage's place, and the one before
  for (int g = p.g0; g < p.g1; ++g) {
    auto stage = [&](auto half) {
      constexpr int J = decltype(half)::value;
      uint8_t* const at = lds + now;
      read(at, 1);
      products(std::integral_constant<int, 2 * J>{});
      issue_b(lds + before, 2 * g + J + TL::D - 1);
      order(std::integral_constant<int, R>{}, std::integral_constant<int, BLOADS>{});
      // the next stage is there, and with the second of a pair its scales
      wait_all_but<AHEAD>();
      barrier();
      before = now;
      now = now == TL::RING - TL::STAGE ? 0 : now + TL::STAGE;
      read(lds + now, 0);
      if constexpr (J == 1) read_scales(g + 1);
      products(std::integral_constant<int, 2 * J + 1>{});
      issue_a(at, 2 * g + J + TL::D);
      if constexpr (J == 0) issue_scales(g + TL::D / 2);
      order(std::integral_constant<int, J == 0 ? R : 2 * R>{},
            std::integral_constant<int, ALOADS + (J == 0 ? TL::SLOADS : 0)>{});
    };
    stage(std::integral_constant<int, 0>{});
    stage(std::integral_constant<int, 1>{});
    keep_scales();
  }
  wait_vmem();  // the loads in flight write this workgroup's LDS
  if (p.part) {
    store_piece(p.part, wave, lane, acc);
    return;
  }
  barrier();  // every wave has read its last fragments: the stages' LDS is free
  const int64_t mw = p.m0 + wm * TL::MI * 32;
  const int nw = p.n0 + wn * TL::NI * (glu ? 16 : 32);
  if constexpr (FIN != kAny) {
    mx_finish<T, FIN == kPlain ? kActNone : FIN, FIN == kPlain>(a, lds + wave * TL::OUT, lane, mw, nw, acc);
  } else {
    static_assert(TL::WAVES * 32 * kAnyPitch * 4 <= TL::RING, "the sums fit");
    float* const sums = reinterpret_cast<float*>(lds) + wave * 32 * kAnyPitch;
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) {
#pragma unroll
      for (int j = 0; j < TL::NI; j += 2) {
        stage_any(sums, lane, 0, acc[i][j], acc[i][j + 1]);
        finish_any_act<T, true, 1>(a, sums, lane, mw + 32 * i, nw + j * (glu ? 16 : 32));
        // the next columns' sums are written behind these reads
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
}

// The place of work unit u behind the whole tiles: a piece of a cut tile's contraction.
template <typename TL>
__device__ __forceinline__ MxPlace piece_at(const GemmArgs& a, int u) {
  const int piece = u % a.parts;
  int tm, tn;
  tile_at<kMxGroup>(a, a.whole + u / a.parts, tm, tn);
  return {(int64_t)tm * TL::BM, tn * (TL::BN / (a.act == kActSwiglu ? 2 : 1)), (int)((int64_t)a.kt * piece / a.parts),
          (int)((int64_t)a.kt * (piece + 1) / a.parts), a.part + (int64_t)u * (TL::BM * TL::BN)};
}
template <typename TL>
__device__ __forceinline__ MxPlace whole_at(const GemmArgs& a, int t) {
  int tm, tn;
  tile_at<kMxGroup>(a, t, tm, tn);
  return {(int64_t)tm * TL::BM, tn * (TL::BN / (a.act == kActSwiglu ? 2 : 1)), 0, a.kt, nullptr};
}

// The product by large tiles, one workgroup a CU, and behind them by small ones that cover what is left: the
// rows past the last whole tile row, and the whole tiles of a last round that would leave most of the card
// idle.
// A stage of 256 columns takes a CU 1.24 us when few work (2980 cycles, of which the matrix instructions need
// 2048), and 1.85 when all do: the power then allows the matrix instructions alone 5600 to 6300 TFLOP/s on
// random codes (8500 on zeros).  8192 x 8192 x 8192 258 to 267 us, 4130 to 4250 TFLOP/s (the library's product of
// the same codes 3180 to 3630); 4416 x 3840 onto 11520 112 us, 3470, with a bias 118; with a swiglu onto 2 x 10240
// 194 us, 3580: of a round's 63000 cycles, 15 stages of the contraction, 18000 are its start and epilogue.
// Kept out: a persistent workgroup that asks for the next tile during the epilogue (3 % for a product alone, and
// with a bias or an activation its registers spilled); 128 x 256 tiles by two workgroups a CU (their operands' way
// to LDS bounds them); rings of five and more stages and other orders of the tiles (no difference); each half
// of the waves on half of the contraction (none either).
template <typename T, int FIN>
__global__ __launch_bounds__(MxBig::NT, 2) void mx_gemm_kernel(MxGemmArgs x) {
  const GemmArgs& a = x.g;
  static_assert(MxBig::NT == MxTail::NT && MxTail::LDS <= MxBig::LDS && MxBig::WAVES * MxBig::OUT <= MxBig::RING &&
                    MxTail::WAVES * MxTail::OUT <= MxTail::RING, "one workgroup size, one LDS");
  __shared__ __align__(1024) uint8_t lds[MxBig::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, bid = blockIdx.x;
  if (bid < a.whole) {
    mx_tile<T, MxBig, FIN>(x, lds, wave, lane, whole_at<MxBig>(a, xcd_share(bid, a.whole)));
    return;
  }
  const int u = xcd_share(bid - a.whole, (int)gridDim.x - a.whole);
  if (a.parts > 1) {
    mx_tile<T, MxBig, FIN>(x, lds, wave, lane, piece_at<MxBig>(a, u));
    return;
  }
  constexpr int KM = MxBig::BM / MxTail::BM, KN = MxBig::BN / MxTail::BN;
  const int cut = (a.tm * a.tn - a.whole) * (KM * KN), width = MxTail::BN / (FIN == kActSwiglu ? 2 : 1);
  MxPlace p;
  if (u < cut) {
    p = whole_at<MxBig>(a, a.whole + u / (KM * KN));
    p.m0 += u % (KM * KN) / KN * MxTail::BM;
    p.n0 += u % KN * width;
    if (p.n0 >= a.n) return;  // a part of the last tile column that lies past the last column
  } else {
    const int64_t from = (int64_t)a.tm * MxBig::BM;
    const int v = u - cut, strip = (int)((a.m - from + MxTail::BM - 1) / MxTail::BM);
    p = {from + v % strip * MxTail::BM, v / strip * width, 0, a.kt, nullptr};
  }
  mx_tile<T, MxTail, FIN>(x, lds, wave, lane, p);
}

// The product by tiles of half the size, where the large ones would be too few for the CUs: a stage of 256
// columns takes 0.86 us with 150 busy CUs and 1.14 with all, the way of its operands to LDS and its
// products one after the other (0.4 us each).  1280 x 10240 onto 3840 41 us, where large tiles in three pieces of the
// contraction and their sums take 50 and whole ones 56.
template <typename T, int FIN>
__global__ __launch_bounds__(MxMid::NT, 2) void mx_mid_kernel(MxGemmArgs x) {
  static_assert(MxMid::WAVES * MxMid::OUT <= MxMid::RING, "the epilogue fits");
  __shared__ __align__(1024) uint8_t lds[MxMid::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  mx_tile<T, MxMid, FIN>(x, lds, wave, lane, whole_at<MxMid>(x.g, xcd_share(blockIdx.x, (int)gridDim.x)));
}

// The product by small tiles, two workgroups a CU: 0.75 us a stage of 256 columns alone on a CU, 1.28 for two, their
// operands' way to LDS (12 to 15 TB/s over the chip).  512 x 3840 onto 3840 11.7 us.
template <typename T, int FIN>
__global__ __launch_bounds__(MxSmall::NT, 2) void mx_small_kernel(MxGemmArgs x) {
  const GemmArgs& a = x.g;
  static_assert(MxSmall::LDS <= 80 * 1024 && MxSmall::WAVES * MxSmall::OUT <= MxSmall::RING, "two workgroups a CU");
  __shared__ __align__(1024) uint8_t lds[MxSmall::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, bid = blockIdx.x;
  if (bid < a.whole)
    mx_tile<T, MxSmall, FIN>(x, lds, wave, lane, whole_at<MxSmall>(a, xcd_share(bid, a.whole)));
  else
    mx_tile<T, MxSmall, FIN>(x, lds, wave, lane,
                             piece_at<MxSmall>(a, xcd_share(bid - a.whole, (int)gridDim.x - a.whole)));
}

// ---------------------------------------------------------------- few rows

// out for groups of 16 * MT rows of x (blockIdx.y), as the linear layers' skinny_kernel: a workgroup
// reads 16 rows of W (of both halves for a swiglu) once, its W waves take 256-column stages in turn
// through rings of D LDS slots of their own, and their sums are added in order.  A slot holds, for each
// group of 16 rows, 2 KiB of codes and 128 bytes of scales.
// QX: x is 16-bit, and its up to kMxQuantRows rows are quantized into LDS first, as mx_quantize_kernel
// does it; each workgroup does so again, while the first stages of W are under way: one row of 3840 onto 11520
// 7.1 us, onto 15360 from 256 columns 4.3, where a kernel before it makes that 8.3 and 5.0.  Of four rows onto
// 11520 it is 8.5 and 8.7, and with more the kernel before is faster.
// What bounds it are the operands' way into LDS (15 TB/s over the chip) and the start: 22 MB of W onto 11520 take
// 6.2 us with up to 16 rows, 4.4 at the rate of a copy.  Operands read to registers as the matrix
// instructions take them, without LDS, were slower from 8 rows on (32 rows 12 us, now 7.6).  Every workgroup
// reads all of x: of the 66 MB that 32 rows onto 11520 take to LDS 44 are x's.  (In QX x's codes lie 128 bytes
// apart without W's permutation: rows 0 and 2, and 1 and 3, share banks.)
template <typename T, int MT, bool GLU, int W, int D, bool QX>
__global__ __launch_bounds__(64 * W) void mx_skinny_kernel(MxGemmArgs args) {
  const GemmArgs& a = args.g;
  constexpr int H = GLU ? 2 : 1, TILES = H + (QX ? 0 : MT), PART = 2048 + 128, STAGE = TILES * PART;
  constexpr int XPART = kMxQuantRows * 136;
  __shared__ __align__(1024) uint8_t lds[W * D * STAGE + (QX ? kMxQuantCols / 256 * XPART : 0)];
  static_assert(H * MT * 1024 <= D * STAGE, "the sums fit");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  uint8_t* const mine = lds + wave * D * STAGE;
  uint8_t* const xlds = lds + W * D * STAGE;
  // pitch: bytes of a row of codes, the same on both sides
  const int64_t pitch = a.ldb * 2, m0 = (int64_t)blockIdx.y * 16 * MT;
  const int m = (int)(a.m - m0), chunks = a.kt;
  const int n0 = blockIdx.x * 16, rows = GLU ? 2 * a.n : a.n;
  const __amdgpu_buffer_rsrc_t xrs = raw_rsrc(static_cast<const uint8_t*>(a.a) + m0 * pitch, 0x7fffffff);
  __amdgpu_buffer_rsrc_t wrs[H];
#pragma unroll
  for (int h = 0; h < H; ++h)
    wrs[h] = raw_rsrc(static_cast<const uint8_t*>(a.b) + ((int64_t)n0 + (int64_t)h * a.n) * pitch, 0x7fffffff);
  // of a load's eight rows, lane l takes row l / 8 and the 16-byte chunk that lies at l % 8;
  // rows past the last read the last one again (what they give is not stored)
  int woff[2], xoff[MT][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = 8 * i + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
    woff[i] = (int)((min(n0 + row, a.n - 1) - n0) * pitch) + c * 16;
#pragma unroll
    for (int j = 0; j < MT; ++j) xoff[j][i] = (int)(min(16 * j + row, m - 1) * pitch) + c * 16;
  }
  // scales: lane l of the lower ones takes four bytes of row l / 2
  const int srow = lane >> 1;
  int wsoff[H], xsoff[MT];
#pragma unroll
  for (int h = 0; h < H; ++h) wsoff[h] = (min(n0 + srow, a.n - 1) + h * a.n) * 8 + 4 * (lane & 1);
#pragma unroll
  for (int j = 0; j < MT; ++j) xsoff[j] = min(16 * j + srow, m - 1) * 8 + 4 * (lane & 1);
  auto issue = [&](uint8_t* stage, int chunk) {
    const int at = chunk * 128;
    const __amdgpu_buffer_rsrc_t wss = raw_rsrc(args.sb + (int64_t)chunk * rows * 8, (uint32_t)rows * 8);
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int i = 0; i < 2; ++i) dma_16(stage + h * PART + i * 1024, wrs[h], woff[i] + at);
      if (lane < 32) __builtin_amdgcn_raw_ptr_buffer_load_lds(wss, stage + h * PART + 2048, 4, wsoff[h], 0, 0, 0);
    }
    if constexpr (QX) return;
    const __amdgpu_buffer_rsrc_t xss = raw_rsrc(args.sa + ((int64_t)chunk * a.m + m0) * 8, (uint32_t)m * 8);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) dma_16(stage + (H + j) * PART + i * 1024, xrs, xoff[j][i] + at);
      if (lane < 32) __builtin_amdgcn_raw_ptr_buffer_load_lds(xss, stage + (H + j) * PART + 2048, 4, xsoff[j], 0, 0, 0);
    }
  };
  const int q = lane >> 4, r = lane & 15;
  // in step s of a stage lane (q, r) multiplies chunk 2 q + s of row r, with byte 2 q + s of its scales
  int at[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) at[s] = r * 128 + (((2 * q + s) ^ ((r >> 1) & 7)) << 4);
  const int sat = 2048 + r * 8 + 2 * q;
  const int xrow = r % kMxQuantRows;  // QX: rows past the last are some other's, and not stored
  f32x4 acc[H][MT] = {};
  // wave i finishes the rows 16 i .. of x and every W-th 16 after: lane (q, r) columns 4 q .. + 3 of
  // row r.  Bias and residual are asked for first (zeros where there are none) and used last.
  constexpr int G = (MT + W - 1) / W;
  uint32_t bias[H][4];
  uint16_t res[G][4];
  if (wave < MT) {
    const __amdgpu_buffer_rsrc_t brs = raw_rsrc(a.bias, a.bias ? (uint32_t)rows * (a.bias_f32 ? 4 : 2) : 0u);
    const __amdgpu_buffer_rsrc_t rrs = raw_rsrc(static_cast<const T*>(a.res) + m0 * a.ldr, a.res ? 0x7fffffffu : 0u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + 4 * q + e, out = n < a.n ? 0 : (int)0x80000000;
#pragma unroll
      for (int h = 0; h < H; ++h)
        bias[h][e] = a.bias_f32 ? load_4(brs, (n + h * a.n) * 4 | out) : load_2(brs, (n + h * a.n) * 2 | out);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int mr = 16 * (wave + W * g) + r;
        res[g][e] = load_2(rrs, mr < m ? (int)((mr * a.ldr + n) * 2) | out : (int)0x80000000);
      }
    }
    keep_order();
  }
  // half a wave quantizes 256 columns of a row; rows 1, 2 or 4 are taken in turn, kAhead in flight
  constexpr int kAhead = 8;
  using V = typename Vec8<T>::type;
  const int shift = m <= 1 ? 0 : m <= 2 ? 1 : 2, units = chunks << shift, col = (lane & 31) * 8;
  V ahead[QX ? kAhead : 1];
  auto ask = [&](int u0) {
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(args.x, 0x7fffffffu);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int u = u0 + 2 * W * i, row = u & ((1 << shift) - 1), c = (u >> shift) * 256 + col;
      const int none = row < m && c < args.kx ? 0 : (int)0x80000000;
      ahead[i] = __builtin_bit_cast(V, load_16(rs, (int)(row * args.ldx + c) * 2 | none));
    }
  };
  auto put = [&](int u0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int u = u0 + 2 * W * i, row = u & ((1 << shift) - 1);
      const int e = block_exponent(quad_max(top_of(ahead[i])));
      const uint32_t codes = e == 255 ? 0u : codes_of(ahead[i], scale_of(e));
      if (u < units) {
        uint8_t* const to = xlds + (u >> shift) * XPART;
        *reinterpret_cast<uint32_t*>(to + row * 128 + (lane & 31) * 4) = codes;
        if ((lane & 3) == 0) to[kMxQuantRows * 128 + row * 8 + (lane & 31) / 4] = (uint8_t)e;
      }
    }
  };
  const int u0 = 2 * wave + (lane >> 5);
  if constexpr (QX) {
    ask(u0);
    keep_order();
  }
#pragma unroll
  for (int d = 0; d < D - 1; ++d)
    if (wave + d * W < chunks) issue(mine + d * STAGE, wave + d * W);
  if constexpr (QX) {
    put(u0);
#pragma unroll 1
    for (int u = u0 + 2 * W * kAhead; u - (lane >> 5) < units; u += 2 * W * kAhead) {
      ask(u);
      put(u);
    }
    __syncthreads();
  }
  int now = 0, free = (D - 1) * STAGE;
#pragma unroll 1
  for (int c = wave; c < chunks; c += W) {
    // this stage has arrived, and the last one's reads are done: its place takes the next loads
    if (c + (D - 1) * W < chunks) {
      wait_all_but<3 * TILES * (D - 2)>();
      hold_memory();
      issue(mine + free, c + (D - 1) * W);
    } else {
      wait_all_but<0>();
      hold_memory();
    }
    const uint8_t* stage = mine + now;
    int ws[H], xs[MT];
#pragma unroll
    for (int h = 0; h < H; ++h) ws[h] = *reinterpret_cast<const uint16_t*>(stage + h * PART + sat);
#pragma unroll
    for (int j = 0; j < MT; ++j)
      xs[j] = *reinterpret_cast<const uint16_t*>(QX ? xlds + c * XPART + kMxQuantRows * 128 + xrow * 8 + 2 * q
                                                    : stage + (H + j) * PART + sat);
    auto step = [&](auto s) {
      constexpr int S = decltype(s)::value;
      i32x4 w[H], x[MT];
#pragma unroll
      for (int h = 0; h < H; ++h) w[h] = operand_at<i32x4>(stage + h * PART + at[S]);
#pragma unroll
      for (int j = 0; j < MT; ++j)
        x[j] = operand_at<i32x4>(QX ? xlds + c * XPART + xrow * 128 + (2 * q + S) * 16
                                    : stage + (H + j) * PART + at[S]);
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[h][j] = mx16<S>(w[h], ws[h], x[j], xs[j], acc[h][j]);
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
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
  auto bias_of = [&](uint32_t v) {
    return a.bias_f32 ? __uint_as_float(v) : (float)__builtin_bit_cast(T, (uint16_t)v);
  };
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int group = wave + W * g, mr = 16 * group + r;
    if (group >= MT) return;
    f32x4 z = {}, z2 = {};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const f32x4* const p = reinterpret_cast<const f32x4*>(lds + w * D * STAGE) + group * 64 + lane;
      z += p[0];
      if (GLU) z2 += p[(H - 1) * MT * 64];
    }
    if (mr >= m) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t n = n0 + 4 * q + e;
      if (n >= a.n) continue;
      const float v = z[e] + bias_of(bias[0][e]), v2 = GLU ? z2[e] + bias_of(bias[H - 1][e]) : 1.0f;
      if (a.z) {
        float* row = a.z + (m0 + mr) * rows;
        row[n] = v;
        if (GLU) row[a.n + n] = v2;
      }
      const float y = act_fwd(a.act, v) * v2 + (float)__builtin_bit_cast(T, res[g][e]);
      static_cast<T*>(a.out)[(m0 + mr) * a.n + n] = (T)y;
    }
  }
}

template <typename T, typename TL>
hipError_t join_mx(const GemmArgs& a, hipStream_t st) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.parts == 1) return e;
  join_kernel<T, TL, kMxGroup><<<(a.tm * a.tn - a.whole) * (TL::WAVES * TL::MI * TL::NI / 2) / 4, 256, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T, int FIN>
hipError_t run_mx_tiles(const MxGemmArgs& x, hipStream_t st) {
  const GemmArgs& a = x.g;
  const int rest = (a.tm * a.tn - a.whole) * a.parts;
  if constexpr (FIN != kAny) {
    if (a.big == 2) {
      mx_mid_kernel<T, FIN><<<a.whole, MxMid::NT, 0, st>>>(x);
      return hipGetLastError();
    }
    if (a.big) {
      mx_gemm_kernel<T, FIN><<<a.whole + (a.parts > 1 ? rest : a.tails), MxBig::NT, 0, st>>>(x);
      return join_mx<T, MxBig>(a, st);
    }
  }
  mx_small_kernel<T, FIN><<<a.whole + rest, MxSmall::NT, 0, st>>>(x);
  return join_mx<T, MxSmall>(a, st);
}

// Waves and LDS slots of a wave.  Up to as many workgroups as the chip holds of them: four waves with deep rings,
// more bytes in flight on a CU (3840 columns of 3840, one row: 3.7 us against 4.9 for the other).  Past that: two
// waves, four and more workgroups a CU (with 64 rows three), so that all run at once (11520 columns: 6.2 us
// against 7.7; with 64 rows 10.7 against 14.5; 15360 of 256: 2.9 against 4.2).
template <int MT, bool GLU, bool QX>
struct SkinnyShape {
  static constexpr int STAGE = ((GLU ? 2 : 1) + (QX ? 0 : MT)) * 2176;
  static constexpr int XLDS = QX ? kMxQuantCols / 256 * kMxQuantRows * 136 : 0;
  static constexpr int fit(int bytes) { return (bytes - XLDS) / STAGE; }
  static constexpr int bound(int d, int lo, int hi) { return d < lo ? lo : d > hi ? hi : d; }
  // LDS: 80 KB (64 rows: all of it), or 40 KB (64 rows: 42.5, the two slots that it needs)
  static constexpr int FEW = bound(fit(80 * 1024) / 4, MT == 4 ? 3 : 2, 4), MANY = bound(fit(40 * 1024) / 2, 2, 3);
  // the same with QX: its sums are those of the codes, bit for bit
  static constexpr int FEW_SLOTS = MT == 4 ? 256 : 512;
};

template <typename T, int MT, bool GLU, bool QX>
hipError_t run_skinny(const MxGemmArgs& x, hipStream_t st) {
  const GemmArgs& a = x.g;
  using S = SkinnyShape<MT, GLU, QX>;
  const dim3 grid((uint32_t)((a.n + 15) / 16), (uint32_t)((a.m + 16 * MT - 1) / (16 * MT)));
  if ((int64_t)grid.x * grid.y > S::FEW_SLOTS) mx_skinny_kernel<T, MT, GLU, 2, S::MANY, QX><<<grid, 128, 0, st>>>(x);
  else mx_skinny_kernel<T, MT, GLU, 4, S::FEW, QX><<<grid, 256, 0, st>>>(x);
  return hipGetLastError();
}

template <typename T>
hipError_t run_mx(const MxGemmArgs& x, hipStream_t st) {
  const GemmArgs& a = x.g;
  if (!a.skinny) {
    if (!a.vec) return run_mx_tiles<T, kAny>(x, st);
    if (a.act == kActSwiglu) return run_mx_tiles<T, kActSwiglu>(x, st);
    if (a.act == kActSilu) return run_mx_tiles<T, kActSilu>(x, st);
    if (a.act == kActGelu) return run_mx_tiles<T, kActGelu>(x, st);
    return a.bias || a.res ? run_mx_tiles<T, kActNone>(x, st) : run_mx_tiles<T, kPlain>(x, st);
  }
  const bool glu = a.act == kActSwiglu;
  if (x.x && glu) return run_skinny<T, 1, true, true>(x, st);
  if (x.x) return run_skinny<T, 1, false, true>(x, st);
  if (glu) return a.skinny == 1 ? run_skinny<T, 1, true, false>(x, st) : run_skinny<T, 2, true, false>(x, st);
  if (a.skinny == 1) return run_skinny<T, 1, false, false>(x, st);
  if (a.skinny == 2) return run_skinny<T, 2, false, false>(x, st);
  if (a.skinny == 3) return run_skinny<T, 3, false, false>(x, st);
  return run_skinny<T, 4, false, false>(x, st);
}

template <typename T>
hipError_t run_quantize(const MxQuantArgs& a, hipStream_t st) {
  const dim3 grid((uint32_t)((a.m + 4 * kQuantRows - 1) / (4 * kQuantRows)), (uint32_t)((a.kp + 511) / 512));
  if (a.vec) mx_quantize_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else mx_quantize_kernel<T, false><<<grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t run_dequantize(const MxDequantArgs& a, hipStream_t st) {
  const dim3 grid((uint32_t)((a.m + 4 * kQuantRows - 1) / (4 * kQuantRows)), (uint32_t)((a.k + 511) / 512));
  if (a.vec) mx_dequantize_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else mx_dequantize_kernel<T, false><<<grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

void mx_gemm_plan(GemmArgs& a) {
  const bool glu = a.act == kActSwiglu;
  a.kt = (int)(a.k / kBK);
  a.thin = 0;
  a.part_floats = 0;
  a.parts = 1;
  a.tm = a.tn = a.whole = 0;
  // The least estimated time, in units of 1.85 us: 256 columns of the contraction for large tiles on every CU.
  // The sums of pieces move at 8 TB/s, their join and the launch cost 5.5 us.  Measured, the choice against each
  // shape alone (small, half, large, in us): 512 x 3840 onto 3840 11.7 (11.6, 16.3, 23.7), 1280 x 10240 onto 3840 40.7
  // (50.7, 41.4, 56.0), 1536 x 3840 onto 3840 19.5 (21.5, 20.0, 26.0), 2048 x 3840 onto 3840 22.5 (24.1, 22.7,
  // 27.2), 3000 x 3840 onto 3840 29.7 (35.4, 37.4, 29.8), 4416 x 3840 onto 11520 111 (139, 136, 123), 4416 x 10240
  // onto 3840 105 (131, 132, 135).
  // The kernel for few rows: 1.5 us a round and 0.7 for each 16 rows of x (and the swiglu's second half), its
  // operands at 15 TB/s.  Where the two meet, few rows and tiles in us: 3840 columns of 3840, 192 rows 10.6 and 10.8,
  // 256 rows 17.9 and 11.0; 11520 columns, 48 rows 9.0 and 10.6, 65 rows 17.7 and 10.9; 15360 columns of 256, 32 rows
  // 3.9 and 3.5, 48 rows 4.6 and 3.6; swiglu to 10240 columns of 3840, 32 rows 10.4 and 10.7, 33 rows 17.9 and 10.7;
  // 1536 columns of 1536, 256 rows 5.4 and 6.0, 667 rows 9.8 and 6.2; 256 columns of 3840, 2000 rows 8.9 and 14.6,
  // 4000 rows 19.3 and 10.4.
  const int64_t rows = glu ? 2 * (int64_t)a.n : a.n;
  auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
  double best = 1e30;
  a.skinny = 0;
  if (a.m <= 16384) {
    a.skinny = (int)std::min<int64_t>(up(a.m, 16), glu ? 2 : 4);
    const int tiles = a.skinny + glu;
    const int64_t groups = up(a.n, 16) * up(a.m, 16 * a.skinny);
    // workgroups that the chip holds, as SkinnyShape has them
    const int few = a.skinny == 4 ? 256 : 512, many = tiles == 4 ? 768 : tiles > 1 ? 1024 : 1536;
    best = ((double)up(groups, groups > few ? many : few) * (1.5 + 0.7 * tiles) +
            (double)groups * (tiles + 1) * a.kt * 2048 / 15e6) / 1.85;
    // less than any tiles take, whole or in pieces
    if (best <= 1.7 + std::min(a.kt * 0.4, 3.0 + a.kt * 0.025)) return;
  }
  auto take = [&](double cost, int big, int64_t tm, int64_t tn, int64_t whole, int parts, int64_t tails, int64_t sums) {
    if (cost + 1.0 >= best) return;
    best = cost + 1.0;
    a.skinny = 0;
    a.big = big;
    a.tm = (int)tm;
    a.tn = (int)tn;
    a.whole = (int)whole;
    a.parts = parts;
    a.tails = (int)tails;
    a.part_floats = sums;
  };
  // a stage of 256 columns of a round of `n` tiles, by shape: what the power allows past 150 busy CUs
  auto some = [](int64_t n, double few, double all) {
    return few + (all - few) * (double)std::max<int64_t>(n - 150, 0) / 106;
  };
  auto big_stage = [&](int64_t n) { return some(n, 0.68, 1.0); };
  auto mid_stage = [&](int64_t n) { return some(n, 0.465, 0.63); };
  auto small_stage = [](int64_t n) { return n <= 256 ? 0.4 : 0.69; };
  // n tiles in rounds of `slots`
  auto rounds_of = [&](int64_t n, int64_t slots, int kt, double start, auto stage) {
    const int64_t rest = n % slots;
    return (double)(n / slots) * (kt * stage(slots) + start) + (rest ? kt * stage(rest) + start : 0.0);
  };
  constexpr double kBig = 1.7, kMid = 1.2, kSmall = 0.7;  // start and epilogue of a round
  if (a.vec) {
    const int64_t tm = up(a.m, MxMid::BM), tn = up(rows, MxMid::BN), tiles = tm * tn;
    take(rounds_of(tiles, 256, a.kt, kMid, mid_stage), 2, tm, tn, tiles, 1, 0, 0);
  }
  // rows that take no 16-byte accesses are the small tiles'
  for (int big = a.vec ? 1 : 0; big >= 0; --big) {
    const int bm = big ? MxBig::BM : MxSmall::BM, bn = big ? MxBig::BN : MxSmall::BN, slots = big ? 256 : 512;
    const int64_t tm = up(a.m, bm), tn = up(rows, bn), tiles = tm * tn, rest = tiles % slots, whole = tiles - rest;
    auto cost = [&](int64_t n, int kt) {
      return big ? rounds_of(n, slots, kt, kBig, big_stage) : rounds_of(n, slots, kt, kSmall, small_stage);
    };
    // whole tiles alone
    take(cost(tiles, a.kt), big, tm, tn, tiles, 1, 0, 0);
    // the last round's tiles in pieces of the contraction, joined by a second kernel
    for (int p = 2; p <= 16 && a.kt / p >= 2 && rest; ++p) {
      const double bytes = (double)rest * p * bm * bn * 4;
      take(cost(whole, a.kt) + cost(rest * p, (int)up(a.kt, p)) + 3.0 + bytes * 2 / 8e6 / 1.85, big, tm, tn, whole, p, 0,
           rest * p * bm * bn);
    }
    if (!big) continue;
    // the rows past the last whole tile row, with or without the last round's tiles, as small ones
    const int64_t fm = a.m / bm, full = fm * tn, strip = up(a.m - fm * bm, MxTail::BM) * up(rows, MxTail::BN);
    const double tail = a.kt * 0.44 + kSmall;
    const int64_t left = full % slots;
    const double one = cost(slots, a.kt), rounds = (double)(full / slots) * one;
    // CUs without a tile in the last round take small ones meanwhile
    const int64_t beside = (slots - left) * (int64_t)(one / tail);
    if (left)
      take(rounds + one + (double)up(std::max<int64_t>(strip - beside, 0), slots) * tail, 1, fm, tn, full, 1, strip, 0);
    take(rounds + (double)up(strip + left * 4, slots) * tail, 1, fm, tn, full - left, 1, strip + left * 4, 0);
  }
}

hipError_t launch_mx_gemm(const MxGemmArgs& a, int f16, hipStream_t st) {
  return f16 ? run_mx<_Float16>(a, st) : run_mx<__bf16>(a, st);
}
hipError_t launch_mx_quantize(const MxQuantArgs& a, int f16, hipStream_t st) {
  return f16 ? run_quantize<_Float16>(a, st) : run_quantize<__bf16>(a, st);
}
hipError_t launch_mx_dequantize(const MxDequantArgs& a, int f16, hipStream_t st) {
  return f16 ? run_dequantize<_Float16>(a, st) : run_dequantize<__bf16>(a, st);
}

}  // namespace sage
