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

// A wave takes 512 columns of kQuantRows rows, a lane eight of each row: four lanes a block.
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

// The scales of MI blocks of 32 rows in one stage: lane (h, r) gets the four bytes of row r that
// belong to the 16-byte chunks 4 h .. 4 h + 3 of its codes; in step s of the stage it multiplies
// chunk 4 h + s with byte s.  Rows past the last read the last one's.
template <int N>
struct Scales {
  int off[N];
  const uint8_t* base;
  int64_t step;  // bytes of a stage's scales
  __device__ __forceinline__ void issue(int (&v)[N], int kt) const {
    const __amdgpu_buffer_rsrc_t rs = raw_rsrc(base + kt * step, 0x7fffffff);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (int)load_4(rs, off[i]);
  }
};

// The product by tiles, as the linear layers' gemm_kernel: three LDS stages of A and two of B,
// the next step's fragments read under this one's products.  A stage is 256 columns.  Scales go
// straight to registers, a stage ahead.
template <typename T, typename TL>
__global__ __launch_bounds__(TL::NT, TL::SIMD) void mx_gemm_kernel(MxGemmArgs x) {
  const GemmArgs& a = x.g;
  __shared__ __align__(1024) uint8_t lds[TL::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const bool glu = a.act == kActSwiglu;
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

  Operand<TL::BM, true, TL::WAVES> A;
  Operand<TL::BN, true, TL::WAVES> B;
  A.init(a.a, a.lda, m0, a.m, wave, lane, false, 0);
  B.init(a.b, a.ldb, n0, a.n, wave, lane, glu, a.n);
  const int wm = wave / TL::WN, wn = wave % TL::WN;
  const int h = lane >> 5, r = lane & 31;
  Scales<TL::MI> SA;
  Scales<TL::NI> SB;
  const int rows = glu ? 2 * a.n : a.n;
  SA.base = x.sa + m0 * 8;
  SA.step = a.m * 8;
  SB.base = x.sb;
  SB.step = (int64_t)rows * 8;
  // fragment addresses: chunk 4 h + s of row r in step s
  int fa[TL::MI][4], fb[TL::NI][4];
  auto frag_at = [&](int row, int s) { return row * 128 + (((4 * h + s) ^ ((row >> 1) & 7)) << 4); };
#pragma unroll
  for (int i = 0; i < TL::MI; ++i) {
    const int row = (wm * TL::MI + i) * 32 + r;
    SA.off[i] = (int)min((int64_t)row, a.m - 1 - m0) * 8 + 4 * h;
#pragma unroll
    for (int s = 0; s < 4; ++s) fa[i][s] = frag_at(row, s);
  }
#pragma unroll
  for (int i = 0; i < TL::NI; ++i) {
    const int row = (wn * TL::NI + i) * 32 + r;
    const int n = n0 + (glu ? (row >> 6) * 32 + r : row);
    SB.off[i] = (min(n, a.n - 1) + (glu && (row >> 5 & 1) ? a.n : 0)) * 8 + 4 * h;
#pragma unroll
    for (int s = 0; s < 4; ++s) fb[i][s] = frag_at(row, s);
  }

  f32x16 acc[TL::MI][TL::NI] = {};
  i32x4 va[2][TL::MI], vb[2][TL::NI];
  int sa[2][TL::MI], sb[2][TL::NI];
  const int64_t end = (int64_t)kt1 * kBK, ka = min(a.k, end);
  auto read = [&](const uint8_t* pa, const uint8_t* pb, int s, int to) {
#pragma unroll
    for (int i = 0; i < TL::NI; ++i) vb[to][i] = operand_at<i32x4>(pb + fb[i][s]);
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) va[to][i] = operand_at<i32x4>(pa + fa[i][s]);
  };
  auto products = [&](int from, auto step) {
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
      for (int j = 0; j < TL::NI; ++j)
        acc[i][j] = mx32<decltype(step)::value>(vb[from][j], sb[0][j], va[from][i], sa[0][i], acc[i][j]);
  };
  constexpr int H = decltype(A)::LOADS / 2;
  static_assert(H * 2 == decltype(B)::LOADS, "as many loads of A as of B");
  auto order = [&]() {
    constexpr int M = TL::MI * TL::NI, R = TL::MI + TL::NI;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      order_mfma();
      if (i < R) order_read();
      if (i % (M / H) == M / H / 2) order_load();
    }
  };
  uint8_t* const lb = lds + TL::B_AT;
  SA.issue(sa[0], kt0);
  SB.issue(sb[0], kt0);
  A.template issue<0, 2 * H>(lds, (int64_t)kt0 * kBK, ka, wave);
  B.template issue<0, 2 * H>(lb, (int64_t)kt0 * kBK, ka, wave);
  A.template issue<0, 2 * H>(lds + TL::A_BYTES, (int64_t)(kt0 + 1) * kBK, ka, wave);
  B.template issue<0, H>(lb + TL::B_BYTES, (int64_t)(kt0 + 1) * kBK, ka, wave);
  wait_loads<3 * H>();
  barrier();
  read(lds, lb, 0, 0);
  int a0 = 0, b0 = 0;        // the present stage's place
  int a2 = 2 * TL::A_BYTES;  // the place of the stage after next
  for (int kt = kt0; kt < kt1; ++kt) {
    uint8_t* const pa = lds + a0;
    uint8_t* const pb = lb + b0;
    const int next = min(kt + 1, kt1 - 1);
    SA.issue(sa[1], next);
    SB.issue(sb[1], next);
    read(pa, pb, 1, 1);
    products(0, std::integral_constant<int, 0>{});
    B.template issue<H, H>(lb + (b0 ^ TL::B_BYTES), (int64_t)(kt + 1) * kBK, ka, wave);
    order();
    read(pa, pb, 2, 0);
    products(1, std::integral_constant<int, 1>{});
    A.template issue<0, H>(lds + a2, (int64_t)(kt + 2) * kBK, ka, wave);
    order();
    read(pa, pb, 3, 1);
    products(0, std::integral_constant<int, 2>{});
    A.template issue<H, H>(lds + a2, (int64_t)(kt + 2) * kBK, ka, wave);
    order();
    wait_loads<2 * H>();
    barrier();
    a2 = a0;
    a0 = a0 == 2 * TL::A_BYTES ? 0 : a0 + TL::A_BYTES;
    b0 ^= TL::B_BYTES;
    read(lds + a0, lb + b0, 0, 0);
    products(1, std::integral_constant<int, 3>{});
    B.template issue<0, H>(pb, (int64_t)(kt + 2) * kBK, ka, wave);
    order();
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) sa[0][i] = sa[1][i];
#pragma unroll
    for (int i = 0; i < TL::NI; ++i) sb[0][i] = sb[1][i];
  }
  wait_vmem();  // the loads in flight write this workgroup's LDS
  if (cut) {
    store_piece<TL>(a, t, piece, wave, lane, acc);
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
      finish_any_act<T, true, TL::MI>(a, mine, lane, mw, nw);
      return;
    }
  }
  finish<T>(a, lane, mw, nw, acc);
}

// ---------------------------------------------------------------- few rows

constexpr int kMxSkinnyWaves = 4;

// Waits for every LDS read and for all but the last N loads.
template <int N>
__device__ __forceinline__ void wait_all_but() {
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
}

// out for at most 16 * MT rows of x, as the linear layers' skinny_kernel: a workgroup reads 16
// rows of W (of both halves for a swiglu) once, its waves take 256-column stages in turn through
// rings of LDS slots of their own, and their sums are added in order.  A slot holds, for each
// group of 16 rows, 2 KiB of codes and 128 bytes of scales.
template <typename T, int MT, bool GLU>
__global__ __launch_bounds__(64 * kMxSkinnyWaves, MT < 4 ? 2 : 1) void mx_skinny_kernel(MxGemmArgs args) {
  const GemmArgs& a = args.g;
  constexpr int H = GLU ? 2 : 1, TILES = H + MT, PART = 2048 + 128, STAGE = TILES * PART;
  constexpr int D = TILES == 2 ? 4 : TILES == 3 ? 3 : 2;
  __shared__ __align__(1024) uint8_t lds[kMxSkinnyWaves * D * STAGE];
  static_assert(sizeof(lds) <= (MT < 4 ? 80 : 160) * 1024 && H * MT * 1024 <= D * STAGE,
                "two workgroups a CU, and the sums fit");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  uint8_t* const mine = lds + wave * D * STAGE;
  const int64_t pitch = a.ldb * 2, m = a.m;  // bytes of a row of codes, the same on both sides
  const int n0 = blockIdx.x * 16, rows = GLU ? 2 * a.n : a.n;
  const __amdgpu_buffer_rsrc_t xrs = raw_rsrc(a.a, 0x7fffffff);
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
    for (int j = 0; j < MT; ++j) xoff[j][i] = (int)(min((int64_t)(16 * j + row), m - 1) * pitch) + c * 16;
  }
  // scales: lane l of the lower ones takes four bytes of row l / 2
  const int srow = lane >> 1;
  int wsoff[H], xsoff[MT];
#pragma unroll
  for (int h = 0; h < H; ++h) wsoff[h] = (min(n0 + srow, a.n - 1) + h * a.n) * 8 + 4 * (lane & 1);
#pragma unroll
  for (int j = 0; j < MT; ++j) xsoff[j] = (int)min((int64_t)(16 * j + srow), m - 1) * 8 + 4 * (lane & 1);
  auto issue = [&](uint8_t* stage, int chunk) {
    const int at = chunk * 128;
    const __amdgpu_buffer_rsrc_t wss = raw_rsrc(args.sb + (int64_t)chunk * rows * 8, (uint32_t)rows * 8);
    const __amdgpu_buffer_rsrc_t xss = raw_rsrc(args.sa + (int64_t)chunk * m * 8, (uint32_t)m * 8);
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int i = 0; i < 2; ++i) dma_16(stage + h * PART + i * 1024, wrs[h], woff[i] + at);
      if (lane < 32) __builtin_amdgcn_raw_ptr_buffer_load_lds(wss, stage + h * PART + 2048, 4, wsoff[h], 0, 0, 0);
    }
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
  f32x4 acc[H][MT] = {};
  const int chunks = a.kt;
  // wave i finishes rows 16 i .. of x: lane (q, r) columns 4 q .. + 3 of row r.  Bias and residual
  // are asked for first (zeros where there are none) and waited for last.
  const int64_t mr = 16 * wave + r;
  uint32_t bias[H][4];
  uint16_t res[4];
  if (wave < MT) {
    const __amdgpu_buffer_rsrc_t brs = raw_rsrc(a.bias, a.bias ? (uint32_t)(a.n * H) * (a.bias_f32 ? 4 : 2) : 0u);
    const __amdgpu_buffer_rsrc_t rrs = raw_rsrc(a.res, a.res ? 0x7fffffffu : 0u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + 4 * q + e, out = n < a.n && mr < m ? 0 : (int)0x80000000;
#pragma unroll
      for (int h = 0; h < H; ++h)
        bias[h][e] = a.bias_f32 ? load_4(brs, (n + h * a.n) * 4 | out) : load_2(brs, (n + h * a.n) * 2 | out);
      res[e] = load_2(rrs, (int)((mr * a.ldr + n) * 2) | out);
    }
    keep_order();
  }
#pragma unroll
  for (int d = 0; d < D - 1; ++d)
    if (wave + d * kMxSkinnyWaves < chunks) issue(mine + d * STAGE, wave + d * kMxSkinnyWaves);
  int now = 0, free = (D - 1) * STAGE;
#pragma unroll 1
  for (int c = wave; c < chunks; c += kMxSkinnyWaves) {
    // this stage has arrived, and the last one's reads are done: its place takes the next loads
    if (c + (D - 1) * kMxSkinnyWaves < chunks) {
      wait_all_but<3 * TILES * (D - 2)>();
      hold_memory();
      issue(mine + free, c + (D - 1) * kMxSkinnyWaves);
    } else {
      wait_all_but<0>();
      hold_memory();
    }
    const uint8_t* stage = mine + now;
    int ws[H], xs[MT];
#pragma unroll
    for (int h = 0; h < H; ++h) ws[h] = *reinterpret_cast<const uint16_t*>(stage + h * PART + sat);
#pragma unroll
    for (int j = 0; j < MT; ++j) xs[j] = *reinterpret_cast<const uint16_t*>(stage + (H + j) * PART + sat);
    auto step = [&](auto s) {
      constexpr int S = decltype(s)::value;
      i32x4 w[H], x[MT];
#pragma unroll
      for (int h = 0; h < H; ++h) w[h] = operand_at<i32x4>(stage + h * PART + at[S]);
#pragma unroll
      for (int j = 0; j < MT; ++j) x[j] = operand_at<i32x4>(stage + (H + j) * PART + at[S]);
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
  if (wave >= MT) return;
  f32x4 z = {}, z2 = {};
#pragma unroll
  for (int w = 0; w < kMxSkinnyWaves; ++w) {
    const f32x4* const p = reinterpret_cast<const f32x4*>(lds + w * D * STAGE) + threadIdx.x;
    z += p[0];
    if (GLU) z2 += p[(H - 1) * MT * 64];
  }
  if (mr >= m) return;
  auto bias_of = [&](uint32_t v) {
    return a.bias_f32 ? __uint_as_float(v) : (float)__builtin_bit_cast(T, (uint16_t)v);
  };
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t n = n0 + 4 * q + e;
    if (n >= a.n) continue;
    const float v = z[e] + bias_of(bias[0][e]), v2 = GLU ? z2[e] + bias_of(bias[H - 1][e]) : 1.0f;
    if (a.z) {
      float* row = a.z + mr * a.n * H;
      row[n] = v;
      if (GLU) row[a.n + n] = v2;
    }
    const float y = act_fwd(a.act, v) * v2 + (float)__builtin_bit_cast(T, res[e]);
    static_cast<T*>(a.out)[mr * a.n + n] = (T)y;
  }
}

using MxBig = Tile<2, 2, 4, 4, 1>;    // 256 x 256, 4 waves of 128 x 128, one workgroup a CU
using MxSmall = Tile<2, 2, 2, 2, 2>;  // 128 x 128, 4 waves of 64 x 64, two workgroups a CU

template <typename T, typename TL>
hipError_t run_mx_tiles(const MxGemmArgs& x, hipStream_t st) {
  const GemmArgs& a = x.g;
  const int tiles = a.tm * a.tn, rest = tiles - a.whole;
  mx_gemm_kernel<T, TL><<<a.whole + rest * a.parts, TL::NT, 0, st>>>(x);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || rest == 0) return e;
  join_kernel<T, TL><<<rest * (TL::WAVES * TL::MI * TL::NI / 2) / 4, 256, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t run_mx(const MxGemmArgs& x, hipStream_t st) {
  const GemmArgs& a = x.g;
  if (!a.skinny) return a.big ? run_mx_tiles<T, MxBig>(x, st) : run_mx_tiles<T, MxSmall>(x, st);
  const uint32_t grid = (uint32_t)((a.n + 15) / 16);
  constexpr int NT = 64 * kMxSkinnyWaves;
  if (a.act == kActSwiglu) {
    if (a.m <= 16) mx_skinny_kernel<T, 1, true><<<grid, NT, 0, st>>>(x);
    else mx_skinny_kernel<T, 2, true><<<grid, NT, 0, st>>>(x);
  } else if (a.m <= 16) mx_skinny_kernel<T, 1, false><<<grid, NT, 0, st>>>(x);
  else if (a.m <= 32) mx_skinny_kernel<T, 2, false><<<grid, NT, 0, st>>>(x);
  else if (a.m <= 48) mx_skinny_kernel<T, 3, false><<<grid, NT, 0, st>>>(x);
  else mx_skinny_kernel<T, 4, false><<<grid, NT, 0, st>>>(x);
  return hipGetLastError();
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
  a.skinny = a.m <= (glu ? 32 : 64);
  a.thin = 0;
  a.part_floats = 0;
  a.parts = 1;
  a.tm = a.tn = a.whole = 0;
  if (a.skinny) return;
  // The tile shape and the split of the last round's tiles with the least estimated time, in
  // stages of the large tile on every CU.
  double best = 1e30;
  for (int big = 1; big >= 0; --big) {
    const int bm = big ? MxBig::BM : MxSmall::BM, bn = (big ? MxBig::BN : MxSmall::BN) / (glu ? 2 : 1);
    const int64_t tm = (a.m + bm - 1) / bm, tn = (a.n + bn - 1) / bn, tiles = tm * tn;
    const int slots = big ? 256 : 512;
    const double start = big ? 7.5 : 3.6;
    for (int p = 1; p <= 16; ++p) {
      // rows that take no 16-byte accesses are finished by the small tiles themselves, and
      // with large ones by the join
      const int64_t rest = !a.vec && (big || p > 1) ? tiles : p == 1 ? 0 : tiles % slots;
      if (p > 1 && (rest == 0 || a.kt / p < 2)) continue;
      const int64_t whole = tiles - rest;
      const double stage = big ? 1.0 : tiles <= 256 && rest * p <= 256 ? 0.37 : 0.63;
      double cost = (double)((whole + slots - 1) / slots) * (a.kt * stage + start);
      if (rest) {
        const double bytes = (double)rest * p * bm * (big ? MxBig::BN : MxSmall::BN) * 4;
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
        a.part_floats = rest * p * bm * (big ? MxBig::BN : MxSmall::BN);
      }
    }
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
