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
#include "sage_tile.h"

namespace sage {

namespace {

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
// TWO: A in two parts (GemmArgs::half); TO: the output's type, where it is not the operands'.
template <typename T, bool AK, bool BKC, typename TL, typename TO = T, bool TWO = false>
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
  // the loads FIRST .. + COUNT - 1 of stage kt
  auto issue_a = [&](auto first, auto count, uint8_t* to, int kt) {
    const int64_t k0 = (int64_t)kt * kBK;
    if constexpr (TWO) {
      const int64_t in = k0 < a.half ? k0 : k0 - a.half, part = k0 < a.half ? 0 : a.plane;
      A.template issue<decltype(first)::value, decltype(count)::value>(to, part + in, part + (k0 < end ? a.k : in), wave);
    } else {
      A.template issue<decltype(first)::value, decltype(count)::value>(to, k0, ka, wave);
    }
  };
  auto issue_b = [&](auto first, auto count, uint8_t* to, int kt) {
    const int64_t k0 = (int64_t)kt * kBK;
    if constexpr (TWO) {
      const int64_t in = k0 < a.half ? k0 : k0 - a.half;
      B.template issue<decltype(first)::value, decltype(count)::value>(to, in, k0 < end ? a.kv : in, wave);
    } else {
      B.template issue<decltype(first)::value, decltype(count)::value>(to, k0, kb, wave);
    }
  };
  const std::integral_constant<int, 0> none;
  const std::integral_constant<int, H> some;
  const std::integral_constant<int, 2 * H> all;
  uint8_t* const lb = lds + TL::B_AT;
  issue_a(none, all, lds, kt0);
  issue_b(none, all, lb, kt0);
  issue_a(none, all, lds + TL::A_BYTES, kt0 + 1);
  issue_b(none, some, lb + TL::B_BYTES, kt0 + 1);
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
    issue_b(some, some, lb + (b0 ^ TL::B_BYTES), kt + 1);
    order();
    read(sa, sb, 2, 0);
    products(1);
    issue_a(none, some, lds + a2, kt + 2);
    order();
    read(sa, sb, 3, 1);
    products(0);
    issue_a(some, some, lds + a2, kt + 2);
    order();
    wait_loads<2 * H>();
    barrier();
    a2 = a0;
    a0 = a0 == 2 * TL::A_BYTES ? 0 : a0 + TL::A_BYTES;
    b0 ^= TL::B_BYTES;
    read(lds + a0, lb + b0, 0, 0);
    products(1);
    issue_b(none, some, sb, kt + 2);
    order();
  }
  wait_vmem();  // the loads in flight write this workgroup's LDS
  if (cut) {
    store_piece(a.part + ((int64_t)(t - a.whole) * a.parts + piece) * (TL::BM * TL::BN), wave, lane, acc);
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
      finish_any_act<TO, AK && BKC, TL::MI>(a, mine, lane, mw, nw);
      return;
    }
  }
  if constexpr (AK && BKC)
    finish<TO>(a, lane, mw, nw, acc);
  else
    finish_wave<TO, kActNone, true>(a, lane, mw, nw, acc);
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
// TWO: dz as two bf16 matrices, the rounded value and the rounded rest, for a product that takes both
// (the MXFP4 layer's dx): 2^-17 of a value is lost, none leaves fp16's range, and dx has its own
// rounding alone (fp16 2.1e-4 of its norm).  The product doubles: a training step of the MXFP4 gelu of
// 4416 x 3840 onto 10240 takes 822 us where one part takes 533, of the swiglu 1625 where 1035.
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

template <typename T, int ACT, bool VEC, bool TWO>
__global__ __launch_bounds__(256) void dact_kernel(DactArgs a) {
  constexpr bool kGlu = ACT == kActSwiglu;
  constexpr int kRows = ACT == kActNone ? 8 : 4;
  using D = std::conditional_t<TWO, __bf16, T>;
  // value j of dz, and of its second part
  auto put = [](Eight<D, VEC>& to, Eight<D, VEC>& rest, int j, float g) {
    to.v[j] = (D)g;
    if constexpr (TWO) rest.v[j] = (D)(fabsf((float)to.v[j]) < INFINITY ? g - (float)to.v[j] : 0.0f);
  };
  __shared__ float sum[kGlu ? 2 : 1][4][512];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = blockIdx.x * 512, wide = kGlu ? 2 * a.n : a.n;
  const int64_t r0 = (int64_t)blockIdx.y * a.chunk, r1 = r0 + a.chunk < a.m ? r0 + a.chunk : a.m;
  float s1[8] = {}, s2[8] = {};
  for (int64_t m0 = r0 + wave; m0 < r1; m0 += 4 * kRows) {
    Eight<T, VEC> d[kRows];
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
      Eight<D, VEC> dz, up, dz_rest, up_rest;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float g = (float)d[u].v[j];
        if constexpr (kGlu) {
          const float zz = z[u].v[j], h = g * act_fwd(ACT, zz);
          g = g * z2[u].v[j] * act_grad(ACT, zz);
          put(up, up_rest, j, h);
          s2[j] += h;
        } else if constexpr (ACT != kActNone) {
          g *= act_grad(ACT, z[u].v[j]);
        }
        put(dz, dz_rest, j, g);
        s1[j] += g;
      }
      if (a.dz && m < r1) {
        D* row = static_cast<D*>(a.dz) + m * a.ldz;
        // the last columns of a row go up to its end
        dz.store(row, n, kGlu ? a.n : (int)a.ldz, lane);
        if constexpr (kGlu) up.store(row + a.n, n, (int)a.ldz - a.n, lane);
        if constexpr (TWO) {
          row += a.plane;
          dz_rest.store(row, n, kGlu ? a.n : (int)a.ldz, lane);
          if constexpr (kGlu) up_rest.store(row + a.n, n, (int)a.ldz - a.n, lane);
        }
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

template <typename T, bool AK, bool BKC, typename TL, typename TO = T, bool TWO = false>
hipError_t run_tiles(const GemmArgs& a, hipStream_t st) {
  const int tiles = a.tm * a.tn, rest = tiles - a.whole;
  gemm_kernel<T, AK, BKC, TL, TO, TWO><<<a.whole + rest * a.parts, TL::NT, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || rest == 0) return e;
  join_kernel<TO, TL><<<rest * (TL::WAVES * TL::MI * TL::NI / 2) / 4, 256, 0, st>>>(a);
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
  if (a.half)
    return a.big ? run_tiles<__bf16, true, false, Big, T, true>(a, st) : run_tiles<__bf16, true, false, Small, T, true>(a, st);
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
  a.kt = (int)(a.half ? 2 * a.half / kBK : (a.k + kBK - 1) / kBK);
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

template <typename T, bool VEC, bool TWO>
void run_act(const DactArgs& a, dim3 grid, hipStream_t st) {
  if (a.act == kActSwiglu) dact_kernel<T, kActSwiglu, VEC, TWO><<<grid, 256, 0, st>>>(a);
  else if (a.act == kActSilu) dact_kernel<T, kActSilu, VEC, TWO><<<grid, 256, 0, st>>>(a);
  else dact_kernel<T, kActGelu, VEC, TWO><<<grid, 256, 0, st>>>(a);
}

template <typename T, bool VEC>
void run_dact(const DactArgs& a, dim3 grid, hipStream_t st) {
  if (a.act == kActNone) dact_kernel<T, kActNone, VEC, false><<<grid, 256, 0, st>>>(a);
  else if (a.plane) run_act<T, VEC, true>(a, grid, st);
  else run_act<T, VEC, false>(a, grid, st);
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
