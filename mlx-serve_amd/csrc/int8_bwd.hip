// The gradient of an int8 product to its activations, on the matrix cores:
//   dx[m,k] = row[m] * sum over n of a[m,n] w[n,k]
// with the scaled gradients a in fp16 parts (int8_quant.hip) and the codes as exact fp16, fp32
// sums; the parts follow one another along the sum, smallest first and the banks within each. A part's
// power of two goes into the codes as they become fp16.
//
// Block: 8 waves as 2 (rows of a) x 4 (columns of w), BM x BN outputs, v_mfma_f32_16x16x32_f16 with
// D[k][m] = w[n][k] a[m][n]. A step is 64 values of n: rows of a are one cache line, the codes 64
// rows of BN bytes, both moved by LDS DMA into a ring of R stages as in int8_gemm.hip (one barrier a
// step, in its middle). The sum runs along the rows of w, so a
// fragment takes one column of eight rows: ds_read_b64_tr_b8 gives lane l of 16 column l % 16 of the
// 8 x 16 bytes that the 16 lanes point at, so w is read as it lies in memory, and no turned copy of
// it is made. Codes become fp16 in registers, five operations for four: u = code + 128 in the low
// byte of 0x64 is 1024 + u, minus 1152; an exponent of 11 less in both is 2^-11 of that, and 22 less 2^-22
// (subnormal, and exact).
//
// What bounds it: the matrix cores at the clock that the card's power allows. dx [4096,4096] of gate
// + up [14336,4096] takes 1360 us in two parts behind the gradient's pass (1440 where launches follow one another
// at once), 1.41 PFLOP/s, where a bf16 library product of 8192^3 runs at 1.25 to 1.42; MFMA instructions are
// busy 78% of the time. Measured with one part, 686 us: without an alias scope of the turned reads (read_tr8) 86
// us more, stored straight from the products' layout 13 us more. A dword of each line asked for in the L2
// ahead of the DMA, which helps short rings in int8_gemm.hip, made it 2 to 8% slower at every size and tile.
#include <algorithm>
#include <atomic>

#include "int8_stage.h"
#include "prefill_tiles.h"

namespace mi {
namespace {

using namespace i8;

constexpr int kBN_ = 64;  // values of n a step
typedef int32_t i32x2_t __attribute__((ext_vector_type(2)));

template <int BM, int BN, int R>
constexpr int lds_bytes() { return R * (BM * 128 + kBN_ * BN); }

// Swizzle of the 16-byte slots of a row of codes. A pass of 32 lanes reads one slot of 16 rows:
// rows 8e .. 8e+7 of quarters q and q + 1 (n = 16 q + 8 e + j): j and the parity of q tell them
// apart, and where a row is 128 bytes its lowest bit already does.
template <int BN>
MI_DEV int nswz(int n) {
  return BN == 256 ? (n & 7) | ((n >> 1) & 8) : ((n >> 1) & 3) | ((n >> 2) & 4);
}

// The fp16 exponent that codes come under, and what is taken off again (1152 of their unit), for part t of
// the gradients.
struct CodeUnit {
  uint32_t c, off;
  MI_DEV explicit CodeUnit(int t) : c(0x64646464u - t * 0x2C2C2C2Cu), off(0xE480E480u - t * 0x2C002C00u) {}
};
static_assert(kPartBits == 0x2C / 4, "a part's bits in fp16's exponent");

// four codes -> fp16, in order
MI_DEV u32x2_t codes_f16(uint32_t w, const CodeUnit& unit) {
  const uint32_t u = w ^ 0x80808080u;
  const f16x2_t off = __builtin_bit_cast(f16x2_t, unit.off);
  const f16x2_t a = __builtin_bit_cast(f16x2_t, perm_b32(unit.c, u, 0x04010400u)) + off;
  const f16x2_t b = __builtin_bit_cast(f16x2_t, perm_b32(unit.c, u, 0x04030402u)) + off;
  return u32x2_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

// (__restrict__ gives the read an alias scope: without one the compiler takes every LDS DMA in flight
// for a write to it and waits for all of them, vmcnt(0), each step.)
MI_DEV i32x2_t read_tr8(const unsigned char* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2_t*)p);
}

// waves a SIMD: 2 (one block a CU), 4 for the small tiles (two blocks)
constexpr int eu_waves(int bm, int bn) { return bm * bn <= 128 * 128 ? 4 : 2; }

template <int BM, int BN, int R, bool SPLIT>
__global__ void __launch_bounds__(512)
    __attribute__((amdgpu_waves_per_eu(eu_waves(BM, BN), eu_waves(BM, BN))))
int8_bwd_kernel(Int8BwdParams P) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int MT = BM / 32, NT = BN / 64;   // 16-row / 16-column tiles of a wave
  constexpr int XI = BM / 64, WI = BN / 128;  // DMA instructions of a wave a step
  constexpr int kStage = BM * 128 + kBN_ * BN, kW = BM * 128;
  constexpr int kRI = 1024 / BN;              // rows of w an instruction moves
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int fr = lane & 15, q = lane >> 4;
  const int M = P.M, N = P.N, K = P.K, ldw = P.ldw, np = P.np;
  const int mtiles = (M + BM - 1) / BM;
  const TileOf at = tile_of_block(mtiles, P.ct1 - P.ct0);
  const int m0 = at.mt * BM, k0 = (P.ct0 + at.nt) * BN, s0 = at.split * P.sps;
  const int seg_steps = np / kBN_;
  const int part_steps = P.banks * seg_steps;
  const int ns = min(P.sps, P.terms * part_steps - s0);
  const int mrows = min(BM, M - m0);
  const int abytes = mrows * np * 2;

  uint32_t xo[XI], wo[WI];
  int wr[WI];
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int r = 8 * (wave * XI + i) + (lane >> 3);
    xo[i] = (uint32_t)(min(r, mrows - 1) * np * 2 + 16 * ((lane & 7) ^ xswz(r)));
  }
#pragma unroll
  for (int i = 0; i < WI; ++i) {
    wr[i] = kRI * (wave * WI + i) + lane / (BN / 16);
    const int c = 16 * ((lane % (BN / 16)) ^ nswz<BN>(wr[i]));
    wo[i] = k0 + c < ldw ? (uint32_t)wr[i] * (uint32_t)ldw + (uint32_t)(k0 + c) : kOOB;
  }
  // where a stage reads: bank and part `seg`, values n .. n + 63 of it
  struct Cursor {
    int st, seg, n;
  };
  auto start = [&](int st) {
    const int g = s0 + st;
    return Cursor{st, g / seg_steps, g % seg_steps * kBN_};
  };
  auto step = [&](Cursor& c) __attribute__((always_inline)) {
    ++c.st;
    c.n += kBN_;
    if (c.n >= np) {
      c.n = 0;
      ++c.seg;
    }
  };
  auto abase = [&](const Cursor& c) { return P.a + ((size_t)c.seg * M + m0) * np; };
  auto wbase = [&](const Cursor& c) { return P.w[c.seg & (P.banks - 1)] + (size_t)c.n * ldw; };
  // stages past the range load through resources of zero records (zeros, no traffic), rows from N
  // on and columns from K on out of bounds
  auto issue = [&](const Cursor& c, int slot, int j) __attribute__((always_inline)) {  // instruction j
    const bool on = c.st < ns;
    unsigned char* b = smem + slot * kStage;
    if (j < XI) {
      dma16(rsrc(abase(c), on ? abytes : 0), b + (wave * XI + j) * 1024, xo[j], c.n * 2);
    } else {
      const int i = j - XI, rows = min(kBN_, N - c.n);
      dma16(rsrc(wbase(c), on ? rows * ldw : 0), b + kW + (wave * WI + i) * 1024, wr[i] < rows ? wo[i] : kOOB, 0);
    }
  };
  f32x4_t acc[NT][MT];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[a][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  u32x4_t X[2][MT], Wf[2];  // Wf: the codes of one tile as fp16, and the next one's
  i32x2_t A[2][NT];
  // half e: values n = 16 q + 8 e .. + 7 of both operands (slot 2q + e of a row of a)
  const int fo0 = fr * 128 + (((2 * q) ^ xswz(fr)) << 4), fo1 = fr * 128 + (((2 * q + 1) ^ xswz(fr)) << 4);
  const int xr = 16 * wm * MT * 128;
  const int nr = 16 * q + (fr >> 1);  // row of w in half 0; half 1 is 8 rows on, same swizzle
  int ao[NT];
#pragma unroll
  for (int a = 0; a < NT; ++a) ao[a] = kW + nr * BN + (((wn * NT + a) ^ nswz<BN>(nr)) << 4) + 8 * (fr & 1);
  auto read_a = [&](int slot, int e) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < NT; ++a) A[e][a] = read_tr8(smem + slot * kStage + ao[a] + e * 8 * BN);
  };
  auto read_x = [&](int slot, int e, int i) __attribute__((always_inline)) {
    X[e][i] = *reinterpret_cast<const u32x4_t*>(smem + slot * kStage + xr + (e ? fo1 : fo0) + 16 * i * 128);
  };
  auto to_f16 = [&](int e, int a, const CodeUnit& u) -> u32x4_t {
    const u32x2_t lo = codes_f16((uint32_t)A[e][a].x, u), hi = codes_f16((uint32_t)A[e][a].y, u);
    return u32x4_t{lo.x, lo.y, hi.x, hi.y};
  };
  // The products of half e, one tile of codes at a time. Beside a tile's MFMAs: the next tile's
  // codes to fp16, and a part of the next half's fragment reads (its codes first: the last tile's
  // neighbour is their first) from stage `rs`, and of the DMA where `dma`. Codes of this stage in unit
  // `u`, of the next half's in `un`.
  auto half = [&](int e, int rs, bool dma, const Cursor& c, int slot, const CodeUnit& u, const CodeUnit& un)
                  __attribute__((always_inline)) {
    constexpr int kX = NT > 1 ? (MT + NT - 2) / (NT - 1) : MT;  // x reads of the tiles after the first
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      if (a == 0) read_a(rs, e ^ 1);
#pragma unroll
      for (int i = 0; i < kX; ++i)
        if (a > 0 && (a - 1) * kX + i < MT) read_x(rs, e ^ 1, (a - 1) * kX + i);
      if (dma) {
#pragma unroll
        for (int j = a; j < XI + WI; j += NT) issue(c, slot, j);
      }
      Wf[(a + 1) & 1] = a + 1 < NT ? to_f16(e, a + 1, u) : to_f16(e ^ 1, 0, un);
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[a][i] = mfma_f16(Wf[a & 1], X[e][i], acc[a][i]);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
        if (i % 4 == 1) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  static_assert(NT % 2 == 0, "a half ends on the tile buffer it began on");

  Cursor ci = start(0);
#pragma unroll
  for (int s = 0; s < R; ++s) {
#pragma unroll
    for (int j = 0; j < XI + WI; ++j) issue(ci, s, j);
    step(ci);
    __builtin_amdgcn_sched_barrier(0);
  }
  wait_vm((R - 1) * (XI + WI));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  read_a(0, 0);
#pragma unroll
  for (int i = 0; i < MT; ++i) read_x(0, 0, i);
  const int order = s0 / part_steps;                // parts before this range's first
  int end = (order + 1) * part_steps - s0;          // of its steps
  CodeUnit unit(P.terms - 1 - order);
  Wf[0] = to_f16(0, 0, unit);
  int slot = 0;
#pragma unroll 1
  for (int t = 0; t < ns; ++t) {
    const int next = slot + 1 == R ? 0 : slot + 1;
    CodeUnit ahead = unit;  // the next step's
    if (t + 1 == end) {
      ahead.c += 0x2C2C2C2Cu;
      ahead.off += 0x2C002C00u;
      end += part_steps;
    }
    half(0, slot, false, ci, slot, unit, unit);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave's reads of stage t
    wait_vm((R - 2) * (XI + WI));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    half(1, next, true, ci, slot, unit, ahead);
    unit = ahead;
    step(ci);
    slot = next;
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // no DMA may outlive the block

  // acc[a][i] register j is [k = 16 (wn NT + a) + 4q + j][m = 16 (wm MT + i) + fr]
  const int mw = m0 + 16 * wm * MT + fr, kw = k0 + 16 * wn * NT + 4 * q;
  if constexpr (SPLIT) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int a = 0; a < NT; ++a)
        if (mw + 16 * i < M && kw + 16 * a < ldw)
          *reinterpret_cast<f32x4_t*>(P.part + ((size_t)at.split * M + mw + 16 * i) * ldw + kw + 16 * a) = acc[a][i];
    return;
  }
  float row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) row[i] = P.row[min(mw + 16 * i, M - 1)];
  auto values = [&](int i, int a, float (&v)[1][4]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[0][j] = acc[a][i][j] * row[i];
  };
  void* const out[1] = {P.dx};
  if (P.vec16 && P.type == kF32) {
    store_tile<4, MT, NT, 1, lds_bytes<BM, BN, R>()>(smem, out, P.type, M, K, m0, k0, values);
  } else if (P.vec16) {
    store_tile<2, MT, NT, 1, lds_bytes<BM, BN, R>()>(smem, out, P.type, M, K, m0, k0, values);
  } else {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int a = 0; a < NT; ++a) {
        float v[1][4];
        values(i, a, v);
        if (mw + 16 * i < M && kw + 16 * a < K)
          store4(P.dx, (int64_t)(mw + 16 * i) * K + kw + 16 * a, P.type, P.vec, K - kw - 16 * a, v[0]);
      }
  }
}

// The ranges' sums, added in their order.
__global__ void __launch_bounds__(256) int8_bwd_reduce_kernel(Int8BwdParams P) {
  const int64_t l4 = P.ldw / 4, total = l4 * P.M;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / l4;
    const int k = (int)(i - m * l4) * 4;
    if (k >= P.K) continue;
    const f32x4_t* p = reinterpret_cast<const f32x4_t*>(P.part) + i;
    const f32x4_t v = add_splits<8>(p[0], p, total, 1, P.ks);
    const float row = P.row[m];
    const float o[4] = {v[0] * row, v[1] * row, v[2] * row, v[3] * row};
    store4(P.dx, m * P.K + k, P.type, P.vec, P.K - k, o);
  }
}

template <int BM, int BN, int R>
hipError_t launch_tile(const Int8BwdParams& P, hipStream_t s) {
  constexpr int lds = lds_bytes<BM, BN, R>();
  static std::atomic<uint64_t> done{0};  // devices whose functions have the attribute
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (e == hipSuccess && !(done.load() & bit)) {
    for (auto k : {int8_bwd_kernel<BM, BN, R, false>, int8_bwd_kernel<BM, BN, R, true>})
      if (e == hipSuccess)
        e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e == hipSuccess) done |= bit;
  }
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)(((P.M + BM - 1) / BM) * (P.ct1 - P.ct0)), (unsigned)P.ks);
  if (P.ks > 1)
    hipLaunchKernelGGL((int8_bwd_kernel<BM, BN, R, true>), grid, dim3(512), lds, s, P);
  else
    hipLaunchKernelGGL((int8_bwd_kernel<BM, BN, R, false>), grid, dim3(512), lds, s, P);
  return hipGetLastError();
}

}  // namespace

// As int8_gemm_plan. Measured, bf16, us with the gradient's own pass, 256x256 / 128x256 / 128x128 / 64x128 tiles:
//   dx [M,4096], sum of 4096   128 rows 36 / 31 / 27 / 31   300 50 / 44 / 47 / 49   1024 82 / 84 / 94 / 113
//                             2048 rows 134 / 138 / 155 / 209
//   dx [M,14336], sum of 4096  300 rows 118 / 116 / 125 / 148   1024 191 / 247 / 275 / 359   2048 376 / 486 / 497 / 688
//   dx [M,4096], gate + up sums of 14336   512 rows 231 / 261 / 291 / 389   4096 1535 / 1992 / 2207 / 3005
// and as planned 28, 44, 84, 138; 117, 191, 375; 228, 1529. 64x128 tiles last for fewer rows and shorter sums.
void int8_bwd_plan(Int8BwdParams& P) {
  const int steps = P.banks * P.terms * (P.np / kBN_);
  constexpr TileCost kTiles[] = {
      {256, 256, 1.47, 0.0, 8.0}, {128, 256, 0.92, 0.0, 4.0}, {128, 128, 0.64, 1.07, 3.0}, {64, 128, 0.5, 0.8, 3.0}};
  double best = 1e30;
  for (const TileCost& t : kTiles) {
    const int64_t tiles = (int64_t)((P.M + t.bm - 1) / t.bm) * ((P.K + t.bn - 1) / t.bn);
    for (int k = 1; k <= std::max(1, steps / 4) && k <= 64; ++k) {
      const int sps = (steps + k - 1) / k, ks = (steps + sps - 1) / sps;
      const double part = ks > 1 ? (double)ks * P.M * P.K * 8 / 4.2e6 + 3.0 : 0.0;
      double cost = tile_us(t, tiles * ks, sps) + part;
      const int tail = t.bm == 256 && ks == 1 ? tail_columns(t, kTiles[1], P.M, (P.K + 255) / 256, steps, &cost) : 0;
      if (cost < best - 1e-9) {
        best = cost;
        P.bm = t.bm;
        P.bn = t.bn;
        P.ks = ks;
        P.sps = sps;
        P.tail = tail;
      }
    }
  }
}

hipError_t launch_int8_bwd(const Int8BwdParams& given, hipStream_t s) {
  Int8BwdParams P = given;
  const int ct = (P.K + P.bn - 1) / P.bn;
  P.ct0 = 0;
  P.ct1 = ct - P.tail;
  hipError_t e = P.bm == 256   ? launch_tile<256, 256, 3>(P, s)
                 : P.bm == 128 ? (P.bn == 256 ? launch_tile<128, 256, 4>(P, s) : launch_tile<128, 128, 3>(P, s))
                               : launch_tile<64, 128, 4>(P, s);
  if (e == hipSuccess && P.tail) {
    P.ct0 = P.ct1;
    P.ct1 = ct;
    e = launch_tile<128, 256, 4>(P, s);
  }
  if (e != hipSuccess || P.ks == 1) return e;
  int64_t g = ((int64_t)P.M * P.ldw / 4 + 255) / 256;
  if (g > 8192) g = 8192;
  hipLaunchKernelGGL(int8_bwd_reduce_kernel, dim3((unsigned)g), dim3(256), 0, s, P);
  return hipGetLastError();
}

}  // namespace mi
