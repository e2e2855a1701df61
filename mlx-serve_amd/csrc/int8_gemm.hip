// Int8 products of more than a few rows, on the matrix cores:
//   acc[m,n] = sum_k x[m,k] w[n,k] (int32, exact), scaled as it is written (int8.h), or for two
//   banks of weights y = silu(gate) * up of the two sums, which meet in the same lane.
//
// Block: 8 waves as 2 (rows of x) x 4 (rows of w), BM x BN outputs, v_mfma_i32_16x16x64_i8 with
// D[n][m] = w[n][k] x[m][k]. With two banks the 16-row tiles of w alternate gate, up. A step is
// 128 codes of K: a row of either operand is one cache line, moved by LDS DMA (16 bytes a lane,
// slots XOR-swizzled by row) into a ring of R stages, and read as fragments half a step ahead
// of the products that take them. Each half step's products (MT x NT of them a wave) carry the
// LDS reads of the next half and the DMA; one barrier a step, in its middle: every wave is past
// its last read of stage t (it sits in registers), so the DMA of stage t + R may go out into it,
// and stage t + 1 has landed. Vector memory operations return in order, so "landed" is an
// exact vmcnt.
//
// What bounds it: large products the matrix cores and the DMA beside them at the clock that the card's
// power allows: 8192 x 4096 x 14336 in 360 to 370 us among other calls, 2.6 POPS (395 to 415 where launches
// follow one another at once), MFMA instructions busy 66% of the time. In turn with it and on the same codes
// a library product to int32, without the scales, took 382 to 391. 64-byte steps in a ring of five stages took
// 444 us against 361 to 377, weights straight into registers 455, four waves of 128 x 128 each (a third
// less read from LDS, one wave a SIMD) 444, 32 x 32 x 32 instructions 410. Up to 256 rows or so the weights
// from HBM bound it: gate + up [14336,4096], 48 rows, 25.9 us (4.5 TB/s; graphs over more weights than the
// last-level cache holds). Two things keep them coming:
// - Rows of a power-of-two pitch meet in the same memory channels. Up to 256 rows a column tile starts
//   3 steps further along K than the one before it and wraps round (int32 sums, exact in any
//   order): 25.9 us against 30.6 there. With more rows tiles share lines in the L2 by reading them
//   at the same time, and it costs up to 2%.
// - A ring of two stages is short for weights from HBM: where all blocks run in one round (AHEAD), each
//   asks the L2 for its lines two steps before it moves them (one dword a line, into a corner of
//   LDS that nothing reads; the blocks of a panel that share a tile of x or w, prefill_tiles.h,
//   each for a part): gate + up 512 rows 59 us against 65, 128 rows 35 against 40. With more rounds
//   (8192 rows 361 / 371) and with three stages (25.9 / 31) it costs time: a line then comes in parts.
//
// K: any multiple of 16. In the last step the slots from K on load out of bounds, as zeros.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "int8_stage.h"
#include "prefill_tiles.h"

namespace mi {
namespace {

using namespace i8;
constexpr int kBK = 128;
constexpr int kStagger = 3;  // steps; 2, 5, 8, 11 and 13 are within 2% of it, 16 (2 KB) is 45% slower

template <int BM, int BN, int R>
constexpr int lds_bytes() { return R * (BM + BN) * kBK + 2048; }

// waves a SIMD: 2 (one block a CU), 4 for the small tiles (two blocks, whose starts and ends overlap)
constexpr int eu_waves(int bm, int bn) { return bm * bn <= 128 * 128 ? 4 : 2; }

template <bool DUAL, int BM, int BN, int R, bool SPLIT, bool AHEAD>
__global__ void __launch_bounds__(512)
    __attribute__((amdgpu_waves_per_eu(eu_waves(BM, BN), eu_waves(BM, BN))))
int8_gemm_kernel(Int8Params P) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int MT = BM / 32, NT = BN / 64;    // 16-row tiles of a wave
  constexpr int XI = BM / 64, WI = BN / 64;    // DMA instructions (8 rows) of a wave a step
  constexpr int kStage = (BM + BN) * kBK, kW = BM * kBK;
  constexpr int kON = DUAL ? BN / 2 : BN;      // columns of y
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int fr = lane & 15, q = lane >> 4;
  const int M = P.M, N = P.N, K = P.K, ldx = (int)P.ldx;
  const int mtiles = (M + BM - 1) / BM;
  const TileOf at = tile_of_block(mtiles, P.ct1 - P.ct0);
  const int m0 = at.mt * BM, n0 = (P.ct0 + at.nt) * kON, s0 = at.split * P.sps;
  const int ns = min(P.sps, (K + kBK - 1) / kBK - s0);
  const int mrows = min(BM, M - m0), nrows = min(kON, N - n0);
  const int xbytes = mrows * ldx, wbytes = nrows * K;
  const int8_t* xb = P.x + (size_t)m0 * ldx;
  const int8_t* wb = P.w + (size_t)n0 * K;
  const int8_t* wb2 = DUAL ? P.w2 + (size_t)n0 * K : wb;

  uint32_t xo[XI], wo[WI];
  int xc[XI], wc[WI];
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int r = 8 * (wave * XI + i) + (lane >> 3);
    xc[i] = 16 * ((lane & 7) ^ xswz(r));
    xo[i] = r < mrows ? (uint32_t)(r * ldx + xc[i]) : kOOB;
  }
#pragma unroll
  for (int i = 0; i < WI; ++i) {
    const int r = 8 * (wave * WI + i) + (lane >> 3);
    const int row = DUAL ? 16 * (r >> 5) + (r & 15) : r;  // tiles alternate gate, up
    wc[i] = 16 * ((lane & 7) ^ xswz(r));
    wo[i] = row < nrows ? (uint32_t)row * (uint32_t)K + wc[i] : kOOB;
  }
  // stages past the range load through a resource of zero records (zeros, no traffic)
  const int first = M <= 256 ? at.nt * kStagger % ns : 0;
  auto place = [&](int st) __attribute__((always_inline)) {  // of step st along K
    return (s0 + st + (st + first < ns ? first : first - ns)) * kBK;
  };
  auto issue = [&](int st, int slot) __attribute__((always_inline)) {
    const bool on = st < ns;
    const int k = place(st);
    unsigned char* b = smem + slot * kStage;
#pragma unroll
    for (int i = 0; i < XI; ++i)
      dma16(rsrc(xb, on ? xbytes : 0), b + (wave * XI + i) * 1024, xc[i] < K - k ? xo[i] : kOOB, k);
#pragma unroll
    for (int i = 0; i < WI; ++i)
      dma16(rsrc(DUAL && ((wave * WI + i) >> 1 & 1) ? wb2 : wb, on ? wbytes : 0),
            b + kW + (wave * WI + i) * 1024, wc[i] < K - k ? wo[i] : kOOB, k);
  };
  // L2 prefetch: waves 0-3 the rows of x, 4-7 those of w (4, 5 gate and 6, 7 up), 64 a wave. The h
  // blocks of a panel that read this w tile split its rows, four of those that read x its.
  constexpr int PF = AHEAD ? 1 : 0;  // instructions a step
  const int h = min(4, mtiles - at.mt / 4 * 4);
  const bool pw = wave >= 4;
  const int8_t* pb = !pw ? xb : DUAL && (wave & 2) ? wb2 : wb;
  const int pr = (wave & (DUAL && pw ? 1 : 3)) * 64 + lane, pn = pw ? min(kON, nrows) : min(BM, mrows);
  const bool mine = pr < pn && (pw ? at.mt % h == (wave & 3) % h : (at.nt & 3) == (wave & 3));
  const uint32_t po = mine ? (uint32_t)pr * (uint32_t)(pw ? K : ldx) : kOOB;
  auto prefetch = [&](int st) __attribute__((always_inline)) {
    if constexpr (PF)
      dma4(rsrc(pb, st < ns ? (pw ? wbytes : xbytes) : 0), smem + R * kStage + wave * 256, po, place(st));
  };

  i32x4_t acc[NT][MT];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[a][i] = i32x4_t{0, 0, 0, 0};
  u32x4_t X[2][MT], A[2][NT];
  // half e of a step: slot 2q + e of a row (both operands take the same 64 codes)
  const int fo0 = fr * kBK + (((2 * q) ^ xswz(fr)) << 4), fo1 = fr * kBK + (((2 * q + 1) ^ xswz(fr)) << 4);
  const int xr = 16 * wm * MT * kBK, wr = kW + 16 * wn * NT * kBK;
  auto frags = [&](int slot, int e) __attribute__((always_inline)) {
    const unsigned char* b = smem + slot * kStage + (e ? fo1 : fo0);
#pragma unroll
    for (int i = 0; i < MT; ++i) X[e][i] = *reinterpret_cast<const u32x4_t*>(b + xr + 16 * i * kBK);
#pragma unroll
    for (int a = 0; a < NT; ++a) A[e][a] = *reinterpret_cast<const u32x4_t*>(b + wr + 16 * a * kBK);
  };
  auto products = [&](int e) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int a = 0; a < NT; ++a) acc[a][i] = mfma_i8(A[e][a], X[e][i], acc[a][i]);
  };

#pragma unroll
  for (int s = 0; s < R; ++s) {
    issue(s, s);
    prefetch(s + R);
    __builtin_amdgcn_sched_barrier(0);
  }
  wait_vm(PF + (R - 1) * (XI + WI + PF));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  frags(0, 0);
  int slot = 0;
#pragma unroll 1
  for (int t = 0; t < ns; ++t) {
    const int next = R == 2 ? slot ^ 1 : slot + 1 == R ? 0 : slot + 1;
    frags(slot, 1);
    products(0);
#pragma unroll
    for (int r = 0; r < MT + NT; ++r) {  // a read, one or two products
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      if (MT * NT >= 2 * (MT + NT)) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave's reads of stage t
    wait_vm(PF + (R - 2) * (XI + WI + PF));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    frags(next, 0);
    issue(t + R, slot);
    prefetch(t + 2 * R);
    products(1);
#pragma unroll
    for (int r = 0; r < MT + NT; ++r) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      if (MT * NT >= 2 * (MT + NT)) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (r % 3 != 2) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    slot = next;
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // no DMA may outlive the block

  // acc[a][i] register j is [n = 16 (wn NT + a) + 4q + j][m = 16 (wm MT + i) + fr]
  constexpr int TA = DUAL ? NT / 2 : NT;  // 16-column tiles of y
  const int mw = m0 + 16 * wm * MT + fr, nw = n0 + 16 * wn * TA + 4 * q;
  if constexpr (SPLIT) {
#pragma unroll
    for (int a = 0; a < TA; ++a)
#pragma unroll
      for (int i = 0; i < MT; ++i)
        if (nw + 16 * a < N && mw + 16 * i < M)
          store_part<DUAL>(P, at.split, mw + 16 * i, nw + 16 * a, acc[DUAL ? 2 * a : a][i], acc[DUAL ? 2 * a + 1 : a][i]);
    return;
  }
  float sx[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) sx[i] = P.sx[min(mw + 16 * i, M - 1)];
  Cols cols[TA];
#pragma unroll
  for (int a = 0; a < TA; ++a) cols[a] = load_cols<DUAL>(P, min(nw + 16 * a, N - 1));
  if (P.vec16) {
    auto emit = [&](auto esz) __attribute__((always_inline)) {
      constexpr int E = decltype(esz)::value;
      auto values = [&](int i, int a, float (&y)[4], float (&g)[4], float (&u)[4]) __attribute__((always_inline)) {
        scaled4<DUAL>(P, acc[DUAL ? 2 * a : a][i], acc[DUAL ? 2 * a + 1 : a][i], sx[i], cols[a], y, g, u);
      };
      if constexpr (DUAL) {
        if (P.gate) {
          void* const out[3] = {P.y, P.gate, P.up};
          store_tile<E, MT, TA, 3, lds_bytes<BM, BN, R>()>(
              smem, out, P.type, M, N, m0, n0,
              [&](int i, int a, float (&v)[3][4]) __attribute__((always_inline)) { values(i, a, v[0], v[1], v[2]); });
          return;
        }
      }
      void* const out[1] = {P.y};
      store_tile<E, MT, TA, 1, lds_bytes<BM, BN, R>()>(
          smem, out, P.type, M, N, m0, n0, [&](int i, int a, float (&v)[1][4]) __attribute__((always_inline)) {
            float g[4], u[4];
            values(i, a, v[0], g, u);
          });
    };
    if (P.type == kF32)
      emit(std::integral_constant<int, 4>{});
    else
      emit(std::integral_constant<int, 2>{});
    return;
  }
#pragma unroll
  for (int a = 0; a < TA; ++a)
#pragma unroll
    for (int i = 0; i < MT; ++i)
      if (nw + 16 * a < N && mw + 16 * i < M)
        finish4<DUAL>(P, mw + 16 * i, nw + 16 * a, acc[DUAL ? 2 * a : a][i], acc[DUAL ? 2 * a + 1 : a][i], sx[i], cols[a]);
}

// The splits' sums, exact in any order, and the scales. (Loads of 8 splits go out before their adds.)
template <bool DUAL>
__global__ void __launch_bounds__(256) int8_reduce_kernel(Int8Params P) {
  constexpr int B = DUAL ? 2 : 1;
  const int64_t n4 = ((int64_t)P.N + 3) / 4, total = n4 * P.M, mn = (int64_t)P.M * P.N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / n4;
    const int n = (int)(i - m * n4) * 4;
    const float sx = P.sx[m];
    const Cols cols = load_cols<DUAL>(P, n);
    i32x4_t v[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int32_t* p = P.part + b * mn + m * P.N + n;
      if (P.N % 4 == 0) {
        v[b] = add_splits<8>(v[b], reinterpret_cast<const i32x4_t*>(p), B * mn / 4, 0, P.ks);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < P.N) v[b][j] = add_splits<8>((int32_t)0, p + j, B * mn, 0, P.ks);
      }
    }
    finish4<DUAL>(P, m, n, v[0], v[1], sx, cols);
  }
}

template <bool DUAL, int BM, int BN, int R, bool SPLIT, bool AHEAD>
hipError_t launch_kernel(const Int8Params& P, dim3 grid, hipStream_t s) {
  constexpr int lds = lds_bytes<BM, BN, R>();
  const auto kernel = int8_gemm_kernel<DUAL, BM, BN, R, SPLIT, AHEAD>;
  static std::atomic<uint64_t> done{0};  // devices whose function has the attribute
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (e == hipSuccess && !(done.load() & bit)) {
    e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e == hipSuccess) done |= bit;
  }
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, grid, dim3(512), lds, s, P);
  return hipGetLastError();
}

template <bool DUAL, int BM, int BN, int R>
hipError_t launch_tile(const Int8Params& P, hipStream_t s) {
  const dim3 grid((unsigned)(((P.M + BM - 1) / BM) * (P.ct1 - P.ct0)), (unsigned)P.ks);
  const bool split = P.ks > 1;
  if constexpr (R == 2) {
    if ((uint64_t)grid.x * grid.y <= 256)
      return split ? launch_kernel<DUAL, BM, BN, R, true, true>(P, grid, s)
                   : launch_kernel<DUAL, BM, BN, R, false, true>(P, grid, s);
  }
  return split ? launch_kernel<DUAL, BM, BN, R, true, false>(P, grid, s)
               : launch_kernel<DUAL, BM, BN, R, false, false>(P, grid, s);
}

template <bool DUAL>
hipError_t launch_gemm(Int8Params P, hipStream_t s) {
  const int cols = DUAL ? P.bn / 2 : P.bn, ct = (P.N + cols - 1) / cols;
  P.ct0 = 0;
  P.ct1 = ct - P.tail;
  hipError_t e = P.bm == 256   ? launch_tile<DUAL, 256, 256, 2>(P, s)
                 : P.bm == 128 ? (P.bn == 256 ? launch_tile<DUAL, 128, 256, 3>(P, s)
                                              : launch_tile<DUAL, 128, 128, 2>(P, s))
                               : launch_tile<DUAL, 64, 128, 3>(P, s);
  if (e == hipSuccess && P.tail) {
    P.ct0 = P.ct1;
    P.ct1 = ct;
    e = launch_tile<DUAL, 128, 256, 3>(P, s);
  }
  if (e != hipSuccess || P.ks == 1) return e;
  int64_t g = ((int64_t)P.M * ((P.N + 3) / 4) + 255) / 256;
  if (g > 8192) g = 8192;
  hipLaunchKernelGGL((int8_reduce_kernel<DUAL>), dim3((unsigned)g), dim3(256), 0, s, P);
  return hipGetLastError();
}

}  // namespace

// Tile and K splits: the fewest estimated microseconds, from the blocks' steps, a split's int32
// partials written and read back with the reduce launch, and the time that the operands take
// from HBM at least. Depends on the sizes alone (not on pointers), so the workspace can be asked
// for ahead. Measured, us, with 256x256 / 128x256 / 128x128 / 64x128 tiles:
//   [14336,4096]  128 rows 33 / 28 / 29 / 22   512 55 / 39 / 44 / 56   2048 119 / 145 / 151 / 183
//   [4096,4096]   128 rows 21 / 23 / 19 / 17   512 33 / 26 / 25 / 19   2048  51 /  40 /  41 /  56
//   [4096,14336]  128 rows 34 / 29 / 28 / 27   512 53 / 45 / 54 / 61   2048 124 / 116 / 130 / 175
//   gate + up [14336,4096] 256 rows 60 / 42 / 47 / 60, 1024 122 / 141 / 156 / 183
double int8_gemm_plan(Int8Params& P) {
  const int steps = (P.K + kBK - 1) / kBK, banks = P.banks;
  constexpr TileCost kTiles[] = {
      {256, 256, 1.55, 0.0, 8.0}, {128, 256, 1.03, 0.0, 4.0}, {128, 128, 0.75, 1.13, 3.0}, {64, 128, 0.5, 0.8, 2.5}};
  double best = 1e30;
  for (const TileCost& t : kTiles) {
    const int on = t.bn / banks;
    const int64_t tiles = (int64_t)((P.M + t.bm - 1) / t.bm) * ((P.N + on - 1) / on);
    for (int k = 1; k <= std::max(1, steps / 4) && k <= 64; ++k) {
      const int sps = (steps + k - 1) / k, ks = (steps + sps - 1) / sps;
      const double part = ks > 1 ? (double)ks * banks * P.M * P.N * 8 / 5e6 + 3.0 : 0.0;
      double cost = tile_us(t, tiles * ks, sps) + part;
      const int tail = t.bm == 256 && ks == 1 ? tail_columns(t, kTiles[1], P.M, (P.N + on - 1) / on, steps, &cost) : 0;
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
  return 3.0 + std::max(best, ((double)banks * P.N + P.M) * P.K / 5e6);
}

hipError_t launch_int8_gemm(const Int8Params& P, hipStream_t s) {
  return P.w2 ? launch_gemm<true>(P, s) : launch_gemm<false>(P, s);
}

}  // namespace mi
