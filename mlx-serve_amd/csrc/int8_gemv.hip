// Int8 products of few rows (up to 128): decode, and short prompts through small matrices. The weights are
// read once, so their bytes bound it.
//
// Block: WK waves that share 16 NT rows of w (of both banks, with two) and split K between them;
// a wave streams its part of those rows straight into registers (one instruction reads 16 rows x 64
// bytes), U chunks of 64 codes ahead, and multiplies them with up to 16 MT rows of x on
// v_mfma_i32_16x16x64_i8 (rows from M on are zeros that cost no traffic). The waves' int32 sums
// meet in LDS, exact in any order; there are no partial sums in memory and one launch.
// x comes from the L2: every block reads it whole, MT / NT times the weight bytes of its tile (halved
// by the second bank), which is why wide calls take two tiles a wave.
//
// One float token (FUSE): each block quantizes it by itself, into LDS, while its first weights are on
// their way: it is a few KB, and a launch of its own costs more (2 us and the gap before it).
//
// Measured in graphs over more weights than the last-level cache (256 MB) holds, us: [14336,4096] 1 token
// 15.7, 2 rows 14.6 (4.0 TB/s), 8 rows 17.0; [4096,14336] 14.5, 13.4 and 15.7; [4096,4096] 6.2, 5.9 and 6.4; gate + up [14336,4096] 1 token 27.5
// (4.3 TB/s), 16 rows 29. Above 16 rows the reads of x from the L2 count: [4096,4096] 16 rows 7.4,
// 64 rows 13.2. (Two chunks that share a line, 16 of each 32 bytes for either, so that the first load
// asks for the whole line, took 0.2 us off one token of [4096,4096] and put up to 1.3 us on 8 rows;
// starts of the blocks along K moved apart, as in int8_gemm.hip, cost 10 to 20%.)
#include <algorithm>
#include <atomic>
#include <cmath>

#include "int8_stage.h"

namespace mi {
namespace {

using namespace i8;

// a 16-byte vector of x's values as codes; E values
template <int T>
MI_DEV uint32_t vec_max(u32x4_t v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == kF32) {
      m = max(m, v[i] & 0x7FFFFFFFu);
    } else {
      m = max(m, max(v[i] & 0x7FFFu, (v[i] >> 16) & 0x7FFFu));
    }
  }
  return m;
}

// The token to codes in xs (K bytes, zeros up to a multiple of 64); returns its scale. Every
// thread of the block calls it; v holds vectors tid, tid + threads, ...
template <int T, int XV, int THREADS>
MI_DEV float quantize_token(const u32x4_t (&v)[XV], int K, unsigned char* xs, uint32_t* part) {
  constexpr int E = T == kF32 ? 4 : 8, W = THREADS / 64;
  const int tid = threadIdx.x;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < XV; ++i) m = max(m, vec_max<T>(v[i]));
#pragma unroll
  for (int d = 32; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
  if ((tid & 63) == 0) part[tid >> 6] = m;
  lds_sync();
#pragma unroll
  for (int i = 0; i < W; ++i) m = max(m, part[i]);
  const RowScale R = row_scale(T == kBF16  ? m << 16
                               : T == kF16 ? __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m)) & 0x7FFFFFFFu
                                           : m);
#pragma unroll
  for (int i = 0; i < XV; ++i) {
    const int c = tid + i * THREADS;
    if (c * E >= (K + 63) / 64 * 64) continue;  // (vectors from K on were loaded as zeros)
#pragma unroll
    for (int h = 0; h < E / 4; ++h) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (T == kF32) {
          f[j] = __uint_as_float(v[i][j]);
        } else {
          const uint16_t b = (uint16_t)(v[i][2 * h + j / 2] >> (16 * (j & 1)));
          f[j] = T == kBF16 ? bf16_bits_to_f32(b) : (float)__builtin_bit_cast(_Float16, b);
        }
      }
      *reinterpret_cast<uint32_t*>(xs + c * E + 4 * h) = codes4(f, R);
    }
  }
  lds_sync();
  return R.s;
}

template <bool DUAL, int MT, int NT, int WK, int U, int XV>
__global__ void __launch_bounds__(WK * 64, MT == 1 ? 8 : MT <= 4 ? 4 : 2) int8_gemv_kernel(Int8Params P) {
  constexpr int B = DUAL ? 2 : 1;
  constexpr bool FUSE = XV > 0;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, q = lane >> 4;
  const int M = P.M, N = P.N, K = P.K, ldx = (int)P.ldx;
  const int n0 = (int)blockIdx.x * 16 * NT;
  const int nrows = min(16 * NT, N - n0);
  const int chunks = (K + 63) / 64, per = (chunks + WK - 1) / WK;
  const int cb = wave * per, ce = min(chunks, cb + per);

  // this wave's part of the end: output tile wave of NT x MT (its scales come ahead of the weights)
  static_assert(NT * MT <= WK, "a wave finishes one tile");
  const int ta = wave / MT, ti = wave % MT;
  const int em = 16 * ti + fr, en = n0 + 16 * ta + 4 * q;
  const bool ends = wave < NT * MT && em < M && en < N;
  Cols cols = {};
  float sx = 0.f;
  if (ends) {
    cols = load_cols<DUAL>(P, en);
    if constexpr (!FUSE) sx = P.sx[em];
  }

  u32x4_t xv[FUSE ? XV : 1];
  if constexpr (FUSE) {  // ahead of the weights: loads return in order
    const __amdgpu_buffer_rsrc_t xr = rsrc(P.xf, K * (P.xf_type == kF32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < XV; ++i)
      xv[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, (tid + i * WK * 64) * 16, 0, 0);
  }
  const __amdgpu_buffer_rsrc_t wr[2] = {rsrc(P.w + (size_t)n0 * K, nrows * K),
                                        rsrc((DUAL ? P.w2 : P.w) + (size_t)n0 * K, nrows * K)};
  const __amdgpu_buffer_rsrc_t xr = rsrc(P.x, FUSE ? 0 : M * ldx);
  uint32_t wo[NT], xo[MT];
#pragma unroll
  for (int a = 0; a < NT; ++a) wo[a] = 16 * a + fr < nrows ? (uint32_t)(16 * a + fr) * (uint32_t)K + 16 * q : kOOB;
#pragma unroll
  for (int i = 0; i < MT; ++i) xo[i] = 16 * i + fr < M ? (uint32_t)((16 * i + fr) * ldx + 16 * q) : kOOB;

  u32x4_t W[U][B * NT], X[U][MT];
  auto load = [&](int u, int c) __attribute__((always_inline)) {
    const bool on = c < ce && 64 * c + 16 * q < K;
#pragma unroll
    for (int k = 0; k < B; ++k)
#pragma unroll
      for (int a = 0; a < NT; ++a)
        W[u][k * NT + a] = __builtin_amdgcn_raw_buffer_load_b128(wr[k], on ? wo[a] + 64 * c : kOOB, 0, 0);
    if constexpr (!FUSE) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
        X[u][i] = __builtin_amdgcn_raw_buffer_load_b128(xr, on ? xo[i] + 64 * c : kOOB, 0, 0);
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, cb + u);
  unsigned char* xs = smem + 256;
  if constexpr (FUSE) {
    uint32_t* part = reinterpret_cast<uint32_t*>(smem);
    sx = P.xf_type == kBF16  ? quantize_token<kBF16, XV, WK * 64>(xv, K, xs, part)
          : P.xf_type == kF16 ? quantize_token<kF16, XV, WK * 64>(xv, K, xs, part)
                              : quantize_token<kF32, XV, WK * 64>(xv, K, xs, part);
  }
  i32x4_t acc[B * NT][MT];
#pragma unroll
  for (int a = 0; a < B * NT; ++a)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[a][i] = i32x4_t{0, 0, 0, 0};
  auto products = [&](int u, int c) __attribute__((always_inline)) {
    if constexpr (FUSE) X[u][0] = *reinterpret_cast<const u32x4_t*>(xs + min(c, chunks - 1) * 64 + 16 * q);
#pragma unroll
    for (int a = 0; a < B * NT; ++a)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[a][i] = mfma_i8(W[u][a], X[u][i], acc[a][i]);
  };
  int c = cb;
  for (; c + U < ce; c += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      products(u, c + u);
      load(u, c + u + U);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) products(u, c + u);
  // waves' sums: [wave][tile][x tile][lane]
  i32x4_t* sums = reinterpret_cast<i32x4_t*>(smem);
  if constexpr (FUSE) lds_sync();  // the codes' last reads
#pragma unroll
  for (int a = 0; a < B * NT; ++a)
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[((wave * B * NT + a) * MT + i) * 64 + lane] = acc[a][i];
  lds_sync();
  if (!ends) return;
  i32x4_t s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int w = 0; w < WK; ++w)
#pragma unroll
    for (int k = 0; k < B; ++k) s[k] += sums[((w * B * NT + k * NT + ta) * MT + ti) * 64 + lane];
  finish4<DUAL>(P, em, en, s[0], s[1], sx, cols);
}

// XV: 16-byte vectors of the float token a thread holds (0: codes)
template <bool DUAL, int MT, int NT, int WK, int U, int XV>
hipError_t launch(const Int8Params& P, hipStream_t s) {
  constexpr int B = DUAL ? 2 : 1;
  size_t lds = (size_t)WK * B * NT * MT * 1024;
  if (XV) lds = std::max(lds, (size_t)256 + (P.K + 63) / 64 * 64);
  if constexpr (WK * B * NT * MT > 64) {  // past 64 KB (the most is 128 KB: 128 rows of two banks)
    static std::atomic<uint64_t> done{0};  // devices whose function has the attribute
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = (uint64_t)1 << (dev & 63);
    if (e == hipSuccess && !(done.load() & bit)) {
      e = hipFuncSetAttribute((const void*)int8_gemv_kernel<DUAL, MT, NT, WK, U, XV>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e == hipSuccess) done |= bit;
    }
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((int8_gemv_kernel<DUAL, MT, NT, WK, U, XV>),
                     dim3((unsigned)((P.N + 16 * NT - 1) / (16 * NT))), dim3(WK * 64), lds, s, P);
  return hipGetLastError();
}

template <bool DUAL, int NT>
hipError_t launch_tiles(const Int8Params& P, hipStream_t s) {
  if (P.M <= 16) return launch<DUAL, 1, NT, 8, DUAL || NT == 2 ? 2 : 4, 0>(P, s);
  if (P.M <= 32) return launch<DUAL, 2, NT, 8, 2, 0>(P, s);
  if (P.M <= 48) return launch<DUAL, 3, NT, 8, 2, 0>(P, s);
  if (P.M <= 64) return launch<DUAL, 4, NT, 8, 2, 0>(P, s);
  if constexpr (NT == 1) {
    if (P.M <= 96) return launch<DUAL, 6, 1, 8, 2, 0>(P, s);
    return launch<DUAL, 8, 1, 8, 2, 0>(P, s);
  }
  return hipErrorInvalidValue;  // (the plan takes one tile above 64 rows)
}

template <bool DUAL>
hipError_t launch_rows(const Int8Params& P, hipStream_t s) {
  constexpr int U = DUAL ? 2 : 4;
  if (P.xf) {
    const int64_t bytes = (int64_t)P.K * (P.xf_type == kF32 ? 4 : 2);
    return bytes <= 8192 ? launch<DUAL, 1, 1, 8, U, 1>(P, s) : launch<DUAL, 1, 1, 8, U, 4>(P, s);
  }
  if constexpr (!DUAL) {
    if (P.nt == 2) return launch_tiles<DUAL, 2>(P, s);
  }
  return launch_tiles<DUAL, 1>(P, s);
}

}  // namespace

// Tiles of a wave, and the estimated microseconds: a CU takes about 32 KB of weights and x in a
// microsecond, over rounds of 256 blocks, and the weights come at 3.6 TB/s at most. Two tiles (one
// bank) halve what is read of x, where they leave a block for each CU. Measured, one / two tiles a
// wave: [14336,4096] 2 rows 14.7 / 16.0 us, 16 rows 20.9 / 17.5; [4096,14336] 16 rows 20.1 / 23.7.
// Against int8_gemm.hip, here / there, 16, 32, 64 and 128 rows: [4096,4096] 7.4 / 10.8, 8.6 / 11.9,
// 13.2 / 15.0, 20.5 / 16.1; [4096,14336] 20.2 / 18.8, 25 / 18.2, 40 / 19.6, 66 / 25.1; gate + up [5632,2048]
// 8.9 / 13.5, 11.2 / 11.8, 15.5 / 12.4, 25.0 / 12.2.
double int8_gemv_plan(Int8Params& P) {
  P.nt = P.banks == 1 && P.M > 8 && P.M <= 64 && P.N >= 32 * 256 ? 2 : 1;
  const double rounds = std::ceil((double)((P.N + 16 * P.nt - 1) / (16 * P.nt)) / 256);
  return 3.5 + std::max(rounds * (16.0 * P.nt * P.banks + P.M) * P.K / 32e3, (double)P.banks * P.N * P.K / 3.6e6);
}

// One token of floats quantized in the launch: four 16-byte vectors a thread. Sizes alone decide, as
// such a call asks for no workspace (pointers off 16 bytes: int8_token_any_kernel).
bool int8_gemv_fuses(int64_t M, int64_t K, int type) {
  return M == 1 && K % 16 == 0 && K * (type == kF32 ? 4 : 2) <= 512 * 4 * 16;
}

hipError_t launch_int8_gemv(const Int8Params& P, hipStream_t s) {
  return P.w2 ? launch_rows<true>(P, s) : launch_rows<false>(P, s);
}

}  // namespace mi
