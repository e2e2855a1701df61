// Int8 products of any size and alignment: 64 x 64 output tiles, operands staged through LDS, byte by
// byte where a 16-byte load could leave the row. The kernels of int8_gemv.hip, int8_gemm.hip and
// int8_bwd.hip take rows on 16 bytes; what is left here are pointers that are not. (Rows of K bytes, no
// multiple of 16, are first copied to such: int8_pad_kernel. Straight from them, 16 rows' gradient
// through a [4001,1001] matrix took 188 us.)
#include "int8.h"

namespace mi {
namespace {

using namespace i8;

constexpr int kT = 64;        // rows of either operand
constexpr int kLd = 64 + 16;  // bytes of a staged row: 16-byte aligned, banks spread

// 16 codes k .. k+15 of a row at any address, zeros from K on
MI_DEV u32x4_t codes16(const int8_t* row, int k, int K) {
  u32x4_t v = {0, 0, 0, 0};
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
    return v;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (k + j < K) v[j / 4] |= (uint32_t)(uint8_t)row[k + j] << (8 * (j % 4));
  return v;
}

// Rows of K codes to rows of ld, a multiple of 16, zeros from K on.
__global__ void __launch_bounds__(256) int8_pad_kernel(int8_t* __restrict__ to, const int8_t* __restrict__ from,
                                                       int64_t rows, int K, int ld) {
  const int64_t per = ld / 16, total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int k = (int)(i - r * per) * 16;
    *reinterpret_cast<u32x4_t*>(to + r * ld + k) = codes16(from + r * K, k, K);
  }
}

// y (or the gate and up products): block of 4 waves, wave w rows 16w .. 16w+15 of the weights
// against all 64 rows of x.
template <bool DUAL>
__global__ void __launch_bounds__(256) int8_any_kernel(Int8Params P) {
  __shared__ __attribute__((aligned(16))) unsigned char xs[kT * kLd];
  __shared__ __attribute__((aligned(16))) unsigned char ws[(DUAL ? 2 : 1) * kT * kLd];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int fr = lane & 15, q = lane >> 4;
  const int ntiles = (P.N + kT - 1) / kT;
  const int64_t m0 = (int64_t)(blockIdx.x / ntiles) * kT;
  const int n0 = (int)(blockIdx.x % ntiles) * kT;
  const int r = tid >> 2, rb = 16 * (tid & 3);  // the row and bytes this thread stages
  const int64_t xm = min(m0 + r, (int64_t)P.M - 1);
  const int64_t wn = min(n0 + r, P.N - 1);
  i32x4_t acc[DUAL ? 2 : 1][4];
#pragma unroll
  for (int b = 0; b < (DUAL ? 2 : 1); ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[b][i] = i32x4_t{0, 0, 0, 0};
  for (int k = 0; k < P.K; k += 64) {
    *reinterpret_cast<u32x4_t*>(xs + r * kLd + rb) = codes16(P.x + xm * P.ldx, k + rb, P.K);
    *reinterpret_cast<u32x4_t*>(ws + r * kLd + rb) = codes16(P.w + wn * P.K, k + rb, P.K);
    if constexpr (DUAL)
      *reinterpret_cast<u32x4_t*>(ws + (kT + r) * kLd + rb) = codes16(P.w2 + wn * P.K, k + rb, P.K);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < (DUAL ? 2 : 1); ++b) {
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(ws + (b * kT + 16 * wave + fr) * kLd + 16 * q);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[b][i] = mfma_i8(w, *reinterpret_cast<const u32x4_t*>(xs + (16 * i + fr) * kLd + 16 * q), acc[b][i]);
    }
    __syncthreads();
  }
  const int n = n0 + 16 * wave + 4 * q;
  if (n >= P.N) return;
  const Cols c = load_cols<DUAL>(P, n);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + 16 * i + fr;
    if (m < P.M) finish4<DUAL>(P, m, n, acc[0][i], acc[DUAL ? 1 : 0][i], P.sx[m], c);
  }
}

// One float token of sizes that int8_gemv.hip would quantize in its launch, on pointers it cannot
// take: the same here, with no workspace. A wave has four columns at a time.
template <int T, bool DUAL>
__global__ void __launch_bounds__(256) int8_token_any_kernel(Int8Params P) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  uint32_t* part = reinterpret_cast<uint32_t*>(smem);
  int8_t* xs = reinterpret_cast<int8_t*>(smem + 16);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t m = 0;
  for (int k = tid; k < P.K; k += 256) m = max(m, __float_as_uint(load_f<T>(P.xf, k)) & 0x7FFFFFFFu);
  for (int d = 32; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
  if (lane == 0) part[wave] = m;
  __syncthreads();
  const RowScale R = row_scale(max(max(part[0], part[1]), max(part[2], part[3])));
  for (int k = tid; k < P.K; k += 256) xs[k] = (int8_t)code_of(load_f<T>(P.xf, k), R);
  __syncthreads();
  const int n = ((int)blockIdx.x * 4 + wave) * 4;
  if (n >= P.N) return;
  int32_t s[2][4] = {};
  for (int j = 0; j < 4 && n + j < P.N; ++j) {
    const int64_t row = (int64_t)(n + j) * P.K;
    for (int k = lane; k < P.K; k += 64) {
      s[0][j] += (int)xs[k] * (int)P.w[row + k];
      if constexpr (DUAL) s[1][j] += (int)xs[k] * (int)P.w2[row + k];
    }
  }
#pragma unroll
  for (int b = 0; b < (DUAL ? 2 : 1); ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      for (int d = 32; d; d >>= 1) s[b][j] += __shfl_xor(s[b][j], d);
  if (lane == 0)
    finish4<DUAL>(P, 0, n, i32x4_t{s[0][0], s[0][1], s[0][2], s[0][3]},
                  i32x4_t{s[1][0], s[1][1], s[1][2], s[1][3]}, R.s, load_cols<DUAL>(P, n));
}

template <int T>
hipError_t launch_token(const Int8Params& P, hipStream_t s) {
  const dim3 grid((unsigned)((P.N + 15) / 16));
  if (P.w2)
    hipLaunchKernelGGL((int8_token_any_kernel<T, true>), grid, dim3(256), 16 + P.K, s, P);
  else
    hipLaunchKernelGGL((int8_token_any_kernel<T, false>), grid, dim3(256), 16 + P.K, s, P);
  return hipGetLastError();
}

// dx: 64 rows x 64 codes of the weight rows' K; 32 values of n a step. The weights' tile is
// turned in LDS (row k, values n) as exact fp16, times the power of two of the gradients' part.
constexpr int kLdB = 40;  // fp16 values of a staged row

template <int T>
__global__ void __launch_bounds__(256) int8_bwd_any_kernel(Int8BwdParams P) {
  __shared__ __attribute__((aligned(16))) uint16_t as[kT * kLdB];
  __shared__ __attribute__((aligned(16))) uint16_t bs[kT * kLdB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int fr = lane & 15, q = lane >> 4;
  const int ktiles = (P.K + kT - 1) / kT;
  const int64_t m0 = (int64_t)(blockIdx.x / ktiles) * kT;
  const int k0 = (int)(blockIdx.x % ktiles) * kT;
  const int ar = tid >> 2, ac = 8 * (tid & 3);   // row of a, 8 values of n
  const int wr = tid >> 3, wc = 8 * (tid & 7);   // value of n, 8 codes of k
  const int64_t am = min(m0 + ar, (int64_t)P.M - 1);
  f32x4_t acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int seg = 0; seg < P.banks * P.terms; ++seg) {
    const uint16_t* a = P.a + (int64_t)seg * P.M * P.np;
    const int8_t* w = P.w[seg % P.banks];
    const float part = 1.f / (float)(1u << kPartBits * (P.terms - 1 - seg / P.banks));
    for (int n = 0; n < P.N; n += 32) {  // a is zero up to np, a multiple of 32
      *reinterpret_cast<u32x4_t*>(as + ar * kLdB + ac) =
          *reinterpret_cast<const u32x4_t*>(a + am * P.np + n + ac);
      const bool on = n + wr < P.N;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = k0 + wc + j;
        const _Float16 f = on && k < P.K ? (_Float16)((float)w[(int64_t)(n + wr) * P.K + k] * part)
                                             : (_Float16)0.f;
        bs[(wc + j) * kLdB + wr] = __builtin_bit_cast(uint16_t, f);
      }
      __syncthreads();
      const u32x4_t b = *reinterpret_cast<const u32x4_t*>(bs + (16 * wave + fr) * kLdB + 8 * q);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[i] = mfma_f16(b, *reinterpret_cast<const u32x4_t*>(as + (16 * i + fr) * kLdB + 8 * q), acc[i]);
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + 16 * i + fr;
    if (m >= P.M) continue;
    const float r = P.row[m];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + 16 * wave + 4 * q + j;
      if (k < P.K) store_f<T>(P.dx, m * P.K + k, acc[i][j] * r);
    }
  }
}

template <int T>
hipError_t launch_bwd(const Int8BwdParams& P, hipStream_t s) {
  const dim3 grid((unsigned)((((int64_t)P.M + kT - 1) / kT) * ((P.K + kT - 1) / kT)));
  hipLaunchKernelGGL((int8_bwd_any_kernel<T>), grid, dim3(256), 0, s, P);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_int8_pad(int8_t* to, const int8_t* from, int64_t rows, int64_t K, int64_t ld, hipStream_t s) {
  const int64_t blocks = (rows * (ld / 16) + 255) / 256;
  hipLaunchKernelGGL(int8_pad_kernel, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, s, to, from,
                     rows, (int)K, (int)ld);
  return hipGetLastError();
}

hipError_t launch_int8_any(const Int8Params& P, hipStream_t s) {
  if (P.xf)
    return P.xf_type == kBF16 ? launch_token<kBF16>(P, s)
           : P.xf_type == kF16 ? launch_token<kF16>(P, s)
                               : launch_token<kF32>(P, s);
  const dim3 grid((unsigned)((((int64_t)P.M + kT - 1) / kT) * ((P.N + kT - 1) / kT)));
  if (P.w2)
    hipLaunchKernelGGL((int8_any_kernel<true>), grid, dim3(256), 0, s, P);
  else
    hipLaunchKernelGGL((int8_any_kernel<false>), grid, dim3(256), 0, s, P);
  return hipGetLastError();
}

hipError_t launch_int8_bwd_any(const Int8BwdParams& P, hipStream_t s) {
  return P.type == kBF16 ? launch_bwd<kBF16>(P, s)
         : P.type == kF16 ? launch_bwd<kF16>(P, s)
                          : launch_bwd<kF32>(P, s);
}

}  // namespace mi
