// Token (row) quantization to int8, and the element-wise half of the SwiGLU gradient.
//
// Quantization: s = max_k |x_k| / 127 rounded once to fp32, q_k the integer nearest to x_k / s,
// ties to even, exactly: t = x * (1/s) is within a few units of 2^-24 of the quotient, so its
// nearest integer q is right unless the quotient lies next to a border, and r = x - q s is exact
// in one fma (x and s have 24 bits, |r| < s, and both are multiples of s's last bit, or q = 0).
// So |r| < s/2 proves q, and the rare others are settled from r.
//
// Memory-bound: a row is read once and held in registers between the maximum and the codes.
#include "int8.h"

namespace mi {
namespace {

using namespace i8;

constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: v + kMagic rounds v to an integer (ties to
                                      // even), whose two's complement is the sum's low bits
constexpr float kTiny = 0x1p-100f;    // below, x and s are scaled by 2^100 (exact)

struct RowScale {
  float s, inv, half;
  bool fin, tiny;  // codes are 0 unless s is finite and not 0
};

MI_DEV RowScale row_scale(uint32_t maxbits) {
  RowScale r;
  r.s = __uint_as_float(maxbits) / 127.f;
  r.fin = r.s > 0.f && r.s < __builtin_inff();
  r.tiny = r.s < kTiny;
  r.inv = r.fin ? 1.f / (r.tiny ? r.s * 0x1p100f : r.s) : 0.f;
  r.half = 0.5f * r.s;
  return r;
}

// any row and value
MI_DEV int code_of(float x, const RowScale& R) {
  if (!R.fin) return 0;
  const float s = R.tiny ? R.s * 0x1p100f : R.s;
  if (R.tiny) x *= 0x1p100f;
  float q = rintf(x * R.inv);
  const float d = fmaf(-q, s, x);
  const float away = d > 0.f ? 1.f : -1.f, h = 0.5f * s;
  if (fabsf(d) > h || (fabsf(d) == h && ((int)q & 1))) q += away;
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

// four codes in a dword
MI_DEV uint32_t codes4(const float (&x)[4], const RowScale& R) {
  uint32_t t[4];
  bool sure = R.fin && !R.tiny;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = fmaf(x[i], R.inv, kMagic);
    t[i] = __float_as_uint(v);
    sure = sure && fabsf(fmaf(-(v - kMagic), R.s, x[i])) < R.half;
  }
  if (!sure) {
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = (uint32_t)code_of(x[i], R);
  }
  return perm_b32(perm_b32(t[3], t[2], 0x0C0C0400u), perm_b32(t[1], t[0], 0x0C0C0400u), 0x05040100u);
}

// Bits of |x| compare as the values do, and a NaN above infinity: the integer maximum keeps it.
template <int T>
MI_DEV uint32_t max_bits(u32x4_t v, uint32_t m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == kF32) {
      m = max(m, v[i] & 0x7FFFFFFFu);
    } else {
      m = max(m, v[i] & 0x7FFFu);
      m = max(m, (v[i] >> 16) & 0x7FFFu);
    }
  }
  return m;
}
template <int T>
MI_DEV uint32_t f32_bits(uint32_t m) {  // of the largest magnitude, as fp32
  if constexpr (T == kBF16) return m << 16;
  if constexpr (T == kF16)
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m)) & 0x7FFFFFFFu;
  return m;
}

// A row for each group of WPR waves; VPT 16-byte vectors a lane.
template <int T, int WPR, int VPT>
__global__ void __launch_bounds__(WPR < 4 ? 256 : WPR * 64)
int8_quantize_kernel(int8_t* __restrict__ q, float* __restrict__ s, const void* __restrict__ x,
                     int64_t rows, int K, int ldq) {
  constexpr int E = T == kF32 ? 4 : 8;  // values of a vector
  constexpr int kRows = WPR < 4 ? 4 / WPR : 1;
  const int tid = threadIdx.x % (WPR * 64);
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / (WPR * 64);
  const bool on = row < rows;
  const int nv = K / E;
  u32x4_t v[VPT];
  uint32_t m = 0;
  const u32x4_t* xr = reinterpret_cast<const u32x4_t*>(x) + (on ? row : 0) * (int64_t)nv;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = tid + i * WPR * 64;
    v[i] = c < nv ? xr[c] : u32x4_t{0, 0, 0, 0};
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) m = max_bits<T>(v[i], m);
#pragma unroll
  for (int d = 32; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
  if constexpr (WPR > 1) {
    __shared__ uint32_t part[16];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    const int w0 = threadIdx.x / (WPR * 64) * WPR;
#pragma unroll
    for (int i = 0; i < WPR; ++i) m = max(m, part[w0 + i]);
  }
  if (!on) return;
  const RowScale R = row_scale(f32_bits<T>(m));
  if (tid == 0) s[row] = R.s;
  int8_t* qr = q + row * ldq;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = tid + i * WPR * 64;
    if (c >= nv) continue;
    if constexpr (T == kF32) {
      const float f[4] = {__uint_as_float(v[i].x), __uint_as_float(v[i].y),
                          __uint_as_float(v[i].z), __uint_as_float(v[i].w)};
      reinterpret_cast<uint32_t*>(qr)[c] = codes4(f, R);
    } else {
      u32x2_t o;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint16_t b = (uint16_t)(v[i][2 * h + j / 2] >> (16 * (j & 1)));
          f[j] = T == kBF16 ? bf16_bits_to_f32(b) : (float)__builtin_bit_cast(_Float16, b);
        }
        o[h] = codes4(f, R);
      }
      reinterpret_cast<u32x2_t*>(qr)[c] = o;
    }
  }
  for (int k = K + 4 * tid; k < ldq; k += 4 * WPR * 64) *reinterpret_cast<uint32_t*>(qr + k) = 0;
}

// Any width and alignment: a block a row, read twice.
template <int T>
__global__ void __launch_bounds__(256)
int8_quantize_any_kernel(int8_t* __restrict__ q, float* __restrict__ s, const void* __restrict__ x,
                         int64_t rows, int64_t K, int64_t ldq) {
  __shared__ uint32_t part[4];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    uint32_t m = 0;
    for (int64_t k = threadIdx.x; k < K; k += 256)
      m = max(m, __float_as_uint(load_f<T>(x, row * K + k)) & 0x7FFFFFFFu);
    for (int d = 32; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    m = max(max(part[0], part[1]), max(part[2], part[3]));
    const RowScale R = row_scale(m);
    if (threadIdx.x == 0) s[row] = R.s;
    for (int64_t k = threadIdx.x; k < ldq; k += 256)
      q[row * ldq + k] = (int8_t)(k < K ? code_of(load_f<T>(x, row * K + k), R) : 0);
  }
}

template <int T, int WPR, int VPT>
hipError_t launch_rows(int8_t* q, float* s, const void* x, int64_t rows, int64_t K, int64_t ldq,
                       hipStream_t st) {
  constexpr int kRows = WPR < 4 ? 4 / WPR : 1;
  hipLaunchKernelGGL((int8_quantize_kernel<T, WPR, VPT>), dim3((unsigned)((rows + kRows - 1) / kRows)),
                     dim3(WPR < 4 ? 256 : WPR * 64), 0, st, q, s, x, rows, (int)K, (int)ldq);
  return hipGetLastError();
}

template <int T>
hipError_t launch_type(int8_t* q, float* s, const void* x, int64_t rows, int64_t K, int64_t ldq,
                       hipStream_t st) {
  constexpr int E = T == kF32 ? 4 : 8;
  const bool vec = K % E == 0 && ldq % E == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)q % E == 0 &&
                   K <= 16 * 64 * 8 * E;
  if (!vec) {
    const unsigned g = (unsigned)(rows < 65536 ? rows : 65536);
    hipLaunchKernelGGL((int8_quantize_any_kernel<T>), dim3(g), dim3(256), 0, st, q, s, x, rows, K, ldq);
    return hipGetLastError();
  }
  const int64_t nv = K / E;
  if (nv <= 64 && rows > 256) return launch_rows<T, 1, 1>(q, s, x, rows, K, ldq, st);
  if (nv <= 256) return launch_rows<T, 4, 1>(q, s, x, rows, K, ldq, st);
  if (nv <= 512 && rows > 256) return launch_rows<T, 4, 2>(q, s, x, rows, K, ldq, st);
  if (nv <= 1024 && rows > 256) return launch_rows<T, 4, 4>(q, s, x, rows, K, ldq, st);
  if (nv <= 2048 && rows > 256) return launch_rows<T, 4, 8>(q, s, x, rows, K, ldq, st);
  if (nv <= 1024) return launch_rows<T, 16, 1>(q, s, x, rows, K, ldq, st);
  if (nv <= 2048) return launch_rows<T, 16, 2>(q, s, x, rows, K, ldq, st);
  if (nv <= 4096) return launch_rows<T, 16, 4>(q, s, x, rows, K, ldq, st);
  return launch_rows<T, 16, 8>(q, s, x, rows, K, ldq, st);
}

// ------------------------------------------------------------- SwiGLU gradient ---
// Values times their channel scale, in bf16 parts for the matrix product that follows: one part,
// rounded, for bf16 gradients; for fp16 and fp32 the leading 8 bits, cut off (so that what is
// left is exact), then the next 8, the last part rounded: 16 and 24 bits in all.
template <int TERMS>
MI_DEV void split_bf16(float v, uint16_t (&p)[TERMS]) {
  if constexpr (TERMS == 1) {
    p[0] = (uint16_t)f32_to_bf16_bits(v);
  } else {
    const bool fin = (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u;
    float r = v;
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
      const bool last = t == TERMS - 1;
      p[t] = last || !fin ? (uint16_t)f32_to_bf16_bits(r) : (uint16_t)(__float_as_uint(r) >> 16);
      r = fin ? r - bf16_bits_to_f32(p[t]) : 0.f;
    }
  }
}

template <int T, int BANKS, int VEC>
__global__ void __launch_bounds__(256) int8_grad_kernel(Int8GradParams P) {
  constexpr int TERMS = T + 1;
  const int np = P.np, N = P.N;
  const int64_t per_row = np / VEC, total = per_row * P.M;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / per_row;
    const int n0 = (int)(i - m * per_row) * VEC;
    const int64_t at = m * N + n0;
    const bool on = n0 < N;  // VEC > 1 only where N is a multiple of it
    uint16_t part[BANKS][TERMS][VEC];
    float dg[VEC], du[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float a = 0.f, b = 0.f;
      dg[j] = du[j] = 0.f;
      if (on) {
        const float dy = load_f<T>(P.dy, at + j);
        if constexpr (BANKS == 1) {
          a = dy * P.sw[n0 + j];
        } else {
          const float g = load_f<T>(P.gate, at + j), u = load_f<T>(P.up, at + j);
          const float sig = sigmoid_f(g);
          dg[j] = dy * u * sig * (1.f + g * (1.f - sig));
          du[j] = dy * g * sig;
          a = dg[j] * P.sw[n0 + j];
          b = du[j] * P.sw2[n0 + j];
        }
      }
      uint16_t p[TERMS];
      split_bf16<TERMS>(a, p);
#pragma unroll
      for (int t = 0; t < TERMS; ++t) part[0][t][j] = p[t];
      if constexpr (BANKS == 2) {
        split_bf16<TERMS>(b, p);
#pragma unroll
        for (int t = 0; t < TERMS; ++t) part[1][t][j] = p[t];
      }
    }
#pragma unroll
    for (int b = 0; b < BANKS; ++b)
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
        uint16_t* o = P.a + ((int64_t)(b * TERMS + t) * P.M + m) * np + n0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = part[b][t][j];
      }
    if (BANKS == 2 && on && P.dgate) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        store_f<T>(P.dgate, at + j, dg[j]);
        store_f<T>(P.dup, at + j, du[j]);
      }
    }
  }
}

template <int T, int BANKS>
hipError_t launch_grad(const Int8GradParams& P, hipStream_t s) {
  const int64_t total = (int64_t)P.M * P.np;
  int64_t g = (total + 255) / 256;
  if (g > 16384) g = 16384;
  hipLaunchKernelGGL((int8_grad_kernel<T, BANKS, 1>), dim3((unsigned)g), dim3(256), 0, s, P);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_int8_quantize(int8_t* q, float* s, const void* x, int64_t rows, int64_t K,
                                int64_t ldq, int type, hipStream_t st) {
  // a launch has fewer than 2^32 threads: at most 2^21 rows of 1024
  constexpr int64_t kChunk = (int64_t)1 << 21;
  const size_t row = (size_t)K * (type == kF32 ? 4 : 2);
  for (int64_t r = 0; r < rows; r += kChunk) {
    const int64_t n = std::min(kChunk, rows - r);
    const void* xr = (const char*)x + (size_t)r * row;
    const hipError_t e = type == kBF16 ? launch_type<kBF16>(q + r * ldq, s + r, xr, n, K, ldq, st)
                         : type == kF16 ? launch_type<kF16>(q + r * ldq, s + r, xr, n, K, ldq, st)
                                        : launch_type<kF32>(q + r * ldq, s + r, xr, n, K, ldq, st);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_int8_grad(const Int8GradParams& P, hipStream_t s) {
  if (P.banks == 1)
    return P.type == kBF16 ? launch_grad<kBF16, 1>(P, s)
           : P.type == kF16 ? launch_grad<kF16, 1>(P, s)
                            : launch_grad<kF32, 1>(P, s);
  return P.type == kBF16 ? launch_grad<kBF16, 2>(P, s)
         : P.type == kF16 ? launch_grad<kF16, 2>(P, s)
                          : launch_grad<kF32, 2>(P, s);
}

}  // namespace mi
