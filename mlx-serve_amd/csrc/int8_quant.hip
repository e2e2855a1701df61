// Token (row) quantization to int8, and the element-wise half of the SwiGLU gradient.
//
// Memory-bound: a row is read once and held in registers between the maximum and the codes. Measured:
// [8192,14336] bf16 63 us, 5.6 TB/s (a copy of 256 MiB: 5.35); one row of 4096 2 us.
#include "int8.h"

namespace mi {
namespace {

using namespace i8;

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
  // Waves a row, measured: 8192 rows of 14336 bf16 values 72 us with 4, 68 with 8 or 16; 8192 rows of 4096
  // 25 us with 1 or 8, 20 with 4.
  if (nv <= 512 && rows > 256) return launch_rows<T, 4, 2>(q, s, x, rows, K, ldq, st);
  if (nv <= 1024 && rows > 256) return launch_rows<T, 8, 2>(q, s, x, rows, K, ldq, st);
  if (nv <= 2048 && rows > 256) return launch_rows<T, 8, 4>(q, s, x, rows, K, ldq, st);
  if (nv <= 1024) return launch_rows<T, 16, 1>(q, s, x, rows, K, ldq, st);
  if (nv <= 2048) return launch_rows<T, 16, 2>(q, s, x, rows, K, ldq, st);
  if (nv <= 4096) return launch_rows<T, 16, 4>(q, s, x, rows, K, ldq, st);
  return launch_rows<T, 16, 8>(q, s, x, rows, K, ldq, st);
}

// ------------------------------------------------------------- SwiGLU gradient ---
// The values that the backward product sums, times their channel scale, as fp16 parts of 11 bits: two, and three where
// the gradient is fp32, which keep its 24. (The scale alone has 24 bits: one part adds 2^-11 of a value to a sum
// of values that may cancel, and half as much again to the error of an fp16 result: 2.9e-4 of its norm,
// 2.1e-4 with two.) fp16's range is met by a power of two for each row, exact both ways: the row's
// largest value goes into 2^14 .. 2^15. Each part is what the one before left, times 2^11, so that it
// has 11 bits wherever the first does: two leave 2^-22 of a value down to 2^-28 of the row's largest, and 2^-50
// of that largest below; three leave nothing of an fp32 value down to 2^-28 (below, where the first part is
// subnormal, the matrix instructions cut the others off at 2^-51). A row with an infinity or a NaN is taken as
// it is.
//
// Memory-bound (three reads, six writes of [M, N] with both outputs); a row is held in
// registers between its maximum and the parts. Measured: [4096,14336] bf16 gate + up 205 us, 5.2 TB/s.

// power of two for a row whose largest finite magnitude has these bits, and its reciprocal
MI_DEV void row_power(uint32_t maxbits, float* scale, float* inv) {
  const int b = maxbits == 0 ? 127 : min(268 - (int)(maxbits >> 23), 253);
  *scale = __uint_as_float((uint32_t)b << 23);
  *inv = __uint_as_float((uint32_t)(254 - b) << 23);
}

template <int TERMS>
MI_DEV void parts_of(float v, uint16_t (&p)[TERMS]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    const _Float16 h = (_Float16)v;
    p[t] = __builtin_bit_cast(uint16_t, h);
    const float f = (float)h;
    const bool fin = (__float_as_uint(f) & 0x7F800000u) != 0x7F800000u;
    v = fin ? (v - f) * (float)(1 << kPartBits) : 0.f;  // (the difference is exact, and at most 2^15 again)
  }
}
// where part t of a bank lies
MI_DEV int64_t part_at(const Int8GradParams& P, int bank, int t, int64_t m) {
  return ((int64_t)((P.terms - 1 - t) * P.banks + bank) * P.M + m) * P.np;
}

template <int T>
struct Grad {
  float a, b, dg, du;
};
template <int T, int BANKS>
MI_DEV Grad<T> gradient(float dy, float g, float u, float sw, float sw2) {
  Grad<T> r;
  if constexpr (BANKS == 1) {
    r.a = dy * sw;
    r.b = r.dg = r.du = 0.f;
  } else {
    const Sigmoid sig = sigmoid_of(g, T == kF32);
    r.dg = dy * u * sig.s * (1.f + g * sig.c);
    r.du = dy * g * sig.s;
    r.a = r.dg * sw;
    r.b = r.du * sw2;
  }
  return r;
}
MI_DEV uint32_t mag(float v) {  // 0 unless finite
  const uint32_t m = __float_as_uint(v) & 0x7FFFFFFFu;
  return m < 0x7F800000u ? m : 0u;
}

// values of a 16-byte vector
template <int T, int E>
MI_DEV void unpack(const void* p, int64_t v, float (&f)[E]) {
  const u32x4_t x = reinterpret_cast<const u32x4_t*>(p)[v];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if constexpr (T == kF32) {
      f[j] = __uint_as_float(x[j]);
    } else {
      const uint16_t h = (uint16_t)(x[j / 2] >> (16 * (j & 1)));
      f[j] = T == kBF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
    }
  }
}
template <int E>
MI_DEV void unpack_f32(const float* p, int n, float (&f)[E]) {
#pragma unroll
  for (int j = 0; j < E; j += 4) {
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(p + n + j);
#pragma unroll
    for (int k = 0; k < 4; ++k) f[j + k] = x[k];
  }
}
template <int T, int E>
MI_DEV void pack_store(void* p, int64_t v, const float (&f)[E]) {
  u32x4_t o = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if constexpr (T == kF32)
      o[j] = __float_as_uint(f[j]);
    else
      o[j / 2] |= (T == kBF16 ? f32_to_bf16_bits(f[j])
                              : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[j])) << (16 * (j & 1));
  }
  reinterpret_cast<u32x4_t*>(p)[v] = o;
}

// A block a row, VPT vectors of 16 bytes a thread; np / E vectors of `a` a row.
template <int T, int BANKS, int WPR, int VPT>
__global__ void __launch_bounds__(WPR * 64) int8_grad_kernel(Int8GradParams P) {
  constexpr int E = T == kF32 ? 4 : 8, TERMS = int8_parts(T);
  __shared__ uint32_t part[WPR];
  const int64_t m = blockIdx.x;
  const int nv = P.N / E, npv = P.np / E;
  float a[VPT][E], b[BANKS == 2 ? VPT : 1][E];
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * WPR * 64;
    const bool on = c < nv;
    float dy[E], g[E], u[E], sw[E], sw2[E], dg[E], du[E];
    if (on) {
      unpack<T, E>(P.dy, m * nv + c, dy);
      unpack_f32<E>(P.sw, c * E, sw);
      if constexpr (BANKS == 2) {
        unpack<T, E>(P.gate, m * nv + c, g);
        unpack<T, E>(P.up, m * nv + c, u);
        unpack_f32<E>(P.sw2, c * E, sw2);
      }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
      a[i][j] = 0.f;
      if constexpr (BANKS == 2) b[i][j] = 0.f;
      if (on) {
        const Grad<T> r = gradient<T, BANKS>(dy[j], BANKS == 2 ? g[j] : 0.f, BANKS == 2 ? u[j] : 0.f,
                                             sw[j], BANKS == 2 ? sw2[j] : 0.f);
        a[i][j] = r.a;
        mx = max(mx, mag(r.a));
        if constexpr (BANKS == 2) {
          b[i][j] = r.b;
          mx = max(mx, mag(r.b));
        }
        dg[j] = r.dg;
        du[j] = r.du;
      }
    }
    if (BANKS == 2 && on && P.dgate) {
      pack_store<T, E>(P.dgate, m * nv + c, dg);
      pack_store<T, E>(P.dup, m * nv + c, du);
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WPR; ++i) mx = max(mx, part[i]);
  float scale, inv;
  row_power(mx, &scale, &inv);
  if (threadIdx.x == 0) P.row[m] = inv;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * WPR * 64;
    if (c >= npv) continue;
#pragma unroll
    for (int k = 0; k < BANKS; ++k) {
      uint16_t p[E][TERMS];
#pragma unroll
      for (int j = 0; j < E; ++j) parts_of<TERMS>((k ? b[BANKS == 2 ? i : 0][j] : a[i][j]) * scale, p[j]);
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
        uint32_t o[E / 2];
#pragma unroll
        for (int j = 0; j < E; j += 2) o[j / 2] = p[j][t] | (uint32_t)p[j + 1][t] << 16;
        uint16_t* q = P.a + part_at(P, k, t, m) + c * E;
        if constexpr (E == 8)
          *reinterpret_cast<u32x4_t*>(q) = u32x4_t{o[0], o[1], o[E / 2 - 2], o[E / 2 - 1]};
        else
          *reinterpret_cast<u32x2_t*>(q) = u32x2_t{o[0], o[1]};
      }
    }
  }
}

// Any width and alignment: a block a row, which is read and computed twice.
template <int T, int BANKS>
__global__ void __launch_bounds__(256) int8_grad_any_kernel(Int8GradParams P) {
  constexpr int TERMS = int8_parts(T);
  __shared__ uint32_t part[4];
  for (int64_t m = blockIdx.x; m < P.M; m += gridDim.x) {
    const int64_t at = m * P.N;
    auto grad = [&](int n) {
      return gradient<T, BANKS>(load_f<T>(P.dy, at + n), BANKS == 2 ? load_f<T>(P.gate, at + n) : 0.f,
                                BANKS == 2 ? load_f<T>(P.up, at + n) : 0.f, P.sw[n], BANKS == 2 ? P.sw2[n] : 0.f);
    };
    uint32_t mx = 0;
    for (int n = threadIdx.x; n < P.N; n += 256) {
      const Grad<T> r = grad(n);
      mx = max(mx, max(mag(r.a), mag(r.b)));
      if (BANKS == 2 && P.dgate) {
        store_f<T>(P.dgate, at + n, r.dg);
        store_f<T>(P.dup, at + n, r.du);
      }
    }
    for (int d = 32; d; d >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
    __syncthreads();
    mx = max(max(part[0], part[1]), max(part[2], part[3]));
    float scale, inv;
    row_power(mx, &scale, &inv);
    if (threadIdx.x == 0) P.row[m] = inv;
    for (int n = threadIdx.x; n < P.np; n += 256) {
      Grad<T> r = {0.f, 0.f, 0.f, 0.f};
      if (n < P.N) r = grad(n);
#pragma unroll
      for (int k = 0; k < BANKS; ++k) {
        uint16_t p[TERMS];
        parts_of<TERMS>((k ? r.b : r.a) * scale, p);
#pragma unroll
        for (int t = 0; t < TERMS; ++t) P.a[part_at(P, k, t, m) + n] = p[t];
      }
    }
  }
}

template <int T, int BANKS, int WPR, int VPT>
hipError_t launch_grad_rows(const Int8GradParams& P, hipStream_t s) {
  hipLaunchKernelGGL((int8_grad_kernel<T, BANKS, WPR, VPT>), dim3((unsigned)P.M), dim3(WPR * 64), 0, s, P);
  return hipGetLastError();
}

template <int T, int BANKS>
hipError_t launch_grad(const Int8GradParams& P, hipStream_t s) {
  const int npv = P.np / (T == kF32 ? 4 : 8);
  if (P.vec && npv <= 4096 && P.M <= 1 << 21) {  // (below 2^32 threads)
    if (npv <= 256) return launch_grad_rows<T, BANKS, 4, 1>(P, s);
    if (npv <= 512) return launch_grad_rows<T, BANKS, 4, 2>(P, s);
    if (npv <= 1024) return launch_grad_rows<T, BANKS, 16, 1>(P, s);
    if (npv <= 2048) return launch_grad_rows<T, BANKS, 16, 2>(P, s);
    return launch_grad_rows<T, BANKS, 16, 4>(P, s);
  }
  hipLaunchKernelGGL((int8_grad_any_kernel<T, BANKS>), dim3((unsigned)(P.M < 65536 ? P.M : 65536)), dim3(256), 0,
                     s, P);
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
