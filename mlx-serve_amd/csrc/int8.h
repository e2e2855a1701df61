// Parameters and device helpers of the int8 (8-bit weights and activations) operators.
#pragma once
#include "mi_common.h"
#include "mi_internal.h"

namespace mi {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

enum FloatType { kBF16 = 0, kF16 = 1, kF32 = 2 };

// The int32 sum of K products of codes is exact up to here: 131071 * 128 * 128 < 2^31.
constexpr int64_t kInt8MaxK = 131071;

// y[m,n] = sx[m] * sw[n] * sum_k x[m,k] w[n,k] (+ bias[n]), or with a second bank (w2)
// y = silu(g) * u of the two products, which go to `gate` and `up` as well where given.
struct Int8Params {
  const int8_t* x;  // [M, ldx]
  const float* sx;  // [M]
  const int8_t* w;  // [N, K]
  const float* sw;  // [N]
  const int8_t* w2;
  const float* sw2;
  const void* bias;  // nullable [N], y's type
  void* y;           // [M, N]
  void* gate;        // nullable
  void* up;
  const void* xf;    // one-launch decode: float x [M, K], quantized in the kernel (x, sx unused)
  int xf_type;
  int64_t ldx;
  int M, N, K;
  int type;  // FloatType of y, bias, gate and up
};

// dx[m,k] = sum over banks and n of a[m,n] w[n,k], a split into `terms` bf16 parts:
// part [(bank * terms + t)][M][np] holds part t of a (zero from n = N on).
struct Int8BwdParams {
  const uint16_t* a;
  const int8_t* w[2];  // [N, K]
  void* dx;            // [M, K]
  float* part;         // splits > 1: fp32 partials [splits][M][K]
  int banks, terms, np;
  int M, N, K;
  int type;
  int splits;
};

// a = dy * sw[n] (one bank), or the two products of the SwiGLU gradient with sw / sw2.
struct Int8GradParams {
  const void* dy;
  const void* gate;  // banks == 2
  const void* up;
  const float* sw;
  const float* sw2;
  void* dgate;  // nullable
  void* dup;
  uint16_t* a;
  int banks, terms, np;
  int M, N;
  int type;
};

hipError_t launch_int8_quantize(int8_t* q, float* s, const void* x, int64_t rows, int64_t K,
                                int64_t ldq, int type, hipStream_t st);
hipError_t launch_int8_any(const Int8Params& P, hipStream_t s);
hipError_t launch_int8_grad(const Int8GradParams& P, hipStream_t s);
hipError_t launch_int8_bwd_any(const Int8BwdParams& P, hipStream_t s);

namespace i8 {

template <int T>
MI_DEV float load_f(const void* p, int64_t i) {
  if constexpr (T == kBF16) return bf16_bits_to_f32(((const uint16_t*)p)[i]);
  if constexpr (T == kF16) return (float)((const _Float16*)p)[i];
  return ((const float*)p)[i];
}
// one rounding, to nearest
template <int T>
MI_DEV void store_f(void* p, int64_t i, float v) {
  if constexpr (T == kBF16)
    ((uint16_t*)p)[i] = (uint16_t)f32_to_bf16_bits(v);
  else if constexpr (T == kF16)
    ((_Float16*)p)[i] = (_Float16)v;
  else
    ((float*)p)[i] = v;
}

// 16 rows x 64 codes of each operand: lane l holds 16 codes of row l % 16, the quarter l / 16
// of the 64 (any order of the 64 that both operands share). D: register r of lane l is
// [A row 4 (l / 16) + r][B row l % 16].
MI_DEV i32x4_t mfma_i8(u32x4_t a, u32x4_t b, i32x4_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a),
                                               __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}

// 1 / (1 + e^-g): e^-g overflows to infinity for g < -88, which gives 0, the limit.
MI_DEV float sigmoid_f(float g) { return 1.f / (1.f + expf(-g)); }

// The products of one output, to memory. Scales are applied in 32 bits, one rounding at the end.
template <int T, bool DUAL>
MI_DEV void finish(const Int8Params& P, int64_t m, int n, int32_t a, int32_t b, float sx,
                   float sw, float sw2, float bias) {
  const int64_t i = m * P.N + n;
  const float g = (float)a * sx * sw;
  if constexpr (!DUAL) {
    store_f<T>(P.y, i, g + bias);
  } else {
    const float u = (float)b * sx * sw2;
    store_f<T>(P.y, i, g * sigmoid_f(g) * u);
    if (P.gate) {
      store_f<T>(P.gate, i, g);
      store_f<T>(P.up, i, u);
    }
  }
}

}  // namespace i8
}  // namespace mi
