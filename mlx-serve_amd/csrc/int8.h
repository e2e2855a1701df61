// Parameters and device helpers of the int8 (8-bit weights and activations) operators.
#pragma once
#include "mi_common.h"
#include "mi_internal.h"

namespace mi {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

enum FloatType { kBF16 = 0, kF16 = 1, kF32 = 2 };

// The int32 sum of K products of codes is exact up to here: 131071 * 128 * 128 < 2^31.
constexpr int64_t kInt8MaxK = 131071;
constexpr int64_t kInt8FewRows = 128;  // rows that int8_gemv.hip can take

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
  int type;   // FloatType of y, bias, gate and up
  int banks;  // 1, or 2 with w2
  // int8_gemm.hip: rows of x and of w (both banks) of a tile; K ranges over blocks and 128-code steps of one, ks > 1
  // through int32 sums [ks][banks][M][N] in `part`
  int bm, bn, ks, sps;
  int ct0, ct1;  // column tiles of a launch
  int tail;      // 256 x 256 tiles: column tiles at the end that 128 x 256 ones take, in a launch of their own
  int32_t* part;
  int nt;    // int8_gemv.hip: 16-row tiles of a wave; 0: another kernel
  bool vec;    // four columns of y, gate and up with one store (N and pointers)
  bool vec16;  // their rows on 16 bytes
};

// dx[m,k] = row[m] * sum over banks, parts and n of 2^(-11 t) a_t[m,n] w[n,k]: the scaled gradients as fp16,
// each row times a power of two (1 / row[m]) that puts its largest value into 2^14 .. 2^15, in `terms`
// parts, each of them what the one before it left times 2^11. The smallest part comes first:
// [(terms - 1 - t) * banks + bank][M][np], zero from n = N on.
constexpr int kPartBits = 11;
__host__ __device__ constexpr int int8_parts(int type) { return type == kF32 ? 3 : 2; }
struct Int8BwdParams {
  const uint16_t* a;
  const float* row;    // [M]
  const int8_t* w[2];  // [N, ldw]
  void* dx;            // [M, K]
  float* part;         // ks > 1: fp32 sums [ks][M][ldw]
  int banks, terms, np;
  int M, N, K, ldw;
  int type;
  int bm, bn, ks, sps;  // int8_bwd.hip: rows and columns of a tile, ranges of sps 64-value steps over the parts
  int ct0, ct1, tail;   // as in Int8Params
  bool vec, vec16;
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
  float* row;
  int banks, terms, np;
  int M, N;
  int type;
  bool vec;  // rows and scales on 16 bytes, N a multiple of 8 (fp32: 4)
};

hipError_t launch_int8_quantize(int8_t* q, float* s, const void* x, int64_t rows, int64_t K,
                                int64_t ldq, int type, hipStream_t st);
void int8_forward_plan(Int8Params& P);  // one of the two below, from the same (int8.cpp)
double int8_gemv_plan(Int8Params& P);  // nt, from M, N, K and banks; returns estimated us
bool int8_gemv_fuses(int64_t M, int64_t K, int type);
hipError_t launch_int8_gemv(const Int8Params& P, hipStream_t s);
double int8_gemm_plan(Int8Params& P);  // bm, ks, sps, from the same; returns estimated us
hipError_t launch_int8_gemm(const Int8Params& P, hipStream_t s);
hipError_t launch_int8_pad(int8_t* to, const int8_t* from, int64_t rows, int64_t K, int64_t ld, hipStream_t s);
hipError_t launch_int8_any(const Int8Params& P, hipStream_t s);
hipError_t launch_int8_grad(const Int8GradParams& P, hipStream_t s);
void int8_bwd_plan(Int8BwdParams& P);  // from M, K, np, banks and terms: bm, bn, ks, sps
hipError_t launch_int8_bwd(const Int8BwdParams& P, hipStream_t s);
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

// Codes of a row: s = max |x| / 127, rounded once, and the integers nearest to x / s (ties to even),
// exactly: x * (1/s) is within a few units of 2^-24 of the quotient, so its nearest integer q is
// right unless the quotient lies next to a border, and r = x - q s is exact in one fma (x and s
// have 24 bits, |r| < s, and both are multiples of s's last bit, or q = 0). So |r| < s/2 proves q,
// and the rare others are settled from r.
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

// 16 rows x 64 codes of each operand: lane l holds 16 codes of row l % 16, the quarter l / 16
// of the 64 (any order of the 64 that both operands share). D: register r of lane l is
// [A row 4 (l / 16) + r][B row l % 16].
MI_DEV i32x4_t mfma_i8(u32x4_t a, u32x4_t b, i32x4_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a),
                                               __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

MI_DEV f32x4_t mfma_f16(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// s = 1 / (1 + e^-g), and 1 - s.
struct Sigmoid {
  float s, c;
};
// For results of 8 or 11 bits, on the hardware's exponential and reciprocal: one ulp each, and 1.25 |g| / 2^24
// from rounding the exponent, 2^-17 in all up to |g| = 88, where a result's own rounding is 2^-11 at best.
// e^-g overflows to infinity for g < -88, which gives 0, the limit. (sigmoid_f32 in its place, five times the
// instructions, took 2003 rows of gate + up [14336,4096] from 281 to 290 us.)
MI_DEV Sigmoid sigmoid_16(float g) {
  const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * g));
  return {s, 1.f - s};
}
// For fp32 results: e = e^-|g| has no large argument and does not overflow, and neither s nor 1 - s
// comes of a difference. e is good to one ulp, the sum, quotient and product round once each.
MI_DEV Sigmoid sigmoid_f32(float g) {
  const float e = expf(-fabsf(g)), t = 1.f / (1.f + e);
  return g < 0.f ? Sigmoid{e * t, t} : Sigmoid{t, e * t};
}
MI_DEV Sigmoid sigmoid_of(float g, bool f32) { return f32 ? sigmoid_f32(g) : sigmoid_16(g); }

// Four neighbouring values, one rounding each; `vec`: with one store.
MI_DEV void store4(void* p, int64_t i, int type, bool vec, int cnt, const float (&v)[4]) {
  if (type == kF32) {
    float* o = (float*)p + i;
    if (vec) {
      *reinterpret_cast<f32x4_t*>(o) = f32x4_t{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < cnt) o[j] = v[j];
    }
    return;
  }
  uint32_t b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    b[j] = type == kBF16 ? f32_to_bf16_bits(v[j]) : __builtin_bit_cast(uint16_t, (_Float16)v[j]);
  uint16_t* o = (uint16_t*)p + i;
  if (vec) {
    *reinterpret_cast<u32x2_t*>(o) = u32x2_t{b[0] | b[1] << 16, b[2] | b[3] << 16};
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < cnt) o[j] = (uint16_t)b[j];
  }
}
MI_DEV float load_rt(const void* p, int64_t i, int type) {
  return type == kBF16 ? load_f<kBF16>(p, i) : type == kF16 ? load_f<kF16>(p, i) : load_f<kF32>(p, i);
}

// Scales and bias of columns n .. n + 3 (those from N on repeat column n).
struct Cols {
  float s[4], s2[4], b[4];
};
template <bool DUAL>
MI_DEV Cols load_cols(const Int8Params& P, int n) {
  Cols c;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = n + j < P.N ? n + j : n;
    c.s[j] = P.sw[k];
    c.s2[j] = DUAL ? P.sw2[k] : 0.f;
    c.b[j] = !DUAL && P.bias ? load_rt(P.bias, k, P.type) : 0.f;
  }
  return c;
}

// The sums of columns n .. n + 3 (those below N) of row m, to memory: scales in 32 bits, one
// rounding at the end.
template <bool DUAL>
MI_DEV void scaled4(const Int8Params& P, i32x4_t a, i32x4_t b, float sx, const Cols& c, float (&y)[4],
                    float (&g)[4], float (&u)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    g[j] = (float)a[j] * sx * c.s[j];
    if constexpr (DUAL) {
      u[j] = (float)b[j] * sx * c.s2[j];
      y[j] = g[j] * sigmoid_of(g[j], P.type == kF32).s * u[j];
    } else {
      y[j] = P.bias ? g[j] + c.b[j] : g[j];
    }
  }
}
template <bool DUAL>
MI_DEV void finish4(const Int8Params& P, int64_t m, int n, i32x4_t a, i32x4_t b, float sx, const Cols& c) {
  const int64_t i = m * P.N + n;
  const int cnt = P.N - n;
  float y[4], u[4], g[4];
  scaled4<DUAL>(P, a, b, sx, c, y, g, u);
  store4(P.y, i, P.type, P.vec, cnt, y);
  if constexpr (DUAL) {
    if (P.gate) {
      store4(P.gate, i, P.type, P.vec, cnt, g);
      store4(P.up, i, P.type, P.vec, cnt, u);
    }
  }
}

// int32 sums of a K range: [split][bank][M][N]
template <bool DUAL>
MI_DEV void store_part(const Int8Params& P, int split, int64_t m, int n, i32x4_t a, i32x4_t b) {
#pragma unroll
  for (int k = 0; k < (DUAL ? 2 : 1); ++k) {
    int32_t* o = P.part + (((int64_t)split * (DUAL ? 2 : 1) + k) * P.M + m) * P.N + n;
    const i32x4_t v = k ? b : a;
    if (P.N % 4 == 0) {
      *reinterpret_cast<i32x4_t*>(o) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < P.N) o[j] = v[j];
    }
  }
}
}  // namespace i8
}  // namespace mi
