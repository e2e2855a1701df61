// C ABI of the int8 operators (include/mi_qmm.h): validation, dispatch, workspace layout. The
// workspace belongs to the caller, so calls on different streams and graphs share nothing.
#include <string>

#include "int8.h"
#include "mi_qmm.h"

namespace mi {
int report_error(int code, const std::string& msg);  // sets mi_last_error() (api.cpp)

// up to 16 rows the few-row kernel, up to 128 the one that should be faster
void int8_forward_plan(Int8Params& P) {
  P.ks = 1;
  const double few = P.M <= kInt8FewRows ? int8_gemv_plan(P) : (P.nt = 0, 0.0);
  if (P.M > 16 && int8_gemm_plan(P) < few) P.nt = 0;
  if (P.nt) P.ks = 1;
}
}  // namespace mi

namespace {

using mi::report_error;

constexpr int64_t kMaxDim = (int64_t)1 << 30;
constexpr int64_t kMaxTiles = (int64_t)1 << 22;  // blocks of up to 512 threads: below 2^32 threads

// A backward call's blocks, and offsets within 256 rows of a gradient or 64 of codes below 2^31.
bool backward_fits(int64_t M, int64_t N, int64_t K) {
  return ((M + 63) / 64) * ((K + 63) / 64) <= kMaxTiles && N < (int64_t)1 << 21 && K < (int64_t)1 << 24;
}

int bad(const char* msg) { return report_error(MI_ERR_INVALID, msg); }
int hip_status(hipError_t e, const char* what) {
  return e == hipSuccess ? MI_OK
                         : report_error(MI_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

int float_type(int dtype) {
  return dtype == MI_DTYPE_BFLOAT16  ? mi::kBF16
         : dtype == MI_DTYPE_FLOAT16 ? mi::kF16
         : dtype == MI_DTYPE_FLOAT32 ? mi::kF32
                                     : -1;
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Shared by the five calls: sizes and the workspace the caller gave. `need` 0: none is used.
int check_sizes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return bad("negative size");
  if (M > kMaxDim || N > kMaxDim || K > kMaxDim) return bad("M, N or K too large");
  return MI_OK;
}
int check_workspace(const void* ws, int64_t given, int64_t need) {
  if (need == 0) return MI_OK;
  if (!ws || given < need)
    return report_error(MI_ERR_WORKSPACE, "this call needs a workspace of " + std::to_string(need) +
                                              " bytes, " + std::to_string(ws ? given : 0) + " given");
  if ((uintptr_t)ws % 16) return bad("the workspace must be aligned to 16 bytes");
  return MI_OK;
}

// Forward workspace: codes [M, ld] and scales of activations that come as floats; where K is no
// multiple of 16 also rows of ld = K rounded up for x and w; then the K ranges' sums of a split
// product. Sizes alone decide what is asked for; a call on pointers that another kernel has to
// take leaves the sums' part unused.
int64_t x_bytes(int64_t M, int64_t K, int x_dtype) {
  return x_dtype == MI_DTYPE_INT8 && K % 16 == 0 ? 0 : up(M * up(K, 16), 256);
}
int64_t sx_bytes(int64_t M, int x_dtype) { return x_dtype == MI_DTYPE_INT8 ? 0 : up(M * 4, 256); }
int64_t w_bytes(int64_t N, int64_t K) { return K % 16 == 0 ? 0 : up(N * up(K, 16), 256); }  // a bank
bool fused_token(int64_t M, int64_t K, int x_dtype) {
  return x_dtype != MI_DTYPE_INT8 && mi::int8_gemv_fuses(M, K, float_type(x_dtype));
}
int64_t forward_need(mi::Int8Params& P, int64_t M, int64_t N, int64_t K, int x_dtype) {
  if (M == 0 || N == 0 || K == 0 || fused_token(M, K, x_dtype)) return 0;
  P.M = (int)M;
  P.N = (int)N;
  P.K = (int)up(K, 16);
  mi::int8_forward_plan(P);
  return x_bytes(M, K, x_dtype) + sx_bytes(M, x_dtype) + P.banks * w_bytes(N, K) +
         (P.ks > 1 ? (int64_t)P.ks * P.banks * M * N * 4 : 0);
}
bool aligned(const void* p, int a) { return (uintptr_t)p % a == 0; }
bool rows_on_16(const mi::Int8Params& P) {
  return ((uintptr_t)P.x | (uintptr_t)P.ldx | (uintptr_t)P.w | (uintptr_t)P.w2 | (uintptr_t)P.K) % 16 == 0;
}
// Blocks of a launch, below 2^32 threads.
bool forward_fits(int64_t M, int64_t N) {
  return ((M + 63) / 64) * ((N + 63) / 64) <= kMaxTiles && (M > mi::kInt8FewRows || N <= (int64_t)1 << 26);
}

int forward(mi::Int8Params& P, const void* x, const float* x_scales, int64_t M, int64_t N,
            int64_t K, int x_dtype, int y_dtype, void* ws, int64_t ws_bytes, hipStream_t s) {
  if (int rc = check_sizes(M, N, K)) return rc;
  if (K == 0) return bad("K must be positive");
  P.type = float_type(y_dtype);
  if (P.type < 0) return report_error(MI_ERR_UNSUPPORTED, "y dtype not supported (bfloat16, float16, float32)");
  const int xt = float_type(x_dtype);
  if (xt < 0 && x_dtype != MI_DTYPE_INT8)
    return report_error(MI_ERR_UNSUPPORTED, "x dtype not supported (int8, bfloat16, float16, float32)");
  if (K > mi::kInt8MaxK)
    return report_error(MI_ERR_UNSUPPORTED, "K over 131071: the int32 sums could overflow");
  if (xt >= 0 && x_scales) return bad("x_scales belong to int8 x");
  if (M == 0 || N == 0) return MI_OK;
  if (!forward_fits(M, N)) return report_error(MI_ERR_UNSUPPORTED, "M * N too large for one call");
  if (!P.y || !x || !P.w || !P.sw || (xt < 0 && !x_scales)) return bad("null tensor pointer");
  P.banks = P.w2 ? 2 : 1;
  const int64_t need = forward_need(P, M, N, K, x_dtype);
  if (int rc = check_workspace(ws, ws_bytes, need)) return rc;
  const int a4 = P.type == mi::kF32 ? 16 : 8;
  P.vec = N % 4 == 0 && aligned(P.y, a4) && aligned(P.gate, a4) && aligned(P.up, a4);
  P.vec16 = N % (P.type == mi::kF32 ? 4 : 8) == 0 && aligned(P.y, 16) && aligned(P.gate, 16) && aligned(P.up, 16);
  P.M = (int)M;
  P.N = (int)N;
  P.K = (int)K;
  P.x = (const int8_t*)x;
  P.sx = x_scales;
  P.ldx = K;
  if (fused_token(M, K, x_dtype)) {
    P.xf = x;
    P.xf_type = xt;
    return hip_status(rows_on_16(P) ? mi::launch_int8_gemv(P, s) : mi::launch_int8_any(P, s),
                      "int8 matmul launch");
  }
  const int64_t ld = up(K, 16);
  char* at = (char*)ws;
  hipError_t e = hipSuccess;
  if (xt >= 0) {
    P.x = (const int8_t*)at;
    P.sx = (const float*)(at + x_bytes(M, K, x_dtype));
    P.ldx = ld;
    e = mi::launch_int8_quantize((int8_t*)at, (float*)P.sx, x, M, K, ld, xt, s);
  } else if (ld != K) {
    P.x = (const int8_t*)at;
    P.ldx = ld;
    e = mi::launch_int8_pad((int8_t*)at, (const int8_t*)x, M, K, ld, s);
  }
  at += x_bytes(M, K, x_dtype) + sx_bytes(M, x_dtype);
  if (ld != K) {
    P.K = (int)ld;  // the zeros behind K add nothing
    for (const int8_t** w : {&P.w, &P.w2}) {
      if (e != hipSuccess || !*w) continue;
      e = mi::launch_int8_pad((int8_t*)at, *w, N, K, ld, s);
      *w = (const int8_t*)at;
      at += w_bytes(N, K);
    }
  }
  P.part = (int32_t*)at;
  if (e != hipSuccess) return hip_status(e, "int8 quantize launch");
  return hip_status(!rows_on_16(P) ? mi::launch_int8_any(P, s)
                    : P.nt         ? mi::launch_int8_gemv(P, s)
                                   : mi::launch_int8_gemm(P, s),
                    "int8 matmul launch");
}

// Backward workspace: the fp16 parts of the scaled gradients, [terms * banks][M][np], the rows' powers of two,
// the codes in rows of ldw where K is no multiple of 16, then the ranges' sums of a split product.
int64_t parts_bytes(const mi::Int8BwdParams& B) { return up((int64_t)B.banks * B.terms * B.M * B.np * 2, 256); }
int64_t rows_bytes(const mi::Int8BwdParams& B) { return up((int64_t)B.M * 4, 256); }
int64_t backward_need(mi::Int8BwdParams& B, int64_t M, int64_t N, int64_t K, int banks, int type) {
  if (M == 0 || N == 0 || K == 0) return 0;
  B.banks = banks;
  B.terms = mi::int8_parts(type);
  B.np = (int)up(N, 64);
  B.M = (int)M;
  B.N = (int)N;
  B.K = (int)K;
  B.ldw = (int)up(K, 16);
  B.type = type;
  mi::int8_bwd_plan(B);
  return parts_bytes(B) + rows_bytes(B) + banks * w_bytes(N, K) + (B.ks > 1 ? (int64_t)B.ks * M * B.ldw * 4 : 0);
}

int backward(mi::Int8GradParams& G, mi::Int8BwdParams& B, int64_t M, int64_t N, int64_t K, int dtype,
             int banks, void* ws, int64_t ws_bytes, hipStream_t s) {
  if (int rc = check_sizes(M, N, K)) return rc;
  if (N == 0) return bad("N must be positive");
  const int type = float_type(dtype);
  if (type < 0) return report_error(MI_ERR_UNSUPPORTED, "dtype not supported (bfloat16, float16, float32)");
  if (M == 0 || K == 0) return MI_OK;
  if (!backward_fits(M, N, K))
    return report_error(MI_ERR_UNSUPPORTED, "M * K or the rows too large for one call");
  if (!G.dy || !G.sw || !B.dx || !B.w[0] || (banks == 2 && (!G.gate || !G.up || !G.sw2 || !B.w[1])))
    return bad("null tensor pointer");
  if (!G.dgate != !G.dup) return bad("dgate and dup go together");
  if (int rc = check_workspace(ws, ws_bytes, backward_need(B, M, N, K, banks, type))) return rc;
  G.a = (uint16_t*)ws;
  G.row = (float*)((char*)ws + parts_bytes(B));
  B.a = G.a;
  B.row = G.row;
  char* at = (char*)G.row + rows_bytes(B);
  G.banks = banks;
  G.terms = B.terms;
  G.np = B.np;
  G.M = B.M;
  G.N = B.N;
  G.type = type;
  G.vec = N % (type == mi::kF32 ? 4 : 8) == 0 && aligned(G.dy, 16) && aligned(G.gate, 16) && aligned(G.up, 16) &&
          aligned(G.dgate, 16) && aligned(G.dup, 16) && aligned(G.sw, 16) && aligned(G.sw2, 16);
  B.vec = K % 4 == 0 && aligned(B.dx, type == mi::kF32 ? 16 : 8);
  B.vec16 = K % (type == mi::kF32 ? 4 : 8) == 0 && aligned(B.dx, 16);
  hipError_t e = mi::launch_int8_grad(G, s);
  for (int b = 0; b < banks && B.ldw != K; ++b) {
    if (e == hipSuccess) e = mi::launch_int8_pad((int8_t*)at, B.w[b], N, K, B.ldw, s);
    B.w[b] = (const int8_t*)at;
    at += w_bytes(N, K);
  }
  B.part = (float*)at;
  if (e != hipSuccess) return hip_status(e, "int8 gradient launch");
  const bool fast = ((uintptr_t)B.w[0] | (uintptr_t)B.w[1]) % 16 == 0;
  return hip_status(fast ? mi::launch_int8_bwd(B, s) : mi::launch_int8_bwd_any(B, s), "int8 backward launch");
}

}  // namespace

extern "C" {

int mi_int8_quantize(int8_t* q, float* scales, const void* x, int64_t rows, int64_t K, int x_dtype,
                     void* stream) {
  if (int rc = check_sizes(0, 0, K)) return rc;
  if (rows < 0) return bad("negative size");
  const int type = float_type(x_dtype);
  if (type < 0) return report_error(MI_ERR_UNSUPPORTED, "x dtype not supported (bfloat16, float16, float32)");
  if (K == 0) return bad("K must be positive");
  if (rows == 0) return MI_OK;
  if (!q || !scales || !x) return bad("null tensor pointer");
  return hip_status(mi::launch_int8_quantize(q, scales, x, rows, K, K, type, (hipStream_t)stream),
                    "int8 quantize launch");
}

int64_t mi_int8_forward_workspace(int64_t M, int64_t N, int64_t K, int banks, int x_dtype) {
  if (M < 0 || N < 0 || K < 0 || banks < 1 || banks > 2 || M > kMaxDim || N > kMaxDim ||
      K > mi::kInt8MaxK || !forward_fits(M, N) || (x_dtype != MI_DTYPE_INT8 && float_type(x_dtype) < 0))
    return -1;
  mi::Int8Params P{};
  P.banks = banks;
  return forward_need(P, M, N, K, x_dtype);
}

int64_t mi_int8_backward_workspace(int64_t M, int64_t N, int64_t K, int banks, int dtype) {
  const int type = float_type(dtype);
  if (M < 0 || N < 0 || K < 0 || banks < 1 || banks > 2 || type < 0 || M > kMaxDim || N > kMaxDim ||
      K > kMaxDim || !backward_fits(M, N, K))
    return -1;
  mi::Int8BwdParams B{};
  return backward_need(B, M, N, K, banks, type);
}

int mi_int8_matmul(void* y, const void* x, const float* x_scales, const int8_t* w,
                   const float* w_scales, const void* bias, int64_t M, int64_t N, int64_t K,
                   int x_dtype, int y_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  mi::Int8Params P{};
  P.y = y;
  P.w = w;
  P.sw = w_scales;
  P.bias = bias;
  return forward(P, x, x_scales, M, N, K, x_dtype, y_dtype, workspace, workspace_bytes,
                 (hipStream_t)stream);
}

int mi_int8_gate_up_swiglu(void* y, void* gate, void* up, const void* x, const float* x_scales,
                           const int8_t* w_gate, const float* s_gate, const int8_t* w_up,
                           const float* s_up, int64_t M, int64_t N, int64_t K, int x_dtype,
                           int y_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!gate != !up) return bad("gate and up go together");
  if (M > 0 && N > 0 && (!w_up || !s_up)) return bad("null tensor pointer");
  mi::Int8Params P{};
  P.y = y;
  P.gate = gate;
  P.up = up;
  P.w = w_gate;
  P.sw = s_gate;
  P.w2 = w_up;
  P.sw2 = s_up;
  return forward(P, x, x_scales, M, N, K, x_dtype, y_dtype, workspace, workspace_bytes,
                 (hipStream_t)stream);
}

int mi_int8_matmul_backward(void* dx, const void* dy, const int8_t* w, const float* w_scales,
                            int64_t M, int64_t N, int64_t K, int dtype, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  mi::Int8GradParams G{};
  mi::Int8BwdParams B{};
  G.dy = dy;
  G.sw = w_scales;
  B.dx = dx;
  B.w[0] = w;
  return backward(G, B, M, N, K, dtype, 1, workspace, workspace_bytes, (hipStream_t)stream);
}

int mi_int8_gate_up_swiglu_backward(void* dx, void* dgate, void* dup, const void* dy,
                                    const void* gate, const void* up, const int8_t* w_gate,
                                    const float* s_gate, const int8_t* w_up, const float* s_up,
                                    int64_t M, int64_t N, int64_t K, int dtype, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  mi::Int8GradParams G{};
  mi::Int8BwdParams B{};
  G.dy = dy;
  G.gate = gate;
  G.up = up;
  G.sw = s_gate;
  G.sw2 = s_up;
  G.dgate = dgate;
  G.dup = dup;
  B.dx = dx;
  B.w[0] = w_gate;
  B.w[1] = w_up;
  return backward(G, B, M, N, K, dtype, 2, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
