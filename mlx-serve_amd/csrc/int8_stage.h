// Staging helpers of the int8 matrix kernels: buffer loads into LDS, waits, the row swizzle.
#pragma once
#include "int8.h"
#include "qmv_common.h"

namespace mi {
namespace i8 {

using qmv_detail::vmcnt_imm;

constexpr int kBufFlags = 0x00020000;   // raw dword access
constexpr uint32_t kOOB = 0x7FFFFFF0u;  // past any resource: the load returns 0
// XOR swizzle of the 16-byte slots of a 128-byte row. A ds_read_b128 pass serves lanes 0-3, 12-15,
// 20-23 and 24-27 of a half together: rows 0-3 and 12-15 of quarter q, 4-11 of quarter q + 1.
// With slots 2q + e these keep apart.
MI_DEV int xswz(int r) { return (r & 2) | ((r >> 2) & 1) | ((r >> 1) & 4); }

MI_DEV void dma16(__amdgpu_buffer_rsrc_t rs, unsigned char* lds, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16,
                                           voff, soff, 0, 0);
}
MI_DEV void dma4(__amdgpu_buffer_rsrc_t rs, unsigned char* lds, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 4,
                                           voff, soff, 0, 0);
}
MI_DEV __amdgpu_buffer_rsrc_t rsrc(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, kBufFlags);
}

// s_waitcnt vmcnt(n); n is a constant after inlining
MI_DEV void wait_vm(int n) {
  switch (n) {
#define C(n) case n: __builtin_amdgcn_s_waitcnt(vmcnt_imm(n)); break;
    C(1) C(2) C(3) C(4) C(5) C(6) C(7) C(8) C(9) C(10) C(11) C(12) C(13) C(14) C(15) C(16) C(17)
    C(18) C(19) C(20) C(21) C(22) C(23) C(24) C(25) C(26) C(27) C(28)
    default: __builtin_amdgcn_s_waitcnt(vmcnt_imm(0)); break;
#undef C
  }
}


// A tile of the matrix kernels for their plans: microseconds a step of a block that has its CU to
// itself, of two that share it (0: a block fills the CU), and beside the steps (start, end).
struct TileCost {
  int bm, bn;
  double alone, paired, ends;
};
// `tiles` blocks of `steps` steps on 256 CUs
inline double tile_us(const TileCost& t, int64_t tiles, int steps) {
  const int64_t per_cu = (tiles + 255) / 256;
  const double one = steps * t.alone + t.ends;
  if (t.paired == 0.0) return (double)per_cu * one;
  return (double)(per_cu / 2) * (steps * t.paired + t.ends) + (per_cu % 2 ? one : 0.0);
}

}  // namespace i8
}  // namespace mi
