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


// A block's finished tile to memory through LDS, in rows of COLS values of ESZ bytes: stored straight
// from the products' layout, a wave writes 32 bytes of each of 16 rows at a time: 2003 rows of gate + up
// [14336,4096] with both projections kept took 296 us, this way 255. Waves 2 x 4 with MT tiles of 16 rows and
// TA tiles of 16 columns each; value(i, a, v) gives OUT x 4 values of the lane's row and columns.
// Passes of 32 IC rows, so that OUT of them fit the staging LDS (its DMA has landed and its reads
// are done, in every wave, after the first barrier). Rows of `out` on 16 bytes.
template <int ESZ, int MT, int TA, int OUT, int LDS, class V>
MI_DEV void store_tile(unsigned char* smem, void* const (&out)[OUT], int type, int M, int N, int m0, int n0,
                       V value) {
  constexpr int IC = MT < 8 / ESZ ? MT : 8 / ESZ;  // 4 (16-bit) or 2
  constexpr int kCols = 64 * TA, kPitch = kCols * ESZ + 16, kRows = 32 * IC;
  constexpr int kChunks = kCols * ESZ / 16;
  static_assert(OUT * kRows * kPitch <= LDS && kRows * kChunks % 512 == 0 && MT % IC == 0, "a pass fits");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave >> 2, wn = wave & 3, fr = lane & 15, q = lane >> 4;
#pragma unroll
  for (int i0 = 0; i0 < MT; i0 += IC) {
    lds_sync();
#pragma unroll
    for (int i = 0; i < IC; ++i)
#pragma unroll
      for (int a = 0; a < TA; ++a) {
        float v[OUT][4];
        value(i0 + i, a, v);
#pragma unroll
        for (int o = 0; o < OUT; ++o) {
          unsigned char* p = smem + (o * kRows + 16 * (wm * IC + i) + fr) * kPitch + (16 * (wn * TA + a) + 4 * q) * ESZ;
          if constexpr (ESZ == 4) {
            *reinterpret_cast<f32x4_t*>(p) = f32x4_t{v[o][0], v[o][1], v[o][2], v[o][3]};
          } else {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              b[j] = type == kBF16 ? f32_to_bf16_bits(v[o][j])
                                   : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[o][j]);
            *reinterpret_cast<u32x2_t*>(p) = u32x2_t{b[0] | b[1] << 16, b[2] | b[3] << 16};
          }
        }
      }
    lds_sync();
#pragma unroll
    for (int o = 0; o < OUT; ++o)
#pragma unroll
      for (int k = 0; k < kRows * kChunks / 512; ++k) {
        const int at = tid + 512 * k, r = at / kChunks, c = at % kChunks;
        const int m = m0 + 16 * (r / (16 * IC) * MT + i0 + r / 16 % IC) + r % 16, n = n0 + c * (16 / ESZ);
        if (m < M && n < N)
          *reinterpret_cast<u32x4_t*>((unsigned char*)out[o] + ((int64_t)m * N + n) * ESZ) =
              *reinterpret_cast<const u32x4_t*>(smem + (o * kRows + r) * kPitch + c * 16);
      }
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

// Whole rounds of big tiles and, for what is left of the last one, small tiles in a launch of their own:
// the column tiles at the end that those take, 0 where it would not pay. `ct` column tiles of `big`
// (256 rows) and `small` (128) alike.
inline int tail_columns(const TileCost& big, const TileCost& small, int64_t M, int64_t ct, int steps, double* us) {
  const int64_t bt = (M + 255) / 256, st = (M + 127) / 128, rounds = bt * ct / 256;
  if (rounds < 1 || bt * ct % 256 == 0 || bt > 256) return 0;
  const int64_t tail = ct - rounds * 256 / bt;
  const double cost = tile_us(big, bt * (ct - tail), steps) + tile_us(small, st * tail, steps) + 2.0;
  if (cost >= *us) return 0;
  *us = cost;
  return (int)tail;
}

}  // namespace i8
}  // namespace mi
