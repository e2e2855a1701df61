// Which kernels an int8 call takes on aligned tensors, from the library's own plans: reads lines
//   f <banks> <rows come as floats of so many bytes, or 0> <M> <N> <K>     forward
//   b <banks> <bytes of a gradient> <M> <N> <K>                            backward
// and prints a line for each, the launches of a call behind one another:
//   token <vectors>             one token quantized in the launch of the few-row kernel
//   few <x tiles> <w tiles>     the few-row kernel
//   tile <rows> <columns> <whole | split | tail>[ ahead]
#include <cstdio>
#include <cstring>

#include "int8.h"

static void tiles(int M, int columns, int bm, int bn, int on, int ks, int tail, bool ahead_kernels) {
  const int ct = (columns + on - 1) / on;
  const long blocks = (long)((M + bm - 1) / bm) * (ct - tail) * ks;
  const bool two = (bm == 256 && bn == 256) || (bm == 128 && bn == 128);  // rings of two stages
  std::printf("tile %d %d %s%s", bm, bn, ks > 1 ? "split" : "whole", ahead_kernels && two && blocks <= 256 ? " ahead" : "");
  if (tail) std::printf(", tile 128 256 tail");
}

int main() {
  char way;
  int banks, bytes, M, N, K;
  while (std::scanf(" %c %d %d %d %d %d", &way, &banks, &bytes, &M, &N, &K) == 6) {
    std::printf("%d: ", banks);
    if (way == 'f') {
      mi::Int8Params P{};
      const int type = bytes == 4 ? mi::kF32 : mi::kBF16;
      if (bytes && mi::int8_gemv_fuses(M, K, type)) {
        std::printf("token %d\n", K * bytes <= 8192 ? 1 : 4);
        continue;
      }
      P.M = M, P.N = N, P.K = (K + 15) / 16 * 16, P.banks = banks;
      mi::int8_forward_plan(P);
      if (P.nt) {
        const int t = (M + 15) / 16;
        std::printf("few %d %d", t <= 4 ? t : t <= 6 ? 6 : 8, P.nt);
      } else {
        tiles(M, N, P.bm, P.bn, P.bn / banks, P.ks, P.tail, true);
      }
    } else {
      mi::Int8BwdParams P{};
      P.banks = banks, P.terms = mi::int8_parts(bytes == 4 ? mi::kF32 : mi::kBF16);
      P.np = (N + 63) / 64 * 64, P.M = M, P.N = N, P.K = K, P.ldw = (K + 15) / 16 * 16;
      mi::int8_bwd_plan(P);
      tiles(M, K, P.bm, P.bn, P.bn, P.ks, P.tail, false);
    }
    std::printf("\n");
  }
  return 0;
}
