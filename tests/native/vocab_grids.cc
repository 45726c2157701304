// Host-only: the grids that calls of cavs_vocab_xent* would launch, over the corners of what they accept and sizes between.  Prints those whose threads reach
// 2^32 along a dimension, and how many calls were looked at.  (The launch itself is replaced: nothing runs.)
#include <cstdio>
#include <cstdlib>
#include <string>

#include "common.h"

namespace {
int bad = 0;
std::string call;
template <typename K, typename... Args>
void seen(K, dim3 grid, dim3 block, size_t, hipStream_t, Args &&...) {
  const unsigned long long t[3] = {1ull * grid.x * block.x, 1ull * grid.y * block.y, 1ull * grid.z * block.z};
  if (t[0] >> 32 || t[1] >> 32 || t[2] >> 32 || !t[0] || !t[1] || grid.y > 65535 || grid.z > 65535) {
    bad++;
    std::printf("%s: grid %u %u %u of %u\n", call.c_str(), grid.x, grid.y, grid.z, block.x);
  }
}
}  // namespace
#define launch seen
#include "vocab_xent.hip"
#undef launch

int main() {
  const int ns[] = {1, 64, 65, 256, 257, 1 << 14, (1 << 20) - 64, 1 << 20}, hs[] = {1, 64, 4096, (1 << 16) - 64, 1 << 16},
            cs[] = {1, 300, 32767, 300000, 525001, (1 << 20) + 1, 1 << 23};
  int calls = 0;
  char *some = nullptr;  // (addresses that nothing reads)
  some += 4096;
  float *f = reinterpret_cast<float *>(some);
  for (int type : {CAVS_F32, CAVS_BF16})
    for (int n : ns)
      for (int H : hs)
        for (int C : cs)
          for (int what = 0; what < 3; what++) {
            const size_t bytes = cavs_vocab_xent_workspace(type, n, H, C, what > 0);
            // (more than a device of 288 GB holds beside its operands: no such call can be made)
            const double size = type == CAVS_F32 ? 4 : 2;
            if (bytes == 0 || bytes + size * ((double)n * H + (double)C * H) > 288e9) continue;
            call = "type " + std::to_string(type) + " n " + std::to_string(n) + " H " + std::to_string(H) + " C " + std::to_string(C) + " call " + std::to_string(what);
            if (what == 0) cavs_vocab_xent_fwd(type, some, H, some, H, f, f, f, f, n, H, C, some, bytes, nullptr);
            else if (what == 1) cavs_vocab_xent(type, some, H, some, H, f, f, f, 1.f, f, f, some, H, some, H, f, n, H, C, some, bytes, nullptr);
            else cavs_vocab_xent_bwd(type, some, H, some, H, f, f, f, f, 1.f, some, H, some, H, f, n, H, C, some, bytes, nullptr);
            calls++;
          }
  std::printf("%d calls, %d grids too large\n", calls, bad);
  return bad != 0;
}
