// Dropout whose mask is never stored: y = r + x / (share kept) where an element stays, r where it does not.  The gradient is the same call on d y.
// Bound by HBM: bf16 16384 x 4096 onto a residual 75 us, 5.4 TB/s (some of it from the last cache), arithmetic 41 % busy; fp32 7331 x 515 8.3 us with the launch.
#include "dropout.h"

namespace cavs {
namespace {

// Rows are pieces of eight columns; a workgroup has whole rows of about kItems pieces (of wide rows one), four of a lane's on their way at a time.
constexpr int kItems = 1024, kAtOnce = 4;

template <class T>
struct DropArgs {
  T *y;
  const T *x, *r;
  long ldy, ldx, ldr;
  int n, w, pieces, rows;  // pieces of a row, rows of a workgroup
  Mask m;
};

template <class T, bool ADD>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs<T> a) {
  const int row0 = blockIdx.x * a.rows, rows = min(a.rows, a.n - row0);
  const int down = 256 / a.pieces, across = 256 - down * a.pieces;
  const unsigned long long step = step_of(a.m);
  int row = threadIdx.x / a.pieces, piece = threadIdx.x - row * a.pieces;
  while (row < rows) {
    int at[kAtOnce], of[kAtOnce];
    Eight<T> x[kAtOnce], r[kAtOnce];
    unsigned id[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) {
      at[k] = row, of[k] = piece;
      if (row < rows) {
        const int left = a.w - 8 * piece;
        x[k].load(a.x + (row0 + row) * a.ldx + 8 * piece, left);
        if constexpr (ADD) r[k].load(a.r + (row0 + row) * a.ldr + 8 * piece, left);
        id[k] = row_id(a.m, row0 + row);
      }
      row += down, piece += across;
      if (piece >= a.pieces) piece -= a.pieces, row++;
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) {
      if (at[k] >= rows) break;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = x[k][e];
      drop8(a.m, draws_of(a.m, step, id[k], of[k]), v);
      if constexpr (ADD) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += r[k][e];
      }
      Eight<T>::store(a.y + (row0 + at[k]) * a.ldy + 8 * of[k], v, a.w - 8 * of[k]);
    }
  }
}

template <class T>
int run_dropout(void *y, int ldy, const void *x, int ldx, const void *r, int ldr, int n, int w, const Mask &m, hipStream_t st) {
  DropArgs<T> a{static_cast<T *>(y), static_cast<const T *>(x), static_cast<const T *>(r), ldy, ldx, ldr, n, w, (int)(((long)w + 7) / 8), 1, m};
  // (few rows: as many workgroups as there are rows or compute units)
  const long per = ((long)n * a.pieces + num_cus() - 1) / num_cus(), items = per < kItems ? per : kItems;
  const long rows = items / a.pieces, least = (n + (long)most_groups(256) - 1) / most_groups(256);
  a.rows = (int)(rows > least ? rows : least);
  const unsigned groups = (unsigned)((n + (long)a.rows - 1) / a.rows);
  launch(r ? dropout_kernel<T, true> : dropout_kernel<T, false>, groups, 256, 0, st, a);
  CAVS_LAUNCH_CHECK();
  return CAVS_OK;
}

__global__ void advance_kernel(unsigned long long *word, unsigned long long by) { *word += by; }

}  // namespace
}  // namespace cavs

using namespace cavs;

extern "C" {

int cavs_dropout(int type, void *y, int ldy, const void *x, int ldx, const void *r, int ldr, int n, int w, const cavs_dropout_mask *mask, void *stream) {
  CAVS_REQUIRE(type == CAVS_F32 || type == CAVS_BF16, "cavs_dropout: type %d is neither CAVS_F32 nor CAVS_BF16", type);
  CAVS_REQUIRE(n >= 0 && w > 0, "cavs_dropout: bad shape n=%d w=%d", n, w);
  CAVS_REQUIRE(ldy >= w && ldx >= w && (!r || ldr >= w), "cavs_dropout: a row stride is below w=%d", w);
  CAVS_REQUIRE(mask && (n == 0 || (y && x)), "cavs_dropout: null pointer");
  Mask m;
  CAVS_REQUIRE(mask_of(mask, &m), "cavs_dropout: p is not in [0, 1)");
  if (n == 0) return CAVS_OK;
  return (type == CAVS_F32 ? run_dropout<float> : run_dropout<u16>)(y, ldy, x, ldx, r, ldr, n, w, m, as_stream(stream));
}

int cavs_dropout_advance(unsigned long long *step_word, unsigned long long by, void *stream) {
  CAVS_REQUIRE(step_word, "cavs_dropout_advance: null pointer");
  launch(advance_kernel, 1, 1, 0, as_stream(stream), step_word, by);
  CAVS_LAUNCH_CHECK();
  return CAVS_OK;
}

}  // extern "C"
