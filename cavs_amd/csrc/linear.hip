// Y = R + drop(act(X W^T + b)) and its gradients: products with everything that follows them in their epilogue.
//
//   forward   Z = X W^T + b, Y = R + drop(act(Z))
//   backward  D = drop(dY . act'(Z)), dX = D W, dW = D^T X, db = sums of D's columns
//
// Tiles are made of the transposed product, so that a lane of the 32x32 instruction holds neighbouring values of a row of the result: after an
// exchange with the lane 32 away eight of them, which is what bias, residual and results are read and written in, and what one call of the dropout's
// generator is for.
//
// Measured, whole calls: bf16 8192 x 8192 x 4096 onto a residual with dropout 386 us, 1420 TFLOP/s (matrix pipe 72 % busy at the clock power leaves, 1.83 GHz); gradients of
// 4096 x 2048 x 8192 through gelu and dropout 245 (products 198, 1390 TFLOP/s; D 50); fp32 gradients of 7088 x 512 x 2048 194 (products 140, 212 TFLOP/s of fp32;
// packing 45; joining parts 12); one token of 2048 x 8192 in bf16 8.6, 3.9 TB/s. Gradients' products are bound by the matrix pipe, D and packing by HBM, few rows by W's bytes.
#include <cmath>

#include "activations.h"
#include "direct_product.h"
#include "dropout.h"

namespace cavs {
namespace {

// ------------------------------------------------------------------ epilogues: eight neighbouring values of a row of the result
// What they read of a row is asked for before any of it is made (hold), where the tile lies inside the result without a look at where it ends.
template <class T>
struct Forward {
  static constexpr bool FAST = sizeof(T) == 2;
  const float *bias;
  int act;
  Mask m;
  const T *R;
  long ldr;
  T *Z;
  long ldz;
  T *Y;
  long ldy;
  typedef Eight<T> Held;
  __device__ __forceinline__ void hold(Held &r, int row, int col, int left) const {
    r.zero();
    if (R) r.load(R + row * ldr + col, left);
  }
  __device__ __forceinline__ void hold_whole(Held &r, int row, int col) const {
    if (R) r.load(R + row * ldr + col);
    else r.zero();
  }
  // bias: of the eight columns, or null
  __device__ __forceinline__ void finish(unsigned long long step, unsigned id, const float *b, const Held &r, int row, int col, int left, float (&v)[8]) const {
    if (b) {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += b[e];
    }
    if (Z) Eight<T>::store(Z + row * ldz + col, v, left);
    if (act) {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = act_of<FAST>(act, v[e]);
    }
    if (m.t) drop8(m, draws_of(m, step, id, col >> 3), v);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] += r[e];
    Eight<T>::store(Y + row * ldy + col, v, left);
  }
  __device__ __forceinline__ const float *biases() const { return bias; }
  __device__ __forceinline__ unsigned long long step() const { return step_of(m); }
  __device__ __forceinline__ unsigned id(int row) const { return m.t ? row_id(m, row) : 0u; }
};
template <class T>
struct Plain {
  T *Y;
  long ldy;
  struct Held {};
  __device__ __forceinline__ void hold(Held &, int, int, int) const {}
  __device__ __forceinline__ void hold_whole(Held &, int, int) const {}
  __device__ __forceinline__ void finish(unsigned long long, unsigned, const float *, const Held &, int row, int col, int left, float (&v)[8]) const {
    Eight<T>::store(Y + row * ldy + col, v, left);
  }
  __device__ __forceinline__ const float *biases() const { return nullptr; }
  __device__ __forceinline__ unsigned long long step() const { return 0; }
  __device__ __forceinline__ unsigned id(int) const { return 0; }
};

// A tile's biases in LDS (of its columns, 0 beyond the last), written before the product and read behind its barriers
template <int BM, class E>
__device__ __forceinline__ void keep_biases(const E &out, float *kept, int m0, int cols) {
  const float *b = out.biases();
  if (!b) return;
  for (int i = threadIdx.x; i < BM; i += blockDim.x) kept[i] = m0 + i < cols ? b[m0 + i] : 0.f;
}
// pieces i < I, j < J of a wavefront's tile: col(i), row(j) within the tile at m0, n0; values(i, j, v)
template <int I, int J, int BM, int BN, class E, class Row, class Col, class Values>
__device__ __forceinline__ void finish_tile(const E &out, const float *kept, int m0, int n0, int cols, int rows, Row &&row, Col &&col, Values &&values) {
  const float *b = out.biases() ? kept : nullptr;
  const unsigned long long step = out.step();
  if (m0 + BM <= cols && n0 + BN <= rows) {
#pragma unroll
    for (int j = 0; j < J; j++) {
      const int r = n0 + row(j);
      const unsigned id = out.id(r);
      typename E::Held held[I];
#pragma unroll
      for (int i = 0; i < I; i++) out.hold_whole(held[i], r, m0 + col(i));
#pragma unroll
      for (int i = 0; i < I; i++) {
        float v[8];
        values(i, j, v);
        out.finish(step, id, b ? b + col(i) : nullptr, held[i], r, m0 + col(i), 8, v);
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < J; j++) {
    const int r = n0 + row(j);
    const unsigned id = r < rows ? out.id(r) : 0u;
#pragma unroll
    for (int i = 0; i < I; i++) {
      float v[8];
      values(i, j, v);  // (an exchange between lanes: all of them take part)
      const int c = m0 + col(i);
      if (r >= rows || c >= cols) continue;
      typename E::Held held;
      out.hold(held, r, c, cols - c);
      out.finish(step, id, b ? b + col(i) : nullptr, held, r, c, cols - c, v);
    }
  }
}

// ------------------------------------------------------------------ operands, packed (nt_product.h)
template <class T>
struct PackJob {
  const T *src;
  long ld;
  int rows, K, orows;  // orows: rows of o, zero beyond those of src
  PackedOut o;
  int across, blocks;  // blocks of 64 columns, of 64 x 64
};
template <int P, class T>
__device__ __forceinline__ void pack_block(const PackJob<T> &g, int block, PackTile &tile) {
  const int r0 = block / g.across * 64, k0 = block % g.across * 64;
  load_tile(tile, g.src, g.ld, r0, k0, g.rows, g.K);
  __syncthreads();
  pack_tile<P>(tile, g.o, PackedOut{}, r0, k0, g.orows, g.K);
}
template <int P, class T>
__global__ __launch_bounds__(256) void pack_kernel(PackJob<T> j0, PackJob<T> j1) {
  __shared__ PackTile tile;
  const int block = blockIdx.y * gridDim.x + blockIdx.x;
  if (block < j0.blocks) pack_block<P>(j0, block, tile);
  else if (block < j0.blocks + j1.blocks) pack_block<P>(j1, block - j0.blocks, tile);
}

// D packed, and sums of its columns over 64 rows each [blocks of rows][N]
template <class T>
struct GradJob {
  const T *dY, *Z;
  long lddy, ldz;
  int act;
  Mask m;
  int n, N, orows, across, blocks;
  PackedOut o;
  float *sums;
};
// and X and W packed, behind it
template <int P, class T>
__global__ __launch_bounds__(256) void grad_kernel(GradJob<T> g, PackJob<T> x, PackJob<T> w) {
  __shared__ PackTile tile;
  __shared__ float part[4][64];
  const int block = blockIdx.y * gridDim.x + blockIdx.x;
  if (block >= g.blocks) {
    if (block < g.blocks + x.blocks) pack_block<P>(x, block - g.blocks, tile);
    else if (block < g.blocks + x.blocks + w.blocks) pack_block<P>(w, block - g.blocks - x.blocks, tile);
    return;
  }
  const int r0 = block / g.across * 64, k0 = block % g.across * 64, piece = threadIdx.x & 7;
  const unsigned long long step = step_of(g.m);
#pragma unroll
  for (int q = 0; q < 2; q++) {
    const int r = (threadIdx.x >> 3) + 32 * q, row = r0 + r, col = k0 + 8 * piece, left = row < g.n ? g.N - col : 0;
    Eight<T> d, z;
    d.zero(), z.zero();
    if (left > 0) {
      d.load(g.dY + row * g.lddy + col, left);
      if (g.act) z.load(g.Z + row * g.ldz + col, left);
    }
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = g.act ? d[e] * slope_of<P == 1>(g.act, z[e]) : d[e];
    if (g.m.t && left > 0) drop8(g.m, draws_of(g.m, step, row_id(g.m, row), col >> 3), v);
#pragma unroll
    for (int e = 0; e < 8; e++) tile[r][8 * piece + e] = e < left ? v[e] : 0.f;
  }
  __syncthreads();
  if (g.o.p) pack_tile<P>(tile, g.o, PackedOut{}, r0, k0, g.orows, g.N);
  if (!g.sums) return;
  const int c = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i++) s += tile[16 * wave + i][c];
  part[wave][c] = s;
  __syncthreads();
  if (wave == 0 && k0 + c < g.N) g.sums[(long)(r0 / 64) * g.N + k0 + c] = (part[0][c] + part[1][c]) + (part[2][c] + part[3][c]);
}

// sums of columns that launches before left over 64 rows each, 64 columns a workgroup, of its first four wavefronts
struct ColumnsJob {
  const float *part;
  int parts, cols;
  float *out;
  int blocks;  // 0: none
};
__device__ __forceinline__ void sum_columns(const ColumnsJob &g, int block, float (*each)[64]) {
  const int c = block * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6, per = (g.parts + 3) / 4, end = min(g.parts, (w + 1) * per);
  float s = 0.f;
  if (w < 4 && c < g.cols)
    for (int p = w * per; p < end; p += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = p + k < end ? g.part[(long)(p + k) * g.cols + c] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; k++) s += v[k];
    }
  if (w < 4) each[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && c < g.cols) g.out[c] = (each[0][threadIdx.x] + each[1][threadIdx.x]) + (each[2][threadIdx.x] + each[3][threadIdx.x]);
}

// ------------------------------------------------------------------ products of packed operands
// result[row, col] = sum over k of A[col, k] B[row, k].  K in `splits` stretches of kchunk, each with sums of its own at part + split * rows * cols; part
// null: straight to the epilogue.
template <class E>
struct Product {
  PackedRef A, B;
  int cols, rows, K, tilesM, tilesN, kchunk;
  float *part;
  E out;
};

// The eight values of block 8 q of a row, q = 0 .. 3 of the 32 columns of a tile of accumulators: lanes below 32 have q = 2 pair, the others 2 pair + 1
__device__ __forceinline__ void exchanged(const floatx16 &t, int pair, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(t[8 * pair + i]), __float_as_uint(t[8 * pair + 4 + i]), false, false);
    v[i] = __uint_as_float(x[0]);
    v[4 + i] = __uint_as_float(x[1]);
  }
}

template <class T, class E>
__device__ __forceinline__ void finish_packed(const Product<E> &g, int split, const float *kept, int m0, int n0, floatx16 (&acc)[T::ACC][T::TM][T::TN]) {
  if constexpr (T::ACC > 1) {
#pragma unroll
    for (int i = 0; i < T::TM; i++)
#pragma unroll
      for (int j = 0; j < T::TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[0][i][j][r] += acc[T::ACC - 1][i][j][r];
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const auto col = [&](int i) { return wave / T::WGN * T::WM + 16 * i + 8 * (lane >> 5); };
  const auto row = [&](int j) { return wave % T::WGN * T::WN + 32 * j + (lane & 31); };
  const auto values = [&](int i, int j, float (&v)[8]) { exchanged(acc[0][i >> 1][j], i & 1, v); };
  if (g.part) {
    const Plain<float> part{g.part + (long)split * g.rows * g.cols, g.cols};
    finish_tile<2 * T::TM, T::TN, T::BM, T::BN>(part, kept, m0, n0, g.cols, g.rows, row, col, values);
  } else {
    finish_tile<2 * T::TM, T::TN, T::BM, T::BN>(g.out, kept, m0, n0, g.cols, g.rows, row, col, values);
  }
}
template <class E>
__device__ __forceinline__ void tile_at(const Product<E> &g, int block, int bm, int bn, int *split, int *m0, int *n0, int *kbeg, int *kend) {
  const int tiles = g.tilesM * g.tilesN;
  *split = block / tiles;
  nt_tile_of(block - *split * tiles, g.tilesM, g.tilesN, m0, n0);
  *m0 *= bm, *n0 *= bn;
  *kbeg = *split * g.kchunk, *kend = min(g.K, *kbeg + g.kchunk);
}

template <class T, class E>
__global__ __launch_bounds__(T::THREADS, T::EU) void packed_forward_kernel(Product<E> g) {
  // (one array: of two the compiler no longer knows that the pieces are not what is on its way from memory, and waits: direct_forward_kernel of
  // 8192 x 8192 x 4096 924 us, 394 so)
  __shared__ __attribute__((aligned(16))) char S[T::LDS + T::BM * 4];
  float *kept = reinterpret_cast<float *>(S + T::LDS);
  int split, m0, n0, kbeg, kend;
  tile_at(g, blockIdx.x, T::BM, T::BN, &split, &m0, &n0, &kbeg, &kend);
  floatx16 acc[T::ACC][T::TM][T::TN];
  if (!g.part) keep_biases<T::BM>(g.out, kept, m0, g.cols);
  nt_multiply<T, false, false>(g.A, g.cols, m0, g.B, g.rows, n0, kbeg, kend, S, acc);
  finish_packed<T>(g, split, kept, m0, n0, acc);
}
// Both gradients in a launch, so that the compute units whose last tile of the one has ended go on with the other: dX = D W (its A turned) and dW = D^T X (both
// turned), `wfirst`: dW is j0.  Behind them db, which waits for no more than they do (in a launch of its own 5 us more).
template <class T, class E>
__global__ __launch_bounds__(T::THREADS, T::EU) void packed_back_kernel(Product<E> j0, Product<E> j1, int blocks0, int blocks, int wfirst, ColumnsJob b) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS];
  if ((int)blockIdx.x >= blocks) {
    sum_columns(b, blockIdx.x - blocks, reinterpret_cast<float(*)[64]>(S));
    return;
  }
  const bool second = (int)blockIdx.x >= blocks0;
  const Product<E> &g = second ? j1 : j0;
  int split, m0, n0, kbeg, kend;
  tile_at(g, second ? blockIdx.x - blocks0 : blockIdx.x, T::BM, T::BN, &split, &m0, &n0, &kbeg, &kend);
  floatx16 acc[T::ACC][T::TM][T::TN];
  if (second != (wfirst != 0)) nt_multiply<T, true, true>(g.A, g.cols, m0, g.B, g.rows, n0, kbeg, kend, S, acc);
  else nt_multiply<T, true, false>(g.A, g.cols, m0, g.B, g.rows, n0, kbeg, kend, S, acc);
  finish_packed<T>(g, split, nullptr, m0, n0, acc);
}

// ------------------------------------------------------------------ products of operands as they lie (direct_product.h)
template <class E>
struct DirectJob {
  DirectRef A, B;
  int cols, rows, K, tilesM, tilesN, kchunk;
  float *part;
  E out;
};
template <class E>
__device__ __forceinline__ void tile_at(const DirectJob<E> &g, int block, int bm, int bn, int *split, int *m0, int *n0, int *kbeg, int *kend) {
  const int tiles = g.tilesM * g.tilesN;
  *split = block / tiles;
  nt_tile_of(block - *split * tiles, g.tilesM, g.tilesN, m0, n0);
  *m0 *= bm, *n0 *= bn;
  *kbeg = *split * g.kchunk, *kend = min(g.K, *kbeg + g.kchunk);
}
template <class T, class E>
__device__ __forceinline__ void finish_direct(const DirectJob<E> &g, int split, const float *kept, int m0, int n0, const floatx4 (&acc)[T::I][2 * T::J]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const auto col = [&](int i) { return T::col(wave, lane, i); };
  const auto row = [&](int j) { return T::row(wave, lane, j); };
  const auto values = [&](int i, int j, float (&v)[8]) { eight_columns(acc[i][2 * j], acc[i][2 * j + 1], v); };
  if (g.part) {
    const Plain<float> part{g.part + (long)split * g.rows * g.cols, g.cols};
    finish_tile<T::I, T::J, T::BM, T::BN>(part, kept, m0, n0, g.cols, g.rows, row, col, values);
  } else {
    finish_tile<T::I, T::J, T::BM, T::BN>(g.out, kept, m0, n0, g.cols, g.rows, row, col, values);
  }
}
template <class T, class E>
__global__ __launch_bounds__(T::THREADS, T::EU) void direct_forward_kernel(DirectJob<E> g) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS + T::BM * 4];
  float *kept = reinterpret_cast<float *>(S + T::LDS);
  int split, m0, n0, kbeg, kend;
  tile_at(g, blockIdx.x, T::BM, T::BN, &split, &m0, &n0, &kbeg, &kend);
  floatx4 acc[T::I][2 * T::J];
  if (!g.part) keep_biases<T::BM>(g.out, kept, m0, g.cols);
  direct_multiply<false, false>(T{}, g.A, g.cols, m0, g.B, g.rows, n0, kbeg, kend, S, acc);
  finish_direct<T>(g, split, kept, m0, n0, acc);
}
// (as packed_back_kernel)
template <class T, class E>
__global__ __launch_bounds__(T::THREADS, T::EU) void direct_back_kernel(DirectJob<E> j0, DirectJob<E> j1, int blocks0, int blocks, int wfirst, ColumnsJob b) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS];
  if ((int)blockIdx.x >= blocks) {
    sum_columns(b, blockIdx.x - blocks, reinterpret_cast<float(*)[64]>(S));
    return;
  }
  const bool second = (int)blockIdx.x >= blocks0;
  const DirectJob<E> &g = second ? j1 : j0;
  int split, m0, n0, kbeg, kend;
  tile_at(g, second ? blockIdx.x - blocks0 : blockIdx.x, T::BM, T::BN, &split, &m0, &n0, &kbeg, &kend);
  floatx4 acc[T::I][2 * T::J];
  if (second != (wfirst != 0)) direct_multiply<true, true>(T{}, g.A, g.cols, m0, g.B, g.rows, n0, kbeg, kend, S, acc);
  else direct_multiply<true, false>(T{}, g.A, g.cols, m0, g.B, g.rows, n0, kbeg, kend, S, acc);
  finish_direct<T>(g, split, nullptr, m0, n0, acc);
}

// D is rounded to bf16 before its two products, once (here and in grad_kernel<1>): what bf16 leaves off would be a second part in both, twice the instructions of the
// matrix pipe, which has 198 of the 245 us of 4096 x 2048 x 8192.  There dX and dW are off by 0.00235 of their norm with it, by 0.00166, their own rounding,
// without.  db is summed before it.
// D as it lies (write: bf16, rows of N), and sums of its columns over 64 rows each [stretches of rows][N]; 256 columns a workgroup
__global__ __launch_bounds__(256) void grad_rows_kernel(GradJob<u16> g, u16 *D) {
  __shared__ float part[8][256];
  const int block = blockIdx.y * gridDim.x + blockIdx.x;
  if (block >= g.blocks) return;
  const int piece = threadIdx.x & 31, line = threadIdx.x >> 5, r0 = block / g.across * 64, col = block % g.across * 256 + 8 * piece;
  const int left = g.N - col;
  const unsigned long long step = step_of(g.m);
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (left > 0) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
      Eight<u16> d[4], z[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int row = min(r0 + line + 8 * (4 * q + i), g.n - 1);  // (N is whole pieces here)
        d[i].load(g.dY + row * g.lddy + col);
        if (g.act) z[i].load(g.Z + row * g.ldz + col);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int row = r0 + line + 8 * (4 * q + i);
        if (row >= g.n) break;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = d[i][e];
        if (g.act) {
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] *= slope_of<true>(g.act, z[i][e]);
        }
        if (g.m.t) drop8(g.m, draws_of(g.m, step, row_id(g.m, row), col >> 3), v);
#pragma unroll
        for (int e = 0; e < 8; e++) s[e] += v[e];
        if (D) Eight<u16>::store(D + (long)row * g.N + col, v, 8);
      }
    }
  }
  if (!g.sums) return;
#pragma unroll
  for (int e = 0; e < 8; e++) part[line][8 * piece + e] = s[e];
  __syncthreads();
  const int c = block % g.across * 256 + threadIdx.x;
  if (c >= g.N) return;
  float t = part[0][threadIdx.x];
#pragma unroll
  for (int i = 1; i < 8; i++) t += part[i][threadIdx.x];
  g.sums[(long)(r0 / 64) * g.N + c] = t;
}

// ------------------------------------------------------------------ few rows: W read once, where it lies
// A workgroup makes sixteen columns of the result: eight wavefronts, each a stretch of K, the rows of W and X as pieces of the 16x16x32 instruction straight from memory
// (fp32: split into parts on the way), 256 k of them asked for at a time.  Their sums meet in LDS.  Sixteen columns, so that W has two workgroups
// a compute unit from 8192 columns on; each reads all of X, or one of 16, 32 or 64 rows each (few_of).
template <class T>
struct FewJob {
  const T *X, *W;
  long ldx, ldw;
  int n, K, N, chunk;  // chunk: k of a wavefront, a multiple of 32
  Forward<T> out;
};
template <int P>
__device__ __forceinline__ void parts_of_eight(const Eight<float> &v, bf16x8 (&o)[P]) {
  u16 t[8][P];
#pragma unroll
  for (int e = 0; e < 8; e++) parts_of<P>(v[e], t[e]);
#pragma unroll
  for (int p = 0; p < P; p++)
    o[p] = __builtin_bit_cast(bf16x8, make_uint4(t[0][p] | (unsigned)t[1][p] << 16, t[2][p] | (unsigned)t[3][p] << 16, t[4][p] | (unsigned)t[5][p] << 16,
                                                 t[6][p] | (unsigned)t[7][p] << 16));
}
__device__ __forceinline__ void parts_of_eight(const Eight<u16> &v, bf16x8 (&o)[1]) {
  typedef unsigned four __attribute__((ext_vector_type(4)));
  o[0] = __builtin_bit_cast(bf16x8, (four)v.a);
}

constexpr int kFewWaves = 8;
// TT: blocks of sixteen rows of X
template <class T, int TT>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(FewJob<T> g) {
  constexpr int P = sizeof(T) == 4 ? 3 : 1, DEPTH = sizeof(T) == 4 ? (TT > 2 ? 2 : 4) : (TT > 2 ? 4 : 8), ACC = P > 1 ? 2 : 1;
  __shared__ float sums[kFewWaves][TT][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = blockIdx.x * 16, x = lane & 15, piece = 8 * (lane >> 4), r0 = blockIdx.y * 16 * TT;
  const int kbeg = wave * g.chunk, kend = min(g.K, kbeg + g.chunk);
  const T *w = g.W + min(c0 + x, g.N - 1) * g.ldw + piece;
  const T *rows[TT];
#pragma unroll
  for (int t = 0; t < TT; t++) rows[t] = g.X + min(r0 + 16 * t + x, g.n - 1) * g.ldx + piece;  // (rows beyond the last: once more the last, not stored)
  // what the epilogue reads, two lanes a row, is asked for first
  const int r = threadIdx.x >> 1, row = r0 + r, col = c0 + 8 * (threadIdx.x & 1), left = r < 16 * TT && row < g.n ? g.N - col : 0;
  Eight<float> bias;
  Eight<T> held;
  bias.zero(), held.zero();
  unsigned long long step = 0;
  unsigned id = 0;
  if (left > 0) {
    if (g.out.bias) bias.load(g.out.bias + col, left);
    g.out.hold(held, row, col, left);
    step = g.out.step(), id = g.out.id(row);
  }
  floatx4 acc[ACC][TT];
#pragma unroll
  for (int a = 0; a < ACC; a++)
#pragma unroll
    for (int t = 0; t < TT; t++) acc[a][t] = floatx4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Eight<T> &wv, const Eight<T> (&xv)[TT]) {
    bf16x8 a[P], b[P];
    parts_of_eight(wv, a);
#pragma unroll
    for (int t = 0; t < TT; t++) {
      parts_of_eight(xv[t], b);
#pragma unroll
      for (int p = 0; p < P; p++)
#pragma unroll
        for (int q = 0; q < P - p; q++)
          acc[p + q ? ACC - 1 : 0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[p], b[q], acc[p + q ? ACC - 1 : 0][t], 0, 0, 0);
    }
  };
  int k = kbeg;
  for (; k + 32 * DEPTH <= kend; k += 32 * DEPTH) {
    Eight<T> wv[DEPTH], xv[DEPTH][TT];
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      wv[d].load(w + k + 32 * d);
#pragma unroll
      for (int t = 0; t < TT; t++) xv[d][t].load(rows[t] + k + 32 * d);
    }
#pragma unroll
    for (int d = 0; d < DEPTH; d++) multiply(wv[d], xv[d]);
  }
  for (; k < kend; k += 32) {
    Eight<T> wv, xv[TT];
    const int left = kend - k - piece;
    wv.zero();
    if (left > 0) wv.load(w + k, left);
#pragma unroll
    for (int t = 0; t < TT; t++) {
      xv[t].zero();
      if (left > 0) xv[t].load(rows[t] + k, left);
    }
    multiply(wv, xv);
  }
#pragma unroll
  for (int t = 0; t < TT; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      float v = acc[0][t][r];
      if constexpr (ACC > 1) v += acc[1][t][r];
      sums[wave][t][x][4 * (lane >> 4) + r] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < TT * 256; i += 64 * kFewWaves) {
    const int t = i >> 8, r = i >> 4 & 15, c = i & 15;
    float v = sums[0][t][r][c];
#pragma unroll
    for (int q = 1; q < kFewWaves; q++) v += sums[q][t][r][c];
    sums[0][t][r][c] = v;  // (nobody else reads this one)
  }
  __syncthreads();
  if (left <= 0) return;
  float v[8], b[8];
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = sums[0][r >> 4][r & 15][8 * (threadIdx.x & 1) + e], b[e] = bias[e];
  g.out.finish(step, id, b, held, row, col, left, v);
}

// what a product left in parts, in their order, to the epilogue; pieces of eight columns
template <class E>
struct PartsJob {
  const float *part;
  int parts, rows, cols;
  E out;
  int blocks;  // 0: none
};
template <class E>
__device__ __forceinline__ void join_block(const PartsJob<E> &g, int block) {
  const int pieces = (g.cols + 7) / 8;
  const long total = (long)g.rows * pieces, i = (long)block * 256 + threadIdx.x;
  if (i >= total) return;
  const int row = (int)(i / pieces), col = 8 * (int)(i - (long)row * pieces), left = g.cols - col;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < g.parts; p += 4) {
    Eight<float> t[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      t[k].zero();
      if (p + k < g.parts) t[k].load(g.part + ((long)(p + k) * g.rows + row) * g.cols + col, left);
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += t[k][e];
  }
  typename E::Held held;
  g.out.hold(held, row, col, left);
  float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (g.out.biases()) {
    Eight<float> t;
    t.load(g.out.biases() + col, left);
#pragma unroll
    for (int e = 0; e < 8; e++) b[e] = t[e];
  }
  g.out.finish(g.out.step(), g.out.id(row), b, held, row, col, left, v);
}
template <class E>
__global__ __launch_bounds__(256) void parts_kernel(PartsJob<E> g) { join_block(g, blockIdx.x); }

// the ends of both gradients and db
template <class E>
__global__ __launch_bounds__(256) void back_ends_kernel(PartsJob<E> x, PartsJob<E> w, ColumnsJob b) {
  __shared__ float each[4][64];
  const int block = blockIdx.x;
  if (block < b.blocks) sum_columns(b, block, each);
  else if (block < b.blocks + x.blocks) join_block(x, block - b.blocks);
  else if (block < b.blocks + x.blocks + w.blocks) join_block(w, block - b.blocks - x.blocks);
}

// ------------------------------------------------------------------ what a call consists of
template <int P> struct Tiles;
template <> struct Tiles<1> {
  using L = NtTile<1, 128, 128, 32, 2, 2>;
  using S = NtTile<1, 64, 64, 64, 2, 2, 3>;
};
template <> struct Tiles<3> {
  using L = NtTile<3, 128, 128, 16, 2, 2>;
  using S = NtTile<3, 64, 64, 32, 2, 2>;
};
// (of the products here that turn operands)
template <class T>
struct Apart : T {
  static constexpr bool APART = true;
};
template <int P, class F>
int with_tile(int size, F &&f) {
  using TT = Tiles<P>;
  if (size) return f(typename TT::L{});
  return f(typename TT::S{});
}

struct Shape {  // of a product
  int size, tm, tn, splits, kchunk;
  double us;
};
// The tile and the stretches of K that a model of the launch finds best: ns a k of a compute unit that has one, two or three workgroups of a tile, as
// measured (fp32, in products of 7088 rows: 128 x 128 at 224, 448 and 672 workgroups, 64 x 64 at 256, 512 and 768); each workgroup costs 200 k more than it multiplies,
// and what products leave in parts is written and read at the rate of a copy, by a launch more.  us of a call with all workgroups whole / in the stretches this
// finds: fp32 gradients of 7088 x 512 x 2048 405 / 245.
template <int P> struct Speeds;
template <> struct Speeds<3> { static constexpr double ns[2][3] = {{26, 26, 29}, {68, 73, 98}}; };
template <> struct Speeds<1> { static constexpr double ns[2][3] = {{6, 6.5, 8}, {14, 15, 20}}; };
// (a dimension of a grid has less than 2^32 threads, with the workgroups that sum columns and of the launch that joins parts too)
inline bool too_many(double groups, int threads, int splits, long results) { return (groups + 16384) * threads >= 4294967296. || (splits > 1 && results >= 1l << 33); }
constexpr int kStretches[] = {1, 2, 3, 4, 5, 6, 8, 12, 16, 24, 32};
template <int P>
Shape shape_of(int cols, int rows, int K) {
  Shape best{};
  double least = INFINITY;
  const int cus = num_cus();
  for (int size = 0; size < 2; size++) {
    Shape s{};
    s.size = size;
    int bm = 0, bn = 0;
    with_tile<P>(size, [&](auto t) { return bm = decltype(t)::BM, bn = decltype(t)::BN, 0; });
    s.tm = tiles_of(cols, bm), s.tn = tiles_of(rows, bn);
    for (int splits : kStretches) {
      if (splits > 1 && K / splits < 256) break;
      s.kchunk = ceil_to((K + splits - 1) / splits, kPlaneAlign);
      s.splits = (K + s.kchunk - 1) / s.kchunk;
      if (too_many((double)s.tm * s.tn * s.splits, 256, s.splits, (long)rows * cols)) continue;
      const long groups = (long)s.tm * s.tn * s.splits, full = groups / (3 * cus), rest = (groups - full * 3 * cus + cus - 1) / cus;
      double us = 1e-3 * (s.kchunk + 200) * (full * Speeds<P>::ns[size][2] + (rest > 0 ? Speeds<P>::ns[size][rest - 1] : 0.));
      if (s.splits > 1) us += 5. + s.splits * (8. * rows * cols) / 4.7e6;
      if (us < least) least = us, best = s, best.us = us;
    }
  }
  return best;
}

// Of operands as they lie: the tile and the stretches of K that a model of the launch finds best.  us a k of a round of tiles, one a compute unit of the wide
// ones (0.0245 with the chip full, 0.0195 with half of it idle: power), two of the narrow (0.0140; one 0.0090); each workgroup costs 256 k more than it
// multiplies, and what products leave in parts is written and read at the rate of a copy, by a launch more.
Shape direct_shape_of(int cols, int rows, int K) {
  Shape best{};
  double least = INFINITY;
  const int cus = num_cus();
  for (int wide = 0; wide < 2; wide++) {
    Shape s{};
    s.size = wide;
    const int side = wide ? WideTile::BM : NarrowTile::BM;
    s.tm = tiles_of(cols, side), s.tn = tiles_of(rows, side);
    for (int splits : kStretches) {
      if (splits > 1 && K / splits < 256) break;
      s.kchunk = ceil_to((K + splits - 1) / splits, 64);
      s.splits = (K + s.kchunk - 1) / s.kchunk;
      if (too_many((double)s.tm * s.tn * s.splits, wide ? WideTile::THREADS : NarrowTile::THREADS, s.splits, (long)rows * cols)) continue;
      const long groups = (long)s.tm * s.tn * s.splits, full = wide ? groups / cus : groups / (2 * cus), rest = groups - full * (wide ? cus : 2 * cus);
      const double k = s.kchunk + 256.;
      double us = full * k * (wide ? 0.0245 : 0.0140);
      if (rest > 0) us += k * (wide ? (full > 0 || rest > cus / 2 ? 0.0225 : 0.0195) : (rest > cus ? 0.0140 : 0.0090));
      if (s.splits > 1) us += 5. + s.splits * (8. * rows * cols) / 4.7e6;
      if (us < least) least = us, best = s, best.us = us;
    }
  }
  return best;
}

// Both gradients in a launch: the same tile, and for each the stretches that a model finds best.  Where all workgroups have a place at once: the mean of them at the
// measured speed of as many as the fullest compute unit has; where not, what there is to multiply at the speed of all places, and a third of a round for the last;
// but no less than the longest by itself.  Parts go through the caches at twice a copy's rate, and take a launch's 5 us.
// us of a call with all workgroups whole / in the stretches this finds / in the best of them: fp32 7088 x 512 x 2048 266 / 187 / 187 (240 with the products in launches
// of their own), 4096 x 1024 x 1024 148 / 116 / 110, 157 x 300 x 777 31 / 21 / 21; bf16 2048 x 1024 x 4096 53 / 47 / 47, 8192 x 512 x 2048 87 / 48 / 48, 100 x 4096 x 4096
// 46 / 29 / 28.
struct Places {  // of a compute unit for workgroups of a tile, ns a k of one where all are taken and of the longest
  int bm, bn, threads, places;
  double ns, longest;
};
template <class Price>
void back_shapes_of(int n, int K, int N, int Kx, int Kw, int align, const Price &price, Shape *dx, Shape *dw) {
  double least = INFINITY;
  const int cus = num_cus();
  for (int size = 0; size < 2; size++) {
    const Places any = price(size, 1., cus);
    Shape x{}, w{};
    x.size = w.size = size;
    x.tm = w.tm = tiles_of(K, any.bm), x.tn = tiles_of(n, any.bn), w.tn = tiles_of(N, any.bn);
    auto set = [&](Shape &s, int of, int splits) {
      s.kchunk = ceil_to((of + splits - 1) / splits, align);
      s.splits = (of + s.kchunk - 1) / s.kchunk;
    };
    for (int sx : kStretches) {
      if (sx > 1 && Kx / sx < 256) break;
      set(x, Kx, sx);
      for (int sw : kStretches) {
        if (sw > 1 && Kw / sw < 256) break;
        set(w, Kw, sw);
        const double gx = (double)x.tm * x.tn * x.splits, gw = (double)w.tm * w.tn * w.splits, kx = x.kchunk + 200., kw = w.kchunk + 200.;
        const Places at = price(size, gx + gw, cus);
        if (too_many(gx + gw, at.threads, x.splits, (long)n * K) || too_many(gx + gw, at.threads, w.splits, (long)N * K)) continue;
        const double groups = gx + gw, all = (double)at.places * cus, work = gx * kx + gw * kw;
        const double even = at.ns * (groups > all ? work / all + 0.35 * std::fmin(kx, kw) : work / groups);
        double us = 1e-3 * std::fmax(even, at.longest * std::fmax(kx, kw));
        if (x.splits > 1) us += x.splits * (8. * n * K) / 9e6;
        if (w.splits > 1) us += w.splits * (8. * N * K) / 9e6;
        if (x.splits > 1 || w.splits > 1) us += 5.;
        if (us < least) least = us, *dx = x, *dw = w;
      }
    }
  }
}

struct Plan {
  int Kp, Np, np;  // as contraction lengths
  Shape fwd, dx, dw;
  size_t x, w, d, part, wpart, sums, bytes;
};
template <int P>
Plan plan_of(int n, int K, int N, int back) {
  Plan p{};
  p.Kp = ceil_to(K, kPlaneAlign), p.Np = ceil_to(N, kPlaneAlign), p.np = ceil_to(n, kPlaneAlign);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  auto parts = [&](const Shape &s, int rows, int cols) { return s.splits > 1 ? (size_t)s.splits * rows * cols * 4 : 0; };
  p.x = take(packed_bytes<P>(p.np, p.Kp));
  p.w = take(packed_bytes<P>(p.Np, p.Kp));
  if (!back) {
    p.fwd = shape_of<P>(N, n, p.Kp);
    p.part = take(parts(p.fwd, n, N));
  } else {
    p.d = take(packed_bytes<P>(p.np, p.Np));
    back_shapes_of(n, K, N, p.Np, p.np, kPlaneAlign, [](int size, double groups, int cus) {
      Places at{};
      with_tile<P>(size, [&](auto t) { return at.bm = decltype(t)::BM, at.bn = decltype(t)::BN, at.threads = decltype(t)::THREADS, 0; });
      at.places = groups <= cus ? 1 : groups <= 2 * cus ? 2 : 3;
      at.ns = Speeds<P>::ns[size][at.places - 1], at.longest = Speeds<P>::ns[size][0];
      return at;
    }, &p.dx, &p.dw);
    p.part = take(parts(p.dx, n, K)), p.wpart = take(parts(p.dw, N, K));
    p.sums = take((size_t)(p.np / 64) * N * 4);
  }
  p.bytes = at;
  return p;
}
Plan direct_plan_of(int n, int K, int N, int back) {
  Plan p{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  auto parts = [&](const Shape &s, int rows, int cols) { return s.splits > 1 ? (size_t)s.splits * rows * cols * 4 : 0; };
  if (!back) {
    p.fwd = direct_shape_of(N, n, K);
    p.part = take(parts(p.fwd, n, N));
  } else {
    p.d = take((size_t)n * N * 2);
    back_shapes_of(n, K, N, N, n, 64, [](int size, double groups, int cus) {
      if (size) return Places{WideTile::BM, WideTile::BN, WideTile::THREADS, 1, groups > cus / 2 ? 24.5 : 19.5, groups > cus / 2 ? 24.5 : 19.5};
      const int places = groups <= cus ? 1 : 2;
      return Places{NarrowTile::BM, NarrowTile::BN, NarrowTile::THREADS, places, places == 1 ? 9. : 14., places == 1 ? 9. : 14.};
    }, &p.dx, &p.dw);
    p.part = take(parts(p.dx, n, K)), p.wpart = take(parts(p.dw, N, K));
    p.sums = take((size_t)tiles_of(n, 64) * N * 4);
  }
  p.bytes = at;
  return p;
}

// Whether a forward pass reads W where it lies (few_rows_kernel) or goes by tiles.  ns a k of its workgroups, one a compute unit: bf16 1.0 + 0.05 a row of X,
// fp32 3.0 + 0.04 and 0.0013 a row squared (8192 x 2048 with 1, 16, 32, 64 rows: 1.0 1.6 2.5 4.2, 3.2 3.7 5.6 10.8); tiles cost what their model says, and what packing W and X takes.  us, without bias and
// what follows it, of few rows (64 a workgroup) / of tiles: bf16 2048 x 8192 with 1 row 6.9 / 10.8, 16 9.5 / 11.7, 64 20 / 15.5; 8192 x 2048 with 16 16 / 13.4; 1000 x 1000 with 157 5.8 / 13.6, 512
// 10.5 / 14.1; 512 x 2048 with 512 12.4 / 8.4; fp32 2048 x 8192 with 1 16 / 46, 32 29 / 48, 64 50 / 48; 300 x 777 with 157 7.1 / 12.3, 512 x 2048 with 256 15.5 / 17.7.
// Rows of a workgroup, 16, 32 or 64, by the same figures: where 64 leave compute units idle W is read by more of them (from the caches).  us, so, of 64 / of what this takes:
// fp32 157 x 300 x 777 7.1 / 5.6, 98 x 1918 x 352 18 / 8.8, 40 x 2048 x 2048 24 / 17, 32 x 8192 x 2048 50 / 35, bf16 64 x 4096 x 640 11 / 9.
struct Few {
  int blocks;  // of sixteen rows of X, of a workgroup: 1, 2 or 4
  double us;
};
Few few_of(int type, int n, int K, int N) {
  Few best{4, INFINITY};
  const double cus = num_cus();
  for (int blocks = 1; blocks <= 4; blocks *= 2) {
    if (tiles_of(n, 16 * blocks) > 65535) continue;  // (a grid's y)
    const double rows = n < 16 * blocks ? n : 16 * blocks, groups = (double)tiles_of(N, 16) * tiles_of(n, 16 * blocks);
    const double us = 2.5 + 1e-3 * K * (type == CAVS_F32 ? 3.0 + (0.04 + 0.0013 * rows) * rows : 1.0 + 0.05 * rows) * std::ceil(groups / cus);
    if (us < best.us) best = Few{blocks, us};
  }
  return best;
}
bool few_rows(int type, int n, int K, int N, double tiles_us) { return few_of(type, n, K, N).us < tiles_us; }
template <int P>
double packed_us(int n, int K, int N) { return 0.8 * (shape_of<P>(N, n, ceil_to(K, kPlaneAlign)).us + 4.5 + (double)K * ((double)n + N) * (P == 3 ? 10 : 4) / 7e6); }
double direct_us(int n, int K, int N) { return direct_shape_of(N, n, K).us + 1.5; }

struct Call {
  const void *X, *W, *R, *Z, *dY;
  int ldx, ldw, ldr, ldz, lddy;
  const float *b;
  int act;
  Mask m;
  void *Zout, *Y, *dX, *dW;
  int ldy, lddx, lddw;
  float *db;
  int n, K, N;
  size_t room;  // bytes of the workspace
};
// (whoever chose the path and whoever sized the workspace agree, or nothing is launched)
int check_room(const Call &c, size_t need) {
  CAVS_REQUIRE(need <= c.room, "cavs_linear: a plan of %zu bytes for n=%d K=%d N=%d, a workspace of %zu", need, c.n, c.K, c.N, c.room);
  return CAVS_OK;
}

inline dim3 grid_of(long blocks) {
  const long most = (1 << 24) - 1, high = (blocks + most - 1) / most;
  return dim3((unsigned)((blocks + high - 1) / high), (unsigned)high);
}
template <int P, class T>
PackJob<T> packing(const void *src, int ld, int rows, int K, int orows, char *o, int Kp) {
  PackJob<T> j{static_cast<const T *>(src), ld, rows, K, orows, {reinterpret_cast<u16 *>(o), Kp}, Kp / 64, 0};
  j.blocks = j.across * tiles_of(orows, 64);
  return j;
}

template <class E>
PartsJob<E> parts_of_product(const float *part, const Shape &s, int rows, int cols, const E &out) {
  const long blocks = ((long)rows * ((cols + 7) / 8) + 255) / 256;
  return PartsJob<E>{part, s.splits, rows, cols, out, s.splits > 1 ? (int)blocks : 0};
}
template <class E>
int join_parts(const float *part, const Shape &s, int rows, int cols, const E &out, hipStream_t st) {
  const PartsJob<E> g = parts_of_product(part, s, rows, cols, out);
  if (g.blocks > 0) {
    launch(parts_kernel<E>, (unsigned)g.blocks, 256, 0, st, g);
    CAVS_LAUNCH_CHECK();
  }
  return CAVS_OK;
}
// what is wanted of both gradients, the longer workgroups first
template <class Job>
struct BackJobs {
  Job j0, j1;
  int blocks0, blocks, wfirst;
};
template <class Job>
BackJobs<Job> back_jobs(const Job &x, const Shape &sx, bool wantx, const Job &w, const Shape &sw, bool wantw) {
  const int bx = wantx ? sx.tm * sx.tn * sx.splits : 0, bw = wantw ? sw.tm * sw.tn * sw.splits : 0;
  const bool wfirst = sw.kchunk > sx.kchunk;
  return wfirst ? BackJobs<Job>{w, x, bw, bx + bw, 1} : BackJobs<Job>{x, w, bx, bx + bw, 0};
}
// db from sums over 64 rows each
ColumnsJob columns_of(const Call &c, const Plan &p, char *ws, int stretches) {
  return ColumnsJob{reinterpret_cast<float *>(ws + p.sums), stretches, c.N, c.db, c.db ? (c.N + 63) / 64 : 0};
}
// what the products leave to do, and db if there were none
template <class T>
int back_ends(const Call &c, const Plan &p, char *ws, const ColumnsJob &b, hipStream_t st) {
  const Plain<T> ox{static_cast<T *>(c.dX), c.lddx}, ow{static_cast<T *>(c.dW), c.lddw};
  PartsJob<Plain<T>> x = parts_of_product(reinterpret_cast<float *>(ws + p.part), p.dx, c.n, c.K, ox);
  PartsJob<Plain<T>> w = parts_of_product(reinterpret_cast<float *>(ws + p.wpart), p.dw, c.N, c.K, ow);
  if (!c.dX) x.blocks = 0;
  if (!c.dW) w.blocks = 0;
  if (x.blocks + w.blocks + b.blocks > 0) {
    launch(back_ends_kernel<Plain<T>>, (unsigned)(x.blocks + w.blocks + b.blocks), 256, 0, st, x, w, b);
    CAVS_LAUNCH_CHECK();
  }
  return CAVS_OK;
}

// rows that begin on 16 bytes and are whole pieces of eight, in reach of 32 bits from the first of a tile
bool lies_well(const void *p, long ld, int w) { return aligned16(p) && ld % 8 == 0 && w % 8 == 0 && ld <= 1 << 22; }

// Whether bf16 operands may lie well at all, whatever their strides and alignment: of what cavs_linear_workspace has room for
bool may_lie_well(int K, int N, int back) { return K % 8 == 0 && (!back || N % 8 == 0); }

int run_direct_fwd(const Call &c, char *ws, hipStream_t st) {
  const Plan p = direct_plan_of(c.n, c.K, c.N, 0);
  if (const int rc = check_room(c, p.bytes)) return rc;
  float *part = reinterpret_cast<float *>(ws + p.part);
  const Forward<u16> out{c.b, c.act, c.m, static_cast<const u16 *>(c.R), c.ldr, static_cast<u16 *>(c.Zout), c.ldz, static_cast<u16 *>(c.Y), c.ldy};
  const DirectJob<Forward<u16>> g{{static_cast<const u16 *>(c.W), c.ldw}, {static_cast<const u16 *>(c.X), c.ldx}, c.N, c.n, c.K, p.fwd.tm, p.fwd.tn, p.fwd.kchunk,
                                  p.fwd.splits > 1 ? part : nullptr, out};
  const unsigned groups = (unsigned)(p.fwd.tm * p.fwd.tn * p.fwd.splits);
  if (p.fwd.size) launch(direct_forward_kernel<WideTile, Forward<u16>>, groups, WideTile::THREADS, 0, st, g);
  else launch(direct_forward_kernel<NarrowTile, Forward<u16>>, groups, NarrowTile::THREADS, 0, st, g);
  CAVS_LAUNCH_CHECK();
  return join_parts(part, p.fwd, c.n, c.N, out, st);
}

int run_direct_bwd(const Call &c, char *ws, hipStream_t st) {
  const Plan p = direct_plan_of(c.n, c.K, c.N, 1);
  if (const int rc = check_room(c, p.bytes)) return rc;
  const bool as_is = !c.act && !c.m.t && lies_well(c.dY, c.lddy, c.N);
  GradJob<u16> g{static_cast<const u16 *>(c.dY), static_cast<const u16 *>(c.Z), c.lddy, c.ldz, c.act, c.m, c.n, c.N, c.n, tiles_of(c.N, 256), 0,
                 {}, c.db ? reinterpret_cast<float *>(ws + p.sums) : nullptr};
  g.blocks = g.across * tiles_of(c.n, 64);
  u16 *made = !as_is && (c.dX || c.dW) ? reinterpret_cast<u16 *>(ws + p.d) : nullptr;
  if (made || c.db) {
    launch(grad_rows_kernel, grid_of(g.blocks), 256, 0, st, g, made);
    CAVS_LAUNCH_CHECK();
  }
  ColumnsJob b = columns_of(c, p, ws, tiles_of(c.n, 64));
  if (c.dX || c.dW) {
    typedef Plain<u16> E;
    const DirectRef D{made ? made : g.dY, made ? (long)c.N : c.lddy}, X{static_cast<const u16 *>(c.X), c.ldx}, W{static_cast<const u16 *>(c.W), c.ldw};
    float *xpart = reinterpret_cast<float *>(ws + p.part), *wpart = reinterpret_cast<float *>(ws + p.wpart);
    const DirectJob<E> x{W, D, c.K, c.n, c.N, p.dx.tm, p.dx.tn, p.dx.kchunk, p.dx.splits > 1 ? xpart : nullptr, E{static_cast<u16 *>(c.dX), c.lddx}};
    const DirectJob<E> w{X, D, c.K, c.N, c.n, p.dw.tm, p.dw.tn, p.dw.kchunk, p.dw.splits > 1 ? wpart : nullptr, E{static_cast<u16 *>(c.dW), c.lddw}};
    const auto j = back_jobs(x, p.dx, c.dX, w, p.dw, c.dW);
    const unsigned groups = (unsigned)(j.blocks + b.blocks);
    if (p.dx.size) launch(direct_back_kernel<WideTile, E>, groups, WideTile::THREADS, 0, st, j.j0, j.j1, j.blocks0, j.blocks, j.wfirst, b);
    else launch(direct_back_kernel<NarrowTile, E>, groups, NarrowTile::THREADS, 0, st, j.j0, j.j1, j.blocks0, j.blocks, j.wfirst, b);
    CAVS_LAUNCH_CHECK();
    b.blocks = 0;
  }
  return back_ends<u16>(c, p, ws, b, st);
}

template <class T>
int run_few(const Call &c, hipStream_t st) {
  const Forward<T> out{c.b, c.act, c.m, static_cast<const T *>(c.R), c.ldr, static_cast<T *>(c.Zout), c.ldz, static_cast<T *>(c.Y), c.ldy};
  const FewJob<T> g{static_cast<const T *>(c.X), static_cast<const T *>(c.W), c.ldx, c.ldw, c.n, c.K, c.N, ceil_to((c.K + kFewWaves - 1) / kFewWaves, 32), out};
  const int blocks = few_of(sizeof(T) == 4 ? CAVS_F32 : CAVS_BF16, c.n, c.K, c.N).blocks;
  const dim3 groups((unsigned)tiles_of(c.N, 16), (unsigned)tiles_of(c.n, 16 * blocks));
  launch(blocks == 1 ? few_rows_kernel<T, 1> : blocks == 2 ? few_rows_kernel<T, 2> : few_rows_kernel<T, 4>, groups, 64 * kFewWaves, 0, st, g);
  CAVS_LAUNCH_CHECK();
  return CAVS_OK;
}

template <int P, class T>
int run_fwd(const Call &c, char *ws, hipStream_t st) {
  const Plan p = plan_of<P>(c.n, c.K, c.N, 0);
  if (const int rc = check_room(c, p.bytes)) return rc;
  const PackJob<T> x = packing<P, T>(c.X, c.ldx, c.n, c.K, c.n, ws + p.x, p.Kp), w = packing<P, T>(c.W, c.ldw, c.N, c.K, c.N, ws + p.w, p.Kp);
  launch(pack_kernel<P, T>, grid_of((long)x.blocks + w.blocks), 256, 0, st, x, w);
  CAVS_LAUNCH_CHECK();
  typedef Forward<T> E;
  float *part = reinterpret_cast<float *>(ws + p.part);
  const E out{c.b, c.act, c.m, static_cast<const T *>(c.R), c.ldr, static_cast<T *>(c.Zout), c.ldz, static_cast<T *>(c.Y), c.ldy};
  const Product<E> g{{w.o.p, p.Kp}, {x.o.p, p.Kp}, c.N, c.n, p.Kp, p.fwd.tm, p.fwd.tn, p.fwd.kchunk, p.fwd.splits > 1 ? part : nullptr, out};
  with_tile<P>(p.fwd.size, [&](auto t) {
    using Tile = decltype(t);
    launch(packed_forward_kernel<Tile, E>, (unsigned)(p.fwd.tm * p.fwd.tn * p.fwd.splits), Tile::THREADS, 0, st, g);
    return 0;
  });
  CAVS_LAUNCH_CHECK();
  return join_parts(part, p.fwd, c.n, c.N, out, st);
}

template <int P, class T>
int run_bwd(const Call &c, char *ws, hipStream_t st) {
  const Plan p = plan_of<P>(c.n, c.K, c.N, 1);
  if (const int rc = check_room(c, p.bytes)) return rc;
  GradJob<T> g{static_cast<const T *>(c.dY), static_cast<const T *>(c.Z), c.lddy, c.ldz, c.act, c.m, c.n, c.N, p.np, p.Np / 64, 0,
               {c.dX || c.dW ? reinterpret_cast<u16 *>(ws + p.d) : nullptr, p.Np}, c.db ? reinterpret_cast<float *>(ws + p.sums) : nullptr};
  g.blocks = g.across * (p.np / 64);
  PackJob<T> x = packing<P, T>(c.X, c.ldx, c.n, c.K, p.np, ws + p.x, p.Kp), w = packing<P, T>(c.W, c.ldw, c.N, c.K, p.Np, ws + p.w, p.Kp);
  if (!c.dW) x.blocks = 0;
  if (!c.dX) w.blocks = 0;
  launch(grad_kernel<P, T>, grid_of((long)g.blocks + x.blocks + w.blocks), 256, 0, st, g, x, w);
  CAVS_LAUNCH_CHECK();
  ColumnsJob b = columns_of(c, p, ws, p.np / 64);
  if (c.dX || c.dW) {
    typedef Plain<T> E;
    const PackedRef X{x.o.p, p.Kp}, W{w.o.p, p.Kp}, D{g.o.p, p.Np};
    float *xpart = reinterpret_cast<float *>(ws + p.part), *wpart = reinterpret_cast<float *>(ws + p.wpart);
    const Product<E> jx{W, D, c.K, c.n, p.Np, p.dx.tm, p.dx.tn, p.dx.kchunk, p.dx.splits > 1 ? xpart : nullptr, E{static_cast<T *>(c.dX), c.lddx}};
    const Product<E> jw{X, D, c.K, c.N, p.np, p.dw.tm, p.dw.tn, p.dw.kchunk, p.dw.splits > 1 ? wpart : nullptr, E{static_cast<T *>(c.dW), c.lddw}};
    const auto j = back_jobs(jx, p.dx, c.dX, jw, p.dw, c.dW);
    with_tile<P>(p.dx.size, [&](auto t) {
      using Tile = decltype(t);
      launch(packed_back_kernel<Apart<Tile>, E>, (unsigned)(j.blocks + b.blocks), Tile::THREADS, 0, st, j.j0, j.j1, j.blocks0, j.blocks, j.wfirst, b);
      return 0;
    });
    CAVS_LAUNCH_CHECK();
    b.blocks = 0;
  }
  return back_ends<T>(c, p, ws, b, st);
}

template <class T>
__global__ __launch_bounds__(256) void no_rows_kernel(T *dW, long ld, float *db, int N, int K) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (db && i < N) db[i] = 0.f;
  if (dW)
    for (long at = i; at < (long)N * K; at += (long)gridDim.x * 256) dW[at / K * ld + at % K] = T(0);
}

constexpr int kMostRows = 1 << 20, kMostK = 1 << 16;
constexpr long kMostOut = 1l << 36;
bool shape_ok(int n, int K, int N) { return n <= kMostRows && N <= kMostRows && K <= kMostK && (long)n * N <= kMostOut && (long)N * K <= kMostOut; }

int check(const char *who, int type, const Call &c, const cavs_dropout_mask *mask, Mask *m) {
  CAVS_REQUIRE(type == CAVS_F32 || type == CAVS_BF16, "%s: type %d is neither CAVS_F32 nor CAVS_BF16", who, type);
  CAVS_REQUIRE(c.n >= 0 && c.K > 0 && c.N > 0, "%s: bad shape n=%d K=%d N=%d", who, c.n, c.K, c.N);
  CAVS_REQUIRE(shape_ok(c.n, c.K, c.N), "%s: unsupported shape n=%d K=%d N=%d (at most 2^20, 2^16, 2^20; n N and N K 2^36)", who, c.n, c.K, c.N);
  CAVS_REQUIRE(c.act >= CAVS_ACT_NONE && c.act <= CAVS_ACT_GELU, "%s: unknown activation %d", who, c.act);
  CAVS_REQUIRE(mask_of(mask, m), "%s: p is not in [0, 1)", who);
  return CAVS_OK;
}
int check_workspace(const char *who, const void *ws, size_t bytes, size_t need) {
  CAVS_REQUIRE(ws && bytes >= need, "%s: workspace of %zu bytes needed, %zu given", who, need, bytes);
  CAVS_REQUIRE(aligned16(ws), "%s: the workspace must be 16-byte aligned", who);
  return CAVS_OK;
}

}  // namespace
}  // namespace cavs

using namespace cavs;

extern "C" {

size_t cavs_linear_workspace(int type, int n, int K, int N, int back) {
  if (n <= 0 || K <= 0 || N <= 0 || !shape_ok(n, K, N) || (type != CAVS_F32 && type != CAVS_BF16)) return 0;
  size_t need = 256;  // (of few rows nothing is used)
  if (type == CAVS_F32) {
    if (back || !few_rows(type, n, K, N, packed_us<3>(n, K, N))) need = plan_of<3>(n, K, N, back).bytes;
    return need;
  }
  if (back || !few_rows(type, n, K, N, packed_us<1>(n, K, N))) need = plan_of<1>(n, K, N, back).bytes;
  if (may_lie_well(K, N, back) && (back || !few_rows(type, n, K, N, direct_us(n, K, N)))) {
    const size_t direct = direct_plan_of(n, K, N, back).bytes;
    need = need > direct ? need : direct;
  }
  return need;
}

int cavs_linear_fwd(int type, const void *X, int ldx, const void *W, int ldw, const float *b, int act, const cavs_dropout_mask *mask, const void *R, int ldr,
                    void *Z, int ldz, void *Y, int ldy, int n, int K, int N, void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "cavs_linear_fwd";
  Call c{};
  c.X = X, c.ldx = ldx, c.W = W, c.ldw = ldw, c.b = b, c.act = act, c.R = R, c.ldr = ldr, c.Zout = Z, c.ldz = ldz, c.Y = Y, c.ldy = ldy, c.n = n, c.K = K, c.N = N;
  c.room = workspace_bytes;
  if (const int rc = check(who, type, c, mask, &c.m)) return rc;
  CAVS_REQUIRE((!X || ldx >= K) && (!W || ldw >= K), "%s: a row stride is below K=%d", who, K);
  CAVS_REQUIRE((!Y || ldy >= N) && (!R || ldr >= N) && (!Z || ldz >= N), "%s: a row stride is below N=%d", who, N);
  if (n == 0) return CAVS_OK;
  CAVS_REQUIRE(X && W && Y, "%s: null pointer", who);
  if (const int rc = check_workspace(who, workspace, workspace_bytes, cavs_linear_workspace(type, n, K, N, 0))) return rc;
  char *w = static_cast<char *>(workspace);
  hipStream_t st = as_stream(stream);
  if (type == CAVS_F32) return few_rows(type, n, K, N, packed_us<3>(n, K, N)) ? run_few<float>(c, st) : run_fwd<3, float>(c, w, st);
  const bool direct = may_lie_well(K, N, 0) && lies_well(X, ldx, K) && lies_well(W, ldw, K);
  if (few_rows(type, n, K, N, direct ? direct_us(n, K, N) : packed_us<1>(n, K, N))) return run_few<u16>(c, st);
  return direct ? run_direct_fwd(c, w, st) : run_fwd<1, u16>(c, w, st);
}

int cavs_linear_bwd(int type, const void *X, int ldx, const void *W, int ldw, const void *Z, int ldz, int act, const cavs_dropout_mask *mask, const void *dY,
                    int lddy, void *dX, int lddx, void *dW, int lddw, float *db, int n, int K, int N, void *workspace, size_t workspace_bytes,
                    void *stream) {
  const char *who = "cavs_linear_bwd";
  Call c{};
  c.X = X, c.ldx = ldx, c.W = W, c.ldw = ldw, c.Z = Z, c.ldz = ldz, c.act = act, c.dY = dY, c.lddy = lddy, c.dX = dX, c.lddx = lddx, c.dW = dW, c.lddw = lddw;
  c.db = db, c.n = n, c.K = K, c.N = N, c.room = workspace_bytes;
  if (const int rc = check(who, type, c, mask, &c.m)) return rc;
  // (of what is read and written: X for dW, W for dX, Z for the slope)
  CAVS_REQUIRE((!dY || lddy >= N) && (!act || !Z || ldz >= N) && (!dW || !X || ldx >= K) && (!dX || !W || ldw >= K) && (!dX || lddx >= K) && (!dW || lddw >= K),
               "%s: a row stride is below its width", who);
  hipStream_t st = as_stream(stream);
  if (!dX && !dW && !db) return CAVS_OK;
  if (n == 0) {  // sums over no rows
    if (!dW && !db) return CAVS_OK;
    const unsigned groups = (unsigned)((N + 255) / 256);
    if (type == CAVS_F32) launch(no_rows_kernel<float>, groups, 256, 0, st, static_cast<float *>(dW), (long)lddw, db, N, K);
    else launch(no_rows_kernel<u16>, groups, 256, 0, st, static_cast<u16 *>(dW), (long)lddw, db, N, K);
    CAVS_LAUNCH_CHECK();
    return CAVS_OK;
  }
  CAVS_REQUIRE(dY && (!act || Z) && (!dW || X) && (!dX || W), "%s: null pointer", who);
  if (const int rc = check_workspace(who, workspace, workspace_bytes, cavs_linear_workspace(type, n, K, N, 1))) return rc;
  char *w = static_cast<char *>(workspace);
  if (type == CAVS_F32) return run_bwd<3, float>(c, w, st);
  const bool direct = may_lie_well(K, N, 1) && (!dW || lies_well(X, ldx, K)) && (!dX || lies_well(W, ldw, K));
  return direct ? run_direct_bwd(c, w, st) : run_bwd<1, u16>(c, w, st);
}

}  // extern "C"
