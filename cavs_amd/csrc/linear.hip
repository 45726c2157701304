// Y = R + drop(act(X W^T + b)) and its gradients: products with everything that follows them in their epilogue.
//
//   forward   Z = X W^T + b, Y = R + drop(act(Z))
//   backward  D = drop(dY) . act'(Z), dX = D W, dW = D^T X, db = sums of D's columns
//
// Tiles are made of the transposed product, so that a lane of the 32x32 instruction holds neighbouring values of a row of the result: after an
// exchange with the lane 32 away eight of them, which is what bias, residual and results are read and written in, and what one call of the dropout's
// generator is for.
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
__global__ __launch_bounds__(256) void pack_kernel(PackJob<T> j0, PackJob<T> j1) {
  __shared__ PackTile tile;
  const int at = blockIdx.y * gridDim.x + blockIdx.x;
  if (at >= j0.blocks + j1.blocks) return;
  const bool second = at >= j0.blocks;
  const PackJob<T> &g = second ? j1 : j0;
  const int block = second ? at - j0.blocks : at, r0 = block / g.across * 64, k0 = block % g.across * 64;
  load_tile(tile, g.src, g.ld, r0, k0, g.rows, g.K);
  __syncthreads();
  pack_tile<P>(tile, g.o, PackedOut{}, r0, k0, g.orows, g.K);
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
template <int P, class T>
__global__ __launch_bounds__(256) void grad_kernel(GradJob<T> g) {
  __shared__ PackTile tile;
  __shared__ float part[4][64];
  const int block = blockIdx.y * gridDim.x + blockIdx.x;
  if (block >= g.blocks) return;
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
    for (int e = 0; e < 8; e++) v[e] = d[e];
    if (g.m.t && left > 0) drop8(g.m, draws_of(g.m, step, row_id(g.m, row), col >> 3), v);
#pragma unroll
    for (int e = 0; e < 8; e++) tile[r][8 * piece + e] = e < left ? g.act ? v[e] * slope_of<P == 1>(g.act, z[e]) : v[e] : 0.f;
  }
  __syncthreads();
  if (g.o.p) pack_tile<P>(tile, g.o, PackedOut{}, r0, k0, g.orows, g.N);
  if (!g.sums) return;
  const int c = threadIdx.x & 63, w = threadIdx.x >> 6;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i++) s += tile[16 * w + i][c];
  part[w][c] = s;
  __syncthreads();
  if (w == 0 && k0 + c < g.N) g.sums[(long)(r0 / 64) * g.N + k0 + c] = (part[0][c] + part[1][c]) + (part[2][c] + part[3][c]);
}

// ------------------------------------------------------------------ products of packed operands
// result[row, col] = sum over k of A[col, k] B[row, k].  K in `splits` stretches of kchunk, each with sums of its own at part + split * rows * cols; part
// null: straight to the epilogue.
template <class E>
struct Product {
  PackedRef A, B;
  int cols, rows, K, tilesM, tilesN, splits, kchunk;
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

template <class T, bool TA, bool TB, class E>
__global__ __launch_bounds__(T::THREADS, T::EU) void packed_product_kernel(Product<E> g) {
  // (one array: of two the compiler no longer knows that the pieces are not what is on its way from memory, and waits: 8192 x 8192 x 4096 924 us, 394 so)
  __shared__ __attribute__((aligned(16))) char S[T::LDS + T::BM * 4];
  float *kept = reinterpret_cast<float *>(S + T::LDS);
  const int tiles = g.tilesM * g.tilesN, split = blockIdx.x / tiles;
  int tm, tn;
  nt_tile_of(blockIdx.x - split * tiles, g.tilesM, g.tilesN, &tm, &tn);
  const int m0 = tm * T::BM, n0 = tn * T::BN, kbeg = split * g.kchunk, kend = min(g.K, kbeg + g.kchunk);
  floatx16 acc[T::ACC][T::TM][T::TN];
  if (!g.part) keep_biases<T::BM>(g.out, kept, m0, g.cols);
  nt_multiply<T, TA, TB>(g.A, g.cols, m0, g.B, g.rows, n0, kbeg, kend, S, acc);
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

// ------------------------------------------------------------------ products of operands as they lie (direct_product.h)
template <class E>
struct DirectJob {
  DirectRef A, B;
  int cols, rows, K, tilesM, tilesN, kchunk;
  float *part;
  E out;
};
template <class T, bool TA, bool TB, class E>
__global__ __launch_bounds__(T::THREADS, T::EU) void direct_product_kernel(DirectJob<E> g) {
  // (one array: of two the compiler no longer knows that the pieces are not what is on its way from memory, and waits: 8192 x 8192 x 4096 924 us, 394 so)
  __shared__ __attribute__((aligned(16))) char S[T::LDS + T::BM * 4];
  float *kept = reinterpret_cast<float *>(S + T::LDS);
  const int tiles = g.tilesM * g.tilesN, split = blockIdx.x / tiles;
  int tm, tn;
  nt_tile_of(blockIdx.x - split * tiles, g.tilesM, g.tilesN, &tm, &tn);
  const int m0 = tm * T::BM, n0 = tn * T::BN, kbeg = split * g.kchunk, kend = min(g.K, kbeg + g.kchunk);
  floatx4 acc[T::I][2 * T::J];
  if (!g.part) keep_biases<T::BM>(g.out, kept, m0, g.cols);
  direct_multiply<TA, TB>(T{}, g.A, g.cols, m0, g.B, g.rows, n0, kbeg, kend, S, acc);
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
        if (g.m.t) drop8(g.m, draws_of(g.m, step, row_id(g.m, row), col >> 3), v);
        if (g.act) {
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] *= slope_of<true>(g.act, z[i][e]);
        }
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

// what products left in parts, in their order, to the epilogue; pieces of eight columns
template <class E>
__global__ __launch_bounds__(256) void parts_kernel(const float *part, int parts, int rows, int cols, E out) {
  const int pieces = (cols + 7) / 8;
  const long total = (long)rows * pieces, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int row = (int)(i / pieces), col = 8 * (int)(i - (long)row * pieces), left = cols - col;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < parts; p += 4) {
    Eight<float> t[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      t[k].zero();
      if (p + k < parts) t[k].load(part + ((long)(p + k) * rows + row) * cols + col, left);
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += t[k][e];
  }
  typename E::Held held;
  out.hold(held, row, col, left);
  float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (out.biases()) {
    Eight<float> t;
    t.load(out.biases() + col, left);
#pragma unroll
    for (int e = 0; e < 8; e++) b[e] = t[e];
  }
  out.finish(out.step(), out.id(row), b, held, row, col, left, v);
}

__global__ __launch_bounds__(256) void column_sums_kernel(const float *part, int parts, int cols, float *out) {
  __shared__ float each[4][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6, per = (parts + 3) / 4, end = min(parts, (w + 1) * per);
  float s = 0.f;
  if (c < cols)
    for (int p = w * per; p < end; p += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = p + k < end ? part[(long)(p + k) * cols + c] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; k++) s += v[k];
    }
  each[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && c < cols) out[c] = (each[0][threadIdx.x] + each[1][threadIdx.x]) + (each[2][threadIdx.x] + each[3][threadIdx.x]);
}

// ------------------------------------------------------------------ what a call consists of
template <int P> struct Tiles;
template <> struct Tiles<1> {
  using L = NtTile<1, 256, 128, 32, 2, 2>;
  using M = NtTile<1, 128, 128, 32, 2, 2>;
  using S = NtTile<1, 64, 64, 64, 2, 2, 3>;
};
template <> struct Tiles<3> {
  using L = NtTile<3, 128, 128, 16, 2, 2>;
  using M = L;
  using S = NtTile<3, 64, 64, 32, 2, 2>;
};
template <int P, class F>
int with_tile(int size, F &&f) {
  using TT = Tiles<P>;
  if (size == 2) return f(typename TT::L{});
  if (size == 1) return f(typename TT::M{});
  return f(typename TT::S{});
}

struct Shape {  // of a product
  int size, tm, tn, splits, kchunk;
};
// The tile and the stretches of K that a model of the launch finds best: ns a k of a compute unit that has one, two or three workgroups of a tile, as
// measured (fp32, in products of 7088 rows: 128 x 128 at 224, 448 and 672 workgroups, 64 x 64 at 256, 512 and 768); each workgroup costs 200 k more than it multiplies,
// and what products leave in parts is written and read at the rate of a copy, by a launch more.  us of a call with all workgroups whole / in the stretches this
// finds: fp32 gradients of 7088 x 512 x 2048 405 / 245.
template <int P> struct Speeds;
template <> struct Speeds<3> { static constexpr int SIZES = 2; static constexpr double ns[2][3] = {{26, 26, 29}, {68, 73, 98}}; };
template <> struct Speeds<1> { static constexpr int SIZES = 3; static constexpr double ns[3][3] = {{6, 6.5, 8}, {14, 15, 20}, {24, 27, 38}}; };
constexpr int kStretches[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
template <int P>
Shape shape_of(int cols, int rows, int K) {
  Shape best{};
  double least = INFINITY;
  const int cus = num_cus();
  for (int size = 0; size < Speeds<P>::SIZES; size++) {
    Shape s{};
    s.size = size;
    int bm = 0, bn = 0;
    with_tile<P>(size, [&](auto t) { return bm = decltype(t)::BM, bn = decltype(t)::BN, 0; });
    s.tm = tiles_of(cols, bm), s.tn = tiles_of(rows, bn);
    for (int splits : kStretches) {
      if (splits > 1 && K / splits < 256) break;
      s.kchunk = ceil_to((K + splits - 1) / splits, kPlaneAlign);
      s.splits = (K + s.kchunk - 1) / s.kchunk;
      const long groups = (long)s.tm * s.tn * s.splits, full = groups / (3 * cus), rest = (groups - full * 3 * cus + cus - 1) / cus;
      double us = 1e-3 * (s.kchunk + 200) * (full * Speeds<P>::ns[size][2] + (rest > 0 ? Speeds<P>::ns[size][rest - 1] : 0.));
      if (s.splits > 1) us += 5. + s.splits * (8. * rows * cols) / 4.7e6;
      if (us < least) least = us, best = s;
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
      const long groups = (long)s.tm * s.tn * s.splits, full = wide ? groups / cus : groups / (2 * cus), rest = groups - full * (wide ? cus : 2 * cus);
      const double k = s.kchunk + 256.;
      double us = full * k * (wide ? 0.0245 : 0.0140);
      if (rest > 0) us += k * (wide ? (full > 0 || rest > cus / 2 ? 0.0225 : 0.0195) : (rest > cus ? 0.0140 : 0.0090));
      if (s.splits > 1) us += 5. + s.splits * (8. * rows * cols) / 4.7e6;
      if (us < least) least = us, best = s;
    }
  }
  return best;
}

struct Plan {
  int Kp, Np, np;  // as contraction lengths
  Shape fwd, dx, dw;
  size_t x, w, d, part, sums, bytes;
};
template <int P>
Plan plan_of(int n, int K, int N, int back) {
  Plan p{};
  p.Kp = ceil_to(K, kPlaneAlign), p.Np = ceil_to(N, kPlaneAlign), p.np = ceil_to(n, kPlaneAlign);
  size_t at = 0, part = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  auto parts = [&](const Shape &s, int rows, int cols) {
    const size_t b = s.splits > 1 ? (size_t)s.splits * rows * cols * 4 : 0;
    part = part > b ? part : b;
  };
  p.x = take(packed_bytes<P>(p.np, p.Kp));
  p.w = take(packed_bytes<P>(p.Np, p.Kp));
  if (!back) {
    p.fwd = shape_of<P>(N, n, p.Kp);
    parts(p.fwd, n, N);
  } else {
    p.d = take(packed_bytes<P>(p.np, p.Np));
    p.dx = shape_of<P>(K, n, p.Np);
    p.dw = shape_of<P>(K, N, p.np);
    parts(p.dx, n, K), parts(p.dw, N, K);
    p.sums = take((size_t)(p.np / 64) * N * 4);
  }
  p.part = take(part);
  p.bytes = at;
  return p;
}
Plan direct_plan_of(int n, int K, int N, int back) {
  Plan p{};
  size_t at = 0, part = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  auto parts = [&](const Shape &s, int rows, int cols) {
    const size_t b = s.splits > 1 ? (size_t)s.splits * rows * cols * 4 : 0;
    part = part > b ? part : b;
  };
  if (!back) {
    p.fwd = direct_shape_of(N, n, K);
    parts(p.fwd, n, N);
  } else {
    p.d = take((size_t)n * N * 2);
    p.dx = direct_shape_of(K, n, N);
    p.dw = direct_shape_of(K, N, n);
    parts(p.dx, n, K), parts(p.dw, N, K);
    p.sums = take((size_t)tiles_of(n, 64) * N * 4);
  }
  p.part = take(part);
  p.bytes = at;
  return p;
}

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
};

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
int join_parts(const float *part, const Shape &s, int rows, int cols, const E &out, hipStream_t st) {
  launch(parts_kernel<E>, (unsigned)(((long)rows * ((cols + 7) / 8) + 255) / 256), 256, 0, st, part, s.splits, rows, cols, out);
  CAVS_LAUNCH_CHECK();
  return CAVS_OK;
}
template <int P, bool TA, bool TB, class E>
int product(const Shape &s, const PackedRef &A, int cols, const PackedRef &B, int rows, int K, float *part, const E &out, hipStream_t st) {
  Product<E> g{A, B, cols, rows, K, s.tm, s.tn, s.splits, s.kchunk, s.splits > 1 ? part : nullptr, out};
  with_tile<P>(s.size, [&](auto t) {
    using T = decltype(t);
    launch(packed_product_kernel<T, TA, TB, E>, s.tm * s.tn * s.splits, T::THREADS, 0, st, g);
    return 0;
  });
  CAVS_LAUNCH_CHECK();
  return g.part ? join_parts(part, s, rows, cols, out, st) : (int)CAVS_OK;
}

template <bool TA, bool TB, class E>
int direct_product(const Shape &s, const DirectRef &A, int cols, const DirectRef &B, int rows, int K, float *part, const E &out, hipStream_t st) {
  DirectJob<E> g{A, B, cols, rows, K, s.tm, s.tn, s.kchunk, s.splits > 1 ? part : nullptr, out};
  const unsigned groups = (unsigned)(s.tm * s.tn * s.splits);
  if (s.size) launch(direct_product_kernel<WideTile, TA, TB, E>, groups, WideTile::THREADS, 0, st, g);
  else launch(direct_product_kernel<NarrowTile, TA, TB, E>, groups, NarrowTile::THREADS, 0, st, g);
  CAVS_LAUNCH_CHECK();
  return g.part ? join_parts(part, s, rows, cols, out, st) : (int)CAVS_OK;
}

// rows that begin on 16 bytes and are whole pieces of eight, in reach of 32 bits from the first of a tile
bool lies_well(const void *p, long ld, int w) { return aligned16(p) && ld % 8 == 0 && w % 8 == 0 && ld <= 1 << 22; }

int run_direct_fwd(const Call &c, char *ws, hipStream_t st) {
  const Plan p = direct_plan_of(c.n, c.K, c.N, 0);
  const Forward<u16> out{c.b, c.act, c.m, static_cast<const u16 *>(c.R), c.ldr, static_cast<u16 *>(c.Zout), c.ldz, static_cast<u16 *>(c.Y), c.ldy};
  return direct_product<false, false>(p.fwd, DirectRef{static_cast<const u16 *>(c.W), c.ldw}, c.N, DirectRef{static_cast<const u16 *>(c.X), c.ldx}, c.n, c.K,
                                      reinterpret_cast<float *>(ws + p.part), out, st);
}

int run_direct_bwd(const Call &c, char *ws, hipStream_t st) {
  const Plan p = direct_plan_of(c.n, c.K, c.N, 1);
  const bool as_is = !c.act && !c.m.t && lies_well(c.dY, c.lddy, c.N);
  GradJob<u16> g{static_cast<const u16 *>(c.dY), static_cast<const u16 *>(c.Z), c.lddy, c.ldz, c.act, c.m, c.n, c.N, c.n, tiles_of(c.N, 256), 0,
                 {}, c.db ? reinterpret_cast<float *>(ws + p.sums) : nullptr};
  g.blocks = g.across * tiles_of(c.n, 64);
  u16 *made = !as_is && (c.dX || c.dW) ? reinterpret_cast<u16 *>(ws + p.d) : nullptr;
  if (made || c.db) {
    launch(grad_rows_kernel, grid_of(g.blocks), 256, 0, st, g, made);
    CAVS_LAUNCH_CHECK();
  }
  const DirectRef D{made ? made : g.dY, made ? (long)c.N : c.lddy}, X{static_cast<const u16 *>(c.X), c.ldx}, W{static_cast<const u16 *>(c.W), c.ldw};
  float *part = reinterpret_cast<float *>(ws + p.part);
  if (c.dX) {
    if (const int rc = direct_product<true, false>(p.dx, W, c.K, D, c.n, c.N, part, Plain<u16>{static_cast<u16 *>(c.dX), c.lddx}, st)) return rc;
  }
  if (c.dW) {
    if (const int rc = direct_product<true, true>(p.dw, X, c.K, D, c.N, c.n, part, Plain<u16>{static_cast<u16 *>(c.dW), c.lddw}, st)) return rc;
  }
  if (c.db) {
    launch(column_sums_kernel, (c.N + 63) / 64, 256, 0, st, g.sums, tiles_of(c.n, 64), c.N, c.db);
    CAVS_LAUNCH_CHECK();
  }
  return CAVS_OK;
}

template <int P, class T>
int run_fwd(const Call &c, char *ws, hipStream_t st) {
  const Plan p = plan_of<P>(c.n, c.K, c.N, 0);
  const PackJob<T> x = packing<P, T>(c.X, c.ldx, c.n, c.K, c.n, ws + p.x, p.Kp), w = packing<P, T>(c.W, c.ldw, c.N, c.K, c.N, ws + p.w, p.Kp);
  launch(pack_kernel<P, T>, grid_of((long)x.blocks + w.blocks), 256, 0, st, x, w);
  CAVS_LAUNCH_CHECK();
  const Forward<T> out{c.b, c.act, c.m, static_cast<const T *>(c.R), c.ldr, static_cast<T *>(c.Zout), c.ldz, static_cast<T *>(c.Y), c.ldy};
  return product<P, false, false>(p.fwd, PackedRef{w.o.p, p.Kp}, c.N, PackedRef{x.o.p, p.Kp}, c.n, p.Kp, reinterpret_cast<float *>(ws + p.part), out, st);
}

template <int P, class T>
int run_bwd(const Call &c, char *ws, hipStream_t st) {
  const Plan p = plan_of<P>(c.n, c.K, c.N, 1);
  GradJob<T> g{static_cast<const T *>(c.dY), static_cast<const T *>(c.Z), c.lddy, c.ldz, c.act, c.m, c.n, c.N, p.np, p.Np / 64, 0,
               {c.dX || c.dW ? reinterpret_cast<u16 *>(ws + p.d) : nullptr, p.Np}, c.db ? reinterpret_cast<float *>(ws + p.sums) : nullptr};
  g.blocks = g.across * (p.np / 64);
  launch(grad_kernel<P, T>, grid_of(g.blocks), 256, 0, st, g);
  CAVS_LAUNCH_CHECK();
  PackJob<T> x = packing<P, T>(c.X, c.ldx, c.n, c.K, p.np, ws + p.x, p.Kp), w = packing<P, T>(c.W, c.ldw, c.N, c.K, p.Np, ws + p.w, p.Kp);
  const PackedRef X{x.o.p, p.Kp}, W{w.o.p, p.Kp}, D{g.o.p, p.Np};
  if (!c.dW) x.blocks = 0;
  if (!c.dX) w.blocks = 0;
  if (c.dX || c.dW) {
    launch(pack_kernel<P, T>, grid_of((long)x.blocks + w.blocks), 256, 0, st, x, w);
    CAVS_LAUNCH_CHECK();
  }
  float *part = reinterpret_cast<float *>(ws + p.part);
  if (c.dX) {
    if (const int rc = product<P, true, false>(p.dx, W, c.K, D, c.n, p.Np, part, Plain<T>{static_cast<T *>(c.dX), c.lddx}, st)) return rc;
  }
  if (c.dW) {
    if (const int rc = product<P, true, true>(p.dw, X, c.K, D, c.N, p.np, part, Plain<T>{static_cast<T *>(c.dW), c.lddw}, st)) return rc;
  }
  if (c.db) {
    launch(column_sums_kernel, (c.N + 63) / 64, 256, 0, st, g.sums, p.np / 64, c.N, c.db);
    CAVS_LAUNCH_CHECK();
  }
  return CAVS_OK;
}

template <class T>
__global__ __launch_bounds__(256) void no_rows_kernel(T *dW, long ld, float *db, int N, int K) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (db && i < N) db[i] = 0.f;
  if (dW)
    for (long at = i; at < (long)N * K; at += (long)gridDim.x * 256) dW[at / K * ld + at % K] = T(0);
}

// (offsets within a tile's rows are below 2^32 bytes, and a launch has less than 2^24 tiles)
constexpr int kMostRows = 1 << 20, kMostK = 1 << 16;
constexpr long kMostOut = 1l << 36;
bool shape_ok(int n, int K, int N) { return n <= kMostRows && N <= kMostRows && K <= kMostK && (long)n * N <= kMostOut && (long)N * K <= kMostOut; }

int check(const char *who, int type, const Call &c, const cavs_dropout_mask *mask, Mask *m) {
  CAVS_REQUIRE(type == CAVS_F32 || type == CAVS_BF16, "%s: type %d is neither CAVS_F32 nor CAVS_BF16", who, type);
  CAVS_REQUIRE(c.n >= 0 && c.K > 0 && c.N > 0, "%s: bad shape n=%d K=%d N=%d", who, c.n, c.K, c.N);
  CAVS_REQUIRE(shape_ok(c.n, c.K, c.N), "%s: unsupported shape n=%d K=%d N=%d (at most 2^20, 2^16, 2^20; n N and N K 2^36)", who, c.n, c.K, c.N);
  CAVS_REQUIRE(c.act >= CAVS_ACT_NONE && c.act <= CAVS_ACT_GELU, "%s: unknown activation %d", who, c.act);
  CAVS_REQUIRE(c.ldx >= c.K && c.ldw >= c.K, "%s: a row stride is below K=%d", who, c.K);
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
  if (type == CAVS_F32) return plan_of<3>(n, K, N, back).bytes;
  const size_t packed = plan_of<1>(n, K, N, back).bytes, direct = K % 8 == 0 && (!back || N % 8 == 0) ? direct_plan_of(n, K, N, back).bytes : 0;
  return packed > direct ? packed : direct;
}

int cavs_linear_fwd(int type, const void *X, int ldx, const void *W, int ldw, const float *b, int act, const cavs_dropout_mask *mask, const void *R, int ldr,
                    void *Z, int ldz, void *Y, int ldy, int n, int K, int N, void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "cavs_linear_fwd";
  Call c{};
  c.X = X, c.ldx = ldx, c.W = W, c.ldw = ldw, c.b = b, c.act = act, c.R = R, c.ldr = ldr, c.Zout = Z, c.ldz = ldz, c.Y = Y, c.ldy = ldy, c.n = n, c.K = K, c.N = N;
  if (const int rc = check(who, type, c, mask, &c.m)) return rc;
  CAVS_REQUIRE(ldy >= N && (!R || ldr >= N) && (!Z || ldz >= N), "%s: a row stride is below N=%d", who, N);
  if (n == 0) return CAVS_OK;
  CAVS_REQUIRE(X && W && Y, "%s: null pointer", who);
  if (const int rc = check_workspace(who, workspace, workspace_bytes, cavs_linear_workspace(type, n, K, N, 0))) return rc;
  char *w = static_cast<char *>(workspace);
  if (type == CAVS_F32) return run_fwd<3, float>(c, w, as_stream(stream));
  return lies_well(X, ldx, K) && lies_well(W, ldw, K) ? run_direct_fwd(c, w, as_stream(stream)) : run_fwd<1, u16>(c, w, as_stream(stream));
}

int cavs_linear_bwd(int type, const void *X, int ldx, const void *W, int ldw, const void *Z, int ldz, int act, const cavs_dropout_mask *mask, const void *dY,
                    int lddy, void *dX, int lddx, void *dW, int lddw, float *db, int n, int K, int N, void *workspace, size_t workspace_bytes,
                    void *stream) {
  const char *who = "cavs_linear_bwd";
  Call c{};
  c.X = X, c.ldx = ldx, c.W = W, c.ldw = ldw, c.Z = Z, c.ldz = ldz, c.act = act, c.dY = dY, c.lddy = lddy, c.dX = dX, c.lddx = lddx, c.dW = dW, c.lddw = lddw;
  c.db = db, c.n = n, c.K = K, c.N = N;
  if (const int rc = check(who, type, c, mask, &c.m)) return rc;
  CAVS_REQUIRE(lddy >= N && (!act || ldz >= N) && (!dX || lddx >= K) && (!dW || lddw >= K), "%s: a row stride is below its width", who);
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
  const bool direct = N % 8 == 0 && (!dW || lies_well(X, ldx, K)) && (!dX || lies_well(W, ldw, K));
  return direct && (long)N <= 1 << 22 ? run_direct_bwd(c, w, st) : run_bwd<1, u16>(c, w, st);
}

}  // extern "C"
