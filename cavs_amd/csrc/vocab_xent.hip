// Softmax cross entropy of X W^T + b over a large vocabulary, and its gradients, without logits in memory.
//
//   z = X W^T + b,  lse_r = log sum_c exp z_rc,  loss_r = lse_r - z_r,label,  d_rc = w_r (exp(z_rc - lse_r) - [c = label_r])
//   dX = d W,  dW = d^T X,  db = sums of d's columns
//
// The vocabulary goes by in pieces.  The first pass over them makes each tile of z in registers and leaves a maximum and a sum of
// exponentials per row and tile; what they come to together is lse.  The second makes the tile again, d from it, and leaves d of a piece
// (packed for its two products, by token and by class), which d X and d W are made of before the next piece overwrites it.
// Statistics, sums and accumulators are fp32; d is rounded to bf16 where the gradients are (half a unit of 2^-8, as their own
// rounding), and is three bf16 parts, all of an fp32's bits, where they are fp32.
#include "nt_product.h"
#include "wave_reduce.h"

namespace cavs {
namespace {

// ------------------------------------------------------------------ operands, packed
// src [rows, K] with its columns as k and, for the products that sum over its rows, with its rows as k.  Either may be left out.  A row whose
// flag says so is zero in the second: 0 times what it holds need not be 0.
enum { KEEP_ALL = 0, KEEP_NONZERO = 1, KEEP_FINITE = 2 };  // rows with flag != 0; rows whose flag is not -inf

template <int P, class Src>
__global__ __launch_bounds__(256) void pack_kernel(const Src *__restrict__ src, long ld, int rows, int K, PackedOut o, PackedOut t, const float *__restrict__ flag,
                                                   int keep) {
  __shared__ PackTile tile;
  const int r0 = blockIdx.y * 64, k0 = blockIdx.x * 64, k = threadIdx.x & 63;
#pragma unroll 8
  for (int i = threadIdx.x >> 6; i < 64; i += 4) {
    const int r = r0 + i;
    tile[i][k] = r < rows && k0 + k < K ? value_of(src + r * ld + k0 + k) : 0.f;
  }
  __syncthreads();
  pack_tile<P>(tile, o, keep == KEEP_ALL ? t : PackedOut{}, r0, k0, rows, K);
  if (!t.p || keep == KEEP_ALL) return;
  __syncthreads();
  for (int i = threadIdx.x >> 6; i < 64; i += 4)
    if (r0 + i < rows && (keep == KEEP_NONZERO ? flag[r0 + i] == 0.f : flag[r0 + i] == -INFINITY)) tile[i][k] = 0.f;
  __syncthreads();
  pack_tile<P>(tile, PackedOut{}, t, r0, k0, rows, K);
}

// ------------------------------------------------------------------ the tile of z
// Vocabulary rows are the tile's rows, tokens its columns: a lane holds 16 TM classes of TN tokens, and a token's sums are
// sums over registers.
// Coordinates of acc[.][i][j][r]: class nt_class, token nt_token.
template <class T>
struct Where {
  int wm, wn, lane, half;
  __device__ inline Where() {
    const int wave = threadIdx.x >> 6;
    lane = threadIdx.x & 63, half = lane >> 5;
    wm = wave / T::WGN, wn = wave % T::WGN;
  }
  __device__ inline int row(int i, int r) const { return wm * T::WM + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3); }
  __device__ inline int col(int j) const { return wn * T::WN + 32 * j + (lane & 31); }
};

// The tile's biases into LDS (-inf for what is no class), and the two sets of accumulators into one.
template <class T>
__device__ inline void biases_of_tile(floatx16 (&acc)[T::ACC][T::TM][T::TN], const float *__restrict__ bias, int m0, int M, float *lb) {
  for (int i = threadIdx.x; i < T::BM; i += T::THREADS) lb[i] = m0 + i >= M ? -INFINITY : bias ? bias[m0 + i] : 0.f;
  if constexpr (T::ACC > 1)
#pragma unroll
    for (int i = 0; i < T::TM; i++)
#pragma unroll
      for (int j = 0; j < T::TN; j++) acc[0][i][j] += acc[T::ACC - 1][i][j];
  __syncthreads();
}
// z of 16 classes: product + bias; those with a bias of -inf: -inf, whatever the product is.  (Biases are read again for each use: all of them in
// registers would take the room of a third workgroup.)
__device__ inline void logits16(const floatx16 &acc, const float *lb, float (&z)[16]) {
  asm volatile("" ::: "memory");
#pragma unroll
  for (int q = 0; q < 4; q++) {
    const float4 b = *reinterpret_cast<const float4 *>(lb + 8 * q);
    z[4 * q] = b.x == -INFINITY ? -INFINITY : acc[4 * q] + b.x;
    z[4 * q + 1] = b.y == -INFINITY ? -INFINITY : acc[4 * q + 1] + b.y;
    z[4 * q + 2] = b.z == -INFINITY ? -INFINITY : acc[4 * q + 2] + b.z;
    z[4 * q + 3] = b.w == -INFINITY ? -INFINITY : acc[4 * q + 3] + b.w;
  }
}

// The row of a lane's classes (counted from its first) that a label's class is; what is no class of this tile is no such row, or one beyond the
// last class, whose label weighs nothing.
template <class T>
__device__ inline int label_row(float label, int first, const Where<T> &w) {
  return label >= 0.f && label < 2147483648.f ? (int)label - first - w.row(0, 0) : -1;
}

struct TileArgs {
  PackedRef W, X;      // of the piece's classes, of the tokens
  int M, n, K;         // classes of the piece, tokens, k (a multiple of kPlaneAlign)
  int tilesM, tilesN;
  const float *bias;   // of the piece, or null
  const float *labels;
  int c0;              // first class of the piece
};

template <class T>
__global__ __launch_bounds__(T::THREADS, T::EU) void stats_kernel(TileArgs a, float2 *__restrict__ stats, float *__restrict__ zlabel) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS];
  int tm, tn;
  nt_tile_of(blockIdx.x, a.tilesM, a.tilesN, &tm, &tn);
  const int m0 = tm * T::BM, n0 = tn * T::BN;
  floatx16 acc[T::ACC][T::TM][T::TN];
  nt_multiply<T>(a.W, a.M, m0, a.X, a.n, n0, 0, a.K, S, acc);
  float *lb = reinterpret_cast<float *>(S);
  float2 *part = reinterpret_cast<float2 *>(S + T::BM * 4);  // [WGM][BN]
  const Where<T> w;
  biases_of_tile<T>(acc, a.bias, m0, a.M, lb);
#pragma unroll
  for (int j = 0; j < T::TN; j++) {
    const int token = n0 + w.col(j);
    const float label = token < a.n ? a.labels[token] : -1.f;
    const int at = label_row(label, a.c0 + m0, w);
    float top = -INFINITY, z[16];
#pragma unroll
    for (int i = 0; i < T::TM; i++) {
      logits16(acc[0][i][j], lb + w.row(i, 0), z);
#pragma unroll
      for (int r = 0; r < 16; r++) top = fmaxf(top, z[r]);
      if (!__any((unsigned)(at - 32 * i) < 32u)) continue;  // (few tiles hold one of their tokens' labels)
#pragma unroll
      for (int r = 0; r < 16; r++)
        if (at == 32 * i + 8 * (r >> 2) + (r & 3)) zlabel[token] = z[r];
    }
    top = fmaxf(top, __shfl_xor(top, 32));
    const float from = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < T::TM; i++) {
      logits16(acc[0][i][j], lb + w.row(i, 0), z);
#pragma unroll
      for (int r = 0; r < 16; r++) sum += __expf(z[r] - from);
    }
    sum += __shfl_xor(sum, 32);
    if (w.half == 0) part[w.wm * T::BN + w.col(j)] = make_float2(top, sum);
  }
  __syncthreads();
  for (int x = threadIdx.x; x < T::BN; x += T::THREADS) {
    if (n0 + x >= a.n) continue;
    float2 s = part[x];
#pragma unroll
    for (int q = 1; q < T::WGM; q++) {
      const float2 o = part[q * T::BN + x];
      const float top = fmaxf(s.x, o.x), from = top == -INFINITY ? 0.f : top;
      s = make_float2(top, s.y * __expf(s.x - from) + o.y * __expf(o.x - from));
    }
    stats[(long)(a.c0 / T::BM + tm) * a.n + n0 + x] = s;
  }
}

// What a row's tiles come to: lse, loss and the weight of its gradient (zero for a row without a class, or without any class that is not
// masked).  Sixteen rows to a workgroup, sixteen lanes to a row's tiles.
__global__ __launch_bounds__(256) void rows_kernel(const float2 *__restrict__ stats, int tiles, const float *__restrict__ zlabel, const float *__restrict__ labels,
                                                   int n, int C, float *__restrict__ loss, float *__restrict__ lse) {
  __shared__ float2 part[16][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, row = blockIdx.x * 16 + x;
  float2 s = make_float2(-INFINITY, 0.f);
  if (row < n)
    for (int t = y; t < tiles; t += 16) {
      const float2 o = stats[(long)t * n + row];
      const float top = fmaxf(s.x, o.x), from = top == -INFINITY ? 0.f : top;
      s = make_float2(top, s.y * __expf(s.x - from) + o.y * __expf(o.x - from));
    }
  part[y][x] = s;
  __syncthreads();
  if (y != 0 || row >= n) return;
  float top = s.x;
  for (int q = 1; q < 16; q++) top = fmaxf(top, part[q][x].x);
  const float from = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int q = 0; q < 16; q++) sum += part[q][x].y * expf(part[q][x].x - from);
  const float all = from + logf(sum), label = labels[row];
  const bool has = label >= 0.f && label < (float)C;
  if (lse) lse[row] = all;
  // (no class left: an infinite loss, not the NaN of -inf - -inf)
  if (loss) loss[row] = !has ? 0.f : all == -INFINITY ? INFINITY : all - zlabel[row];
}

__global__ __launch_bounds__(256) void weights_kernel(const float *__restrict__ labels, const float *__restrict__ lse, const float *__restrict__ dloss, int n,
                                                      int C, float *__restrict__ weight) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= n) return;
  const float label = labels[row];
  const bool has = label >= 0.f && label < (float)C && lse[row] != -INFINITY;
  weight[row] = has ? dloss ? dloss[row] : 1.f : 0.f;
}

// d of a tile: e = p - [label] for the product with W, by token, and e times the token's weight for that with X, by class (zero between the last
// class or token and the end of the steps); and the sums of the latter over the tile's tokens.
// What multiplies all of a row's d, or all of d, stays out of what is rounded: next to the label, where p is small, e is -1 and a bit, which bf16
// holds well, while any factor in it is a rounding error that all of its kind share.
template <class T>
__global__ __launch_bounds__(T::THREADS, T::EU) void dlogits_kernel(TileArgs a, const float *__restrict__ lse, const float *__restrict__ weight, PackedOut d,
                                                                    PackedOut t, float *__restrict__ sums, int ld_sums) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS];
  int tm, tn;
  nt_tile_of(blockIdx.x, a.tilesM, a.tilesN, &tm, &tn);
  const int m0 = tm * T::BM, n0 = tn * T::BN;
  floatx16 acc[T::ACC][T::TM][T::TN];
  nt_multiply<T>(a.W, a.M, m0, a.X, a.n, n0, 0, a.K, S, acc);
  float *lb = reinterpret_cast<float *>(S);
  float *part = lb + T::BM;  // [WGN][BM]
  const Where<T> w;
  char *turn = S + 4 * T::BM * (1 + T::WGN) + (threadIdx.x >> 6) * kTurn;
  static_assert(4 * T::BM * (1 + T::WGN) + T::WAVES * kTurn <= T::LDS, "");
  biases_of_tile<T>(acc, a.bias, m0, a.M, lb);
  int at[T::TN];
  float g[T::TN], all[T::TN];
#pragma unroll
  for (int j = 0; j < T::TN; j++) {
    const int token = n0 + w.col(j);
    const bool in = token < a.n;
    g[j] = in ? weight[token] : 0.f, all[j] = in ? lse[token] : 0.f;
    at[j] = g[j] != 0.f ? label_row(a.labels[token], a.c0 + m0, w) : -1;
  }
#pragma unroll
  for (int i = 0; i < T::TM; i++) {
    const int cb = (m0 + w.wm * T::WM) / 32 + i;
    float sum[16] = {};
#pragma unroll
    for (int j = 0; j < T::TN; j++) {
      const int xb = (n0 + w.wn * T::WN) / 32 + j;
      float x[16];
      logits16(acc[0][i][j], lb + w.row(i, 0), x);
#pragma unroll
      for (int r = 0; r < 16; r++) x[r] = g[j] == 0.f ? 0.f : __expf(x[r] - all[j]);
      if (__any((unsigned)(at[j] - 32 * i) < 32u)) {  // (few tiles hold one of their tokens' labels)
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] -= at[j] == 32 * i + 8 * (r >> 2) + (r & 3) ? 1.f : 0.f;
      }
      Parts16<T::P> e;
      if (d.p && 32 * xb < a.n && 32 * cb < d.K) {
#pragma unroll
        for (int r = 0; r < 16; r++) parts_of<T::P>(x[r], e.v[r]);
        put_rows<T::P>(d, xb, cb, e, w.lane);
      }
#pragma unroll
      for (int r = 0; r < 16; r++) x[r] *= g[j], sum[r] += x[r];
      if (t.p && 32 * cb < a.M && 32 * xb < t.K) {
#pragma unroll
        for (int r = 0; r < 16; r++) parts_of<T::P>(x[r], e.v[r]);
        put_columns<T::P>(t, cb, xb, e, w.lane, turn);
      }
    }
    if (!sums) continue;
#pragma unroll
    for (int r = 0; r < 16; r++) {
      float x = sum[r];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor(x, o);
      if ((w.lane & 31) == 0) part[w.wn * T::BM + w.row(i, r)] = x;
    }
  }
  if (!sums) return;
  __syncthreads();
  for (int x = threadIdx.x; x < T::BM; x += T::THREADS) {
    if (m0 + x >= a.M) continue;
    float s = part[x];
#pragma unroll
    for (int q = 1; q < T::WGN; q++) s += part[q * T::BM + x];
    sums[(long)tn * ld_sums + m0 + x] = s;
  }
}

// ------------------------------------------------------------------ the products with d
// out[row, col] = scale * A B^T.  K in `splits` stretches of kchunk, each with sums of its own (unscaled) at part + split * M * N; part null:
// straight to out.
template <class Out>
struct ProductJob {
  PackedRef A, B;
  int M, N, K, tilesM, tilesN, splits, kchunk;
  float *part;
  int add;  // what is there already is added to (`part`)
  Out *out;
  long ldo;
  float scale;
};

template <class T, class Out>
__global__ __launch_bounds__(T::THREADS, T::EU) void product_kernel(ProductJob<Out> j0, ProductJob<Out> j1, int blocks0) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS];
  const bool second = (int)blockIdx.x >= blocks0;
  const ProductJob<Out> &g = second ? j1 : j0;
  int block = second ? blockIdx.x - blocks0 : blockIdx.x, tm, tn;
  const int tiles = g.tilesM * g.tilesN, split = block / tiles;
  nt_tile_of(block - split * tiles, g.tilesM, g.tilesN, &tm, &tn);
  const int m0 = tm * T::BM, n0 = tn * T::BN, kbeg = split * g.kchunk, kend = min(g.K, kbeg + g.kchunk);
  floatx16 acc[T::ACC][T::TM][T::TN];
  nt_multiply<T>(g.A, g.M, m0, g.B, g.N, n0, kbeg, kend, S, acc);
  const Where<T> w;
  float *part = g.part ? g.part + (long)split * g.M * g.N : nullptr;
#pragma unroll
  for (int j = 0; j < T::TN; j++) {
    const int col = n0 + w.col(j);
    if (col >= g.N) continue;
#pragma unroll
    for (int i = 0; i < T::TM; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int row = m0 + w.row(i, r);
        if (row >= g.M) continue;
        float x = acc[0][i][j][r];
        if constexpr (T::ACC > 1) x += acc[T::ACC - 1][i][j][r];
        if (part) {
          float *o = part + (long)row * g.N + col;
          *o = g.add ? *o + x : x;
        } else {
          store_as(g.out + row * g.ldo + col, g.scale * x);
        }
      }
  }
}

// out[r, 0 .. w) = scale * factor[r] * sum of `parts` pieces, in their order
template <class Out>
__global__ __launch_bounds__(256) void parts_kernel(const float *__restrict__ part, int parts, int rows, int w, float scale, const float *__restrict__ factor,
                                                    Out *__restrict__ out, long ldo) {
  const long total = (long)rows * w;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    float s = parts > 0 ? part[i] : 0.f;
    for (int p = 1; p < parts; p++) s += part[p * total + i];
    const long r = i / w;
    store_as(out + r * ldo + (i - r * w), (factor ? scale * factor[r] : scale) * s);
  }
}

// ------------------------------------------------------------------ what a call consists of
template <int P> struct Tiles;
template <> struct Tiles<1> {
  using L = NtTile<1, 256, 128, 32, 2, 2>;
  using M = NtTile<1, 128, 128, 32, 2, 2>;
  using S = NtTile<1, 64, 64, 64, 2, 2>;
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
template <int P>
void tile_sides(int size, int *bm, int *bn) {
  with_tile<P>(size, [&](auto t) { return *bm = decltype(t)::BM, *bn = decltype(t)::BN, 0; });
}
// the largest tile that still gives most compute units one
template <int P>
int tile_size(long M, long N) {
  for (int size = 2; size > 0; size--) {
    int bm, bn;
    tile_sides<P>(size, &bm, &bn);
    if ((M + bm - 1) / bm * ((N + bn - 1) / bn) >= num_cus() * 3 / 4) return size;
  }
  return 0;
}

struct Call {
  const void *X, *W;
  int ldx, ldw;
  const float *b, *labels, *dloss;
  float scale;
  float *loss, *lse;
  const float *lse_given;
  void *dX, *dW;
  int lddx, lddw;
  float *db;
  int n, H, C;
};

constexpr int kPieceBytes = 256 << 20;  // d of a piece, in both orders
constexpr size_t kKeepBytes = 512 << 20;  // of W packed: kept from the first pass for the second
constexpr int kSplits = 8;

// Sizes and places of a call's workspace.
struct Plan {
  int P, size, bm, bn, Hp, np, piece, pieces, tiles;  // tiles: of the whole vocabulary
  int grads, keep, psize, pm, pn, xsplits, xchunk, wsplits, wchunk;
  size_t stats, zlabel, lse, weight, x, w, xt, wt, d, dt, sums, xpart, wpart, bytes;
};

template <int P>
Plan plan_of(int n, int H, int C, int grads) {
  Plan p{};
  p.P = P, p.grads = grads;
  p.Hp = ceil_to(H, kPlaneAlign), p.np = ceil_to(n, kPlaneAlign);
  long most = grads ? kPieceBytes / (4l * P * p.np) : (128l << 20) / (2l * P * p.Hp);
  most = most < 1024 ? 1024 : most > 1 << 20 ? 1 << 20 : most;
  p.pieces = (int)((C + most - 1) / most);
  p.piece = ceil_to((C + p.pieces - 1) / p.pieces, 256);
  p.pieces = tiles_of(C, p.piece);
  const int rows = p.piece < C ? p.piece : C;
  p.size = tile_size<P>(rows, n);
  tile_sides<P>(p.size, &p.bm, &p.bn);
  p.tiles = tiles_of(C, p.bm);
  p.keep = packed_bytes<P>(C, p.Hp) <= kKeepBytes;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  p.stats = take((size_t)p.tiles * n * 8);
  p.zlabel = take((size_t)n * 4);
  p.lse = take((size_t)n * 4);
  p.weight = take((size_t)n * 4);
  p.x = take(packed_bytes<P>(n, p.Hp));
  p.w = take(packed_bytes<P>(grads && p.keep ? C : rows, p.Hp));
  if (grads) {
    const int rp = ceil_to(rows, kPlaneAlign);
    p.psize = tile_size<P>((long)rows + n, H);
    tile_sides<P>(p.psize, &p.pm, &p.pn);
    // few tiles: K in several stretches, none of them short
    auto split = [&](long tiles, int K, int *chunk) {
      int s = (int)(num_cus() / (tiles > 0 ? tiles : 1));
      s = s > kSplits ? kSplits : s;
      s = s > K / 512 ? K / 512 : s;
      s = s < 1 ? 1 : s;
      *chunk = ceil_to((K + s - 1) / s, kPlaneAlign);
      return (K + *chunk - 1) / *chunk;
    };
    p.xsplits = split((long)tiles_of(n, p.pm) * tiles_of(H, p.pn), rp, &p.xchunk);
    p.wsplits = split((long)tiles_of(rows, p.pm) * tiles_of(H, p.pn), p.np, &p.wchunk);
    p.xt = take(packed_bytes<P>(H, p.np));
    p.wt = take(packed_bytes<P>(H, rp));
    p.d = take(packed_bytes<P>(n, rp));
    p.dt = take(packed_bytes<P>(rows, p.np));
    p.sums = take((size_t)tiles_of(n, p.bn) * C * 4);
    p.xpart = take((size_t)p.xsplits * n * H * 4);
    p.wpart = take(p.wsplits > 1 ? (size_t)p.wsplits * rows * H * 4 : 0);
  }
  p.bytes = at;
  return p;
}

template <int P, class Src>
void pack(const void *src, long ld, int rows, int K, PackedOut o, PackedOut t, const float *flag, int keep, hipStream_t st) {
  launch(pack_kernel<P, Src>, dim3(tiles_of(K, 64), tiles_of(rows, 64)), 256, 0, st, static_cast<const Src *>(src), ld, rows, K, o, t, flag, keep);
}

template <int P, class Src>
int run(const Call &c, const Plan &p, char *ws, hipStream_t st) {
  const int n = c.n, H = c.H, C = c.C;
  auto f32 = [&](size_t at) { return reinterpret_cast<float *>(ws + at); };
  auto pl = [&](size_t at) { return reinterpret_cast<u16 *>(ws + at); };
  auto ref = [](const PackedOut &o) { return PackedRef{o.p, o.K}; };
  const PackedOut none{}, X{pl(p.x), p.Hp};
  const bool keep = p.grads && p.keep;
  pack<P, Src>(c.X, c.ldx, n, H, X, none, nullptr, KEEP_ALL, st);
  float *lse = c.lse ? c.lse : f32(p.lse);
  auto piece_w = [&](int c0) { return PackedOut{pl(p.w + (keep ? packed_bytes<P>(c0, p.Hp) : 0)), p.Hp}; };
  auto source = [&](int c0) { return static_cast<const Src *>(c.W) + (long)c0 * c.ldw; };
  auto tile_args = [&](int c0, int rows) {
    return TileArgs{ref(piece_w(c0)), ref(X), rows, n, p.Hp, tiles_of(rows, p.bm), tiles_of(n, p.bn), c.b ? c.b + c0 : nullptr, c.labels, c0};
  };
  if (!c.lse_given) {
    for (int c0 = 0; c0 < C; c0 += p.piece) {
      const int rows = C - c0 < p.piece ? C - c0 : p.piece;
      pack<P, Src>(source(c0), c.ldw, rows, H, piece_w(c0), none, nullptr, KEEP_ALL, st);
      const TileArgs a = tile_args(c0, rows);
      with_tile<P>(p.size, [&](auto t) {
        using T = decltype(t);
        launch(stats_kernel<T>, a.tilesM * a.tilesN, T::THREADS, 0, st, a, reinterpret_cast<float2 *>(ws + p.stats), f32(p.zlabel));
        return 0;
      });
    }
    launch(rows_kernel, (n + 15) / 16, 256, 0, st, reinterpret_cast<const float2 *>(ws + p.stats), p.tiles, f32(p.zlabel), c.labels, n, C, c.loss, lse);
  }
  if (p.grads) {
    const float *all = c.lse_given ? c.lse_given : lse;
    float *weight = f32(p.weight);
    launch(weights_kernel, (n + 255) / 256, 256, 0, st, c.labels, all, c.dloss, n, C, weight);
    const PackedOut xt{pl(p.xt), p.np};
    if (c.dW) pack<P, Src>(c.X, c.ldx, n, H, none, xt, weight, KEEP_NONZERO, st);
    bool first = true;
    for (int c0 = 0; c0 < C; c0 += p.piece, first = false) {
      const int rows = C - c0 < p.piece ? C - c0 : p.piece, rp = ceil_to(rows, kPlaneAlign);
      const PackedOut wt{pl(p.wt), rp};
      // (what the first pass packed may still be there)
      const bool make = c.lse_given || (!keep && p.pieces > 1);
      if (c.dX || make)
        pack<P, Src>(source(c0), c.ldw, rows, H, make ? piece_w(c0) : none, c.dX ? wt : none, c.b ? c.b + c0 : nullptr, c.b ? KEEP_FINITE : KEEP_ALL, st);
      const TileArgs a = tile_args(c0, rows);
      const PackedOut d{c.dX ? pl(p.d) : nullptr, rp}, dt{c.dW ? pl(p.dt) : nullptr, p.np};
      with_tile<P>(p.size, [&](auto t) {
        using T = decltype(t);
        launch(dlogits_kernel<T>, a.tilesM * a.tilesN, T::THREADS, 0, st, a, all, weight, d, dt, c.db ? f32(p.sums) + c0 : nullptr, C);
        return 0;
      });
      auto job = [&](const PackedOut &A, const PackedOut &B, int M, int K, int chunk, float *part, bool add, void *out, long ldo) {
        return ProductJob<Src>{ref(A), ref(B), M, H, K, tiles_of(M, p.pm), tiles_of(H, p.pn), (K + chunk - 1) / chunk, chunk, part, add,
                               static_cast<Src *>(out), ldo, c.scale};
      };
      ProductJob<Src> jx{}, jw{};
      // (a last piece shorter than the others fills fewer stretches: those beyond keep what they have)
      if (c.dX) jx = job(d, wt, n, rp, p.xchunk, f32(p.xpart), !first, nullptr, 0);
      Src *dW = c.dW ? static_cast<Src *>(c.dW) + (long)c0 * c.lddw : nullptr;
      if (c.dW) jw = job(dt, xt, rows, p.np, p.wchunk, p.wsplits > 1 ? f32(p.wpart) : nullptr, false, dW, c.lddw);
      const int bx = c.dX ? jx.tilesM * jx.tilesN * jx.splits : 0, bw = c.dW ? jw.tilesM * jw.tilesN * jw.splits : 0;
      if (bx + bw > 0)
        with_tile<P>(p.psize, [&](auto t) {
          using T = decltype(t);
          launch(product_kernel<T, Src>, bx + bw, T::THREADS, 0, st, jx, jw, bx);
          return 0;
        });
      if (c.dW && p.wsplits > 1) launch(parts_kernel<Src>, 2048, 256, 0, st, f32(p.wpart), p.wsplits, rows, H, c.scale, nullptr, dW, (long)c.lddw);
    }
    if (c.dX) launch(parts_kernel<Src>, 2048, 256, 0, st, f32(p.xpart), p.xsplits, n, H, c.scale, weight, static_cast<Src *>(c.dX), (long)c.lddx);
    if (c.db) launch(parts_kernel<float>, 512, 256, 0, st, f32(p.sums), tiles_of(n, p.bn), 1, C, c.scale, nullptr, c.db, (long)C);
  }
  CAVS_LAUNCH_CHECK();
  return CAVS_OK;
}

constexpr int kMostRows = 1 << 20, kMostH = 1 << 16, kMostClasses = 1 << 23;  // (offsets within a tile's rows are below 2^32 bytes)

bool plan(int type, int n, int H, int C, int grads, Plan *p) {
  if (n <= 0 || H <= 0 || C <= 0 || n > kMostRows || H > kMostH || C > kMostClasses || (type != CAVS_F32 && type != CAVS_BF16)) return false;
  *p = type == CAVS_F32 ? plan_of<3>(n, H, C, grads) : plan_of<1>(n, H, C, grads);
  return true;
}

int check_and_run(const char *who, int type, const Call &c, int grads, void *ws, size_t ws_bytes, void *stream) {
  CAVS_REQUIRE(type == CAVS_F32 || type == CAVS_BF16, "%s: type %d is neither CAVS_F32 nor CAVS_BF16", who, type);
  CAVS_REQUIRE(c.n >= 0 && c.H > 0 && c.C > 0, "%s: bad shape n=%d H=%d C=%d", who, c.n, c.H, c.C);
  CAVS_REQUIRE(c.H <= kMostH && c.n <= kMostRows && c.C <= kMostClasses, "%s: unsupported shape n=%d H=%d C=%d (at most 2^20, 2^16, 2^23)", who, c.n, c.H, c.C);
  CAVS_REQUIRE(c.ldx >= c.H && c.ldw >= c.H && (!c.dX || c.lddx >= c.H) && (!c.dW || c.lddw >= c.H), "%s: a row stride is below H=%d", who, c.H);
  CAVS_REQUIRE(c.W && (c.n == 0 || (c.X && c.labels)), "%s: null pointer", who);
  if (c.n == 0) {  // sums over no rows
    hipStream_t st = as_stream(stream);
    if (c.dW && type == CAVS_F32) launch(parts_kernel<float>, 2048, 256, 0, st, nullptr, 0, c.C, c.H, 0.f, nullptr, static_cast<float *>(c.dW), (long)c.lddw);
    if (c.dW && type == CAVS_BF16) launch(parts_kernel<u16>, 2048, 256, 0, st, nullptr, 0, c.C, c.H, 0.f, nullptr, static_cast<u16 *>(c.dW), (long)c.lddw);
    if (c.db) launch(parts_kernel<float>, 64, 256, 0, st, nullptr, 0, 1, c.C, 0.f, nullptr, c.db, (long)c.C);
    CAVS_LAUNCH_CHECK();
    return CAVS_OK;
  }
  Plan p;
  plan(type, c.n, c.H, c.C, grads, &p);
  CAVS_REQUIRE(ws && ws_bytes >= p.bytes, "%s: workspace of %zu bytes needed, %zu given", who, p.bytes, ws_bytes);
  CAVS_REQUIRE(aligned16(ws), "%s: the workspace must be 16-byte aligned", who);
  char *w = static_cast<char *>(ws);
  return type == CAVS_F32 ? run<3, float>(c, p, w, as_stream(stream)) : run<1, u16>(c, p, w, as_stream(stream));
}

}  // namespace
}  // namespace cavs

using namespace cavs;

extern "C" {

size_t cavs_vocab_xent_workspace(int type, int n, int H, int C, int grads) {
  Plan p;
  return plan(type, n, H, C, grads, &p) ? p.bytes : 0;
}

int cavs_vocab_xent_fwd(int type, const void *X, int ldx, const void *W, int ldw, const float *b, const float *labels, float *loss, float *lse, int n, int H,
                        int C, void *workspace, size_t workspace_bytes, void *stream) {
  Call c{};
  c.X = X, c.ldx = ldx, c.W = W, c.ldw = ldw, c.b = b, c.labels = labels, c.loss = loss, c.lse = lse, c.n = n, c.H = H, c.C = C;
  CAVS_REQUIRE(loss || lse || n == 0, "cavs_vocab_xent_fwd: neither loss nor lse is wanted");
  return check_and_run("cavs_vocab_xent_fwd", type, c, 0, workspace, workspace_bytes, stream);
}

int cavs_vocab_xent_bwd(int type, const void *X, int ldx, const void *W, int ldw, const float *b, const float *labels, const float *lse, const float *dloss,
                        float scale, void *dX, int lddx, void *dW, int lddw, float *db, int n, int H, int C, void *workspace, size_t workspace_bytes,
                        void *stream) {
  Call c{X, W, ldx, ldw, b, labels, dloss, scale, nullptr, nullptr, lse, dX, dW, lddx, lddw, db, n, H, C};
  CAVS_REQUIRE(lse || n == 0, "cavs_vocab_xent_bwd: null pointer");
  return check_and_run("cavs_vocab_xent_bwd", type, c, 1, workspace, workspace_bytes, stream);
}

int cavs_vocab_xent(int type, const void *X, int ldx, const void *W, int ldw, const float *b, const float *labels, const float *dloss, float scale, float *loss,
                    float *lse, void *dX, int lddx, void *dW, int lddw, float *db, int n, int H, int C, void *workspace, size_t workspace_bytes, void *stream) {
  Call c{X, W, ldx, ldw, b, labels, dloss, scale, loss, lse, nullptr, dX, dW, lddx, lddw, db, n, H, C};
  return check_and_run("cavs_vocab_xent", type, c, 1, workspace, workspace_bytes, stream);
}

}  // extern "C"
