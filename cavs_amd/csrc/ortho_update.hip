// Momentum, orthogonalised by Newton-Schulz products, for several matrices at once.
//
//   M <- mu M + G,  U = G + mu M or M,  X = U / (|U| + eps);  `steps` times  X <- (a I + b A + c A A) X, A = X X^T
//
// on the side that is smaller: m x n with m <= n.  Three products a step, each one launch over all matrices: A and a I + b A + c A A are
// symmetric, so only blocks on the diagonal and below are made, and those below are stored twice.  What a launch makes is
// what the next ones read, packed as bf16 parts (nt_product.h): X by rows (for A) and by columns (for the product
// with it), A and the polynomial by rows, which are their columns.
//
// A singular value next to 0 grows a-fold a step, 485-fold in five, and so does a rounding error made beside it.  With three parts X, A and the
// polynomial keep an fp32's bits and the result is as far off as in fp32.  Where nothing but a result rounded to bf16 is wanted, two parts do for as long as
// what they leave off, 2^-17 of the largest, has grown to no more than half a step of bf16, 2^-8.  (Error of the result, a bf16 gradient of
// rank 3 to the last bit, 96 x 160, two / three parts: 5 steps 0.0020 / 0.0017 of its norm, 6 steps 0.0028 / 0.0017, 8 steps 0.042 / 0.0018, 10 steps
// 0.48 / 0.0083; rounding alone 0.0017.  One part, 2^-9, would come out as large as the result.)
#include "nt_product.h"

namespace cavs {
namespace {

constexpr int kMats = 16;       // matrices of a launch
constexpr int kNormBlocks = 256; // workgroups that add up a matrix's squares

struct Mat {
  const void *G;
  float *M, *W;
  void *O;
  long ldg, ldm, ldw, ldo;
  int rows, cols;      // as the caller has them
  int m, n, mp, np;    // of X, and padded to whole steps
  u16 *X, *Xt[2], *A, *Q;  // packed: [m, np], [n, mp] (read, written), [m, mp], [m, mp]
  float shrink;        // sqrt(max(1, outputs / inputs))
};

struct Common {
  int count, nesterov;
  float a, b, c, eps, momentum, lr, decay;
  const int *guard;
  double *squares;     // [kMats][kNormBlocks]
  int *arrived;        // a counter for every tile of a launch, zero between launches
  int counters;
  float *part;         // tiles of stretches of K
};

__device__ inline bool held_back(const Common &c) { return c.guard && *c.guard != 0; }

// M <- mu M + G, and the squares of U, added up in 64 bits in a fixed order
struct NormArgs {
  Mat m[kMats];
  Common c;
};
template <class Src>
__global__ __launch_bounds__(256) void norm_kernel(NormArgs g) {
  const Common &c = g.c;
  const int who = blockIdx.y;
  if (who == 0)
    for (int i = blockIdx.x * 256 + threadIdx.x; i < c.counters; i += gridDim.x * 256) c.arrived[i] = 0;
  if (held_back(c)) return;
  const Mat &t = g.m[who];
  double sum = 0.;
  // lanes along a row, four neighbouring values each, as many rows at a time as there are lanes left; four loads of a lane on their way.  (One value a
  // load: bf16 of 8192 x 4096 and 4096 x 4096 184 us, 46 now.)
  typedef Src four __attribute__((ext_vector_type(4), aligned(sizeof(Src))));
  typedef float four32 __attribute__((ext_vector_type(4), aligned(4)));
  int across = 16;
  while (across < 256 && 16 * across < t.cols) across *= 2;
  const int high = 256 / across, x = threadIdx.x % across, y = threadIdx.x / across;
  for (long r0 = (long)blockIdx.x * high; r0 < t.rows; r0 += (long)gridDim.x * high) {
    const long r = r0 + y;
    if (r >= t.rows) continue;
    const Src *G = static_cast<const Src *>(t.G) + r * t.ldg;
    float *M = t.M ? t.M + r * t.ldm : nullptr;
    for (int k0 = 4 * x; k0 < t.cols; k0 += 16 * across) {
      four gr[4];
      four32 mo[4];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int k = k0 + 4 * q * across;
        if (k + 4 <= t.cols) {
          gr[q] = *reinterpret_cast<const four *>(G + k);
          if (M) mo[q] = *reinterpret_cast<const four32 *>(M + k);
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            gr[q][e] = k + e < t.cols ? G[k + e] : Src(0);
            if (M) mo[q][e] = k + e < t.cols ? M[k + e] : 0.f;
          }
        }
      }
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int k = k0 + 4 * q * across;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const Src one = gr[q][e];
          const float v = value_of(&one);
          float u = v;
          if (M) {
            mo[q][e] = fmaf(c.momentum, mo[q][e], v);
            u = c.nesterov ? fmaf(c.momentum, mo[q][e], v) : mo[q][e];
          }
          sum += (double)u * u;  // (zero beyond the last column)
        }
        if (M && k + 4 <= t.cols) {
          *reinterpret_cast<four32 *>(M + k) = mo[q];
        } else if (M) {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (k + e < t.cols) M[k + e] = mo[q][e];
        }
      }
    }
  }
  __shared__ double s[256];
  s[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) c.squares[who * kNormBlocks + blockIdx.x] = s[0];
}

// X by rows and by columns, 64 x 64 at a time
struct StartArgs {
  Mat m[kMats];
  Common c;
  int first[kMats + 1];
};
template <int P, class Src>
__global__ __launch_bounds__(256) void start_kernel(StartArgs g) {
  __shared__ PackTile tile;
  const Common &c = g.c;
  if (held_back(c)) return;
  int who = 0;
  while (who + 1 < c.count && (int)blockIdx.x >= g.first[who + 1]) who++;
  const Mat &t = g.m[who];
  const bool flat = t.rows <= t.cols;
  const int across = (flat ? t.np : t.mp) / 64, block = blockIdx.x - g.first[who];
  const int r0 = block / across * 64, k0 = block % across * 64, k = threadIdx.x & 63;
  // (all of a lane's values on their way while the norm is made)
  float gr[16], mo[16];
  auto in = [&](int i) { return r0 + (int)(threadIdx.x >> 6) + 4 * i < t.rows && k0 + k < t.cols; };
  auto at = [&](int i, long ld) { return (long)(r0 + (threadIdx.x >> 6) + 4 * i) * ld + k0 + k; };
#pragma unroll
  for (int i = 0; i < 16; i++) gr[i] = in(i) ? value_of(static_cast<const Src *>(t.G) + at(i, t.ldg)) : 0.f;
#pragma unroll
  for (int i = 0; i < 16; i++) mo[i] = t.M && in(i) ? t.M[at(i, t.ldm)] : 0.f;
  __shared__ double s[kNormBlocks];
  s[threadIdx.x] = c.squares[who * kNormBlocks + threadIdx.x];
  for (int o = kNormBlocks / 2; o > 0; o >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
  }
  __syncthreads();
  const double by = s[0] == 0. ? 0. : 1. / (sqrt(s[0]) + (double)c.eps);  // (nothing stays nothing, with eps = 0 too)
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const float u = !t.M ? gr[i] : c.nesterov ? fmaf(c.momentum, mo[i], gr[i]) : mo[i];
    tile[(threadIdx.x >> 6) + 4 * i][k] = in(i) ? (float)((double)u * by) : 0.f;
  }
  __syncthreads();
  const PackedOut X{t.X, t.np}, Xt{t.Xt[0], t.mp};
  pack_tile<P>(tile, flat ? X : Xt, flat ? Xt : X, r0, k0, t.rows, t.cols);
}

enum { GRAM = 0, POLYNOMIAL = 1, APPLY = 2, LAST = 3 };

struct ProductArgs {
  Mat m[kMats];
  Common c;
  int first[kMats + 1];              // workgroups
  int tilesN[kMats], splits[kMats], chunk[kMats], tiles0[kMats];  // tiles0: of the counters
  long part0[kMats];
};

// Tile `t` of those of a symmetric m x m result that reach the diagonal or below
template <class T>
__device__ inline void lower_tile(int t, int m, int *tm, int *tn) {
  const int tilesN = (m + T::BN - 1) / T::BN;
  int row = 0;
  for (;; row++) {
    const int here = min(tilesN, (row * T::BM + T::BM + T::BN - 1) / T::BN);
    if (t < here) break;
    t -= here;
  }
  *tm = row, *tn = t;
}
template <class T>
int lower_tiles(int m) {
  const int tilesM = (m + T::BM - 1) / T::BM, tilesN = (m + T::BN - 1) / T::BN;
  int all = 0;
  for (int row = 0; row < tilesM; row++) {
    const int here = (row * T::BM + T::BM + T::BN - 1) / T::BN;
    all += here < tilesN ? here : tilesN;
  }
  return all;
}

template <class T, class Src, int STAGE>
__global__ __launch_bounds__(T::THREADS, T::EU) void ortho_product_kernel(ProductArgs g) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS];
  const Common &c = g.c;
  if (held_back(c)) return;
  int who = 0;
  while (who + 1 < c.count && (int)blockIdx.x >= g.first[who + 1]) who++;
  const Mat &t = g.m[who];
  const int m = t.m, n = t.n, splits = g.splits[who];
  int block = blockIdx.x - g.first[who];
  const int tiles = (g.first[who + 1] - g.first[who]) / splits, split = block / tiles, id = block - split * tiles;
  constexpr bool SYM = STAGE == GRAM || STAGE == POLYNOMIAL;
  int tm, tn;
  if constexpr (SYM) lower_tile<T>(xcd_remap(id, tiles), m, &tm, &tn);
  else nt_tile_of(id, tiles / g.tilesN[who], g.tilesN[who], &tm, &tn);  // (the plan's, for this matrix's orientation)
  const int m0 = tm * T::BM, n0 = tn * T::BN;
  // The last product is made so that a row of the result is a row of the accumulators, whichever side of X is the longer one in the caller's.
  const bool turned = STAGE == LAST && t.rows <= t.cols;
  const PackedRef X{t.X, t.np}, Xt{t.Xt[0], t.mp}, A1{t.A, t.mp}, Q{t.Q, t.mp};
  const PackedRef &A = STAGE == GRAM ? X : STAGE == POLYNOMIAL ? A1 : turned ? Q : Xt, &B = STAGE == GRAM ? X : STAGE == POLYNOMIAL ? A1 : turned ? Xt : Q;
  const int K = STAGE == GRAM ? t.np : t.mp, kbeg = split * g.chunk[who], kend = min(K, kbeg + g.chunk[who]);
  const int M = SYM || turned ? m : n, N = turned ? n : m;
  floatx16 acc[T::ACC][T::TM][T::TN];
  nt_multiply<T>(A, M, m0, B, N, n0, kbeg, kend, S, acc);
  if constexpr (T::ACC > 1)
#pragma unroll
    for (int i = 0; i < T::TM; i++)
#pragma unroll
      for (int j = 0; j < T::TN; j++) acc[0][i][j] += acc[T::ACC - 1][i][j];

  if (splits > 1) {
    // Each stretch of K leaves its tile; whoever is the last to arrive adds them up in their order and goes on.  Past this XCD's L2, as the
    // others may be anywhere; the count goes up once the stores have arrived.  (Fences instead, which write back and drop all of an L2: 105 us a
    // launch where this takes 20.)
    float *here = c.part + g.part0[who] + (long)id * splits * (T::BM * T::BN) + threadIdx.x;
    auto at = [&](int s, int e) { return here + (long)s * (T::BM * T::BN) + e * T::THREADS; };
#pragma unroll
    for (int e = 0; e < T::TM * T::TN * 16; e++)
      __hip_atomic_store(at(split, e), acc[0][e / 16 / T::TN][e / 16 % T::TN][e % 16], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    int *last = reinterpret_cast<int *>(S);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      int *counter = c.arrived + g.tiles0[who] + id;
      const bool all = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == splits - 1;
      if (all) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      *last = all;
    }
    __syncthreads();
    if (!*last) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T::TM; i++)
#pragma unroll
      for (int j = 0; j < T::TN; j++) {
        float sum[16] = {};
        for (int s = 0; s < splits; s += 4) {  // four stretches' loads on their way at a time
          float v[4][16];
#pragma unroll
          for (int k = 0; k < 4; k++)
#pragma unroll
            for (int r = 0; r < 16; r++)
              v[k][r] = __hip_atomic_load(at(s + k < splits ? s + k : s, (i * T::TN + j) * 16 + r), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
          for (int k = 0; k < 4; k++)
#pragma unroll
            for (int r = 0; r < 16; r++) sum[r] += s + k < splits ? v[k][r] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < 16; r++) acc[0][i][j][r] = sum[r];
      }
  }

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  char *turn = S + wave * kTurn;
#pragma unroll
  for (int i = 0; i < T::TM; i++)
#pragma unroll
    for (int j = 0; j < T::TN; j++) {
      // the block of 32 rows and of 32 columns; this lane's column, the first of its rows
      const int rb = (m0 + wave / T::WGN * T::WM) / 32 + i, cb = (n0 + wave % T::WGN * T::WN) / 32 + j;
      const int col = 32 * cb + (lane & 31), row0 = 32 * rb + 4 * (lane >> 5);
      auto row = [&](int r) { return row0 + 8 * (r >> 2) + (r & 3); };
      float x[16];
#pragma unroll
      for (int r = 0; r < 16; r++) x[r] = acc[0][i][j][r];
      if constexpr (SYM) {
        // blocks above the diagonal are the mirror images of those below; of one on it both halves are here
        if (32 * cb >= m || 32 * rb >= t.mp || rb < cb) continue;
        if constexpr (STAGE == POLYNOMIAL) {
          // (A's parts by its columns' rows: A is symmetric)
#pragma unroll
          for (int q = 0; q < 4; q++) {
            float A4[4] = {};
#pragma unroll
            for (int p = T::P - 1; p >= 0; p--) {
              const uint2 v = *reinterpret_cast<const uint2 *>(t.A + (((long)cb * (t.mp / 16) + 2 * rb + (q >> 1)) * T::P + p) * 512 +
                                                               ((lane & 31) + 32 * (q & 1)) * 8 + 4 * (lane >> 5));
              A4[0] += __uint_as_float(v.x << 16), A4[1] += __uint_as_float(v.x & 0xffff0000u);
              A4[2] += __uint_as_float(v.y << 16), A4[3] += __uint_as_float(v.y & 0xffff0000u);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) x[4 * q + k] = fmaf(c.c, x[4 * q + k], c.b * A4[k]) + (row(4 * q + k) == col ? c.a : 0.f);
          }
        }
        Parts16<T::P> e;
#pragma unroll
        for (int r = 0; r < 16; r++) parts_of<T::P>(row(r) < m ? x[r] : 0.f, e.v[r]);
        const PackedOut o{STAGE == GRAM ? t.A : t.Q, t.mp};
        put_rows<T::P>(o, cb, rb, e, lane);
        if (rb > cb && 32 * rb < m) put_columns<T::P>(o, rb, cb, e, lane, turn);
      } else if constexpr (STAGE == APPLY) {
        Parts16<T::P> e;
#pragma unroll
        for (int r = 0; r < 16; r++) parts_of<T::P>(row(r) < n && col < m ? x[r] : 0.f, e.v[r]);
        if (32 * cb < m && 32 * rb < t.np) put_rows<T::P>(PackedOut{t.X, t.np}, cb, rb, e, lane);
        if (32 * rb < n && 32 * cb < t.mp) put_columns<T::P>(PackedOut{t.Xt[1], t.mp}, rb, cb, e, lane, turn);
      } else {
        if (col >= t.cols) continue;
        float w[16];  // (all of them on their way before the first is stored)
        if (t.W)
#pragma unroll
          for (int r = 0; r < 16; r++) w[r] = row(r) < t.rows ? t.W[row(r) * t.ldw + col] : 0.f;
#pragma unroll
        for (int r = 0; r < 16; r++) {
          if (row(r) >= t.rows) continue;
          if (t.O) store_as(static_cast<Src *>(t.O) + row(r) * t.ldo + col, x[r]);
          if (t.W) t.W[row(r) * t.ldw + col] = fmaf(1.f - c.lr * c.decay, w[r], -c.lr * t.shrink * x[r]);
        }
      }
    }
}

// ------------------------------------------------------------------ what a call consists of
template <int P> struct Tiles;
template <> struct Tiles<2> {
  using L = NtTile<2, 128, 128, 16, 2, 2, 3>;
  using S = NtTile<2, 64, 64, 32, 2, 2, 3>;
};
template <> struct Tiles<3> {
  using L = NtTile<3, 128, 128, 16, 2, 2>;
  using S = NtTile<3, 64, 64, 32, 2, 2, 3>;
};

struct Plan {
  size_t squares, arrived, part, bytes;
  int counters;
};

struct Shape {
  int m, n, mp, np;
  explicit Shape(const cavs_ortho_desc &d) {
    m = d.rows < d.cols ? d.rows : d.cols, n = d.rows < d.cols ? d.cols : d.rows;
    mp = ceil_to(m, kPlaneAlign), np = ceil_to(n, kPlaneAlign);
  }
};

// One launch's tiles; where they are few, K in stretches, none of them short
template <class T>
struct LaunchPlan {
  int first[kMats + 1], tilesN[kMats], splits[kMats], chunk[kMats], tiles0[kMats];
  long part0[kMats], parts;
  int tiles;
  LaunchPlan(const cavs_ortho_desc *d, int count, int stage) {
    long work = 0;  // tiles times k
    tiles = 0;
    int own[kMats], K[kMats];
    for (int i = 0; i < count; i++) {
      const Shape s(d[i]);
      const bool turned = stage == LAST && d[i].rows <= d[i].cols;
      tilesN[i] = tiles_of(turned ? s.n : s.m, T::BN);
      own[i] = stage == GRAM || stage == POLYNOMIAL ? lower_tiles<T>(s.m) : tilesN[i] * tiles_of(turned ? s.m : s.n, T::BM);
      K[i] = stage == GRAM ? s.np : s.mp;
      tiles0[i] = tiles;
      tiles += own[i];
      work += (long)own[i] * K[i];
    }
    // (of 300 x 512 and 512 x 512, four each, 204 tiles: all of K at once 285 us a call, in two stretches 307; of 128 x 512, two, 6 tiles: 159, in
    // stretches of 256 154, of 128 144)
    const bool few = 2 * tiles <= num_cus();
    const int step = ceil_to((int)(work / (2l * num_cus())) + 128, kPlaneAlign);
    first[0] = 0, parts = 0;
    for (int i = 0; i < count; i++) {
      splits[i] = !few || K[i] <= step ? 1 : (K[i] + step - 1) / step;
      chunk[i] = splits[i] == 1 ? K[i] : ceil_to((K[i] + splits[i] - 1) / splits[i], kPlaneAlign);
      splits[i] = (K[i] + chunk[i] - 1) / chunk[i];
      first[i + 1] = first[i] + own[i] * splits[i];
      part0[i] = parts;
      if (splits[i] > 1) parts += (long)own[i] * splits[i] * T::BM * T::BN;
    }
  }
};

// The tiles with the shorter longest way: as many as the fullest compute unit gets, times what one takes (a small one a third longer for its
// size).  Eight of 1024 x 1024: 288 large tiles 85 us, 1088 small ones 72; their last product, 512 large tiles 112 us.
template <int P, class F>
auto with_tile(const cavs_ortho_desc *d, int count, int stage, F &&f) {
  using L = typename Tiles<P>::L;
  using S = typename Tiles<P>::S;
  const int large = LaunchPlan<L>(d, count, stage).tiles, small = LaunchPlan<S>(d, count, stage).tiles;
  if ((long)tiles_of(large, num_cus()) * L::BM * L::BN * 3 > (long)tiles_of(small, num_cus()) * S::BM * S::BN * 4) return f(S{});
  return f(L{});
}

// what a matrix takes, packed: X, two Xt, A and the polynomial
template <int P>
size_t room_of(const Shape &s) {
  return packed_bytes<P>(s.m, s.np) + 2 * packed_bytes<P>(s.n, s.mp) + 2 * packed_bytes<P>(s.m, s.mp);
}

template <int P>
Plan plan_of(const cavs_ortho_desc *d, int count) {
  Plan p{};
  size_t most = 0;
  long parts = 0;
  for (int at = 0; at < count; at += kMats) {  // (batches come one after the other, in the same room)
    const int k = count - at < kMats ? count - at : kMats;
    size_t bytes = 0;
    for (int i = 0; i < k; i++) bytes += (room_of<P>(Shape(d[at + i])) + 255) & ~(size_t)255;
    most = bytes > most ? bytes : most;
    for (int stage = GRAM; stage <= LAST; stage++)
      with_tile<P>(d + at, k, stage, [&](auto t) {
        const LaunchPlan<decltype(t)> l(d + at, k, stage);
        parts = l.parts > parts ? l.parts : parts;
        p.counters = l.tiles > p.counters ? l.tiles : p.counters;
        return 0;
      });
  }
  p.squares = most;
  p.arrived = p.squares + sizeof(double) * kMats * kNormBlocks;
  p.part = (p.arrived + sizeof(int) * p.counters + 255) & ~(size_t)255;
  p.bytes = p.part + sizeof(float) * parts;
  return p;
}

template <int P, class Src, int STAGE>
void product(const cavs_ortho_desc *d, int count, const Mat *m, const Common &c, hipStream_t st) {
  with_tile<P>(d, count, STAGE, [&](auto tile) {
    using T = decltype(tile);
    const LaunchPlan<T> l(d, count, STAGE);
    ProductArgs a{};
    a.c = c;
    for (int i = 0; i < count; i++) {
      a.m[i] = m[i];
      a.tilesN[i] = l.tilesN[i], a.splits[i] = l.splits[i], a.chunk[i] = l.chunk[i], a.tiles0[i] = l.tiles0[i], a.part0[i] = l.part0[i];
    }
    for (int i = 0; i <= count; i++) a.first[i] = l.first[i];
    launch(ortho_product_kernel<T, Src, STAGE>, l.first[count], T::THREADS, 0, st, a);
    return 0;
  });
}

template <int P, class Src>
int run(const cavs_ortho_desc *d, int count, const cavs_ortho_options &o, bool in_out, const Plan &p, char *ws, hipStream_t st) {
  Common c{};
  c.nesterov = o.nesterov, c.a = o.a, c.b = o.b, c.c = o.c, c.eps = o.eps, c.momentum = o.momentum, c.lr = o.lr, c.decay = o.weight_decay, c.guard = o.guard;
  c.squares = reinterpret_cast<double *>(ws + p.squares);
  c.arrived = reinterpret_cast<int *>(ws + p.arrived);
  c.counters = p.counters;
  c.part = reinterpret_cast<float *>(ws + p.part);
  for (int at = 0; at < count; at += kMats) {
    const int k = count - at < kMats ? count - at : kMats;
    const cavs_ortho_desc *b = d + at;
    c.count = k;
    StartArgs s{};
    NormArgs nm{};
    char *room = ws;
    for (int i = 0; i < k; i++) {
      const Shape h(b[i]);
      char *next = room;
      auto take = [&](size_t bytes) {
        u16 *here = reinterpret_cast<u16 *>(next);
        next += bytes;
        return here;
      };
      Mat t{b[i].G, b[i].M, b[i].W, b[i].O, b[i].ldg, b[i].ldm, b[i].ldw, b[i].ldo, b[i].rows, b[i].cols, h.m, h.n, h.mp, h.np};
      t.X = take(packed_bytes<P>(h.m, h.np)), t.Xt[0] = take(packed_bytes<P>(h.n, h.mp)), t.Xt[1] = take(packed_bytes<P>(h.n, h.mp));
      t.A = take(packed_bytes<P>(h.m, h.mp)), t.Q = take(packed_bytes<P>(h.m, h.mp));
      const int outputs = in_out ? b[i].cols : b[i].rows, inputs = in_out ? b[i].rows : b[i].cols;
      t.shrink = outputs > inputs ? (float)__builtin_sqrt((double)outputs / inputs) : 1.f;
      room += (room_of<P>(h) + 255) & ~(size_t)255;
      s.m[i] = nm.m[i] = t;
      s.first[i + 1] = s.first[i] + tiles_of(b[i].rows, 64) * tiles_of(b[i].cols, 64);
    }
    s.c = nm.c = c;
    launch(norm_kernel<Src>, dim3(kNormBlocks, k), 256, 0, st, nm);
    launch(start_kernel<P, Src>, s.first[k], 256, 0, st, s);
    for (int step = 0; step < o.steps; step++) {
      product<P, Src, GRAM>(b, k, s.m, c, st);
      product<P, Src, POLYNOMIAL>(b, k, s.m, c, st);
      if (step + 1 < o.steps) product<P, Src, APPLY>(b, k, s.m, c, st);
      else product<P, Src, LAST>(b, k, s.m, c, st);
      for (int i = 0; i < k; i++) {
        u16 *x = s.m[i].Xt[0];
        s.m[i].Xt[0] = s.m[i].Xt[1], s.m[i].Xt[1] = x;
      }
    }
  }
  CAVS_LAUNCH_CHECK();
  return CAVS_OK;
}

constexpr int kMostSide = 1 << 16;

// How far the steps carry an error of X: the largest slope of their map at singular values up to 1 (with coefficients that orthogonalise, a^steps, at 0)
double growth(const cavs_ortho_options &o) {
  double most = 1.;
  for (int i = 0; i <= 16; i++) {
    double x = i / 16., slope = 1.;
    for (int step = 0; step < o.steps; step++) {
      const double s = x * x;
      slope *= o.a + s * (3. * o.b + s * 5. * o.c);
      x *= o.a + s * (o.b + s * o.c);
      if (!(fabs(slope) <= most)) most = fabs(slope);
    }
  }
  return most;
}

// whether two parts hold what is wanted
bool two_parts(int type, int count, const cavs_ortho_desc *d, const cavs_ortho_options &o) {
  for (int i = 0; i < count; i++)
    if (d[i].W) return false;
  return type == CAVS_BF16 && growth(o) <= 512.;  // (2^-8 over 2^-17)
}

bool sizes_ok(int type, int count, const cavs_ortho_desc *d) {
  if ((type != CAVS_F32 && type != CAVS_BF16) || count < 0 || (count > 0 && !d)) return false;
  for (int i = 0; i < count; i++)
    if (d[i].rows <= 0 || d[i].cols <= 0 || d[i].rows > kMostSide || d[i].cols > kMostSide) return false;
  return true;
}

int check_and_run(const char *who, int type, int count, const cavs_ortho_desc *d, const cavs_ortho_options *o, bool in_out, void *workspace, size_t workspace_bytes,
                  void *stream) {
  CAVS_REQUIRE(type == CAVS_F32 || type == CAVS_BF16, "%s: type %d is neither CAVS_F32 nor CAVS_BF16", who, type);
  CAVS_REQUIRE(count >= 0 && (count == 0 || d) && o, "%s: bad count %d or null pointer", who, count);
  CAVS_REQUIRE(o->steps >= 1 && o->steps <= 64, "%s: %d steps (1 to 64)", who, o->steps);
  CAVS_REQUIRE(o->eps >= 0.f, "%s: eps is negative or not a number", who);
  for (int i = 0; i < count; i++) {
    const cavs_ortho_desc &e = d[i];
    CAVS_REQUIRE(e.rows > 0 && e.cols > 0 && e.rows <= kMostSide && e.cols <= kMostSide, "%s: matrix %d: unsupported shape %d x %d (1 to 2^16)", who, i,
                 e.rows, e.cols);
    CAVS_REQUIRE(e.G, "%s: matrix %d: null pointer", who, i);
    CAVS_REQUIRE(e.O || e.W, "%s: matrix %d: neither O nor W is wanted", who, i);
    CAVS_REQUIRE(e.ldg >= e.cols && (!e.M || e.ldm >= e.cols) && (!e.W || e.ldw >= e.cols) && (!e.O || e.ldo >= e.cols),
                 "%s: matrix %d: a row stride is below its %d columns", who, i, e.cols);
  }
  if (count == 0) return CAVS_OK;
  const bool two = two_parts(type, count, d, *o);
  Plan p = plan_of<3>(d, count);
  const size_t need = p.bytes;
  if (two) p = plan_of<2>(d, count);
  CAVS_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes needed, %zu given", who, need, workspace_bytes);
  CAVS_REQUIRE(aligned16(workspace), "%s: the workspace must be 16-byte aligned", who);
  char *ws = static_cast<char *>(workspace);
  hipStream_t st = as_stream(stream);
  if (type == CAVS_F32) return run<3, float>(d, count, *o, in_out, p, ws, st);
  return two ? run<2, u16>(d, count, *o, in_out, p, ws, st) : run<3, u16>(d, count, *o, in_out, p, ws, st);
}

}  // namespace
}  // namespace cavs

using namespace cavs;

extern "C" {

size_t cavs_ortho_update_workspace(int type, int count, const cavs_ortho_desc *d) {
  if (count <= 0 || !sizes_ok(type, count, d)) return 0;
  return plan_of<3>(d, count).bytes;  // (two parts take less, whatever the options)
}

int cavs_ortho_update(int type, int count, const cavs_ortho_desc *d, const cavs_ortho_options *o, void *workspace, size_t workspace_bytes, void *stream) {
  return check_and_run("cavs_ortho_update", type, count, d, o, false, workspace, workspace_bytes, stream);
}

int cavs_ortho_update_in_out(int type, int count, const cavs_ortho_desc *d, const cavs_ortho_options *o, void *workspace, size_t workspace_bytes, void *stream) {
  return check_and_run("cavs_ortho_update_in_out", type, count, d, o, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
