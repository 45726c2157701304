// Softmax cross entropy of X W^T + b over a large vocabulary, and its gradients, without logits in memory.
//
//   z = X W^T + b,  lse_r = log sum_c exp z_rc,  loss_r = lse_r - z_r,label,  d_rc = w_r (exp(z_rc - lse_r) - [c = label_r])
//   dX = d W,  dW = d^T X,  db = sums of d's columns
//
// The vocabulary goes by in pieces.  The first pass over them makes each tile of z in registers and leaves a maximum and a sum of
// exponentials per row and tile; what they come to together is lse.  The second makes the tile again, d from it, and leaves d of a piece (of all classes
// where that is 512 MB or less), packed by token, which d X and d W are made of before the next piece overwrites it.  (d^T is read from the same bytes: packed in
// both orders, half as many classes to a piece, fp32 10000 x 512 with 7088 tokens took 1869 us, and takes 1520.)
// Statistics, sums and accumulators are fp32; d is rounded to bf16 where the gradients are (half a unit of 2^-8, as their own
// rounding), and is three bf16 parts, all of an fp32's bits, where they are fp32.
#include <type_traits>

#include "nt_product.h"
#include "wave_reduce.h"

namespace cavs {
namespace {

// ------------------------------------------------------------------ operands, packed
// src [rows, K] with its columns as k and, for a product that sums over them, with its rows as k; either may be left out.  What takes no part is zero
// where it is summed over, as 0 times what it holds need not be 0: a row whose bias is -inf (its z is -inf whatever is there), and in X's second order a row
// that sends nothing back.
// `weight`: up to 64 bf16 rows come times their weights as two parts, the second behind the first along k (see dlogits_kernel).
__device__ inline bool is_class(float label, int classes) { return label >= 0.f && label < (float)classes; }
// A label that names a masked class: the loss is infinite and, as it is of a row whose classes are all masked, sends nothing back.  (Without its -1 in d the
// rest would be no loss's gradient; with it d X would need a row of W that may hold anything.)
__device__ inline bool is_open_class(float label, const float *bias, int classes) {
  return is_class(label, classes) && !(bias && bias[(int)label] == -INFINITY);
}

struct PackJob {
  const void *src;
  long ld;
  int rows, K;
  PackedOut o, t;
  int orows;                      // rows of o, zero beyond those of src
  const float *bias;              // of rows, or null
  const float *labels, *weight;   // of rows, for t, or null
  const float *class_bias;        // of the classes, or null
  int classes;
  int across, blocks;             // blocks of 64 columns, of 64 x 64
};

template <int P, class Src>
__global__ __launch_bounds__(256) void pack_kernel(PackJob j0, PackJob j1) {
  __shared__ PackTile tile;
  const int at = blockIdx.y * gridDim.x + blockIdx.x;
  if (at >= j0.blocks + j1.blocks) return;
  const bool second = at >= j0.blocks;
  const PackJob &g = second ? j1 : j0;
  const int block = second ? at - j0.blocks : at;
  const int r0 = block / g.across * 64, k0 = block % g.across * 64, k = threadIdx.x & 63;
  const Src *src = static_cast<const Src *>(g.src);
  __shared__ bool open[64];  // (looked up beside the tile's loads: a label, and its class's bias)
  __shared__ float weight[64];
  if (g.labels && threadIdx.x < 64) {
    const int r = r0 + threadIdx.x;
    open[threadIdx.x] = r < g.rows && is_open_class(g.labels[r], g.class_bias, g.classes);
    weight[threadIdx.x] = g.weight && r < g.rows ? g.weight[r] : 1.f;
  }
  load_tile(tile, src, g.ld, r0, k0, g.rows, g.K);
  __syncthreads();
  if (g.bias) {
    for (int i = threadIdx.x >> 6; i < 64; i += 4)
      if (r0 + i < g.rows && g.bias[r0 + i] == -INFINITY) tile[i][k] = 0.f;
    __syncthreads();
  }
  pack_tile<P>(tile, g.o, PackedOut{}, r0, k0, g.orows, g.K);
  if (!g.t.p) return;
  if (g.labels) {
    __syncthreads();
    for (int i = threadIdx.x >> 6; i < 64; i += 4) {
      if (!open[i]) tile[i][k] = 0.f;
      else if (g.weight) tile[i][k] *= weight[i];
    }
    __syncthreads();
  }
  pack_tile<P>(tile, PackedOut{}, g.t, r0, k0, g.rows, g.K);
  if constexpr (P == 1) {
    if (!g.weight) return;
    __syncthreads();
    for (int i = threadIdx.x >> 6; i < 64; i += 4) {
      const float rest = tile[i][k] - bf16_float(bf16_bits(tile[i][k]));
      tile[i][k] = fabsf(rest) < INFINITY ? rest : 0.f;
    }
    __syncthreads();
    pack_tile<P>(tile, PackedOut{}, g.t, r0 + 64, k0, g.rows, g.K);
  }
}

// ------------------------------------------------------------------ the tile of z
// 32 values of a row as they lie in memory, as pieces of eight k for the matrix instruction
template <class Src>
struct RawRow;
template <>
struct RawRow<u16> {
  typedef unsigned four __attribute__((ext_vector_type(4), aligned(2)));
  four v[4];
  __device__ inline void load(const u16 *p) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = *reinterpret_cast<const four *>(p + 8 * i);
  }
  __device__ inline void load(const u16 *p, int left) {  // 32 values of which `left` are there
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (8 * i + 8 <= left) v[i] = *reinterpret_cast<const four *>(p + 8 * i);
      else
#pragma unroll
        for (int e = 0; e < 4; e++)
          v[i][e] = (8 * i + 2 * e < left ? p[8 * i + 2 * e] : 0u) | (8 * i + 2 * e + 1 < left ? (unsigned)p[8 * i + 2 * e + 1] << 16 : 0u);
    }
  }
  template <int P>
  __device__ inline void pieces(int s, bf16x8 (&o)[P]) const { o[0] = __builtin_bit_cast(bf16x8, v[s]); }
};
template <>
struct RawRow<float> {
  typedef float four __attribute__((ext_vector_type(4), aligned(4)));
  four v[8];
  __device__ inline void load(const float *p) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = *reinterpret_cast<const four *>(p + 4 * i);
  }
  __device__ inline void load(const float *p, int left) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (4 * i + 4 <= left) v[i] = *reinterpret_cast<const four *>(p + 4 * i);
      else
#pragma unroll
        for (int e = 0; e < 4; e++) v[i][e] = 4 * i + e < left ? p[4 * i + e] : 0.f;
    }
  }
  template <int P>
  __device__ inline void pieces(int s, bf16x8 (&o)[P]) const {
    unsigned short part[8][P];
#pragma unroll
    for (int e = 0; e < 8; e++) parts_of<P>(v[2 * s + e / 4][e % 4], part[e]);
#pragma unroll
    for (int p = 0; p < P; p++)
      o[p] = __builtin_bit_cast(bf16x8, make_uint4(part[0][p] | (unsigned)part[1][p] << 16, part[2][p] | (unsigned)part[3][p] << 16,
                                                   part[4][p] | (unsigned)part[5][p] << 16, part[6][p] | (unsigned)part[7][p] << 16));
  }
};

// A tile whose rows of W are read where they lie: four wavefronts of 32 classes each, 32 TN tokens.  For losses alone, of tokens so few that packing W, which
// writes and reads half as much again (bf16) or three times as much (fp32), would be most of the work.
template <int P_, int TN_>
struct RawTile {
  static constexpr bool RAW = true;
  static constexpr int P = P_, BM = 128, BN = 32 * TN_, WGM = 4, WGN = 1, WAVES = 4, THREADS = 256, WM = 32, WN = BN, TM = 1, TN = TN_;
  static constexpr int ACC = P > 1 ? 2 : 1, EU = 2, STAGE = TN * 4 * P * 1024, LDS = 2 * STAGE > 16384 ? 2 * STAGE : 16384;
};
// acc = the tile's product: 64 k at a time, a lane's 32 k of its class on their way from memory while those before are multiplied; X packed, by way of
// LDS, two stages.  A lane's k are 32 in a row (see RawRow's users below): its pieces of X are those of its k.
template <class T, class Src>
__device__ __forceinline__ void raw_multiply(const Src *W, long ldw, int M, int m0, const PackedRef &X, int n, int n0, int H, char *S,
                                             floatx16 (&acc)[T::ACC][T::TM][T::TN]) {
  constexpr int P = T::P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x = lane & 31, half = lane >> 5;
#pragma unroll
  for (int s = 0; s < T::ACC; s++)
#pragma unroll
    for (int j = 0; j < T::TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[s][0][j][r] = 0.f;
  const Src *row = W + min(m0 + 32 * wave + x, M - 1) * ldw + 32 * half;
  const int chunks = (H + 63) / 64;
  auto fetch_w = [&](RawRow<Src> &r, int chunk) {
    if (64 * chunk + 64 <= H) r.load(row + 64 * chunk);
    else r.load(row + 64 * chunk, H - 64 * chunk - 32 * half);
  };
  // this wavefront's blocks of a stage: every fourth of TN x 4 x P
  auto fetch_x = [&](int chunk, char *to) {
#ifdef __HIP_DEVICE_COMPILE__
    const auto rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<u16 *>(X.p), 0, 0xffffffffu, 0x00020000);
#pragma unroll
    for (int c = 0; c < T::TN * P; c++) {
      const int at = 4 * c + wave, j = at / (4 * P);
      const unsigned off = (unsigned)(min(n0 / 32 + j, (n - 1) / 32) * (X.K / 16) + 4 * chunk) * (P * 1024) + at % (4 * P) * 1024;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (__attribute__((address_space(3))) void *)(to + at * 1024), 16, 16 * lane, off, 0, 0);
    }
#endif
  };
  RawRow<Src> now, next;
  fetch_x(0, S);
  fetch_w(now, 0);
  int at = 0;
  for (int chunk = 0; chunk < chunks; chunk++) {
    nt_arrive<0>();
    if (chunk + 1 < chunks) {
      fetch_x(chunk + 1, S + (T::STAGE - at));
      fetch_w(next, chunk + 1);
    }
#pragma unroll
    for (int s = 0; s < 4; s++) {
      bf16x8 w[P], t[T::TN][P];
#pragma unroll
      for (int j = 0; j < T::TN; j++)
#pragma unroll
        for (int p = 0; p < P; p++)
          t[j][p] = *reinterpret_cast<const bf16x8 *>(S + at + ((j * 4 + 2 * half + (s >> 1)) * P + p) * 1024 + (x + 32 * (s & 1)) * 16);
      now.template pieces<P>(s, w);
#pragma unroll
      for (int q = P - 1; q >= 0; q--)
#pragma unroll
        for (int p = 0; p <= q; p++)
#pragma unroll
          for (int j = 0; j < T::TN; j++)
            acc[q ? T::ACC - 1 : 0][0][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[p], t[j][q - p], acc[q ? T::ACC - 1 : 0][0][j], 0, 0, 0);
    }
    now = next;
    at = T::STAGE - at;
  }
  nt_arrive<0>();
}

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
  const void *raw;     // the piece's rows of W as they lie, and H
  long ldw;
  int H;
};
// acc and the tile's place
template <class T>
__device__ __forceinline__ void product_of_tile(const TileArgs &a, char *S, floatx16 (&acc)[T::ACC][T::TM][T::TN], int *m0, int *n0, int *tn) {
  int tm;
  if constexpr (T::RAW) {
    using Src = std::conditional_t<T::P == 1, u16, float>;
    const int t = xcd_remap(blockIdx.x, a.tilesM * a.tilesN);
    tm = t / a.tilesN, *tn = t - tm * a.tilesN;  // (tiles of the same classes together: W comes from memory once)
    *m0 = tm * T::BM, *n0 = *tn * T::BN;
    raw_multiply<T, Src>(static_cast<const Src *>(a.raw), a.ldw, a.M, *m0, a.X, a.n, *n0, a.H, S, acc);
  } else {
    nt_tile_of(blockIdx.x, a.tilesM, a.tilesN, &tm, tn);
    *m0 = tm * T::BM, *n0 = *tn * T::BN;
    nt_multiply<T>(a.W, a.M, *m0, a.X, a.n, *n0, 0, a.K, S, acc);
  }
}

template <class T>
__global__ __launch_bounds__(T::THREADS, T::EU) void stats_kernel(TileArgs a, float2 *__restrict__ stats, float *__restrict__ zlabel) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS];
  int m0, n0, tn;
  floatx16 acc[T::ACC][T::TM][T::TN];
  product_of_tile<T>(a, S, acc, &m0, &n0, &tn);
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
    stats[(long)((a.c0 + m0) / T::BM) * a.n + n0 + x] = s;
  }
}

__device__ inline float2 joined(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x), from = top == -INFINITY ? 0.f : top;
  return make_float2(top, a.y * __expf(a.x - from) + b.y * __expf(b.x - from));
}
// ------------------------------------------------------------------ few tokens
// Up to 64 tokens: W read where it lies, once; what bounds it is memory.  A workgroup has 32 classes at a time, each of its
// four wavefronts a quarter of k: 64 lanes with 64 or 128 bytes each under way are what a CU needs to keep memory busy, and a few thousand
// classes give every CU such wavefronts.  A lane reads 32 k of one row in one go, 64 at a time for its row (a line of memory is used up by one or two
// lanes one after the other); the instruction does not mind which k it adds up as long as both operands agree.  The four sums of a product
// meet in LDS.  Up to 32 tokens X is read as W is, and the launch that would pack it is saved; two blocks of 32 come packed, the lane's pieces
// those of its k (64 tokens, bf16 50000 x 2048: 70 us, as they lie 86).
// us of a call, this / packed and in tiles (n = 1, 32, 64 / any up to 64):  bf16 32000 x 1024 16, 22, 31 / 55, 50000 x 2048 38 (5.4 TB/s), 56, 70 / 225;
// fp32 21701 x 300 19, 22, 28 / 28, 50000 x 2048 114, 131, 169 / 442.  Beyond 64 W has to be read again, or wavefronts get few: bf16 32000 x 1024,
// 96 tokens 55 / 55, 128 61 / 56.
struct DirectArgs {
  const void *W, *X;
  long ldw, ldx;
  PackedRef packed;     // X, where it is packed
  int H, C, n, blocks;  // blocks: of 32 classes
  const float *bias, *labels;
  float2 *stats;  // a row of n for every workgroup
  float *zlabel, *z;  // z: null, or all of it for the gradients, block of 32 classes by block of 32 tokens by wavefront by lane
};
template <int P, class Src, int TN, bool PACKED>
__global__ __launch_bounds__(256, P == 1 ? 4 : 2) void direct_stats_kernel(DirectArgs a) {
  constexpr int ACC = P > 1 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float sums[4][TN * 16][64];
  __shared__ float2 part[4][32 * TN];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x = lane & 31, half = lane >> 5;
  const int chunks = (a.H + 63) / 64, first = chunks * wave / 4, end = chunks * (wave + 1) / 4;
  auto fetch = [&](RawRow<Src> &r, const Src *row, int chunk) {
    const int k = 64 * chunk;
    if (k + 64 <= a.H) r.load(row + k);
    else r.load(row + k, a.H - k - 32 * half);
  };
  const Src *token_row[TN];
  const u16 *pieces[TN];
#pragma unroll
  for (int j = 0; j < TN; j++) {
    token_row[j] = static_cast<const Src *>(a.X) + min(32 * j + x, a.n - 1) * a.ldx + 32 * half;
    pieces[j] = a.packed.p + (long)min(j, (a.n - 1) / 32) * (a.packed.K / 16) * P * 512 + (2 * half * P) * 512 + x * 8;
  }
  float2 all = make_float2(-INFINITY, 0.f);  // of token threadIdx.x
  for (int block = blockIdx.x; block < a.blocks; block += gridDim.x) {
    const Src *row = static_cast<const Src *>(a.W) + (long)min(32 * block + x, a.C - 1) * a.ldw + 32 * half;
    floatx16 acc[ACC][TN];
#pragma unroll
    for (int s = 0; s < ACC; s++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[s][j][r] = 0.f;
    RawRow<Src> now, next, t[TN];
    if (first < end) fetch(now, row, first);
    for (int chunk = first; chunk < end; chunk++) {
      if constexpr (!PACKED)
#pragma unroll
        for (int j = 0; j < TN; j++) fetch(t[j], token_row[j], chunk);
      if (chunk + 1 < end) fetch(next, row, chunk + 1);
#pragma unroll
      for (int s = 0; s < 4; s++) {
        bf16x8 w[P], u[TN][P];
#pragma unroll
        for (int j = 0; j < TN; j++) {
          if constexpr (PACKED) {
#pragma unroll
            for (int p = 0; p < P; p++) u[j][p] = *reinterpret_cast<const bf16x8 *>(pieces[j] + ((4 * chunk + (s >> 1)) * P + p) * 512 + 256 * (s & 1));
          } else {
            t[j].template pieces<P>(s, u[j]);
          }
        }
        now.template pieces<P>(s, w);
#pragma unroll
        for (int q = P - 1; q >= 0; q--)
#pragma unroll
          for (int p = 0; p <= q; p++)
#pragma unroll
            for (int j = 0; j < TN; j++) acc[q ? ACC - 1 : 0][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[p], u[j][q - p], acc[q ? ACC - 1 : 0][j], 0, 0, 0);
      }
      now = next;
    }
    if constexpr (ACC > 1)
#pragma unroll
      for (int j = 0; j < TN; j++) acc[0][j] += acc[1][j];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) sums[wave][16 * j + r][lane] = acc[0][j][r];
    __syncthreads();
    // this wavefront's rows of the block: 8 wave + 4 half + 0 .. 3
    const int c = 32 * block + 8 * wave + 4 * half;
    float b[4];
#pragma unroll
    for (int k = 0; k < 4; k++) b[k] = c + k >= a.C ? -INFINITY : a.bias ? a.bias[c + k] : 0.f;
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int token = 32 * j + x;
      const float label = token < a.n ? a.labels[token] : -1.f;
      float z[4], top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int r = 16 * j + 4 * wave + k;
        z[k] = (sums[0][r][lane] + sums[1][r][lane]) + (sums[2][r][lane] + sums[3][r][lane]);
        z[k] = b[k] == -INFINITY ? -INFINITY : z[k] + b[k];
        top = fmaxf(top, z[k]);
        if (is_class(label, a.C) && (int)label == c + k) a.zlabel[token] = z[k];
      }
      if (a.z) *reinterpret_cast<float4 *>(a.z + (((long)block * TN + j) * 4 + wave) * 256 + 4 * lane) = make_float4(z[0], z[1], z[2], z[3]);
      top = fmaxf(top, __shfl_xor(top, 32));
      const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int k = 0; k < 4; k++) sum += __expf(z[k] - from);
      sum += __shfl_xor(sum, 32);
      if (half == 0) part[wave][32 * j + x] = make_float2(top, sum);
    }
    __syncthreads();
    if (threadIdx.x < 32 * TN) all = joined(all, joined(joined(part[0][threadIdx.x], part[1][threadIdx.x]), joined(part[2][threadIdx.x], part[3][threadIdx.x])));
  }
  if (threadIdx.x < 32 * TN && (int)threadIdx.x < a.n) a.stats[(long)blockIdx.x * a.n + threadIdx.x] = all;
}

// What a row's tiles come to: lse, loss and the weight of its gradient (zero for a row without a class, or whose class is
// masked).  Sixteen lanes to a row, or all of a workgroup where rows are few.
struct RowArgs {
  const float2 *stats;
  int tiles, n, C;
  const float *zlabel, *labels, *bias, *dloss;
  float *loss, *lse, *weight;
};
__device__ inline float weight_of(bool open, float lse, const float *dloss, int row) {
  return open && lse != -INFINITY ? dloss ? dloss[row] : 1.f : 0.f;
}
template <int ROWS>
__global__ __launch_bounds__(256) void rows_kernel(RowArgs a) {
  constexpr int LANES = 256 / ROWS;
  __shared__ float2 part[LANES][ROWS];
  const int x = threadIdx.x % ROWS, y = threadIdx.x / ROWS, row = blockIdx.x * ROWS + x;
  float2 s = make_float2(-INFINITY, 0.f);
  const float label = y == 0 && row < a.n ? a.labels[row] : -1.f;
  const bool open = is_open_class(label, a.bias, a.C);  // (two loads one after the other, on their way beside the statistics)
  if (row < a.n)
    for (int t = y; t < a.tiles; t += 4 * LANES) {
      float2 v[4];
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = t + k * LANES < a.tiles ? a.stats[(long)(t + k * LANES) * a.n + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < 4; k++) s = joined(s, v[k]);
    }
  part[y][x] = s;
  for (int half = LANES / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (y < half) part[y][x] = joined(part[y][x], part[y + half][x]);
  }
  if (y != 0 || row >= a.n) return;
  s = part[0][x];
  const float all = (s.x == -INFINITY ? 0.f : s.x) + logf(s.y);
  if (a.lse) a.lse[row] = all;
  // (no class left: an infinite loss, not the NaN of -inf - -inf)
  if (a.loss) a.loss[row] = !is_class(label, a.C) ? 0.f : all == -INFINITY || !open ? INFINITY : all - a.zlabel[row];
  if (a.weight) a.weight[row] = weight_of(open, all, a.dloss, row);
}

__global__ __launch_bounds__(256) void weights_kernel(const float *__restrict__ labels, const float *__restrict__ lse, const float *__restrict__ bias,
                                                      const float *__restrict__ dloss, int n, int C, float *__restrict__ weight) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row < n) weight[row] = weight_of(is_open_class(labels[row], bias, C), lse[row], dloss, row);
}

// d = weight * (p - [label]) of a tile, packed by token (zero between the last class or token and the end of the steps), and its sums over the tile's
// tokens.  `scale`, which multiplies all of d, stays out of what is rounded: next to the label, where p is small, p - 1 is -1 and a bit, which bf16 holds
// well, while a factor in it is a rounding error that all of its kind share.  So is a token's weight for that token: of up to 64 bf16 ones (`beside`) it stays
// out as well.  d W has it as a factor of its rows then, and d^T X with X, in two parts, for which d is there twice (64 tokens, 25040 x 1000: 123 us a call
// without weights, 128 with them); of thousands of tokens that would be a quarter more operations and twice the d.  Errors of dX and dW, 25040 x 1000:
// 64 tokens 0.0019 of their norm, 65 0.0024, 2371 0.0024 and 0.0023; rounding the gradients alone 0.0017.
template <class T>
__global__ __launch_bounds__(T::THREADS, T::EU) void dlogits_kernel(TileArgs a, const float *__restrict__ lse, const float *__restrict__ weight, PackedOut d,
                                                                    float *__restrict__ sums, int ld_sums, float sums_scale, int beside) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS];
  int m0, n0, tn;
  floatx16 acc[T::ACC][T::TM][T::TN];
  product_of_tile<T>(a, S, acc, &m0, &n0, &tn);
  float *lb = reinterpret_cast<float *>(S);
  float *part = lb + T::BM;  // [WGN][BM]
  const Where<T> w;
  static_assert(4 * T::BM * (1 + T::WGN) <= T::LDS, "");
  const int tokens = (a.n + kPlaneAlign - 1) / kPlaneAlign * kPlaneAlign;
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
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const float v = g[j] * x[r];
        sum[r] += v;
        if (T::P > 1 || !beside) x[r] = v;
      }
      if (d.p && 32 * xb < tokens && 32 * cb < d.K) {
        Parts16<T::P> e;
#pragma unroll
        for (int r = 0; r < 16; r++) parts_of<T::P>(x[r], e.v[r]);
        put_rows<T::P>(d, xb, cb, e, w.lane);
        if (T::P == 1 && beside) put_rows<T::P>(d, xb + 2, cb, e, w.lane);
        asm volatile("" ::: "memory");  // (one block after the other: a lane has no registers for two)
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
    sums[(long)tn * ld_sums + m0 + x] = sums_scale * s;
  }
}

// ------------------------------------------------------------------ the gradients of few tokens
// d of up to 64 tokens from the z that direct_stats_kernel left (a float a token and class, beside W's row of H), packed as dlogits_kernel packs it,
// and its sums over the tokens.  A wavefront has a block of 32 classes.
struct FewLogitsArgs {
  const float *z;
  const float *lse, *weight, *labels;
  int n, C, c0;
  PackedOut d;  // null: not wanted; of the piece that begins with class c0
  int blocks;   // of 32 classes
  float *sums;  // of the piece, or null
  float scale;  // of the sums
  int beside;   // as dlogits_kernel's
};
template <int P>
__global__ __launch_bounds__(256) void few_dlogits_kernel(FewLogitsArgs a) {
  const int lane = threadIdx.x & 63, x = lane & 31, half = lane >> 5, cb = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (cb >= a.blocks) return;
  const int c = a.c0 + 32 * cb, TN = (a.n + 31) / 32;
  float sum[16] = {};
#pragma unroll
  for (int j = 0; j < kPlaneAlign / 32; j++) {
    const int token = 32 * j + x;
    float e[16] = {};
    if (j < TN && c < a.C) {
      const bool in = token < a.n;
      const float g = in ? a.weight[token] : 0.f, all = in ? a.lse[token] : 0.f, label = in ? a.labels[token] : -1.f;
      const int at = is_class(label, a.C) ? (int)label - c - 4 * half : -1;
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const float4 z = *reinterpret_cast<const float4 *>(a.z + (((long)(c / 32) * TN + j) * 4 + q) * 256 + 4 * lane);
        const float v[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float x = g == 0.f ? 0.f : __expf(v[k] - all) - (at == 8 * q + k ? 1.f : 0.f), gx = g * x;
          sum[4 * q + k] += gx;
          e[4 * q + k] = P == 1 && a.beside ? x : gx;
        }
      }
    }
    if (a.d.p) {
      Parts16<P> o;
#pragma unroll
      for (int r = 0; r < 16; r++) parts_of<P>(e[r], o.v[r]);
      put_rows<P>(a.d, j, cb, o, lane);
      if (P == 1 && a.beside) put_rows<P>(a.d, j + 2, cb, o, lane);
    }
  }
  if (!a.sums) return;
#pragma unroll
  for (int r = 0; r < 16; r++) {
    float v = sum[r];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor(v, o);
    const int row = 8 * (r >> 2) + 4 * half + (r & 3);
    if (x == 0 && c + row < a.C) a.sums[32 * cb + row] = a.scale * v;
  }
}

// Sums over classes of d times W, W's rows read where they lie, once: what bounds it is memory.  A lane has F neighbouring columns of eight classes
// of a step, a load of 4 F or 2 F bytes each; the instruction takes its eight classes of one column at a time, so those are F operands, of
// columns F apart, by renaming registers.  A workgroup has 32 F columns, up to 32 TN tokens and a stretch of the classes, of which each wavefront takes
// every fourth step of sixteen; what they sum up meets in LDS and goes to part [stretch, n, H].  Rows of classes that are masked are zero.
// (F as large as accumulators leave room for: with loads of 4 bytes a wavefront has 2 KB under way, too little.  bf16 81664 x 4096, 12 tokens: W's 669 MB in
// 119 us, 5.6 TB/s; with stretches for one and a half rounds of workgroups 212.)
struct FewArgs {
  const void *W;
  long ldw;
  PackedRef d;  // by token; its k the piece's classes
  int M, n, H;  // classes of the piece
  const float *bias;
  int across, chunk;  // blocks of 32 F columns, classes of a stretch (a multiple of 64)
  float *part;
  int add;
};
template <int P, int TN>
constexpr int few_columns() { return (P == 1 ? 8 : 4) / TN; }
template <int P, class Src, int TN>
__global__ __launch_bounds__(256, 2) void few_dx_kernel(FewArgs a) {
  constexpr int ACC = P > 1 ? 2 : 1, F = few_columns<P, TN>();
  __shared__ __attribute__((aligned(16))) float sums[4][32][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x = lane & 31, half = lane >> 5;
  const int h0 = 32 * F * (blockIdx.x % a.across), stretch = blockIdx.x / a.across;
  const int kend = min(a.d.K, (stretch + 1) * a.chunk);
  const u16 *dp[TN];
#pragma unroll
  for (int j = 0; j < TN; j++) dp[j] = a.d.p + (long)min(j, (a.n - 1) / 32) * (a.d.K / 16) * P * 512 + lane * 8;
  floatx16 acc[ACC][TN][F];
#pragma unroll
  for (int s = 0; s < ACC; s++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int f = 0; f < F; f++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[s][j][f][r] = 0.f;
  // F columns from h0 + F x on, of eight classes.  Towards the end of a row the last F there are, moved down once they have come: what a lane holds beyond the
  // last column goes nowhere.  (Value by value there, few workgroups kept all the others waiting: fp32 40806 x 4052, 12 tokens 338 us, 218 now.)
  const bool edge = h0 + 32 * F > a.H, wide = a.H >= F;
  const int h = h0 + F * x, from = edge ? min(h, a.H - F) : h, beyond = h - from;
  constexpr int WORDS = F * sizeof(Src) / 4;
  typedef unsigned words __attribute__((ext_vector_type(WORDS == 1 ? 2 : WORDS), aligned(sizeof(Src))));
  struct Eight {
    unsigned v[8][WORDS];
    bf16x8 d[TN][P];
    float b[8];
  };
  auto fetch = [&](Eight &o, int k0) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int c = min(k0 + 8 * half + e, a.M - 1);
      const Src *row = static_cast<const Src *>(a.W) + c * a.ldw;
      o.b[e] = a.bias ? a.bias[c] : 0.f;
      if (wide) {
        static_assert(WORDS > 1, "a lane's columns are eight bytes or more");
        const words v = *reinterpret_cast<const words *>(row + from);
#pragma unroll
        for (int i = 0; i < WORDS; i++) o.v[e][i] = v[i];
      } else {
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
          if constexpr (sizeof(Src) == 4) {
            o.v[e][i] = h + i < a.H ? __float_as_uint(value_of(row + h + i)) : 0u;
          } else {
            const unsigned lo = h + 2 * i < a.H ? row[h + 2 * i] : 0u, hi = h + 2 * i + 1 < a.H ? row[h + 2 * i + 1] : 0u;
            o.v[e][i] = lo | hi << 16;
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int p = 0; p < P; p++) o.d[j][p] = *reinterpret_cast<const bf16x8 *>(dp[j] + ((long)(k0 / 16) * P + p) * 512);
  };
  auto mask = [&](Eight &o, int k0) {
    if (edge && wide)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        unsigned(&v)[WORDS] = o.v[e];
        if constexpr (sizeof(Src) == 2) {
          if (beyond & 1)
#pragma unroll
            for (int i = 0; i < WORDS; i++) v[i] = v[i] >> 16 | (i + 1 < WORDS ? v[i + 1] << 16 : 0u);
        }
        const int words_beyond = sizeof(Src) == 2 ? beyond >> 1 : beyond;
#pragma unroll
        for (int by = 1; by < WORDS; by *= 2)
          if (words_beyond & by)
#pragma unroll
            for (int i = 0; i + by < WORDS; i++) v[i] = v[i + by];
      }
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (k0 + 8 * half + e >= a.M || o.b[e] == -INFINITY)
#pragma unroll
        for (int i = 0; i < WORDS; i++) o.v[e][i] = 0;
  };
  Eight now, next;
  int k = stretch * a.chunk + 16 * wave;
  if (k < kend) fetch(now, k);
  for (; k < kend; k += 64) {
    if (k + 64 < kend) fetch(next, k + 64);
    mask(now, k);
#pragma unroll
    for (int f = 0; f < F; f++) {
      bf16x8 w[P];
      if constexpr (sizeof(Src) == 4) {
        u16 part[8][P];
#pragma unroll
        for (int e = 0; e < 8; e++) parts_of<P>(__uint_as_float(now.v[e][f]), part[e]);
#pragma unroll
        for (int p = 0; p < P; p++)
          w[p] = __builtin_bit_cast(bf16x8, make_uint4(part[0][p] | (unsigned)part[1][p] << 16, part[2][p] | (unsigned)part[3][p] << 16,
                                                       part[4][p] | (unsigned)part[5][p] << 16, part[6][p] | (unsigned)part[7][p] << 16));
      } else {
        unsigned u[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const unsigned lo = now.v[2 * e][f / 2], hi = now.v[2 * e + 1][f / 2];
          u[e] = f % 2 ? lo >> 16 | (hi & 0xffff0000u) : (lo & 0xffffu) | hi << 16;
        }
        w[0] = __builtin_bit_cast(bf16x8, make_uint4(u[0], u[1], u[2], u[3]));
      }
#pragma unroll
      for (int q = P - 1; q >= 0; q--)
#pragma unroll
        for (int p = 0; p <= q; p++)
#pragma unroll
          for (int j = 0; j < TN; j++)
            acc[q ? ACC - 1 : 0][j][f] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(now.d[j][p], w[q - p], acc[q ? ACC - 1 : 0][j][f], 0, 0, 0);
    }
    now = next;
  }
  float *part = a.part + (long)stretch * a.n * a.H;
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int f0 = 0; f0 < F; f0 += 2) {
      __syncthreads();
#pragma unroll
      for (int f = 0; f < 2; f++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          float v = acc[0][j][f0 + f][r];
          if constexpr (ACC > 1) v += acc[1][j][f0 + f][r];
          sums[wave][16 * f + r][lane] = v;
        }
      __syncthreads();
      // this wavefront's rows of the block: 8 wave + 4 half + 0 .. 3
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int token = 32 * j + 8 * wave + 4 * half + i;
        if (token >= a.n) continue;
#pragma unroll
        for (int f = 0; f < 2; f++) {
          const int r = 16 * f + 4 * wave + i, h = h0 + F * x + f0 + f;
          if (h >= a.H) continue;
          float v = (sums[0][r][lane] + sums[1][r][lane]) + (sums[2][r][lane] + sums[3][r][lane]);
          float *o = part + (long)token * a.H + h;
          *o = a.add ? *o + v : v;
        }
      }
    }
}

// ------------------------------------------------------------------ the products with d
// out[row, col] = scale * factor[row] * A B^T.  K in `splits` stretches of kchunk, each with sums of its own (unscaled) at part + split * M * N; part null:
// straight to out.  A launch is d W, d's rows the tile's rows, and d^T X, d's classes the tile's rows and its tokens what is summed over.
template <class Out>
struct ProductJob {
  PackedRef A, B;
  int M, N, K, tilesM, tilesN, splits, kchunk;
  float *part;
  int add;  // what is there already is added to (`part`)
  Out *out;
  long ldo;
  float scale;
  const float *factor;  // of out's rows, or null
};

// STREAM: `out` goes past the caches.  TB: W by class.
template <class T, class Out, bool STREAM, bool TB>
__global__ __launch_bounds__(T::THREADS, T::EU) void product_kernel(ProductJob<Out> j0, ProductJob<Out> j1, int blocks0) {
  __shared__ __attribute__((aligned(16))) char S[T::LDS];
  const bool second = (int)blockIdx.x >= blocks0;
  const ProductJob<Out> &g = second ? j1 : j0;
  int block = second ? blockIdx.x - blocks0 : blockIdx.x, tm, tn;
  const int tiles = g.tilesM * g.tilesN, split = block / tiles;
  nt_tile_of(block - split * tiles, g.tilesM, g.tilesN, &tm, &tn);
  const int m0 = tm * T::BM, n0 = tn * T::BN, kbeg = split * g.kchunk, kend = min(g.K, kbeg + g.kchunk);
  floatx16 acc[T::ACC][T::TM][T::TN];
  if (second) nt_multiply<T, true>(g.A, g.M, m0, g.B, g.N, n0, kbeg, kend, S, acc);
  else nt_multiply<T, false, TB>(g.A, g.M, m0, g.B, g.N, n0, kbeg, kend, S, acc);
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
        } else if constexpr (STREAM) {
          stream_as(g.out + row * g.ldo + col, (g.factor ? g.scale * g.factor[row] : g.scale) * x);
        } else {
          store_as(g.out + row * g.ldo + col, (g.factor ? g.scale * g.factor[row] : g.scale) * x);
        }
      }
  }
}

// out[r, 0 .. w) = scale * factor[r] * sum of `parts` pieces, in their order
struct SumJob {
  const float *part;
  int parts, rows, w;
  const float *factor;
  void *out;
  long ldo;
  int blocks;
};
template <class Out>
__device__ inline void sum_parts(const SumJob &g, float scale, int block) {
  const long total = (long)g.rows * g.w;
  Out *out = static_cast<Out *>(g.out);
  for (long i = (long)block * 256 + threadIdx.x; i < total; i += (long)g.blocks * 256) {
    float s = 0.f;
    for (int p = 0; p < g.parts; p += 8) {  // (eight loads on their way at a time)
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = p + k < g.parts ? g.part[(p + k) * total + i] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; k++) s += v[k];
    }
    const long r = i / g.w;
    store_as(out + r * g.ldo + (i - r * g.w), (g.factor ? scale * g.factor[r] : scale) * s);
  }
}
// d X, d W and d b (fp32) of what the launches before left in parts
template <class Out>
__global__ __launch_bounds__(256) void sums_kernel(SumJob x, SumJob w, SumJob b, float scale) {
  int block = blockIdx.x;
  if (block < x.blocks) return sum_parts<Out>(x, scale, block);
  block -= x.blocks;
  if (block < w.blocks) return sum_parts<Out>(w, scale, block);
  sum_parts<float>(b, scale, block - w.blocks);
}

// ------------------------------------------------------------------ what a call consists of
template <int P> struct Tiles;
template <> struct Tiles<1> {
  using L = NtTile<1, 256, 128, 32, 2, 2>;
  using M = NtTile<1, 128, 128, 32, 2, 2>;
  using S = NtTile<1, 64, 64, 64, 2, 2, 3>;  // (171 x 2216 x 192 43 us of a call, two stages 49)
};
template <> struct Tiles<3> {
  using L = NtTile<3, 128, 128, 16, 2, 2>;
  using M = L;
  using S = NtTile<3, 64, 64, 32, 2, 2>;  // (500 x 512 x 3000 74 us of a call, three stages, which leave a unit two workgroups, 86; 171 x 2216 x 192 95, 91)
};

template <int P, class F>
int with_product_tile(int size, F &&f) {
  using TT = Tiles<P>;
  if (size == 2) return f(typename TT::L{});
  if (size == 1) return f(typename TT::M{});
  return f(typename TT::S{});
}
// sizes 0 .. 2: packed operands, small to large; 3: W as it lies
template <int P, class F>
int with_tile(int size, F &&f) {
  if (size == 3) return f(RawTile<P, P == 1 ? 4 : 2>{});
  return with_product_tile<P>(size, f);
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

constexpr int kPieceBytes = 256 << 20;  // d of a piece, where it is not all of d
// d at once: W is packed once then, and d W goes without sums from piece to piece (bf16 50000 x 2048, 4096 tokens, 410 MB: 3219 us, in two
// pieces 3454; fp32 10000 x 512, 7088 tokens, 427 MB: 1592 us, 1622)
constexpr int kWholeBytes = 512 << 20;
constexpr size_t kKeepBytes = 512 << 20;  // of W packed: kept from the first pass for the second
constexpr int kSplits = 64;
constexpr int kMostBlocks = (1 << 24) - 1;  // workgroups of 256 along one dimension of a grid, whose threads are to be below 2^32
constexpr int kFewRows = 64, kRawRows = 256;

// What the two products of a piece take, us, with their K in so many stretches.  Workgroups go to the compute unit that is free first, those of d W
// before those of d^T X; a unit multiplies at one speed whatever it holds, but for the end, where a long workgroup is left alone.  Each
// costs 256 k more than it multiplies, and what they leave in parts is written and read at the rate of a copy.
struct Stretches {
  int tiles, K, chunk, n;
  void set(int s) { chunk = ceil_to((K + s - 1) / s, kPlaneAlign), n = (K + chunk - 1) / chunk; }
};
inline double products_us(const Stretches &x, const Stretches &w, double us_per_k, double part_bytes) {
  const long cus = num_cus(), nx = (long)x.tiles * x.n, nw = (long)w.tiles * w.n, a = x.chunk + 256, b = w.chunk + 256;
  const long more = nx % cus, low = nx / cus * a, high = low + a;  // `more` units with one of d W's more than the others
  long t = nx > 0 && more == 0 ? low : nx > 0 ? high : 0;
  if (nw > 0) {
    const long mean = (nx * a + nw * b) / cus;
    long i = mean > low ? (mean - low) / b : 0, j = mean > high ? (mean - high) / b : 0;
    for (;;) {  // the first moment by which all of d^T X's have ended
      const long ti = low + i * b, tj = high + j * b, at = ti < tj ? ti : tj;
      if (more * (at > high ? (at - high) / b : 0) + (cus - more) * (at > low ? (at - low) / b : 0) >= nw) {
        t = at > t ? at : t;
        break;
      }
      i += ti == at, j += tj == at;
    }
  }
  const double longest = a > b && nx > 0 ? a : b, alone = longest - (t - longest) / 2;
  return (t + (alone > 0 ? 1.5 * alone : 0.)) * us_per_k + part_bytes / 4.7e6;
}

// Sizes and places of a call's workspace.
struct Plan {
  int P, size, bm, bn, Hp, np, piece, pieces, tiles;  // tiles: of the whole vocabulary
  int few;  // tokens: W read where it lies, z kept for the gradients
  int raw;  // losses of not many tokens: W read where it lies
  int facross;  // few_dx_kernel's
  int one_order;  // W packed by class alone
  int grads, keep, psize, pm, pn, xsplits, xchunk, wsplits, wchunk;
  size_t stats, zlabel, lse, weight, z, x, w, xt, wt, d, sums, xpart, wpart, bytes;
};

template <int P>
Plan plan_of(int n, int H, int C, int grads) {
  Plan p{};
  p.P = P, p.grads = grads;
  p.Hp = ceil_to(H, kPlaneAlign), p.np = ceil_to(n, kPlaneAlign);
  long most = grads ? ((long)C * 2 * P * p.np <= kWholeBytes ? kWholeBytes : kPieceBytes) / (2l * P * p.np) : (128l << 20) / (2l * P * p.Hp);
  most = most < 1024 ? 1024 : most > 1 << 20 ? 1 << 20 : most;
  p.pieces = (int)((C + most - 1) / most);
  p.piece = ceil_to((C + p.pieces - 1) / p.pieces, 256);
  int rows = p.piece < C ? p.piece : C;
  // Few tokens: W read where it lies and z kept, packing W and making z twice would be most of the work.  Gradients take two launches more that way, which
  // long rows or many classes pay for.  us with gradients packed / as it lies, 1, 24 and 64 tokens:
  //   fp32  300 x 1024 53 / 39, 54 / 42, 57 / 47   1000 x 512 41 / 36, 42 / 39, 44 / 43   12000 x 300 58 / 57, 61 / 60, 63 / 66   21701 x 300 79 / 72, 81 / 77,
  //         87 / 82   12000 x 512 70 / 61, 72 / 65, 77 / 71   32000 x 128 79 / 64, 82 / 71, 84 / 77   40806 x 4050 1417 / 679 (12)
  //   bf16  1000 x 512 28 / 30, 30 / 33, 31 / 41   4000 x 1024 49 / 39, 48 / 43, 51 / 55   12000 x 1024 63 / 56, 64 / 64, 66 / 71   32000 x 128 54 / 51, 57 / 59,
  //         59 / 63   81792 x 72 95 / 78, 99 / 85, 100 / 93   124416 x 2176 858 / 475 (64)
  const bool many = C >= 128 * num_cus();
  p.few = n <= kFewRows && (!grads || many || (P == 3 ? H >= 512 || (long)C * H >= 5000000 : H >= 1024 && (n <= 32 || (long)C * H >= 16000000)));
  // Losses of up to 256 tokens under a vocabulary with a tile of 128 classes for every second compute unit.  us packed / as it lies, 96 and 256 tokens:
  //   bf16 124416 x 2176 361 / 283, 423 / 313, 45376 x 1024 53 / 33, 74 / 42, 21701 x 300 20 / 18, 23 / 19, 10000 x 512 20 / 20, 23 / 21; fp32 45376 x 1024
  //   171 / 139, 217 / 181, 21701 x 300 31 / 27, 42 / 40, 1000 x 128 13 / 15
  p.raw = !grads && !p.few && n <= kRawRows && C >= 64 * num_cus();
  p.size = p.raw ? 3 : tile_size<P>(rows, n);
  tile_sides<P>(p.size, &p.bm, &p.bn);
  while ((long)tiles_of(rows, p.bm) * tiles_of(n, p.bn) > kMostBlocks) rows = p.piece = ceil_to(rows / 2, 256);  // (losses alone of a million tokens)
  p.pieces = tiles_of(C, p.piece);
  p.tiles = tiles_of(C, p.bm);
  if (p.few) p.tiles = tiles_of(C, 32) < 4 * num_cus() ? tiles_of(C, 32) : 4 * num_cus();
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
  p.z = take(p.few && grads ? (size_t)tiles_of(C, 32) * tiles_of(n, 32) * 4096 : 0);
  p.x = take(p.few && n <= 32 ? 0 : packed_bytes<P>(n, p.Hp));
  p.w = take(p.few || p.raw ? 0 : packed_bytes<P>(ceil_to(grads && p.keep ? C : rows, kPlaneAlign), p.Hp));
  if (grads) {
    const int rp = ceil_to(rows, kPlaneAlign);
    p.psize = tile_size<P>((long)rows + n, H);
    tile_sides<P>(p.psize, &p.pm, &p.pn);
    // What the model finds best, of all sizes up to eight workgroups a compute unit.  us of a call, this / all at once, with 2 CUs / tiles
    // stretches where tiles are fewer than half the CUs: fp32 10000 x 512, 7088 tokens 1628 / 1733; 21701 x 300, 1000 tokens 396 / 419; 8000 x 64, 4000
    // tokens 194 / 210; 45376 x 1024, 96 tokens 486 / 513; bf16 25040 x 1000, 2371 tokens 614 / 618; 3000 x 128, 7000 tokens 93 / 97.  (The best
    // of a sweep is up to 3 % faster.)
    Stretches x{p.few ? 0 : tiles_of(n, p.pm) * tiles_of(H, p.pn), rp, rp, 1}, w{tiles_of(rows, p.pm) * tiles_of(H, p.pn), p.np, p.np, 1};
    const double us_per_k = 2. * p.pm * p.pn * (P == 3 ? 6 / 1450e6 : 1 / 1300e6) * num_cus();  // (the pipe's rates that large products reach)
    auto most_of = [&](const Stretches &g) {
      const int s = 8 * num_cus() / (g.tiles > 0 ? g.tiles : 8 * num_cus());
      return s < kSplits ? s : kSplits;
    };
    double best = INFINITY;
    const int sizes[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    for (int sx : sizes)
      for (int sw : sizes) {
        if ((sx > 1 && sx > most_of(x)) || (sw > 1 && sw > most_of(w))) break;
        x.set(sx), w.set(sw);
        double bytes = 0.;
        if (p.pieces > 1 || x.n > 1) bytes += x.n * (4. * n * H) * (1. + (p.pieces > 1) + 1. / p.pieces);
        if (w.n > 1) bytes += w.n * (8. * rows * H);
        const double us = products_us(x, w, us_per_k, bytes);
        if (us < best) best = us, p.xsplits = x.n, p.xchunk = x.chunk, p.wsplits = w.n, p.wchunk = w.chunk;
      }
    if (p.few) {
      p.facross = tiles_of(H, 32 * (n <= 32 ? few_columns<P, 1>() : few_columns<P, 2>()));
      // stretches for the two workgroups that a compute unit holds, of 128 classes or more (few classes: 64)
      int stretches = 2 * num_cus() / p.facross, least = rp <= 2048 ? 64 : 128;
      stretches = stretches > rp / least ? rp / least : stretches;
      stretches = stretches < 1 ? 1 : stretches;
      p.xchunk = ceil_to((rp + stretches - 1) / stretches, kPlaneAlign);
      p.xsplits = (rp + p.xchunk - 1) / p.xchunk;
    }
    const int twice = P == 1 && n <= kFewRows ? 2 : 1;  // (see dlogits_kernel)
    p.xt = take(packed_bytes<P>(H, twice * p.np));
    // W in one order, d W reading it by transposing loads, or packed with its classes as k too, whichever costs less.  us of a call, one order / two: bf16
    // 30000 x 1024 with 512 tokens 243 / 258, 1000 375 / 387, 2000 633 / 631, 3000 899 / 864; 50000 x 2048 with 1000 1042 / 1063, 4096 3317 / 3295; 128000 x
    // 4096 with 8192 32500 / 31450; 10000 x 512 with 7000 429 / 442; fp32 45376 x 1024 with 96 430 / 480, 10000 x 512 with 7088 1555 / 1556.  Narrow rows and
    // few tokens, a tile or three of d W, each a long way: fp32 81792 x 72 with 96 177 / 152, 300 276 / 270, 1000 635 / 675; bf16 112 / 103 with 96.
    p.one_order = (H > 128 || n > 512) && (P == 3 || n <= 2000 || H <= 512);
    p.wt = take(p.few || p.one_order ? 0 : packed_bytes<P>(H, rp));
    p.d = take(packed_bytes<P>(twice * p.np, rp));
    p.sums = take((size_t)tiles_of(n, p.bn) * C * 4);
    p.xpart = take((size_t)p.xsplits * n * H * 4);
    p.wpart = take(p.wsplits > 1 ? (size_t)p.wsplits * rows * H * 4 : 0);
  }
  p.bytes = at;
  return p;
}

inline PackJob packing(PackJob j) {
  j.across = tiles_of(j.K, 64);
  j.blocks = j.o.p || j.t.p ? j.across * tiles_of(j.rows, 64) : 0;
  return j;
}
template <int P, class Src>
void pack(const PackJob &a, const PackJob &b, hipStream_t st) {
  const int blocks = a.blocks + b.blocks, high = (blocks + kMostBlocks - 1) / kMostBlocks;
  if (blocks > 0) launch(pack_kernel<P, Src>, dim3((blocks + high - 1) / high, high), 256, 0, st, a, b);
}
template <class Out>
void sums(SumJob x, SumJob w, SumJob b, float scale, hipStream_t st) {
  for (SumJob *j : {&x, &w, &b}) {
    const long blocks = j->out ? ((long)j->rows * j->w + 255) / 256 : 0;
    j->blocks = (int)(blocks > 2048 ? 2048 : blocks);
  }
  if (x.blocks + w.blocks + b.blocks > 0) launch(sums_kernel<Out>, x.blocks + w.blocks + b.blocks, 256, 0, st, x, w, b, scale);
}

template <int P, class Src>
int run(const Call &c, const Plan &p, char *ws, hipStream_t st) {
  const int n = c.n, H = c.H, C = c.C;
  auto f32 = [&](size_t at) { return reinterpret_cast<float *>(ws + at); };
  auto pl = [&](size_t at) { return reinterpret_cast<u16 *>(ws + at); };
  auto ref = [](const PackedOut &o) { return PackedRef{o.p, o.K}; };
  const PackedOut none{}, X{pl(p.x), p.Hp};
  const bool keep = p.grads && p.keep, one = p.pieces == 1;
  float *lse = c.lse ? c.lse : f32(p.lse), *weight = f32(p.weight);
  auto piece_w = [&](int c0) { return PackedOut{pl(p.w + (keep ? packed_bytes<P>(c0, p.Hp) : 0)), p.Hp}; };
  auto rows_of = [&](int c0) { return C - c0 < p.piece ? C - c0 : p.piece; };
  auto piece_wt = [&](int rows) { return c.dX && !p.one_order ? PackedOut{pl(p.wt), ceil_to(rows, kPlaneAlign)} : none; };
  auto job_w = [&](int c0, bool o, bool t) {
    const int rows = rows_of(c0);
    return packing({static_cast<const Src *>(c.W) + (long)c0 * c.ldw, c.ldw, rows, H, o && !p.raw ? piece_w(c0) : none, t && p.grads ? piece_wt(rows) : none,
                    ceil_to(rows, kPlaneAlign), c.b ? c.b + c0 : nullptr, nullptr, nullptr, nullptr, 0, 0, 0});
  };
  const bool beside = P == 1 && c.dloss && n <= kFewRows;  // weights are not in d
  const int wk = beside ? 2 * p.np : p.np;                  // what d^T X sums over
  const PackedOut xt{p.grads && c.dW ? pl(p.xt) : nullptr, wk};
  // X in one launch with what there is of W by then
  PackJob jx = packing({c.X, c.ldx, n, H, p.few && n <= 32 ? none : X, xt, n, nullptr, c.labels, beside ? c.dloss : nullptr, c.b, C, 0, 0});
  auto tile_args = [&](int c0) {
    const int rows = rows_of(c0);
    return TileArgs{ref(piece_w(c0)), ref(X), rows, n, p.Hp, tiles_of(rows, p.bm), tiles_of(n, p.bn), c.b ? c.b + c0 : nullptr, c.labels, c0,
                    static_cast<const Src *>(c.W) + (long)c0 * c.ldw, c.ldw, H};
  };
  if (p.few) {
    pack<P, Src>(jx, PackJob{}, st);
    const DirectArgs a{c.W, c.X, c.ldw, c.ldx, ref(X), H, C, n, tiles_of(C, 32), c.b, c.labels, reinterpret_cast<float2 *>(ws + p.stats), f32(p.zlabel),
                       p.grads ? f32(p.z) : nullptr};
    if (n <= 32) launch(direct_stats_kernel<P, Src, 1, false>, p.tiles, 256, 0, st, a);
    else launch(direct_stats_kernel<P, Src, 2, true>, p.tiles, 256, 0, st, a);
  }
  if (!c.lse_given) {
    for (int c0 = 0; c0 < C && !p.few; c0 += p.piece) {
      pack<P, Src>(jx, job_w(c0, true, one), st);
      jx = PackJob{};
      const TileArgs a = tile_args(c0);
      with_tile<P>(p.size, [&](auto t) {
        using T = decltype(t);
        launch(stats_kernel<T>, a.tilesM * a.tilesN, T::THREADS, 0, st, a, reinterpret_cast<float2 *>(ws + p.stats), f32(p.zlabel));
        return 0;
      });
    }
    const RowArgs r{reinterpret_cast<const float2 *>(ws + p.stats), p.tiles, n, C, f32(p.zlabel), c.labels, c.b, c.dloss, c.loss, lse, p.grads ? weight : nullptr};
    if (n <= 1024) launch(rows_kernel<1>, n, 256, 0, st, r);
    else launch(rows_kernel<16>, (n + 15) / 16, 256, 0, st, r);
  } else {
    launch(weights_kernel, (n + 255) / 256, 256, 0, st, c.labels, c.lse_given, c.b, c.dloss, n, C, weight);
  }
  if (p.grads) {
    const float *all = c.lse_given ? c.lse_given : lse;
    const int token_tiles = tiles_of(n, p.bn);
    const bool x_parts = p.few || !one || p.xsplits > 1, w_parts = p.wsplits > 1, b_parts = !p.few && token_tiles > 1;
    bool first = true;
    for (int c0 = 0; c0 < C; c0 += p.piece, first = false) {
      const int rows = rows_of(c0), rp = ceil_to(rows, kPlaneAlign);
      // (what the first pass packed may still be there)
      if (!p.few) pack<P, Src>(jx, job_w(c0, c.lse_given || !(keep || one), c.lse_given || !one), st);
      jx = PackJob{};
      const TileArgs a = tile_args(c0);
      const PackedOut d{c.dX || c.dW ? pl(p.d) : nullptr, rp};
      if (p.few && (d.p || c.db)) {
        const FewLogitsArgs f{f32(p.z), all, weight, c.labels, n, C, c0, d, rp / 32, c.db ? c.db + c0 : nullptr, c.scale, beside};
        launch(few_dlogits_kernel<P>, (rp / 32 + 3) / 4, 256, 0, st, f);
      } else if (d.p || c.db) {
        with_product_tile<P>(p.size, [&](auto t) {
          using T = decltype(t);
          launch(dlogits_kernel<T>, a.tilesM * a.tilesN, T::THREADS, 0, st, a, all, weight, d, !c.db ? nullptr : b_parts ? f32(p.sums) + c0 : c.db + c0, C,
                 b_parts ? 1.f : c.scale, (int)beside);
          return 0;
        });
      }
      auto job = [&](const PackedOut &A, const PackedOut &B, int M, int K, int chunk, float *part, bool add, void *out, long ldo, const float *factor) {
        return ProductJob<Src>{ref(A), ref(B), M, H, K, tiles_of(M, p.pm), tiles_of(H, p.pn), (K + chunk - 1) / chunk, chunk, part, add,
                               static_cast<Src *>(out), ldo, c.scale, factor};
      };
      ProductJob<Src> px{}, pw{};
      // (a last piece shorter than the others fills fewer stretches: those beyond keep what they have)
      if (c.dX && !p.few) px = job(d, p.one_order ? piece_w(c0) : piece_wt(rows), n, rp, p.xchunk, x_parts ? f32(p.xpart) : nullptr, !first, c.dX, c.lddx, beside ? weight : nullptr);
      Src *dW = c.dW ? static_cast<Src *>(c.dW) + (long)c0 * c.lddw : nullptr;
      if (c.dW) pw = job(d, xt, rows, wk, beside ? wk : p.wchunk, w_parts ? f32(p.wpart) : nullptr, false, dW, c.lddw, nullptr);
      // (d W of more than the last cache holds, in whole lines of 128 bytes: bf16 124416 x 2176, 64 tokens 533 us of a call, streaming 469, 81664 x 4096, 12
      // tokens 544, 456; lines in parts the other way, fp32 40806 x 4050, 12 tokens 823, 940)
      const bool stream = p.few && c.dW && (size_t)C * H * sizeof(Src) > 256u << 20 && (uintptr_t)c.dW % 128 == 0 && c.lddw * sizeof(Src) % 128 == 0 && H * sizeof(Src) % 128 == 0;
      const int bx = c.dX && !p.few ? px.tilesM * px.tilesN * px.splits : 0, bw = c.dW ? pw.tilesM * pw.tilesN * pw.splits : 0;
      if (bx + bw > 0)
        with_product_tile<P>(p.psize, [&](auto t) {
          using T = decltype(t);
          if constexpr (std::is_same_v<T, typename Tiles<P>::L>)  // (so large a d W has tiles enough)
            if (stream) return launch(product_kernel<T, Src, true, true>, bx + bw, T::THREADS, 0, st, px, pw, bx), 0;
          if (p.one_order) launch(product_kernel<T, Src, false, true>, bx + bw, T::THREADS, 0, st, px, pw, bx);
          else launch(product_kernel<T, Src, false, false>, bx + bw, T::THREADS, 0, st, px, pw, bx);
          return 0;
        });
      if (c.dX && p.few) {
        const FewArgs f{static_cast<const Src *>(c.W) + (long)c0 * c.ldw, c.ldw, ref(d), rows, n, H, c.b ? c.b + c0 : nullptr, p.facross, p.xchunk,
                        f32(p.xpart), !first};
        const int grid = p.facross * ((rp + p.xchunk - 1) / p.xchunk);
        if (n <= 32) launch(few_dx_kernel<P, Src, 1>, grid, 256, 0, st, f);
        else launch(few_dx_kernel<P, Src, 2>, grid, 256, 0, st, f);
      }
      const bool last = c0 + p.piece >= C;
      SumJob sx{}, sw{}, sb{};
      if (last && c.dX && x_parts) sx = {f32(p.xpart), p.xsplits, n, H, beside ? weight : nullptr, c.dX, c.lddx, 0};
      if (dW && w_parts) sw = {f32(p.wpart), p.wsplits, rows, H, nullptr, dW, c.lddw, 0};
      if (last && c.db && b_parts) sb = {f32(p.sums), token_tiles, 1, C, nullptr, c.db, C, 0};
      sums<Src>(sx, sw, sb, c.scale, st);
    }
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
    const SumJob w{nullptr, 0, c.C, c.H, nullptr, c.dW, c.lddw, 0}, b{nullptr, 0, 1, c.C, nullptr, c.db, c.C, 0};
    if (type == CAVS_F32) sums<float>({}, w, b, 0.f, st);
    else sums<u16>({}, w, b, 0.f, st);
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
