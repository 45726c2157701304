// Products C = A B^T of operands packed for the bf16 matrix pipe.
//
// An operand of type bf16 is one part.  A float is the sum of bf16 parts, h = bf16(x), m = bf16(x - h), l = bf16(x - h - m); three of
// them hold all its bits, two hold 16.  A product of operands of P parts adds up the P (P + 1) / 2 products of weight 2^-8(P-1) and
// above: six of nine, three of four.  The products of the first parts go into one set of accumulators and all the others, a 2^-8
// smaller, into a second: the pipe loses an addend of less than about an eighth of its accumulator's last place, and beside their own
// kind the small ones are not lost.  (gemm_split.h splits on the way into LDS; here whoever makes an operand writes its parts,
// as the same operand goes into several products, and a tile's loads go to LDS without passing through registers.)
//
// A packed operand [rows, K] is blocks of 32 rows by 16 k, 1 KB a part: lane l of a wavefront finds its piece for the 32x32x16 instruction,
// eight k of row l % 32, at byte 16 l.  Blocks follow each other part by part, then along k, then along the rows.  So a wavefront's load is 1 KB in
// one piece, and LDS is read in the order it was written.  (Rows of bf16 as they lie in memory, 32 or 128 bytes of each to a tile: the loads of a
// 128 x 128 x 16 tile alone took 2277 us of 7088 x 4096 x 3584, all of it takes 865 now.)  K is padded with zeros to whole steps: the loops
// below know no k that is not there.  Blocks of rows beyond the last read the last one again; what comes of them is not stored.
//
// A workgroup is four wavefronts and its LDS two stages, so that a CU holds three of them that know nothing of each other: while one waits
// for its loads the others multiply.  TFLOP/s of the bf16 pipe, random operands (power holds the clock at 1.9 GHz):
//   one part     8192 x 8192 x 4096   256 x 128 x 32 1342    256 x 256 x 32, eight wavefronts 1349    128 x 128 x 32 1213
//   three parts  7088 x 4096 x 3584   128 x 128 x 16 1444 (241 of the fp32 product)   256 x 128 x 32, eight wavefronts 1351
//   two parts    4096 x 4096 x 4096   128 x 128 x 16, three stages 1323   256 x 128 x 32, eight wavefronts 1369 (too few tiles of smaller matrices)
#pragma once
#include "gemm_common.h"

namespace cavs {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16;

constexpr int kPlaneAlign = 64;  // of K, in elements

struct PackedRef {
  const u16 *p;
  int K;  // a multiple of kPlaneAlign
};
struct PackedOut {
  u16 *p;
  int K;
};
template <int P>
constexpr size_t packed_bytes(long rows, int K) { return (size_t)((rows + 31) / 32 * 32) * K * 2 * P; }

// bf16 of a float (to nearest), its bits
__device__ inline u16 bf16_bits(float x) { return __builtin_bit_cast(u16, (__bf16)x); }
__device__ inline float bf16_float(u16 b) { return __uint_as_float((unsigned)b << 16); }

// The parts of x.  A finite x that bf16 would round to infinity (above 3.39e38) has bf16's largest value as its first part; what is left are 16 bits, which
// the other two hold.  Of an infinity or a NaN the last part is NaN, and so is what it is multiplied into.  The one part of type bf16 is what bf16 makes of x.
template <int P>
__device__ inline void parts_of(float x, u16 (&o)[P]) {
  if constexpr (P == 1) {
    o[0] = bf16_bits(x);
  } else {
    constexpr float most = 3.38953139e38f;  // (2^128 - 2^120)
    float rest = x;
    o[0] = bf16_bits(__builtin_amdgcn_fmed3f(x, -most, most));
#pragma unroll
    for (int p = 1; p < P; p++) {
      rest -= bf16_float(o[p - 1]);
      o[p] = bf16_bits(rest);
    }
  }
}

// NS: stages in LDS.
template <int P_, int BM_, int BN_, int BK_, int WGM_, int WGN_, int NS_ = 2>
struct NtTile {
  static constexpr int P = P_, BM = BM_, BN = BN_, BK = BK_, WGM = WGM_, WGN = WGN_, NS = NS_;
  static constexpr bool RAW = false;  // (an operand of another layout)
  static constexpr int WAVES = WGM * WGN, THREADS = 64 * WAVES;
  static constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 32, TN = WN / 32;
  static constexpr int STEPS = BK / 16, ROWB = 1024 * P * STEPS;    // bytes a row of blocks takes of a stage
  static constexpr int CA = BM / 32 * P * STEPS / WAVES, CB = BN / 32 * P * STEPS / WAVES;  // blocks a wavefront loads per stage
  static constexpr int PA = BM / 32 * ROWB, STAGE = (BM + BN) / 32 * ROWB, LDS = NS * STAGE;
  static constexpr int LOADS = CA + CB;
  static constexpr int ACC = P > 1 ? 2 : 1;
  static constexpr int GROUPS = 160 * 1024 / LDS;                   // workgroups a CU's LDS has room for
  static constexpr int EU = GROUPS * WAVES / 4 < 4 ? GROUPS * WAVES / 4 : WM < 64 ? 4 : 3;  // wavefronts a SIMD is to hold
  static_assert(BM / 32 * P * STEPS % WAVES == 0 && BN / 32 * P * STEPS % WAVES == 0, "a tile's loads are the same for every wavefront");
  static_assert(kPlaneAlign % BK == 0, "operands end on a step");
  static_assert(NS >= 2 && LDS <= 160 * 1024, "stages");
};

// Until at most N of this wavefront's loads are on their way and all it read from LDS is there; then until every wavefront is here.  (A barrier
// by itself waits for neither, and __syncthreads would wait for all loads.)
template <int N>
__device__ __forceinline__ void nt_arrive() {
  if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A piece (eight k of row l % 32) from where its two half blocks of sixteen rows lie
__device__ __forceinline__ bf16x8 turned_piece(const char *from, int lane) {
  const int group = lane >> 4 & 1, half = lane >> 5;
  const char *p = from + group * 512 + half * 256 + 8 * (lane & 15);
#ifdef __HIP_DEVICE_COMPILE__
  typedef short four __attribute__((ext_vector_type(4)));
  const four lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) four *)(p + 128 * (half ^ group)));
  const four hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) four *)(p + 128 * (half ^ group ^ 1)));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
  return *reinterpret_cast<const bf16x8 *>(p);
#endif
}

// acc[ACC][TM][TN] of the tile at rows m0 of A and n0 of B over k in [kbeg, kend), both multiples of BK.  S: T::LDS bytes.
// TA: what is given is A^T, packed with A's rows as its k and with all of A's k as rows (its last block of rows whole, and as many as kend
// asks for).  A step's half blocks of 16 of its rows by 16 k, 512 bytes, come to LDS row by row, and the transposing load makes of four neighbouring
// values of four rows, sixteen lanes at a time, four k of sixteen rows of A.  (Bit 7 of a place is turned over by bit 3 of the row and
// bit 4 of k: of the four groups of lanes no two that could go together meet in a bank.)  TB: the same of B.
// NS stages in a ring: while one is multiplied the others are on their way from memory; a step's one barrier says that the stage to come
// has arrived and that nobody reads the one before it any more, so that its place takes the load of the stage NS - 1 ahead.
template <class T, bool TA = false, bool TB = false>
__device__ __forceinline__ void nt_multiply(const PackedRef &A, int M, int m0, const PackedRef &B, int N, int n0, int kbeg, int kend, char *S,
                                            floatx16 (&acc)[T::ACC][T::TM][T::TN]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WGN, wn = wave % T::WGN;
#pragma unroll
  for (int s = 0; s < T::ACC; s++)
#pragma unroll
    for (int i = 0; i < T::TM; i++)
#pragma unroll
      for (int j = 0; j < T::TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[s][i][j][r] = 0.f;

  // Blocks c = 0, 1, .. of a stage, in the order they have in memory: row of blocks by row of blocks, step by step, part by part.  This wavefront
  // loads every WAVES-th, each lane the 16 bytes it will read.
  constexpr int PER = T::P * T::STEPS;
  unsigned sa[T::CA], sb[T::CB], la[T::CA], lb[T::CB];
  const long rowa = (long)(A.K / 16) * T::P * 1024, rowb = (long)(B.K / 16) * T::P * 1024;
  auto source = [&](bool turned, int at, int blocks, int K, int rows, int first, unsigned row, unsigned *of_lane, unsigned *of_wave) {
    if (!turned) {
      *of_lane = 16 * lane;
      *of_wave = (unsigned)min(at / PER, (rows - 1 - first) / 32) * row + at % PER * 1024;
    } else {  // two half blocks, of neighbouring sixteens of rows: step by step, part by part, down the tile
      const int which = at / blocks, step = which / T::P, sixteen = at % blocks * 2 + (lane >> 5), place = lane & 31;
      const int here = place ^ 8 * ((place >> 4) ^ (lane >> 5));
      *of_lane = min(sixteen, K / 16 - 1 - first / 16) * (T::P * 1024) + (here & 1) * 512 + (here >> 1) * 16;
      *of_wave = (step >> 1) * row + (step & 1) * 256 + which % T::P * 1024;
    }
  };
#pragma unroll
  for (int c = 0; c < T::CA; c++) source(TA, c * T::WAVES + wave, T::BM / 32, A.K, M, m0, (unsigned)rowa, &la[c], &sa[c]);
#pragma unroll
  for (int c = 0; c < T::CB; c++) source(TB, c * T::WAVES + wave, T::BN / 32, B.K, N, n0, (unsigned)rowb, &lb[c], &sb[c]);
  auto begin = [&](bool turned, const u16 *p, int first, long row) {
    return reinterpret_cast<const char *>(p) + (turned ? kbeg / 32 * row + (long)(first / 16) * (T::P * 1024) : first / 32 * row + (long)(kbeg / 16) * (T::P * 1024));
  };
  [[maybe_unused]] const char *pa = begin(TA, A.p, m0, rowa), *pb = begin(TB, B.p, n0, rowb);

  auto fetch = [&](int kt, char *to) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass knows no such load)
    const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(TA ? pa + (long)(kt * T::STEPS / 2) * rowa : pa), 0, 0xffffffffu, 0x00020000);
    const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(TB ? pb + (long)(kt * T::STEPS / 2) * rowb : pb), 0, 0xffffffffu, 0x00020000);
    const unsigned on = (unsigned)kt * (PER * 1024), half = kt * T::STEPS % 2 * 256;
#pragma unroll
    for (int c = 0; c < T::CA; c++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void *)(to + (c * T::WAVES + wave) * 1024), 16, la[c], sa[c] + (TA ? half : on), 0, 0);
#pragma unroll
    for (int c = 0; c < T::CB; c++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (__attribute__((address_space(3))) void *)(to + T::PA + (c * T::WAVES + wave) * 1024), 16, lb[c],
                                               sb[c] + (TB ? half : on), 0, 0);
#endif
  };
  const int a0 = wm * (T::WM / 32) * T::ROWB + 16 * lane, b0 = T::PA + wn * (T::WN / 32) * T::ROWB + 16 * lane;
  // A's parts from the last to the first, each with those of B that it meets: one part of A and what there is of B by then are all that registers hold
  auto step = [&](const char *from, int s) {
    bf16x8 b[T::P][T::TN];
#pragma unroll
    for (int p = T::P - 1; p >= 0; p--) {
      bf16x8 a[T::TM];
#pragma unroll
      for (int i = 0; i < T::TM; i++) {
        if constexpr (!TA) a[i] = *reinterpret_cast<const bf16x8 *>(from + a0 + (i * T::ROWB + (s * T::P + p) * 1024));
        else a[i] = turned_piece(from + wm * (T::WM / 32) * 1024 + ((s * T::P + p) * (T::BM / 32) + i) * 1024, lane);
      }
#pragma unroll
      for (int j = 0; j < T::TN; j++) {
        const int q = T::P - 1 - p;
        if constexpr (!TB) b[q][j] = *reinterpret_cast<const bf16x8 *>(from + b0 + (j * T::ROWB + (s * T::P + q) * 1024));
        else b[q][j] = turned_piece(from + T::PA + wn * (T::WN / 32) * 1024 + ((s * T::P + q) * (T::BN / 32) + j) * 1024, lane);
      }
#pragma unroll
      for (int q = T::P - 1 - p; q >= 0; q--)
#pragma unroll
        for (int i = 0; i < T::TM; i++)
#pragma unroll
          for (int j = 0; j < T::TN; j++)
            acc[p + q ? T::ACC - 1 : 0][i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[q][j], acc[p + q ? T::ACC - 1 : 0][i][j], 0, 0, 0);
    }
  };
  const int nk = (kend - kbeg) / T::BK;
#pragma unroll
  for (int q = 0; q < T::NS - 1; q++)
    if (q < nk) fetch(q, S + q * T::STAGE);
  int at = 0;
  for (int kt = 0; kt < nk; kt++) {
    if (kt + T::NS - 2 < nk) nt_arrive<(T::NS - 2) * T::LOADS>();
    else nt_arrive<0>();
    if (kt + T::NS - 1 < nk) fetch(kt + T::NS - 1, S + (at == 0 ? (T::NS - 1) * T::STAGE : at - T::STAGE));
#pragma unroll
    for (int s = 0; s < T::STEPS; s++) {
      step(S + at, s);
      // (one part, 256 x 128: the compiler's own pattern for a product's loop, 2.5 % faster; the others are as fast without)
      if constexpr (T::P == 1 && T::BM == 256) __builtin_amdgcn_iglp_opt(1);
    }
    at = at == (T::NS - 1) * T::STAGE ? 0 : at + T::STAGE;
  }
  nt_arrive<0>();  // (LDS is free for what follows)
}

// The tiles of a launch over tilesM x tilesN: eight tiles of A at a time, down each tile of B, the tiles that one XCD runs together reading
// few panels of either operand.
__device__ inline void nt_tile_of(int block, int tilesM, int tilesN, int *tm, int *tn) {
  const int t = xcd_remap(block, tilesM * tilesN);
  const int band = t / (8 * tilesN), in = t - band * 8 * tilesN, high = min(8, tilesM - 8 * band);
  *tm = 8 * band + in % high;
  *tn = in / high;
}

// The 32 x 32 values a wavefront holds of an accumulator (lane l, element r: c = l % 32, r' = 8 (r / 4) + 4 (l / 32) + r % 4), as parts, into a
// packed operand: with x = c, k = r' ("rows", 16-byte pieces of two halves), or with x = r', k = c ("columns", by way of LDS: kTurn bytes
// of the wavefront's own).  xb, kb: the block of 32 rows, of 32 k.
constexpr int kTurn = 4 * 528;
template <int P>
struct Parts16 {
  u16 v[16][P];
};
template <int P>
__device__ inline void put_rows(const PackedOut &o, int xb, int kb, const Parts16<P> &t, int lane) {
#pragma unroll
  for (int p = 0; p < P; p++)
#pragma unroll
    for (int q = 0; q < 4; q++)
      *reinterpret_cast<uint2 *>(o.p + (((long)xb * (o.K / 16) + 2 * kb + (q >> 1)) * P + p) * 512 + ((lane & 31) + 32 * (q & 1)) * 8 + 4 * (lane >> 5)) =
          make_uint2(t.v[4 * q][p] | (unsigned)t.v[4 * q + 1][p] << 16, t.v[4 * q + 2][p] | (unsigned)t.v[4 * q + 3][p] << 16);
}
template <int P>
__device__ inline void put_columns(const PackedOut &o, int xb, int kb, const Parts16<P> &t, int lane, char *turn) {
  // eight k of a row are a piece; pieces of the same eight k lie together, 16 bytes further for the next eight so that all banks take part
  u16 *in = reinterpret_cast<u16 *>(turn + (lane >> 3 & 3) * 528 + (lane >> 5) * 64 + (lane & 7) * 2);
#pragma unroll
  for (int p = 0; p < P; p++) {
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int r = 0; r < 16; r++) in[(8 * (r >> 2) + (r & 3)) * 8] = t.v[r][p];
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");  // (a wavefront's own accesses to LDS happen in their order)
#pragma unroll
    for (int b = 0; b < 2; b++)
      *reinterpret_cast<uint4 *>(o.p + (((long)xb * (o.K / 16) + 2 * kb + b) * P + p) * 512 + lane * 8) =
          *reinterpret_cast<const uint4 *>(turn + (2 * b + (lane >> 5)) * 528 + (lane & 31) * 16);
  }
}

// 64 x 64 values in LDS as parts, into packed operands: rows r0 .. of `o` with k = k0 .., and rows k0 .. of `t` with k = r0 ..; 256 threads.
// What lies beyond `rows` and `cols` is zero in the tile.
typedef float PackTile[64][65];
template <int P>
__device__ inline void pack_tile(const PackTile &tile, const PackedOut &o, const PackedOut &t, int r0, int k0, int rows, int cols) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = lane & 31, h = lane >> 5;
#pragma unroll
  for (int b = 0; b < 2; b++) {  // a block of 32 rows; the wavefront's 16 k
    auto put = [&](const PackedOut &to, int row0, int col0, int all, auto &&at) {
      if (row0 + 32 * b >= all || col0 + 16 * wave >= to.K) return;
      u16 part[8][P];
#pragma unroll
      for (int e = 0; e < 8; e++) parts_of<P>(at(32 * b + x, 16 * wave + 8 * h + e), part[e]);
#pragma unroll
      for (int p = 0; p < P; p++)
        *reinterpret_cast<uint4 *>(to.p + (((long)(row0 / 32 + b) * (to.K / 16) + col0 / 16 + wave) * P + p) * 512 + lane * 8) =
            make_uint4(part[0][p] | (unsigned)part[1][p] << 16, part[2][p] | (unsigned)part[3][p] << 16, part[4][p] | (unsigned)part[5][p] << 16,
                       part[6][p] | (unsigned)part[7][p] << 16);
    };
    if (o.p) put(o, r0, k0, rows, [&](int r, int k) { return tile[r][k]; });
    if (t.p) put(t, k0, r0, cols, [&](int r, int k) { return tile[k][r]; });
  }
}

// an operand's element as a float
__device__ inline float value_of(const float *p) { return *p; }
__device__ inline float value_of(const u16 *p) { return bf16_float(*p); }

// rows r0 .. r0 + 63, columns k0 .. k0 + 63 of src [rows, K] into a tile, zero beyond; 256 threads, four neighbouring values of a lane at a time
// (one at a time the bf16 rows of 124416 x 2176 took 612 us to pack)
template <class Src>
__device__ inline void load_tile(PackTile &tile, const Src *src, long ld, int r0, int k0, int rows, int K) {
  typedef Src four __attribute__((ext_vector_type(4), aligned(sizeof(Src))));
  const int k = 4 * (threadIdx.x & 15);
  four v[4];
#pragma unroll
  for (int q = 0; q < 4; q++) {
    const int r = r0 + (threadIdx.x >> 4) + 16 * q;
    const Src *p = src + r * ld + k0 + k;
    if (r < rows && k0 + k + 4 <= K) {
      v[q] = *reinterpret_cast<const four *>(p);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[q][e] = r < rows && k0 + k + e < K ? p[e] : Src(0);
    }
  }
#pragma unroll
  for (int q = 0; q < 4; q++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const Src one = v[q][e];
      tile[(threadIdx.x >> 4) + 16 * q][k + e] = value_of(&one);
    }
}

__device__ inline void store_as(float *o, float x) { *o = x; }
__device__ inline void stream_as(float *o, float x) { __builtin_nontemporal_store(x, o); }
__device__ inline void stream_as(u16 *o, float x) { __builtin_nontemporal_store(bf16_bits(x), o); }
__device__ inline void store_as(u16 *o, float x) { *o = bf16_bits(x); }

constexpr int ceil_to(int x, int to) { return (x + to - 1) / to * to; }
inline int tiles_of(int x, int side) { return (x + side - 1) / side; }


}  // namespace cavs
