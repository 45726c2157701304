// Products of bf16 matrices as they lie in memory: result[row, col] = sum over k of A[col, k] B[row, k], tiles of the transposed product, so that a lane
// holds neighbouring columns of a row of the result.
//
// An operand is given [rows, k] or, "turned", [k, rows]; its rows in memory begin on 16 bytes and are whole pieces of eight values.  64 k of a tile go to LDS
// without passing through registers, 16 bytes a lane, 1 KB a wavefront's load: what lies there in the order of the lanes is put into an order that
// spreads over the banks by what each lane asks for.
//   [rows, k]: 128 bytes of a row are eight pieces; piece q of row r is at q ^ (r / 2 % 8).  Sixteen lanes that read a piece of sixteen rows meet no bank twice.
//   [k, rows]: 256 bytes of a line of k are 128 rows in pieces of eight; piece q of line k is at q ^ (4 (k % 4) + 2 (k / 8 % 2)).  The transposing load takes
//   four lines of sixteen rows for each sixteen lanes.
// The transposing loads are assembly with their wait in it: the compiler takes the builtin for a reader of whatever is on its way from memory and waits for
// all of that first (256 x 256 tiles, 4096 x 8192 x 8192: 570 us with the builtin, 399 so).
#pragma once
#include "nt_product.h"

namespace cavs {

typedef float floatx4 __attribute__((ext_vector_type(4)));

struct DirectRef {
  const u16 *p;
  long ld;  // of a row, or of a line of k
};

__device__ __forceinline__ void lds_from(const char *p, unsigned bytes, unsigned at, char *to) {
#ifdef __HIP_DEVICE_COMPILE__
  const unsigned long long v = reinterpret_cast<unsigned long long>(p);
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
  const auto r = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char *>((unsigned long long)hi << 32 | lo), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)to, 16, at, 0, 0, 0);
#endif
}

// What this wavefront loads of 128 rows by 64 k, KB by KB (of 16): blocks first, first + 1, ..  Relative to the tile's first row and k, bytes.
template <int C, bool TURNED>
struct DirectSource {
  unsigned v[C];
  short k[C];  // the first k of each
  __device__ __forceinline__ void set(const DirectRef &o, int row0, int left, int block, int lane) {  // left: rows there are, from the tile's first
#pragma unroll
    for (int c = 0; c < C; c++) {
      if constexpr (!TURNED) {
        const int r = (block + c) * 8 + (lane >> 3), q = (lane & 7) ^ (r >> 1 & 7);
        v[c] = (unsigned)min(row0 + r, left - 1) * (unsigned)(o.ld * 2) + q * 16;
        k[c] = q * 8;
      } else {
        const int line = (block + c) * 4 + (lane >> 4), q = (lane & 15) ^ (4 * (line & 3) + 2 * (line >> 3 & 1));
        v[c] = (unsigned)line * (unsigned)(o.ld * 2) + min(row0 / 8 + q, left / 8 - 1) * 16;
        k[c] = line;
      }
    }
  }
  // whole stages; a buffer of no bytes: nothing is read
  __device__ __forceinline__ void load(const char *p, unsigned bytes, char *to) const {
#pragma unroll
    for (int c = 0; c < C; c++) lds_from(p, bytes, v[c], to + c * 1024);
  }
  // the first `rest` k, zeros behind them
  __device__ __forceinline__ void load_rest(const char *p, int rest, char *to, int lane) const {
#pragma unroll
    for (int c = 0; c < C; c++) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (k[c] < rest) x = *reinterpret_cast<const uint4 *>(p + v[c]);
      *reinterpret_cast<uint4 *>(to + c * 1024 + lane * 16) = x;
    }
  }
};

// Where a lane finds its pieces for the 16x16x32 instruction: row l % 16, eight k from 8 (l / 16) on, of blocks t of sixteen rows from `row0` on (a multiple
// of 32) and steps s of 32 k.
template <int T, bool TURNED>
struct DirectPieces {
  unsigned at[TURNED ? T : 2];
  __device__ __forceinline__ void set(int row0, int lane) {
    if constexpr (!TURNED) {
#pragma unroll
      for (int s = 0; s < 2; s++) at[s] = (row0 + (lane & 15)) * 128 + ((4 * s + (lane >> 4)) ^ (lane >> 1 & 7)) * 16;
    } else {
      const int x = 4 * (lane >> 2 & 3) + 2 * (lane >> 4 & 1);
#pragma unroll
      for (int t = 0; t < T; t++) at[t] = (8 * (lane >> 4) + (lane >> 2 & 3)) * 256 + ((row0 / 8 + 2 * t + (lane >> 1 & 1)) ^ x) * 16 + 8 * (lane & 1);
    }
  }
  __device__ __forceinline__ bf16x8 piece(const char *from, int t, int s) const {  // not turned
    return *reinterpret_cast<const bf16x8 *>(from + at[s] + t * 2048);
  }
};

// turned pieces, all there when this returns (as is all that was read before): two or four blocks of sixteen rows, both steps
__device__ __forceinline__ void turned_pieces(const char *from, const DirectPieces<2, true> &a, bf16x8 (&o)[2][2]) {
#ifdef __HIP_DEVICE_COMPILE__
  const unsigned base = lds_address(from);
  u32x2 t[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:1024\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:1024\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:8192\n\tds_read_b64_tr_b16 %5, %8 offset:9216\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:8192\n\tds_read_b64_tr_b16 %7, %9 offset:9216\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]), "=&v"(t[3]), "=&v"(t[4]), "=&v"(t[5]), "=&v"(t[6]), "=&v"(t[7])
      : "v"(base + a.at[0]), "v"(base + a.at[1])
      : "memory");
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll
    for (int i = 0; i < 2; i++) o[i][s] = both(t[4 * s + 2 * i], t[4 * s + 2 * i + 1]);
#endif
}
__device__ __forceinline__ void turned_pieces(const char *from, const DirectPieces<4, true> &a, bf16x8 (&o)[4][2]) {
#ifdef __HIP_DEVICE_COMPILE__
  const unsigned base = lds_address(from);
  u32x2 t[16];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:1024\n\t"
      "ds_read_b64_tr_b16 %2, %17\n\tds_read_b64_tr_b16 %3, %17 offset:1024\n\t"
      "ds_read_b64_tr_b16 %4, %18\n\tds_read_b64_tr_b16 %5, %18 offset:1024\n\t"
      "ds_read_b64_tr_b16 %6, %19\n\tds_read_b64_tr_b16 %7, %19 offset:1024\n\t"
      "ds_read_b64_tr_b16 %8, %16 offset:8192\n\tds_read_b64_tr_b16 %9, %16 offset:9216\n\t"
      "ds_read_b64_tr_b16 %10, %17 offset:8192\n\tds_read_b64_tr_b16 %11, %17 offset:9216\n\t"
      "ds_read_b64_tr_b16 %12, %18 offset:8192\n\tds_read_b64_tr_b16 %13, %18 offset:9216\n\t"
      "ds_read_b64_tr_b16 %14, %19 offset:8192\n\tds_read_b64_tr_b16 %15, %19 offset:9216\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]), "=&v"(t[3]), "=&v"(t[4]), "=&v"(t[5]), "=&v"(t[6]), "=&v"(t[7]), "=&v"(t[8]), "=&v"(t[9]), "=&v"(t[10]),
        "=&v"(t[11]), "=&v"(t[12]), "=&v"(t[13]), "=&v"(t[14]), "=&v"(t[15])
      : "v"(base + a.at[0]), "v"(base + a.at[1]), "v"(base + a.at[2]), "v"(base + a.at[3])
      : "memory");
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll
    for (int i = 0; i < 4; i++) o[i][s] = both(t[8 * s + 2 * i], t[8 * s + 2 * i + 1]);
#endif
}
template <int T, bool TURNED>
__device__ __forceinline__ void pieces_of(const char *from, const DirectPieces<T, TURNED> &a, bf16x8 (&o)[T][2]) {
  if constexpr (TURNED) turned_pieces(from, a, o);
  else
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int t = 0; t < T; t++) o[t][s] = a.piece(from, t, s);
}

// 256 x 256 x 64, eight wavefronts, each four quarters of 64 x 32.  Two wavefronts share a SIMD and take turns: while one reads its pieces from LDS and asks for
// two KB from memory, the other multiplies; a barrier, and they change places.  A quarter is all of a stage's k, so of the four halves of a stage each (A0, A1:
// 128 rows of A, B0, B1 of B) is read into registers in one turn, and its place takes the load of the stage after the next two turns later: what a turn
// reads was asked for six turns of both before (a load's way takes about two).
// One wavefront a SIMD with 128 x 128 and all four halves at once was slower (453 us against 411), as were tiles of 32 k in rings of five (480).
struct WideTile {
  static constexpr int BM = 256, BN = 256, THREADS = 512, I = 8, J = 2, EU = 2;  // I blocks of sixteen columns, J of 32 rows of the result a wavefront
  static constexpr int HALF = 16384, STAGE = 4 * HALF, LDS = 2 * STAGE;
  __device__ static __forceinline__ int col(int wave, int lane, int i) { return (i >> 2) * 128 + (wave & 1) * 64 + (i & 3) * 16 + 8 * (lane >> 5); }
  __device__ static __forceinline__ int row(int wave, int lane, int j) { return j * 128 + (wave >> 1) * 32 + (lane & 31); }
};

// until every wavefront is here (nothing is moved across it)
__device__ __forceinline__ void turn_over() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// acc of the tile at rows m0 of A (M of them) and n0 of B (N) over k in [kbeg, kend).  S: LDS.
template <bool TA, bool TB>
__device__ __forceinline__ void direct_multiply(const WideTile &, const DirectRef &A, int M, int m0, const DirectRef &B, int N, int n0, int kbeg, int kend, char *S,
                                                floatx4 (&acc)[8][4]) {
  constexpr int A0 = 0, A1 = WideTile::HALF, B0 = 2 * WideTile::HALF, B1 = 3 * WideTile::HALF, ST = WideTile::STAGE;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = wave >> 2, mine = 2048 * wave;
#pragma unroll
  for (int i = 0; i < 8; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  DirectSource<2, TA> a0, a1;
  DirectSource<2, TB> b0, b1;
  a0.set(A, 0, M - m0, 2 * wave, lane), a1.set(A, 128, M - m0, 2 * wave, lane);
  b0.set(B, 0, N - n0, 2 * wave, lane), b1.set(B, 128, N - n0, 2 * wave, lane);
  const char *pa = reinterpret_cast<const char *>(TA ? A.p + kbeg * A.ld + m0 : A.p + m0 * A.ld + kbeg);
  const char *pb = reinterpret_cast<const char *>(TB ? B.p + kbeg * B.ld + n0 : B.p + n0 * B.ld + kbeg);
  const long da = TA ? 128 * A.ld : 128, db = TB ? 128 * B.ld : 128;
  const int rest = (kend - kbeg) & 63, full = (kend - kbeg) / 64;
  const unsigned bytes = full > 0 ? 0xffffffffu : 0u;
  int asked = 0;
  auto step_on = [&]() {  // (behind the last stage: once more the last, into places that nobody reads)
    if (++asked < full) pa += da, pb += db;
  };
  // k that are no whole stage come first
  if (rest) {
    b0.load_rest(pb, rest, S + B0 + mine, lane), a0.load_rest(pa, rest, S + A0 + mine, lane);
    b1.load_rest(pb, rest, S + B1 + mine, lane), a1.load_rest(pa, rest, S + A1 + mine, lane);
    pa += 2 * rest * (TA ? A.ld : 1), pb += 2 * rest * (TB ? B.ld : 1);
  } else {
    b0.load(pb, bytes, S + B0 + mine), a0.load(pa, bytes, S + A0 + mine), b1.load(pb, bytes, S + B1 + mine), a1.load(pa, bytes, S + A1 + mine);
    step_on();
  }
  b0.load(pb, bytes, S + ST + B0 + mine), a0.load(pa, bytes, S + ST + A0 + mine), b1.load(pb, bytes, S + ST + B1 + mine);
  const char *qa = pa;
  step_on();

  DirectPieces<4, TA> la;
  DirectPieces<2, TB> lb;
  la.set((wave & 1) * 64, lane), lb.set((wave >> 1) * 32, lane);
  bf16x8 a[4][2], bx[2][2], by[2][2], bz[2][2];
  auto multiply = [&](int ia, int jb, const bf16x8 (&b)[2][2]) {
    turn_over();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[4 * ia + i][2 * jb + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i][s], b[j][s], acc[4 * ia + i][2 * jb + j], 0, 0, 0);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (what this turn's place may be overwritten with waits for these reads)
    turn_over();
  };
  nt_arrive<6>();  // (the first stage is there)
  pieces_of(S + B0, lb, bx);
  nt_arrive<6>();
  if (group) __builtin_amdgcn_s_barrier();
  // A turn's own loads and those of the four before may be on their way; what the next turn reads was asked for before them.
  auto arrived = []() { asm volatile("s_waitcnt vmcnt(10)" ::: "memory"); };
  auto stage = [&](char *here, char *next, const bf16x8 (&b)[2][2], bf16x8 (&bn)[2][2]) {
    a1.load(qa, bytes, next + A1 + mine);
    pieces_of(here + A0, la, a);
    arrived();
    multiply(0, 0, b);
    b0.load(pb, bytes, here + B0 + mine);
    pieces_of(here + B1, lb, bz);
    arrived();
    multiply(0, 1, bz);
    a0.load(pa, bytes, here + A0 + mine);
    pieces_of(here + A1, la, a);
    arrived();
    multiply(1, 1, bz);
    b1.load(pb, bytes, here + B1 + mine);
    pieces_of(next + B0, lb, bn);
    arrived();
    multiply(1, 0, b);
    qa = pa;
    step_on();
  };
  for (int left = full + (rest > 0);;) {
    stage(S, S + ST, bx, by);
    if (--left == 0) break;
    stage(S + ST, S, by, bx);
    if (--left == 0) break;
  }
  if (!group) __builtin_amdgcn_s_barrier();
  nt_arrive<0>();
}

// 128 x 128 x 64, four wavefronts of 64 x 64, two workgroups a compute unit: for products that have too few wide tiles.
struct NarrowTile {
  static constexpr int BM = 128, BN = 128, THREADS = 256, I = 4, J = 2, EU = 2;
  static constexpr int HALF = 16384, STAGE = 2 * HALF, LDS = 2 * STAGE;
  __device__ static __forceinline__ int col(int wave, int lane, int i) { return (wave & 1) * 64 + i * 16 + 8 * (lane >> 5); }
  __device__ static __forceinline__ int row(int wave, int lane, int j) { return (wave >> 1) * 64 + j * 32 + (lane & 31); }
};
template <bool TA, bool TB>
__device__ __forceinline__ void direct_multiply(const NarrowTile &, const DirectRef &A, int M, int m0, const DirectRef &B, int N, int n0, int kbeg, int kend,
                                                char *S, floatx4 (&acc)[4][4]) {
  constexpr int PB = NarrowTile::HALF, ST = NarrowTile::STAGE;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = 4096 * wave;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  DirectSource<4, TA> sa;
  DirectSource<4, TB> sb;
  sa.set(A, 0, M - m0, 4 * wave, lane), sb.set(B, 0, N - n0, 4 * wave, lane);
  const char *pa = reinterpret_cast<const char *>(TA ? A.p + kbeg * A.ld + m0 : A.p + m0 * A.ld + kbeg);
  const char *pb = reinterpret_cast<const char *>(TB ? B.p + kbeg * B.ld + n0 : B.p + n0 * B.ld + kbeg);
  const long da = TA ? 128 * A.ld : 128, db = TB ? 128 * B.ld : 128;
  const int rest = (kend - kbeg) & 63;
  int full = (kend - kbeg) / 64;
  auto ask = [&](char *to) {
    sa.load(pa, 0xffffffffu, to + mine), sb.load(pb, 0xffffffffu, to + PB + mine);
    pa += da, pb += db, full--;
  };
  if (rest) {
    sa.load_rest(pa, rest, S + mine, lane), sb.load_rest(pb, rest, S + PB + mine, lane);
    pa += 2 * rest * (TA ? A.ld : 1), pb += 2 * rest * (TB ? B.ld : 1);
  } else {
    ask(S);
  }
  DirectPieces<4, TA> la;
  DirectPieces<4, TB> lb;
  la.set((wave & 1) * 64, lane), lb.set((wave >> 1) * 64, lane);
  char *here = S, *next = S + ST;
  for (;;) {
    nt_arrive<0>();
    const bool more = full > 0;
    if (more) ask(next);
    bf16x8 a[4][2], b[4][2];
    if constexpr (TA && !TB) {  // (those that the compiler waits for first)
      pieces_of(here + PB, lb, b);
      pieces_of(here, la, a);
    } else {
      pieces_of(here, la, a);
      pieces_of(here + PB, lb, b);
    }
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i][s], b[j][s], acc[i][j], 0, 0, 0);
    if (!more) break;
    char *t = here;
    here = next, next = t;
  }
  nt_arrive<0>();
}

// Eight neighbouring columns of a row from the accumulators of a block of sixteen columns and two of sixteen rows: lane l's are of row l % 32, columns 8 (l / 32) ..
__device__ __forceinline__ void eight_columns(const floatx4 &t, const floatx4 &u, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(t[e]), __float_as_uint(u[e]), false, false);
    v[e] = __uint_as_float(x[0]);
    v[4 + e] = __uint_as_float(x[1]);
  }
}

}  // namespace cavs
