// Products C = A B^T of operands laid out for the bf16 matrix pipe: `P` planes of bf16, k-contiguous.
//
// An operand of type bf16 is one plane.  A float is the sum of bf16 parts, h = bf16(x), m = bf16(x - h), l = bf16(x - h - m); three of
// them hold all its bits, two hold 16.  A product of operands of P parts adds up the P (P + 1) / 2 products of weight 2^-8(P-1) and
// above: six of nine, three of four.  The products of the first parts go into one set of accumulators and all the others, a 2^-8
// smaller, into a second: the pipe loses an addend of less than about an eighth of its accumulator's last place, and beside their own
// kind the small ones are not lost.  (gemm_split.h splits on the way into LDS; here whoever makes an operand writes its
// planes, as the same operand goes into several products, and a tile's loads go to LDS without passing through registers.)
//
// Planes are zero from K up to `ld`, a multiple of 64: the loops below know no k that is not there.  Rows beyond the last read the last
// one again; what comes of them is not stored.
#pragma once
#include "gemm_common.h"

namespace cavs {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16;

constexpr int kPlaneAlign = 64;  // of K, in elements

struct PlanesRef {
  const u16 *p;
  long plane;  // elements from one plane to the next
  int ld;      // of a row: a multiple of kPlaneAlign
};

// bf16 of a float (to nearest), its bits
__device__ inline u16 bf16_bits(float x) { return __builtin_bit_cast(u16, (__bf16)x); }
__device__ inline float bf16_float(u16 b) { return __uint_as_float((unsigned)b << 16); }

// The parts of x.  Where x has no part (an infinity, a NaN, a finite value that rounds to infinity) the first is what bf16 makes of it and
// the others are zero.
template <int P>
__device__ inline void parts_of(float x, u16 (&o)[P]) {
  o[0] = bf16_bits(x);
  if constexpr (P > 1) {
    float rest = x - bf16_float(o[0]);
    if (!(fabsf(rest) < INFINITY)) rest = 0.f;
#pragma unroll
    for (int p = 1; p < P; p++) {
      o[p] = bf16_bits(rest);
      rest -= bf16_float(o[p]);
    }
  }
}

template <int P_, int BM_, int BN_, int BK_, int WGM_, int WGN_>
struct NtTile {
  static constexpr int P = P_, BM = BM_, BN = BN_, BK = BK_, WGM = WGM_, WGN = WGN_;
  static constexpr int WAVES = WGM * WGN, THREADS = 64 * WAVES;
  static constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 32, TN = WN / 32;
  static constexpr int ROWB = 2 * BK, PPR = BK / 8;           // bytes of a row of a tile, 16-byte pieces of it
  static constexpr int RPC = 1024 / ROWB;                     // rows a wavefront loads with one instruction
  static constexpr int CA = BM / RPC / WAVES, CB = BN / RPC / WAVES;  // such instructions per wavefront, plane and operand
  static constexpr int PA = BM * ROWB, PB = BN * ROWB, STAGE = P * (PA + PB), LDS = 2 * STAGE;
  static constexpr int ACC = P > 1 ? 2 : 1;
  static constexpr int EU = THREADS == 512 || WM == 64 ? 2 : P == 1 ? 4 : 3;  // wavefronts a SIMD is to hold: what LDS has room for
  static_assert(BM % (RPC * WAVES) == 0 && BN % (RPC * WAVES) == 0, "a tile's loads are the same for every wavefront");
  static_assert(kPlaneAlign % BK == 0, "planes end on a step");
};

// Byte of a tile's row x where its piece `oct` (8 k) lies: pieces change places so that sixteen rows read at one k touch all banks once.
template <class T>
__device__ inline int nt_at(int x, int oct) {
  return x * T::ROWB + ((oct ^ ((x * T::ROWB >> 8) & (T::PPR - 1))) << 4);
}

// acc[ACC][TM][TN] of the tile at rows m0 of A and n0 of B over k in [kbeg, kend), both multiples of BK.  S: T::LDS bytes.
// Two stages: while one is multiplied the other is on its way from memory; a step's one barrier says that the stage to come has arrived
// and that nobody reads the one before it any more.
template <class T>
__device__ __forceinline__ void nt_multiply(const PlanesRef &A, int M, int m0, const PlanesRef &B, int N, int n0, int kbeg, int kend, char *S,
                                            floatx16 (&acc)[T::ACC][T::TM][T::TN]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WGN, wn = wave % T::WGN;
  static_assert((32 * T::ROWB >> 8) % T::PPR == 0, "");
#pragma unroll
  for (int s = 0; s < T::ACC; s++)
#pragma unroll
    for (int i = 0; i < T::TM; i++)
#pragma unroll
      for (int j = 0; j < T::TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[s][i][j][r] = 0.f;

  // what this lane loads: piece lane % PPR of row lane / PPR of a wavefront's stretch of rows, as it lies in LDS
  int va[T::CA], vb[T::CB];
  auto offset = [&](int x, int x0, int X, int ld) {
    const int piece = (lane % T::PPR) ^ ((x * T::ROWB >> 8) & (T::PPR - 1));
    return (int)((unsigned)min(x, X - 1 - x0) * (unsigned)ld * 2u) + 16 * piece;
  };
#pragma unroll
  for (int c = 0; c < T::CA; c++) va[c] = offset((c * T::WAVES + wave) * T::RPC + lane / T::PPR, m0, M, A.ld);
#pragma unroll
  for (int c = 0; c < T::CB; c++) vb[c] = offset((c * T::WAVES + wave) * T::RPC + lane / T::PPR, n0, N, B.ld);
  [[maybe_unused]] const u16 *pa = A.p + (long)m0 * A.ld + kbeg, *pb = B.p + (long)n0 * B.ld + kbeg;

  auto fetch = [&](int kt, char *to) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass knows no such load)
    const unsigned off = (unsigned)kt * T::ROWB;
#pragma unroll
    for (int p = 0; p < T::P; p++) {
      const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<u16 *>(pa + p * A.plane), 0, 0xffffffffu, 0x00020000);
      const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<u16 *>(pb + p * B.plane), 0, 0xffffffffu, 0x00020000);
#pragma unroll
      for (int c = 0; c < T::CA; c++)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void *)(to + p * (T::PA + T::PB) + (c * T::WAVES + wave) * 1024), 16,
                                                 va[c], off, 0, 0);
#pragma unroll
      for (int c = 0; c < T::CB; c++)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (__attribute__((address_space(3))) void *)(to + p * (T::PA + T::PB) + T::PA + (c * T::WAVES + wave) * 1024),
                                                 16, vb[c], off, 0, 0);
    }
#endif
  };
  // where this lane's first piece of either operand lies; that of step s is at the address with s in its bits 5 and up (rows are
  // multiples of ROWB, their order of pieces repeats within 32 rows)
  const int half = lane >> 5, a0 = nt_at<T>(wm * T::WM + (lane & 31), half), b0 = T::PA + nt_at<T>(wn * T::WN + (lane & 31), half);
  auto multiply = [&](const char *from) {
#pragma unroll
    for (int s = 0; s < T::BK / 16; s++) {
      bf16x8 a[T::TM][T::P], b[T::TN][T::P];
#pragma unroll
      for (int p = 0; p < T::P; p++) {
#pragma unroll
        for (int i = 0; i < T::TM; i++) a[i][p] = *reinterpret_cast<const bf16x8 *>(from + (a0 ^ (32 * s)) + (p * (T::PA + T::PB) + 32 * i * T::ROWB));
#pragma unroll
        for (int j = 0; j < T::TN; j++) b[j][p] = *reinterpret_cast<const bf16x8 *>(from + (b0 ^ (32 * s)) + (p * (T::PA + T::PB) + 32 * j * T::ROWB));
      }
#pragma unroll
      for (int w = T::P - 1; w >= 0; w--)  // the parts' weights, the small products first
#pragma unroll
        for (int p = 0; p <= w; p++)
#pragma unroll
          for (int i = 0; i < T::TM; i++)
#pragma unroll
            for (int j = 0; j < T::TN; j++)
              acc[w ? T::ACC - 1 : 0][i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i][p], b[j][w - p], acc[w ? T::ACC - 1 : 0][i][j], 0, 0, 0);
    }
  };
  const int nk = (kend - kbeg) / T::BK;
  if (nk > 0) fetch(0, S);
  int at = 0;
  for (int kt = 0; kt < nk; kt++) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (a barrier by itself need not wait for loads that go to LDS)
    __syncthreads();
    if (kt + 1 < nk) fetch(kt + 1, S + (T::STAGE - at));
    multiply(S + at);
    at = T::STAGE - at;
  }
  __syncthreads();  // (LDS is free for what follows)
}

// The tiles of a launch over tilesM x tilesN: eight tiles of A at a time, down each tile of B, the tiles that one XCD runs together reading
// few panels of either operand.
__device__ inline void nt_tile_of(int block, int tilesM, int tilesN, int *tm, int *tn) {
  const int t = xcd_remap(block, tilesM * tilesN);
  const int band = t / (8 * tilesN), in = t - band * 8 * tilesN, high = min(8, tilesM - 8 * band);
  *tm = 8 * band + in % high;
  *tn = in / high;
}

// Four neighbouring values of a row: x[0..3] to o[0..3], `left` of them (4 or more: all), as one store where the row allows it.
__device__ inline void store4(float *o, const float (&x)[4], int left, bool vec) {
  if (vec && left >= 4) {
    *reinterpret_cast<float4 *>(o) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (k < left) o[k] = x[k];
  }
}
__device__ inline void store4(u16 *o, const float (&x)[4], int left, bool vec) {
  const u16 a = bf16_bits(x[0]), b = bf16_bits(x[1]), c = bf16_bits(x[2]), d = bf16_bits(x[3]);
  if (vec && left >= 4) {
    *reinterpret_cast<uint2 *>(o) = make_uint2(a | (unsigned)b << 16, c | (unsigned)d << 16);
  } else {
    if (left > 0) o[0] = a;
    if (left > 1) o[1] = b;
    if (left > 2) o[2] = c;
    if (left > 3) o[3] = d;
  }
}

// an operand's element as a float
__device__ inline float value_of(const float *p) { return *p; }
__device__ inline float value_of(const u16 *p) { return bf16_float(*p); }

constexpr int ceil_to(int x, int to) { return (x + to - 1) / to * to; }

}  // namespace cavs
