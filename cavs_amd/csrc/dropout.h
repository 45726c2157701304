// Which elements a dropout keeps, from a counter-based generator: Philox4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) of
// seven rounds, the fewest its authors found to pass all their tests.  The key is the seed, the counter (column / 8, the row's id, step): its 128 bits are the
// draws of eight neighbouring columns, 16 bits each, so that a lane that holds eight values makes one.  An element stays if its draw is at least
// round(65536 p).  (With 32 bits a draw eight values would need two calls.  A wavefront's 512 values of bf16, read and written, are 110 ns of a compute unit's share of a
// copy's rate, 4.74 TB/s; a call is 14 products of 16 cycles and some 45 instructions of 4, 400 cycles of one of its four SIMDs, 45 ns.)
#pragma once
#include "rows8.h"

namespace cavs {

struct Mask {  // of a call
  unsigned k0, k1;
  unsigned long long step;
  const unsigned long long *word;
  const int *ids;
  unsigned t;
  float scale;
};

// false: p is not in [0, 1).  m null: nothing is dropped.
inline bool mask_of(const cavs_dropout_mask *m, Mask *o) {
  *o = Mask{0, 0, 0, nullptr, nullptr, 0, 1.f};
  if (!m) return true;
  if (!(m->p >= 0.f && m->p < 1.f)) return false;
  const int t = (int)((double)m->p * 65536. + 0.5);
  o->t = t > 65535 ? 65535 : t;
  o->scale = (float)(65536. / (65536 - (int)o->t));
  o->k0 = (unsigned)m->seed, o->k1 = (unsigned)(m->seed >> 32);
  o->step = m->step, o->word = m->step_word, o->ids = m->ids;
  return true;
}

__device__ __forceinline__ unsigned long long step_of(const Mask &m) { return m.word ? m.step + *m.word : m.step; }
__device__ __forceinline__ unsigned row_id(const Mask &m, int row) { return m.ids ? (unsigned)m.ids[row] : (unsigned)row; }

struct Draws {
  unsigned w[4];
  __device__ __forceinline__ unsigned operator[](int e) const { return e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu; }
};
__device__ __forceinline__ Draws draws_of(const Mask &m, unsigned long long step, unsigned row, unsigned block) {
  unsigned c0 = block, c1 = row, c2 = (unsigned)step, c3 = (unsigned)(step >> 32), k0 = m.k0, k1 = m.k1;
#pragma unroll
  for (int r = 0; r < 7; r++) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(b >> 32) ^ c1 ^ k0, c1 = (unsigned)b;
    c2 = (unsigned)(a >> 32) ^ c3 ^ k1, c3 = (unsigned)a;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return Draws{{c0, c1, c2, c3}};
}
// what is dropped becomes 0, whatever it was
__device__ __forceinline__ void drop8(const Mask &m, const Draws &d, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = d[e] >= m.t ? v[e] * m.scale : 0.f;
}

}  // namespace cavs
