// Eight neighbouring values of a row, fp32 or bf16, as floats.  Rows begin anywhere their type may: the vector loads and stores ask for no more alignment than
// an element has (global memory takes them so), and a row's end goes value by value.
#pragma once
#include "common.h"

namespace cavs {

typedef unsigned short u16;

// the offsets that a grid of `threads` threads a workgroup may have along x: threads of a dimension are to be below 2^32
constexpr unsigned most_groups(unsigned threads) { return 0xffffffffu / threads; }

__device__ __forceinline__ float from_bits16(unsigned b) { return __uint_as_float(b << 16); }
__device__ __forceinline__ unsigned to_bits16(float x) { return __builtin_bit_cast(u16, (__bf16)x); }

// A type's eight values as they lie: a load that is not waited for until they are looked at.
template <class T>
struct Eight;
template <>
struct Eight<float> {
  typedef float four __attribute__((ext_vector_type(4), aligned(4)));
  four a, b;
  __device__ __forceinline__ void load(const float *p) {
    a = *reinterpret_cast<const four *>(p);
    b = *reinterpret_cast<const four *>(p + 4);
  }
  __device__ __forceinline__ void load(const float *p, int count) {
    if (count >= 8) return load(p);
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] = e < count ? p[e] : 0.f, b[e] = 4 + e < count ? p[4 + e] : 0.f;
  }
  __device__ __forceinline__ void zero() { a = 0.f, b = 0.f; }
  __device__ __forceinline__ float operator[](int e) const { return e < 4 ? a[e] : b[e - 4]; }
  __device__ __forceinline__ static void store(float *p, const float (&v)[8], int count) {
    if (count >= 8) {
      *reinterpret_cast<four *>(p) = four{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<four *>(p + 4) = four{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e < count) p[e] = v[e];
    }
  }
};
template <>
struct Eight<u16> {
  typedef unsigned four __attribute__((ext_vector_type(4), aligned(2)));
  four a;
  __device__ __forceinline__ void load(const u16 *p) { a = *reinterpret_cast<const four *>(p); }
  __device__ __forceinline__ void load(const u16 *p, int count) {
    if (count >= 8) return load(p);
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] = (2 * e < count ? p[2 * e] : 0u) | (2 * e + 1 < count ? (unsigned)p[2 * e + 1] << 16 : 0u);
  }
  __device__ __forceinline__ void zero() { a = 0u; }
  __device__ __forceinline__ float operator[](int e) const { return e & 1 ? __uint_as_float(a[e >> 1] & 0xffff0000u) : __uint_as_float(a[e >> 1] << 16); }
  __device__ __forceinline__ static void store(u16 *p, const float (&v)[8], int count) {
    if (count >= 8) {
      four o;
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = to_bits16(v[2 * e]) | to_bits16(v[2 * e + 1]) << 16;
      *reinterpret_cast<four *>(p) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e < count) p[e] = to_bits16(v[e]);
    }
  }
};

}  // namespace cavs
