// Norms after and before a block, with its gate and residual scale:
//   z = post(y),  s = r + scale gate . z,  x = pre(s)
// where a norm of v [w] is nothing, (v / sqrt(mean v^2 + eps)) weight + bias, or ((v - mean v) / sqrt(var v + eps)) weight + bias.  With v^ what is between
// the brackets, h = d x . weight and D = d s + the gradient that comes through x:
//   D = d s + rstd (h - [mean h] - s^ mean(h s^)),  d r = D,  d gate = scale z D,  d z = scale gate . D,  d y from d z as D from d x,
//   d weight = sum over rows of d x . v^,  d bias = sum over rows of d x
//
// A row is held by L lanes, eight neighbouring values of each in registers, so that memory is read and written once.  The sums of a row are made in 64
// bits: of values and squares at once (mean and variance from one trip across the lanes; a mean of 2^13 deviations costs nothing, beyond that 1 / deviation is off by
// 2^-52 (mean / deviation)^2 of it, 2^-12 at 2^20), and squares of any float fit.  Bound by HBM, of few rows by the trips across the lanes: fp32 7088 x 512 forward 11.5 us, 5.0 TB/s; bf16 gradients of 16384 x 4096 169, 4.8 TB/s, arithmetic 64 %
// busy; fp32 gradients of 2371 x 1001 with everything 25, 3.0 TB/s (198 workgroups of three turns, and a launch for the sums).
#include <cmath>
#include <type_traits>

#include "rows8.h"

namespace cavs {
namespace {

constexpr int kMostW = 16384;

struct Norm {  // as cavs_norm_desc
  int n, w;
  const void *y, *r, *gate_rows;
  long ldy, ldr, ldg;
  const float *gate;
  float scale, eps;
  int post, pre;
  const float *post_w, *post_b, *pre_w, *pre_b;
};

// ------------------------------------------------------------------ sums over the lanes of a row
__device__ __forceinline__ double two(unsigned lo, unsigned hi) { return __longlong_as_double((long long)((unsigned long long)hi << 32 | lo)); }
template <int CTRL>
__device__ __forceinline__ double moved(double v) {
  const int lo = __double2loint(v), hi = __double2hiint(v);
  return two(__builtin_amdgcn_update_dpp(0, lo, CTRL, 0xf, 0xf, true), __builtin_amdgcn_update_dpp(0, hi, CTRL, 0xf, 0xf, true));
}
// of lanes 32 or 16 apart: v's in the lower half (the even rows of sixteen), w's in the upper
__device__ __forceinline__ double crossed32(double v, double w) {
  const auto a = __builtin_amdgcn_permlane32_swap(__double2loint(v), __double2loint(w), false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(__double2hiint(v), __double2hiint(w), false, false);
  return two(a[0], b[0]) + two(a[1], b[1]);
}
__device__ __forceinline__ double crossed16(double v, double w) {
  const auto a = __builtin_amdgcn_permlane16_swap(__double2loint(v), __double2loint(w), false, false);
  const auto b = __builtin_amdgcn_permlane16_swap(__double2hiint(v), __double2hiint(w), false, false);
  return two(a[0], b[0]) + two(a[1], b[1]);
}
// over N neighbouring lanes, N up to 16, every lane with the result: its neighbour, the pair beside, the four, the eight
template <int N>
__device__ __forceinline__ double near_sum(double v) {
  if constexpr (N >= 2) v += moved<0xb1>(v);    // quad_perm 1 0 3 2
  if constexpr (N >= 4) v += moved<0x4e>(v);    // quad_perm 2 3 0 1
  if constexpr (N >= 8) v += moved<0x141>(v);   // row_half_mirror
  if constexpr (N >= 16) v += moved<0x140>(v);  // row_mirror
  return v;
}
__device__ __forceinline__ double of_lane(double v, int lane) {
  return two(__builtin_amdgcn_readlane(__double2loint(v), lane), __builtin_amdgcn_readlane(__double2hiint(v), lane));
}
// K sums of the L lanes of a row, every lane with the results.  Of a wavefront up to four sums go down together, a quarter of the lanes to each (crossed),
// so that they cost one sum's trip.  L above 64: `lds` [groups of the workgroup][K][L / 64], which may be written again after the next barrier but one.
template <int L, int K>
__device__ __forceinline__ void row_sums(double (&v)[K], double *lds) {
  if constexpr (L < 64) {
#pragma unroll
    for (int k = 0; k < K; k++) {
      if constexpr (L == 32) v[k] = crossed16(v[k], v[k]);
      v[k] = near_sum<16>(v[k]);
    }
  } else {
    constexpr int Q = (K + 3) / 4;
    double t[Q];
#pragma unroll
    for (int q = 0; q < Q; q++) {
      const int k = 4 * q;
      const double a = crossed32(v[k], k + 1 < K ? v[k + 1 < K ? k + 1 : 0] : 0.), b = k + 2 < K ? crossed32(v[k + 2 < K ? k + 2 : 0], k + 3 < K ? v[k + 3 < K ? k + 3 : 0] : 0.) : 0.;
      t[q] = near_sum<16>(crossed16(a, b));  // (of sums k, k + 2, k + 1, k + 3: rows of sixteen 0 .. 3)
    }
    if constexpr (L == 64) {
#pragma unroll
      for (int k = 0; k < K; k++) v[k] = of_lane(t[k / 4], 16 * ((k & 1) * 2 + (k >> 1 & 1)));
    } else {
      constexpr int W = L / 64;
      const int lane = threadIdx.x & 63, wave = threadIdx.x % L / 64, at = (lane >> 5) + (lane >> 4 & 1) * 2;
      lds += threadIdx.x / L * (K * W);
#pragma unroll
      for (int q = 0; q < Q; q++)
        if ((lane & 15) == 0 && 4 * q + at < K) lds[(4 * q + at) * W + wave] = t[q];
      __syncthreads();
      // lane l: of sum l / W the part of wavefront l % W
      constexpr int ROUNDS = (K * W + 63) / 64;
#pragma unroll
      for (int r = 0; r < ROUNDS; r++) {
        const int i = r * 64 + lane;
        const double x = near_sum<W>(i < K * W ? lds[i] : 0.);
#pragma unroll
        for (int k = 0; k < 64 / W; k++)
          if (r * (64 / W) + k < K) v[r * (64 / W) + k] = of_lane(x, k * W);
      }
    }
  }
}

// v^ = ((v - mean) - rest) rstd: mean as a float and what it leaves off, so that the difference is a float's own however far the values are from 0; in quarters, as a
// difference may be twice the largest float, and 1 / deviation of the largest is no normal one.  Where nothing is centred: v rstd (bf16 gradients of 16384 x 4096 with
// norms on both sides 168 us, in quarters 170).
struct Stats {
  float mean, rest, rstd4;  // a quarter of the mean, 4 / deviation
  float rstd;
  __device__ __forceinline__ void of(double sum, double squares, int w, bool centred, float eps) {
    const double inv = 1. / w, m = centred ? sum * inv : 0., v = squares * inv - m * m;
    mean = (float)(0.25 * m);
    rest = (float)(0.25 * m - (double)mean);
    const double a = (v > 0. ? v : v == v ? 0. : v) + (double)eps;
    const double y = __builtin_amdgcn_rsq(a);  // (2^-23, and a step of Newton's makes 2^-45 of it)
    const double z = y * (1.5 - 0.5 * a * y * y);
    rstd = (float)z;
    rstd4 = (float)(4. * z);
  }
  template <bool CENTRED = true>
  __device__ __forceinline__ float hat(float v) const { return CENTRED ? (fmaf(v, 0.25f, -mean) - rest) * rstd4 : v * rstd; }
};

template <int L>
constexpr int threads_of() { return L > 256 ? L : 256; }
template <int L>
constexpr int sums_lds(int k) { return L > 64 ? k * threads_of<L>() / 64 : 1; }

// A lane's eight columns.  Of the last piece of a row that is no multiple of eight they are the row's last eight, `skip` of which are the lane's before it: a load is
// always whole and none waits for another (with its end value by value, each array of a row waited for the one before: d of 16384 x 4096 with norms on
// both sides 272 us, without that wait 180).  SMALL: rows of less than eight values.
template <bool SMALL>
struct Place {
  int col, skip, w;
  __device__ __forceinline__ void set(int c, int width) {
    w = width;
    col = SMALL ? c : min(c, w - 8);
    skip = SMALL ? (c < w ? 0 : 8) : c - col;
  }
  __device__ __forceinline__ bool has(int e) const { return SMALL ? col + e < w : e >= skip; }
  template <class T>
  __device__ __forceinline__ void load(Eight<T> &o, const T *row) const {
    if constexpr (SMALL) o.load(row + col, w - col);
    else o.load(row + col);
  }
  template <class T>
  __device__ __forceinline__ void store(T *row, const float (&v)[8]) const {
    if (!SMALL && skip == 0) {
      Eight<T>::store(row + col, v, 8);
    } else if (skip < 8) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (has(e)) row[col + e] = as<T>(v[e]);
    }
  }
  template <class T>
  __device__ __forceinline__ static T as(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return (u16)to_bits16(v);
  }
  // weights; 0 where a column is not this lane's
  __device__ __forceinline__ void weights(float (&o)[8], const float *p, float none) const {
    Eight<float> t;
    if (p) load(t, p);
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] = !has(e) ? 0.f : p ? t[e] : none;
  }
};

// ------------------------------------------------------------------ forward
template <class T, int L, int V, bool SMALL>
__global__ __launch_bounds__(threads_of<L>()) void norm_fwd_kernel(Norm a, T *s, long lds_, T *x, long ldx) {
  __shared__ double part[2][sums_lds<L>(2)];
  const int lane = threadIdx.x % L, at = blockIdx.x * (threads_of<L>() / L) + threadIdx.x / L, row = min(at, a.n - 1);
  const bool on = at < a.n;  // (rows of more than a wavefront's lanes go through the barriers together)
  Place<SMALL> c[V];
  float v[V][8];
  Eight<T> y[V], r[V], g[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    c[i].set(8 * (i * L + lane), a.w);
    c[i].load(y[i], static_cast<const T *>(a.y) + row * a.ldy);
    r[i].zero(), g[i].zero();
  }
  if (a.r) {
#pragma unroll
    for (int i = 0; i < V; i++) c[i].load(r[i], static_cast<const T *>(a.r) + row * a.ldr);
  }
  if (a.gate_rows) {
#pragma unroll
    for (int i = 0; i < V; i++) c[i].load(g[i], static_cast<const T *>(a.gate_rows) + row * a.ldg);
  }
  auto stats = [&](int kind, double *lds) {
    double t[2] = {0., 0.};
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) t[0] += v[i][e], t[1] += (double)v[i][e] * v[i][e];
    row_sums<L>(t, lds);
    Stats o;
    o.of(t[0], t[1], a.w, kind == CAVS_NORM_LAYER, a.eps);
    return o;
  };
#pragma unroll
  for (int i = 0; i < V; i++)
#pragma unroll
    for (int e = 0; e < 8; e++) v[i][e] = c[i].has(e) ? y[i][e] : 0.f;
  Stats post{}, pre{};
  if (a.post) post = stats(a.post, part[0]);
#pragma unroll
  for (int i = 0; i < V; i++) {
    float w[8], b[8];
    if (a.post) {
      c[i].weights(w, a.post_w, 1.f), c[i].weights(b, a.post_b, 0.f);
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = post.hat(v[i][e]) * w[e] + b[e];
    }
    if (a.gate_rows) {
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = g[i][e];
    } else {
      c[i].weights(w, a.gate, 1.f);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) v[i][e] = c[i].has(e) ? v[i][e] * (a.scale * w[e]) + r[i][e] : 0.f;
    if (s && on) c[i].store(s + row * lds_, v[i]);
  }
  if (!x) return;
  if (a.pre) pre = stats(a.pre, part[1]);
#pragma unroll
  for (int i = 0; i < V; i++) {
    float w[8], b[8];
    if (a.pre) {
      c[i].weights(w, a.pre_w, 1.f), c[i].weights(b, a.pre_b, 0.f);
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = pre.hat(v[i][e]) * w[e] + b[e];
    }
    if (on) c[i].store(x + row * ldx, v[i]);
  }
}

// ------------------------------------------------------------------ backward
struct Back {
  const void *s, *ds, *dx;
  long lds, ldds, lddx;
  void *dy, *dr, *dg;
  long lddy, lddr, lddg;
  float *part;  // [workgroups][sums][w]: pre_w, gate, (POST) post_w, (FULL) pre_b, (both) post_b; null: none wanted
};

// A workgroup takes every gridDim.x-th row (group of rows), its lanes the same columns of each: the sums over rows are in registers until it ends. The weights
// are in LDS (of the widest rows in memory), which leaves registers for two workgroups of 512 a compute unit where there are no more than the sums below:
// while one waits for a row's sums the other has its loads on their way.
// what is summed over rows: weights of both norms and the gate, and (FULL) biases.  FULL is for norms that take the mean off, or gradients of biases; what they need
// besides of a row's sums and of registers is left out otherwise (rms norms on both sides, bf16 16384 x 4096 with / without it
// 260 / 221 us, and 180 with two workgroups a compute unit then).
constexpr int back_sums(bool post, bool full) { return full ? (post ? 5 : 3) : (post ? 3 : 2); }
// One workgroup of 512 a compute unit, with the registers to have its next row on the way while it computes this one, where what it computes leaves no room for two:
// us of two / of one so: norms on both sides, fp32 2371 x 1001 with biases 41 / 26, bf16 32768 x 512 without 51 / 44; 16384 x 4096 without 180 / 221.
constexpr bool back_ahead(int lanes, bool post, bool full) { return post && lanes <= 512 && (full || lanes <= 64); }
template <int L>
constexpr int back_threads() { return L > 512 ? L : 512; }

template <class T, int L, int V, bool POST, bool FULL, bool SMALL>
__global__ __launch_bounds__(back_threads<L>(), back_ahead(L, POST, FULL) ? 2 : 4) void norm_bwd_kernel(Norm a, Back b) {
  typedef float four __attribute__((ext_vector_type(4)));
  constexpr int THREADS = back_threads<L>(), G = THREADS / L, S = back_sums(POST, FULL), WAVES = L > 64 ? THREADS / 64 : 1, KINDS = POST ? 4 : 2;
  constexpr int PRE_W = 0, GATE = 1, POST_W = 2, PRE_B = POST ? 3 : 2, POST_B = 4;  // of the sums over rows
  constexpr int SS = 0, HS = 1, YY = 2, S1 = POST ? 3 : 2, H1 = S1 + 1, Y1 = H1 + 1, K = FULL ? (POST ? 6 : 4) : (POST ? 3 : 2);  // of those of a row
  constexpr bool KEPT = V == 1, AHEAD = back_ahead(L, POST, FULL);
  __shared__ double part[2][K * WAVES];
  __shared__ four kept[KEPT ? KINDS : 1][2][KEPT ? L : 1];  // pre_w, gate, post_w, post_b
  __shared__ float merged[G > 1 ? (G - 1) * 8 * L * V : 1];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  Place<SMALL> c[V];
#pragma unroll
  for (int i = 0; i < V; i++) c[i].set(8 * (i * L + lane), a.w);
  auto weights = [&](int kind, int i, float (&o)[8]) {
    if constexpr (KEPT) {
      const four lo = kept[kind][0][lane], hi = kept[kind][1][lane];
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = lo[e], o[4 + e] = hi[e];
    } else {
      c[i].weights(o, kind == 0 ? a.pre_w : kind == 1 ? a.gate : kind == 2 ? a.post_w : a.post_b, kind == 3 ? 0.f : 1.f);
    }
  };
  if constexpr (KEPT) {
    for (int k = group; k < KINDS; k += G) {
      float o[8];
      c[0].weights(o, k == 0 ? a.pre_w : k == 1 ? a.gate : k == 2 ? a.post_w : a.post_b, k == 3 ? 0.f : 1.f);
      kept[k][0][lane] = four{o[0], o[1], o[2], o[3]}, kept[k][1][lane] = four{o[4], o[5], o[6], o[7]};
    }
    __syncthreads();
  }
  float acc[S][V][8];
#pragma unroll
  for (int k = 0; k < S; k++)
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) acc[k][i][e] = 0.f;
  const double inv = 1. / a.w;
  const bool whole = a.w == 8 * L * V;
  int turn = 0;
  struct Row {
    Eight<T> s[V], ds[V], dx[V], y[V], g[V];
  } now;
  auto fetch = [&](Row &o, int first) {
    const int row = min(first + group, a.n - 1);  // (a group without a row goes along with the last: nothing of it is stored or added)
#pragma unroll
    for (int i = 0; i < V; i++) o.s[i].zero(), o.ds[i].zero(), o.dx[i].zero(), o.y[i].zero(), o.g[i].zero();
    auto load = [&](Eight<T> (&to)[V], const void *p, long ld) {
      if (!p) return;
#pragma unroll
      for (int i = 0; i < V; i++) c[i].load(to[i], static_cast<const T *>(p) + row * ld);
    };
    load(o.s, a.pre ? b.s : nullptr, b.lds), load(o.dx, b.dx, b.lddx), load(o.y, a.y, a.ldy), load(o.ds, b.ds, b.ldds), load(o.g, a.gate_rows, a.ldg);
  };
  if constexpr (AHEAD) fetch(now, blockIdx.x * G);
  for (int first = blockIdx.x * G; first < a.n; first += gridDim.x * G, turn ^= 1) {
    const int row = min(first + group, a.n - 1);
    const bool on = first + group < a.n;
    Row next;
    if constexpr (AHEAD) fetch(next, min(first + (int)gridDim.x * G, a.n - 1));
    else fetch(now, first);
    const Eight<T>(&s)[V] = now.s, (&ds)[V] = now.ds, (&dx)[V] = now.dx, (&y)[V] = now.y, (&g)[V] = now.g;
    double t[K];
#pragma unroll
    for (int k = 0; k < K; k++) t[k] = 0.;
#pragma unroll
    for (int i = 0; i < V; i++) {
      float pw[8], sv[8], yv[8];
      weights(0, i, pw);
#pragma unroll
      for (int e = 0; e < 8; e++) sv[e] = s[i][e], yv[e] = y[i][e];
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (!c[i].has(e)) sv[e] = 0.f, yv[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const double v = sv[e];
        const float h = dx[i][e] * pw[e];
        t[SS] += v * v, t[HS] += h * v;
        if constexpr (FULL) t[S1] += v, t[H1] += h;
        if constexpr (POST) {
          const double u = yv[e];
          t[YY] += u * u;
          if constexpr (FULL) t[Y1] += u;
        }
      }
    }
    row_sums<L>(t, part[POST ? 0 : turn]);  // (of two calls a row, or one: never the place of the call before)
    Stats pre{0.f, 0.f, 4.f, 1.f}, post{};
    float h1 = 0.f, h2 = 0.f;  // means of h and of h s^ (no norm: s is 0 here, and D = ds + dx)
    const bool centred = FULL && a.pre == CAVS_NORM_LAYER, post_centred = FULL && POST && a.post == CAVS_NORM_LAYER;
    if (a.pre) {
      pre.of(centred ? t[FULL ? S1 : 0] : 0., t[SS], a.w, centred, a.eps);
      const double m = centred ? t[FULL ? S1 : 0] * inv : 0., hm = centred ? t[FULL ? H1 : 0] * inv : 0.;
      h1 = (float)hm;
      h2 = (float)((t[HS] * inv - m * hm) * pre.rstd);
    }
    if constexpr (POST) post.of(post_centred ? t[FULL ? Y1 : 0] : 0., t[YY], a.w, post_centred, a.eps);
    float dz[V][8];
    double q[FULL ? 2 : 1] = {};
#pragma unroll
    for (int i = 0; i < V; i++) {
      float w[8], D[8];
      weights(0, i, w);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float hat = pre.hat<FULL>(s[i][e]), d = dx[i][e];
        D[e] = ds[i][e] + pre.rstd * ((d * w[e] - h1) - hat * h2);
        if (on) {
          acc[PRE_W][i][e] += d * hat;
          if constexpr (FULL) acc[PRE_B][i][e] += d;
        }
      }
      if (b.dr && on) c[i].store(static_cast<T *>(b.dr) + row * b.lddr, D);
      if (a.gate_rows) {
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = g[i][e];
      } else {
        weights(1, i, w);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) D[e] *= a.scale, dz[i][e] = D[e] * w[e];
      if constexpr (POST) {
        float qb[8];
        weights(2, i, w), weights(3, i, qb);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float zh = post.hat<FULL>(y[i][e]);
          D[e] *= zh * w[e] + qb[e];
          if (on) {
            acc[POST_W][i][e] += dz[i][e] * zh;
            if constexpr (FULL) acc[POST_B][i][e] += dz[i][e];
          }
          dz[i][e] *= w[e];
          q[0] += (double)dz[i][e] * y[i][e];
          if constexpr (FULL) q[FULL ? 1 : 0] += dz[i][e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) D[e] *= y[i][e];
        if (b.dy && on) c[i].store(static_cast<T *>(b.dy) + row * b.lddy, dz[i]);
      }
      if (b.dg && on) c[i].store(static_cast<T *>(b.dg) + row * b.lddg, D);
      if (on) {
#pragma unroll
        for (int e = 0; e < 8; e++) acc[GATE][i][e] += D[e];
      }
    }
    if constexpr (POST) {
      row_sums<L>(q, part[1]);
      const double m = post_centred ? t[FULL ? Y1 : 0] * inv : 0., gm = post_centred ? q[FULL ? 1 : 0] * inv : 0.;
      const float g1 = (float)gm, g2 = (float)((q[0] * inv - m * gm) * post.rstd);
      if (b.dy && on) {
#pragma unroll
        for (int i = 0; i < V; i++) {
#pragma unroll
          for (int e = 0; e < 8; e++) dz[i][e] = post.rstd * ((dz[i][e] - g1) - post.hat<FULL>(y[i][e]) * g2);
          c[i].store(static_cast<T *>(b.dy) + row * b.lddy, dz[i]);
        }
      }
    }
    if constexpr (AHEAD) now = next;
  }
  if (!b.part) return;
#pragma unroll
  for (int k = 0; k < S; k++) {
    if constexpr (G > 1) {  // the groups of a workgroup in their order
      __syncthreads();
      if (group > 0) {
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) merged[((group - 1) * V * 8 + i * 8 + e) * L + lane] = acc[k][i][e];
      }
      __syncthreads();
      if (group > 0) continue;
#pragma unroll 1
      for (int q = 1; q < G; q++)
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) acc[k][i][e] += merged[((q - 1) * V * 8 + i * 8 + e) * L + lane];
    }
#pragma unroll
    for (int i = 0; i < V; i++) c[i].store(b.part + ((long)blockIdx.x * S + k) * a.w, acc[k][i]);
  }
}

// out[k][c] = the sum of the workgroups' parts, in their order: sixteen stretches of them side by side, 64 columns a workgroup
struct SumOut {
  float *o[5];
};
__global__ __launch_bounds__(1024) void norm_sums_kernel(const float *part, int groups, int sums, int w, SumOut out) {
  __shared__ float each[16][64];
  const int k = blockIdx.y, c = blockIdx.x * 64 + (threadIdx.x & 63), stretch = threadIdx.x >> 6;
  float *o = out.o[k];
  if (!o) return;
  const int per = (groups + 15) / 16, end = min(groups, (stretch + 1) * per);
  float s = 0.f;
  if (c < w) {
    for (int g = stretch * per; g < end; g += 8) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; q++) v[q] = g + q < end ? part[((long)(g + q) * sums + k) * w + c] : 0.f;
#pragma unroll
      for (int q = 0; q < 8; q++) s += v[q];
    }
  }
  each[stretch][threadIdx.x & 63] = s;
  __syncthreads();
  if (stretch || c >= w) return;
#pragma unroll
  for (int q = 1; q < 16; q++) s += each[q][threadIdx.x];
  o[c] = s;
}

// ------------------------------------------------------------------ what a call consists of
// lanes of a row: the fewest that hold it eight values each
template <class F>
int with_lanes(int w, F &&f) {
  if (w < 8) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{}, std::true_type{});
#define CAVS_NORM_LANES(L, V) \
  if (w <= 8 * L * V) return f(std::integral_constant<int, L>{}, std::integral_constant<int, V>{}, std::false_type{});
  CAVS_NORM_LANES(16, 1)
  CAVS_NORM_LANES(32, 1)
  CAVS_NORM_LANES(64, 1)
  CAVS_NORM_LANES(128, 1)
  CAVS_NORM_LANES(256, 1)
  CAVS_NORM_LANES(512, 1)
  CAVS_NORM_LANES(1024, 1)
  CAVS_NORM_LANES(1024, 2)
#undef CAVS_NORM_LANES
  return CAVS_EUNSUPPORTED;
}

// workgroups of the backward pass: what the compute units hold at once, each the same number of rows but for the last
int back_groups(int n, int w, bool post, bool full) {
  int groups = 0;
  with_lanes(w, [&](auto l, auto, auto) {
    constexpr int L = decltype(l)::value, T = back_threads<L>(), G = T / L;
    const long most = (back_ahead(L, post, full) ? 1 : 1024 / T) * num_cus(), wanted = (n + (long)G - 1) / G, turns = (wanted + most - 1) / most;
    groups = (int)((wanted + turns - 1) / turns);
    return CAVS_OK;
  });
  return groups;
}

template <class T>
int run_fwd(const Norm &a, void *s, int lds, void *x, int ldx, hipStream_t st) {
  return with_lanes(a.w, [&](auto l, auto v, auto small) {
    constexpr bool SMALL = decltype(small)::value;
    constexpr int L = decltype(l)::value, V = decltype(v)::value, G = threads_of<L>() / L;
    launch(norm_fwd_kernel<T, L, V, SMALL>, (unsigned)((a.n + (long)G - 1) / G), threads_of<L>(), 0, st, a, static_cast<T *>(s), (long)lds, static_cast<T *>(x), (long)ldx);
    CAVS_LAUNCH_CHECK();
    return (int)CAVS_OK;
  });
}

template <class T>
int run_bwd(const Norm &a, const Back &b, const SumOut &o, bool full, int groups, hipStream_t st) {
  return with_lanes(a.w, [&](auto l, auto v, auto small) {
    constexpr bool SMALL = decltype(small)::value;
    constexpr int L = decltype(l)::value, V = decltype(v)::value;
    const auto kernel = a.post ? (full ? norm_bwd_kernel<T, L, V, true, true, SMALL> : norm_bwd_kernel<T, L, V, true, false, SMALL>)
                               : (full ? norm_bwd_kernel<T, L, V, false, true, SMALL> : norm_bwd_kernel<T, L, V, false, false, SMALL>);
    launch(kernel, groups, back_threads<L>(), 0, st, a, b);
    CAVS_LAUNCH_CHECK();
    if (b.part) {
      const int sums = back_sums(a.post, full);
      launch(norm_sums_kernel, dim3((a.w + 63) / 64, sums), 1024, 0, st, b.part, groups, sums, a.w, o);
      CAVS_LAUNCH_CHECK();
    }
    return (int)CAVS_OK;
  });
}

__global__ void zeros_kernel(SumOut o, int w) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  for (int k = 0; k < 5; k++)
    if (o.o[k] && c < w) o.o[k][c] = 0.f;
}

int check(const char *who, int type, const cavs_norm_desc *d, Norm *o) {
  CAVS_REQUIRE(type == CAVS_F32 || type == CAVS_BF16, "%s: type %d is neither CAVS_F32 nor CAVS_BF16", who, type);
  CAVS_REQUIRE(d, "%s: null pointer", who);
  CAVS_REQUIRE(d->n >= 0 && d->w > 0, "%s: bad shape n=%d w=%d", who, d->n, d->w);
  CAVS_REQUIRE(d->w <= kMostW && d->n <= (int)most_groups(1024), "%s: unsupported shape n=%d w=%d (at most 2^22 - 1, 16384)", who, d->n, d->w);
  CAVS_REQUIRE(d->post >= CAVS_NORM_NONE && d->post <= CAVS_NORM_LAYER && d->pre >= CAVS_NORM_NONE && d->pre <= CAVS_NORM_LAYER, "%s: unknown norm", who);
  CAVS_REQUIRE((!d->y || d->ldy >= d->w) && (!d->r || d->ldr >= d->w) && (!d->gate_rows || d->ldg >= d->w), "%s: a row stride is below w=%d", who, d->w);
  CAVS_REQUIRE(!(d->gate && d->gate_rows), "%s: a gate is a row of values or a matrix, not both", who);
  CAVS_REQUIRE(d->eps > 0.f && d->eps < INFINITY, "%s: eps is not a positive number", who);
  *o = Norm{d->n, d->w, d->y, d->r, d->gate_rows, d->ldy, d->ldr, d->ldg, d->gate, d->scale, d->eps, d->post, d->pre, d->post_w, d->post_b, d->pre_w, d->pre_b};
  if (!o->post) o->post_w = o->post_b = nullptr;  // (a norm that is not there has no weights, whatever the descriptor holds)
  if (!o->pre) o->pre_w = o->pre_b = nullptr;
  return CAVS_OK;
}

}  // namespace
}  // namespace cavs

using namespace cavs;

extern "C" {

size_t cavs_norm_residual_workspace(int n, int w) {
  if (n <= 0 || w <= 0 || w > kMostW || n > (int)most_groups(1024)) return 0;
  return (size_t)back_groups(n, w, false, false) * 5 * w * 4;
}

int cavs_norm_residual_fwd(int type, const cavs_norm_desc *d, void *s, int lds, void *x, int ldx, void *stream) {
  const char *who = "cavs_norm_residual_fwd";
  Norm a;
  if (const int rc = check(who, type, d, &a)) return rc;
  CAVS_REQUIRE((!s || lds >= a.w) && (!x || ldx >= a.w), "%s: a row stride is below w=%d", who, a.w);
  CAVS_REQUIRE(s || x || a.n == 0, "%s: neither s nor x is wanted", who);
  if (a.n == 0) return CAVS_OK;
  CAVS_REQUIRE(a.y, "%s: null pointer", who);
  return (type == CAVS_F32 ? run_fwd<float> : run_fwd<u16>)(a, s, lds, x, ldx, as_stream(stream));
}

int cavs_norm_residual_bwd(int type, const cavs_norm_desc *d, const void *s, int lds, const void *ds, int ldds, const void *dx, int lddx,
                           const cavs_norm_grads *g, void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "cavs_norm_residual_bwd";
  Norm a;
  if (const int rc = check(who, type, d, &a)) return rc;
  CAVS_REQUIRE(g, "%s: null pointer", who);
  CAVS_REQUIRE((!s || lds >= a.w) && (!ds || ldds >= a.w) && (!dx || lddx >= a.w) && (!g->dy || g->lddy >= a.w) && (!g->dr || g->lddr >= a.w) &&
                   (!g->dgate_rows || g->lddg >= a.w),
               "%s: a row stride is below w=%d", who, a.w);
  CAVS_REQUIRE(a.pre || (!g->dpre_w && !g->dpre_b), "%s: gradients of a norm that is not there", who);
  CAVS_REQUIRE(a.post || (!g->dpost_w && !g->dpost_b), "%s: gradients of a norm that is not there", who);
  CAVS_REQUIRE((a.gate || !g->dgate) && (a.gate_rows || !g->dgate_rows), "%s: gradients of a gate that is not there", who);
  SumOut o{{g->dpre_w, g->dgate, g->dpost_w, g->dpre_b, g->dpost_b}};
  const bool sums = g->dpre_w || g->dpre_b || g->dgate || g->dpost_w || g->dpost_b;
  hipStream_t st = as_stream(stream);
  if (a.n == 0) {  // sums over no rows
    if (sums) {
      launch(zeros_kernel, (a.w + 255) / 256, 256, 0, st, o, a.w);
      CAVS_LAUNCH_CHECK();
    }
    return CAVS_OK;
  }
  CAVS_REQUIRE(ds || dx, "%s: neither ds nor dx is given", who);
  CAVS_REQUIRE(!a.pre || s || !dx, "%s: null pointer", who);
  if (!g->dy && !g->dgate && !g->dgate_rows && !g->dpost_w && !g->dpost_b) a.post = CAVS_NORM_NONE;  // (nothing behind it is wanted)
  const bool needs_y = g->dgate || g->dgate_rows || a.post;
  CAVS_REQUIRE(!needs_y || a.y, "%s: null pointer", who);
  if (!dx) a.pre = CAVS_NORM_NONE, a.pre_w = nullptr;  // (nothing comes through it)
  if (!a.post) o.o[2] = o.o[3], o.o[3] = o.o[4] = nullptr;  // (in the order of the sums there are)
  const bool full = a.pre == CAVS_NORM_LAYER || a.post == CAVS_NORM_LAYER || g->dpre_b || g->dpost_b;
  const int groups = back_groups(a.n, a.w, a.post, full);
  Back b{s, ds, dx, lds, ldds, lddx, g->dy, g->dr, g->dgate_rows, g->lddy, g->lddr, g->lddg, nullptr};
  if (!needs_y) a.y = nullptr;  // (not read)
  if (sums) {
    CAVS_REQUIRE(workspace && workspace_bytes >= (size_t)groups * 5 * a.w * 4, "%s: workspace of %zu bytes needed, %zu given", who, (size_t)groups * 5 * a.w * 4,
                 workspace_bytes);
    CAVS_REQUIRE(aligned16(workspace), "%s: the workspace must be 16-byte aligned", who);
    b.part = static_cast<float *>(workspace);
  }
  return (type == CAVS_F32 ? run_bwd<float> : run_bwd<u16>)(a, b, o, full, groups, st);
}

}  // extern "C"
