// Norms after and before a block, with its gate and residual scale:
//   z = post(y),  s = r + scale gate . z,  x = pre(s)
// where a norm of v [w] is nothing, (v / sqrt(mean v^2 + eps)) weight + bias, or ((v - mean v) / sqrt(var v + eps)) weight + bias.  With v^ what is between
// the brackets, h = d x . weight and D = d s + the gradient that comes through x:
//   D = d s + rstd (h - [mean h] - s^ mean(h s^)),  d r = D,  d gate = scale z D,  d z = scale gate . D,  d y from d z as D from d x,
//   d weight = sum over rows of d x . v^,  d bias = sum over rows of d x
//
// A row is held by L lanes, eight neighbouring values of each in registers, so that memory is read and written once.  The sums of a row are made in 64
// bits: of values and squares at once (mean and variance from one trip across the lanes, without loss for any mean below 2^20 deviations), and squares of any float
// fit.  Bound by HBM; of few rows by the trips across the lanes.
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
__device__ __forceinline__ double rotated(double v) {
  const int lo = __double2loint(v), hi = __double2hiint(v);
  return two(__builtin_amdgcn_update_dpp(0, lo, CTRL, 0xf, 0xf, true), __builtin_amdgcn_update_dpp(0, hi, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ double crossed32(double v) {
  const unsigned lo = __double2loint(v), hi = __double2hiint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(lo, lo, false, false), b = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
  return two(a[0], b[0]) + two(a[1], b[1]);
}
__device__ __forceinline__ double crossed16(double v) {
  const unsigned lo = __double2loint(v), hi = __double2hiint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), b = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
  return two(a[0], b[0]) + two(a[1], b[1]);
}
// of sixteen, 32 or 64 neighbouring lanes, every lane with the result
template <int L>
__device__ __forceinline__ double lanes_sum(double v) {
  if constexpr (L >= 64) v = crossed32(v);
  if constexpr (L >= 32) v = crossed16(v);
  v += rotated<0x128>(v);  // row_ror:8, 4, 2, 1
  v += rotated<0x124>(v);
  v += rotated<0x122>(v);
  return v + rotated<0x121>(v);
}
// K sums of the L lanes of a row.  L above 64: a workgroup is a row; `lds` [K][L / 64] is written here and may be written again after the next barrier but one.
template <int L, int K>
__device__ __forceinline__ void row_sums(double (&v)[K], double *lds) {
#pragma unroll
  for (int k = 0; k < K; k++) v[k] = lanes_sum<L>(v[k]);
  if constexpr (L > 64) {
    constexpr int W = L / 64;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; k++) lds[k * W + (threadIdx.x >> 6)] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
      v[k] = 0.;
#pragma unroll
      for (int i = 0; i < W; i++) v[k] += lds[k * W + i];
    }
  }
}

// v^ = ((v - mean) - rest) rstd: mean as a float and what it leaves off, so that the difference is a float's own however far the values are from 0
struct Stats {
  float mean, rest, rstd;
  __device__ __forceinline__ void of(double sum, double squares, int w, int kind, float eps) {
    const double inv = 1. / w, m = kind == CAVS_NORM_LAYER ? sum * inv : 0., v = squares * inv - m * m;
    mean = (float)m;
    rest = (float)(m - (double)mean);
    const double a = (v > 0. ? v : v == v ? 0. : v) + (double)eps;
    const double y = __builtin_amdgcn_rsq(a);  // (2^-23, and a step of Newton's makes 2^-45 of it)
    rstd = (float)(y * (1.5 - 0.5 * a * y * y));
  }
  __device__ __forceinline__ float hat(float v) const { return ((v - mean) - rest) * rstd; }
};

template <int L>
constexpr int threads_of() { return L > 64 ? L : 256; }

__device__ __forceinline__ void weights8(float (&o)[8], const float *p, int c, int left, float none) {
  if (!p || left <= 0) {
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] = e < left ? none : 0.f;
    return;
  }
  Eight<float> t;
  t.load(p + c, left);
#pragma unroll
  for (int e = 0; e < 8; e++) o[e] = t[e];
}

// ------------------------------------------------------------------ forward
template <class T, int L, int V>
__global__ __launch_bounds__(threads_of<L>()) void norm_fwd_kernel(Norm a, T *s, long lds_, T *x, long ldx) {
  __shared__ double part[2][2 * (L > 64 ? L / 64 : 1)];
  const int lane = threadIdx.x % L, row = blockIdx.x * (threads_of<L>() / L) + threadIdx.x / L;
  if (row >= a.n) return;  // (a whole workgroup's, where one is a row)
  float v[V][8];
  Eight<T> y[V], r[V], g[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = 8 * (i * L + lane), left = a.w - c;
    y[i].zero(), r[i].zero(), g[i].zero();
    if (left > 0) {
      y[i].load(static_cast<const T *>(a.y) + row * a.ldy + c, left);
      if (a.r) r[i].load(static_cast<const T *>(a.r) + row * a.ldr + c, left);
      if (a.gate_rows) g[i].load(static_cast<const T *>(a.gate_rows) + row * a.ldg + c, left);
    }
  }
  auto stats = [&](int kind, double *lds) {
    double t[2] = {0., 0.};
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) t[0] += v[i][e], t[1] += (double)v[i][e] * v[i][e];
    row_sums<L, 2>(t, lds);
    Stats o;
    o.of(t[0], t[1], a.w, kind, a.eps);
    return o;
  };
#pragma unroll
  for (int i = 0; i < V; i++)
#pragma unroll
    for (int e = 0; e < 8; e++) v[i][e] = y[i][e];
  Stats post{}, pre{};
  if (a.post) post = stats(a.post, part[0]);
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = 8 * (i * L + lane), left = a.w - c;
    float w[8], b[8], gate[8];
    if (a.post) {
      weights8(w, a.post_w, c, left, 1.f), weights8(b, a.post_b, c, left, 0.f);
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = post.hat(v[i][e]) * w[e] + b[e];
    }
    weights8(gate, a.gate, c, left, 1.f);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      v[i][e] *= a.scale * (a.gate_rows ? g[i][e] : gate[e]);
      v[i][e] = 8 * (i * L + lane) + e < a.w ? v[i][e] + r[i][e] : 0.f;
    }
    if (s && left > 0) Eight<T>::store(s + row * lds_ + c, v[i], left);
  }
  if (!x) return;
  if (a.pre) pre = stats(a.pre, part[1]);
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = 8 * (i * L + lane), left = a.w - c;
    if (left <= 0) continue;
    float w[8], b[8];
    if (a.pre) {
      weights8(w, a.pre_w, c, left, 1.f), weights8(b, a.pre_b, c, left, 0.f);
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = pre.hat(v[i][e]) * w[e] + b[e];
    }
    Eight<T>::store(x + row * ldx + c, v[i], left);
  }
}

// ------------------------------------------------------------------ backward
struct Back {
  const void *s, *ds, *dx;
  long lds, ldds, lddx;
  void *dy, *dr, *dg;
  long lddy, lddr, lddg;
  float *part;  // [workgroups][sums][w]: pre_w, pre_b, gate, post_w, post_b; null: none wanted
  int sums;     // 3 or 5
};

// A workgroup takes every gridDim.x-th row (group of rows), its lanes the same columns of each: the sums over rows are in registers until it ends.
template <class T, int L, int V, bool POST>
__global__ __launch_bounds__(threads_of<L>()) void norm_bwd_kernel(Norm a, Back b) {
  constexpr int G = threads_of<L>() / L, S = POST ? 5 : 3;
  __shared__ double part[2][8 * (L > 64 ? L / 64 : 1)];
  __shared__ float merged[G > 1 ? G - 1 : 1][G > 1 ? 8 * L * V : 1];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  float acc[S][V][8], pw[V][8], qw[V][8], qb[V][8], gate[V][8];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = 8 * (i * L + lane), left = a.w - c;
    weights8(pw[i], a.pre_w, c, left, 1.f);
    if constexpr (POST) weights8(qw[i], a.post_w, c, left, 1.f), weights8(qb[i], a.post_b, c, left, 0.f);
    weights8(gate[i], a.gate, c, left, 1.f);
#pragma unroll
    for (int e = 0; e < 8; e++)
#pragma unroll
      for (int k = 0; k < S; k++) acc[k][i][e] = 0.f;
  }
  const double inv = 1. / a.w;
  for (int first = blockIdx.x * G; first < a.n; first += gridDim.x * G) {
    const int row = first + group;
    const bool on = row < a.n;
    Eight<T> s[V], ds[V], dx[V], y[V], g[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = 8 * (i * L + lane), left = on ? a.w - c : 0;
      s[i].zero(), ds[i].zero(), dx[i].zero(), y[i].zero(), g[i].zero();
      if (left > 0) {
        if (a.pre) s[i].load(static_cast<const T *>(b.s) + row * b.lds + c, left);
        if (b.dx) dx[i].load(static_cast<const T *>(b.dx) + row * b.lddx + c, left);
        if (b.ds) ds[i].load(static_cast<const T *>(b.ds) + row * b.ldds + c, left);
        if (a.y) y[i].load(static_cast<const T *>(a.y) + row * a.ldy + c, left);
        if (a.gate_rows) g[i].load(static_cast<const T *>(a.gate_rows) + row * a.ldg + c, left);
      }
    }
    double t[6] = {0., 0., 0., 0., 0., 0.};
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const double v = s[i][e], h = dx[i][e] * pw[i][e];
        t[0] += v, t[1] += v * v, t[2] += h, t[3] += h * v;
        if constexpr (POST) t[4] += y[i][e], t[5] += (double)y[i][e] * y[i][e];
      }
    if constexpr (!POST) {
      double u[4] = {t[0], t[1], t[2], t[3]};
      row_sums<L, 4>(u, part[0]);
#pragma unroll
      for (int k = 0; k < 4; k++) t[k] = u[k];
    } else {
      row_sums<L, 6>(t, part[0]);
    }
    Stats pre{}, post{};
    float h1 = 0.f, h2 = 0.f;  // means of h and of h s^
    if (a.pre) {
      pre.of(t[0], t[1], a.w, a.pre, a.eps);
      const double m = a.pre == CAVS_NORM_LAYER ? t[0] * inv : 0.;
      h1 = a.pre == CAVS_NORM_LAYER ? (float)(t[2] * inv) : 0.f;
      h2 = (float)((t[3] - m * t[2]) * inv * pre.rstd);
    }
    if constexpr (POST) post.of(t[4], t[5], a.w, a.post, a.eps);
    float D[V][8], dz[V][8];
    double q[2] = {0., 0.};
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = 8 * (i * L + lane), left = on ? a.w - c : 0;
      float dgate[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        D[i][e] = ds[i][e];
        if (a.pre) {
          const float hat = pre.hat(s[i][e]), d = dx[i][e];
          D[i][e] += pre.rstd * ((d * pw[i][e] - h1) - hat * h2);
          acc[0][i][e] += d * hat;
          acc[1][i][e] += d;
        } else {
          D[i][e] += dx[i][e];
        }
        const float gt = a.gate_rows ? g[i][e] : gate[i][e];
        float z = y[i][e], zh = 0.f;
        if constexpr (POST) {
          zh = post.hat(z);
          z = zh * qw[i][e] + qb[i][e];
        }
        const float scaled = a.scale * D[i][e];
        dgate[e] = scaled * z;
        acc[2][i][e] += dgate[e];
        dz[i][e] = scaled * gt;
        if constexpr (POST) {
          acc[3][i][e] += dz[i][e] * zh;
          acc[4][i][e] += dz[i][e];
          const double h = dz[i][e] * qw[i][e];
          q[0] += h, q[1] += h * y[i][e];
        }
      }
      if (left > 0) {
        if (b.dr) Eight<T>::store(static_cast<T *>(b.dr) + row * b.lddr + c, D[i], left);
        if (b.dg) Eight<T>::store(static_cast<T *>(b.dg) + row * b.lddg + c, dgate, left);
        if constexpr (!POST) {
          if (b.dy) Eight<T>::store(static_cast<T *>(b.dy) + row * b.lddy + c, dz[i], left);
        }
      }
    }
    if constexpr (POST) {
      row_sums<L, 2>(q, part[1]);
      const double m = a.post == CAVS_NORM_LAYER ? t[4] * inv : 0.;
      const float g1 = a.post == CAVS_NORM_LAYER ? (float)(q[0] * inv) : 0.f, g2 = (float)((q[1] - m * q[0]) * inv * post.rstd);
#pragma unroll
      for (int i = 0; i < V; i++) {
        const int c = 8 * (i * L + lane), left = on ? a.w - c : 0;
        if (left <= 0 || !b.dy) continue;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = post.rstd * ((dz[i][e] * qw[i][e] - g1) - post.hat(y[i][e]) * g2);
        Eight<T>::store(static_cast<T *>(b.dy) + row * b.lddy + c, o, left);
      }
    }
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
          for (int e = 0; e < 8; e++) merged[group - 1][(i * 8 + e) * L + lane] = acc[k][i][e];
      }
      __syncthreads();
      if (group > 0) continue;
#pragma unroll
      for (int q = 1; q < G; q++)
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) acc[k][i][e] += merged[q - 1][(i * 8 + e) * L + lane];
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = 8 * (i * L + lane), left = a.w - c;
      if (left > 0) Eight<float>::store(b.part + ((long)blockIdx.x * S + k) * a.w + c, acc[k][i], left);
    }
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
// lanes of a row: the fewest that hold it eight values each, of 128 values and more as many as leave at most half of them idle
template <class F>
int with_lanes(int w, F &&f) {
#define CAVS_NORM_LANES(L, V) \
  if (w <= 8 * L * V) return f(std::integral_constant<int, L>{}, std::integral_constant<int, V>{});
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

// workgroups of the backward pass: what the compute units hold at once
int back_groups(int n, int w) {
  int groups = 0;
  with_lanes(w, [&](auto l, auto) {
    constexpr int L = decltype(l)::value, T = threads_of<L>(), G = T / L;
    const int most = (1024 / T > 0 ? 1024 / T : 1) * num_cus(), wanted = (int)((n + (long)G - 1) / G);
    groups = wanted < most ? wanted : most;
    return CAVS_OK;
  });
  return groups;
}

template <class T>
int run_fwd(const Norm &a, void *s, int lds, void *x, int ldx, hipStream_t st) {
  return with_lanes(a.w, [&](auto l, auto v) {
    constexpr int L = decltype(l)::value, V = decltype(v)::value, G = threads_of<L>() / L;
    launch(norm_fwd_kernel<T, L, V>, (unsigned)((a.n + (long)G - 1) / G), threads_of<L>(), 0, st, a, static_cast<T *>(s), (long)lds, static_cast<T *>(x), (long)ldx);
    CAVS_LAUNCH_CHECK();
    return (int)CAVS_OK;
  });
}

template <class T>
int run_bwd(const Norm &a, const Back &b, const SumOut &o, int groups, hipStream_t st) {
  return with_lanes(a.w, [&](auto l, auto v) {
    constexpr int L = decltype(l)::value, V = decltype(v)::value;
    launch(a.post ? norm_bwd_kernel<T, L, V, true> : norm_bwd_kernel<T, L, V, false>, groups, threads_of<L>(), 0, st, a, b);
    CAVS_LAUNCH_CHECK();
    if (b.part) {
      launch(norm_sums_kernel, dim3((a.w + 63) / 64, b.sums), 1024, 0, st, b.part, groups, b.sums, a.w, o);
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
  return CAVS_OK;
}

}  // namespace
}  // namespace cavs

using namespace cavs;

extern "C" {

size_t cavs_norm_residual_workspace(int n, int w) {
  if (n <= 0 || w <= 0 || w > kMostW || n > (int)most_groups(1024)) return 0;
  return (size_t)back_groups(n, w) * 5 * w * 4;
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
  const SumOut o{{g->dpre_w, g->dpre_b, g->dgate, g->dpost_w, g->dpost_b}};
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
  if (!dx) a.pre = CAVS_NORM_NONE;  // (nothing comes through it)
  const int groups = back_groups(a.n, a.w);
  Back b{s, ds, dx, lds, ldds, lddx, g->dy, g->dr, g->dgate_rows, g->lddy, g->lddr, g->lddg, nullptr, a.post ? 5 : 3};
  if (!needs_y) a.y = nullptr;  // (not read)
  if (sums) {
    CAVS_REQUIRE(workspace && workspace_bytes >= (size_t)groups * 5 * a.w * 4, "%s: workspace of %zu bytes needed, %zu given", who, (size_t)groups * 5 * a.w * 4,
                 workspace_bytes);
    CAVS_REQUIRE(aligned16(workspace), "%s: the workspace must be 16-byte aligned", who);
    b.part = static_cast<float *>(workspace);
  }
  return (type == CAVS_F32 ? run_bwd<float> : run_bwd<u16>)(a, b, o, groups, st);
}

}  // extern "C"
