// Group norm with an activation, channels last, and its gradients.  x [B, R, C], a
// group of cpg = C / G neighbouring channels:
//
//   mean, var over a sample's R rows and the group's channels,  rs = 1 / sqrt(var + eps)
//   xh = (x - mean) * rs,  n = xh * w + b,  y = act(n)
//
//   dn = dy * act'(n),  s1[b, c] = sum over rows of dn,  s2[b, c] = sum over rows of dn * xh
//   db = sum over samples of s1,  dw = sum over samples of s2
//   dx = rs * (dn * w - m1 - xh * m2),  m1, m2 = means over the group of w * s1, w * s2
//
// Bound by HBM, and by launches where a sample is small.  A lane keeps its 16 bytes of
// channels through all rows of its workgroup, so parameters and sums live in registers
// and rows are read whole.  The statistics are of centred values: a lane takes batches
// of rows, whose mean and centred squares are exact to fp32 whatever the mean, and joins
// them with the running pair (Chan, Golub & LeVeque, "Updating formulae and a pairwise
// algorithm for computing sample variances", 1979); lanes, groups and workgroups are
// joined the same way.  All sums in fp32 and in a fixed order, no atomics.
//
// Large samples: workgroups leave partial sums, a second kernel joins them, a third
// reads x again, in the opposite order of rows, so that the rows read last are still in
// the cache.  Small samples: one workgroup each, one launch.
#include <algorithm>
#include <cmath>

#include "nsw_gemm_common.h"
#include "nsw_grad.h"

namespace nsw {

namespace {

constexpr int NT = 256;            // threads of a workgroup
constexpr int64_t MOST_BLOCKS = 1 << 22;   // of the kernels that loop over groups or columns of all samples: a launch has fewer than 2^32 lanes

struct GnArgs {
  const void *x, *dy, *w, *b;
  void *y, *dx, *dw, *db;
  float* stats;                    // [B, G, 2] mean, rs
  float* part;                     // of the workgroups: [B P][G][2] mean and centred squares, or [B P][2][C] s1, s2
  float* sums;                     // [B, 2, C] s1, s2
  int64_t B, R, per;               // samples, rows of a sample, rows of a workgroup
  int P, C, G, cpg, RL;            // workgroups of a sample, ..., rows in flight at once
  int tpg;                         // lanes that join a group's sums (a power of two)
  FastDiv dcpg, dcv;
  float eps;
};

// A lane's place: 16-byte column pieces cv(k), k < CPT, of row slot rl.
template <typename T, int CPT>
struct Place {
  static constexpr int VEC = Vec16<T>::N;
  int rl, cv0, CV;
  bool in;                          // the lane has a row slot
  __device__ __forceinline__ Place(const GnArgs& a) {
    CV = a.C / VEC;
    if constexpr (CPT == 1) {
      rl = (int)a.dcv.div(threadIdx.x);
      cv0 = (int)threadIdx.x - rl * CV;
    } else {
      rl = 0;
      cv0 = (int)threadIdx.x;
    }
    in = rl < a.RL;
  }
  __device__ __forceinline__ bool has(int k) const { return in && (CPT == 1 || cv0 + NT * k < CV); }
  __device__ __forceinline__ int col(int k) const { return (cv0 + NT * k) * VEC; }
};

// act of a result that is rounded to T
template <typename T, int ACT>
__device__ __forceinline__ float act_for(float n) {
  if constexpr (ACT == NSW_ACT_NONE) return n;
  else return gate_act<T, ACT>(n);
}

template <int ACT>
__device__ __forceinline__ float act_slope(float n) {
  if constexpr (ACT == NSW_ACT_NONE) {
    return 1.f;
  } else {
    float a, d;
    gate_act_grad<ACT>(n, a, d);
    return d;
  }
}

// Running mean and centred squares of U more rows' values v (n rows so far).
template <typename T, int CPT, int U>
__device__ __forceinline__ void take_rows(const float (&v)[U][CPT][Vec16<T>::N], float& n, float (&mean)[CPT][Vec16<T>::N],
                                          float (&m2)[CPT][Vec16<T>::N]) {
  const float f = (float)U / (n + (float)U), g = n * f;
#pragma unroll
  for (int k = 0; k < CPT; ++k)
#pragma unroll
    for (int e = 0; e < Vec16<T>::N; ++e) {
      float s = v[0][k][e];
#pragma unroll
      for (int u = 1; u < U; ++u) s += v[u][k][e];
      const float m = s * (1.f / (float)U);
      float q = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) q = fmaf(v[u][k][e] - m, v[u][k][e] - m, q);
      const float d = m - mean[k][e];
      mean[k][e] = fmaf(d, f, mean[k][e]);
      m2[k][e] += fmaf(d * g, d, q);
    }
  n += (float)U;
}

template <int CPT> constexpr int UNROLL = CPT == 1 ? 8 : 4;

// f(row, U rows' values) over rows r0 + rl, r0 + rl + RL, ... below r1, in batches of U and then one by one.
template <typename T, int CPT, int U, class F>
__device__ __forceinline__ int64_t in_batches(const T* base, int64_t r, int64_t r1, const GnArgs& a, const Place<T, CPT>& at, F f) {
  for (; r + (int64_t)(U - 1) * a.RL < r1; r += (int64_t)U * a.RL) {
    float v[U][CPT][Vec16<T>::N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < CPT; ++k)
        if (CPT == 1 || at.has(k)) load16(base + (r + (int64_t)u * a.RL) * a.C + at.col(k), v[u][k]);
        else
#pragma unroll
          for (int e = 0; e < Vec16<T>::N; ++e) v[u][k][e] = 0.f;
    f(r, v);
  }
  return r;
}

// Rows r0 + rl, r0 + rl + RL, ... below r1 of a slot.
__device__ __forceinline__ int64_t rows_of_slot(int64_t rows, int rl, int RL) { return rows > rl ? (rows - rl + RL - 1) / RL : 0; }

// Statistics of rows [r0, r1) of a sample: (mean, centred squares) of group g to out(g, mean, m2).
// lds: 2 RL C floats.
template <typename T, int CPT, class F>
__device__ __forceinline__ void chunk_stats(const GnArgs& a, const T* base, int64_t r0, int64_t r1, float* lds, F out) {
  constexpr int VEC = Vec16<T>::N, U = UNROLL<CPT>;
  const Place<T, CPT> at(a);
  float mean[CPT][VEC] = {}, m2[CPT][VEC] = {}, n = 0.f;
  if (at.in) {
    int64_t r = in_batches<T, CPT, U>(base, r0 + at.rl, r1, a, at, [&](int64_t, auto& v) { take_rows<T, CPT, U>(v, n, mean, m2); });
    in_batches<T, CPT, 1>(base, r, r1, a, at, [&](int64_t, auto& v) { take_rows<T, CPT, 1>(v, n, mean, m2); });
  }
  const int half = a.RL * a.C;
#pragma unroll
  for (int k = 0; k < CPT; ++k)
    if (at.has(k)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        lds[at.rl * a.C + at.col(k) + e] = mean[k][e];
        lds[half + at.rl * a.C + at.col(k) + e] = m2[k][e];
      }
    }
  __syncthreads();
  const int lane = (int)threadIdx.x & (a.tpg - 1), count = a.RL * a.cpg;
  const int64_t rows = r1 - r0;
  const float total = 1.f / ((float)rows * (float)a.cpg);
  for (int g0 = 0; g0 < a.G; g0 += NT / a.tpg) {            // the same turns on every lane: the shuffles need them all
    const int g = g0 + (int)threadIdx.x / a.tpg;
    float s = 0.f;
    if (g < a.G)
      for (int i = lane; i < count; i += a.tpg) {
        const int rl = (int)a.dcpg.div((uint32_t)i), c = g * a.cpg + i - rl * a.cpg;
        s = fmaf((float)rows_of_slot(rows, rl, a.RL), lds[rl * a.C + c], s);
      }
    for (int off = a.tpg >> 1; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    const float m = s * total;
    float q = 0.f;
    if (g < a.G)
      for (int i = lane; i < count; i += a.tpg) {
        const int rl = (int)a.dcpg.div((uint32_t)i), c = g * a.cpg + i - rl * a.cpg;
        const float d = lds[rl * a.C + c] - m, nr = (float)rows_of_slot(rows, rl, a.RL);
        if (nr > 0.f) q += fmaf(nr * d, d, lds[half + rl * a.C + c]);
      }
    for (int off = a.tpg >> 1; off >= 1; off >>= 1) q += __shfl_xor(q, off, 64);
    if (g < a.G && lane == 0) out(g, m, q);
  }
}

__device__ __forceinline__ float root_of(float m2, float n, float eps) { return 1.0f / sqrtf(m2 / n + eps); }

// 259,200 rows of 512, bf16: 265 MB in 65 us, 4.1 TB/s.
template <typename T, int CPT>
__global__ __launch_bounds__(NT) void group_norm_stats_kernel(GnArgs a) {
  extern __shared__ float lds[];
  const int64_t s = (int64_t)blockIdx.x / a.P, p = (int64_t)blockIdx.x - s * a.P;
  const int64_t r0 = p * a.per, r1 = r0 + a.per < a.R ? r0 + a.per : a.R;
  float* part = a.part + (int64_t)blockIdx.x * a.G * 2;
  chunk_stats<T, CPT>(a, (const T*)a.x + s * a.R * a.C, r0, r1, lds, [&](int g, float m, float q) {
    part[2 * g] = m;
    part[2 * g + 1] = q;
  });
}

// (mean, rs) of each sample's groups from the workgroups' pairs, a wave each.
__global__ __launch_bounds__(NT) void group_norm_join_kernel(GnArgs a) {
  const int lane = (int)threadIdx.x & 63;
  auto rows = [&](int p) { return (float)((p + 1) * a.per < a.R ? a.per : a.R - p * a.per); };
  for (int64_t i = (int64_t)blockIdx.x * (NT / 64) + (int)threadIdx.x / 64; i < a.B * a.G; i += (int64_t)gridDim.x * (NT / 64)) {
    const int64_t s = i / a.G;
    const f32x2* part = (const f32x2*)a.part + s * a.P * a.G + (i - s * a.G);
    float t = 0.f;
    for (int p = lane; p < a.P; p += 64) t = fmaf(rows(p), part[(int64_t)p * a.G][0], t);
    const float m = wave_sum(t) / (float)a.R;
    float q = 0.f;
    for (int p = lane; p < a.P; p += 64) {
      const f32x2 v = part[(int64_t)p * a.G];
      const float d = v[0] - m;
      q += fmaf(rows(p) * (float)a.cpg * d, d, v[1]);
    }
    q = wave_sum(q);
    if (lane == 0) {
      a.stats[2 * i] = m;
      a.stats[2 * i + 1] = root_of(q, (float)a.R * (float)a.cpg, a.eps);
    }
  }
}

// A lane's channels: mean and rs of their groups (of sample stats [G, 2]), weight, bias.
template <typename T, int CPT>
struct Channels {
  static constexpr int VEC = Vec16<T>::N;
  float mean[CPT][VEC], rs[CPT][VEC], w[CPT][VEC], b[CPT][VEC];
  __device__ __forceinline__ Channels(const GnArgs& a, const Place<T, CPT>& at, const float* stats) {
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
      const int c = at.has(k) ? at.col(k) : 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int g = (int)a.dcpg.div((uint32_t)(c + e));
        mean[k][e] = stats[2 * g];
        rs[k][e] = stats[2 * g + 1];
        w[k][e] = 1.f;
        b[k][e] = 0.f;
      }
      if (a.w != nullptr) load16((const T*)a.w + c, w[k]);
      if (a.b != nullptr) load16((const T*)a.b + c, b[k]);
    }
  }
  __device__ __forceinline__ float hat(int k, int e, float x) const { return (x - mean[k][e]) * rs[k][e]; }
  __device__ __forceinline__ float n(int k, int e, float hat) const { return fmaf(hat, w[k][e], b[k][e]); }
};

template <typename T, int CPT, int ACT>
__device__ __forceinline__ void apply_rows(const GnArgs& a, const T* base, T* out, int64_t r0, int64_t r1, const float* stats) {
  constexpr int U = CPT == 1 ? 4 : 2;
  const Place<T, CPT> at(a);
  if (!at.in) return;
  const Channels<T, CPT> ch(a, at, stats);
  auto body = [&](int64_t r, auto& v) {
    constexpr int N = sizeof(v) / sizeof(v[0]);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int k = 0; k < CPT; ++k) {
        if (CPT > 1 && !at.has(k)) continue;
        float o[Vec16<T>::N];
#pragma unroll
        for (int e = 0; e < Vec16<T>::N; ++e) o[e] = act_for<T, ACT>(ch.n(k, e, ch.hat(k, e, v[u][k][e])));
        store16(out + (r + (int64_t)u * a.RL) * a.C + at.col(k), o);
      }
  };
  const int64_t r = in_batches<T, CPT, U>(base, r0 + at.rl, r1, a, at, body);
  in_batches<T, CPT, 1>(base, r, r1, a, at, body);
}

// The same rows read, in part from the cache, and written: 86 us, 6.2 TB/s.
template <typename T, int CPT, int ACT>
__global__ __launch_bounds__(NT) void group_norm_apply_kernel(GnArgs a) {
  const int64_t i = (int64_t)gridDim.x - 1 - blockIdx.x;    // the rows read last first
  const int64_t s = i / a.P, p = i - s * a.P;
  const int64_t r0 = p * a.per, r1 = r0 + a.per < a.R ? r0 + a.per : a.R;
  apply_rows<T, CPT, ACT>(a, (const T*)a.x + s * a.R * a.C, (T*)a.y + s * a.R * a.C, r0, r1, a.stats + s * a.G * 2);
}

// A sample to a workgroup, statistics and results.
template <typename T, int CPT, int ACT>
__global__ __launch_bounds__(NT) void group_norm_small_kernel(GnArgs a) {
  extern __shared__ float lds[];
  const int64_t s = blockIdx.x;
  const T* base = (const T*)a.x + s * a.R * a.C;
  float* mine = lds + 2 * a.RL * a.C;                       // [G, 2]
  chunk_stats<T, CPT>(a, base, 0, a.R, lds, [&](int g, float m, float q) {
    const float r = root_of(q, (float)a.R * (float)a.cpg, a.eps);
    mine[2 * g] = m;
    mine[2 * g + 1] = r;
    a.stats[(s * a.G + g) * 2] = m;
    a.stats[(s * a.G + g) * 2 + 1] = r;
  });
  __syncthreads();
  apply_rows<T, CPT, ACT>(a, base, (T*)a.y + s * a.R * a.C, 0, a.R, mine);
}

// --------------------------------------------------------------- gradients ---

// f(row, U rows of x, U rows of dy) as in_batches.
template <typename T, int CPT, int U, class F>
__device__ __forceinline__ int64_t in_pairs(const T* x, const T* dy, int64_t r, int64_t r1, const GnArgs& a,
                                            const Place<T, CPT>& at, F f) {
  for (; r + (int64_t)(U - 1) * a.RL < r1; r += (int64_t)U * a.RL) {
    float v[U][CPT][Vec16<T>::N], d[U][CPT][Vec16<T>::N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < CPT; ++k) {
        const int64_t o = (r + (int64_t)u * a.RL) * a.C + at.col(k);
        if (CPT == 1 || at.has(k)) {
          load16(x + o, v[u][k]);
          load16(dy + o, d[u][k]);
        } else {
#pragma unroll
          for (int e = 0; e < Vec16<T>::N; ++e) v[u][k][e] = d[u][k][e] = 0.f;
        }
      }
    f(r, v, d);
  }
  return r;
}

// s1, s2 of rows [r0, r1) of a sample to out(column of [2, C], value).  lds: 2 RL C floats; a thread reads
// its column's slots before out, which may put the value in the place of the first.
template <typename T, int CPT, int ACT, class F>
__device__ __forceinline__ void chunk_sums(const GnArgs& a, const T* x, const T* dy, int64_t r0, int64_t r1, const float* stats,
                                           float* lds, F out) {
  constexpr int VEC = Vec16<T>::N, U = CPT == 1 ? 4 : 2;
  const Place<T, CPT> at(a);
  const int half = a.RL * a.C;
  if (at.in) {
    const Channels<T, CPT> ch(a, at, stats);
    float s1[CPT][VEC] = {}, s2[CPT][VEC] = {};
    auto body = [&](int64_t, auto& v, auto& d) {
      constexpr int N = sizeof(v) / sizeof(v[0]);
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int k = 0; k < CPT; ++k)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float h = ch.hat(k, e, v[u][k][e]);
            const float dn = d[u][k][e] * act_slope<ACT>(ch.n(k, e, h));
            s1[k][e] += dn;
            s2[k][e] = fmaf(dn, h, s2[k][e]);
          }
    };
    const int64_t r = in_pairs<T, CPT, U>(x, dy, r0 + at.rl, r1, a, at, body);
    in_pairs<T, CPT, 1>(x, dy, r, r1, a, at, body);
#pragma unroll
    for (int k = 0; k < CPT; ++k)
      if (at.has(k)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          lds[at.rl * a.C + at.col(k) + e] = s1[k][e];
          lds[half + at.rl * a.C + at.col(k) + e] = s2[k][e];
        }
      }
  }
  __syncthreads();
  for (int c = (int)threadIdx.x; c < 2 * a.C; c += NT) {
    const float* col = c < a.C ? lds + c : lds + half + (c - a.C);
    float t = col[0];
    for (int rl = 1; rl < a.RL; ++rl) t += col[rl * a.C];
    out(c, t);
  }
}

// 2 x 64,800 rows of 1024, bf16: 531 MB in 127 us, 4.2 TB/s.
template <typename T, int CPT, int ACT>
__global__ __launch_bounds__(NT) void group_norm_sums_kernel(GnArgs a) {
  extern __shared__ float lds[];
  const int64_t s = (int64_t)blockIdx.x / a.P, p = (int64_t)blockIdx.x - s * a.P;
  const int64_t r0 = p * a.per, r1 = r0 + a.per < a.R ? r0 + a.per : a.R;
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.C;
  chunk_sums<T, CPT, ACT>(a, (const T*)a.x + s * a.R * a.C, (const T*)a.dy + s * a.R * a.C, r0, r1, a.stats + s * a.G * 2, lds,
                          [&](int c, float t) { part[c] = t; });
}

// sums [B, 2, C] from the workgroups' partial rows.
__global__ __launch_bounds__(NT) void group_norm_sums_join_kernel(GnArgs a, int blocks) {
  __shared__ __attribute__((aligned(16))) float red[32][36];
  for (int64_t i = blockIdx.x; i < a.B * blocks; i += gridDim.x) {
    const int64_t s = i / blocks;
    column_sums_block<float>(a.part + s * a.P * 2 * a.C, a.sums + s * 2 * a.C, a.P, 2 * a.C, (int)(i - s * blocks), red);
    __syncthreads();
  }
}

// db and dw from sums, 32 of their 2 C columns to a workgroup, every 32nd sample to a lane.
constexpr int PARAMS = 32;
template <typename T>
__device__ __forceinline__ void params_block(const GnArgs& a, int block) {
  __shared__ __attribute__((aligned(16))) float red[32][PARAMS + 4];
  const int cl = ((int)threadIdx.x & 7) * 4, grp = (int)threadIdx.x >> 3, c = block * PARAMS + cl;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  if (c < 2 * a.C)
#pragma unroll 4
    for (int64_t s = grp; s < a.B; s += 32) t += *reinterpret_cast<const f32x4*>(a.sums + s * 2 * a.C + c);
  *reinterpret_cast<f32x4*>(&red[grp][cl]) = t;
  __syncthreads();
  T* out = (T*)(c < a.C ? a.db : a.dw);
  if (grp != 0 || c >= 2 * a.C || out == nullptr) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) t += *reinterpret_cast<const f32x4*>(&red[i][cl]);
  const float v[4] = {t[0], t[1], t[2], t[3]};
  store4<T>(out + (c < a.C ? c : c - a.C), v);
}

template <typename T>
__global__ __launch_bounds__(NT) void group_norm_params_kernel(GnArgs a) {
  params_block<T>(a, (int)blockIdx.x);
}

// dx of rows [r0, r1) of a sample with its s1, s2 [C].  means: 2 G floats of LDS.
template <typename T, int CPT, int ACT>
__device__ __forceinline__ void gradient_rows(const GnArgs& a, const T* x, const T* dy, T* dx, int64_t r0, int64_t r1,
                                              const float* stats, const float* s1, const float* s2, float* means) {
  constexpr int VEC = Vec16<T>::N, U = CPT == 1 ? 4 : 2;
  const int lane = (int)threadIdx.x & (a.tpg - 1);
  const float inv = 1.f / ((float)a.R * (float)a.cpg);
  for (int g0 = 0; g0 < a.G; g0 += NT / a.tpg) {
    const int g = g0 + (int)threadIdx.x / a.tpg;
    float m1 = 0.f, m2 = 0.f;
    if (g < a.G)
      for (int i = lane; i < a.cpg; i += a.tpg) {
        const int c = g * a.cpg + i;
        const float w = a.w == nullptr ? 1.f : to_f32(((const T*)a.w)[c]);
        m1 = fmaf(w, s1[c], m1);
        m2 = fmaf(w, s2[c], m2);
      }
    for (int off = a.tpg >> 1; off >= 1; off >>= 1) {
      m1 += __shfl_xor(m1, off, 64);
      m2 += __shfl_xor(m2, off, 64);
    }
    if (g < a.G && lane == 0) {
      means[2 * g] = m1 * inv;
      means[2 * g + 1] = m2 * inv;
    }
  }
  __syncthreads();
  const Place<T, CPT> at(a);
  if (!at.in) return;
  const Channels<T, CPT> ch(a, at, stats);
  float m1[CPT][VEC], m2[CPT][VEC];
#pragma unroll
  for (int k = 0; k < CPT; ++k) {
    const int c = at.has(k) ? at.col(k) : 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int g = (int)a.dcpg.div((uint32_t)(c + e));
      m1[k][e] = means[2 * g];
      m2[k][e] = means[2 * g + 1];
    }
  }
  auto body = [&](int64_t r, auto& v, auto& d) {
    constexpr int N = sizeof(v) / sizeof(v[0]);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int k = 0; k < CPT; ++k) {
        if (CPT > 1 && !at.has(k)) continue;
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float h = ch.hat(k, e, v[u][k][e]);
          const float dn = d[u][k][e] * act_slope<ACT>(ch.n(k, e, h));
          o[e] = ch.rs[k][e] * fmaf(-h, m2[k][e], fmaf(dn, ch.w[k][e], -m1[k][e]));
        }
        store16(dx + (r + (int64_t)u * a.RL) * a.C + at.col(k), o);
      }
  };
  const int64_t r = in_pairs<T, CPT, U>(x, dy, r0 + at.rl, r1, a, at, body);
  in_pairs<T, CPT, 1>(x, dy, r, r1, a, at, body);
}

// The first workgroups form the parameters' gradients, the rest dx (2 x 64,800 rows of 1024,
// bf16: 796 MB in 144 us, 5.5 TB/s).
template <typename T, int CPT, int ACT>
__global__ __launch_bounds__(NT) void group_norm_gradient_kernel(GnArgs a, int params) {
  extern __shared__ float lds[];
  if ((int)blockIdx.x < params) {
    params_block<T>(a, (int)blockIdx.x);
    return;
  }
  const int64_t i = (int64_t)gridDim.x - 1 - blockIdx.x;    // the rows read last first
  const int64_t s = i / a.P, p = i - s * a.P;
  const int64_t r0 = p * a.per, r1 = r0 + a.per < a.R ? r0 + a.per : a.R;
  const int64_t o = s * a.R * a.C;
  gradient_rows<T, CPT, ACT>(a, (const T*)a.x + o, (const T*)a.dy + o, (T*)a.dx + o, r0, r1, a.stats + s * a.G * 2,
                             a.sums + s * 2 * a.C, a.sums + (s * 2 + 1) * a.C, lds);
}

template <typename T, int CPT, int ACT>
__global__ __launch_bounds__(NT) void group_norm_small_gradient_kernel(GnArgs a) {
  extern __shared__ float lds[];
  const int64_t s = blockIdx.x, o = s * a.R * a.C;
  const int half = a.RL * a.C;
  float* means = lds + 2 * half;                            // [G, 2]
  const float* stats = a.stats + s * a.G * 2;
  chunk_sums<T, CPT, ACT>(a, (const T*)a.x + o, (const T*)a.dy + o, 0, a.R, stats, lds, [&](int c, float t) {
    lds[c < a.C ? c : half + c - a.C] = t;
    a.sums[s * 2 * a.C + c] = t;
  });
  if (a.dx == nullptr) return;
  __syncthreads();
  gradient_rows<T, CPT, ACT>(a, (const T*)a.x + o, (const T*)a.dy + o, (T*)a.dx + o, 0, a.R, stats, lds, lds + half, means);
}

// ------------------------------------------------------------------- plans ---

// Rows in flight of a workgroup, workgroups of a sample and their rows; one workgroup:
// the small kernels.
struct Plan {
  int RL, P;
  int64_t per;
};

// Bytes of a sample up to which one workgroup takes it: more of them where there are workgroups
// for all compute units.  One workgroup against several, us of the forward and the backward pass, bf16,
// C = 192: one sample of 48 KB 12.4 + 15.6 and 15.5 + 14.8, of 96 KB 15.8 + 23.4 and 15.7 + 15.0; 128 of 96 KB
// 17.8 + 26.9 and 21.4 + 24.4, of 192 KB 29.8 + 52.6 and 26.4 + 36.2; 256 of 192 KB 33 + 56 and 37 + 57.
int64_t small_of(int64_t B) { return (B >= 256 ? 192 : B >= 128 ? 96 : 64) << 10; }

Plan plan(int64_t B, int64_t R, int64_t C, int dtype, int per_cu) {
  const int64_t es = (int64_t)dtype_size(dtype), CV = C * es / 16;
  const int RL = (int)std::max<int64_t>(1, NT / CV);
  if (R * C * es <= small_of(B)) return {RL, 1, R};
  const int64_t turns = (R + 8 * RL - 1) / (8 * RL);
  const int64_t want = std::max<int64_t>(2, (256 * per_cu + B - 1) / B);
  const int64_t each = std::max<int64_t>(1, (turns + want - 1) / want);
  return {RL, (int)((turns + each - 1) / each), each * 8 * RL};
}

// Workgroups a compute unit: few where each leaves sums to be joined, many where it only writes rows.
constexpr int STATS_PER_CU = 2, APPLY_PER_CU = 16;

GnArgs common(int64_t B, int64_t R, int64_t C, int64_t G, int dtype, float eps) {
  GnArgs a{};
  a.B = B; a.R = R; a.C = (int)C; a.G = (int)G; a.cpg = (int)(C / G); a.eps = eps;
  a.dcpg = FastDiv::make((uint32_t)a.cpg);
  a.dcv = FastDiv::make((uint32_t)(C * (int64_t)dtype_size(dtype) / 16));
  a.tpg = 1;
  while (a.tpg < 64 && a.tpg * 2 * a.G <= NT) a.tpg *= 2;
  return a;
}

void set(GnArgs& a, const Plan& p) {
  a.RL = p.RL; a.P = p.P; a.per = p.per;
}

int check_sizes(const char* what, int64_t B, int64_t R, int64_t C, int64_t G, int dtype) {
  NSW_CHECK_ARG(dtype == NSW_DTYPE_BF16 || dtype == NSW_DTYPE_F32, "%s: unknown dtype %d", what, dtype);
  const int64_t vec = dtype == NSW_DTYPE_BF16 ? 8 : 4;
  NSW_CHECK_ARG(C > 0 && C % vec == 0 && C <= vec * 512, "%s: C=%lld must be a multiple of %lld, at most %lld", what,
                (long long)C, (long long)vec, (long long)(vec * 512));
  NSW_CHECK_ARG(G > 0 && C % G == 0, "%s: C=%lld must be a multiple of the %lld groups", what, (long long)C, (long long)G);
  NSW_CHECK_ARG(B >= 0 && B < (1LL << 20) && R >= 0 && R < (1LL << 40), "%s: B=%lld, R=%lld out of range", what, (long long)B,
                (long long)R);
  return NSW_OK;
}

// f(T, CPT) for the dtype and width.
template <class F>
int with_cols(int dtype, int64_t C, F f) {
  const int64_t CV = C * (int64_t)dtype_size(dtype) / 16;
  auto by = [&](auto t) {
    if (CV <= NT) return f(t, std::integral_constant<int, 1>{});
    return f(t, std::integral_constant<int, 2>{});
  };
  return dtype == NSW_DTYPE_BF16 ? by(bf16{}) : by(float{});
}

template <class F>
int with_act(int act, F f) {
  switch (act) {
    case NSW_ACT_SILU: return f(std::integral_constant<int, NSW_ACT_SILU>{});
    case NSW_ACT_GELU: return f(std::integral_constant<int, NSW_ACT_GELU>{});
    case NSW_ACT_GELU_TANH: return f(std::integral_constant<int, NSW_ACT_GELU_TANH>{});
    default: return f(std::integral_constant<int, NSW_ACT_NONE>{});
  }
}

bool known_act(int act) {
  return act == NSW_ACT_SILU || act == NSW_ACT_GELU || act == NSW_ACT_GELU_TANH || act == NSW_ACT_NONE;
}

bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p % 16) return false;
  return true;
}

// Floats of LDS for the lanes' sums, two of each slot and channel.
size_t slots_lds(const GnArgs& a) { return (size_t)2 * a.RL * a.C * sizeof(float); }

}  // namespace

}  // namespace nsw

using namespace nsw;

extern "C" size_t nsw_group_norm_workspace_size(int64_t B, int64_t R, int64_t C, int64_t groups, int dtype) {
  if (check_sizes("nsw_group_norm_workspace_size", B, R, C, groups, dtype) != NSW_OK) return 0;
  const Plan p = plan(std::max<int64_t>(B, 1), R, C, dtype, STATS_PER_CU);
  return p.P == 1 ? 16 : (size_t)(B * p.P * groups * 2) * sizeof(float);
}

extern "C" int nsw_group_norm(const void* x, const void* weight, const void* bias, void* y, float* stats, int64_t B, int64_t R,
                              int64_t C, int64_t groups, float eps, int act, int dtype, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* what = "nsw_group_norm";
  if (int rc = check_sizes(what, B, R, C, groups, dtype)) return rc;
  NSW_CHECK_ARG(known_act(act), "%s: unknown activation %d", what, act);
  NSW_CHECK_ARG(eps >= 0.f && std::isfinite(eps), "%s: eps=%g", what, (double)eps);
  if (B == 0 || R == 0) return NSW_OK;
  NSW_CHECK_ARG(x && y && stats, "%s: x, y and stats are required", what);
  NSW_CHECK_ARG(aligned16({x, weight, bias, y, stats, workspace}), "%s: pointers must be 16-byte aligned", what);
  const size_t need = nsw_group_norm_workspace_size(B, R, C, groups, dtype);
  NSW_CHECK_ARG(workspace != nullptr && workspace_bytes >= need, "%s: workspace of %zu bytes needed, got %zu", what, need,
                workspace ? workspace_bytes : (size_t)0);
  GnArgs a = common(B, R, C, groups, dtype, eps);
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.stats = stats; a.part = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  const Plan ps = plan(B, R, C, dtype, STATS_PER_CU), pa = plan(B, R, C, dtype, APPLY_PER_CU);
  return with_cols(dtype, C, [&](auto t, auto cpt) {
    using T = decltype(t);
    constexpr int CPT = decltype(cpt)::value;
    set(a, ps);
    if (ps.P > 1) {
      hipLaunchKernelGGL((group_norm_stats_kernel<T, CPT>), dim3((unsigned)(B * ps.P)), dim3(NT), slots_lds(a), st, a);
      hipLaunchKernelGGL(group_norm_join_kernel, dim3((unsigned)std::min<int64_t>((B * groups + 3) / 4, MOST_BLOCKS)), dim3(NT), 0, st, a);
      set(a, pa);
    }
    return with_act(act, [&](auto ac) {
      constexpr int ACT = decltype(ac)::value;
      if (ps.P > 1)
        hipLaunchKernelGGL((group_norm_apply_kernel<T, CPT, ACT>), dim3((unsigned)(B * pa.P)), dim3(NT), 0, st, a);
      else
        hipLaunchKernelGGL((group_norm_small_kernel<T, CPT, ACT>), dim3((unsigned)B), dim3(NT),
                           slots_lds(a) + (size_t)2 * a.G * sizeof(float), st, a);
      return check_launch(what);
    });
  });
}

extern "C" size_t nsw_group_norm_backward_workspace_size(int64_t B, int64_t R, int64_t C, int64_t groups, int dtype) {
  if (check_sizes("nsw_group_norm_backward_workspace_size", B, R, C, groups, dtype) != NSW_OK) return 0;
  const Plan p = plan(std::max<int64_t>(B, 1), R, C, dtype, STATS_PER_CU);
  return (size_t)(std::max<int64_t>(B, 1) * (p.P > 1 ? p.P + 1 : 1) * 2 * C) * sizeof(float);
}

extern "C" int nsw_group_norm_backward(const void* dy, const void* x, const float* stats, const void* weight, const void* bias,
                                       void* dx, void* dweight, void* dbias, int64_t B, int64_t R, int64_t C, int64_t groups,
                                       int act, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "nsw_group_norm_backward";
  if (int rc = check_sizes(what, B, R, C, groups, dtype)) return rc;
  NSW_CHECK_ARG(known_act(act), "%s: unknown activation %d", what, act);
  const bool rows = B > 0 && R > 0;
  NSW_CHECK_ARG(!rows || (dy && x && stats), "%s: dy, x and stats are required", what);
  NSW_CHECK_ARG(aligned16({dy, x, stats, weight, bias, dx, dweight, dbias, workspace}), "%s: pointers must be 16-byte aligned",
                what);
  const size_t need = nsw_group_norm_backward_workspace_size(B, R, C, groups, dtype);
  NSW_CHECK_ARG(workspace != nullptr && workspace_bytes >= need, "%s: workspace of %zu bytes needed, got %zu", what, need,
                workspace ? workspace_bytes : (size_t)0);
  if (!dx && !dweight && !dbias) return NSW_OK;
  const Plan ps = plan(std::max<int64_t>(B, 1), R, C, dtype, STATS_PER_CU), pa = plan(std::max<int64_t>(B, 1), R, C, dtype, APPLY_PER_CU);
  GnArgs a = common(B, R, C, groups, dtype, 0.f);
  a.x = x; a.dy = dy; a.w = weight; a.b = bias; a.dx = dx; a.dw = dweight; a.db = dbias; a.stats = (float*)stats;
  a.sums = (float*)workspace;
  a.part = a.sums + std::max<int64_t>(B, 1) * 2 * C;
  hipStream_t st = (hipStream_t)stream;
  const int params = dweight || dbias ? (int)((2 * C + PARAMS - 1) / PARAMS) : 0;
  return with_cols(dtype, C, [&](auto t, auto cpt) {
    using T = decltype(t);
    constexpr int CPT = decltype(cpt)::value;
    if (!rows) {                                            // zeros
      a.B = 0;
      if (params) hipLaunchKernelGGL((group_norm_params_kernel<T>), dim3((unsigned)params), dim3(NT), 0, st, a);
      return check_launch(what);
    }
    return with_act(act, [&](auto ac) {
      constexpr int ACT = decltype(ac)::value;
      set(a, ps);
      if (ps.P == 1) {
        hipLaunchKernelGGL((group_norm_small_gradient_kernel<T, CPT, ACT>), dim3((unsigned)B), dim3(NT),
                           slots_lds(a) + (size_t)2 * a.G * sizeof(float), st, a);
        if (params) hipLaunchKernelGGL((group_norm_params_kernel<T>), dim3((unsigned)params), dim3(NT), 0, st, a);
        return check_launch(what);
      }
      const int blocks = (int)((2 * C + 31) / 32);
      hipLaunchKernelGGL((group_norm_sums_kernel<T, CPT, ACT>), dim3((unsigned)(B * ps.P)), dim3(NT), slots_lds(a), st, a);
      hipLaunchKernelGGL(group_norm_sums_join_kernel, dim3((unsigned)std::min<int64_t>(B * blocks, MOST_BLOCKS)), dim3(NT), 0, st, a, blocks);
      set(a, pa);
      if (dx == nullptr)
        hipLaunchKernelGGL((group_norm_params_kernel<T>), dim3((unsigned)params), dim3(NT), 0, st, a);
      else
        hipLaunchKernelGGL((group_norm_gradient_kernel<T, CPT, ACT>), dim3((unsigned)(B * pa.P + params)), dim3(NT),
                           (size_t)2 * a.G * sizeof(float), st, a, params);
      return check_launch(what);
    });
  });
}
