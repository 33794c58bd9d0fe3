// The norms around a branch of a pre-norm block, with its gate and residual:
//
//   n = branch * ro * post_w      ro = 1 / sqrt(mean(branch^2) + eps)   (post_w NULL: n = branch)
//   y = alpha * skip + gate * n   gate of the row's sample              (gate NULL: 1)
//   z = y * ry * norm_w           ry = 1 / sqrt(mean(y^2) + eps)        (norm_w NULL: no z)
//
// and the gradients of all of it.  Values are held in fp32 from the loads to the
// stores: z is of the unrounded y.  The backward pass forms y again from branch and
// skip (the same bytes as reading y, without y's rounding):
//
//   t  = dz * norm_w,  d  = dy + ry * (t - yh * mean(t * yh))     yh = y * ry
//   dskip = alpha * d
//   s  = d * gate * post_w,  dbranch = ro * (s - oh * mean(s * oh))   oh = branch * ro
//   S[sample, c] = sum over the sample's rows of d * oh,  Q[c] = sum over rows of dz * yh
//   dgate = post_w * S,  dpost_w = sum over samples of gate * S,  dnorm_w = Q
//
// Bound by HBM: one pass over the rows, each element read and written once.  A
// workgroup takes a range of one sample's rows, a row at a time on LPR lanes (narrow
// rows, several to a wave), a wave, or the whole workgroup (wide rows), so that a
// lane's columns stay the same: the parameters live in registers, and so do the
// lane's sums for S and Q, which go to a partial row of the workgroup and from there
// through a second kernel in a fixed order (no atomics: the same bits every time).
// The next row's loads are issued before the present row's arithmetic.  129600 x 1024
// bf16: forward 178 us (6.0 TB/s), backward 302 + 6 us (5.2 TB/s, the second kernel included).
#include <algorithm>

#include "nsw_common.h"

namespace nsw {

namespace {

constexpr int NT = 256;   // threads of a workgroup

struct NormArgs {
  const void *branch, *skip, *post_w, *gate, *norm_w;
  const void *dy, *dz;
  void *y, *z, *dbranch, *dskip;
  float* part;            // [G P][2][C] sums of the workgroups: S, Q
  int64_t R;              // rows of a sample
  int64_t per;            // rows of a workgroup
  int P;                  // workgroups of a sample
  int C;
  float alpha, eps;
};

// LPR lanes hold a row of up to LPR * CH 16-byte pieces; LPR = NT: the workgroup.
template <typename T, int LPR_, int CH_> struct RowCfg {
  static constexpr int LPR = LPR_, CH = CH_, VEC = Vec16<T>::N;
  static constexpr bool WG = LPR_ == NT;
  static constexpr int RPS = NT / LPR_;              // rows in flight at once
  static constexpr int WIDTH = LPR_ * CH_ * VEC;     // widest row
};

template <class CFG>
struct Lane {
  int lr, slot;
  __device__ __forceinline__ Lane() : lr((int)threadIdx.x % CFG::LPR), slot((int)threadIdx.x / CFG::LPR) {}
  __device__ __forceinline__ int col(int k) const { return (lr + CFG::LPR * k) * CFG::VEC; }
};

// Sums over the lanes of a row, on each of them.  Workgroup rows: the waves' sums
// meet in LDS, red[turn & 1]; two turns apart a barrier lies between a buffer's reads
// and its next writes.
template <class CFG, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[2][4], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = row16_sum(v[i]);
    if constexpr (CFG::LPR == 32) v[i] = rows2_sum(v[i]);
    if constexpr (CFG::LPR >= 64) v[i] = rows4_sum(v[i]);
  }
  if constexpr (CFG::WG) {
    float(*r)[4] = red[turn & 1];
    ++turn;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i][threadIdx.x >> 6] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (r[i][0] + r[i][1]) + (r[i][2] + r[i][3]);
  }
}

template <typename T>
__device__ __forceinline__ void widen(const u32x4& raw, float* out) {
  if constexpr (sizeof(T) == 2) {
    const bf16x8 v = __builtin_bit_cast(bf16x8, raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (float)v[i];
  } else {
    const f32x4 v = __builtin_bit_cast(f32x4, raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = v[i];
  }
}

template <typename T>
__device__ __forceinline__ u32x4 narrow(const float* in) {
  if constexpr (sizeof(T) == 2) {
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (bf16)in[i];
    return __builtin_bit_cast(u32x4, v);
  } else {
    return __builtin_bit_cast(u32x4, f32x4{in[0], in[1], in[2], in[3]});
  }
}

// Results past L2 (1-4% faster: 259200 x 512 forward 183 -> 180 us, 129600 x 1024
// backward 329 -> 322), but not those of workgroup-wide rows (8000 x 8192 backward 188 ->
// 196).
template <typename T, class CFG>
__device__ __forceinline__ void put(T* p, const u32x4& v) {
  if constexpr (CFG::WG) *reinterpret_cast<u32x4*>(p) = v;
  else __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
}

// The lane's pieces of row `row` (zeros past the row's end).
template <typename T, class CFG>
__device__ __forceinline__ void load_row(const void* p, int64_t row, int C, const Lane<CFG>& ln, u32x4 (&raw)[CFG::CH]) {
#pragma unroll
  for (int k = 0; k < CFG::CH; ++k) {
    const int c = ln.col(k);
    raw[k] = u32x4{0, 0, 0, 0};
    if (c < C) raw[k] = *reinterpret_cast<const u32x4*>((const T*)p + row * C + c);
  }
}

// A parameter's values for the lane's columns (1 where there is none; 0 past the end).
template <typename T, class CFG>
__device__ __forceinline__ void load_param(const void* p, int C, const Lane<CFG>& ln, float (&w)[CFG::CH][CFG::VEC]) {
#pragma unroll
  for (int k = 0; k < CFG::CH; ++k) {
    const int c = ln.col(k);
#pragma unroll
    for (int e = 0; e < CFG::VEC; ++e) w[k][e] = c < C ? 1.f : 0.f;
    if (p != nullptr && c < C) load16<T>((const T*)p + c, w[k]);
  }
}

template <typename T, class CFG>
__global__ __launch_bounds__(NT) void residual_norm_kernel(NormArgs a) {
  constexpr int CH = CFG::CH, VEC = CFG::VEC;
  __shared__ float red[2][2][4];
  int turn = 0;
  const Lane<CFG> ln;
  const int C = a.C, g = (int)(blockIdx.x / (unsigned)a.P), p = (int)(blockIdx.x % (unsigned)a.P);
  const int64_t base = g * a.R, r0 = base + p * a.per, r1 = r0 + a.per < base + a.R ? r0 + a.per : base + a.R;
  const bool post = a.post_w != nullptr, pre = a.norm_w != nullptr;
  const float inv = 1.f / (float)C;
  float wg[CH][VEC], wn[CH][VEC];
  {   // gate * post_w: one factor of the normalised branch
    float w[CH][VEC];
    load_param<T, CFG>(a.post_w, C, ln, w);
    load_param<T, CFG>(a.gate == nullptr ? nullptr : (const T*)a.gate + (int64_t)g * C, C, ln, wg);
    load_param<T, CFG>(a.norm_w, C, ln, wn);
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) wg[k][e] *= w[k][e];
  }
  u32x4 ro_[CH], rx_[CH];
  auto fetch = [&](int64_t row, u32x4(&o)[CH], u32x4(&x)[CH]) {
    row = row < r1 ? row : r1 - 1;
    load_row<T, CFG>(a.branch, row, C, ln, o);
    load_row<T, CFG>(a.skip, row, C, ln, x);
  };
  fetch(r0 + ln.slot, ro_, rx_);
  for (int64_t r = r0; r < r1; r += CFG::RPS) {
    const int64_t row = r + ln.slot;
    u32x4 no_[CH], nx_[CH];
    fetch(row + CFG::RPS, no_, nx_);
    float o[CH][VEC], y[CH][VEC];
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      widen<T>(ro_[k], o[k]);
      widen<T>(rx_[k], y[k]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[0] = fmaf(o[k][e], o[k][e], s[0]);
    }
    float ro = 1.f;
    if (post) {
      row_sums<CFG>(s, red, turn);
      ro = 1.f / sqrtf(s[0] * inv + a.eps);
    }
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        y[k][e] = fmaf(a.alpha, y[k][e], (o[k][e] * ro) * wg[k][e]);
        s[0] = fmaf(y[k][e], y[k][e], s[0]);
      }
    const bool ok = row < r1;
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (ok && ln.col(k) < C) put<T, CFG>((T*)a.y + row * C + ln.col(k), narrow<T>(y[k]));
    if (pre) {
      row_sums<CFG>(s, red, turn);
      const float ry = 1.f / sqrtf(s[0] * inv + a.eps);
#pragma unroll
      for (int k = 0; k < CH; ++k) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[k][e] = (y[k][e] * ry) * wn[k][e];
        if (ok && ln.col(k) < C) put<T, CFG>((T*)a.z + row * C + ln.col(k), narrow<T>(y[k]));
      }
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      ro_[k] = no_[k];
      rx_[k] = nx_[k];
    }
  }
}

// The workgroup's sum of v over the slots of its lanes' columns, into dst [C].
template <class CFG>
__device__ __forceinline__ void store_part(float (&v)[CFG::CH][CFG::VEC], float* buf, float* dst, int C, const Lane<CFG>& ln) {
  if constexpr (CFG::RPS == 1) {
#pragma unroll
    for (int k = 0; k < CFG::CH; ++k)
      if (ln.col(k) < C) {
#pragma unroll
        for (int e = 0; e < CFG::VEC; e += 4)
          *reinterpret_cast<f32x4*>(dst + ln.col(k) + e) = f32x4{v[k][e], v[k][e + 1], v[k][e + 2], v[k][e + 3]};
      }
  } else {
    __syncthreads();   // the buffer's earlier use
#pragma unroll
    for (int k = 0; k < CFG::CH; ++k)
#pragma unroll
      for (int e = 0; e < CFG::VEC; e += 4)
        *reinterpret_cast<f32x4*>(buf + ln.slot * CFG::WIDTH + ln.col(k) + e) =
            f32x4{v[k][e], v[k][e + 1], v[k][e + 2], v[k][e + 3]};
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += NT) {
      float t = 0.f;
#pragma unroll
      for (int s = 0; s < CFG::RPS; ++s) t += buf[s * CFG::WIDTH + c];
      dst[c] = t;
    }
  }
}

template <typename T, class CFG>
__global__ __launch_bounds__(NT) void residual_norm_backward_kernel(NormArgs a) {
  constexpr int CH = CFG::CH, VEC = CFG::VEC;
  __shared__ float red[2][2][4];
  __shared__ __attribute__((aligned(16))) float buf[CFG::RPS == 1 ? 4 : CFG::RPS * CFG::WIDTH];
  int turn = 0;
  const Lane<CFG> ln;
  const int C = a.C, g = (int)(blockIdx.x / (unsigned)a.P), p = (int)(blockIdx.x % (unsigned)a.P);
  const int64_t base = g * a.R, r0 = base + p * a.per, r1 = r0 + a.per < base + a.R ? r0 + a.per : base + a.R;
  const bool post = a.post_w != nullptr, pre = a.norm_w != nullptr, has_dy = a.dy != nullptr;
  const float inv = 1.f / (float)C;
  float wg[CH][VEC], wn[CH][VEC], S[CH][VEC], Q[CH][VEC];
  {   // gate * post_w: the factor of the normalised branch, and of d on its way back
    float w[CH][VEC];
    load_param<T, CFG>(a.post_w, C, ln, w);
    load_param<T, CFG>(a.gate == nullptr ? nullptr : (const T*)a.gate + (int64_t)g * C, C, ln, wg);
    load_param<T, CFG>(a.norm_w, C, ln, wn);
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        wg[k][e] *= w[k][e];
        S[k][e] = 0.f;
        Q[k][e] = 0.f;
      }
  }
  u32x4 ro_[CH], rx_[CH], ry_[CH], rz_[CH];
  auto fetch = [&](int64_t row, u32x4(&o)[CH], u32x4(&x)[CH], u32x4(&dy)[CH], u32x4(&dz)[CH]) {
    row = row < r1 ? row : r1 - 1;
    load_row<T, CFG>(a.branch, row, C, ln, o);
    if (pre) load_row<T, CFG>(a.skip, row, C, ln, x);
    if (has_dy) load_row<T, CFG>(a.dy, row, C, ln, dy);
    if (pre) load_row<T, CFG>(a.dz, row, C, ln, dz);
  };
#pragma unroll
  for (int k = 0; k < CH; ++k) rx_[k] = ry_[k] = rz_[k] = u32x4{0, 0, 0, 0};
  if (r0 < r1) fetch(r0 + ln.slot, ro_, rx_, ry_, rz_);
  for (int64_t r = r0; r < r1; r += CFG::RPS) {
    const int64_t row = r + ln.slot;
    const bool ok = row < r1;
    u32x4 no_[CH], nx_[CH], ny_[CH], nz_[CH];
#pragma unroll
    for (int k = 0; k < CH; ++k) nx_[k] = ny_[k] = nz_[k] = u32x4{0, 0, 0, 0};
    fetch(row + CFG::RPS, no_, nx_, ny_, nz_);
    float oh[CH][VEC], d[CH][VEC];
    float s1[1] = {0.f};
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      widen<T>(ro_[k], oh[k]);
      widen<T>(ry_[k], d[k]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s1[0] = fmaf(oh[k][e], oh[k][e], s1[0]);
    }
    float ro = 1.f;
    if (post) {
      row_sums<CFG>(s1, red, turn);
      ro = 1.f / sqrtf(s1[0] * inv + a.eps);
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) oh[k][e] *= ro;
    }
    if (pre) {
      float y[CH][VEC], dz[CH][VEC];
      float s2[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        widen<T>(rx_[k], y[k]);
        widen<T>(rz_[k], dz[k]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          y[k][e] = fmaf(a.alpha, y[k][e], oh[k][e] * wg[k][e]);
          s2[0] = fmaf(y[k][e], y[k][e], s2[0]);
          s2[1] = fmaf(dz[k][e] * wn[k][e], y[k][e], s2[1]);
        }
      }
      row_sums<CFG>(s2, red, turn);
      const float ry = 1.f / sqrtf(s2[0] * inv + a.eps);
      const float m = (s2[1] * ry) * inv;          // mean(t * yh)
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float yh = y[k][e] * ry;
          d[k][e] = fmaf(ry, fmaf(-yh, m, dz[k][e] * wn[k][e]), d[k][e]);
          Q[k][e] = fmaf(ok ? dz[k][e] : 0.f, ok ? yh : 0.f, Q[k][e]);
        }
    }
    float s3[1] = {0.f};
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float ds[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        ds[e] = a.alpha * d[k][e];
        S[k][e] = fmaf(ok ? d[k][e] : 0.f, ok ? oh[k][e] : 0.f, S[k][e]);
        d[k][e] *= wg[k][e];
        s3[0] = fmaf(d[k][e], oh[k][e], s3[0]);
      }
      if (ok && ln.col(k) < C) put<T, CFG>((T*)a.dskip + row * C + ln.col(k), narrow<T>(ds));
    }
    if (post) {
      row_sums<CFG>(s3, red, turn);
      const float m = s3[0] * inv;
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[k][e] = ro * fmaf(-oh[k][e], m, d[k][e]);
    }
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (ok && ln.col(k) < C) put<T, CFG>((T*)a.dbranch + row * C + ln.col(k), narrow<T>(d[k]));
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      ro_[k] = no_[k];
      rx_[k] = nx_[k];
      ry_[k] = ny_[k];
      rz_[k] = nz_[k];
    }
  }
  float* dst = a.part + (int64_t)blockIdx.x * 2 * C;
  store_part<CFG>(S, buf, dst, C, ln);
  store_part<CFG>(Q, buf, dst + C, C, ln);
}

// Team of a sample's partial rows among the 16-column groups of 4 lanes: all of them
// where there are more than 16 rows, else 1, 4 or 16 groups of one wave, so that few
// rows need no barrier and many samples go side by side.
constexpr int PT = 1024, NG = PT / 4;  // threads of residual_norm_params_kernel, its groups
__host__ __device__ constexpr int team_of(int P) { return P == 1 ? 1 : P <= 4 ? 4 : P <= 16 ? 16 : NG; }

// dgate and dpost_w (blockIdx.z 0) and dnorm_w (1) from the workgroups' partial rows
// [G P][2][C], 16 columns to a workgroup: 4 lanes hold 4 columns each, a team takes its
// rows in turn and adds up, always in the same order.  Many samples are split over
// gridDim.y workgroups, which leave their sums in over [gridDim.y][2][C] for
// residual_norm_split_kernel.  Bound by latency: with 64 groups, all of them on each
// sample and both sums in turn the backward pass of 16199 x 200 fp32 took 24.0 us, 19.8
// so; of 20000 samples of 2 rows of 256 bf16 491 us, 100 so.
template <typename T>
__global__ __launch_bounds__(PT) void residual_norm_params_kernel(const float* __restrict__ part, int G, int P, int C,
                                                                  const T* __restrict__ post_w, const T* __restrict__ gate,
                                                                  T* __restrict__ dpost, T* __restrict__ dgate,
                                                                  T* __restrict__ dnorm, float* __restrict__ over) {
  const int per = (G + (int)gridDim.y - 1) / (int)gridDim.y, g0 = (int)blockIdx.y * per, g1 = g0 + per < G ? g0 + per : G;
  const bool split = gridDim.y > 1;
  float* mine = over + (int64_t)blockIdx.y * 2 * C;
  __shared__ __attribute__((aligned(16))) float red[2][PT / 64][16];
  int turn = 0;
  const int cl = ((int)threadIdx.x & 3) * 4, grp = (int)threadIdx.x >> 2;
  const int c = (int)blockIdx.x * 16 + cl;
  const bool in = c < C;
  // over a team of 4 groups, over the wave's 4 of those, over the waves
  auto over4 = [](f32x4& t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = t[e];                                       // not t[e] itself: a bit cast of an element reads element 0
      x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, false));
      x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x124, 0xf, 0xf, false));
      t[e] = x;
    }
  };
  auto over16 = [](f32x4& t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = rows4_sum(t[e]);
  };
  // a buffer is written again two turns later, past the barrier of the turn between
  auto over_waves = [&](f32x4& t) {
    float(*r)[16] = red[turn & 1];
    ++turn;
    if ((threadIdx.x & 63) < 4) *reinterpret_cast<f32x4*>(&r[threadIdx.x >> 6][cl]) = t;
    __syncthreads();
    t = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < PT / 64; ++w) t += *reinterpret_cast<const f32x4*>(&r[w][cl]);
  };
  // the sum over rows p0, p0 + step .. below p1 of partial array h
  auto rows = [&](int64_t p0, int64_t p1, int step, int h) {
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
    if (in) {
#pragma unroll 4
      for (int64_t p = p0; p < p1; p += step) t += *reinterpret_cast<const f32x4*>(part + (p * 2 + h) * C + c);
    }
    return t;
  };
  if (blockIdx.z == 1) {
    if (dnorm == nullptr) return;
    f32x4 q = rows((int64_t)g0 * P + grp, (int64_t)(g1 > g0 ? g1 : g0) * P, NG, 1);
    over4(q);
    over16(q);
    over_waves(q);
    if (grp != 0 || !in) return;
    const float v[4] = {q[0], q[1], q[2], q[3]};
    if (split) store4<float>(mine + C + c, v);
    else store4<T>(dnorm + c, v);
    return;
  }
  if (dpost == nullptr && dgate == nullptr) return;
  const int team = team_of(P), at = grp % team;
  float w[4] = {1.f, 1.f, 1.f, 1.f};
  f32x4 dp = {0.f, 0.f, 0.f, 0.f};
  if (post_w != nullptr && in) load4<T>(post_w + c, w);
  for (int gb = g0; gb < g1; gb += NG / team) {
    const int g = gb + grp / team;
    f32x4 s = g < g1 ? rows((int64_t)g * P + at, (int64_t)(g + 1) * P, team, 0) : f32x4{0.f, 0.f, 0.f, 0.f};
    if (team >= 4) over4(s);
    if (team >= 16) over16(s);
    if (team == NG) over_waves(s);
    if (at != 0 || g >= g1 || !in) continue;
    float gt[4] = {1.f, 1.f, 1.f, 1.f}, dg[4];
    if (gate != nullptr) load4<T>(gate + (int64_t)g * C + c, gt);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dg[e] = w[e] * s[e];
      dp[e] = fmaf(gt[e], s[e], dp[e]);
    }
    if (dgate != nullptr) store4<T>(dgate + (int64_t)g * C + c, dg);
  }
  if (dpost == nullptr) return;
  if (team < NG) {                                          // over the teams; lanes that lead none hold zeros
    over4(dp);
    over16(dp);
    over_waves(dp);
  }
  if (grp != 0 || !in) return;
  const float v[4] = {dp[0], dp[1], dp[2], dp[3]};
  if (split) store4<float>(mine + c, v);
  else store4<T>(dpost + c, v);
}

// dpost_w and dnorm_w from the Y split sums, in order; a lane 4 columns of one of them.
template <typename T>
__global__ __launch_bounds__(NT) void residual_norm_split_kernel(const float* __restrict__ over, int Y, int C,
                                                                 T* __restrict__ dpost, T* __restrict__ dnorm) {
  const int i = ((int)blockIdx.x * NT + (int)threadIdx.x) * 4;
  if (i >= 2 * C) return;
  T* out = i < C ? dpost : dnorm;
  if (out == nullptr) return;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int y = 0; y < Y; ++y) t += *reinterpret_cast<const f32x4*>(over + (int64_t)y * 2 * C + i);
  const float v[4] = {t[0], t[1], t[2], t[3]};
  store4<T>(out + (i < C ? i : i - C), v);
}

// Workgroups that share the samples of the parameters' sums: one where the samples go
// side by side or are at most 3 (bf16 backward, us one / shared: 2 x 1000 x 512 11.5 /
// 12.1, 3 x 1000 x 512 14.0 / 13.3, 8 x 500 x 256 17.6 / 10.5), else as many as it takes,
// at most 64.
inline int sample_split(int64_t G, int P) {
  const int64_t side = NG / team_of(P);
  return G <= std::max<int64_t>(3, side) ? 1 : (int)std::min<int64_t>(64, (G + side - 1) / side);
}

// Workgroups of a sample: enough to fill the chip `per_cu` times over in all, each
// with at least one turn of rows.
struct Split {
  int64_t per;
  int P;
};
inline Split split_rows(int64_t R, int64_t G, int rps, int per_cu) {
  const int64_t turns = (R + rps - 1) / rps;
  const int64_t want = std::max<int64_t>(1, (256 * per_cu + G - 1) / G);
  const int64_t each = std::max<int64_t>(1, (turns + want - 1) / want);
  return {each * rps, (int)((turns + each - 1) / each)};
}

// Workgroups to a compute unit.  Forward: many, so that the last ones to finish are
// short (259200 x 512 bf16, us: 4 216, 16 208, 32 197, 128 183).  Backward: as many as
// its registers let run at once, since each leaves partial rows for the second kernel
// (bf16, us with it: 259200 x 512 2 407, 4 340, 8 340; 129600 x 1024 1 373, 2 328, 4 335).
constexpr int FWD_PER_CU = 128;
template <typename T, class CFG>
constexpr int BWD_PER_CU = CFG::CH == 1 ? 4 : (sizeof(T) == 2 ? 4 : 8) / CFG::CH;

// f(RowCfg) for the narrowest shape that holds C.
template <typename T, class F>
int with_cfg(int64_t C, F f) {
  if (C <= RowCfg<T, 16, 1>::WIDTH) return f(RowCfg<T, 16, 1>{});
  if (C <= RowCfg<T, 32, 1>::WIDTH) return f(RowCfg<T, 32, 1>{});
  if (C <= RowCfg<T, 64, 1>::WIDTH) return f(RowCfg<T, 64, 1>{});
  if (C <= RowCfg<T, 64, 2>::WIDTH) return f(RowCfg<T, 64, 2>{});
  if (C <= RowCfg<T, NT, 2>::WIDTH) return f(RowCfg<T, NT, 2>{});
  return f(RowCfg<T, NT, 4>{});
}

int check_norm(const char* what, int64_t rows, int64_t C, int64_t G, int dtype, const void* gate) {
  NSW_CHECK_ARG(dtype == NSW_DTYPE_BF16 || dtype == NSW_DTYPE_F32, "%s: unknown dtype %d", what, dtype);
  const int64_t vec = dtype == NSW_DTYPE_BF16 ? 8 : 4;
  NSW_CHECK_ARG(rows >= 0 && rows < (1LL << 40), "%s: rows=%lld out of range", what, (long long)rows);
  NSW_CHECK_ARG(C > 0 && C % vec == 0 && C <= vec * 1024, "%s: C=%lld must be a multiple of %lld, at most %lld", what,
                (long long)C, (long long)vec, (long long)(vec * 1024));
  NSW_CHECK_ARG(G >= 1 && G <= 65536 && rows % G == 0, "%s: rows=%lld must be a multiple of the gate's rows G=%lld (at most 65536)",
                what, (long long)rows, (long long)G);
  NSW_CHECK_ARG(gate != nullptr || G == 1, "%s: G=%lld without a gate", what, (long long)G);
  return NSW_OK;
}

template <typename T>
int64_t backward_parts(int64_t rows, int64_t C, int64_t G) {
  int64_t n = 0;
  with_cfg<T>(C, [&](auto cfg) {
    n = (int64_t)split_rows(rows / G, G, decltype(cfg)::RPS, BWD_PER_CU<T, decltype(cfg)>).P * G;
    return 0;
  });
  return n;
}

template <typename T>
int launch_forward(NormArgs a, int64_t rows, int64_t G, hipStream_t st) {
  if (rows == 0) return NSW_OK;
  return with_cfg<T>(a.C, [&](auto cfg) {
    using CFG = decltype(cfg);
    const Split s = split_rows(rows / G, G, CFG::RPS, FWD_PER_CU);
    a.R = rows / G; a.per = s.per; a.P = s.P;
    hipLaunchKernelGGL((residual_norm_kernel<T, CFG>), dim3((unsigned)(G * s.P)), dim3(NT), 0, st, a);
    return check_launch("nsw_residual_norm");
  });
}

template <typename T>
int launch_backward(NormArgs a, int64_t rows, int64_t G, void* dpost, void* dgate, void* dnorm, hipStream_t st) {
  const char* what = "nsw_residual_norm_backward";
  int P = 0;
  int rc = with_cfg<T>(a.C, [&](auto cfg) {
    using CFG = decltype(cfg);
    const Split s = split_rows(rows / G, G, CFG::RPS, BWD_PER_CU<T, CFG>);
    a.R = rows / G; a.per = s.per; a.P = P = s.P;
    if (rows == 0) return (int)NSW_OK;
    hipLaunchKernelGGL((residual_norm_backward_kernel<T, CFG>), dim3((unsigned)(G * s.P)), dim3(NT), 0, st, a);
    return check_launch(what);
  });
  if (rc || (!dpost && !dgate && !dnorm)) return rc;
  const int Y = sample_split(G, P);
  float* over = a.part + std::max<int64_t>((int64_t)P * G, 1) * 2 * a.C;
  hipLaunchKernelGGL((residual_norm_params_kernel<T>), dim3((unsigned)((a.C + 15) / 16), (unsigned)Y, 2), dim3(PT), 0, st, a.part,
                     (int)G, P, a.C, (const T*)a.post_w, (const T*)a.gate, (T*)dpost, (T*)dgate, (T*)dnorm, over);
  rc = check_launch(what);
  if (rc || Y == 1 || (!dpost && !dnorm)) return rc;
  hipLaunchKernelGGL((residual_norm_split_kernel<T>), dim3((unsigned)((2 * a.C / 4 + NT - 1) / NT)), dim3(NT), 0, st, over, Y,
                     a.C, (T*)dpost, (T*)dnorm);
  return check_launch(what);
}

bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p % 16) return false;
  return true;
}

}  // namespace

}  // namespace nsw

using namespace nsw;

extern "C" int nsw_residual_norm(const void* branch, const void* skip, const void* post_w, const void* gate,
                                 const void* norm_w, void* y, void* z, int64_t rows, int64_t C, int64_t G, float alpha,
                                 float eps, int dtype, void* stream) {
  const char* what = "nsw_residual_norm";
  if (int rc = check_norm(what, rows, C, G, dtype, gate)) return rc;
  NSW_CHECK_ARG(rows == 0 || (branch && skip && y), "%s: branch, skip and y are required", what);
  NSW_CHECK_ARG(rows == 0 || (norm_w != nullptr) == (z != nullptr), "%s: z is written where norm_w is given", what);
  NSW_CHECK_ARG(aligned16({branch, skip, post_w, gate, norm_w, y, z}), "%s: pointers must be 16-byte aligned", what);
  NormArgs a{};
  a.branch = branch; a.skip = skip; a.post_w = post_w; a.gate = gate; a.norm_w = norm_w;
  a.y = y; a.z = z; a.C = (int)C; a.alpha = alpha; a.eps = eps;
  return dtype == NSW_DTYPE_BF16 ? launch_forward<bf16>(a, rows, G, (hipStream_t)stream)
                                 : launch_forward<float>(a, rows, G, (hipStream_t)stream);
}

extern "C" size_t nsw_residual_norm_backward_workspace_size(int64_t rows, int64_t C, int64_t G, int dtype) {
  if (check_norm("nsw_residual_norm_backward_workspace_size", rows, C, G, dtype, &rows) != NSW_OK) return 0;
  const int64_t n = dtype == NSW_DTYPE_BF16 ? backward_parts<bf16>(rows, C, G) : backward_parts<float>(rows, C, G);
  const int64_t Y = sample_split(G, (int)(n / G));
  return (size_t)((std::max<int64_t>(n, 1) + (Y > 1 ? Y : 0)) * 2 * C) * sizeof(float);
}

extern "C" int nsw_residual_norm_backward(const void* dy, const void* dz, const void* branch, const void* skip,
                                          const void* post_w, const void* gate, const void* norm_w, void* dbranch,
                                          void* dskip, void* dpost_w, void* dgate, void* dnorm_w, int64_t rows, int64_t C,
                                          int64_t G, float alpha, float eps, int dtype, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  const char* what = "nsw_residual_norm_backward";
  if (int rc = check_norm(what, rows, C, G, dtype, gate)) return rc;
  NSW_CHECK_ARG(rows == 0 || (branch && skip && dbranch && dskip), "%s: branch, skip, dbranch and dskip are required", what);
  NSW_CHECK_ARG(rows == 0 || dy || dz, "%s: dy or dz is required", what);
  NSW_CHECK_ARG(rows == 0 || (norm_w != nullptr) == (dz != nullptr), "%s: dz and norm_w go together", what);
  NSW_CHECK_ARG((!dpost_w || post_w) && (!dgate || gate) && (!dnorm_w || norm_w),
                "%s: a gradient of a parameter that is not given", what);
  NSW_CHECK_ARG(aligned16({dy, dz, branch, skip, post_w, gate, norm_w, dbranch, dskip, dpost_w, dgate, dnorm_w, workspace}),
                "%s: pointers must be 16-byte aligned", what);
  const size_t need = nsw_residual_norm_backward_workspace_size(rows, C, G, dtype);
  NSW_CHECK_ARG(workspace != nullptr && workspace_bytes >= need, "%s: workspace of %zu bytes needed, got %zu", what, need,
                workspace ? workspace_bytes : (size_t)0);
  NormArgs a{};
  a.branch = branch; a.skip = skip; a.post_w = post_w; a.gate = gate; a.norm_w = norm_w;
  a.dy = dy; a.dz = dz; a.dbranch = dbranch; a.dskip = dskip; a.part = (float*)workspace;
  a.C = (int)C; a.alpha = alpha; a.eps = eps;
  return dtype == NSW_DTYPE_BF16 ? launch_backward<bf16>(a, rows, G, dpost_w, dgate, dnorm_w, (hipStream_t)stream)
                                 : launch_backward<float>(a, rows, G, dpost_w, dgate, dnorm_w, (hipStream_t)stream);
}
