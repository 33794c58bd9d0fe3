// Gradients of window attention with a learned position bias.  With p_ij = exp(z_ij - m_i) /
// l_i formed again from q, k and the forward pass's row statistics:
//
//   D_i = do_i o_i,  dz_ij = p_ij (do_i v_j - D_i)
//   dv_j = sum_i p_ij do_i,  dk_j = scale sum_i dz_ij q_i,  dq_i = scale sum_j dz_ij k_j
//   dtable[b, head] = sum of dz_ij over the windows and the pairs whose bucket is b
//
// keys_kernel: a wave owns KB 16-key blocks of a window (their k and v as fragments in
// registers, dk and dv in accumulators), the workgroup's four waves step together over 32-query
// tiles in LDS.  S = Q K^T puts a key on a lane, so that p and dz are the right operands of
// dv^T = do^T p and dk^T = q^T dz as they lie.  Windows that one workgroup holds (ALL) also
// form dq there: dz goes through LDS, keys by queries, and a wave takes 16 columns of dq over
// all keys, k^T in registers: five products a pair, every operand read once.  Longer windows:
// queries_kernel forms dq with p once more (two products more, no sums across workgroups).
//
// The bias's gradient is added up in LDS over all windows that a workgroup takes, of one head.
// Each group of 16 lanes has accumulators of its own: within it the keys, so the displacements,
// differ, and a wave's additions keep their order: no two lanes meet, the same bits in
// every run.  With many displacements the groups of a wave take turns in one accumulator, with
// more the waves do.  bias_sum_kernel and bias_table_kernel add the workgroups' sums and
// those of a bucket, in order.
//
// bf16: p and dz are rounded to bf16 for the products (dtable: not rounded).
#include <algorithm>

#include "nsw_position_attention.h"

namespace nsw {

namespace posattn {

namespace {

constexpr int QT = 32;              // queries of a tile

// Bytes of LDS of keys_kernel without the accumulators.
template <typename T, int HD, int KB, bool ALL>
constexpr size_t tile_bytes() {
  typedef Dim<T, HD> D;
  const size_t work = (2 * QT * D::STR + (ALL ? 64 * KB * (QT + 16 / sizeof(T)) : 0)) * sizeof(T);
  const size_t keys = ALL ? 64 * KB * D::STR * sizeof(T) : 0;      // k of the window, before the steps
  return (work > keys ? work : keys) + 4 * QT * sizeof(float);
}

template <typename T, int HD, int KB, bool ALL, bool MASK>
__global__ __launch_bounds__(NT, 1) void keys_kernel(Args a) {
  typedef Dim<T, HD> D;
  constexpr int ND = D::ND, ZS = QT + 16 / (int)sizeof(T);         // floats or bf16 of a key's dz in LDS
  constexpr int NKS = 2 * KB;                                      // 32-key steps of the workgroup's keys
  constexpr int DQ = ALL ? (2 * ND + 3) / 4 : 0;                   // 16 x 16 blocks of dq of a wave
  constexpr int KD = ALL ? (ND + 3) / 4 : 0;                       // 16-column blocks of k^T of a wave
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* Qs = (T*)smem;
  T* Gs = Qs + QT * D::STR;
  T* Zs = Gs + QT * D::STR;
  float* rows = (float*)(smem + tile_bytes<T, HD, KB, ALL>()) - 4 * QT;
  int* qinfo = (int*)rows;
  float *mrow = rows + QT, *lrow = rows + 2 * QT, *drow = rows + 3 * QT;
  float* rel = rows + 4 * QT;
  float* acc = rel + ((a.R + 3) & ~3);

  // a head's parts side by side
  const int part = (int)blockIdx.x % a.NP, kc = (int)blockIdx.x / a.NP % a.nqc, head = (int)blockIdx.x / a.NP / a.nqc;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fg = lane >> 4;
  const int L = a.L, C = a.C;
  const int64_t ld = 3 * (int64_t)C;
  const int kw = kc * 64 * KB + wave * 16 * KB;                    // the wave's first key
  const bool bias = a.part != nullptr, alone = L == 1;           // one token: p is 1 whatever z, dz exactly 0
  load_rel<T>(a, head, rel);
  if (bias)
    for (int i = tid; i < a.copies * a.RS; i += NT) acc[i] = 0.f;
  float* mine = acc + (a.copies == 16 ? (wave * 4 + fg) * a.RS : a.copies == 4 ? wave * a.RS : 0);

  for (int64_t win = part; win < a.Bw; win += a.NP) {
    const T* base = (const T*)a.qkv + win * L * ld + head * a.hd;
    T* dbase = (T*)a.dqkv + win * L * ld + head * a.hd;
    const T* gbase = (const T*)a.dout + win * L * (int64_t)C + head * a.hd;
    const T* obase = (const T*)a.out + win * L * (int64_t)C + head * a.hd;
    const f32x2* stats = (const f32x2*)a.stats + (win * a.heads + head) * L;
    const int wi = (int)(win % a.nW);
    const bool shifted = !MASK && wi >= a.band0;
    const float* mask = MASK ? a.mask + (int64_t)wi * L * L : nullptr;

    TileCopy<T, HD, QT> qc, gc, oc;
    f32x2 st = {0.f, 0.f};
    auto load_tile = [&](int q0) {
      qc.load(base + (int64_t)q0 * ld, ld, L - q0, a.hd);
      gc.load(gbase + (int64_t)q0 * C, C, L - q0, a.hd);
      oc.load(obase + (int64_t)q0 * C, C, L - q0, a.hd);
      if (tid < QT) st = q0 + tid < L ? stats[q0 + tid] : f32x2{-INFINITY, 0.f};
    };
    load_tile(0);

    typename D::Frag kf[KB][D::NS], vf[KB][D::NS];
    int kinfo[KB];
    f32x4 dk[KB][ND], dv[KB][ND];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const int key = kw + 16 * b + fr;
      kinfo[b] = info_of(a, key, shifted) - a.off;
#pragma unroll
      for (int s = 0; s < D::NS; ++s) {
        typename D::Frag z = {};
        kf[b][s] = key < L ? row_frag<T, HD>(base + (int64_t)key * ld + C, s, fg, a.hd) : z;
        vf[b][s] = key < L ? row_frag<T, HD>(base + (int64_t)key * ld + 2 * C, s, fg, a.hd) : z;
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) dk[b][d] = dv[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // k^T of the window, through LDS, for dq
    typename D::TFrag kt[ALL ? KD : 1][ALL ? NKS : 1];
    if constexpr (ALL) {
      wg_barrier();                                                // the steps of the window before are done
      TileCopy<T, HD, 64 * KB> all;
      all.load(base + C, ld, L, a.hd);
      all.store(Qs);
      wg_barrier();
#pragma unroll
      for (int i = 0; i < KD; ++i) {
        const int d = (wave + 4 * i) % ND;
#pragma unroll
        for (int s = 0; s < NKS; ++s) kt[i][s] = col_frag<T, D::STR>(Qs + 32 * s * D::STR, 16 * d, fr, fg);
      }
    }

    for (int q0 = 0; q0 < L; q0 += QT) {
      wg_barrier();                                                // the tile before (ALL: and its dz) is read
      qc.store(Qs);
      gc.store(Gs);
      row_dots<T, HD, QT>(gc, oc, drow);
      if (tid < QT) {
        qinfo[tid] = info_of(a, q0 + tid, shifted);
        mrow[tid] = st[0] == -INFINITY ? INFINITY : st[0];         // an empty row, or none: p = 0
        lrow[tid] = st[0] == -INFINITY ? 0.f : st[1];
      }
      wg_barrier();
      if (q0 + QT < L) load_tile(q0 + QT);

      f32x4 P[2][KB], Z[2][KB];                                    // queries 16 qb + 4 fg + r, key fr of block b
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        typename D::Frag qf[D::NS], gf[D::NS];
#pragma unroll
        for (int s = 0; s < D::NS; ++s) {
          qf[s] = row_frag<T, HD>(Qs + (16 * qb + fr) * D::STR, s, fg, HD);
          gf[s] = row_frag<T, HD>(Gs + (16 * qb + fr) * D::STR, s, fg, HD);
        }
        const int4 qi = *reinterpret_cast<const int4*>(qinfo + 16 * qb + 4 * fg);
        const int qn[4] = {qi.x, qi.y, qi.z, qi.w};
        const f32x4 m4 = *reinterpret_cast<const f32x4*>(mrow + 16 * qb + 4 * fg);
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(lrow + 16 * qb + 4 * fg);
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(drow + 16 * qb + 4 * fg);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          f32x4 s4 = {0.f, 0.f, 0.f, 0.f}, g4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < D::NS; ++s) {
            s4 = mma(qf[s], kf[b][s], s4);
            g4 = mma(gf[s], vf[b][s], g4);
          }
          const int key = kw + 16 * b + fr;
          int at[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            at[r] = (qn[r] - kinfo[b]) & (MAX_R - 1);
            float z = fmaf(s4[r], a.scale, rel[at[r]]);
            if constexpr (MASK) {
              const int q = q0 + 16 * qb + 4 * fg + r;
              if (q < L && key < L) z += mask[(int64_t)q * L + key];
            } else if (shifted) {
              z += (qn[r] ^ (kinfo[b] + a.off)) >> 30 ? -100.f : 0.f;
            }
            const float p = key < L ? __builtin_amdgcn_exp2f(fmaf(z - m4[r], LOG2E, -l4[r])) : 0.f;
            P[qb][b][r] = p;
            Z[qb][b][r] = alone ? 0.f : p * (g4[r] - d4[r]);
          }
          if (bias) {
            // 32-bit LDS additions without a result; the lanes of a group lie at different displacements
            auto add = [&](int r) { __hip_atomic_fetch_add(mine + at[r], Z[qb][b][r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); };
            if (a.copies == 16) {
              if (key < L) {
#pragma unroll
                for (int r = 0; r < 4; ++r) add(r);
              }
            } else if (a.copies == 4) {
#pragma unroll
              for (int g = 0; g < 4; ++g)
                if (fg == g && key < L) {
#pragma unroll
                  for (int r = 0; r < 4; ++r) add(r);
                }
            } else {
              for (int w = 0; w < 4; ++w) {
                if (w == wave) {
#pragma unroll
                  for (int g = 0; g < 4; ++g)
                    if (fg == g && key < L) {
#pragma unroll
                      for (int r = 0; r < 4; ++r) add(r);
                    }
                }
                wg_barrier();
              }
            }
          }
        }
      }
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const typename D::TFrag pf = pair_frag<T>(P[0][b], P[1][b]), zf = pair_frag<T>(Z[0][b], Z[1][b]);
        if constexpr (ALL) {
          T* zrow = Zs + (wave * 16 * KB + 16 * b + fr) * ZS + 4 * fg;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            typedef __attribute__((ext_vector_type(4))) T T4;
            *reinterpret_cast<T4*>(zrow + 16 * h) = T4{zf[4 * h], zf[4 * h + 1], zf[4 * h + 2], zf[4 * h + 3]};
          }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          dv[b][d] = mma(col_frag<T, D::STR>(Gs, 16 * d, fr, fg), pf, dv[b][d]);
          dk[b][d] = mma(col_frag<T, D::STR>(Qs, 16 * d, fr, fg), zf, dk[b][d]);
        }
      }
      if constexpr (ALL) {
        wg_barrier();                                              // dz of all keys is there
#pragma unroll
        for (int i = 0; i < DQ; ++i) {
          const int t = wave + 4 * i, d = t % ND, qb = t / ND;     // ND 1: waves 2 and 3 have none
          if (t < 2 * ND) {
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < NKS; ++s) o = mma(kt[ND > 4 ? i % KD : 0][s], col_frag<T, ZS>(Zs + 32 * s * ZS, 16 * qb, fr, fg), o);
            const int q = q0 + 16 * qb + fr;
            if (q < L) store_quad<T, HD>(dbase + (int64_t)q * ld, 16 * d + 4 * fg, a.hd, o, a.scale);
          }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const int key = kw + 16 * b + fr;
      if (key < L) {
        T* row = dbase + (int64_t)key * ld;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          store_quad<T, HD>(row + C, 16 * d + 4 * fg, a.hd, dk[b][d], a.scale);
          store_quad<T, HD>(row + 2 * C, 16 * d + 4 * fg, a.hd, dv[b][d], 1.f);
        }
      }
    }
  }
  if (bias) {
    wg_barrier();
    float* dst = a.part + (int64_t)blockIdx.x * a.R;
    for (int r = tid; r < a.R; r += NT) {
      float t = acc[r];
      for (int c = 1; c < a.copies; ++c) t += acc[c * a.RS + r];
      dst[r] = t;
    }
  }
}

// dq of QB 64-query blocks of a (window, head), over 64-key tiles, as forward_kernel.
template <typename T, int HD, int QB, bool MASK>
__global__ __launch_bounds__(NT, 2) void queries_kernel(Args a) {
  typedef Dim<T, HD> D;
  constexpr int KT = 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* Ks = (T*)smem;
  T* Vs = Ks + KT * D::STR;
  int* kinfo = (int*)(Vs + KT * D::STR);
  float* rel = (float*)(kinfo + KT);

  const uint32_t blk = (uint32_t)xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const uint32_t item = a.dnqc.div(blk);
  const int qc = (int)(blk - item * (uint32_t)a.nqc);
  const int64_t win = a.dheads.div(item);
  const int head = (int)(item - (uint32_t)win * (uint32_t)a.heads);
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fg = lane >> 4;
  const int L = a.L, C = a.C;
  const int64_t ld = 3 * (int64_t)C;
  const T* base = (const T*)a.qkv + win * L * ld + head * a.hd;
  const int wi = (int)(win % a.nW);
  const bool shifted = !MASK && wi >= a.band0;
  const float* mask = MASK ? a.mask + (int64_t)wi * L * L : nullptr;
  const int q0 = qc * 64 * QB + wave * 16;

  TileCopy<T, HD, KT> kc, vc;
  kc.load(base + C, ld, L, a.hd);
  vc.load(base + 2 * C, ld, L, a.hd);
  typename D::Frag qf[QB][D::NS], gf[QB][D::NS];
  int qinfo[QB];
  float m[QB], l2[QB], dots[QB];
  f32x4 O[QB][D::ND];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int q = q0 + 64 * i + fr, qr = q < L ? q : L - 1;
    qinfo[i] = info_of(a, qr, shifted) + a.off;
    const T* grow = (const T*)a.dout + (win * L + qr) * (int64_t)C + head * a.hd;
    const T* orow = (const T*)a.out + (win * L + qr) * (int64_t)C + head * a.hd;
    float t = 0.f;
#pragma unroll
    for (int s = 0; s < D::NS; ++s) {
      qf[i][s] = row_frag<T, HD>(base + qr * ld, s, fg, a.hd);
      gf[i][s] = row_frag<T, HD>(grow, s, fg, a.hd);
      const typename D::Frag of = row_frag<T, HD>(orow, s, fg, a.hd);
#pragma unroll
      for (int e = 0; e < D::EL; ++e) t = fmaf((float)gf[i][s][e], (float)of[e], t);
    }
    dots[i] = rows4_sum(t);
    const f32x2 st = ((const f32x2*)a.stats)[(win * a.heads + head) * L + qr];
    m[i] = st[0] == -INFINITY ? INFINITY : st[0];
    l2[i] = st[0] == -INFINITY ? 0.f : st[1];
#pragma unroll
    for (int d = 0; d < D::ND; ++d) O[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  load_rel<T>(a, head, rel);

  for (int k0 = 0; k0 < L; k0 += KT) {
    if (k0) wg_barrier();
    kc.store(Ks);
    vc.store(Vs);
    if (tid < KT) kinfo[tid] = info_of(a, k0 + tid, shifted);
    wg_barrier();
    const int left = L - k0;
    if (left > KT) {
      kc.load(base + (int64_t)(k0 + KT) * ld + C, ld, left - KT, a.hd);
      vc.load(base + (int64_t)(k0 + KT) * ld + 2 * C, ld, left - KT, a.hd);
    }
    f32x4 Z[QB][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      typename D::Frag kf[D::NS], vf[D::NS];
#pragma unroll
      for (int s = 0; s < D::NS; ++s) {
        kf[s] = row_frag<T, HD>(Ks + (16 * kb + fr) * D::STR, s, fg, HD);
        vf[s] = row_frag<T, HD>(Vs + (16 * kb + fr) * D::STR, s, fg, HD);
      }
      const int4 ki = *reinterpret_cast<const int4*>(kinfo + 16 * kb + 4 * fg);
      const int kn[4] = {ki.x, ki.y, ki.z, ki.w};
#pragma unroll
      for (int i = 0; i < QB; ++i) {
        f32x4 s4 = {0.f, 0.f, 0.f, 0.f}, g4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < D::NS; ++s) {
          s4 = mma(kf[s], qf[i][s], s4);
          g4 = mma(vf[s], gf[i][s], g4);
        }
        const int q = q0 + 64 * i + fr;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float z = fmaf(s4[r], a.scale, rel[(qinfo[i] - kn[r]) & (MAX_R - 1)]);
          const int key = k0 + 16 * kb + 4 * fg + r;
          if constexpr (MASK) {
            if (q < L && key < L) z += mask[(int64_t)q * L + key];
          } else if (shifted) {
            z += ((qinfo[i] - a.off) ^ kn[r]) >> 30 ? -100.f : 0.f;
          }
          const float p = key < L ? __builtin_amdgcn_exp2f(fmaf(z - m[i], LOG2E, -l2[i])) : 0.f;
          Z[i][kb][r] = p * (g4[r] - dots[i]);                   // L > 64 here
        }
      }
    }
    typename D::TFrag kf[D::ND];
#pragma unroll
    for (int d = 0; d < D::ND; ++d) kf[d] = col_frag<T, D::STR>(Ks, 16 * d, fr, fg);
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const typename D::TFrag zf = pair_frag<T>(Z[i][0], Z[i][1]);
#pragma unroll
      for (int d = 0; d < D::ND; ++d) O[i][d] = mma(kf[d], zf, O[i][d]);
    }
  }
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int q = q0 + 64 * i + fr;
    if (q < L) {
      T* row = (T*)a.dqkv + (win * L + q) * ld + head * a.hd;
#pragma unroll
      for (int d = 0; d < D::ND; ++d) store_quad<T, HD>(row, 16 * d + 4 * fg, a.hd, O[i][d], a.scale);
    }
  }
}

// sums[h, r] = the head's parts at displacement r, in order.
__global__ __launch_bounds__(NT) void bias_sum_kernel(const float* __restrict__ part, float* __restrict__ sums, int P, int R) {
  // 64 displacements to a workgroup, four groups of lanes that take every fourth part
  __shared__ float red[4][64];
  const int r = (int)blockIdx.x * 64 + ((int)threadIdx.x & 63), grp = (int)threadIdx.x >> 6;
  const float* p = part + (int64_t)blockIdx.y * P * R;
  float t = 0.f;
  if (r < R)
#pragma unroll 8
    for (int i = grp; i < P; i += 4) t += p[(int64_t)i * R + r];
  red[grp][threadIdx.x & 63] = t;
  __syncthreads();
  if (grp == 0 && r < R) sums[(int64_t)blockIdx.y * R + r] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// dtable[b, h] = sum of sums[h, r] over the displacements of bucket b, ascending: a lane a bucket.
template <typename T>
__global__ __launch_bounds__(NT) void bias_table_kernel(const float* __restrict__ sums, const int* __restrict__ buckets,
                                                        T* __restrict__ dtable, int R, int nb, int heads) {
  __shared__ __attribute__((aligned(16))) float v[1024];
  __shared__ __attribute__((aligned(16))) int at[1024];
  const int b = (int)blockIdx.x * NT + (int)threadIdx.x, h = (int)blockIdx.y;
  float t = 0.f;
  for (int r0 = 0; r0 < R; r0 += 1024) {
    __syncthreads();
    for (int i = (int)threadIdx.x; i < 1024; i += NT) {
      const int r = r0 + i;
      v[i] = r < R ? sums[(int64_t)h * R + r] : 0.f;
      at[i] = r < R ? buckets[r] : -1;
    }
    __syncthreads();
    const int n = R - r0 < 1024 ? R - r0 : 1024;
    for (int i = 0; i < n; i += 4) {
      const int4 k = *reinterpret_cast<const int4*>(at + i);
      const f32x4 x = *reinterpret_cast<const f32x4*>(v + i);
      if (k.x == b) t += x[0];
      if (k.y == b) t += x[1];
      if (k.z == b) t += x[2];
      if (k.w == b) t += x[3];
    }
  }
  if (b < nb) dtable[(int64_t)b * heads + h] = from_f32<T>(t);
}

// Key blocks of a wave in keys_kernel, and whether the workgroup holds the window.
struct KeysPlan {
  int KB;
  bool all;
};
template <typename T, int HD>
KeysPlan keys_plan(int L) {
  constexpr int MOST = HD == 128 ? (sizeof(T) == 4 ? 1 : 2) : 3;
  const int KB = L <= 64 ? 1 : MOST >= 3 && L > 128 ? 3 : MOST >= 2 ? 2 : 1;
  return {KB, L <= 64 * KB};
}

// Accumulators in LDS: one for each 16 lanes, each wave, or the workgroup, within 96 KB.
void set_copies(Args& a) {
  a.RS = (a.R + 51) / 64 * 64 + 12;                        // 12 mod 64: the groups' lanes fall in different banks
  a.copies = 16 * a.RS * 4 <= (96 << 10) ? 16 : 4 * a.RS * 4 <= (96 << 10) ? 4 : 1;
}

// Workgroups that share a head's windows: about four to a compute unit in all.
void set_parts(Args& a, int KB) {
  a.nqc = (a.L + 64 * KB - 1) / (64 * KB);
  const int64_t want = std::max<int64_t>(1, 1024 / ((int64_t)a.heads * a.nqc));
  a.NP = (int)std::min<int64_t>(std::max<int64_t>(a.Bw, 1), want);
}

template <typename F>
int with_kind(int dtype, int hd, F f) {
  auto by = [&](auto t) {
    switch (hd) {
      case 4: case 8: case 16: return f(t, std::integral_constant<int, 16>{});
      case 32: return f(t, std::integral_constant<int, 32>{});
      case 64: return f(t, std::integral_constant<int, 64>{});
      default: return f(t, std::integral_constant<int, 128>{});
    }
  };
  return dtype == NSW_DTYPE_BF16 ? by(bf16{}) : by(float{});
}

template <typename T, int HD, int KB, bool ALL>
int launch_keys(const Args& a, hipStream_t st) {
  const size_t lds = tile_bytes<T, HD, KB, ALL>() + (size_t)((a.R + 3) & ~3) * 4 + (a.part ? (size_t)a.copies * a.RS * 4 : 0);
  const dim3 grid((unsigned)(a.NP * a.nqc * a.heads));
  if (a.mask) hipLaunchKernelGGL((keys_kernel<T, HD, KB, ALL, true>), grid, dim3(NT), lds, st, a);
  else hipLaunchKernelGGL((keys_kernel<T, HD, KB, ALL, false>), grid, dim3(NT), lds, st, a);
  return check_launch("nsw_position_attention_backward");
}

template <typename T, int HD>
int launch_queries(Args a, hipStream_t st) {
  typedef Dim<T, HD> D;
  constexpr int QB = HD == 128 && sizeof(T) == 4 ? 1 : 2;
  a.nqc = (a.L + 64 * QB - 1) / (64 * QB);
  a.dnqc = FastDiv::make((uint32_t)a.nqc);
  const int64_t grid = a.Bw * a.heads * a.nqc;
  if (grid >= (1LL << 31)) return set_error(NSW_ERR_INVALID, "nsw_position_attention_backward: too large");
  const size_t lds = (size_t)2 * 32 * D::STR * sizeof(T) + 32 * sizeof(int) + (size_t)a.R * sizeof(float);
  if (a.mask) hipLaunchKernelGGL((queries_kernel<T, HD, QB, true>), dim3((unsigned)grid), dim3(NT), lds, st, a);
  else hipLaunchKernelGGL((queries_kernel<T, HD, QB, false>), dim3((unsigned)grid), dim3(NT), lds, st, a);
  return check_launch("nsw_position_attention_backward");
}

}  // namespace

size_t backward_workspace(const Args& a0, int dtype) {
  Args a = a0;
  with_kind(dtype, a.hd, [&](auto t, auto hd) {
    set_parts(a, keys_plan<decltype(t), decltype(hd)::value>(a.L).KB);
    return 0;
  });
  return (size_t)a.heads * ((size_t)a.NP * a.nqc + 1) * a.R * sizeof(float);
}

int launch_backward(Args a, void* dtable, float* workspace, int dtype, hipStream_t st) {
  const char* what = "nsw_position_attention_backward";
  return with_kind(dtype, a.hd, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    const KeysPlan p = keys_plan<T, HD>(a.L);
    set_parts(a, p.KB);
    set_copies(a);
    float* sums = workspace;                               // [heads, R], then the parts
    a.part = dtable ? workspace + (size_t)a.heads * a.R : nullptr;
    int rc = NSW_OK;
    if (a.Bw > 0) {
      if (p.KB == 1) rc = p.all ? launch_keys<T, HD, 1, true>(a, st) : launch_keys<T, HD, 1, false>(a, st);
      if constexpr (!(HD == 128 && sizeof(T) == 4))
        if (p.KB == 2) rc = p.all ? launch_keys<T, HD, 2, true>(a, st) : launch_keys<T, HD, 2, false>(a, st);
      if constexpr (HD != 128)
        if (p.KB == 3) rc = p.all ? launch_keys<T, HD, 3, true>(a, st) : launch_keys<T, HD, 3, false>(a, st);
      if (rc == NSW_OK && !p.all) rc = launch_queries<T, HD>(a, st);
    }
    if (rc || !dtable) return rc;
    const int P = a.Bw > 0 ? a.NP * a.nqc : 0;
    hipLaunchKernelGGL(bias_sum_kernel, dim3((unsigned)((a.R + 63) / 64), (unsigned)a.heads), dim3(NT), 0, st, a.part, sums, P, a.R);
    hipLaunchKernelGGL((bias_table_kernel<T>), dim3((unsigned)((a.nb + NT - 1) / NT), (unsigned)a.heads), dim3(NT), 0, st, sums,
                       a.buckets, (T*)dtable, a.R, a.nb, a.heads);
    return check_launch(what);
  });
}

}  // namespace posattn

}  // namespace nsw
