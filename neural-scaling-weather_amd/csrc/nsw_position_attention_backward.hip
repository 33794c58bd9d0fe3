// Gradients of window attention with a learned position bias.  With p_ij = exp(z_ij - m_i) /
// l_i formed again from q, k and the forward pass's row statistics:
//
//   D_i = do_i o_i,  dz_ij = p_ij (do_i v_j - D_i)
//   dv_j = sum_i p_ij do_i,  dk_j = scale sum_i dz_ij q_i,  dq_i = scale sum_j dz_ij k_j
//   dtable[b, head] = sum of dz_ij over the windows and the pairs whose bucket is b
//
// Both kernels put a key on a lane (S = Q K^T), so that p and dz are the right operands of
// dv^T = do^T p and dk^T = q^T dz as they lie.  They take the windows of one head in turn and
// add dz up over them, pair by pair, so that displacements are looked at once a workgroup and not
// once a window (float additions in LDS, one for each pair of each window, took 1100 us of
// 1795 at 400 windows of 9 x 18 and 16 heads of 64).
//
// windows_kernel, for windows of up to 16 WAVES tokens: a wave owns 16 keys (k and v in
// fragments, dk and dv in accumulators), the workgroup steps over 32-query tiles in LDS; dz
// goes through LDS, keys by queries, to the waves that form dq from it and k: five products
// a pair, every operand read once.  The sums of dz stay in registers.
//
// keys_kernel and queries_kernel, for longer ones: a wave owns KB 16-key blocks, dq comes from a
// kernel of its own that forms p once more (two products more, no sums across workgroups), the
// sums of dz are read and written in memory, each by one lane.
//
// pairs_kernel adds up the pairs of a displacement, table_kernel the displacements of a
// bucket: no atomics, the same bits in every run.
//
// bf16: p and dz are rounded to bf16 for the products (dtable: not rounded).
#include <algorithm>

#include "nsw_position_attention.h"

namespace nsw {

namespace posattn {

namespace {

constexpr int QT = 32;              // queries of a tile

// Row statistics of a tile's queries as the kernels use them: p = exp2(z - m - l), not of one
// sum m + l, which would lose l where a mask or a bias makes |m| large; rows without keys, or
// past the window, p = 0.
__device__ __forceinline__ void put_stats(const f32x2& st, float* mrow, float* lrow) {
  const bool none = st[0] == -INFINITY;
  *mrow = none ? INFINITY : st[0];
  *lrow = none ? 0.f : st[1];
}

// Statistics of query q0 + i of a window, of n queries from q0 on; none behind them.
__device__ __forceinline__ f32x2 load_stats(const Args& a, int64_t win, int head, int q0, int n, int i) {
  typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
  const Rows x = At::stats(a, win, head, q0, a.L - q0);
  const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(x.r, i < n ? (uint32_t)i * x.ldb : NOWHERE, 0, 0);
  const f32x2 st = __builtin_bit_cast(f32x2, v);
  return i < n ? st : f32x2{-INFINITY, 0.f};
}

// p and dz of four pairs from their products: s = q k, g = do v.
__device__ __forceinline__ void weigh(f32x4& s, f32x4& g, const f32x4& m, const f32x4& l, const f32x4& d) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    s[r] = __builtin_amdgcn_exp2f(s[r] - m[r] - l[r]);
    g[r] = s[r] * (g[r] - d[r]);
  }
}

template <typename T>
__device__ __forceinline__ void put4(T* p, const typename FragOf<T, 8>::type& f, int h) {
  typedef __attribute__((ext_vector_type(4))) T T4;
  *reinterpret_cast<T4*>(p) = T4{f[4 * h], f[4 * h + 1], f[4 * h + 2], f[4 * h + 3]};
}

// ------------------------------------------------- windows in a workgroup ---

template <typename T, int HD, int WAVES> struct Windows {
  typedef Dim<T, HD> D;
  static constexpr int KEYS = 16 * WAVES, STEPS = WAVES / 2;
  static constexpr int ZS = QT + (sizeof(T) == 2 ? 16 : 4);        // values of a key's dz in LDS
  static constexpr int QG = 2 * QT * D::STR;                       // a tile of q and do
  static constexpr int ZT = KEYS * ZS;
  static constexpr size_t TILES = (size_t)(2 * QG + 2 * KEYS * D::STR + 2 * ZT) * sizeof(T);
  static constexpr size_t LDS = TILES + 2 * 4 * QT * sizeof(float);
};

// 180 x 360 x 1024 of 9 x 18 windows, 16 heads, bf16: 470-500 us, 1.3 GB at 2.8 TB/s, five
// products at 0.22 PFLOP/s.  One workgroup of twelve waves a compute unit; vector instructions
// 120 us of issue, matrix units 56, the rest LDS instructions (106 thousand a compute unit in 1.1
// million cycles: every wave reads the tile of q and do twice, for 16 keys; bank conflicts are 5%
// of the cycles) and the barrier of each 32-query step.
template <typename T, int HD, int WAVES, bool MASK>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void windows_kernel(Args a) {
  typedef Dim<T, HD> D;
  typedef Windows<T, HD, WAVES> X;
  constexpr int N = 64 * WAVES, ND = D::ND;
  constexpr int TASKS = (2 * ND + WAVES - 1) / WAVES;              // 16 x 16 blocks of a tile's dq of a wave
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* QGs = (T*)smem;                                               // [2][q rows, do rows]
  T* Ks = QGs + 2 * X::QG;
  T* Vs = Ks + X::KEYS * D::STR;
  T* Zs = Vs + X::KEYS * D::STR;                                   // [2][keys]
  float* rows = (float*)(smem + X::TILES);                         // [2][infos, m, l, D]
  float* rel = rows + 2 * 4 * QT;

  const int part = (int)blockIdx.x % a.NP, head = (int)blockIdx.x / a.NP;   // a head's parts side by side
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fg = lane >> 4;
  const int L = a.L, steps = (L + QT - 1) / QT;
  const int key = 16 * wave + fr;
  const bool keys = 16 * wave < L, bias = a.part != nullptr, alone = L == 1;   // alone: p is 1 whatever z, dz exactly 0
  const float zs = a.scale * LOG2E;
  // the waves that bring in a tile's q, and its do and o: the last of them own few keys or none
  const bool bring_q = wave / 4 == (WAVES == 12 ? 2 : 0), bring_g = wave / 4 == (WAVES == 4 ? 0 : 1);
  load_rel<T>(a, head, rel);
  f32x4 sums[2 * X::STEPS];
#pragma unroll
  for (int i = 0; i < 2 * X::STEPS; ++i) sums[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (!keys) {                                                     // dz of no keys: zeros, whatever the step
    typename D::TFrag z = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) put4<T>(Zs + i / 2 * X::ZT + key * X::ZS + 16 * (i % 2) + 4 * fg, z, 0);
  }

  // what a window needs first, in registers: k, v and the first tile
  TileCopy<T, HD, X::KEYS, N> kc, vc;
  TileCopy<T, HD, QT> qc, gc, oc;
  Lost<T, HD, QT> lost;
  f32x2 st;
  // rows of the window from q0 on, n of them (none: zeros, so that nothing is kept from before)
  auto load_tile = [&](int64_t win, int q0, int n) {
    const At at(a, win, head, (int)sizeof(T));
    qc.load(at.qkv(a.qkv, 0, q0, bring_q ? n : 0), a.hd);
    gc.load(at.out(a.dout, q0, bring_g ? n : 0), a.hd);
    oc.load(at.out(a.out, q0, bring_g ? n : 0), a.hd);
    lost.load(At::stats(a, win, head, q0, bring_g ? n : 0), a.hd);
    st = load_stats(a, win, head, q0, tid < QT ? n : 0, tid);
  };
  auto load_window = [&](int64_t win) {
    const int n = win < a.Bw ? L : 0;
    const At at(a, win, head, (int)sizeof(T));
    kc.load(at.qkv(a.qkv, 1, 0, n), a.hd);
    vc.load(at.qkv(a.qkv, 2, 0, n), a.hd);
    load_tile(win, 0, n);
  };
  auto store_tile = [&](int step, bool shifted) {
    T* q = QGs + (step & 1) * X::QG;
    float* r = rows + (step & 1) * 4 * QT;
    if (bring_q) qc.store(q);
    if (bring_g) {
      gc.store(q + QT * D::STR);
      row_dots(gc, oc, lost, r + 3 * QT);
    }
    if (tid < QT) {
      ((int*)r)[tid] = info_of(a, QT * step + tid, shifted) + rel_base(a, rel);
      put_stats(st, r + QT + tid, r + 2 * QT + tid);
    }
  };

  load_window(part);
  for (int64_t win = part; win < a.Bw; win += a.NP) {
    const At at(a, win, head, (int)sizeof(T));
    const Rows dq = at.qkv(a.dqkv, 0, 0, L);
    const int wi = (int)(win % a.nW);
    const bool shifted = !MASK && wi >= a.band0;
    const Plane mask(MASK ? a.mask + (int64_t)wi * L * L : nullptr, MASK ? L : 0);
    const int kinfo = info_of(a, key, shifted);
    wg_barrier();                                                  // the window before is done with the LDS
    kc.store(Ks);
    vc.store(Vs);
    store_tile(0, shifted);
    wg_barrier();
    f32x4 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    // dq of a step's tile, from dz of all keys and k
    auto queries = [&](int step) {
      const T* z = Zs + (step & 1) * X::ZT;
#pragma unroll
      for (int i = 0; i < TASKS; ++i) {
        const int t = wave + WAVES * i, d = t % ND, qb = t / ND;
        if (t < 2 * ND) {
          f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < WAVES / 2; ++s) {
            o = mma(col_frag<T, D::STR>(Ks + 32 * s * D::STR, 16 * d, fr, fg), col_frag<T, X::ZS>(z + 32 * s * X::ZS, 16 * qb, fr, fg), o);
            if (s % 3 == 2) __builtin_amdgcn_sched_barrier(0);
          }
          store_quad<T, HD>(dq, (uint32_t)(QT * step + 16 * qb + fr), 16 * d + 4 * fg, a.hd, o, a.scale);
        }
      }
    };

#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      load_tile(win, QT * (step + 1), L - QT * (step + 1));
      if (keys) {
        const T *Qs = QGs + (step & 1) * X::QG, *Gs = Qs + QT * D::STR;
        const float* r0 = rows + (step & 1) * 4 * QT;
        f32x4 P[2], Z[2], B[2];                                    // queries 16 qb + 4 fg + r, key fr
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          P[qb] = Z[qb] = f32x4{0.f, 0.f, 0.f, 0.f};
          const int4 qi = *reinterpret_cast<const int4*>(r0 + 16 * qb + 4 * fg);
          B[qb] = biases({qi.x, qi.y, qi.z, qi.w}, {kinfo, kinfo, kinfo, kinfo}, shifted);
        }
#pragma unroll
        for (int s = 0; s < D::NS; ++s) {
          const typename D::Frag kf = row_frag<T, HD>(Ks + key * D::STR, s, fg), vf = row_frag<T, HD>(Vs + key * D::STR, s, fg);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) {
            P[qb] = mma(row_frag<T, HD>(Qs + (16 * qb + fr) * D::STR, s, fg), kf, P[qb]);
            Z[qb] = mma(row_frag<T, HD>(Gs + (16 * qb + fr) * D::STR, s, fg), vf, Z[qb]);
          }
        }
        logits(P[0], zs, B[0]);
        logits(P[1], zs, B[1]);
        if (shifted) {                                             // one branch (one a block: 180 x 360 x 1024 20 us more)
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) {
            const int4 qi = *reinterpret_cast<const int4*>(r0 + 16 * qb + 4 * fg);
            add_shift(P[qb], {qi.x, qi.y, qi.z, qi.w}, {kinfo, kinfo, kinfo, kinfo});
            asm volatile("" : "+v"(P[qb]));
          }
        }
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const f32x4 m4 = *reinterpret_cast<const f32x4*>(r0 + QT + 16 * qb + 4 * fg);
          const f32x4 l4 = *reinterpret_cast<const f32x4*>(r0 + 2 * QT + 16 * qb + 4 * fg);
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(r0 + 3 * QT + 16 * qb + 4 * fg);
          if constexpr (MASK) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              P[qb][r] += in_units(mask.get(QT * step + 16 * qb + 4 * fg + r, key));
            }
          }
          if (16 * wave + 16 > L) {
            if (key >= L) P[qb] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            asm volatile("" : "+v"(P[qb]));                        // a branch of these waves, no selects of all
          }
          weigh(P[qb], Z[qb], m4, l4, d4);
          if (alone) {
            Z[qb] = f32x4{0.f, 0.f, 0.f, 0.f};
            asm volatile("" : "+v"(Z[qb]));
          }
        }
        const typename D::TFrag pf = pair_frag<T>(P[0], P[1]), zf = pair_frag<T>(Z[0], Z[1]);
        T* z = Zs + (step & 1) * X::ZT + key * X::ZS + 4 * fg;
        put4<T>(z, zf, 0);
        put4<T>(z + 16, zf, 1);
        if (bias) {
          // the step's two sums, by branches: a register's index cannot vary
#pragma unroll
          for (int i = 0; i < X::STEPS; ++i)
            if (step == i) {
              sums[2 * i] += Z[0];
              sums[2 * i + 1] += Z[1];
              asm volatile("" : "+v"(sums[2 * i]), "+v"(sums[2 * i + 1]));   // not by selects in every step
            }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          dv[d] = mma(col_frag<T, D::STR>(Gs, 16 * d, fr, fg), pf, dv[d]);
          dk[d] = mma(col_frag<T, D::STR>(Qs, 16 * d, fr, fg), zf, dk[d]);
          if (d % 2) __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (step > 0) queries(step - 1);
      if (step + 1 < steps) store_tile(step + 1, shifted);
      wg_barrier();                                                // this step's dz and the next tile are there
    }
    load_window(win + a.NP);
    queries(steps - 1);
    const Rows dkr = at.qkv(a.dqkv, 1, 0, L), dvr = at.qkv(a.dqkv, 2, 0, L);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      store_quad<T, HD>(dkr, (uint32_t)key, 16 * d + 4 * fg, a.hd, dk[d], a.scale);
      store_quad<T, HD>(dvr, (uint32_t)key, 16 * d + 4 * fg, a.hd, dv[d], 1.f);
    }
  }
  if (bias) {
    const Plane dst(a.part + (int64_t)blockIdx.x * L * L, L);
#pragma unroll
    for (int i = 0; i < 2 * X::STEPS; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) dst.put(16 * i + 4 * fg + r, key, sums[i][r]);
  }
}

// ---------------------------------------------------------- longer windows ---

template <typename T, int HD>
constexpr size_t keys_lds() { return 2 * (2 * QT * Dim<T, HD>::STR * sizeof(T) + 4 * QT * sizeof(float)); }

// dk, dv and the sums of dz of 64 KB keys of a head, its windows in turn, over 32-query tiles in two
// buffers; two workgroups a compute unit (two frames of 90 x 180 x 512, 8 heads, with a mask, bf16:
// 848 us with one, 262 with two; 2 x 1999 tokens 158).  Bound by vector instructions and, with
// few keys a window, by the reading and writing of the sums.
// 512-byte rows: one workgroup a compute unit rather than 129 registers in memory (8 windows of
// 20 x 25 with 8 heads of 128, fp32: the pass 423 -> 360 us).
template <typename T, int HD, int KB, bool MASK>
__global__ __launch_bounds__(NT, HD * (int)sizeof(T) >= 512 ? 1 : 2) void keys_kernel(Args a) {
  typedef Dim<T, HD> D;
  constexpr int ND = D::ND, QG = 2 * QT * D::STR;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* QGs = (T*)smem;                                               // [2][q rows, do rows]
  float* rows = (float*)(QGs + 2 * QG);                            // [2][infos, m, l, D]
  float* rel = rows + 2 * 4 * QT;

  // a head's parts side by side
  const int part = (int)blockIdx.x % a.NP, kc = (int)blockIdx.x / a.NP % a.nqc, head = (int)blockIdx.x / a.NP / a.nqc;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fg = lane >> 4;
  const int L = a.L, steps = (L + QT - 1) / QT;
  const int kw = kc * 64 * KB + wave * 16 * KB;                    // the wave's first key
  const bool bias = a.part != nullptr;
  const float zs = a.scale * LOG2E;
  load_rel<T>(a, head, rel);
  const Plane sums(bias ? a.part + ((int64_t)head * a.NP + part) * L * L : nullptr, bias ? L : 0);

  for (int64_t win = part; win < a.Bw; win += a.NP) {
    const At at(a, win, head, (int)sizeof(T));
    const int wi = (int)(win % a.nW);
    const bool shifted = !MASK && wi >= a.band0;
    const Plane mask(MASK ? a.mask + (int64_t)wi * L * L : nullptr, MASK ? L : 0);

    TileCopy<T, HD, QT> qc, gc, oc;
    Lost<T, HD, QT> lost;
    f32x2 st;
    auto load_tile = [&](int q0) {
      qc.load(at.qkv(a.qkv, 0, q0, L - q0), a.hd);
      gc.load(at.out(a.dout, q0, L - q0), a.hd);
      oc.load(at.out(a.out, q0, L - q0), a.hd);
      lost.load(At::stats(a, win, head, q0, L - q0), a.hd);
      st = load_stats(a, win, head, q0, tid < QT ? L - q0 : 0, tid);
    };
    auto store_tile = [&](int step) {
      T* q = QGs + (step & 1) * QG;
      float* r = rows + (step & 1) * 4 * QT;
      qc.store(q);
      gc.store(q + QT * D::STR);
      row_dots(gc, oc, lost, r + 3 * QT);
      if (tid < QT) {
        ((int*)r)[tid] = info_of(a, QT * step + tid, shifted) + rel_base(a, rel);
        put_stats(st, r + QT + tid, r + 2 * QT + tid);
      }
    };
    load_tile(0);
    const Rows krows = at.qkv(a.qkv, 1, 0, L), vrows = at.qkv(a.qkv, 2, 0, L);
    typename D::Frag kf[KB][D::NS], vf[KB][D::NS];
    int kinfo[KB];
    f32x4 dk[KB][ND], dv[KB][ND];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const int key = kw + 16 * b + fr;                            // past the window: zeros
      kinfo[b] = info_of(a, key, shifted);
#pragma unroll
      for (int s = 0; s < D::NS; ++s) {
        kf[b][s] = row_frag<T, HD>(krows, (uint32_t)key, s, fg, a.hd);
        vf[b][s] = row_frag<T, HD>(vrows, (uint32_t)key, s, fg, a.hd);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) dk[b][d] = dv[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    wg_barrier();                                                  // the window before is done with the LDS
    store_tile(0);
    wg_barrier();

#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      const int q0 = QT * step;
      load_tile(q0 + QT);
      const T *Qs = QGs + (step & 1) * QG, *Gs = Qs + QT * D::STR;
      const float* r0 = rows + (step & 1) * 4 * QT;
      f32x4 P[2][KB], Z[2][KB];                                    // queries 16 qb + 4 fg + r, key fr of block b
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        typename D::Frag qf[D::NS], gf[D::NS];
#pragma unroll
        for (int s = 0; s < D::NS; ++s) {
          qf[s] = row_frag<T, HD>(Qs + (16 * qb + fr) * D::STR, s, fg);
          gf[s] = row_frag<T, HD>(Gs + (16 * qb + fr) * D::STR, s, fg);
        }
        const int4 qi = *reinterpret_cast<const int4*>(r0 + 16 * qb + 4 * fg);
        f32x4 B[KB], old[KB], M[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          B[b] = biases({qi.x, qi.y, qi.z, qi.w}, {kinfo[b], kinfo[b], kinfo[b], kinfo[b]}, shifted);
          if constexpr (MASK) {
#pragma unroll
            for (int r = 0; r < 4; ++r) M[b][r] = mask.get(q0 + 16 * qb + 4 * fg + r, kw + 16 * b + fr);
          }
          old[b] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (bias && win != part) {
#pragma unroll
            for (int r = 0; r < 4; ++r) old[b][r] = sums.get(q0 + 16 * qb + 4 * fg + r, kw + 16 * b + fr);
          }
        }
        const f32x4 m4 = *reinterpret_cast<const f32x4*>(r0 + QT + 16 * qb + 4 * fg);
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(r0 + 2 * QT + 16 * qb + 4 * fg);
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(r0 + 3 * QT + 16 * qb + 4 * fg);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          P[qb][b] = Z[qb][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < D::NS; ++s) {
            P[qb][b] = mma(qf[s], kf[b][s], P[qb][b]);
            Z[qb][b] = mma(gf[s], vf[b][s], Z[qb][b]);
          }
        }
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const int key = kw + 16 * b + fr;
          logits(P[qb][b], zs, B[b]);
          if (shifted) add_shift(P[qb][b], {qi.x, qi.y, qi.z, qi.w}, {kinfo[b], kinfo[b], kinfo[b], kinfo[b]});
          if constexpr (MASK) {
#pragma unroll
            for (int r = 0; r < 4; ++r) P[qb][b][r] += in_units(M[b][r]);
          }
          if (kw + 16 * b + 16 > L) {
            if (key >= L) P[qb][b] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            asm volatile("" : "+v"(P[qb][b]));                     // a branch of these waves, no selects of all
          }
          weigh(P[qb][b], Z[qb][b], m4, l4, d4);
          if (bias) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sums.put(q0 + 16 * qb + 4 * fg + r, key, old[b][r] + Z[qb][b][r]);
          }
        }
      }
      typename D::TFrag pf[KB], zf[KB];
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        pf[b] = pair_frag<T>(P[0][b], P[1][b]);
        zf[b] = pair_frag<T>(Z[0][b], Z[1][b]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const typename D::TFrag gt = col_frag<T, D::STR>(Gs, 16 * d, fr, fg), qt = col_frag<T, D::STR>(Qs, 16 * d, fr, fg);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          dv[b][d] = mma(gt, pf[b], dv[b][d]);
          dk[b][d] = mma(qt, zf[b], dk[b][d]);
        }
      }
      if (step + 1 < steps) store_tile(step + 1);
      wg_barrier();                                                // the next tile is there
    }
    const Rows dkr = at.qkv(a.dqkv, 1, 0, L), dvr = at.qkv(a.dqkv, 2, 0, L);
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        store_quad<T, HD>(dkr, (uint32_t)(kw + 16 * b + fr), 16 * d + 4 * fg, a.hd, dk[b][d], a.scale);
        store_quad<T, HD>(dvr, (uint32_t)(kw + 16 * b + fr), 16 * d + 4 * fg, a.hd, dv[b][d], 1.f);
      }
  }
}

constexpr int WQ = 8, QKT = 64;                                    // of queries_kernel: waves of 16 queries, keys of a tile

// dq of 128 queries of a (window, head), over key tiles, as the forward pass (two frames of 90 x 180
// x 512, bf16: 138 us where four waves of 32 queries took 158; 2 x 1999 tokens 54 against 69).
template <typename T, int HD, bool MASK>
__global__ __launch_bounds__(64 * WQ, HD * (int)sizeof(T) <= 128 ? 4 : 2) void queries_kernel(Args a) {
  typedef Dim<T, HD> D;
  constexpr int KT = QKT;
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
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fg = lane >> 4;
  const int L = a.L;
  const At at(a, win, head, (int)sizeof(T));
  const int wi = (int)(win % a.nW);
  const bool shifted = !MASK && wi >= a.band0;
  const Plane mask(MASK ? a.mask + (int64_t)wi * L * L : nullptr, MASK ? L : 0);
  const int query = (qc * WQ + wave) * 16 + fr;            // past the window: zeros

  TileCopy<T, HD, KT, 64 * WQ> kc, vc;
  kc.load(at.qkv(a.qkv, 1, 0, L), a.hd);
  vc.load(at.qkv(a.qkv, 2, 0, L), a.hd);
  const Rows qrows = at.qkv(a.qkv, 0, 0, L), grows = at.out(a.dout, 0, L), orows = at.out(a.out, 0, L), srows = At::stats(a, win, head, 0, L);
  typename D::Frag q[D::NS], g[D::NS];
  const int qinfo = info_of(a, query, shifted) + rel_base(a, rel);
  const float zs = a.scale * LOG2E;
  float m, l, dot = 0.f;
#pragma unroll
  for (int s = 0; s < D::NS; ++s) {
    q[s] = row_frag<T, HD>(qrows, (uint32_t)query, s, fg, a.hd);
    g[s] = row_frag<T, HD>(grows, (uint32_t)query, s, fg, a.hd);
    const typename D::Frag o = row_frag<T, HD>(orows, (uint32_t)query, s, fg, a.hd);
    if constexpr (sizeof(T) == 2) {
      const int ch = 4 * s + fg;
      const uint32_t at = HD > 16 || 8 * ch < a.hd ? (uint32_t)query * srows.ldb + 8u + 4u * ch : NOWHERE;
      const uint32_t bits = lost_word(srows, at);
#pragma unroll
      for (int e = 0; e < D::EL; ++e) dot = fmaf((float)g[s][e], found((float)o[e], bits, e), dot);
    } else {
#pragma unroll
      for (int e = 0; e < D::EL; ++e) dot = fmaf(g[s][e], o[e], dot);
    }
  }
  dot = rows4_sum(dot);
  put_stats(load_stats(a, win, head, 0, L, query), &m, &l);
  const f32x4 m4 = {m, m, m, m}, l4 = {l, l, l, l}, d4 = {dot, dot, dot, dot};
  f32x4 O[D::ND];
#pragma unroll
  for (int d = 0; d < D::ND; ++d) O[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  load_rel<T>(a, head, rel);

  for (int k0 = 0; k0 < L; k0 += KT) {
    if (k0) wg_barrier();                                  // the tile before is read
    kc.store(Ks);
    vc.store(Vs);
    if (tid < KT) kinfo[tid] = info_of(a, k0 + tid, shifted);
    wg_barrier();
    const int left = L - k0;                               // keys from k0 on
    kc.load(at.qkv(a.qkv, 1, k0 + KT, left - KT), a.hd);
    vc.load(at.qkv(a.qkv, 2, k0 + KT, left - KT), a.hd);
    auto tile = [&](auto shift, auto tail) {
#pragma unroll
      for (int ks = 0; ks < KT / 32; ++ks) {
        if (decltype(tail)::value && 32 * ks >= left) break;
        f32x4 Z[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const int k = 32 * ks + 16 * kb;
          const int4 ki = *reinterpret_cast<const int4*>(kinfo + k + 4 * fg);
          const int kn[4] = {ki.x, ki.y, ki.z, ki.w};
          const f32x4 bias = biases({qinfo, qinfo, qinfo, qinfo}, kn, decltype(shift)::value);
          f32x4 s4 = {0.f, 0.f, 0.f, 0.f}, g4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < D::NS; ++s) {
            s4 = mma(row_frag<T, HD>(Ks + (k + fr) * D::STR, s, fg), q[s], s4);
            g4 = mma(row_frag<T, HD>(Vs + (k + fr) * D::STR, s, fg), g[s], g4);
          }
          logits(s4, zs, bias);
          if (decltype(shift)::value) add_shift(s4, {qinfo, qinfo, qinfo, qinfo}, kn);
          if constexpr (MASK) {
            const f32x4 x = mask.get4(query, k0 + k + 4 * fg);
#pragma unroll
            for (int r = 0; r < 4; ++r) s4[r] += in_units(x[r]);
          }
          if (decltype(tail)::value && k + 16 > left) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (k + 4 * fg + r >= left) s4[r] = -INFINITY;
          }
          weigh(s4, g4, m4, l4, d4);
          Z[kb] = g4;
        }
        const typename D::TFrag zf = pair_frag<T>(Z[0], Z[1]);
#pragma unroll
        for (int d = 0; d < D::ND; ++d) O[d] = mma(col_frag<T, D::STR>(Ks + 32 * ks * D::STR, 16 * d, fr, fg), zf, O[d]);
      }
    };
    if (shifted) tile(std::true_type{}, std::true_type{});
    else if (left < KT) tile(std::false_type{}, std::true_type{});
    else tile(std::false_type{}, std::false_type{});
  }
  const Rows dq = at.qkv(a.dqkv, 0, 0, L);
#pragma unroll
  for (int d = 0; d < D::ND; ++d) store_quad<T, HD>(dq, (uint32_t)query, 16 * d + 4 * fg, a.hd, O[d], a.scale);
}

// Work of a workgroup of pairs_kernel: `queries` of a window's queries (a multiple of eight) and
// `parts` of the parts; `shares` of them, qshares of the queries.
struct Shares { int queries, parts, qshares, shares; };

// out[h, y, r] = sum over the pairs of displacement r whose query lies in share y's queries, and
// over its parts: a lane a displacement, neighbours on neighbouring keys, eight queries at a time
// (2 x 1999 tokens, 8 heads: 256 MB in 69 us; sixteen at a time measured the same).
__global__ __launch_bounds__(NT) void pairs_kernel(Args a, float* __restrict__ out, Shares sh) {
  constexpr int U = 8;
  const int r = (int)blockIdx.x * NT + (int)threadIdx.x, h = (int)blockIdx.y, y = (int)blockIdx.z;
  const int w2 = 2 * a.W - 1, a2 = 2 * a.A - 1;
  const int dw = r % w2 - (a.W - 1), da = r / w2 % a2 - (a.A - 1), dt = r / w2 / a2 - (a.TW - 1);
  const int back = (dt * a.A + da) * a.W + dw;             // tokens between query and key
  const int64_t LL = (int64_t)a.L * a.L;
  const int i0 = y % sh.qshares * sh.queries, i1 = i0 + sh.queries < a.L ? i0 + sh.queries : a.L;
  const int p0 = y / sh.qshares * sh.parts, p1 = p0 + sh.parts < a.NP ? p0 + sh.parts : a.NP;
  int w = i0 % a.W, i = i0 / a.W % a.A, t = i0 / (a.W * a.A);
  float s[U] = {};
  for (int q0 = i0; q0 < i1; q0 += U) {
    uint32_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = q0 + u;
      const bool there = q < i1 && r < a.R && (unsigned)(w - dw) < (unsigned)a.W && (unsigned)(i - da) < (unsigned)a.A &&
                         (unsigned)(t - dt) < (unsigned)a.TW;
      at[u] = there ? (uint32_t)(q * a.L + q - back) * 4u : NOWHERE;
      if (++w == a.W) {
        w = 0;
        if (++i == a.A) {
          i = 0;
          ++t;
        }
      }
    }
    for (int p = p0; p < p1; ++p) {
      const Plane x(a.part + ((int64_t)h * a.NP + p) * LL, a.L);
#pragma unroll
      for (int u = 0; u < U; ++u) s[u] += __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(x.r, at[u], 0, 0));
    }
  }
  if (r < a.R) out[((int64_t)h * gridDim.z + y) * a.R + r] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// dtable[b, h] = sum over the displacements of bucket b of their shares' sums: a workgroup 64
// buckets of a head, a wave a sixteenth of the displacements, ascending, the sixteenths in order.
constexpr int TT = 1024;
template <typename T>
__global__ __launch_bounds__(TT) void table_kernel(const float* __restrict__ sums, const int* __restrict__ buckets,
                                                   T* __restrict__ dtable, int R, int shares, int nb, int heads) {
  extern __shared__ __attribute__((aligned(16))) float v[];        // [Rp], then their buckets [Rp], Rp a multiple of 64
  __shared__ float red[TT / 64][64];
  const int Rp = (R + 63) / 64 * 64;
  int* at = (int*)(v + Rp);
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, b = (int)blockIdx.x * 64 + lane, h = (int)blockIdx.y;
  for (int r = (int)threadIdx.x; r < Rp; r += TT) {
    float s = 0.f;
    if (r < R)
#pragma unroll 8
      for (int y = 0; y < shares; ++y) s += sums[((int64_t)h * shares + y) * R + r];
    v[r] = s;
    at[r] = r < R ? buckets[r] : -1;
  }
  __syncthreads();
  float t[4] = {};
  for (int r = wave * (Rp / 16); r < (wave + 1) * (Rp / 16); r += 4) {
    const int4 k = *reinterpret_cast<const int4*>(at + r);
    const f32x4 x = *reinterpret_cast<const f32x4*>(v + r);
    t[0] += k.x == b ? x[0] : 0.f;
    t[1] += k.y == b ? x[1] : 0.f;
    t[2] += k.z == b ? x[2] : 0.f;
    t[3] += k.w == b ? x[3] : 0.f;
  }
  red[wave][lane] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  if (wave == 0 && b < nb) {
    float s = red[0][lane];
#pragma unroll
    for (int i = 1; i < TT / 64; ++i) s += red[i][lane];
    dtable[(int64_t)b * heads + h] = from_f32<T>(s);
  }
}

// Waves of windows_kernel for windows of L tokens; 0: longer than it takes (twelve waves do
// not hold the accumulators of 256-byte rows, the LDS not k and v of 128 rows of 512 bytes).
template <typename T, int HD> constexpr int MOST_WAVES = HD * (int)sizeof(T) >= 512 ? 4 : HD * (int)sizeof(T) >= 256 ? 8 : 12;
template <typename T, int HD>
int waves_of(int L) {
  const int w = L <= 64 ? 4 : L <= 128 ? 8 : 12;
  return L <= 192 && w <= MOST_WAVES<T, HD> ? w : 0;
}

// 16-key blocks of a wave of keys_kernel.
template <typename T, int HD> constexpr int KEY_BLOCKS = HD * (int)sizeof(T) >= 256 ? 1 : 2;

// Workgroups that share a head's windows, one at least: in all 256 times four of 4 waves, two of 8
// or one of 12 (windows_kernel; where the LDS holds fewer, from 128-byte rows on, the others
// then follow) or two (keys_kernel), each with the same number of windows as near as can be.
// Their sums of dz: 1 GiB at most, or heads L^2 floats where that is more.
void set_parts(Args& a, int waves, int keys) {
  a.nqc = waves ? 1 : (a.L + keys - 1) / keys;
  const int64_t all = waves ? 256 * (16 / waves) : 512;
  const int64_t want = std::max<int64_t>(1, all / ((int64_t)a.heads * a.nqc));
  const int64_t Bw = std::max<int64_t>(a.Bw, 1), each = (Bw + want - 1) / want;
  a.NP = (int)((Bw + each - 1) / each);
}

// Shares of pairs_kernel: up to 32 of the queries, and, while that is fewer than 1024 workgroups,
// of the parts, 64 in all (2048 windows of 7x7, four heads, 256 parts: the pass 183 -> 119 us).
Shares shares_of(const Args& a) {
  const int64_t others = (int64_t)((a.R + NT - 1) / NT) * a.heads;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(32, 2048 / others));
  Shares s;
  s.queries = (int)(((a.L + want - 1) / want + 7) / 8 * 8);
  s.qshares = (a.L + s.queries - 1) / s.queries;
  const int64_t more = std::max<int64_t>(1, std::min<int64_t>(64 / s.qshares, 1024 / (others * s.qshares)));
  s.parts = (int)((a.NP + more - 1) / more);
  s.shares = s.qshares * ((a.NP + s.parts - 1) / s.parts);
  return s;
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

template <typename T, int HD, int WAVES>
int launch_windows(const Args& a, hipStream_t st) {
  const size_t lds = Windows<T, HD, WAVES>::LDS + (size_t)a.R * sizeof(float);
  const dim3 grid((unsigned)(a.NP * a.heads));
  if (a.mask) hipLaunchKernelGGL((windows_kernel<T, HD, WAVES, true>), grid, dim3(64 * WAVES), lds, st, a);
  else hipLaunchKernelGGL((windows_kernel<T, HD, WAVES, false>), grid, dim3(64 * WAVES), lds, st, a);
  return check_launch("nsw_position_attention_backward");
}

template <typename T, int HD>
int launch_keys(const Args& a, hipStream_t st) {
  constexpr int KB = KEY_BLOCKS<T, HD>;
  const size_t lds = keys_lds<T, HD>() + (size_t)a.R * sizeof(float);
  const dim3 grid((unsigned)(a.NP * a.nqc * a.heads));
  if (a.mask) hipLaunchKernelGGL((keys_kernel<T, HD, KB, true>), grid, dim3(NT), lds, st, a);
  else hipLaunchKernelGGL((keys_kernel<T, HD, KB, false>), grid, dim3(NT), lds, st, a);
  return check_launch("nsw_position_attention_backward");
}

template <typename T, int HD>
int launch_queries(Args a, hipStream_t st) {
  typedef Dim<T, HD> D;
  a.nqc = (a.L + 16 * WQ - 1) / (16 * WQ);
  a.dnqc = FastDiv::make((uint32_t)a.nqc);
  const int64_t grid = a.Bw * a.heads * a.nqc;
  const size_t lds = (size_t)QKT * (2 * D::STR * sizeof(T) + sizeof(int)) + (size_t)a.R * sizeof(float);
  if (a.mask) hipLaunchKernelGGL((queries_kernel<T, HD, true>), dim3((unsigned)grid), dim3(64 * WQ), lds, st, a);
  else hipLaunchKernelGGL((queries_kernel<T, HD, false>), dim3((unsigned)grid), dim3(64 * WQ), lds, st, a);
  return check_launch("nsw_position_attention_backward");
}

}  // namespace

size_t backward_workspace(const Args& a0, int dtype) {
  Args a = a0;
  with_kind(dtype, a.hd, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    set_parts(a, waves_of<T, HD>(a.L), 64 * KEY_BLOCKS<T, HD>);
    return 0;
  });
  return (size_t)a.heads * ((size_t)shares_of(a).shares * a.R + (size_t)a.NP * a.L * a.L) * sizeof(float);
}

int launch_backward(Args a, void* dtable, float* workspace, int dtype, hipStream_t st) {
  const char* what = "nsw_position_attention_backward";
  return with_kind(dtype, a.hd, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    const int waves = waves_of<T, HD>(a.L);
    set_parts(a, waves, 64 * KEY_BLOCKS<T, HD>);
    const Shares sh = shares_of(a);
    float* sums = workspace;                               // [heads, shares, R], then the parts
    a.part = dtable ? workspace + (size_t)a.heads * sh.shares * a.R : nullptr;
    int rc = NSW_OK;
    if (a.Bw > 0) {
      if (waves == 4) rc = launch_windows<T, HD, 4>(a, st);
      if constexpr (MOST_WAVES<T, HD> >= 8)
        if (waves == 8) rc = launch_windows<T, HD, 8>(a, st);
      if constexpr (MOST_WAVES<T, HD> >= 12)
        if (waves == 12) rc = launch_windows<T, HD, 12>(a, st);
      if (waves == 0) {
        rc = launch_keys<T, HD>(a, st);
        if (rc == NSW_OK) rc = launch_queries<T, HD>(a, st);
      }
    }
    if (rc || !dtable) return rc;
    if (a.Bw > 0)
      hipLaunchKernelGGL(pairs_kernel, dim3((unsigned)((a.R + NT - 1) / NT), (unsigned)a.heads, (unsigned)sh.shares), dim3(NT), 0, st, a,
                         sums, sh);
    const size_t lds = (size_t)((a.R + 63) / 64 * 64) * 8;
    hipLaunchKernelGGL((table_kernel<T>), dim3((unsigned)((a.nb + 63) / 64), (unsigned)a.heads), dim3(TT), lds, st, sums, a.buckets,
                       (T*)dtable, a.R, a.Bw > 0 ? sh.shares : 0, a.nb, a.heads);
    return check_launch(what);
  });
}

}  // namespace posattn

}  // namespace nsw
