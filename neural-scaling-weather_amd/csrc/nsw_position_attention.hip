// Window attention with a learned position bias, forward:
//
//   z_ij = scale q_i k_j + table[bucket[r(i, j)], head] + mask_ij,  o_i = softmax_j(z_ij) v_j
//
// r(i, j) the displacement between tokens i and j of a window of T x A x W tokens, a
// difference of two codes (one subtraction; the bias is then one LDS read).  A row whose
// mask leaves nothing (every z_ij = -inf) gives zeros.
//
// Windows of up to 192 tokens (fewer with 256-byte rows) go through whole_kernel, whose waves
// hold a row's logits with all keys; longer ones through forward_kernel, which steps over key
// tiles with the running maximum m and sum of each row, so any length goes (180 x 360 x 1024 of
// 9 x 18 windows, bf16: 142 us against 210 when this was chosen, 105 for the bytes at a copy's
// rate; 147 with the lost bits in the statistics).
// S^T = K Q^T puts a query on a lane, whose probabilities are then the right operand of
// O^T = V^T P^T as they lie.  Logits in units of log2 e (the factor is in the scale and in the
// bias's LDS copy), so that a probability is one subtraction and exp2.  fp32 statistics and sums; bf16: probabilities
// (at most 1) are rounded to bf16 for the product with v, and their sum is of the rounded
// ones, by a product with ones on the matrix units (the gradients' sum, in stats, is not).  stats
// keeps m and log2 of the sum apart, since their sum would lose the second where |m| is large.
#include <algorithm>
#include <cmath>

#include "nsw_position_attention.h"

namespace nsw {

int check_geom(int64_t B, int64_t T, int64_t H, int64_t W, int64_t ws0, int64_t ws1, const char* what);

namespace posattn {

namespace {

// A row's maximum and log2 of its sum.
__device__ __forceinline__ void store_stats(const Rows& stats, uint32_t at, float m, float t) {
  typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
  const f32x2 v = {m, __builtin_amdgcn_logf(t)};
  __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), stats.r, at, 0, 0);
}

// ------------------------------------------------- windows in a workgroup ---

template <typename T, int HD, int NKB> struct Whole {
  static constexpr int STEPS = (NKB + 1) / 2, KEYS = 32 * STEPS;   // 32-key steps
  static constexpr size_t KV = (size_t)2 * KEYS * Dim<T, HD>::STR * sizeof(T);
  static constexpr int BUFS = 2 * KV <= (128 << 10) ? 2 : 1;
  static constexpr size_t LDS = BUFS * KV + 2 * KEYS * sizeof(int);
  static constexpr int END = NKB <= 4 ? 0 : NKB <= 8 ? 4 : NKB <= 11 ? 8 : 11;   // first block in which a window may end (launch_hd)
};

// Windows of up to 16 NKB tokens of one head in turn.  A wave owns 16 queries and holds their
// logits with all keys, so that a row's maximum is known before its probabilities are formed,
// and, as the pairs are the same in every window, their biases too.  Logits are whole before the
// maximum is taken from them, so that the difference at the maximum is exactly 0 however large
// a bias is (products that start from the biases over the scale, a probability one multiply-add:
// infinite or 0 at biases of 1e10, and no faster, 154 us against 147).  k and v lie in LDS, loaded
// while the window before is computed, in a second buffer where it fits (one barrier a window).
// Four waves with three blocks of queries each, biases looked up: 185 us where this took 142.
// 6,400 windows of 162 tokens and one head in 147 us: 572 MB at 3.9 TB/s (a copy: 5.1), vector
// instructions 56 us of issue, matrix units 24, three waves a SIMD.  The shift is added to whole
// logits: added to the biases, two sets of them live at once, and the registers that go to
// memory make it 275 us.
template <typename T, int HD, int NKB, bool MASK>
__global__ __launch_bounds__(64 * NKB, (NKB + 3) / 4) void whole_kernel(Args a) {
  typedef Dim<T, HD> D;
  typedef Whole<T, HD, NKB> X;
  constexpr int N = 64 * NKB;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* KVs = (T*)smem;                                               // [BUFS][k rows, v rows]
  int* kinfo = (int*)(smem + X::BUFS * X::KV);                     // [2][KEYS]: without and with the shift's classes
  float* rel = (float*)(kinfo + 2 * X::KEYS);

  const int part = (int)blockIdx.x % a.NP, head = (int)blockIdx.x / a.NP;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fg = lane >> 4;
  const int L = a.L, query = 16 * wave + fr;
  const bool queries = 16 * wave < L;
  const float zs = a.scale * LOG2E;

  TileCopy<T, HD, X::KEYS, N> kc, vc;
  typename D::Frag qn[D::NS];
  auto load_window = [&](int64_t win) {
    const int n = win < a.Bw ? L : 0;
    const At at(a, win, head, (int)sizeof(T));
    kc.load(at.qkv(a.qkv, 1, 0, n), a.hd);
    vc.load(at.qkv(a.qkv, 2, 0, n), a.hd);
    const Rows q = at.qkv(a.qkv, 0, 0, n);
#pragma unroll
    for (int s = 0; s < D::NS; ++s) qn[s] = row_frag<T, HD>(q, (uint32_t)query, s, fg, a.hd);
  };
  load_window(part);
  load_rel<T>(a, head, rel);
  for (int i = tid; i < X::KEYS; i += N) {
    kinfo[i] = info_of(a, i, false);
    kinfo[X::KEYS + i] = info_of(a, i, true);
  }
  constexpr bool ONES = sizeof(T) == 2;
  typename D::TFrag ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (T)1.f;
  wg_barrier();
  // keys past the window: no weight
  f32x4 bias[NKB];
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb) {
    const int qi = info_of(a, query, false) + rel_base(a, rel);
    const int4 k = *reinterpret_cast<const int4*>(kinfo + 16 * kb + 4 * fg);
    bias[kb] = biases({qi, qi, qi, qi}, {k.x, k.y, k.z, k.w}, false);
#pragma unroll
    for (int r = 0; r < 4; ++r) bias[kb][r] = 16 * kb + 4 * fg + r < L ? bias[kb][r] : -INFINITY;
  }

  int turn = 0;
  for (int64_t win = part; win < a.Bw; win += a.NP, turn ^= 1) {
    const int wi = (int)(win % a.nW);
    const bool shifted = !MASK && wi >= a.band0;
    const Plane mask(MASK ? a.mask + (int64_t)wi * L * L : nullptr, MASK ? L : 0);
    const At at(a, win, head, (int)sizeof(T));
    T* Ks = KVs + (X::BUFS == 2 ? turn : 0) * (int)(X::KV / sizeof(T));
    T* Vs = Ks + X::KEYS * D::STR;
    if constexpr (X::BUFS == 1) wg_barrier();                      // the window before is read
    kc.store(Ks);
    vc.store(Vs);
    typename D::Frag q[D::NS];
#pragma unroll
    for (int s = 0; s < D::NS; ++s) q[s] = qn[s];
    wg_barrier();                                                  // two buffers: the window two before is read, too
    load_window(win + a.NP);
    if (!queries) continue;
    f32x4 S[NKB];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
      S[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < D::NS; ++s) S[kb] = mma(row_frag<T, HD>(Ks + (16 * kb + fr) * D::STR, s, fg), q[s], S[kb]);
      logits(S[kb], zs, bias[kb]);
      // block after block, which the registers hold (180 x 360 x 1024: 147 us, 160 in the compiler's order; with a
      // mask its own order is the faster one, 274 against 305)
      if constexpr (!MASK) __builtin_amdgcn_sched_barrier(0);
    }
    if (shifted) {
      const int qc = info_of(a, query, true);
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        const int4 k = *reinterpret_cast<const int4*>(kinfo + X::KEYS + 16 * kb + 4 * fg);
        add_shift(S[kb], {qc, qc, qc, qc}, {k.x, k.y, k.z, k.w});
      }
    }
    if constexpr (MASK) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        const f32x4 m4 = mask.get4(query, 16 * kb + 4 * fg);
#pragma unroll
        for (int r = 0; r < 4; ++r) S[kb][r] += in_units(m4[r]);
      }
      // past the window the next query's values were read
#pragma unroll
      for (int kb = X::END; kb < NKB; ++kb)
        if (16 * kb < L && 16 * kb + 16 > L) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * kb + 4 * fg + r >= L) S[kb][r] = -INFINITY;
        }
    }
    float mx = S[0][0];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, S[kb][r]);
    mx = rows4_max(mx);
    const float to = mx == -INFINITY ? 0.f : mx;
    float l = 0.f;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        S[kb][r] = __builtin_amdgcn_exp2f(S[kb][r] - to);
        l += S[kb][r];
      }
    f32x4 O[D::ND], Z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < D::ND; ++d) O[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < X::STEPS; ++ks) {
      const f32x4 none = {0.f, 0.f, 0.f, 0.f};
      const typename D::TFrag pf = pair_frag<T>(S[2 * ks], 2 * ks + 1 < NKB ? S[2 * ks + 1 < NKB ? 2 * ks + 1 : 0] : none);
#pragma unroll
      for (int d = 0; d < D::ND; ++d) O[d] = mma(col_frag<T, D::STR>(Vs + 32 * ks * D::STR, 16 * d, fr, fg), pf, O[d]);
      if constexpr (ONES) Z = mma(ones, pf, Z);
    }
    const float sum = rows4_sum(l), t = ONES ? Z[0] : sum;
    const float inv = t > 0.f ? 1.f / t : t == 0.f ? 0.f : t;      // an empty row: zeros; NaN stays
    const Rows orows = at.out(a.o, 0, L);
#pragma unroll
    for (int d = 0; d < D::ND; ++d) store_quad<T, HD>(orows, (uint32_t)query, 16 * d + 4 * fg, a.hd, O[d], inv);
    const Rows srows = At::stats(a, win, head, 0, L);
#pragma unroll
    for (int d = 0; d < D::ND; ++d) store_lost<T, HD>(srows, (uint32_t)query, 16 * d + 4 * fg, a.hd, O[d], inv);
    store_stats(srows, fg == 0 ? (uint32_t)query * srows.ldb : NOWHERE, mx, sum);
  }
}

// ---------------------------------------------------------- longer windows ---

constexpr int WAVES = 8;                                           // of forward_kernel, 16 queries each
constexpr int64_t MOST_BLOCKS = 1 << 23;                           // a launch has fewer than 2^32 lanes

// A workgroup takes 128 queries of a (window, head) over 64-key tiles, the next tile in
// registers meanwhile, two workgroups a compute unit (2 x 1999 tokens, 8 heads of 64, bf16: 45 us
// where four waves of 32 queries took 78; 55 with the unrounded sums and lost bits, 0.3 PFLOP/s,
// bound by vector instructions: a bias, a logit, a maximum, exp2 and a sum for each pair).
template <typename T, int HD, bool MASK>
__global__ __launch_bounds__(64 * WAVES, 2) void forward_kernel(Args a) {
  typedef Dim<T, HD> D;
  constexpr int KT = 64;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* Ks = (T*)smem;
  T* Vs = Ks + KT * D::STR;
  int* kinfo = (int*)(Vs + KT * D::STR);
  float* rel = (float*)(kinfo + KT);

  const uint32_t b = (uint32_t)xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const uint32_t item = a.dnqc.div(b);
  const int qc = (int)(b - item * (uint32_t)a.nqc);
  const int64_t win = a.dheads.div(item);
  const int head = (int)(item - (uint32_t)win * (uint32_t)a.heads);
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fg = lane >> 4;
  const int L = a.L;
  const At at(a, win, head, (int)sizeof(T));
  const int wi = (int)(win % a.nW);
  const bool shifted = !MASK && wi >= a.band0;
  const Plane mask(MASK ? a.mask + (int64_t)wi * L * L : nullptr, MASK ? L : 0);
  const int query = (qc * WAVES + wave) * 16 + fr;         // past the window: zeros

  TileCopy<T, HD, KT, 64 * WAVES> kc, vc;
  kc.load(at.qkv(a.qkv, 1, 0, L), a.hd);
  vc.load(at.qkv(a.qkv, 2, 0, L), a.hd);
  const Rows qrows = at.qkv(a.qkv, 0, 0, L);
  typename D::Frag q[D::NS];
#pragma unroll
  for (int s = 0; s < D::NS; ++s) q[s] = row_frag<T, HD>(qrows, (uint32_t)query, s, fg, a.hd);
  const int qinfo = info_of(a, query, shifted) + rel_base(a, rel);
  load_rel<T>(a, head, rel);

  const float zs = a.scale * LOG2E;
  constexpr bool ONES = sizeof(T) == 2;
  typename D::TFrag ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (T)1.f;
  f32x4 O[D::ND], Z = {0.f, 0.f, 0.f, 0.f};                // Z: the rows' sums (ONES)
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < D::ND; ++d) O[d] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int k0 = 0; k0 < L; k0 += KT) {
    if (k0) wg_barrier();                                  // the tile before is read
    kc.store(Ks);
    vc.store(Vs);
    if (tid < KT) kinfo[tid] = info_of(a, k0 + tid, shifted);
    wg_barrier();
    const int left = L - k0;                               // keys from k0 on
    kc.load(at.qkv(a.qkv, 1, k0 + KT, left - KT), a.hd);
    vc.load(at.qkv(a.qkv, 2, k0 + KT, left - KT), a.hd);
    // whole tiles without a shift run without branches between the lanes' loads and products
    auto tile = [&](auto shift, auto tail) {
      f32x4 S[4];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        if (!decltype(tail)::value || 16 * kb < left) {
          const int4 ki = *reinterpret_cast<const int4*>(kinfo + 16 * kb + 4 * fg);
          const int kn[4] = {ki.x, ki.y, ki.z, ki.w};
          const f32x4 bias = biases({qinfo, qinfo, qinfo, qinfo}, kn, decltype(shift)::value);
          S[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < D::NS; ++s) S[kb] = mma(row_frag<T, HD>(Ks + (16 * kb + fr) * D::STR, s, fg), q[s], S[kb]);
          logits(S[kb], zs, bias);
          if (decltype(shift)::value) add_shift(S[kb], {qinfo, qinfo, qinfo, qinfo}, kn);
          if constexpr (MASK) {
            const f32x4 m4 = mask.get4(query, k0 + 16 * kb + 4 * fg);
#pragma unroll
            for (int r = 0; r < 4; ++r) S[kb][r] += in_units(m4[r]);
          }
          if (decltype(tail)::value && 16 * kb + 16 > left) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (16 * kb + 4 * fg + r >= left) S[kb][r] = -INFINITY;
          }
        } else {
          S[kb] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        }
      }
      float mx = S[0][0];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, S[kb][r]);
      mx = fmaxf(m, rows4_max(mx));
      const float to = mx == -INFINITY ? 0.f : mx;
      const float f = __builtin_amdgcn_exp2f(m - to);
      m = mx;
      float t = 0.f;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          S[kb][r] = __builtin_amdgcn_exp2f(S[kb][r] - to);
          t += S[kb][r];
        }
      l = fmaf(l, f, t);
      Z *= f;
#pragma unroll
      for (int d = 0; d < D::ND; ++d) O[d] *= f;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        if (!decltype(tail)::value || 32 * ks < left) {
          const typename D::TFrag pf = pair_frag<T>(S[2 * ks], S[2 * ks + 1]);
#pragma unroll
          for (int d = 0; d < D::ND; ++d) O[d] = mma(col_frag<T, D::STR>(Vs + 32 * ks * D::STR, 16 * d, fr, fg), pf, O[d]);
          if constexpr (ONES) Z = mma(ones, pf, Z);
        }
    };
    if (shifted) tile(std::true_type{}, std::true_type{});
    else if (left < KT) tile(std::false_type{}, std::true_type{});
    else tile(std::false_type{}, std::false_type{});
  }
  const Rows orows = at.out(a.o, 0, L);
  const float sum = rows4_sum(l), t = ONES ? Z[0] : sum;
  const float inv = t > 0.f ? 1.f / t : t == 0.f ? 0.f : t;        // an empty row: zeros; NaN stays
#pragma unroll
  for (int d = 0; d < D::ND; ++d) store_quad<T, HD>(orows, (uint32_t)query, 16 * d + 4 * fg, a.hd, O[d], inv);
  const Rows srows = At::stats(a, win, head, 0, L);
#pragma unroll
  for (int d = 0; d < D::ND; ++d) store_lost<T, HD>(srows, (uint32_t)query, 16 * d + 4 * fg, a.hd, O[d], inv);
  store_stats(srows, fg == 0 ? (uint32_t)query * srows.ldb : NOWHERE, m, sum);
}

template <typename T, int HD>
int launch_long(Args a, hipStream_t st) {
  typedef Dim<T, HD> D;
  a.nqc = (a.L + 16 * WAVES - 1) / (16 * WAVES);
  a.dnqc = FastDiv::make((uint32_t)a.nqc);
  const int64_t grid = a.Bw * a.heads * a.nqc;
  if (grid >= MOST_BLOCKS) return set_error(NSW_ERR_INVALID, "nsw_position_attention: too large");
  const size_t lds = (size_t)2 * 64 * D::STR * sizeof(T) + 64 * sizeof(int) + (size_t)a.R * sizeof(float);
  if (a.mask != nullptr) hipLaunchKernelGGL((forward_kernel<T, HD, true>), dim3((unsigned)grid), dim3(64 * WAVES), lds, st, a);
  else hipLaunchKernelGGL((forward_kernel<T, HD, false>), dim3((unsigned)grid), dim3(64 * WAVES), lds, st, a);
  return check_launch("nsw_position_attention");
}

template <typename T, int HD, int NKB>
int launch_whole(Args a, hipStream_t st) {
  typedef Whole<T, HD, NKB> X;
  const int64_t all = 256 * (16 / NKB);                            // four waves to a SIMD, where the LDS holds as many
  const int64_t want = std::max<int64_t>(1, all / a.heads), each = (a.Bw + want - 1) / want;
  a.NP = (int)((a.Bw + each - 1) / each);
  const dim3 grid((unsigned)(a.NP * a.heads)), block(64 * NKB);
  const size_t lds = X::LDS + (size_t)a.R * sizeof(float);
  if (a.mask != nullptr) hipLaunchKernelGGL((whole_kernel<T, HD, NKB, true>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((whole_kernel<T, HD, NKB, false>), grid, block, lds, st, a);
  return check_launch("nsw_position_attention");
}

// Longest window of whole_kernel, in blocks of 64 tokens: what the LDS holds of k and v and the
// registers of twelve waves of a row.  Beyond 128 tokens 11 blocks of 16 where they suffice: what 12
// need of registers goes to memory (400 windows of 162 tokens and 16 heads: head dim 64 147 us
// against 163, 16 75 against 79, fp32 32 285 against 284, with a mask 342 against 430).
template <typename T, int HD> constexpr int MOST_WHOLE = HD * (int)sizeof(T) >= 512 ? 1 : HD * (int)sizeof(T) >= 256 ? 2 : 3;

template <typename T, int HD>
int launch_hd(const Args& a, hipStream_t st) {
  if (a.L <= 64) return launch_whole<T, HD, 4>(a, st);
  if constexpr (MOST_WHOLE<T, HD> >= 2)
    if (a.L <= 128) return launch_whole<T, HD, 8>(a, st);
  if constexpr (MOST_WHOLE<T, HD> >= 3) {
    if (a.L <= 176) return launch_whole<T, HD, 11>(a, st);
    if (a.L <= 192) return launch_whole<T, HD, 12>(a, st);
  }
  return launch_long<T, HD>(a, st);
}

template <typename T>
int launch_t(const Args& a, hipStream_t st) {
  switch (a.hd) {
    case 4: case 8: case 16: return launch_hd<T, 16>(a, st);
    case 32: return launch_hd<T, 32>(a, st);
    case 64: return launch_hd<T, 64>(a, st);
    default: return launch_hd<T, 128>(a, st);
  }
}

// The arguments of both passes, checked.
int make_args(Args& a, const char* what, int64_t Bw, int64_t L, int64_t C, int64_t heads, float scale, int64_t nb, int64_t T,
              int64_t A, int64_t W, const float* mask, int64_t nW, int64_t H_img, int64_t W_img, int64_t s0, int64_t s1, int dtype) {
  NSW_CHECK_ARG(dtype == NSW_DTYPE_BF16 || dtype == NSW_DTYPE_F32, "%s: unknown dtype %d", what, dtype);
  NSW_CHECK_ARG(Bw >= 0 && heads > 0 && C > 0 && C % heads == 0 && C % 8 == 0 && C < (1 << 18),
                "%s: Bw=%lld, C=%lld, heads=%lld (C a multiple of 8 and of heads)", what, (long long)Bw, (long long)C, (long long)heads);
  const int64_t hd = C / heads;
  NSW_CHECK_ARG(hd == 4 || hd == 8 || hd == 16 || hd == 32 || hd == 64 || hd == 128, "%s: head_dim=%lld unsupported (4, 8, 16, 32, 64, 128)",
                what, (long long)hd);
  NSW_CHECK_ARG(T > 0 && A > 0 && W > 0 && T <= MAX_R && A <= MAX_R && W <= MAX_R && L == T * A * W,
                "%s: L=%lld is not the %lld x %lld x %lld tokens of a window", what, (long long)L, (long long)T, (long long)A, (long long)W);
  const int64_t R = (2 * T - 1) * (2 * A - 1) * (2 * W - 1);
  NSW_CHECK_ARG(R <= MAX_R, "%s: %lld displacements in a window, at most %d", what, (long long)R, MAX_R);
  NSW_CHECK_ARG(nb > 0 && nb < (1 << 24), "%s: %lld buckets", what, (long long)nb);
  NSW_CHECK_ARG(std::isfinite(scale), "%s: scale=%g", what, (double)scale);
  NSW_CHECK_ARG(Bw < (1LL << 31) && Bw * heads < (1LL << 31) && (L <= 64 || Bw * heads * ((L + 127) / 128) < MOST_BLOCKS) &&
                    L * 3 * C * (int64_t)dtype_size(dtype) < (1LL << 31),
                "%s: too large", what);
  a.Bw = Bw; a.L = (int)L; a.C = (int)C; a.heads = (int)heads; a.hd = (int)hd; a.R = (int)R; a.nb = (int)nb;
  a.TW = (int)T; a.A = (int)A; a.W = (int)W; a.scale = scale;
  a.ns = dtype == NSW_DTYPE_BF16 ? 2 + (int)((hd + 7) / 8) : 2;
  a.off = (int)(((T - 1) * (2 * A - 1) + A - 1) * (2 * W - 1) + W - 1);
  a.dAW = FastDiv::make((uint32_t)(A * W)); a.dW = FastDiv::make((uint32_t)W); a.dheads = FastDiv::make((uint32_t)heads);
  a.mask = mask; a.nW = 1; a.band0 = 1; a.thr = 0;
  if (mask) {
    NSW_CHECK_ARG(nW > 0 && Bw % nW == 0 && nW < (1LL << 31), "%s: Bw=%lld not a multiple of the mask's %lld windows", what,
                  (long long)Bw, (long long)nW);
    a.nW = (int)nW; a.band0 = a.nW;
  } else if (s0 != 0 || s1 != 0) {
    if (int rc = check_geom(1, T, H_img, W_img, A, W, what)) return rc;
    NSW_CHECK_ARG(s0 >= 0 && s0 < A && s1 >= 0 && s1 < W, "%s: shift must lie in [0, window)", what);
    const int64_t across = W_img / W, n = (H_img / A) * across;
    NSW_CHECK_ARG(Bw % n == 0, "%s: Bw=%lld not a multiple of the image's %lld windows", what, (long long)Bw, (long long)n);
    a.nW = (int)n; a.band0 = (int)(n - across); a.thr = (int)(A - s0);
  }
  return NSW_OK;
}

bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p % 16) return false;
  return true;
}

}  // namespace

int launch_forward(Args a, int dtype, hipStream_t st) { return dtype == NSW_DTYPE_BF16 ? launch_t<bf16>(a, st) : launch_t<float>(a, st); }

}  // namespace posattn

}  // namespace nsw

using namespace nsw;

extern "C" int nsw_position_attention(const void* qkv, const void* table, const int32_t* buckets, const float* mask, int64_t nW_mask,
                                      void* o, float* stats, int64_t Bw, int64_t L, int64_t C, int64_t num_heads, float scale,
                                      int64_t num_buckets, int64_t T, int64_t ws0, int64_t ws1, int64_t H, int64_t W, int64_t s0,
                                      int64_t s1, int dtype, void* stream) {
  const char* what = "nsw_position_attention";
  posattn::Args a{};
  if (int rc = posattn::make_args(a, what, Bw, L, C, num_heads, scale, num_buckets, T, ws0, ws1, mask, nW_mask, H, W, s0, s1, dtype))
    return rc;
  if (Bw == 0) return NSW_OK;
  NSW_CHECK_ARG(qkv && table && buckets && o && stats, "%s: qkv, table, buckets, o and stats are required", what);
  NSW_CHECK_ARG(posattn::aligned16({qkv, o, stats}) && (uintptr_t)mask % 4 == 0 && (uintptr_t)buckets % 4 == 0,
                "%s: qkv, o and stats must be 16-byte aligned", what);
  a.qkv = qkv; a.table = table; a.buckets = buckets; a.o = o; a.stats = stats;
  return posattn::launch_forward(a, dtype, (hipStream_t)stream);
}

extern "C" size_t nsw_position_attention_backward_workspace_size(int64_t Bw, int64_t L, int64_t C, int64_t num_heads, int64_t T,
                                                                 int64_t ws0, int64_t ws1, int dtype) {
  posattn::Args a{};
  if (posattn::make_args(a, "nsw_position_attention_backward_workspace_size", Bw, L, C, num_heads, 1.f, 1, T, ws0, ws1, nullptr, 0, 0,
                         0, 0, 0, dtype))
    return 0;
  return posattn::backward_workspace(a, dtype);
}

extern "C" int nsw_position_attention_backward(const void* dout, const void* qkv, const void* o, const float* stats, const void* table,
                                               const int32_t* buckets, const float* mask, int64_t nW_mask, void* dqkv, void* dtable,
                                               int64_t Bw, int64_t L, int64_t C, int64_t num_heads, float scale, int64_t num_buckets,
                                               int64_t T, int64_t ws0, int64_t ws1, int64_t H, int64_t W, int64_t s0, int64_t s1,
                                               int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "nsw_position_attention_backward";
  posattn::Args a{};
  if (int rc = posattn::make_args(a, what, Bw, L, C, num_heads, scale, num_buckets, T, ws0, ws1, mask, nW_mask, H, W, s0, s1, dtype))
    return rc;
  NSW_CHECK_ARG(Bw == 0 || (dout && qkv && o && stats && table && buckets && dqkv),
                "%s: dout, qkv, o, stats, table, buckets and dqkv are required", what);
  NSW_CHECK_ARG(dtable == nullptr || buckets, "%s: buckets are required", what);
  NSW_CHECK_ARG(posattn::aligned16({dout, qkv, o, stats, dqkv, workspace}) && (uintptr_t)mask % 4 == 0 && (uintptr_t)buckets % 4 == 0,
                "%s: dout, qkv, o, stats, dqkv and the workspace must be 16-byte aligned", what);
  const size_t need = dtable ? posattn::backward_workspace(a, dtype) : 0;
  NSW_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need), "%s: workspace of %zu bytes needed, got %zu", what,
                need, workspace ? workspace_bytes : (size_t)0);
  a.dout = dout; a.qkv = qkv; a.out = o; a.stats = (float*)stats; a.table = table; a.buckets = buckets; a.dqkv = dqkv;
  return posattn::launch_backward(a, dtable, (float*)workspace, dtype, (hipStream_t)stream);
}
