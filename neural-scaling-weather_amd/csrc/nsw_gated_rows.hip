// nsw_gated_linear for few rows, and the gradients of its sums (EPI_GATED_GRAD of the
// GEMM): the weights' bytes and the latency count.  A workgroup
// of eight waves takes 16 hidden columns (16 gate and 16 up rows of w) and 16 MB rows of
// x; the waves share out k in steps of 128 bytes of a row, operands straight from global
// memory (lane (i, g): 32 bytes of row i, so a row's 128-byte line is four lanes'
// loads), and their sums meet in LDS in a fixed order.  bf16 on v_mfma_f32_16x16x32_bf16,
// fp32 on v_mfma_f32_16x16x4_f32: any order of k serves as long as both operands have it.
#include <algorithm>
#include <type_traits>

#include "nsw_gemm_common.h"

namespace nsw {

namespace {

template <typename T, int MB, bool GRAD>
__global__ __launch_bounds__(512) void gated_rows_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                         const T* __restrict__ bias, const T* __restrict__ dh,
                                                         T* __restrict__ y, float* __restrict__ colsum, int64_t M, int H,
                                                         int K, int act) {
  constexpr int NW = 8, STEP = 128 / (int)sizeof(T);        // k of a step
  constexpr int U = MB == 4 ? 2 : 4;                        // steps whose loads are in flight together
  constexpr int PIECE = 16 / (int)sizeof(T);                // values of a 16-byte load
  __shared__ f32x4 red[NW][2][MB][64];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int i = lane & 15, g = lane >> 4, n0 = (int)blockIdx.x * 16;   // H is a multiple of 16
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MB);
  const T* wg = w + (int64_t)(n0 + i) * K;
  const T* wu = wg + (int64_t)H * K;
  const T* xp[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) xp[mb] = x + (m0 + mb * 16 + i < M ? m0 + mb * 16 + i : M - 1) * K;
  f32x4 acc[2][MB];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) acc[j][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = (K + STEP - 1) / STEP;
  // the lane's two 16-byte pieces of step s (zeros past the row's end)
  auto load = [&](const T* row, int s, u32x4 (&f)[2]) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int k = s * STEP + (2 * g + p) * PIECE;
      f[p] = u32x4{0, 0, 0, 0};
      if (k < K) f[p] = *reinterpret_cast<const u32x4*>(row + k);
    }
  };
  auto mul = [&](const u32x4 (&a)[2], const u32x4 (&b)[2], f32x4& c) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if constexpr (sizeof(T) == 2) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[p]), __builtin_bit_cast(bf16x8, b[p]), c, 0, 0, 0);
      } else {
        const f32x4 av = __builtin_bit_cast(f32x4, a[p]), bv = __builtin_bit_cast(f32x4, b[p]);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(av[e], bv[e], c, 0, 0, 0);
      }
    }
  };
  for (int s0 = wave; s0 < steps; s0 += U * NW) {
    u32x4 fg[U][2], fu[U][2], fx[U][MB][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * NW;
      if (s >= steps) break;
      load(wg, s, fg[u]);
      load(wu, s, fu[u]);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) load(xp[mb], s, fx[u][mb]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * NW >= steps) break;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        mul(fg[u], fx[u][mb], acc[0][mb]);
        mul(fu[u], fx[u][mb], acc[1][mb]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) red[wave][j][mb][lane] = acc[j][mb];
  __syncthreads();
  // lane (i, g) of row block mb holds columns n0 + 4 g + r of row m0 + mb 16 + i
  if (wave >= MB) return;
  const int64_t m = m0 + wave * 16 + i;
  const int n = n0 + 4 * g;
  if (!GRAD && m >= M) return;                              // GRAD: every lane takes part in the column sums
  f32x4 t[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    t[j] = red[0][j][wave][lane];
#pragma unroll
    for (int v = 1; v < NW; ++v) t[j] += red[v][j][wave][lane];
  }
  float b[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, o[2][4], d4[4] = {0.f, 0.f, 0.f, 0.f};
  if (bias != nullptr) {
    load4<T>(bias + n, b[0]);
    load4<T>(bias + H + n, b[1]);
  }
  if (GRAD && m < M) load4<T>(dh + m * H + n, d4);
  auto form = [&](auto f) {
    constexpr int ACT = decltype(f)::value;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float gt = t[0][e] + b[0][e], up = t[1][e] + b[1][e];
      if constexpr (GRAD) {
        float a, d;
        gate_act_grad<ACT>(gt, a, d);
        o[0][e] = d4[e] * up * d;
        o[1][e] = d4[e] * a;
      } else {
        o[0][e] = gate_act<T, ACT>(gt) * up;
      }
    }
  };
  if (act == NSW_ACT_SILU) form(std::integral_constant<int, NSW_ACT_SILU>{});
  else if (act == NSW_ACT_GELU) form(std::integral_constant<int, NSW_ACT_GELU>{});
  else form(std::integral_constant<int, NSW_ACT_GELU_TANH>{});
  if constexpr (GRAD) {
    if (m < M) {
      store4<T>(y + m * 2 * H + n, o[0]);
      store4<T>(y + m * 2 * H + H + n, o[1]);
    }
    if (colsum != nullptr) {                                // row blockIdx.y MB + wave of [.., 2H]
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f32x4 c;
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = row16_sum(m < M ? o[j][e] : 0.f);
        if (i == 0) *reinterpret_cast<f32x4*>(colsum + ((int64_t)blockIdx.y * MB + wave) * 2 * H + j * H + n) = c;
      }
    }
  } else {
    store4<T>(y + m * H + n, o[0]);
  }
}

}  // namespace

static int row_blocks(int64_t M) { return M <= 16 ? 1 : M <= 32 ? 2 : 4; }

template <typename T, bool GRAD>
static int launch_rows(const void* x, const void* w, const void* bias, const void* dh, void* y, float* colsum, int64_t M,
                       int64_t H, int64_t K, int act, hipStream_t st, const char* what) {
  const int mb = row_blocks(M);
  const dim3 grid((unsigned)(H / 16), (unsigned)((M + 16 * mb - 1) / (16 * mb))), block(512);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, block, 0, st, (const T*)x, (const T*)w, (const T*)bias, (const T*)dh, (T*)y, colsum, M,
                       (int)H, (int)K, act);
  };
  if (mb == 1) go(gated_rows_kernel<T, 1, GRAD>);
  else if (mb == 2) go(gated_rows_kernel<T, 2, GRAD>);
  else go(gated_rows_kernel<T, 4, GRAD>);
  return check_launch(what);
}

// Whether few-row workgroups are estimated faster than the GEMM (us, fits to measured
// times; silu and bias, us this kernel / the GEMM):
//   1024 -> 4096 bf16   M 1: 5.5 / 9.6    64: 9.1 / 10.0    128: 15.4 / 10.1
//   512 -> 1360 bf16    M 1: 3.5 / 6.2   128: 5.6 / 7.0     256: 9.9 / 7.1
//   1024 -> 4096 fp32   M 1: 9.8 / 43    128: 38 / 44       256: 74 / 45
// A workgroup reads its weights once more for each 64 rows; the GEMM's time is that of
// one round of small tiles, which walk the whole of k one stage at a time.
bool gated_few_rows(int64_t M, int64_t H, int64_t K, int dtype) {
  const int64_t wgs = H / 16 * ((M + 63) / 64);
  const double steps = (double)(K * (int64_t)dtype_size(dtype)) / 128;
  if (dtype == NSW_DTYPE_BF16) return std::max(2.5 + 0.35 * steps, 3 + (double)wgs * (0.004 + 0.0014 * steps)) < 4 + 0.0059 * (double)K;
  return std::max(3 + 0.5 * steps, 3 + (double)wgs * (0.004 + 0.0022 * steps)) < 6.5 + 0.0335 * (double)K;
}

// Rows of gated_rows' colsum.
int64_t gated_rows_parts(int64_t M) {
  const int64_t mb = row_blocks(M);
  return (M + 16 * mb - 1) / (16 * mb) * mb;
}

// As gemm_gated (dh and colsum NULL: forward).
int gated_rows(const void* x, const void* w, const void* bias, const void* dh, void* y, float* colsum, int64_t M, int64_t H,
               int64_t K, int act, int dtype, hipStream_t st, const char* what) {
  if (dtype == NSW_DTYPE_BF16)
    return dh ? launch_rows<bf16, true>(x, w, bias, dh, y, colsum, M, H, K, act, st, what)
              : launch_rows<bf16, false>(x, w, bias, dh, y, colsum, M, H, K, act, st, what);
  return dh ? launch_rows<float, true>(x, w, bias, dh, y, colsum, M, H, K, act, st, what)
            : launch_rows<float, false>(x, w, bias, dh, y, colsum, M, H, K, act, st, what);
}

}  // namespace nsw
