// Gradients of the linear products: dx = dy . w, dw = dy^T . x and db = column sums
// of dy, for nsw_linear (dy given) and for nsw_gated_linear (dy formed from dh by
// EPI_GATED_GRAD).  Every operand is read as it lies: bf16 by grad_products, fp32 by the
// forward GEMM's kernel with turned operands (EPI_BATCH), dx and dw side by side in pieces
// of their contractions, the pieces' products added in a fixed order.  fp32, 16200 rows,
// 192 -> 768, kernels in a loop of passes: 76 us for the sums formed again, 144 for dx and dw
// (132 TFLOP/s of fp32 in six bf16 products a value; the matrix units busy in two thirds of the
// cycles, the vector ones, which split the operands, in four fifths), 5 for the parts; on
// transposed copies dx and dw took 40 more.
#include <algorithm>

#include "nsw_gemm_common.h"
#include "nsw_grad.h"

namespace nsw {

int gemm_gated(const void* x, const void* w, const void* bias, const void* dh, void* y, float* colsum, int64_t M,
               int64_t H, int64_t K, int act, int dtype, void* stream, const char* what);
int64_t gated_grad_parts(int64_t M, int64_t H, int64_t K, int dtype);
double gemm_f32_pair_us(const BatchOf& a, const BatchOf& b, int& tile);
int gemm_f32_pair(const BatchOf& a, const BatchOf& b, int tile, hipStream_t st, const char* what);
int grad_products(const void* dy, const void* x, const void* w, void* dx, void* dw, const ColumnSums& sums, int64_t M, int64_t N,
                  int64_t K, char* ws, hipStream_t st, const char* what);
int64_t grad_products_workspace(int64_t M, int64_t N, int64_t K);

namespace {

constexpr int NT = 256;

// Parts a by the first `na` workgroups, b by the next nb, column sums by the others.
template <typename T>
__global__ __launch_bounds__(NT) void finish_kernel(Parts a, unsigned na, Parts b, unsigned nb, ColumnSums sums, int N) {
  __shared__ __attribute__((aligned(16))) float red[32][36];
  unsigned id = blockIdx.x;
  if (id >= na + nb) {
    column_sums_block<T>(sums.part, (T*)sums.out, (int)sums.parts, N, (int)(id - na - nb), red);
    return;
  }
  const bool first = id < na;
  const Parts& p = first ? a : b;
  const int64_t i = ((int64_t)(first ? id : id - na) * NT + threadIdx.x) * 4;
  if (i >= p.n) return;
  const float* part = (const float*)p.part + i;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < p.S; ++s) t += *reinterpret_cast<const f32x4*>(part + s * p.n);
  const float v[4] = {t[0], t[1], t[2], t[3]};
  store4<T>((T*)p.out + i, v);
}

// part[b][c] = the sum of rows b per .. of x [R, C]: 32 columns to a workgroup, as
// column_sums_block.
template <typename T>
__global__ __launch_bounds__(NT) void column_parts_kernel(const T* __restrict__ x, float* __restrict__ part, int64_t R, int C,
                                                          int64_t per) {
  __shared__ __attribute__((aligned(16))) float red[32][36];
  const int cl = ((int)threadIdx.x & 7) * 4, grp = (int)threadIdx.x >> 3;
  const int c = (int)blockIdx.x * 32 + cl;
  const int64_t r0 = blockIdx.y * per, r1 = r0 + per < R ? r0 + per : R;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  if (c < C)
#pragma unroll 4
    for (int64_t r = r0 + grp; r < r1; r += 32) {
      float v[4];
      load4<T>(x + r * C + c, v);
      t += f32x4{v[0], v[1], v[2], v[3]};
    }
  *reinterpret_cast<f32x4*>(&red[grp][cl]) = t;
  __syncthreads();
  if (grp == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < 32; ++i) t += *reinterpret_cast<const f32x4*>(&red[i][cl]);
    *reinterpret_cast<f32x4*>(part + (int64_t)blockIdx.y * C + c) = t;
  }
}

int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }
int64_t column_part_rows(int64_t M) { return std::max<int64_t>(256, (M + 63) / 64); }

// fp32: how the contractions of dx (N values, pieces of Px) and dw (M rows, pieces of P)
// are cut, and the tile: by the estimated time of both side by side, whichever is asked
// for (a gradient's bits do not depend on what else is), the pieces' products written and
// read once more.  No piece of dw's operands passes the GEMM's 2 GiB; where dy does, dx
// goes in pieces of rows, by itself.
struct PlanF32 {
  int64_t S = 0, P = 0, Sx = 1, Px = 0, rows = 0;      // rows: of dx in one launch
  int tile = 0, tilex = 0;                             // of both (of dw, where they run apart), of dx apart
  bool together = true;
  PlanF32() = default;
  PlanF32(int64_t M, int64_t N, int64_t K) {
    auto pieces = [](int64_t D, int64_t step, int64_t most, int64_t s, int64_t& n) {
      auto up = [&](int64_t v) { return (v + step - 1) / step * step; };
      const int64_t p = std::min(most, std::max<int64_t>(up((D + s - 1) / s), up(64)));
      n = (D + p - 1) / p;
      return p;
    };
    const int64_t most = std::max<int64_t>(((1LL << 31) - 1) / (std::max(N, K) * 4) / 64 * 64, 64);
    rows = std::max<int64_t>(1, ((1LL << 31) - 1) / (N * 4));
    together = rows >= M;
    Px = N;
    double best = 0;
    auto next = [](int64_t s) { return s == 1 ? 2 : s & (s - 1) ? s / 3 * 4 : s / 2 * 3; };   // 1 2 3 4 6 8 12 ..
    const int64_t tiles = ((M + 63) / 64) * ((K + 127) / 128);
    for (int64_t sx = 1; sx <= (together ? 64 : 1); sx = next(sx)) {
      int64_t nx;
      const int64_t px = pieces(N, 32, N, sx, nx);
      if (nx < sx || (sx > 1 && tiles * sx > 2048)) break;   // no more pieces to be had, or enough
      const BatchOf bx{nullptr, nullptr, nullptr, M, K, px, together ? nx : 0, N, N, K, px, px * K, 0};
      for (int64_t s = 1; s <= 64; s = next(s)) {
        int64_t n;
        const int64_t p = pieces(M, 64, most, s, n);
        int t;
        const BatchOf bw{nullptr, nullptr, nullptr, N, K, p, n, M, N, K, p * N, p * K, 1};
        double us = gemm_f32_pair_us(bw, bx, t);
        if (n > 1 || nx > 1) us += 4 + (double)((n > 1 ? n * N : 0) + (nx > 1 ? nx * M : 0)) * (double)K * 8 / 4e6;
        if (S == 0 || us < best) {
          best = us;
          S = n;
          P = p;
          Sx = nx;
          Px = px;
          tile = t;
        }
        if (n < s) break;
      }
    }
    if (!together) gemm_f32_pair_us(BatchOf{nullptr, nullptr, nullptr, rows, K, N, 1, N, N, K, N, N * K, 0}, BatchOf{}, tilex);
  }
};

// Workspace of the two products and the column sums.
struct GradSpace {
  PlanF32 f;
  int64_t prodx = 0, prodw = 0, part = 0, bytes = 0;
  GradSpace(int64_t M, int64_t N, int64_t K, int64_t parts, int dtype) {
    if (dtype == NSW_DTYPE_F32) {
      f = PlanF32(M, N, K);
      prodw = prodx + align256(f.Sx > 1 ? f.Sx * M * K * 4 : 0);
      part = prodw + align256(f.S > 1 ? f.S * N * K * 4 : 0);
    } else {
      part = grad_products_workspace(M, N, K);
    }
    bytes = part + align256(parts * N * 4);
  }
};

bool bad_sizes(int64_t M, int64_t N, int64_t K, int dtype) {
  if (dtype != NSW_DTYPE_BF16 && dtype != NSW_DTYPE_F32) return true;
  const int64_t g = dtype == NSW_DTYPE_BF16 ? 32 : 16;   // one step of dx's contraction
  return M <= 0 || N <= 0 || K <= 0 || M >= (1LL << 31) || N >= (1LL << 31) || K >= (1LL << 31) || N % g || K % 16;
}

bool bad_gated_sizes(int64_t M, int64_t H, int64_t K, int dtype) {
  return H <= 0 || H >= (1LL << 30) || H % 16 || bad_sizes(M, 2 * H, K, dtype) || (dtype == NSW_DTYPE_BF16 && K % 32);
}

// fp32: both products side by side, then parts with the column sums.
int linear_grads_f32(const char* dy, const void* x, const void* w, char* dx, void* dw, const ColumnSums& sums, int64_t M,
                     int64_t N, int64_t K, const GradSpace& sp, char* ws, hipStream_t st, const char* what) {
  const PlanF32& p = sp.f;
  char* px = p.Sx > 1 ? ws + sp.prodx : dx;
  void* pw = p.S > 1 ? ws + sp.prodw : dw;
  BatchOf bx{}, bw{};
  if (dx) bx = BatchOf{dy, w, px, M, K, p.Px, p.Sx, N, N, K, p.Px, p.Px * K, 0};
  if (dw) bw = BatchOf{dy, x, pw, N, K, p.P, p.S, M, N, K, p.P * N, p.P * K, 1};
  if (dx && !p.together) {
    for (int64_t m = 0; m < M; m += p.rows) {
      bx.x = dy + m * N * 4;
      bx.y = dx + m * K * 4;
      bx.M = std::min(p.rows, M - m);
      if (int rc = gemm_f32_pair(bx, BatchOf{}, p.tilex, st, what)) return rc;
    }
    bx.batch = 0;
  }
  const bool dw_first = p.P >= p.Px;                       // the longer ones
  if (int rc = gemm_f32_pair(dw_first ? bw : bx, dw_first ? bx : bw, p.tile, st, what)) return rc;
  return finish_grads(Parts{px, dx, M * K, dx ? (int)p.Sx : 0}, Parts{pw, dw, N * K, dw ? (int)p.S : 0}, sums, N,
                      NSW_DTYPE_F32, st, what);
}

int linear_grads(const void* dy, const void* x, const void* w, void* dx, void* dw, void* db, int64_t parts, int64_t M,
                 int64_t N, int64_t K, int dtype, const GradSpace& sp, char* ws, hipStream_t st, const char* what) {
  const ColumnSums sums{(const float*)(ws + sp.part), db, parts};
  return dtype == NSW_DTYPE_BF16 ? grad_products(dy, x, w, dx, dw, sums, M, N, K, ws, st, what)
                                 : linear_grads_f32((const char*)dy, x, w, (char*)dx, dw, sums, M, N, K, sp, ws, st, what);
}

}  // namespace

int finish_grads(const Parts& a, const Parts& b, const ColumnSums& sums, int64_t N, int dtype, hipStream_t st, const char* what) {
  auto blocks = [](const Parts& p) { return p.S > 1 ? (unsigned)((p.n / 4 + NT - 1) / NT) : 0u; };
  const unsigned na = blocks(a), nb = blocks(b), ns = sums.out ? (unsigned)((N + 31) / 32) : 0u;
  if (na + nb + ns == 0) return NSW_OK;
  const dim3 grid(na + nb + ns);
  if (dtype == NSW_DTYPE_BF16) hipLaunchKernelGGL((finish_kernel<bf16>), grid, dim3(NT), 0, st, a, na, b, nb, sums, (int)N);
  else hipLaunchKernelGGL((finish_kernel<float>), grid, dim3(NT), 0, st, a, na, b, nb, sums, (int)N);
  return check_launch(what);
}

}  // namespace nsw

using namespace nsw;

extern "C" size_t nsw_linear_backward_workspace_size(int64_t M, int64_t N, int64_t K, int dtype) {
  if (bad_sizes(M, N, K, dtype)) return 0;
  const int64_t per = column_part_rows(M);
  return (size_t)GradSpace(M, N, K, (M + per - 1) / per, dtype).bytes;
}

extern "C" int nsw_linear_backward(const void* dy, const void* x, const void* w, void* dx, void* dw, void* db, int64_t M,
                                   int64_t N, int64_t K, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "nsw_linear_backward";
  NSW_CHECK_ARG(!bad_sizes(M, N, K, dtype), "%s: M=%lld, N=%lld, K=%lld in dtype %d: N and K must be multiples of 32 and 16 (bf16) / 16 (fp32)",
                what, (long long)M, (long long)N, (long long)K, dtype);
  NSW_CHECK_ARG(dy && (x || !dw) && w, "%s: dy, w and, for dw, x are required", what);
  const int64_t per = column_part_rows(M), parts = (M + per - 1) / per;
  const GradSpace sp(M, N, K, parts, dtype);
  NSW_CHECK_ARG(workspace != nullptr && workspace_bytes >= (size_t)sp.bytes, "%s: workspace of %lld bytes needed", what,
                (long long)sp.bytes);
  NSW_CHECK_ARG((((uintptr_t)dy | (uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)db |
                  (uintptr_t)workspace) % 16) == 0, "%s: pointers must be 16-byte aligned", what);
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  if (db) {
    float* part = (float*)(ws + sp.part);
    const dim3 grid((unsigned)((N + 31) / 32), (unsigned)parts);
    if (dtype == NSW_DTYPE_BF16)
      hipLaunchKernelGGL((column_parts_kernel<bf16>), grid, dim3(NT), 0, st, (const bf16*)dy, part, M, (int)N, per);
    else
      hipLaunchKernelGGL((column_parts_kernel<float>), grid, dim3(NT), 0, st, (const float*)dy, part, M, (int)N, per);
    if (int rc = check_launch(what)) return rc;
  }
  return linear_grads(dy, x, w, dx, dw, db, parts, M, N, K, dtype, sp, ws, st, what);
}

extern "C" size_t nsw_gated_linear_backward_workspace_size(int64_t M, int64_t H, int64_t K, int dtype) {
  if (bad_gated_sizes(M, H, K, dtype)) return 0;
  // dy [M, 2H] first
  return (size_t)(align256(M * 2 * H * (int64_t)dtype_size(dtype)) +
                  GradSpace(M, 2 * H, K, gated_grad_parts(M, H, K, dtype), dtype).bytes);
}

extern "C" int nsw_gated_linear_backward(const void* dh, const void* x, const void* w, const void* bias, void* dx, void* dw,
                                         void* db, int64_t M, int64_t H, int64_t K, int act, int dtype, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  const char* what = "nsw_gated_linear_backward";
  NSW_CHECK_ARG(!bad_gated_sizes(M, H, K, dtype), "%s: M=%lld, H=%lld, K=%lld in dtype %d: H must be a multiple of 16, K of 32 (bf16) / 16 (fp32)",
                what, (long long)M, (long long)H, (long long)K, dtype);
  NSW_CHECK_ARG(dh && x && w, "%s: dh, x and w are required", what);
  const int64_t parts = gated_grad_parts(M, H, K, dtype), dy_bytes = align256(M * 2 * H * (int64_t)dtype_size(dtype));
  const GradSpace sp(M, 2 * H, K, parts, dtype);
  NSW_CHECK_ARG(workspace != nullptr && workspace_bytes >= (size_t)(dy_bytes + sp.bytes), "%s: workspace of %lld bytes needed",
                what, (long long)(dy_bytes + sp.bytes));
  NSW_CHECK_ARG((((uintptr_t)dh | (uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)dx | (uintptr_t)dw |
                  (uintptr_t)db | (uintptr_t)workspace) % 16) == 0, "%s: pointers must be 16-byte aligned", what);
  NSW_CHECK_ARG(act == NSW_ACT_SILU || act == NSW_ACT_GELU || act == NSW_ACT_GELU_TANH, "%s: unknown activation %d", what, act);
  if (!dx && !dw && !db) return NSW_OK;
  char* dy = (char*)workspace;
  char* ws = dy + dy_bytes;
  int rc = gemm_gated(x, w, bias, dh, dy, db ? (float*)(ws + sp.part) : nullptr, M, H, K, act, dtype, stream, what);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  return linear_grads(dy, x, w, dx, dw, db, parts, M, 2 * H, K, dtype, sp, ws, st, what);
}
