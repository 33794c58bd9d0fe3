// Gradients of the linear products: dx = dy . w, dw = dy^T . x and db = column sums
// of dy, for nsw_linear (dy given) and for nsw_gated_linear (dy formed from dh by
// EPI_GATED_GRAD).
#include <algorithm>

#include "nsw_gemm_common.h"

namespace nsw {

int gemm_gated(const void* x, const void* w, const void* bias, const void* dh, void* y, float* colsum, int64_t M,
               int64_t H, int64_t K, int act, int dtype, void* stream, const char* what);
int64_t gated_grad_parts(int64_t M, int64_t H, int64_t K, int dtype);
int gemm_plain(const void* x, const void* w, void* y, int64_t M, int64_t N, int64_t K, int dtype, void* stream,
               const char* what);

namespace {

constexpr int NT = 256;

// out[c][r] = in[r][c] for in [R, C]; rows R .. Rp of the transpose's columns are
// zeros.  64 x 64 values through LDS, 16-byte accesses on both sides (C and Rp are
// multiples of 16 bytes).
template <typename T>
__global__ __launch_bounds__(NT) void transpose_kernel(const T* __restrict__ in, T* __restrict__ out, int R, int C, int Rp) {
  constexpr int V = Vec16<T>::N, L = 64 / V;      // values of a piece, pieces of a tile row
  __shared__ T t[64][64 + (sizeof(T) == 2 ? 2 : 1)];
  const int c0 = (int)blockIdx.x * 64, r0 = (int)blockIdx.y * 64;
  const int pl = (int)threadIdx.x % L, rw = (int)threadIdx.x / L;
  for (int r = rw; r < 64; r += NT / L) {
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
    if (r0 + r < R && c0 + pl * V < C) load16<T>(in + (int64_t)(r0 + r) * C + c0 + pl * V, v);
#pragma unroll
    for (int e = 0; e < V; ++e) t[r][pl * V + e] = from_f32<T>(v[e]);
  }
  __syncthreads();
  for (int c = rw; c < 64; c += NT / L) {
    if (c0 + c >= C || r0 + pl * V >= Rp) continue;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = to_f32(t[pl * V + e][c]);
    store16<T>(out + (int64_t)(c0 + c) * Rp + r0 + pl * V, v);
  }
}

// part[b][c] = the sum of rows b per .. of x [R, C]: 32 columns to a workgroup, as
// column_sums_kernel.
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

// out[c] = sum over p of part[p][c], in a fixed order.
template <typename T>
__global__ __launch_bounds__(NT) void column_sums_kernel(const float* __restrict__ part, T* __restrict__ out, int P, int C) {
  __shared__ __attribute__((aligned(16))) float red[32][36];
  const int cl = ((int)threadIdx.x & 7) * 4, grp = (int)threadIdx.x >> 3;
  const int c = (int)blockIdx.x * 32 + cl;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  if (c < C)
#pragma unroll 4
    for (int p = grp; p < P; p += 32) t += *reinterpret_cast<const f32x4*>(part + (int64_t)p * C + c);
  *reinterpret_cast<f32x4*>(&red[grp][cl]) = t;
  __syncthreads();
  if (grp == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < 32; ++i) t += *reinterpret_cast<const f32x4*>(&red[i][cl]);
    const float v[4] = {t[0], t[1], t[2], t[3]};
    store4<T>(out + c, v);
  }
}

template <typename T>
int transpose(const void* in, void* out, int64_t R, int64_t C, int64_t Rp, hipStream_t st, const char* what) {
  const int64_t gy = (Rp + 63) / 64;
  NSW_CHECK_ARG(gy < 65536, "%s: too many rows", what);
  hipLaunchKernelGGL((transpose_kernel<T>), dim3((unsigned)((C + 63) / 64), (unsigned)gy), dim3(NT), 0, st, (const T*)in,
                     (T*)out, (int)R, (int)C, (int)Rp);
  return check_launch(what);
}

template <typename T>
int column_sums(const float* part, void* out, int64_t P, int64_t C, hipStream_t st, const char* what) {
  hipLaunchKernelGGL((column_sums_kernel<T>), dim3((unsigned)((C + 31) / 32)), dim3(NT), 0, st, part, (T*)out, (int)P, (int)C);
  return check_launch(what);
}

int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }
int64_t granule(int dtype) { return dtype == NSW_DTYPE_BF16 ? 32 : 16; }
int64_t column_part_rows(int64_t M) { return std::max<int64_t>(256, (M + 63) / 64); }

// Workspace: w^T, dy^T and x^T (rows padded to the product's step), partial column sums.
struct GradSpace {
  int64_t Mp, wt, dyt, xt, part, bytes;
  GradSpace(int64_t M, int64_t N, int64_t K, int64_t parts, int dtype) {
    const int64_t es = (int64_t)dtype_size(dtype), g = granule(dtype);
    Mp = (M + g - 1) / g * g;
    wt = 0;
    dyt = wt + align256(N * K * es);
    xt = dyt + align256(N * Mp * es);
    part = xt + align256(K * Mp * es);
    bytes = part + align256(parts * N * 4);
  }
};

bool bad_sizes(int64_t M, int64_t N, int64_t K, int dtype) {
  if (dtype != NSW_DTYPE_BF16 && dtype != NSW_DTYPE_F32) return true;
  const int64_t g = granule(dtype);
  return M <= 0 || N <= 0 || K <= 0 || M >= (1LL << 31) || N >= (1LL << 31) || K >= (1LL << 31) || N % g || K % g;
}

template <typename T>
int linear_grads(const void* dy, const void* x, const void* w, void* dx, void* dw, void* db, int64_t parts, int64_t M,
                 int64_t N, int64_t K, int dtype, char* ws, hipStream_t st, const char* what) {
  const GradSpace sp(M, N, K, parts, dtype);
  int rc = NSW_OK;
  if (dx) {
    if ((rc = transpose<T>(w, ws + sp.wt, N, K, N, st, what))) return rc;
    if ((rc = gemm_plain(dy, ws + sp.wt, dx, M, K, N, dtype, st, what))) return rc;
  }
  if (dw) {
    if ((rc = transpose<T>(dy, ws + sp.dyt, M, N, sp.Mp, st, what))) return rc;
    if ((rc = transpose<T>(x, ws + sp.xt, M, K, sp.Mp, st, what))) return rc;
    if ((rc = gemm_plain(ws + sp.dyt, ws + sp.xt, dw, N, K, sp.Mp, dtype, st, what))) return rc;
  }
  if (db) rc = column_sums<T>((const float*)(ws + sp.part), db, parts, N, st, what);
  return rc;
}

}  // namespace

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
  const size_t need = nsw_linear_backward_workspace_size(M, N, K, dtype);
  NSW_CHECK_ARG(need > 0, "%s: M=%lld, N=%lld, K=%lld in dtype %d: N and K must be multiples of 32 (bf16) / 16 (fp32)",
                what, (long long)M, (long long)N, (long long)K, dtype);
  NSW_CHECK_ARG(dy && x && w, "%s: dy, x and w are required", what);
  NSW_CHECK_ARG(workspace != nullptr && workspace_bytes >= need, "%s: workspace of %zu bytes needed", what, need);
  NSW_CHECK_ARG((((uintptr_t)dy | (uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)db |
                  (uintptr_t)workspace) % 16) == 0, "%s: pointers must be 16-byte aligned", what);
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  const int64_t per = column_part_rows(M), parts = (M + per - 1) / per;
  if (db) {
    float* part = (float*)(ws + GradSpace(M, N, K, parts, dtype).part);
    const dim3 grid((unsigned)((N + 31) / 32), (unsigned)parts);
    if (dtype == NSW_DTYPE_BF16)
      hipLaunchKernelGGL((column_parts_kernel<bf16>), grid, dim3(NT), 0, st, (const bf16*)dy, part, M, (int)N, per);
    else
      hipLaunchKernelGGL((column_parts_kernel<float>), grid, dim3(NT), 0, st, (const float*)dy, part, M, (int)N, per);
    if (int rc = check_launch(what)) return rc;
  }
  if (dtype == NSW_DTYPE_BF16) return linear_grads<bf16>(dy, x, w, dx, dw, db, parts, M, N, K, dtype, ws, st, what);
  return linear_grads<float>(dy, x, w, dx, dw, db, parts, M, N, K, dtype, ws, st, what);
}

extern "C" size_t nsw_gated_linear_backward_workspace_size(int64_t M, int64_t H, int64_t K, int dtype) {
  if (H <= 0 || H >= (1LL << 30) || H % 16 || bad_sizes(M, 2 * H, K, dtype)) return 0;
  // dy [M, 2H] first
  return (size_t)(align256(M * 2 * H * (int64_t)dtype_size(dtype)) +
                  GradSpace(M, 2 * H, K, gated_grad_parts(M, H, K, dtype), dtype).bytes);
}

extern "C" int nsw_gated_linear_backward(const void* dh, const void* x, const void* w, const void* bias, void* dx, void* dw,
                                         void* db, int64_t M, int64_t H, int64_t K, int act, int dtype, void* workspace,
                                         size_t workspace_bytes, void* stream) {
  const char* what = "nsw_gated_linear_backward";
  const size_t need = nsw_gated_linear_backward_workspace_size(M, H, K, dtype);
  NSW_CHECK_ARG(need > 0, "%s: M=%lld, H=%lld, K=%lld in dtype %d: H must be a multiple of 16, K of 32 (bf16) / 16 (fp32)",
                what, (long long)M, (long long)H, (long long)K, dtype);
  NSW_CHECK_ARG(dh && x && w, "%s: dh, x and w are required", what);
  NSW_CHECK_ARG(workspace != nullptr && workspace_bytes >= need, "%s: workspace of %zu bytes needed", what, need);
  NSW_CHECK_ARG((((uintptr_t)dh | (uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)dx | (uintptr_t)dw |
                  (uintptr_t)db | (uintptr_t)workspace) % 16) == 0, "%s: pointers must be 16-byte aligned", what);
  NSW_CHECK_ARG(act == NSW_ACT_SILU || act == NSW_ACT_GELU || act == NSW_ACT_GELU_TANH, "%s: unknown activation %d", what, act);
  if (!dx && !dw && !db) return NSW_OK;
  const int64_t parts = gated_grad_parts(M, H, K, dtype);
  char* ws = (char*)workspace;
  char* dy = ws;
  ws += align256(M * 2 * H * (int64_t)dtype_size(dtype));
  const GradSpace sp(M, 2 * H, K, parts, dtype);
  int rc = gemm_gated(x, w, bias, dh, dy, db ? (float*)(ws + sp.part) : nullptr, M, H, K, act, dtype, stream, what);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NSW_DTYPE_BF16) return linear_grads<bf16>(dy, x, w, dx, dw, db, parts, M, 2 * H, K, dtype, ws, st, what);
  return linear_grads<float>(dy, x, w, dx, dw, db, parts, M, 2 * H, K, dtype, ws, st, what);
}
