// Pieces that the linear gradients' files share.
#pragma once

#include "nsw_common.h"

namespace nsw {

// out[c] = sum over p of part[p][c] for 32 columns, in a fixed order, by 256 threads.
template <typename T>
__device__ __forceinline__ void column_sums_block(const float* __restrict__ part, T* __restrict__ out, int P, int C, int block,
                                                  float (*red)[36]) {
  const int cl = ((int)threadIdx.x & 7) * 4, grp = (int)threadIdx.x >> 3;
  const int c = block * 32 + cl;
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

// Column sums to be made of `parts` partial rows [parts, C] (out NULL: none).
struct ColumnSums {
  const float* part;
  void* out;
  int64_t parts;
};

// Parts [S][n] to add up into out [n], in order (n a multiple of 4).
struct Parts {
  const void* part;
  void* out;
  int64_t n;
  int S;
};
// The last launch of a pass: parts of a and b (none where S < 2) and the column sums [N].
int finish_grads(const Parts& a, const Parts& b, const ColumnSums& sums, int64_t N, int dtype, hipStream_t st, const char* what);

}  // namespace nsw
