// Window attention with a learned position bias: what its forward and backward kernels share.
#pragma once

#include "nsw_common.h"

namespace nsw {

namespace posattn {

constexpr int NT = 256;             // threads of a workgroup, four waves
constexpr int MAX_R = 8192;         // displacements of a window
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const void *qkv, *table, *dout, *out;
  void *o, *dqkv;
  float* stats;                     // [Bw, heads, L, 2]: row maximum m of z log2 e, log2 of the row's sum of exp2(z log2 e - m)
  const int* buckets;               // [R]
  const float* mask;                // [nW, L, L] or NULL
  float* part;                      // [heads, NP, L, L]: dz summed over the windows of a workgroup, or NULL
  int64_t Bw;
  int nW;                           // windows of the mask, or of an image
  int L, C, heads, hd, R, off, nb;
  int TW, A, W;                     // extent of a window (frames are the outermost)
  int nqc;                          // workgroups that share a window's queries (keys in the backward pass)
  int NP;                           // backward: workgroups that share a head's windows
  int band0, thr;                   // shift mask: first window of the last band (none: nW), its first row of the other class
  float scale;
  FastDiv dAW, dW, dheads, dnqc;
};

// Code of token p = (t, a, w) (past the window: of its last) in bytes of a float table:
// displacements are differences of codes.  Bit 30: the token's class under the shift mask.
__device__ __forceinline__ int info_of(const Args& a, int p, bool shifted) {
  if (p >= a.L) p = a.L - 1;
  const int t = (int)a.dAW.div((uint32_t)p), r = p - t * a.A * a.W, i = (int)a.dW.div((uint32_t)r);
  const int code = (t * (2 * a.A - 1) + i) * (2 * a.W - 1) + (r - i * a.W);
  return 4 * code | (shifted && i >= a.thr ? 1 << 30 : 0);
}

// Four logits in units of log2 e from products s: z_r = s_r zs + rel[q_r - k_r] + mask, q and k the
// infos with the middle displacement's offset added to q's, rel and the masks times log2 e.
// SHIFT: -100 between the classes.  R <= 8192 = 2^13, so that their bits fall out of the offset.
template <bool SHIFT>
__device__ __forceinline__ void logits(f32x4& s, float zs, const float* rel, const int (&q)[4], const int (&k)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int d = q[r] - k[r];
    if constexpr (SHIFT) {
      s[r] = fmaf(s[r], zs, *reinterpret_cast<const float*>((const char*)rel + (d & (4 * MAX_R - 4))));
      s[r] += (q[r] ^ k[r]) >> 30 ? -100.f * LOG2E : 0.f;
    } else {
      s[r] = fmaf(s[r], zs, *reinterpret_cast<const float*>((const char*)rel + d));
    }
  }
}

// A mask value times log2 e: the lowest floats stay finite, so that a row of them is uniform, as
// in fp32 on the formula.
__device__ __forceinline__ float mask_units(float m) {
  const float v = m * LOG2E;
  return v == -INFINITY && m != -INFINITY ? -3.402823466e38f : v;
}

// ------------------------------------------------------------- fragments ---
// Operands of D += A B with 16 x 16 results: lane (fr = lane % 16, fg = lane / 16) holds
// row fr of A or column fr of B at EL values of k of its own, and rows 4 fg .. 4 fg + 3 of
// column fr of the result.  bf16: one v_mfma_f32_16x16x32_bf16 for 32 k, 8 a lane; fp32:
// EL v_mfma_f32_16x16x4_f32, step j taking value j of each lane.  Any assignment of k to
// (fg, j) serves as long as A and B share it.
template <typename T, int EL> struct FragOf;
template <int EL> struct FragOf<bf16, EL> { typedef bf16x8 type; };
template <> struct FragOf<float, 4> { typedef f32x4 type; };
typedef __attribute__((ext_vector_type(8))) float f32x8;
template <> struct FragOf<float, 8> { typedef f32x8 type; };

__device__ __forceinline__ f32x4 mma(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const f32x8& a, const f32x8& b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f32x4 mma(const f32x4& a, const f32x4& b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// Rows of HD values (head dims below 16: 16, the rest zeros), padded in LDS: a fragment
// read of 16 rows and a transposing read of 4 rows meet few banks twice.
template <typename T, int HD_> struct Dim {
  static constexpr int HD = HD_;
  static constexpr int EPC = 16 / (int)sizeof(T);          // values of a 16-byte chunk
  static constexpr int CPR = HD / EPC;                     // chunks of a row
  static constexpr int STR = HD + (sizeof(T) == 2 ? 8 : 4);
  static constexpr int NS = HD >= 32 ? HD / 32 : 1;        // k-steps of a product over the head dim
  static constexpr int ND = HD / 16;                       // 16-wide blocks of the head dim
  static constexpr int EL = sizeof(T) == 2 || HD >= 32 ? 8 : 4;
  typedef typename FragOf<T, EL>::type Frag;               // over the head dim
  typedef typename FragOf<T, 8>::type TFrag;               // over 32 tokens
};

// 16 bytes of a row of hd values (head dim 4 in bf16: 8 bytes and zeros), zeros past its end.
// The row begins `off` bytes behind base; 32-bit offsets on one base of the wave leave the
// lanes one register for an address (a window's rows end below 4 GiB: checked by the host).
template <typename T, int HD>
__device__ __forceinline__ u32x4 load_chunk(const char* base, uint32_t off, int ch, int hd) {
  constexpr int EPC = 16 / (int)sizeof(T);
  const char* p = base + (off + 16u * (uint32_t)ch);
  if constexpr (HD > 16) {
    return *reinterpret_cast<const u32x4*>(p);
  } else {
    if ((ch + 1) * EPC <= hd) return *reinterpret_cast<const u32x4*>(p);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (ch * EPC < hd) {
      const uint64_t h = *reinterpret_cast<const uint64_t*>(p);
      v[0] = (uint32_t)h;
      v[1] = (uint32_t)(h >> 32);
    }
    return v;
  }
}

// Fragment over the head dim, k-step s, of a row in memory: bf16 values 32 s + 8 fg .., fp32 the
// same or (head dim 16) 4 fg ..
template <typename T, int HD>
__device__ __forceinline__ typename Dim<T, HD>::Frag row_frag(const char* base, uint32_t off, int s, int fg, int hd) {
  typedef typename Dim<T, HD>::Frag F;
  if constexpr (sizeof(T) == 4 && HD >= 32) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(base + (off + 128u * (uint32_t)s + 32u * (uint32_t)fg));
    const f32x4 hi = *reinterpret_cast<const f32x4*>(base + (off + 128u * (uint32_t)s + 32u * (uint32_t)fg + 16u));
    return F{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  } else {
    return __builtin_bit_cast(F, load_chunk<T, HD>(base, off, 4 * s + fg, hd));
  }
}

// The same of a row of a tile in LDS.
template <typename T, int HD>
__device__ __forceinline__ typename Dim<T, HD>::Frag row_frag(const T* row, int s, int fg) {
  typedef typename Dim<T, HD>::Frag F;
  if constexpr (sizeof(T) == 2) {
    if constexpr (HD >= 32) return *reinterpret_cast<const F*>(row + 32 * s + 8 * fg);
    const F z = {};
    return fg < 2 ? *reinterpret_cast<const F*>(row + 8 * fg) : z;
  } else if constexpr (HD >= 32) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(row + 32 * s + 8 * fg), hi = *reinterpret_cast<const f32x4*>(row + 32 * s + 8 * fg + 4);
    return F{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  } else {
    return *reinterpret_cast<const F*>(row + 4 * fg);
  }
}

// Fragment over 32 rows of a tile in LDS (stride STR), column block of 16 at col: the rows
// in the order that a pair of results holds them, j < 4 row 4 fg + j, else 16 + 4 fg + j - 4.
// bf16: two transposing reads; within a group of 16 lanes lane i addresses row 4 fg + i / 4
// at 4 (i % 4) and receives column i of rows 4 fg .. 4 fg + 3.
template <typename T, int STR>
__device__ __forceinline__ typename FragOf<T, 8>::type col_frag(const T* tile, int col, int fr, int fg) {
  if constexpr (sizeof(T) == 2) {
    typedef short i16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) i16x4* lds_ptr;
    const T* p = tile + (4 * fg + (fr >> 2)) * STR + col + 4 * (fr & 3);
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 16 * STR));
    typedef short i16x8 __attribute__((ext_vector_type(8)));
    const i16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8, v);
  } else {
    const T* p = tile + 4 * fg * STR + col + fr;
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = p[j * STR];
      v[4 + j] = p[(16 + j) * STR];
    }
    return v;
  }
}

// The fragment over 32 rows that two results hold (rows 0 .. 15 in lo, 16 .. 31 in hi).
// bf16: each value rounded to 8 bits.
template <typename T>
__device__ __forceinline__ typename FragOf<T, 8>::type pair_frag(const f32x4& lo, const f32x4& hi) {
  typename FragOf<T, 8>::type f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[j] = (T)lo[j];
    f[4 + j] = (T)hi[j];
  }
  return f;
}

// rel[r] = the head's bias of displacement r times log2 e; buckets that the table does not have: 0.
template <typename T>
__device__ __forceinline__ void load_rel(const Args& a, int head, float* rel) {
  for (int r = (int)threadIdx.x; r < a.R; r += (int)blockDim.x) {
    const int b = a.buckets[r];
    rel[r] = (unsigned)b < (unsigned)a.nb ? to_f32(((const T*)a.table)[(int64_t)b * a.heads + head]) * LOG2E : 0.f;
  }
}

// A tile of ROWS rows of HD values from memory (row r at base + r ldb bytes, rows from `rows`
// on zeros) by way of registers: load() and later store() into LDS.
template <typename T, int HD, int ROWS, int NT = posattn::NT>
struct TileCopy {
  typedef Dim<T, HD> D;
  static constexpr int N = (ROWS * D::CPR + NT - 1) / NT;
  u32x4 v[N];
  __device__ __forceinline__ void load(const char* base, uint32_t ldb, int rows, int hd) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int i = (int)threadIdx.x + NT * c, r = i / D::CPR, ch = i % D::CPR;
      v[c] = u32x4{0u, 0u, 0u, 0u};
      if (r < rows && (ROWS * D::CPR % NT == 0 || r < ROWS)) v[c] = load_chunk<T, HD>(base, (uint32_t)r * ldb, ch, hd);
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int i = (int)threadIdx.x + NT * c, r = i / D::CPR, ch = i % D::CPR;
      if (ROWS * D::CPR % NT == 0 || r < ROWS) *reinterpret_cast<u32x4*>(tile + r * D::STR + ch * D::EPC) = v[c];
    }
  }
};

// Dot products of the rows of two tiles held by TileCopy, to dst[row] in LDS.
template <typename T, int HD, int ROWS, int NT>
__device__ __forceinline__ void row_dots(const TileCopy<T, HD, ROWS, NT>& x, const TileCopy<T, HD, ROWS, NT>& y, float* dst) {
  typedef Dim<T, HD> D;
#pragma unroll
  for (int c = 0; c < TileCopy<T, HD, ROWS, NT>::N; ++c) {
    const int i = (int)threadIdx.x + NT * c, r = i / D::CPR, ch = i % D::CPR;
    float s = 0.f;
    if constexpr (sizeof(T) == 2) {
      const bf16x8 u = __builtin_bit_cast(bf16x8, x.v[c]), w = __builtin_bit_cast(bf16x8, y.v[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf((float)u[e], (float)w[e], s);
    } else {
      const f32x4 u = __builtin_bit_cast(f32x4, x.v[c]), w = __builtin_bit_cast(f32x4, y.v[c]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = fmaf(u[e], w[e], s);
    }
#pragma unroll
    for (int off = D::CPR / 2; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    if (ch == 0 && (ROWS * D::CPR % NT == 0 || r < ROWS)) dst[r] = s;
  }
}

// 4 values of a result to column d of a row of hd values, off bytes behind base.
template <typename T, int HD>
__device__ __forceinline__ void store_quad(char* base, uint32_t off, int d, int hd, const f32x4& v, float f) {
  if (HD > 16 || d < hd) {
    const float x[4] = {v[0] * f, v[1] * f, v[2] * f, v[3] * f};
    store4((T*)(base + (off + (uint32_t)(d * (int)sizeof(T)))), x);
  }
}

int launch_forward(Args a, int dtype, hipStream_t st);
int launch_backward(Args a, void* dtable, float* workspace, int dtype, hipStream_t st);
size_t backward_workspace(const Args& a, int dtype);

}  // namespace posattn

}  // namespace nsw
