// Window attention with a learned position bias: what its forward and backward kernels share.
#pragma once

#include <type_traits>

#include "nsw_common.h"

namespace nsw {

namespace posattn {

constexpr int NT = 256;             // threads of a workgroup, four waves
constexpr int MAX_R = 8192;         // displacements of a window
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const void *qkv, *table, *dout, *out;
  void *o, *dqkv;
  float* stats;                     // [Bw, heads, L, ns]: row maximum m of z log2 e, log2 of the row's sum of exp2(z log2 e - m), lost bits
  int ns;
  const int* buckets;               // [R]
  const float* mask;                // [nW, L, L] or NULL
  float* part;                      // [heads, NP, L, L]: dz summed over the windows of a workgroup, or NULL
  int64_t Bw;
  int nW;                           // windows of the mask, or of an image
  int L, C, heads, hd, R, off, nb;
  int TW, A, W;                     // extent of a window (frames are the outermost)
  int nqc;                          // workgroups that share a window's queries (keys in the backward pass)
  int NP;                           // workgroups that share a head's windows
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

// The byte address in LDS of rel, to which the queries' infos are moved together with the middle
// displacement: a pair's bias then lies at the difference of its two infos.
__device__ __forceinline__ int rel_base(const Args& a, const float* rel) {
  return (int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const float*)rel + 4 * a.off;
}

// Biases of four pairs in units of log2 e from the infos of their queries (moved) and keys; with a
// shift the bits of the classes have to be kept out of the address.
__device__ __forceinline__ f32x4 biases(const int (&q)[4], const int (&k)[4], bool shifted) {
  typedef __attribute__((address_space(3))) const float* lds_ptr;
  f32x4 b;
  if (shifted) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      b[r] = *(lds_ptr)(uintptr_t)((uint32_t)(q[r] - k[r]) & 0x3fffffffu);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) b[r] = *(lds_ptr)(uintptr_t)(uint32_t)(q[r] - k[r]);
  }
  return b;
}

// Logits in units of log2 e from products.  A shift or mask is added to them, in every kernel in this
// order: the backward pass then forms each z to the bit as the forward pass did, and a row's
// probabilities add up to 1 however large its logits are (shift and bias added first in one of
// them: off by an fp32 step of |z|, 0.3% at 1e5).
__device__ __forceinline__ void logits(f32x4& s, float zs, const f32x4& bias) {
#pragma unroll
  for (int r = 0; r < 4; ++r) s[r] = fmaf(s[r], zs, bias[r]);
}

// The shift's -100 between pairs of two classes.
__device__ __forceinline__ void add_shift(f32x4& s, const int (&q)[4], const int (&k)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) s[r] += (q[r] ^ k[r]) >> 30 ? -100.f * LOG2E : 0.f;
}

// A value of a mask or table times log2 e: finite ones stay finite (2.36e38 and what lies beyond
// become the largest float), so that a row of the lowest or the highest floats is uniform, as in
// fp32 on the formula.
__device__ __forceinline__ float in_units(float x) {
  constexpr float MOST = 3.402823466e38f;
  const float v = x * LOG2E;
  return fabsf(x) <= MOST ? __builtin_amdgcn_fmed3f(v, -MOST, MOST) : v;
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
  static constexpr int STR = HD + (sizeof(T) == 4 ? 4 : HD == 16 ? 0 : 16);   // bf16: 8 times an odd number of banks
  static constexpr int NS = HD >= 32 ? HD / 32 : 1;        // k-steps of a product over the head dim
  static constexpr int ND = HD / 16;                       // 16-wide blocks of the head dim
  static constexpr int EL = sizeof(T) == 2 || HD >= 32 ? 8 : 4;
  typedef typename FragOf<T, EL>::type Frag;               // over the head dim
  typedef typename FragOf<T, 8>::type TFrag;               // over 32 tokens
};

// n rows of a tensor, `ldb` bytes apart, of which this head has `bytes`: a buffer descriptor on
// a base that is the same for the wave.  A lane's address is one 32-bit offset, what lies behind
// the last row reads as zeros and is not written (rows of a window end below 2 GiB: checked by
// the host), so no lane branches around its loads.
struct Rows {
  __amdgpu_buffer_rsrc_t r;
  uint32_t ldb;
  __device__ __forceinline__ Rows(const void* p, uint32_t ldb_, int n, int bytes) : ldb(ldb_) {
    const uint64_t u = (uint64_t)p;
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32));
    const int num = __builtin_amdgcn_readfirstlane(n > 0 ? (int)((uint32_t)(n - 1) * ldb + (uint32_t)bytes) : 0);
    r = __builtin_amdgcn_make_buffer_rsrc((void*)(hi << 32 | lo), 0, num, 0x00020000);
  }
};
constexpr uint32_t NOWHERE = 0xfffffff0u;   // an offset behind every row

// 16 bytes, chunk ch, of a row of hd values, zeros past its end (head dims 4 and 8 among 16).
template <typename T, int HD>
__device__ __forceinline__ u32x4 load_chunk(const Rows& x, uint32_t off, int ch, int hd) {
  constexpr int EPC = 16 / (int)sizeof(T);
  const uint32_t at = off + 16u * (uint32_t)ch;
  if constexpr (HD > 16) {
    return __builtin_amdgcn_raw_buffer_load_b128(x.r, at, 0, 0);
  } else {
    if (hd >= EPC) return __builtin_amdgcn_raw_buffer_load_b128(x.r, ch * EPC < hd ? at : NOWHERE, 0, 0);
    typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;      // bf16, head dim 4: 8 bytes
    const u32x2 h = __builtin_amdgcn_raw_buffer_load_b64(x.r, ch == 0 ? at : NOWHERE, 0, 0);
    return u32x4{h[0], h[1], 0u, 0u};
  }
}

// Fragment over the head dim, k-step s, of a row in memory: bf16 values 32 s + 8 fg .., fp32 the
// same or (head dim 16) 4 fg ..
template <typename T, int HD>
__device__ __forceinline__ typename Dim<T, HD>::Frag row_frag(const Rows& x, uint32_t row, int s, int fg, int hd) {
  typedef typename Dim<T, HD>::Frag F;
  const uint32_t off = row * x.ldb;
  if constexpr (sizeof(T) == 4 && HD >= 32) {
    const f32x4 lo = __builtin_bit_cast(f32x4, load_chunk<T, HD>(x, off, 8 * s + 2 * fg, hd));
    const f32x4 hi = __builtin_bit_cast(f32x4, load_chunk<T, HD>(x, off, 8 * s + 2 * fg + 1, hd));
    return F{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  } else {
    return __builtin_bit_cast(F, load_chunk<T, HD>(x, off, 4 * s + fg, hd));
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
    rel[r] = (unsigned)b < (unsigned)a.nb ? in_units(to_f32(((const T*)a.table)[(int64_t)b * a.heads + head])) : 0.f;
  }
}

// A tile of ROWS rows of HD values from memory by way of registers: load() and later store()
// into LDS, by NT threads, a workgroup's or four waves of a larger one.
template <typename T, int HD, int ROWS, int NT = posattn::NT>
struct TileCopy {
  typedef Dim<T, HD> D;
  static constexpr int N = (ROWS * D::CPR + NT - 1) / NT;
  u32x4 v[N];
  __device__ __forceinline__ void load(const Rows& x, int hd) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int i = (int)threadIdx.x % NT + NT * c, r = i / D::CPR, ch = i % D::CPR;
      v[c] = u32x4{0u, 0u, 0u, 0u};
      if (ROWS * D::CPR % NT == 0 || r < ROWS) v[c] = load_chunk<T, HD>(x, (uint32_t)r * x.ldb, ch, hd);
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int i = (int)threadIdx.x % NT + NT * c, r = i / D::CPR, ch = i % D::CPR;
      if (ROWS * D::CPR % NT == 0 || r < ROWS) *reinterpret_cast<u32x4*>(tile + r * D::STR + ch * D::EPC) = v[c];
    }
  }
};

// D = do o of the gradients cancels against do v, and the rounding of o to bf16 would be most of
// dz's error (dtable 2.5e-3 off where its own rounding is 1.7e-3).  The forward pass therefore
// leaves, behind a row's statistics, what each value of o lost, in sixteenths of a step and 4
// bits: a quarter of o's bytes.  A step is 2^16 of fp32's pattern, whatever the exponent: the
// difference of the two patterns is rounded to 2^12, -7 .. 6 of it are written as 1 .. 14, so that
// no word of them is a float's NaN, and none zero, which is what lies past a window's rows.
__device__ __forceinline__ uint32_t lost_of(float x) {
  const int d = __builtin_bit_cast(int, x) - __builtin_bit_cast(int, (float)(bf16)x) + 0x8800;
  return (uint32_t)(d < 0x1000 ? 0x1000 : d > 0xefff ? 0xefff : d) >> 12;
}
// the value from its bf16 and the e-th 4 bits of a word
__device__ __forceinline__ float found(float b, uint32_t bits, int e) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, b) - 0x8000u + ((bits >> 4 * e & 15u) << 12));
}
__device__ __forceinline__ uint32_t lost_word(const Rows& stats, uint32_t at) {
  const uint32_t v = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(stats.r, at, 0, 0);
  return v ? v : 0x88888888u;
}

// The lost bits that belong to a TileCopy of o: a word to 8 values.
template <typename T, int HD, int ROWS, int NT = posattn::NT>
struct Lost {
  typedef Dim<T, HD> D;
  static constexpr int N = sizeof(T) == 2 ? TileCopy<T, HD, ROWS, NT>::N : 0;
  uint32_t v[N > 0 ? N : 1];
  __device__ __forceinline__ void load(const Rows& stats, int hd) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int i = (int)threadIdx.x % NT + NT * c, r = i / D::CPR, ch = i % D::CPR;
      const uint32_t at = (HD > 16 || 8 * ch < hd) && (ROWS * D::CPR % NT == 0 || r < ROWS) ? (uint32_t)r * stats.ldb + 8u + 4u * ch : NOWHERE;
      v[c] = lost_word(stats, at);
    }
  }
};

// Dot products of the rows of two tiles held by TileCopy, of the second with its lost bits, to
// dst[row] in LDS.
template <typename T, int HD, int ROWS, int NT>
__device__ __forceinline__ void row_dots(const TileCopy<T, HD, ROWS, NT>& x, const TileCopy<T, HD, ROWS, NT>& y,
                                         const Lost<T, HD, ROWS, NT>& lost, float* dst) {
  typedef Dim<T, HD> D;
#pragma unroll
  for (int c = 0; c < TileCopy<T, HD, ROWS, NT>::N; ++c) {
    const int i = (int)threadIdx.x % NT + NT * c, r = i / D::CPR, ch = i % D::CPR;
    float s = 0.f;
    if constexpr (sizeof(T) == 2) {
      const bf16x8 u = __builtin_bit_cast(bf16x8, x.v[c]), w = __builtin_bit_cast(bf16x8, y.v[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf((float)u[e], found((float)w[e], lost.v[c], e), s);
    } else {
      const f32x4 u = __builtin_bit_cast(f32x4, x.v[c]), w = __builtin_bit_cast(f32x4, y.v[c]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = fmaf(u[e], w[e], s);
    }
    // the row's lanes: pairs, quads, eights (half rows mirrored), sixteens (rows mirrored), 32
    auto add = [&](auto ctrl) {
      s += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, s), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    add(std::integral_constant<int, 0xB1>{});
    if constexpr (D::CPR >= 4) add(std::integral_constant<int, 0x4E>{});
    if constexpr (D::CPR >= 8) add(std::integral_constant<int, 0x141>{});
    if constexpr (D::CPR >= 16) add(std::integral_constant<int, 0x140>{});
    if constexpr (D::CPR >= 32) s = rows2_sum(s);
    if (ch == 0 && (ROWS * D::CPR % NT == 0 || r < ROWS)) dst[r] = s;
  }
}

// 4 values of a result to column d of a row of hd values.
template <typename T, int HD>
__device__ __forceinline__ void store_quad(const Rows& x, uint32_t row, int d, int hd, const f32x4& v, float f) {
  const uint32_t at = HD > 16 || d < hd ? row * x.ldb + (uint32_t)(d * (int)sizeof(T)) : NOWHERE;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
    const bf16x4 o = {(bf16)(v[0] * f), (bf16)(v[1] * f), (bf16)(v[2] * f), (bf16)(v[3] * f)};
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, o), x.r, at, 0, 0);
  } else {
    const f32x4 o = {v[0] * f, v[1] * f, v[2] * f, v[3] * f};
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), x.r, at, 0, 0);
  }
}

// What 4 values v f of a result lost in store_quad, to the row's statistics.
template <typename T, int HD>
__device__ __forceinline__ void store_lost(const Rows& stats, uint32_t row, int d, int hd, const f32x4& v, float f) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t b = lost_of(v[0] * f) | lost_of(v[1] * f) << 4 | lost_of(v[2] * f) << 8 | lost_of(v[3] * f) << 12;
    const uint32_t at = HD > 16 || d < (hd + 7) / 8 * 8 ? row * stats.ldb + 8u + (uint32_t)(d / 2) : NOWHERE;
    __builtin_amdgcn_raw_buffer_store_b16((unsigned short)b, stats.r, at, 0, 0);
  }
}

// Where a window's rows begin in each tensor, for one head.
struct At {
  uint32_t ldb, ob;                 // bytes of a row of qkv, of o
  int64_t q, o;                     // byte offsets
  int bytes;                        // of a head in a row
  __device__ __forceinline__ At(const Args& a, int64_t win, int head, int es) {
    ob = (uint32_t)a.C * (uint32_t)es;
    ldb = 3u * ob;
    bytes = a.hd * es;
    q = win * a.L * (int64_t)ldb + head * bytes;
    o = win * a.L * (int64_t)ob + head * bytes;
  }
  // rows [r0, r0 + n) of part 0 (q), 1 (k), 2 (v) of qkv or its gradient; of o or its gradient
  __device__ __forceinline__ Rows qkv(const void* p, int part, int r0, int n) const {
    return Rows((const char*)p + q + (int64_t)r0 * ldb + part * (int64_t)ob, ldb, n, bytes);
  }
  // rows [r0, r0 + n) of the statistics
  __device__ __forceinline__ static Rows stats(const Args& a, int64_t win, int head, int r0, int n) {
    return Rows(a.stats + ((win * a.heads + head) * a.L + r0) * a.ns, 4u * (uint32_t)a.ns, n, 4 * a.ns);
  }
  __device__ __forceinline__ Rows out(const void* p, int r0, int n) const { return Rows((const char*)p + o + (int64_t)r0 * ob, ob, n, bytes); }
};

// A window's fp32 matrix [L, L], of a mask or of sums: element (q, k), pairs outside the window
// nowhere.
struct Plane {
  __amdgpu_buffer_rsrc_t r;
  int L;
  __device__ __forceinline__ Plane(const float* p, int L_) : L(L_) { r = Rows(p, (uint32_t)L_ * 4u, L_, L_ * 4).r; }
  __device__ __forceinline__ uint32_t at(int q, int k) const { return k < L ? (uint32_t)(q * L + k) * 4u : NOWHERE; }
  __device__ __forceinline__ float get(int q, int k) const { return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, at(q, k), 0, 0)); }
  // keys k .. k + 3 of query q; what lies past the window is of another row or zero
  __device__ __forceinline__ f32x4 get4(int q, int k) const { return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at(q, k), 0, 0)); }
  __device__ __forceinline__ void put(int q, int k, float v) const { __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), r, at(q, k), 0, 0); }
};

int launch_forward(Args a, int dtype, hipStream_t st);
int launch_backward(Args a, void* dtable, float* workspace, int dtype, hipStream_t st);
size_t backward_workspace(const Args& a, int dtype);

}  // namespace posattn

}  // namespace nsw
