// bf16 products of the linear gradients, out[r, c] = sum over d of X(r, d) W(d, c),
// without a transposed copy of any operand:
//   dx = dy . w     X = dy [R, D] rows, W = w [D, C] (contraction along its rows)
//   dw = dy^T . x   X = dy [D, R], W = x [D, C] (both along their rows)
//
// The tile, ring and schedule are mainloop_256's of the forward GEMM (256 x 256 results,
// eight waves of 128 x 64, x in 3 slots and w in 2 of 32 KB, a stage of 64 d, copies by
// the first four waves, the next step's fragments read under the present one's MFMAs).
// An operand along whose rows the contraction runs is staged as it lies in memory, 64 d
// rows of 256 columns (512 bytes), and turned while it is read: ds_read_b64_tr_b16
// gives each of 16 lanes one column of a 4 (d) x 16 block.  Its 32-byte units (16
// columns) are XOR-swizzled with f(d) = (d & 3) | ((d >> 3) & 1) << 2, so that the eight
// rows that 32 lanes read (d .. d+3 and d+8 .. d+11) lie in distinct banks.
//
// The contraction of dw is the batch: long, with few results.  It is split S ways over
// workgroups; the parts (fp32) are added in a fixed order by a second kernel.
#include <algorithm>

#include "nsw_gemm_common.h"
#include "nsw_gemm_tiles.h"

namespace nsw {

int add_parts(const void* part, void* out, int64_t n, int S, int dtype, hipStream_t st, const char* what);

namespace {

typedef __attribute__((ext_vector_type(4))) short s16x4;
constexpr int GB = 256;                 // tile rows and columns
constexpr int GSLOT = 32 * 1024;        // one operand's stage
constexpr int GD = 64;                  // contraction of a stage

struct GradArgs {
  const bf16 *x, *w;
  void* out;                            // bf16 [R, C], or fp32 [S, R, C]
  int64_t ldx, ldw;                     // row lengths (elements)
  int R, C;
  int64_t D, per;                       // contraction, and that of one part (a multiple of 64)
  int S;
};

__device__ __forceinline__ void mfma_b(f32x4& acc, const bf16x8& a, const bf16x8& b) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}

// Copies of one operand's stages.  T: as it lies, contraction along the rows: copy j of
// the wave is stage rows 2 (wave 8 + j) and the next, lane i 16-byte slot i % 32 of the
// row i / 32.  Not T: 128 bytes of d of 256 rows, as the forward GEMM.  Row d >= D, and
// what lies past the operand's end, reads as zero (the descriptor's range check); rows r
// past the edge repeat the last one, columns past the edge are never stored.
template <bool T> struct OperandCopy {
  u32x4 rsrc;
  uint32_t v[T ? 4 : 8];
  uint32_t ld2;                         // T: bytes of a row
  __device__ __forceinline__ void init(const bf16* p, int64_t ld, int64_t d0, int64_t d1, int c0, int count, int wave,
                                       int lane) {
    if constexpr (T) {
      ld2 = (uint32_t)ld * 2u;
      rsrc = make_rsrc(p + d0 * ld + c0, (uint32_t)(((d1 - d0) * ld - c0) * 2));
      const int kr = wave * 16 + lane / 32, f = (kr & 3) | ((kr >> 3) & 1) << 2;
#pragma unroll
      for (int q = 0; q < 4; ++q) {     // q = (j & 1) | (j >> 2) << 1
        const int chunk = (lane % 32) ^ (f << 1) ^ ((q & 1) << 2) ^ ((q >> 1) << 3);
        v[q] = (uint32_t)kr * ld2 + (uint32_t)chunk * 16u;
      }
    } else {
      const uint32_t rb = (uint32_t)ld * 2u;
      const int rows = count - c0 < GB ? count - c0 : GB;
      rsrc = make_rsrc(p + (int64_t)c0 * ld + d0, (uint32_t)(((int64_t)rows * ld - d0) * 2));
      ld2 = rb;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = wave * 64 + j * 8 + lane / 8;
        v[j] = (uint32_t)(r < rows ? r : rows - 1) * rb + (uint32_t)((lane % 8) ^ row_swizzle(r)) * 16u;
      }
    }
  }
  // copy j of stage st to `lds` (the wave's part of the slot).  The scalar offset is the
  // stage's start, always below the descriptor's size: the range check subtracts it
  __device__ __forceinline__ void copy(uint32_t lds, int st, int j) const {
    if constexpr (T)
      dma16(rsrc, lds + j * 1024, v[(j & 1) | (j >> 2) << 1] + (uint32_t)(2 * j) * ld2, (uint32_t)st * GD * ld2);
    else
      dma16(rsrc, lds + j * 1024, v[j], (uint32_t)st * (GD * 2));
  }
};

// Fragments of 16 rows (columns).  `at` is the lane's offset in a slot for the wave's
// first unit; unit n after it is at ^ (n << 5) (T: the unit's bits hold the swizzle) or
// n 2 KB further, the stage's second half of d 16 KB further or, not T, at chunk ^ 4.
template <bool T>
__device__ __forceinline__ uint32_t frag_at(int unit, int lane) {
  const int i = lane & 15, fg = lane >> 4;
  if constexpr (T) {
    const int f = (i >> 2) | (fg & 1) << 2;
    return (uint32_t)((fg * 8 + (i >> 2)) * 512 + ((unit ^ f) << 5) + (i & 3) * 8);
  } else {
    return (uint32_t)((unit * 16 + i) * ROWB + (fg ^ row_swizzle(i)) * 16);
  }
}
template <bool T>
__device__ __forceinline__ bf16x8 grad_frag(const char* slot, uint32_t at, int n, int sub) {
  if constexpr (T) {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    typedef __attribute__((address_space(3))) char* lds_char;
    const lds_char p = (lds_char)slot + (at ^ (uint32_t)(n << 5)) + sub * (32 * 512);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * 512));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    return *reinterpret_cast<const bf16x8*>(slot + (at ^ (sub ? 64u : 0u)) + n * (16 * ROWB));
  }
}

// Schedule as mainloop_256; COPY: a wave that issues the copies.
template <bool XT, bool COPY>
__device__ __forceinline__ void grad_loop(char* smem, const GradArgs& a, int r0, int c0, int64_t d0, int64_t d1,
                                          f32x4 (&acc)[4][8], int wave, int lane) {
  constexpr int NC = 8, CPG = 4, UNR = 12;
  OperandCopy<XT> cx;
  OperandCopy<true> cw;
  if constexpr (COPY) {
    cx.init(a.x, a.ldx, d0, d1, r0, a.R, wave, lane);
    cw.init(a.w, a.ldw, d0, d1, c0, a.C, wave, lane);
  }
  const uint32_t base = (uint32_t)(uintptr_t)smem + wave * (NC * 1024);
  const int nk = (int)((d1 - d0 + 31) / 32), nst = (nk + 1) / 2;
#define NSW_XS(s) (((s) % 3) * GSLOT)
#define NSW_WS(s) ((3 + (s) % 2) * GSLOT)
  if constexpr (COPY) {
#pragma unroll
    for (int j = 0; j < NC; ++j) cx.copy(base + NSW_XS(0), 0, j);
#pragma unroll
    for (int j = 0; j < NC; ++j) cw.copy(base + NSW_WS(0), 0, j);
    if (nst > 1) {
#pragma unroll
      for (int j = 0; j < NC; ++j) cx.copy(base + NSW_XS(1), 1, j);
#pragma unroll
      for (int j = 0; j < NC; ++j) cw.copy(base + NSW_WS(1), 1, j);
      NSW_WAIT_VMCNT(2 * NC);
    } else {
      NSW_WAIT_VMCNT(0);
    }
  }
  wg_barrier();
  uint32_t ax = frag_at<XT>((wave / 4) * 8, lane), aw = frag_at<true>((wave % 4) * 4, lane);
  bf16x8 fa[2][4], fb[2][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) fa[0][i] = grad_frag<true>(smem + NSW_WS(0), aw, i, 0);
#pragma unroll
  for (int i = 0; i < 8; ++i) fb[0][i] = grad_frag<XT>(smem + NSW_XS(0), ax, i, 0);
#define NSW_GSTEP(U)                                                                                   \
  {                                                                                                    \
    const int k = kt + U;                                                                              \
    if (k < nk) {                                                                                      \
      constexpr int sub_ = (U) % 2, su_ = (U) / 2, nsub_ = ((U) + 1) % 2, nsu_ = ((U) + 1) / 2;        \
      const int st = k >> 1;                                                                           \
      if (sub_ == 1 && k + 1 < nk) {                                                                   \
        if constexpr (COPY) NSW_WAIT_VMCNT(NC);                                                        \
        NSW_WAIT_LGKMCNT0();                                                                           \
        wg_barrier();                                                                                  \
      }                                                                                                \
      /* the fragments' addresses are formed anew in each step: kept, they spill */                   \
      asm volatile("" : "+v"(ax), "+v"(aw));                                                           \
      const int cst_ = st + 2 < nst ? st + 2 : nst - 1;                                                \
      const uint32_t wdst_ = base + (k + 1 < nk ? NSW_WS(su_ + 2) : NSW_XS(su_ + 1));                  \
      _Pragma("unroll") for (int nb = 0; nb < 4; ++nb) {                                               \
        if constexpr (COPY) {                                                                          \
          if (nb < 2) {                                                                                \
            _Pragma("unroll") for (int c_ = 0; c_ < CPG; ++c_) {                                       \
              const int j_ = nb * CPG + c_;                                                            \
              if (sub_ == 1) cw.copy(wdst_, cst_, j_);                                                 \
              else cx.copy(base + NSW_XS(su_ + 2), cst_, j_);                                          \
            }                                                                                          \
          }                                                                                            \
        }                                                                                              \
        _Pragma("unroll") for (int q = 0; q < 2; ++q)                                                  \
          fb[((U) + 1) & 1][nb * 2 + q] = grad_frag<XT>(smem + NSW_XS(nsu_), ax, nb * 2 + q, nsub_);        \
        _Pragma("unroll") for (int mb = 0; mb < 8; ++mb) mfma_b(acc[nb][mb], fa[(U) & 1][nb], fb[(U) & 1][mb]); \
        fa[((U) + 1) & 1][nb] = grad_frag<true>(smem + NSW_WS(nsu_), aw, nb, nsub_);                   \
        if constexpr (XT) {                                                                            \
          _Pragma("unroll") for (int q = 0; q < 4; ++q) {                                              \
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                         \
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                         \
          }                                                                                            \
          _Pragma("unroll") for (int q = 0; q < 2; ++q) {                                              \
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                         \
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);                                         \
          }                                                                                            \
        } else {                                                                                       \
          _Pragma("unroll") for (int q = 0; q < 4; ++q) {                                              \
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                         \
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);                                         \
          }                                                                                            \
        }                                                                                              \
      }                                                                                                \
    }                                                                                                  \
  }
  for (int kt = 0; kt < nk; kt += UNR) {
    NSW_GSTEP(0) NSW_GSTEP(1) NSW_GSTEP(2) NSW_GSTEP(3) NSW_GSTEP(4) NSW_GSTEP(5)
    NSW_GSTEP(6) NSW_GSTEP(7) NSW_GSTEP(8) NSW_GSTEP(9) NSW_GSTEP(10) NSW_GSTEP(11)
  }
#undef NSW_GSTEP
#undef NSW_XS
#undef NSW_WS
}

// XT: X's contraction runs along its rows; OT: bf16 (S = 1) or the fp32 parts.
template <bool XT, typename OT>
__global__ __launch_bounds__(512, 2) void grad_kernel(GradArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[5 * GSLOT];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  // part-major, inside a part groups of GROUP_M row blocks x all column blocks as the
  // forward GEMM: the tiles of one XCD walk the same d range over shared panels
  const int MT = (a.R + GB - 1) / GB, NT = (a.C + GB - 1) / GB;
  const int id = xcd_remap(blockIdx.x, MT * NT * a.S);
  const int part = id / (MT * NT), tile = id - part * (MT * NT);
  const int gm0 = tile / (GROUP_M * NT) * GROUP_M, gsz = MT - gm0 < GROUP_M ? MT - gm0 : GROUP_M, tin = tile - gm0 * NT;
  const int r0 = (gm0 + tin % gsz) * GB, c0 = tin / gsz * GB;
  const int64_t d0 = part * a.per, d1 = d0 + a.per < a.D ? d0 + a.per : a.D;
  f32x4 acc[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (wave < 4) grad_loop<XT, true>(smem, a, r0, c0, d0, d1, acc, wave, lane);
  else grad_loop<XT, false>(smem, a, r0, c0, d0, d1, acc, wave, lane);
  NSW_WAIT_VMCNT(0);       // the copies past the last stage
  wg_barrier();            // the ring is no longer read
  // lane (frow, fg) of block (nb, mb) holds out[mb 16 + frow][nb 16 + 4 fg + r]: 32 rows
  // at a time through an LDS part of the wave's own, out in whole 64-column rows
  constexpr int STRIDE = 64 * (int)sizeof(OT) + 16, VEC = 16 / (int)sizeof(OT), LPR = 64 / VEC, RPI = 64 / LPR;
  char* stg = smem + wave * 32 * STRIDE;
  const int frow = lane & 15, fg = lane >> 4, crow = lane / LPR, ccol = lane % LPR * VEC;
  const int rw = r0 + (wave / 4) * 128, cw = c0 + (wave % 4) * 64 + ccol;
  OT* out = (OT*)a.out + (int64_t)part * a.R * a.C;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
        const f32x4 t = acc[nb][h * 2 + mb];
        const float v[4] = {t[0], t[1], t[2], t[3]};
        store4<OT>(reinterpret_cast<OT*>(stg + (mb * 16 + frow) * STRIDE) + nb * 16 + 4 * fg, v);
      }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int r = rw + h * 32 + i * RPI + crow;
      const u32x4 v = *reinterpret_cast<const u32x4*>(stg + (i * RPI + crow) * STRIDE + ccol * (int)sizeof(OT));
      if (r < a.R && cw < a.C) *reinterpret_cast<u32x4*>(out + (int64_t)r * a.C + cw) = v;
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  }
}

}  // namespace

// Parts of the contraction, and the d of one: by estimated time, a stage STG us a round
// of 256 workgroups, FIX us for a workgroup's start and end, the parts' bytes written and
// read at 4.5 TB/s.
void grad_split(int64_t R, int64_t C, int64_t D, int64_t ld, int& S, int64_t& per) {
  const int64_t tiles = ((R + GB - 1) / GB) * ((C + GB - 1) / GB), stages = (D + GD - 1) / GD;
  double best = 0;
  S = 0;
  for (int64_t s = 1; s <= 64 && s <= stages; ++s) {
    const int64_t each = (stages + s - 1) / s;
    // 32-bit offsets inside a part
    if (each * GD * ld * 2 >= (1LL << 31) && s < 64 && s < stages) continue;
    const int64_t parts = (stages + each - 1) / each;
    static const double STG = getenv("NSW_STG") ? atof(getenv("NSW_STG")) : 1.2, FIX = getenv("NSW_FIX") ? atof(getenv("NSW_FIX")) : 5; // EXPERIMENT
    double t = (double)((tiles * parts + 255) / 256) * (FIX + STG * (double)each);
    if (parts > 1) t += 3 + (double)(parts * R * C) * 8 / 4.5e6;
    if (S == 0 || t < best) {
      best = t;
      S = (int)parts;
      per = each * GD;
    }
  }
}

int64_t grad_product_workspace(int64_t R, int64_t C, int64_t D, int64_t ld) {
  int S;
  int64_t per;
  grad_split(R, C, D, ld, S, per);
  return S > 1 ? (int64_t)S * R * C * 4 : 0;
}

// out [R, C] = X . W, X [R, D] (xt 0) or [D, R] (xt 1), W [D, C].
int grad_product(const void* x, const void* w, void* out, int64_t R, int64_t C, int64_t D, int xt, void* ws, hipStream_t st,
                 const char* what) {
  GradArgs a{};
  a.x = (const bf16*)x; a.w = (const bf16*)w;
  a.ldx = xt ? R : D; a.ldw = C;
  a.R = (int)R; a.C = (int)C; a.D = D;
  const int64_t ld = std::max<int64_t>(C, xt ? R : 0);
  grad_split(R, C, D, ld, a.S, a.per);
  NSW_CHECK_ARG(a.per * ld * 2 < (1LL << 31) && (xt || GB * D * 2 < (1LL << 31)), "%s: rows too long (32-bit offsets)", what);
  const int64_t grid = ((R + GB - 1) / GB) * ((C + GB - 1) / GB) * a.S;
  NSW_CHECK_ARG(grid < (1LL << 31), "%s: too many tiles", what);
  a.out = a.S > 1 ? ws : out;
  const dim3 g((unsigned)grid), b(512);
  if (a.S > 1) {
    if (xt) hipLaunchKernelGGL((grad_kernel<true, float>), g, b, 0, st, a);
    else hipLaunchKernelGGL((grad_kernel<false, float>), g, b, 0, st, a);
    if (int rc = check_launch(what)) return rc;
    return add_parts(ws, out, R * C, a.S, NSW_DTYPE_BF16, st, what);
  } else {
    if (xt) hipLaunchKernelGGL((grad_kernel<true, bf16>), g, b, 0, st, a);
    else hipLaunchKernelGGL((grad_kernel<false, bf16>), g, b, 0, st, a);
  }
  return check_launch(what);
}

}  // namespace nsw
