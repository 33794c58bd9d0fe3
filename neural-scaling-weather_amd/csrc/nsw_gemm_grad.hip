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
// workgroups; the parts (fp32) are added in a fixed order by a second kernel.  Tiles of
// 256 x 256 run at 1.48 PFLOP/s (64800 x 8192 -> 1024: dx 731 us, dw 739 + 23), the matrix
// units busy in 85% of the cycles at a clock of 1.65 GHz (of 2.4), which the chip's power sets
// as for the forward GEMM; products too small for that take 128 x 128 and share one launch.
#include <algorithm>

#include "nsw_gemm_common.h"
#include "nsw_gemm_tiles.h"
#include "nsw_grad.h"

namespace nsw {

namespace {

typedef __attribute__((ext_vector_type(4))) short s16x4;
constexpr int GD = 64;                  // contraction of a stage
constexpr int gslot(int gb) { return gb * GD * 2; }   // bytes of one operand's stage, GB x GB tile

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

// Copies of one operand's stages by four waves, NC of 1 KB each a stage.  T: as it lies,
// contraction along the rows: a copy is RPC rows of GB columns.  Not T: 128 bytes of d of
// GB rows, as the forward GEMM.  Row d >= D, and what lies past the operand's end, reads
// as zero (the descriptor's range check); rows r past the edge repeat the last one,
// columns past the edge are never stored.
template <bool T, int GB> struct OperandCopy {
  static constexpr int NC = gslot(GB) / 4096, RPC = 512 / GB, LPR = 64 / RPC;
  // T: the swizzle of copy j's rows differs from copy 0's by these bits of f
  static constexpr int swz(int j) { return GB == 256 ? (j & 1) << 1 | ((j >> 2) & 1) << 2 : ((j >> 1) & 1) << 2; }
  static constexpr int slot_of(int j) { return GB == 256 ? (j & 1) | (j >> 2) << 1 : (j >> 1) & 1; }
  static constexpr int NV = T ? (GB == 256 ? 4 : 2) : NC;
  u32x4 rsrc;
  uint32_t v[NV];
  uint32_t ld2;                         // T: bytes of a row
  __device__ __forceinline__ void init(const bf16* p, int64_t ld, int64_t d0, int64_t d1, int c0, int count, int wave,
                                       int lane) {
    ld2 = (uint32_t)ld * 2u;
    if constexpr (T) {
      rsrc = make_rsrc(p + d0 * ld + c0, (uint32_t)(((d1 - d0) * ld - c0) * 2));
      const int kr = wave * (NC * RPC) + lane / LPR, f = (kr & 3) | ((kr >> 3) & 1) << 2;
#pragma unroll
      for (int j = 0; j < NC; ++j)
        v[slot_of(j)] = (uint32_t)kr * ld2 + (uint32_t)((lane % LPR) ^ ((f ^ swz(j)) << 1)) * 16u;
    } else {
      const int rows = count - c0 < GB ? count - c0 : GB;
      rsrc = make_rsrc(p + (int64_t)c0 * ld + d0, (uint32_t)(((int64_t)rows * ld - d0) * 2));
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int r = (wave * NC + j) * 8 + lane / 8;
        v[j] = (uint32_t)(r < rows ? r : rows - 1) * ld2 + (uint32_t)((lane % 8) ^ row_swizzle(r)) * 16u;
      }
    }
  }
  // copy j of stage st to `lds` (the wave's part of the slot).  The scalar offset is the
  // stage's start, always below the descriptor's size: the range check subtracts it
  __device__ __forceinline__ void copy(uint32_t lds, int st, int j) const {
    if constexpr (T)
      dma16(rsrc, lds + j * 1024, v[slot_of(j)] + (uint32_t)(RPC * j) * ld2, (uint32_t)st * GD * ld2);
    else
      dma16(rsrc, lds + j * 1024, v[j], (uint32_t)st * (GD * 2));
  }
};

// Fragments of 16 rows (columns).  `at` is the lane's offset in a slot for the wave's
// first unit; unit n after it is at ^ (n << 5) (T: the unit's bits hold the swizzle) or
// n 2 KB further, the stage's second half of d 32 rows further or, not T, at chunk ^ 4.
template <bool T, int GB>
__device__ __forceinline__ uint32_t frag_at(int unit, int lane) {
  const int i = lane & 15, fg = lane >> 4;
  if constexpr (T) {
    const int f = (i >> 2) | (fg & 1) << 2;
    return (uint32_t)((fg * 8 + (i >> 2)) * (GB * 2) + ((unit ^ f) << 5) + (i & 3) * 8);
  } else {
    return (uint32_t)((unit * 16 + i) * ROWB + (fg ^ row_swizzle(i)) * 16);
  }
}
template <bool T, int GB>
__device__ __forceinline__ bf16x8 grad_frag(const char* slot, uint32_t at, int n, int sub) {
  if constexpr (T) {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    typedef __attribute__((address_space(3))) char* lds_char;
    const lds_char p = (lds_char)slot + (at ^ (uint32_t)(n << 5)) + sub * (32 * GB * 2);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * GB * 2));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    return *reinterpret_cast<const bf16x8*>(slot + (at ^ (sub ? 64u : 0u)) + n * (16 * ROWB));
  }
}

// Schedule as mainloop_256; COPY: a wave that issues the copies.
template <bool XT, bool COPY>
__device__ __forceinline__ void grad_loop(char* smem, const GradArgs& a, int r0, int c0, int64_t d0, int64_t d1,
                                          f32x4 (&acc)[4][8], int wave, int lane) {
  constexpr int GB = 256, GSLOT = gslot(GB), NC = OperandCopy<XT, GB>::NC, CPG = NC / 2, UNR = 12;
  OperandCopy<XT, GB> cx;
  OperandCopy<true, GB> cw;
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
  uint32_t ax = frag_at<XT, GB>((wave / 4) * 8, lane), aw = frag_at<true, GB>((wave % 4) * 4, lane);
  bf16x8 fa[2][4], fb[2][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) fa[0][i] = grad_frag<true, GB>(smem + NSW_WS(0), aw, i, 0);
#pragma unroll
  for (int i = 0; i < 8; ++i) fb[0][i] = grad_frag<XT, GB>(smem + NSW_XS(0), ax, i, 0);
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
          fb[((U) + 1) & 1][nb * 2 + q] = grad_frag<XT, GB>(smem + NSW_XS(nsu_), ax, nb * 2 + q, nsub_);        \
        _Pragma("unroll") for (int mb = 0; mb < 8; ++mb) mfma_b(acc[nb][mb], fa[(U) & 1][nb], fb[(U) & 1][mb]); \
        fa[((U) + 1) & 1][nb] = grad_frag<true, GB>(smem + NSW_WS(nsu_), aw, nb, nsub_);                   \
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

// A wave's results out: lane (frow, fg) of block (nb, mb) holds out[mb 16 + frow][nb 16 + 4
// fg + r]; 32 rows at a time through an LDS part of the wave's own, in whole 64-column rows.
template <typename OT, int MB>
__device__ __forceinline__ void grad_write_out(char* smem, const f32x4 (&acc)[4][MB], const GradArgs& a, int part, int rw,
                                               int cw0, int wave, int lane) {
  constexpr int STRIDE = 64 * (int)sizeof(OT) + 16, VEC = 16 / (int)sizeof(OT), LPR = 64 / VEC, RPI = 64 / LPR;
  char* stg = smem + wave * 32 * STRIDE;
  const int frow = lane & 15, fg = lane >> 4, crow = lane / LPR, ccol = lane % LPR * VEC, cw = cw0 + ccol;
  OT* out = (OT*)a.out + (int64_t)part * a.R * a.C;
#pragma unroll
  for (int h = 0; h < MB / 2; ++h) {
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

// XT: X's contraction runs along its rows; OT: bf16 (S = 1) or the fp32 parts.
template <bool XT, typename OT>
__global__ __launch_bounds__(512, 2) void grad_kernel(GradArgs a) {
  constexpr int GB = 256;
  __shared__ __attribute__((aligned(1024))) char smem[5 * gslot(GB)];
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
  grad_write_out<OT, 8>(smem, acc, a, part, r0 + (wave / 4) * 128, c0 + (wave % 4) * 64, wave, lane);
}

// 128 x 128 results, four waves of 64 x 64, two workgroups a CU: where 256 x 256 leaves
// compute units idle.  A ring of two stages, one barrier a stage (mainloop_ring of the
// forward GEMM).
template <bool XT>
__device__ __forceinline__ void grad_small_tile(char* smem, const GradArgs& a, int bid) {
  constexpr int GB = 128, GSLOT = gslot(GB);
  using CX = OperandCopy<XT, GB>;
  using CW = OperandCopy<true, GB>;
  constexpr int NC = CX::NC;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  constexpr int GM = GROUP_M * 2;                           // tile order as grad_kernel
  const int MT = (a.R + GB - 1) / GB, NT = (a.C + GB - 1) / GB;
  const int id = xcd_remap(bid, MT * NT * a.S);
  const int part = id / (MT * NT), tile = id - part * (MT * NT);
  const int gm0 = tile / (GM * NT) * GM, gsz = MT - gm0 < GM ? MT - gm0 : GM, tin = tile - gm0 * NT;
  const int r0 = (gm0 + tin % gsz) * GB, c0 = tin / gsz * GB;
  const int64_t d0 = part * a.per, d1 = d0 + a.per < a.D ? d0 + a.per : a.D;
  CX cx;
  CW cw;
  cx.init(a.x, a.ldx, d0, d1, r0, a.R, wave, lane);
  cw.init(a.w, a.ldw, d0, d1, c0, a.C, wave, lane);
  const uint32_t base = (uint32_t)(uintptr_t)smem + wave * (NC * 1024);
  const int nk = (int)((d1 - d0 + 31) / 32), nst = (nk + 1) / 2;
  // slot s: x at 2 s GSLOT, w behind it
  auto copy = [&](int st, int slot) {
#pragma unroll
    for (int j = 0; j < NC; ++j) cx.copy(base + 2 * slot * GSLOT, st, j);
#pragma unroll
    for (int j = 0; j < NC; ++j) cw.copy(base + (2 * slot + 1) * GSLOT, st, j);
  };
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint32_t ax = frag_at<XT, GB>((wave / 2) * 4, lane), aw = frag_at<true, GB>((wave % 2) * 4, lane);
  copy(0, 0);
  for (int st = 0; st < nst; ++st) {
    wait_copies();
    wg_barrier();          // stage st has landed, and no wave reads stage st - 1 any more
    const int slot = st & 1;
    if (st + 1 < nst) copy(st + 1, slot ^ 1);
    const char* xs = smem + 2 * slot * GSLOT;
    const char* ws = xs + GSLOT;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      if (sub == 1 && 2 * st + 1 >= nk) break;              // the unused half of the last stage
      bf16x8 fa[4];
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) fa[nb] = grad_frag<true, GB>(ws, aw, nb, sub);
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) {
        const bf16x8 fb = grad_frag<XT, GB>(xs, ax, mb, sub);
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) mfma_b(acc[nb][mb], fa[nb], fb);
      }
    }
  }
  wg_barrier();            // the ring is no longer read
  const int rw = r0 + (wave / 2) * 64, cw0 = c0 + (wave % 2) * 64;
  if (a.S > 1) grad_write_out<float, 4>(smem, acc, a, part, rw, cw0, wave, lane);
  else grad_write_out<bf16, 4>(smem, acc, a, part, rw, cw0, wave, lane);
}

// Workgroups [0, na) the product with the longer parts, nb of the other, then the column
// sums: products that leave compute units idle run side by side in one launch (gated
// backward of 300 rows, 256 -> 512: 15.0 us, 20.3 one after the other; 1000, 512 -> 1360:
// 30 / 42).  na is a multiple of 8, so that a workgroup's place in its product keeps its XCD.
__global__ __launch_bounds__(256, 2) void grad_small_kernel(GradArgs dw, GradArgs dx, int na, int nb, int dw_first,
                                                            ColumnSums sums, int N) {
  __shared__ __attribute__((aligned(1024))) char smem[4 * gslot(128)];
  int id = (int)blockIdx.x;
  if (id >= na + nb) {
    column_sums_block<bf16>(sums.part, (bf16*)sums.out, (int)sums.parts, N, id - na - nb, reinterpret_cast<float(*)[36]>(smem));
    return;
  }
  const bool is_dw = (id < na) == (dw_first != 0);
  const GradArgs& a = is_dw ? dw : dx;
  if (id >= na) id -= na;
  if (id >= (a.R + 127) / 128 * ((a.C + 127) / 128) * a.S) return;
  if (is_dw) grad_small_tile<true>(smem, dw, id);
  else grad_small_tile<false>(smem, dx, id);
}

}  // namespace

namespace {

// Tile (256 or 128), parts of the contraction and the d of one, by estimated time: a round
// of workgroups costs fa + fb us a stage with every slot taken, pa + pb while at most the
// share f0 of the slots is (between them linear); parts are written and read at 4.5 TB/s
// and a launch more.  Measured, us, 256 x 256 / 128 x 128 with the parts each is best at:
//   dx = dy [M, N] . w [N, K]   M 500, N 1024, K 256: 12.2 / 8.2     12961, 2720, 512: 49 / 43
//                               64800, 1024, 1024: 114 / 138         64800, 8192, 1024: 772 / 1091 (1.4 PFLOP/s)
//   dw = dy^T . x               M 500, N 1024, K 256: 12.5 / 7.3     2000, 8192, 1024: 40 / 34
//                               64800, 1024, 1024: 118 / 150         64800, 8192, 1024: 758 / 1148
struct GradCost {
  int gb, slots;
  double fa, fb, pa, pb, f0;
  double us(double wgs, double stages) const {
    const double t = wgs / slots, r = (double)(int64_t)t, f = t - r, full = fa + fb * stages, part = pa + pb * stages;
    return r * full + (f > 0 ? part + std::max(0.0, f - f0) / (1 - f0) * (full - part) : 0);
  }
};
struct GradPlan {
  int gb = 256, S = 0;
  int64_t per = 0;
  double us = 0;
};
constexpr GradCost BIG_COST{256, 256, 8.5, 1.4, 5.5, 0.96, 0}, SMALL_COST{128, 512, 4.5, 0.97, 3.6, 0.56, 0.4};
int64_t tiles(int64_t R, int64_t C, int gb) { return ((R + gb - 1) / gb) * ((C + gb - 1) / gb); }
// A second launch, and the parts through memory.
double parts_us(int64_t S, int64_t n) { return S > 1 ? 3 + (double)(S * n) * 8 / 4.5e6 : 0; }

GradPlan grad_plan(int64_t R, int64_t C, int64_t D, int64_t ld) {
  const int64_t stages = (D + GD - 1) / GD;
  GradPlan p;
  for (const GradCost& c : {BIG_COST, SMALL_COST}) {
    const int64_t n = tiles(R, C, c.gb);
    for (int64_t s = 1; s <= 64 && s <= stages; ++s) {
      const int64_t each = (stages + s - 1) / s, parts = (stages + each - 1) / each;
      // 32-bit offsets inside a part (at the most parts there are, the caller refuses)
      if (each * GD * ld * 2 >= (1LL << 31) && s < 64 && s < stages) continue;
      const double t = c.us((double)(n * parts), (double)each) + parts_us(parts, R * C);
      if (p.S == 0 || t < p.us) p = GradPlan{c.gb, (int)parts, each * GD, t};
    }
  }
  return p;
}

// Both products side by side on 128 x 128 tiles, each in parts of a length of its own;
// where that is not estimated 3% faster than one after the other (x, w), those are left.
// More workgroups than slots: 2 us and 0.8 a stage each, shared out, and 0.35 of the
// shorter one at the end.  Fits to twelve shapes and all pairs of lengths: what it picks
// is within 10% of the best pair, 1% at the median.  Measured, us, this / one after the
// other as before (two launches):
//   M 12961, N 2720, K 512: 88 / 91   2000, 8192, 1024: 71 / 82   64800, 512, 256: 46 / 57
//   2000, 1024, 256: 15 / 22          64800, 2048, 512: 281 / 234 (left one after the other)
void pair_plan(int64_t M, int64_t N, int64_t K, GradPlan& x, GradPlan& w) {
  const int64_t sx = (N + GD - 1) / GD, sw = (M + GD - 1) / GD, nx = tiles(M, K, 128), nw = tiles(N, K, 128);
  const int64_t ld = std::max(N, K);
  double best = 0.97 * (x.us + w.us);
  constexpr GradCost pair{128, SMALL_COST.slots, 2, 0.8, SMALL_COST.pa, SMALL_COST.pb, SMALL_COST.f0};
  auto next = [](int64_t e, int64_t s) { return e == s ? s + 1 : std::min(s, e & (e - 1) ? e / 3 * 4 : e / 2 * 3); };   // 2 3 4 6 8 .. s
  for (int64_t ex = std::min<int64_t>(2, sx); ex <= sx; ex = next(ex, sx)) {
    const int64_t Sx = (sx + ex - 1) / ex;
    if (Sx > 8 || ex * GD * K * 2 >= (1LL << 31)) continue;
    const double tx = pair.fa + pair.fb * (double)ex;
    for (int64_t ew = std::min<int64_t>(2, sw); ew <= sw; ew = next(ew, sw)) {
      const int64_t Sw = (sw + ew - 1) / ew;
      if (Sw > 64 || ew * GD * ld * 2 >= (1LL << 31)) continue;
      const double tw = pair.fa + pair.fb * (double)ew, ax = (double)(nx * Sx), aw = (double)(nw * Sw);
      double t = ax + aw <= SMALL_COST.slots
                     ? pair.us(ax + aw, (double)std::max(ex, ew))
                     : std::max({(ax * tx + aw * tw) / SMALL_COST.slots + 0.35 * std::min(tx, tw), tx, tw});
      if (Sx > 1 || Sw > 1) t += 4 + (double)((Sx > 1 ? Sx * M * K : 0) + (Sw > 1 ? Sw * N * K : 0)) * 8 / 6e6;
      if (t < best) {
        best = t;
        x = GradPlan{128, (int)Sx, ex * GD, t};
        w = GradPlan{128, (int)Sw, ew * GD, t};
      }
    }
  }
}
// The plans of both, whichever is asked for: a gradient's bits do not depend on what else is.
void plan_products(int64_t M, int64_t N, int64_t K, GradPlan& x, GradPlan& w) {
  x = grad_plan(M, K, N, K);
  w = grad_plan(N, K, M, std::max(N, K));
  pair_plan(M, N, K, x, w);
}
int64_t plan_bytes(const GradPlan& p, int64_t n) { return p.S > 1 ? (p.S * n * 4 + 255) / 256 * 256 : 0; }

}  // namespace

int64_t grad_products_workspace(int64_t M, int64_t N, int64_t K) {
  GradPlan x, w;
  plan_products(M, N, K, x, w);
  return plan_bytes(x, M * K) + plan_bytes(w, N * K);
}

// dx [M, K] = dy . w and dw [N, K] = dy^T . x, where not NULL, and the column sums.
int grad_products(const void* dy, const void* x, const void* w, void* dx, void* dw, const ColumnSums& sums, int64_t M, int64_t N,
                  int64_t K, char* ws, hipStream_t st, const char* what) {
  GradPlan px, pw;
  plan_products(M, N, K, px, pw);
  GradArgs ax{}, aw{};
  ax.x = (const bf16*)dy; ax.w = (const bf16*)w; ax.ldx = N; ax.ldw = K;
  ax.R = (int)M; ax.C = (int)K; ax.D = N; ax.S = px.S; ax.per = px.per;
  ax.out = px.S > 1 ? ws : dx;
  aw.x = (const bf16*)dy; aw.w = (const bf16*)x; aw.ldx = N; aw.ldw = K;
  aw.R = (int)N; aw.C = (int)K; aw.D = M; aw.S = pw.S; aw.per = pw.per;
  aw.out = pw.S > 1 ? ws + plan_bytes(px, M * K) : dw;
  NSW_CHECK_ARG((!dx || (ax.per * K * 2 < (1LL << 31) && px.gb * N * 2 < (1LL << 31))) &&
                    (!dw || aw.per * std::max(N, K) * 2 < (1LL << 31)), "%s: rows too long (32-bit offsets)", what);
  const int64_t gx = dx ? tiles(M, K, px.gb) * px.S : 0, gw = dw ? tiles(N, K, pw.gb) * pw.S : 0, gs = sums.out ? (N + 31) / 32 : 0;
  NSW_CHECK_ARG(gx + gw + gs < (1LL << 31) - 8, "%s: too many tiles", what);
  if (dx && px.gb == 256) {
    if (px.S > 1) hipLaunchKernelGGL((grad_kernel<false, float>), dim3((unsigned)gx), dim3(512), 0, st, ax);
    else hipLaunchKernelGGL((grad_kernel<false, bf16>), dim3((unsigned)gx), dim3(512), 0, st, ax);
    if (int rc = check_launch(what)) return rc;
  }
  if (dw && pw.gb == 256) {
    if (pw.S > 1) hipLaunchKernelGGL((grad_kernel<true, float>), dim3((unsigned)gw), dim3(512), 0, st, aw);
    else hipLaunchKernelGGL((grad_kernel<true, bf16>), dim3((unsigned)gw), dim3(512), 0, st, aw);
    if (int rc = check_launch(what)) return rc;
  }
  const int64_t nx = px.gb == 128 ? gx : 0, nw = pw.gb == 128 ? gw : 0;
  ColumnSums late = sums;                                   // with the parts, if nothing runs beside them here
  if (nx + nw > 0) {
    late.out = nullptr;
    const bool dw_first = pw.per >= px.per;
    const int64_t na = ((dw_first ? nw : nx) + 7) / 8 * 8, nb = dw_first ? nx : nw;
    hipLaunchKernelGGL(grad_small_kernel, dim3((unsigned)(na + nb + gs)), dim3(256), 0, st, aw, ax, (int)na, (int)nb,
                       (int)dw_first, sums, (int)N);
    if (int rc = check_launch(what)) return rc;
  }
  return finish_grads(Parts{ax.out, dx, M * K, dx ? px.S : 0}, Parts{aw.out, dw, N * K, dw ? pw.S : 0}, late, N, NSW_DTYPE_BF16, st,
                      what);
}

}  // namespace nsw
