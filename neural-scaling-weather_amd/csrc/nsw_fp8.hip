// Products in 8-bit floating point: rows of e4m3 values with one power-of-two scale
// (E8M0: the exponent + 127 in a byte) for each 1 x 128 block of x and each 128 x 128
// block of w,
//   y[m, n] = epilogue(sum over blocks kb of 2^(ex[m, kb] + ew[n / 128, kb]) sum over
//                      the block's k of xq[m, k] wq[n, k]),
// and the quantiser that makes them: a block's scale is the smallest power of two that
// brings its largest finite magnitude to at most 448, e4m3's largest.
//
// Powers of two, because gfx950's scaled matrix instructions (v_mfma_scale_f32_*_
// f8f6f4) apply them inside the product, at the rate of the plain 8-bit ones: no
// vector instruction touches a partial sum, and scaling adds no rounding.  The
// hardware's own blocks are 32 k; a block of 128 passes the same scale four times.
//
// The 8-bit instructions add in groups of 8 consecutive k: within a group a product
// keeps only its bits at or above 2^-13 of the largest product's power of two
// (measured: next to 2^16, 2^3 counts and 2^2 does not, of either sign); groups and the
// accumulator are added in fp32.  A result is off by at most 7 2^-13 of its sum of
// magnitudes from that, by 2.4e-4 of itself on normal rows: 1/7 of the rounding to
// bf16 that follows, and far below e4m3's own 2^-4 a value.  For fp32 results that is
// too much: there the values are widened to bf16 (exact) for the 16-bit instructions,
// whose sums are fp32 throughout, and each block's sum is scaled as it is added.
//
// The instructions are issued "transposed", as in the 16-bit GEMM: A is the weight
// fragment, B the activation fragment, so that a lane holds four consecutive output
// columns of one row.
#include <algorithm>
#include <type_traits>

#include "nsw_gemm_common.h"

namespace nsw {

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr int BLK = 128;                 // values of a block along k
constexpr int MAX_KB = 126;              // longest rows: 16128 values
constexpr int QT = 256;                  // threads of the quantisers

// ---------------------------------------------------------------- quantiser ---

// Eight values: load (zeros past the row's end), largest finite magnitude, e4m3 of
// them under inverse scale inv (a value that is not finite becomes NaN).
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int k, int K, float (&v)[8]) {
  constexpr int VEC = Vec16<T>::N;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e += VEC)
    if (k + e < K) load16<T>(row + k + e, v + e);
}
__device__ __forceinline__ float top8(const float (&v)[8]) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = fabsf(v[e]);
    m = fmaxf(m, a < INFINITY ? a : 0.f);
  }
  return m;
}
__device__ __forceinline__ uint2 pack8(const float (&v)[8], float inv) {
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = fabsf(v[e]) < INFINITY ? v[e] * inv : __builtin_nanf("");
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(s[4], s[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(s[6], s[7], hi, true);
  return uint2{(uint32_t)lo, (uint32_t)hi};
}
// E8M0 byte of the smallest 2^e with top <= 448 * 2^e: top = 1.f 2^x and 448 = 1.75
// 2^8, so e = x - 8, one more where 1.f > 1.75; at least 2^-127 (blocks of zeros, and
// of values below 2^-118, which round to that scale's grid).
__device__ __forceinline__ int scale_byte(float top) {
  const uint32_t b = __builtin_bit_cast(uint32_t, top);
  const int s = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return s < 0 ? 0 : s;
}
__device__ __forceinline__ float inverse_scale(int byte) { return __builtin_bit_cast(float, (uint32_t)(254 - byte) << 23); }

__device__ __forceinline__ float row16_max(float x) {
  x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, false)));
  x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x124, 0xf, 0xf, false)));
  x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x122, 0xf, 0xf, false)));
  x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x121, 0xf, 0xf, false)));
  return x;
}

// 1 x 128 blocks, 16 lanes each; block b of the R * Kb is row b / Kb.  Bound by HBM
// (64800 x 1024 bf16 in 34 us: 5.8 TB/s), with four blocks' loads in flight a lane.
template <typename T>
__global__ __launch_bounds__(QT) void quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                           uint8_t* __restrict__ scale, uint32_t blocks, int K, int Kb,
                                                           FastDiv by_kb) {
  constexpr int U = 4;                                      // blocks in flight per 16 lanes
  const int l = (int)threadIdx.x & 15;
  const int64_t b0 = ((int64_t)blockIdx.x * (QT / 16) + (threadIdx.x >> 4)) * U;
  float v[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t b = b0 + u < blocks ? (uint32_t)(b0 + u) : blocks - 1, r = by_kb.div(b);
    load8<T>(x + (int64_t)r * K, (int)(b - r * (uint32_t)Kb) * BLK + l * 8, K, v[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int s = scale_byte(row16_max(top8(v[u])));
    const uint2 p = pack8(v[u], inverse_scale(s));
    if (b0 + u < blocks) {
      *reinterpret_cast<uint2*>(q + (b0 + u) * BLK + l * 8) = p;
      if (l == 0) scale[b0 + u] = (uint8_t)s;
    }
  }
}

// 128 x 128 blocks, a workgroup each (1336 x 1000 fp32 5 us, a launch's latency).
template <typename T>
__global__ __launch_bounds__(QT) void quantize_tiles_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                            uint8_t* __restrict__ scale, int64_t R, int K, int Kb) {
  __shared__ float tops[QT / 16];
  constexpr int U = 128 / (QT / 16);                        // rows of a thread
  const int l = (int)threadIdx.x & 15, g = (int)threadIdx.x >> 4;
  const int kb = (int)blockIdx.x;
  const int64_t r0 = (int64_t)blockIdx.y * 128 + g;
  float v[U][8], m = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + u * (QT / 16);
    load8<T>(x + (r < R ? r : 0) * K, r < R ? kb * BLK + l * 8 : K, K, v[u]);
    m = fmaxf(m, top8(v[u]));
  }
  m = row16_max(m);
  if (l == 0) tops[g] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < QT / 16; ++i) m = fmaxf(m, tops[i]);
  const int s = scale_byte(m);
  const float inv = inverse_scale(s);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + u * (QT / 16);
    if (r < R) *reinterpret_cast<uint2*>(q + (r * Kb + kb) * BLK + l * 8) = pack8(v[u], inv);
  }
  if (threadIdx.x == 0) scale[(int64_t)blockIdx.y * Kb + kb] = (uint8_t)s;
}

// ------------------------------------------------------------------ product ---

struct Fp8Args {
  const uint8_t *xq, *xs, *wq, *ws;
  const void *bias, *residual;
  void* y;
  int64_t M;
  int N, K, Kb;      // K = 128 Kb
};

// Epilogue of one value before the residual.
template <typename T, int EPI>
__device__ __forceinline__ float finish(float v, float b) {
  if constexpr (EPI != EPI_NONE) v += b;
  if constexpr (EPI == EPI_BIAS_GELU) v = sizeof(T) == 2 ? gelu_erf_bf16(v) : gelu_erf(v);
  if constexpr (EPI == EPI_BIAS_GELU_TANH) v = gelu_tanh(v);
  return v;
}

// 32 e4m3 values as four bf16 fragments (every e4m3 value is a bf16 value).
__device__ __forceinline__ void widen32(const i32x8& f, bf16x8 (&o)[4]) {
#pragma unroll
  for (int g = 0; g < 4; ++g)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * g + h], 1.f, false);
      const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * g + h], 1.f, true);
      o[g][4 * h] = lo[0]; o[g][4 * h + 1] = lo[1]; o[g][4 * h + 2] = hi[0]; o[g][4 * h + 3] = hi[1];
    }
}

// v under the E8M0 scales a and b (255 is NaN, as for the scaled instructions).
__device__ __forceinline__ float scaled(float v, int a, int b) {
  return a == 255 || b == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(v, a + b - 254);
}

// Between a wave's LDS writes and its reads of what other lanes wrote (LDS accesses
// of a wave are served in order; only the compiler has to keep them so).
__device__ __forceinline__ void wave_fence() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

// Tile of WGM x WGN wavefronts, each MB x NB blocks of 32 x 32 results; operands in a
// ring of NST stages of 128 k (one scale block), one barrier a stage as mainloop_ring
// of the 16-bit GEMM; the tile's scales wait in LDS behind the ring.
template <int WGM_, int WGN_, int MB_, int NB_, int NST_, int LDS_>
struct Tile8 {
  static constexpr int WGM = WGM_, WGN = WGN_, MB = MB_, NB = NB_, NST = NST_, LDS = LDS_, NW = WGM * WGN;
  static constexpr int WTM = MB * 32, WTN = NB * 32, BM = WGM * WTM, BN = WGN * WTN;
  static constexpr int SLOT = (BM + BN) * BLK, RING = NST * SLOT;
  static constexpr int NBLK = (BN + 127) / 128;             // weight scale rows a tile meets
  static constexpr int MINW = NW * (160 * 1024 / LDS) / 4;
  static_assert(BN % 128 == 0 || 128 % BN == 0, "weight scales");
  static_assert(RING + MAX_KB * (BM + NBLK) <= LDS, "the scales of the longest rows fit behind the ring");
};
// 128 x 128, two workgroups a CU, so that one's epilogue runs beside the other's main loop
// (16384 x 4096 -> 1024 bf16 69 us, 2.0 PFLOP/s, with bias and GELU 74)
using Mid8 = Tile8<2, 2, 2, 2, 2, 80 * 1024>;

// The tile's scales into LDS: [Kb][BM] bytes of its rows, [Kb][NBLK] of its weight blocks.
template <class TC>
__device__ __forceinline__ void load_scales(const Fp8Args& a, uint8_t* xsl, uint8_t* wsl, int64_t m0, int n0, int rows) {
  constexpr int NW = TC::NW;
  {
    constexpr int TPR = NW * 64 / TC::BM, U = 8;            // threads of a row, loads in flight
    static_assert(TPR * TC::BM == NW * 64, "whole threads to a row");
    const int r = (int)threadIdx.x % TC::BM;
    const uint8_t* p = a.xs + (m0 + (r < rows ? r : rows - 1)) * a.Kb;
    for (int k0 = (int)threadIdx.x / TC::BM; k0 < a.Kb; k0 += U * TPR) {
      uint8_t b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) b[u] = p[k0 + u * TPR < a.Kb ? k0 + u * TPR : 0];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k0 + u * TPR < a.Kb) xsl[(k0 + u * TPR) * TC::BM + r] = b[u];
    }
  }
  for (int i = threadIdx.x; i < a.Kb * TC::NBLK; i += NW * 64) {
    const int kb = i / TC::NBLK, b = i - kb * TC::NBLK;
    const int nb = n0 / 128 + b, last = (a.N - 1) / 128;
    wsl[kb * TC::NBLK + b] = a.ws[(int64_t)(nb < last ? nb : last) * a.Kb + kb];
  }
}

// Epilogue: lane (frow, half) of block (nb, mb) holds y[mb 32 + frow][nb 32 + 8 q + 4
// half + r] in element 4 q + r.  Each wave stages 32 rows of its columns in an LDS part
// of its own and copies them out in whole rows of 16-byte pieces.  With a residual the
// staged values stay fp32, so that the sum is rounded once.
template <typename T, int EPI, class TC>
__device__ __forceinline__ void write_out(const Fp8Args& a, char* smem, f32x16 (&acc)[TC::NB][TC::MB], int64_t m0, int n0,
                                          int wave, int lane) {
  constexpr int MB = TC::MB, NB = TC::NB, NW = TC::NW;
  const int wm = wave / TC::WGN, wn = wave % TC::WGN, frow = lane & 31, half = lane >> 5;
  constexpr bool RES = EPI == EPI_BIAS_RESIDUAL;
  using ST = std::conditional_t<RES, float, T>;
  constexpr int STRIDE = TC::WTN * (int)sizeof(ST) + 16, VEC = Vec16<T>::N, LPR = TC::WTN / VEC, RPI = 64 / LPR;
  static_assert(NW * 32 * STRIDE <= TC::LDS, "staging fits in the LDS");
  char* stg = smem + wave * 32 * STRIDE;
  const int nw = n0 + wn * TC::WTN;
  const int crow = lane / LPR, ccol = lane % LPR * VEC;
  const bool cin = nw + ccol < a.N;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int64_t mr = m0 + wm * TC::WTM + mb * 32;
    u32x4 res[RES ? 32 / RPI : 1];
    if constexpr (RES) {   // in one batch, ahead of the staging
#pragma unroll
      for (int i = 0; i < 32 / RPI; ++i) {
        const int64_t m = mr + i * RPI + crow;
        res[i] = *reinterpret_cast<const u32x4*>((const T*)a.residual + (m < a.M ? m : a.M - 1) * a.N + (cin ? nw + ccol : 0));
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = nb * 32 + 8 * q + 4 * half;
        float b[4] = {0.f, 0.f, 0.f, 0.f}, o[4];
        if constexpr (EPI != EPI_NONE) load4<T>((const T*)a.bias + (nw + c < a.N ? nw + c : 0), b);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = finish<T, EPI>(acc[nb][mb][4 * q + r], b[r]);
        store4<ST>(reinterpret_cast<ST*>(stg + frow * STRIDE) + c, o);
      }
    wave_fence();
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int64_t m = mr + i * RPI + crow;
      const char* src = stg + (i * RPI + crow) * STRIDE + ccol * (int)sizeof(ST);
      if (m < a.M && cin) {
        T* yp = (T*)a.y + m * a.N + nw + ccol;
        if constexpr (RES) {
          float o[VEC], rv[VEC];
          load16<T>(reinterpret_cast<const T*>(&res[i]), rv);
#pragma unroll
          for (int e = 0; e < VEC; e += 4) load16<float>(reinterpret_cast<const float*>(src) + e, o + e);
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[e] += rv[e];
          store16<T>(yp, o);
        } else {
          __builtin_nontemporal_store(*reinterpret_cast<const u32x4*>(src), reinterpret_cast<u32x4*>(yp));
        }
      }
    }
    wave_fence();
  }
}

template <typename T, int EPI, class TC>
__global__ __launch_bounds__(TC::NW * 64, TC::MINW) void linear_fp8_kernel(Fp8Args a) {
  constexpr int MB = TC::MB, NB = TC::NB, NW = TC::NW, NST = TC::NST;
  __shared__ __attribute__((aligned(1024))) char smem[TC::LDS];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int wm = wave / TC::WGN, wn = wave % TC::WGN;
  const int MT = (int)((a.M + TC::BM - 1) / TC::BM), NT = (a.N + TC::BN - 1) / TC::BN;
  // XCD x works on a contiguous range of tiles, groups of GM row blocks x all column
  // blocks, column-major inside, so that its L2 holds both panels
  constexpr int GM = GROUP_M * 256 / TC::BM;
  const int tile = xcd_remap(blockIdx.x, MT * NT);
  const int gm0 = tile / (GM * NT) * GM, gsz = MT - gm0 < GM ? MT - gm0 : GM;
  const int tin = tile - gm0 * NT;
  const int64_t m0 = (int64_t)(gm0 + tin % gsz) * TC::BM;
  const int n0 = tin / gsz * TC::BN;
  const int rows = a.M - m0 < TC::BM ? (int)(a.M - m0) : TC::BM, cols = a.N - n0 < TC::BN ? a.N - n0 : TC::BN;

  // operand copies: copy j of the wave covers 8 stage rows, lane i row i / 8, 16-byte
  // slot i % 8, swizzled as the 16-bit GEMM's; rows past the edge repeat the last one
  constexpr int CX = TC::BM / 8 / NW, CW = TC::BN / 8 / NW, NC = CX + CW;
  static_assert(CX * NW * 8 == TC::BM && CW * NW * 8 == TC::BN, "copies split evenly over the waves");
  const u32x4 rx = make_rsrc(a.xq + m0 * a.K, (uint32_t)rows * (uint32_t)a.K);
  const u32x4 rw = make_rsrc(a.wq + (int64_t)n0 * a.K, (uint32_t)cols * (uint32_t)a.K);
  uint32_t v[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int r = (j < CX ? wave * CX + j : wave * CW + j - CX) * 8 + lane / 8, end = j < CX ? rows : cols;
    v[j] = (uint32_t)(r < end ? r : end - 1) * (uint32_t)a.K + (uint32_t)((lane % 8) ^ row_swizzle(r)) * 16u;
  }
  const uint32_t lds = (uint32_t)(uintptr_t)smem;
  auto copy = [&](int s, int slot) {
#pragma unroll
    for (int j = 0; j < NC; ++j)
      dma16(j < CX ? rx : rw,
            lds + slot * TC::SLOT + (j < CX ? (wave * CX + j) * 1024 : TC::BM * BLK + (wave * CW + j - CX) * 1024), v[j],
            (uint32_t)s * BLK);
  };
  const int nst = a.Kb;
#pragma unroll
  for (int s = 0; s < NST - 1; ++s)
    if (s < nst) copy(s, s);
  uint8_t* xsl = reinterpret_cast<uint8_t*>(smem) + TC::RING;
  uint8_t* wsl = xsl + a.Kb * TC::BM;
  load_scales<TC>(a, xsl, wsl, m0, n0, rows);

  f32x16 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  const int frow = lane & 31, half = lane >> 5;
  const int xrow = wm * TC::WTM + frow, wrow = TC::BM + wn * TC::WTN + frow;
  const int wblk = (n0 % 128 + wn * TC::WTN) / 128;         // the wave's columns lie in one weight block
  auto frag = [&](const char* st, int row, int t) {
    i32x8 f;
    const u32x4 lo = *reinterpret_cast<const u32x4*>(st + row * BLK + ((4 * t + 2 * half) ^ row_swizzle(row)) * 16);
    const u32x4 hi = *reinterpret_cast<const u32x4*>(st + row * BLK + ((4 * t + 2 * half + 1) ^ row_swizzle(row)) * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = (int)lo[e];
      f[4 + e] = (int)hi[e];
    }
    return f;
  };
  int slot = 0;
  for (int s = 0; s < nst; ++s) {
    if (nst - 1 - s >= NST - 2) wait_copies<(NST - 2) * NC>();
    else wait_copies<0>();
    wg_barrier();
    if (s + NST - 1 < nst) copy(s + NST - 1, slot == 0 ? NST - 1 : slot - 1);
    const char* st = smem + slot * TC::SLOT;
    int sx[MB];
    const int sw = wsl[s * TC::NBLK + wblk];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) sx[mb] = xsl[s * TC::BM + xrow + mb * 32];
    if constexpr (sizeof(T) == 4) {
      f32x16 part[NB][MB];                                  // the block's sums
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) part[i][j][e] = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x8 wa[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) widen32(frag(st, wrow + nb * 32, t), wa[nb]);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          bf16x8 xb[4];
          widen32(frag(st, xrow + mb * 32, t), xb);
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              part[nb][mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wa[nb][g], xb[g], part[nb][mb], 0, 0, 0);
        }
      }
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            acc[nb][mb][e] += scaled(part[nb][mb][e], sw, sx[mb]);
    } else
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      i32x8 fa[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) fa[nb] = frag(st, wrow + nb * 32, t);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const i32x8 fb = frag(st, xrow + mb * 32, t);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          acc[nb][mb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[nb], fb, acc[nb][mb], 0, 0, 0, sw, 0, sx[mb]);
      }
    }
    slot = slot + 1 == NST ? 0 : slot + 1;
  }
  wg_barrier();                                             // the ring is no longer read

  write_out<T, EPI, TC>(a, smem, acc, m0, n0, wave, lane);
}

// The large bf16 products: waves of 64 x 128 results, WGM x 2 of them.  Stages of 64 k
// (64 bytes of a row) in a ring of NST; the fragments of stage s + 1 are read under the
// matrix instructions of stage s, the w fragment of an n block into the registers that
// block has just released.  A stage's one barrier frees the slot of the stage before it
// for the copies of stage s + NST - 1; the reads of stage s may still be in flight there,
// those of stage s - 1 are over, because its matrix instructions have been issued.
// 8192^3 in 435 us, 2.53 PFLOP/s, the matrix units busy in 72% of the cycles at a clock of
// 1.71 GHz (of 2.4); 64800 x 4096 -> 1024 242 us; 64800 x 1024 -> 4096 300, with bias and
// GELU 363 (matrix units busy in 40%): there the epilogue is two fifths of a tile's time.
// Reads pinned a whole stage ahead, and four waves of 128 x 128 with a third less LDS
// traffic, measure the same within 2%.
template <int WGM_, int NST_, int LDS_>
struct Deep8 {
  static constexpr int WGM = WGM_, WGN = 2, MB = 2, NB = 4, NST = NST_, NW = WGM * WGN, KS = 64, LDS = LDS_;
  static constexpr int WTM = MB * 32, WTN = NB * 32, BM = WGM * WTM, BN = WGN * WTN;
  static constexpr int SLOT = (BM + BN) * KS, RING = NST * SLOT, NBLK = BN / 128;
  static constexpr int KB = (LDS - RING) / (BM + NBLK);     // longest rows: their scales fit behind the ring
  static constexpr int MINW = NW * (160 * 1024 / LDS) / 4;
};
using Big8 = Deep8<4, 4, 160 * 1024>;                       // 256 x 256, one workgroup a CU

// 16-byte slot of chunk c of a 64-byte stage row: conflict-free fragment reads whether 8
// lanes share 32 banks or 16 lanes 64.
__device__ __forceinline__ int swizzle64(int row) { return ((row >> 1) & 3) ^ ((row >> 3) & 1); }

template <typename T, int EPI, class TC>
__global__ __launch_bounds__(TC::NW * 64, TC::MINW) void linear_fp8_deep_kernel(Fp8Args a) {
  constexpr int MB = TC::MB, NB = TC::NB, NW = TC::NW, NST = TC::NST;
  __shared__ __attribute__((aligned(1024))) char smem[TC::LDS];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int wm = wave / TC::WGN, wn = wave % TC::WGN;
  const int MT = (int)((a.M + TC::BM - 1) / TC::BM), NT = (a.N + TC::BN - 1) / TC::BN;
  constexpr int GM = GROUP_M * 256 / TC::BM;                // tile order as linear_fp8_kernel
  const int tile = xcd_remap(blockIdx.x, MT * NT);
  const int gm0 = tile / (GM * NT) * GM, gsz = MT - gm0 < GM ? MT - gm0 : GM;
  const int tin = tile - gm0 * NT;
  const int64_t m0 = (int64_t)(gm0 + tin % gsz) * TC::BM;
  const int n0 = tin / gsz * TC::BN;
  const int rows = a.M - m0 < TC::BM ? (int)(a.M - m0) : TC::BM, cols = a.N - n0 < TC::BN ? a.N - n0 : TC::BN;

  // copy j of the wave: 16 stage rows, lane i row i / 4, 16-byte slot i % 4
  constexpr int CX = TC::BM / 16 / NW, CW = TC::BN / 16 / NW, NC = CX + CW;
  const u32x4 rx = make_rsrc(a.xq + m0 * a.K, (uint32_t)rows * (uint32_t)a.K);
  const u32x4 rw = make_rsrc(a.wq + (int64_t)n0 * a.K, (uint32_t)cols * (uint32_t)a.K);
  uint32_t v[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int r = (j < CX ? wave * CX + j : wave * CW + j - CX) * 16 + lane / 4, end = j < CX ? rows : cols;
    v[j] = (uint32_t)(r < end ? r : end - 1) * (uint32_t)a.K + (uint32_t)((lane % 4) ^ swizzle64(r)) * 16u;
  }
  const uint32_t lds = (uint32_t)(uintptr_t)smem;
  auto copy = [&](int s, int slot, int lo, int hi) {
#pragma unroll
    for (int j = 0; j < NC; ++j)
      if (j >= lo && j < hi)
        dma16(j < CX ? rx : rw,
              lds + slot * TC::SLOT + (j < CX ? (wave * CX + j) * 1024 : TC::BM * TC::KS + (wave * CW + j - CX) * 1024), v[j],
              (uint32_t)s * TC::KS);
  };
  const int ns = a.Kb * 2;                                  // stages; past the end the last one again, never used
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) copy(s < ns ? s : ns - 1, s, 0, NC);
  uint8_t* xsl = reinterpret_cast<uint8_t*>(smem) + TC::RING;
  uint8_t* wsl = xsl + a.Kb * TC::BM;
  load_scales<TC>(a, xsl, wsl, m0, n0, rows);

  const int frow = lane & 31, half = lane >> 5, nw = n0 + wn * TC::WTN;
  f32x16 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  // lane's offset of a fragment's first chunk in a slot; its second chunk is at ^ 16
  const uint32_t at = (uint32_t)(frow * TC::KS + ((2 * half) ^ swizzle64(frow)) * 16);
  const char* xp = smem + wm * TC::WTM * TC::KS;
  const char* wp = smem + (TC::BM + wn * TC::WTN) * TC::KS;
  auto frag = [&](const char* p) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(p + at), hi = *reinterpret_cast<const u32x4*>(p + (at ^ 16u));
    i32x8 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = (int)lo[e];
      f[4 + e] = (int)hi[e];
    }
    return f;
  };
  const uint8_t* xsp = xsl + wm * TC::WTM + frow;
  const uint8_t* wsp = wsl + wn;
  static_assert(TC::WTN == 128, "a wave's columns are one weight block");

  wait_copies<(NST - 2) * NC>();
  wg_barrier();
  i32x8 fa[NB], fb[2][MB];
  int sx[2][MB], sw[2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) fa[nb] = frag(wp + nb * 32 * TC::KS);
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    fb[0][mb] = frag(xp + mb * 32 * TC::KS);
    sx[0][mb] = xsp[mb * 32];
  }
  sw[0] = wsp[0];
  // stage s = s0 + u: slots, register sets and scale sets by constants
  constexpr int UNR = NST % 4 == 0 ? NST : NST % 2 == 0 ? 2 * NST : 4 * NST;
  for (int s0 = 0; s0 < ns; s0 += UNR) {
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int s = s0 + u;
      if (s < ns) {
        const int cs = s + NST - 1 < ns ? s + NST - 1 : ns - 1, kn = (s + 1 < ns ? s + 1 : s) >> 1;
        wait_copies<(NST - 3) * NC>();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const char* xn = xp + (u + 1) % NST * TC::SLOT;
        const char* wn_ = wp + (u + 1) % NST * TC::SLOT;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          copy(cs, (u + NST - 1) % NST, nb * NC / NB, (nb + 1) * NC / NB);
          if (nb < MB) fb[(u + 1) & 1][nb] = frag(xn + nb * 32 * TC::KS);
          if ((u & 1) == 1 && nb == 0) {                    // the next block's scales
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) sx[((u + 1) >> 1) & 1][mb] = xsp[kn * TC::BM + mb * 32];
            sw[((u + 1) >> 1) & 1] = wsp[kn * TC::NBLK];
          }
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
            acc[nb][mb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[nb], fb[u & 1][mb], acc[nb][mb], 0, 0, 0,
                                                                          sw[(u >> 1) & 1], 0, sx[(u >> 1) & 1][mb]);
          fa[nb] = frag(wn_ + nb * 32 * TC::KS);
        }
      }
    }
  }
  wait_copies();                                            // those past the last stage
  wg_barrier();                                             // the ring is no longer read
  write_out<T, EPI, TC>(a, smem, acc, m0, n0, wave, lane);
}

// Few rows: the weights' bytes and the latency count.  A workgroup of eight waves takes
// 16 columns and 16 MB rows; the waves share out the k blocks (one v_mfma_scale_f32_
// 16x16x128 or four of the 16-bit ones each), operands straight from global memory (lane
// (i, g): 32 bytes of row i, so a row's 128-byte line is four lanes' loads), and their
// sums meet in LDS in a fixed order.
template <typename T, int EPI, int MB>
__global__ __launch_bounds__(512) void linear_fp8_rows_kernel(Fp8Args a) {
  constexpr int NW = 8, U = MB == 4 ? 2 : 4;                // k blocks whose loads are in flight together
  __shared__ f32x4 red[NW][MB][64];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int i = lane & 15, g = lane >> 4, n0 = (int)blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MB);
  const uint8_t* wp = a.wq + (int64_t)(n0 + i < a.N ? n0 + i : a.N - 1) * a.K + g * 32;
  const uint8_t* wsp = a.ws + (int64_t)(n0 / 128) * a.Kb;
  const uint8_t *xp[MB], *xsp[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int64_t m = m0 + mb * 16 + i < a.M ? m0 + mb * 16 + i : a.M - 1;
    xp[mb] = a.xq + m * a.K + g * 32;
    xsp[mb] = a.xs + m * a.Kb;
  }
  auto load = [&](const uint8_t* p) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(p), hi = *reinterpret_cast<const u32x4*>(p + 16);
    i32x8 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = (int)lo[e];
      f[4 + e] = (int)hi[e];
    }
    return f;
  };
  f32x4 acc[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) acc[mb] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave; k0 < a.Kb; k0 += U * NW) {
    i32x8 fw[U], fx[U][MB];
    int sw[U], sx[U][MB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = k0 + u * NW;
      if (kb >= a.Kb) break;
      fw[u] = load(wp + (int64_t)kb * BLK);
      sw[u] = wsp[kb];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        fx[u][mb] = load(xp[mb] + (int64_t)kb * BLK);
        sx[u][mb] = xsp[mb][kb];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u * NW >= a.Kb) break;
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
          acc[mb] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[u], fx[u][mb], acc[mb], 0, 0, 0, sw[u], 0, sx[u][mb]);
      } else {
        bf16x8 w4[4], x4[4];
        widen32(fw[u], w4);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          widen32(fx[u][mb], x4);
          f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < 4; ++q) part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w4[q], x4[q], part, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[mb][e] += scaled(part[e], sw[u], sx[u][mb]);
        }
      }
    }
  }
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) red[wave][mb][lane] = acc[mb];
  __syncthreads();
  // lane (i, g) of block mb holds y[m0 + mb 16 + i][n0 + 4 g + r]
  if (wave >= MB) return;
  const int64_t m = m0 + wave * 16 + i;
  const int n = n0 + 4 * g;
  if (m >= a.M || n >= a.N) return;
  f32x4 t = red[0][wave][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) t += red[w][wave][lane];
  float b[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f}, o[4];
  if constexpr (EPI != EPI_NONE) load4<T>((const T*)a.bias + n, b);
  if constexpr (EPI == EPI_BIAS_RESIDUAL) load4<T>((const T*)a.residual + m * a.N + n, r);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = finish<T, EPI>(t[e], b[e]) + r[e];
  store4<T>((T*)a.y + m * a.N + n, o);
}

template <typename T, int EPI, int MB>
int launch_rows(const Fp8Args& a, hipStream_t st, const char* what) {
  hipLaunchKernelGGL((linear_fp8_rows_kernel<T, EPI, MB>), dim3((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 16 * MB - 1) / (16 * MB))),
                     dim3(512), 0, st, a);
  return check_launch(what);
}

int64_t tiles(int64_t M, int64_t N, int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); }

// Rows of the results of one workgroup: 16, 32 or 64 (the kernel for few rows), 128 or 256.
// Kernel by estimated time (us, fits to measured ones within 15%; bias and GELU, us
// few rows / 128 x 128 / 256 x 256):
//   1024 -> 4096 bf16   M 64: 4.9 / 9.1 / -    256: 14.5 / 9.3 / -    16384: - / 97 / 97     64800: - / 378 / 363
//   4096 -> 1024 bf16   M 64: 14.5 / 23.1 / -  512: 27.5 / 24.0 / -   8192: - / 39 / 47      16384: - / 74 / 64
//   1024 -> 4096 fp32   M 64: 5.0 / 15.0 / -   512: 27.9 / 15.4 / -
// Few rows: every workgroup reads its weights once more for each 64 rows.
template <typename T>
int tile_rows(int64_t M, int64_t N, int64_t Kb) {
  const double kb = (double)Kb;
  const int mr = M <= 16 ? 1 : M <= 32 ? 2 : 4;
  const double few = 2.3 + 0.0015 * kb * (double)tiles(M, N, 16 * mr, 16);
  const double mid = sizeof(T) == 2 ? std::max(4.5 + 0.61 * kb, (double)tiles(M, N, 128, 128) / 512 * (3.9 + 1.085 * kb))
                                    : std::max(5.5 + 1.0 * kb, (double)tiles(M, N, 128, 128) / 512 * (4 + 1.9 * kb));
  if (few < mid && M <= 64 * 65535LL) return 16 * mr;       // the grid's y
  if (sizeof(T) == 2 && 6 + (double)((tiles(M, N, Big8::BM, Big8::BN) + 255) / 256) * (8.5 + 1.53 * kb) < mid) return Big8::BM;
  return Mid8::BM;
}

template <typename T, int EPI>
int launch_fp8(const Fp8Args& a, hipStream_t st, const char* what) {
  const int rows = tile_rows<T>(a.M, a.N, a.Kb);
  if (rows == 16) return launch_rows<T, EPI, 1>(a, st, what);
  if (rows == 32) return launch_rows<T, EPI, 2>(a, st, what);
  if (rows == 64) return launch_rows<T, EPI, 4>(a, st, what);
  if constexpr (sizeof(T) == 2) {
    using TC = Big8;
    static_assert(TC::KB >= MAX_KB, "the longest rows' scales fit");
    if (rows == TC::BM) {
      const int64_t n = tiles(a.M, a.N, TC::BM, TC::BN);
      NSW_CHECK_ARG(n < (1LL << 31), "%s: too many tiles", what);
      hipLaunchKernelGGL((linear_fp8_deep_kernel<T, EPI, TC>), dim3((unsigned)n), dim3(TC::NW * 64), 0, st, a);
      return check_launch(what);
    }
  }
  using TC = Mid8;
  const int64_t n = tiles(a.M, a.N, TC::BM, TC::BN);
  NSW_CHECK_ARG(n < (1LL << 31), "%s: too many tiles", what);
  hipLaunchKernelGGL((linear_fp8_kernel<T, EPI, TC>), dim3((unsigned)n), dim3(TC::NW * 64), 0, st, a);
  return check_launch(what);
}

template <typename T>
int dispatch_fp8(const Fp8Args& a, int epilogue, hipStream_t st, const char* what) {
  switch (epilogue) {
    case NSW_EPI_NONE: return launch_fp8<T, EPI_NONE>(a, st, what);
    case NSW_EPI_BIAS: return launch_fp8<T, EPI_BIAS>(a, st, what);
    case NSW_EPI_BIAS_GELU: return launch_fp8<T, EPI_BIAS_GELU>(a, st, what);
    case NSW_EPI_BIAS_GELU_TANH: return launch_fp8<T, EPI_BIAS_GELU_TANH>(a, st, what);
    case NSW_EPI_BIAS_RESIDUAL: return launch_fp8<T, EPI_BIAS_RESIDUAL>(a, st, what);
    default: return set_error(NSW_ERR_INVALID, "%s: unknown epilogue %d", what, epilogue);
  }
}

template <typename T>
int launch_quantize(const void* x, void* q, void* scale, int64_t R, int64_t K, int rows, hipStream_t st, const char* what) {
  const int64_t Kb = (K + BLK - 1) / BLK;
  if (rows == 1) {
    const int64_t blocks = R * Kb, per = QT / 16 * 4, grid = (blocks + per - 1) / per;
    NSW_CHECK_ARG(blocks < (1LL << 32), "%s: too many blocks", what);
    hipLaunchKernelGGL((quantize_rows_kernel<T>), dim3((unsigned)grid), dim3(QT), 0, st, (const T*)x, (uint8_t*)q,
                       (uint8_t*)scale, (uint32_t)blocks, (int)K, (int)Kb, FastDiv::make((uint32_t)Kb));
  } else {
    NSW_CHECK_ARG((R + 127) / 128 < 65536, "%s: too many rows", what);
    hipLaunchKernelGGL((quantize_tiles_kernel<T>), dim3((unsigned)Kb, (unsigned)((R + 127) / 128)), dim3(QT), 0, st,
                       (const T*)x, (uint8_t*)q, (uint8_t*)scale, R, (int)K, (int)Kb);
  }
  return check_launch(what);
}

}  // namespace

}  // namespace nsw

using namespace nsw;

extern "C" int nsw_quantize_fp8(const void* x, void* q, void* scale, int64_t R, int64_t K, int rows_per_scale, int dtype,
                                void* stream) {
  const char* what = "nsw_quantize_fp8";
  NSW_CHECK_ARG(dtype == NSW_DTYPE_BF16 || dtype == NSW_DTYPE_F32, "%s: unknown dtype %d", what, dtype);
  NSW_CHECK_ARG(rows_per_scale == 1 || rows_per_scale == 128, "%s: a scale for 1 or 128 rows, got %d", what, rows_per_scale);
  const int64_t vec = dtype == NSW_DTYPE_BF16 ? 8 : 4;
  NSW_CHECK_ARG(R > 0 && R < (1LL << 40) && K > 0 && K < (1LL << 30) && K % vec == 0,
                "%s: R=%lld, K=%lld: K must be a positive multiple of %lld", what, (long long)R, (long long)K, (long long)vec);
  NSW_CHECK_ARG(x && q && scale, "%s: x, q and scale are required", what);
  NSW_CHECK_ARG((((uintptr_t)x | (uintptr_t)q) % 16) == 0, "%s: x and q must be 16-byte aligned", what);
  hipStream_t st = (hipStream_t)stream;
  return dtype == NSW_DTYPE_BF16 ? launch_quantize<bf16>(x, q, scale, R, K, rows_per_scale, st, what)
                                 : launch_quantize<float>(x, q, scale, R, K, rows_per_scale, st, what);
}

extern "C" int nsw_linear_fp8_tile_rows(int64_t M, int64_t N, int64_t K, int dtype) {
  if (M <= 0 || M >= (1LL << 38) || N <= 0 || N >= (1LL << 30) || N % 8 || K <= 0 || K % BLK || K > MAX_KB * BLK) return 0;
  return dtype == NSW_DTYPE_BF16 ? tile_rows<bf16>(M, N, K / BLK) : dtype == NSW_DTYPE_F32 ? tile_rows<float>(M, N, K / BLK) : 0;
}

extern "C" int nsw_linear_fp8(const void* xq, const void* xs, const void* wq, const void* ws, const void* bias,
                              const void* residual, void* y, int64_t M, int64_t N, int64_t K, int epilogue, int dtype,
                              void* stream) {
  const char* what = "nsw_linear_fp8";
  NSW_CHECK_ARG(dtype == NSW_DTYPE_BF16 || dtype == NSW_DTYPE_F32, "%s: unknown dtype %d", what, dtype);
  NSW_CHECK_ARG(M > 0 && M < (1LL << 38) && N > 0 && N < (1LL << 30) && K > 0 && K < (1LL << 30),
                "%s: M, N, K must be positive", what);
  NSW_CHECK_ARG(K % BLK == 0, "%s: K=%lld must be a multiple of 128 (rows are padded with zeros)", what, (long long)K);
  NSW_CHECK_ARG(K <= MAX_KB * BLK, "%s: K=%lld, at most %d", what, (long long)K, MAX_KB * BLK);
  NSW_CHECK_ARG(N % 8 == 0, "%s: N=%lld must be a multiple of 8", what, (long long)N);
  NSW_CHECK_ARG(xq && xs && wq && ws && y, "%s: xq, xs, wq, ws and y are required", what);
  NSW_CHECK_ARG(epilogue == NSW_EPI_NONE || bias, "%s: epilogue %d needs a bias", what, epilogue);
  NSW_CHECK_ARG(epilogue != NSW_EPI_BIAS_RESIDUAL || residual, "%s: residual epilogue needs a residual", what);
  NSW_CHECK_ARG((((uintptr_t)xq | (uintptr_t)wq | (uintptr_t)bias | (uintptr_t)residual | (uintptr_t)y) % 16) == 0,
                "%s: xq, wq, bias, residual and y must be 16-byte aligned", what);
  Fp8Args a{};
  a.xq = (const uint8_t*)xq; a.xs = (const uint8_t*)xs; a.wq = (const uint8_t*)wq; a.ws = (const uint8_t*)ws;
  a.bias = bias; a.residual = residual; a.y = y; a.M = M; a.N = (int)N; a.K = (int)K; a.Kb = (int)(K / BLK);
  return dtype == NSW_DTYPE_BF16 ? dispatch_fp8<bf16>(a, epilogue, (hipStream_t)stream, what)
                                 : dispatch_fp8<float>(a, epilogue, (hipStream_t)stream, what);
}
