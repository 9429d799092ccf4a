// 16-bit products on bf16 / fp16 MFMA (gfx950), shared by the forward and the
// backward passes of the linear layers.
//
// C[m, n] = sum over k of A(m, k) W(n, k), float32 sums. Each operand is read
// either along k (KC: element (r, k) at r * ld + k; the forward's x and w, dx's
// dz) or along its rows (RC: at k * ld + r; dx's w, dw's dz and x).
//
//   workgroup tile  BN x BM = (32*WN*FN) x (32*WM*FM), WN x WM waves
//   wave tile       FN x FM MFMA blocks of 32 x 32 (v_mfma_f32_32x32x16)
//
// C^T layout: a lane's accumulators belong to one m and 4 consecutive n per
// register quad. Operands go from global memory straight into a ring of S LDS
// stages of 64 k (global_load_lds_dwordx4), one barrier per stage, fragments
// read one k-step ahead: the structure of the int8 GEMM (gemm.hip), whose stage
// of 128 k-bytes is the same number of bytes and of MFMA cycles.
//
// KC stage: [rows][64 k], 16-byte chunk c of row r at c ^ ((r / 2) % 8); a
//   fragment (8 k of one row) is one 16-byte read.
// RC stage: [64 k][rows]; a fragment is two ds_read_b64_tr_b16, each of which
//   takes a 4 (k) x 16 (rows) block per 16 lanes and hands every lane the 4 k
//   of its row. 16-row pair of chunks p of line k sits at p ^ (k & 3), and in
//   lines of whole 256 bytes with bit 2 flipped for odd p: the four lines of a
//   block fall on different banks, and so do the two blocks of a 32-row fragment.
//
// The contraction's end inside a stage: loads clamp to the last k (rows to the
// last row), and the last stage's fragments are masked. Of two terms the first
// ends on whole stages: A has zeros up to there, and w's lines are read as zeros.
#pragma once

#include "colsum.h"

namespace dc {

// One DMA of 16 bytes per lane into LDS (see dma16) from an address of each lane's own.
__device__ __forceinline__ void dma16_at(const void* lane, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(lane),
               "{m0}"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}

// As in gemm.hip: vmcnt(n) with the other counters left unconstrained, and lgkmcnt(0) (gfx9
// encoding: vmcnt bits 3:0 and 15:14, expcnt 6:4, lgkmcnt 11:8)
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt has 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}
__device__ __forceinline__ void wait_lgkmcnt0() { __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4)); }

// Sets a kernel's dynamic LDS limit, once per instantiation and device
// (`done`: its flags); threads that race on a first call each set it (the call
// is idempotent).
inline int reserve_lds(const void* fn, int bytes, std::atomic<bool> (&done)[64], const char* what) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
  if (done[dev].load(std::memory_order_acquire)) return DC_OK;
  hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) {
    set_error("%s: cannot reserve %d bytes of LDS: %s", what, bytes, hipGetErrorString(e));
    return DC_EHIP;
  }
  done[dev].store(true, std::memory_order_release);
  return DC_OK;
}

struct Gemm16 {
  const uint16_t *a, *a2;   // a2: the second term's (terms == 2) or second problem's A
  const uint16_t *w, *w2;   // w2: the second term's W, or the gate's
  int64_t lda, ldw, ldw2;
  int M, N;                 // outputs; N counts channels of a gated product once
  int K;                    // k of a term
  int ka;                   // k that a term's A rows (KC) can be read to, a multiple of 8
  int nk1, nk;              // stages of the first term, and of all
  const uint16_t* zeros;    // two terms: 16 bytes of zeros, 16-byte aligned
  int wlim, alim;           // rows of W and A that loads may touch (RC: rounded up to 8)
  int tiles_m, tiles_n;
  int problems;             // 2: a second product (a2, out2) in the same launch
  int act, bias_dtype;
  const void *bias, *bias2;
  const uint16_t* res;
  uint16_t *out, *out2;
  uint8_t *z, *z2;          // store_saved8
  int64_t ldr, ldo;
  // split-K: blockIdx.y takes `kstages` stages and writes float32 sums to
  // part + (y * problems + problem) * M * width, row stride `width`
  float* part;
  int splits, kstages, width;
};

// How a product runs: the tile (an index of the tile list) and its k slices.
struct Plan16 {
  int tile, splits, kstages;
};

template <int WN_, int WM_, int FN_, int FM_, int S_, int OCC_>
struct Tile16 {
  static constexpr int WN = WN_, WM = WM_, FN = FN_, FM = FM_, S = S_;
  static constexpr int OCC = OCC_;                 // waves per SIMD the registers must allow
  static constexpr int NW = WN * WM, NT = 64 * NW;
  static constexpr int BN = 32 * WN * FN, BM = 32 * WM * FM;
  static constexpr int STAGE = (BN + BM) * 128;    // bytes
  static constexpr int LW = BN / 8 / NW, LA = BM / 8 / NW;   // DMA instructions per wave and stage
  static constexpr int LDS = S * STAGE;
  static_assert(BN % (8 * NW) == 0 && BM % (8 * NW) == 0, "whole DMA instructions per wave");
  static_assert(LDS <= 160 * 1024, "LDS per CU");
};

template <int DT>
__device__ __forceinline__ v16f mfma16(v4i w, v4i a, v16f c) {
  if constexpr (DT == DC_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, a), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, a), c, 0, 0, 0);
}

__device__ __forceinline__ float bias_at(const void* b, int dtype, int64_t n) {
  if (!b) return 0.0f;
  if (dtype == DC_F32) return static_cast<const float*>(b)[n];
  const uint32_t u = static_cast<const uint16_t*>(b)[n];
  return dtype == DC_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
}

typedef short v4s __attribute__((ext_vector_type(4)));
__device__ __forceinline__ int2 lds_read_tr(const uint8_t* p) {
  return __builtin_bit_cast(int2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                      (__attribute__((address_space(3))) v4s*)(const_cast<uint8_t*>(p))));
}

// Where 16-row pair `p` of line k of an RC stage sits (its own inverse but for
// bit 2: see rc_logical). R: rows of the stage.
template <int R>
__device__ __forceinline__ int rc_physical(int p, int k) {
  const int q = p ^ (k & 3);
  return R % 128 == 0 ? q ^ ((p & 1) << 2) : q;
}
template <int R>
__device__ __forceinline__ int rc_logical(int q, int k) {
  const int p = q ^ (k & 3);
  return R % 128 == 0 ? p ^ ((p & 1) << 2) : p;
}

// Keeps the `valid` (0 .. 8) first of a fragment's 8 values.
__device__ __forceinline__ v4i keep_first(v4i f, int valid) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = valid - 2 * j;
    f[j] = n >= 2 ? f[j] : n == 1 ? (f[j] & 0xffff) : 0;
  }
  return f;
}

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// One wave's FN x FM blocks leave through its share of the LDS ring, 32 rows at
// a time, float32: put(row, chunk, v) gets 8 consecutive columns of one row
// (chunk: which 8 of the 32 * FN), lanes along the row.
template <int FN, int FM, class Put>
__device__ __forceinline__ void rows_f32(const v16f (&acc)[FN][FM], uint8_t* stage, int lane, Put&& put) {
  constexpr int RP = 32 * FN * 4 + 16, CH = 4 * FN;
  const int hf = lane >> 5, l32 = lane & 31;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    if (j) wave_lds_fence();   // the last block has been read
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(stage + l32 * RP + 4 * (32 * i + 8 * g + 4 * hf)) =
            make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
    wave_lds_fence();
#pragma unroll
    for (int q = lane; q < 32 * CH; q += 64) {
      const int r = q / CH, c = q % CH;
      const float4 lo = *reinterpret_cast<const float4*>(stage + r * RP + 32 * c);
      const float4 hi = *reinterpret_cast<const float4*>(stage + r * RP + 32 * c + 16);
      const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      put(32 * j + r, c, v);
    }
  }
}

// The same with the lane's column fixed and a gated tile's value and gate
// columns together: put(row, values, gates), 8 columns of one row.
template <int FN, int FM, bool GATED, class Put>
__device__ __forceinline__ void rows_pre(const v16f (&acc)[FN][FM], uint8_t* stage, int lane, Put&& put) {
  constexpr int RP = 32 * FN * 4 + 16, CH = GATED ? 2 * FN : 4 * FN;
  const int hf = lane >> 5, l32 = lane & 31;
  const int c = lane % CH, at = GATED ? c / 4 * 256 + c % 4 * 32 : 32 * c;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    if (j) wave_lds_fence();
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(stage + l32 * RP + 4 * (32 * i + 8 * g + 4 * hf)) =
            make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
    wave_lds_fence();
#pragma unroll
    for (int k = 0; k < 32 * CH / 64; ++k) {
      const int r = lane / CH + k * (64 / CH);
      float v[8], g[8];
#pragma unroll
      for (int q = 0; q < 8; q += 4) {
        const float4 x = *reinterpret_cast<const float4*>(stage + r * RP + at + 4 * q);
        v[q] = x.x, v[q + 1] = x.y, v[q + 2] = x.z, v[q + 3] = x.w;
        if constexpr (GATED) {
          const float4 y = *reinterpret_cast<const float4*>(stage + r * RP + at + 128 + 4 * q);
          g[q] = y.x, g[q + 1] = y.y, g[q + 2] = y.z, g[q + 3] = y.w;
        }
      }
      put(32 * j + r, v, g);
    }
  }
}

// Rounded to 16 bits before LDS: put(row, chunk, uint4).
template <int DT, int FN, int FM, class Put>
__device__ __forceinline__ void rows_h16(const v16f (&acc)[FN][FM], uint8_t* stage, int lane, Put&& put) {
  constexpr int RP = 32 * FN * 2 + 16, CH = 4 * FN;
  const int hf = lane >> 5, l32 = lane & 31;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    if (j) wave_lds_fence();
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v16f& a = acc[i][j];
        const v2f lo = {a[4 * g], a[4 * g + 1]}, hi = {a[4 * g + 2], a[4 * g + 3]};
        uint2 u;
        if constexpr (DT == DC_BF16)
          u = make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, v2bf)),
                         __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, v2bf)));
        else
          u = make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, v2h)),
                         __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, v2h)));
        *reinterpret_cast<uint2*>(stage + l32 * RP + 2 * (32 * i + 8 * g + 4 * hf)) = u;
      }
    wave_lds_fence();
#pragma unroll
    for (int q = lane; q < 32 * CH; q += 64) {
      const int r = q / CH, c = q % CH;
      put(32 * j + r, c, *reinterpret_cast<const uint4*>(stage + r * RP + 16 * c));
    }
  }
}

// EPI: 0 the sums alone (backward), 1 bias / activation / residual, 2 gated.
enum { EPI_NONE = 0, EPI_LINEAR = 1, EPI_GATED = 2 };

template <class T, int DT, bool A_RC, bool W_RC, int EPI>
__global__ void __launch_bounds__(T::NT, T::OCC) linear16_kernel(Gemm16 p) {
  constexpr int FN = T::FN, FM = T::FM, BN = T::BN, BM = T::BM, S = T::S, L = T::LW + T::LA;
  constexpr bool GATED = EPI == EPI_GATED;
  constexpr int ON = GATED ? BN / 2 : BN;   // output channels of the tile
  static_assert(!GATED || (FN % 2 == 0 && !W_RC), "value and gate blocks alternate");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int l32 = lane & 31, hf = lane >> 5;
  const int wn = w % T::WN, wm = w / T::WN;

  // tile: XCD-contiguous ranges (workgroups are dealt round-robin over 8), then 8 m-tiles per sweep along n
  const int nwg = gridDim.x, per = nwg / 8, rest = nwg % 8, xcd = blockIdx.x % 8;
  int logical = xcd * per + min(xcd, rest) + blockIdx.x / 8;
  const int per_problem = p.tiles_m * p.tiles_n;
  const int problem = logical >= per_problem ? 1 : 0;
  logical -= problem * per_problem;
  const int band = 8 * p.tiles_n, first = logical / band * 8, high = min(p.tiles_m - first, 8);
  const int m0 = (first + logical % band % high) * BM, n0 = logical % band / high * ON;
  if (problem) p.a = p.a2, p.out = p.out2;

  int kt = 0, kend = p.nk;
  if (p.splits > 1) {
    kt = blockIdx.y * p.kstages;
    kend = min(kt + p.kstages, p.nk);
  }

  // The bias of W row `lane` of the wave's 64 (gated: 32 value, then 32 gate
  // rows), as loaded: issued ahead of the operands, converted after the main loop.
  uint32_t bias_raw = 0u;
  if constexpr (EPI != EPI_NONE) {
    static_assert(FN == 2, "a lane per W row of the wave");
    const void* b = GATED && hf ? p.bias2 : p.bias;
    const int n = min(GATED ? n0 + 32 * wn + l32 : n0 + 64 * wn + lane, p.N - 1);
    if (p.bias_dtype == DC_F32) {
      if (b) bias_raw = static_cast<const uint32_t*>(b)[n];
    } else {
      if (b) bias_raw = static_cast<const uint16_t*>(b)[n];
    }
  }

  // DMA sources: byte offsets from the tile's first row (KC) or column (RC)
  uint32_t woff[T::LW], aoff[T::LA];
  auto off_kc = [&](int u, int r0, int lim, int64_t ld) __attribute__((always_inline)) {
    const int r = 8 * (w + T::NW * u) + lane / 8;
    return (uint32_t)((min(r0 + r, lim - 1) - r0) * (uint32_t)ld * 2 + 16 * ((lane % 8) ^ ((r >> 1) & 7)));
  };
  // line and column of chunk `lane` of DMA instruction u of an RC stage of R rows
  auto rc_line = [&](int u, int R) __attribute__((always_inline)) { return (64 * (w + T::NW * u) + lane) / (R / 8); };
  auto rc_col = [&](int u, auto R_, int r0, int lim) __attribute__((always_inline)) {
    constexpr int R = decltype(R_)::value;
    const int q = (64 * (w + T::NW * u) + lane) % (R / 8);
    const int col = 16 * rc_logical<R>(q >> 1, rc_line(u, R)) + 8 * (q & 1);
    return min(r0 + col, lim - 8) - r0;
  };
  typedef std::integral_constant<int, BN> RW;
  typedef std::integral_constant<int, BM> RA;
#pragma unroll
  for (int u = 0; u < T::LW; ++u) {
    if constexpr (W_RC) {
      woff[u] = (uint32_t)rc_line(u, BN) * (uint32_t)p.ldw * 2 + 2 * rc_col(u, RW{}, n0, p.wlim);
    } else if constexpr (GATED) {
      // 8 rows of one 32-row block, value and gate blocks in turn
      const int r = 8 * (w + T::NW * u) + lane / 8, blk = r / 32, ch = n0 + blk / 2 * 32 + r % 32;
      const uint32_t ld = (uint32_t)((blk & 1) ? p.ldw2 : p.ldw);
      woff[u] = (min(ch, p.wlim - 1) - n0) * ld * 2 + 16 * ((lane % 8) ^ ((r >> 1) & 7));
    } else {
      woff[u] = off_kc(u, n0, p.wlim, p.ldw);
    }
  }
#pragma unroll
  for (int u = 0; u < T::LA; ++u) {
    if constexpr (A_RC) aoff[u] = (uint32_t)rc_line(u, BM) * (uint32_t)p.lda * 2 + 2 * rc_col(u, RA{}, m0, p.alim);
    else aoff[u] = off_kc(u, m0, p.alim, p.lda);
  }
  const uint16_t* at0 = A_RC ? p.a + m0 : p.a + (int64_t)m0 * p.lda;
  const uint16_t* at1 = A_RC || !p.a2 ? at0 : p.a2 + (int64_t)m0 * p.lda;
  const uint16_t* wt0 = W_RC ? p.w + n0 : p.w + (int64_t)n0 * p.ldw;
  const uint16_t* wt1 = !p.w2 ? wt0 : W_RC ? p.w2 + n0 : p.w2 + (int64_t)n0 * p.ldw2;
  const uint32_t lds0 = lds_addr(smem) + 1024 * w;
  auto issue = [&](int s, int slot) __attribute__((always_inline)) {
    const bool second = s >= p.nk1;
    const int k0 = 64 * (second ? s - p.nk1 : s);
    const uint16_t* ab = (second ? at1 : at0) + (A_RC ? k0 * p.lda : k0);
    const uint16_t* wb = (!GATED && second ? wt1 : wt0) + (W_RC ? k0 * p.ldw : k0);
    const uint16_t* gb = GATED ? wt1 + k0 : wb;
    const uint32_t d = lds0 + slot * T::STAGE;
    const int left = p.K - k0;   // k of the term from this stage on
    if (left >= 64) {
#pragma unroll
      for (int u = 0; u < T::LW; ++u)
        dma16(GATED && (((w + T::NW * u) / 4) & 1) ? gb : wb, woff[u], d + 1024 * T::NW * u);
#pragma unroll
      for (int u = 0; u < T::LA; ++u) dma16(ab, aoff[u], d + BN * 128 + 1024 * T::NW * u);
    } else {
      // the term ends in this stage: chunks (KC) and lines (RC) past it read the last ones again
      const int last = (left + 7) / 8 - 1, lasta = min(8, (p.ka - k0) / 8) - 1;
#pragma unroll
      for (int u = 0; u < T::LW; ++u) {
        const int r = 8 * (w + T::NW * u) + lane / 8, c = (lane % 8) ^ ((r >> 1) & 7), ln = rc_line(u, BN);
        const uint32_t o = W_RC ? woff[u] - (uint32_t)(ln - min(ln, left - 1)) * (uint32_t)p.ldw * 2
                                : woff[u] - 16 * (c - min(c, last));
        if constexpr (W_RC && !A_RC) {
          // where a first term ends, its A holds zeros that meet w's lines past the
          // end: zeros too, as 0 times an infinite w would be NaN
          const uint8_t* at = reinterpret_cast<const uint8_t*>(wb) + o;
          if (p.zeros && ln >= left) at = reinterpret_cast<const uint8_t*>(p.zeros);
          dma16_at(at, d + 1024 * T::NW * u);
        } else {
          dma16(GATED && (((w + T::NW * u) / 4) & 1) ? gb : wb, o, d + 1024 * T::NW * u);
        }
      }
#pragma unroll
      for (int u = 0; u < T::LA; ++u) {
        const int r = 8 * (w + T::NW * u) + lane / 8, c = (lane % 8) ^ ((r >> 1) & 7), ln = rc_line(u, BM);
        const uint32_t o = A_RC ? aoff[u] - (uint32_t)(ln - min(ln, left - 1)) * (uint32_t)p.lda * 2
                                : aoff[u] - 16 * (c - min(c, lasta));
        dma16(ab, o, d + BN * 128 + 1024 * T::NW * u);
      }
    }
  };

  // fragment reads: per-lane base of each block, plus immediates
  const int swz = (l32 >> 1) & 7;
  uint32_t wbase[W_RC ? FN : 1], abase[A_RC ? FM : 1];
  const int kline = 8 * hf + ((lane & 15) >> 2);   // RC: this lane's line of a k-step's first read
  if constexpr (W_RC) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
      wbase[i] = kline * BN * 2 + 32 * rc_physical<BN>(2 * (wn * FN + i) + ((lane >> 4) & 1), kline) + 8 * (lane & 3);
  } else {
    wbase[0] = (wn * 32 * FN + l32) * 128;
  }
  if constexpr (A_RC) {
#pragma unroll
    for (int j = 0; j < FM; ++j)
      abase[j] = BN * 128 + kline * BM * 2 + 32 * rc_physical<BM>(2 * (wm * FM + j) + ((lane >> 4) & 1), kline) +
                 8 * (lane & 3);
  } else {
    abase[0] = BN * 128 + (wm * 32 * FM + l32) * 128;
  }
  int kc[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) kc[ks] = 16 * ((2 * ks + hf) ^ swz);

  v16f acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = v16f{0};
  v4i wf[2][FN], af[2][FM];
  auto frags = [&](int buf, int slot, int ks) __attribute__((always_inline)) {
    const uint8_t* b = smem + slot * T::STAGE;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if constexpr (W_RC) {
        const int2 lo = lds_read_tr(b + wbase[i] + ks * 16 * BN * 2);
        const int2 hi = lds_read_tr(b + wbase[i] + (ks * 16 + 4) * BN * 2);
        wf[buf][i] = v4i{lo.x, lo.y, hi.x, hi.y};
      } else {
        wf[buf][i] = *reinterpret_cast<const v4i*>(b + wbase[0] + kc[ks] + 32 * 128 * i);
      }
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      if constexpr (A_RC) {
        const int2 lo = lds_read_tr(b + abase[j] + ks * 16 * BM * 2);
        const int2 hi = lds_read_tr(b + abase[j] + (ks * 16 + 4) * BM * 2);
        af[buf][j] = v4i{lo.x, lo.y, hi.x, hi.y};
      } else {
        af[buf][j] = *reinterpret_cast<const v4i*>(b + abase[0] + kc[ks] + 32 * 128 * j);
      }
    }
  };
  // the last stage's fragments past the contraction's end, zeroed
  auto mask = [&](int buf, int ks, int left) __attribute__((always_inline)) {
    const int valid = max(0, min(8, left - 16 * ks - 8 * hf));
#pragma unroll
    for (int i = 0; i < FN; ++i) wf[buf][i] = keep_first(wf[buf][i], valid);
#pragma unroll
    for (int j = 0; j < FM; ++j) af[buf][j] = keep_first(af[buf][j], valid);
  };
  auto mfmas = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = mfma16<DT>(wf[buf][i], af[buf][j], acc[i][j]);
  };
  // waits until at most the newest n stages of this wave's loads are in flight
  auto wait_left = [&](int n) __attribute__((always_inline)) {
    static_assert(S <= 4, "wait_left handles up to 3 stages in flight");
    if (S > 3 && n >= 3) wait_vmcnt<3 * L>();
    else if (S > 2 && n >= 2) wait_vmcnt<2 * L>();
    else if (n >= 1) wait_vmcnt<L>();
    else wait_vmcnt<0>();
  };
  auto sync = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

#pragma unroll
  for (int s = 0; s < S; ++s)
    if (kt + s < kend) issue(kt + s, s);
  wait_left(min(kend - kt, S) - 1);
  sync();
  int slot = 0;
  if (kt + 1 < kend) frags(0, 0, 0);
  // stage kt in `slot`; MORE: stage kt + S exists
  auto stage = [&](auto more) __attribute__((always_inline)) {
    constexpr bool MORE = decltype(more)::value;
#pragma unroll
    for (int ks = 0; ks < 3; ++ks) {
      frags((ks + 1) & 1, slot, ks + 1);
      mfmas(ks & 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    const int next = slot == S - 1 ? 0 : slot + 1;
    if constexpr (MORE) wait_vmcnt<(S - 2) * L>();
    else wait_left(kend - 2 - kt);
    wait_lgkmcnt0();
    sync();
    frags(0, next, 0);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MORE) issue(kt + S, slot);
    mfmas(1);
    __builtin_amdgcn_sched_barrier(0);
    slot = next;
    ++kt;
  };
  while (kt + S < kend) stage(std::true_type{});
  while (kt + 1 < kend) stage(std::false_type{});
  if (kt < kend) {
    const int left = p.K - 64 * (kt >= p.nk1 ? kt - p.nk1 : kt);
    frags(0, slot, 0);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks < 3) frags((ks + 1) & 1, slot, ks + 1);
      if (left < 64) mask(ks & 1, ks, left);
      mfmas(ks & 1);
    }
  }
  __syncthreads();   // every wave is done reading the ring

  // epilogue
  constexpr int WAVE_BYTES = S * T::STAGE / T::NW / 16 * 16;
  static_assert(32 * (32 * FN * 4 + 16) <= WAVE_BYTES, "one 32-row block must fit the wave's LDS share");
  uint8_t* share = smem + w * WAVE_BYTES;
  const int mb = m0 + wm * 32 * FM;                    // the wave's first row
  const int nb = n0 + wn * 32 * (GATED ? FN / 2 : FN);   // and first output channel
  if (p.splits > 1) {
    float* part = p.part + ((int64_t)blockIdx.y * p.problems + problem) * p.M * p.width;
    rows_f32<FN, FM>(acc, share, lane, [&](int r, int c, const float (&v)[8]) __attribute__((always_inline)) {
      const int m = mb + r;
      if (m >= p.M) return;
      if constexpr (GATED) {
        const int n = nb + c / 8 * 32 + c % 4 * 8;   // 4 chunks of values, then 4 of gates
        store8_n(part + (int64_t)m * p.width + (c / 4 & 1) * p.N + n, p.N - n, v);
      } else {
        const int n = nb + 8 * c;
        store8_n(part + (int64_t)m * p.width + n, p.N - n, v);
      }
    });
    return;
  }
  if constexpr (EPI != EPI_NONE) {
    // the wave's biases through the end of its LDS share; each lane's 8 columns
    // are the same in every step
    constexpr int CH = GATED ? 2 * FN : 4 * FN;   // output chunks of a row
    static_assert(32 * (32 * FN * 4 + 16) + 256 <= WAVE_BYTES, "the biases follow a staged block");
    const int oc = lane % CH;
    float* b_l = reinterpret_cast<float*>(share + WAVE_BYTES - 256);
    asm volatile("" : "+v"(bias_raw));   // not converted, and waited for, where it is loaded
    b_l[lane] = p.bias_dtype == DC_F32 ? __uint_as_float(bias_raw) : h16_to_f32<DT>(bias_raw);
    wave_lds_fence();
    float bv[8], bg[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bv[e] = b_l[8 * oc + e], bg[e] = GATED ? b_l[32 + 8 * oc + e] : 0.0f;
    const int n = nb + 8 * oc;
    // one uniform branch around the whole of it, so that the steps of a block overlap
    with_act(p.act, [&](auto act_) __attribute__((always_inline)) {
      constexpr int ACT = decltype(act_)::value;
      auto put = [&](int r, float (&v)[8], float (&g)[8]) __attribute__((always_inline)) {
        const int m = mb + r;
        if (m >= p.M || n >= p.N) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] += bv[e];
          if constexpr (GATED) g[e] += bg[e];
        }
        if (p.z) {
          store_saved8(p.z, p.M, p.N, m, n, v);
          if constexpr (GATED) store_saved8(p.z2, p.M, p.N, m, n, g);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (GATED) v[e] *= act_value<ACT>(g[e]);
          else v[e] = act_value<ACT>(v[e]);
        }
        if (!GATED && p.res) {
          float s[8];
          load8_n<DT>(p.res + (int64_t)m * p.ldr + n, p.N - n, s);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += s[e];
        }
        store_chunk16(p.out + (int64_t)m * p.ldo + n, p.N - n, pack8<DT>(v));
      };
      rows_pre<FN, FM, GATED>(acc, share, lane, put);
    });
  } else {
    rows_h16<DT, FN, FM>(acc, share, lane, [&](int r, int c, uint4 v) __attribute__((always_inline)) {
      const int m = mb + r;
      const int n = nb + 8 * c;
      if (m < p.M) store_chunk16(p.out + (int64_t)m * p.ldo + n, p.N - n, v);
    });
  }
}

// ---------------------------------------------------------------- split-K join

// Sums the slices' partials in order and applies the epilogue: a thread takes 8
// columns of a row.
template <int DT, int EPI>
__global__ void __launch_bounds__(256) linear16_join_kernel(Gemm16 p) {
  constexpr bool GATED = EPI == EPI_GATED;
  const int n8 = (p.N + 7) / 8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= (int64_t)n8 * p.M) return;
  const int64_t m = idx / n8;
  const int n = (int)(idx % n8) * 8, left = p.N - n, problem = blockIdx.y;
  const int64_t plane = (int64_t)p.M * p.width;
  const float* src = p.part + problem * plane + m * p.width + n;
  float v[8] = {0}, g[8] = {0};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    float x[8];
    load8_n(src + s * p.problems * plane, left, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += x[e];
    if constexpr (GATED) {
      load8_n(src + s * p.problems * plane + p.N, left, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] += x[e];
    }
  }
  if constexpr (EPI != EPI_NONE) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= left) break;
      v[e] += bias_at(p.bias, p.bias_dtype, n + e);
      if constexpr (GATED) g[e] += bias_at(p.bias2, p.bias_dtype, n + e);
    }
    if (p.z) {
      store_saved8(p.z, p.M, p.N, m, n, v);
      if constexpr (GATED) store_saved8(p.z2, p.M, p.N, m, n, g);
    }
    with_act(p.act, [&](auto act_) __attribute__((always_inline)) {
      constexpr int ACT = decltype(act_)::value;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (GATED) v[e] *= act_value<ACT>(g[e]);
        else v[e] = act_value<ACT>(v[e]);
      }
    });
    if (!GATED && p.res) {
      float r[8];
      load8_n<DT>(p.res + m * p.ldr + n, left, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += r[e];
    }
  }
  store_chunk16((problem ? p.out2 : p.out) + m * p.ldo + n, left, pack8<DT>(v));
}

// ---------------------------------------------------------------- launch

template <class T, int DT, bool A_RC, bool W_RC, int EPI>
int launch16(const char* who, Gemm16 p, const Plan16& plan, hipStream_t st) {
  constexpr int ON = EPI == EPI_GATED ? T::BN / 2 : T::BN;
  p.tiles_n = (p.N + ON - 1) / ON;
  p.tiles_m = (p.M + T::BM - 1) / T::BM;
  p.splits = plan.splits, p.kstages = plan.kstages;
  const int64_t tiles = (int64_t)p.tiles_n * p.tiles_m * p.problems;
  if (tiles > 0x7fffffff) return fail(DC_EINVAL, "linear16: problem too large");
  static std::atomic<bool> attr_set[64];
  auto kernel = &linear16_kernel<T, DT, A_RC, W_RC, EPI>;
  if (int e = reserve_lds(reinterpret_cast<const void*>(kernel), T::LDS, attr_set, "linear16_kernel")) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, p.splits > 1 ? p.splits : 1), dim3(T::NT), T::LDS, st, p);
  if (int e = launch_status(who)) return e;
  if (p.splits > 1) {
    const int64_t chunks = (int64_t)((p.N + 7) / 8) * p.M;
    hipLaunchKernelGGL((linear16_join_kernel<DT, EPI>), dim3((unsigned)((chunks + 255) / 256), p.problems), dim3(256),
                       0, st, p);
    return launch_status(who);
  }
  return DC_OK;
}

// Tiles (n x m); EPI_GATED ones hold half as many channels.
typedef Tile16<4, 2, 2, 4, 2, 2> T256x256;    // 8 waves of 64 x 128, 128 KB: 1 per CU
typedef Tile16<4, 2, 2, 3, 2, 2> T256x192;    // 8 waves of 64 x 96, 112 KB: 1 per CU
typedef Tile16<4, 2, 2, 2, 3, 2> T256x128;    // 8 waves of 64 x 64, 144 KB: 1 per CU
typedef Tile16<2, 4, 2, 2, 3, 2> T128x256;    // 8 waves of 64 x 64, 144 KB: 1 per CU
typedef Tile16<2, 2, 2, 3, 2, 2> T128x192;    // 4 waves of 64 x 96, 80 KB: 2 per CU
typedef Tile16<2, 2, 2, 2, 2, 2> T128x128;    // 4 waves of 64 x 64, 64 KB: 2 per CU
typedef Tile16<2, 4, 2, 1, 3, 2> T128x128d;   // 8 waves of 64 x 32, 96 KB: 1 per CU
typedef Tile16<1, 4, 2, 1, 3, 2> T64x128;     // 4 waves of 64 x 32, 72 KB: 2 per CU
typedef Tile16<1, 2, 2, 1, 3, 2> T64x64;      // 2 waves of 64 x 32, 48 KB: 3 per CU
enum {
  TILE_256x256, TILE_256x192, TILE_256x128, TILE_128x256, TILE_128x192, TILE_128x128, TILE_128x128D, TILE_64x128,
  TILE_64x64
};

template <int DT, bool A_RC, bool W_RC, int EPI>
int run_tile16(const char* who, const Gemm16& p, const Plan16& plan, hipStream_t st) {
  switch (plan.tile) {
    case TILE_256x256: return launch16<T256x256, DT, A_RC, W_RC, EPI>(who, p, plan, st);
    case TILE_256x192: return launch16<T256x192, DT, A_RC, W_RC, EPI>(who, p, plan, st);
    case TILE_256x128: return launch16<T256x128, DT, A_RC, W_RC, EPI>(who, p, plan, st);
    case TILE_128x256: return launch16<T128x256, DT, A_RC, W_RC, EPI>(who, p, plan, st);
    case TILE_128x192: return launch16<T128x192, DT, A_RC, W_RC, EPI>(who, p, plan, st);
    case TILE_128x128: return launch16<T128x128, DT, A_RC, W_RC, EPI>(who, p, plan, st);
    case TILE_128x128D: return launch16<T128x128d, DT, A_RC, W_RC, EPI>(who, p, plan, st);
    case TILE_64x128: return launch16<T64x128, DT, A_RC, W_RC, EPI>(who, p, plan, st);
    default: return launch16<T64x64, DT, A_RC, W_RC, EPI>(who, p, plan, st);
  }
}

// Tile and k slices of a product with `rows` W rows (a gated product's value
// and gate rows both), M rows of A and nk stages.
Plan16 plan16(int64_t M, int64_t rows, int64_t nk, int problems);
// Float32 scratch of its slices.
inline size_t plan16_bytes(const Plan16& plan, int64_t M, int64_t rows, int problems) {
  return plan.splits > 1 ? sizeof(float) * (size_t)plan.splits * problems * (size_t)M * (size_t)rows : 0;
}

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// A matrix argument: `rows` x `width` values of unit stride along a row.
struct Mat16 {
  const void* p;
  int64_t ld, rows, width;
};
// Whether the product kernels can read it in place: 16-byte chunks of whole
// rows, at 32-bit offsets within a tile. Otherwise it is copied to scratch.
inline bool in_place(const Mat16& m) {
  return aligned16(m.p) && m.ld % 8 == 0 && m.width % 8 == 0 && m.ld < (1 << 22);
}

// Hands out a call's scratch in 256-byte steps; with no base, only measures it.
struct Scratch16 {
  uint8_t* base;
  size_t used = 0;
  void* take(size_t bytes) {
    uint8_t* p = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
  // the operand as the kernels read it: itself, or room for its padded copy
  Mat16 operand(const Mat16& m) {
    if (in_place(m)) return m;
    const int64_t w8 = round_up(m.width, 8);
    return {take(2 * (size_t)m.rows * (size_t)w8), w8, m.rows, w8};
  }
};
// Adds an operand's padded copy, if it has one, to those a call makes.
inline void add_pad(PadJobs& jobs, const Mat16& from, const Mat16& to) {
  if (to.p == from.p || from.rows == 0) return;
  jobs.job[jobs.count++] = {static_cast<const uint16_t*>(from.p), static_cast<uint16_t*>(const_cast<void*>(to.p)),
                            from.ld, from.rows, from.width};
}

// Whether a forward product (`rows` weight rows, of all its weights) runs on the
// kernel for few rows of x: at most 16, and, as one launch without partial sums
// is its gain, not where a workgroup's chain of k steps gets long or the weights'
// bytes swamp a launch. Over 1500 random products of 1 to 16 rows the rule is
// 1.3% off the better of the two (always this kernel 7.8%, never 8.6%): 1 x 1024
// -> 256 8.0 us (tiles 10.5), 1 x 4096 -> 4096 8.9 (11.5); 16 x 8192 -> 1024 17.0
// (11.9), 1 x 2048 -> 2 x 8192 15.1 (13.8).
inline bool skinny16(int64_t M, int64_t rows, int64_t K, bool gated) {
  return M <= 16 && rows * K <= 24 * 1000 * 1000 && (gated ? 2 : 1) * K <= (M <= 8 ? 10240 : 5120);
}
// It reads its operands in place at any alignment.
int run_skinny16(const char* who, const Gemm16& p, int dtype, hipStream_t st);

int refuse(int code, const char* who, const char* msg);
// What every product checks: sizes, type, activation.
int check_product(const char* who, int dtype, int act, int64_t M, int64_t N, int64_t K);
int check_scratch(const char* who, size_t need, const void* ws, size_t ws_bytes);

}  // namespace dc
