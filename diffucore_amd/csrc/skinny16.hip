// Forward products of few rows (single tokens, a sampler's conditioning): the
// weights' bytes are all that counts, each read once.
//
//   y = act(x w^T + b) + res,  h = (x wv^T + bv) act(x wg^T + bg),  M <= 16
//
// A workgroup holds 16 channels (gated: 16 value and 16 gate rows) and all of
// x's rows; its 8 waves split k between them and join in LDS, so one launch
// does it and no partial sums go to memory. Operands go straight from global
// memory to the registers of v_mfma_f32_16x16x32 (lane: row l % 16, 8 k from
// 8 (l / 16)), 16 bytes a lane at any alignment, several k steps in flight.
// Bound by the weights' bytes and, below about 20 MB, by the launch: 1 x 4096 ->
// 4096 bf16 8.9 us a call (11.5 on tiles, whose split k takes a second launch),
// 1 x 1280 -> 1280 7.8 (10.5), of which the call's host side is 7.7.
#include "linear16.h"

namespace dc {

constexpr int SKINNY_WAVES = 8, SKINNY_CH = 16;

template <int DT>
__device__ __forceinline__ v4f mfma16x16(uint4 w, uint4 x, v4f c) {
  if constexpr (DT == DC_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, x), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, x), c, 0, 0, 0);
}

template <int DT, bool GATED>
__global__ void __launch_bounds__(64 * SKINNY_WAVES) skinny16_kernel(Gemm16 p) {
  constexpr int NW = GATED ? 2 : 1, U = GATED ? 4 : 8;   // weight rows per channel; k steps in flight
  __shared__ v4f red[SKINNY_WAVES][NW][64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, r = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * SKINNY_CH;
  const uint16_t* wrow[NW];
  wrow[0] = p.w + (int64_t)min(n0 + r, p.N - 1) * p.ldw;
  if constexpr (GATED) wrow[NW - 1] = p.w2 + (int64_t)min(n0 + r, p.N - 1) * p.ldw2;
  const uint16_t* xrow = p.a + (int64_t)min(r, p.M - 1) * p.lda;
  v4f acc[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};

  const int steps = (p.K + 31) / 32, per = (steps + SKINNY_WAVES - 1) / SKINNY_WAVES;
  const int whole = p.K / 32;   // steps that lie in the row
  int s = wave * per;
  const int end = min(s + per, steps);
  for (; s + U <= min(end, whole); s += U) {
    uint4 w[U][NW], x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = 32 * (s + u) + 8 * kq;
#pragma unroll
      for (int i = 0; i < NW; ++i) w[u][i] = load_chunk16(wrow[i] + k, 8);
      x[u] = load_chunk16(xrow + k, 8);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NW; ++i) acc[i] = mfma16x16<DT>(w[u][i], x[u], acc[i]);
  }
  for (; s < end; ++s) {
    const int k = 32 * s + 8 * kq, left = p.K - k;   // past the row's end both are 0
    uint4 w[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) w[i] = load_chunk16(wrow[i] + k, left);
    const uint4 x = load_chunk16(xrow + k, left);
#pragma unroll
    for (int i = 0; i < NW; ++i) acc[i] = mfma16x16<DT>(w[i], x, acc[i]);
  }
#pragma unroll
  for (int i = 0; i < NW; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave) return;
  // the first wave finishes: this lane's row and 4 channels
  const int m = r, n = n0 + 4 * kq;
  v4f v = red[0][0][lane], g = red[0][NW - 1][lane];
#pragma unroll
  for (int q = 1; q < SKINNY_WAVES; ++q) {
    v += red[q][0][lane];
    if constexpr (GATED) g += red[q][NW - 1][lane];
  }
  if (m >= p.M) return;
  with_act(p.act, [&](auto act_) __attribute__((always_inline)) {
    constexpr int ACT = decltype(act_)::value;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e >= p.N) break;
      const int64_t at = (int64_t)m * p.N + n + e;
      float y = v[e] + bias_at(p.bias, p.bias_dtype, n + e);
      if (p.z) store_saved1(p.z, p.M, p.N, at, y);
      if constexpr (GATED) {
        const float gate = g[e] + bias_at(p.bias2, p.bias_dtype, n + e);
        if (p.z) store_saved1(p.z2, p.M, p.N, at, gate);
        y *= act_value<ACT>(gate);
      } else {
        y = act_value<ACT>(y);
        if (p.res) y += h16_to_f32<DT>(p.res[m * p.ldr + n + e]);
      }
      p.out[m * p.ldo + n + e] = (uint16_t)f32_to_h16<DT>(y);
    }
  });
}

template <int DT, bool GATED>
static void launch_skinny(const Gemm16& p, hipStream_t st) {
  hipLaunchKernelGGL((skinny16_kernel<DT, GATED>), dim3((unsigned)((p.N + SKINNY_CH - 1) / SKINNY_CH)),
                     dim3(64 * SKINNY_WAVES), 0, st, p);
}

int run_skinny16(const char* who, const Gemm16& p, int dtype, hipStream_t st) {
  const bool gated = p.w2;
  if (dtype == DC_BF16) gated ? launch_skinny<DC_BF16, true>(p, st) : launch_skinny<DC_BF16, false>(p, st);
  else gated ? launch_skinny<DC_F16, true>(p, st) : launch_skinny<DC_F16, false>(p, st);
  return launch_status(who);
}

}  // namespace dc
