// Column sums over rows: per-workgroup partial sums in scratch, then one pass
// that adds them in a fixed order (no atomics: the same bits on every run).
#pragma once

#include "act.h"

namespace dc {

// out_s[w] = sum over p of part[(p * sections + s) * width + w], stored as
// `out_dtype` (DC_F16 / DC_BF16 / DC_F32); NULL outputs are skipped.
int reduce_partials(const float* part, int P, int sections, int64_t width, void* out0, void* out1, int out_dtype,
                    hipStream_t st, const char* what);

inline bool float_dtype(int dt) { return dt == DC_F16 || dt == DC_BF16 || dt == DC_F32; }

// 8 consecutive 16-bit values as floats.
template <int DT>
__device__ __forceinline__ void unpack8(uint4 u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = h16_to_f32<DT>(w[i] & 0xffffu);
    f[2 * i + 1] = h16_to_f32<DT>(w[i] >> 16);
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const v2f x = {f[2 * i], f[2 * i + 1]};
    if constexpr (DT == DC_BF16) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, v2bf));
    else w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, v2h));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Up to 8 16-bit values from p (n of them, the rest 0), at any element alignment.
template <int DT>
__device__ __forceinline__ void load8_n(const uint16_t* p, int64_t n, float (&f)[8]) {
  if (n >= 8) {
    unpack8<DT>(load16_any(p), f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < n ? h16_to_f32<DT>(p[e]) : 0.0f;
  }
}

// Up to 8 floats from p (n of them, the rest 0), at any element alignment.
__device__ __forceinline__ void load8_n(const float* p, int64_t n, float (&f)[8]) {
  if (n >= 8) {
#pragma unroll
    for (int q = 0; q < 8; q += 4) {
      const U32x4 u = *reinterpret_cast<const U32x4*>(p + q);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[q + e] = __uint_as_float(u.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < n ? p[e] : 0.0f;
  }
}

}  // namespace dc
