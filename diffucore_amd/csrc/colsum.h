// Column sums over rows: per-workgroup partial sums in scratch, then one pass
// that adds them in a fixed order (no atomics: the same bits on every run).
#pragma once

#include "act.h"

namespace dc {

// out_s[w] = sum over p of part[(p * sections + s) * width + w], stored as
// `out_dtype` (DC_F16 / DC_BF16 / DC_F32); NULL outputs are skipped.
int reduce_partials(const float* part, int P, int sections, int64_t width, void* out0, void* out1, int out_dtype,
                    hipStream_t st, const char* what);

// The elementwise half of a feed-forward backward pass: dz of dy and the
// pre-activations (zg: gated; neither: none), rows of lddz = N rounded up to 64
// with zeros past N, and the sums of dz over rows before rounding (NULL: not
// asked for). `part`: act16_bwd_part_bytes of scratch for the sums.
struct ActBwd {
  const void* dy;
  int64_t lddy;
  const float *zv, *zg;
  int64_t ldz;
  int act;
  void *dzv, *dzg;
  int64_t lddz;
  void *dbv, *dbg;
  int db_dtype, dtype;
  int64_t M, N;
  float* part;
};
int act16_bwd(const char* who, const ActBwd& a, hipStream_t st);
size_t act16_bwd_part_bytes(int64_t M, int64_t N, bool gated);

// dst [M, W rounded up to 8] (16-byte aligned) = src [M, W] and zeros.
int pad_rows16(const char* who, const void* src, int64_t lds, void* dst, int64_t M, int64_t W, hipStream_t st);

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

// 8 values from p, of which n are left in the row (the rest 0), at any element alignment.
template <int DT>
__device__ __forceinline__ void load8_n(const uint16_t* p, int64_t n, float (&f)[8]) {
  unpack8<DT>(load_chunk16(p, n), f);
}
__device__ __forceinline__ void load8_n(const float* p, int64_t n, float (&f)[8]) {
  const float4 a = load_chunk32(p, n), b = load_chunk32(p + 4, n - 4);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
__device__ __forceinline__ void store8_n(float* p, int64_t n, const float (&f)[8]) {
  store_chunk32(p, n, make_float4(f[0], f[1], f[2], f[3]));
  store_chunk32(p + 4, n - 4, make_float4(f[4], f[5], f[6], f[7]));
}

}  // namespace dc
