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
// pre-activations (zg: gated; neither: none), rows of lddz = dz_width(N) with
// zeros past N, and the sums of dz over rows before rounding (NULL: not
// asked for). `part`: act16_bwd_part_bytes of scratch for the sums.
// A dz row: whole stages of 64, with 8 zeros past N rounded up to 8 unless N is
// a multiple of 64.
inline int64_t dz_width(int64_t N) { return (N + 63) / 64 * 64 + (N % 64 > 56 ? 64 : 0); }

struct ActBwd {
  const void* dy;
  int64_t lddy;
  const uint8_t *zv, *zg;   // saved (saved16_bytes each)
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

// Up to three copies dst [rows, width rounded up to 8] (16-byte aligned) = src
// [rows, width] (any alignment) and zeros, in one launch.
struct PadJob {
  const uint16_t* src;
  uint16_t* dst;
  int64_t ld, rows, width;
};
struct PadJobs {
  PadJob job[3];
  uint32_t first[3];
  int count = 0;
  int run(const char* who, hipStream_t st);
};

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

// Pre-activations kept for the backward pass: the upper 24 bits (16 significant)
// of a float32, as a plane of 16-bit halves [M, N] and then a plane of bytes
// [M, N]. Cutting loses less than 2^-15 of a value, always towards 0: the value is
// first made larger by 2^-16 of itself, which leaves it off by at most 2^-16 to
// either side, in one multiplication that keeps inf and NaN what they are (rounding
// by an integer add would turn some NaN into 0). float32 would cost a third more
// traffic (linear 4608 x 2048 -> 8192 with gradients 555 us, 509 so), bf16 or fp16 a
// rounding as large as the result's own.
constexpr float SAVED_CENTRE = 1.0f + 1.0f / 65536;
inline size_t saved16_bytes(int64_t M, int64_t N) { return 3 * (size_t)M * (size_t)N; }

__device__ __forceinline__ void store_saved8(uint8_t* z, int64_t M, int64_t N, int64_t m, int64_t n,
                                             const float (&z8)[8]) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = z8[e] * SAVED_CENTRE;
  uint32_t h[4], l[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = __float_as_uint(f[2 * i]), b = __float_as_uint(f[2 * i + 1]);
    h[i] = __builtin_amdgcn_perm(b, a, 0x07060302);   // the upper halves of a and b
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i]), 0x0c0c0501);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(f[4 * i + 3]), __float_as_uint(f[4 * i + 2]), 0x0c0c0501);
    l[i] = ab | cd << 16;                             // byte 1 of each
  }
  store_chunk16(reinterpret_cast<uint16_t*>(z) + m * N + n, N - n, make_uint4(h[0], h[1], h[2], h[3]));
  store_chunk8(z + 2 * M * N + m * N + n, N - n, make_uint2(l[0], l[1]));
}
__device__ __forceinline__ void store_saved1(uint8_t* z, int64_t M, int64_t N, int64_t at, float v) {
  const float f = v * SAVED_CENTRE;
  reinterpret_cast<uint16_t*>(z)[at] = (uint16_t)(__float_as_uint(f) >> 16);
  z[2 * M * N + at] = (uint8_t)(__float_as_uint(f) >> 8);
}
__device__ __forceinline__ void load_saved8(const uint8_t* z, int64_t M, int64_t N, int64_t m, int64_t n,
                                            float (&f)[8]) {
  const uint4 u = load_chunk16(reinterpret_cast<const uint16_t*>(z) + m * N + n, N - n);
  const uint2 v = load_chunk8(z + 2 * M * N + m * N + n, N - n);
  const uint32_t h[4] = {u.x, u.y, u.z, u.w}, l[2] = {v.x, v.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = l[i / 2] >> (16 * (i % 2));
    f[2 * i] = __uint_as_float(h[i] << 16 | (b & 0xffu) << 8);
    f[2 * i + 1] = __uint_as_float((h[i] & 0xffff0000u) | (b & 0xff00u));
  }
}

}  // namespace dc
