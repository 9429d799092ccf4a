// Layer norm over the last dim and its backward pass on gfx950.
//
//   y = xh w + b,  xh = (x - mean) r,  r = 1 / sqrt(mean((x - mean)^2) + eps)
//   dxh = dy w,  dx = r (dxh - mean(dxh) - xh mean(dxh xh))
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Memory-bound (8 to 20 operations an element): each pass reads its rows once
// and keeps them in registers. A row belongs to G lanes, C chunks of 16 bytes
// each (chunk c * G + lane); G and C are the smallest that cover the row, so
// narrow rows share a wave (G = 8 .. 32) and wide ones take a workgroup
// (G = 256). Statistics are two passes over the registers, in float32: the
// squared deviations never cancel. The backward pass walks rows with a fixed
// set of workgroups, every lane summing dw and db of its own columns in
// registers; the workgroups' partial rows are joined in order by a second
// launch. Rows past 1536 chunks (12288 16-bit, 6144 float32 values) are re-read
// from the caches instead (wide kernels).
#include "colsum.h"

namespace dc {

constexpr int NORM_MAX_C = 6;

struct NormArgs {
  const void* x;
  const void* dy;
  const void* w;
  const void* b;
  void* out;        // y or dx
  float* stats;     // forward: written, backward: read; [2][M]
  float* part;      // backward: [P][2][D] or NULL
  int64_t ldx, lddy, ldo;
  int64_t M;
  int D;
  int w_dtype;      // DC_NONE: no w, no b
  float eps;
};

template <int DT>
struct Elem {
  static constexpr int VEC = DT == DC_F32 ? 4 : 8;
  typedef typename std::conditional<DT == DC_F32, float, uint16_t>::type T;
};

template <int DT>
__device__ __forceinline__ float elem_f32(typename Elem<DT>::T v) {
  if constexpr (DT == DC_F32) return v;
  else return h16_to_f32<DT>(v);
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T f32_elem(float v) {
  if constexpr (DT == DC_F32) return v;
  else return (uint16_t)f32_to_h16<DT>(v);
}

// One 16-byte chunk of a row, `n` values left in the row (0 past its end).
template <int DT>
__device__ __forceinline__ void load_chunk(const void* base, int64_t at, int n, float (&f)[Elem<DT>::VEC]) {
  constexpr int V = Elem<DT>::VEC;
  const auto* p = static_cast<const typename Elem<DT>::T*>(base) + at;
  if (n >= V) {
    if constexpr (DT == DC_F32) {
      const U32x4 u = *reinterpret_cast<const U32x4*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(u.v[e]);
    } else {
      unpack8<DT>(load16_any(p), f);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = e < n ? elem_f32<DT>(p[e]) : 0.0f;
  }
}
template <int DT>
__device__ __forceinline__ void store_chunk(void* base, int64_t at, int n, const float (&f)[Elem<DT>::VEC]) {
  constexpr int V = Elem<DT>::VEC;
  auto* p = static_cast<typename Elem<DT>::T*>(base) + at;
  if (n >= V) {
    if constexpr (DT == DC_F32) {
      U32x4 u;
#pragma unroll
      for (int e = 0; e < 4; ++e) u.v[e] = __float_as_uint(f[e]);
      *reinterpret_cast<U32x4*>(p) = u;
    } else {
      store16_any(p, pack8<DT>(f));
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) p[e] = f32_elem<DT>(f[e]);
  }
}

// V partial sums into a float row, `n` values left in it.
template <int V>
__device__ __forceinline__ void store_chunk_f32(float* row, int col, int n, const float (&f)[V]) {
  if (n >= V) {
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      U32x4 u;
#pragma unroll
      for (int e = 0; e < 4; ++e) u.v[e] = __float_as_uint(f[q + e]);
      *reinterpret_cast<U32x4*>(row + col + q) = u;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) row[col + e] = f[e];
  }
}

// V weights (or biases) of any type from column `col`, `n` left in the row.
template <int V>
__device__ __forceinline__ void load_params(const void* w, int dtype, int col, int n, float (&f)[V]) {
  if (dtype == DC_F32) {
    const float* p = static_cast<const float*>(w) + col;
    if (n >= V) {
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        const U32x4 u = *reinterpret_cast<const U32x4*>(p + q);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[q + e] = __uint_as_float(u.v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = e < n ? p[e] : 0.0f;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(w) + col;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint32_t u = e < n ? p[e] : 0u;
      f[e] = dtype == DC_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
    }
  }
}

// Sum over the G lanes of a row (all lanes get it): butterfly in the wave, then
// the waves through LDS.
template <int G>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (G > 64) {
    __syncthreads();   // the last use of red is over
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < G / 64; ++i) v += red[i];
  }
  return v;
}

template <int DT, int G, int C>
__global__ void __launch_bounds__(256) norm_fwd_kernel(NormArgs p) {
  constexpr int V = Elem<DT>::VEC, RPB = 256 / G;
  __shared__ float red[4];
  const int l = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / G;
  const bool live = row < p.M;
  float v[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * G + l) * V;
    load_chunk<DT>(p.x, row * p.ldx + col, live ? p.D - col : 0, v[c]);
  }
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) s += v[c][e];
  const float inv = 1.0f / (float)p.D;
  const float mean = row_sum<G>(s, red) * inv;
  float q = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = (c * G + l) * V + e < p.D ? v[c][e] - mean : 0.0f;
      q = __builtin_fmaf(d, d, q);
    }
  const float rstd = 1.0f / __builtin_sqrtf(row_sum<G>(q, red) * inv + p.eps);
  if (!live) return;
  if (p.stats && l == 0) p.stats[row] = mean, p.stats[p.M + row] = rstd;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * G + l) * V, n = p.D - col;
    if (n <= 0) continue;
    float w[V], b[V];
    if (p.w) load_params<V>(p.w, p.w_dtype, col, n, w);
    if (p.b) load_params<V>(p.b, p.w_dtype, col, n, b);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float y = (v[c][e] - mean) * rstd;
      if (p.w) y *= w[e];
      if (p.b) y += b[e];
      v[c][e] = y;
    }
    store_chunk<DT>(p.out, row * p.ldo + col, n, v[c]);
  }
}

template <int DT, int G, int C>
__global__ void __launch_bounds__(256) norm_bwd_kernel(NormArgs p) {
  constexpr int V = Elem<DT>::VEC, RPB = 256 / G;
  __shared__ float red[4];
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int l = threadIdx.x % G;
  float w[C][V], dw[C][V], db[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * G + l) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) w[c][e] = 1.0f, dw[c][e] = db[c][e] = 0.0f;
    if (p.w && col < p.D) load_params<V>(p.w, p.w_dtype, col, p.D - col, w[c]);
  }
  const float inv = 1.0f / (float)p.D;
  // every lane of a workgroup makes the same number of trips (row_sum has barriers)
  const int64_t step = (int64_t)gridDim.x * RPB, trips = (p.M + step - 1) / step;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / G;
  for (int64_t i = 0; i < trips; ++i, row += step) {
    const bool live = row < p.M;
    float mean = 0.0f, rstd = 0.0f;
    if (live) mean = p.stats[row], rstd = p.stats[p.M + row];
    float x[C][V], g[C][V];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * G + l) * V, n = live ? p.D - col : 0;
      load_chunk<DT>(p.x, row * p.ldx + col, n, x[c]);
      load_chunk<DT>(p.dy, row * p.lddy + col, n, g[c]);
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // past the row's end the gradient loaded is 0, and so is its share of every sum
        const float xh = (x[c][e] - mean) * rstd;
        dw[c][e] = __builtin_fmaf(g[c][e], xh, dw[c][e]);
        db[c][e] += g[c][e];
        g[c][e] *= w[c][e];
        x[c][e] = xh;
        s1 += g[c][e];
        s2 = __builtin_fmaf(g[c][e], xh, s2);
      }
    if (!p.out) continue;
    s1 = row_sum<G>(s1, red) * inv;
    s2 = row_sum<G>(s2, red) * inv;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * G + l) * V, n = live ? p.D - col : 0;
      if (n <= 0) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) g[c][e] = rstd * (g[c][e] - s1 - x[c][e] * s2);
      store_chunk<DT>(p.out, row * p.ldo + col, n, g[c]);
    }
  }
  if (!p.part) return;
  float* out = p.part + (int64_t)blockIdx.x * 2 * p.D;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * G + l) * V;
      store_chunk_f32<V>(out, col, p.D - col, dw[c]);
      store_chunk_f32<V>(out + p.D, col, p.D - col, db[c]);
    }
  } else {
    // the row groups of a wave by butterfly, then the waves one after the other through LDS
#pragma unroll
    for (int o = G; o < 64; o <<= 1)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) dw[c][e] += __shfl_xor(dw[c][e], o), db[c][e] += __shfl_xor(db[c][e], o);
    float* acc = reinterpret_cast<float*>(smem);   // [2][C * G * V]
    constexpr int W = C * G * V;
    for (int wv = 0; wv < 4; ++wv) {
      if ((int)threadIdx.x >> 6 == wv && (threadIdx.x & 63) < G) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int at = (c * G + l) * V + e;
            acc[at] = wv ? acc[at] + dw[c][e] : dw[c][e];
            acc[W + at] = wv ? acc[W + at] + db[c][e] : db[c][e];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < p.D; i += 256) out[i] = acc[i], out[p.D + i] = acc[W + i];
  }
}

// ---------------------------------------------------------------- wide rows

// A workgroup a row, the row read again for each of its passes.
template <int DT>
__global__ void __launch_bounds__(256) norm_fwd_wide_kernel(NormArgs p) {
  constexpr int V = Elem<DT>::VEC;
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const float inv = 1.0f / (float)p.D;
  float s = 0.0f, q = 0.0f, v[V];
  for (int col = threadIdx.x * V; col < p.D; col += 256 * V) {
    load_chunk<DT>(p.x, row * p.ldx + col, p.D - col, v);
#pragma unroll
    for (int e = 0; e < V; ++e) s += v[e];
  }
  const float mean = row_sum<256>(s, red) * inv;
  for (int col = threadIdx.x * V; col < p.D; col += 256 * V) {
    load_chunk<DT>(p.x, row * p.ldx + col, p.D - col, v);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = col + e < p.D ? v[e] - mean : 0.0f;
      q = __builtin_fmaf(d, d, q);
    }
  }
  const float rstd = 1.0f / __builtin_sqrtf(row_sum<256>(q, red) * inv + p.eps);
  if (p.stats && threadIdx.x == 0) p.stats[row] = mean, p.stats[p.M + row] = rstd;
  for (int col = threadIdx.x * V; col < p.D; col += 256 * V) {
    const int n = p.D - col;
    float w[V], b[V];
    load_chunk<DT>(p.x, row * p.ldx + col, n, v);
    if (p.w) load_params<V>(p.w, p.w_dtype, col, n, w);
    if (p.b) load_params<V>(p.b, p.w_dtype, col, n, b);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float y = (v[e] - mean) * rstd;
      if (p.w) y *= w[e];
      if (p.b) y += b[e];
      v[e] = y;
    }
    store_chunk<DT>(p.out, row * p.ldo + col, n, v);
  }
}

template <int DT>
__global__ void __launch_bounds__(256) norm_dx_wide_kernel(NormArgs p) {
  constexpr int V = Elem<DT>::VEC;
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const float inv = 1.0f / (float)p.D, mean = p.stats[row], rstd = p.stats[p.M + row];
  float s1 = 0.0f, s2 = 0.0f, x[V], g[V], w[V];
  auto load = [&](int col) __attribute__((always_inline)) {
    const int n = p.D - col;
    load_chunk<DT>(p.x, row * p.ldx + col, n, x);
    load_chunk<DT>(p.dy, row * p.lddy + col, n, g);
    if (p.w) load_params<V>(p.w, p.w_dtype, col, n, w);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      x[e] = (x[e] - mean) * rstd;
      if (p.w) g[e] *= w[e];
    }
  };
  for (int col = threadIdx.x * V; col < p.D; col += 256 * V) {
    load(col);
#pragma unroll
    for (int e = 0; e < V; ++e) s1 += g[e], s2 = __builtin_fmaf(g[e], x[e], s2);
  }
  s1 = row_sum<256>(s1, red) * inv;
  s2 = row_sum<256>(s2, red) * inv;
  for (int col = threadIdx.x * V; col < p.D; col += 256 * V) {
    load(col);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = rstd * (g[e] - s1 - x[e] * s2);
    store_chunk<DT>(p.out, row * p.ldo + col, p.D - col, g);
  }
}

// dw and db of 256 chunks of columns over a block of rows.
template <int DT>
__global__ void __launch_bounds__(256) norm_dw_wide_kernel(NormArgs p, int64_t rows) {
  constexpr int V = Elem<DT>::VEC;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (at >= p.D) return;
  const int col = (int)at, n = p.D - col;
  const int64_t r0 = blockIdx.y * rows, r1 = min(r0 + rows, p.M);
  float dw[V] = {0}, db[V] = {0};
  for (int64_t row = r0; row < r1; ++row) {
    float x[V], g[V];
    load_chunk<DT>(p.x, row * p.ldx + col, n, x);
    load_chunk<DT>(p.dy, row * p.lddy + col, n, g);
    const float mean = p.stats[row], rstd = p.stats[p.M + row];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      dw[e] = __builtin_fmaf(g[e], (x[e] - mean) * rstd, dw[e]);
      db[e] += g[e];
    }
  }
  float* out = p.part + (int64_t)blockIdx.y * 2 * p.D;
  store_chunk_f32<V>(out, col, n, dw);
  store_chunk_f32<V>(out + p.D, col, n, db);
}

// ---------------------------------------------------------------- dispatch

// The smallest row group that covers `chunks` with at most 6 chunks a lane: one
// row's reductions then cross as few lanes as they can, and no lane of the
// group idles over more than one chunk. G = 0: wide.
struct NormPlan {
  int G, C;
};
static NormPlan norm_plan(int64_t D, int dtype) {
  const int64_t vec = dtype == DC_F32 ? 4 : 8, chunks = (D + vec - 1) / vec;
  const int groups[] = {8, 16, 32, 64, 256};
  for (int g : groups)
    if (chunks <= (int64_t)g * NORM_MAX_C) return {g, (int)((chunks + g - 1) / g)};
  return {0, 0};
}

// Workgroups of the backward pass, each with one partial row of dw and db: as
// many as are resident at once, fewer when there are few rows.
static int64_t norm_blocks(int64_t M, const NormPlan& r) {
  const int64_t most = 2LL * device_cus();
  const int64_t rpb = r.G ? 256 / r.G : 1, all = (M + rpb - 1) / rpb;
  return all < most ? all : most;
}

template <int DT, int G>
static int launch_norm(const NormArgs& p, int C, bool bwd, hipStream_t st) {
  constexpr int RPB = 256 / G;
  constexpr int V = Elem<DT>::VEC;
  auto go = [&](auto c_) {
    constexpr int c = decltype(c_)::value;
    if (!bwd) {
      hipLaunchKernelGGL((norm_fwd_kernel<DT, G, c>), dim3((unsigned)((p.M + RPB - 1) / RPB)), dim3(256), 0, st, p);
    } else {
      const unsigned lds = RPB > 1 && p.part ? 2 * c * G * V * 4 : 0;
      hipLaunchKernelGGL((norm_bwd_kernel<DT, G, c>), dim3((unsigned)norm_blocks(p.M, {G, c})), dim3(256), lds, st, p);
    }
  };
  switch (C) {
    case 1: go(std::integral_constant<int, 1>{}); break;
    case 2: go(std::integral_constant<int, 2>{}); break;
    case 3: go(std::integral_constant<int, 3>{}); break;
    case 4: go(std::integral_constant<int, 4>{}); break;
    case 5: go(std::integral_constant<int, 5>{}); break;
    default: go(std::integral_constant<int, 6>{}); break;
  }
  return launch_status(bwd ? "dc_layer_norm_bwd" : "dc_layer_norm");
}

template <int DT>
static int run_norm(const NormArgs& p, bool bwd, hipStream_t st) {
  const NormPlan r = norm_plan(p.D, DT);
  switch (r.G) {
    case 8: return launch_norm<DT, 8>(p, r.C, bwd, st);
    case 16: return launch_norm<DT, 16>(p, r.C, bwd, st);
    case 32: return launch_norm<DT, 32>(p, r.C, bwd, st);
    case 64: return launch_norm<DT, 64>(p, r.C, bwd, st);
    case 256: return launch_norm<DT, 256>(p, r.C, bwd, st);
    default: break;
  }
  if (!bwd) {
    hipLaunchKernelGGL((norm_fwd_wide_kernel<DT>), dim3((unsigned)p.M), dim3(256), 0, st, p);
    return launch_status("dc_layer_norm");
  }
  if (p.out) {
    hipLaunchKernelGGL((norm_dx_wide_kernel<DT>), dim3((unsigned)p.M), dim3(256), 0, st, p);
    if (int e = launch_status("dc_layer_norm_bwd")) return e;
  }
  if (p.part) {
    const int64_t P = norm_blocks(p.M, r), rows = (p.M + P - 1) / P;
    const int64_t span = 256 * Elem<DT>::VEC;
    hipLaunchKernelGGL((norm_dw_wide_kernel<DT>), dim3((unsigned)((p.D + span - 1) / span), (unsigned)P), dim3(256),
                       0, st, p, rows);
    return launch_status("dc_layer_norm_bwd");
  }
  return DC_OK;
}

static int check_norm(const char* who, int x_dtype, const void* w, const void* b, int w_dtype, int64_t M, int64_t D) {
  const char* msg = nullptr;
  if (M < 0 || D <= 0 || M > 0x7fffffff || D > (1 << 24)) msg = "M must be 0 .. 2^31 - 1 and D 1 .. 2^24";
  else if (!float_dtype(x_dtype)) msg = "x_dtype must be DC_F16, DC_BF16 or DC_F32";
  else if ((w || b) && !float_dtype(w_dtype)) msg = "w_dtype must be DC_F16, DC_BF16 or DC_F32";
  if (!msg) return DC_OK;
  set_error("%s: %s", who, msg);
  return DC_EINVAL;
}

static int dispatch_norm(const NormArgs& p, int dtype, bool bwd, hipStream_t st) {
  switch (dtype) {
    case DC_F16: return run_norm<DC_F16>(p, bwd, st);
    case DC_BF16: return run_norm<DC_BF16>(p, bwd, st);
    default: return run_norm<DC_F32>(p, bwd, st);
  }
}

}  // namespace dc

using namespace dc;

extern "C" int dc_layer_norm(const void* x, int64_t ldx, int x_dtype, const void* w, const void* b, int w_dtype,
                             float eps, void* y, int64_t ldy, float* stats, int64_t M, int64_t D, void* stream) {
  clear_error();
  if (int e = check_norm("dc_layer_norm", x_dtype, w, b, w_dtype, M, D)) return e;
  if (M == 0) return DC_OK;
  if (!x || !y) return fail(DC_EINVAL, "dc_layer_norm: null pointer");
  if (ldx < D || ldy < D) return fail(DC_EINVAL, "dc_layer_norm: row stride < D");
  NormArgs p{};
  p.x = x, p.w = w, p.b = b, p.out = y, p.stats = stats, p.ldx = ldx, p.ldo = ldy, p.M = M, p.D = (int)D;
  p.w_dtype = w_dtype, p.eps = eps;
  return dispatch_norm(p, x_dtype, false, (hipStream_t)stream);
}

extern "C" size_t dc_layer_norm_bwd_workspace_bytes(int64_t M, int64_t D, int x_dtype) {
  if (M <= 0 || D <= 0 || M > 0x7fffffff || D > (1 << 24) || !float_dtype(x_dtype)) return 0;
  return sizeof(float) * 2 * (size_t)D * (size_t)norm_blocks(M, norm_plan(D, x_dtype));
}

extern "C" int dc_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, int x_dtype, const void* w,
                                 int w_dtype, const float* stats, void* dx, int64_t lddx, void* dw, void* db,
                                 int64_t M, int64_t D, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  const char* who = "dc_layer_norm_bwd";
  if (int e = check_norm(who, x_dtype, w ? w : dw, db, w_dtype, M, D)) return e;
  hipStream_t st = (hipStream_t)stream;
  const bool sums = dw || db;
  if (M == 0) return sums ? reduce_partials(nullptr, 0, 2, D, dw, db, w_dtype, st, who) : DC_OK;
  if (!dx && !sums) return DC_OK;
  if (!dy || !x || !stats) return fail(DC_EINVAL, "dc_layer_norm_bwd: null pointer");
  if (lddy < D || ldx < D || (dx && lddx < D)) return fail(DC_EINVAL, "dc_layer_norm_bwd: row stride < D");
  const size_t need = dc_layer_norm_bwd_workspace_bytes(M, D, x_dtype);
  if (sums && (!ws || ws_bytes < need || !aligned16(ws))) {
    set_error("%s: workspace too small or not 16-byte aligned (needs %zu bytes)", who, need);
    return DC_EWORKSPACE;
  }
  NormArgs p{};
  p.x = x, p.dy = dy, p.w = w, p.out = dx, p.stats = const_cast<float*>(stats);
  p.part = sums ? static_cast<float*>(ws) : nullptr;
  p.ldx = ldx, p.lddy = lddy, p.ldo = lddx, p.M = M, p.D = (int)D, p.w_dtype = w_dtype;
  if (int e = dispatch_norm(p, x_dtype, true, st)) return e;
  return sums ? reduce_partials(p.part, (int)norm_blocks(M, norm_plan(D, x_dtype)), 2, D, dw, db, w_dtype, st, who)
              : DC_OK;
}
