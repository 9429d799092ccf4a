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
// launch. Rows past 1536 chunks (12288 16-bit, 6144 float32 values), and those
// short of one, are re-read from the caches instead (wide kernels).
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
  static constexpr int VEC = DT == DC_F32 ? 4 : 8;   // values of a 16-byte chunk
};

// One 16-byte chunk of a row as loaded, `n` values left in the row (0 past its end).
template <int DT>
__device__ __forceinline__ uint4 load_raw(const void* base, int64_t at, int n) {
  if constexpr (DT == DC_F32) {
    const float4 f = load_chunk32(static_cast<const float*>(base) + at, n);
    return make_uint4(__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w));
  } else {
    return load_chunk16(static_cast<const uint16_t*>(base) + at, n);
  }
}
template <int DT>
__device__ __forceinline__ void unpack_raw(uint4 u, float (&f)[Elem<DT>::VEC]) {
  if constexpr (DT == DC_F32) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  } else {
    unpack8<DT>(u, f);
  }
}
template <int DT>
__device__ __forceinline__ void load_chunk(const void* base, int64_t at, int n, float (&f)[Elem<DT>::VEC]) {
  unpack_raw<DT>(load_raw<DT>(base, at, n), f);
}
template <int DT>
__device__ __forceinline__ void store_chunk(void* base, int64_t at, int n, const float (&f)[Elem<DT>::VEC]) {
  if constexpr (DT == DC_F32) store_chunk32(static_cast<float*>(base) + at, n, make_float4(f[0], f[1], f[2], f[3]));
  else store_chunk16(static_cast<uint16_t*>(base) + at, n, pack8<DT>(f));
}

// V partial sums into a float row, `n` values left in it.
template <int V>
__device__ __forceinline__ void store_chunk_f32(float* row, int col, int n, const float (&f)[V]) {
#pragma unroll
  for (int q = 0; q < V; q += 4)
    store_chunk32(row + col + q, n - q, make_float4(f[q], f[q + 1], f[q + 2], f[q + 3]));
}

// V weights (or biases) of any type from column `col`, `n` left in the row.
template <int V>
__device__ __forceinline__ void load_params(const void* w, int dtype, int col, int n, float (&f)[V]) {
  if (dtype == DC_F32) {
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      const float4 u = load_chunk32(static_cast<const float*>(w) + col + q, n - q);
      f[q] = u.x, f[q + 1] = u.y, f[q + 2] = u.z, f[q + 3] = u.w;
    }
    return;
  }
  const uint16_t* p = static_cast<const uint16_t*>(w) + col;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const uint32_t u = e < n ? p[e] : 0u;
    f[e] = dtype == DC_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
  }
}

__device__ __forceinline__ float param_at(const void* w, int dtype, int i) {
  if (dtype == DC_F32) return static_cast<const float*>(w)[i];
  const uint32_t u = static_cast<const uint16_t*>(w)[i];
  return dtype == DC_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
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

// A row's chunks without branches, so that all its loads are in flight at once.
// Chunks c < C - 1 lie in the row. The last one may lie past it (zeros then) or,
// with TAIL (D not a whole number of chunks), hold its end: it is read from the
// row's last 16 bytes and shifted into place.
template <int DT, int G, int C, bool TAIL>
__device__ __forceinline__ void load_row(const void* base, int64_t at, int l, int D, uint4 (&r)[C]) {
  constexpr int V = Elem<DT>::VEC, ES = DT == DC_F32 ? 4 : 2;
  const uint8_t* row = static_cast<const uint8_t*>(base) + at * ES;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * G + l) * V;
    const int from = c < C - 1 ? col : TAIL ? min(col, D - V) : col < D ? col : 0;
    const auto u = load_words<uint16_t, 4>(reinterpret_cast<const uint16_t*>(row + (int64_t)from * ES));
    r[c] = make_uint4(u.v[0], u.v[1], u.v[2], u.v[3]);
  }
}
// The last chunk put in order; apart from the loads, so that it waits for none of the next ones.
template <int DT, int G, int C, bool TAIL>
__device__ __forceinline__ void end_row(uint4& z, int l, int D) {
  constexpr int V = Elem<DT>::VEC, ES = DT == DC_F32 ? 4 : 2;
  const int col = ((C - 1) * G + l) * V;
  if constexpr (TAIL) {
    const int shift = max(col - (D - V), 0) * ES;   // bytes to drop in front: a multiple of the element's
    const bool w1 = shift & 4, w2 = shift & 8;
    if (w1) z = make_uint4(z.y, z.z, z.w, 0u);
    if (w2) z = make_uint4(z.z, z.w, 0u, 0u);
    if constexpr (DT != DC_F32) {
      if (shift & 2)
        z = make_uint4(z.x >> 16 | z.y << 16, z.y >> 16 | z.z << 16, z.z >> 16 | z.w << 16, z.w >> 16);
    }
  }
  if (col >= D) z = make_uint4(0u, 0u, 0u, 0u);
}
template <int DT, int G, int C, bool TAIL>
__device__ __forceinline__ void store_part(void* base, int64_t at, int c, int l, int D,
                                           const float (&f)[Elem<DT>::VEC]) {
  constexpr int V = Elem<DT>::VEC;
  const int col = (c * G + l) * V;
  if (c < C - 1 || (!TAIL && col < D)) store_chunk<DT>(base, at + col, V, f);
  else if (TAIL) store_chunk<DT>(base, at + col, D - col, f);
}

// Weights (and biases) as float32 in LDS, so that a lane's share of them costs
// no registers: [W] weights (1 without), then [W] biases, W = C * G * V.
template <int W>
__device__ __forceinline__ void stage_params(const NormArgs& p, float* lds, bool bias) {
  for (int i = threadIdx.x; i < W; i += 256) {
    lds[i] = p.w && i < p.D ? param_at(p.w, p.w_dtype, i) : 1.0f;
    if (bias) lds[W + i] = p.b && i < p.D ? param_at(p.b, p.w_dtype, i) : 0.0f;
  }
  __syncthreads();
}
template <int V>
__device__ __forceinline__ void read_params(const float* lds, float (&f)[V]) {
#pragma unroll
  for (int q = 0; q < V; q += 4) {
    const float4 u = *reinterpret_cast<const float4*>(lds + q);
    f[q] = u.x, f[q + 1] = u.y, f[q + 2] = u.z, f[q + 3] = u.w;
  }
}
// V values of w (or b) from column col: LDS for row groups of a wave, the
// caches for a workgroup's wide rows.
template <int V, bool STAGED>
__device__ __forceinline__ void get_params(const float* lds, const void* w, int dtype, int col, int D, float none,
                                           float (&f)[V]) {
  if constexpr (STAGED) {
    read_params<V>(lds + col, f);
  } else if (w) {
    load_params<V>(w, dtype, col, D - col, f);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = none;
  }
}

template <int DT, int G, int C, bool TAIL>
__global__ void __launch_bounds__(256) norm_fwd_kernel(NormArgs p) {
  constexpr int V = Elem<DT>::VEC, RPB = 256 / G, W = C * G * V;
  constexpr bool STAGED = G <= 64;
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) float par[STAGED ? 2 * W : 4];
  const int l = threadIdx.x % G;
  const float inv = 1.0f / (float)p.D;
  if constexpr (STAGED) stage_params<W>(p, par, true);
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / G; row < p.M; row += (int64_t)gridDim.x * RPB) {
    uint4 r[C];
    load_row<DT, G, C, TAIL>(p.x, row * p.ldx, l, p.D, r);
    end_row<DT, G, C, TAIL>(r[C - 1], l, p.D);
    float v[C][V], s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      unpack_raw<DT>(r[c], v[c]);
#pragma unroll
      for (int e = 0; e < V; ++e) s += v[c][e];
    }
    const float mean = row_sum<G>(s, red) * inv;
    float q = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = c < C - 1 || (c * G + l) * V + e < p.D ? v[c][e] - mean : 0.0f;
        q = __builtin_fmaf(d, d, q);
      }
    const float rstd = 1.0f / __builtin_sqrtf(row_sum<G>(q, red) * inv + p.eps);
    if (p.stats && l == 0) p.stats[row] = mean, p.stats[p.M + row] = rstd;
    asm volatile("" ::: "memory");   // the parameters are read again for each row, not kept
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * G + l) * V;
      float w[V], b[V];
      get_params<V, STAGED>(par, p.w, p.w_dtype, col, p.D, 1.0f, w);
      get_params<V, STAGED>(par + W, p.b, p.w_dtype, col, p.D, 0.0f, b);
#pragma unroll
      for (int e = 0; e < V; ++e) v[c][e] = (v[c][e] - mean) * rstd * w[e] + b[e];
      store_part<DT, G, C, TAIL>(p.out, row * p.ldo, c, l, p.D, v[c]);
    }
  }
}

// Waves per SIMD that the backward's registers allow, and so its workgroups per
// CU: its sums and the row as loaded take 3 registers a value of the lane (4 in
// float32), the rest about 48, with barriers in the loop (G = 256) 72.
constexpr int bwd_occ(int dtype, int G, int C) {
  const int need = (dtype == DC_F32 ? 4 * 4 : 3 * 8) * C + (G == 256 ? 72 : 48), occ = 512 / need;
  return occ < 2 ? 2 : occ > 6 ? 6 : occ;
}

template <int DT, int G, int C, bool TAIL>
__global__ void __launch_bounds__(256, bwd_occ(DT, G, C)) norm_bwd_kernel(NormArgs p) {
  constexpr int V = Elem<DT>::VEC, RPB = 256 / G, W = C * G * V;
  __shared__ float red[4];
  // the weights, and (the rows done) the waves' sums of dw and db
  __shared__ __attribute__((aligned(16))) float par[RPB > 1 ? 2 * W : W];
  const int l = threadIdx.x % G;
  float dw[C][V], db[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[c][e] = db[c][e] = 0.0f;
  stage_params<W>(p, par, false);
  const float inv = 1.0f / (float)p.D;
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / G; row < p.M; row += (int64_t)gridDim.x * RPB) {
    // the row as loaded: its float32 form would take twice the registers until dx
    uint4 rx[C], rg[C];
    load_row<DT, G, C, TAIL>(p.x, row * p.ldx, l, p.D, rx);
    load_row<DT, G, C, TAIL>(p.dy, row * p.lddy, l, p.D, rg);
    const float mean = p.stats[row], rstd = p.stats[p.M + row];
    end_row<DT, G, C, TAIL>(rx[C - 1], l, p.D);
    end_row<DT, G, C, TAIL>(rg[C - 1], l, p.D);
    float s1 = 0.0f, s2 = 0.0f;
    asm volatile("" ::: "memory");   // the weights are read again for each row, not kept
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float w[V], x[V], g[V];
      read_params<V>(par + (c * G + l) * V, w);
      unpack_raw<DT>(rx[c], x);
      unpack_raw<DT>(rg[c], g);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // past the row's end the gradient is 0, and so is its share of every sum
        const float xh = (x[e] - mean) * rstd;
        // pinned: the compiler otherwise keeps the products to add them at the loop's end
        dw[c][e] = materialize(__builtin_fmaf(g[e], xh, dw[c][e]));
        db[c][e] = materialize(db[c][e] + g[e]);
        g[e] *= w[e];
        s1 += g[e];
        s2 = __builtin_fmaf(g[e], xh, s2);
      }
    }
    s1 = row_sum<G>(s1, red) * inv;
    s2 = row_sum<G>(s2, red) * inv;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      // read and unpacked again, not kept
      asm volatile("" : "+v"(rx[c].x), "+v"(rx[c].y), "+v"(rx[c].z), "+v"(rx[c].w), "+v"(rg[c].x), "+v"(rg[c].y),
                   "+v"(rg[c].z), "+v"(rg[c].w) : : "memory");
      float w[V], x[V], g[V];
      read_params<V>(par + (c * G + l) * V, w);
      unpack_raw<DT>(rx[c], x);
      unpack_raw<DT>(rg[c], g);
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = rstd * (g[e] * w[e] - s1 - (x[e] - mean) * rstd * s2);
      if (p.out) store_part<DT, G, C, TAIL>(p.out, row * p.ldo, c, l, p.D, g);
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
    __syncthreads();   // the weights have been read
    for (int wv = 0; wv < 4; ++wv) {
      if ((int)threadIdx.x >> 6 == wv && (threadIdx.x & 63) < G) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int at = (c * G + l) * V + e;
            par[at] = wv ? par[at] + dw[c][e] : dw[c][e];
            par[W + at] = wv ? par[W + at] + db[c][e] : db[c][e];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < p.D; i += 256) out[i] = par[i], out[p.D + i] = par[W + i];
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
  if (D < vec) return {0, 0};   // no 16 bytes to read: one by one
  const int groups[] = {8, 16, 32, 64, 256};
  for (int g : groups)
    if (chunks <= (int64_t)g * NORM_MAX_C) return {g, (int)((chunks + g - 1) / g)};
  return {0, 0};
}

// Workgroups: as many as stay resident, fewer when there are few rows. The
// backward pass writes a partial row of dw and db for each.
static int64_t norm_blocks(int64_t M, int G, int per_cu) {
  const int64_t most = (int64_t)per_cu * device_cus();
  const int64_t rpb = G ? 256 / G : 1, all = (M + rpb - 1) / rpb;
  return all < most ? all : most;
}
// A partial row costs about what 2 / 3 of a row of float32 does (once written,
// once read), so past two workgroups per CU each takes 8 rows a group or more
// (4099 x 2731 float32: 1280 workgroups' partials took 11 us to join, 512 5 us).
static int64_t bwd_blocks(int64_t M, const NormPlan& r, int dtype) {
  const int64_t most = norm_blocks(M, r.G, r.G ? bwd_occ(dtype, r.G, r.C) : 4), two = norm_blocks(M, r.G, 2);
  const int64_t rpb = r.G ? 256 / r.G : 1, by_rows = M / (8 * rpb);
  return by_rows < two ? two : by_rows < most ? by_rows : most;
}
constexpr int FWD_BLOCKS = 8;

template <int DT, int G, bool TAIL>
static int launch_norm(const NormArgs& p, int C, bool bwd, hipStream_t st) {
  auto go = [&](auto c_) {
    constexpr int c = decltype(c_)::value;
    const unsigned blocks = (unsigned)(bwd ? bwd_blocks(p.M, {G, c}, DT) : norm_blocks(p.M, G, FWD_BLOCKS));
    if (bwd) hipLaunchKernelGGL((norm_bwd_kernel<DT, G, c, TAIL>), dim3(blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((norm_fwd_kernel<DT, G, c, TAIL>), dim3(blocks), dim3(256), 0, st, p);
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
  const bool tail = p.D % Elem<DT>::VEC;
  switch (r.G) {
    case 8: return tail ? launch_norm<DT, 8, true>(p, r.C, bwd, st) : launch_norm<DT, 8, false>(p, r.C, bwd, st);
    case 16: return tail ? launch_norm<DT, 16, true>(p, r.C, bwd, st) : launch_norm<DT, 16, false>(p, r.C, bwd, st);
    case 32: return tail ? launch_norm<DT, 32, true>(p, r.C, bwd, st) : launch_norm<DT, 32, false>(p, r.C, bwd, st);
    case 64: return tail ? launch_norm<DT, 64, true>(p, r.C, bwd, st) : launch_norm<DT, 64, false>(p, r.C, bwd, st);
    case 256: return tail ? launch_norm<DT, 256, true>(p, r.C, bwd, st) : launch_norm<DT, 256, false>(p, r.C, bwd, st);
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
    const int64_t P = bwd_blocks(p.M, r, DT), rows = (p.M + P - 1) / P;
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
  return sizeof(float) * 2 * (size_t)D * (size_t)bwd_blocks(M, norm_plan(D, x_dtype), x_dtype);
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
  const int64_t P = bwd_blocks(M, norm_plan(D, x_dtype), x_dtype);
  return sums ? reduce_partials(p.part, (int)P, 2, D, dw, db, w_dtype, st, who) : DC_OK;
}
