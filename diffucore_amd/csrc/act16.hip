// The elementwise half of the feed-forward backward passes on gfx950: output
// gradient times the activation's slope, written as the 16-bit operand of the
// two products that follow, with the bias gradients' column sums taken from
// the float32 values on the way.
//
//   linear  dz = dy act'(z)                          reads 2 + 3 bytes an element, writes 2
//   gated   dzv = dy act(zg), dzg = dy zv act'(zg)   reads 2 + 6, writes 4
//   sums    db = sum over rows of dy                 reads 2
//
// The pre-activations z are kept in 24 bits. Rounded to 16 they cost a third
// rounding of the same size as dz's own and the result's (bf16 gated gradients
// 0.0031 off in relative L2 where the rounding of the result alone is 0.0017,
// 0.0024 with 24 bits or 32).
//
// Memory-bound: one pass, 16 bytes a lane and access. A workgroup takes 8 * TX
// columns (TX lanes of 8 columns) and every TYth row of a block of rows, sums
// its rows in registers, joins its TY row lanes through LDS and writes one
// partial row; reduce_partials adds those in order.
#include "colsum.h"

namespace dc {

struct ActBwdArgs {
  const uint16_t* dy;
  const uint8_t* za;    // linear: z; gated: the value's pre-activation (store_saved8)
  const uint8_t* zg;
  uint16_t* da;         // linear: dz; gated: the value's gradient
  uint16_t* dg;
  float* part;          // [P][1 or 2][N], NULL: no sums
  int64_t lddy, lddz;
  int M, N, pad;        // pad: columns of dz to fill (its row stride)
  int tx_log, rows;     // log2 TX; rows per workgroup
  int act;
};

// MODE 0: sums of dy alone, 1: linear, 2: gated
template <int DT, int MODE, int ACT>
__device__ __forceinline__ void act_bwd_rows(const ActBwdArgs& p, int64_t col, int ty, int TY, float (&sa)[8],
                                             float (&sg)[8]) {
  const int64_t r0 = (int64_t)blockIdx.y * p.rows, r1 = min(r0 + p.rows, (int64_t)p.M);
  const int64_t n = p.N - col;   // columns left: 8 or more, or a row's tail
  for (int64_t r = r0 + ty; r < r1; r += TY) {
    float dy[8], a[8], g[8];
    load8_n<DT>(p.dy + r * p.lddy + col, n, dy);
    if constexpr (MODE == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sa[e] += dy[e];
    } else {
      load_saved8(p.za, p.M, p.N, r, col, a);
      if constexpr (MODE == 2) load_saved8(p.zg, p.M, p.N, r, col, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float value;
        if constexpr (MODE == 1) {
          a[e] = dy[e] * act_slope<ACT>(a[e], value);
        } else {
          const float slope = act_slope<ACT>(g[e], value);
          g[e] = dy[e] * a[e] * slope;
          a[e] = dy[e] * value;
        }
        // the row's tail: dz holds zeros there, whatever a gradient of 0 times a slope gives
        if (e >= n) a[e] = 0.0f, g[e] = 0.0f;
        sa[e] += a[e];
        if constexpr (MODE == 2) sg[e] += g[e];
      }
      *reinterpret_cast<uint4*>(p.da + r * p.lddz + col) = pack8<DT>(a);
      if constexpr (MODE == 2) *reinterpret_cast<uint4*>(p.dg + r * p.lddz + col) = pack8<DT>(g);
    }
  }
}

template <int DT, int MODE>
__global__ void __launch_bounds__(256) act_bwd_kernel(ActBwdArgs p) {
  __shared__ float red[256 * 8];
  const int t = threadIdx.x, TX = 1 << p.tx_log, TY = 256 >> p.tx_log;
  const int tx = t & (TX - 1), ty = t >> p.tx_log;
  const int64_t col = 8 * ((int64_t)blockIdx.x * TX + tx);
  float sa[8] = {0}, sg[8] = {0};
  if (col < (MODE == 0 ? p.N : p.pad)) {
    if constexpr (MODE == 0) act_bwd_rows<DT, 0, DC_ACT_NONE>(p, col, ty, TY, sa, sg);
    else with_act(p.act, [&](auto a) { act_bwd_rows<DT, MODE, decltype(a)::value>(p, col, ty, TY, sa, sg); });
  }
  if (!p.part) return;
#pragma unroll
  for (int s = 0; s < (MODE == 2 ? 2 : 1); ++s) {
    float (&v)[8] = s ? sg : sa;
    if (s) __syncthreads();   // the first section's sums have been read
#pragma unroll
    for (int e = 0; e < 8; ++e) red[e * 256 + t] = v[e];
    __syncthreads();
    for (int i = t; i < 8 * TX; i += 256) {
      const int e = i >> p.tx_log, x = i & (TX - 1);
      const int64_t c = 8 * ((int64_t)blockIdx.x * TX + x) + e;
      float sum = 0.0f;
      for (int y = 0; y < TY; ++y) sum += red[e * 256 + y * TX + x];
      if (c < p.N) p.part[((int64_t)blockIdx.y * (MODE == 2 ? 2 : 1) + s) * p.N + c] = sum;
    }
  }
}

// One workgroup: 32 columns, 8 lanes down the partials.
__global__ void __launch_bounds__(256) reduce_partials_kernel(const float* __restrict__ part, int P, int sections,
                                                              int64_t width, void* out0, void* out1, int out_dtype) {
  __shared__ float red[8][32];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, s = blockIdx.y;
  void* out = s ? out1 : out0;
  if (!out) return;
  const int64_t c = (int64_t)blockIdx.x * 32 + x;
  float sum = 0.0f;
  if (c < width) {
    const float* src = part + s * width + c;
    const int64_t step = sections * width;
#pragma unroll 8
    for (int q = y; q < P; q += 8) sum += src[q * step];
  }
  red[y][x] = sum;
  __syncthreads();
  if (y == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += red[i][x];
    if (out_dtype == DC_F32) static_cast<float*>(out)[c] = sum;
    else static_cast<uint16_t*>(out)[c] =
        (uint16_t)(out_dtype == DC_BF16 ? f32_to_bf16_bits(sum) : f32_to_f16_bits(sum));
  }
}

int reduce_partials(const float* part, int P, int sections, int64_t width, void* out0, void* out1, int out_dtype,
                    hipStream_t st, const char* what) {
  if (width == 0) return DC_OK;
  hipLaunchKernelGGL(reduce_partials_kernel, dim3((unsigned)((width + 31) / 32), sections), dim3(256), 0, st, part, P,
                     sections, width, out0, out1, out_dtype);
  return launch_status(what);
}

// The split of an [M, N] pass: TX lanes of 8 columns, the most (a power of two,
// 64 at most) that leave no more than an eighth of them idle past the row's end,
// but 16 where rows have as many; and row blocks so that about 8 workgroups per
// CU run, down to one row a lane. 777 x 2731 gated bf16 18.6 -> 11.9 us, 1001 x
// 577 fp16 10.8 -> 5.4 against 4 rows a lane on 64 lanes.
struct ActBwdPlan {
  int tx_log, rows, col_blocks, row_blocks;
};
static ActBwdPlan act_bwd_plan(int64_t M, int64_t N) {
  ActBwdPlan r;
  const int64_t chunks = dz_width(N) / 8;   // of a row of dz
  for (r.tx_log = 6; r.tx_log > 3; --r.tx_log) {
    const int64_t TX = 1LL << r.tx_log, idle = (chunks + TX - 1) / TX * TX - chunks;
    if (8 * idle <= chunks || (r.tx_log == 4 && chunks >= 16)) break;
  }
  const int64_t TX = 1LL << r.tx_log, TY = 256 >> r.tx_log, most = (M + TY - 1) / TY;
  r.col_blocks = (int)((chunks + TX - 1) / TX);
  int64_t want = (8LL * device_cus() + r.col_blocks - 1) / r.col_blocks;
  if (want > most) want = most;
  if (want < 1) want = 1;
  if (want > 512) want = 512;
  r.rows = (int)((M + want - 1) / want);
  if (r.rows < 1) r.rows = 1;
  r.row_blocks = (int)((M + r.rows - 1) / r.rows);
  if (r.row_blocks < 1) r.row_blocks = 1;
  return r;
}

size_t act16_bwd_part_bytes(int64_t M, int64_t N, bool gated) {
  const ActBwdPlan r = act_bwd_plan(M, N);
  return sizeof(float) * (size_t)r.row_blocks * (gated ? 2 : 1) * (size_t)N;
}

template <int MODE>
static int run_act_bwd(const char* who, ActBwdArgs p, int dtype, void* db0, void* db1, int db_dtype, hipStream_t st) {
  const ActBwdPlan r = act_bwd_plan(p.M, p.N);
  p.tx_log = r.tx_log, p.rows = r.rows;
  const dim3 grid(r.col_blocks, r.row_blocks);
  if (dtype == DC_BF16) hipLaunchKernelGGL((act_bwd_kernel<DC_BF16, MODE>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((act_bwd_kernel<DC_F16, MODE>), grid, dim3(256), 0, st, p);
  if (int e = launch_status(who)) return e;
  return p.part ? reduce_partials(p.part, r.row_blocks, MODE == 2 ? 2 : 1, p.N, db0, db1, db_dtype, st, who) : DC_OK;
}

int act16_bwd(const char* who, const ActBwd& a, hipStream_t st) {
  ActBwdArgs p{};
  p.dy = static_cast<const uint16_t*>(a.dy), p.lddy = a.lddy, p.M = (int)a.M, p.N = (int)a.N;
  p.za = a.zv, p.zg = a.zg, p.act = a.act;
  p.da = static_cast<uint16_t*>(a.dzv), p.dg = static_cast<uint16_t*>(a.dzg), p.lddz = a.lddz, p.pad = (int)a.lddz;
  p.part = a.dbv || a.dbg ? a.part : nullptr;
  if (a.zg) return run_act_bwd<2>(who, p, a.dtype, a.dbv, a.dbg, a.db_dtype, st);
  if (a.zv) return run_act_bwd<1>(who, p, a.dtype, a.dbv, nullptr, a.db_dtype, st);
  return run_act_bwd<0>(who, p, a.dtype, a.dbv, nullptr, a.db_dtype, st);
}

// ---------------------------------------------------------------- padded copies

// dst [rows, W rounded up to 8] = src [rows, W] and zeros, for each job: a thread
// a chunk of 8.
__global__ void __launch_bounds__(256) pad_rows_kernel(PadJobs p) {
  const int j = p.count > 2 && blockIdx.x >= p.first[2] ? 2 : p.count > 1 && blockIdx.x >= p.first[1] ? 1 : 0;
  const PadJob job = j == 0 ? p.job[0] : j == 1 ? p.job[1] : p.job[2];
  const uint32_t first = j == 0 ? 0u : j == 1 ? p.first[1] : p.first[2];
  const int64_t chunks = (job.width + 7) / 8, i = (int64_t)(blockIdx.x - first) * 256 + threadIdx.x;
  if (i >= job.rows * chunks) return;
  const int64_t r = i / chunks, c = i % chunks;
  reinterpret_cast<uint4*>(job.dst)[i] = load_chunk16(job.src + r * job.ld + 8 * c, job.width - 8 * c);
}

int PadJobs::run(const char* who, hipStream_t st) {
  if (!count) return DC_OK;
  int64_t blocks = 0;
  for (int j = 0; j < count; ++j) {
    first[j] = (uint32_t)blocks;
    blocks += (job[j].rows * ((job[j].width + 7) / 8) + 255) / 256;
    if (blocks > 0x7fffffff) return fail(DC_EINVAL, "linear16: operands too large to pad");
  }
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)blocks), dim3(256), 0, st, *this);
  return launch_status(who);
}

}  // namespace dc
