// Backward passes of the feed-forward operators: the elementwise half
// (act16.hip), then on the kernel of linear16.h
//   dx = dz w (+ dzg wg)     dz along k, w along its rows
//   dw = dz^T x              both along their rows, k the rows of the batch
#include "linear16.h"

namespace dc {

struct Backward16 {
  Mat16 dy, x, wv, wg, dz, dzg, xs, wvs, wgs;   // ..s: as the kernels read them
  Plan16 dx_plan, dw_plan;
  float* part;
  int problems;
  bool z;
  size_t bytes;

  // want_dx / want_dw / want_db as the call asks; z: there are pre-activations
  Backward16(const Mat16& dy_, const Mat16& x_, const Mat16& wv_, const Mat16& wg_, bool z_, bool want_dx, int want_dw,
             bool want_db, void* base)
      : dy(dy_), x(x_), wv(wv_), wg(wg_), z(z_) {
    const int64_t M = dy.rows, N = dy.width, K = x.width, ldz = dz_width(N);
    const bool gated = wg.p;
    Scratch16 s{static_cast<uint8_t*>(base)};
    if (z) {
      dz = {s.take(2 * (size_t)M * ldz), ldz, M, ldz};
      if (gated) dzg = {s.take(2 * (size_t)M * ldz), ldz, M, ldz};
      else dzg = {};
    } else {
      dz = want_dx || want_dw ? s.operand(dy) : dy;
      dzg = {};
    }
    xs = want_dw ? s.operand(x) : x;
    wvs = want_dx ? s.operand(wv) : wv;
    wgs = want_dx && gated ? s.operand(wg) : wg;
    // the passes run one after the other: their partial sums share one place
    const int64_t nk = round_up(N, 64) / 64;
    problems = want_dw == 2 ? 2 : 1;
    dx_plan = plan16(M, K, gated ? 2 * nk : nk, 1);
    dw_plan = plan16(N, K, round_up(M, 64) / 64, problems);
    size_t most = want_db ? act16_bwd_part_bytes(M, N, gated) : 0;
    if (want_dx) most = max_of(most, plan16_bytes(dx_plan, M, K, 1));
    if (want_dw) most = max_of(most, plan16_bytes(dw_plan, N, K, problems));
    part = static_cast<float*>(s.take(most));
    bytes = s.used;
  }
  int pad(const char* who, hipStream_t st) const {
    PadJobs jobs;
    add_pad(jobs, x, xs), add_pad(jobs, wv, wvs);
    if (wg.p) add_pad(jobs, wg, wgs);
    else if (!z) add_pad(jobs, dy, dz);
    return jobs.run(who, st);
  }
  static size_t max_of(size_t a, size_t b) { return a > b ? a : b; }
};

static int run_dx(const char* who, const Backward16& b, void* dx, int64_t lddx, int dtype, hipStream_t st) {
  const int64_t M = b.dy.rows, N = b.dy.width, K = b.x.width, N64 = round_up(N, 64);
  Gemm16 p{};
  p.a = static_cast<const uint16_t*>(b.dz.p), p.a2 = static_cast<const uint16_t*>(b.dzg.p), p.lda = b.dz.ld;
  p.w = static_cast<const uint16_t*>(b.wvs.p), p.ldw = b.wvs.ld;
  p.w2 = static_cast<const uint16_t*>(b.wgs.p), p.ldw2 = b.wgs.ld;
  p.M = (int)M, p.N = (int)K, p.K = (int)N, p.ka = (int)b.dz.width;
  p.nk1 = (int)(N64 / 64), p.nk = b.wg.p ? 2 * p.nk1 : p.nk1;
  p.alim = (int)M, p.wlim = (int)round_up(K, 8);
  if (b.wg.p && N % 64) p.zeros = p.a + round_up(N, 8);   // of dz's first row
  p.out = static_cast<uint16_t*>(dx), p.ldo = lddx;
  p.problems = 1, p.part = b.part, p.width = (int)K;
  return dtype == DC_BF16 ? run_tile16<DC_BF16, false, true, EPI_NONE>(who, p, b.dx_plan, st)
                          : run_tile16<DC_F16, false, true, EPI_NONE>(who, p, b.dx_plan, st);
}

// dw of dz, or of both halves' dz (dw2).
static int run_dw(const char* who, const Backward16& b, const void* dz, void* dw, const void* dz2, void* dw2,
                  int64_t lddw, int dtype, hipStream_t st) {
  const int64_t M = b.dy.rows, N = b.dy.width, K = b.x.width;
  Gemm16 p{};
  p.a = static_cast<const uint16_t*>(dz), p.a2 = static_cast<const uint16_t*>(dz2), p.lda = b.dz.ld;
  p.w = static_cast<const uint16_t*>(b.xs.p), p.ldw = b.xs.ld;
  p.M = (int)N, p.N = (int)K, p.K = (int)M, p.nk = p.nk1 = (int)(round_up(M, 64) / 64);
  p.alim = (int)round_up(N, 8), p.wlim = (int)round_up(K, 8);
  p.out = static_cast<uint16_t*>(dw), p.out2 = static_cast<uint16_t*>(dw2), p.ldo = lddw;
  p.problems = b.problems, p.part = b.part, p.width = (int)K;
  return dtype == DC_BF16 ? run_tile16<DC_BF16, true, true, EPI_NONE>(who, p, b.dw_plan, st)
                          : run_tile16<DC_F16, true, true, EPI_NONE>(who, p, b.dw_plan, st);
}

// Zeros: a product over no rows.
__global__ void __launch_bounds__(256) zero_rows_kernel(uint16_t* p, int64_t ld, int64_t rows, int64_t width) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * width; i += (int64_t)gridDim.x * 256)
    p[i / width * ld + i % width] = 0;
}
static int zero_rows(const char* who, void* p, int64_t ld, int64_t rows, int64_t width, hipStream_t st) {
  hipLaunchKernelGGL(zero_rows_kernel, dim3(1024), dim3(256), 0, st, static_cast<uint16_t*>(p), ld, rows, width);
  return launch_status(who);
}

}  // namespace dc

using namespace dc;

extern "C" size_t dc_linear16_bwd_workspace_bytes(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                                  const void* w, int64_t ldw, int act, int want, int64_t M, int64_t N,
                                                  int64_t K) {
  if (M <= 0 || N <= 0 || check_product("dc_linear16_bwd", DC_F16, act, M, N, K)) return 0;
  return Backward16({dy, lddy, M, N}, {x, ldx, M, K}, {w, ldw, N, K}, {}, act != DC_ACT_NONE, want & DC_WANT_DX,
                    want & DC_WANT_DW ? 1 : 0, want & DC_WANT_DB, nullptr).bytes;
}

extern "C" int dc_linear16_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int64_t ldw,
                               const void* z, int act, void* dx, int64_t lddx, void* dw, int64_t lddw,
                               void* db, int db_dtype, int dtype, int64_t M, int64_t N, int64_t K, void* ws,
                               size_t ws_bytes, void* stream) {
  clear_error();
  const char* who = "dc_linear16_bwd";
  if (int e = check_product(who, dtype, act, M, N, K)) return e;
  if (db && !float_dtype(db_dtype)) return refuse(DC_EINVAL, who, "bad db_dtype");
  if ((dx && lddx < K) || (dw && lddw < K)) return refuse(DC_EINVAL, who, "row stride less than the row");
  hipStream_t st = (hipStream_t)stream;
  if (M == 0 || N == 0) {
    if (dx && M)
      if (int e = zero_rows(who, dx, lddx, M, K, st)) return e;
    if (dw && N)
      if (int e = zero_rows(who, dw, lddw, N, K, st)) return e;
    return db ? reduce_partials(nullptr, 0, 1, N, db, nullptr, db_dtype, st, who) : DC_OK;
  }
  if (!dx && !dw && !db) return DC_OK;
  const bool act_z = act != DC_ACT_NONE;
  if (!dy || !x || !w || (act_z && !z)) return refuse(DC_EINVAL, who, "null pointer");
  if (lddy < N || ldx < K || ldw < K)
    return refuse(DC_EINVAL, who, "row stride less than the row");
  const Backward16 b({dy, lddy, M, N}, {x, ldx, M, K}, {w, ldw, N, K}, {}, act_z, dx, dw ? 1 : 0, db, ws);
  if (int e = check_scratch(who, b.bytes, ws, ws_bytes)) return e;
  if (int e = b.pad(who, st)) return e;
  if (act_z || db) {
    const ActBwd a{dy, lddy, static_cast<const uint8_t*>(act_z ? z : nullptr), nullptr, act,
                   const_cast<void*>(act_z ? b.dz.p : nullptr), nullptr, dz_width(N), db, nullptr, db_dtype, dtype,
                   M, N, b.part};
    if (int e = act16_bwd(who, a, st)) return e;
  }
  if (dx)
    if (int e = run_dx(who, b, dx, lddx, dtype, st)) return e;
  if (!dw) return DC_OK;
  return run_dw(who, b, b.dz.p, dw, nullptr, nullptr, lddw, dtype, st);
}

extern "C" size_t dc_gated16_bwd_workspace_bytes(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                                 const void* wv, int64_t ldwv, const void* wg, int64_t ldwg, int want,
                                                 int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || !wg || check_product("dc_gated16_bwd", DC_F16, DC_ACT_NONE, M, N, K)) return 0;
  return Backward16({dy, lddy, M, N}, {x, ldx, M, K}, {wv, ldwv, N, K}, {wg, ldwg, N, K}, true, want & DC_WANT_DX,
                    (want & DC_WANT_DW ? 1 : 0) + (want & DC_WANT_DW2 ? 1 : 0), want & DC_WANT_DB, nullptr).bytes;
}

extern "C" int dc_gated16_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* wv, int64_t ldwv,
                              const void* wg, int64_t ldwg, const void* zv, const void* zg, int act,
                              void* dx, int64_t lddx, void* dwv, void* dwg, int64_t lddw, void* dbv, void* dbg,
                              int db_dtype, int dtype, int64_t M, int64_t N, int64_t K, void* ws, size_t ws_bytes,
                              void* stream) {
  clear_error();
  const char* who = "dc_gated16_bwd";
  if (int e = check_product(who, dtype, act, M, N, K)) return e;
  if ((dbv || dbg) && !float_dtype(db_dtype)) return refuse(DC_EINVAL, who, "bad db_dtype");
  if ((dx && lddx < K) || ((dwv || dwg) && lddw < K)) return refuse(DC_EINVAL, who, "row stride less than the row");
  hipStream_t st = (hipStream_t)stream;
  if (M == 0 || N == 0) {
    if (dx && M)
      if (int e = zero_rows(who, dx, lddx, M, K, st)) return e;
    if (dwv && N)
      if (int e = zero_rows(who, dwv, lddw, N, K, st)) return e;
    if (dwg && N)
      if (int e = zero_rows(who, dwg, lddw, N, K, st)) return e;
    return dbv || dbg ? reduce_partials(nullptr, 0, 2, N, dbv, dbg, db_dtype, st, who) : DC_OK;
  }
  if (!dx && !dwv && !dwg && !dbv && !dbg) return DC_OK;
  if (!dy || !x || !wv || !wg || !zv || !zg) return refuse(DC_EINVAL, who, "null pointer");
  if (lddy < N || ldx < K || ldwv < K || ldwg < K)
    return refuse(DC_EINVAL, who, "row stride less than the row");
  const int dws = (dwv ? 1 : 0) + (dwg ? 1 : 0);
  const Backward16 b({dy, lddy, M, N}, {x, ldx, M, K}, {wv, ldwv, N, K}, {wg, ldwg, N, K}, true, dx, dws, dbv || dbg,
                     ws);
  if (int e = check_scratch(who, b.bytes, ws, ws_bytes)) return e;
  if (int e = b.pad(who, st)) return e;
  const ActBwd a{dy, lddy, static_cast<const uint8_t*>(zv), static_cast<const uint8_t*>(zg), act,
                 const_cast<void*>(b.dz.p), const_cast<void*>(b.dzg.p), b.dz.ld, dbv, dbg, db_dtype, dtype, M, N,
                 b.part};
  if (int e = act16_bwd(who, a, st)) return e;
  if (dx)
    if (int e = run_dx(who, b, dx, lddx, dtype, st)) return e;
  if (!dws) return DC_OK;
  if (dws == 2) return run_dw(who, b, b.dz.p, dwv, b.dzg.p, dwg, lddw, dtype, st);
  return run_dw(who, b, dwv ? b.dz.p : b.dzg.p, dwv ? dwv : dwg, nullptr, nullptr, lddw, dtype, st);
}
