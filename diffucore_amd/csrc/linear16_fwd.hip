// Forward products of the feed-forward operators:
//   linear  y = act(x w^T + b) + res
//   gated   h = (x wv^T + bv) act(x wg^T + bg)
// on the kernel of linear16.h. A gated tile's W rows are 32-row blocks of value
// and gate rows in turn, so value and gate of an output meet in one lane.
#include "linear16.h"

namespace dc {

int refuse(int code, const char* who, const char* msg) {
  set_error("%s: %s", who, msg);
  return code;
}

// Sizes and types every product checks.
int check_product(const char* who, int dtype, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return refuse(DC_EINVAL, who, "negative size");
  if (M > 0x3fffffff || N > 0x3fffffff || K > 0x3fffffff) return refuse(DC_EINVAL, who, "size too large");
  if (dtype != DC_F16 && dtype != DC_BF16) return refuse(DC_EINVAL, who, "dtype must be DC_F16 or DC_BF16");
  return DC_OK;
}

int check_scratch(const char* who, size_t need, const void* ws, size_t ws_bytes) {
  if (!need || (ws && aligned16(ws) && ws_bytes >= need)) return DC_OK;
  set_error("%s: workspace too small or not 16-byte aligned (needs %zu bytes)", who, need);
  return DC_EWORKSPACE;
}

static bool plain_act(int act) {
  return act == DC_ACT_NONE || act == DC_ACT_GELU_ERF || act == DC_ACT_GELU_TANH || act == DC_ACT_SILU ||
         act == DC_ACT_QUICK_GELU;
}

Plan16 plan16(int64_t M, int64_t rows, int64_t nk, int problems) {
  const int64_t cus = device_cus();
  const auto tiles = [&](int bn, int bm) { return ((rows + bn - 1) / bn) * ((M + bm - 1) / bm) * problems; };
  const int64_t t128 = tiles(128, 128);
  Plan16 r{TILE_256x256, 1, (int)nk};
  if (t128 <= cus / 2) r.tile = tiles(64, 128) < cus / 2 ? TILE_64x64 : TILE_64x128;
  else if (t128 <= cus) r.tile = TILE_128x128D;
  else if (t128 <= 2 * cus) r.tile = TILE_128x128;
  if (t128 > cus / 2) return r;
  const int64_t used = r.tile == TILE_64x64 ? tiles(64, 64) : tiles(64, 128);
  int64_t s = 2 * cus / used;
  if (s > nk / 8) s = nk / 8;
  if (s > 16) s = 16;
  if (s < 2) return r;
  r.kstages = (int)((nk + s - 1) / s);
  r.splits = (int)((nk + r.kstages - 1) / r.kstages);
  return r;
}

}  // namespace dc

using namespace dc;

extern "C" size_t dc_linear16_workspace_bytes(int op, int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > 0x3fffffff || N > 0x3fffffff || K > 0x3fffffff) return 0;
  const int64_t mk = round_up(M, 64) / 64, nk = round_up(N, 64) / 64, kk = round_up(K, 64) / 64;
  switch (op) {
    case DC_LINEAR16_FWD: return plan16_bytes(plan16(M, N, kk, 1), M, N, 1);
    case DC_LINEAR16_GATED: return plan16_bytes(plan16(M, 2 * N, kk, 1), M, 2 * N, 1);
    case DC_LINEAR16_DX: return plan16_bytes(plan16(M, K, nk, 1), M, K, 1);
    case DC_LINEAR16_DX2: return plan16_bytes(plan16(M, K, 2 * nk, 1), M, K, 1);
    case DC_LINEAR16_DW: return plan16_bytes(plan16(N, K, mk, 1), N, K, 1);
    case DC_LINEAR16_DW2: return plan16_bytes(plan16(N, K, mk, 2), N, K, 2);
    default: return 0;
  }
}

extern "C" int dc_linear16(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype,
                           const void* res, int64_t ldr, int act, void* out, int64_t ldo, float* z, int64_t ldz,
                           int dtype, int64_t M, int64_t N, int64_t K, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  const char* who = "dc_linear16";
  if (int e = check_product(who, dtype, M, N, K)) return e;
  if (!plain_act(act)) return refuse(DC_EINVAL, who, "bad act");
  if (M == 0 || N == 0) return DC_OK;
  if (K == 0) return refuse(DC_EINVAL, who, "K must be positive");
  if (!x || !w || !out) return refuse(DC_EINVAL, who, "null pointer");
  if (bias && !float_dtype(bias_dtype)) return refuse(DC_EINVAL, who, "bad bias_dtype");
  if (ldo < N || (res && ldr < N) || (z && ldz < N)) return refuse(DC_EINVAL, who, "row stride < N");
  if (K % 8 || bad_operand(x, ldx, K) || bad_operand(w, ldw, K))
    return refuse(DC_EUNSUPPORTED, who, "needs K, ldx, ldw multiples of 8 and 16-byte aligned x, w");
  Gemm16 p{};
  p.a = static_cast<const uint16_t*>(x), p.lda = ldx;
  p.w = static_cast<const uint16_t*>(w), p.ldw = ldw;
  p.M = (int)M, p.N = (int)N, p.K = (int)K, p.nk = p.nk1 = (int)(round_up(K, 64) / 64);
  p.ka = (int)K, p.alim = (int)M, p.wlim = (int)N;
  p.bias = bias, p.bias_dtype = bias_dtype, p.act = act, p.res = static_cast<const uint16_t*>(res), p.ldr = ldr;
  p.out = static_cast<uint16_t*>(out), p.ldo = ldo, p.z = z, p.ldz = ldz;
  const Plan16 plan = plan16(M, N, p.nk, 1);
  p.problems = 1, p.part = static_cast<float*>(ws), p.width = (int)N;
  if (int e = check_scratch(who, plan16_bytes(plan, M, N, 1), ws, ws_bytes)) return e;
  hipStream_t st = (hipStream_t)stream;
  return dtype == DC_BF16 ? run_tile16<DC_BF16, false, false, EPI_LINEAR>(who, p, plan, st)
                          : run_tile16<DC_F16, false, false, EPI_LINEAR>(who, p, plan, st);
}

extern "C" int dc_gated16(const void* x, int64_t ldx, const void* wv, int64_t ldwv, const void* wg, int64_t ldwg,
                          const void* bv, const void* bg, int bias_dtype, int act, void* out, int64_t ldo, float* zv,
                          float* zg, int64_t ldz, int dtype, int64_t M, int64_t N, int64_t K, void* ws, size_t ws_bytes,
                          void* stream) {
  clear_error();
  const char* who = "dc_gated16";
  if (int e = check_product(who, dtype, M, N, K)) return e;
  if (!plain_act(act)) return refuse(DC_EINVAL, who, "bad act");
  if (M == 0 || N == 0) return DC_OK;
  if (K == 0) return refuse(DC_EINVAL, who, "K must be positive");
  if (!x || !wv || !wg || !out) return refuse(DC_EINVAL, who, "null pointer");
  if ((bv || bg) && !float_dtype(bias_dtype)) return refuse(DC_EINVAL, who, "bad bias_dtype");
  if (!zv != !zg) return refuse(DC_EINVAL, who, "zv and zg go together");
  if (ldo < N || (zv && ldz < N)) return refuse(DC_EINVAL, who, "row stride < N");
  if (K % 8 || bad_operand(x, ldx, K) || bad_operand(wv, ldwv, K) || bad_operand(wg, ldwg, K))
    return refuse(DC_EUNSUPPORTED, who, "needs K and row strides multiples of 8 and 16-byte aligned x, wv, wg");
  Gemm16 p{};
  p.a = static_cast<const uint16_t*>(x), p.lda = ldx;
  p.w = static_cast<const uint16_t*>(wv), p.ldw = ldwv;
  p.w2 = static_cast<const uint16_t*>(wg), p.ldw2 = ldwg;
  p.M = (int)M, p.N = (int)N, p.K = (int)K, p.nk = p.nk1 = (int)(round_up(K, 64) / 64);
  p.ka = (int)K, p.alim = (int)M, p.wlim = (int)N;
  p.bias = bv, p.bias2 = bg, p.bias_dtype = bias_dtype, p.act = act;
  p.out = static_cast<uint16_t*>(out), p.ldo = ldo;
  p.z = zv, p.z2 = zg, p.ldz = ldz;
  const Plan16 plan = plan16(M, 2 * N, p.nk, 1);
  p.problems = 1, p.part = static_cast<float*>(ws), p.width = (int)(2 * N);
  if (int e = check_scratch(who, plan16_bytes(plan, M, 2 * N, 1), ws, ws_bytes)) return e;
  hipStream_t st = (hipStream_t)stream;
  return dtype == DC_BF16 ? run_tile16<DC_BF16, false, false, EPI_GATED>(who, p, plan, st)
                          : run_tile16<DC_F16, false, false, EPI_GATED>(who, p, plan, st);
}

