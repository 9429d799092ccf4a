// Backward products of the feed-forward operators, on the kernel of linear16.h:
//   dx = dz w (+ dz2 w2)   dz along k, w along its rows
//   dw = dz^T x            both along their rows, k the rows of the batch
#include "linear16.h"

using namespace dc;

extern "C" int dc_linear16_dx(const void* dz, int64_t lddz, const void* w, int64_t ldw, const void* dz2,
                              const void* w2, int64_t ldw2, void* dx, int64_t lddx, int dtype,
                              int64_t M, int64_t N, int64_t K, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  const char* who = "dc_linear16_dx";
  if (int e = check_product(who, dtype, M, N, K)) return e;
  if (M == 0 || K == 0) return DC_OK;
  if (N == 0) return refuse(DC_EINVAL, who, "N must be positive");
  if (!dz || !w || !dx || !dz2 != !w2) return refuse(DC_EINVAL, who, "null pointer");
  if (lddx < K) return refuse(DC_EINVAL, who, "row stride < K");
  const int64_t N64 = round_up(N, 64), width = dz2 ? N64 : round_up(N, 8), K8 = round_up(K, 8);
  if (bad_operand(dz, lddz, width) || bad_operand(w, ldw, K8) ||
      (dz2 && (bad_operand(dz2, lddz, width) || bad_operand(w2, ldw2, K8))))
    return refuse(DC_EUNSUPPORTED, who, "needs row strides in multiples of 8 that cover the padded rows, and "
                                        "16-byte aligned dz, w");
  Gemm16 p{};
  p.a = static_cast<const uint16_t*>(dz), p.lda = lddz;
  p.a2 = static_cast<const uint16_t*>(dz2);
  p.w = static_cast<const uint16_t*>(w), p.ldw = ldw;
  p.w2 = static_cast<const uint16_t*>(w2), p.ldw2 = ldw2;
  p.M = (int)M, p.N = (int)K, p.K = (int)N, p.nk1 = (int)(N64 / 64), p.nk = dz2 ? 2 * p.nk1 : p.nk1;
  p.ka = (int)width, p.alim = (int)M, p.wlim = (int)K8;
  p.out = static_cast<uint16_t*>(dx), p.ldo = lddx;
  const Plan16 plan = plan16(M, K, p.nk, 1);
  p.problems = 1, p.part = static_cast<float*>(ws), p.width = (int)K;
  if (int e = check_scratch(who, plan16_bytes(plan, M, K, 1), ws, ws_bytes)) return e;
  hipStream_t st = (hipStream_t)stream;
  return dtype == DC_BF16 ? run_tile16<DC_BF16, false, true, EPI_NONE>(who, p, plan, st)
                          : run_tile16<DC_F16, false, true, EPI_NONE>(who, p, plan, st);
}

extern "C" int dc_linear16_dw(const void* dz, int64_t lddz, const void* x, int64_t ldx, const void* dz2, void* dw,
                              int64_t lddw, void* dw2, int dtype, int64_t M, int64_t N, int64_t K, void* ws, size_t ws_bytes,
                              void* stream) {
  clear_error();
  const char* who = "dc_linear16_dw";
  if (int e = check_product(who, dtype, M, N, K)) return e;
  if (N == 0 || K == 0) return DC_OK;
  if (!dw || !dz2 != !dw2 || (M && (!dz || !x))) return refuse(DC_EINVAL, who, "null pointer");
  if (lddw < K) return refuse(DC_EINVAL, who, "row stride < K");
  const int64_t N8 = round_up(N, 8), K8 = round_up(K, 8);
  if (M && (bad_operand(dz, lddz, N8) || bad_operand(x, ldx, K8) || (dz2 && bad_operand(dz2, lddz, N8))))
    return refuse(DC_EUNSUPPORTED, who, "needs row strides in multiples of 8 that cover the padded rows, and "
                                        "16-byte aligned dz, x");
  Gemm16 p{};
  p.a = static_cast<const uint16_t*>(dz), p.lda = lddz;
  p.a2 = static_cast<const uint16_t*>(dz2);
  p.w = static_cast<const uint16_t*>(x), p.ldw = ldx;
  p.M = (int)N, p.N = (int)K, p.K = (int)M, p.nk = p.nk1 = (int)(round_up(M, 64) / 64);
  p.alim = (int)N8, p.wlim = (int)K8;
  p.out = static_cast<uint16_t*>(dw), p.out2 = static_cast<uint16_t*>(dw2), p.ldo = lddw;
  const int problems = dz2 ? 2 : 1;
  const Plan16 plan = plan16(N, K, p.nk, problems);
  p.problems = problems, p.part = static_cast<float*>(ws), p.width = (int)K;
  if (int e = check_scratch(who, plan16_bytes(plan, N, K, problems), ws, ws_bytes)) return e;
  hipStream_t st = (hipStream_t)stream;
  return dtype == DC_BF16 ? run_tile16<DC_BF16, true, true, EPI_NONE>(who, p, plan, st)
                          : run_tile16<DC_F16, true, true, EPI_NONE>(who, p, plan, st);
}
