// Forward products of the feed-forward operators:
//   linear  y = act(x w^T + b) + res
//   gated   h = (x wv^T + bv) act(x wg^T + bg)
// on the kernel of linear16.h. A gated tile's W rows are 32-row blocks of value
// and gate rows in turn, so value and gate of an output meet in one wave.
#include "linear16.h"

namespace dc {

int refuse(int code, const char* who, const char* msg) {
  set_error("%s: %s", who, msg);
  return code;
}

int check_product(const char* who, int dtype, int act, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K <= 0) return refuse(DC_EINVAL, who, "bad M/N/K");
  if (M > 0x3fffffff || N > 0x1fffffff || K >= (1 << 22))
    return refuse(DC_EINVAL, who, "size too large (M < 2^30, N < 2^29, K < 2^22)");
  if (dtype != DC_F16 && dtype != DC_BF16) return refuse(DC_EINVAL, who, "dtype must be DC_F16 or DC_BF16");
  if (act != DC_ACT_NONE && act != DC_ACT_GELU_ERF && act != DC_ACT_GELU_TANH && act != DC_ACT_SILU &&
      act != DC_ACT_QUICK_GELU)
    return refuse(DC_EINVAL, who, "bad act");
  return DC_OK;
}

int check_scratch(const char* who, size_t need, const void* ws, size_t ws_bytes) {
  if (!need || (ws && aligned16(ws) && ws_bytes >= need)) return DC_OK;
  set_error("%s: workspace too small or not 16-byte aligned (needs %zu bytes)", who, need);
  return DC_EWORKSPACE;
}

// Tile and k slices by the least of a fitted time, in us:
//   T = fixed + h (round + stage * stages)  [+ 3.2 + 0.34 per MB of partial sums when k is split]
// where a round fills every CU with `per` workgroups of the tile and h counts
// rounds; a last round in which the busiest CU holds j < per of them counts
// level[j - 1], and any level that is not full on every CU counts up to `slack`
// less (the clock rises and memory frees as CUs fall idle). Fitted to 10500 random
// products of 17 to 16384 rows, 16 to 20480 channels and 64 to 8192 of k (all
// three operand layouts, with and without kept pre-activations, 9 tiles, up to 16
// slices; operands rotated through memory): rms error of a time 9 to 14%, and the
// pick is 1.9% off the best of all tiles and slices on average. A rule that went by
// the number of 128 x 128 tiles was 6.9% off. At 256 x 256 / 256 x 192 / 128 x 192 /
// 128 x 128, us: 4608 x 2048 -> 8192 196 / 159 / 161 / 171, gated 8192 x 640 -> 2560
// 76 / 80 / 68 / 72, 8192 x 2560 -> 640 62 / 51 / 41 / 38, dw of 4608 x (2048, 8192)
// 131 / 190 / 158 / 153.
struct TileCost {
  int tile, bn, bm, per;
  float fixed, round, stage, slack, level[2];
};
static constexpr TileCost COSTS[] = {
    {TILE_256x256, 256, 256, 1, 1.47f, 7.95f, 1.840f, 0.315f, {}},
    {TILE_256x192, 256, 192, 1, 2.85f, 5.39f, 1.485f, 0.341f, {}},
    {TILE_256x128, 256, 128, 1, 3.00f, 4.57f, 1.001f, 0.312f, {}},
    {TILE_128x256, 128, 256, 1, 3.01f, 4.60f, 1.016f, 0.334f, {}},
    {TILE_128x192, 128, 192, 2, 4.76f, 4.50f, 1.490f, 0.232f, {0.675f}},
    {TILE_128x128, 128, 128, 2, 3.35f, 3.45f, 1.129f, 0.202f, {0.792f}},
    {TILE_128x128D, 128, 128, 1, 3.83f, 2.93f, 0.586f, 0.316f, {}},
    {TILE_64x128, 64, 128, 2, 5.21f, 1.77f, 0.768f, 0.232f, {0.549f}},
    {TILE_64x64, 64, 64, 3, 5.75f, 1.42f, 0.671f, 0.108f, {0.395f, 0.646f}},
};

Plan16 plan16(int64_t M, int64_t rows, int64_t nk, int problems) {
  const int64_t cus = device_cus();
  const float mb = (float)((double)M * (double)rows * problems * 4e-6);
  Plan16 best{TILE_256x256, 1, (int)nk};
  float least = 1e30f;
  for (const TileCost& c : COSTS) {
    const int64_t tiles = (rows + c.bn - 1) / c.bn * ((M + c.bm - 1) / c.bm) * problems;
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16}) {
      // slices of 4 stages or more, of products that leave CUs idle
      if (s > 1 && (tiles > cus || nk < 4 * s)) break;
      const int64_t stages = (nk + s - 1) / s, splits = stages ? (nk + stages - 1) / stages : 1;
      const int64_t units = tiles * splits, slots = cus * c.per;
      const int64_t rest = units % slots, j = (rest + cus - 1) / cus;   // j: on the busiest CU of the last round
      float h = (float)(units / slots);
      if (j) h += (j < c.per ? c.level[j - 1] : 1.0f) * (1.0f - c.slack * (1.0f - (float)rest / (float)(cus * j)));
      float t = c.fixed + h * (c.round + c.stage * (float)stages);
      if (splits > 1) t += 3.2f + 0.34f * mb * (float)splits;
      if (t < least) least = t, best = {c.tile, (int)splits, (int)stages};
    }
  }
  return best;
}

// A forward call's scratch: copies of the operands that need one, split-K sums.
struct Forward16 {
  Mat16 x, w, w2, xs, ws, w2s;   // as given, and as the kernel reads them
  Plan16 plan;
  float* part = nullptr;
  size_t bytes = 0;
  bool skinny;
  Forward16(const Mat16& x_, const Mat16& w_, const Mat16& w2_, int64_t M, int64_t N, int64_t K, void* base)
      : x(x_), w(w_), w2(w2_), xs(x_), ws(w_), w2s(w2_), skinny(skinny16(M, w2_.p ? 2 * N : N, K, w2_.p)) {
    if (skinny) return;
    Scratch16 s{static_cast<uint8_t*>(base)};
    xs = s.operand(x), ws = s.operand(w), w2s = w2.p ? s.operand(w2) : w2;
    const int64_t rows = w2.p ? 2 * N : N;
    plan = plan16(M, rows, round_up(K, 64) / 64, 1);
    part = static_cast<float*>(s.take(plan16_bytes(plan, M, rows, 1)));
    bytes = s.used;
  }
  int pad(const char* who, hipStream_t st) const {
    PadJobs jobs;
    add_pad(jobs, x, xs), add_pad(jobs, w, ws);
    if (w2.p) add_pad(jobs, w2, w2s);
    return jobs.run(who, st);
  }
  Gemm16 args(int64_t M, int64_t N, int64_t K) const {
    Gemm16 p{};
    p.a = static_cast<const uint16_t*>(xs.p), p.lda = xs.ld;
    p.w = static_cast<const uint16_t*>(ws.p), p.ldw = ws.ld;
    p.w2 = static_cast<const uint16_t*>(w2s.p), p.ldw2 = w2s.ld;
    // zeros past K where K is not a multiple of 8: the contraction runs over them
    p.K = p.ka = (int)(skinny ? K : round_up(K, 8));
    p.M = (int)M, p.N = (int)N, p.nk = p.nk1 = (int)(round_up(K, 64) / 64);
    p.alim = (int)M, p.wlim = (int)N, p.problems = 1, p.part = part, p.width = (int)(w2.p ? 2 * N : N);
    return p;
  }
};

}  // namespace dc

using namespace dc;

extern "C" size_t dc_saved16_bytes(int64_t M, int64_t N) { return M > 0 && N > 0 ? saved16_bytes(M, N) : 0; }

extern "C" size_t dc_linear16_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M,
                                              int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || check_product("dc_linear16", DC_F16, DC_ACT_NONE, M, N, K)) return 0;
  return Forward16({x, ldx, M, K}, {w, ldw, N, K}, {}, M, N, K, nullptr).bytes;
}

extern "C" int dc_linear16(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype,
                           const void* res, int64_t ldr, int act, void* out, int64_t ldo, void* z, int dtype,
                           int64_t M, int64_t N, int64_t K, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  const char* who = "dc_linear16";
  if (int e = check_product(who, dtype, act, M, N, K)) return e;
  if (M == 0 || N == 0) return DC_OK;
  if (!x || !w || !out) return refuse(DC_EINVAL, who, "null pointer");
  if (bias && bias_dtype != dtype && bias_dtype != DC_F32)
    return refuse(DC_EINVAL, who, "bias_dtype must be dtype or DC_F32");
  if (ldx < K || ldw < K || ldo < N || (res && ldr < N))
    return refuse(DC_EINVAL, who, "row stride less than the row");
  const Forward16 f({x, ldx, M, K}, {w, ldw, N, K}, {}, M, N, K, ws);
  if (int e = check_scratch(who, f.bytes, ws, ws_bytes)) return e;
  hipStream_t st = (hipStream_t)stream;
  if (int e = f.pad(who, st)) return e;
  Gemm16 p = f.args(M, N, K);
  p.bias = bias, p.bias_dtype = bias_dtype, p.act = act, p.res = static_cast<const uint16_t*>(res), p.ldr = ldr;
  p.out = static_cast<uint16_t*>(out), p.ldo = ldo, p.z = static_cast<uint8_t*>(z);
  if (f.skinny) return run_skinny16(who, p, dtype, st);
  return dtype == DC_BF16 ? run_tile16<DC_BF16, false, false, EPI_LINEAR>(who, p, f.plan, st)
                          : run_tile16<DC_F16, false, false, EPI_LINEAR>(who, p, f.plan, st);
}

extern "C" size_t dc_gated16_workspace_bytes(const void* x, int64_t ldx, const void* wv, int64_t ldwv, const void* wg,
                                             int64_t ldwg, int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || !wg || check_product("dc_gated16", DC_F16, DC_ACT_NONE, M, N, K)) return 0;
  return Forward16({x, ldx, M, K}, {wv, ldwv, N, K}, {wg, ldwg, N, K}, M, N, K, nullptr).bytes;
}

extern "C" int dc_gated16(const void* x, int64_t ldx, const void* wv, int64_t ldwv, const void* wg, int64_t ldwg,
                          const void* bv, const void* bg, int bias_dtype, int act, void* out, int64_t ldo, void* zv,
                          void* zg, int dtype, int64_t M, int64_t N, int64_t K, void* ws,
                          size_t ws_bytes, void* stream) {
  clear_error();
  const char* who = "dc_gated16";
  if (int e = check_product(who, dtype, act, M, N, K)) return e;
  if (M == 0 || N == 0) return DC_OK;
  if (!x || !wv || !wg || !out) return refuse(DC_EINVAL, who, "null pointer");
  if ((bv || bg) && bias_dtype != dtype && bias_dtype != DC_F32)
    return refuse(DC_EINVAL, who, "bias_dtype must be dtype or DC_F32");
  if (!zv != !zg) return refuse(DC_EINVAL, who, "zv and zg go together");
  if (ldx < K || ldwv < K || ldwg < K || ldo < N)
    return refuse(DC_EINVAL, who, "row stride less than the row");
  const Forward16 f({x, ldx, M, K}, {wv, ldwv, N, K}, {wg, ldwg, N, K}, M, N, K, ws);
  if (int e = check_scratch(who, f.bytes, ws, ws_bytes)) return e;
  hipStream_t st = (hipStream_t)stream;
  if (int e = f.pad(who, st)) return e;
  Gemm16 p = f.args(M, N, K);
  p.bias = bv, p.bias2 = bg, p.bias_dtype = bias_dtype, p.act = act;
  p.out = static_cast<uint16_t*>(out), p.ldo = ldo, p.z = static_cast<uint8_t*>(zv), p.z2 = static_cast<uint8_t*>(zg);
  if (f.skinny) return run_skinny16(who, p, dtype, st);
  return dtype == DC_BF16 ? run_tile16<DC_BF16, false, false, EPI_GATED>(who, p, f.plan, st)
                          : run_tile16<DC_F16, false, false, EPI_GATED>(who, p, f.plan, st);
}
