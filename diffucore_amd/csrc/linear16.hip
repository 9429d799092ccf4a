// 16-bit products of the feed-forward operators on bf16 / fp16 MFMA (gfx950):
//   forward   y = act(x w^T + b) + res, and h = (x wv^T + bv) act(x wg^T + bg)
//   backward  dx = dz w (+ dz2 w2), dw = dz^T x
//
// All three are C[m, n] = sum over k of A(m, k) W(n, k) with operands read at
// (row stride, k stride): the forward's are contiguous along k, dx reads w and
// dw both operands contiguous along the rows. Sums are float32.
//
// One kernel: 64 (n) x 64 (m) tiles, 32 of k at a time through LDS, 2 waves of
// 64 (n) x 32 (m) on v_mfma_f32_32x32x16. C^T layout: a lane's accumulators
// belong to one m and 4 consecutive n per register quad. A gated tile holds 32
// channels: its first MFMA block is their value rows, its second their gate
// rows, so value and gate of an output meet in one lane.
#include "colsum.h"

namespace dc {

struct Gemm16 {
  const uint16_t *a, *a2;       // a2, w2: the second term (dx2) or the second problem (dw2)
  const uint16_t *w, *w2;       // gated: value and gate weights
  int64_t ars, aks, wrs, wks;   // row and k strides
  int64_t w2rs;
  int M, N, K;
  int K1;                       // k where the second term starts (== K: one term)
  int Kr;                       // k of a term that its operands have
  const void *bias, *bias2;
  int bias_dtype, act;
  const uint16_t* res;
  uint16_t *out, *out2;
  float *z, *z2;
  int64_t ldr, ldo, ldz;
  int gated;
};

__device__ __forceinline__ float bias_at(const void* b, int dtype, int n) {
  if (!b) return 0.0f;
  if (dtype == DC_F32) return static_cast<const float*>(b)[n];
  const uint32_t u = static_cast<const uint16_t*>(b)[n];
  return dtype == DC_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
}

template <int DT>
__device__ __forceinline__ v16f mfma16(uint4 w, uint4 a, v16f c) {
  if constexpr (DT == DC_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, a), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, a), c, 0, 0, 0);
}

template <int DT>
__global__ void __launch_bounds__(128) linear16_kernel(Gemm16 p) {
  constexpr int KB = 32, P = KB + 8;
  __shared__ __attribute__((aligned(16))) uint16_t lw[64 * P], la[64 * P];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, l32 = lane & 31, hf = lane >> 5;
  const int BN = p.gated ? 32 : 64;
  const int n0 = blockIdx.x * BN, m0 = blockIdx.y * 64;
  const uint16_t* a = p.a;
  uint16_t* out = p.out;
  if (blockIdx.z) a = p.a2, out = p.out2;
  v16f acc[2] = {v16f{0}, v16f{0}};
  for (int k0 = 0; k0 < p.K; k0 += KB) {
    const bool second = k0 >= p.K1;   // K1 is a multiple of 32
    const int kk = second ? k0 - p.K1 : k0, kn = p.Kr;
    const uint16_t* as = second ? p.a2 : a;
    for (int i = t; i < 64 * KB; i += 128) {
      const int r = p.aks == 1 ? i / KB : i % 64, k = p.aks == 1 ? i % KB : i / 64;
      la[r * P + k] = m0 + r < p.M && kk + k < kn ? as[(m0 + r) * p.ars + (kk + k) * p.aks] : 0;
    }
    for (int i = t; i < 64 * KB; i += 128) {
      const int r = p.wks == 1 ? i / KB : i % 64, k = p.wks == 1 ? i % KB : i / 64;
      const bool two = p.gated ? r >= 32 : second;
      const int n = n0 + (p.gated ? r % 32 : r);
      const uint16_t* ws = two ? p.w2 : p.w;
      const int64_t rs = two ? p.w2rs : p.wrs;
      const int64_t at = p.wks == 1 ? n * rs + kk + k : n + (kk + k) * (two ? p.w2rs : p.wks);
      lw[r * P + k] = n < p.N && kk + k < kn ? ws[at] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < KB / 16; ++ks) {
      const uint4 af = *reinterpret_cast<const uint4*>(la + (32 * wv + l32) * P + 16 * ks + 8 * hf);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 wf = *reinterpret_cast<const uint4*>(lw + (32 * i + l32) * P + 16 * ks + 8 * hf);
        acc[i] = mfma16<DT>(wf, af, acc[i]);
      }
    }
    __syncthreads();
  }
  const int m = m0 + 32 * wv + l32;
  if (m >= p.M) return;
  with_act(p.act, [&](auto act_) {
    constexpr int ACT = decltype(act_)::value;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int nl = 8 * (r / 4) + 4 * hf + r % 4;
      if (p.gated) {
        const int n = n0 + nl;
        if (n >= p.N) continue;
        const float v = acc[0][r] + bias_at(p.bias, p.bias_dtype, n), g = acc[1][r] + bias_at(p.bias2, p.bias_dtype, n);
        if (p.z) {
          p.z[m * p.ldz + n] = v;
          p.z2[m * p.ldz + n] = g;
        }
        out[m * p.ldo + n] = (uint16_t)f32_to_h16<DT>(v * act_value<ACT>(g));
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = n0 + 32 * i + nl;
          if (n >= p.N) continue;
          const float v = acc[i][r] + bias_at(p.bias, p.bias_dtype, n);
          if (p.z) p.z[m * p.ldz + n] = v;
          float y = act_value<ACT>(v);
          if (p.res) y += h16_to_f32<DT>(p.res[m * p.ldr + n]);
          out[m * p.ldo + n] = (uint16_t)f32_to_h16<DT>(y);
        }
      }
    }
  });
}

static int run_linear16(const char* who, const Gemm16& p, int dtype, int problems, hipStream_t st) {
  const int bn = p.gated ? 32 : 64;
  const dim3 grid((unsigned)((p.N + bn - 1) / bn), (unsigned)((p.M + 63) / 64), problems);
  if (grid.y > 65535) return fail(DC_EINVAL, "linear16: too many rows");
  if (dtype == DC_BF16) hipLaunchKernelGGL((linear16_kernel<DC_BF16>), grid, dim3(128), 0, st, p);
  else hipLaunchKernelGGL((linear16_kernel<DC_F16>), grid, dim3(128), 0, st, p);
  return launch_status(who);
}

static int refuse(int code, const char* who, const char* msg) {
  set_error("%s: %s", who, msg);
  return code;
}

static bool plain_act(int act) {
  return act == DC_ACT_NONE || act == DC_ACT_GELU_ERF || act == DC_ACT_GELU_TANH || act == DC_ACT_SILU ||
         act == DC_ACT_QUICK_GELU;
}

// Sizes and types every product checks.
static int check_product(const char* who, int dtype, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return refuse(DC_EINVAL, who, "negative size");
  if (M > 0x3fffffff || N > 0x3fffffff || K > 0x3fffffff) return refuse(DC_EINVAL, who, "size too large");
  if (dtype != DC_F16 && dtype != DC_BF16) return refuse(DC_EINVAL, who, "dtype must be DC_F16 or DC_BF16");
  return DC_OK;
}

static int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// A product's operand: `width` contiguous values a row.
static bool bad_operand(const void* p, int64_t ld, int64_t width) {
  return !aligned16(p) || ld % 8 || width % 8 || ld < width;
}

}  // namespace dc

using namespace dc;

extern "C" size_t dc_linear16_workspace_bytes(int, int64_t, int64_t, int64_t) { return 0; }

extern "C" int dc_linear16(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype,
                           const void* res, int64_t ldr, int act, void* out, int64_t ldo, float* z, int64_t ldz,
                           int dtype, int64_t M, int64_t N, int64_t K, void*, size_t, void* stream) {
  clear_error();
  const char* who = "dc_linear16";
  if (int e = check_product(who, dtype, M, N, K)) return e;
  if (!plain_act(act)) return refuse(DC_EINVAL, who, "bad act");
  if (M == 0 || N == 0) return DC_OK;
  if (K == 0) return refuse(DC_EINVAL, who, "K must be positive");
  if (!x || !w || !out) return refuse(DC_EINVAL, who, "null pointer");
  if (bias && !float_dtype(bias_dtype)) return refuse(DC_EINVAL, who, "bad bias_dtype");
  if (ldo < N || (res && ldr < N) || (z && ldz < N)) return refuse(DC_EINVAL, who, "row stride < N");
  if (bad_operand(x, ldx, K) || bad_operand(w, ldw, K))
    return refuse(DC_EUNSUPPORTED, who, "needs K, ldx, ldw multiples of 8 and 16-byte aligned x, w");
  Gemm16 p{};
  p.a = static_cast<const uint16_t*>(x), p.ars = ldx, p.aks = 1;
  p.w = static_cast<const uint16_t*>(w), p.wrs = ldw, p.wks = 1;
  p.M = (int)M, p.N = (int)N, p.K = p.K1 = p.Kr = (int)K;
  p.bias = bias, p.bias_dtype = bias_dtype, p.act = act, p.res = static_cast<const uint16_t*>(res), p.ldr = ldr;
  p.out = static_cast<uint16_t*>(out), p.ldo = ldo, p.z = z, p.ldz = ldz;
  return run_linear16(who, p, dtype, 1, (hipStream_t)stream);
}

extern "C" int dc_gated16(const void* x, int64_t ldx, const void* wv, int64_t ldwv, const void* wg, int64_t ldwg,
                          const void* bv, const void* bg, int bias_dtype, int act, void* out, int64_t ldo, float* zv,
                          float* zg, int64_t ldz, int dtype, int64_t M, int64_t N, int64_t K, void*, size_t,
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
  if (bad_operand(x, ldx, K) || bad_operand(wv, ldwv, K) || bad_operand(wg, ldwg, K))
    return refuse(DC_EUNSUPPORTED, who, "needs K and row strides multiples of 8 and 16-byte aligned x, wv, wg");
  Gemm16 p{};
  p.a = static_cast<const uint16_t*>(x), p.ars = ldx, p.aks = 1;
  p.w = static_cast<const uint16_t*>(wv), p.wrs = ldwv, p.wks = 1;
  p.w2 = static_cast<const uint16_t*>(wg), p.w2rs = ldwg, p.gated = 1;
  p.M = (int)M, p.N = (int)N, p.K = p.K1 = p.Kr = (int)K;
  p.bias = bv, p.bias2 = bg, p.bias_dtype = bias_dtype, p.act = act;
  p.out = static_cast<uint16_t*>(out), p.ldo = ldo;
  p.z = zv, p.z2 = zg, p.ldz = ldz;
  return run_linear16(who, p, dtype, 1, (hipStream_t)stream);
}

extern "C" int dc_linear16_dx(const void* dz, int64_t lddz, const void* w, int64_t ldw, const void* dz2,
                              const void* w2, int64_t ldw2, void* dx, int64_t lddx, int dtype,
                              int64_t M, int64_t N, int64_t K, void*, size_t, void* stream) {
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
  p.a = static_cast<const uint16_t*>(dz), p.ars = lddz, p.aks = 1;
  p.a2 = static_cast<const uint16_t*>(dz2);
  p.w = static_cast<const uint16_t*>(w), p.wks = ldw, p.wrs = 1;
  p.w2 = static_cast<const uint16_t*>(w2), p.w2rs = ldw2;
  p.M = (int)M, p.N = (int)K, p.K1 = dz2 ? (int)N64 : (int)N, p.K = dz2 ? (int)(N64 + N) : (int)N, p.Kr = (int)N;
  p.out = static_cast<uint16_t*>(dx), p.ldo = lddx;
  return run_linear16(who, p, dtype, 1, (hipStream_t)stream);
}

extern "C" int dc_linear16_dw(const void* dz, int64_t lddz, const void* x, int64_t ldx, const void* dz2, void* dw,
                              int64_t lddw, void* dw2, int dtype, int64_t M, int64_t N, int64_t K, void*, size_t,
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
  p.a = static_cast<const uint16_t*>(dz), p.aks = lddz, p.ars = 1;
  p.a2 = static_cast<const uint16_t*>(dz2);
  p.w = static_cast<const uint16_t*>(x), p.wks = ldx, p.wrs = 1;
  p.M = (int)N, p.N = (int)K, p.K = p.K1 = p.Kr = (int)M;
  p.out = static_cast<uint16_t*>(dw), p.out2 = static_cast<uint16_t*>(dw2), p.ldo = lddw;
  return run_linear16(who, p, dtype, dz2 ? 2 : 1, (hipStream_t)stream);
}
