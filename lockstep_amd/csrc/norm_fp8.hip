// The residual's addition, the contract's float RMS norm and fp8 rows of its output, in one kernel.
//
//   h = T(x + r)                       the residual stream, rounded once to x's type (h = x without r)
//   rs = sN / sqrt(max(S + ne, 2^-126))   S the sum of h^2 by the pinned tree of the float norm (norm.hip)
//   y = fl32(fl32(h * rs) * g)         in binary32: what rmsnorm_float rounds to bf16
//   (q, s) = fp8 rows of y             quantised from binary32, not from a rounded copy (fp8_quant.h)
//
// A row is W waves of 64 lanes; lane l of wave w holds groups of eight (w C + c) 64 + l, c < C, so a wave's
// loads and stores are contiguous and 16 lanes (a DPP row) hold 128 values, one block of scales.  The tree
// pairs neighbouring groups first, so it runs over the lanes' bits, then c, then w; groups past the row are
// -0, which changes no sum.  Bound by HBM: x and r read, h, codes and scales written.
#include <type_traits>

#include "fp8_quant.h"
#include "lsk_common.h"
#include "row_tiles.h"

namespace lsk {

struct NormFp8Args {
  const void* x;
  const void* r;  // or null
  int64_t ldx, ldr, R;
  int N;
  const void* g;  // [N]
  int g_dtype;
  float sN, ne;
  void* h;  // [R, N] or null, row stride ldh
  int64_t ldh;
  uint8_t* q;  // [R, N]
  float* scale;
  int64_t sm, sb;
  void* out;  // [R, N] bf16 or null
};

// Pairwise sum over the lanes of a wave, neighbours first, in every lane.
LSK_DEV float wave_tree(float v) {
  auto add = [&](int o) { v = f32_add(v, __int_as_float(o)); };
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xb1, 0xf, 0xf, false));   // quad [1,0,3,2]
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4e, 0xf, 0xf, false));   // quad [2,3,0,1]
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, false));  // half-row mirror
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, false));  // row mirror
  auto row = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
  return f32_add(f32_add(row(0), row(16)), f32_add(row(32), row(48)));
}

template <int DT, bool VEC>
LSK_DEV void store8(void* o, int64_t i, const float (&v)[8]) {
  if constexpr (VEC) {
    store_eight((char*)o + i * (DT == LSK_F32 ? 4 : 2), DT, v);
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      store_out(o, DT, i + t, v[t]);
      __asm__ volatile("" ::: "memory");  // (no 16-byte stores: store16_split)
    }
  }
}

template <int DT, bool VEC, int C>
__global__ __launch_bounds__(1024) void add_rmsnorm_fp8_kernel(NormFp8Args p) {
  __shared__ float red[16];
  const int lane = threadIdx.x & 63, wave = wave_id(), W = blockDim.x >> 6;
  const int64_t m = blockIdx.x;
  const int G = p.N / 8, g0 = wave * C * 64 + lane;
  // (one switch on the gain's type for all of a lane's loads)
  auto gain = [&](auto& g, int first) {
    auto load = [&](auto gdt) {
#pragma unroll
      for (int c = 0; c < (int)(sizeof(g) / sizeof(g[0])); ++c)
        if (g0 + 64 * (first + c) < G) load8<decltype(gdt)::value, VEC>(p.g, 8 * (g0 + 64 * (first + c)), g[c]);
    };
    if (p.g_dtype == LSK_F32) load(std::integral_constant<int, LSK_F32>{});
    else if (p.g_dtype == LSK_BF16) load(std::integral_constant<int, LSK_BF16>{});
    else load(std::integral_constant<int, LSK_F16>{});
  };
  constexpr bool kEarly = C <= 4;  // (eight groups' residuals and gains beside the values would not fit the registers)
  constexpr int kE = kEarly ? C : 1;
  float v[C][8], r[kE][8], g[kE][8];
  auto residual = [&](int c, float (&w)[8]) {
#pragma unroll
    for (int t = 0; t < 8; ++t) w[t] = 0.0f;
    if (p.r && g0 + 64 * c < G) load8<DT, VEC>(p.r, m * p.ldr + 8 * (g0 + 64 * c), w);
  };
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int t = 0; t < 8; ++t) v[c][t] = 0.0f;
    if (g0 + 64 * c < G) load8<DT, VEC>(p.x, m * p.ldx + 8 * (g0 + 64 * c), v[c]);
    if constexpr (kEarly) residual(c, r[c]);
  }
  if constexpr (kEarly) gain(g, 0);
  float S[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if constexpr (!kEarly) residual(c, r[0]);
    if (p.r)
#pragma unroll
      for (int t = 0; t < 8; ++t) v[c][t] = round_out(DT, f32_add(v[c][t], r[kEarly ? c : 0][t]));
    float s = f32_mul(v[c][0], v[c][0]);
#pragma unroll
    for (int t = 1; t < 8; ++t) s = f32_add(s, f32_mul(v[c][t], v[c][t]));
    S[c] = g0 + 64 * c < G ? s : -0.0f;
    if (p.h && g0 + 64 * c < G) store8<DT, VEC>(p.h, m * p.ldh + 8 * (g0 + 64 * c), v[c]);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) S[c] = wave_tree(S[c]);
#pragma unroll
  for (int h = 1; h < C; h *= 2)
#pragma unroll
    for (int c = 0; c < C; c += 2 * h) S[c] = f32_add(S[c], S[c + h]);
  float sum = S[0];
  if (W > 1) {
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = i < W ? red[i] : -0.0f;
#pragma unroll
    for (int h = 1; h < 16; h *= 2)
#pragma unroll
      for (int i = 0; i < 16; i += 2 * h) w[i] = f32_add(w[i], w[i + h]);
    sum = w[0];
  }
  if (p.ne != 0.0f) sum = f32_add(sum, p.ne);
  sum = sum < 0x1p-126f ? 0x1p-126f : sum;  // (a NaN stays)
  const float rs = f32_div(p.sN, __builtin_sqrtf(sum));
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int grp = g0 + 64 * c;
    if constexpr (!kEarly) gain(g, c);
    float y[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      y[t] = f32_mul(f32_mul(v[c][t], rs), g[kEarly ? c : 0][t]);
      if (grp >= G) y[t] = 0.0f;  // (beside a row's end: not to weigh in the block's maximum, a NaN sum's NaNs among them)
    }
    float s;
    const uint2 code = quantize_row_fp8(y, s);
    if (grp < G) {
      *(uint2*)(p.q + m * p.N + 8 * grp) = code;
      if ((lane & 15) == 0) p.scale[m * p.sm + (grp >> 4) * p.sb] = s;
      if (p.out) store8<LSK_BF16, true>(p.out, m * p.N + 8 * grp, y);
    }
  }
}

}  // namespace lsk

extern "C" int lsk_add_rmsnorm_fp8(const void* x, int x_dtype, int64_t ldx, const void* residual, int64_t ldr, int64_t R,
                                   int64_t N, const void* g, int g_dtype, float sN, double eps, void* h, int64_t ldh,
                                   uint8_t* q, float* scale, int64_t scale_m, int64_t scale_b, void* out, void* stream) {
  LSK_REQUIRE(lsk::is_float_dtype(x_dtype), "lsk_add_rmsnorm_fp8: x_dtype must be f32, bf16 or f16");
  LSK_REQUIRE(lsk::is_float_dtype(g_dtype), "lsk_add_rmsnorm_fp8: the gain must be f32, bf16 or f16");
  LSK_REQUIRE(R >= 0 && N >= 0 && N % 16 == 0 && N <= 65536, "lsk_add_rmsnorm_fp8: R=%lld, N=%lld (N a multiple of 16 up to 65536)",
              (long long)R, (long long)N);
  if (R == 0 || N == 0) return LSK_OK;
  LSK_REQUIRE(x && g && q && scale, "lsk_add_rmsnorm_fp8: null pointer");
  LSK_REQUIRE(R == 1 || (ldx >= N && (!residual || ldr >= N) && (!h || ldh >= N)), "lsk_add_rmsnorm_fp8: leading dimension below N");
  LSK_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0, "lsk_add_rmsnorm_fp8: codes and out must be 16-byte aligned");
  // One group a lane while 16 waves hold the row (MI355X, 1, 2, 4 and 8 groups a lane: 8192 rows of 4096 53.6, 58.5, 63.5,
  // 64.3 us, 512 of them 6.6, 7.3, 10.4, 15.3, 16384 of 1024 27.3, 28.3, 28.2, 28.4; 235 MB in 53.6 us are 4.4 TB/s, a
  // large copy reaches 5.0).
  int64_t P = 64;
  while (P < N / 8) P *= 2;
  int C = 1;
  while (P / 64 > 16 * C) C *= 2;
  const int W = (int)(P / 64 / C);
  LSK_REQUIRE(R <= 0x7fffffff && grid_ok(R, 64 * W), "lsk_add_rmsnorm_fp8: grid too large");
  lsk::NormFp8Args p{x, residual, ldx, ldr, R, (int)N, g, g_dtype, sN, 0.0f, h, ldh, q, scale, scale_m, scale_b, out};
  if (!(sN > 0.0f)) p.sN = (float)__builtin_sqrt((double)N);  // the width constant fl32(sqrt(N))
  p.ne = (float)((double)N * eps);  // one binary64 product, one rounding
  const int size = x_dtype == LSK_F32 ? 4 : 2;
  auto even = [&](const void* a, int64_t ld) { return !a || ((uintptr_t)a % 16 == 0 && (R == 1 || ld * size % 16 == 0)); };
  const bool vec = even(x, ldx) && even(residual, ldr) && even(h, ldh) && (uintptr_t)g % 16 == 0;
  auto run = [&](auto dt, auto v, auto c) {
    hipLaunchKernelGGL((lsk::add_rmsnorm_fp8_kernel<decltype(dt)::value, decltype(v)::value, decltype(c)::value>),
                       dim3((unsigned)R), dim3(64 * W), 0, (hipStream_t)stream, p);
  };
  auto with_c = [&](auto dt, auto v) {
    if (C == 1) run(dt, v, std::integral_constant<int, 1>{});
    else if (C == 2) run(dt, v, std::integral_constant<int, 2>{});
    else if (C == 4) run(dt, v, std::integral_constant<int, 4>{});
    else run(dt, v, std::integral_constant<int, 8>{});
  };
  auto with_dt = [&](auto dt) { vec ? with_c(dt, std::true_type{}) : with_c(dt, std::false_type{}); };
  if (x_dtype == LSK_F32) with_dt(std::integral_constant<int, LSK_F32>{});
  else if (x_dtype == LSK_BF16) with_dt(std::integral_constant<int, LSK_BF16>{});
  else with_dt(std::integral_constant<int, LSK_F16>{});
  return lsk::check_launch("add_rmsnorm_fp8_kernel");
}
