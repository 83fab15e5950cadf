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

// Pairwise sum over 16 lanes (a DPP row) or all of a wave, neighbours first, in every lane of them.
LSK_DEV float row_tree(float v) {
  auto add = [&](int o) { v = f32_add(v, __int_as_float(o)); };
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xb1, 0xf, 0xf, false));   // quad [1,0,3,2]
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4e, 0xf, 0xf, false));   // quad [2,3,0,1]
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, false));  // half-row mirror
  add(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, false));  // row mirror
  return v;
}

LSK_DEV float wave_tree(float v) {
  v = row_tree(v);
  auto row = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
  return f32_add(f32_add(row(0), row(16)), f32_add(row(32), row(48)));
}

// A wave's groups first .. first + 63 of kWords / 2 times eight bytes each, those before G, to o + their bytes: through its
// part of LDS, so that each store of eight bytes a lane fills whole lines.  (Stores past the caches at a lane's own
// bytes fill parts of lines: 8192 rows of 4096 in binary32 113 -> 77 us on MI355X, in 16 bits level.)
template <int kWords>
LSK_DEV void store_groups(void* o, int first, int G, const uint32_t (&w)[kWords], char* strip) {
  constexpr int kParts = kWords / 2;
  const int lane = threadIdx.x & 63;
  uint64_t* const mine = (uint64_t*)strip + kParts * lane;
#pragma unroll
  for (int t = 0; t < kParts; ++t) mine[t] = (uint64_t)w[2 * t + 1] << 32 | w[2 * t];
  wave_lds_fence();
#pragma unroll
  for (int t = 0; t < kParts; ++t) {
    const int u = 64 * t + lane;
    if (first + u / kParts < G) __builtin_nontemporal_store(((const uint64_t*)strip)[u], (uint64_t*)o + kParts * first + u);
    __asm__ volatile("" ::: "memory");  // (no 16-byte stores: store16_split)
  }
  wave_lds_fence();
}

// Eight values of type DT as they lie in memory.
template <int DT>
LSK_DEV void words_of(const float (&v)[8], uint32_t (&w)[DT == LSK_F32 ? 8 : 4], bool nan) {
#pragma unroll
  for (int t = 0; t < (DT == LSK_F32 ? 8 : 4); ++t) {
    if constexpr (DT == LSK_F32) w[t] = __float_as_uint(v[t]);
    else if constexpr (DT == LSK_BF16)
      w[t] = nan ? pack_bf16x2(v[2 * t], v[2 * t + 1]) : pack_bf16x2_nonan(v[2 * t], v[2 * t + 1]);
    else
      w[t] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * t]) |
             (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * t + 1]) << 16;
  }
}

template <int DT, bool VEC, int C>
__global__ __launch_bounds__(1024) void add_rmsnorm_fp8_kernel(NormFp8Args p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float red[16];
  const int lane = threadIdx.x & 63, wave = wave_id(), W = blockDim.x >> 6;
  const int64_t m = blockIdx.x;
  const int G = p.N / 8, g0 = wave * C * 64 + lane;
  char* const strip = smem + wave * 64 * (DT == LSK_F32 ? 32 : 16);
  // f(the gain's type, a compile-time value)
  auto with_gain = [&](auto f) {
    if (p.g_dtype == LSK_F32) f(std::integral_constant<int, LSK_F32>{});
    else if (p.g_dtype == LSK_BF16) f(std::integral_constant<int, LSK_BF16>{});
    else f(std::integral_constant<int, LSK_F16>{});
  };
  constexpr bool kEarly = C <= 4;  // (eight groups' residuals and gains beside the values would not fit the registers)
  constexpr int kE = kEarly ? C : 1;
  constexpr int kWords = DT == LSK_F32 ? 8 : 4;  // of a group in x's type
  float v[C][8], y[8];
  uint32_t gw[kE][8] = {};  // gains as they lie in memory
  Raw8<DT, VEC> x[kE], r[kE];
  auto load = [&](int c, int e) {
    const bool in = g0 + 64 * c < G;
    x[e] = raw8<DT, VEC>(p.x, m * p.ldx + 8 * (g0 + 64 * c), in);
    r[e] = raw8<DT, VEC>(p.r ? p.r : p.x, m * p.ldr + 8 * (g0 + 64 * c), in && p.r);
  };
  auto load_gain = [&](int c, int e) {
    const bool in = g0 + 64 * c < G, wide = p.g_dtype == LSK_F32;
    const int i = in ? 8 * (g0 + 64 * c) : 0;
    if constexpr (VEC) {  // (without a branch; 16-bit gains twice)
      const v4u32* const at = (const v4u32*)((const char*)p.g + i * (wide ? 4 : 2));
      const v4u32 lo = at[0], hi = at[wide ? 1 : 0];
#pragma unroll
      for (int t = 0; t < 4; ++t) gw[e][t] = in ? lo[t] : 0, gw[e][4 + t] = in ? hi[t] : 0;
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t)
        gw[e][t] = !in ? 0 : wide ? ((const uint32_t*)p.g)[i + t] : ((const uint16_t*)p.g)[i + t];
    }
  };
  if constexpr (kEarly) {
#pragma unroll
    for (int c = 0; c < C; ++c) load(c, c);
#pragma unroll
    for (int c = 0; c < C; ++c) load_gain(c, c);
    __asm__ volatile("" ::: "memory");  // (the residual's loads stay ahead of the branch that uses them)
  }
  float S[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int e = kEarly ? c : 0;
    if constexpr (!kEarly) load(c, e);
    raw8_values(x[e], v[c]);
    auto square = [&] {
      float s = f32_mul(v[c][0], v[c][0]);
#pragma unroll
      for (int t = 1; t < 8; ++t) s = f32_add(s, f32_mul(v[c][t], v[c][t]));
      return s;
    };
    float s;
    uint32_t w[kWords];
    if (p.r) {  // (uniform)
      raw8_values(r[e], y);
#pragma unroll
      for (int t = 0; t < 8; ++t) y[t] = f32_add(v[c][t], y[t]);
      auto rounded = [&](bool nan) {
        words_of<DT>(y, w, nan);
        Raw8<DT, true> h;
#pragma unroll
        for (int t = 0; t < kWords; ++t) h.w[t] = w[t];
        raw8_values(h, v[c]);
      };
      rounded(false);
      s = square();
      if (DT == LSK_BF16 && __builtin_amdgcn_ballot_w64(s != s)) rounded(true);  // (a NaN makes the sum one)
    } else {
      if (p.h) words_of<DT>(v[c], w, true);
      s = square();
    }
    if (p.h) store_groups((char*)p.h + m * p.ldh * (DT == LSK_F32 ? 4 : 2), g0 - lane + 64 * c, G, w, strip);
    S[c] = g0 + 64 * c < G ? s : -0.0f;
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
    sum = row_tree((lane & 15) < W ? red[lane & 15] : -0.0f);
  }
  if (p.ne != 0.0f) sum = f32_add(sum, p.ne);
  sum = sum < 0x1p-126f ? 0x1p-126f : sum;  // (a NaN stays)
  const float rs = f32_div(p.sN, __builtin_sqrtf(sum));
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int grp = g0 + 64 * c;
    const int e = kEarly ? c : 0;
    if constexpr (!kEarly) load_gain(c, e);
    // (beside a row's end v and the gain are 0, and so is y, unless the sum is a NaN, when all of the row's are)
    with_gain([&](auto gdt) {
      Raw8<decltype(gdt)::value, VEC> raw;
#pragma unroll
      for (int t = 0; t < decltype(raw)::kWords; ++t) raw.w[t] = gw[e][t];
      raw8_values(raw, y);
    });
#pragma unroll
    for (int t = 0; t < 8; ++t) y[t] = f32_mul(f32_mul(v[c][t], rs), y[t]);
    float s;
    const uint2 code = quantize_row_fp8(y, s);
    if (grp < G) {
      *(uint2*)(p.q + m * p.N + 8 * grp) = code;
      if ((lane & 15) == 0) p.scale[m * p.sm + (grp >> 4) * p.sb] = s;
    }
    if (p.out) {
      const float any = ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));  // (a NaN where one of them is)
      uint32_t w[4];
      words_of<LSK_BF16>(y, w, __builtin_amdgcn_ballot_w64(any != any) != 0);
      store_groups((uint16_t*)p.out + m * p.N, grp - lane, G, w, strip);
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
  const int size = x_dtype == LSK_F32 ? 4 : 2;
  auto even = [&](const void* a, int64_t ld) { return !a || ((uintptr_t)a % 16 == 0 && (R == 1 || ld * size % 16 == 0)); };
  LSK_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && even(h, ldh),
              "lsk_add_rmsnorm_fp8: codes, out and h must be 16-byte aligned, h's rows too");
  // One group a lane while 16 waves hold the row, two for long 16-bit rows enough to fill the machine (MI355X, bf16, 1, 2, 4
  // and 8 groups a lane: 8192 rows of 4096 49.0, 46.2, 48.8, 58.5 us, of 3584 44.0, 41.7, 44.3, 56.6, 512 of 4096 5.1, 5.5,
  // 7.3, 11.3, 32 of them 3.9, 4.5, 5.8, 10.1, 16384 of 1024 21.8, 22.2, 27.0, 46.9; f32, 8192 of 4096 76.8, 77.7, 81.3, 95.4;
  // 235 MB in 46.2 us are 5.1 TB/s, what a large copy reaches).
  int64_t P = 64;
  while (P < N / 8) P *= 2;
  int C = size == 2 && R >= 2048 && N >= 2048 ? 2 : 1;
  while (P / 64 > 16 * C) C *= 2;
  const int W = (int)(P / 64 / C);
  LSK_REQUIRE(R <= 0x7fffffff && grid_ok(R, 64 * W), "lsk_add_rmsnorm_fp8: grid too large");
  lsk::NormFp8Args p{x, residual, ldx, ldr, R, (int)N, g, g_dtype, sN, 0.0f, h, ldh, q, scale, scale_m, scale_b, out};
  if (!(sN > 0.0f)) p.sN = (float)__builtin_sqrt((double)N);  // the width constant fl32(sqrt(N))
  p.ne = (float)((double)N * eps);  // one binary64 product, one rounding
  const bool vec = even(x, ldx) && even(residual, ldr) && (uintptr_t)g % 16 == 0;
  auto run = [&](auto dt, auto v, auto c) {
    hipLaunchKernelGGL((lsk::add_rmsnorm_fp8_kernel<decltype(dt)::value, decltype(v)::value, decltype(c)::value>),
                       dim3((unsigned)R), dim3(64 * W), (size_t)(64 * W * 8 * size), (hipStream_t)stream, p);
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
