// Products of block-scaled fp8 (e4m3) rows and weights, their quantisers and the way back.
//
// With a binary32 scale per 128 values of an activation row and per 128 x 128 of a weight,
//   y[m, n] = sum_b sa[m, b] sw[n / 128, b] sum_{k in b} qa[m, k] qw[n, k]  (+ bias[n]).
// A block's inner sum comes from the matrix core (fp8_tile.h), starting from +0; the outer sum is one chain
// of FMAs over ascending b, acc = fma(inner, fl32(sa * sw), acc), in every kernel here, so a row's result is
// the same bits whatever the other rows are and however many.  Scales stay where they are: any strides for
// the rows', so that the quantiser can lay them block by block ([ceil(K / 128)][M]), which is what a tile's
// loads want.
#include <hip/hip_runtime.h>

#include "fp8_quant.h"
#include "fp8_tile.h"
#include "lsk_common.h"
#include "mfma_tile.h"
#include "row_tiles.h"

namespace lsk {

// ---------------------------------------------------------------- the quantisers
// 16 lanes per 128 values of a row (a lane holds eight), 16 of these to a thread block: `rows` rows of it by
// 16 / rows blocks, kQuantDeep times along K with their loads in flight together.  With 16 rows a block its
// scales are 64-byte runs of the block-by-block layout; few rows spread over K instead.  Bound by HBM.
constexpr int kQuantDeep = 4;
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_fp8_kernel(const void* __restrict__ x, int64_t ldx, int64_t M, int K,
                                                                int rows, uint8_t* __restrict__ q,
                                                                float* __restrict__ scale, int64_t sm, int64_t sb) {
  const int g = threadIdx.x >> 4, per = 16 / rows, step = per * kQuantDeep;
  const int nb = (K + 127) / 128, across = (nb + step - 1) / step;
  const int64_t rb = blockIdx.x / across, row = rb * rows + g % rows;
  const int b0 = (int)(blockIdx.x - rb * across) * step + g / rows, c = 8 * (threadIdx.x & 15);
  if (row >= M) return;  // (16 lanes alike, as everywhere below)
  float v[kQuantDeep][8];
#pragma unroll
  for (int z = 0; z < kQuantDeep; ++z) {
    const int k = 128 * (b0 + per * z) + c;
#pragma unroll
    for (int t = 0; t < 8; ++t) v[z][t] = 0.0f;
    if (k < K) load8<DT, VEC>(x, row * ldx + k, v[z]);
  }
#pragma unroll
  for (int z = 0; z < kQuantDeep; ++z) {
    const int b = b0 + per * z, k = 128 * b + c;
    if (b >= nb) break;
    float s;
    const uint2 w = quantize_row_fp8(v[z], s);
    if (k < K) *(uint2*)(q + row * K + k) = w;
    if (c == 0) scale[row * sm + b * sb] = s;
  }
}

static int64_t quantize_rows_blocks(int64_t M, int64_t K, int& rows) {
  rows = 16;
  while (rows > 1 && rows / 2 >= M) rows /= 2;
  const int64_t step = 16 / rows * kQuantDeep, nb = (K + 127) / 128;
  return (M + rows - 1) / rows * ((nb + step - 1) / step);
}

// (the caller has checked the grid)
static int quantize_rows_launch(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* q, float* scale,
                                int64_t sm, int64_t sb, hipStream_t s) {
  int rows;
  const dim3 grid((unsigned)quantize_rows_blocks(M, K, rows)), blk(256);
  by_input(x, x_dtype, ldx, [&](auto dt, auto vec) {
    hipLaunchKernelGGL((quantize_rows_fp8_kernel<decltype(dt)::value, decltype(vec)::value>), grid, blk, 0, s, x, ldx, M,
                       (int)K, rows, q, scale, sm, sb);
  });
  return check_launch("quantize_rows_fp8_kernel");
}

// A 128 x 128 block of a weight a thread block, 16 rows at a time, held in registers between its maximum and
// its codes.  Bound by HBM.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void quantize_weight_fp8_kernel(const void* __restrict__ x, int64_t ldx, int64_t N,
                                                                  int K, uint8_t* __restrict__ q,
                                                                  float* __restrict__ scale) {
  __shared__ uint32_t tops[4];
  const int nb = (K + 127) / 128;
  const int64_t rb = blockIdx.x / nb;
  const int b = (int)(blockIdx.x - rb * nb), k = 128 * b + 8 * (threadIdx.x & 15);
  const int64_t row0 = 128 * rb + (threadIdx.x >> 4);
  float v[8][8];
#pragma unroll
  for (int z = 0; z < 8; ++z) {
#pragma unroll
    for (int t = 0; t < 8; ++t) v[z][t] = 0.0f;
    if (k < K && row0 + 16 * z < N) load8<DT, VEC>(x, (row0 + 16 * z) * ldx + k, v[z]);
  }
  uint32_t top = 0;
#pragma unroll
  for (int z = 0; z < 8; ++z) {
    const uint32_t t = top8(v[z]);
    top = top > t ? top : t;
  }
  top = wave_max_u32(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) top = top > tops[w] ? top : tops[w];
  const Fp8Scale s = fp8_scale(top);
  if (threadIdx.x == 0) scale[blockIdx.x] = s.s;
#pragma unroll
  for (int z = 0; z < 8; ++z)
    if (k < K && row0 + 16 * z < N) *(uint2*)(q + (row0 + 16 * z) * K + k) = quantize8_fp8(v[z], s.inv);
}

// Codes times scales: eight values a thread, whole lines in and out.
template <int ODT>
__global__ __launch_bounds__(256) void dequant_fp8_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                          int64_t sm, int64_t sb, int row_shift, int64_t total, int K8,
                                                          void* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / K8;
    const int c = (int)(i - row * K8);
    const uint2 w = ((const uint2*)q)[i];
    const float s = scale[(row >> row_shift) * sm + (c >> 4) * sb];
    float v[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int u = (int)(h ? w.y : w.x);
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(u, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(u, true);
      v[4 * h] = f32_mul(a[0], s), v[4 * h + 1] = f32_mul(a[1], s);
      v[4 * h + 2] = f32_mul(b[0], s), v[4 * h + 3] = f32_mul(b[1], s);
    }
    if constexpr (ODT == LSK_F16) {
      // (the product is a binary32 number first: the compiler would round it to f16 in one instruction)
#pragma unroll
      for (int t = 0; t < 8; ++t) __asm__("" : "+v"(v[t]));
    }
    store_eight((char*)out + i * (ODT == LSK_F32 ? 32 : 16), ODT, v);
  }
}

// ---------------------------------------------------------------- the products
struct Fp8Args {
  const uint8_t* a;  // codes [M, K], row stride lda
  const float* sa;   // scales: element (m, b) at m * sm + b * sb
  const uint8_t* w;  // codes [N, K], row stride ldw
  const float* sw;   // scales [ceil(N / 128), ceil(K / 128)], row stride ldsw
  int64_t lda, sm, sb, ldw, ldsw;
  int64_t M, N;
  int K;
  const float* bias;  // [N] or null
  void* out;
  int out_dtype;
  int64_t ldo;
  // one projection of every expert: rows offs[e] .. offs[e + 1] - 1 through w_ptrs[e], ws_ptrs[e] and
  // b_ptrs[e] (or null)
  const int32_t* offs;  // [E + 1]
  int E;
  const int64_t* w_ptrs;
  const int64_t* ws_ptrs;
  const int64_t* b_ptrs;
};

// A BM x BN tile: tiles walk kGroupM row tiles down a column of weight tiles inside each XCD's run
// of them, so the row tiles that share a weight tile run together on one L2.
template <int BM, int BN, int WM, int WN, int RING, bool EXACT, bool GROUPED>
__global__ __launch_bounds__(WM * WN * 64) void fp8_tile_kernel(Fp8Args p, int64_t mtiles, int vec) {
  using C = Fp8Cfg<BM, BN, WM, WN, RING>;
  constexpr int kGroupM = 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int ntiles = (int)((p.N + BN - 1) / BN);
  // logical tile L: row tile mt, first weight row n0
  int mt, n0;
  auto place = [&](int L) {
    const int first = L / (kGroupM * ntiles) * kGroupM;
    const int gsize = (int)mtiles - first < kGroupM ? (int)mtiles - first : kGroupM;
    const int in = L - first * ntiles;
    mt = first + in % gsize;
    n0 = in / gsize * BN;
  };
  int m0, m1;
  if constexpr (GROUPED) {  // (the grid holds the most tiles there can be: the ones there are go to every XCD)
    ExpertTiles tiles(p.offs, p.E, (int)p.M, BM);
    mtiles = tiles.count();
    if (blockIdx.x >= mtiles * ntiles) return;
    place(xcd_logical_id(blockIdx.x, (int)mtiles * ntiles));
    int e;
    if (!tiles.find(mt, e, m0, m1)) return;
    p.w = (const uint8_t*)wave_uniform64(p.w_ptrs[e]);
    p.sw = (const float*)wave_uniform64(p.ws_ptrs[e]);
    p.bias = p.b_ptrs ? (const float*)wave_uniform64(p.b_ptrs[e]) : nullptr;
  } else {
    place(xcd_logical_id(blockIdx.x, (int)mtiles * ntiles));
    m0 = mt * BM, m1 = (int)p.M;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int rows_a = m1 - m0 < BM ? m1 - m0 : BM, rows_w = (int)p.N - n0 < BN ? (int)p.N - n0 : BN;
  const int nb = (p.K + 127) / 128, blocks_w = (rows_w + 127) / 128;

  Fp8Rows<C> t;
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a + (int64_t)m0 * p.lda, (int64_t)(rows_a - 1) * p.lda + p.K);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.w + (int64_t)n0 * p.ldw, (int64_t)(rows_w - 1) * p.ldw + p.K);
  const __amdgpu_buffer_rsrc_t rsa =
      make_rsrc(p.sa + m0 * p.sm, nb ? 4 * ((rows_a - 1) * p.sm + (nb - 1) * p.sb + 1) : 0);
  const __amdgpu_buffer_rsrc_t rsb = make_rsrc(p.sw + (n0 >> 7) * p.ldsw, nb ? 4 * ((blocks_w - 1) * p.ldsw + nb) : 0);
  t.sta = (uint32_t)(4 * p.sb);
#pragma unroll
  for (int j = 0; j < C::kLA; ++j) {
    int row, kb;
    pp_slot<C::kThreads, 8>(tid, j, row, kb);
    t.a[j] = row < rows_a ? (uint32_t)(row * p.lda) : kOob;
  }
#pragma unroll
  for (int j = 0; j < C::kLB; ++j) {
    int row, kb;
    pp_slot<C::kThreads, 8>(tid, j, row, kb);
    t.b[j] = row < rows_w ? (uint32_t)(row * p.ldw) : kOob;
  }
  t.s = tid < BM ? (tid < rows_a ? (uint32_t)(4 * tid * p.sm) : kOob)
                 : (tid - BM < blocks_w ? (uint32_t)(4 * (tid - BM) * p.ldsw) : kOob);

  typename C::Acc acc;
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j) acc[i][j] = v4f{0, 0, 0, 0};
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass does not instantiate the main loop twice)
  fp8_mainloop<BM, BN, WM, WN, RING, EXACT>(acc, ra, rb, rsa, rsb, t, p.K, smem);
#endif
  __syncthreads();

  // a 16-row strip at a time through the wave's part of LDS, out of it four consecutive columns a lane
  const int wm = wave / C::kWN, wn = wave % C::kWN;
  float* strip = (float*)(smem + wave * 16 * C::kLdc * 4);
  constexpr int kLanes = C::WTN / 4, kRows = 64 / kLanes;  // lanes a row, rows an instruction
  const int col = wn * C::WTN + lane % kLanes * 4, size = p.out_dtype == LSK_F32 ? 4 : 2;
  float b[4] = {0, 0, 0, 0};
  if (p.bias)
#pragma unroll
    for (int z = 0; z < 4; ++z)
      if (col + z < rows_w) b[z] = p.bias[n0 + col + z];
  int row = wm * C::WTM + lane / kLanes;
  const int64_t step = (int64_t)kRows * p.ldo * size;
  char* o = (char*)p.out + ((int64_t)(m0 + row) * p.ldo + n0 + col) * size;
  const bool whole = vec && col + 4 <= rows_w;
#pragma unroll
  for (int i = 0; i < C::TM; ++i) {
#pragma unroll
    for (int j = 0; j < C::TN; ++j) *(v4f*)(strip + (lane & 15) * C::kLdc + j * 16 + 4 * (lane >> 4)) = acc[i][j];
    // (a wave's own LDS operations run in order)
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += kRows, row += kRows, o += step) {
      v4f v = *(const v4f*)(strip + (r0 + lane / kLanes) * C::kLdc + lane % kLanes * 4);
      if (row >= rows_a || col >= rows_w) continue;
      if (p.bias)
#pragma unroll
        for (int z = 0; z < 4; ++z) v[z] = f32_add(v[z], b[z]);
      if (whole) {
        store_quad(o, p.out_dtype, v);
      } else {
        for (int z = 0; z < 4 && col + z < rows_w; ++z) store_out(o, p.out_dtype, z, v[z]);
      }
    }
  }
}

static int64_t fp8_row_tiles(const Fp8Args& p, int bm) {
  return p.offs ? expert_tiles_max(p.M, p.E, bm) : (p.M + bm - 1) / bm;
}

template <int BM, int BN, int WM, int WN, int RING>
static int fp8_tile_launch(const Fp8Args& p, hipStream_t s) {
  using C = Fp8Cfg<BM, BN, WM, WN, RING>;
  const int64_t mtiles = fp8_row_tiles(p, BM), blocks = mtiles * ((p.N + BN - 1) / BN);
  LSK_REQUIRE(grid_ok(blocks, C::kThreads) && blocks <= 0x7fffffff, "fp8 product: grid too large");
  const int vec = out_vec_ok(p.out, p.out_dtype, p.ldo);
  auto run = [&](auto kern) {
    if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes) != hipSuccess)
      return set_error("fp8_tile_kernel: cannot reserve LDS"), LSK_ERR_HIP;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(C::kThreads), C::kSmemBytes, s, p, mtiles, vec);
    return check_launch("fp8_tile_kernel");
  };
  if (p.out_dtype == LSK_F32)  // binary32 outputs from products kept whole (fp8_block)
    return p.offs ? run(fp8_tile_kernel<BM, BN, WM, WN, RING, true, true>)
                  : run(fp8_tile_kernel<BM, BN, WM, WN, RING, true, false>);
  return p.offs ? run(fp8_tile_kernel<BM, BN, WM, WN, RING, false, true>)
                : run(fp8_tile_kernel<BM, BN, WM, WN, RING, false, false>);
}

// The products address a tile's rows and scales with 31-bit offsets.
static bool fp8_reach(const Fp8Args& p) {
  const int64_t nb = (p.K + 127) / 128;
  return 256 * p.lda < 0x7fffffff && 256 * p.ldw < 0x7fffffff && 4 * (256 * p.sm + nb * p.sb) < 0x7fffffff &&
         4 * (4 * p.ldsw + nb) < 0x7fffffff;
}

static int fp8_product(const Fp8Args& p, hipStream_t s) {
  LSK_REQUIRE(fp8_reach(p), "fp8 product: M=%lld N=%lld K=%d beyond 31-bit offsets", (long long)p.M, (long long)p.N, p.K);
  return fp8_tile_launch<64, 64, 2, 2, 2>(p, s);
}

}  // namespace lsk

static int fp8_quant_check(const char* who, const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const void* q,
                           const void* scale) {
  LSK_REQUIRE(lsk::is_float_dtype(x_dtype), "%s: x_dtype must be f32, bf16 or f16", who);
  LSK_REQUIRE(M >= 0 && K >= 0 && K % 16 == 0 && K < (1 << 24), "%s: bad sizes (K=%lld a multiple of 16 below 2^24)", who,
              (long long)K);
  if (M == 0 || K == 0) return LSK_OK;
  LSK_REQUIRE(M == 1 || ldx >= K, "%s: ldx below K", who);
  LSK_REQUIRE(x && q && scale, "%s: null pointer", who);
  LSK_REQUIRE((uintptr_t)q % 16 == 0, "%s: codes must be 16-byte aligned", who);
  return LSK_OK;
}

extern "C" int lsk_quantize_rows_fp8(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* q,
                                     float* scale, int64_t scale_m, int64_t scale_b, void* stream) {
  const int rc = fp8_quant_check("lsk_quantize_rows_fp8", x, x_dtype, M, K, ldx, q, scale);
  if (rc || M == 0 || K == 0) return rc;
  int rows;
  LSK_REQUIRE(M <= (1LL << 40) && grid_ok(lsk::quantize_rows_blocks(M, K, rows), 256), "lsk_quantize_rows_fp8: grid too large");
  return lsk::quantize_rows_launch(x, x_dtype, M, K, ldx, q, scale, scale_m, scale_b, (hipStream_t)stream);
}

extern "C" int lsk_quantize_weight_fp8(const void* x, int x_dtype, int64_t N, int64_t K, int64_t ldx, uint8_t* q,
                                       float* scale, void* stream) {
  const int rc = fp8_quant_check("lsk_quantize_weight_fp8", x, x_dtype, N, K, ldx, q, scale);
  if (rc || N == 0 || K == 0) return rc;
  const int64_t blocks = (N + 127) / 128 * ((K + 127) / 128);
  LSK_REQUIRE(N <= (1LL << 40) && grid_ok(blocks, 256), "lsk_quantize_weight_fp8: grid too large");
  const dim3 grid((unsigned)blocks), blk(256);
  lsk::by_input(x, x_dtype, ldx, [&](auto dt, auto vec) {
    hipLaunchKernelGGL((lsk::quantize_weight_fp8_kernel<decltype(dt)::value, decltype(vec)::value>), grid, blk, 0,
                       (hipStream_t)stream, x, ldx, N, (int)K, q, scale);
  });
  return lsk::check_launch("quantize_weight_fp8_kernel");
}

extern "C" int lsk_dequant_fp8(const uint8_t* q, const float* scale, int64_t scale_m, int64_t scale_b, int block_rows,
                               int64_t M, int64_t K, void* out, int out_dtype, void* stream) {
  LSK_REQUIRE(lsk::is_float_dtype(out_dtype), "lsk_dequant_fp8: out_dtype must be f32, bf16 or f16");
  LSK_REQUIRE(M >= 0 && K >= 0 && K % 16 == 0 && K < (1 << 24) && M <= (1LL << 40),
              "lsk_dequant_fp8: bad sizes (K=%lld a multiple of 16 below 2^24)", (long long)K);
  LSK_REQUIRE(block_rows == 1 || block_rows == 128, "lsk_dequant_fp8: scales for 1 or 128 rows, got %d", block_rows);
  if (M == 0 || K == 0) return LSK_OK;
  LSK_REQUIRE(q && scale && out, "lsk_dequant_fp8: null pointer");
  LSK_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0, "lsk_dequant_fp8: codes and out must be 16-byte aligned");
  const int64_t total = M * (K / 8), blocks = (total + 255) / 256;
  const dim3 grid((unsigned)(blocks < (1 << 22) ? blocks : (1 << 22))), blk(256);
  const int shift = block_rows == 128 ? 7 : 0;
  auto run = [&](auto odt) {
    hipLaunchKernelGGL((lsk::dequant_fp8_kernel<decltype(odt)::value>), grid, blk, 0, (hipStream_t)stream, q, scale, scale_m,
                       scale_b, shift, total, (int)(K / 8), out);
  };
  if (out_dtype == LSK_F32) run(std::integral_constant<int, LSK_F32>{});
  else if (out_dtype == LSK_BF16) run(std::integral_constant<int, LSK_BF16>{});
  else run(std::integral_constant<int, LSK_F16>{});
  return lsk::check_launch("dequant_fp8_kernel");
}

static int fp8_check(const char* who, int64_t M, int64_t N, int64_t K, int out_dtype, int64_t ldo) {
  LSK_REQUIRE(M >= 0 && N >= 0 && K >= 0 && K % 16 == 0, "%s: bad sizes M=%lld N=%lld K=%lld (K a multiple of 16)", who,
              (long long)M, (long long)N, (long long)K);
  LSK_REQUIRE(M <= 0x7fffffff && N <= 0x7fffffff && K < (1 << 22), "%s: sizes beyond 31 bits (K beyond 2^22)", who);
  LSK_REQUIRE(lsk::is_float_dtype(out_dtype), "%s: out_dtype must be f32, bf16 or f16", who);
  LSK_REQUIRE(ldo >= N, "%s: ldo below N", who);
  return LSK_OK;
}

static int fp8_scales_check(const char* who, int64_t sm, int64_t sb) {
  LSK_REQUIRE(sm >= 0 && sb >= 0 && sm < (1LL << 31) && sb < (1LL << 31), "%s: bad scale strides", who);
  return LSK_OK;
}

extern "C" int lsk_gemm_fp8(const uint8_t* a, const float* a_scale, int64_t scale_m, int64_t scale_b, int64_t M, int64_t K,
                            const uint8_t* w, const float* w_scale, int64_t N, const float* bias, void* out, int out_dtype,
                            int64_t ldo, void* stream) {
  int rc = fp8_check("lsk_gemm_fp8", M, N, K, out_dtype, ldo);
  if (rc || (rc = fp8_scales_check("lsk_gemm_fp8", scale_m, scale_b))) return rc;
  if (M == 0 || N == 0) return LSK_OK;
  LSK_REQUIRE(out && (K == 0 || (a && a_scale && w && w_scale)), "lsk_gemm_fp8: null pointer");
  LSK_REQUIRE((uintptr_t)a % 16 == 0 && (uintptr_t)w % 16 == 0, "lsk_gemm_fp8: codes must be 16-byte aligned");
  lsk::Fp8Args p{};
  p.a = a, p.sa = a_scale, p.w = w, p.sw = w_scale;
  p.lda = p.ldw = K, p.sm = scale_m, p.sb = scale_b, p.ldsw = (K + 127) / 128;
  p.M = M, p.N = N, p.K = (int)K;
  p.bias = bias, p.out = out, p.out_dtype = out_dtype, p.ldo = ldo;
  return lsk::fp8_product(p, (hipStream_t)stream);
}

// The quantised rows come first in the workspace, then their scales, block by block.
extern "C" int64_t lsk_linear_fp8_workspace(int64_t M, int64_t N, int64_t K) {
  return lsk::up256(M * K) + lsk::up256(4 * M * ((K + 127) / 128));
}

extern "C" int lsk_linear_fp8(const void* x, int x_dtype, int64_t ldx, int64_t M, int64_t K, const uint8_t* w,
                              const float* w_scale, int64_t N, const float* bias, void* out, int out_dtype, int64_t ldo,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = fp8_check("lsk_linear_fp8", M, N, K, out_dtype, ldo);
  if (rc) return rc;
  LSK_REQUIRE(lsk::is_float_dtype(x_dtype), "lsk_linear_fp8: x_dtype must be f32, bf16 or f16");
  if (M == 0 || N == 0) return LSK_OK;
  LSK_REQUIRE(out && (K == 0 || (x && w && w_scale)), "lsk_linear_fp8: null pointer");
  LSK_REQUIRE(M == 1 || ldx >= K, "lsk_linear_fp8: ldx below K");
  LSK_REQUIRE((uintptr_t)w % 16 == 0, "lsk_linear_fp8: codes must be 16-byte aligned");
  const int64_t need = lsk_linear_fp8_workspace(M, N, K);
  LSK_REQUIRE(lsk::work_ok(workspace, workspace_bytes, need),
              "lsk_linear_fp8: workspace of %lld bytes (256-byte aligned) needed", (long long)need);
  hipStream_t s = (hipStream_t)stream;
  uint8_t* q = (uint8_t*)workspace;
  float* qs = (float*)(q + lsk::up256(M * K));
  lsk::Fp8Args p{};
  p.a = q, p.sa = qs, p.w = w, p.sw = w_scale;
  p.lda = p.ldw = K, p.sm = 1, p.sb = M, p.ldsw = (K + 127) / 128;
  p.M = M, p.N = N, p.K = (int)K;
  p.bias = bias, p.out = out, p.out_dtype = out_dtype, p.ldo = ldo;
  int rows;
  LSK_REQUIRE(K == 0 || grid_ok(lsk::quantize_rows_blocks(M, K, rows), 256), "lsk_linear_fp8: grid too large");
  if (K > 0 && (rc = lsk::quantize_rows_launch(x, x_dtype, M, K, ldx, q, qs, 1, M, s))) return rc;
  return lsk::fp8_product(p, s);
}

extern "C" int lsk_grouped_gemm_fp8(const uint8_t* a, const float* a_scale, int64_t scale_m, int64_t scale_b,
                                    const int32_t* offs, int64_t E, int64_t R, const int64_t* w_ptrs, int64_t ldw,
                                    const int64_t* ws_ptrs, int64_t ldsw, const int64_t* b_ptrs, int64_t N, int64_t K,
                                    void* out, int out_dtype, int64_t ldo, void* stream) {
  int rc = fp8_check("lsk_grouped_gemm_fp8", R, N, K, out_dtype, ldo);
  if (rc || (rc = fp8_scales_check("lsk_grouped_gemm_fp8", scale_m, scale_b))) return rc;
  LSK_REQUIRE(E >= 1 && E <= (1 << 20), "lsk_grouped_gemm_fp8: E=%lld not in [1, 2^20]", (long long)E);
  if (R == 0 || N == 0) return LSK_OK;
  LSK_REQUIRE(out && offs && w_ptrs && ws_ptrs && (K == 0 || (a && a_scale)), "lsk_grouped_gemm_fp8: null pointer");
  LSK_REQUIRE((uintptr_t)a % 16 == 0 && ldw >= K && ldw % 16 == 0 && ldsw >= (K + 127) / 128,
              "lsk_grouped_gemm_fp8: codes in rows of 16-byte multiples, strides that cover K");
  lsk::Fp8Args p{};
  p.a = a, p.sa = a_scale;
  p.lda = K, p.sm = scale_m, p.sb = scale_b, p.ldw = ldw, p.ldsw = ldsw;
  p.M = R, p.N = N, p.K = (int)K;
  p.out = out, p.out_dtype = out_dtype, p.ldo = ldo;
  p.offs = offs, p.E = (int)E, p.w_ptrs = w_ptrs, p.ws_ptrs = ws_ptrs, p.b_ptrs = b_ptrs;
  return lsk::fp8_product(p, (hipStream_t)stream);
}
