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

#define LSK_HD __host__ __device__ inline

namespace lsk {

// ---------------------------------------------------------------- the quantisers
// 16 lanes per 128 values of a row (a lane holds eight), 16 of these to a thread block: `rows` rows of it by
// 16 / rows blocks, kQuantDeep times along K with their loads in flight together.  With 16 rows a block its
// scales are 64-byte runs of the block-by-block layout; few rows spread over K instead.  Bound by HBM: 8192 bf16 rows of
// 4096, 102 MB, in 22.4 us on MI355X (25.4 with each load waited for), 4.5 TB/s.
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
  Raw8<DT, VEC> raw[kQuantDeep];
#pragma unroll
  for (int z = 0; z < kQuantDeep; ++z) {
    const int k = 128 * (b0 + per * z) + c;
    raw[z] = raw8<DT, VEC>(x, row * ldx + k, k < K);
  }
#pragma unroll
  for (int z = 0; z < kQuantDeep; ++z) {
    const int b = b0 + per * z, k = 128 * b + c;
    if (b >= nb) break;
    float v[8], s;
    raw8_values(raw[z], v);
    const uint2 w = quantize_row_fp8(v, s);
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
// its codes.  Bound by HBM: 28672 x 4096 in bf16, 352 MB, in 65 us on MI355X (72 with each load waited for), 5.4 TB/s.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void quantize_weight_fp8_kernel(const void* __restrict__ x, int64_t ldx, int64_t N,
                                                                  int K, uint8_t* __restrict__ q,
                                                                  float* __restrict__ scale) {
  __shared__ uint32_t tops[4];
  const int nb = (K + 127) / 128;
  const int64_t rb = blockIdx.x / nb;
  const int b = (int)(blockIdx.x - rb * nb), k = 128 * b + 8 * (threadIdx.x & 15);
  const int64_t row0 = 128 * rb + (threadIdx.x >> 4);
  Raw8<DT, VEC> raw[8];
#pragma unroll
  for (int z = 0; z < 8; ++z) raw[z] = raw8<DT, VEC>(x, (row0 + 16 * z) * ldx + k, k < K && row0 + 16 * z < N);
  uint32_t top = 0;
  float v[8];
#pragma unroll
  for (int z = 0; z < 8; ++z) {
    raw8_values(raw[z], v);
    const uint32_t t = top8(v);
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
  for (int z = 0; z < 8; ++z) {
    raw8_values(raw[z], v);
    if (k < K && row0 + 16 * z < N) *(uint2*)(q + (row0 + 16 * z) * K + k) = quantize8_fp8(v, s.inv);
  }
}

// Codes times scales, four times eight bytes of outputs a thread, so that a wave's stores are whole lines side by side
// (MI355X, against eight consecutive values a thread: 28672 x 4096 to bf16 64 -> 54 us, to f32 466 -> 100; lines filled by
// two stores past the caches reach HBM in parts).  Bound by HBM: 352 MB in 54 us are 6.5 TB/s.  `per` of these units to a
// row; part: 2^22 / per, rounded up.
template <int ODT>
__global__ __launch_bounds__(256) void dequant_fp8_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                          int64_t sm, int64_t sb, int row_shift, int64_t total, uint32_t per,
                                                          uint32_t part, void* __restrict__ out) {
  constexpr int V = ODT == LSK_F32 ? 2 : 4, kStep = 4;
  typedef std::conditional_t<V == 2, uint16_t, uint32_t> Codes;
  for (int64_t base = (int64_t)blockIdx.x * (256 * kStep); base < total; base += (int64_t)gridDim.x * (256 * kStep)) {
    const int64_t row0 = base >> 32 ? base / per : (int64_t)((uint32_t)base / per);
    const uint32_t c0 = (uint32_t)(base - row0 * per) + threadIdx.x;
    const bool wide = per >= 256 * kStep;  // (one row's end at most lies among a block's units)
    int u[kStep];
    float s[kStep];
#pragma unroll
    for (int z = 0; z < kStep; ++z) {
      // (short rows: t < 2^11, and 2^22 / per rounded up is off by less than per / 2^22)
      const uint32_t t = c0 + 256 * z, down = wide ? t >= per : t * part >> 22, c = t - down * per;
      u[z] = 0, s[z] = 0.0f;
      if (base + 256 * z + threadIdx.x < total) {
        u[z] = (int)((const Codes*)q)[base + 256 * z + threadIdx.x];
        s[z] = scale[((row0 + down) >> row_shift) * sm + c / (128 / V) * sb];
      }
    }
#pragma unroll
    for (int z = 0; z < kStep; ++z) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(u[z], false);
      float v[4] = {f32_mul(a[0], s[z]), f32_mul(a[1], s[z]), 0.0f, 0.0f};
      if constexpr (V == 4) {
        const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(u[z], true);
        v[2] = f32_mul(b[0], s[z]), v[3] = f32_mul(b[1], s[z]);
      }
      uint64_t w;
      if constexpr (ODT == LSK_F32) {
        w = (uint64_t)__float_as_uint(v[1]) << 32 | __float_as_uint(v[0]);
      } else if constexpr (ODT == LSK_BF16) {
        const float any = (v[0] + v[1]) + (v[2] + v[3]);  // (a NaN where one of them is)
        uint32_t lo = pack_bf16x2_nonan(v[0], v[1]), hi = pack_bf16x2_nonan(v[2], v[3]);
        if (__builtin_amdgcn_ballot_w64(any != any)) lo = pack_bf16x2(v[0], v[1]), hi = pack_bf16x2(v[2], v[3]);
        w = (uint64_t)hi << 32 | lo;
      } else {
        uint16_t h[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          // (the product is a binary32 number first: the compiler would round it to f16 in one instruction)
          __asm__("" : "+v"(v[t]));
          h[t] = __builtin_bit_cast(uint16_t, (_Float16)v[t]);
        }
        w = (uint64_t)((uint32_t)h[2] | (uint32_t)h[3] << 16) << 32 | ((uint32_t)h[0] | (uint32_t)h[1] << 16);
      }
      if (base + 256 * z + threadIdx.x < total) __builtin_nontemporal_store(w, (uint64_t*)out + base + 256 * z + threadIdx.x);
    }
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

// Few rows: a block computes NG x 16 output columns of up to MT x 16 rows over all of K, streaming its
// weight rows from HBM.  Four waves bring the codes in, KS x 256 values (256 bytes of a row, whole lines)
// a stage, by direct global -> LDS loads RING - 1 stages ahead; waves multiply a group of 16 weight
// rows by a row tile each.  Bound by HBM, that is by bytes in flight: with a few thousand weight rows there is
// a block of 16 of them a CU, which is why waves that do not multiply load.  K is not split over waves or
// blocks: every kernel here sums an output in one chain, and a split by the number of rows would make a
// row's bits depend on its batch.  The products of the rows' scales with the weight's (a block's columns share
// one weight scale) are put into LDS whole at the start; their loads go out before the ring's, which they would
// wait for otherwise.
// (MI355X: 32 rows on 4096 x 14336 17.2 us, 688 KB a CU, rows and weights, at 40 B/ns; 128 rows over 32 experts of
// 2880 x 2880 49 us, 4.9 TB/s; one row on 28672 x 4096 26, 4.5 TB/s.  With one block of 16 weight rows a CU the depth of the
// ring counts: the product of one row of 18944 with 3584 columns takes 22.3 us with four stages in the ring, 17.8 with six.)
// DT >= 0: the block's rows of x (at most 16; vec: 16-byte aligned) are quantised by every block into LDS
// itself, which saves a launch and the wait for it; x comes from the L2.
template <int NG, int MT, int KS, bool FUSE>
struct Fp8StreamCfg {
  static constexpr int kPartW = NG * 4096, kPart = kPartW + (FUSE ? 0 : MT * 4096), kStage = KS * kPart;  // bytes
  static constexpr int kPer = KS * (NG + (FUSE ? 0 : MT));  // loads per thread per stage
  static constexpr int kPre = 16;                            // scales of a thread loaded ahead of the ring
  static_assert(NG * MT <= 4, "a wave multiplies at most one weight group with one row tile");
  static_assert(NG <= 8 && 128 % (16 * NG) == 0, "a block's columns share a weight scale");
};

// Parts of 256 values, whole stages of them; floats from one row of scales to the next (two of four banks
// further each row: 16 rows' pairs read at once lie in 32 banks), bytes from one row of codes to the next.
LSK_HD int fp8_parts(int K, int ks) { return ((K + 255) / 256 + ks - 1) / ks * ks; }
LSK_HD int fp8_scale_pitch(int K, int ks) { return 2 * fp8_parts(K, ks) | 2; }
LSK_HD int fp8_fused_pitch(int K, int ks) { return fp8_parts(K, ks) * 256 + 16; }
template <int NG, int MT, int KS, int RING, bool FUSE>
static int64_t fp8_stream_lds(int K, int rows) {
  return RING * Fp8StreamCfg<NG, MT, KS, FUSE>::kStage + (FUSE ? (int64_t)rows * fp8_fused_pitch(K, KS) : 0) +
         (int64_t)(FUSE ? rows : MT * 16) * fp8_scale_pitch(K, KS) * 4;
}

template <int NG, int MT, int KS, int RING, int DT, bool EXACT, bool GROUPED>
__global__ __launch_bounds__(256) void fp8_stream_kernel(Fp8Args p, const void* __restrict__ x, int64_t ldx, int vec) {
  constexpr bool FUSE = DT >= 0;
  using C = Fp8StreamCfg<NG, MT, KS, FUSE>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), r = lane & 15, q = lane >> 4;
  const int ngroups = (int)((p.N + 16 * NG - 1) / (16 * NG));
  const int tile = blockIdx.x / ngroups, n0 = (blockIdx.x - tile * ngroups) * 16 * NG;
  int64_t m0 = (int64_t)tile * 16 * MT, m1 = p.M;
  if constexpr (GROUPED) {
    int e, first, end;
    if (!ExpertTiles(p.offs, p.E, (int)p.M, 16 * MT).find(tile, e, first, end)) return;
    m0 = first;
    m1 = end;
    p.w = (const uint8_t*)wave_uniform64(p.w_ptrs[e]);
    p.sw = (const float*)wave_uniform64(p.ws_ptrs[e]);
    p.bias = p.b_ptrs ? (const float*)wave_uniform64(p.b_ptrs[e]) : nullptr;
  }
  const int rows_a = m1 - m0 < 16 * MT ? (int)(m1 - m0) : 16 * MT;
  const int rows_w = p.N - n0 < 16 * NG ? (int)p.N - n0 : 16 * NG;
  const int nb = (p.K + 127) / 128, parts = fp8_parts(p.K, KS), nk = parts / KS;
  const int sp = fp8_scale_pitch(p.K, KS), fp = fp8_fused_pitch(p.K, KS);
  char* const fused = smem + RING * C::kStage;  // FUSE: the rows' codes
  float* const scales = (float*)(fused + (FUSE ? rows_a * fp : 0));
  const float* const sw = p.sw + (int64_t)(n0 >> 7) * p.ldsw;

  // the scales' table: row m of it, block b; 0 past the rows and past K
  constexpr int kRows = 16 * MT;
  const int total = FUSE ? 0 : kRows * 2 * parts;
  const float* const sa = p.sa + m0 * p.sm;
  float pa[C::kPre], pw[C::kPre];
  if constexpr (!FUSE) {
#pragma unroll
    for (int z = 0; z < C::kPre; ++z) {
      const int i = tid + 256 * z, m = i % kRows, b = i / kRows;
      pa[z] = pw[z] = 0.0f;
      if (256 * z < total && m < rows_a && b < nb) pa[z] = sa[m * p.sm + b * p.sb], pw[z] = sw[b];
    }
  }

  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w + (int64_t)n0 * p.ldw, (int64_t)(rows_w - 1) * p.ldw + p.K);
  const __amdgpu_buffer_rsrc_t ra = FUSE ? rw : make_rsrc(p.a + m0 * p.lda, (int64_t)(rows_a - 1) * p.lda + p.K);
  // a thread's 16-byte slot j of a part: row 16 j + tid / 16, chunk c of its 256 bytes in place c ^ row % 16
  const int row = tid >> 4, kc = 16 * ((tid & 15) ^ row);
  auto issue = [&](int kt) {
    char* base = smem + (kt % RING) * C::kStage + wave * 1024;
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      const int k = 256 * (KS * kt + u);
      const bool in = k + kc < p.K;
#pragma unroll
      for (int j = 0; j < NG; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_void_t)(base + u * C::kPart + j * 4096), 16,
                                                 in && 16 * j + row < rows_w ? (uint32_t)((16 * j + row) * (int)p.ldw + kc) : kOob,
                                                 k, 0, 0);
      if constexpr (!FUSE) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void_t)(base + u * C::kPart + C::kPartW + j * 4096), 16,
                                                   in && 16 * j + row < rows_a ? (uint32_t)((16 * j + row) * (int)p.lda + kc) : kOob,
                                                   k, 0, 0);
      }
    }
  };
  compiler_fence();
#pragma unroll
  for (int s = 0; s < RING - 1; ++s) issue(s);

  if constexpr (!FUSE) {
#pragma unroll
    for (int z = 0; z < C::kPre; ++z) {
      const int i = tid + 256 * z;
      if (i < total) scales[i % kRows * sp + i / kRows] = f32_mul(pa[z], pw[z]);
    }
    for (int i = tid + 256 * C::kPre; i < total; i += 256) {
      const int m = i % kRows, b = i / kRows;
      scales[m * sp + b] = m < rows_a && b < nb ? f32_mul(sa[m * p.sm + b * p.sb], sw[b]) : 0.0f;
    }
  } else {
    // 16 lanes a block of 128 values, the rows end to end (zeros past K), kBatch loads of a thread in flight
    const int slots = 32 * parts, all = rows_a * slots;  // pieces of eight values
    constexpr int kBatch = 4;
    auto quantize = [&](auto aligned) {
      for (int i0 = tid; i0 < all; i0 += 256 * kBatch) {
        constexpr bool VEC = decltype(aligned)::value;
        Raw8<DT, VEC> raw[kBatch];
        int m[kBatch];
#pragma unroll
        for (int z = 0; z < kBatch; ++z) {
          const int i = i0 + 256 * z;
          m[z] = (int)((uint32_t)i / (uint32_t)slots);
          const int k = 8 * (i - m[z] * slots);
          raw[z] = raw8<DT, VEC>(x, (m0 + m[z]) * ldx + k, i < all && k < p.K);
        }
#pragma unroll
        for (int z = 0; z < kBatch; ++z) {
          const int i = i0 + 256 * z, c = i - m[z] * slots;
          if (i >= all) continue;  // (16 lanes alike: `slots` is a multiple of 32)
          float v[8], s;
          raw8_values(raw[z], v);
          *(uint2*)(fused + m[z] * fp + 8 * c) = quantize_row_fp8(v, s);
          if ((c & 15) == 0) scales[m[z] * sp + (c >> 4)] = (c >> 4) < nb ? f32_mul(s, sw[c >> 4]) : 0.0f;
        }
      }
    };
    if (vec) quantize(std::true_type{});
    else quantize(std::false_type{});
  }

  // wave w multiplies weight group w % NG with row tile w / NG
  const int g = wave % NG, mt = wave / NG;
  const bool multiplies = wave < NG * MT;
  v4f acc = v4f{0, 0, 0, 0};
  // (rows past the end: whatever lies there, their results are not stored)
  const int ar = FUSE ? min(r, rows_a - 1) : 16 * mt + r;
  const float* const ars = scales + ar * sp;
  const char* const arc = FUSE ? fused + ar * fp : smem + C::kPartW + ar * 256;
  // a stage's fragments are read a stage ahead where the ring is deep enough, so that the LDS works under the
  // matrix core's and the FMAs' chain
  struct Frag {
    v2f_t s[KS];
    v8i w[KS][2], a[KS][2];
  };
  auto read = [&](int kt, Frag& f) {
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      const int slot = (kt % RING) * C::kStage + u * C::kPart, part = KS * kt + u;
      const char* base = smem + slot + (16 * g + r) * 256;
      f.s[u] = *(const v2f_t*)(ars + 2 * part);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c0 = 16 * ((8 * h + q) ^ r), c1 = 16 * ((8 * h + 4 + q) ^ r);
        f.w[u][h] = fp8_operand(*(const v4i*)(base + c0), *(const v4i*)(base + c1));
        const char* a = FUSE ? arc + 256 * part + 128 * h + 16 * q : arc + slot;
        f.a[u][h] = FUSE ? fp8_operand(*(const v4i*)a, *(const v4i*)(a + 64))
                         : fp8_operand(*(const v4i*)(a + c0), *(const v4i*)(a + c1));
      }
    }
  };
  auto multiply = [&](const Frag& f) {
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) acc = fp8_scaled(fp8_block<EXACT>(f.w[u][h], f.a[u][h]), f.s[u][h], acc);
  };
  Frag f[2];
  if constexpr (RING >= 4) {
    wait_vm<(RING - 2) * C::kPer>();
    wait_lgkm0();
    phase_barrier();
    if (multiplies) read(0, f[0]);
    auto step = [&](int kt, Frag& now, Frag& next) {
      compiler_fence();  // (the reads of the stage before stay on their side of the barrier)
      wait_vm<(RING - 3) * C::kPer>();
      phase_barrier();
      issue(kt + RING - 1);
      if (multiplies) {
        if (kt + 1 < nk) read(kt + 1, next);
        multiply(now);
      }
    };
    int kt = 0;
    for (; kt + 2 <= nk; kt += 2) {
      step(kt, f[0], f[1]);
      step(kt + 1, f[1], f[0]);
    }
    if (kt < nk) step(kt, f[0], f[1]);
  } else {
    for (int kt = 0; kt < nk; ++kt) {
      wait_vm<(RING - 2) * C::kPer>();
      wait_lgkm0();
      phase_barrier();
      issue(kt + RING - 1);
      if (multiplies) {
        read(kt, f[0]);
        multiply(f[0]);
      }
    }
  }
  wait_vm<0>();
  if (!multiplies) return;
  float b[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int64_t n = n0 + 16 * g + 4 * q + t;
    b[t] = p.bias && n < p.N ? p.bias[n] : 0.0f;
  }
  const int row_out = 16 * mt + r;
  if (row_out >= rows_a) return;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int64_t n = n0 + 16 * g + 4 * q + t;
    float y = acc[t];
    __asm__("" : "+v"(y));  // (a binary32 sum first, as the tiles have it: not one FMA that rounds to f16)
    if (n < p.N) store_out(p.out, p.out_dtype, (m0 + row_out) * p.ldo + n, p.bias ? f32_add(y, b[t]) : y);
  }
}

// ---------------------------------------------------------------- tiles
// The tile's outputs: a 16-row strip at a time through the wave's part of LDS, out of it four consecutive columns a lane.
// LINES: rows begin on lines of 128 bytes, and whole lines go past the caches (store_quad; MI355X, builds in turn, past them
// and not: 4096 rows of 28672 x 4096 422 us, 434; 4096 of 4096 x 2048 34.6, 36.8; 32768 over 128 experts of 1536 x 2048 186,
// 196); lines that two rows share are put together in the L2 (3102 rows of 13016 x 128 40.6, 34.5; 4000 of 4600 x 2880
// 82.4, 84.0).
template <class C, int ODT, bool LINES>
LSK_DEV void fp8_tile_out(const Fp8Args& p, const typename C::Acc& acc, char* smem, int m0, int n0, int rows_a, int rows_w,
                          int vec) {
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int wm = wave / C::kWN, wn = wave % C::kWN;
  float* strip = (float*)(smem + wave * 16 * C::kLdc * 4);
  constexpr int kLanes = C::WTN / 4, kRows = 64 / kLanes;  // lanes a row, rows an instruction
  const int col = wn * C::WTN + lane % kLanes * 4, size = ODT == LSK_F32 ? 4 : 2;
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
    wave_lds_fence();
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += kRows, row += kRows, o += step) {
      v4f v = *(const v4f*)(strip + (r0 + lane / kLanes) * C::kLdc + lane % kLanes * 4);
      if (row >= rows_a || col >= rows_w) continue;
      if (p.bias)
#pragma unroll
        for (int z = 0; z < 4; ++z) v[z] = f32_add(v[z], b[z]);
      if (whole) {
        store_quad<LINES>(o, ODT, v);
        __asm__ volatile("" ::: "memory");  // (no 16-byte stores: store16_split)
      } else {
        for (int z = 0; z < 4 && col + z < rows_w; ++z) store_out(o, ODT, z, v[z]);
      }
    }
    wave_lds_fence();
  }
}

// A BM x BN tile: tiles walk kGroupM row tiles down a column of weight tiles inside each XCD's run
// of them, so the row tiles that share a weight tile run together on one L2.
template <int BM, int BN, int WM, int WN, int RING, bool EXACT, bool GROUPED>
__global__ __launch_bounds__(WM * WN * 64) void fp8_tile_kernel(Fp8Args p, int64_t mtiles, int vec) {
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

  auto tile = [&](auto config) {
    using C = decltype(config);
    Fp8Tile t;
    t.ra = make_rsrc(p.a + (int64_t)m0 * p.lda, (int64_t)(rows_a - 1) * p.lda + p.K);
    t.rb = make_rsrc(p.w + (int64_t)n0 * p.ldw, (int64_t)(rows_w - 1) * p.ldw + p.K);
    t.rsa = make_rsrc(p.sa + m0 * p.sm, nb ? 4 * ((rows_a - 1) * p.sm + (nb - 1) * p.sb + 1) : 0);
    t.rsb = make_rsrc(p.sw + (n0 >> 7) * p.ldsw, nb ? 4 * ((blocks_w - 1) * p.ldsw + nb) : 0);
    t.lda = (int)p.lda, t.ldb = (int)p.ldw, t.rows_a = rows_a, t.rows_b = rows_w;
    t.sta = (uint32_t)(4 * p.sb);
    t.s = tid < C::kBM ? (tid < rows_a ? (uint32_t)(4 * tid * p.sm) : kOob)
                       : (tid - C::kBM < blocks_w ? (uint32_t)(4 * (tid - C::kBM) * p.ldsw) : kOob);

    typename C::Acc acc;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j) acc[i][j] = v4f{0, 0, 0, 0};
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass does not instantiate the main loop twice)
    fp8_mainloop<C::kBM, C::kBN, C::kWM, C::kWN, C::kRing, EXACT>(acc, t, p.K, smem);
#endif
    __syncthreads();

    auto out = [&](auto odt) {
      if (vec == 2) fp8_tile_out<C, decltype(odt)::value, true>(p, acc, smem, m0, n0, rows_a, rows_w, vec);
      else fp8_tile_out<C, decltype(odt)::value, false>(p, acc, smem, m0, n0, rows_a, rows_w, vec);
    };
    if constexpr (EXACT) out(std::integral_constant<int, LSK_F32>{});
    else if (p.out_dtype == LSK_BF16) out(std::integral_constant<int, LSK_BF16>{});
    else out(std::integral_constant<int, LSK_F16>{});
  };
  // A half-empty tile's rows over all eight waves, 64 each, rather than over one group of four.  (MI355X, builds in turn:
  // 16384 rows over 128 experts of 1536 x 2048 145.1 -> 141.2 us, 32768 of them 188.8 -> 185.8, 16384 over 32 of 5760 x 2880
  // 421 -> 416; the requests in flight bound such tiles as much as the products.)
  if constexpr (BM == 256) {
    if (rows_a <= 128) return tile(Fp8Cfg<128, BN, WM, WN, RING>{});
  }
  tile(Fp8Cfg<BM, BN, WM, WN, RING>{});
}

// E: the experts, 0 for a dense product.
static int64_t fp8_row_tiles(int64_t M, int64_t E, int bm) { return E ? expert_tiles_max(M, E, bm) : (M + bm - 1) / bm; }

template <int BM, int BN, int WM, int WN, int RING>
static int fp8_tile_launch(const Fp8Args& p, hipStream_t s) {
  using C = Fp8Cfg<BM, BN, WM, WN, RING>;
  const int64_t mtiles = fp8_row_tiles(p.M, p.E, BM), blocks = mtiles * ((p.N + BN - 1) / BN);
  LSK_REQUIRE(grid_ok(blocks, C::kThreads) && blocks <= 0x7fffffff, "fp8 product: grid too large");
  const int64_t pitch = p.ldo * (p.out_dtype == LSK_F32 ? 4 : 2);
  const int vec = !out_vec_ok(p.out, p.out_dtype, p.ldo) ? 0 : (uintptr_t)p.out % 128 == 0 && pitch % 128 == 0 ? 2 : 1;
  auto run = [&](auto kern) {
    if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes) != hipSuccess)
      return set_error("fp8_tile_kernel: cannot reserve LDS"), LSK_ERR_HIP;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(C::kThreads), C::kSmemBytes, s, p, mtiles, vec);
    return check_launch("fp8_tile_kernel");
  };
  if constexpr (C::kThreads == 256) {
    if (p.out_dtype == LSK_F32)  // from products kept whole (fp8_block)
      return p.offs ? run(fp8_tile_kernel<BM, BN, WM, WN, RING, true, true>)
                    : run(fp8_tile_kernel<BM, BN, WM, WN, RING, true, false>);
  }
  return p.offs ? run(fp8_tile_kernel<BM, BN, WM, WN, RING, false, true>)
                : run(fp8_tile_kernel<BM, BN, WM, WN, RING, false, false>);
}

// The products address a tile's rows and scales with 31-bit offsets.
static bool fp8_reach(const Fp8Args& p) {
  const int64_t nb = (p.K + 127) / 128;
  return 256 * p.lda < 0x7fffffff && 256 * p.ldw < 0x7fffffff && 4 * (256 * p.sm + nb * p.sb) < 0x7fffffff &&
         4 * (4 * p.ldsw + nb) < 0x7fffffff;
}

template <int NG, int MT, int KS, int RING, int DT>
static int fp8_stream_launch(const Fp8Args& p, const void* x, int64_t ldx, hipStream_t s) {
  const int64_t tiles = fp8_row_tiles(p.M, p.E, 16 * MT);
  const int64_t blocks = tiles * ((p.N + 16 * NG - 1) / (16 * NG));
  LSK_REQUIRE(grid_ok(blocks, 256) && blocks <= 0x7fffffff, "fp8 product: grid too large");
  const int64_t lds = fp8_stream_lds<NG, MT, KS, RING, (DT >= 0)>(p.K, (int)(p.M < 16 ? p.M : 16));
  LSK_REQUIRE(lds <= 160 * 1024, "fp8 product: K=%d too long for few rows", p.K);
  const int vec = x && (uintptr_t)x % 16 == 0 && (ldx * (DT == LSK_F32 ? 4 : 2)) % 16 == 0;
  auto run = [&](auto kern) {
    if (lds > 65536 &&
        hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess)
      return set_error("fp8_stream_kernel: cannot reserve LDS"), LSK_ERR_HIP;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), (size_t)lds, s, p, x, ldx, vec);
    return check_launch("fp8_stream_kernel");
  };
  const bool exact = p.out_dtype == LSK_F32;  // (fp8_block)
  if constexpr (DT < 0) {
    if (p.offs)
      return exact ? run(fp8_stream_kernel<NG, MT, KS, RING, DT, true, true>)
                   : run(fp8_stream_kernel<NG, MT, KS, RING, DT, false, true>);
  }
  return exact ? run(fp8_stream_kernel<NG, MT, KS, RING, DT, true, false>)
               : run(fp8_stream_kernel<NG, MT, KS, RING, DT, false, false>);
}

// ---------------------------------------------------------------- which launch
// About how long a product takes on each of the launches, in us: the CU with the most blocks, ceil(blocks / 256) of
// them, works through them `resident` at a time, a round of o blocks at once in round[o - 1] + k[o - 1] a block of 128
// values of K; every million outputs cost `out` and `area` a block of K, every 10^9 weights read `weights`, and every
// 10^9 bytes of a block's operands `spill` where the rows (of an expert) outgrow an XCD's 4 MB of L2.  Fitted to 902
// products with bf16 outputs on MI355X (1 to 4096 rows of 17 to 37888 columns, K = 16 to 18944; 1 to 32768 rows over 2 to
// 128 experts), 256 x 256 tiles of at most 128 rows then still computed as full ones; binary32 outputs, which are other
// instructions and twice the bytes, choose by the same constants.  On products that it was not fitted to, what it picks is
// slower than the best of these launches by (755 dense, 380 by expert of each):
//   bf16 outputs      2.6 % on average, dense, and 2.4 % by expert; nine of ten within 9.3 and 8.3 %; at most 45 % (221 rows of
//                     3136 x 4864, 23.7 us on 32 x 32 blocks, 16.4 on 64 x 64 tiles) and 26 % (2 rows over 44 experts)
//   binary32 outputs  2.5 and 2.9 %; nine of ten within 7.1 and 9.8 %; at most 28 % (348 rows of 125 x 736, 8.1 and 6.3 us)
//                     and 25 % (2405 rows over 23 experts of 2091 x 3904, 104 and 83 us)
// All of them give the same bits.
struct Fp8Cost {
  int bm, bn, resident;  // resident 0: as many as the LDS holds at this K, to four
  double base, out, area, weights, spill, round[4], k[4];
};
enum {  // fp8_launch's order
  kTile256, kTile128, kTile64x128, kTile64, kTile64Deep, kTile128x64, kStream1, kStream2, kStream4, kStream1Deep, kStream1x2,
  kStream2x2, kStream2x2Deep, kLaunches
};
constexpr Fp8Cost kFp8Costs[kLaunches] = {
    {256, 256, 1, 2.6, 0.044, 0.042, 45, 0, {8.6}, {0.93}},
    {128, 128, 2, 2.0, 0, 0.06, 54, 0, {4.4, 5.5}, {0.556, 0.526}},
    {64, 128, 3, 2.7, 0.19, 0.056, 97, 3.1, {1.8, 2.8, 2.5}, {0.43, 0.383, 0.662}},
    {64, 64, 4, 3.2, 0.19, 0.118, 85, 4.3, {0.54, 0.94, 2.1, 1.8}, {0.364, 0.256, 0.22, 0.374}},
    {64, 64, 2, 2.4, 0.58, 0.003, 84, 8.6, {1.7, 1.7}, {0.284, 0.369}},
    {128, 64, 1, 2.5, 0.72, 0.004, 23, 0, {2.0}, {0.427}},
    {16, 16, 0, 2.6, 15.7, 0.55, 0, 0, {2.2, 1.5}, {0.068, 0.087}},
    {16, 32, 0, 3.1, 4.2, 0, 54, 0, {1.9, 1.8, 0.1, 0}, {0.114, 0.141, 0.382, 0.481}},
    {16, 64, 0, 3.0, 3.3, 0.33, 75, 0, {1.7, 0, 0.6, 0}, {0.158, 0.255, 0.313, 0.313}},
    {16, 16, 0, 2.7, 14.2, 0, 14, 0, {2.0}, {0.086}},
    {32, 16, 0, 2.6, 1.6, 0, 95, 6.3, {2.9}, {0.083}},
    {32, 32, 0, 3.5, 0.11, 0.008, 97, 7.6, {1.6, 1.9, 2.3}, {0.135, 0.17, 0.24}},
    {32, 32, 0, 1.9, 0.126, 0.014, 63, 0, {3.5}, {0.116}},
};

template <int NG, int MT, int KS, int RING>
static int fp8_stream_resident(int64_t K) {  // blocks of a CU, to four (0: the scales of all of K do not fit)
  const int64_t n = 160 * 1024 / fp8_stream_lds<NG, MT, KS, RING, false>((int)K, 16);
  return (int)(n < 4 ? n : 4);
}

static int fp8_launch(int which, const Fp8Args& p, hipStream_t s) {
  switch (which) {
    case kTile256: return fp8_tile_launch<256, 256, 2, 4, 2>(p, s);
    case kTile128: return fp8_tile_launch<128, 128, 2, 2, 2>(p, s);
    case kTile64x128: return fp8_tile_launch<64, 128, 2, 2, 2>(p, s);
    case kTile64: return fp8_tile_launch<64, 64, 2, 2, 2>(p, s);
    case kTile64Deep: return fp8_tile_launch<64, 64, 2, 2, 4>(p, s);
    case kTile128x64: return fp8_tile_launch<128, 64, 2, 2, 4>(p, s);
    case kStream1: return fp8_stream_launch<1, 1, 2, 4, -1>(p, nullptr, 0, s);
    case kStream2: return fp8_stream_launch<2, 1, 1, 3, -1>(p, nullptr, 0, s);
    case kStream4: return fp8_stream_launch<4, 1, 1, 2, -1>(p, nullptr, 0, s);
    case kStream1Deep: return fp8_stream_launch<1, 1, 2, 6, -1>(p, nullptr, 0, s);
    case kStream1x2: return fp8_stream_launch<1, 2, 2, 4, -1>(p, nullptr, 0, s);
    case kStream2x2: return fp8_stream_launch<2, 2, 1, 3, -1>(p, nullptr, 0, s);
    default: return fp8_stream_launch<2, 2, 2, 4, -1>(p, nullptr, 0, s);
  }
}

static int fp8_resident(int which, int64_t K) {
  switch (which) {
    case kStream1: return fp8_stream_resident<1, 1, 2, 4>(K);
    case kStream2: return fp8_stream_resident<2, 1, 1, 3>(K);
    case kStream4: return fp8_stream_resident<4, 1, 1, 2>(K);
    case kStream1Deep: return fp8_stream_resident<1, 1, 2, 6>(K);
    case kStream1x2: return fp8_stream_resident<1, 2, 2, 4>(K);
    case kStream2x2: return fp8_stream_resident<2, 2, 1, 3>(K);
    case kStream2x2Deep: return fp8_stream_resident<2, 2, 2, 4>(K);
    default: return kFp8Costs[which].resident;
  }
}

// E > 0: rows over E experts, `live` of which get some were all as likely, half a tile of each part empty.
static double fp8_us(int which, int64_t M, int64_t N, int64_t K, int64_t E) {
  const Fp8Cost& c = kFp8Costs[which];
  const int o = fp8_resident(which, K);
  if (o < 1) return 1e30;
  const double live = E ? E * (1.0 - __builtin_exp(-(double)M / E)) : 1.0;
  double down = (double)((M + c.bm - 1) / c.bm);
  if (E) down = (double)M / c.bm + live / 2 > live ? (double)M / c.bm + live / 2 : live;
  const double blocks = __builtin_ceil(down * ((N + c.bn - 1) / c.bn)), nk = (double)((K + 127) / 128);
  const double most = __builtin_ceil(blocks / 256), full = __builtin_floor(most / o), outs = blocks * 1e-6 * c.bm * c.bn;
  const int rest = (int)(most - full * o);
  const bool spills = (double)M * K > 4e6 * (E ? E : 1);
  return c.base + outs * (c.out + c.area * nk) + live * N * K * 1e-9 * c.weights +
         (spills ? blocks * (c.bm + c.bn) * K * 1e-9 * c.spill : 0) + full * (c.round[o - 1] + c.k[o - 1] * nk) +
         (rest ? c.round[rest - 1] + c.k[rest - 1] * nk : 0);
}

// The launch of a product: of those whose grid holds it the one that is likely to take the shortest; -1 where none holds it.
static int fp8_choice(int64_t M, int64_t N, int64_t K, int64_t E, int out_dtype) {
  int best = -1;
  double us = 1e30;
  for (int c = 0; c < kLaunches; ++c) {
    if (K == 0 && c >= kStream1) break;
    if (c == kTile256 && out_dtype == LSK_F32) continue;  // (products kept whole need more registers than it has)
    const Fp8Cost& f = kFp8Costs[c];
    if (!grid_ok(fp8_row_tiles(M, E, f.bm) * ((N + f.bn - 1) / f.bn), c == kTile256 ? 512 : 256)) continue;
    const double t = fp8_us(c, M, N, K, E);
    if (t < us) us = t, best = c;
  }
  return best;
}

static int fp8_check_launch(const Fp8Args& p, int which) {
  LSK_REQUIRE(fp8_reach(p), "fp8 product: M=%lld N=%lld K=%d beyond 31-bit offsets", (long long)p.M, (long long)p.N, p.K);
  LSK_REQUIRE(which >= 0, "fp8 product: grid too large");
  return LSK_OK;
}

static int fp8_product(const Fp8Args& p, hipStream_t s) {
  const int which = fp8_choice(p.M, p.N, p.K, p.E, p.out_dtype), rc = fp8_check_launch(p, which);
  return rc ? rc : fp8_launch(which, p, s);
}

// The columns of a block that quantises its rows itself: one group of 16 while a block a CU and a few more hold them,
// else two, then four; the borders, 300 and 1600 groups, are thresholds.  (MI355X, in a graph, us with 16, 32 and 64:
// one row of 3584 on 4608 columns, 288 groups, 7.7, 8.3, 10.7, four rows 10.5, 10.0, 12.5, one of 768 4.7, 4.4, 4.5; one of
// 2048 on 4800, 300 groups, 6.4, 6.3, 7.6, on 5120 6.5, 6.3, 7.7, on 16384 11.0, 8.8, 8.8; one of 4096 on 25600, 1600
// groups, 28.0, 27.4, 24.5, on 28672 30.2, 28.8, 26.2; one of 3584 on 37888 29.0, 24.7, 25.0; sixteen of 1024 on 28672
// 21.3, 15.6, 11.1; 64 of 512 on 2048 5.7, 5.3, 5.3, 128 of 256 on 1024 5.7, 4.4, 4.6.  So up to 12 % from the best of
// the three for up to 16 rows, and 30 % for more, which always take 16.)
static int fp8_fused_columns(int64_t N) {
  const int64_t groups = (N + 15) / 16;
  return groups <= 300 ? 16 : groups <= 1600 ? 32 : 64;
}

// Whether a linear's rows are quantised in the product's launch, by every block: up to 16 while they hold few values, more
// while the blocks, of 16 rows each, are two a CU at most.  (MI355X, in a graph, us in one launch and in two: one row of 3584
// on 4608 columns 7.7, 9.8, of 14336 on 4096 19.7, 18.2, of 18944 on 3584 25.1, 21.1; 4 of 2048 on 1024 5.8, 8.3, of 5120 on
// 4096 11.1, 11.4, of 8192 on 4096 16.0, 13.5, of 4096 on 12000 17.3, 16.3; 12 of 1536 on 2048 7.7, 8.4; 16 of 1024 on 2048
// 6.8, 8.1, of 2048 10.2, 8.9; 64 of 512 on 2048 5.7, 8.3, 128 of 256 on 1024 5.7, 6.8, 200 of 1024 on 512 8.0, 8.6, and with
// more blocks 128 of 256 on 2048 8.8, 6.7, 96 of 1024 on 2048 10.0, 8.6.  A launch and a workspace less are 4 us of a
// caller's time besides, which is why one long row stays in one launch; in a replayed graph it is up to 19 % slower there.)
static bool fp8_fuses(int64_t M, int64_t N, int64_t K) {
  const int columns = fp8_fused_columns(N);
  if (K == 0 || !grid_ok((M + 15) / 16 * ((N + columns - 1) / columns), 256)) return false;
  return M <= 16 ? M * K <= (N <= 4096 ? 20480 : 16384) : K <= 1024 && M <= 16 * 512 && (M + 15) / 16 * ((N + 15) / 16) <= 512;
}

static int fp8_stream_fused(const Fp8Args& p, const void* x, int x_dtype, int64_t ldx, hipStream_t s) {
  const int columns = fp8_fused_columns(p.N);
  auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (columns == 16) return fp8_stream_launch<1, 1, 2, 4, DT>(p, x, ldx, s);
    if (columns == 32) return fp8_stream_launch<2, 1, 1, 3, DT>(p, x, ldx, s);
    return fp8_stream_launch<4, 1, 1, 2, DT>(p, x, ldx, s);
  };
  if (x_dtype == LSK_F32) return run(std::integral_constant<int, LSK_F32>{});
  if (x_dtype == LSK_BF16) return run(std::integral_constant<int, LSK_BF16>{});
  return run(std::integral_constant<int, LSK_F16>{});
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
  const int v = out_dtype == LSK_F32 ? 2 : 4;
  const int64_t total = M * (K / v), blocks = (total + 1023) / 1024;
  const dim3 grid((unsigned)(blocks < (1 << 22) ? blocks : (1 << 22))), blk(256);
  const int shift = block_rows == 128 ? 7 : 0;
  auto run = [&](auto odt) {
    hipLaunchKernelGGL((lsk::dequant_fp8_kernel<decltype(odt)::value>), grid, blk, 0, (hipStream_t)stream, q, scale, scale_m,
                       scale_b, shift, total, (uint32_t)(K / v), (uint32_t)(((1 << 22) + K / v - 1) / (K / v)), out);
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

// (a stride that nothing steps by may be any size)
static int fp8_scales_check(const char* who, int64_t M, int64_t K, int64_t& sm, int64_t& sb) {
  LSK_REQUIRE(sm >= 0 && sb >= 0, "%s: bad scale strides", who);
  if (M <= 1) sm = 0;
  if (K <= 128) sb = 0;
  LSK_REQUIRE(sm < (1LL << 31) && sb < (1LL << 31), "%s: bad scale strides", who);
  return LSK_OK;
}

extern "C" int lsk_gemm_fp8(const uint8_t* a, const float* a_scale, int64_t scale_m, int64_t scale_b, int64_t M, int64_t K,
                            const uint8_t* w, const float* w_scale, int64_t N, const float* bias, void* out, int out_dtype,
                            int64_t ldo, void* stream) {
  int rc = fp8_check("lsk_gemm_fp8", M, N, K, out_dtype, ldo);
  if (rc || (rc = fp8_scales_check("lsk_gemm_fp8", M, K, scale_m, scale_b))) return rc;
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
  if (lsk::fp8_fuses(M, N, K)) return 0;
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
  if (lsk::fp8_fuses(M, N, K)) {
    LSK_REQUIRE(lsk::fp8_reach(p), "lsk_linear_fp8: N=%lld K=%lld beyond 31-bit offsets", (long long)N, (long long)K);
    return lsk::fp8_stream_fused(p, x, x_dtype, ldx, s);
  }
  int rows;
  LSK_REQUIRE(K == 0 || grid_ok(lsk::quantize_rows_blocks(M, K, rows), 256), "lsk_linear_fp8: grid too large");
  const int which = lsk::fp8_choice(M, N, K, 0, out_dtype);
  if ((rc = lsk::fp8_check_launch(p, which))) return rc;  // (before anything is launched)
  if (K > 0 && (rc = lsk::quantize_rows_launch(x, x_dtype, M, K, ldx, q, qs, 1, M, s))) return rc;
  return lsk::fp8_launch(which, p, s);
}

extern "C" int lsk_grouped_gemm_fp8(const uint8_t* a, const float* a_scale, int64_t scale_m, int64_t scale_b,
                                    const int32_t* offs, int64_t E, int64_t R, const int64_t* w_ptrs, int64_t ldw,
                                    const int64_t* ws_ptrs, int64_t ldsw, const int64_t* b_ptrs, int64_t N, int64_t K,
                                    void* out, int out_dtype, int64_t ldo, void* stream) {
  int rc = fp8_check("lsk_grouped_gemm_fp8", R, N, K, out_dtype, ldo);
  if (rc || (rc = fp8_scales_check("lsk_grouped_gemm_fp8", R, K, scale_m, scale_b))) return rc;
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

extern "C" int lsk_fp8_launch(int64_t M, int64_t N, int64_t K, int64_t E, int out_dtype) {
  if (M < 1 || N < 1 || K < 0 || K % 16 || E < 0 || M > 0x7fffffff || N > 0x7fffffff || K >= (1 << 22) || E > (1 << 20) ||
      !lsk::is_float_dtype(out_dtype))
    return -1;
  return lsk::fp8_choice(M, N, K, E, out_dtype);
}
