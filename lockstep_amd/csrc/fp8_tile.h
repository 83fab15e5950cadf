// Main loop of the fp8 products' tiles on gfx950's matrix core.
//
// A block computes a BM x BN tile of A * W^T over all of K, a stage of 128 values (one block of the scales)
// at a time through a ring of LDS stages that direct global -> LDS loads fill.  A stage's products are one
// v_mfma_f32_16x16x128_f8f6f4 per 16 x 16 outputs from +0, added to the running sum times the two scales
// with one FMA an output (fp8.hip): four VALU cycles of every eight of the matrix core, in its shadow.
//
// Lane l of that instruction supplies 32 bytes of row l % 16 of either operand: bytes 16 q .. + 15 and
// 64 + 16 q .. + 15 of the 128, q = l / 16 (any division of the 128 that both operands share gives the
// product; this one makes each half one 16-byte LDS read without bank conflicts).  Weight rows go in as
// the instruction's rows and activation rows as its columns, so register r of lane l holds output row
// l % 16 and column 4 (l / 16) + r: four consecutive outputs of one row, and one activation scale a lane.
#pragma once
#include <type_traits>

#include "mfma_tile.h"
#include "pp_tile.h"

namespace lsk {

typedef int v8i __attribute__((ext_vector_type(8)));

LSK_DEV v8i fp8_operand(v4i lo, v4i hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

// The sums of products of one block of 128 values, from +0.  EXACT: the values widened to bf16 (which holds
// e4m3) and multiplied there, products kept whole and summed in binary32.  The fp8 instruction sums eight
// products at a time on the scale of the largest, keeping 13 bits below it (MI355X: 2^16 + 2^3 is kept, 2^2
// dropped): 1.4e-5 of the result on normal data, nothing next to a bf16's or f16's 2^-9 or 2^-12, but not what a
// binary32 output is for.
template <bool EXACT>
LSK_DEV v4f fp8_block(v8i w, v8i a) {
  const v4f zero = {0, 0, 0, 0};
  if constexpr (!EXACT) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, zero, 0, 0, 0, 0, 0, 0);
  } else {
    typedef __bf16 v8b __attribute__((ext_vector_type(8)));
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    v4f p = zero;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      v8b x, y;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const v2b x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)w[k + h], 1.0f, false);
        const v2b x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)w[k + h], 1.0f, true);
        const v2b y0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)a[k + h], 1.0f, false);
        const v2b y1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)a[k + h], 1.0f, true);
        x[4 * h] = x0[0], x[4 * h + 1] = x0[1], x[4 * h + 2] = x1[0], x[4 * h + 3] = x1[1];
        y[4 * h] = y0[0], y[4 * h + 1] = y0[1], y[4 * h + 2] = y1[0], y[4 * h + 3] = y1[1];
      }
      p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, p, 0, 0, 0);
    }
    return p;
  }
}

// acc + p * s, one rounding an output.
LSK_DEV v4f fp8_scaled(v4f p, float s, v4f acc) {
#pragma unroll
  for (int t = 0; t < 4; ++t) acc[t] = __builtin_fmaf(p[t], s, acc[t]);
  return acc;
}

template <int BM, int BN, int WM, int WN, int RING>
struct Fp8Cfg {
  static_assert(WM * WN == 8 || WM * WN == 4, "eight waves (ping-pong) or four");
  static_assert(RING >= 2 && (WM * WN == 4 || RING == 2), "ring of stages");
  static constexpr int kThreads = WM * WN * 64, kBM = BM, kBN = BN, kWM = WM, kWN = WN, kRing = RING;
  static constexpr int kNB = BN > 128 ? BN / 128 : 1;  // weight scales of a stage
  static_assert(BM % 64 == 0 && BM + kNB <= kThreads, "one scale a thread");
  static constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
  static_assert(WTM % 16 == 0 && WTN % 16 == 0 && 128 % WTN == 0, "a wave's columns share a weight scale");
  static constexpr int kStageA = BM * 128, kStageB = BN * 128, kStage = kStageA + kStageB + kThreads * 4;  // bytes
  static constexpr int kLA = kStageA / 16 / kThreads, kLB = kStageB / 16 / kThreads;
  static constexpr int kPer = kLA + kLB + 1;  // loads per thread per stage
  static_assert(kStageA % (16 * kThreads) == 0 && kStageB % (16 * kThreads) == 0, "tile / threads");
  static constexpr int kMainBytes = kRing * kStage;
  static constexpr int kLdc = WTN + 4;  // floats a row of a staged 16-row strip
  static constexpr int kEpiBytes = WM * WN * 16 * kLdc * 4;
  static constexpr int kSmemBytes = kMainBytes > kEpiBytes ? kMainBytes : kEpiBytes;
  static_assert(kSmemBytes <= 160 * 1024, "LDS");
  typedef v4f Acc[TM][TN];
};

// Where a tile's operands lie: resources over its rows from its first one on, the bytes from a row to the next, how
// many rows there are, and this thread's scale in the resource over the tile's scales (kOob: none) with the bytes
// between the scales of two stages.
struct Fp8Tile {
  __amdgpu_buffer_rsrc_t ra, rb, rsa, rsb;
  int lda, ldb, rows_a, rows_b;
  uint32_t s, sta;
};

template <int BM, int BN, int WM, int WN, int RING, bool EXACT>
LSK_DEV void fp8_mainloop(typename Fp8Cfg<BM, BN, WM, WN, RING>::Acc& acc, const Fp8Tile& t, int K, char* smem) {
  using C = Fp8Cfg<BM, BN, WM, WN, RING>;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int wm = wave / C::kWN, wn = wave % C::kWN;
  const int nk = (K + 127) / 128;
  const bool sc_a = wave * 64 < C::kBM;  // (a wave's scales are all the rows' or all the weights')
  const __amdgpu_buffer_rsrc_t rs = sc_a ? t.rsa : t.rsb;
  const uint32_t st = sc_a ? t.sta : 4;

  // A thread loads one chunk of every kThreads / 8-th row, the same chunk of each: its first row's offset is a
  // lane's, the rest is added by a scalar, which the range check leaves out.
  constexpr int kStep = C::kThreads / 8;
  static_assert(kStep % 16 == 0, "rows a step apart share their swizzle");
  int r0, kc;
  pp_slot<C::kThreads, 8>(tid, 0, r0, kc);
  const uint32_t offa = (uint32_t)(r0 * t.lda + kc), offb = (uint32_t)(r0 * t.ldb + kc);
  // Load l of stage s (chunks past K, and past the last stage, read zeros, and so do rows past the last).
  auto load = [&](int s, int l) {
    char* base = smem + (s % C::kRing) * C::kStage + wave * 1024;
    const int k0 = s * 128;
    const bool in = k0 + kc < K;
    if (l < C::kLA)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(t.ra, (lds_void_t)(base + l * C::kThreads * 16), 16,
                                               in && r0 + l * kStep < t.rows_a ? offa : kOob, k0 + l * kStep * t.lda, 0, 0);
    else if (l < C::kLA + C::kLB)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(t.rb, (lds_void_t)(base + l * C::kThreads * 16), 16,
                                               in && r0 + (l - C::kLA) * kStep < t.rows_b ? offb : kOob,
                                               k0 + (l - C::kLA) * kStep * t.ldb, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t)(base + C::kStageA + C::kStageB - wave * 768), 4,
                                               s < nk ? t.s : kOob, (int)((uint32_t)s * st), 0, 0);
  };
  auto issue = [&](int s) {
#pragma unroll
    for (int l = 0; l < C::kPer; ++l) load(s, l);
  };

  const int lr = lane & 15, q = lane >> 4, sw = pp_swz<8>(lr);
  const int offA = (wm * C::WTM + lr) * 128, offB = C::kStageA + (wn * C::WTN + lr) * 128;
  const int offS = C::kStageA + C::kStageB, sA = offS + 4 * (wm * C::WTM + lr), sB = offS + 4 * (C::kBM + wn * C::WTN / 128);
  const int lo = 16 * (q ^ sw), hi = 16 * ((q + 4) ^ sw);

  struct Frag {
    v8i a[C::TM], b[C::TN];
    float s[C::TM];
  };
  auto read = [&](int kt, Frag& f) {
    const char* base = smem + (kt % C::kRing) * C::kStage;
    const float sb = *(const float*)(base + sB);
#pragma unroll
    for (int i = 0; i < C::TM; ++i) f.s[i] = f32_mul(*(const float*)(base + sA + i * 64), sb);
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
      f.b[j] = fp8_operand(*(const v4i*)(base + offB + j * 2048 + lo), *(const v4i*)(base + offB + j * 2048 + hi));
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
      f.a[i] = fp8_operand(*(const v4i*)(base + offA + i * 2048 + lo), *(const v4i*)(base + offA + i * 2048 + hi));
  };
  // Three products ahead of the FMAs that use them: a result takes the matrix core's eight passes and three more to
  // come back, and a wave that waited for each would leave the core idle as long (MI355X, builds in turn, in the compiler's
  // order, two and three ahead: 256 x 256 tiles, 4096 rows of 28672 x 4096, 436, 442, 422 us; 128 x 128, 2048 of 4096 x 4096,
  // 39.7, 38.9, 37.8; by expert, where loads bound the tiles, 16384 over 32 of 5760 x 2880 398, 422, 416).
  constexpr int kTiles = C::TM * C::TN, kDepth = kTiles < 3 ? kTiles : 3;
  constexpr int kEvery = kTiles / C::kPer > 0 ? kTiles / C::kPer : 1;  // products to a load
  static_assert(C::kThreads == 256 || kTiles >= C::kPer, "a stage's loads fit among its products");
  // with: the loads of stage s among the products.  (Every caller raises the wave's priority for them: the SIMD's other
  // waves read and issue loads meanwhile, and take their slots otherwise; without and with, builds in turn: 256 x 256 tiles
  // on 4096 rows of 28672 x 4096 429, 422 us, 128 x 128 on 2048 of 4096 x 4096 41.6, 37.8; by expert 16384 rows over 32 of
  // 5760 x 2880 410, 416.)
  auto multiply = [&](const Frag& f, auto with, int s) {
    constexpr bool kWith = decltype(with)::value;
    if constexpr (EXACT) {
      if (kWith) issue(s);
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int j = 0; j < C::TN; ++j) acc[i][j] = fp8_scaled(fp8_block<true>(f.b[j], f.a[i]), f.s[i], acc[i][j]);
    } else {
      v4f p[kDepth + 1];
#pragma unroll
      for (int n = 0; n < kDepth; ++n) p[n] = fp8_block<false>(f.b[n % C::TN], f.a[n / C::TN]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const int z = n + kDepth;
        if (z < kTiles) p[z % (kDepth + 1)] = fp8_block<false>(f.b[z % C::TN], f.a[z / C::TN]);
        if constexpr (kWith)
          if (n % kEvery == 0 && n / kEvery < C::kPer) load(s, n / kEvery);
        acc[n / C::TN][n % C::TN] = fp8_scaled(p[n % (kDepth + 1)], f.s[n / C::TN], acc[n / C::TN][n % C::TN]);
        __builtin_amdgcn_sched_barrier(0);  // (in this order)
      }
    }
  };

  Frag f;
  if constexpr (C::kThreads == 256) {
    if constexpr (RING < 4) {
      // One barrier a stage: a wave's own loads of stage kt are complete when at most the RING - 2 younger
      // stages are outstanding, every wave's at the barrier; the slot of stage kt - 1, which every wave has read
      // by then, takes stage kt + RING - 1.
#pragma unroll
      for (int s = 0; s < RING - 1; ++s) issue(s);
      for (int kt = 0; kt < nk; ++kt) {
        wait_vm<(RING - 2) * C::kPer>();
        phase_barrier();
        issue(kt + RING - 1);
        read(kt, f);
        __builtin_amdgcn_s_setprio(1);
        multiply(f, std::false_type{}, 0);
        __builtin_amdgcn_s_setprio(0);
      }
    } else {
      // The same with a stage's fragments read a stage ahead of its products.
      Frag g;
#pragma unroll
      for (int s = 0; s < RING - 1; ++s) issue(s);
      wait_vm<(RING - 2) * C::kPer>();
      phase_barrier();
      read(0, f);
      auto step = [&](int kt, Frag& now, Frag& next) {
        compiler_fence();  // (the reads of the stage before stay on their side of the barrier)
        wait_vm<(RING - 3) * C::kPer>();
        phase_barrier();
        issue(kt + RING - 1);
        read(kt + 1, next);
        __builtin_amdgcn_s_setprio(1);
        multiply(now, std::false_type{}, 0);
        __builtin_amdgcn_s_setprio(0);
      };
      int kt = 0;
      for (; kt + 2 <= nk; kt += 2) {
        step(kt, f, g);
        step(kt + 1, g, f);
      }
      if (kt < nk) step(kt, f, g);
    }
    wait_vm<0>();
  } else {
    // Two groups of four waves, half a period apart: while one multiplies stage kt the other reads its fragments
    // (group 0 reads in period 2 kt and multiplies in 2 kt + 1, group 1 a period later).  Both request stage kt + 1 in
    // period 2 kt, into the slot of stage kt - 1, which group 1 has read by the end of 2 kt - 1, and wait for it at the
    // end of 2 kt + 1.  Group 0 issues behind its reads and group 1 one request to every three products.  (All of
    // group 1's ahead of its products is no worse, builds in turn: so and ahead, 4096 rows of 28672 x 4096 422, 416 us, 32768
    // over 128 experts of 1536 x 2048 186, 181.)
    issue(0);
    wait_vm<0>();
    phase_barrier();
    if (wave < 4) {
      for (int kt = 0; kt < nk; ++kt) {
        read(kt, f);
        __builtin_amdgcn_sched_barrier(0);
        issue(kt + 1);
        wait_lgkm0();
        phase_barrier();
        __builtin_amdgcn_s_setprio(1);
        multiply(f, std::false_type{}, 0);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);  // (the wait stays behind the products)
        wait_vm<0>();
        phase_barrier();
      }
      phase_barrier();
    } else {
      issue(1);
      phase_barrier();
      for (int kt = 0; kt < nk; ++kt) {
        read(kt, f);
        wait_lgkm0();
        wait_vm<0>();
        phase_barrier();
        __builtin_amdgcn_s_setprio(1);
        multiply(f, std::true_type{}, kt + 2);
        __builtin_amdgcn_s_setprio(0);
        phase_barrier();
      }
      wait_vm<0>();
    }
  }
}

}  // namespace lsk
