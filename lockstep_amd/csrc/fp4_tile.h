// Main loops of the MXFP4 products' tiles on gfx950's block-scaled matrix core.
//
// A block computes a BM x BN tile of A * W^T over all of K.  With eight waves it does so as pp_tile.h
// does for int8: two groups of four waves half a period apart, one reading its operands from LDS while the
// other multiplies, K staged 128 (or 256) values at a time through a ring of LDS stages that direct
// global -> LDS loads fill RING - 1 stages ahead.  A 128-value stage of a row is 64 bytes of codes and
// one dword of four scale bytes.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 on fp4: lane l supplies the 16 code bytes of block l / 32 of the
// 64 values and that block's scale byte, for row l % 32 of either operand.  Weight rows go in as the
// instruction's rows and activation rows as its columns, so register r of lane l holds output row
// l % 32 and columns 8 (r / 4) + 4 (l / 32) + r % 4: four consecutive outputs of one row.  Every output
// is one chain over ascending K (fp4.hip).
//
// The scales come transposed, [stage of 128 values][row] dwords, so that a stage's scales of a tile
// are two contiguous runs and one load instruction a wave; lane l takes the bytes of its half by a
// shift, the instruction's byte selector the block within it.
#pragma once
#include <type_traits>

#include "mfma_tile.h"
#include "pp_tile.h"

namespace lsk {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

LSK_DEV v8i fp4_operand(v4i x) { return v8i{x[0], x[1], x[2], x[3], 0, 0, 0, 0}; }

template <int BM, int BN, int WM, int WN, int RING, int BKB>
struct Fp4Cfg {
  static_assert(WM * WN == 8 || WM * WN == 4, "eight waves (ping-pong) or four");
  static_assert(RING >= (WM * WN == 8 ? 3 : 2), "ring of stages");
  static_assert(BKB == 64 || BKB == 128, "stages of 128 or 256 values");
  static constexpr int kThreads = WM * WN * 64, kBM = BM, kBN = BN, kWM = WM, kWN = WN;
  static_assert(BM + BN <= kThreads, "one scale dword per thread and 128 values");
  static constexpr int kRing = RING, kAhead = RING - 1;
  static constexpr int kChunks = BKB / 16, kSub = BKB / 64;  // 16-byte chunks and 128-value parts of a stage
  static constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 32, TN = WTN / 32;
  static constexpr int kStageA = BM * BKB, kStageB = BN * BKB, kScale = kThreads * 4 * kSub;
  static constexpr int kStage = kStageA + kStageB + kScale;
  static constexpr int kLA = kStageA / 16 / kThreads, kLB = kStageB / 16 / kThreads;
  static constexpr int kPer = kLA + kLB + kSub;  // loads per thread per stage
  static constexpr int kMainBytes = kRing * kStage;
  static constexpr int kLdc = WTN + 4;           // floats a row of a staged 32-row strip
  static constexpr int kEpiBytes = WM * WN * 32 * kLdc * 4;
  static constexpr int kSmemBytes = kMainBytes > kEpiBytes ? kMainBytes : kEpiBytes;
  static_assert(kStageA % (16 * kThreads) == 0 && kStageB % (16 * kThreads) == 0, "tile / threads");
  static_assert(WTM % 32 == 0 && WTN % 32 == 0, "wave tile must be a multiple of 32");
  static_assert(kSmemBytes <= 160 * 1024, "LDS");
  typedef v16f Acc[TM][TN];
};

// This thread's part of a tile's loads: its rows' offsets in the resources over the tile's codes (kOob:
// no row), its dword's offset in the one over the transposed scales from the tile's first row on, and
// the bytes between the scales of two stages.
template <class C>
struct Fp4Rows {
  uint32_t a[C::kLA], b[C::kLB], s;
  uint32_t sta, stb;
};

template <int BM, int BN, int WM, int WN, int RING, int BKB>
LSK_DEV void fp4_mainloop(typename Fp4Cfg<BM, BN, WM, WN, RING, BKB>::Acc& acc, __amdgpu_buffer_rsrc_t ra, __amdgpu_buffer_rsrc_t rb,
                          __amdgpu_buffer_rsrc_t rsa, __amdgpu_buffer_rsrc_t rsb,
                          const Fp4Rows<Fp4Cfg<BM, BN, WM, WN, RING, BKB>>& t, int K, char* smem) {
  using C = Fp4Cfg<BM, BN, WM, WN, RING, BKB>;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int group = wave >> 2, wm = wave / C::kWN, wn = wave % C::kWN;
  const int Kb = K / 2, nk = (Kb + BKB - 1) / BKB;
  // (whether this wave's scale dwords are the activations' or the weights': BM is a multiple of 64)
  const bool sc_a = wave * 64 < C::kBM;
  const __amdgpu_buffer_rsrc_t rs = sc_a ? rsa : rsb;
  const uint32_t st = sc_a ? t.sta : t.stb;

  int ka[C::kLA], kb[C::kLB];
#pragma unroll
  for (int j = 0; j < C::kLA; ++j) {
    int r;
    pp_slot<C::kThreads, C::kChunks>(tid, j, r, ka[j]);
  }
#pragma unroll
  for (int j = 0; j < C::kLB; ++j) {
    int r;
    pp_slot<C::kThreads, C::kChunks>(tid, j, r, kb[j]);
  }
  const int nst = (K + 127) / 128;
  auto issue = [&](int s, auto check) {
    constexpr bool kCheck = decltype(check)::value;
    char* base = smem + (s % C::kRing) * C::kStage;
    const int k0 = s * BKB;
#pragma unroll
    for (int j = 0; j < C::kLA; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void_t)(base + (j * C::kThreads + wave * 64) * 16), 16,
                                               (!kCheck || k0 + ka[j] < Kb) ? t.a[j] + (uint32_t)(k0 + ka[j]) : kOob, 0, 0,
                                               0);
#pragma unroll
    for (int j = 0; j < C::kLB; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rb, (lds_void_t)(base + C::kStageA + (j * C::kThreads + wave * 64) * 16), 16,
          (!kCheck || k0 + kb[j] < Kb) ? t.b[j] + (uint32_t)(k0 + kb[j]) : kOob, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < C::kSub; ++u)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (lds_void_t)(base + C::kStageA + C::kStageB + (u * C::kThreads + wave * 64) * 4), 4,
          (!kCheck || s * C::kSub + u < nst) ? t.s : kOob, (int)((uint32_t)(s * C::kSub + u) * st), 0, 0);
  };

  const int lr = lane & 31, sw = pp_swz<C::kChunks>(lr), kg = lane >> 5;
  const int offA = (wm * C::WTM + lr) * BKB, offB = C::kStageA + (wn * C::WTN + lr) * BKB;
  const int offS = C::kStageA + C::kStageB + 4 * lr;
  const int sA = offS + 4 * wm * C::WTM, sB = offS + 4 * (C::kBM + wn * C::WTN);
  int slot[2 * C::kSub];
#pragma unroll
  for (int ks = 0; ks < 2 * C::kSub; ++ks) slot[ks] = 16 * ((2 * ks + kg) ^ sw);

  if constexpr (C::kThreads == 256) {
    // Four waves, one barrier a stage.  RING > 2: a stage's fragments are read into registers a stage ahead,
    // so that the LDS works under the matrix core's chain (200 rows of 3584 x 18944 on 64 x 64 tiles 28.4 ->
    // 24.2 us on MI355X).  A wave's own loads of stage kt + 1 are complete when at most the RING - 3 younger
    // stages are outstanding, every wave's at the barrier; the slot of stage kt - 1, whose fragments every
    // wave has multiplied, takes stage kt + RING - 1.  RING 2 reads a stage when it multiplies it, and loads
    // the next one meanwhile: with two or three blocks a CU the other blocks fill the gaps (777 rows of 4608
    // x 3584 on 64 x 128 tiles 16.6 us, 18.4 with the longer ring).  Past the last stage the loads read
    // zeros, so the count of outstanding loads is the same to the end.
    struct Frag {
      v4i a[2 * C::kSub][C::TM], b[2 * C::kSub][C::TN];
      int xa[C::kSub][C::TM], xb[C::kSub][C::TN];
    };
    auto read = [&](int kt, Frag& f) {
      const char* base = smem + (kt % RING) * C::kStage;
#pragma unroll
      for (int u = 0; u < C::kSub; ++u) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i) f.xa[u][i] = *(const int*)(base + sA + u * 4 * C::kThreads + i * 128);
#pragma unroll
        for (int j = 0; j < C::TN; ++j) f.xb[u][j] = *(const int*)(base + sB + u * 4 * C::kThreads + j * 128);
      }
#pragma unroll
      for (int h = 0; h < 2 * C::kSub; ++h) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i) f.a[h][i] = *(const v4i*)(base + offA + i * 32 * BKB + slot[h]);
#pragma unroll
        for (int j = 0; j < C::TN; ++j) f.b[h][j] = *(const v4i*)(base + offB + j * 32 * BKB + slot[h]);
      }
    };
    auto multiply = [&](Frag& f) {
#pragma unroll
      for (int u = 0; u < C::kSub; ++u) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i) f.xa[u][i] = (int)((uint32_t)f.xa[u][i] >> (8 * kg));
#pragma unroll
        for (int j = 0; j < C::TN; ++j) f.xb[u][j] = (int)((uint32_t)f.xb[u][j] >> (8 * kg));
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int j = 0; j < C::TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(f.b[2 * u][j]), fp4_operand(f.a[2 * u][i]),
                                                                        acc[i][j], 4, 4, 0, f.xb[u][j], 0, f.xa[u][i]);
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int j = 0; j < C::TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(f.b[2 * u + 1][j]),
                                                                        fp4_operand(f.a[2 * u + 1][i]), acc[i][j], 4, 4, 2,
                                                                        f.xb[u][j], 2, f.xa[u][i]);
      }
    };
    if constexpr (RING == 2) {
      Frag f;
      issue(0, std::true_type{});
      for (int kt = 0; kt < nk; ++kt) {
        wait_vm<0>();
        phase_barrier();
        issue(kt + 1, std::true_type{});
        read(kt, f);
        multiply(f);
      }
    } else {
      Frag f[2];
#pragma unroll
      for (int s = 0; s < RING - 1; ++s) issue(s, std::true_type{});
      wait_vm<(RING - 2) * C::kPer>();
      phase_barrier();
      read(0, f[0]);
      auto step = [&](int kt, Frag& now, Frag& next) {
        compiler_fence();  // (the reads of the stage before stay on their side of the barrier)
        wait_vm<(RING - 3) * C::kPer>();
        phase_barrier();
        issue(kt + RING - 1, std::true_type{});
        read(kt + 1, next);
        multiply(now);
      };
      int kt = 0;
      for (; kt + 2 <= nk; kt += 2) {
        step(kt, f[0], f[1]);
        step(kt + 1, f[1], f[0]);
      }
      if (kt < nk) step(kt, f[0], f[1]);
    }
    wait_vm<0>();
  } else {
    using Chk = std::true_type;
    using NoChk = std::false_type;
    using W0 = std::integral_constant<int, 0>;
    auto step = [&](int kt, auto wait_n, bool do_issue, auto check) {
      constexpr int kWait = decltype(wait_n)::value;
      if (do_issue) issue(kt + C::kAhead, check);
      const char* base = smem + (kt % C::kRing) * C::kStage;
      v4i fa[2 * C::kSub][C::TM], fb[2 * C::kSub][C::TN];
      int xa[C::kSub][C::TM], xb[C::kSub][C::TN];
#pragma unroll
      for (int u = 0; u < C::kSub; ++u) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i) xa[u][i] = *(const int*)(base + sA + u * 4 * C::kThreads + i * 128);
#pragma unroll
        for (int j = 0; j < C::TN; ++j) xb[u][j] = *(const int*)(base + sB + u * 4 * C::kThreads + j * 128);
      }
#pragma unroll
      for (int ks = 0; ks < 2 * C::kSub; ++ks) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i) fa[ks][i] = *(const v4i*)(base + offA + i * 32 * BKB + slot[ks]);
#pragma unroll
        for (int j = 0; j < C::TN; ++j) fb[ks][j] = *(const v4i*)(base + offB + j * 32 * BKB + slot[ks]);
      }
      wait_vm<kWait>();
      wait_lgkm0();
#pragma unroll
      for (int u = 0; u < C::kSub; ++u) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i) xa[u][i] = (int)((uint32_t)xa[u][i] >> (8 * kg));
#pragma unroll
        for (int j = 0; j < C::TN; ++j) xb[u][j] = (int)((uint32_t)xb[u][j] >> (8 * kg));
      }
      phase_barrier();
#pragma unroll
      for (int u = 0; u < C::kSub; ++u) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int j = 0; j < C::TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(fb[2 * u][j]), fp4_operand(fa[2 * u][i]),
                                                                        acc[i][j], 4, 4, 0, xb[u][j], 0, xa[u][i]);
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int j = 0; j < C::TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                fp4_operand(fb[2 * u + 1][j]), fp4_operand(fa[2 * u + 1][i]), acc[i][j], 4, 4, 2, xb[u][j], 2, xa[u][i]);
      }
      phase_barrier();
    };

#pragma unroll
    for (int s = 0; s < C::kAhead; ++s)
      if (s < nk) issue(s, Chk{});
    wait_vm<0>();
    phase_barrier();
    if (group == 1) phase_barrier();
    if (nk >= C::kAhead) {
      using WSteady = std::integral_constant<int, (C::kAhead - 1) * C::kPer>;
      const int nfull = Kb / BKB;
      int kt = 0;
      for (; kt + C::kAhead < nfull; ++kt) step(kt, WSteady{}, true, NoChk{});
      for (; kt + C::kAhead < nk; ++kt) step(kt, WSteady{}, true, Chk{});
      step(kt, std::integral_constant<int, (C::kAhead - 2) * C::kPer>{}, false, NoChk{});
      step(kt + 1, std::integral_constant<int, (C::kAhead >= 3 ? C::kAhead - 3 : 0) * C::kPer>{}, false, NoChk{});
      if (C::kAhead >= 3) step(kt + 2, std::integral_constant<int, (C::kAhead >= 4 ? C::kAhead - 4 : 0) * C::kPer>{}, false, NoChk{});
      if (C::kAhead >= 4) step(kt + 3, W0{}, false, NoChk{});
    } else {
      for (int kt = 0; kt < nk; ++kt) step(kt, W0{}, false, NoChk{});
    }
    if (group == 0) phase_barrier();
  }
}

}  // namespace lsk
