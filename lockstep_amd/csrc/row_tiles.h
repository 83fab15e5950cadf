// What the products of quantised rows share (MXFP4: fp4.hip, fp8: fp8.hip): their inputs by type and
// alignment, the row tiles of expert-sorted rows, the outputs' stores and the workspaces' checks.
#pragma once
#include <type_traits>

#include "lsk_common.h"

namespace lsk {

// Eight elements from element i on, in 16-byte loads (VEC: aligned for them) or one by one.
template <int DT, bool VEC>
LSK_DEV void load8(const void* x, int64_t i, float (&v)[8]) {
  if constexpr (VEC) {
    load8_as_f32<DT>((const char*)x + i * (DT == LSK_F32 ? 4 : 2), 0, v);
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = load_as_f32(x, DT, i + t);
  }
}

// The same in two steps, so that the loads of many stand under one another's latency: raw8 loads, zeros where `in` does
// not hold (x's first eight elements are read there and left), raw8_values converts.  (Under a condition each load was
// waited for before the next went out: the norm of 8192 rows of 4096, fp8 rows out, 55 us, so 47.)
template <int DT, bool VEC>
struct Raw8 {
  static constexpr int kWords = VEC && DT != LSK_F32 ? 4 : 8;
  uint32_t w[kWords];
};

template <int DT, bool VEC>
LSK_DEV Raw8<DT, VEC> raw8(const void* x, int64_t i, bool in) {
  Raw8<DT, VEC> r;
  i = in ? i : 0;
  if constexpr (VEC) {
    const v4u32* const p = (const v4u32*)((const char*)x + i * (DT == LSK_F32 ? 4 : 2));
#pragma unroll
    for (int h = 0; h < Raw8<DT, VEC>::kWords / 4; ++h) {
      const v4u32 a = p[h];
#pragma unroll
      for (int t = 0; t < 4; ++t) r.w[4 * h + t] = in ? a[t] : 0;
    }
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const uint32_t a = DT == LSK_F32 ? ((const uint32_t*)x)[i + t] : ((const uint16_t*)x)[i + t];
      r.w[t] = in ? a : 0;
    }
  }
  return r;
}

template <int DT, bool VEC>
LSK_DEV void raw8_values(const Raw8<DT, VEC>& r, float (&v)[8]) {
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const uint32_t w = VEC && DT != LSK_F32 ? (t & 1 ? r.w[t / 2] >> 16 : r.w[t / 2] & 0xffff) : r.w[t];
    if constexpr (DT == LSK_F32) v[t] = __uint_as_float(w);
    else if constexpr (DT == LSK_BF16) v[t] = __uint_as_float(w << 16);
    else v[t] = (float)__builtin_bit_cast(_Float16, (uint16_t)w);
  }
}

// f(dtype, vec) with the dtype and the alignment of x's rows as compile-time values.
template <class F>
inline void by_input(const void* x, int x_dtype, int64_t ldx, F f) {
  const int size = x_dtype == LSK_F32 ? 4 : 2;
  const bool vec = (uintptr_t)x % 16 == 0 && (ldx * size) % 16 == 0;
  auto with = [&](auto dt) { vec ? f(dt, std::true_type{}) : f(dt, std::false_type{}); };
  if (x_dtype == LSK_F32) with(std::integral_constant<int, LSK_F32>{});
  else if (x_dtype == LSK_BF16) with(std::integral_constant<int, LSK_BF16>{});
  else with(std::integral_constant<int, LSK_F16>{});
}

// Inclusive scans over the wave by DPP row shifts and broadcasts (lanes without a source keep `ident`).
template <class Op>
LSK_DEV int wave_scan(int v, int ident, Op op) {
  v = op(v, __builtin_amdgcn_update_dpp(ident, v, 0x111, 0xf, 0xf, false));  // row_shr:1
  v = op(v, __builtin_amdgcn_update_dpp(ident, v, 0x112, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(ident, v, 0x114, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(ident, v, 0x118, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(ident, v, 0x142, 0xa, 0xf, false));  // row_bcast:15
  v = op(v, __builtin_amdgcn_update_dpp(ident, v, 0x143, 0xc, 0xf, false));  // row_bcast:31
  return v;
}

// Row tiles of expert-sorted rows, bm rows each, counted over the experts in order.  Offsets that
// decrease or leave [0, R] are taken as min(R, max(0, offs[0..j])), so that experts come out empty or
// shortened and no row outside [0, R) is touched.  Every wave looks its tile up itself, 64 experts a
// step: no table to build in a launch of its own.
struct ExpertTiles {
  const int32_t* offs;
  int E, R, bm;
  int carry, lo, hi, n, sum;  // of the last 64 experts looked at, one a lane; carry: the rows before them
  LSK_DEV ExpertTiles(const int32_t* o, int e, int r, int b) : offs(o), E(e), R(r), bm(b) { restart(); }
  LSK_DEV void restart() {
    carry = min(max(offs[0], 0), R);
    look(0);
  }
  LSK_DEV void look(int e0) {
    const int lane = threadIdx.x & 63;
    hi = wave_scan(min(max(offs[min(e0 + lane + 1, E)], 0), R), 0, [](int a, int b) { return max(a, b); });
    hi = max(hi, carry);
    lo = __shfl_up(hi, 1, 64);
    if (lane == 0) lo = carry;
    n = (int)((unsigned)(hi - lo + bm - 1) / (unsigned)bm);
    sum = wave_scan(n, 0, [](int a, int b) { return a + b; });
  }
  LSK_DEV void next(int e0) {
    carry = __builtin_amdgcn_readlane(hi, 63);
    look(e0);
  }
  // how many tiles there are
  LSK_DEV int count() {
    int total = __builtin_amdgcn_readlane(sum, 63);
    for (int e0 = 64; e0 < E; e0 += 64) {
      next(e0);
      total += __builtin_amdgcn_readlane(sum, 63);
    }
    if (E > 64) restart();
    return total;
  }
  // tile t: its expert, first row and the end of the expert's rows; false past the last tile
  LSK_DEV bool find(int t, int& e, int& m0, int& m1) {
    for (int e0 = 0;;) {
      const uint64_t past = __builtin_amdgcn_ballot_w64(sum > t);
      if (past) {
        const int l = __builtin_ctzll(past);
        e = e0 + l;
        m0 = __builtin_amdgcn_readlane(lo, l) +
             (t - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l))) * bm;
        m1 = __builtin_amdgcn_readlane(hi, l);
        return true;
      }
      t -= __builtin_amdgcn_readlane(sum, 63);
      e0 += 64;
      if (e0 >= E) return false;
      next(e0);
    }
  }
};
inline int64_t expert_tiles_max(int64_t R, int64_t E, int64_t bm) { return R / bm + (E < R ? E : R); }

// Four outputs to consecutive places (8-byte, for binary32 16-byte aligned), rounded to the type; a NaN
// to bf16 becomes 0x7FC0, off the common path (v0 + v1 + v2 + v3 is a NaN where one of them is).
// Non-temporal: an output stays in no L2 past its launch, and within it leaves the L2 to the operands
// (4096 rows of 28672 x 4096 321 -> 293 us on MI355X, 777 of 4608 x 3584 21.9 -> 20.6).
// NT false: as any other store, for rows that share their lines with others' (fp8.hip).
template <bool NT = true>
LSK_DEV void store_quad(char* o, int dtype, v4f v) {
  auto put = [&](char* at, uint32_t lo, uint32_t hi) {
    if constexpr (NT) __builtin_nontemporal_store((uint64_t)hi << 32 | lo, (uint64_t*)at);
    else *(uint64_t*)at = (uint64_t)hi << 32 | lo;
  };
  if (dtype == LSK_F32) {
    put(o, __float_as_uint(v[0]), __float_as_uint(v[1]));
    __asm__ volatile("" ::: "memory");  // (no 16-byte stores: store16_split)
    put(o + 8, __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else if (dtype == LSK_BF16) {
    const float s = (v[0] + v[1]) + (v[2] + v[3]);
    uint32_t lo = pack_bf16x2_nonan(v[0], v[1]), hi = pack_bf16x2_nonan(v[2], v[3]);
    if (__builtin_amdgcn_ballot_w64(s != s)) lo = pack_bf16x2(v[0], v[1]), hi = pack_bf16x2(v[2], v[3]);
    put(o, lo, hi);
    __asm__ volatile("" ::: "memory");  // (merged with the one below, a store is no longer a non-temporal one)
  } else {
    put(o, (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[0]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[1]) << 16),
        (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[3]) << 16));
  }
}

inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

inline bool is_float_dtype(int d) { return d == LSK_F32 || d == LSK_BF16 || d == LSK_F16; }

inline bool work_ok(const void* w, int64_t have, int64_t need) {
  return have >= need && (need == 0 || (w && (uintptr_t)w % 256 == 0));
}

}  // namespace lsk
