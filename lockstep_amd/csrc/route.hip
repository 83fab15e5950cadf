// The choice of experts by softmax or sigmoid scores (beside the table scores of the contract's router, moe.hip).
//
// Per token, with logits l over E experts:
//   p_e = exp(l_e - max l) / sum exp(l - max l)   or   1 / (1 + exp(-l_e)),      c_e = p_e + bias_e
// The E experts lie in `groups` runs of one size; a group counts the sum of its `group_top` (1 or 2) largest c,
// the `keep` groups that count most stay, and of their experts the k largest c are chosen, larger ones first;
// of equals (groups and experts) the lower index.  The weights are p of the chosen, over their sum when
// renormalised, times `factor`.
//
// All of it in 64 bits, so that two experts whose scores differ in less than binary32 holds are still told apart;
// gfx950 computes 64-bit FMAs at the rate of 32-bit ones.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "lsk_common.h"

namespace lsk {

struct RouteArgs {
  const void* g;
  int g_dtype;
  int64_t ldg, T;
  int E, k, groups, keep, group_top;
  int sigmoid, renorm;
  double factor;
  const float* bias;
  int64_t* idx;
  void* w;
  int w_dtype;
};

// c as a whole number that orders the same: 0 is not to be chosen, 1 a NaN, above them -infinity and the rest.
LSK_DEV uint64_t rank_of(double c) {
  const uint64_t u = (uint64_t)__double_as_longlong(c + 0.0);  // (-0 becomes +0)
  return c != c ? 1 : (u >> 63 ? ~u : u | 1ull << 63);
}

// The largest rank of the wave and, of the lanes that hold it, the lowest index.
LSK_DEV void wave_best(uint64_t& r, int& i) {
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t ro = (uint64_t)__shfl_xor((unsigned long long)r, o, 64);
    const int io = __shfl_xor(i, o, 64);
    if (ro > r || (ro == r && io < i)) r = ro, i = io;
  }
}
LSK_DEV double wave_sum(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

LSK_DEV double lane_value(double v, int l) {  // l the same in every lane
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, l);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), l);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
// The value of the lane that a DPP control names; without one (or in a row that the mask leaves out), `old`.
template <int CTRL, int ROWS = 0xf>
LSK_DEV double dpp_value(double old, double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v), o = (uint64_t)__double_as_longlong(old);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)o, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)(o >> 32), (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
// The larger one; a NaN is passed over.
LSK_DEV double larger(double a, double b) { return __builtin_fmax(a, b); }
constexpr double kOut = __builtin_nan("");  // not to be chosen, where no score is a NaN

// larger() over the wave, in every lane.
LSK_DEV double wave_larger(double v) {
  v = larger(v, dpp_value<0xb1>(v, v));        // quad [1,0,3,2]
  v = larger(v, dpp_value<0x4e>(v, v));        // quad [2,3,0,1]
  v = larger(v, dpp_value<0x141>(v, v));       // half-row mirror
  v = larger(v, dpp_value<0x140>(v, v));       // row mirror
  v = larger(v, dpp_value<0x142, 0xa>(v, v));  // row bcast 15
  v = larger(v, dpp_value<0x143, 0xc>(v, v));  // row bcast 31
  return lane_value(v, 63);
}

// The choice among c (no NaNs but kOut), a round for each of the k: the largest upper word of rank_of over the wave, of
// those that hold it the largest lower word where there are several (scores within 2^-20 of each other), and of those the
// lowest expert.  Lane z gets the z-th expert and its score.  (A maximum of whole numbers over the wave is one instruction
// a step, of 64-bit numbers three: 8192 tokens, 256 experts, 8 of them: 13.6 us with those.)
template <int EPL>
LSK_DEV void choose(const RouteArgs& p, const double (&s)[EPL], const double (&c)[EPL], double& chosen, int& expert, double& sum) {
  const int lane = threadIdx.x & 63;
  uint32_t hi[EPL], lo[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const uint64_t r = c[j] != c[j] ? 0 : rank_of(c[j]);
    hi[j] = (uint32_t)(r >> 32), lo[j] = (uint32_t)r;
  }
  for (int z = 0; z < p.k; ++z) {
    uint32_t top = hi[0];
#pragma unroll
    for (int j = 1; j < EPL; ++j) top = top > hi[j] ? top : hi[j];
    top = wave_max_u32(top);
    uint64_t at[EPL];
    int n = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) at[j] = __builtin_amdgcn_ballot_w64(hi[j] == top), n += __builtin_popcountll(at[j]);
    if (n > 1) {
      uint32_t low = 0;
#pragma unroll
      for (int j = 0; j < EPL; ++j) low = hi[j] == top && lo[j] > low ? lo[j] : low;
      low = wave_max_u32(low);
#pragma unroll
      for (int j = 0; j < EPL; ++j) at[j] &= __builtin_amdgcn_ballot_w64(lo[j] == low);
    }
    double v = 0;
    int e = 0;
#pragma unroll
    for (int j = EPL - 1; j >= 0; --j) {  // (the lowest j last)
      if (!at[j]) continue;
      const int l = __builtin_ctzll(at[j]);
      v = lane_value(s[j], l);
      e = l + 64 * j;
    }
    sum = z ? sum + v : v;
    if (lane == z) chosen = v, expert = e;
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (e == lane + 64 * j) hi[j] = lo[j] = 0;
  }
}

// The groups that stay (no NaNs in c; a sum may be one, of both infinities): 64 / groups lanes, rounded down to a power of two, look a group over from LDS for
// its two largest; then lane g compares group g with every other.
LSK_DEV uint64_t kept_groups(const RouteArgs& p, const double* c) {
  const int lane = threadIdx.x & 63, size = p.E / p.groups;
  int per = 1;
  while (2 * per * p.groups <= 64) per *= 2;
  const int g = lane / per;
  double a = kOut, b = kOut;  // the two largest
  auto put = [&](double x, double y) {  // two more, x the larger
    const double lo = __builtin_fmin(a, x);  // (of a and nothing: a, which then is x: nothing)
    const bool none = a != a || x != x;
    a = larger(a, x);
    b = larger(larger(b, y), none ? kOut : lo);
  };
  if (g < p.groups)
    for (int i = lane % per; i < size; i += per) put(c[g * size + i], kOut);
  if (per > 1) put(dpp_value<0xb1>(kOut, a), dpp_value<0xb1>(kOut, b));
  if (per > 2) put(dpp_value<0x4e>(kOut, a), dpp_value<0x4e>(kOut, b));
  if (per > 4) put(dpp_value<0x141>(kOut, a), dpp_value<0x141>(kOut, b));  // (a quad's lanes hold the same by now)
  if (per > 8) put(dpp_value<0x140>(kOut, a), dpp_value<0x140>(kOut, b));
  if (per > 16) put(__shfl_xor(a, 16, 64), __shfl_xor(b, 16, 64));
  const double sum = p.group_top == 2 ? a + b : a;
  // (bring group g's to lane g)
  const double mine = __shfl(sum, lane * per & 63, 64);
  int ahead = 0;
  for (int h = 0; h < p.groups; ++h) {
    const double o = lane_value(sum, h * per);
    ahead += (o == o && mine != mine) || o > mine || ((o == mine || (o != o && mine != mine)) && h < lane);
  }
  return __builtin_amdgcn_ballot_w64(lane < p.groups && ahead < p.keep);
}

// The same two where scores are NaNs: by rank_of, the slow way.
template <int EPL>
LSK_DEV void choose_ranked(const RouteArgs& p, const double (&s)[EPL], const double (&c)[EPL], double& chosen, int& expert,
                           double& total) {
  const int lane = threadIdx.x & 63;
  uint64_t r[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) r[j] = lane + 64 * j < p.E ? rank_of(c[j]) : 0;
  if (p.keep < p.groups) {
    const int size = p.E / p.groups;
    double mine = 0;
    for (int g = 0; g < p.groups; ++g) {
      double sum = 0;
      int skip = -1;
      for (int z = 0; z < p.group_top; ++z) {
        uint64_t best = 0;
        int at = 1 << 30;
        double v = 0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const int e = lane + 64 * j;
          if (e / size == g && e != skip && r[j] > best) best = r[j], at = e;
        }
        wave_best(best, at);
#pragma unroll
        for (int j = 0; j < EPL; ++j)
          if (lane + 64 * j == at) v = c[j];
        v = __shfl(v, at & 63, 64);
        sum = z ? sum + v : v;
        skip = at;
      }
      if (lane == g) mine = sum;
    }
    uint64_t gr = lane < p.groups ? rank_of(mine) : 0, kept = 0;
    for (int z = 0; z < p.keep; ++z) {
      uint64_t best = gr;
      int at = lane;
      wave_best(best, at);
      kept |= 1ull << at;
      if (lane == at) gr = 0;
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = lane + 64 * j;
      if (e < p.E && !(kept >> (e / size) & 1)) r[j] = 0;
    }
  }
  for (int z = 0; z < p.k; ++z) {
    uint64_t best = 0;
    int at = 1 << 30;
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (r[j] > best) best = r[j], at = lane + 64 * j;
    wave_best(best, at);
    double v = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (lane + 64 * j == at) v = s[j], r[j] = 0;
    v = __shfl(v, at & 63, 64);
    total = z ? total + v : v;
    if (lane == z) chosen = v, expert = at;
  }
}

// A wave a token; lane l holds experts l, l + 64, ...
template <int EPL, bool GROUPS>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs p) {
  __shared__ double values[GROUPS ? 4 : 1][GROUPS ? 64 * EPL : 1];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= p.T) return;
  double s[EPL], c[EPL];
  double top = -__builtin_inf();
  // All of a lane's loads go out together: conversions wait until they are on their way, and what lies past E comes from
  // E's last place.  (MI355X, each waited for before the next, and so: 4096 tokens of 384 experts 14.2, 11.8 us, 8192 of
  // 256 in groups 18.1, 16.7, 32 of 256 in groups 7.5, 6.9, 32 of 128 4.9, 4.9.)
  const bool wide = p.g_dtype == LSK_F32;
  uint32_t raw[EPL];
  float bias[EPL] = {};
  if (wide) {  // (uniform, as the others)
    const uint32_t* const row = (const uint32_t*)p.g + t * p.ldg;
#pragma unroll
    for (int j = 0; j < EPL; ++j) raw[j] = row[min(lane + 64 * j, p.E - 1)];
  } else {
    const uint16_t* const row = (const uint16_t*)p.g + t * p.ldg;
#pragma unroll
    for (int j = 0; j < EPL; ++j) raw[j] = row[min(lane + 64 * j, p.E - 1)];
  }
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) bias[j] = p.bias[min(lane + 64 * j, p.E - 1)];
  }
  __asm__ volatile("" ::: "memory");  // (none behind the branches below)
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const float v = wide ? __uint_as_float(raw[j])
                         : p.g_dtype == LSK_BF16 ? __uint_as_float(raw[j] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)raw[j]);
    s[j] = lane + 64 * j < p.E ? (double)v : -__builtin_inf();
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) top = larger(top, s[j]);
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] = 1.0 / (1.0 + exp(-s[j]));
  } else {
    top = wave_larger(top);
    double sum = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      // (nothing above -infinity: every score is 0; a NaN makes the sum one)
      s[j] = s[j] == -__builtin_inf() ? 0.0 : exp(s[j] - top);
      sum += s[j];
    }
    sum = wave_sum(sum);
    const double scale = 1.0 / sum;
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] = sum == 0.0 ? 0.0 : s[j] * scale;
  }
  bool nan = false;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane + 64 * j;
    c[j] = s[j] + (double)bias[j];
    nan |= e < p.E && c[j] != c[j];
    if (e >= p.E) c[j] = kOut;
  }
  double chosen = 0, sum = 0;
  int expert = 0;
  if (__builtin_amdgcn_ballot_w64(nan)) {
    choose_ranked<EPL>(p, s, c, chosen, expert, sum);
  } else {
    if constexpr (GROUPS) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) values[wave][lane + 64 * j] = c[j];
      wave_lds_fence();
      const uint64_t kept = kept_groups(p, values[wave]);
      const uint32_t recip = (1u << 20) / (uint32_t)(p.E / p.groups) + 1;  // e / size for e < 1024, size < 1024
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (!(kept >> ((lane + 64 * j) * recip >> 20 & 63) & 1)) c[j] = kOut;
    }
    choose<EPL>(p, s, c, chosen, expert, sum);
  }
  if (lane < p.k) {
    double w = p.renorm ? (sum == 0.0 ? 0.0 : chosen / sum) : chosen;
    w *= p.factor;
    const int64_t o = t * p.k + lane;
    p.idx[o] = expert;
    if (p.w_dtype == LSK_F32) ((float*)p.w)[o] = (float)w;
    else store_out(p.w, p.w_dtype, o, (float)w);
  }
}

}  // namespace lsk

extern "C" int lsk_route_experts(const void* g, int g_dtype, int64_t ldg, int64_t T, int64_t E, int k, int sigmoid,
                                 const float* bias, int groups, int keep_groups, int group_top, int renormalize,
                                 double factor, int64_t* idx, void* w, int w_dtype, void* stream) {
  LSK_REQUIRE(g_dtype == LSK_F32 || g_dtype == LSK_BF16 || g_dtype == LSK_F16, "lsk_route_experts: logits must be f32, bf16 or f16");
  LSK_REQUIRE(w_dtype == LSK_F32 || w_dtype == LSK_BF16 || w_dtype == LSK_F16, "lsk_route_experts: weights must be f32, bf16 or f16");
  LSK_REQUIRE(T >= 0 && E >= 1 && E <= 1024, "lsk_route_experts: T=%lld, E=%lld (E in [1, 1024])", (long long)T, (long long)E);
  LSK_REQUIRE(groups >= 1 && groups <= 64 && E % groups == 0 && keep_groups >= 1 && keep_groups <= groups,
              "lsk_route_experts: %d of %d groups over %lld experts (at most 64 of one size)", keep_groups, groups, (long long)E);
  LSK_REQUIRE(group_top == 1 || (group_top == 2 && (keep_groups == groups || E / groups >= 2)),
              "lsk_route_experts: a group counts its 1 or 2 largest, and holds as many");
  LSK_REQUIRE(k >= 1 && k <= 64 && k <= E / groups * keep_groups, "lsk_route_experts: k=%d not in [1, min(64, %lld)]", k,
              (long long)(E / groups * keep_groups));
  if (T == 0) return LSK_OK;
  LSK_REQUIRE(g && idx && w, "lsk_route_experts: null pointer");
  LSK_REQUIRE(T == 1 || ldg >= E, "lsk_route_experts: ldg below E");
  LSK_REQUIRE(T < (1LL << 40) && grid_ok((T + 3) / 4, 256), "lsk_route_experts: grid too large");
  lsk::RouteArgs p{g, g_dtype, ldg, T, (int)E, k, groups, keep_groups, group_top, sigmoid != 0, renormalize != 0, factor, bias,
                   idx, w, w_dtype};
  const dim3 grid((unsigned)((T + 3) / 4)), blk(256);
  hipStream_t s = (hipStream_t)stream;
  auto run = [&](auto epl) {
    if (keep_groups < groups) hipLaunchKernelGGL((lsk::route_kernel<decltype(epl)::value, true>), grid, blk, 0, s, p);
    else hipLaunchKernelGGL((lsk::route_kernel<decltype(epl)::value, false>), grid, blk, 0, s, p);
  };
  if (E <= 64) run(std::integral_constant<int, 1>{});
  else if (E <= 128) run(std::integral_constant<int, 2>{});
  else if (E <= 256) run(std::integral_constant<int, 4>{});
  else if (E <= 512) run(std::integral_constant<int, 8>{});
  else run(std::integral_constant<int, 16>{});
  return lsk::check_launch("route_kernel");
}
