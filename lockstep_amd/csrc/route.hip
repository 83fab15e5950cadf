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

// A wave a token; lane l holds experts l, l + 64, ...
template <int EPL>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs p) {
  __shared__ double score[4][64];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= p.T) return;
  double s[EPL], c[EPL];
  uint64_t r[EPL];
  double top = -__builtin_inf();
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane + 64 * j;
    s[j] = e < p.E ? (double)load_as_f32(p.g, p.g_dtype, t * p.ldg + e) : -__builtin_inf();
    top = s[j] > top ? s[j] : top;
  }
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] = 1.0 / (1.0 + exp(-s[j]));
  } else {
    for (int o = 32; o > 0; o >>= 1) {
      const double q = __shfl_xor(top, o, 64);
      top = q > top ? q : top;
    }
    double sum = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      // (nothing above -infinity: every score is 0; a NaN makes the sum one)
      s[j] = s[j] == -__builtin_inf() ? 0.0 : exp(s[j] - top);
      sum += s[j];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] = sum == 0.0 ? 0.0 : s[j] / sum;
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane + 64 * j;
    c[j] = e < p.E && p.bias ? s[j] + (double)p.bias[e] : s[j];
    r[j] = e < p.E ? rank_of(c[j]) : 0;
  }
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
        const int own = at;
        wave_best(best, at);
#pragma unroll
        for (int j = 0; j < EPL; ++j)
          if (lane + 64 * j == at) v = c[j];
        v = __shfl(v, at & 63, 64);
        (void)own;
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
  double chosen = 0;  // lane z: the z-th chosen expert's score
  int expert = 0;
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
    if (lane == z) chosen = v, expert = at;
  }
  double sum = 0;
  score[wave][lane] = chosen;
  for (int z = 0; z < p.k; ++z) sum += score[wave][z];  // (a wave's own LDS operations run in order)
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
  auto run = [&](auto epl) { hipLaunchKernelGGL((lsk::route_kernel<decltype(epl)::value>), grid, blk, 0, s, p); };
  if (E <= 64) run(std::integral_constant<int, 1>{});
  else if (E <= 128) run(std::integral_constant<int, 2>{});
  else if (E <= 256) run(std::integral_constant<int, 4>{});
  else if (E <= 512) run(std::integral_constant<int, 8>{});
  else run(std::integral_constant<int, 16>{});
  return lsk::check_launch("route_kernel");
}
