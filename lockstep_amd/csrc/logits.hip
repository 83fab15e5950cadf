// Penalties for repeated tokens, biases and allowed-token masks on a head's logits, one pass.
//
// Per row and token v, with n = how often v stands in the row's output and `seen` = v stands in its
// prompt or output:
//   l = fl32(l + bias[v]);  seen: l = l > 0 ? fl32(l / r) : fl32(l * r);
//   l = fl32(l - fl32(f * n));  n > 0: l = fl32(l - p);  mask bit 0: l = -inf;  out = round(l)
// A block owns a run of one row's tokens: it counts the row's history into a table of that run in LDS
// (a word per token: the output count, and the top bit for the prompt; integer atomics, so the order
// of tokens changes nothing), then streams the logits past it.  Every block of a row reads the whole
// history, which stays in the L2.
#include <hip/hip_runtime.h>

#include "lsk_common.h"

namespace lsk {

struct PenaltyArgs {
  const void* logits;
  int64_t ldl;
  int64_t B, V;
  const void *prompt, *output;            // [B, Lp] / [B, Lo] int32 or int64, or null
  int64_t ldp, Lp, ldo_tok, Lo;
  const void *prompt_lens, *output_lens;  // [B] int32 or int64, or null (all Lp / Lo)
  int p64, o64, pl64, ol64;               // 1: 64-bit entries
  const float *rep, *freq, *pres;         // [B] or null (1, 0, 0)
  const float* bias;                      // null, or row b at bias + b * ldb
  int64_t ldb;
  const uint32_t* mask;                   // null, or row b at mask + b * ldm: bit v % 32 of word v / 32
  int64_t ldm;
  void* out;
  int64_t ldo;
  int chunk;                              // tokens of a block, a multiple of 8
};

constexpr uint32_t kInPrompt = 0x80000000u;

LSK_DEV int64_t int_at(const void* p, int wide, int64_t i) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

template <int DT>
LSK_DEV float logit_at(const void* p, int64_t i) { return load_as_f32(p, DT, i); }

template <int DT>
__global__ __launch_bounds__(512) void penalize_logits_kernel(PenaltyArgs p) {
  extern __shared__ uint32_t count[];
  const int tid = threadIdx.x, chunks = (int)((p.V + p.chunk - 1) / p.chunk);
  const int64_t b = blockIdx.x / chunks, v0 = (int64_t)(blockIdx.x - b * chunks) * p.chunk;
  const int n = (int)(p.V - v0 < p.chunk ? p.V - v0 : p.chunk);
  const bool counted = p.prompt || p.output;
  if (counted) {
    for (int i = tid; i < n; i += 512) count[i] = 0;
    __syncthreads();
    if (p.prompt) {
      int64_t len = p.prompt_lens ? int_at(p.prompt_lens, p.pl64, b) : p.Lp;
      len = len < p.Lp ? len : p.Lp;
      for (int64_t i = tid; i < len; i += 512) {
        const int64_t t = int_at(p.prompt, p.p64, b * p.ldp + i) - v0;
        if (t >= 0 && t < n) atomicOr(&count[t], kInPrompt);
      }
    }
    if (p.output) {
      int64_t len = p.output_lens ? int_at(p.output_lens, p.ol64, b) : p.Lo;
      len = len < p.Lo ? len : p.Lo;
      for (int64_t i = tid; i < len; i += 512) {
        const int64_t t = int_at(p.output, p.o64, b * p.ldo_tok + i) - v0;
        if (t >= 0 && t < n) atomicAdd(&count[t], 1u);
      }
    }
    __syncthreads();
  }
  const float rep = p.rep ? p.rep[b] : 1.0f, freq = p.freq ? p.freq[b] : 0.0f, pres = p.pres ? p.pres[b] : 0.0f;
  for (int i = tid; i < n; i += 512) {
    const int64_t v = v0 + i;
    float l = logit_at<DT>(p.logits, b * p.ldl + v);
    if (p.bias) l = f32_add(l, p.bias[b * p.ldb + v]);
    const uint32_t c = counted ? count[i] : 0;
    if (c) {
      if (p.rep) l = l > 0.0f ? f32_div(l, rep) : f32_mul(l, rep);
      const uint32_t k = c & ~kInPrompt;
      if (k) {
        if (p.freq) l = l - f32_mul(freq, (float)k);
        if (p.pres) l = l - pres;
      }
    }
    if (p.mask && !((p.mask[b * p.ldm + (v >> 5)] >> (v & 31)) & 1u)) l = -__builtin_inff();
    store_out(p.out, DT, b * p.ldo + v, l);
  }
}

}  // namespace lsk

extern "C" int lsk_penalize_logits(const void* logits, int dtype, int64_t ldl, int64_t B, int64_t V, const void* prompt,
                                   int64_t ldp, int64_t Lp, const void* prompt_lens, const void* output, int64_t ldo_tok,
                                   int64_t Lo, const void* output_lens, int wide, const float* repetition,
                                   const float* frequency, const float* presence, const float* bias, int64_t ldb,
                                   const int32_t* mask, int64_t ldm, void* out, int64_t ldo, void* stream) {
  LSK_REQUIRE(dtype == LSK_F32 || dtype == LSK_BF16 || dtype == LSK_F16,
              "lsk_penalize_logits: dtype must be f32, bf16 or f16");
  LSK_REQUIRE(B >= 0 && V >= 0 && B <= 0x7fffffff && V <= 0x7fffffff, "lsk_penalize_logits: bad sizes B=%lld V=%lld",
              (long long)B, (long long)V);
  LSK_REQUIRE(Lp >= 0 && Lo >= 0 && Lo <= 0x7fffffff, "lsk_penalize_logits: bad history lengths %lld, %lld",
              (long long)Lp, (long long)Lo);
  if (B == 0 || V == 0) return LSK_OK;
  LSK_REQUIRE(logits && out, "lsk_penalize_logits: null pointer");
  LSK_REQUIRE(B == 1 || (ldl >= V && ldo >= V), "lsk_penalize_logits: row strides below V");
  LSK_REQUIRE(!mask || B == 1 || ldm >= 0, "lsk_penalize_logits: negative mask stride");
  lsk::PenaltyArgs p{};
  p.logits = logits, p.ldl = ldl, p.B = B, p.V = V;
  p.prompt = Lp ? prompt : nullptr, p.ldp = ldp, p.Lp = Lp, p.prompt_lens = prompt_lens;
  p.output = Lo ? output : nullptr, p.ldo_tok = ldo_tok, p.Lo = Lo, p.output_lens = output_lens;
  p.p64 = wide & 1, p.o64 = (wide >> 1) & 1, p.pl64 = (wide >> 2) & 1, p.ol64 = (wide >> 3) & 1;
  p.rep = repetition, p.freq = frequency, p.pres = presence;
  p.bias = bias, p.ldb = ldb, p.mask = (const uint32_t*)mask, p.ldm = ldm;
  p.out = out, p.ldo = ldo;
  p.chunk = 8192;
  const int64_t blocks = B * ((V + p.chunk - 1) / p.chunk);
  LSK_REQUIRE(blocks <= 0x7fffffff, "lsk_penalize_logits: grid too large");
  const size_t smem = p.prompt || p.output ? 4 * (size_t)p.chunk : 0;
  const dim3 grid((unsigned)blocks), blk(512);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == LSK_F32) hipLaunchKernelGGL(lsk::penalize_logits_kernel<LSK_F32>, grid, blk, smem, s, p);
  else if (dtype == LSK_BF16) hipLaunchKernelGGL(lsk::penalize_logits_kernel<LSK_BF16>, grid, blk, smem, s, p);
  else hipLaunchKernelGGL(lsk::penalize_logits_kernel<LSK_F16>, grid, blk, smem, s, p);
  return lsk::check_launch("penalize_logits_kernel");
}
