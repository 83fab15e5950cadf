// Penalties for repeated tokens, biases and allowed-token masks on a head's logits, one pass.
//
// Per row and token v, with n = how often v stands in the row's output and `seen` = v stands in its
// prompt or output:
//   l = fl32(l + bias[v]);  seen: l = l > 0 ? fl32(l / r) : fl32(l * r);
//   n > 0: l = fl32(fl32(l - fl32(f * n)) - p);  mask bit 0: l = -inf;  out = round(l)
// A block owns a run of one row's tokens.  It requests its first logits, counts the row's history into
// a table of that run in LDS meanwhile (the output count, and the top bit for the prompt; integer
// atomics, so the order of tokens changes nothing), and then streams the run: a vector of tokens none
// of which stands in the history, without bias and mask, is a copy.  Bound by HBM.  Every block of a
// row reads the whole history, which stays in the L2: runs are as long as the LDS of two blocks a CU
// allows, and shorter where there are too few rows to fill the part with them.
#include <hip/hip_runtime.h>

#include <type_traits>

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
  int chunk;                              // tokens of a block
};

LSK_DEV int64_t int_at(const void* p, int wide, int64_t i) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// The count table: 16-bit entries, two a word, while no count can reach the prompt's bit (Lo < 2^15),
// else 32-bit ones.
template <int BITS>
struct CountTable {
  uint32_t* w;
  static constexpr uint32_t kPrompt = 1u << (BITS - 1), kAll = BITS == 32 ? 0xffffffffu : 0xffffu;
  LSK_DEV int word(int i) const { return BITS == 32 ? i : i >> 1; }
  LSK_DEV int shift(int i) const { return BITS == 32 ? 0 : (i & 1) * 16; }
  LSK_DEV void mark_prompt(int i) { atomicOr(&w[word(i)], kPrompt << shift(i)); }
  LSK_DEV void count(int i) { atomicAdd(&w[word(i)], 1u << shift(i)); }
  LSK_DEV uint32_t at(int i) const { return (w[word(i)] >> shift(i)) & kAll; }
};

// f(local token) for each token of a row's history that lies in the block's run [v0, v0 + n).
template <class F>
LSK_DEV void each_token(const void* tok, int wide, int64_t ld, int64_t L, const void* lens, int lwide, int64_t b,
                        int64_t v0, int n, F f) {
  if (!tok) return;
  int64_t len = lens ? int_at(lens, lwide, b) : L;
  len = len < L ? len : L;
  for (int64_t i = threadIdx.x; i < len; i += blockDim.x) {
    const int64_t t = int_at(tok, wide, b * ld + i) - v0;
    if (t >= 0 && t < n) f((int)t);
  }
}

// PLAIN: without bias and mask, where a token outside the history keeps its bits, a NaN's payload too.
template <int DT, int BITS, bool PLAIN>
__global__ __launch_bounds__(1024, 8) void penalize_logits_kernel(PenaltyArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint32_t smem[];
  constexpr int VEC = DT == LSK_F32 ? 4 : 8, SIZE = DT == LSK_F32 ? 4 : 2;
  const int tid = threadIdx.x, nt = blockDim.x, chunks = (int)((p.V + p.chunk - 1) / p.chunk);
  const int64_t b = blockIdx.x / chunks, v0 = (int64_t)(blockIdx.x - b * chunks) * p.chunk;
  const int n = (int)(p.V - v0 < p.chunk ? p.V - v0 : p.chunk);
  const bool counted = p.prompt || p.output;
  const char* in = (const char*)p.logits + (b * p.ldl + v0) * SIZE;
  char* out = (char*)p.out + (b * p.ldo + v0) * SIZE;
  const float* bias = !PLAIN && p.bias ? p.bias + b * p.ldb + v0 : nullptr;
  const uint32_t* mask = !PLAIN && p.mask ? p.mask + b * p.ldm : nullptr;
  // the run's first 16-byte boundary, where the vectors start (rows of in and out that differ modulo
  // 16 bytes go token by token); the table starts `pad` entries in, so that vectors of it are whole too
  const bool vec = ((uintptr_t)in & 15) == ((uintptr_t)out & 15) && (uintptr_t)in % SIZE == 0;
  int head = vec ? (int)((16 - ((uintptr_t)in & 15)) & 15) / SIZE : n;
  head = head < n ? head : n;
  const int pad = (VEC - head % VEC) % VEC;
  CountTable<BITS> table{smem};

  // a thread's first vectors, on their way while the history is counted
  constexpr int kAhead = 5;
  const int nvec = (n - head) / VEC;
  v4u32 ahead[kAhead];
#pragma unroll
  for (int z = 0; z < kAhead; ++z)
    if (tid + z * nt < nvec) ahead[z] = *(const v4u32*)(in + (int64_t)(head + (tid + z * nt) * VEC) * SIZE);

  if (counted) {
    const int words = ((n + pad) * BITS + 31) / 32;
    for (int i = tid; i < (words + 3) / 4; i += nt) ((uint4*)smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    each_token(p.prompt, p.p64, p.ldp, p.Lp, p.prompt_lens, p.pl64, b, v0, n, [&](int t) { table.mark_prompt(t + pad); });
    each_token(p.output, p.o64, p.ldo_tok, p.Lo, p.output_lens, p.ol64, b, v0, n, [&](int t) { table.count(t + pad); });
    __syncthreads();
  }
  const float rep = p.rep ? p.rep[b] : 1.0f, freq = p.freq ? p.freq[b] : 0.0f, pres = p.pres ? p.pres[b] : 0.0f;
  // the penalties of a token with count word c != 0
  auto penalized = [&](float l, uint32_t c) {
    if (p.rep) l = l > 0.0f ? f32_div(l, rep) : f32_mul(l, rep);
    const uint32_t k = c & (CountTable<BITS>::kPrompt - 1);
    if (k) {
      if (p.freq) l = l - f32_mul(freq, (float)k);
      if (p.pres) l = l - pres;
    }
    return l;
  };
  auto one = [&](int i) {
    const uint32_t c = counted ? table.at(i + pad) : 0;
    if (PLAIN && !c) {
      if constexpr (DT == LSK_F32) ((uint32_t*)out)[i] = ((const uint32_t*)in)[i];
      else ((uint16_t*)out)[i] = ((const uint16_t*)in)[i];
      return;
    }
    float l = load_as_f32(in, DT, i);
    if (bias) l = f32_add(l, bias[i]);
    if (c) l = penalized(l, c);
    const int64_t v = v0 + i;
    if (mask && !((mask[v >> 5] >> (v & 31)) & 1u)) l = -__builtin_inff();
    store_out(out, DT, i, l);
  };
  for (int i = tid; i < head; i += nt) one(i);

  auto vector = [&](int g, v4u32 raw) {
    const int i = head + g * VEC;
    uint32_t cw[VEC * BITS / 32] = {};
    bool any = false;
    if (counted) {
      const uint4* c = (const uint4*)((const char*)smem + (int64_t)(i + pad) * (BITS / 8));
#pragma unroll
      for (int q = 0; q < VEC * BITS / 128; ++q) {
        const uint4 u = c[q];
        cw[4 * q] = u.x, cw[4 * q + 1] = u.y, cw[4 * q + 2] = u.z, cw[4 * q + 3] = u.w;
        any = any || (u.x | u.y | u.z | u.w);
      }
      if constexpr (VEC * BITS < 128) {
        const uint2 u = *(const uint2*)c;
        cw[0] = u.x, cw[1] = u.y;
        any = u.x | u.y;
      }
    }
    if (PLAIN && !any) {
      if (in != out) store16_split(out + (int64_t)i * SIZE, raw);
      return;
    }
    const uint32_t rw[4] = {raw[0], raw[1], raw[2], raw[3]};
    uint32_t o[4];
    auto value = [&](int z) {
      if constexpr (DT == LSK_F32) return __uint_as_float(rw[z]);
      else if constexpr (DT == LSK_BF16) return bf16_to_f32((uint16_t)(rw[z / 2] >> (z % 2 * 16)));
      else return (float)__builtin_bit_cast(_Float16, (uint16_t)(rw[z / 2] >> (z % 2 * 16)));
    };
    auto counted_at = [&](int z) -> uint32_t {
      return BITS == 32 ? cw[z] : (cw[z * BITS / 32] >> (z * BITS % 32)) & 0xffffu;
    };
    if constexpr (PLAIN) {  // the counted tokens alone, in their places among the others' bits
#pragma unroll
      for (int z = 0; z < 4; ++z) o[z] = rw[z];
#pragma unroll
      for (int z = 0; z < VEC; ++z) {
        const uint32_t c = counted_at(z);
        if (!c) continue;
        const float l = penalized(value(z), c);
        if constexpr (DT == LSK_F32) {
          o[z] = __float_as_uint(l);
        } else {
          const uint32_t h = DT == LSK_BF16 ? f32_to_bf16(l) : __builtin_bit_cast(uint16_t, (_Float16)l);
          o[z / 2] = z % 2 ? (o[z / 2] & 0xffffu) | h << 16 : (o[z / 2] & 0xffff0000u) | h;
        }
      }
    } else {
      float l[VEC];
#pragma unroll
      for (int z = 0; z < VEC; ++z) l[z] = value(z);
      if (bias) {
        float bv[VEC];
        __builtin_memcpy(bv, bias + i, VEC * 4);
#pragma unroll
        for (int z = 0; z < VEC; ++z) l[z] = f32_add(l[z], bv[z]);
      }
      if (any) {
#pragma unroll
        for (int z = 0; z < VEC; ++z) {
          const uint32_t c = counted_at(z);
          if (c) l[z] = penalized(l[z], c);
        }
      }
      if (mask) {
        const int64_t v = v0 + i;
        const uint64_t lo = mask[v >> 5], hi = mask[(v + VEC - 1) >> 5];
        const uint32_t m = (uint32_t)(((hi << 32) | lo) >> (v & 31));  // (VEC bits at most: inside 64)
#pragma unroll
        for (int z = 0; z < VEC; ++z)
          if (!((m >> z) & 1u)) l[z] = -__builtin_inff();
      }
      if constexpr (DT == LSK_F32) {
#pragma unroll
        for (int z = 0; z < 4; ++z) o[z] = __float_as_uint(l[z]);
      } else if constexpr (DT == LSK_BF16) {
#pragma unroll
        for (int z = 0; z < 4; ++z) o[z] = pack_bf16x2(l[2 * z], l[2 * z + 1]);
      } else {
#pragma unroll
        for (int z = 0; z < 4; ++z)
          o[z] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)l[2 * z]) |
                 ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)l[2 * z + 1]) << 16);
      }
    }
    store16_split(out + (int64_t)i * SIZE, o[0], o[1], o[2], o[3]);
  };
#pragma unroll
  for (int z = 0; z < kAhead; ++z)
    if (tid + z * nt < nvec) vector(tid + z * nt, ahead[z]);
  for (int g = tid + kAhead * nt; g < nvec; g += nt) vector(g, *(const v4u32*)(in + (int64_t)(head + g * VEC) * SIZE));
  for (int i = head + nvec * VEC + tid; i < n; i += nt) one(i);
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
  LSK_REQUIRE(B == 1 || out != logits || ldo == ldl, "lsk_penalize_logits: in place with two row strides");
  LSK_REQUIRE(!mask || B == 1 || ldm >= 0, "lsk_penalize_logits: negative mask stride");
  lsk::PenaltyArgs p{};
  p.logits = logits, p.ldl = ldl, p.B = B, p.V = V;
  p.prompt = Lp ? prompt : nullptr, p.ldp = ldp, p.Lp = Lp, p.prompt_lens = prompt_lens;
  p.output = Lo ? output : nullptr, p.ldo_tok = ldo_tok, p.Lo = Lo, p.output_lens = output_lens;
  p.p64 = wide & 1, p.o64 = (wide >> 1) & 1, p.pl64 = (wide >> 2) & 1, p.ol64 = (wide >> 3) & 1;
  p.rep = repetition, p.freq = frequency, p.pres = presence;
  p.bias = bias, p.ldb = ldb, p.mask = (const uint32_t*)mask, p.ldm = ldm;
  p.out = out, p.ldo = ldo;
  // 16-bit counts while they cannot reach the prompt's bit; runs of up to 76 KB of them (two blocks a
  // CU), at least 512 blocks where runs of 1024 tokens give as many
  const bool narrow = Lo < (1 << 15), counted = p.prompt || p.output;
  const int64_t most = counted && !narrow ? 19456 : 38912;
  int64_t chunks = (512 + B - 1) / B;
  if (chunks > (V + 1023) / 1024) chunks = (V + 1023) / 1024;
  if (chunks < (V + most - 1) / most) chunks = (V + most - 1) / most;
  p.chunk = (int)(((V + chunks - 1) / chunks + 31) / 32 * 32);
  const int64_t blocks = B * ((V + p.chunk - 1) / p.chunk);
  const int threads = p.chunk >= 8192 ? 1024 : 256;
  LSK_REQUIRE(grid_ok(blocks, threads), "lsk_penalize_logits: grid too large");
  const size_t smem = counted ? ((size_t)p.chunk + 8) * (narrow ? 2 : 4) + 16 : 0;
  const dim3 grid((unsigned)blocks), blk(threads);
  hipStream_t s = (hipStream_t)stream;
  auto run = [&](auto kern) {
    if (smem > 65536 &&
        hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != hipSuccess)
      return lsk::set_error("lsk_penalize_logits: cannot reserve LDS"), LSK_ERR_HIP;
    hipLaunchKernelGGL(kern, grid, blk, smem, s, p);
    return lsk::check_launch("penalize_logits_kernel");
  };
  auto with = [&](auto dt) {
    constexpr int kDt = decltype(dt)::value;
    if (!p.bias && !p.mask)
      return narrow ? run(lsk::penalize_logits_kernel<kDt, 16, true>) : run(lsk::penalize_logits_kernel<kDt, 32, true>);
    return narrow ? run(lsk::penalize_logits_kernel<kDt, 16, false>) : run(lsk::penalize_logits_kernel<kDt, 32, false>);
  };
  if (dtype == LSK_F32) return with(std::integral_constant<int, LSK_F32>{});
  if (dtype == LSK_BF16) return with(std::integral_constant<int, LSK_BF16>{});
  return with(std::integral_constant<int, LSK_F16>{});
}
