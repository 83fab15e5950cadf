// MXFP4 activations and weights: the quantiser and the products on the block-scaled matrix core.
//
// A value of an MXFP4 row is fp4(code) * 2^(s - 127): sixteen E2M1 codes {0, 0.5, 1, 1.5, 2, 3, 4, 6}
// with a sign, one E8M0 byte s per 32 values along K.  With both operands in that form
//   y[m, n] = sum_b 2^(sa[m, b] + sw[n, b] - 254) sum_{j in b} fa[m, j] fw[n, j]
// runs on v_mfma_scale_f32_16x16x128_f8f6f4 and v_mfma_scale_f32_32x32x64_f8f6f4 as it lies in
// memory: a lane holds the 16 code bytes of one block of one row and that block's scale byte.
//
// Every output is one chain of such instructions over ascending K from +0.  Chained 32x32x64 and
// 16x16x128 give the same bits (MI355X: tested with scale bytes from one octave to all that a byte holds,
// through subnormal sums and overflows), so a row's result depends neither on the tile that computes it nor
// on the other rows of the call.
#include <hip/hip_runtime.h>

#include "lsk_common.h"
#include "fp4_tile.h"
#include "mfma_tile.h"

#define LSK_HD __host__ __device__ inline

namespace lsk {

// ---------------------------------------------------------------- the quantiser
// Eight values of a block (the block's other 24 in the three neighbouring lanes of a quad) to eight
// codes; s = the block's scale byte.  The largest magnitude's exponent E (biased) comes from its
// bits, so s = E - 2 puts it in [4, 8) of its scale; the conversion instruction divides by 2^(s -
// 127), rounds to nearest with ties to the even code and takes magnitudes above 6 to 6 (checked on
// MI355X against the definition over every bf16 pattern and as many random binary32 at each of 255
// scales).  A block that holds an infinity or a NaN gets s = 255, which makes every product with it
// NaN, and code 7 at those elements, 0 elsewhere.
LSK_DEV uint32_t quantize8_mxfp4(const float (&v)[8], uint32_t& s) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(v[i]) & 0x7fffffffu;
    top = top > u ? top : u;
  }
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, false);  // quad [1,0,3,2]
  top = top > o ? top : o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, false);  // quad [2,3,0,1]
  top = top > o ? top : o;
  const uint32_t E = top >> 23;
  if (E == 255) {
    s = 255;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(v[i]);
      if ((u & 0x7f800000u) == 0x7f800000u) w |= (7u | ((u >> 28) & 8u)) << (4 * i);
    }
    return w;
  }
  s = E > 2 ? E - 2 : 0;
  const float sc = __uint_as_float(s ? s << 23 : 0x00400000u);  // 2^(s - 127)
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], sc, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], sc, 3);
  return w;
}

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

// Where block b of row r of `rows` keeps its scale byte in the transposed form the tiles read:
// [b / 4][row] dwords, byte b % 4.  Bytes past the last block are 0 (a 255 there would make NaNs of
// the zero codes beside it).
LSK_DEV void store_scale_t(uint8_t* t, int64_t rows, int64_t r, int b, int nb, uint32_t s) {
  uint8_t* d = t + ((b >> 2) * rows + r) * 4;
  d[b & 3] = (uint8_t)s;
  if (b == nb - 1)
    for (int z = (b & 3) + 1; z < 4; ++z) d[z] = 0;
}

// A thread per eight values, a quad of lanes per block: total = M * K / 8 threads' worth of work (a
// multiple of 4, so quads lie wholly inside or outside it).  Bound by HBM: s_x bytes read and 17/32
// written a value.  TS: the scales transposed.
template <int DT, bool VEC, bool TS>
LSK_DEV void quantize_run(const void* __restrict__ x, int64_t ldx, int64_t M, int64_t total, int K8, int block,
                          int blocks, uint8_t* __restrict__ packed, uint8_t* __restrict__ scale) {
  for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < total; i += (int64_t)blocks * 256) {
    const int64_t row = i / K8;
    const int c = (int)(i - row * K8);
    float v[8];
    load8<DT, VEC>(x, row * ldx + 8 * c, v);
    uint32_t s;
    ((uint32_t*)packed)[i] = quantize8_mxfp4(v, s);
    if constexpr (TS) {
      if ((c & 3) == 0) store_scale_t(scale, M, row, c >> 2, K8 >> 2, s);
    } else if ((i & 3) == 0) {
      scale[i >> 2] = (uint8_t)s;
    }
  }
}

// The same with transposed scales for K % 128 == 0: 16 rows by 512 values a block, 16 lanes a row, so that
// a block stores 16 rows' dwords of a stage side by side (scattered over blocks, a line of 32 rows was
// written in pieces from several XCDs).
template <int DT, bool VEC>
LSK_DEV void quantize_rows16(const void* __restrict__ x, int64_t ldx, int64_t M, int K, int64_t block,
                             uint8_t* __restrict__ packed, uint32_t* __restrict__ sat) {
  const int chunks = (K + 511) / 512, tid = threadIdx.x;
  const int64_t rb = block / chunks, row = rb * 16 + (tid >> 4);
  const int k0 = (int)(block - rb * chunks) * 512 + 8 * (tid & 15);
  float v[4][8];
#pragma unroll
  for (int z = 0; z < 4; ++z)
    if (row < M && k0 + 128 * z < K) load8<DT, VEC>(x, row * ldx + k0 + 128 * z, v[z]);
#pragma unroll
  for (int z = 0; z < 4; ++z) {
    if (row >= M || k0 + 128 * z >= K) continue;  // (16 lanes alike)
    uint32_t s;
    *(uint32_t*)(packed + (row * K + k0 + 128 * z) / 2) = quantize8_mxfp4(v[z], s);
    uint32_t w = s << (2 * (tid & 12));  // the four bytes of a dword, from 16 lanes
    w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x124, 0xf, 0xf, false);  // row_ror:4
    w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x128, 0xf, 0xf, false);  // row_ror:8
    if ((tid & 15) == 0) sat[(int64_t)((k0 >> 7) + z) * M + row] = w;
  }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void quantize_mxfp4_kernel(const void* __restrict__ x, int64_t ldx, int64_t M,
                                                             int64_t total, int K8, uint8_t* __restrict__ packed,
                                                             uint8_t* __restrict__ scale) {
  quantize_run<DT, VEC, false>(x, ldx, M, total, K8, blockIdx.x, gridDim.x, packed, scale);
}

// f(dtype, vec) with the dtype and the alignment of x's rows as compile-time values.
template <class F>
static void by_input(const void* x, int x_dtype, int64_t ldx, F f) {
  const int size = x_dtype == LSK_F32 ? 4 : 2;
  const bool vec = (uintptr_t)x % 16 == 0 && (ldx * size) % 16 == 0;
  auto with = [&](auto dt) { vec ? f(dt, std::true_type{}) : f(dt, std::false_type{}); };
  if (x_dtype == LSK_F32) with(std::integral_constant<int, LSK_F32>{});
  else if (x_dtype == LSK_BF16) with(std::integral_constant<int, LSK_BF16>{});
  else with(std::integral_constant<int, LSK_F16>{});
}

static int quantize_launch(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* packed,
                           uint8_t* scale, hipStream_t s) {
  const int64_t total = M * (K / 8), blocks = (total + 255) / 256;
  const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536)), blk(256);
  by_input(x, x_dtype, ldx, [&](auto dt, auto vec) {
    hipLaunchKernelGGL((quantize_mxfp4_kernel<decltype(dt)::value, decltype(vec)::value>), grid, blk, 0, s, x, ldx, M,
                       total, (int)(K / 8), packed, scale);
  });
  return check_launch("quantize_mxfp4_kernel");
}

// ---------------------------------------------------------------- the products
struct Fp4Args {
  const uint8_t* a;   // codes [M, K/2], row stride lda bytes
  const uint8_t* sa;  // scales [M, K/32], row stride ldsa
  const uint8_t* w;   // codes [N, K/2], row stride ldw
  const uint8_t* sw;  // scales [N, K/32], row stride ldsw
  int64_t lda, ldsa, ldw, ldsw;
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

// Few rows: a block computes NG x 16 output columns of up to MT x 16 rows over all of K, streaming its
// weight rows from HBM.  Four waves bring the codes in, KS x 512 values (256 bytes of a row, whole lines)
// a stage, by direct global -> LDS loads RING - 1 stages ahead; waves multiply a group of 16 weight
// rows by a row tile each, on 16x16x128 instructions (weight rows as their rows, activation rows as
// their columns, so a lane ends with four consecutive outputs of a row).  Bound by HBM, that is by
// bytes in flight: with a few thousand weight rows there is a block of 16 of them a CU, which is why
// waves that do not multiply load.  K is not split over waves or blocks: every kernel here sums an output in
// one chain, and a split by the number of rows would make a row's bits depend on its batch.  (One at places
// that depend on K alone, in every kernel, would not; it needs a second set of accumulators, for which the
// 256 x 256 tiles, at 204 of 256 registers, have no room.)  The scales of the block's rows are copied into LDS whole at the start.
// DT >= 0: the rows of x (at most 16; vec: 16-byte aligned) are quantised by every block into LDS
// itself, which saves a launch and the wait for it; x comes from the L2.
template <int NG, int MT, int KS, bool FUSE>
struct Fp4StreamCfg {
  static constexpr int kPartW = NG * 4096, kPart = kPartW + (FUSE ? 0 : MT * 4096), kStage = KS * kPart;  // bytes
  static constexpr int kPer = KS * (NG + (FUSE ? 0 : MT));  // loads per thread per stage
  static constexpr int kMW = NG * MT > 4 ? NG * MT / 4 : 1;  // row tiles of a wave
  static_assert(NG * MT <= 4 || NG == 4, "a wave's row tiles share its weight rows");
};

// Bytes from one row of scales to the next in LDS: whole stages, in an odd number of 16-byte pieces (512
// values each), so that 16 rows read at once lie in 16 bank groups.
LSK_HD int scale_pieces(int nb, int ks) { return ((nb + 15) / 16 + ks - 1) / ks * ks; }
LSK_HD int scale_pitch(int nb, int ks) { return scale_pieces(nb, ks) * 16 | 16; }
// Bytes of LDS of such a block: the ring, the rows' codes (FUSE: `rows` of them) and the scales.
LSK_HD int fused_pitch(int K, int ks) { return scale_pieces(K / 32, ks) * 256 + 16; }
template <int NG, int MT, int KS, int RING, bool FUSE>
static int64_t fp4_stream_lds(int K, int rows) {
  return RING * Fp4StreamCfg<NG, MT, KS, FUSE>::kStage + (FUSE ? (int64_t)rows * fused_pitch(K, KS) : 0) +
         (int64_t)(NG * 16 + (FUSE ? rows : MT * 16)) * scale_pitch(K / 32, KS);
}

template <int NG, int MT, int KS, int RING, int DT, bool GROUPED>
__global__ __launch_bounds__(256) void fp4_stream_kernel(Fp4Args p, const void* __restrict__ x, int64_t ldx,
                                                         int vec) {
  constexpr bool FUSE = DT >= 0;
  using C = Fp4StreamCfg<NG, MT, KS, FUSE>;
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
    p.sw = (const uint8_t*)wave_uniform64(p.ws_ptrs[e]);
    p.bias = p.b_ptrs ? (const float*)wave_uniform64(p.b_ptrs[e]) : nullptr;
  }
  const int rows_a = m1 - m0 < 16 * MT ? (int)(m1 - m0) : 16 * MT;
  const int rows_w = p.N - n0 < 16 * NG ? (int)p.N - n0 : 16 * NG;
  const int nb = p.K / 32, Kb = p.K / 2, pieces = scale_pieces(nb, KS), nk = pieces / KS;
  const int sp = scale_pitch(nb, KS), fp = fused_pitch(p.K, KS);
  char* const fused = smem + RING * C::kStage;  // FUSE: the rows' codes
  char* const scw = fused + (FUSE ? rows_a * fp : 0);
  char* const sca = scw + NG * 16 * sp;

  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w + (int64_t)n0 * p.ldw, (int64_t)(rows_w - 1) * p.ldw + Kb);
  const __amdgpu_buffer_rsrc_t ra = FUSE ? rw : make_rsrc(p.a + m0 * p.lda, (int64_t)(rows_a - 1) * p.lda + Kb);
  // a thread's 16-byte slot j of a part: row 16 j + tid / 16, chunk c of its 256 bytes in place c ^ row % 16
  const int row = tid >> 4, kc = 16 * ((tid & 15) ^ row);
  auto issue = [&](int kt) {
    char* base = smem + (kt % RING) * C::kStage + wave * 1024;
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      const int k = 256 * (KS * kt + u);
      const bool in = k + kc < Kb;
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
#pragma unroll
  for (int s = 0; s < RING - 1; ++s) issue(s);

  // The scales: 16 threads a row, a 16-byte piece each, every row's first 32 pieces in flight at once and
  // no branch around a load but uniform ones.  A row's last piece comes from the 16 bytes that end it,
  // shifted down; zeros past it.
  constexpr int kRows = NG + (FUSE ? 0 : MT);  // row sets of 16
  const int c0 = tid & 15;
  auto scale_src = [&](int j) {
    return j < NG ? p.sw + n0 * p.ldsw + (uint32_t)(min(16 * j + row, rows_w - 1) * (int)p.ldsw)
                  : p.sa + m0 * p.ldsa + (uint32_t)(min(16 * (j - NG) + row, rows_a - 1) * (int)p.ldsa);
  };
  auto store_piece = [&](int j, int c, uint64_t lo, uint64_t hi) {
    if (c >= pieces) return;
    const int sh = 8 * max(16 * c + 16 - nb, 0);
    if (sh >= 128) lo = hi = 0;
    else if (sh >= 64) lo = hi >> (sh - 64), hi = 0;
    else if (sh > 0) lo = lo >> sh | hi << (64 - sh), hi >>= sh;
    *(ulonglong2*)(scw + (16 * j + row) * sp + 16 * c) = make_ulonglong2(lo, hi);
  };
  if (nb >= 16) {
    for (int cc = 0; cc < pieces; cc += 32) {
      uint64_t v[2][kRows][2];
#pragma unroll
      for (int j = 0; j < kRows; ++j) __builtin_memcpy(v[0][j], scale_src(j) + min(16 * (cc + c0), nb - 16), 16);
      if (cc + 16 < pieces) {
#pragma unroll
        for (int j = 0; j < kRows; ++j) __builtin_memcpy(v[1][j], scale_src(j) + min(16 * (cc + 16 + c0), nb - 16), 16);
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) store_piece(j, cc + c0, v[0][j][0], v[0][j][1]);
      if (cc + 16 < pieces) {
#pragma unroll
        for (int j = 0; j < kRows; ++j) store_piece(j, cc + 16 + c0, v[1][j][0], v[1][j][1]);
      }
    }
  } else {
    for (int j = 0; j < kRows; ++j)
      for (int c = c0; c < pieces * 16; c += 16) (scw + (16 * j + row) * sp)[c] = c < nb ? (char)scale_src(j)[c] : 0;
  }
  if constexpr (FUSE) {
    // (codes past K stay as they were: the weights beside them are zeros; scales past K are written 0)
    const int K8 = p.K / 8, all = rows_a * K8;
    auto load = [&](int m, int c, float (&v)[8]) {
      if (vec) load8<DT, true>(x, (m0 + m) * ldx + 8 * c, v);
      else load8<DT, false>(x, (m0 + m) * ldx + 8 * c, v);
    };
    auto put = [&](int m, int c, const float (&v)[8]) {
      uint32_t sc;
      *(uint32_t*)(fused + m * fp + 4 * c) = quantize8_mxfp4(v, sc);
      if ((c & 3) == 0) sca[m * sp + (c >> 2)] = (char)sc;
    };
    if (rows_a == 1) {
      for (int c = tid; c < K8; c += 256) {
        float v[8];
        load(0, c, v);
        put(0, c, v);
      }
    } else {  // the rows end to end, kBatch loads of a thread in flight
      constexpr int kBatch = 4;
      for (int i0 = tid; i0 < all; i0 += 256 * kBatch) {
        float v[kBatch][8];
        int m[kBatch];
#pragma unroll
        for (int z = 0; z < kBatch; ++z) {
          const int i = i0 + 256 * z;
          m[z] = (int)((uint32_t)i / (uint32_t)K8);
          if (i < all) load(m[z], i - m[z] * K8, v[z]);
        }
#pragma unroll
        for (int z = 0; z < kBatch; ++z)
          if (i0 + 256 * z < all) put(m[z], i0 + 256 * z - m[z] * K8, v[z]);  // (a quad of lanes alike)
      }
    }
    const int past = 16 * pieces - nb;
    for (int i = tid; i < rows_a * past; i += 256) {
      const int m = (int)((uint32_t)i / (uint32_t)past);
      sca[m * sp + nb + i - m * past] = 0;
    }
  }

  // wave w multiplies weight group w % NG with row tiles w / NG (and, NG * MT > 4, the next ones)
  constexpr int MW = C::kMW;
  const int g = wave % NG, mt = wave / NG * MW;
  const bool multiplies = NG * MT >= 4 || wave < NG * MT;
  v4f acc[MW];
  const char *ars[MW], *arc[MW];
#pragma unroll
  for (int m = 0; m < MW; ++m) {
    acc[m] = v4f{0, 0, 0, 0};
    // (rows past the end: whatever lies there, their results are not stored)
    const int ar = FUSE ? min(r, rows_a - 1) : 16 * (mt + m) + r;
    ars[m] = sca + ar * sp;
    arc[m] = FUSE ? fused + ar * fp : smem + C::kPartW + ar * 256;
  }
  const char* wrs = scw + (16 * g + r) * sp;
  // a stage's fragments are read a stage ahead where the ring is deep enough (fp4_tile.h)
  struct Frag {
    v4u32 sw[KS], sa[KS][MW];
    v4i w[KS][4], a[KS][MW][4];
  };
  auto read = [&](int kt, Frag& f) {
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      const int slot = (kt % RING) * C::kStage + u * C::kPart, part = KS * kt + u;
      const char* base = smem + slot + (16 * g + r) * 256;
      f.sw[u] = *(const v4u32*)(wrs + 16 * part);
#pragma unroll
      for (int m = 0; m < MW; ++m) f.sa[u][m] = *(const v4u32*)(ars[m] + 16 * part);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int c = 16 * ((4 * s + q) ^ r);
        f.w[u][s] = *(const v4i*)(base + c);
#pragma unroll
        for (int m = 0; m < MW; ++m)
          f.a[u][m][s] = FUSE ? *(const v4i*)(arc[m] + 256 * part + 64 * s + 16 * q) : *(const v4i*)(arc[m] + slot + c);
      }
    }
  };
  auto multiply = [&](const Frag& f) {
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int m = 0; m < MW; ++m)
          acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(f.w[u][s]), fp4_operand(f.a[u][m][s]), acc[m],
                                                                    4, 4, 0, (int)(f.sw[u][s] >> (8 * q)), 0,
                                                                    (int)(f.sa[u][m][s] >> (8 * q)));
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
#pragma unroll
  for (int m = 0; m < MW; ++m) {
    const int row_out = 16 * (mt + m) + r;
    if (row_out >= rows_a) continue;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t n = n0 + 16 * g + 4 * q + t;
      if (n < p.N) store_out(p.out, p.out_dtype, (m0 + row_out) * p.ldo + n, p.bias ? f32_add(acc[m][t], b[t]) : acc[m][t]);
    }
  }
}

// ---------------------------------------------------------------- tiles
// Scales [rows, nb] bytes (row stride lds) to the transposed form: 64 rows by 128 bytes a block, read in
// whole lines (eight lanes a row), turned in LDS, stored 64 rows' dwords side by side.
constexpr int kTurnPitch = 33;  // dwords
LSK_DEV void transpose_scales(const uint8_t* __restrict__ s, int64_t lds, int64_t rows, int nb, int64_t block,
                              uint32_t* __restrict__ t, uint32_t* turn) {
  const int64_t rblocks = (rows + 63) / 64, c = block / rblocks, r0 = (block - c * rblocks) * 64;
  const int nst = (nb + 3) / 4, tid = threadIdx.x, at = (int)(128 * c) + 16 * (tid & 7);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = 32 * half + (tid >> 3);
    const uint8_t* p = s + (r0 + row < rows ? r0 + row : rows - 1) * lds;
    uint64_t v[2] = {0, 0};
    if (at < nb) {
      if (nb >= 16) {  // the last piece from the 16 bytes that end the row, shifted down
        const int sh = 8 * max(at + 16 - nb, 0);
        __builtin_memcpy(v, p + min(at, nb - 16), 16);
        if (sh >= 64) v[0] = v[1] >> (sh - 64), v[1] = 0;
        else if (sh > 0) v[0] = v[0] >> sh | v[1] << (64 - sh), v[1] >>= sh;
      } else {
        for (int z = 0; z < nb; ++z) (z < 8 ? v[0] : v[1]) |= (uint64_t)p[z] << (8 * (z & 7));
      }
    }
    uint32_t* d = turn + row * kTurnPitch + 4 * (tid & 7);
    d[0] = (uint32_t)v[0], d[1] = (uint32_t)(v[0] >> 32), d[2] = (uint32_t)v[1], d[3] = (uint32_t)(v[1] >> 32);
  }
  __syncthreads();
  const int row = tid & 63;
  if (r0 + row >= rows) return;
#pragma unroll
  for (int z = 0; z < 8; ++z) {
    const int d = 4 * z + (tid >> 6);
    if (32 * (int)c + d < nst) t[(32 * c + d) * rows + r0 + row] = turn[row * kTurnPitch + d];
  }
}
inline int64_t transpose_blocks(int64_t rows, int64_t K) { return ((rows + 63) / 64) * ((K / 32 + 127) / 128); }

// What the tiles need beside the codes, in one launch: the rows quantised with transposed scales (DT an
// input type) or their scales transposed (DT < 0), and the weights' scales transposed, every expert's
// in turn.
struct Fp4Prep {
  const void* x;
  int64_t ldx, M, total;
  int K;
  uint8_t* q;
  const uint8_t* sa;
  int64_t ldsa;
  uint32_t* sat;
  int64_t ablocks;
  const uint8_t* sw;
  const int64_t* ws_ptrs;
  int64_t ldsw, N, wblocks;  // blocks of one weight
  uint32_t* swt;
};
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void fp4_prep_kernel(Fp4Prep p) {
  __shared__ uint32_t turn[64 * kTurnPitch];
  if (blockIdx.x < p.ablocks) {
    if constexpr (DT >= 0)
      if (p.K % 128 == 0) quantize_rows16<DT, VEC>(p.x, p.ldx, p.M, p.K, blockIdx.x, p.q, p.sat);
      else quantize_run<DT, VEC, true>(p.x, p.ldx, p.M, p.total, p.K / 8, blockIdx.x, (int)p.ablocks, p.q, (uint8_t*)p.sat);
    else
      transpose_scales(p.sa, p.ldsa, p.M, p.K / 32, blockIdx.x, p.sat, turn);
    return;
  }
  const int64_t b = blockIdx.x - p.ablocks, e = b / p.wblocks;
  transpose_scales(p.ws_ptrs ? (const uint8_t*)p.ws_ptrs[e] : p.sw, p.ldsw, p.N, p.K / 32, b - e * p.wblocks,
                   p.swt + e * p.N * ((p.K + 127) / 128), turn);
}

// Four outputs to consecutive places (8-byte, for binary32 16-byte aligned), rounded to the type; a NaN
// to bf16 becomes 0x7FC0, off the common path (v0 + v1 + v2 + v3 is a NaN where one of them is).
// Non-temporal: an output stays in no L2 past its launch, and within it leaves the L2 to the operands
// (4096 rows of 28672 x 4096 321 -> 293 us on MI355X, 777 of 4608 x 3584 21.9 -> 20.6).
LSK_DEV void store_quad(char* o, int dtype, v4f v) {
  auto put = [&](char* at, uint32_t lo, uint32_t hi) {
    __builtin_nontemporal_store((uint64_t)hi << 32 | lo, (uint64_t*)at);
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
  } else {
    put(o, (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[0]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[1]) << 16),
        (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[3]) << 16));
  }
}

// A BM x BN tile: tiles walk kGroupM row tiles down a column of weight tiles inside each XCD's run
// of them, so the row tiles that share a weight tile run together on one L2.
template <int BM, int BN, int WM, int WN, int RING, int BKB, bool GROUPED>
__global__ __launch_bounds__(WM * WN * 64) void fp4_tile_kernel(Fp4Args p, const uint32_t* __restrict__ sat,
                                                       const uint32_t* __restrict__ swt, int64_t mtiles, int vec) {
  using C = Fp4Cfg<BM, BN, WM, WN, RING, BKB>;
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
  const int nst = (p.K + 127) / 128;
  int m0, m1;
  if constexpr (GROUPED) {  // (the grid holds the most tiles there can be: the ones there are go to every XCD)
    ExpertTiles tiles(p.offs, p.E, (int)p.M, BM);
    mtiles = tiles.count();
    if (blockIdx.x >= mtiles * ntiles) return;
    place(xcd_logical_id(blockIdx.x, (int)mtiles * ntiles));
    int e;
    if (!tiles.find(mt, e, m0, m1)) return;
    p.w = (const uint8_t*)wave_uniform64(p.w_ptrs[e]);
    p.bias = p.b_ptrs ? (const float*)wave_uniform64(p.b_ptrs[e]) : nullptr;
    swt += (int64_t)e * nst * p.N;
  } else {
    place(xcd_logical_id(blockIdx.x, (int)mtiles * ntiles));
    m0 = mt * BM, m1 = (int)p.M;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int rows_a = m1 - m0 < BM ? m1 - m0 : BM, rows_w = (int)p.N - n0 < BN ? (int)p.N - n0 : BN;

  Fp4Rows<C> t;
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a + (int64_t)m0 * p.lda, (int64_t)(rows_a - 1) * p.lda + p.K / 2);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.w + (int64_t)n0 * p.ldw, (int64_t)(rows_w - 1) * p.ldw + p.K / 2);
  t.sta = (uint32_t)(4 * p.M), t.stb = (uint32_t)(4 * p.N);
  const __amdgpu_buffer_rsrc_t rsa = make_rsrc(sat + m0, 4 * ((int64_t)nst * p.M - m0));
  const __amdgpu_buffer_rsrc_t rsb = make_rsrc(swt + n0, 4 * ((int64_t)nst * p.N - n0));
#pragma unroll
  for (int j = 0; j < C::kLA; ++j) {
    int row, kb;
    pp_slot<C::kThreads, C::kChunks>(tid, j, row, kb);
    t.a[j] = row < rows_a ? (uint32_t)(row * p.lda) : kOob;
  }
#pragma unroll
  for (int j = 0; j < C::kLB; ++j) {
    int row, kb;
    pp_slot<C::kThreads, C::kChunks>(tid, j, row, kb);
    t.b[j] = row < rows_w ? (uint32_t)(row * p.ldw) : kOob;
  }
  t.s = tid < BM ? (tid < rows_a ? 4u * tid : kOob) : (tid - BM < rows_w ? 4u * (tid - BM) : kOob);

  typename C::Acc acc;
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass does not instantiate the main loop twice)
  fp4_mainloop<BM, BN, WM, WN, RING, BKB>(acc, ra, rb, rsa, rsb, t, p.K, smem);
#endif
  __syncthreads();

  // a 32-row strip at a time through the wave's part of LDS, out of it four consecutive columns a lane
  const int wm = wave / C::kWN, wn = wave % C::kWN;
  float* strip = (float*)(smem + wave * 32 * C::kLdc * 4);
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
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int h = 0; h < 4; ++h)
        *(v4f*)(strip + (lane & 31) * C::kLdc + j * 32 + 8 * h + 4 * (lane >> 5)) =
            v4f{acc[i][j][4 * h], acc[i][j][4 * h + 1], acc[i][j][4 * h + 2], acc[i][j][4 * h + 3]};
    // (a wave's own LDS operations run in order)
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += kRows, row += kRows, o += step) {
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

static int64_t fp4_row_tiles(const Fp4Args& p, int bm) {
  return p.offs ? expert_tiles_max(p.M, p.E, bm) : (p.M + bm - 1) / bm;
}

// (fp4_tiles has checked the grid)
template <int BM, int BN, int WM, int WN, int RING, int BKB>
static int fp4_tile_launch(const Fp4Args& p, const uint32_t* sat, const uint32_t* swt, hipStream_t s) {
  using C = Fp4Cfg<BM, BN, WM, WN, RING, BKB>;
  const int64_t mtiles = fp4_row_tiles(p, BM), blocks = mtiles * ((p.N + BN - 1) / BN);
  const int vec = out_vec_ok(p.out, p.out_dtype, p.ldo);
  auto run = [&](auto kern) {
    if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes) != hipSuccess)
      return set_error("fp4_tile_kernel: cannot reserve LDS"), LSK_ERR_HIP;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(C::kThreads), C::kSmemBytes, s, p, sat, swt, mtiles, vec);
    return check_launch("fp4_tile_kernel");
  };
  return p.offs ? run(fp4_tile_kernel<BM, BN, WM, WN, RING, BKB, true>)
                : run(fp4_tile_kernel<BM, BN, WM, WN, RING, BKB, false>);
}

// Whether the products of M rows (of E experts: E > 0) run on the tiles: where the streaming blocks would be
// many, by groups of 16 columns of 32 rows, since each streams its weight rows again for its 32; and where a
// block's scales of all of K do not fit the LDS.  (MI355X, GPU us of a linear on streaming blocks and on
// tiles, groups: 64 rows of 8192 x 2048 8.9, 9.6 at 1024; 64 of 12000 x 2048 11.1, 10.2, 256 of 3584 x 14336 43,
// 25 at 1500 - 1800; 128 of 3584 x 14336 19, 24 at 896; 24 of 28672 x 2048 11.0, 12.2 at 1792, 17 of 37888 x 2048
// 17.6, 15.2 at 2368.  By expert: 192 rows over 4 of 4096 x 1024 7.7, 10.0 at 2560; 128 over 4 of 5760 x 2880 20,
// 16 at 2880; 16 rows each over 32 of 5760 x 2880 69, 70, 24 each 80, 72.)  The counts are what one round of
// blocks takes with two of them a CU; by expert, where the count is the most tiles there can be and part of
// them stay empty, a fitted two and a half.  A long K, whose scales leave the LDS room for one, halves them (64
// rows of 7000 x 18944 31.6 on streaming blocks, 28.7 on tiles).
constexpr int64_t kStreamK = 32768;
template <int NG, int MT, int KS, int RING, int DT>
static int fp4_stream_per_cu(int64_t K, int rows) {  // blocks that a CU's LDS holds, counted to two
  return 2 * fp4_stream_lds<NG, MT, KS, RING, (DT >= 0)>((int)K, rows) <= 160 * 1024 ? 2 : 1;
}
static bool fp4_takes_tiles(int64_t M, int64_t N, int64_t K, int64_t E) {
  if (K == 0 || K > kStreamK) return K > 0;
  const int64_t groups = (E ? expert_tiles_max(M, E, 32) : (M + 31) / 32) * ((N + 15) / 16);
  const int64_t of4 = fp4_stream_per_cu<4, 2, 1, 2, -1>(K, 16), of2 = fp4_stream_per_cu<2, 2, 1, 3, -1>(K, 16);
  if (E) return M > 16 * E && groups > 1280 * of4;
  return M > 16 && groups > (M <= 32 ? 1024 * of4 : 512 * of2);
}
// The tiles address a tile's rows and the transposed scales with 31-bit offsets.
static bool fp4_tiles_reach(int64_t M, int64_t N, int64_t K) {
  const int64_t nst = (K + 127) / 128;
  return 4 * nst * M < 0x7fffffff && 4 * nst * N < 0x7fffffff && 256 * (K / 2) < 0x7fffffff;
}

static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// Bytes of the transposed scales of M rows and of E weights of N rows.
static int64_t fp4_prep_bytes(int64_t M, int64_t N, int64_t K, int64_t E) {
  const int64_t nst = (K + 127) / 128;
  return up256(4 * nst * M) + up256(4 * nst * N * E);
}

// About how long a product takes on tiles of one size, in us: the CU with the most blocks, ceil(tiles / 256)
// of them, works through them `blocks` at a time, a round of o blocks at once in round[o] + k[o] * K / 1000
// (round[0]: the launches); every million outputs costs `out` and `area` * K / 1000, and every 10^9 weights
// of experts (E > 0, whose last rows take half a tile each) `weights`.  Fitted to 368 products on MI355X (65
// to 4096 rows, 512 to 28672 columns, K = 96 to 14336; 100 to 16384 rows over 4 to 128 experts).  The tile it
// picks is 0.4 % slower than the best of the five on average and 17 % at most; thresholds on the number of
// tiles were 5 % and 44 % (4096 rows of 4608 x 512 on 1.1 rounds of 256 x 256).  Dense weight bytes are no term
// of it, so it says less than they take where they bound the product (64 rows of 152064 x 3584: 39 us by the
// fit, 78 measured); its choice past 28672 columns is an extrapolation.
struct Fp4TileCost {
  int bm, bn, blocks;
  double out, area, weights, round[4], k[4];
};
constexpr Fp4TileCost kFp4Tiles[5] = {
    {256, 256, 1, 0.053, 0.16, 0, {4.9, 9.9}, {0, 4.9}},
    {128, 256, 2, 0.11, 0.15, 21, {6.5, 4.5, 4.8}, {0, 4.1, 7.0}},
    {128, 128, 2, 0.12, 0.15, 27, {6.5, 3.7, 4.2}, {0, 2.9, 3.4}},
    {64, 128, 3, 0.13, 0.15, 50, {7.3, 0.88, 1.6, 2.4}, {0, 2.4, 2.6, 3.4}},
    {64, 64, 2, 0.71, 0.11, 50, {6.6, 0.56, 0.99}, {0, 1.3, 1.7}},
};
static double fp4_tile_us(const Fp4TileCost& t, int64_t M, int64_t N, int64_t K, int64_t E) {
  const int64_t down = E ? (M / t.bm + E / 2 > E ? M / t.bm + E / 2 : E) : (M + t.bm - 1) / t.bm;
  const int64_t tiles = down * ((N + t.bn - 1) / t.bn), most = (tiles + 255) / 256;
  const double kk = K * 1e-3, outs = tiles * 1e-6 * t.bm * t.bn;
  const int o = t.blocks, rest = (int)(most % o);
  return t.round[0] + outs * (t.out + t.area * kk) + E * N * kk * 1e-6 * t.weights +
         (double)(most / o) * (t.round[o] + t.k[o] * kk) + (rest ? t.round[rest] + t.k[rest] * kk : 0);
}
static int fp4_cheapest_tile(int64_t M, int64_t N, int64_t K, int64_t E) {
  int best = 0;
  for (int c = 1; c < 5; ++c)
    if (fp4_tile_us(kFp4Tiles[c], M, N, K, E) < fp4_tile_us(kFp4Tiles[best], M, N, K, E)) best = c;
  return best;
}

// The tiles' products: p.a / p.sa the rows (x null), or x to be quantised into q first.
static int fp4_tiles(Fp4Args p, const void* x, int x_dtype, int64_t ldx, uint8_t* q, char* work, hipStream_t s) {
  const int64_t nst = (p.K + 127) / 128, E = p.offs ? p.E : 1;
  LSK_REQUIRE(fp4_tiles_reach(p.M, p.N, p.K), "mxfp4 product: M=%lld N=%lld K=%d beyond 31-bit offsets", (long long)p.M,
              (long long)p.N, p.K);
  Fp4Prep r{};
  r.M = p.M, r.K = p.K;
  r.sat = (uint32_t*)work, r.swt = (uint32_t*)(work + up256(4 * nst * p.M));
  r.sw = p.sw, r.ws_ptrs = p.offs ? p.ws_ptrs : nullptr, r.ldsw = p.ldsw, r.N = p.N;
  r.wblocks = transpose_blocks(p.N, p.K);
  if (x) {
    r.x = x, r.ldx = ldx, r.total = p.M * (p.K / 8), r.q = q;
    r.ablocks = (r.total + 255) / 256 < 65536 ? (r.total + 255) / 256 : 65536;
    if (p.K % 128 == 0) r.ablocks = (p.M + 15) / 16 * ((p.K + 511) / 512);
    p.a = q;
  } else {
    r.sa = p.sa, r.ldsa = p.ldsa, r.ablocks = transpose_blocks(p.M, p.K);
  }
  const int tile = fp4_cheapest_tile(p.M, p.N, p.K, p.offs ? E : 0);
  const Fp4TileCost& size = kFp4Tiles[tile];
  const int64_t blocks = fp4_row_tiles(p, size.bm) * ((p.N + size.bn - 1) / size.bn);
  LSK_REQUIRE(grid_ok(r.ablocks + r.wblocks * E, 256) && grid_ok(blocks, tile < 2 ? 512 : 256),
              "mxfp4 product: grid too large");
  const dim3 grid((unsigned)(r.ablocks + r.wblocks * E)), blk(256);
  if (x)
    by_input(x, x_dtype, ldx, [&](auto dt, auto vec) {
      hipLaunchKernelGGL((fp4_prep_kernel<decltype(dt)::value, decltype(vec)::value>), grid, blk, 0, s, r);
    });
  else
    hipLaunchKernelGGL((fp4_prep_kernel<-1, false>), grid, blk, 0, s, r);
  const int rc = check_launch("fp4_prep_kernel");
  if (rc) return rc;
  switch (tile) {  // (all give the same bits)
    case 0: return fp4_tile_launch<256, 256, 2, 4, 4, 64>(p, r.sat, r.swt, s);
    case 1: return fp4_tile_launch<128, 256, 2, 4, 3, 64>(p, r.sat, r.swt, s);
    case 2: return fp4_tile_launch<128, 128, 2, 2, 2, 128>(p, r.sat, r.swt, s);
    case 3: return fp4_tile_launch<64, 128, 2, 2, 2, 128>(p, r.sat, r.swt, s);
    default: return fp4_tile_launch<64, 64, 2, 2, 4, 128>(p, r.sat, r.swt, s);
  }
}

template <int NG, int MT, int KS, int RING, int DT>
static int fp4_stream_launch(const Fp4Args& p, const void* x, int64_t ldx, hipStream_t s) {
  const int64_t tiles = p.offs ? expert_tiles_max(p.M, p.E, 16 * MT) : (p.M + 16 * MT - 1) / (16 * MT);
  const int64_t blocks = tiles * ((p.N + 16 * NG - 1) / (16 * NG));
  LSK_REQUIRE(grid_ok(blocks, 256), "mxfp4 product: grid too large");
  const int64_t lds = fp4_stream_lds<NG, MT, KS, RING, (DT >= 0)>(p.K, (int)(p.M < 16 ? p.M : 16));
  LSK_REQUIRE(lds <= 160 * 1024, "mxfp4 product: K=%d too long for few rows", p.K);
  const int vec = x && (uintptr_t)x % 16 == 0 && (ldx * (DT == LSK_F32 ? 4 : 2)) % 16 == 0;
  auto run = [&](auto kern) {
    if (lds > 65536 &&
        hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess)
      return set_error("fp4_stream_kernel: cannot reserve LDS"), LSK_ERR_HIP;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), (size_t)lds, s, p, x, ldx, vec);
    return check_launch("fp4_stream_kernel");
  };
  if constexpr (DT < 0) {
    if (p.offs) return run(fp4_stream_kernel<NG, MT, KS, RING, DT, true>);
  }
  return run(fp4_stream_kernel<NG, MT, KS, RING, DT, false>);
}

// The launch shape by the number of 16-row weight groups over all row tiles: one group a block while
// there are few (long stages, a deep ring: nothing else hides the latency), else blocks of two, then of
// four with the shortest ring, several of which share a CU: each for one round of blocks, as many a CU as its
// LDS holds, counted to two.  For row tiles of 16 the second bound is fixed: three blocks of two groups a CU, which
// fit up to K = 7168 or so; at 14336 two do and at 32768 one, so just below the bound such products take up to
// three rounds (16 rows of 20000 x 14336 32.8 us where the weights' bytes take 25, of 24000 x 32768 110 and 69; not
// measured against blocks of four there).  (MI355X, kernel us for NG x KS x RING = 1 x 2 x 4, 2 x 1 x 3: 24 rows of 4096 x 14336
// 11.0, 12.4; 16 of 4096 x 7168 7.3, 8.1; calls 64 of 3584 x 2048 11.4, 8.3.  Calls for 1 x 1 x 4, 2 x 1 x 3, 4 x
// 1 x 2: 8 of 28672 x 4096 16.8, 16.9, 14.0; by expert, 4 rows of 5760 x 2880 13.9, 10.0, 10.4; 256 rows over 32
// experts of 2880 x 2880 50, 41, 36; 64 over 2 of 5760 x 2880 -, 12.6, 10.1.)
template <int MT, int DT>
static int fp4_stream_shape(const Fp4Args& p, const void* x, int64_t ldx, hipStream_t s) {
  const int64_t tiles = p.offs ? expert_tiles_max(p.M, p.E, 16 * MT) : (p.M + 16 * MT - 1) / (16 * MT);
  const int64_t groups = tiles * ((p.N + 15) / 16);
  const int rows = (int)(p.M < 16 ? p.M : 16);
  if (groups <= 256 * fp4_stream_per_cu<1, MT, 2, 4, DT>(p.K, rows)) return fp4_stream_launch<1, MT, 2, 4, DT>(p, x, ldx, s);
  if (groups <= (MT == 1 ? 1536 : 512 * fp4_stream_per_cu<2, 2, 1, 3, -1>(p.K, 16)))
    return fp4_stream_launch<2, MT, 1, 3, DT>(p, x, ldx, s);
  return fp4_stream_launch<4, MT, 1, 2, DT>(p, x, ldx, s);
}

// Row tiles of 16 while that holds all rows (of an expert: twice the average, the skew of a routing).
static int fp4_stream(const Fp4Args& p, hipStream_t s) {
  const int64_t per = p.offs ? 2 * p.M / p.E : p.M;
  return per <= 16 ? fp4_stream_shape<1, -1>(p, nullptr, 0, s) : fp4_stream_shape<2, -1>(p, nullptr, 0, s);
}

// Whether a linear's few rows are quantised in the product's launch: one row whose codes fit the LDS beside
// the ring, or up to 16 of few values together, since every block quantises them all.  (MI355X, GPU us in one
// launch and in two, N = 4608: one row of 4096 5.2, 7.0, of 18944 11.7, 11.7 (N = 1024); 4 of 1024 4.6, 6.2,
// of 4096 7.9, 7.1, of 8192 13.6, 9.0; 16 of 512 5.7, 6.4, of 1024 7.0, 6.3.  A launch less is 3 us of a
// caller's time besides, but nothing in a replayed graph.  The rule does not look at N, and the border was set at
// 4608: in a graph, 16 rows of 1024 take 10.1, 8.5 at N = 28672 and 32.8, 24.6 at 152064, 4 of 4096 15.6, 14.0
// and 78, 68, 8 of 1024 8.0, 8.3 and 22.2, 23.8, 16 of 512 6.2, 6.7 and 20.1, 19.9.)
static bool fp4_fuses(int64_t M, int64_t K) {
  return K > 0 && (M == 1 ? K <= 24576 : M <= 16 && M * K <= 16384);
}

static int fp4_stream_fused(const Fp4Args& p, const void* x, int x_dtype, int64_t ldx, hipStream_t s) {
  if (x_dtype == LSK_F32) return fp4_stream_shape<1, LSK_F32>(p, x, ldx, s);
  if (x_dtype == LSK_BF16) return fp4_stream_shape<1, LSK_BF16>(p, x, ldx, s);
  return fp4_stream_shape<1, LSK_F16>(p, x, ldx, s);
}

static bool is_float_dtype(int d) { return d == LSK_F32 || d == LSK_BF16 || d == LSK_F16; }

static bool work_ok(const void* w, int64_t have, int64_t need) {
  return have >= need && (need == 0 || (w && (uintptr_t)w % 256 == 0));
}

}  // namespace lsk

extern "C" int lsk_quantize_mxfp4(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* packed,
                                  uint8_t* scale, void* stream) {
  LSK_REQUIRE(lsk::is_float_dtype(x_dtype), "lsk_quantize_mxfp4: x_dtype must be f32, bf16 or f16");
  LSK_REQUIRE(M >= 0 && K >= 0 && K % 32 == 0 && K <= 0x7fffffff, "lsk_quantize_mxfp4: K=%lld not a multiple of 32",
              (long long)K);
  if (M == 0 || K == 0) return LSK_OK;
  LSK_REQUIRE(M <= 0x7fffffffffLL / K * 32, "lsk_quantize_mxfp4: M=%lld too large", (long long)M);
  LSK_REQUIRE(M == 1 || ldx >= K, "lsk_quantize_mxfp4: ldx below K");
  LSK_REQUIRE(x && packed && scale, "lsk_quantize_mxfp4: null pointer");
  LSK_REQUIRE((uintptr_t)packed % 4 == 0, "lsk_quantize_mxfp4: packed must be 4-byte aligned");
  return lsk::quantize_launch(x, x_dtype, M, K, ldx, packed, scale, (hipStream_t)stream);
}

static int mxfp4_check(const char* who, int64_t M, int64_t N, int64_t K, int out_dtype, int64_t ldo) {
  LSK_REQUIRE(M >= 0 && N >= 0 && K >= 0 && K % 32 == 0, "%s: bad sizes M=%lld N=%lld K=%lld (K a multiple of 32)", who,
              (long long)M, (long long)N, (long long)K);
  LSK_REQUIRE(M <= 0x7fffffff && N <= 0x7fffffff && K < (1 << 24), "%s: sizes beyond 31 bits (K beyond 2^24)", who);
  LSK_REQUIRE(lsk::is_float_dtype(out_dtype), "%s: out_dtype must be f32, bf16 or f16", who);
  LSK_REQUIRE(ldo >= N, "%s: ldo below N", who);
  return LSK_OK;
}

extern "C" int64_t lsk_gemm_mxfp4_workspace(int64_t M, int64_t N, int64_t K) {
  return lsk::fp4_takes_tiles(M, N, K, 0) ? lsk::fp4_prep_bytes(M, N, K, 1) : 0;
}

#define LSK_REQUIRE_WORK(who, need)                                                                                  \
  LSK_REQUIRE(lsk::work_ok(workspace, workspace_bytes, need), who ": workspace of %lld bytes (256-byte aligned) needed", \
              (long long)(need))

extern "C" int lsk_gemm_mxfp4(const uint8_t* a, const uint8_t* a_scale, int64_t M, int64_t K, const uint8_t* w,
                              const uint8_t* w_scale, int64_t N, const float* bias, void* out, int out_dtype,
                              int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = mxfp4_check("lsk_gemm_mxfp4", M, N, K, out_dtype, ldo);
  if (rc) return rc;
  if (M == 0 || N == 0) return LSK_OK;
  LSK_REQUIRE(out && (K == 0 || (a && a_scale && w && w_scale)), "lsk_gemm_mxfp4: null pointer");
  LSK_REQUIRE((uintptr_t)a % 16 == 0 && (uintptr_t)w % 16 == 0, "lsk_gemm_mxfp4: codes must be 16-byte aligned");
  LSK_REQUIRE_WORK("lsk_gemm_mxfp4", lsk_gemm_mxfp4_workspace(M, N, K));
  lsk::Fp4Args p{};
  p.a = a, p.sa = a_scale, p.w = w, p.sw = w_scale;
  p.lda = p.ldw = K / 2, p.ldsa = p.ldsw = K / 32;
  p.M = M, p.N = N, p.K = (int)K;
  p.bias = bias, p.out = out, p.out_dtype = out_dtype, p.ldo = ldo;
  if (lsk::fp4_takes_tiles(M, N, K, 0)) return lsk::fp4_tiles(p, nullptr, 0, 0, nullptr, (char*)workspace, (hipStream_t)stream);
  return lsk::fp4_stream(p, (hipStream_t)stream);
}

// The quantised rows come first in the workspace, then their scales (the row kernels) or the tiles' part.
extern "C" int64_t lsk_linear_mxfp4_workspace(int64_t M, int64_t N, int64_t K) {
  if (lsk::fp4_fuses(M, K)) return 0;
  return lsk::up256(M * (K / 2)) +
         (lsk::fp4_takes_tiles(M, N, K, 0) ? lsk::fp4_prep_bytes(M, N, K, 1) : lsk::up256(M * (K / 32)));
}

extern "C" int lsk_linear_mxfp4(const void* x, int x_dtype, int64_t ldx, int64_t M, int64_t K, const uint8_t* w,
                                const uint8_t* w_scale, int64_t N, const float* bias, void* out, int out_dtype,
                                int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = mxfp4_check("lsk_linear_mxfp4", M, N, K, out_dtype, ldo);
  if (rc) return rc;
  LSK_REQUIRE(lsk::is_float_dtype(x_dtype), "lsk_linear_mxfp4: x_dtype must be f32, bf16 or f16");
  if (M == 0 || N == 0) return LSK_OK;
  LSK_REQUIRE(out && (K == 0 || (x && w && w_scale)), "lsk_linear_mxfp4: null pointer");
  LSK_REQUIRE(M == 1 || ldx >= K, "lsk_linear_mxfp4: ldx below K");
  LSK_REQUIRE((uintptr_t)w % 16 == 0, "lsk_linear_mxfp4: codes must be 16-byte aligned");
  LSK_REQUIRE_WORK("lsk_linear_mxfp4", lsk_linear_mxfp4_workspace(M, N, K));
  hipStream_t s = (hipStream_t)stream;
  uint8_t* q = (uint8_t*)workspace;
  uint8_t* rest = q + lsk::up256(M * (K / 2));
  lsk::Fp4Args p{};
  p.a = q, p.sa = rest, p.w = w, p.sw = w_scale;
  p.lda = p.ldw = K / 2, p.ldsa = p.ldsw = K / 32;
  p.M = M, p.N = N, p.K = (int)K;
  p.bias = bias, p.out = out, p.out_dtype = out_dtype, p.ldo = ldo;
  if (lsk::fp4_takes_tiles(M, N, K, 0)) return lsk::fp4_tiles(p, x, x_dtype, ldx, q, (char*)rest, s);
  if (lsk::fp4_fuses(M, K)) return lsk::fp4_stream_fused(p, x, x_dtype, ldx, s);
  if (K > 0 && (rc = lsk::quantize_launch(x, x_dtype, M, K, ldx, q, rest, s))) return rc;
  return lsk::fp4_stream(p, s);
}

extern "C" int64_t lsk_grouped_gemm_mxfp4_workspace(int64_t R, int64_t E, int64_t N, int64_t K) {
  return lsk::fp4_takes_tiles(R, N, K, E) ? lsk::fp4_prep_bytes(R, N, K, E) : 0;
}

extern "C" int lsk_grouped_gemm_mxfp4(const uint8_t* a, const uint8_t* a_scale, const int32_t* offs, int64_t E, int64_t R,
                                      const int64_t* w_ptrs, int64_t ldw, const int64_t* ws_ptrs, int64_t lds,
                                      const int64_t* b_ptrs, int64_t N, int64_t K, void* out, int out_dtype, int64_t ldo,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = mxfp4_check("lsk_grouped_gemm_mxfp4", R, N, K, out_dtype, ldo);
  if (rc) return rc;
  LSK_REQUIRE(E >= 1 && E <= (1 << 20), "lsk_grouped_gemm_mxfp4: E=%lld not in [1, 2^20]", (long long)E);
  if (R == 0 || N == 0) return LSK_OK;
  LSK_REQUIRE(out && offs && w_ptrs && ws_ptrs && (K == 0 || (a && a_scale)), "lsk_grouped_gemm_mxfp4: null pointer");
  LSK_REQUIRE((uintptr_t)a % 16 == 0 && ldw >= K / 2 && ldw % 16 == 0 && lds >= K / 32,
              "lsk_grouped_gemm_mxfp4: codes in rows of 16-byte multiples, strides that cover K");
  LSK_REQUIRE(ldw < (1 << 23) && lds < (1 << 23), "lsk_grouped_gemm_mxfp4: row strides beyond 2^23 bytes");
  LSK_REQUIRE_WORK("lsk_grouped_gemm_mxfp4", lsk_grouped_gemm_mxfp4_workspace(R, E, N, K));
  lsk::Fp4Args p{};
  p.a = a, p.sa = a_scale;
  p.lda = K / 2, p.ldsa = K / 32, p.ldw = ldw, p.ldsw = lds;
  p.M = R, p.N = N, p.K = (int)K;
  p.out = out, p.out_dtype = out_dtype, p.ldo = ldo;
  p.offs = offs, p.E = (int)E, p.w_ptrs = w_ptrs, p.ws_ptrs = ws_ptrs, p.b_ptrs = b_ptrs;
  if (lsk::fp4_takes_tiles(R, N, K, E)) return lsk::fp4_tiles(p, nullptr, 0, 0, nullptr, (char*)workspace, (hipStream_t)stream);
  return lsk::fp4_stream(p, (hipStream_t)stream);
}
