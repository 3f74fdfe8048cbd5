// The feed-forward block's matrix products for one element type, built with
// -DFST_T=<bf16|f16|float> -DFST_NAME=<bf16|f16|f32>, and with -DFST_EXPERTS=1
// for mixtures of experts (names experts_<type>): the tokens then lie in runs, one for
// each expert, and a tile of tokens is of one run.
//
// Two kernels carry it:
//  * ffn_product: tokens times a weight, contraction along the rows of both
//    (gate and up projections with the activation and the product h = act(a) u
//    as its epilogue; the output projection; the gradient of h with the
//    activation's derivative as its epilogue; the gradient of x);
//  * ffn_outer: the weights' gradients, contraction over the tokens.
// Matrix cores accumulate in float32. bf16 and f16 run 16x16x32 steps, float32
// four 16x16x4 steps over the same 16 bytes of a lane, so that tiles, loads and
// LDS layouts are the same bytes for every type.
#include "fst_ffn.h"

#include <algorithm>
#include <type_traits>

namespace fst {

namespace {

typedef FST_T T;
constexpr int ES = sizeof(T);
constexpr bool F32 = ES == 4;
#ifndef FST_EXPERTS
#define FST_EXPERTS 0
#endif
constexpr bool EXPERTS = FST_EXPERTS;

// What loads past an operand's end read: 16 zero bytes.
__device__ const u32x4 kZero16 = {0, 0, 0, 0};

template <typename U>
struct Mma;
template <>
struct Mma<bf16> {
  typedef bf16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<f16> {
  typedef f16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
  // Element e of lane group g is k = 4 g + e for both operands: four steps of
  // four k, in an order of their own.
  static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
};

// All of this wave's loads into LDS but the newest N have landed and its LDS
// reads are done; then the workgroup's.
template <int N>
__device__ __forceinline__ void stage_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// 16 bytes a lane into LDS, lane l's at dst + 16 l (dst is wave-uniform), from a
// buffer (zeros past its range) or an address. Written out because the compiler
// waits for every load into LDS in flight before the transposing LDS reads it
// makes from their builtin, and for all LDS reads at once; these loads have no
// output register, and stage_wait counts them. m0, which they take the LDS address
// from, is reserved: nothing else of these kernels uses it.
__device__ __forceinline__ unsigned lds_offset(const unsigned char* dst) {
  return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)dst);
}
__device__ __forceinline__ void load_to_lds(u32x4 buffer, const unsigned char* dst, int voff, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds_offset(dst)),
               "v"(voff), "s"(buffer), "s"(soff)
               : "memory");
}
__device__ __forceinline__ void load_to_lds(const char* from, const unsigned char* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_offset(dst)), "v"(from)
               : "memory");
}

// act(a), and with D its derivative. sigmoid from the hardware's exp2 and
// reciprocal (1 ulp each). Phi(a) = erfc(-a / sqrt 2) / 2 with Abramowitz and
// Stegun's formula 7.1.26 for erfc (absolute error 1.5e-7), whose exp(-a^2 / 2)
// is also the density in the derivative.
template <int KIND, bool D>
__device__ __forceinline__ float activate(float a, float& slope) {
  if constexpr (KIND == FST_GELU) {
    const float x = fabsf(a) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f));
    const float e = __expf(-x * x);
    const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float q = 0.5f * p * e;  // Phi(-|a|)
    const float phi = a < 0.f ? q : 1.f - q;
    if constexpr (D) slope = fmaf(a * e, 0.39894228040143268f, phi);
    return a * phi;
  } else {
    float z = a, dz = 1.f;  // the sigmoid's argument and its derivative
    if constexpr (KIND == FST_GELU_TANH) {
      const float c = 1.59576912160573071f, s = a * a;  // 2 sqrt(2 / pi)
      z = c * a * fmaf(0.044715f, s, 1.f);
      // Finite, so that 0 * dz is 0: from |a| = 10 on the factor beside it is.
      if constexpr (D) dz = c * fmaf(3.f * 0.044715f, fminf(s, 1e30f), 1.f);
    }
    const float g = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    const float h = a * g;
    if constexpr (D) slope = fmaf(h * (1.f - g), dz, g);  // in this order: a * dz may overflow
    return h;
  }
}

// The same for N elements in place: one choice of the kind for all of them.
template <int KIND, bool D, int N>
__device__ __forceinline__ void activate_each(float* v, float* slope) {
  float unused;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = activate<KIND, D>(v[e], D ? slope[e] : unused);
}
template <bool D, int N>
__device__ __forceinline__ void activate_run(int kind, float* v, float* slope) {
  if (kind == FST_SILU)
    activate_each<FST_SILU, D, N>(v, slope);
  else if (kind == FST_GELU)
    activate_each<FST_GELU, D, N>(v, slope);
  else
    activate_each<FST_GELU_TANH, D, N>(v, slope);
}

// N consecutive elements: loads and stores of `n` of them (a multiple of 8).
template <int N>
__device__ __forceinline__ void load_run(const T* p, int n, float* v) {
  constexpr int V = kVec<T>;
#pragma unroll
  for (int q = 0; q < N / V; ++q) {
    typename Piece<T>::V x;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (T)0.f;
    if (q * V < n) x = *reinterpret_cast<const typename Piece<T>::V*>(p + q * V);
#pragma unroll
    for (int i = 0; i < V; ++i) v[q * V + i] = (float)x[i];
  }
}
template <int N>
__device__ __forceinline__ void store_run(T* p, int n, const float* v) {
  constexpr int V = kVec<T>;
#pragma unroll
  for (int q = 0; q < N / V; ++q)
    if (q * V < n) *reinterpret_cast<typename Piece<T>::V*>(p + q * V) = pack_piece<T>(v + q * V);
}

// Workgroup -> tile. Workgroups go to the eight XCDs in turn; each XCD takes a
// contiguous run of the tiles, ordered in blocks of up to eight token tiles
// by all feature tiles, so that what runs at one time on an XCD shares a few
// token tiles and a few of the weight's through its L2.
__device__ __forceinline__ bool pick_tile(int wg, int nf, int nt, int& f, int& t) {
  const int total = nf * nt, per = (total + 7) >> 3;
  const int i = wg >> 3, at = (wg & 7) * per + i;
  if (i >= per || at >= total) return false;
  const int block = at / (8 * nf), in = at - block * 8 * nf;
  const int tall = min(8, nt - 8 * block);
  f = in / tall;
  t = 8 * block + in - f * tall;
  return true;
}

// Experts: the workgroup's feature tile, expert, and the rows t0 .. end - 1 of its tile
// of BT tokens; expert = p.experts: rows outside every run (past the last one, or before
// the first, where a table is part of a longer one), where they are asked for.
// Workgroup wg of a grid over all tiles, or token tile `at` of a row of the grid (at >=
// 0). Offsets are taken within the rows and in order, so that no table makes a tile reach
// outside. Each wave adds up the runs' tiles by itself, 64 experts at a time. The rows of
// no run come after all tiles, so that every XCD has its share of the products.
struct ExpertTile {
  int ft, expert, t0, end;
};

template <int BT>
__device__ __forceinline__ bool expert_tile(const FfnProduct& p, int wg, int nf, int at, ExpertTile& tile) {
  const int lane = threadIdx.x & 63;
  int start, stop, count, upto;  // of expert e0 + lane: its rows, its tiles, and those up to its last
  const auto bound = [&](int i) { return min(max(p.offsets[i], 0), p.tokens); };
  const auto scan = [&](int e0) __attribute__((always_inline)) {
    const int e = e0 + lane;
    start = e < p.experts ? bound(e) : 0;
    stop = e < p.experts ? max(start, bound(e + 1)) : 0;
    count = upto = (stop - start + BT - 1) / BT;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int below = __shfl_up(upto, d);
      if (lane >= d) upto += below;
    }
  };
  scan(0);
  int total = __builtin_amdgcn_readlane(upto, 63);
  for (int e0 = 64; e0 < p.experts; e0 += 64) {
    scan(e0);
    total += __builtin_amdgcn_readlane(upto, 63);
  }
  int tt = at, behind = at - total;  // place among the tiles of no run
  bool run;
  if (at < 0) {
    run = pick_tile(wg, nf, total, tile.ft, tt);
    behind = wg - (nf * total + 7) / 8 * 8;
  } else {
    run = tt < total;
  }
  if (!run) {
    if (!p.tail || behind < 0) return false;
    const int head = bound(0), heads = (head + BT - 1) / BT, row = at < 0 ? behind / nf : behind;
    const bool before = row < heads;
    tile.ft = at < 0 ? behind % nf : 0;
    tile.expert = p.experts;
    tile.end = before ? head : p.tokens;
    tile.t0 = (int)min((long)tile.end, before ? (long)row * BT : max(head, bound(p.experts)) + (long)(row - heads) * BT);
    return tile.t0 < tile.end;
  }
  if (p.experts > 64) scan(0);
  for (int e0 = 0; e0 < p.experts; e0 += 64) {
    if (e0) scan(e0);
    const int sum = __builtin_amdgcn_readlane(upto, 63);
    if (tt < sum) {
      const int src = __builtin_ctzll(__ballot(upto > tt)), from = __builtin_amdgcn_readlane(start, src);
      tile.expert = e0 + src;
      tile.t0 = from + (tt - __builtin_amdgcn_readlane(upto - count, src)) * BT;
      tile.end = __builtin_amdgcn_readlane(stop, src);
      return tile.t0 >= from && tile.t0 < tile.end;
    }
    tt -= sum;
  }
  return false;
}

// WF x WT waves of NI x NJ subtiles of 16 features by 16 tokens. The weight is
// the matrix core's row operand, so a lane ends up with 4 GS consecutive
// features of its tokens: slot m = 4 a + r of subtile s of a group of GS holds
// feature 4 GS a + 4 s + r, which the loads into LDS arrange. LDS rows are 128
// bytes of k (whole lines of memory: 64-byte rows measured a fifth slower);
// 16-byte part c of row r sits at c ^ ((r >> 1) & 7), so that the 16 rows of a
// read pass cover the banks once. ST stages: the loads of ST - 1 k steps run while
// a step is multiplied, one barrier a step. ST = 5: LDS holds five halves of stages
// (one operand's), and the rows of the step after the next are on their way beside the
// next step's weights (256 x 768 padded, D = 384, F = 1024 bf16: step 1222 -> 1198 us,
// forward 360 -> 349; 65536 tokens, D = 1024, F = 2752: 4.06 -> 4.03 ms).
//
// kFfnRedo runs two contractions after each other, a and u from x and then dh
// from dy, and holds all three.
//
// Bound by the matrix cores and the way to them: with 65536 tokens, D = 1024, F = 2752
// in bf16 gate and up take 692 us (1.07 PFLOP/s), the output product 326 (1.13), dx 616
// (1.20), kFfnRedo 1188 (0.93), where a library product of 8192 a side reaches 1.35
// and one of the gate's shape 1.10. The matrix cores are busy half of the cycles, as
// the LDS is (reads and the loads into it); no bank conflicts; four of five lines
// come from L2. At K = 384 (100500 tokens, F = 1024: 208, 110, 204 and 353 us) a
// workgroup's six steps stand beside its first loads and its stores (147 of 238 us
// without an epilogue, before activations were chosen once per run). Measured and
// slower or no faster: four waves of 128 x 128 (690 -> 830 us, the output product as
// fast, with its LDS reads written ahead by hand), stores as whole lines
// through LDS (236 -> 253 at K = 384), a workgroup that goes from tile to tile with the
// next tile's first loads in flight (gate 210 -> 201 at K = 384, 690 -> 710 wide, kFfnRedo
// spills and takes 413 and 1290), a higher wave priority around the products.
// float32 (128 x 128 tiles; 16384 tokens, D = 512, F = 1408: 390, 185, 365 and kFfnGrad 270
// us): matrix cores busy 80 to 85 % of the cycles, 63 % in kFfnGrad, which reads a and u
// in its epilogue.
template <int MODE, int WF, int WT, int NI, int NJ, int ST>
struct Product {
  static constexpr int WAVES = WF * WT;
  // Weights whose rows share a stage's feature rows, side by side in each wave's NI.
  static constexpr int MATS = MODE == kFfnGate || MODE == kFfnRedo ? 2 : 1;
  static constexpr int NF = NI / MATS;             // feature subtiles of a wave
  static constexpr int GS = NF % 4 == 0 ? 4 : 2;   // subtiles of a group
  static constexpr int FEATURES = 16 * NF * WF;    // of the output, a workgroup
  static constexpr int BF = 16 * NI * WF, BT = 16 * NJ * WT;
  static constexpr int LW = BF / (8 * WAVES), LT = BT / (8 * WAVES), LD = FEATURES / (8 * WAVES);
  static constexpr bool HALVES = ST == 5;
  // A unit of LDS: a stage, or either operand's half of one.
  static constexpr int UNIT = (HALVES ? std::max(BF, BT) : BF + BT) * 128;
  static constexpr int KE = 128 / ES;              // k of a step
  // Loads of a wave that are newer than a step's (at least: dh's steps have fewer).
  static constexpr int NEWER = HALVES ? LT : (ST - 2) * (LT + (MODE == kFfnRedo && LD < LW ? LD : LW));
  static_assert(NF % 2 == 0 && BF % (8 * WAVES) == 0 && BT % (8 * WAVES) == 0 && FEATURES % (8 * WAVES) == 0, "tile");
};

__device__ __forceinline__ u32x4 read16(const unsigned char* p) { return *reinterpret_cast<const u32x4*>(p); }

template <int MODE, int WF, int WT, int NI, int NJ, int ST, int OCC>
__global__ __launch_bounds__(64 * WF * WT, OCC) void ffn_product(FfnProduct p) {
  typedef Product<MODE, WF, WT, NI, NJ, ST> C;
  constexpr int NF = C::NF, GS = C::GS, NE = 4 * GS, WAVES = C::WAVES;
  constexpr bool REDO = MODE == kFfnRedo;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[ST][C::UNIT];
  const int nf = (p.F + C::FEATURES - 1) / C::FEATURES;
#if FST_EXPERTS
  ExpertTile tile;
  if (!expert_tile<C::BT>(p, p.first + blockIdx.x, nf, -1, tile)) return;
  const int f0 = tile.ft * C::FEATURES, t0 = tile.t0, tokens = tile.end;
  if (MODE == kFfnOut && tile.expert == p.experts) {  // rows of no expert
    constexpr int PARTS = C::FEATURES * ES / 16;
    for (int i = threadIdx.x; i < PARTS * C::BT; i += 64 * WAVES) {
      const int t = t0 + i / PARTS, f = f0 + i % PARTS * kVec<T>;
      if (t < tokens && f < p.F) *reinterpret_cast<u32x4*>(static_cast<T*>(p.out[0]) + (long)t * p.ldo + f) = u32x4{0, 0, 0, 0};
    }
    return;
  }
  const long w_at = (long)tile.expert * p.w_next * ES;
#else
  const int tokens = p.count ? *p.count : p.tokens;
  const int nt = (tokens + C::BT - 1) / C::BT;
  int ft, tt;
  if (!pick_tile(p.first + blockIdx.x, nf, nt, ft, tt)) return;
  const int f0 = ft * C::FEATURES, t0 = tt * C::BT;
  constexpr long w_at = 0;
#endif
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wf = wave % WF, wt = wave / WF, g = lane >> 4, n = lane & 15;

  // Loads: each fills 8 rows, lane l the 16 bytes at 16 l: row l / 8, part l & 7
  // of the layout above. Load i of a wave takes the rows 8 (i WAVES + wave) ..
  const int row8 = lane >> 3, m = 8 * (wave & 1) + row8;  // row of its subtile: WAVES is even
  const int part = (lane & 7) ^ ((m >> 1) & 7);
  const int row_bytes = (int)p.ldw * ES;
  // The feature of row m of feature subtile i (of a workgroup).
  auto feature = [&](int i) { return (i / GS) * 16 * GS + NE * (m >> 2) + 4 * (i % GS) + (m & 3); };
  int voff[C::LW], mat[C::LW];
#pragma unroll
  for (int i = 0; i < C::LW; ++i) {
    const int sub = (i * WAVES + wave) >> 1, of = sub % NI;
    mat[i] = of / NF;
    voff[i] = feature(sub / NI * NF + of % NF) * row_bytes + part * 16;
  }
  // Rows of the weights past F read as zeros (range of the buffer; the scalar
  // offset moves along k only and stays inside a row, as the range check
  // subtracts it from the buffer's size).
  const int range = (p.F - f0) * row_bytes;
  auto weight = [&](int k) {
    const uint64_t at = (uint64_t)p.w[k] + w_at + (uint64_t)f0 * row_bytes;  // a 48-bit address, stride 0
    return u32x4{(unsigned)at, (unsigned)(at >> 32) & 0xffffu, (unsigned)range, 0x00020000u};
  };
  const u32x4 wr0 = weight(0), wr1 = weight(C::MATS - 1), wr2 = weight(REDO ? 2 : 0);
  const char *xp[C::LT], *yp[REDO ? C::LT : 1];
#pragma unroll
  for (int i = 0; i < C::LT; ++i) {
    // Tokens past the last repeat it; their columns are not stored.
    const int t = min(t0 + 8 * (i * WAVES + wave) + row8, tokens - 1);
    const long r = p.rows_in ? p.rows_in[t] : t;
    xp[i] = static_cast<const char*>(p.x) + (r * p.ldx) * ES + part * 16;
    if constexpr (REDO) yp[i] = static_cast<const char*>(p.dy) + (r * p.lddy) * ES + part * 16;
  }
  const int steps = (p.K + C::KE - 1) / C::KE;
  const int tail = p.K % C::KE * ES;  // bytes of the last step, 0: all

  // Loads of k step s into stage b: x's contraction, and dh's. Parts past K are
  // zeros in both operands.
  const int total = REDO ? 2 * steps : steps;
  auto cut_at = [&](int s) { return tail != 0 && s == steps - 1 && part * 16 >= tail; };
  // Step v's rows of x, or dy after x's steps, and the weights'.
  auto issue_rows = [&](int v, unsigned char* dst) __attribute__((always_inline)) {
    const bool second = REDO && v >= steps;
    const int s = second ? v - steps : v;
    const bool cut = cut_at(s);
#pragma unroll
    for (int i = 0; i < C::LT; ++i) {
      const char* row = second ? yp[REDO ? i : 0] : xp[i];
      load_to_lds(cut ? reinterpret_cast<const char*>(&kZero16) : row + s * 128l, dst + (i * WAVES + wave) * 1024);
    }
  };
  auto issue_weights = [&](int v, unsigned char* dst) __attribute__((always_inline)) {
    if (REDO && v >= steps) {
      const int s = v - steps;
      const bool cut = cut_at(s);
#pragma unroll
      for (int i = 0; i < C::LD; ++i)
        load_to_lds(wr2, dst + (i * WAVES + wave) * 1024,
                    cut ? (int)0x80000000 : feature((i * WAVES + wave) >> 1) * row_bytes + part * 16, s * 128);
    } else {
      const bool cut = cut_at(v);
#pragma unroll
      for (int i = 0; i < C::LW; ++i)
        load_to_lds(C::MATS == 2 && mat[i] ? wr1 : wr0, dst + (i * WAVES + wave) * 1024, cut ? (int)0x80000000 : voff[i],
                    v * 128);
    }
  };

  f32x4 acc[NI][NJ], dh[REDO ? NF : 1][REDO ? NJ : 1];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
#pragma unroll
    for (int i = 0; i < NI; ++i) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (REDO) {
#pragma unroll
      for (int i = 0; i < NF; ++i) dh[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  const int rd = n * 128, swz = (n >> 1) & 7;
  if constexpr (C::HALVES) {
    issue_rows(0, lds[0]);
    issue_weights(0, lds[1]);
    if (total > 1) issue_rows(1, lds[2]);
  } else {
#pragma unroll
    for (int v = 0; v < ST - 1; ++v) {
      if (v < total) {
        issue_weights(v, lds[v]);
        issue_rows(v, lds[v] + C::BF * 128);
      }
    }
  }
  // Step v: it has landed, what the step before it read is free and loaded anew.
  const unsigned char *at_rows, *at_weights;
  int b = 0;
  auto step = [&](int v) __attribute__((always_inline)) {
    if (v + (C::HALVES ? 1 : ST - 2) < total)
      stage_wait<C::NEWER>();
    else
      stage_wait<0>();
    const auto unit = [&](int i) { return lds[b + i < ST ? b + i : b + i - ST]; };
    at_rows = unit(0) + rd + (C::HALVES ? 0 : C::BF * 128);
    at_weights = unit(C::HALVES ? 1 : 0) + rd;
    if constexpr (C::HALVES) {
      if (v + 1 < total) issue_weights(v + 1, unit(3));
      if (v + 2 < total) issue_rows(v + 2, unit(4));
      b = b + 2 < ST ? b + 2 : b + 2 - ST;
    } else {
      if (v + ST - 1 < total) {
        issue_weights(v + ST - 1, unit(ST - 1));
        issue_rows(v + ST - 1, unit(ST - 1) + C::BF * 128);
      }
      b = b == ST - 1 ? 0 : b + 1;
    }
  };
  for (int v = 0; v < steps; ++v) {
    step(v);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = ((4 * k + g) ^ swz) << 4;
      u32x4 fw[NI], fx[NJ];
#pragma unroll
      for (int i = 0; i < NI; ++i) fw[i] = read16(at_weights + c + (wf * NI + i) * 2048);
#pragma unroll
      for (int j = 0; j < NJ; ++j) fx[j] = read16(at_rows + c + (wt * NJ + j) * 2048);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[i][j] = Mma<T>::run(fw[i], fx[j], acc[i][j]);
    }
  }
  if constexpr (REDO) {
    for (int v = steps; v < total; ++v) {
      step(v);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c = ((4 * k + g) ^ swz) << 4;
        u32x4 fw[NF], fx[NJ];
#pragma unroll
        for (int i = 0; i < NF; ++i) fw[i] = read16(at_weights + c + (wf * NF + i) * 2048);
#pragma unroll
        for (int j = 0; j < NJ; ++j) fx[j] = read16(at_rows + c + (wt * NJ + j) * 2048);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < NF; ++i) dh[i][j] = Mma<T>::run(fw[i], fx[j], dh[i][j]);
      }
    }
  }

  // Epilogue: NE features of one token at a time.
#pragma unroll
  for (int q = 0; q < NF / GS; ++q) {
    const int f = f0 + (wf * (NF / GS) + q) * 16 * GS + NE * g;
    const int left = min(NE, p.F - f);
    if (left <= 0) continue;
    float b0[NE], b1[NE];  // zeros for experts, which have no biases
#pragma unroll
    for (int e = 0; e < NE; ++e) b0[e] = b1[e] = 0.f;
    if (!EXPERTS && MODE != kFfnGrad && p.bias[0]) load_run<NE>(static_cast<const T*>(p.bias[0]) + f, left, b0);
    if (!EXPERTS && C::MATS == 2 && p.bias[1]) load_run<NE>(static_cast<const T*>(p.bias[1]) + f, left, b1);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int t = t0 + (wt * NJ + j) * 16 + n;
      if (t >= tokens) continue;
      float v[NE], u[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        v[e] = acc[GS * q + (e >> 2)][j][e & 3];
        if constexpr (MODE != kFfnGrad && !EXPERTS) v[e] += b0[e];
        if constexpr (C::MATS == 2) {
          u[e] = acc[NF + GS * q + (e >> 2)][j][e & 3];
          if constexpr (!EXPERTS) u[e] += b1[e];
        }
      }
      if constexpr (MODE == kFfnGate) {
        const long at = (long)t * p.ldo + f;
        if (F32 && p.out[1]) {
          store_run<NE>(static_cast<T*>(p.out[1]) + at, left, v);
          store_run<NE>(static_cast<T*>(p.out[2]) + at, left, u);
        }
        activate_run<false, NE>(p.act, v, nullptr);
#pragma unroll
        for (int e = 0; e < NE; ++e) v[e] *= u[e];
        store_run<NE>(static_cast<T*>(p.out[0]) + at, left, v);
      } else if constexpr (MODE == kFfnOut) {
        const long r = p.rows_out ? p.rows_out[t] : t;
        store_run<NE>(static_cast<T*>(p.out[0]) + r * p.ldo + f, left, v);
      } else {
        float d[NE];
#pragma unroll
        for (int e = 0; e < NE; ++e) d[e] = REDO ? dh[REDO ? GS * q + (e >> 2) : 0][REDO ? j : 0][e & 3] : v[e];
        if constexpr (!REDO) {
          load_run<NE>(static_cast<const T*>(p.gate) + (long)t * p.F + f, left, v);
          load_run<NE>(static_cast<const T*>(p.up) + (long)t * p.F + f, left, u);
        }
        float slope[NE];
        activate_run<true, NE>(p.act, v, slope);
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const float act = v[e];
          v[e] = d[e] * u[e] * slope[e];
          u[e] = d[e] * act;
        }
        T* out = static_cast<T*>(p.out[0]) + (long)t * p.ldo + f;
        store_run<NE>(out, left, v);
        store_run<NE>(out + p.F, left, u);
      }
    }
  }
}

// The same products for at most 16 NJ rows. Eight waves share 16 features (of each
// weight) by the tokens and split k between them in contiguous runs, straight from memory
// into registers: no stage waits for another, and the longest chain is an eighth
// of k. The partial sums meet in LDS and are added in the waves' order.
template <int MODE, int NJ>
__global__ __launch_bounds__(512, MODE == kFfnRedo && NJ == 4 ? 2 : 4) void ffn_few(FfnProduct p) {
  constexpr bool REDO = MODE == kFfnRedo;
  constexpr int MATS = MODE == kFfnGate || REDO ? 2 : 1, ACCS = REDO ? 3 : MATS, KE = 64 / ES, AHEAD = NJ == 1 ? 4 : 2;
  __shared__ f32x4 lds[8][ACCS * NJ][64];
#if FST_EXPERTS
  ExpertTile tile;
  if (!expert_tile<16 * NJ>(p, 0, 0, blockIdx.y, tile)) return;
  const int t0 = tile.t0, tokens = tile.end;
  if (MODE == kFfnOut && tile.expert == p.experts) {  // rows of no expert
    constexpr int PARTS = 16 * ES / 16;
    const int t = t0 + threadIdx.x / PARTS, f = blockIdx.x * 16 + threadIdx.x % PARTS * kVec<T>;
    if ((int)threadIdx.x < PARTS * 16 * NJ && t < tokens && f < p.F)
      *reinterpret_cast<u32x4*>(static_cast<T*>(p.out[0]) + (long)t * p.ldo + f) = u32x4{0, 0, 0, 0};
    return;
  }
  const long w_at = (long)tile.expert * p.w_next * ES;
#else
  const int tokens = p.count ? *p.count : p.tokens;
  if (tokens <= 0) return;
  constexpr int t0 = 0;
  constexpr long w_at = 0;
#endif
  const int f0 = blockIdx.x * 16, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int row_bytes = (int)p.ldw * ES;
  const int steps = (p.K + KE - 1) / KE, per = (steps + 7) / 8;
  const int s0 = wave * per, s1 = min(s0 + per, steps);

  f32x4 acc[ACCS][NJ];
#pragma unroll
  for (int a = 0; a < ACCS; ++a)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[a][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // acc[A0 .. A0 + MM) += the weights W0 .. against the tokens' rows of x.
  auto contract = [&](auto first, auto count, int w0, const void* x, long ldx) __attribute__((always_inline)) {
    constexpr int A0 = decltype(first)::value, MM = decltype(count)::value;
    const char *wp[MM], *xp[NJ];
#pragma unroll
    for (int a = 0; a < MM; ++a)
      wp[a] = static_cast<const char*>(p.w[w0 + a]) + w_at + (long)min(f0 + n, p.F - 1) * row_bytes + g * 16;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int t = min(t0 + 16 * j + n, tokens - 1);  // past the last token: not stored
      const long r = p.rows_in ? p.rows_in[t] : t;
      xp[j] = static_cast<const char*>(x) + r * ldx * ES + g * 16;
    }
    for (int s = s0; s < s1; s += AHEAD) {
      u32x4 fw[AHEAD][MM], fx[AHEAD][NJ];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        // Steps past the run and parts past K read zeros.
        const bool in = s + q < s1 && (s + q) * KE + g * (16 / ES) < p.K;
        const char* zero = reinterpret_cast<const char*>(&kZero16);
#pragma unroll
        for (int a = 0; a < MM; ++a) fw[q][a] = *reinterpret_cast<const u32x4*>(in ? wp[a] + (s + q) * 64 : zero);
#pragma unroll
        for (int j = 0; j < NJ; ++j) fx[q][j] = *reinterpret_cast<const u32x4*>(in ? xp[j] + (s + q) * 64 : zero);
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int a = 0; a < MM; ++a) acc[A0 + a][j] = Mma<T>::run(fw[q][a], fx[q][j], acc[A0 + a][j]);
    }
  };
  contract(std::integral_constant<int, 0>{}, std::integral_constant<int, MATS>{}, 0, p.x, p.ldx);
  if constexpr (REDO) contract(std::integral_constant<int, 2>{}, std::integral_constant<int, 1>{}, 2, p.dy, p.lddy);
#pragma unroll
  for (int a = 0; a < ACCS; ++a)
#pragma unroll
    for (int j = 0; j < NJ; ++j) lds[wave][a * NJ + j][lane] = acc[a][j];
  __syncthreads();
  if (wave >= NJ) return;
  // Wave j: features 4 g .. 4 g + 3 of token n of subtile j.
  const int f = f0 + 4 * g, t = t0 + 16 * wave + n;
  if (f >= p.F || t >= tokens) return;
  float v[ACCS][4];
#pragma unroll
  for (int a = 0; a < ACCS; ++a) {
    f32x4 sum = lds[0][a * NJ + wave][lane];
#pragma unroll
    for (int w = 1; w < 8; ++w) sum += lds[w][a * NJ + wave][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[a][e] = sum[e];
      if (!EXPERTS && MODE != kFfnGrad && a < MATS && p.bias[a < 2 ? a : 0])
        v[a][e] += (float)static_cast<const T*>(p.bias[a < 2 ? a : 0])[f + e];
    }
  }
  typedef T T4 __attribute__((ext_vector_type(4)));
  auto store = [&](void* out, long at, const float* q) {
    T4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (T)q[e];
    *reinterpret_cast<T4*>(static_cast<T*>(out) + at) = o;
  };
  const long r = MODE == kFfnOut && p.rows_out ? p.rows_out[t] : t, at = r * p.ldo + f;
  if constexpr (MODE == kFfnGate) {
    if (F32 && p.out[1]) {
      store(p.out[1], at, v[0]);
      store(p.out[2], at, v[1]);
    }
    activate_run<false, 4>(p.act, v[0], nullptr);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[0][e] *= v[1][e];
    store(p.out[0], at, v[0]);
  } else if constexpr (MODE == kFfnOut) {
    store(p.out[0], at, v[0]);
  } else {
    float act[4], slope[4], da[4], du[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) act[e] = REDO ? v[0][e] : (float)static_cast<const T*>(p.gate)[(long)t * p.F + f + e];
    activate_run<true, 4>(p.act, act, slope);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float u = REDO ? v[MATS - 1][e] : (float)static_cast<const T*>(p.up)[(long)t * p.F + f + e];
      const float dh = v[ACCS - 1][e];
      da[e] = dh * u * slope[e];
      du[e] = dh * act[e];
    }
    store(p.out[0], at, da);
    store(p.out[0], at + p.F, du);
  }
}

// ---------------------------------------------------------------------------
// Weights' gradients. LDS holds rows of tokens, features along them: 16-bit
// types read them transposed (ds_read_tr16), float32 element by element. A
// stage is 32 tokens of the tile's M features of a and N of b, and all stages but
// one are in flight: a token's row is a few lines far from the next row's, part of
// which always comes from beyond L2 (two stages of 64 tokens took 1365 us, their
// loads alone 876, the products alone 763: 65536 tokens, D = 1024, F = 2752 bf16; four
// of 32 take 1092). float32, bound by the matrix cores, runs two. 32-byte (float32:
// 64-byte) slices of 16 features are stored in an order that depends on the row, so
// that the rows of a read pass cover the banks once.
// ---------------------------------------------------------------------------
constexpr int KT = 32, OUTER_STAGES = F32 ? 2 : 4;

// One operand's side: FEATS features, loaded by NT threads. MAP: the tokens' rows
// come from a list, of which LDS holds the entries of a few steps (RowList).
template <int FEATS, int NT, bool MAP>
struct OuterSide {
  static constexpr int ROW = FEATS * ES;  // bytes of a token's row
  static constexpr int PARTS = ROW / 16;
  static constexpr int LOADS = KT * PARTS / NT;
  static_assert(KT * PARTS % NT == 0, "whole loads");

  const char* base[LOADS];  // this lane's part of row 0 in each load
  unsigned ld[LOADS];       // row stride in bytes; 0 where the features do not exist
  int r[LOADS];             // its row of the stage

  // Order of the slices of row r, in 16-byte parts.
  static __device__ __forceinline__ int swizzle(int r) {
    return F32 ? (r & 3) << 2 : (r & 7) << 1;
  }
  __device__ __forceinline__ void init(const void* p, long ld_elems, int f0, int count, int tid) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int at = i * NT + tid;
      r[i] = at / PARTS;
      const int f = f0 + ((at % PARTS) ^ swizzle(r[i])) * kVec<T>;
      const bool in = f < count;
      base[i] = in ? static_cast<const char*>(p) + (long)f * ES : reinterpret_cast<const char*>(&kZero16);
      ld[i] = in ? (unsigned)(ld_elems * ES) : 0;
    }
  }
  // rows: the step's entries of the list (MAP).
  __device__ __forceinline__ void issue(int t0, int t1, const int32_t* rows, unsigned char* dst, int wave) const {
    const bool whole = t0 + KT <= t1;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const unsigned row = MAP ? rows[r[i]] : t0 + r[i];
      const char* q = base[i] + (uint64_t)row * ld[i];
      if (!whole) q = t0 + r[i] < t1 ? q : reinterpret_cast<const char*>(&kZero16);
      load_to_lds(q, dst + i * NT * 16 + wave * 1024);
    }
  }
  // Subtile `sub` (16 features) of the stage's tokens as a matrix-core operand.
  // 16-bit: tokens 4 g + .., 16 + 4 g + .. in the lane's eight slots; float32: step
  // e (of four) holds token 4 e + g.
  static __device__ __forceinline__ u32x4 frag(const unsigned char* tile, int sub, int g, int n) {
    if constexpr (F32) {
      u32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * e + g;
        v[e] = *reinterpret_cast<const unsigned*>(tile + r * ROW + (((sub << 2) ^ swizzle(g)) << 4) + 4 * n);
      }
      return v;
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
      const int r = 4 * g + (n >> 2), at = (((sub << 1) ^ swizzle(r)) << 4) + 8 * (n & 3);
      const unsigned char* p = tile + r * ROW + at;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 16 * ROW));
      const u32x2 a = __builtin_bit_cast(u32x2, lo), c = __builtin_bit_cast(u32x2, hi);
      return u32x4{a[0], a[1], c[0], c[1]};
    }
  }
};

// Experts: a piece of an expert's run.
struct OuterRun {
  int expert, piece;
};

template <int WM, int WN, int NI, int NJ, bool MA, bool MB>
__device__ __forceinline__ void outer_tile(const FfnOuter& p, const FfnOuters& all, int wg, unsigned char* lds,
                                           int32_t* list, OuterRun at_run = {}) {
  constexpr int TM = 16 * NI * WM, TN = 16 * NJ * WN, NT = 64 * WM * WN;
  typedef OuterSide<TM, NT, MA> SideA;
  typedef OuterSide<TN, NT, MB> SideB;
  constexpr int A_BYTES = KT * SideA::ROW, STAGE = A_BYTES + KT * SideB::ROW;
  const int nm = (p.M + TM - 1) / TM, nn = (p.N + TN - 1) / TN;
#if FST_EXPERTS
  // Tile wg of an expert's piece of its run.
  const int split = at_run.expert * p.splits + at_run.piece, tile = wg;
  const int first = min(max(all.offsets[at_run.expert], 0), all.tokens);
  const int end = max(min(all.offsets[at_run.expert + 1], all.tokens), first);
  const int run = ((end - first + p.splits - 1) / p.splits + KT - 1) / KT * KT;
  const int t0 = (int)min(first + (long)at_run.piece * run, (long)end), t1 = (int)min((long)t0 + run, (long)end);
#else
  // Consecutive workgroups of an XCD take the tiles of one run of tokens.
  const int total = nm * nn * p.splits, per = (total + 7) >> 3;
  const int i8 = wg >> 3, at = (wg & 7) * per + i8;
  if (i8 >= per || at >= total) return;
  const int split = at / (nm * nn), tile = at - split * nm * nn;
  const int tokens = all.count ? *all.count : all.tokens;
  const int run = ((tokens + p.splits - 1) / p.splits + KT - 1) / KT * KT;
  const int t0 = (int)min((long)split * run, (long)tokens), t1 = (int)min((long)t0 + run, (long)tokens);
#endif
  const int m0 = tile % nm * TM, n0 = tile / nm * TN;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM, g = lane >> 4, n = lane & 15;
  SideA a;
  SideB bb;
  a.init(p.a, p.lda, m0, p.M, tid);
  bb.init(p.b, p.ldb, n0, p.N, tid);
  // The bias' gradient: the columns of b against a row of ones, in the first
  // waves of the first tile of m. Sums of 256 tokens are added up apart: one chain over
  // a run had a float32 column's rounding grow with its length.
  const bool sums = p.bias && m0 == 0 && wm == 0;
  const unsigned one = F32 ? 0x3f800000u : (__is_same(T, bf16) ? 0x3f803f80u : 0x3c003c00u);
  const u32x4 ones = {one, one, one, one};
  f32x4 acc[NI][NJ], sum[NJ];
  float whole[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    whole[j] = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // The list's rows of the tokens, in LDS by chunks of NT, two at a time: loaded as
  // the stages are, a chunk ahead of the steps that use it, so that no load waits
  // for a load (rows read into registers a step ahead had the compiler wait for
  // everything in flight: 585 against 335 us, 256 x 768 padded, D = 384, F = 1024).
  constexpr bool MAP = MA || MB;
  const auto load_rows = [&](int t) __attribute__((always_inline)) {
    const int32_t* from = all.rows + min(t + tid, t1 - 1);
    const int32_t* dst = list + ((t - t0) & (2 * NT - 1)) + 64 * wave;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(
                     lds_offset(reinterpret_cast<const unsigned char*>(dst))),
                 "v"(from)
                 : "memory");
  };
  const auto issue = [&](int t, unsigned char* dst) __attribute__((always_inline)) {
    const int32_t* rows = MAP ? list + ((t - t0) & (2 * NT - 1)) : nullptr;
    a.issue(t, t1, rows, dst, wave);
    bb.issue(t, t1, rows, dst + A_BYTES, wave);
  };
  if (MAP && t0 < t1) {
    load_rows(t0);
    stage_wait<0>();
  }
#pragma unroll
  for (int q = 0; q < OUTER_STAGES - 1; ++q)
    if (t0 + q * KT < t1) issue(t0 + q * KT, lds + q * STAGE);
  constexpr int LOADS = SideA::LOADS + SideB::LOADS;  // a step's; those of the list only tighten the wait
  static_assert(NT >= (2 * OUTER_STAGES - 1) * KT, "a chunk of the list has landed before its first step is loaded");
  int b = 0;
  for (int t = t0; t < t1; t += KT) {
    // A wave has issued two steps' loads since this step's.
    if (t + (OUTER_STAGES - 2) * KT < t1)
      stage_wait<(OUTER_STAGES - 2) * LOADS>();
    else
      stage_wait<0>();
    if (MAP && ((t - t0) & (NT - 1)) == 0 && t + NT < t1) load_rows(t + NT);
    if (t + (OUTER_STAGES - 1) * KT < t1) issue(t + (OUTER_STAGES - 1) * KT, lds + (b == 0 ? OUTER_STAGES - 1 : b - 1) * STAGE);
    const unsigned char* now = lds + b * STAGE;
#pragma unroll
    for (int k = 0; k < KT * ES / 64; ++k) {
      u32x4 fa[NI], fb[NJ];
#pragma unroll
      for (int i = 0; i < NI; ++i) fa[i] = SideA::frag(now + k * (64 / ES) * SideA::ROW, wm * NI + i, g, n);
#pragma unroll
      for (int j = 0; j < NJ; ++j) fb[j] = SideB::frag(now + A_BYTES + k * (64 / ES) * SideB::ROW, wn * NJ + j, g, n);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[i][j] = Mma<T>::run(fa[i], fb[j], acc[i][j]);
      if (sums) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) sum[j] = Mma<T>::run(ones, fb[j], sum[j]);
      }
    }
    if (sums && ((t - t0) & 255) == 256 - KT) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        whole[j] += sum[j][0];
        sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
    b = b == OUTER_STAGES - 1 ? 0 : b + 1;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int nr = n0 + (wn * NJ + j) * 16 + n;
    if (nr >= p.N) continue;
    if (EXPERTS && !p.part) {
      const bool low = nr < p.half;
      T* out = static_cast<T*>(p.direct[low ? 0 : 1]);
      if (!out) continue;
      out += ((long)split * (low ? p.half : p.N - p.half) + (low ? nr : nr - p.half)) * p.M;
      typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int m = m0 + (wm * NI + i) * 16 + 4 * g;
        T4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)acc[i][j][e];
        if (m < p.M) *reinterpret_cast<T4*>(out + m) = o;
      }
      continue;
    }
    float* out = p.part + ((long)split * p.N + nr) * p.M;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int m = m0 + (wm * NI + i) * 16 + 4 * g;
      if (m < p.M) *reinterpret_cast<f32x4*>(out + m) = acc[i][j];
    }
    if (sums && g == 0) p.bias[(long)split * p.N + nr] = whole[j] + sum[j][0];
  }
}

// Experts: the weights' tiles are numbered expert by expert, `tiles` to each. XCD x takes
// those whose work begins in the x-th eighth of all: a tile's is its expert's tokens, and
// as much as kTileTokens of them for its start and its stores. As many tiles to each
// left an XCD with the largest loads running alone (65536 rows over 32 experts of 0 to 1.5
// times the mean, D = 1024, F = 1376 bf16: 777 us, so 679).
constexpr int kTileTokens = 128;

__device__ __forceinline__ void tiles_of_xcd(const FfnOuters& ps, int tiles, int xcd, int& first, int& last) {
  const int lane = threadIdx.x & 63;
  int upto, work;  // of expert e0 + lane: the work of a column of tiles up to it, and its own
  const auto scan = [&](int e0) __attribute__((always_inline)) {
    const int e = e0 + lane;
    const int from = e < ps.experts ? min(max(ps.offsets[e], 0), ps.tokens) : 0;
    const int to = e < ps.experts ? min(max(ps.offsets[e + 1], 0), ps.tokens) : 0;
    work = upto = e < ps.experts ? max(to - from, 0) + kTileTokens : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int below = __shfl_up(upto, d);
      if (lane >= d) upto += below;
    }
  };
  long all = 0;
  for (int e0 = 0; e0 < ps.experts; e0 += 64) {
    scan(e0);
    all += __builtin_amdgcn_readlane(upto, 63);
  }
  // The first tile whose work begins at `share` of all or later.
  const auto tile_at = [&](long share) __attribute__((always_inline)) {
    long before = 0;
    for (int e0 = 0; e0 < ps.experts; e0 += 64) {
      if (ps.experts > 64) scan(e0);
      const long sum = __builtin_amdgcn_readlane(upto, 63);
      if (share < tiles * (before + sum)) {
        const int src = __builtin_ctzll(__ballot(share < tiles * (before + upto)));
        const long own = __builtin_amdgcn_readlane(work, src);
        const long left = share - tiles * (before + __builtin_amdgcn_readlane(upto - work, src));
        return (e0 + src) * tiles + (int)min(max((left + own - 1) / own, 0l), (long)tiles);
      }
      before += sum;
    }
    return ps.experts * tiles;
  };
  first = tile_at(xcd * (tiles * all) / 8);
  last = xcd == 7 ? ps.experts * tiles : tile_at((xcd + 1) * (tiles * all) / 8);
}

// A workgroup's tile is DT of D by FT of F (or 2 F) features: D is the first
// problem's m and the second's n. PADDED: the tokens' rows of x (the first's a) and
// dy (the second's b) come from the list.
template <int DT, int FT, int WF, bool PADDED, int OCC>
__global__ __launch_bounds__(128 * WF, OCC) void ffn_outer(FfnOuters ps) {
  constexpr int ND = DT / 16, NF = FT / 16;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[OUTER_STAGES * KT * ES * (DT + FT)];
  __shared__ __attribute__((aligned(256))) int32_t list[PADDED ? 2 * 128 * WF : 1];
  const int wg = blockIdx.x;
#if FST_EXPERTS
  // Both problems' tiles of a piece of a run one after the other: they share its rows.
  const auto tiles = [](const FfnOuter& p, int m, int n) { return p.splits ? ((p.M + m - 1) / m) * ((p.N + n - 1) / n) : 0; };
  const int one = tiles(ps.p[0], DT, FT), piece = one + tiles(ps.p[1], FT, DT), splits = max(ps.p[0].splits, ps.p[1].splits);
  int at, last;
  tiles_of_xcd(ps, piece * splits, wg & 7, at, last);
  for (at += wg >> 3; at < last; at += gridDim.x >> 3) {
    const int run = at / piece, tile = at - run * piece;
    const OuterRun r{run / splits, run % splits};
    if (tile < one)
      outer_tile<2, WF, ND / 2, NF / WF, false, false>(ps.p[0], ps, tile, lds, list, r);
    else
      outer_tile<2, WF, NF / 2, ND / WF, false, false>(ps.p[1], ps, tile - one, lds, list, r);
    __syncthreads();  // before the next tile is loaded over what this one read
  }
#else
  if (wg < ps.first)
    outer_tile<2, WF, ND / 2, NF / WF, PADDED, false>(ps.p[0], ps, wg, lds, list);
  else
    outer_tile<2, WF, NF / 2, ND / WF, false, PADDED>(ps.p[1], ps, wg - ps.first, lds, list);
#endif
}

// Tiles of t tokens, at most: each run, and the rows before and behind them, may end in a
// tile of its own.
long token_tiles(const FfnProduct& p, int t) {
  if (EXPERTS) return p.tokens / t + std::min(p.tokens, p.experts) + (p.tail ? 2 : 0);
  return (p.tokens + t - 1) / t;
}

// A launch takes fewer than 2^32 lanes, which narrow rows pass at 2^30 of them: as many
// launches as that needs.
template <int MODE, int WF, int WT, int NI, int NJ, int ST, int OCC>
void launch(FfnProduct p, hipStream_t st) {
  typedef Product<MODE, WF, WT, NI, NJ, ST> C;
  constexpr long most = (1l << 31) / (64 * WF * WT);
  const long tiles = (long)((p.F + C::FEATURES - 1) / C::FEATURES) * token_tiles(p, C::BT);
  // Experts: the tiles of no run begin at a multiple of eight.
  const long grid = (tiles + 7) / 8 * 8 + (EXPERTS ? 8 : 0);
  for (long first = 0; first < grid; first += most) {
    p.first = (int)first;
    ffn_product<MODE, WF, WT, NI, NJ, ST, OCC><<<(unsigned)std::min(grid - first, most), 64 * WF * WT, 0, st>>>(p);
  }
}

constexpr int kFewTokens = 64;

// Tokens that share weights: all, or an expert's if the loads are even.
int tokens_of_run(const FfnProduct& p) { return EXPERTS ? (p.tokens + p.experts - 1) / p.experts : p.tokens; }

template <int MODE>
void launch_few(const FfnProduct& p, hipStream_t st) {
  const unsigned nf = (unsigned)((p.F + 15) / 16);
  const auto grid = [&](int t) { return EXPERTS ? dim3(nf, (unsigned)token_tiles(p, t)) : dim3(nf); };
  if (tokens_of_run(p) <= 16)
    ffn_few<MODE, 1><<<grid(16), 512, 0, st>>>(p);
  else
    ffn_few<MODE, 4><<<grid(64), 512, 0, st>>>(p);
}

// The tiles of a product: 256 x 256 features (of all weights) by tokens, one
// workgroup of eight waves a CU; 128 x 128, four waves, two a CU; 64 x 64, four
// waves, two a CU with four stages (in calls this small the operands come from far:
// with two stages 9.4 and 17.6 us where four take 7.3 and 12.8, [1024, 384] at K = 1024
// and 2048). A k step (64 elements of 16 bits) of n workgroups on every CU takes about
// 1.65 n, 0.54 n (one alone 0.64) and 0.24 n (alone 0.28) us, measured on [tokens, F,
// K] = [65536, 2752, 1024], [7640, 768, 2048], [1024, 384, 2048] (bf16, in one run: large 362 /
// 58 / 48 us, middle 405 / 33 / 21, small - / 45 / 13). Up to 64 tokens the waves split k
// instead (ffn_few: 4 tokens, D = 768, F = 2048 7.4 + 15.3 us in 64 x 64 tiles, 6.2 + 5.6;
// 187 tokens, D = 384, F = 1024 5.7 + 7.0 against 6.4 + 7.2). float32 is bound by the
// matrix cores four times as long in each: as fast in the middle tile as in the
// large one, which it does without. kFfnRedo has no small tile: one round of the
// middle one takes 0.35 us a step, of a small one 0.36, more rounds less by more.
enum Tile { kLarge, kMiddle, kSmall, kFew };

Tile pick(const FfnProduct& p, int mats, bool redo) {
  // float32 pays for all 64 rows of a tile, of which a few experts' runs fill an eighth (rows
  // over 64 experts, D = 1024, F = 1376, forward, in small tiles / split over the waves: 256 rows
  // 346 / 237 us, 512 336 / 257, 1024 331 / 356); 16-bit types do not (512 rows 115 / 135).
  if (p.tokens <= kFewTokens || (EXPERTS && F32 && tokens_of_run(p) <= 12)) return kFew;
  const auto load = [&](int f, int t) {
    // Experts: each run ends in half a tile.
    const long down = EXPERTS ? p.tokens / t + (std::min(p.tokens, p.experts) + 1) / 2 : (p.tokens + t - 1) / t;
    const long tiles = (long)((p.F + f - 1) / f) * down;
    return (double)((tiles + 255) / 256);
  };
  const double nl = load(256 / mats, redo ? 192 : 256), nm = load(128 / mats, redo ? 64 : 128), ns = load(64 / mats, 64);
  // Many runs leave partly filled rounds, and float32's tiles cost what their products do:
  // 2.3 n and 0.62 n us a step of middle and small ones (16384 tokens over 8 experts, D =
  // 512, F = 704: output product 148 and 123 us, its gradient 181 and 138, dx 284 and 237,
  // the gate 229 and 232).
  if (EXPERTS && F32) return 2.3 * nm <= 0.62 * ns * (mats == 2 ? 1.03 : 1.0) ? kMiddle : kSmall;
  // Two weights' 64 x 64 tile has a quarter of each operand's rows reused less.
  const double large = 1.65 * nl * (redo ? 0.75 : 1.0), middle = (nm > 1 ? 0.54 * nm : 0.64) * (redo ? 0.55 : 1.0),
               small = (ns > 1 ? 0.24 * ns : 0.28) * (mats == 2 ? 1.3 : 1.0);
  if (!F32 && large <= middle && (redo || large <= small)) return kLarge;
  return redo || middle <= small ? kMiddle : kSmall;
}

template <int DT, int FT, int WF, int OCC>
void launch_outer(FfnOuters& ps, hipStream_t st) {
  const auto tiles = [&](const FfnOuter& p, int m, int n) {
    return (p.splits * (EXPERTS ? ps.experts : 1) * ((p.M + m - 1) / m) * ((p.N + n - 1) / n) + 7) / 8 * 8;
  };
  ps.first = tiles(ps.p[0], DT, FT);
  const int grid = ps.first + tiles(ps.p[1], FT, DT);
  if constexpr (!EXPERTS) {
    if (ps.rows) {
      ffn_outer<DT, FT, WF, true, OCC><<<grid, 128 * WF, 0, st>>>(ps);
      return;
    }
  }
  ffn_outer<DT, FT, WF, false, OCC><<<grid, 128 * WF, 0, st>>>(ps);
}

}  // namespace

#define FST_CAT2(a, b) a##b
#define FST_CAT(a, b) FST_CAT2(a, b)

static Tile tile_of(int mode, const FfnProduct& p) {
  return pick(p, mode == kFfnGate || mode == kFfnRedo ? 2 : 1, mode == kFfnRedo);
}

int FST_CAT(ffn_tile_, FST_NAME)(int mode, const FfnProduct& p) {
  constexpr int side[] = {256, 128, 64, 16};
  return side[tile_of(mode, p)];
}

int FST_CAT(ffn_product_, FST_NAME)(int mode, const FfnProduct& p, hipStream_t st) {
  const Tile tile = tile_of(mode, p);
  if constexpr (!F32) {
    if (tile == kLarge) {
      if (mode == kFfnGate)
        launch<kFfnGate, 2, 4, 8, 4, 5, 1>(p, st);
      else if (mode == kFfnOut)
        launch<kFfnOut, 2, 4, 8, 4, 5, 1>(p, st);
      else
        launch<kFfnRedo, 2, 4, 8, 3, 5, 1>(p, st);
      return hipGetLastError() == hipSuccess ? FST_OK : FST_ELAUNCH;
    }
  }
  constexpr int BACK = F32 ? kFfnGrad : kFfnRedo;
  if (tile == kFew) {
    if (mode == kFfnGate)
      launch_few<kFfnGate>(p, st);
    else if (mode == kFfnOut)
      launch_few<kFfnOut>(p, st);
    else
      launch_few<BACK>(p, st);
  } else if (tile == kMiddle) {
    if (mode == kFfnGate)
      launch<kFfnGate, 2, 2, 4, 4, 2, 2>(p, st);
    else if (mode == kFfnOut)
      launch<kFfnOut, 2, 2, 4, 4, 2, 2>(p, st);
    else
      launch<BACK, 2, 2, 4, F32 ? 4 : 2, 2, 2>(p, st);
  } else {
    // float32 experts run them in large calls too, where two stages and four workgroups a CU
    // keep the matrix cores busier than four and two (pick's example: output product 134
    // -> 123 us, its gradient 154 -> 138, dx 254 -> 237).
    constexpr int ST = EXPERTS && F32 ? 2 : 4, OCC = EXPERTS && F32 ? 4 : 2;
    if (mode == kFfnGate)
      launch<kFfnGate, 1, 4, 4, 1, ST, OCC>(p, st);
    else if (mode == kFfnOut)
      launch<kFfnOut, 2, 2, 2, 2, ST, OCC>(p, st);
    else if constexpr (F32)
      launch<kFfnGrad, 2, 2, 2, 2, ST, OCC>(p, st);
  }
  return hipGetLastError() == hipSuccess ? FST_OK : FST_ELAUNCH;
}

int FST_CAT(ffn_outer_, FST_NAME)(FfnOuters& p, int tile, hipStream_t st) {
  if constexpr (!F32) {
    if (tile == 256) launch_outer<256, 256, 4, 1>(p, st);
  }
  if (tile == 128) launch_outer<128, 128, 2, 2>(p, st);
  return hipGetLastError() == hipSuccess ? FST_OK : FST_ELAUNCH;
}

}  // namespace fst
