// The feed-forward block's matrix products for one element type, built with
// -DFST_T=<bf16|f16|float> -DFST_NAME=<bf16|f16|f32>.
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

namespace fst {

namespace {

typedef FST_T T;
constexpr int ES = sizeof(T);
constexpr bool F32 = ES == 4;

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* glb_ptr;

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

// 16 bytes a lane from the buffer into LDS (wave-uniform base, lane l's at 16 l).
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, unsigned char* dst, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)dst, 16, voff, soff, 0, 0);
}

// act(a), and with D its derivative. sigmoid from the hardware's exp2 and
// reciprocal (1 ulp each). Phi(a) = erfc(-a / sqrt 2) / 2 with Abramowitz and
// Stegun's formula 7.1.26 for erfc (absolute error 1.5e-7), whose exp(-a^2 / 2)
// is also the density in the derivative.
template <bool D>
__device__ __forceinline__ float activate(int kind, float a, float& slope) {
  if (kind == FST_GELU) {
    const float x = fabsf(a) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f));
    const float e = __expf(-x * x);
    const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float q = 0.5f * p * e;  // Phi(-|a|)
    const float phi = a < 0.f ? q : 1.f - q;
    if constexpr (D) slope = fmaf(a * e, 0.39894228040143268f, phi);
    return a * phi;
  }
  float z = a, dz = 1.f;  // the sigmoid's argument and its derivative
  if (kind == FST_GELU_TANH) {
    const float c = 1.59576912160573071f, s = a * a;  // 2 sqrt(2 / pi)
    z = c * a * fmaf(0.044715f, s, 1.f);
    if constexpr (D) dz = c * fmaf(3.f * 0.044715f, s, 1.f);
  }
  const float g = __builtin_amdgcn_rcpf(1.f + __expf(-z));
  if constexpr (D) slope = g * fmaf(a * dz, 1.f - g, 1.f);
  return a * g;
}

// 16 consecutive elements: loads and stores of `n` of them (a multiple of 8).
__device__ __forceinline__ void load16(const T* p, int n, float* v) {
  constexpr int V = kVec<T>;
#pragma unroll
  for (int q = 0; q < 16 / V; ++q) {
    typename Piece<T>::V x;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (T)0.f;
    if (q * V < n) x = *reinterpret_cast<const typename Piece<T>::V*>(p + q * V);
#pragma unroll
    for (int i = 0; i < V; ++i) v[q * V + i] = (float)x[i];
  }
}
__device__ __forceinline__ void store16(T* p, int n, const float* v) {
  constexpr int V = kVec<T>;
#pragma unroll
  for (int q = 0; q < 16 / V; ++q)
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

// Workgroups of 256 threads: WF x WT waves of NI x NJ subtiles of 16 features by
// 16 tokens. The weight is the matrix core's row operand, so a lane ends up
// with the same 16 consecutive features (of each 64) of its tokens: slot m =
// 4 a + r of subtile s of a group holds feature 16 a + 4 s + r, which the
// loads into LDS arrange. LDS rows are 64 bytes of k; 16-byte part c of row r
// sits at c ^ ((r >> 2) & 3), so that the 16 rows of a read pass cover the
// banks once. Three stages: the loads of two k steps are in flight while a
// third is multiplied, one barrier a step.
template <int MODE, int WF, int WT, int NI, int NJ>
struct Product {
  static constexpr int BF = 16 * NI * WF, BT = 16 * NJ * WT, ROWS = BF + BT;
  static constexpr int FEATURES = MODE == kFfnGate ? BF / 2 : BF;  // of the output
  static constexpr int LW = BF / 64, LT = BT / 64;
  static constexpr int STAGE = ROWS * 64;
  static constexpr int KE = 64 / ES;  // k of a step
};

template <int MODE, int WF, int WT, int NI, int NJ>
__global__ __launch_bounds__(256, 2) void ffn_product(FfnProduct p) {
  typedef Product<MODE, WF, WT, NI, NJ> C;
  static_assert(WF * WT == 4 && NI % (MODE == kFfnGate ? 8 : 4) == 0, "waves and feature groups");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[3][C::STAGE];
  const int tokens = p.count ? *p.count : p.tokens;
  const int nf = (p.F + C::FEATURES - 1) / C::FEATURES, nt = (tokens + C::BT - 1) / C::BT;
  int ft, tt;
  if (!pick_tile(blockIdx.x, nf, nt, ft, tt)) return;
  const int f0 = ft * C::FEATURES, t0 = tt * C::BT;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wf = wave % WF, wt = wave / WF, g = lane >> 4, n = lane & 15;

  // Loads: wave w fills subtile w of each group of 64 rows, lane l the 16 bytes
  // at 16 l of it: row l / 4, part (l & 3) of the layout above.
  const int row = lane >> 2, part = (lane & 3) ^ ((row >> 2) & 3);
  const int wrow = 16 * (row >> 2) + 4 * wave + (row & 3);
  const int row_bytes = (int)p.ldw * ES;
  // The scalar offset moves along k only and stays inside a row: the range
  // check subtracts it from the buffer's size.
  int voff[C::LW];
#pragma unroll
  for (int i = 0; i < C::LW; ++i) voff[i] = (wrow + 64 * (MODE == kFfnGate ? i >> 1 : i)) * row_bytes + part * 16;
  // Rows of the weight past F read as zeros (range of the buffer).
  const int range = (p.F - f0) * row_bytes;
  const __amdgpu_buffer_rsrc_t wr0 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(p.w[0]) + (long)f0 * row_bytes), (short)0, range, 0x00020000);
  const __amdgpu_buffer_rsrc_t wr1 = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(p.w[MODE == kFfnGate]) + (long)f0 * row_bytes), (short)0, range, 0x00020000);
  const char* xp[C::LT];
#pragma unroll
  for (int i = 0; i < C::LT; ++i) {
    // Tokens past the last repeat it; their columns are not stored.
    const int t = min(t0 + 64 * i + 16 * wave + row, tokens - 1);
    const long r = p.rows_in ? p.rows_in[t] : t;
    xp[i] = static_cast<const char*>(p.x) + (r * p.ldx) * ES + part * 16;
  }
  const int steps = (p.K + C::KE - 1) / C::KE;
  const int tail = p.K % C::KE * ES;  // bytes of the last step, 0: all

  auto issue = [&](int s, int b) __attribute__((always_inline)) {
    unsigned char* base = lds[b] + wave * 1024;
    // Parts past K are zeros in both operands.
    const bool cut = tail != 0 && s == steps - 1 && part * 16 >= tail;
#pragma unroll
    for (int i = 0; i < C::LW; ++i) {
      load_to_lds(MODE == kFfnGate && (i & 1) ? wr1 : wr0, base + i * 4096, cut ? (int)0x80000000 : voff[i], s * 64);
    }
#pragma unroll
    for (int i = 0; i < C::LT; ++i) {
      const char* q = cut ? reinterpret_cast<const char*>(&kZero16) : xp[i];
      __builtin_amdgcn_global_load_lds((glb_ptr)q, (lds_ptr)(base + (C::LW + i) * 4096), 16, 0, 0);
      xp[i] += 64;
    }
  };

  f32x4 acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  issue(0, 0);
  if (steps > 1) issue(1, 1);
  int b = 0;
  const int rd = n * 64 + ((g ^ ((n >> 2) & 3)) << 4);
  for (int s = 0; s < steps; ++s) {
    if (s + 1 < steps)
      stage_wait<C::LW + C::LT>();
    else
      stage_wait<0>();
    if (s + 2 < steps) issue(s + 2, b == 0 ? 2 : b - 1);
    const unsigned char* base = lds[b] + rd;
    u32x4 fw[NI], fx[NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i) fw[i] = *reinterpret_cast<const u32x4*>(base + (wf * NI + i) * 1024);
#pragma unroll
    for (int j = 0; j < NJ; ++j) fx[j] = *reinterpret_cast<const u32x4*>(base + (WF * NI + wt * NJ + j) * 1024);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i][j] = Mma<T>::run(fw[i], fx[j], acc[i][j]);
    b = b == 2 ? 0 : b + 1;
  }

  // Epilogue: 16 features of one token at a time.
  constexpr int GROUPS = MODE == kFfnGate ? NI / 8 : NI / 4;
  float unused;
#pragma unroll
  for (int q = 0; q < GROUPS; ++q) {
    const int f = f0 + (wf * GROUPS + q) * 64 + 16 * g;
    const int left = min(16, p.F - f);
    if (left <= 0) continue;
    float b0[16], b1[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) b0[e] = b1[e] = 0.f;
    if (MODE != kFfnGrad && p.bias[0]) load16(static_cast<const T*>(p.bias[0]) + f, left, b0);
    if (MODE == kFfnGate && p.bias[1]) load16(static_cast<const T*>(p.bias[1]) + f, left, b1);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int t = t0 + (wt * NJ + j) * 16 + n;
      if (t >= tokens) continue;
      float v[16];
      if constexpr (MODE == kFfnGate) {
        float u[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          v[e] = acc[8 * q + (e >> 2)][j][e & 3] + b0[e];
          u[e] = acc[8 * q + 4 + (e >> 2)][j][e & 3] + b1[e];
        }
        const long at = (long)t * p.ldo + f;
        if (p.out[1]) {
          store16(static_cast<T*>(p.out[1]) + at, left, v);
          store16(static_cast<T*>(p.out[2]) + at, left, u);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = activate<false>(p.act, v[e], unused) * u[e];
        store16(static_cast<T*>(p.out[0]) + at, left, v);
      } else if constexpr (MODE == kFfnOut) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[4 * q + (e >> 2)][j][e & 3] + b0[e];
        const long r = p.rows_out ? p.rows_out[t] : t;
        store16(static_cast<T*>(p.out[0]) + r * p.ldo + f, left, v);
      } else {
        float u[16];
        load16(static_cast<const T*>(p.gate) + (long)t * p.F + f, left, v);
        load16(static_cast<const T*>(p.up) + (long)t * p.F + f, left, u);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float dh = acc[4 * q + (e >> 2)][j][e & 3];
          float slope;
          const float act = activate<true>(p.act, v[e], slope);
          v[e] = dh * u[e] * slope;
          u[e] = dh * act;
        }
        T* out = static_cast<T*>(p.out[0]) + (long)t * p.ldo + f;
        store16(out, left, v);
        store16(out + p.F, left, u);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Weights' gradients. LDS holds rows of tokens, features along them: 16-bit
// types read them transposed (ds_read_tr16), float32 element by element. A
// stage is KT tokens of kOuterM features of a and kOuterN of b: 8 + 16 KB.
// 32-byte (float32: 64-byte) slices of 16 features are stored in the order
// slice ^ (row & 7) (float32: ^ (row & 3)), so that the rows of a read pass
// cover the banks once.
// ---------------------------------------------------------------------------
constexpr int KT = F32 ? 16 : 32;

template <int FEATS>
struct OuterSide {
  static constexpr int ROW = FEATS * ES;           // bytes of a token's row
  static constexpr int PARTS = ROW / 16;           // 16-byte parts of it
  static constexpr int ROWS_PER_LOAD = 256 / PARTS;
  static constexpr int LOADS = KT / ROWS_PER_LOAD;
  static __device__ __forceinline__ int swizzle(int row) { return F32 ? (row & 3) << 2 : (row & 7) << 1; }

  const char* base;        // this lane's part of row 0
  const int32_t* rows;
  long ld;                 // bytes
  bool in;                 // its features exist
  int r0;                  // its row of a load

  __device__ __forceinline__ void init(const void* p, const int32_t* map, long ld_elems, int f0, int count, int tid) {
    r0 = tid / PARTS;
    // ROWS_PER_LOAD is a multiple of the swizzle's period or the row's low
    // bits are those of r0 in every load.
    const int part = (tid % PARTS) ^ swizzle(r0);
    const int f = f0 + part * kVec<T>;
    in = f < count;
    base = static_cast<const char*>(p) + (in ? (long)f * ES : 0);
    rows = map;
    ld = ld_elems * ES;
  }
  __device__ __forceinline__ void issue(int t0, int t1, unsigned char* dst, int wave) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int t = t0 + i * ROWS_PER_LOAD + r0;
      const bool ok = in && t < t1;
      const long r = ok ? (rows ? rows[t] : t) : 0;
      const char* q = ok ? base + r * ld : reinterpret_cast<const char*>(&kZero16);
      __builtin_amdgcn_global_load_lds((glb_ptr)q, (lds_ptr)(dst + i * 4096 + wave * 1024), 16, 0, 0);
    }
  }
  // Subtile `sub` (16 features) as a matrix-core operand. 16-bit: tokens 4 g +
  // .., 16 + 4 g + .. in the lane's eight slots; float32: step e (of four)
  // holds token 4 e + g.
  static __device__ __forceinline__ u32x4 frag(const unsigned char* tile, int sub, int g, int n) {
    if constexpr (F32) {
      u32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * e + g;
        v[e] = *reinterpret_cast<const unsigned*>(tile + r * ROW + (((sub << 2) ^ swizzle(r)) << 4) + 4 * n);
      }
      return v;
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
      const int r = 4 * g + (n >> 2), at = (((sub << 1) ^ swizzle(r)) << 4) + 8 * (n & 3);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(tile + r * ROW + at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(tile + (r + 16) * ROW + at));
      const u32x2 a = __builtin_bit_cast(u32x2, lo), c = __builtin_bit_cast(u32x2, hi);
      return u32x4{a[0], a[1], c[0], c[1]};
    }
  }
};

__global__ __launch_bounds__(256, 2) void ffn_outer(FfnOuters ps) {
  typedef OuterSide<kOuterM> SideA;
  typedef OuterSide<kOuterN> SideB;
  constexpr int NI = 4, NJ = 8, A_BYTES = KT * SideA::ROW, STAGE = A_BYTES + KT * SideB::ROW;
  constexpr int LOADS = SideA::LOADS + SideB::LOADS;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[3][STAGE];
  const int k = (int)blockIdx.x >= ps.first[0];
  const FfnOuter& p = ps.p[k];
  const int splits = ps.splits[k];
  const int nm = (p.M + kOuterM - 1) / kOuterM, nn = (p.N + kOuterN - 1) / kOuterN;
  int at = (int)blockIdx.x - (k ? ps.first[0] : 0);
  // Consecutive workgroups of an XCD take the tiles of one run of tokens.
  const int total = nm * nn * splits, per = (total + 7) >> 3;
  const int i8 = at >> 3;
  at = (at & 7) * per + i8;
  if (i8 >= per || at >= total) return;
  const int split = at / (nm * nn), tile = at - split * nm * nn;
  const int m0 = tile % nm * kOuterM, n0 = tile / nm * kOuterN;
  const int tokens = ps.count ? *ps.count : ps.tokens;
  const int run = ((tokens + splits - 1) / splits + KT - 1) / KT * KT;
  const long ta = min((long)split * run, (long)tokens), tb = min(ta + run, (long)tokens);
  const int t0 = (int)ta, t1 = (int)tb;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1, g = lane >> 4, n = lane & 15;
  SideA a;
  SideB bb;
  a.init(p.a, p.rows_a, p.lda, m0, p.M, tid);
  bb.init(p.b, p.rows_b, p.ldb, n0, p.N, tid);
  auto issue = [&](int s, int buf) __attribute__((always_inline)) {
    a.issue(t0 + s * KT, t1, lds[buf], wave);
    bb.issue(t0 + s * KT, t1, lds[buf] + A_BYTES, wave);
  };
  // The bias' gradient: the columns of b against a row of ones, in the first
  // waves of the first tile of m.
  const bool sums = p.bias && m0 == 0 && wm == 0;
  const unsigned one = F32 ? 0x3f800000u : (__is_same(T, bf16) ? 0x3f803f80u : 0x3c003c00u);
  const u32x4 ones = {one, one, one, one};
  f32x4 acc[NI][NJ], sum[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NI; ++i) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int steps = (t1 - t0 + KT - 1) / KT;
  if (steps > 0) issue(0, 0);
  if (steps > 1) issue(1, 1);
  int b = 0;
  for (int s = 0; s < steps; ++s) {
    if (s + 1 < steps)
      stage_wait<LOADS>();
    else
      stage_wait<0>();
    if (s + 2 < steps) issue(s + 2, b == 0 ? 2 : b - 1);
    u32x4 fa[NI], fb[NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i) fa[i] = SideA::frag(lds[b], wm * NI + i, g, n);
#pragma unroll
    for (int j = 0; j < NJ; ++j) fb[j] = SideB::frag(lds[b] + A_BYTES, wn * NJ + j, g, n);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i][j] = Mma<T>::run(fa[i], fb[j], acc[i][j]);
    if (sums) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) sum[j] = Mma<T>::run(ones, fb[j], sum[j]);
    }
    b = b == 2 ? 0 : b + 1;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int nr = n0 + (wn * NJ + j) * 16 + n;
    if (nr >= p.N) continue;
    float* out = p.part + ((long)split * p.N + nr) * p.M;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int m = m0 + (wm * NI + i) * 16 + 4 * g;
      if (m < p.M) *reinterpret_cast<f32x4*>(out + m) = acc[i][j];
    }
    if (sums && g == 0) p.bias[(long)split * p.N + nr] = sum[j][0];
  }
}

template <int MODE, int WF, int WT, int NI, int NJ>
void launch(const FfnProduct& p, hipStream_t st) {
  typedef Product<MODE, WF, WT, NI, NJ> C;
  const long tiles = (long)((p.F + C::FEATURES - 1) / C::FEATURES) * ((p.tokens + C::BT - 1) / C::BT);
  ffn_product<MODE, WF, WT, NI, NJ><<<(unsigned)((tiles + 7) / 8 * 8), 256, 0, st>>>(p);
}

}  // namespace

#define FST_CAT2(a, b) a##b
#define FST_CAT(a, b) FST_CAT2(a, b)

int FST_CAT(ffn_product_, FST_NAME)(int mode, const FfnProduct& p, hipStream_t st) {
  if (mode == kFfnGate)
    launch<kFfnGate, 2, 2, 8, 4>(p, st);
  else if (mode == kFfnOut)
    launch<kFfnOut, 2, 2, 4, 8>(p, st);
  else
    launch<kFfnGrad, 2, 2, 4, 8>(p, st);
  return hipGetLastError() == hipSuccess ? FST_OK : FST_ELAUNCH;
}

int FST_CAT(ffn_outer_, FST_NAME)(FfnOuters& ps, hipStream_t st) {
  int grid = 0;
  for (int k = 0; k < 2; ++k) {
    const FfnOuter& p = ps.p[k];
    const int tiles = ps.splits[k] * ((p.M + kOuterM - 1) / kOuterM) * ((p.N + kOuterN - 1) / kOuterN);
    grid += (tiles + 7) / 8 * 8;
    ps.first[k] = grid;
  }
  if (grid == 0) return FST_OK;
  ffn_outer<<<grid, 256, 0, st>>>(ps);
  return hipGetLastError() == hipSuccess ? FST_OK : FST_ELAUNCH;
}

}  // namespace fst
