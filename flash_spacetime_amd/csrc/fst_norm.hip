// Layer norm of token rows, forward and backward.
//
//   s = x + r rounded to the rows' type (s = x without a residual),
//   y = (s - m) rstd w + b,  m = mean(s),  rstd = 1 / sqrt(mean((s - m)^2) + eps),
//   g = dy w,  xhat = (s - m) rstd,
//   dx = rstd (g - mean(g) - xhat mean(g xhat)) + ds,  dw = sum dy xhat,  db = sum dy.
//
// A row is held in registers by a group of LPR lanes, so memory is read once
// and written once; the bound is HBM bandwidth (256 x 768 padded rows of 384 bf16 with a
// residual, half of them tokens: forward 78 us, 5.9 TB/s of what it has to move, backward
// 105, 3.7; 60001 rows of 512 f32 40 and 64 us, 6.2 and 5.8 TB/s, some of it from the
// last level cache) or, in calls of few rows, the launch. Statistics, sums and
// gradients are float32; each output is rounded once.
#include "fst_block.h"

namespace fst {

namespace {

constexpr int kNormMax = 16384;  // features of a row

struct NormArgs {
  const void *x, *r, *w, *b;  // r, w, b may be null
  const int32_t* lens;        // padded batches: valid rows of each event; or null
  void *y, *s;                // s: where r is given
  float2* stats;              // (mean, rstd) per row, or null
  long rows;
  long ldx, ldr;
  int L, n;
  float eps;
};

struct NormGradArgs {
  const void *s, *dy, *ds, *w;  // ds, w may be null
  const int32_t* lens;
  const float2* stats;
  void* dx;
  float* part;  // [blocks][2][n] partial dw, db; or null
  long rows;
  long lds_, lddy, ldds;
  int L, n;
};

// Sum over the LPR lanes of a row's group (16, 32, 64 lanes of a wave, or a
// whole workgroup of LPR / 64 waves through LDS); every lane gets it. The
// order of the additions is fixed.
__device__ __forceinline__ float row16_sum(float x) {
#define FST_ROR(x, n) __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + n, 0xf, 0xf, false))
  x += FST_ROR(x, 8);
  x += FST_ROR(x, 4);
  x += FST_ROR(x, 2);
  x += FST_ROR(x, 1);
#undef FST_ROR
  return x;
}

template <int LPR>
__device__ __forceinline__ float group_sum(float x, float* red) {
  x = row16_sum(x);
  if constexpr (LPR >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if constexpr (LPR >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    __syncthreads();  // the sums before are read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int i = 1; i < W; ++i) x += red[i];
  }
  return x;
}

// Lane l's pieces of a row: elements (l + LPR i) V .. + V - 1, i < NC, zeros past
// its end. EDGE: the row's length is no whole number of pieces or rows start
// off 16 bytes; pieces are then read at element alignment, the one that the row
// ends in as the row's last V elements. Those are moved to their places, and what is
// past the end cleared, when the piece is used: a load under a lane's own condition
// would have to land before the next is issued (16 x 500 rows of 1367 f16, backward
// 22.9 us so, 20.0 as it is).
template <typename T, int LPR, int NC, bool EDGE>
struct Pieces {
  static constexpr int V = kVec<T>, E = NC * V;
  static constexpr bool SHORT = EDGE && NC == 1 && LPR == 16;  // rows may have fewer than V elements
  typename Piece<T>::V p[NC];

  static __device__ __forceinline__ int at(int l, int i) { return (l + LPR * i) * V; }
  __device__ __forceinline__ void load(const T* row, int l, int n) {
    if (SHORT && n < V) {
#pragma unroll
      for (int j = 0; j < V; ++j) p[0][j] = l == 0 && j < n ? row[j] : (T)0.f;
      return;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = at(l, i);
      if constexpr (EDGE) {
        p[i] = *reinterpret_cast<const typename Piece<T>::VU*>(row + min(c, n - V));
      } else if (c < n) {
        p[i] = *reinterpret_cast<const typename Piece<T>::V*>(row + c);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) p[i][j] = (T)0.f;
      }
    }
  }
  __device__ __forceinline__ void get(float* v, int l, int n) const {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      typename Piece<T>::V q = p[i];
      if (EDGE && at(LPR, i) > n && !(SHORT && n < V)) {
        const int c = at(l, i);
        const unsigned __int128 x = __builtin_bit_cast(unsigned __int128, q);
        const int past = (V - n % V) % V;  // elements of the last piece past the row's end
        q = __builtin_bit_cast(typename Piece<T>::V, c >= n ? 0 : c + V > n ? x >> (8 * (int)sizeof(T) * past) : x);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = (float)q[j];
    }
  }
  static __device__ __forceinline__ void store(T* row, int l, int n, const float* v) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = at(l, i);
      const typename Piece<T>::V q = pack_piece<T>(v + i * V);
      if (EDGE ? c + V <= n : c < n) {
        if constexpr (EDGE)
          *reinterpret_cast<typename Piece<T>::VU*>(row + c) = q;
        else
          *reinterpret_cast<typename Piece<T>::V*>(row + c) = q;
      } else if (EDGE && c < n) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < n % V) row[c + j] = q[j];
      }
    }
  }
};

// Parameters may be float32 or of the rows' type; null stands for `fill`.
// Elements past the row's end are 0. Whole pieces come in 16-byte loads (by
// elements, a workgroup's first microseconds were these loads: one event of 187
// rows of 384 took 8.0 us).
template <typename T>
__device__ __forceinline__ void load_param(const void* p, bool f32, int c, int n, float fill, float* v) {
  constexpr int V = kVec<T>;
  typedef f32x4 f32x4u __attribute__((aligned(4)));
  if (!p || c + V > n) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      v[i] = c + i >= n ? 0.f : !p ? fill : f32 ? static_cast<const float*>(p)[c + i] : (float)static_cast<const T*>(p)[c + i];
  } else if (f32) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const f32x4 q = *reinterpret_cast<const f32x4u*>(static_cast<const float*>(p) + c + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i + j] = q[j];
    }
  } else {
    const typename Piece<T>::V q = *reinterpret_cast<const typename Piece<T>::VU*>(static_cast<const T*>(p) + c);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)q[i];
  }
}

__device__ __forceinline__ bool row_valid(const int32_t* lens, long row, int L) {
  if (!lens) return true;
  const unsigned b = (unsigned)row / (unsigned)L;  // rows < 2^31
  return (int)((unsigned)row - b * (unsigned)L) < event_len(lens, (int)b, L);
}

// Both kernels walk the rows a group at a time, with the next row's pieces in
// flight while a row is worked on, and the length that says whether the row after
// it is a token before those.
template <typename T, int LPR, int NC, bool EDGE>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void norm_fwd(NormArgs a, int w_f32) {
  typedef Pieces<T, LPR, NC, EDGE> P;
  constexpr int V = P::V, E = P::E, NT = LPR > 256 ? LPR : 256, G = NT / LPR;
  __shared__ float red[LPR > 64 ? LPR / 64 : 1];
  const int l = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int n = a.n;
  const float inv_n = 1.f / (float)n;
  const long step = (long)gridDim.x * G;
  long row = (long)blockIdx.x * G + grp;
  auto is_token = [&](long r) { return r < a.rows && row_valid(a.lens, r, a.L); };
  P x0, x1, r0, r1;
  auto fetch = [&](long r, P& x, P& q) {
    x.load(static_cast<const T*>(a.x) + r * a.ldx, l, n);
    if (a.r) q.load(static_cast<const T*>(a.r) + r * a.ldr, l, n);
  };
  bool now = is_token(row), next = is_token(row + step);
  if (now) fetch(row, x0, r0);
  float w[E], b[E];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    load_param<T>(a.w, w_f32, P::at(l, i), n, 1.f, w + i * V);
    load_param<T>(a.b, w_f32, P::at(l, i), n, 0.f, b + i * V);
  }
  for (; row < a.rows; row += step) {
    const bool later = is_token(row + 2 * step);
    if (next) fetch(row + step, x1, r1);
    T* y = static_cast<T*>(a.y) + row * n;
    T* so = static_cast<T*>(a.s) + row * n;
    float v[E];
    float2 st = make_float2(0.f, 0.f);
    if (now) {
      x0.get(v, l, n);
      if (a.r) {
        float q[E];
        r0.get(q, l, n);
        // The norm is of the sum as it is returned, so that the backward, which
        // has only that, differentiates the same function.
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = (float)(T)(v[i] + q[i]);
        P::store(so, l, n, v);
      }
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) sum += v[i];
      const float m = group_sum<LPR>(sum, red) * inv_n;
      // Second pass in registers: the deviations' own mean corrects m's rounding
      // (rows whose mean is large beside their spread), their squares give the
      // variance.
      float d1 = 0.f, d2 = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float d = P::at(l, i / V) + i % V < n ? v[i] - m : 0.f;
        v[i] = d;
        d1 += d;
        d2 = fmaf(d, d, d2);
      }
      d1 = group_sum<LPR>(d1, red) * inv_n;
      d2 = group_sum<LPR>(d2, red) * inv_n;
      const float rstd = 1.f / sqrtf(fmaxf(fmaf(-d1, d1, d2), 0.f) + a.eps);
      st = make_float2(m + d1, rstd);
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = fmaf((v[i] - d1) * rstd, w[i], b[i]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = 0.f;
      if (a.r) P::store(so, l, n, v);
    }
    P::store(y, l, n, v);
    if (a.stats && l == 0) a.stats[row] = st;
    x0 = x1;
    r0 = r1;
    now = next;
    next = later;
  }
}

template <typename T, int LPR, int NC, bool EDGE>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void norm_bwd(NormGradArgs a, int w_f32) {
  typedef Pieces<T, LPR, NC, EDGE> P;
  constexpr int V = P::V, E = P::E, NT = LPR > 256 ? LPR : 256, G = NT / LPR;
  __shared__ float red[LPR > 64 ? LPR / 64 : 1];
  // Partial sums of the workgroup's row groups (G > 1): [G][E][LPR].
  __shared__ float acc[G > 1 ? NT * E : 1];
  const int l = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int n = a.n;
  const float inv_n = 1.f / (float)n;
  const long step = (long)gridDim.x * G;
  long row = (long)blockIdx.x * G + grp;
  auto is_token = [&](long r) { return r < a.rows && row_valid(a.lens, r, a.L); };
  struct Row {
    P s, dy, ds;
    float2 st;
  } r0, r1;
  auto fetch = [&](long r, Row& q) {
    q.st = a.stats[r];
    q.s.load(static_cast<const T*>(a.s) + r * a.lds_, l, n);
    q.dy.load(static_cast<const T*>(a.dy) + r * a.lddy, l, n);
    if (a.ds) q.ds.load(static_cast<const T*>(a.ds) + r * a.ldds, l, n);
  };
  bool now = is_token(row), next = is_token(row + step);
  if (now) fetch(row, r0);
  float w[E], dw[E], db[E];
#pragma unroll
  for (int i = 0; i < NC; ++i) load_param<T>(a.w, w_f32, P::at(l, i), n, 1.f, w + i * V);
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = db[i] = 0.f;
  for (; row < a.rows; row += step) {
    const bool later = is_token(row + 2 * step);
    if (next) fetch(row + step, r1);
    float g[E];
    if (now) {
      float v[E];
      r0.s.get(v, l, n);
      r0.dy.get(g, l, n);
      const float2 st = r0.st;
      float c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        v[i] = (v[i] - st.x) * st.y;  // xhat; past the row's end its dy is 0
        dw[i] = fmaf(g[i], v[i], dw[i]);
        db[i] += g[i];
        g[i] *= w[i];
        c1 += g[i];
        c2 = fmaf(g[i], v[i], c2);
      }
      if (a.dx) {
        c1 = group_sum<LPR>(c1, red) * inv_n;
        c2 = group_sum<LPR>(c2, red) * inv_n;
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] = st.y * (g[i] - c1 - v[i] * c2);
        if (a.ds) {
          r0.ds.get(v, l, n);
#pragma unroll
          for (int i = 0; i < E; ++i) g[i] += v[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = 0.f;
    }
    if (a.dx) P::store(static_cast<T*>(a.dx) + row * n, l, n, g);
    r0 = r1;
    now = next;
    next = later;
  }
  if (!a.part) return;
  float* out = a.part + (long)blockIdx.x * 2 * n;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float* v = k ? db : dw;
    if constexpr (G > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < E; ++i) acc[(grp * E + i) * LPR + l] = v[i];
      __syncthreads();
      // Element i of lane l, summed over the groups in order.
      for (int t = threadIdx.x; t < E * LPR; t += NT) {
        const int i = t / LPR, ll = t % LPR, c = (ll + LPR * (i / V)) * V + i % V;
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < G; ++q) sum += acc[(q * E + i) * LPR + ll];
        if (c < n) out[k * n + c] = sum;
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = (l + LPR * (i / V)) * V + i % V;
        if (c < n) out[k * n + c] = v[i];
      }
    }
  }
}

// dw | db = the column sums of part [blocks][2 n], in a fixed order: 32 columns a
// workgroup, 32 threads a column, eight loads of each in flight.
template <typename T>
__global__ __launch_bounds__(1024) void norm_grad_sum(const float* part, int blocks, int n, void* dw, void* db,
                                                      int w_f32) {
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c;
  float sum = 0.f;
  if (col < 2 * n) {
    const float* in = part + col;
    int i = k;
    for (; i + 224 < blocks; i += 256) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = in[(long)(i + 32 * j) * 2 * n];
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[j];
    }
    for (; i < blocks; i += 32) sum += in[(long)i * 2 * n];
  }
  red[k][c] = sum;
  __syncthreads();
  if (k == 0 && col < 2 * n) {
#pragma unroll
    for (int i = 1; i < 32; ++i) sum += red[i][c];
    void* out = col < n ? dw : db;
    const int at = col < n ? col : col - n;
    if (out) {
      if (w_f32)
        static_cast<float*>(out)[at] = sum;
      else
        static_cast<T*>(out)[at] = (T)sum;
    }
  }
}

// The lanes a row takes: the fewest whose share is at most three 16-byte
// pieces a lane (four in float32: half as many elements), of which the backward
// holds s, dy, w, dw, db and the next row's three without spilling (but for
// float32 rows of more than 8192). Fewer lanes leave fewer idle: 256 x 768 rows
// of 384 bf16, padded, by 16 / 32 / 64 lanes: forward 96 / 99 / 106 us, backward
// 97 / 123 / 182.
struct NormPlan {
  int lpr, nc;
  bool edge;
};

template <typename T>
constexpr int kMostPieces = sizeof(T) == 4 ? 4 : 3;

// Whether plan_norm gives some row L lanes of C pieces.
template <typename T>
constexpr bool planned(int L, int C) {
  const int fewer = L == 16 ? 0 : L == 32 ? 16 : L == 64 ? 32 : L == 256 ? 64 : 256;
  return C <= kMostPieces<T> && L * C > kMostPieces<T> * fewer && L * (C - 1) * kVec<T> < kNormMax;
}

bool plan_norm(int dtype, int n, NormPlan& p) {
  const int v = 16 / (int)elem_size(dtype), most = dtype == FST_F32 ? kMostPieces<float> : kMostPieces<bf16>;
  if (n > kNormMax) return false;
  const int pieces = (n + v - 1) / v;
  for (int lpr : {16, 32, 64, 256, 1024}) {
    if (pieces <= most * lpr) {
      p.lpr = lpr;
      p.nc = (pieces + lpr - 1) / lpr;
      return true;
    }
  }
  return false;
}

// Most workgroups. The forward's are those that its registers let run at once:
// each loads the parameters and then has a row ahead in flight, which is lost on those
// that would start after others (8000 rows of 1367 f16 3 / 4 / 8 a CU 15.2 / 18.0 / 21.1
// us; 4000 of 16384 bf16 2 / 8 a CU 54 / 72). The backward's each write one partial of
// dw and db; two a CU keep enough rows in flight (768 or 1024 are slower by what
// the partials cost).
constexpr int kNormBlocks = 512;

int norm_forward_blocks(const NormPlan& p, int dtype) {
  if (p.lpr == 1024) return 512;
  const int registers = 22 + p.nc * (dtype == FST_F32 ? 30 : 44);  // of a lane: 54 .. 154
  return 256 * (512 / registers);
}

int norm_rows_per_block(const NormPlan& p) { return p.lpr > 256 ? 1 : 256 / p.lpr; }

int norm_blocks(const NormPlan& p, long rows, int most) {
  const long need = (rows + norm_rows_per_block(p) - 1) / norm_rows_per_block(p);
  return (int)(need < most ? need : most);
}

bool aligned16(const void* p, long ld, size_t es) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * es % 16 == 0; }

template <typename T>
void launch_fwd(const NormPlan& p, const NormArgs& a, int blocks, int w_f32, hipStream_t st) {
  const int threads = p.lpr > 256 ? p.lpr : 256;
#define FST_CASE(L, C)                                                                   \
  if constexpr (planned<T>(L, C)) {                                                      \
    if (p.lpr == L && p.nc == C) {                                                        \
      if (p.edge)                                                                        \
        norm_fwd<T, L, C, true><<<blocks, threads, 0, st>>>(a, w_f32);                   \
      else                                                                               \
        norm_fwd<T, L, C, false><<<blocks, threads, 0, st>>>(a, w_f32);                  \
    }                                                                                    \
  }
#define FST_CASES(L) FST_CASE(L, 1) FST_CASE(L, 2) FST_CASE(L, 3) FST_CASE(L, 4)
  FST_CASES(16)
  FST_CASES(32)
  FST_CASES(64)
  FST_CASES(256)
  FST_CASES(1024)
#undef FST_CASES
#undef FST_CASE
}

template <typename T>
void launch_bwd(const NormPlan& p, const NormGradArgs& a, int blocks, int w_f32, hipStream_t st) {
  const int threads = p.lpr > 256 ? p.lpr : 256;
#define FST_CASE(L, C)                                                                   \
  if constexpr (planned<T>(L, C)) {                                                      \
    if (p.lpr == L && p.nc == C) {                                                        \
      if (p.edge)                                                                        \
        norm_bwd<T, L, C, true><<<blocks, threads, 0, st>>>(a, w_f32);                   \
      else                                                                               \
        norm_bwd<T, L, C, false><<<blocks, threads, 0, st>>>(a, w_f32);                  \
    }                                                                                    \
  }
#define FST_CASES(L) FST_CASE(L, 1) FST_CASE(L, 2) FST_CASE(L, 3) FST_CASE(L, 4)
  FST_CASES(16)
  FST_CASES(32)
  FST_CASES(64)
  FST_CASES(256)
  FST_CASES(1024)
#undef FST_CASES
#undef FST_CASE
}

int check_norm(int dtype, int param_dtype, int B, int L, int N, NormPlan& p) {
  if (dtype != FST_BF16 && dtype != FST_F32 && dtype != FST_F16)
    return fail(FST_EINVAL, "dtype must be FST_BF16, FST_F16 or FST_F32, got %d", dtype);
  if (param_dtype != dtype && param_dtype != FST_F32)
    return fail(FST_EINVAL, "param_dtype must be dtype or FST_F32, got %d", param_dtype);
  if (B < 0 || L < 0) return fail(FST_EINVAL, "negative size (B=%d, L=%d)", B, L);
  if (N < 1) return fail(FST_EINVAL, "need at least one feature, got N=%d", N);
  if ((long)B * L > 0x7fffffffL) return fail(FST_EUNSUPPORTED, "more than 2^31 - 1 rows");
  if (!plan_norm(dtype, N, p))
    return fail(FST_EUNSUPPORTED, "rows of N=%d features: at most %d", N, kNormMax);
  return FST_OK;
}

}  // namespace

}  // namespace fst

using namespace fst;

extern "C" {

int fst_layer_norm_forward(int dtype, int param_dtype, int B, int L, int N, const void* x, int64_t x_stride,
                           const void* residual, int64_t residual_stride, const void* weight, const void* bias,
                           const int32_t* seqlens, float eps, void* y, void* sum, float* stats, void* stream) {
  clear_error();
  NormPlan p;
  const int rc = check_norm(dtype, param_dtype, B, L, N, p);
  if (rc != FST_OK) return rc;
  const long rows = (long)B * L;
  if (rows == 0) return FST_OK;
  if (!x || !y || (residual && !sum)) return fail(FST_EINVAL, "null tensor pointer");
  if (x_stride < N || (residual && residual_stride < N)) return fail(FST_EINVAL, "row stride below N=%d", N);
  if (!(eps >= 0.f)) return fail(FST_EINVAL, "eps must not be negative");
  const size_t es = elem_size(dtype);
  NormArgs a{x, residual, weight, bias, seqlens, y, sum, reinterpret_cast<float2*>(stats),
             rows, (long)x_stride, (long)residual_stride, L, N, eps};
  p.edge = !aligned16(x, x_stride, es) || !aligned16(y, N, es) ||
           (residual && (!aligned16(residual, residual_stride, es) || !aligned16(sum, N, es)));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int w_f32 = param_dtype == FST_F32, blocks = norm_blocks(p, rows, norm_forward_blocks(p, dtype));
  if (dtype == FST_BF16)
    launch_fwd<bf16>(p, a, blocks, w_f32, st);
  else if (dtype == FST_F16)
    launch_fwd<f16>(p, a, blocks, w_f32, st);
  else
    launch_fwd<float>(p, a, blocks, w_f32, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(FST_ELAUNCH, "layer norm launch failed (%s)", hipGetErrorString(e));
  return FST_OK;
}

size_t fst_layer_norm_backward_workspace_bytes(int dtype, int B, int L, int N) {
  NormPlan p;
  if (check_norm(dtype, dtype, B, L, N, p) != FST_OK) return 0;
  return align256((size_t)norm_blocks(p, (long)B * L, kNormBlocks) * 2 * N * sizeof(float));
}

int fst_layer_norm_backward(int dtype, int param_dtype, int B, int L, int N, const void* s, int64_t s_stride,
                            const void* weight, const int32_t* seqlens, const float* stats, const void* dy,
                            int64_t dy_stride, const void* dsum, int64_t dsum_stride, void* dx, void* dweight,
                            void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  NormPlan p;
  const int rc = check_norm(dtype, param_dtype, B, L, N, p);
  if (rc != FST_OK) return rc;
  const long rows = (long)B * L;
  const bool sums = dweight || dbias;
  if (!dx && !sums) return FST_OK;
  if (rows > 0) {
    if (!s || !dy || !stats) return fail(FST_EINVAL, "null tensor pointer");
    if (s_stride < N || dy_stride < N || (dsum && dsum_stride < N)) return fail(FST_EINVAL, "row stride below N=%d", N);
  }
  const int blocks = norm_blocks(p, rows, kNormBlocks);
  const size_t need = align256((size_t)blocks * 2 * N * sizeof(float));
  if (sums && need > 0 && (!workspace || workspace_bytes < need))
    return fail(FST_EWORKSPACE, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, need);
  const size_t es = elem_size(dtype);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int w_f32 = param_dtype == FST_F32;
  float* part = sums ? static_cast<float*>(workspace) : nullptr;
  if (rows > 0) {
    NormGradArgs a{s, dy, dsum, weight, seqlens, reinterpret_cast<const float2*>(stats), dx, part,
                   rows, (long)s_stride, (long)dy_stride, (long)dsum_stride, L, N};
    p.edge = N * es % 16 != 0 || !aligned16(s, s_stride, es) || !aligned16(dy, dy_stride, es) ||
             (dx && !aligned16(dx, N, es)) || (dsum && !aligned16(dsum, dsum_stride, es));
    if (dtype == FST_BF16)
      launch_bwd<bf16>(p, a, blocks, w_f32, st);
    else if (dtype == FST_F16)
      launch_bwd<f16>(p, a, blocks, w_f32, st);
    else
      launch_bwd<float>(p, a, blocks, w_f32, st);
  }
  if (sums) {
    const int grid = (2 * N + 31) / 32;
    if (dtype == FST_BF16)
      norm_grad_sum<bf16><<<grid, 1024, 0, st>>>(part, blocks, N, dweight, dbias, w_f32);
    else if (dtype == FST_F16)
      norm_grad_sum<f16><<<grid, 1024, 0, st>>>(part, blocks, N, dweight, dbias, w_f32);
    else
      norm_grad_sum<float><<<grid, 1024, 0, st>>>(part, blocks, N, dweight, dbias, w_f32);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(FST_ELAUNCH, "layer norm backward launch failed (%s)", hipGetErrorString(e));
  return FST_OK;
}

}  // extern "C"
