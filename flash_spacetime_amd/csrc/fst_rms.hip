// Root-mean-square norm of token rows, forward and backward, and with an output in
// 8 bits.
//
//   s = x + r rounded to the rows' type (s = x without a residual),
//   rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w,
//   g = dy w,  xhat = s rstd,  dx = rstd (g - xhat mean(g xhat)) + ds,  dw = sum dy xhat;
//   8 bits: scale = max |y| / 448 of the row, q = y / scale rounded to e4m3.
//
// A row is held in registers by a group of lanes (fst_rows.h), so memory is read
// once and written once and the bound is HBM bandwidth, or the launch in calls of
// few rows (256 x 768 padded rows of 384 bf16 with a residual, half of them tokens:
// forward 79 us, 5.8 TB/s of what it has to move, backward 94, 4.1; 65536 rows of 1024
// f16 with a residual to 8 bits 86 us, 5.5). Statistics, sums and scales are float32;
// each output is rounded once.
#include "fst_rows.h"

namespace fst {

namespace {

struct RmsArgs {
  const void *x, *r, *w;  // r, w may be null
  const int32_t* lens;    // padded batches: valid rows of each event; or null
  void *y, *s;            // y: rows of T, or of bytes (8 bits); s: where r is given
  float* aside;           // rstd per row, or null; 8 bits: the rows' scales
  long rows;
  long ldx, ldr;
  int L, n;
  float eps;
};

struct RmsGradArgs {
  const void *s, *dy, *ds, *w;  // ds, w may be null
  const int32_t* lens;
  const float* rstd;
  void* dx;
  float* part;  // [blocks][n] partial dw; or null
  long rows;
  long lds_, lddy, ldds;
  int L, n;
};

// The largest e4m3 value, and the least scale: its reciprocal is finite, and a row of
// zeros has one.
constexpr float kTop8 = 448.f, kLeastScale = 0x1p-126f;

// Bytes of a row from its values over `scale`, piece by piece; inv: the rounded reciprocal
// of scale, or both 0 (rows of zeros, and what is finite beside an infinite value). The
// product with inv alone is a unit or two off, and values next to a border between two
// bytes fell to its other side; the remainder v - q scale is exact in a multiply-add,
// and q corrected by it is the quotient rounded to float32 (Markstein, IBM J. Res. Dev. 34,
// 1990). The row's largest value comes out as 448 (1 + 2^-23) at most, which rounds to
// 448; NaN stays NaN.
template <typename P, bool EDGE>
__device__ __forceinline__ void store8(unsigned char* row, int l, int n, const float* v, float scale, float inv) {
  const auto over = [&](float x) {
    const float q = x * inv;
    return fmaf(fmaf(-q, scale, x), inv, q);
  };
  constexpr int V = P::V;
  typedef unsigned char Bytes __attribute__((ext_vector_type(V)));
  typedef Bytes BytesU __attribute__((aligned(1)));
#pragma unroll
  for (int i = 0; i < P::E / V; ++i) {
    const int c = P::at(l, i);
    unsigned word[V / 4];
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float* q = v + i * V + j;
      int o = __builtin_amdgcn_cvt_pk_fp8_f32(over(q[0]), over(q[1]), 0, false);
      o = __builtin_amdgcn_cvt_pk_fp8_f32(over(q[2]), over(q[3]), o, true);
      word[j / 4] = (unsigned)o;
    }
    const Bytes o = __builtin_bit_cast(Bytes, word);
    if (EDGE ? c + V <= n : c < n) {
      if constexpr (EDGE)
        *reinterpret_cast<BytesU*>(row + c) = o;
      else
        *reinterpret_cast<Bytes*>(row + c) = o;
    } else if (EDGE && c < n) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n % V) row[c + j] = o[j];
    }
  }
}

// Both kernels walk the rows a group at a time, and ask for the length that says
// whether the next row is a token before they need it. The forward also has the next
// row's pieces in flight while a row is worked on; the backward holds so much of a row
// that a third wave on a SIMD is worth more (256 x 768 padded rows of 384 bf16 with a
// residual: two rows in flight and two waves 106 us, one and three 93).
template <typename T, int LPR, int NC, bool EDGE, bool Q8>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void rms_fwd(RmsArgs a, int w_f32) {
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
  float w[E];
#pragma unroll
  for (int i = 0; i < NC; ++i) load_param<T>(a.w, w_f32, P::at(l, i), n, 1.f, w + i * V);
  for (; row < a.rows; row += step) {
    const bool later = is_token(row + 2 * step);
    if (next) fetch(row + step, x1, r1);
    float v[E], aside = 0.f, scale = 0.f, inv = 0.f;
    if (now) {
      x0.get(v, l, n);
      if (a.r) {
        float q[E];
        r0.get(q, l, n);
        // The norm is of the sum as it is returned, so that the backward, which
        // has only that, differentiates the same function.
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = (float)(T)(v[i] + q[i]);
        P::store(static_cast<T*>(a.s) + row * n, l, n, v);
      }
      float sum = 0.f;  // elements past the row's end are 0
#pragma unroll
      for (int i = 0; i < E; ++i) sum = fmaf(v[i], v[i], sum);
      const float rstd = 1.f / sqrtf(fmaf(group_sum<LPR>(sum, red), inv_n, a.eps));
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = v[i] * rstd * w[i];
      aside = rstd;
      if constexpr (Q8) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) top = fmaxf(top, fabsf(v[i]));
        aside = fmaxf(group_max<LPR>(top, red) / kTop8, kLeastScale);
        if (aside < __builtin_inff()) scale = aside, inv = 1.f / aside;
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = 0.f;
      if (a.r) P::store(static_cast<T*>(a.s) + row * n, l, n, v);
    }
    if constexpr (Q8)
      store8<P, EDGE>(static_cast<unsigned char*>(a.y) + row * n, l, n, v, scale, inv);
    else
      P::store(static_cast<T*>(a.y) + row * n, l, n, v);
    if (a.aside && l == 0) a.aside[row] = aside;
    x0 = x1;
    r0 = r1;
    now = next;
    next = later;
  }
}

template <typename T, int LPR, int NC, bool EDGE>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256, LPR > 256 ? 1 : 3) void rms_bwd(RmsGradArgs a, int w_f32) {
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
  bool now = is_token(row);
  float w[E], dw[E];
#pragma unroll
  for (int i = 0; i < NC; ++i) load_param<T>(a.w, w_f32, P::at(l, i), n, 1.f, w + i * V);
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = 0.f;
  for (; row < a.rows; row += step) {
    const bool next = is_token(row + step);
    float g[E];
    if (now) {
      P s, dy, ds;
      const float rstd = a.rstd[row];
      s.load(static_cast<const T*>(a.s) + row * a.lds_, l, n);
      dy.load(static_cast<const T*>(a.dy) + row * a.lddy, l, n);
      if (a.ds) ds.load(static_cast<const T*>(a.ds) + row * a.ldds, l, n);
      float v[E];
      s.get(v, l, n);
      dy.get(g, l, n);
      float c = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        v[i] *= rstd;  // xhat; past the row's end 0, as dy
        dw[i] = fmaf(g[i], v[i], dw[i]);
        g[i] *= w[i];
        c = fmaf(g[i], v[i], c);
      }
      if (a.dx) {
        c = group_sum<LPR>(c, red) * inv_n;
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] = rstd * fmaf(-v[i], c, g[i]);
        if (a.ds) {
          ds.get(v, l, n);
#pragma unroll
          for (int i = 0; i < E; ++i) g[i] += v[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = 0.f;
    }
    if (a.dx) P::store(static_cast<T*>(a.dx) + row * n, l, n, g);
    now = next;
  }
  if (!a.part) return;
  float* out = a.part + (long)blockIdx.x * n;
  if constexpr (G > 1) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E; ++i) acc[(grp * E + i) * LPR + l] = dw[i];
    __syncthreads();
    // Element i of lane l, summed over the groups in order.
    for (int t = threadIdx.x; t < E * LPR; t += NT) {
      const int i = t / LPR, ll = t % LPR, c = (ll + LPR * (i / V)) * V + i % V;
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < G; ++q) sum += acc[(q * E + i) * LPR + ll];
      if (c < n) out[c] = sum;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = (l + LPR * (i / V)) * V + i % V;
      if (c < n) out[c] = dw[i];
    }
  }
}

// Most workgroups of the backward, each of which writes one partial of dw: those that
// run at once.
constexpr int kRmsBlocks = 768;

// The forward's: a group has one row or two (a wide model's 65536 rows of 1024 f16 to 8
// bits, 800 / 1024 / 16384 workgroups: 93 / 88 / 85 us).
int rms_forward_blocks(const RowPlan& p) { return p.lpr == 1024 ? 512 : 16384; }

int check_rms(int dtype, int param_dtype, int B, int L, int N, RowPlan& p) {
  if (dtype != FST_BF16 && dtype != FST_F32 && dtype != FST_F16)
    return fail(FST_EINVAL, "dtype must be FST_BF16, FST_F16 or FST_F32, got %d", dtype);
  if (param_dtype != dtype && param_dtype != FST_F32)
    return fail(FST_EINVAL, "param_dtype must be dtype or FST_F32, got %d", param_dtype);
  if (B < 0 || L < 0) return fail(FST_EINVAL, "negative size (B=%d, L=%d)", B, L);
  if (N < 1) return fail(FST_EINVAL, "need at least one feature, got N=%d", N);
  if ((long)B * L > 0x7fffffffL) return fail(FST_EUNSUPPORTED, "more than 2^31 - 1 rows");
  if (!plan_rows(dtype, N, p)) return fail(FST_EUNSUPPORTED, "rows of N=%d features: at most %d", N, kRowMax);
  return FST_OK;
}

template <typename T, bool Q8>
void launch_fwd(const RowPlan& p, const RmsArgs& a, int w_f32, hipStream_t st) {
  const int threads = p.lpr > 256 ? p.lpr : 256, blocks = row_blocks(p, a.rows, rms_forward_blocks(p));
  by_plan<T>(p, [&](auto lanes, auto pieces, auto edge) {
    rms_fwd<T, lanes(), pieces(), edge(), Q8><<<blocks, threads, 0, st>>>(a, w_f32);
  });
}

template <bool Q8>
int forward(int dtype, int param_dtype, int B, int L, int N, const void* x, int64_t x_stride, const void* residual,
            int64_t residual_stride, const void* weight, const int32_t* seqlens, float eps, void* y, void* sum,
            float* aside, void* stream) {
  clear_error();
  RowPlan p;
  const int rc = check_rms(dtype, param_dtype, B, L, N, p);
  if (rc != FST_OK) return rc;
  const long rows = (long)B * L;
  if (rows == 0) return FST_OK;
  if (!x || !y || (residual && !sum) || (Q8 && !aside)) return fail(FST_EINVAL, "null tensor pointer");
  if (x_stride < N || (residual && residual_stride < N)) return fail(FST_EINVAL, "row stride below N=%d", N);
  if (!(eps >= 0.f)) return fail(FST_EINVAL, "eps must not be negative");
  const size_t es = elem_size(dtype);
  const RmsArgs a{x, residual, weight, seqlens, y, sum, aside, rows, (long)x_stride, (long)residual_stride, L, N, eps};
  // Bytes go out as many at a time as elements come in: 8 or 4.
  p.edge = !aligned16(x, x_stride, es) || N * es % 16 != 0 || reinterpret_cast<uintptr_t>(y) % 16 != 0 ||
           (residual && (!aligned16(residual, residual_stride, es) || !aligned16(sum, N, es)));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int w_f32 = param_dtype == FST_F32;
  if (dtype == FST_BF16)
    launch_fwd<bf16, Q8>(p, a, w_f32, st);
  else if (dtype == FST_F16)
    launch_fwd<f16, Q8>(p, a, w_f32, st);
  else
    launch_fwd<float, Q8>(p, a, w_f32, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(FST_ELAUNCH, "RMS norm launch failed (%s)", hipGetErrorString(e));
  return FST_OK;
}

template <typename T>
void launch_bwd(const RowPlan& p, const RmsGradArgs& a, int blocks, int w_f32, hipStream_t st) {
  const int threads = p.lpr > 256 ? p.lpr : 256;
  by_plan<T>(p, [&](auto lanes, auto pieces, auto edge) {
    rms_bwd<T, lanes(), pieces(), edge()><<<blocks, threads, 0, st>>>(a, w_f32);
  });
}

}  // namespace

}  // namespace fst

using namespace fst;

extern "C" {

int fst_rms_norm_forward(int dtype, int param_dtype, int B, int L, int N, const void* x, int64_t x_stride,
                         const void* residual, int64_t residual_stride, const void* weight, const int32_t* seqlens,
                         float eps, void* y, void* sum, float* rstd, void* stream) {
  return forward<false>(dtype, param_dtype, B, L, N, x, x_stride, residual, residual_stride, weight, seqlens, eps, y, sum,
                        rstd, stream);
}

int fst_rms_norm_fp8(int dtype, int param_dtype, int B, int L, int N, const void* x, int64_t x_stride,
                     const void* residual, int64_t residual_stride, const void* weight, const int32_t* seqlens,
                     float eps, void* q, float* scale, void* sum, void* stream) {
  return forward<true>(dtype, param_dtype, B, L, N, x, x_stride, residual, residual_stride, weight, seqlens, eps, q, sum,
                       scale, stream);
}

size_t fst_rms_norm_backward_workspace_bytes(int dtype, int B, int L, int N) {
  RowPlan p;
  if (check_rms(dtype, dtype, B, L, N, p) != FST_OK) return 0;
  return align256((size_t)row_blocks(p, (long)B * L, kRmsBlocks) * N * sizeof(float));
}

int fst_rms_norm_backward(int dtype, int param_dtype, int B, int L, int N, const void* s, int64_t s_stride,
                          const void* weight, const int32_t* seqlens, const float* rstd, const void* dy,
                          int64_t dy_stride, const void* dsum, int64_t dsum_stride, void* dx, void* dweight,
                          void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  RowPlan p;
  const int rc = check_rms(dtype, param_dtype, B, L, N, p);
  if (rc != FST_OK) return rc;
  const long rows = (long)B * L;
  if (!dx && !dweight) return FST_OK;
  if (rows > 0) {
    if (!s || !dy || !rstd) return fail(FST_EINVAL, "null tensor pointer");
    if (s_stride < N || dy_stride < N || (dsum && dsum_stride < N)) return fail(FST_EINVAL, "row stride below N=%d", N);
  }
  const int blocks = row_blocks(p, rows, kRmsBlocks);
  const size_t need = align256((size_t)blocks * N * sizeof(float));
  if (dweight && need > 0 && (!workspace || workspace_bytes < need))
    return fail(FST_EWORKSPACE, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, need);
  const size_t es = elem_size(dtype);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int w_f32 = param_dtype == FST_F32;
  float* part = dweight ? static_cast<float*>(workspace) : nullptr;
  if (rows > 0) {
    const RmsGradArgs a{s, dy, dsum, weight, seqlens, rstd, dx, part,
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
  if (dweight) {
    const int grid = (N + 31) / 32;
    if (dtype == FST_BF16)
      column_sums<bf16><<<grid, 1024, 0, st>>>(part, blocks, N, N, dweight, nullptr, w_f32);
    else if (dtype == FST_F16)
      column_sums<f16><<<grid, 1024, 0, st>>>(part, blocks, N, N, dweight, nullptr, w_f32);
    else
      column_sums<float><<<grid, 1024, 0, st>>>(part, blocks, N, N, dweight, nullptr, w_f32);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(FST_ELAUNCH, "RMS norm backward launch failed (%s)", hipGetErrorString(e));
  return FST_OK;
}

}  // extern "C"
