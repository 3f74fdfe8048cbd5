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
#include "fst_rows.h"

namespace fst {

namespace {

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

// Most workgroups. The forward's are those that its registers let run at once:
// each loads the parameters and then has a row ahead in flight, which is lost on those
// that would start after others (8000 rows of 1367 f16 3 / 4 / 8 a CU 15.2 / 18.0 / 21.1
// us; 4000 of 16384 bf16 2 / 8 a CU 54 / 72). The backward's each write one partial of
// dw and db; two a CU keep enough rows in flight (768 or 1024 are slower by what
// the partials cost).
constexpr int kNormBlocks = 512;

int norm_forward_blocks(const RowPlan& p, int dtype) {
  if (p.lpr == 1024) return 512;
  const int registers = 22 + p.nc * (dtype == FST_F32 ? 30 : 44);  // of a lane: 54 .. 154
  return 256 * (512 / registers);
}

template <typename T>
void launch_fwd(const RowPlan& p, const NormArgs& a, int blocks, int w_f32, hipStream_t st) {
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
void launch_bwd(const RowPlan& p, const NormGradArgs& a, int blocks, int w_f32, hipStream_t st) {
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

int check_norm(int dtype, int param_dtype, int B, int L, int N, RowPlan& p) {
  if (dtype != FST_BF16 && dtype != FST_F32 && dtype != FST_F16)
    return fail(FST_EINVAL, "dtype must be FST_BF16, FST_F16 or FST_F32, got %d", dtype);
  if (param_dtype != dtype && param_dtype != FST_F32)
    return fail(FST_EINVAL, "param_dtype must be dtype or FST_F32, got %d", param_dtype);
  if (B < 0 || L < 0) return fail(FST_EINVAL, "negative size (B=%d, L=%d)", B, L);
  if (N < 1) return fail(FST_EINVAL, "need at least one feature, got N=%d", N);
  if ((long)B * L > 0x7fffffffL) return fail(FST_EUNSUPPORTED, "more than 2^31 - 1 rows");
  if (!plan_rows(dtype, N, p))
    return fail(FST_EUNSUPPORTED, "rows of N=%d features: at most %d", N, kRowMax);
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
  RowPlan p;
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
  const int w_f32 = param_dtype == FST_F32, blocks = row_blocks(p, rows, norm_forward_blocks(p, dtype));
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
  RowPlan p;
  if (check_norm(dtype, dtype, B, L, N, p) != FST_OK) return 0;
  return align256((size_t)row_blocks(p, (long)B * L, kNormBlocks) * 2 * N * sizeof(float));
}

int fst_layer_norm_backward(int dtype, int param_dtype, int B, int L, int N, const void* s, int64_t s_stride,
                            const void* weight, const int32_t* seqlens, const float* stats, const void* dy,
                            int64_t dy_stride, const void* dsum, int64_t dsum_stride, void* dx, void* dweight,
                            void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  RowPlan p;
  const int rc = check_norm(dtype, param_dtype, B, L, N, p);
  if (rc != FST_OK) return rc;
  const long rows = (long)B * L;
  const bool sums = dweight || dbias;
  if (!dx && !sums) return FST_OK;
  if (rows > 0) {
    if (!s || !dy || !stats) return fail(FST_EINVAL, "null tensor pointer");
    if (s_stride < N || dy_stride < N || (dsum && dsum_stride < N)) return fail(FST_EINVAL, "row stride below N=%d", N);
  }
  const int blocks = row_blocks(p, rows, kNormBlocks);
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
      column_sums<bf16><<<grid, 1024, 0, st>>>(part, blocks, N, 2 * N, dweight, dbias, w_f32);
    else if (dtype == FST_F16)
      column_sums<f16><<<grid, 1024, 0, st>>>(part, blocks, N, 2 * N, dweight, dbias, w_f32);
    else
      column_sums<float><<<grid, 1024, 0, st>>>(part, blocks, N, 2 * N, dweight, dbias, w_f32);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(FST_ELAUNCH, "layer norm backward launch failed (%s)", hipGetErrorString(e));
  return FST_OK;
}

}  // extern "C"
