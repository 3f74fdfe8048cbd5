// Gated feed-forward block: C ABI, and the small kernels around its matrix
// products (fst_ffn_inst.hip).
//
//   a = x Wg^T + bg,  u = x Wu^T + bu,  h = act(a) u,  y = h Wd^T + bd;
//   dh = dy Wd,  da = dh u act'(a),  du = dh act(a),  dx = da Wg + du Wu,
//   dWg = da^T x,  dWu = du^T x,  dWd = dy^T h,  biases: column sums of da, du, dy.
//
// Forward: gate and up projections with the activation in one product, then the
// output product. Backward: da and du (side by side in one row, so that the
// products after them are one each), dx, and the weights' gradients, summed over
// runs of the tokens in order. h is kept from the forward; a and u are formed
// again (4 T F D operations beside the backward's 12) except in float32, which
// keeps them: rounded to 16 bits they had moved the gradients to 1.3 times
// the distance from 64 bits (bf16 0.0031 of their norm against 0.0024), and at D =
// 384 writing and reading them took as long as the products do.
// Padded batches are gathered on the way: a list of the valid rows is the
// products' token axis, so padding costs nothing but its zeros.
#include "fst_ffn.h"

namespace fst {

namespace {

// Zeros into the padding rows of event e, by thread `at` of `step`.
__device__ __forceinline__ void zero_padding(unsigned char* out, long row_bytes, int e, int L, int len, long at, long step) {
  u32x4* pad = reinterpret_cast<u32x4*>(out + ((long)e * L + len) * row_bytes);
  const long parts = (L - len) * (row_bytes / 16);
  for (long i = at; i < parts; i += step) pad[i] = u32x4{0, 0, 0, 0};
}

// Valid rows of a padded batch in order (map[0]: their number, map[1 ..]: the
// rows), and zeros into the padding rows of out. Workgroup x takes `per`
// consecutive events, its y-th slice of their rows.
__global__ __launch_bounds__(256) void ffn_rows(const int32_t* seqlens, int B, int L, int per, int32_t* map,
                                                unsigned char* out, long row_bytes) {
  __shared__ int red[256];
  const int e0 = blockIdx.x * per, e1 = min(e0 + per, B), tid = threadIdx.x;
  int sum = 0;
  for (int e = tid; e < e0; e += 256) sum += event_len(seqlens, e, L);
  red[tid] = sum;
  __syncthreads();
  for (int h = 128; h > 0; h >>= 1) {
    if (tid < h) red[tid] += red[tid + h];
    __syncthreads();
  }
  int off = red[0];
  const long at = (long)blockIdx.y * 256 + tid, step = (long)gridDim.y * 256;
  for (int e = e0; e < e1; ++e) {
    const int len = event_len(seqlens, e, L);
    for (long l = at; l < len; l += step) map[1 + off + l] = (int32_t)((long)e * L + l);
    zero_padding(out, row_bytes, e, L, len, at, step);
    off += len;
  }
  if (e1 == B && e0 < B && at == 0) map[0] = off;
}

// out[c * ldo + r] = in[r * C + c] for up to three matrices [R, C]; the workgroups
// after theirs write zeros into the padding rows of `pad` (seqlens given), `slices`
// of them for an event and every `groups`-th after it.
struct Transposes {
  const void* in[3];
  void* out[3];
  long ldo[3];
  int R[3], C[3], first[3];  // workgroups before the next matrix
  const int32_t* seqlens;
  unsigned char* pad;
  long row_bytes;
  int B, L, groups, slices;
};

// A workgroup turns a 64 x 64 tile through LDS, 16 bytes at a time in memory (by
// elements it took 9.6 us at 3 x 384 x 1024, 20 at 3 x 1024 x 2752). R and C are
// multiples of 8.
template <typename E>
__global__ __launch_bounds__(256) void ffn_transpose(Transposes p) {
  constexpr int V = 16 / sizeof(E), PER = 64 / V;  // elements of a piece; pieces of a tile's row
  typedef E Part __attribute__((ext_vector_type(V)));
  __shared__ __attribute__((aligned(16))) E tile[64][64 + V];
  if ((int)blockIdx.x >= p.first[2]) {
    const int at = (int)blockIdx.x - p.first[2], slice = at % p.slices;
    for (long e = at / p.slices; e < p.B; e += p.groups)
      zero_padding(p.pad, p.row_bytes, (int)e, p.L, event_len(p.seqlens, (int)e, p.L), (long)slice * 256 + threadIdx.x,
                   (long)p.slices * 256);
    return;
  }
  const int k = (int)blockIdx.x >= p.first[0] ? ((int)blockIdx.x >= p.first[1] ? 2 : 1) : 0;
  const int wg = (int)blockIdx.x - (k ? p.first[k - 1] : 0);
  const int R = p.R[k], C = p.C[k], nc = (C + 63) / 64;
  const int r0 = wg / nc * 64, c0 = wg % nc * 64;
  const E* in = static_cast<const E*>(p.in[k]);
  E* out = static_cast<E*>(p.out[k]);
#pragma unroll
  for (int i = threadIdx.x; i < 64 * PER; i += 256) {
    const int r = i / PER, c = i % PER * V;
    if (r0 + r < R && c0 + c < C) {
      const Part v = *reinterpret_cast<const Part*>(in + (long)(r0 + r) * C + c0 + c);
#pragma unroll
      for (int j = 0; j < V; ++j) tile[c + j][r] = v[j];
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < 64 * PER; i += 256) {
    const int c = i / PER, r = i % PER * V;
    if (c0 + c < C && r0 + r < R)
      *reinterpret_cast<Part*>(out + (c0 + c) * p.ldo[k] + r0 + r) = *reinterpret_cast<const Part*>(&tile[c][r]);
  }
}

// Gradients = the sums of their partials over the token runs, in order.
struct GradSums {
  const float* part[6];
  void* out[6];
  long stride[6];  // between the runs' partials
  long count[6];   // elements, a multiple of 4
  int splits[6], first[6];
};

template <typename T>
__global__ __launch_bounds__(256) void ffn_grad_sum(GradSums p) {
  int k = 0;
#pragma unroll
  for (int i = 0; i < 5; ++i) k += (int)blockIdx.x >= p.first[i];
  const long e = ((long)((int)blockIdx.x - (k ? p.first[k - 1] : 0)) * 256 + threadIdx.x) * 4;
  if (e >= p.count[k]) return;
  const float* in = p.part[k] + e;
  f32x4 sum = *reinterpret_cast<const f32x4*>(in);
  for (int s = 1; s < p.splits[k]; ++s) sum += *reinterpret_cast<const f32x4*>(in + s * p.stride[k]);
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (T)sum[i];
  *reinterpret_cast<T4*>(static_cast<T*>(p.out[k]) + e) = o;
}

int check_ffn(int dtype, int activation, int B, int L, int D, int F) {
  if (dtype != FST_BF16 && dtype != FST_F32 && dtype != FST_F16)
    return fail(FST_EINVAL, "dtype must be FST_BF16, FST_F16 or FST_F32, got %d", dtype);
  if (activation != FST_SILU && activation != FST_GELU && activation != FST_GELU_TANH)
    return fail(FST_EINVAL, "unknown activation %d", activation);
  if (B < 0 || L < 0) return fail(FST_EINVAL, "negative size (B=%d, L=%d)", B, L);
  if (D < 8 || F < 8 || D % 8 || F % 8)
    return fail(FST_EUNSUPPORTED, "features must be multiples of 8, got D=%d, F=%d", D, F);
  if (D > 65536 || F > 65536 || (long)D * F >= 1l << 28)
    return fail(FST_EUNSUPPORTED, "a weight of D=%d by F=%d: at most 65536 each and 2^28 - 1 elements", D, F);
  if ((long)B * L > 0x7fffffffL - 65536) return fail(FST_EUNSUPPORTED, "too many rows (B=%d, L=%d)", B, L);
  return FST_OK;
}

// A row stride in elements that the kernels do not take.
bool bad_stride(int64_t stride, int n, size_t es) { return stride < n || stride * es % 16 || stride >= (int64_t)(1ul << 32) / (int64_t)es; }

bool misaligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16) return true;
  return false;
}

ffn_product_fn product_of(int dtype) {
  return dtype == FST_BF16 ? ffn_product_bf16 : dtype == FST_F16 ? ffn_product_f16 : ffn_product_f32;
}
ffn_outer_fn outer_of(int dtype) {
  return dtype == FST_BF16 ? ffn_outer_bf16 : dtype == FST_F16 ? ffn_outer_f16 : ffn_outer_f32;
}

// Slices of an event's padding rows: about 1024 workgroups in all.
int slices_of(int events, int L) {
  const int most = (L + 31) / 32, want = events < 1024 ? 1024 / events : 1;
  return want < most ? want : most;
}

void launch_rows(const int32_t* seqlens, int B, int L, int32_t* map, void* out, int D, size_t es, hipStream_t st) {
  const int wgs = B < 1024 ? B : 1024, per = (B + wgs - 1) / wgs;
  ffn_rows<<<dim3((B + per - 1) / per, slices_of(wgs, L)), 256, 0, st>>>(seqlens, B, L, per, map,
                                                                        static_cast<unsigned char*>(out), (long)D * es);
}

// Tile (features a side) and token runs of the weights' gradients [2 F, D] and [D,
// F]: the least of the rounds of workgroups over the chip, at the rates a full
// chip reached (PFLOP/s, bf16: 1.1 in large tiles, one a CU: 65536 tokens, D = 1024,
// F = 2752, 9 runs 1105 us; 0.8 in small ones, two a CU: 4 runs 1412; 100500 tokens of
// 196608, D = 384, F = 1024, 7 runs 334 where large tiles leave a third empty and take 360),
// plus the runs' partials written and read. float32 is as fast in small tiles and
// has only those.
struct OuterPlan {
  int tile, splits;
};

OuterPlan plan_outer(int dtype, long tokens, int D, int F) {
  OuterPlan best{128, 1};
  double least = -1;
  for (const int e : {128, 256}) {
    if (e == 256 && dtype == FST_F32) continue;
    const long tiles = (long)((D + e - 1) / e) * ((2 * F + e - 1) / e + (F + e - 1) / e), slots = e == 256 ? 256 : 512;
    const double rate = (dtype == FST_F32 ? 0.12e15 : e == 256 ? 1.1e15 : 0.8e15) / slots;
    for (int s = 1; s <= 64 && (s == 1 || s * 256l <= tokens); ++s) {
      const double work = (double)tokens / s * 2 * e * e / rate;
      const double t = (double)((tiles * s + slots - 1) / slots) * work + s * 24.0 * D * F / 5e12;
      if (least < 0 || t < least) best = OuterPlan{e, s}, least = t;
    }
  }
  return best;
}

struct GradLayout {
  size_t wdt, w2t, dadu, part0, part1, bias0, bias1, total;
  OuterPlan outer;
};

GradLayout grad_layout(int dtype, long rows, int D, int F) {
  GradLayout l;
  const size_t es = elem_size(dtype), df = (size_t)D * F;
  l.outer = plan_outer(dtype, rows, D, F);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += align256(bytes);
    return at;
  };
  l.wdt = take(df * es);
  l.w2t = take(2 * df * es);
  l.dadu = take((size_t)rows * 2 * F * es);
  l.part0 = take(l.outer.splits * 2 * df * 4);
  l.part1 = take(l.outer.splits * df * 4);
  l.bias0 = take((size_t)l.outer.splits * 2 * F * 4);
  l.bias1 = take((size_t)l.outer.splits * D * 4);
  l.total = off;
  return l;
}

}  // namespace

}  // namespace fst

using namespace fst;

extern "C" {

int fst_ffn_forward(int dtype, int activation, int B, int L, int D, int F, const void* x, int64_t x_stride,
                    const void* w_gate, const void* w_up, const void* w_down, const void* b_gate, const void* b_up,
                    const void* b_down, const int32_t* seqlens, void* hidden, void* gate, void* up, int32_t* rowmap,
                    void* y, void* stream) {
  clear_error();
  int rc = check_ffn(dtype, activation, B, L, D, F);
  if (rc != FST_OK) return rc;
  const long rows = (long)B * L;
  if (rows == 0) return FST_OK;
  if (!x || !w_gate || !w_up || !w_down || !hidden || !y || (seqlens && !rowmap) || !gate != !up)
    return fail(FST_EINVAL, "null tensor pointer");
  if (gate && ffn_redo(dtype)) return fail(FST_EINVAL, "gate and up are kept in float32 only");
  const size_t es = elem_size(dtype);
  if (bad_stride(x_stride, D, es)) return fail(FST_EINVAL, "x's row stride must be at least D, whole 16 bytes and below 2^32");
  if (misaligned({x, w_gate, w_up, w_down, b_gate, b_up, b_down, hidden, gate, up, y}))
    return fail(FST_EINVAL, "pointers must be multiples of 16 bytes");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (seqlens) launch_rows(seqlens, B, L, rowmap, y, D, es, st);
  FfnProduct p{};
  p.count = seqlens ? rowmap : nullptr;
  p.tokens = (int)rows;
  p.act = activation;
  p.w[0] = w_gate;
  p.w[1] = w_up;
  p.bias[0] = b_gate;
  p.bias[1] = b_up;
  p.x = x;
  p.ldx = x_stride;
  p.rows_in = seqlens ? rowmap + 1 : nullptr;
  p.out[0] = hidden;
  p.out[1] = gate;
  p.out[2] = up;
  p.ldo = F;
  p.ldw = p.K = D;
  p.F = F;
  rc = product_of(dtype)(kFfnGate, p, st);
  if (rc == FST_OK) {
    p.w[0] = w_down;
    p.bias[0] = b_down;
    p.x = hidden;
    p.rows_in = nullptr;
    p.rows_out = seqlens ? rowmap + 1 : nullptr;
    p.out[0] = y;
    p.ldo = D;
    p.ldx = p.ldw = p.K = F;
    p.F = D;
    rc = product_of(dtype)(kFfnOut, p, st);
  }
  if (rc != FST_OK) return fail(rc, "feed-forward launch failed");
  return FST_OK;
}

int fst_ffn_tiles(int dtype, int B, int L, int D, int F, int32_t* tiles) {
  clear_error();
  const int rc = check_ffn(dtype, FST_SILU, B, L, D, F);
  if (rc != FST_OK) return rc;
  if (!tiles) return fail(FST_EINVAL, "null pointer");
  const ffn_tile_fn tile_of = dtype == FST_BF16 ? ffn_tile_bf16 : dtype == FST_F16 ? ffn_tile_f16 : ffn_tile_f32;
  FfnProduct p{};
  p.tokens = B * L;
  p.F = F;
  tiles[0] = tile_of(kFfnGate, p);
  tiles[2] = tile_of(ffn_redo(dtype) ? kFfnRedo : kFfnGrad, p);
  p.F = D;
  tiles[1] = tiles[3] = tile_of(kFfnOut, p);
  const OuterPlan outer = plan_outer(dtype, (long)B * L, D, F);
  tiles[4] = outer.tile;
  tiles[5] = outer.splits;
  return FST_OK;
}

size_t fst_ffn_backward_workspace_bytes(int dtype, int B, int L, int D, int F) {
  if (check_ffn(dtype, FST_SILU, B, L, D, F) != FST_OK) return 0;
  return grad_layout(dtype, (long)B * L, D, F).total;
}

int fst_ffn_backward(int dtype, int activation, int B, int L, int D, int F, const void* x, int64_t x_stride,
                     const void* w_gate, const void* w_up, const void* w_down, const void* b_gate, const void* b_up,
                     const int32_t* seqlens, const void* hidden, const void* gate, const void* up,
                     const int32_t* rowmap, const void* dy, int64_t dy_stride, void* dx, void* dw_gate, void* dw_up, void* dw_down, void* db_gate,
                     void* db_up, void* db_down, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = check_ffn(dtype, activation, B, L, D, F);
  if (rc != FST_OK) return rc;
  const long rows = (long)B * L;
  const bool first = dw_gate || dw_up || db_gate || db_up, second = dw_down || db_down;
  if (!first && !second && !dx) return FST_OK;
  const size_t es = elem_size(dtype);
  if (rows > 0) {
    if (!x || !w_gate || !w_up || !w_down || !hidden || !dy || (seqlens && !rowmap) || (!ffn_redo(dtype) && !(gate && up)))
      return fail(FST_EINVAL, "null tensor pointer");
    if (bad_stride(x_stride, D, es) || bad_stride(dy_stride, D, es))
      return fail(FST_EINVAL, "row strides of x and dy must be at least D, whole 16 bytes and below 2^32");
  }
  if (misaligned({x, w_gate, w_up, w_down, b_gate, b_up, hidden, gate, up, dy, dx, dw_gate, dw_up, dw_down, db_gate, db_up, db_down,
                  workspace}))
    return fail(FST_EINVAL, "pointers must be multiples of 16 bytes");
  const GradLayout l = grad_layout(dtype, rows, D, F);
  if (!workspace || workspace_bytes < l.total)
    return fail(FST_EWORKSPACE, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, l.total);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int32_t* map = seqlens ? rowmap + 1 : nullptr;

  if (rows > 0 && (first || dx)) {
    Transposes t{};
    int grid = 0;
    auto add = [&](int k, const void* in, size_t out, int R, int C, long ldo) {
      t.in[k] = in;
      t.out[k] = ws + out;
      t.R[k] = R;
      t.C[k] = C;
      t.ldo[k] = ldo;
      if (in) grid += ((R + 63) / 64) * ((C + 63) / 64);
      t.first[k] = grid;
    };
    add(0, w_down, l.wdt, D, F, D);
    add(1, dx ? w_gate : nullptr, l.w2t, F, D, 2l * F);
    add(2, dx ? w_up : nullptr, l.w2t + F * es, F, D, 2l * F);
    if (seqlens && dx) {
      t.seqlens = seqlens;
      t.pad = static_cast<unsigned char*>(dx);
      t.row_bytes = (long)D * es;
      t.B = B;
      t.L = L;
      t.groups = B < 16384 ? B : 16384;
      t.slices = slices_of(t.groups, L);
      grid += t.groups * t.slices;
    }
    if (es == 2)
      ffn_transpose<uint16_t><<<grid, 256, 0, st>>>(t);
    else
      ffn_transpose<uint32_t><<<grid, 256, 0, st>>>(t);
    FfnProduct p{};
    p.count = seqlens ? rowmap : nullptr;
    p.tokens = (int)rows;
    p.act = activation;
    if (ffn_redo(dtype)) {
      p.w[0] = w_gate;
      p.w[1] = w_up;
      p.w[2] = ws + l.wdt;
      p.bias[0] = b_gate;
      p.bias[1] = b_up;
      p.x = x;
      p.ldx = x_stride;
      p.dy = dy;
      p.lddy = dy_stride;
    } else {
      p.w[0] = ws + l.wdt;
      p.x = dy;
      p.ldx = dy_stride;
      p.gate = gate;
      p.up = up;
    }
    p.rows_in = map;
    p.out[0] = ws + l.dadu;
    p.ldo = 2l * F;
    p.ldw = p.K = D;
    p.F = F;
    rc = product_of(dtype)(ffn_redo(dtype) ? kFfnRedo : kFfnGrad, p, st);
    if (rc == FST_OK && dx) {
      p.w[0] = ws + l.w2t;
      p.bias[0] = nullptr;
      p.x = ws + l.dadu;
      p.rows_in = nullptr;
      p.rows_out = map;
      p.out[0] = dx;
      p.ldo = D;
      p.ldx = p.ldw = p.K = 2 * F;
      p.F = D;
      rc = product_of(dtype)(kFfnOut, p, st);
    }
    if (rc != FST_OK) return fail(rc, "feed-forward backward launch failed");
  }
  if (first || second) {
    FfnOuters o{};
    if (rows > 0) {  // without rows the forward has written no map
      o.count = seqlens ? rowmap : nullptr;
      o.rows = map;
    }
    o.tokens = (int)rows;
    float *p0 = reinterpret_cast<float*>(ws + l.part0), *p1 = reinterpret_cast<float*>(ws + l.part1);
    float *b0 = reinterpret_cast<float*>(ws + l.bias0), *b1 = reinterpret_cast<float*>(ws + l.bias1);
    o.p[0] = FfnOuter{x, ws + l.dadu, (long)x_stride, 2l * F, D, 2 * F, first ? l.outer.splits : 0, p0,
                      db_gate || db_up ? b0 : nullptr};
    o.p[1] = FfnOuter{hidden, dy, F, (long)dy_stride, F, D, second ? l.outer.splits : 0, p1, db_down ? b1 : nullptr};
    rc = outer_of(dtype)(o, l.outer.tile, st);
    if (rc != FST_OK) return fail(rc, "feed-forward weight gradient launch failed");
    const long df = (long)D * F;
    const float* part[6] = {p0, p0 + df, p1, b0, b0 + F, b1};
    void* out[6] = {dw_gate, dw_up, dw_down, db_gate, db_up, db_down};
    const long stride[6] = {2 * df, 2 * df, df, 2l * F, 2l * F, D}, count[6] = {df, df, df, F, F, D};
    GradSums s{};
    int grid = 0;
    for (int k = 0; k < 6; ++k) {
      s.part[k] = part[k];
      s.out[k] = out[k];
      s.stride[k] = stride[k];
      s.count[k] = count[k];
      s.splits[k] = l.outer.splits;
      if (out[k]) grid += (int)((count[k] + 1023) / 1024);
      s.first[k] = grid;
    }
    if (dtype == FST_BF16)
      ffn_grad_sum<bf16><<<grid, 256, 0, st>>>(s);
    else if (dtype == FST_F16)
      ffn_grad_sum<f16><<<grid, 256, 0, st>>>(s);
    else
      ffn_grad_sum<float><<<grid, 256, 0, st>>>(s);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(FST_ELAUNCH, "feed-forward backward launch failed (%s)", hipGetErrorString(e));
  return FST_OK;
}

}  // extern "C"
