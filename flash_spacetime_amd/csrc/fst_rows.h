// Rows of features held in registers by groups of lanes, for the kernels that work on
// whole rows: the norms (fst_norm.hip, fst_rms.hip) and the experts' row movers
// (fst_experts.hip).
#pragma once

#include "fst_block.h"

#include <type_traits>

namespace fst {

namespace {

constexpr int kRowMax = 16384;  // features of a row

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

// The largest of the group's values, NaN left out of the comparison; every lane gets it.
template <int LPR>
__device__ __forceinline__ float group_max(float x, float* red) {
#define FST_ROR_MAX(n) \
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + n, 0xf, 0xf, false)))
  FST_ROR_MAX(8);
  FST_ROR_MAX(4);
  FST_ROR_MAX(2);
  FST_ROR_MAX(1);
#undef FST_ROR_MAX
  if constexpr (LPR >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  if constexpr (LPR >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    __syncthreads();  // what was reduced before is read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int i = 1; i < W; ++i) x = fmaxf(x, red[i]);
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

// dw | db = the column sums of part [blocks][2 n], in a fixed order: 32 columns a
// workgroup, 32 threads a column, eight loads of each in flight.
template <typename T>
__global__ __launch_bounds__(1024) void column_sums(const float* part, int blocks, int n, int cols, void* dw, void* db,
                                                      int w_f32) {
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c;
  float sum = 0.f;
  if (col < cols) {
    const float* in = part + col;
    int i = k;
    for (; i + 224 < blocks; i += 256) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = in[(long)(i + 32 * j) * cols];
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[j];
    }
    for (; i < blocks; i += 32) sum += in[(long)i * cols];
  }
  red[k][c] = sum;
  __syncthreads();
  if (k == 0 && col < cols) {
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
struct RowPlan {
  int lpr, nc;
  bool edge;
};

template <typename T>
constexpr int kMostPieces = sizeof(T) == 4 ? 4 : 3;

// Whether plan_rows gives some row L lanes of C pieces.
template <typename T>
constexpr bool planned(int L, int C) {
  const int fewer = L == 16 ? 0 : L == 32 ? 16 : L == 64 ? 32 : L == 256 ? 64 : 256;
  return C <= kMostPieces<T> && L * C > kMostPieces<T> * fewer && L * (C - 1) * kVec<T> < kRowMax;
}

bool plan_rows(int dtype, int n, RowPlan& p) {
  const int v = 16 / (int)elem_size(dtype), most = dtype == FST_F32 ? kMostPieces<float> : kMostPieces<bf16>;
  if (n > kRowMax) return false;
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

int rows_per_block(const RowPlan& p) { return p.lpr > 256 ? 1 : 256 / p.lpr; }

int row_blocks(const RowPlan& p, long rows, int most) {
  const long need = (rows + rows_per_block(p) - 1) / rows_per_block(p);
  return (int)(need < most ? need : most);
}

// f(lanes, pieces, edge) as constants of the plan's kernel for rows of T.
template <typename T, typename F>
void by_plan(const RowPlan& p, F f) {
  const auto pieces = [&](auto lanes, auto count) {
    if constexpr (planned<T>(lanes(), count())) {
      if (p.lpr == lanes() && p.nc == count()) {
        if (p.edge)
          f(lanes, count, std::true_type{});
        else
          f(lanes, count, std::false_type{});
      }
    }
  };
  const auto lanes = [&](auto l) {
    pieces(l, std::integral_constant<int, 1>{});
    pieces(l, std::integral_constant<int, 2>{});
    pieces(l, std::integral_constant<int, 3>{});
    pieces(l, std::integral_constant<int, 4>{});
  };
  lanes(std::integral_constant<int, 16>{});
  lanes(std::integral_constant<int, 32>{});
  lanes(std::integral_constant<int, 64>{});
  lanes(std::integral_constant<int, 256>{});
  lanes(std::integral_constant<int, 1024>{});
}

bool aligned16(const void* p, long ld, size_t es) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * es % 16 == 0; }

}  // namespace

}  // namespace fst
