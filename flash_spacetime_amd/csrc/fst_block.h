// Shared pieces of the transformer-block operators beside the attention: layer
// norm (fst_norm.hip) and the gated feed-forward block (fst_ffn*.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/flash_spacetime.h"

namespace fst {

// The last failure's message (fst_last_error); returns `code` (fst_capi.hip).
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Elements of a 16-byte piece.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
struct Piece {
  typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef V VU __attribute__((aligned(sizeof(T))));  // at any element's address
};

// Floats -> 16 bytes of T.
template <typename T>
__device__ __forceinline__ typename Piece<T>::V pack_piece(const float* v) {
  typename Piece<T>::V o;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) o[i] = (T)v[i];
  return o;
}

// Valid tokens of event b of a padded batch: its length within [0, L].
__device__ __forceinline__ int event_len(const int32_t* seqlens, int b, int L) {
  const int n = seqlens[b];
  return n < 0 ? 0 : (n > L ? L : n);
}

inline size_t align256(size_t x) { return (x + 255) / 256 * 256; }

inline size_t elem_size(int dtype) { return dtype == FST_F32 ? 4 : 2; }

}  // namespace fst
