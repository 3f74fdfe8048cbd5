// Parameters of the feed-forward block's kernels (fst_ffn_inst.hip), and the
// sizes their launches share with the host side (fst_ffn.hip).
#pragma once

#include "fst_block.h"

namespace fst {

// What a product writes.
enum FfnMode {
  kFfnGate = 0,  // a = x Wg^T + bg, u = x Wu^T + bu: h = act(a) u (and a, u)
  kFfnOut = 1,   // x W^T + b
  kFfnGrad = 2,  // dh = x W^T: da = dh u act'(a), du = dh act(a), one row of 2 F, from a and u as kept
  kFfnRedo = 3,  // the same with a and u formed again (x Wg^T + bg, x Wu^T + bu; dh = dy W^T)
};

// Whether the backward forms a and u again: rounded to 16 bits they would move
// every gradient by as much as its own rounding does. float32 keeps them.
inline bool ffn_redo(int dtype) { return dtype != FST_F32; }

// C[token, f] = sum_k x[token, k] w[f, k]: both operands contiguous along k.
struct FfnProduct {
  const void* w[3];        // [F, K], rows ldw apart; w[1]: up, w[2]: dh's (kFfnRedo)
  const void* bias[2];     // [F] or null
  const void *x, *dy;      // rows of K, ldx, lddy apart; dy with kFfnRedo
  void* out[3];            // kFfnGate: h, a, u (a, u may be null); else out[0]
  const void *gate, *up;   // kFfnGrad: a, u [tokens, F]
  const int32_t* count;    // tokens, on the device (seqlens given); or null
  const int32_t* rows_in;  // row of x (and dy) of each token, or null (the token's own)
  const int32_t* rows_out; // row of out[0] of each token (kFfnOut), or null
  long ldx, lddy, ldo, ldw;  // elements
  int tokens;              // tokens, or the most there can be
  int F, K, act;
};

// C[n, m] = sum_token b[token, n] a[token, m], and sum_token b[token, n]: the
// gradient of a weight (and of the bias beside it), m contiguous in C. The tokens
// are taken in `splits` equal runs, each with a partial of its own, summed in
// order afterwards.
struct FfnOuter {
  const void *a, *b;
  long lda, ldb;   // elements; in bytes below 2^32
  int M, N, splits;
  float* part;     // [splits][N][M]
  float* bias;     // [splits][N], or null
};

// The block's two: (x, [da | du]) and (h, dy), in one launch. Either may have no
// splits: it is not asked for.
struct FfnOuters {
  FfnOuter p[2];
  const int32_t* count;  // tokens, on the device (seqlens given); or null
  const int32_t* rows;   // rows of x and dy of the tokens, or null
  int tokens;
  int first;             // workgroups of the first
};

typedef int (*ffn_product_fn)(int mode, const FfnProduct&, hipStream_t);
typedef int (*ffn_outer_fn)(FfnOuters&, int tile, hipStream_t);
typedef int (*ffn_tile_fn)(int mode, const FfnProduct&);

#define FST_FFN_DECL(name)                                      \
  int ffn_product_##name(int mode, const FfnProduct&, hipStream_t); \
  int ffn_outer_##name(FfnOuters&, int tile, hipStream_t);          \
  int ffn_tile_##name(int mode, const FfnProduct&);
FST_FFN_DECL(bf16)
FST_FFN_DECL(f16)
FST_FFN_DECL(f32)
#undef FST_FFN_DECL

}  // namespace fst
