// Parameters of the feed-forward block's kernels (fst_ffn_inst.hip), and the
// sizes their launches share with the host side (fst_ffn.hip).
#pragma once

#include "fst_block.h"

namespace fst {

// What a product writes.
enum FfnMode {
  kFfnGate = 0,  // a = x Wg^T + bg, u = x Wu^T + bu: h = act(a) u (and a, u)
  kFfnOut = 1,   // x W^T + b
  kFfnGrad = 2,  // dh = x W^T: da = dh u act'(a), du = dh act(a), one row of 2 F
};

// C[token, f] = sum_k x[token, k] w[f, k]: both operands contiguous along k.
struct FfnProduct {
  const void* w[2];        // [F, K], rows ldw apart; w[1] with kFfnGate
  const void* bias[2];     // [F] or null
  const void* x;           // rows of K, ldx apart
  void* out[3];            // kFfnGate: h, a, u (a, u may be null); else out[0]
  const void *gate, *up;   // kFfnGrad: a, u [tokens, F]
  const int32_t* count;    // tokens, on the device (seqlens given); or null
  const int32_t* rows_in;  // row of x of each token, or null (the token's own)
  const int32_t* rows_out; // row of out[0] of each token (kFfnOut), or null
  long ldx, ldo, ldw;      // elements
  int tokens;              // tokens, or the most there can be
  int F, K, act;
};

// C[n, m] = sum_token b[token, n] a[token, m], and sum_token b[token, n]: the
// gradient of a weight (and of the bias beside it), m contiguous in C.
// Workgroups with part >= 0 rows take `splits` equal runs of the tokens; each
// writes its own partial, summed in order afterwards.
struct FfnOuter {
  const void *a, *b;
  const int32_t *rows_a, *rows_b;  // rows of the tokens, or null
  long lda, ldb;
  int M, N;
  float* part;     // [splits][N][M]
  float* bias;     // [splits][N]
};

struct FfnOuters {
  FfnOuter p[2];
  int first[2];    // workgroups of the problems: [0, first[0]), [first[0], first[1])
  int splits[2];
  const int32_t* count;
  int tokens;
};

typedef int (*ffn_product_fn)(int mode, const FfnProduct&, hipStream_t);
typedef int (*ffn_outer_fn)(FfnOuters&, hipStream_t);

#define FST_FFN_DECL(name)                                      \
  int ffn_product_##name(int mode, const FfnProduct&, hipStream_t); \
  int ffn_outer_##name(FfnOuters&, hipStream_t);
FST_FFN_DECL(bf16)
FST_FFN_DECL(f16)
FST_FFN_DECL(f32)
#undef FST_FFN_DECL

// Tile of an outer product, in elements of M and N.
constexpr int kOuterM = 128, kOuterN = 256;

}  // namespace fst
