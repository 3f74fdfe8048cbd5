// Mixture of experts around its feed-forward (fst_ffn*.hip): the router, the
// tokens' slots sorted by expert, and rows moved to the experts' order and back.
//
//   route: of each token's E logits the K largest (ties: the lowest index), and
//     their softmax, over the chosen or over all:  w_k = exp(l_k - m) / sum.
//     Backward over the chosen: dl_k = w_k (dw_k - sum_j w_j dw_j), else 0; over all:
//     dl_e = [e chosen] w_e dw_e - p_e sum_j w_j dw_j, with p the softmax.
//   sort: a stable counting sort of the T K slots by expert.
//   spread: out[place[t, k]] = w[t, k] x[t] (w: 1), dw[t, k] = x[t] . back[place[t, k]].
//   gather: out[t] = sum_k w[t, k] rows[place[t, k]] (w: 1).
//
// The movers are bound by memory (or the launch, in calls of few tokens): they read each
// row once, hold it in registers (fst_rows.h) and write it to its K places, or
// read K rows and write their sum (256 x 768 padded, half of it tokens, two slots, 384
// bf16, of what each has to move: spread 64 us, 5.9 TB/s; weighted gather 77, 4.0; spread
// with dots 106, 5.1; gather 65, 4.7). The router is bound by its instructions and its
// waves' chain of loads (64 f32 logits, K = 4, the same batch: 13.4 us, 2.4 TB/s; its
// gradient 13.1, 4.6), the sort by the chain of its steps (786432 slots: 5.3 + 11.2 us). Sums are float32 in a fixed order; every output is
// rounded once. Places outside the rows are skipped, whoever wrote them; given the order
// beside them, spread writes every row once, zeros into those that no slot has (own_place:
// 0.5 us of 74 in passes of spread alone).
#include "fst_rows.h"

#include <algorithm>

namespace fst {

namespace {

constexpr int kMostExperts = 512, kMostChosen = 16;
constexpr long kMostSlots = 0x7fffffffL - 65536;  // and rows

// --- router -----------------------------------------------------------------

struct RouteArgs {
  const void* logits;
  const int32_t* lens;
  float* weights;
  int32_t* experts;
  long first, rows, ld;  // first: of the launch
  int L, E, K, chosen, wide;
};

struct RouteGradArgs {
  const void* logits;
  const int32_t* lens;
  const float *weights, *dw;
  const int32_t* experts;
  void* dlogits;
  long first, rows, ld;
  int L, E, K, chosen, wide, wide_out;
};

// A logit as an unsigned in its order, NaN above all. The two zeros are one. Keys up to
// -inf's cannot be chosen; 0 stands for what was.
constexpr unsigned kNotChosen = 0x007fffffu;
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned u = __float_as_uint(v + 0.f);
  return v != v ? 0xffffffffu : u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// x reduced with f over groups of G = 8, 16 or 64 lanes, pairs first: every lane gets it.
template <int G, typename F>
__device__ __forceinline__ unsigned group_reduce(unsigned x, F f) {
#define FST_WITH(pattern) f(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, pattern, 0xf, 0xf, false))
  x = FST_WITH(0xb1);   // the other of a pair
  x = FST_WITH(0x4e);   // the other pair of four
  x = FST_WITH(0x141);  // the other four of eight
  if constexpr (G >= 16) x = FST_WITH(0x140);
#undef FST_WITH
  if constexpr (G == 64) {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = f(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = f(b[0], b[1]);
  }
  return x;
}
template <int G>
__device__ __forceinline__ float lanes_sum(float x) {
  return __uint_as_float(group_reduce<G>(__float_as_uint(x), [](unsigned a, unsigned b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// Lane l of a row's G holds its logits l NC .. + NC - 1; -inf past the last. wide: rows and
// their ends on multiples of 16 bytes.
template <typename T, int NC>
constexpr bool kWideLogits = NC * sizeof(T) >= 16;

template <typename T, int NC>
__device__ __forceinline__ void load_logits(const T* row, int l, int E, bool wide, float* v) {
  constexpr int V = kVec<T>;
  if constexpr (kWideLogits<T, NC>) {
    if (wide) {
#pragma unroll
      for (int i = 0; i < NC; i += V) {
        const bool in = l * NC + i < E;
        typename Piece<T>::V q;
        if (in) q = *reinterpret_cast<const typename Piece<T>::V*>(row + l * NC + i);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i + j] = in ? (float)q[j] : -__builtin_inff();
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) v[i] = l * NC + i < E ? (float)row[l * NC + i] : -__builtin_inff();
}

template <typename T, int G, int NC>
__global__ __launch_bounds__(256) void expert_route(RouteArgs a) {
  const int l = threadIdx.x % G;
  const long row = a.first + (long)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (row >= a.rows) return;
  float w = 0.f;
  int expert = -1;  // lane k: the k-th largest
  if (row_valid(a.lens, row, a.L)) {
    float v[NC];
    load_logits<T, NC>(static_cast<const T*>(a.logits) + row * a.ld, l, a.E, a.wide, v);
    unsigned key[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) key[i] = order_key(v[i]);
    float top = 0.f, mine = 0.f;
    for (int k = 0; k < a.K; ++k) {
      unsigned best = key[0], at = l * NC;
#pragma unroll
      for (int i = 1; i < NC; ++i)
        if (key[i] > best) best = key[i], at = l * NC + i;
      const unsigned most = group_reduce<G>(best, [](unsigned x, unsigned y) { return max(x, y); });
      if (most <= kNotChosen) break;  // nothing left to choose: the same for all lanes of the row
      at = group_reduce<G>(best == most ? at : 0xffffffffu, [](unsigned x, unsigned y) { return min(x, y); });
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if ((int)at == l * NC + i) key[i] = 0;
      const float value = key_value(most);
      if (k == 0) top = value;
      if (l == k) mine = value, expert = (int)at;
    }
    w = expert >= 0 ? expf(mine - top) : 0.f;
    float sum = 0.f;
    if (a.chosen) {
      sum = w;
    } else {
#pragma unroll
      for (int i = 0; i < NC; ++i) sum += !(v[i] == -__builtin_inff()) ? expf(v[i] - top) : 0.f;
    }
    sum = lanes_sum<G>(sum);
    w = expert >= 0 ? w / sum : 0.f;
  }
  if (l < a.K) {
    a.weights[row * a.K + l] = w;
    a.experts[row * a.K + l] = expert;
  }
}

template <typename T, int G, int NC>
__global__ __launch_bounds__(256) void expert_route_grad(RouteGradArgs a) {
  const int l = threadIdx.x % G;
  const long row = a.first + (long)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (row >= a.rows) return;
  float d[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) d[i] = 0.f;
  if (row_valid(a.lens, row, a.L)) {
    int expert = -1;
    float w = 0.f, g = 0.f;
    if (l < a.K) expert = a.experts[row * a.K + l];
    if (expert >= 0) w = a.weights[row * a.K + l], g = a.dw[row * a.K + l];
    const float mean = lanes_sum<G>(w * g);
    g = a.chosen ? w * (g - mean) : w * g;
    if (!a.chosen) {
      float v[NC], top = -__builtin_inff(), sum = 0.f;
      load_logits<T, NC>(static_cast<const T*>(a.logits) + row * a.ld, l, a.E, a.wide, v);
#pragma unroll
      for (int i = 0; i < NC; ++i) top = fmaxf(top, v[i]);
      top = key_value(group_reduce<G>(order_key(top), [](unsigned x, unsigned y) { return max(x, y); }));
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        v[i] = v[i] == -__builtin_inff() ? 0.f : expf(v[i] - top);
        sum += v[i];
      }
      sum = lanes_sum<G>(sum);
#pragma unroll
      for (int i = 0; i < NC; ++i) d[i] = sum == 0.f ? 0.f : -mean * (v[i] / sum);
    }
    for (int k = 0; k < a.K; ++k) {
      const int at = __shfl(expert, k, G);
      const float add = __shfl(g, k, G);
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (at == l * NC + i) d[i] += add;
    }
  }
  T* out = static_cast<T*>(a.dlogits) + row * a.E + l * NC;
  if constexpr (kWideLogits<T, NC>) {
    if (a.wide_out) {
#pragma unroll
      for (int i = 0; i < NC; i += kVec<T>)
        if (l * NC + i < a.E) *reinterpret_cast<typename Piece<T>::V*>(out + i) = pack_piece<T>(d + i);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if (l * NC + i < a.E) out[i] = (T)d[i];
}

// f(lanes, logits a lane). A lane's own logits are compared at a few instructions each,
// lanes with each other at as many a step for all of them: few lanes with eight logits
// each (but one for each of the K). 256 x 768 padded tokens of 64 f32 logits, K = 4:
// 16 lanes of four 18.7 us, eight of eight 13.4.
template <typename F>
void by_experts(int E, int K, F f) {
  const auto with = [&](auto lanes, auto count) { f(lanes, count); };
#define FST_LANES(l, c) with(std::integral_constant<int, l>{}, std::integral_constant<int, c>{})
  if (E <= 64 && K <= 8) {
    if (E <= 8)
      FST_LANES(8, 1);
    else if (E <= 16)
      FST_LANES(8, 2);
    else
      FST_LANES(8, 8);
  } else if (E <= 16) {
    FST_LANES(16, 1);
  } else if (E <= 128) {
    FST_LANES(16, 8);
  } else {
    FST_LANES(64, 8);
  }
#undef FST_LANES
}

// launch(grid) for every run of rows that one launch takes: the lanes of all of them have to
// stay below 2^32, which 64 a row pass at 67 million rows.
template <typename A, typename F>
void by_runs(A& a, int lanes, F launch) {
  constexpr long kLanes = 1l << 31;
  for (a.first = 0; a.first < a.rows; a.first += kLanes / lanes)
    launch((unsigned)((std::min(a.rows - a.first, kLanes / lanes) * lanes + 255) / 256));
}

int check_route(int dtype, int B, int L, int E, int K) {
  if (dtype != FST_BF16 && dtype != FST_F32 && dtype != FST_F16)
    return fail(FST_EINVAL, "dtype must be FST_BF16, FST_F16 or FST_F32, got %d", dtype);
  if (B < 0 || L < 0) return fail(FST_EINVAL, "negative size (B=%d, L=%d)", B, L);
  if (E < 1 || K < 1 || K > E) return fail(FST_EINVAL, "top_k must be 1 .. experts, got %d of %d", K, E);
  if (E > kMostExperts || K > kMostChosen)
    return fail(FST_EUNSUPPORTED, "at most %d experts and %d of them a token, got %d, %d", kMostExperts, kMostChosen, E, K);
  if ((long)B * L > kMostSlots / K) return fail(FST_EUNSUPPORTED, "too many slots (B=%d, L=%d, top_k=%d)", B, L, K);
  return FST_OK;
}

// --- sort -------------------------------------------------------------------

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64, kMostBins = kMostExperts + 1;

struct SortArgs {
  const int32_t* experts;
  int32_t *order, *place, *offsets;
  int32_t* counts;  // [blocks][E + 1], or null: one workgroup
  int slots, E, chunk, bits;
};

// A slot's bin: its expert, or E where that is none.
__device__ __forceinline__ int bin_of(int expert, int E) { return (unsigned)expert < (unsigned)E ? expert : E; }

// Four of a wave's slots from `at` on, a lane's 64 apart: their bins, -1 past the end.
__device__ __forceinline__ void load_bins(const SortArgs& a, int at, int end, int* bin) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < 4; ++j) bin[j] = at + 64 * j + lane < end ? a.experts[at + 64 * j + lane] : -1;
#pragma unroll
  for (int j = 0; j < 4; ++j) bin[j] = at + 64 * j + lane < end ? bin_of(bin[j], a.E) : -1;
}

// Among the wave's 64 slots: how many of this one's bin come before it, and how many there
// are. Ballots over the bin's bits tell; an atomic addition for each slot would run 64
// deep where all are of one bin, as padding is.
__device__ __forceinline__ void rank_of(int bin, int bits, int& rank, int& count) {
  unsigned long long same = __ballot(bin >= 0);
  for (int b = 0; b < bits; ++b) {
    const bool set = (bin >> b) & 1;
    const unsigned long long those = __ballot(set);
    same &= set ? those : ~those;
  }
  rank = __builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0));
  count = __popcll(same);
}

__global__ __launch_bounds__(kSortThreads) void expert_count(SortArgs a) {
  __shared__ int count[kMostBins];
  for (int i = threadIdx.x; i <= a.E; i += kSortThreads) count[i] = 0;
  __syncthreads();
  const int s0 = blockIdx.x * a.chunk, s1 = s0 + min(a.chunk, a.slots - s0);
  for (int s = s0 + (threadIdx.x >> 6) * 256; s < s1; s += kSortWaves * 256) {
    int bin[4];
    load_bins(a, s, s1, bin);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int rank, n;
      rank_of(bin[j], a.bits, rank, n);
      if (bin[j] >= 0 && rank == 0) atomicAdd(&count[bin[j]], n);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i <= a.E; i += kSortThreads) a.counts[(long)blockIdx.x * (a.E + 1) + i] = count[i];
}

// Each wave of a workgroup takes a run of its chunk. A slot's row: those of smaller
// bins, of its bin in the chunks before and in the waves before, and those before it in
// its wave. All integers: the order of the additions does not matter.
__global__ __launch_bounds__(kSortThreads) void expert_place(SortArgs a) {
  __shared__ int next[kSortWaves][kMostBins];  // counts, then the next row, of each wave and bin
  __shared__ int total[kMostBins], before[kMostBins];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = a.E + 1;
  const int c0 = blockIdx.x * a.chunk, c1 = c0 + min(a.chunk, a.slots - c0);
  const int run = ((c1 - c0 + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int s0 = min(c0 + wave * run, c1), s1 = min(s0 + run, c1);
  int bin[4], rank[4], count[4];
  load_bins(a, s0, s1, bin);
  volatile int* mine = next[wave];
  for (int i = lane; i < bins; i += 64) mine[i] = 0;
  for (int i = tid; i < bins; i += kSortThreads) total[i] = before[i] = 0;
  __syncthreads();
  if (a.counts) {
    // Thread (part, bin): every parts-th workgroup's count, all loads in flight (sort_plan:
    // at most 32).
    const int width = 1 << a.bits, parts = max(kSortThreads / width, 1), e = tid & (width - 1), blocks = gridDim.x;
    if (e < bins && tid / width < parts) {
      int n[32], all = 0, low = 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const int b = tid / width + j * parts;
        n[j] = b < blocks ? a.counts[(long)b * bins + e] : 0;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        all += n[j];
        low += tid / width + j * parts < (int)blockIdx.x ? n[j] : 0;
      }
      atomicAdd(&total[e], all);
      atomicAdd(&before[e], low);
    }
  }
  for (int s = s0; s < s1; s += 256) {
    if (s > s0) load_bins(a, s, s1, bin);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      rank_of(bin[j], a.bits, rank[j], count[j]);
      if (bin[j] >= 0 && rank[j] == 0) mine[bin[j]] = mine[bin[j]] + count[j];
    }
  }
  __syncthreads();
  if (!a.counts) {
    for (int i = tid; i < bins; i += kSortThreads) {
      int n = 0;
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) n += next[w][i];
      total[i] = n;
    }
    __syncthreads();
  }
  if (wave == 0) {  // total -> rows of smaller bins
    int carry = 0;
    for (int i = lane; i - lane < bins; i += 64) {
      const int n = i < bins ? total[i] : 0;
      int sum = n;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
      }
      if (i < bins) {
        total[i] = carry + sum - n;
        if (blockIdx.x == 0) a.offsets[i] = carry + sum - n;
      }
      carry += __shfl(sum, 63);
    }
  }
  __syncthreads();
  // Sixteen threads a bin, one for each wave.
  static_assert(kSortWaves == 16, "a row of lanes");
  for (int i = tid >> 4; i < bins; i += kSortThreads / 16) {
    const int w = tid & 15, n = next[w][i];
    int sum = n;
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
      const int up = __shfl_up(sum, d, 16);
      if (w >= d) sum += up;
    }
    next[w][i] = total[i] + before[i] + sum - n;
  }
  __syncthreads();
  for (int s = s0; s < s1; s += 256) {
    if (run > 256) {
      load_bins(a, s, s1, bin);
#pragma unroll
      for (int j = 0; j < 4; ++j) rank_of(bin[j], a.bits, rank[j], count[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (bin[j] < 0) continue;
      const int row = mine[bin[j]] + rank[j], slot = s + 64 * j + lane;
      if (rank[j] == 0) mine[bin[j]] = row + count[j];  // after every lane's read: LDS keeps a wave's order
      a.place[slot] = bin[j] < a.E ? row : -1;
      a.order[row] = bin[j] < a.E ? slot : -1;
    }
  }
}

struct SortPlan {
  int blocks, chunk;
};

// Up to 8192 slots one workgroup does all; more are counted first, by chunks of which
// every workgroup then adds up all counts (16384 of them at most).
SortPlan sort_plan(int slots, int E) {
  if (slots <= 8192) return SortPlan{1, slots};
  long blocks = 16384 / (E + 1);
  blocks = blocks > 256 ? 256 : blocks;
  const long need = (slots + 2047l) / 2048;
  blocks = blocks > need ? need : blocks;
  const long chunk = ((slots + blocks - 1) / blocks + 1023) / 1024 * 1024;
  return SortPlan{(int)((slots + chunk - 1) / chunk), (int)chunk};
}

// --- rows to the experts and back -------------------------------------------

struct MoveArgs {
  const void* in;       // spread: the tokens' rows; gather: the experts'
  const void* back;     // spread: the experts' rows the dots are with, or null
  const void* weights;  // [tokens, K], or null
  const int32_t* place;
  const int32_t* used;   // rows of the experts, on the device (null: all)
  const int32_t* order;  // spread: the slot of each of the first order_rows rows, or null
  void *out, *dw;
  long tokens, rows, ld, ldb;
  int K, n, order_rows;
};

// Rows that a place may name.
__device__ __forceinline__ int place_end(const MoveArgs& a) {
  return a.used ? min(max(*a.used, 0), (int)a.rows) : (int)a.rows;
}

// Lanes of a wave that work on one row.
template <int LPR>
constexpr int kRowLanes = LPR < 64 ? LPR : 64;

// Lane k of the row's lanes in a wave: the k-th place of token t (-1: none, and past
// the K).
template <int LPR>
__device__ __forceinline__ int load_place(const MoveArgs& a, long t, int end) {
  const int k = threadIdx.x % kRowLanes<LPR>;
  if (t >= a.tokens || k >= a.K) return -1;
  const int r = a.place[t * a.K + k];
  return (unsigned)r < (unsigned)end ? r : -1;
}
// The same where the order gives that row to the slot, else -1: only such a slot writes it,
// and rows that no slot writes are found by the rows (zero_free_rows). So every row has one
// writer, whatever the tables hold: places may have been taken out since the sort.
template <int LPR>
__device__ __forceinline__ int own_place(const MoveArgs& a, int place, long t) {
  if (!a.order || place < 0) return place;
  return place < a.order_rows && a.order[place] == (int)(t * a.K) + (int)(threadIdx.x % kRowLanes<LPR>) ? place : -1;
}
// Zeros into the rows below `end` that own_place gives to no slot: a lane looks at one of
// 64 rows, and the wave clears those found.
template <typename T, int NT>
__device__ __forceinline__ void zero_free_rows(const MoveArgs& a, int end) {
  const int lane = threadIdx.x & 63;
  const long slots = a.tokens * a.K;
  for (long r0 = ((long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6)) * 64; r0 < end; r0 += (long)gridDim.x * NT) {
    const long r = r0 + lane;
    bool none = r < end;
    if (none && r < a.order_rows) {
      const int slot = a.order[r];
      none = slot < 0 || slot >= slots || a.place[slot] != r;
    }
    for (unsigned long long m = __ballot(none); m; m &= m - 1) {
      T* row = static_cast<T*>(a.out) + (r0 + __builtin_ctzll(m)) * a.n;
      for (int c = lane; c < a.n; c += 64) row[c] = (T)0.f;
    }
  }
}
template <int LPR>
__device__ __forceinline__ bool any_place(int place) {
  const unsigned long long b = __ballot(place >= 0);
  if constexpr (LPR >= 64) return b != 0;
  return ((b >> (threadIdx.x & 63 & ~(LPR - 1))) & ((1ull << (LPR & 63)) - 1)) != 0;
}
template <int LPR>
__device__ __forceinline__ int place_at(int place, int k) {
  return __shfl(place, k, kRowLanes<LPR>);
}
// Lane k's weight of token t, whatever its place (1 without weights): asked for with the
// place, a token ahead, so that neither waits for the other.
template <typename T, int LPR>
__device__ __forceinline__ float load_weight(const MoveArgs& a, long t, bool f32) {
  const int k = threadIdx.x % kRowLanes<LPR>;
  if (!a.weights || t >= a.tokens || k >= a.K) return 1.f;
  const long i = t * a.K + k;
  return f32 ? static_cast<const float*>(a.weights)[i] : (float)static_cast<const T*>(a.weights)[i];
}
template <int LPR>
__device__ __forceinline__ float weight_at(float weight, int k) {
  return __shfl(weight, k, kRowLanes<LPR>);
}

// A group walks the tokens with the next one's row, and the places of the one after it,
// in flight; a token without places is not read.
template <typename T, int LPR, int NC, bool EDGE, bool DOT>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void expert_spread(MoveArgs a, int w_f32) {
  typedef Pieces<T, LPR, NC, EDGE> P;
  constexpr int E = P::E, NT = LPR > 256 ? LPR : 256, G = NT / LPR;
  __shared__ float red[LPR > 64 ? LPR / 64 : 1];
  const int l = threadIdx.x % LPR, n = a.n;
  const long step = (long)gridDim.x * G;
  const long first = (long)blockIdx.x * G + threadIdx.x / LPR;
  const int end = place_end(a);
  P x0, x1;
  long t = first;
  int now = load_place<LPR>(a, t, end), next = load_place<LPR>(a, t + step, end);
  float weight_next = load_weight<T, LPR>(a, t, w_f32);
  if (any_place<LPR>(now)) x0.load(static_cast<const T*>(a.in) + t * a.ld, l, n);
  int own_next = own_place<LPR>(a, now, t);
  for (; t < a.tokens; t += step) {
    const int later = load_place<LPR>(a, t + 2 * step, end);
    if (any_place<LPR>(next)) x1.load(static_cast<const T*>(a.in) + (t + step) * a.ld, l, n);
    const int own = own_next;
    own_next = own_place<LPR>(a, next, t + step);
    const float weight = weight_next;
    weight_next = load_weight<T, LPR>(a, t + step, w_f32);
    float v[E];
    if (any_place<LPR>(now)) x0.get(v, l, n);
    for (int k = 0; k < a.K; ++k) {
      const int to = place_at<LPR>(own, k);
      float dot = 0.f;
      if constexpr (DOT) {
        const int r = place_at<LPR>(now, k);
        if (r >= 0) {
          P y;
          float q[E];
          y.load(static_cast<const T*>(a.back) + r * a.ldb, l, n);
          y.get(q, l, n);
#pragma unroll
          for (int i = 0; i < E; ++i) dot = fmaf(v[i], q[i], dot);
          dot = group_sum<LPR>(dot, red);
        }
      }
      if (a.out && to >= 0) {
        T* out = static_cast<T*>(a.out) + (long)to * n;
        if (a.weights) {
          const float w = weight_at<LPR>(weight, k);
          float q[E];
#pragma unroll
          for (int i = 0; i < E; ++i) q[i] = w * v[i];
          P::store(out, l, n, q);
        } else {
          P::store(out, l, n, v);
        }
      }
      if (DOT && l == 0) {
        if (w_f32)
          static_cast<float*>(a.dw)[t * a.K + k] = dot;
        else
          static_cast<T*>(a.dw)[t * a.K + k] = (T)dot;
      }
    }
    x0 = x1;
    now = next;
    next = later;
  }
  if (!a.out) return;
  float zero[E];
#pragma unroll
  for (int i = 0; i < E; ++i) zero[i] = 0.f;
  for (long r = end + first; r < a.rows; r += step) P::store(static_cast<T*>(a.out) + r * n, l, n, zero);
  if (a.order) zero_free_rows<T, NT>(a, end);
}

// Two of a token's rows are in flight at a time, the next token's places before
// them. A token without places is zeros.
template <typename T, int LPR, int NC, bool EDGE>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void expert_gather(MoveArgs a, int w_f32) {
  typedef Pieces<T, LPR, NC, EDGE> P;
  constexpr int E = P::E, NT = LPR > 256 ? LPR : 256, G = NT / LPR;
  const int l = threadIdx.x % LPR, n = a.n;
  const long step = (long)gridDim.x * G;
  long t = (long)blockIdx.x * G + threadIdx.x / LPR;
  const int end = place_end(a);
  int now = load_place<LPR>(a, t, end);
  float weight_next = load_weight<T, LPR>(a, t, w_f32);
  for (; t < a.tokens; t += step) {
    const int next = load_place<LPR>(a, t + step, end);
    const float weight = weight_next;
    weight_next = load_weight<T, LPR>(a, t + step, w_f32);
    float sum[E];
#pragma unroll
    for (int i = 0; i < E; ++i) sum[i] = 0.f;
    for (int k = 0; k < a.K; k += 2) {
      const int ra = place_at<LPR>(now, k), rb = k + 1 < a.K ? place_at<LPR>(now, k + 1) : -1;
      P xa, xb;
      if (ra >= 0) xa.load(static_cast<const T*>(a.in) + ra * a.ld, l, n);
      if (rb >= 0) xb.load(static_cast<const T*>(a.in) + rb * a.ld, l, n);
      auto add = [&](const P& x, int k) __attribute__((always_inline)) {
        float q[E];
        x.get(q, l, n);
        const float w = weight_at<LPR>(weight, k);
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] = fmaf(w, q[i], sum[i]);
      };
      if (ra >= 0) add(xa, k);
      if (rb >= 0) add(xb, k + 1);
    }
    P::store(static_cast<T*>(a.out) + t * n, l, n, sum);
    now = next;
  }
}

// Most workgroups: a group then has one token or two, and a row's wait is covered by the
// other groups (256 x 768 padded, 384 bf16, two slots a token, spread / weighted gather /
// spread with dots / gather: 2048 workgroups 70 / 87 / 124 / 74 us, 16384 65 / 76 / 112 / 64).
constexpr int kMoveBlocks = 16384;

int check_move(int dtype, int weight_dtype, int64_t tokens, int K, int N, int64_t rows, RowPlan& p) {
  if (dtype != FST_BF16 && dtype != FST_F32 && dtype != FST_F16)
    return fail(FST_EINVAL, "dtype must be FST_BF16, FST_F16 or FST_F32, got %d", dtype);
  if (weight_dtype != dtype && weight_dtype != FST_F32)
    return fail(FST_EINVAL, "weight_dtype must be dtype or FST_F32, got %d", weight_dtype);
  if (tokens < 0 || rows < 0) return fail(FST_EINVAL, "negative size (%ld tokens, %ld rows)", (long)tokens, (long)rows);
  if (K < 1 || N < 1) return fail(FST_EINVAL, "need at least one slot and one feature, got %d, %d", K, N);
  if (K > kMostChosen) return fail(FST_EUNSUPPORTED, "at most %d slots a token, got %d", kMostChosen, K);
  if (rows > kMostSlots || tokens > kMostSlots / K) return fail(FST_EUNSUPPORTED, "too many rows");
  if (!plan_rows(dtype, N, p)) return fail(FST_EUNSUPPORTED, "rows of N=%d features: at most %d", N, kRowMax);
  return FST_OK;
}

template <typename T>
void launch_spread(const RowPlan& p, const MoveArgs& a, int w_f32, hipStream_t st) {
  const long most = a.out && a.rows > a.tokens ? a.rows : a.tokens;
  const int threads = p.lpr > 256 ? p.lpr : 256, blocks = row_blocks(p, most, kMoveBlocks);
  by_plan<T>(p, [&](auto lanes, auto pieces, auto edge) {
    if (a.back)
      expert_spread<T, lanes(), pieces(), edge(), true><<<blocks, threads, 0, st>>>(a, w_f32);
    else
      expert_spread<T, lanes(), pieces(), edge(), false><<<blocks, threads, 0, st>>>(a, w_f32);
  });
}

template <typename T>
void launch_gather(const RowPlan& p, const MoveArgs& a, int w_f32, hipStream_t st) {
  const int threads = p.lpr > 256 ? p.lpr : 256, blocks = row_blocks(p, a.tokens, kMoveBlocks);
  by_plan<T>(p, [&](auto lanes, auto pieces, auto edge) {
    expert_gather<T, lanes(), pieces(), edge()><<<blocks, threads, 0, st>>>(a, w_f32);
  });
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(FST_ELAUNCH, "%s launch failed (%s)", what, hipGetErrorString(e));
  return FST_OK;
}

}  // namespace

}  // namespace fst

using namespace fst;

extern "C" {

int fst_expert_route(int dtype, int B, int L, int E, int K, int normalize, const void* logits, int64_t logits_stride,
                     const int32_t* seqlens, float* weights, int32_t* experts, void* stream) {
  clear_error();
  const int rc = check_route(dtype, B, L, E, K);
  if (rc != FST_OK) return rc;
  const long rows = (long)B * L;
  if (rows == 0) return FST_OK;
  if (!logits || !weights || !experts) return fail(FST_EINVAL, "null tensor pointer");
  if (logits_stride < E) return fail(FST_EINVAL, "row stride below E=%d", E);
  const size_t es = elem_size(dtype);
  const bool wide = aligned16(logits, logits_stride, es) && E * es % 16 == 0;
  RouteArgs a{logits, seqlens, weights, experts, 0, rows, (long)logits_stride, L, E, K, normalize != 0, wide};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  by_experts(E, K, [&](auto lanes, auto count) {
    by_runs(a, lanes(), [&](unsigned grid) {
      if (dtype == FST_BF16)
        expert_route<bf16, lanes(), count()><<<grid, 256, 0, st>>>(a);
      else if (dtype == FST_F16)
        expert_route<f16, lanes(), count()><<<grid, 256, 0, st>>>(a);
      else
        expert_route<float, lanes(), count()><<<grid, 256, 0, st>>>(a);
    });
  });
  return launched("expert route");
}

int fst_expert_route_backward(int dtype, int B, int L, int E, int K, int normalize, const void* logits,
                              int64_t logits_stride, const int32_t* seqlens, const float* weights,
                              const int32_t* experts, const float* dweights, void* dlogits, void* stream) {
  clear_error();
  const int rc = check_route(dtype, B, L, E, K);
  if (rc != FST_OK) return rc;
  const long rows = (long)B * L;
  if (rows == 0) return FST_OK;
  if ((!normalize && !logits) || !weights || !experts || !dweights || !dlogits) return fail(FST_EINVAL, "null tensor pointer");
  if (!normalize && logits_stride < E) return fail(FST_EINVAL, "row stride below E=%d", E);
  const size_t es = elem_size(dtype);
  const bool whole = E * es % 16 == 0, wide = whole && aligned16(logits, logits_stride, es);
  RouteGradArgs a{logits, seqlens, weights, dweights, experts, dlogits, 0, rows, (long)logits_stride, L, E, K, normalize != 0,
                  wide, whole && aligned16(dlogits, E, es)};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  by_experts(E, K, [&](auto lanes, auto count) {
    by_runs(a, lanes(), [&](unsigned grid) {
      if (dtype == FST_BF16)
        expert_route_grad<bf16, lanes(), count()><<<grid, 256, 0, st>>>(a);
      else if (dtype == FST_F16)
        expert_route_grad<f16, lanes(), count()><<<grid, 256, 0, st>>>(a);
      else
        expert_route_grad<float, lanes(), count()><<<grid, 256, 0, st>>>(a);
    });
  });
  return launched("expert route backward");
}

static int check_sort(int slots, int E) {
  if (slots < 0) return fail(FST_EINVAL, "negative size (%d slots)", slots);
  if (E < 1) return fail(FST_EINVAL, "need at least one expert, got %d", E);
  if (E > kMostExperts) return fail(FST_EUNSUPPORTED, "at most %d experts, got %d", kMostExperts, E);
  if (slots > kMostSlots) return fail(FST_EUNSUPPORTED, "too many slots (%d)", slots);
  return FST_OK;
}

size_t fst_expert_sort_workspace_bytes(int slots, int E) {
  if (check_sort(slots, E) != FST_OK) return 0;
  const SortPlan p = sort_plan(slots, E);
  return p.blocks > 1 ? align256((size_t)p.blocks * (E + 1) * sizeof(int32_t)) : 0;
}

int fst_expert_sort(int slots, int E, const int32_t* experts, int32_t* order, int32_t* place, int32_t* offsets,
                    void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const int rc = check_sort(slots, E);
  if (rc != FST_OK) return rc;
  if (!offsets || (slots > 0 && (!experts || !order || !place))) return fail(FST_EINVAL, "null tensor pointer");
  const SortPlan p = sort_plan(slots, E);
  const size_t need = fst_expert_sort_workspace_bytes(slots, E);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(FST_EWORKSPACE, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, need);
  int bits = 0;
  while (E >> bits) ++bits;
  const SortArgs a{experts, order, place, offsets, p.blocks > 1 ? static_cast<int32_t*>(workspace) : nullptr,
                   slots, E, p.chunk, bits};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (p.blocks > 1) expert_count<<<p.blocks, kSortThreads, 0, st>>>(a);
  expert_place<<<p.blocks, kSortThreads, 0, st>>>(a);
  return launched("expert sort");
}

int fst_expert_spread_order(int dtype, int weight_dtype, int64_t tokens, int K, int N, int64_t rows, const void* x,
                            int64_t x_stride, const int32_t* place, const int32_t* order, int64_t order_rows,
                            const int32_t* used, const void* weights, const void* back, int64_t back_stride, void* out,
                            void* dweights, void* stream) {
  clear_error();
  RowPlan p;
  const int rc = check_move(dtype, weight_dtype, tokens, K, N, rows, p);
  if (rc != FST_OK) return rc;
  if (tokens == 0) back = dweights = nullptr;  // no dots: an empty result has no address
  if (!out && !dweights) return FST_OK;
  if ((out && !used) || (tokens > 0 && (!x || !place)) || (rows > 0 && !back != !dweights))
    return fail(FST_EINVAL, "null tensor pointer");
  if (x_stride < N || (back && back_stride < N)) return fail(FST_EINVAL, "row stride below N=%d", N);
  if (order_rows < 0) return fail(FST_EINVAL, "negative size (%ld rows of the order)", (long)order_rows);
  if (tokens == 0 && rows == 0) return FST_OK;
  const size_t es = elem_size(dtype);
  const MoveArgs a{x, dweights ? (back ? back : x) : nullptr, weights, place, used, order, out, dweights,
                   (long)tokens, (long)rows, (long)x_stride, (long)back_stride, K, N, (int)(order_rows < rows ? order_rows : rows)};
  p.edge = N * es % 16 != 0 || !aligned16(x, x_stride, es) || (back && !aligned16(back, back_stride, es)) ||
           reinterpret_cast<uintptr_t>(out) % 16 != 0;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int w_f32 = weight_dtype == FST_F32;
  if (dtype == FST_BF16)
    launch_spread<bf16>(p, a, w_f32, st);
  else if (dtype == FST_F16)
    launch_spread<f16>(p, a, w_f32, st);
  else
    launch_spread<float>(p, a, w_f32, st);
  return launched("expert spread");
}

int fst_expert_spread(int dtype, int weight_dtype, int64_t tokens, int K, int N, int64_t rows, const void* x,
                      int64_t x_stride, const int32_t* place, const int32_t* used, const void* weights,
                      const void* back, int64_t back_stride, void* out, void* dweights, void* stream) {
  return fst_expert_spread_order(dtype, weight_dtype, tokens, K, N, rows, x, x_stride, place, nullptr, 0, used, weights, back,
                                 back_stride, out, dweights, stream);
}

int fst_expert_gather_order(int dtype, int weight_dtype, int64_t tokens, int K, int N, int64_t rows, const void* x,
                            int64_t x_stride, const int32_t* place, const int32_t* used, const void* weights, void* out,
                            void* stream) {
  clear_error();
  RowPlan p;
  const int rc = check_move(dtype, weight_dtype, tokens, K, N, rows, p);
  if (rc != FST_OK) return rc;
  if (tokens == 0) return FST_OK;
  if (!out || !place || (rows > 0 && !x)) return fail(FST_EINVAL, "null tensor pointer");
  if (x_stride < N) return fail(FST_EINVAL, "row stride below N=%d", N);
  const size_t es = elem_size(dtype);
  const MoveArgs a{x, nullptr, weights, place, used, nullptr, out, nullptr, (long)tokens, (long)rows, (long)x_stride, 0, K, N, 0};
  p.edge = N * es % 16 != 0 || !aligned16(x, x_stride, es) || reinterpret_cast<uintptr_t>(out) % 16 != 0;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int w_f32 = weight_dtype == FST_F32;
  if (dtype == FST_BF16)
    launch_gather<bf16>(p, a, w_f32, st);
  else if (dtype == FST_F16)
    launch_gather<f16>(p, a, w_f32, st);
  else
    launch_gather<float>(p, a, w_f32, st);
  return launched("expert gather");
}

int fst_expert_gather(int dtype, int weight_dtype, int64_t tokens, int K, int N, int64_t rows, const void* x,
                      int64_t x_stride, const int32_t* place, const void* weights, void* out, void* stream) {
  return fst_expert_gather_order(dtype, weight_dtype, tokens, K, N, rows, x, x_stride, place, nullptr, weights, out, stream);
}

}  // extern "C"
