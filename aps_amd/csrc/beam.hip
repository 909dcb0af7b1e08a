// One step of a beam search: the best K continuations of B hypotheses over a vocabulary of V, for N
// utterances at once, and the reordering of the decoder's states.
//
//   total[n, b, v] = score[n, b] + x[n, b, v] - log sum_v' exp(x[n, b, v'])
//
// The K largest of B V, ties to the lowest b V + v.  A hypothesis' own K largest logits hold every one
// of its candidates that can be selected, so the logits are read ONCE: a workgroup takes up to 8 192 of a
// row into registers, forms their maximum, their sum of exponentials and their K largest
// (`beam_rows_kernel`); a workgroup per utterance merges the B * splits * K candidates
// (`beam_merge_kernel`).  Sum and totals are in 64 bits: two candidates may lie closer than the
// rounding of a 32-bit log-softmax.  A row is cut by its tokens' numbers, wherever it lies in memory, so rows of
// equal logits have equal sums to the last bit and the tie between their hypotheses goes to the first.
#include "common.h"

namespace aps {
namespace beam {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any element: a global load takes them in one instruction wherever they begin
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned { u32x4 v; };
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kMaxBeam = 64, kTokenBits = 24, kCandidates = 1024, kHeld = 4;
constexpr float kLargest = 3.4028234663852886e38f;

// e^d for d <= 0 in 64 bits: 2^(i / 32) from a table, i the whole part of 32 d log2(e) and |f| <= 1/2 the rest, times
// e^(f ln(2) / 32) by its series to f^5 (cut off below 3e-15).  d is a difference from the largest logit, formed before
// anything is multiplied: it is 0 for that logit whatever its size, where d log2(e) taken as a difference of two
// products is the rounding error of the second (1e22 for the largest finite f32).  Relative error below
// 4e-15 + |d| 2^-52.  Table and series: as many operations as a series to f^8 alone, which is good to 1e-9.
constexpr int kOctave = 32;
constexpr double kStep = 46.16624130844683;  // kOctave log2(e)
__device__ __forceinline__ double exp_neg(double d, const double* table) {
  const double y = fmax(d * kStep, -34500.);           // (2^-1078: 0)
  const double t = y + 6755399441055744.;              // 1.5 * 2^52: the low bits are the nearest integer
  const int i = (int)(uint32_t)__double_as_longlong(t);
  const double f = y - (t - 6755399441055744.);
  double p = 3.9737099845494154e-11;  // (ln(2) / 32)^k / k!
  p = fma(p, f, 9.172562701824643e-09);
  p = fma(p, f, 1.6938509724371819e-06);
  p = fma(p, f, 2.3459619820224677e-04);
  p = fma(p, f, 2.166084939249829e-02);
  p = fma(p, f, 1.0);
  return ldexp(p * table[i & (kOctave - 1)], i >> 5);
}

// order-preserving integers: larger value, larger integer
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double from_ordered(uint64_t u) {
  return __longlong_as_double((long long)((u >> 63) ? (u & 0x7fffffffffffffffull) : ~u));
}

// A lower bound of the K-th largest of a wavefront's 64 unsigned values, K in 1 .. 64: the largest
// multiple of 2^LOW that at least K of them reach, a bit at a time by ballots (a sort by lane exchanges
// took three times as long)
template <int LOW>
__device__ __forceinline__ uint32_t wave_kth(uint32_t v, int K) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= LOW; --bit) {
    const uint32_t c = t | (1u << bit);
    if (__popcll(__ballot(v >= c)) >= K) t = c;
  }
  return t;
}

// Exclusive sum over the workgroup's threads, in no particular order of wavefronts, from *counter on
__device__ __forceinline__ int place(int n, int lane, int* counter) {
  int upto = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(upto, o, 64);
    if (lane >= o) upto += v;
  }
  int base = 0;
  if (lane == 63 && upto) base = atomicAdd(counter, upto);  // (the order of arrival does not matter: ranked later)
  return __shfl(base, 63, 64) + upto - n;
}

struct RowsArgs {
  const void* x;
  int64_t stride;          // elements between rows
  const float* score;      // [N B]
  const uint8_t* done;     // [N B] or null
  uint64_t* keys;          // [N B][splits][K]: ordered(x) << 32 | ~token, 0 = none
  float* top;              // [N B][splits]
  double* sum;             // [N B][splits]
  int64_t eos;
  int32_t V, K, splits;
};

template <typename T>
__device__ __forceinline__ void widen(u32x4 raw, float* to) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 v = __builtin_bit_cast(f32x4, raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = v[i];
  } else if constexpr (__is_same(T, __bf16)) {
    const bf16x8 v = __builtin_bit_cast(bf16x8, raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = (float)v[i];
  } else {
    const f16x8 v = __builtin_bit_cast(f16x8, raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = (float)v[i];
  }
}

// NaN counts as ruled out, +inf as the largest finite value
__device__ __forceinline__ float tame(float x) { return x != x ? -INFINITY : fminf(x, kLargest); }
// (-0 and 0 tie)
__device__ __forceinline__ uint64_t key_of(float x, int token) {
  return ((uint64_t)ordered(x + 0.f) << 32) | (uint32_t)~token;
}

// A workgroup takes 256 PER elements of a row: 32 a thread where there are rows enough to fill the chip,
// 8 (a shorter chain of dependent work) where there are not.
template <typename T, int PER>
__global__ __launch_bounds__(kThreads) void beam_rows_kernel(RowsArgs a) {
  constexpr int VE = 16 / (int)sizeof(T), NV = PER / VE, TILE = kThreads * PER;
  __shared__ __align__(16) uint64_t s_cand[kCandidates];
  __shared__ double s_sum[4], s_table[kOctave];
  __shared__ float s_top[4];
  __shared__ uint32_t s_kth[4];
  __shared__ uint64_t s_best[4];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t row = blockIdx.x;
  const int split = blockIdx.y, V = a.V, K = a.K;
  uint64_t* out = a.keys + (row * a.splits + split) * K;
  if (tid == 0) s_count = 0;
  if (tid < kOctave) s_table[tid] = exp2(tid * (1. / kOctave));
  const uint64_t none = (uint64_t)ordered(-INFINITY) << 32;  // key of a ruled-out token, its index apart
  const bool done = a.done && a.done[row];
  const bool dead = !(a.score[row] > -INFINITY);  // (NaN too)
  if (done || dead) {
    // no logit is looked at: a finished hypothesis goes on with eos at its own score, an unused one with
    // nothing; what is ruled out comes lowest token first, from the first split
    const bool ends = done && !dead;
    if (tid < K) {
      uint64_t key = 0;
      if (split == 0) {
        const int64_t token = ends ? (tid == 0 ? a.eos : tid - 1 + (tid > a.eos)) : tid;
        if (token < V) key = (ends && tid == 0 ? (uint64_t)ordered(0.f) << 32 : none) | (uint32_t)~(uint32_t)token;
      }
      out[tid] = key;
    }
    if (tid == 0) {
      a.top[row * a.splits + split] = ends && split == 0 ? 0.f : -INFINITY;
      a.sum[row * a.splits + split] = 1.;
    }
    return;
  }
  const T* base = static_cast<const T*>(a.x) + row * a.stride;
  const int first = split * TILE + tid * VE;  // vector j of the thread: tokens first + j * 256 VE ..
  float x[PER];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = first + j * kThreads * VE;
    float* to = x + j * VE;
    if (e0 + VE <= V) {
      widen<T>(reinterpret_cast<const Unaligned<T>*>(base + e0)->v, to);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) to[i] = e0 + i < V ? (float)base[e0 + i] : -INFINITY;
    }
  }
  float best = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    x[i] = tame(x[i]);
    best = fmaxf(best, x[i]);
  }
  // K of the threads' maxima are at least `least`, so the K largest elements are too
  const uint32_t kth = wave_kth<12>(ordered(best), K);
  const float wtop = wave_max(best);
  if (lane == 0) s_top[wv] = wtop, s_kth[wv] = kth;
  __syncthreads();
  const float top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  const uint32_t bound = max(max(s_kth[0], s_kth[1]), max(s_kth[2], s_kth[3]));
  // (ruled-out tokens are not collected: if they are needed at all, it is the lowest few)
  const float least = bound <= ordered(-kLargest) ? -kLargest : from_ordered(bound);
  uint32_t hits = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) hits |= x[i] >= least ? 1u << i : 0u;
  int at = place(__popc(hits), lane, &s_count);
  for (; hits; hits &= hits - 1) {  // few: read again rather than picked out of the registers
    const int i = __ffs(hits) - 1, e = first + i / VE * (kThreads * VE) + i % VE;
    if (at < kCandidates) s_cand[at] = key_of(tame((float)base[e]), e);
    ++at;
  }
  double sum = 0.;
  if (top > -INFINITY) {
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += exp_neg((double)x[i] - (double)top, s_table);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) s_sum[wv] = sum;
  __syncthreads();
  const int count = s_count;
  if (tid == 0) {
    a.top[row * a.splits + split] = top;
    a.sum[row * a.splits + split] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  }
  if (count <= kCandidates) {
    for (int c = tid; c < count; c += kThreads) {
      const uint64_t key = s_cand[c];
      int rank = 0;
#pragma unroll 8
      for (int o = 0; o < count; ++o) rank += s_cand[o] > key;
      if (rank < K) out[rank] = key;
    }
    if (count < K) {
      // Of the split's first K + count tokens at most `count` are not ruled out: the lowest ones of the rest
      // follow, then nothing.  (K + count < 128: two wavefronts)
      const int lo = split * TILE, hi = min(V, lo + TILE);
      bool out_of = false;
      if (tid < 128 && lo + tid < hi) out_of = tame((float)base[lo + tid]) == -INFINITY;
      const uint64_t mask = __ballot(out_of);
      if (lane == 0) s_best[wv] = mask;
      __syncthreads();
      const int below = __popcll(mask & ((1ull << lane) - 1)) + (wv == 1 ? __popcll(s_best[0]) : 0);
      if (out_of && count + below < K) out[count + below] = none | (uint32_t)~(uint32_t)(lo + tid);
      for (int c = count + __popcll(s_best[0]) + __popcll(s_best[1]) + tid; c < K; c += kThreads) out[c] = 0;
    }
    return;
  }
  // a great many equal values: K rounds of the largest key below the last
  uint64_t last = ~0ull;
  for (int k = 0; k < K; ++k) {
    uint64_t mx = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int e = first + j * kThreads * VE + i;
        if (!(x[j * VE + i] > -INFINITY)) continue;  // (there are more than K others)
        const uint64_t key = key_of(x[j * VE + i], e);
        if (key < last && key > mx) mx = key;
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor(mx, o, 64);
      mx = other > mx ? other : mx;
    }
    if (lane == 0) s_best[wv] = mx;
    __syncthreads();
    last = s_best[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) last = s_best[w] > last ? s_best[w] : last;
    if (tid == 0) out[k] = last;
    __syncthreads();
  }
}

struct MergeArgs {
  const uint64_t* keys;
  const float* top;
  const double* sum;
  const float* score;
  const uint8_t* done;
  float* new_score;     // [N, K]
  int64_t *parent, *token;
  uint8_t* new_done;
  int64_t eos;
  int32_t B, K, splits;
};

__global__ __launch_bounds__(kThreads) void beam_merge_kernel(MergeArgs a) {
  __shared__ uint64_t s_key[kCandidates], s_tie[kCandidates];
  // of a hypothesis: its score, its largest logit, log sum exp(logit - largest).  The last two stay apart: beside a
  // logit of 1e30 their sum would lose the logarithm.
  __shared__ double s_score[kMaxBeam], s_top[kMaxBeam], s_log[kMaxBeam];
  __shared__ uint32_t s_kth[4];
  __shared__ uint64_t s_best[4], s_best_tie[4];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t n = blockIdx.x;
  const int B = a.B, K = a.K, S = a.splits;
  if (tid == 0) s_count = 0;
  if (tid < B) {
    const int64_t row = n * B + tid;
    float top = -INFINITY;
    for (int s = 0; s < S; ++s) top = fmaxf(top, a.top[row * S + s]);
    double sum = 0.;
    if (top > -INFINITY)
      for (int s = 0; s < S; ++s)
        if (a.top[row * S + s] > -INFINITY)
          sum += a.sum[row * S + s] * exp((double)a.top[row * S + s] - (double)top);
    s_top[tid] = top > -INFINITY ? (double)top : 0.;
    s_log[tid] = top > -INFINITY ? log(sum) : 0.;
    s_score[tid] = (double)tame(a.score[row]);
  }
  const uint64_t* keys = a.keys + n * B * S * K;
  const int total = B * S * K;
  // the first candidates of each thread are on their way while the sums are formed
  uint64_t held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = tid + i * kThreads < total ? keys[tid + i * kThreads] : 0;
  __syncthreads();
  // Candidate c of the utterance: its total as an ordered integer (0: none), and what decides between equal totals,
  // the larger the better: the lower hypothesis, then the larger logit (64 bits may round two to one total, where the
  // row has kept the larger ones), then the lower token
  auto candidate = [&](int c, uint64_t key, uint64_t& tie) -> uint64_t {
    if (!key) return 0;
    const int b = c / (S * K);
    tie = (uint64_t)(kMaxBeam - 1 - b) << 56 | (key >> 32) << kTokenBits | ((uint32_t)key & ((1 << kTokenBits) - 1));
    const float x = from_ordered((uint32_t)(key >> 32));
    return ordered(x > -INFINITY ? s_score[b] + ((double)x - s_top[b] - s_log[b]) + 0. : (double)-INFINITY);
  };
  uint64_t best = 0;
  uint64_t held_tie[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    held_tie[i] = 0;
    held[i] = candidate(tid + i * kThreads, held[i], held_tie[i]);
    best = held[i] > best ? held[i] : best;
  }
  for (int c = tid + kHeld * kThreads; c < total; c += kThreads) {
    uint64_t tie;
    const uint64_t v = candidate(c, keys[c], tie);
    best = v > best ? v : best;
  }
  const uint32_t kth = wave_kth<0>((uint32_t)(best >> 32), K);  // (bounds the totals by their upper halves)
  if (lane == 0) s_kth[wv] = kth;
  __syncthreads();
  const uint32_t bound = max(max(s_kth[0], s_kth[1]), max(s_kth[2], s_kth[3]));
  const uint64_t least = bound ? (uint64_t)bound << 32 : 1;  // (0 is no candidate)
  int mine = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) mine += held[i] >= least;
  for (int c = tid + kHeld * kThreads; c < total; c += kThreads) {
    uint64_t tie;
    mine += candidate(c, keys[c], tie) >= least;
  }
  int at = place(mine, lane, &s_count);
  auto collect = [&](uint64_t v, uint64_t tie) {
    if (v < least) return;
    if (at < kCandidates) s_key[at] = v, s_tie[at] = tie;
    ++at;
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) collect(held[i], held_tie[i]);
  for (int c = tid + kHeld * kThreads; c < total; c += kThreads) {
    uint64_t tie = 0;
    const uint64_t v = candidate(c, keys[c], tie);
    collect(v, tie);
  }
  __syncthreads();
  const int count = s_count;
  auto put = [&](int rank, uint64_t v, uint64_t tie) {
    const int64_t b = kMaxBeam - 1 - (int64_t)(tie >> 56), token = ~(uint32_t)tie & ((1 << kTokenBits) - 1);
    const int64_t at = n * K + rank;
    a.new_score[at] = (float)from_ordered(v);
    a.parent[at] = b;
    a.token[at] = token;
    a.new_done[at] = (a.done && a.done[n * B + b]) || token == a.eos;
  };
  if (count <= kCandidates) {
    for (int c = tid; c < count; c += kThreads) {
      const uint64_t v = s_key[c];
      const uint64_t tie = s_tie[c];
      int rank = 0;
#pragma unroll 8
      for (int o = 0; o < count; ++o) rank += s_key[o] > v || (s_key[o] == v && s_tie[o] > tie);
      if (rank < K) put(rank, v, tie);
    }
    return;
  }
  uint64_t last = ~0ull, last_tie = ~0ull;
  for (int k = 0; k < K; ++k) {
    uint64_t mx = 0, mx_tie = 0;
    for (int c = tid; c < total; c += kThreads) {
      uint64_t tie = 0;
      const uint64_t v = candidate(c, keys[c], tie);
      if (!v || !(v < last || (v == last && tie < last_tie))) continue;
      if (v > mx || (v == mx && tie > mx_tie)) mx = v, mx_tie = tie;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t v = __shfl_xor(mx, o, 64), tie = __shfl_xor(mx_tie, o, 64);
      if (v > mx || (v == mx && tie > mx_tie)) mx = v, mx_tie = tie;
    }
    if (lane == 0) s_best[wv] = mx, s_best_tie[wv] = mx_tie;
    __syncthreads();
    last = s_best[0], last_tie = s_best_tie[0];
#pragma unroll
    for (int w = 1; w < 4; ++w)
      if (s_best[w] > last || (s_best[w] == last && s_best_tie[w] > last_tie)) last = s_best[w], last_tie = s_best_tie[w];
    if (tid == 0) put(k, last, last_tie);
    __syncthreads();
  }
}

// ---- states: row n K + k of a result is row n B + parent[n, k] of its source, for several tensors in
// one launch.  A tensor is [outer, rows, inner bytes]; a parent outside [0, B) gives zeros.
constexpr int kStates = 16, kUnits = 4;  // tensors a launch, units a thread
struct ReorderArgs {
  const char* src[kStates];
  char* dst[kStates];
  uint32_t unit[kStates];    // bytes a thread moves at once: 16, 8, 4, 2 or 1
  uint32_t inner[kStates];   // units a row
  int64_t units[kStates];    // outer * N * K * inner
  int64_t first[kStates];    // first block
  const int64_t* parent;
  uint32_t rows_in, rows_out, B, K;  // N B, N K
  int32_t count;
};

template <typename U, typename I>
__device__ __forceinline__ void move_units(const ReorderArgs& a, int s, int64_t i0) {
  U v[kUnits];
  int64_t at[kUnits];
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const int64_t i = i0 + j * 256;
    at[j] = i < a.units[s] ? i : -1;
    v[j] = U{};
    if (at[j] < 0) continue;
    const I flat = (I)i / a.inner[s];
    const uint32_t col = (uint32_t)((I)i - flat * a.inner[s]);
    const I outer = flat / a.rows_out;
    const uint32_t row = (uint32_t)(flat - outer * a.rows_out);
    const uint32_t n = row / a.K;
    const int64_t p = a.parent[row];
    if (p < 0 || p >= a.B) continue;
    v[j] = reinterpret_cast<const U*>(a.src[s])[((uint64_t)outer * a.rows_in + (uint64_t)n * a.B + p) * a.inner[s] + col];
  }
#pragma unroll
  for (int j = 0; j < kUnits; ++j)
    if (at[j] >= 0) reinterpret_cast<U*>(a.dst[s])[at[j]] = v[j];
}

__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a) {
  int s = 0;
  while (s + 1 < a.count && (int64_t)blockIdx.x >= a.first[s + 1]) ++s;
  const int64_t i0 = ((int64_t)blockIdx.x - a.first[s]) * (256 * kUnits) + threadIdx.x;
  const bool narrow = a.units[s] <= 0x7fffffff;  // (index arithmetic in 32 bits)
  switch (a.unit[s]) {
#define APS_MOVE(BYTES, U)                              \
  case BYTES:                                           \
    if (narrow) move_units<U, uint32_t>(a, s, i0);      \
    else move_units<U, uint64_t>(a, s, i0);             \
    break;
    APS_MOVE(16, u32x4)
    APS_MOVE(8, uint64_t)
    APS_MOVE(4, uint32_t)
    APS_MOVE(2, uint16_t)
    APS_MOVE(1, uint8_t)
#undef APS_MOVE
  }
}

// Elements a thread of the rows kernel takes.  32: 2 048 workgroups read 512 rows of 32 000 f32 logits in 25 us
// (2.6 TB/s; the 64-bit exponentials keep the vector pipe busy for about half of that).  8 for what would be fewer
// than two workgroups a CU: 8 rows of 4 233 in 5.7 us, with 32 in 7.5; 45 of 10 007 (bf16) in 6.0, with 32 in 7.9.
static int per_thread(int64_t rows, int64_t V) { return rows * ((V + 8191) / 8192) < 512 ? 8 : 32; }
static int64_t splits_of(int64_t rows, int64_t V) {
  const int64_t tile = kThreads * per_thread(rows, V);
  return (V + tile - 1) / tile;
}
static bool sizes_fit(int64_t N, int64_t B, int64_t V, int64_t K) {
  return N >= 1 && B >= 1 && B <= kMaxBeam && K >= 1 && K <= kMaxBeam && V >= 1 && V <= (1 << kTokenBits) &&
         K <= B * V && N <= 0x7fffffff / B;
}

template <typename T>
static void launch_rows(const RowsArgs& a, dim3 grid, bool wide, hipStream_t st) {
  if (wide) hipLaunchKernelGGL((beam_rows_kernel<T, 32>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((beam_rows_kernel<T, 8>), grid, dim3(kThreads), 0, st, a);
}

}  // namespace beam
}  // namespace aps

using namespace aps::beam;

extern "C" int64_t aps_beam_select_workspace(int64_t N, int64_t B, int64_t V, int64_t K) {
  if (!sizes_fit(N, B, V, K)) return -1;
  return N * B * splits_of(N * B, V) * (K * 8 + 16);
}

extern "C" int aps_beam_select(const void* logits, int64_t row_stride, const float* scores, const uint8_t* finished,
                               int64_t eos, float* new_scores, int64_t* parent, int64_t* token,
                               uint8_t* new_finished, int64_t N, int64_t B, int64_t V, int64_t K, int32_t dtype,
                               void* workspace, void* stream) {
  APS_CHECK_ARG(logits && scores && new_scores && parent && token && new_finished && workspace);
  APS_CHECK_ARG(sizes_fit(N, B, V, K) && row_stride >= V && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0);
  APS_CHECK_ARG(!finished || (eos >= 0 && eos < V));
  if (dtype < 0 || dtype > 2) return APS_ERR_UNSUPPORTED;
  const int64_t elem = dtype == 0 ? 4 : 2, S = splits_of(N * B, V);
  APS_CHECK_ARG((reinterpret_cast<uintptr_t>(logits) & (elem - 1)) == 0);
  RowsArgs r{};
  r.x = logits, r.stride = row_stride, r.score = scores, r.done = finished, r.eos = eos;
  r.V = (int32_t)V, r.K = (int32_t)K, r.splits = (int32_t)S;
  r.keys = static_cast<uint64_t*>(workspace);
  r.sum = reinterpret_cast<double*>(r.keys + N * B * S * K);
  r.top = reinterpret_cast<float*>(r.sum + N * B * S);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(N * B), (unsigned)S);
  const bool wide = per_thread(N * B, V) == 32;
  if (dtype == 0) launch_rows<float>(r, grid, wide, st);
  else if (dtype == 1) launch_rows<__bf16>(r, grid, wide, st);
  else launch_rows<_Float16>(r, grid, wide, st);
  if (aps_launch_status() != APS_OK) return APS_ERR_LAUNCH;
  MergeArgs m{};
  m.keys = r.keys, m.top = r.top, m.sum = r.sum, m.score = scores, m.done = finished, m.eos = eos;
  m.new_score = new_scores, m.parent = parent, m.token = token, m.new_done = new_finished;
  m.B = (int32_t)B, m.K = (int32_t)K, m.splits = (int32_t)S;
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)N), dim3(kThreads), 0, st, m);
  return aps_launch_status();
}

extern "C" int aps_beam_reorder(const void* const* src, void* const* dst, const int64_t* outer,
                                const int64_t* inner_bytes, int64_t count, const int64_t* parent, int64_t N,
                                int64_t K, int64_t B, void* stream) {
  APS_CHECK_ARG(src && dst && outer && inner_bytes && parent && count >= 0 && N >= 1 && K >= 1 && B >= 1);
  APS_CHECK_ARG(N <= 0x7fffffff / K && N <= 0x7fffffff / B);
  for (int64_t s0 = 0; s0 < count; s0 += kStates) {
    ReorderArgs a{};
    int64_t blocks = 0;
    for (int64_t s = s0; s < count && s < s0 + kStates; ++s) {
      APS_CHECK_ARG(outer[s] >= 0 && inner_bytes[s] >= 0);
      if (outer[s] == 0 || inner_bytes[s] == 0) continue;
      APS_CHECK_ARG(src[s] && dst[s] && inner_bytes[s] < 0x7fffffff);
      const uintptr_t at = reinterpret_cast<uintptr_t>(src[s]) | reinterpret_cast<uintptr_t>(dst[s]) | (uintptr_t)inner_bytes[s];
      const int i = a.count++;
      a.unit[i] = at & 1 ? 1 : (at & 3 ? 2 : (at & 7 ? 4 : (at & 15 ? 8 : 16)));
      a.src[i] = static_cast<const char*>(src[s]), a.dst[i] = static_cast<char*>(dst[s]);
      a.inner[i] = (uint32_t)(inner_bytes[s] / a.unit[i]);
      a.units[i] = outer[s] * N * K * a.inner[i];
      a.first[i] = blocks;
      blocks += (a.units[i] + 256 * kUnits - 1) / (256 * kUnits);
    }
    if (!a.count) continue;
    APS_CHECK_ARG(blocks < 0x7fffffff);
    a.parent = parent, a.rows_in = (uint32_t)(N * B), a.rows_out = (uint32_t)(N * K), a.B = (uint32_t)B, a.K = (uint32_t)K;
    hipLaunchKernelGGL(beam_reorder_kernel, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    if (aps_launch_status() != APS_OK) return APS_ERR_LAUNCH;
  }
  return APS_OK;
}
