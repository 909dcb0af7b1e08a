// Forward attention of a batch of packed sequences, a workgroup per (tile of 128 query rows, key head).
//
//   o_r = sum_j softmax_j(scale q_r . k_j) v_j,   j <= position of r (causal) or every key
//
// A query "row" is a (token, query head of the key head's group) pair, token-major: the G = Hq / Hkv
// heads that share keys share the key / value tiles too, whatever G is.  Wavefront w owns rows 32 w ..
// 32 w + 31 of the tile, one row per lane pair (l, l + 32): S^T = K Q^T leaves a row's scores in the
// registers of its lane pair, the softmax needs one exchange between the two halves, and S^T's
// registers are the operand of O^T = V^T P^T as they stand (attention_tile.h).  K and V go through two
// LDS buffers, the next tile's global loads being in flight during this tile's products: one barrier
// per tile.  Running maximum, sum and output stay in fp32; the output is rescaled only when the running
// maximum grows by more than 2^8 (the weights are then at most 2^8, exact to the same relative error).
//
// Measured (MI355X): 6 prompts of 660 - 8 192 tokens, 32 heads over 8 of 128, bf16, causal: 1.16 - 1.36 ms by card, 800 -
// 940 TFLOP/s; a large bf16 matrix product of the library reaches 1 157.  The matrix pipe is busy 45 % of the cycles
// (at 1.8 GHz: the card is at its power limit), the vector pipe, half of it the exponentials, about as much; the
// two wavefronts of a SIMD overlap the two only in part.  Wave priorities around the products or around the softmax
// cost 6 %.  Short sequences are bound by the chain bounds -> rows -> first tiles, about 5 us.
#ifndef APS_AMD_ATTENTION_ROWS_H_
#define APS_AMD_ATTENTION_ROWS_H_

#include "attention_tile.h"

namespace aps {
namespace att {

struct RowsArgs {
  const void *q, *k, *v;  // packed: k, v [total, Hkv, D] by strides; paged: pages [P, page, Hkv, D]
  void* out;              // [total, Hq, D]
  void* rest;             // packed, 16-bit: what the rounding of `out` took away, [total, Hq, D]; or null
  float* lse;             // [total, Hq] log2 of the softmax sum, +inf for a row that sees nothing; or null
  Index cu;               // [N + 1]
  Index kv_lens;          // paged: [N] keys of each sequence, its new tokens included
  const int32_t* table;   // paged: [N, table_stride]
  int64_t table_stride;
  int64_t total, N, tiles;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;  // strides in elements (paged: of a slot, of a head)
  int64_t num_pages, max_keys;           // paged
  int32_t page_shift;                    // paged: log2 of the page size
  int32_t G, Hkv;
  int32_t causal, zero_tail;
  int32_t by_cost;        // packed: tiles in the order of find_tile_by_cost
  float c;                // scale * log2(e) > 0
  // split over the keys (paged): partial results [split][total * Hq]{D floats} and {max, sum}
  float* part_o;
  float* part_ml;
  int32_t splits;
};

// Position of the first of a sequence's `len` new tokens, the last of its kv_lens[n] positions.  Whatever the array
// holds it lies in [-len, max_keys]: a token behind the table's `max_keys` positions keeps its place there, without a
// page of its own, and one before 0 sees nothing.
__device__ __forceinline__ int first_position(const Index& kv_lens, int64_t n, int len, int64_t max_keys) {
  const int64_t kv = kv_lens.at(n);
  return (int)((kv < 0 ? 0 : (kv > max_keys + len ? max_keys + len : kv)) - len);
}

// off + i, at most `most`
__device__ __forceinline__ int clipped(int off, int i, int most) { return (int)min((int64_t)off + i, (int64_t)most); }

// keys of a tile (f32: three planes; D = 32: a chunk for every thread)
template <typename T, int D>
constexpr int key_tile() { return sizeof(T) == 2 || D == 32 ? 64 : 32; }
constexpr int kRowTile = 128;

// Rows of no sequence (behind the last one; before the first, if cu_seqlens does not begin at 0) are
// cleared, by the workgroups that have no tile: number `first` of `step` of them
template <typename T, int D>
__device__ __forceinline__ void clear_rows(T* out, const Index& cu, int64_t N, int64_t total, int H, int64_t first,
                                           int64_t step) {
  int lead, unused;
  seq_range(cu, 0, total, lead, unused);
  const int64_t tail = max(tail_of(cu, N, total), (int64_t)lead);
  for (int64_t i = first; i < lead + total - tail; i += step) {
    T* row = out + (i < lead ? i : tail + i - lead) * (int64_t)H * D;
    for (int i = threadIdx.x; i < H * D / vec_elems<T>(); i += blockDim.x)
      reinterpret_cast<u32x4*>(row)[i] = u32x4{0, 0, 0, 0};
  }
}

// The next tile of keys (then of values, in the same registers) on its way from global memory to LDS:
// thread t carries chunk t % CH of rows t / CH + i * (256 / CH).  Paged rows outside [0, end) are zeros, packed ones
// the last key's, so nothing that lies there (an unwritten page, the next sequence) can reach a product.  16-bit rows of D = 128:
// the keys are in flight during a tile's scores and the values, in the same registers, during its second
// product, which is what keeps the kernel in 256 registers (a spilled register's reload waits for every load
// issued before it).  Otherwise both are in flight during the whole tile.
template <typename T, int D, bool PAGED>
struct KvStage {
  static constexpr int CH = D / kChunk, BK = key_tile<T, D>(), PER = BK * CH / 256, STEP = 256 / CH, PLANE = BK * D * 2;
  static constexpr bool TURNS = sizeof(T) == 2 && D == 128;  // keys, then values
  Raw<T> r[TURNS ? PER : 2 * PER];
  int32_t page[PER];  // paged: the table's entries for the rows of the tile behind the next one
  int slot[PER];      // paged: slots of the next tile's rows: -1 behind the end, -2 for a page outside the cache

  // The table is read a tile ahead of `resolve`, before the loads of the tile in between: memory answers in order, so
  // a look at an entry that was asked for behind them would wait for them all.
  __device__ __forceinline__ void locate(const RowsArgs& a, int seq, int key0, int end) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int key = min(key0 + (int)threadIdx.x / CH + i * STEP, end - 1);
        page[i] = a.table[(int64_t)seq * a.table_stride + (key >> a.page_shift)];
      }
    }
  }
  __device__ __forceinline__ void resolve(const RowsArgs& a, int key0, int end) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int key = key0 + (int)threadIdx.x / CH + i * STEP;
        slot[i] = page[i] < 0 || page[i] >= a.num_pages ? -2 : (page[i] << a.page_shift) + (key & ((1 << a.page_shift) - 1));
        if (key >= end) slot[i] = -1;
      }
    }
  }
  // base: the key head's row 0 (packed: of the sequence); row_stride in elements
  template <int WHICH>  // 0 keys, 1 values
  __device__ __forceinline__ void load(const T* base, int64_t row_stride, int key0, int end) {
    Raw<T>* r = this->r + (TURNS ? 0 : WHICH * PER);
    const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        r[i] = zero_raw<T>();
        if (slot[i] >= 0) r[i] = load_raw<T>(reinterpret_cast<const char*>(base + slot[i] * row_stride + c * kChunk));
      }
    } else {
      // (rows behind the end read the last one: only offsets lie behind the branch, since two ways with loads on both
      // meet in a wait for them)
      const char* at = reinterpret_cast<const char*>(base + key0 * row_stride);
      const uint32_t chunk_at = c * (kChunk * (int)sizeof(T));
      const int last = end - 1 - key0;
      uint32_t lane_at[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) lane_at[i] = (uint32_t)(r0 * (int)row_stride * (int)sizeof(T)) + chunk_at;
      if (last < BK - 1) {
        rare();
#pragma unroll
        for (int i = 0; i < PER; ++i)
          lane_at[i] = (uint32_t)(min(r0, max(last - i * STEP, 0)) * (int)row_stride * (int)sizeof(T)) + chunk_at;
      }
#pragma unroll
      for (int i = 0; i < PER; ++i)
        r[i] = load_chunk<T>(at + min(i * STEP, last) * (row_stride * (int)sizeof(T)), lane_at[i]);
    }
  }
  template <int WHICH>
  __device__ __forceinline__ void store(char* tile) const {
    const Raw<T>* r = this->r + (TURNS ? 0 : WHICH * PER);
    const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
#pragma unroll
    for (int i = 0; i < PER; ++i) store_chunk<T, D, PLANE>(tile, r0 + i * STEP, c, r[i]);
  }
  // Values on their way to a tile that some row sees only in part (f32: to any tile, a plane that is 0 times
  // infinity being NaN): 0 * infinity is not 0, so a non-finite value would reach the rows it is hidden from.  It
  // goes to LDS as 0 and is added to the rows that see it in the end (`add_non_finite`).  True if there was one.
  __device__ __forceinline__ bool sanitize() {
    Raw<T>* v = r + (TURNS ? 0 : PER);
    bool any = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = only_finite<T>(v[i], any);
    return any;
  }
  __device__ __forceinline__ void mark(uint8_t* hidden) const {
    if constexpr (PAGED) {
      if (threadIdx.x % CH == 0) {
#pragma unroll
        for (int i = 0; i < PER; ++i) hidden[threadIdx.x / CH + i * STEP] = slot[i] == -2;
      }
    }
  }
};

// the non-finite values of keys [from, to) to the rows that see them (seldom: straight from global memory)
template <typename T, int D, bool PAGED>
__device__ __forceinline__ void add_non_finite(const RowsArgs& a, const T* base, int seq, int from, int to, int pos,
                                               int half, f32x16* acc) {
  for (int key = from; key < to; ++key) {
    int64_t row = key;
    if constexpr (PAGED) {
      const int32_t p = a.table[(int64_t)seq * a.table_stride + (key >> a.page_shift)];
      if (p < 0 || p >= a.num_pages) continue;
      row = ((int64_t)p << a.page_shift) + (key & ((1 << a.page_shift) - 1));
    }
    if (key > pos) continue;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = (float)base[row * a.v_t + d * 32 + result_row(i, half)];
        acc[d][i] += finite(x) ? 0.f : x;
      }
  }
}

// wavefronts a SIMD has registers for
template <typename T, int D>
constexpr int rows_waves() { return D * planes<T>() >= 384 ? 1 : (D * planes<T>() >= 96 ? 2 : 3); }

template <typename T, int D, bool PAGED>
__global__ __launch_bounds__(256, (rows_waves<T, D>())) void attention_rows_kernel(RowsArgs a) {
  constexpr int BK = key_tile<T, D>(), NS = D / 16, NKB = BK / 32, NDB = D / 32, PLANE = BK * D * 2, TILE = planes<T>() * PLANE;
  constexpr bool ALWAYS = sizeof(T) == 4;  // non-finite values are taken out of every tile
  __shared__ __align__(16) char lds[4 * TILE];
  __shared__ uint8_t s_hidden[2][64];  // paged: keys without a page
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int h = blockIdx.x % a.Hkv;
  // the last tiles of a sequence see the most keys: they go first
  const int number = blockIdx.x / a.Hkv, want = !PAGED && a.by_cost ? number : (int)a.tiles - 1 - number;
  const SeqTile t = !PAGED && a.by_cost ? find_tile_by_cost(a.cu, (int)a.N, a.total, a.G, kRowTile, want, lane)
                                        : find_tile(a.cu, a.N, a.total, a.G, kRowTile, want, lane);
  const int Hq = a.Hkv * a.G;
  if (t.seq < 0) {
    if (a.zero_tail && h == 0 && blockIdx.y == 0)
      clear_rows<T, D>(static_cast<T*>(a.out), a.cu, a.N, a.total, Hq, want - t.used, a.tiles - t.used);
    return;
  }
  int kv = t.len, off = 0;  // keys; position of the sequence's first query
  if constexpr (PAGED) {
    off = first_position(a.kv_lens, t.seq, t.len, a.max_keys);
    kv = max(clipped(off, t.len, (int)a.max_keys), 0);
  }
  // the last key that token i of the sequence sees
  auto place = [&](int i) { return PAGED ? clipped(off, i, kv - 1) : i; };
  const int rows = t.len * a.G;
  const int row0 = t.tile * kRowTile + wv * 32;
  const int row = row0 + (lane & 31);
  const bool live = row < rows;
  const int tok = live ? row / a.G : 0, head = h * a.G + (live ? row - tok * a.G : 0);
  const int pos = live ? (a.causal ? place(tok) : kv - 1) : -1;
  // keys the tile / the wavefront can see; the least position in the wavefront (no mask below it)
  const int tile_last = min(t.tile * kRowTile + kRowTile, rows) - 1;
  const int last = min(row0 + 32, rows) - 1;
  int end = kv, wave_end = kv, wave_min = kv - 1;
  if (a.causal) {
    end = place(tile_last / a.G) + 1;
    wave_end = row0 < rows ? place(last / a.G) + 1 : 0;
    wave_min = place(row0 / a.G);
  } else if (row0 >= rows) {
    wave_end = 0;
  }
  const T* qp = static_cast<const T*>(a.q) + (t.start + tok) * a.q_t + head * a.q_h;
  Frag<T> qf[NS];  // (a row behind the last one: the sequence's first token, into a column that is not stored)
#pragma unroll
  for (int s = 0; s < NS; ++s)
    qf[s] = operand<T>(load_raw<T>(reinterpret_cast<const char*>(qp + (2 * s + half) * kChunk)));

  int tile_lo = 0, tile_hi = (max(end, 0) + BK - 1) / BK;
  if constexpr (PAGED) {
    if (a.splits > 1) {
      const int per = (tile_hi + a.splits - 1) / a.splits;
      tile_lo = min(tile_hi, per * (int)blockIdx.y);
      tile_hi = min(tile_hi, tile_lo + per);
    }
  }
  f32x16 acc[NDB];
#pragma unroll
  for (int d = 0; d < NDB; ++d) acc[d] = f32x16{0};
  float m = -INFINITY, l = 0.f;  // m: the reference the weights are taken against, in units of log2

  const T* kb = static_cast<const T*>(a.k) + h * a.k_h + (PAGED ? 0 : t.start * a.k_t);
  const T* vb = static_cast<const T*>(a.v) + h * a.v_h + (PAGED ? 0 : t.start * a.v_t);
  KvStage<T, D, PAGED> st;
  bool bad = false;  // a non-finite value in a tile that some row sees only in part
  // tiles that every row of the workgroup sees whole: no mask, no branch; then the others
  const int block_min = a.causal ? place(t.tile * kRowTile / a.G) : kv - 1;
  const int clear = min(tile_hi, (block_min + 1) / BK);
  if (tile_lo < tile_hi) {
    st.locate(a, t.seq, tile_lo * BK, end);
    st.resolve(a, tile_lo * BK, end);
    st.locate(a, t.seq, (tile_lo + 1) * BK, end);
    st.template load<0>(kb, a.k_t, tile_lo * BK, end);
    if (!st.TURNS) st.template load<1>(vb, a.v_t, tile_lo * BK, end);
    st.template store<0>(lds);
    st.mark(s_hidden[0]);
    if (st.TURNS) st.template load<1>(vb, a.v_t, tile_lo * BK, end);
    if (ALWAYS || tile_lo >= clear) bad |= st.sanitize();
    st.template store<1>(lds + TILE);
  }
  loads_done();
  __syncthreads();
  const LaneAt<T, D, PLANE> at_lane(lane);
  // one tile out of buffer `which`
  auto step = [&](int kt, int buf, auto edge) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge)::value;
    const char* tk = lds + buf * 2 * TILE;
    const char* tv = tk + TILE;
    char* nk = lds + (buf ^ 1) * 2 * TILE;
    const bool more = kt + 1 < tile_hi;
    const int k0 = kt * BK;
    const bool sees = !EDGE || k0 < wave_end;
    Frag<T> pf[NKB * 2];
    constexpr bool TURNS = KvStage<T, D, PAGED>::TURNS;
    if (more) {
      st.resolve(a, k0 + BK, end);
      st.locate(a, t.seq, k0 + 2 * BK, end);
      st.template load<0>(kb, a.k_t, k0 + BK, end);
      if (!TURNS) {
        st.template load<1>(vb, a.v_t, k0 + BK, end);
        st.mark(s_hidden[buf ^ 1]);
      }
    }
    if (sees) {
      f32x16 s[NKB];
#pragma unroll
      for (int b = 0; b < NKB; ++b) s[b] = f32x16{0};
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int b = 0; b < NKB; ++b) s[b] = mma<T>(at_lane.frag(tk, b * 32, i), qf[i], s[b]);
      if (EDGE && k0 + BK - 1 > wave_min) {
#pragma unroll
        for (int b = 0; b < NKB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (k0 + b * 32 + result_row(i, half) > pos) s[b][i] = -INFINITY;
      }
      if constexpr (PAGED) {
        const uint64_t hidden = __ballot(lane < BK && s_hidden[buf][lane]);
        if (hidden) {
          rare();
#pragma unroll
          for (int b = 0; b < NKB; ++b) {
            const uint32_t mine = (uint32_t)(hidden >> (b * 32)) >> (half * 4);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if ((mine >> ((i >> 2) * 8 + (i & 3))) & 1) s[b][i] = -INFINITY;
          }
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < NKB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
      top = fmaxf(top, __shfl_xor(top, 32, 64)) * a.c;
      if (__any(top > m + 8.f)) {
        rare();
        // (lane by lane: what a row comes to does not depend on the rows beside it)
        const float to = top > m + 8.f ? top : m;
        const float f = m == -INFINITY ? 1.f : exp2_fast(m - to);
        m = to;
        l *= f;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] *= f;
      }
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int b = 0; b < NKB; ++b) {
        float p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          p[i] = exp2_fast(fmaf(s[b][i], a.c, -ref));
          l += p[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) pf[b * 2 + i] = pack<T>(p + i * 8);
      }
    }
    if (TURNS && more) {
      st.template store<0>(nk);
      st.mark(s_hidden[buf ^ 1]);
      st.template load<1>(vb, a.v_t, k0 + BK, end);
    }
    if (sees) {
#pragma unroll
      for (int b = 0; b < NKB; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int d = 0; d < NDB; ++d) acc[d] = mma<T>(at_lane.frag_t(tv, b * 32, i, d), pf[b * 2 + i], acc[d]);
    }
    if (more) {
      if (!TURNS) st.template store<0>(nk);
      if (ALWAYS || EDGE || kt + 1 >= clear) {
        if (!ALWAYS) rare();
        bad |= st.sanitize();
      }
      st.template store<1>(nk + TILE);
    }
    __syncthreads();
  };
  int kt = tile_lo;
  for (; kt < clear; ++kt) step(kt, (kt - tile_lo) & 1, std::false_type());
  for (; kt < tile_hi; ++kt) step(kt, (kt - tile_lo) & 1, std::true_type());
  l += __shfl_xor(l, 32, 64);
  if ((ALWAYS || clear < tile_hi) && __syncthreads_or(bad)) {
    rare();
    add_non_finite<T, D, PAGED>(a, vb, t.seq, (ALWAYS ? tile_lo : max(clear, tile_lo)) * BK, min(end, tile_hi * BK), pos, half, acc);
  }
  if (!live) return;
  const int64_t at = (t.start + tok) * Hq + head;
  if constexpr (PAGED) {
    if (a.splits > 1) {  // unnormalised; combined by attention_combine_kernel
      const int64_t slot = (int64_t)blockIdx.y * a.total * Hq + at;
      float* po = a.part_o + slot * D;
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          store4<float>(po + d * 32 + result_row(i, half), f32x4{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]});
      if (half == 0) *reinterpret_cast<float2*>(a.part_ml + slot * 2) = make_float2(m, l);
      return;
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  T* po = static_cast<T*>(a.out) + at * D;
  T* pr = a.rest ? static_cast<T*>(a.rest) + at * D : nullptr;
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const f32x4 x = f32x4{acc[d][i] * inv, acc[d][i + 1] * inv, acc[d][i + 2] * inv, acc[d][i + 3] * inv};
      store4<T>(po + d * 32 + result_row(i, half), x);
      if (sizeof(T) == 2 && !PAGED && pr) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = x[e] - (float)(T)x[e];
        store4<T>(pr + d * 32 + result_row(i, half), y);
      }
    }
  if (a.lse && half == 0) a.lse[at] = l > 0.f ? m + log2_fast(l) : (l != l ? l : INFINITY);
}

// sizes every attention entry point takes: rows of a sequence are counted in 32 bits (token x head of
// the group), the grid in 31
static inline bool sizes_fit(int64_t total, int64_t N, int64_t Hq, int64_t Hkv) {
  if (total < 0 || N < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || Hq > 65536) return false;
  if (total > (int64_t)0x7fff0000 / (Hq / Hkv)) return false;
  return ((total * (Hq / Hkv) + 31) / 32 + N + 1) * Hkv < 0x7fffffff;  // (32: the smallest tile of any launch; 16 x more rows in the decode form are checked there)
}

// strides of a 16-byte-chunked tensor: whole chunks, and small enough for 32-bit offsets within a tile
static inline bool strides_fit(int64_t t, int64_t h, int64_t e) {
  const int64_t most = kMaxStride / (16 / e);
  return t % e == 0 && h % e == 0 && t >= 0 && t <= most && h >= 0 && h <= most;
}

// a scale whose product with log2(e) is a normal f32
static inline bool scale_fits(float scale) {
  const float c = scale * kLog2e;
  return c >= 1.17549435e-38f && c <= 3.4028234663852886e38f;
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace att
}  // namespace aps

#define APS_ATT_DISPATCH(FN, ...)                                                                      \
  if (dtype == kTypeF32 && head_dim == 32) FN<float, 32>(__VA_ARGS__);                                 \
  else if (dtype == kTypeF32 && head_dim == 64) FN<float, 64>(__VA_ARGS__);                            \
  else if (dtype == kTypeF32 && head_dim == 128) FN<float, 128>(__VA_ARGS__);                          \
  else if (dtype == kTypeBf16 && head_dim == 32) FN<__bf16, 32>(__VA_ARGS__);                          \
  else if (dtype == kTypeBf16 && head_dim == 64) FN<__bf16, 64>(__VA_ARGS__);                          \
  else if (dtype == kTypeBf16 && head_dim == 128) FN<__bf16, 128>(__VA_ARGS__);                        \
  else if (dtype == kTypeF16 && head_dim == 32) FN<_Float16, 32>(__VA_ARGS__);                         \
  else if (dtype == kTypeF16 && head_dim == 64) FN<_Float16, 64>(__VA_ARGS__);                         \
  else if (dtype == kTypeF16 && head_dim == 128) FN<_Float16, 128>(__VA_ARGS__);                       \
  else return APS_ERR_UNSUPPORTED

#endif  // APS_AMD_ATTENTION_ROWS_H_
