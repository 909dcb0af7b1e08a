// Attention over sequences packed end to end, and its gradients:
//   P_rj = exp(scale q_r . k_j - lse_r),  o_r = sum_j P_rj v_j                    (attention_rows.h)
//   D_r  = do_r . o_r        (16-bit: of o and of what its rounding took away, which the forward pass keeps for it.
//          D_r enters every dS_rj, and sequences of 64 tokens would lose more by o's rounding than by that of
//          dS: dq off by 3.0e-3 instead of 2.3e-3 in bf16, where rounding the result alone is 1.7e-3.  Writing
//          and reading it takes 7 + 5 us of 400 on the 12 sequences named below.)
//   dS_rj = P_rj (do_r . v_j - D_r) scale
//   dq_r = sum_j dS_rj k_j,   dk_j = sum_r dS_rj q_r,   dv_j = sum_r P_rj do_r
// with r over the rows (token, head of the group) that see key j: the sums over a group's heads are part
// of the same accumulation.  Two launches, neither with atomics, so the gradients are bit-reproducible:
// the first walks the keys for a tile of rows (D_r, dq), the second walks the rows for a tile of keys
// (dk, dv); P is formed again in each from the saved lse.
//
// P and dS are rounded to the tensors' type between the products (attention_tile.h: `pack`).  f16 has 30 binary
// orders: dS, of the size of do / (row length), would fall below its normal numbers with upstream gradients of 1e-3 and
// pass its largest with 1e4, and P of long rows is small too.  So f16 takes both times powers of two, which come out
// again in f32 at the end: P times 2^14 where it is rounded (dv), dS times 2^(14 - e), 2^e > |do_r| |v| for the largest
// v the row sees (o_r, in D_r, is a mean of them all), so that |dS| <= 2 |do_r| |v| becomes at most 2^15.  A launch
// ahead leaves the largest norm of every 128 keys' values.  (On the 3 sequences named below that launch takes 6 us, dq
// goes from 184 to 187 us and dk / dv from 269 to 273; maxima by atomics in LDS: 291.)  For dq, e goes
// by the row's own norm; for dk by the largest of the rows that see the key tile (the dq launch leaves one for
// every 32 rows).
#include "attention_rows.h"

namespace aps {
namespace att {

struct GradArgs {
  const void *q, *k, *v, *o, *rest, *go;  // rest (16-bit): what the rounding of o took away
  const float* lse;    // [total, Hq]
  float* delta;        // [total, Hq]
  float* row_norm;     // f16: largest |do_r|^2 of 32 rows, at [h][start G + first row]; of the [Hkv][total G] few are used
  float* value_norm;   // f16: largest |v_j|^2 of 128 keys, at [h][start + first key]
  void *gq, *gk, *gv;  // [total, Hq | Hkv, D]
  Index cu;
  int64_t total, N, tiles;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, go_t, go_h;
  int32_t G, Hkv, causal, by_cost;
  float c, scale;
};

template <typename T>
constexpr bool narrow() { return __is_same(T, _Float16); }  // P and dS are scaled
constexpr int kNormKeys = 128, kOrders = 14;

// (an infinity or a NaN is left out: it makes NaN of what it reaches, whatever the factor)
__device__ __forceinline__ float finite_or_zero(float x) { return finite(x) ? x : 0.f; }
// the least e with |do| |v| < 2^e, from the norms' squares
__device__ __forceinline__ int order_of(float do2, float v2) { return (__builtin_amdgcn_frexp_expf(do2 * v2) + 1) >> 1; }

template <typename T, int D>
__global__ __launch_bounds__(256) void attention_value_norms_kernel(GradArgs a) {
  constexpr int CH = D / kChunk, STEP = 256 / CH;
  __shared__ float s_max[4];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, h = blockIdx.x % a.Hkv;
  const SeqTile t = find_tile(a.cu, a.N, a.total, 1, kNormKeys, blockIdx.x / a.Hkv, lane);
  if (t.seq < 0) return;
  const int key0 = t.tile * kNormKeys;
  const T* v = static_cast<const T*>(a.v) + (t.start + key0) * a.v_t + h * a.v_h + threadIdx.x % CH * kChunk;
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < kNormKeys / STEP; ++i) {
    const int key = min((int)threadIdx.x / CH + i * STEP, t.len - 1 - key0);  // (behind the end: the last one again)
    const Raw<T> r = load_raw<T>(reinterpret_cast<const char*>(v + key * a.v_t));
    float s = dot_raw<T>(r, r);
#pragma unroll
    for (int o = 1; o < CH; o <<= 1) s += __shfl_xor(s, o, 64);
    most = fmaxf(most, finite_or_zero(s));
  }
  most = wave_max(most);
  if (lane == 0) s_max[wv] = most;
  __syncthreads();
  if (threadIdx.x == 0)
    a.value_norm[h * a.total + t.start + key0] = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
}

// dq: the forward kernel's walk, with V as the left operand of dP^T = V dO^T beside S^T = K Q^T and K
// read transposed for dq^T = K^T dS^T.  (The 12 sequences named at the next kernel: 99 - 107 us by card, 620 - 670
// TFLOP/s; the 3: 187 us, 790.)
template <typename T, int D>
__global__ __launch_bounds__(256, (D * planes<T>() >= 192 ? 1 : 2)) void attention_rows_backward_kernel(GradArgs a) {
  constexpr int BK = key_tile<T, D>(), NS = D / 16, NKB = BK / 32, NDB = D / 32, PLANE = BK * D * 2, TILE = planes<T>() * PLANE;
  __shared__ __align__(16) char lds[4 * TILE];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int h = blockIdx.x % a.Hkv;
  const int number = blockIdx.x / a.Hkv, want = a.by_cost ? number : (int)a.tiles - 1 - number;
  const SeqTile t = a.by_cost ? find_tile_by_cost(a.cu, (int)a.N, a.total, a.G, kRowTile, want, lane)
                              : find_tile(a.cu, a.N, a.total, a.G, kRowTile, want, lane);
  const int Hq = a.Hkv * a.G;
  if (t.seq < 0) {
    if (h == 0)
      clear_rows<T, D>(static_cast<T*>(a.gq), a.cu, a.N, a.total, Hq, want - t.used, a.tiles - t.used);
    return;
  }
  const int kv = t.len, rows = t.len * a.G;
  const int row0 = t.tile * kRowTile + wv * 32, row = row0 + (lane & 31);
  const bool live = row < rows;
  const int tok = live ? row / a.G : 0, head = h * a.G + (live ? row - tok * a.G : 0);
  const int pos = live ? (a.causal ? tok : kv - 1) : -1;
  const int last = min(row0 + 32, rows) - 1;
  const int end = a.causal ? (min(t.tile * kRowTile + kRowTile, rows) - 1) / a.G + 1 : kv;
  const int wave_end = row0 >= rows ? 0 : (a.causal ? last / a.G + 1 : kv);
  const int wave_min = a.causal ? row0 / a.G : kv - 1;
  const int64_t at = (t.start + tok) * Hq + head;
  const T* qp = static_cast<const T*>(a.q) + (t.start + tok) * a.q_t + head * a.q_h;
  const T* gp = static_cast<const T*>(a.go) + (t.start + tok) * a.go_t + head * a.go_h;
  const T* op = static_cast<const T*>(a.o) + at * D;
  // (a row behind the last one computes with the sequence's first token, into a column that is not stored: loads
  // without a branch, so that all of them are under way together)
  Frag<T> qf[NS], gf[NS];
  float delta = 0.f;
  Raw<T> g[NS], o[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int c = (2 * s + half) * kChunk;
    qf[s] = operand<T>(load_raw<T>(reinterpret_cast<const char*>(qp + c)));
    g[s] = load_raw<T>(reinterpret_cast<const char*>(gp + c));
    o[s] = load_raw<T>(reinterpret_cast<const char*>(op + c));
  }
  if constexpr (sizeof(T) == 2) {
    const T* rp = static_cast<const T*>(a.rest) + at * D;
    Raw<T> r[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) r[s] = load_raw<T>(reinterpret_cast<const char*>(rp + (2 * s + half) * kChunk));
#pragma unroll
    for (int s = 0; s < NS; ++s) delta += dot_raw<T>(g[s], r[s]);
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) delta += dot_raw<T>(g[s], o[s]), gf[s] = operand<T>(g[s]);
  delta += __shfl_xor(delta, 32, 64);
  const float lse = a.lse[at];
  if (live && half == 0) a.delta[at] = delta;
  float times = 1.f, back = a.scale;  // f16: the factor of dS, and what takes it out again
  if constexpr (narrow<T>()) {
    float own = 0.f, most = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) own += dot_raw<T>(g[s], g[s]);
    own = finite_or_zero(own + __shfl_xor(own, 32, 64));
    for (int key = lane * kNormKeys; key < end; key += 64 * kNormKeys)
      most = fmaxf(most, a.value_norm[h * a.total + t.start + key]);
    const int order = order_of(own, wave_max(most));
    times = ldexpf(1.f, kOrders - order), back = ldexpf(a.scale, order - kOrders);
    delta *= times;
    const float rows_most = wave_max(live ? own : 0.f);
    if (lane == 0 && row0 < rows) a.row_norm[h * a.total * a.G + t.start * a.G + row0] = rows_most;
  }

  f32x16 acc[NDB];
#pragma unroll
  for (int d = 0; d < NDB; ++d) acc[d] = f32x16{0};
  const int tile_hi = (end + BK - 1) / BK;
  const T* kb = static_cast<const T*>(a.k) + h * a.k_h + t.start * a.k_t;
  const T* vb = static_cast<const T*>(a.v) + h * a.v_h + t.start * a.v_t;
  KvStage<T, D, false> st;
  st.template load<0>(kb, a.k_t, 0, end);
  if (!st.TURNS) st.template load<1>(vb, a.v_t, 0, end);
  st.template store<0>(lds);
  if (st.TURNS) st.template load<1>(vb, a.v_t, 0, end);
  st.template store<1>(lds + TILE);
  __syncthreads();
  const LaneAt<T, D, PLANE> at_lane(lane);
  auto step = [&](int kt, int buf, auto masked) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(masked)::value;
    const char* tk = lds + buf * 2 * TILE;
    const char* tv = tk + TILE;
    char* nk = lds + (buf ^ 1) * 2 * TILE;
    const bool more = kt + 1 < tile_hi;
    const int k0 = kt * BK;
    const bool sees = !EDGE || k0 < wave_end;
    // 32 keys at a time; the next tile's keys are in flight during the first half, its values during the second
    constexpr bool TURNS = KvStage<T, D, false>::TURNS;
    if (more) {
      st.template load<0>(kb, a.k_t, k0 + BK, end);
      if (!TURNS) st.template load<1>(vb, a.v_t, k0 + BK, end);
    }
#pragma unroll
    for (int b = 0; b < NKB; ++b) {
      if (TURNS && b == 1 && more) {
        st.template store<0>(nk);
        st.template load<1>(vb, a.v_t, k0 + BK, end);
      }
      f32x16 s = f32x16{0}, g = f32x16{0};
      if (sees) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          s = mma<T>(at_lane.frag(tk, b * 32, i), qf[i], s);
          g = mma<T>(at_lane.frag(tv, b * 32, i), gf[i], g);
        }
      }
      if (TURNS && NKB == 1 && more) {  // (a single half: the values follow behind the first two products)
        st.template store<0>(nk);
        st.template load<1>(vb, a.v_t, k0 + BK, end);
      }
      if (!sees) continue;
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        p[i] = exp2_fast(fmaf(s[i], a.c, -lse)) * (narrow<T>() ? fmaf(g[i], times, -delta) : g[i] - delta);
      if (EDGE && k0 + BK - 1 > wave_min) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + b * 32 + result_row(i, half) > pos) p[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Frag<T> pf = pack<T>(p + i * 8);
#pragma unroll
        for (int d = 0; d < NDB; ++d) acc[d] = mma<T>(at_lane.frag_t(tk, b * 32, i, d), pf, acc[d]);
      }
    }
    if (more) {
      if (!TURNS) st.template store<0>(nk);
      st.template store<1>(nk + TILE);
    }
    __syncthreads();
  };
  // tiles that every row of the workgroup sees whole, without a mask or a branch; then the others
  const int clear = min(tile_hi, ((a.causal ? t.tile * kRowTile / a.G : kv - 1) + 1) / BK);
  int kt = 0;
  for (; kt < clear; ++kt) step(kt, kt & 1, std::false_type());
  for (; kt < tile_hi; ++kt) step(kt, kt & 1, std::true_type());
  if (!live) return;
  T* po = static_cast<T*>(a.gq) + at * D;
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      store4<T>(po + d * 32 + result_row(i, half),
                f32x4{acc[d][i] * back, acc[d][i + 1] * back, acc[d][i + 2] * back, acc[d][i + 3] * back});
}

// dk, dv: a workgroup per (tile of keys, key head), a wavefront per 32 keys whose K and V rows stay in
// registers as right operands; Q and dO go through LDS with the rows' lse, D_r and positions beside them.
// S = Q K^T and dP = dO V^T have the rows in the registers, so P and dS are the right operands of
// dv^T = dO^T P and dk^T = Q^T dS as they stand.  Two of the four wavefronts share 32 keys and take
// alternate blocks of 32 rows, their sums meeting in LDS at the end: a tile of 64 keys, because the first
// keys of a causal sequence are seen by every row of the group and the longest tile is what the launch
// waits for (12 sequences of 195 - 2 048 tokens, 16 heads over 4 of 128, bf16: 439 us with tiles of 128, 373 with
// 64 when it was changed).  f32 with D = 128 has no registers for the larger row tile: four times 32 keys there.
// The 12 sequences take 198 - 218 us by card now, 410 - 450 TFLOP/s: 604 tiles on 256 CUs whose longest walks 128
// row tiles of 1.6 us, one wavefront a SIMD, LDS and the waits for it half of each; 3 sequences of 3 582 - 4 500,
// 16 heads of 64, f16, two wavefronts a SIMD: 268 - 274 us, 720 TFLOP/s.
template <typename T, int D>
constexpr int grad_rows() { return D * planes<T>() >= 384 ? 32 : 64; }
template <typename T, int D>
constexpr int grad_keys() { return 32 * 4 / (grad_rows<T, D>() / 32); }

template <typename T, int D>
__global__ __launch_bounds__(256, (D * planes<T>() >= 128 ? 1 : 2)) void attention_keys_backward_kernel(GradArgs a) {
  constexpr int BR = grad_rows<T, D>(), RG = BR / 32, KG = 4 / RG, CH = D / kChunk, NS = D / 16, NDB = D / 32;
  constexpr int PLANE = BR * D * 2, TILE = planes<T>() * PLANE, PER = BR * CH / 256, STEP = 256 / CH;
  constexpr bool TIGHT = D * planes<T>() >= 384, AHEAD = D * planes<T>() >= 128 && !TIGHT;
  __shared__ __align__(16) char lds[4 * TILE];
  __shared__ __align__(16) float s_lse[2][BR], s_delta[2][BR];
  __shared__ __align__(16) int s_pos[2][BR];
  __shared__ float s_most[4];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int h = blockIdx.x % a.Hkv;
  const int want = blockIdx.x / a.Hkv;  // the first keys are seen by the most rows: they go first
  const SeqTile t = find_tile(a.cu, a.N, a.total, 1, grad_keys<T, D>(), want, lane);
  const int Hq = a.Hkv * a.G;
  if (t.seq < 0) {
    if (h == 0) {
      clear_rows<T, D>(static_cast<T*>(a.gk), a.cu, a.N, a.total, a.Hkv, want - t.used, a.tiles - t.used);
      clear_rows<T, D>(static_cast<T*>(a.gv), a.cu, a.N, a.total, a.Hkv, want - t.used, a.tiles - t.used);
    }
    return;
  }
  const int tile0 = t.tile * grad_keys<T, D>(), key0 = tile0 + wv % KG * 32, key = key0 + (lane & 31);
  const bool live = key < t.len;
  Frag<T> kf[NS], vf[NS];
  {
    const T* kp = static_cast<const T*>(a.k) + (t.start + (live ? key : 0)) * a.k_t + h * a.k_h;
    const T* vp = static_cast<const T*>(a.v) + (t.start + (live ? key : 0)) * a.v_t + h * a.v_h;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = (2 * s + half) * kChunk;
      kf[s] = operand<T>(live ? load_raw<T>(reinterpret_cast<const char*>(kp + c)) : zero_raw<T>());
      vf[s] = operand<T>(live ? load_raw<T>(reinterpret_cast<const char*>(vp + c)) : zero_raw<T>());
    }
  }
  f32x16 gk[NDB], gv[NDB];
#pragma unroll
  for (int d = 0; d < NDB; ++d) gk[d] = gv[d] = f32x16{0};

  // Row tiles: `toks` whole tokens of G <= BR heads each, or BR heads of one token.  A thread's place in a
  // tile is then the same in every tile, and a tile's place is a scalar: no division in the loop.  (BR % G
  // rows of a tile stay empty: none for the usual groups of 1, 2, 4, 8; 1 of 64 for 3, 4 of 64 for 5.)
  const int toks = a.G <= BR ? BR / a.G : 1, segs = a.G <= BR ? 1 : (a.G + BR - 1) / BR;
  const int lo = a.causal ? tile0 / toks * segs : 0, hi = (t.len + toks - 1) / toks * segs;
  const int span = a.G <= BR ? a.G : BR;  // heads of a token in a tile
  auto place = [&](int j, int& tok, int& head) {
    tok = j / span, head = j - tok * span;
    if (tok >= toks) tok = 1 << 30;  // an empty row
  };
  auto at_of = [&](int tok, int head, int64_t s_t, int64_t s_h) {
    return (uint32_t)((tok * (int)s_t + head * (int)s_h) * (int)sizeof(T) + threadIdx.x % CH * (kChunk * (int)sizeof(T)));
  };
  uint32_t q_at[PER], g_at[PER];
  int tok_i[PER], head_i[PER], tok_s, head_s;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    place(threadIdx.x / CH + i * STEP, tok_i[i], head_i[i]);
    q_at[i] = at_of(min(tok_i[i], BR), head_i[i], a.q_t, a.q_h);
    g_at[i] = at_of(min(tok_i[i], BR), head_i[i], a.go_t, a.go_h);
  }
  place(threadIdx.x & (BR - 1), tok_s, head_s);
  const char* qb = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + t.start * a.q_t + (int64_t)h * a.G * a.q_h);
  const char* gb = reinterpret_cast<const char*>(static_cast<const T*>(a.go) + t.start * a.go_t + (int64_t)h * a.G * a.go_h);
  float times = 1.f, back_k = a.scale, back_v = 1.f;  // f16: the factors of dS (beyond P's) and what takes them out again
  Raw<T> qr[PER], gr[PER];
  float r_lse, r_delta;
  int r_pos;
  auto load = [&](int rt) {
    const int tok0 = segs == 1 ? rt * toks : rt / segs, head0 = segs == 1 ? 0 : (rt - tok0 * segs) * BR;
    const char* q0 = qb + (tok0 * a.q_t + head0 * a.q_h) * (int)sizeof(T);
    const char* g0 = gb + (tok0 * a.go_t + head0 * a.go_h) * (int)sizeof(T);
    const bool whole = toks * span == BR && tok0 + toks <= t.len && head0 + span <= a.G;
    if constexpr (TIGHT) {  // (320 registers hold operands and sums: none for a second set of offsets)
      if (whole) {
#pragma unroll
        for (int i = 0; i < PER; ++i) qr[i] = load_chunk<T>(q0, q_at[i]), gr[i] = load_chunk<T>(g0, g_at[i]);
      } else {
        rare();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          qr[i] = gr[i] = zero_raw<T>();
          if (tok_i[i] < t.len - tok0 && head0 + head_i[i] < a.G)
            qr[i] = load_chunk<T>(q0, q_at[i]), gr[i] = load_chunk<T>(g0, g_at[i]);
        }
      }
    } else {
      // An empty row reads the tile's last token's, which lies in the tile anyway (32-bit offsets hold within a tile, not
      // to the end of a long sequence), and gets the weight 0 by lse = inf: only offsets lie behind the branch.
      // (With loads on both of its ways, those met in a wait for all but the
      // last pair: 253 us against 217 on the 12 sequences.)
      uint32_t qo[PER], go[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) qo[i] = q_at[i], go[i] = g_at[i];
      if (!whole) {
        rare();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int tok = min(tok_i[i], min(toks, t.len - tok0) - 1), head = min(head_i[i], a.G - 1 - head0);
          qo[i] = at_of(tok, head, a.q_t, a.q_h), go[i] = at_of(tok, head, a.go_t, a.go_h);
        }
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) qr[i] = load_chunk<T>(q0, qo[i]), gr[i] = load_chunk<T>(g0, go[i]);
    }
    if (threadIdx.x < BR) {
      r_lse = INFINITY, r_delta = 0.f, r_pos = -1;
      if (tok_s < t.len - tok0 && head0 + head_s < a.G) {
        const int64_t at = (t.start + tok0 + tok_s) * Hq + h * a.G + head0 + head_s;
        r_lse = a.lse[at], r_delta = a.delta[at], r_pos = a.causal ? tok0 + tok_s : t.len - 1;
      }
    }
  };
  auto store = [&](int buf) {
    char* tq = lds + buf * 2 * TILE;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      store_chunk<T, D, PLANE>(tq, threadIdx.x / CH + i * STEP, threadIdx.x % CH, qr[i]);
      store_chunk<T, D, PLANE>(tq + TILE, threadIdx.x / CH + i * STEP, threadIdx.x % CH, gr[i]);
    }
    if (threadIdx.x < BR) {
      s_lse[buf][threadIdx.x] = narrow<T>() ? r_lse - kOrders : r_lse;
      s_delta[buf][threadIdx.x] = narrow<T>() ? r_delta * times : r_delta;
      s_pos[buf][threadIdx.x] = r_pos;
    }
  };
  load(lo);
  if constexpr (narrow<T>()) {
    float most = 0.f, value = 0.f;
    const float* norms = a.row_norm + (h * a.total + t.start) * a.G;
    for (int r = (a.causal ? tile0 * a.G / 32 + (int)threadIdx.x : (int)threadIdx.x) * 32; r < t.len * a.G; r += 256 * 32)
      most = fmaxf(most, norms[r]);
    for (int key = lane * kNormKeys; key < t.len; key += 64 * kNormKeys)
      value = fmaxf(value, a.value_norm[h * a.total + t.start + key]);
    most = wave_max(most);
    if (lane == 0) s_most[wv] = most;
    __syncthreads();
    most = fmaxf(fmaxf(s_most[0], s_most[1]), fmaxf(s_most[2], s_most[3]));
    const int order = order_of(most, wave_max(value));
    times = ldexpf(1.f, -order), back_k = ldexpf(a.scale, order - kOrders), back_v = ldexpf(1.f, -kOrders);
  }
  store(0);
  __syncthreads();
  const int b = wv / KG, own = b * 32 * D * 2;  // this wavefront's block of 32 rows of a tile
  const LaneAt<T, D, PLANE> at_lane(lane);
  auto step = [&](int rt, int buf, auto masked) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(masked)::value;
    const char* tq = lds + buf * 2 * TILE;
    const char* tg = tq + TILE;
    const bool more = rt + 1 < hi;
    if (more) load(rt + 1);
    // (every wavefront multiplies every block, masked ones too: a branch around the products makes the
    // compiler move the 128 accumulators between the register files in every iteration)
    // One wavefront a SIMD (AHEAD): nothing hides an LDS read but distance, so the fragments of the first products
    // are all requested before them, and those of the second ones' first half before the weights are formed.
    Frag<T> qa[NS], ga[NS], qt[NDB], gt[NDB];
    f32x4 lse[4], dl[4];
#pragma unroll
    for (int i = 0; i < NS; ++i) qa[i] = at_lane.frag(tq + own, 0, i), ga[i] = at_lane.frag(tg + own, 0, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lse[j] = *reinterpret_cast<const f32x4*>(&s_lse[buf][b * 32 + j * 8 + half * 4]);
      dl[j] = *reinterpret_cast<const f32x4*>(&s_delta[buf][b * 32 + j * 8 + half * 4]);
    }
    if (AHEAD) __builtin_amdgcn_sched_barrier(0);
    f32x16 s = f32x16{0}, g = f32x16{0};
#pragma unroll
    for (int i = 0; i < NS; ++i) s = mma<T>(qa[i], kf[i], s), g = mma<T>(ga[i], vf[i], g);
#pragma unroll
    for (int d = 0; d < NDB; ++d) gt[d] = at_lane.frag_t(tg + own, 0, 0, d), qt[d] = at_lane.frag_t(tq + own, 0, 0, d);
    if (AHEAD) __builtin_amdgcn_sched_barrier(0);
    float p[16], ds[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = exp2_fast(fmaf(s[i], a.c, -lse[i >> 2][i & 3]));
      ds[i] = p[i] * (narrow<T>() ? fmaf(g[i], times, -dl[i >> 2][i & 3]) : g[i] - dl[i >> 2][i & 3]);
    }
    if (EDGE) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key > s_pos[buf][b * 32 + result_row(i, half)]) p[i] = 0.f, ds[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Frag<T> pf = pack<T>(p + i * 8), df = pack<T>(ds + i * 8);
#pragma unroll
      for (int d = 0; d < NDB; ++d) {
        gv[d] = mma<T>(i ? at_lane.frag_t(tg + own, 0, i, d) : gt[d], pf, gv[d]);
        gk[d] = mma<T>(i ? at_lane.frag_t(tq + own, 0, i, d) : qt[d], df, gk[d]);
      }
    }
    if (more) store(buf ^ 1);
    __syncthreads();
  };
  // Only the first row tiles of a causal sequence need a mask: a row behind the last one has lse = inf, so
  // its weights are zeros, and a column behind the last key is not stored.
  const int masked = a.causal ? min(hi, (tile0 + grad_keys<T, D>() - 2 + toks) / toks * segs) : lo;
  int rt = lo;
  for (; rt < masked; ++rt) step(rt, (rt - lo) & 1, std::true_type());
  for (; rt < hi; ++rt) step(rt, (rt - lo) & 1, std::false_type());
  if constexpr (RG > 1) {  // the second half of the rows joins the first (the tiles are free by now)
    float* meet = reinterpret_cast<float*>(lds) + (int64_t)(wv % KG) * (NDB * 32 * 64) + lane;
    static_assert(KG * NDB * 32 * 64 * 4 <= sizeof(lds), "the sums of half the wavefronts fit the tiles");
    if (wv >= KG) {
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          meet[(d * 32 + i) * 64] = gk[d][i];
          meet[(d * 32 + 16 + i) * 64] = gv[d][i];
        }
    }
    __syncthreads();
    if (wv >= KG) return;
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        gk[d][i] += meet[(d * 32 + i) * 64];
        gv[d][i] += meet[(d * 32 + 16 + i) * 64];
      }
  }
  if (!live) return;
  T* pk = static_cast<T*>(a.gk) + ((t.start + key) * a.Hkv + h) * D;
  T* pv = static_cast<T*>(a.gv) + ((t.start + key) * a.Hkv + h) * D;
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int c = d * 32 + result_row(i, half);
      store4<T>(pk + c, f32x4{gk[d][i] * back_k, gk[d][i + 1] * back_k, gk[d][i + 2] * back_k, gk[d][i + 3] * back_k});
      store4<T>(pv + c, f32x4{gv[d][i] * back_v, gv[d][i + 1] * back_v, gv[d][i + 2] * back_v, gv[d][i + 3] * back_v});
    }
}

template <typename T, int D>
static void launch_rows(const RowsArgs& a, unsigned grid, hipStream_t st) {
  hipLaunchKernelGGL((attention_rows_kernel<T, D, false>), dim3(grid), dim3(256), 0, st, a);
}
template <typename T, int D>
static void launch_rows_backward(const GradArgs& a, unsigned grid, hipStream_t st) {
  if constexpr (narrow<T>()) {
    const int64_t tiles = (a.total + kNormKeys - 1) / kNormKeys + a.N;
    hipLaunchKernelGGL((attention_value_norms_kernel<T, D>), dim3((unsigned)(tiles * a.Hkv)), dim3(256), 0, st, a);
  }
  hipLaunchKernelGGL((attention_rows_backward_kernel<T, D>), dim3(grid), dim3(256), 0, st, a);
}
template <typename T, int D>
static void launch_keys_backward(GradArgs a, hipStream_t st) {
  a.tiles = (a.total + grad_keys<T, D>() - 1) / grad_keys<T, D>() + a.N + 1;
  hipLaunchKernelGGL((attention_keys_backward_kernel<T, D>), dim3((unsigned)(a.tiles * a.Hkv)), dim3(256), 0, st, a);
}

}  // namespace att
}  // namespace aps

using namespace aps;
using namespace aps::att;

// Tiles by cost where the card takes two to eight rounds of them (512 workgroups at two a CU).  The 12 sequences (1 248
// workgroups): forward 93.6 -> 86.0 us, dq 108 -> 101; the 3 (1 568): 149.7 -> 145.4 and 191 -> 183.  One round needs no
// order; over many rounds the ends even out, and neighbours of one sequence share its keys in the L2: 6 prompts
// (5 968) take 1 354 us in the sequences' order and 1 381 by cost.
static inline int tiles_by_cost(int32_t causal, int64_t N, unsigned grid) {
  return causal != 0 && N > 1 && N <= 64 && grid > 512 && grid <= 4096;
}

extern "C" int aps_attention_packed(const void* q, const void* k, const void* v, const void* cu_seqlens,
                                    int32_t cu_wide, void* out, void* out_rest, float* lse, int64_t total, int64_t N,
                                    int64_t Hq, int64_t Hkv, int64_t head_dim, int64_t q_t, int64_t q_h,
                                    int64_t k_t, int64_t k_h, int64_t v_t, int64_t v_h, int32_t dtype,
                                    int32_t causal, float scale, void* stream) {
  if (total == 0) return APS_OK;
  APS_CHECK_ARG(q && k && v && cu_seqlens && out && sizes_fit(total, N, Hq, Hkv) && scale_fits(scale));
  const int64_t e = dtype == kTypeF32 ? 4 : 8;
  APS_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(out_rest));
  APS_CHECK_ARG(strides_fit(q_t, q_h, e) && strides_fit(k_t, k_h, e) && strides_fit(v_t, v_h, e));
  RowsArgs a{};
  a.q = q, a.k = k, a.v = v, a.out = out, a.rest = dtype == kTypeF32 ? nullptr : out_rest, a.lse = lse;
  a.cu = Index{cu_seqlens, cu_wide};
  a.total = total, a.N = N;
  a.G = (int32_t)(Hq / Hkv), a.Hkv = (int32_t)Hkv;
  a.tiles = (total * a.G + kRowTile - 1) / kRowTile + N + 1;
  a.q_t = q_t, a.q_h = q_h, a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h;
  a.causal = causal != 0, a.zero_tail = 1, a.splits = 1;
  a.c = scale * kLog2e;
  const unsigned grid = (unsigned)(a.tiles * Hkv);
  a.by_cost = tiles_by_cost(causal, N, grid);
  hipStream_t st = static_cast<hipStream_t>(stream);
  APS_ATT_DISPATCH(launch_rows, a, grid, st);
  return aps_launch_status();
}

extern "C" int64_t aps_attention_packed_backward_workspace(int64_t total, int64_t Hq) {
  return total < 0 || Hq < 1 ? -1 : 3 * total * Hq * (int64_t)sizeof(float);
}

extern "C" int aps_attention_packed_backward(const void* q, const void* k, const void* v, const void* out,
                                             const void* out_rest, const void* g_out, const float* lse, const void* cu_seqlens,
                                             int32_t cu_wide, void* g_q, void* g_k, void* g_v, int64_t total,
                                             int64_t N, int64_t Hq, int64_t Hkv, int64_t head_dim, int64_t q_t,
                                             int64_t q_h, int64_t k_t, int64_t k_h, int64_t v_t, int64_t v_h,
                                             int64_t go_t, int64_t go_h, int32_t dtype, int32_t causal,
                                             float scale, void* workspace, void* stream) {
  if (total == 0) return APS_OK;
  APS_CHECK_ARG(q && k && v && out && g_out && lse && cu_seqlens && g_q && g_k && g_v && workspace);
  APS_CHECK_ARG(dtype == kTypeF32 || out_rest);
  APS_CHECK_ARG(sizes_fit(total, N, Hq, Hkv) && scale_fits(scale));
  const int64_t e = dtype == kTypeF32 ? 4 : 8;
  APS_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(out_rest) && aligned16(g_out));
  APS_CHECK_ARG(aligned16(g_q) && aligned16(g_k) && aligned16(g_v));
  APS_CHECK_ARG(strides_fit(q_t, q_h, e) && strides_fit(k_t, k_h, e) && strides_fit(v_t, v_h, e));
  APS_CHECK_ARG(strides_fit(go_t, go_h, e));
  GradArgs a{};
  a.q = q, a.k = k, a.v = v, a.o = out, a.rest = out_rest, a.go = g_out, a.lse = lse;
  a.delta = static_cast<float*>(workspace), a.row_norm = a.delta + total * Hq, a.value_norm = a.row_norm + total * Hq;
  a.gq = g_q, a.gk = g_k, a.gv = g_v;
  a.cu = Index{cu_seqlens, cu_wide};
  a.total = total, a.N = N;
  a.G = (int32_t)(Hq / Hkv), a.Hkv = (int32_t)Hkv;
  a.q_t = q_t, a.q_h = q_h, a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h, a.go_t = go_t, a.go_h = go_h;
  a.causal = causal != 0, a.scale = scale, a.c = scale * kLog2e;
  hipStream_t st = static_cast<hipStream_t>(stream);
  a.tiles = (total * a.G + kRowTile - 1) / kRowTile + N + 1;
  const unsigned grid = (unsigned)(a.tiles * Hkv);
  a.by_cost = tiles_by_cost(causal, N, grid);
  APS_ATT_DISPATCH(launch_rows_backward, a, grid, st);
  if (aps_launch_status() != APS_OK) return APS_ERR_LAUNCH;
  APS_ATT_DISPATCH(launch_keys_backward, a, st);
  return aps_launch_status();
}
