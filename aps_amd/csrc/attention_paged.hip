// Attention of new tokens over a paged key / value cache, and the write of their keys and values into
// it.  Pages [P, page, Hkv, D] hold the keys (values) of `page` consecutive positions of one sequence;
// table[n, j] is the page of positions j * page ... of sequence n.  The new tokens of sequence n are
// the last of its kv_lens[n] positions: query i of L sits at kv_lens[n] - L + i and sees the keys up to
// there.
//
// Two kernels share the work.  Many rows per key head (a row: a token and a head of the group): the
// 128-row kernel of attention_rows.h with page lookups.  Few rows (single tokens): the cache is read
// once and that is all that counts -- `attention_decode_kernel` below.  Either splits the keys over
// workgroups when there are few tiles; the partial results meet in a second launch, in split order.
#include "attention_rows.h"

namespace aps {
namespace att {

template <typename T>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mma16<__bf16>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma16<_Float16>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma16<float>(u32x4 a, u32x4 b, f32x4 c) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
  return c;
}

// element e of a run of values held as 32-bit words
template <typename T>
__device__ __forceinline__ float value_at(const uint32_t* w, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
  else return (float)__builtin_bit_cast(T, (uint16_t)((e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffff));
}

// A workgroup owns 16 R rows of one (sequence, key head) and a range of its keys; each of its four
// wavefronts walks that range in chunks of 32 keys with a softmax of its own, straight from global
// memory to the matrix operands: no LDS, no barrier until the four meet at the end.
//   S^T = K Q^T: 16 keys x 16 rows, a lane's 16-byte chunk of a key row is its operand.
//   O^T = V^T P^T: lane (g = lane / 16, c = lane % 16) reads elements c D/16 .. of the 8 keys
//   {4 g + i, 16 + 4 g + i} -- the keys whose weights it holds -- and regroups the 16-bit values by key
//   pairs in registers; the e-th product then holds elements {c' D/16 + e} of the output.
// 64 (16-bit, D = 128) registers of loads are in flight per wavefront, which with two wavefronts on a
// SIMD covers the latency of the memory; the matrix work of a 16-row tile is below the load time for
// every type (f32, the slowest: 2 048 cycles per 16 KB on a SIMD, 8 TB/s need 5 000).
// Measured: 16 contexts of 1 367 - 16 000 keys, 32 heads over 8 of 128, bf16: 124 us for 588 MB, 4.7 TB/s (a large
// copy: 5.07); 16 of 4 000, 8 heads of 64: 26 us for 131 MB (f32: 49 for 262 MB).
constexpr int kDecodeChunk = 32, kDecodeLeast = 8;  // keys a step; steps a split has at least

template <typename T, int D, int R>
__global__ __launch_bounds__(256, (sizeof(T) * D * R >= 1024 ? 1 : 2)) void attention_decode_kernel(RowsArgs a) {
  constexpr int E = vec_elems<T>(), NS = D / (4 * E), VE = D / 16, VB = VE * (int)sizeof(T), VW = VB / 4;
  constexpr int ROWS = 16 * R;
  __shared__ __align__(16) float s_o[4][ROWS][D + 4];
  __shared__ float s_m[4][ROWS], s_l[4][ROWS];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
  const int h = blockIdx.x % a.Hkv;
  const int want = blockIdx.x / a.Hkv;
  const SeqTile t = find_tile(a.cu, a.N, a.total, a.G, ROWS, want, lane);
  const int Hq = a.Hkv * a.G;
  if (t.seq < 0) {
    if (a.zero_tail && h == 0 && blockIdx.y == 0)
      clear_rows<T, D>(static_cast<T*>(a.out), a.cu, a.N, a.total, Hq, want - t.used, a.tiles - t.used);
    return;
  }
  const int off = first_position(a.kv_lens, t.seq, t.len, a.max_keys), kv = max(clipped(off, t.len, (int)a.max_keys), 0);
  const int rows = t.len * a.G, row0 = t.tile * ROWS;
  const int end = clipped(off, (min(row0 + ROWS, rows) - 1) / a.G + 1, kv);
  const int least = clipped(off, row0 / a.G, kv - 1);  // the tile's first position: keys up to it need no mask
  int pos[R];
  u32x4 qf[R][NS];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + r * 16 + c;
    const bool live = row < rows;
    const int tok = live ? row / a.G : 0, head = h * a.G + (live ? row - tok * a.G : 0);
    pos[r] = live ? clipped(off, tok, kv - 1) : -1;
    const T* qp = static_cast<const T*>(a.q) + (t.start + tok) * a.q_t + head * a.q_h;
#pragma unroll
    for (int s = 0; s < NS; ++s)
      qf[r][s] = live ? *reinterpret_cast<const u32x4*>(qp + (s * 4 + g) * E) : u32x4{0, 0, 0, 0};
  }
  const int chunks = (max(end, 0) + kDecodeChunk - 1) / kDecodeChunk;
  int lo = 0, hi = chunks;
  if (a.splits > 1) {
    const int use = min(a.splits, (chunks + kDecodeLeast - 1) / kDecodeLeast);
    const int per = use > 0 ? (chunks + use - 1) / use : 0;
    lo = min(chunks, per * (int)blockIdx.y);
    hi = min(chunks, lo + per);
  }
  f32x4 acc[R][VE];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[r][e] = f32x4{0};
  }
  const int32_t* table = a.table + (int64_t)t.seq * a.table_stride;
  // The table's entry for key (lane % 32) of a chunk is asked for a chunk ahead and not looked at before its turn (memory
  // answers in order: before this chunk's loads are asked for, or it would wait for them too)
  auto page_of = [&](int chunk) { return table[min(chunk * kDecodeChunk + (lane & 31), end - 1) >> a.page_shift]; };
  int32_t next = lo + wv < hi ? page_of(lo + wv) : -1;
  for (int ch = lo + wv; ch < hi; ch += 4) {
    // slot of key (lane % 32); -1 past the end or for a page outside the cache (which has < 2^31 slots)
    const int key = ch * kDecodeChunk + (lane & 31);
    const int slot = key >= end || next < 0 || next >= a.num_pages
                         ? -1 : (next << a.page_shift) + (key & ((1 << a.page_shift) - 1));
    next = page_of(ch + 4);
    u32x4 kf[2][NS];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int row = __shfl(slot, b * 16 + c, 64);
      const T* kp = static_cast<const T*>(a.k) + (int64_t)row * a.k_t + h * a.k_h;
#pragma unroll
      for (int s = 0; s < NS; ++s)
        kf[b][s] = row >= 0 ? *reinterpret_cast<const u32x4*>(kp + (s * 4 + g) * E) : u32x4{0, 0, 0, 0};
    }
    uint32_t vr[8][VW];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int row = __shfl(slot, (j >> 2) * 16 + g * 4 + (j & 3), 64);
      const T* vp = static_cast<const T*>(a.v) + (int64_t)row * a.v_t + h * a.v_h + c * VE;
      if constexpr (VW >= 4) {
#pragma unroll
        for (int w = 0; w < VW / 4; ++w) {
          const u32x4 x = row >= 0 ? reinterpret_cast<const u32x4*>(vp)[w] : u32x4{0, 0, 0, 0};
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[j][w * 4 + e] = x[e];
        }
      } else if constexpr (VW == 2) {
        const u32x2 x = row >= 0 ? *reinterpret_cast<const u32x2*>(vp) : u32x2{0, 0};
        vr[j][0] = x.x, vr[j][1] = x.y;
      } else {
        vr[j][0] = row >= 0 ? *reinterpret_cast<const uint32_t*>(vp) : 0u;
      }
    }
    const int k0 = ch * kDecodeChunk;
    // (a chunk past `end` or with a missing page is masked, so its zeros carry no weight)
    const bool mask = k0 + kDecodeChunk - 1 > least || __any(slot < 0);
    if (mask) {
      // Some row may not see all of the chunk, and 0 * infinity is not 0: a non-finite value is taken out of the
      // products and added to the rows that see it (element c VE + e belongs to lanes 4 g + i = c)
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < VE; ++e) bad |= !finite(value_at<T>(vr[j], e));
      if (__any(bad)) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float x = value_at<T>(vr[j], e);
            if (!finite(x)) {
              if constexpr (sizeof(T) == 2) vr[j][e >> 1] &= (e & 1) ? 0xffffu : 0xffff0000u;
              else vr[j][e] = 0;
            }
            for (uint64_t left = __ballot(!finite(x)); left; left &= left - 1) {
              const int from = __builtin_ctzll(left), fg = from >> 4, fc = from & 15;
              const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), from));
              const int key = k0 + (j >> 2) * 16 + fg * 4 + (j & 3);
#pragma unroll
              for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (g * 4 + i == fc && key <= pos[r]) acc[r][e][i] += v;
            }
          }
      }
    }
    // V by element: 16-bit, va[e] = element e of the 8 keys
    u32x4 va[VE];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = vr[2 * j][e >> 1], y = vr[2 * j + 1][e >> 1];
          va[e][j] = (e & 1) ? __builtin_amdgcn_perm(y, x, 0x07060302) : __builtin_amdgcn_perm(y, x, 0x05040100);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      f32x4 s[2] = {f32x4{0}, f32x4{0}};
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) s[b] = mma16<T>(kf[b][i], qf[r][i], s[b]);
      if (mask) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool there = __shfl(slot, b * 16 + g * 4 + i, 64) >= 0;
            if (!there || k0 + b * 16 + g * 4 + i > pos[r]) s[b][i] = -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[b][i]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64)) * a.c;
      if (__any(top > m[r] + 8.f)) {
        const float to = top > m[r] + 8.f ? top : m[r];
        const float f = m[r] == -INFINITY ? 1.f : exp2_fast(m[r] - to);
        m[r] = to;
        l[r] *= f;
#pragma unroll
        for (int e = 0; e < VE; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][e][i] *= f;
      }
      const float ref = m[r] == -INFINITY ? 0.f : m[r];
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = exp2_fast(fmaf(s[i >> 2][i & 3], a.c, -ref));
        l[r] += p[i];
      }
      if constexpr (sizeof(T) == 2) {
        const Frag<T> pf = pack<T>(p);
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[r][e] = mma16<T>(va[e], pf.p[0], acc[r][e]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < VE; ++e)
            acc[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[j][e]), p[j], acc[r][e], 0, 0, 0);
      }
    }
  }
  // the four wavefronts' results meet: register i of acc[e] is element (4 g + i) VE + e of row c
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] += __shfl_xor(l[r], 16, 64);
    l[r] += __shfl_xor(l[r], 32, 64);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e) s_o[wv][r * 16 + c][(g * 4 + i) * VE + e] = acc[r][e][i];
    if (g == 0) s_m[wv][r * 16 + c] = m[r], s_l[wv][r * 16 + c] = l[r];
  }
  __syncthreads();
  constexpr int PER = D / 4;  // threads a row
  for (int i = threadIdx.x; i < ROWS * PER; i += 256) {
    const int r = i / PER, d = (i % PER) * 4, row = row0 + r;
    if (row >= rows) continue;
    const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    f32x4 o = f32x4{0};
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = top == -INFINITY ? 0.f : exp2_fast(s_m[w][r] - top);
      const f32x4 x = *reinterpret_cast<const f32x4*>(&s_o[w][r][d]);
      sum += f * s_l[w][r];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += f * x[e];
    }
    const int tok = row / a.G;
    const int64_t at = (t.start + tok) * Hq + h * a.G + row - tok * a.G;
    if (a.splits > 1) {
      const int64_t slot = (int64_t)blockIdx.y * a.total * Hq + at;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + slot * 2) = make_float2(top, sum);
      if (sum != 0.f) store4<float>(a.part_o + slot * D + d, o);
      continue;
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    store4<T>(static_cast<T*>(a.out) + at * D + d, f32x4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv});
  }
}

// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s, D / 4 threads a row; rows behind the last
// sequence are not touched
template <typename T, int D>
__global__ __launch_bounds__(256) void attention_combine_kernel(RowsArgs a) {
  constexpr int PER = D / 4;
  const int Hq = a.Hkv * a.G, d = (threadIdx.x % PER) * 4;
  const int64_t row = (int64_t)blockIdx.x * (256 / PER) + threadIdx.x / PER, all = a.total * Hq;
  if (row >= tail_of(a.cu, a.N, a.total) * Hq) return;
  int s0, e0;
  seq_range(a.cu, 0, a.total, s0, e0);
  if (row < (int64_t)s0 * Hq) return;  // rows before the first sequence belong to none either
  // eight splits at a time, their loads in flight together
  float top = -INFINITY, sum = 0.f;
  f32x4 o = f32x4{0};
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    float2 ml[8];
    f32x4 x[8];
    float to = top;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ml[j] = make_float2(-INFINITY, 0.f);
      if (s0 + j < a.splits) ml[j] = *reinterpret_cast<const float2*>(a.part_ml + ((s0 + j) * all + row) * 2);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = f32x4{0};
      if (ml[j].y != 0.f) x[j] = *reinterpret_cast<const f32x4*>(a.part_o + ((s0 + j) * all + row) * D + d);
      to = fmaxf(to, ml[j].x);
    }
    const float f0 = to == -INFINITY ? 0.f : exp2_fast(top - to);
    sum *= f0;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= f0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = ml[j].y == 0.f ? 0.f : exp2_fast(ml[j].x - to);
      sum += f * ml[j].y;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += f * x[j][e];
    }
    top = to;
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  store4<T>(static_cast<T*>(a.out) + row * D + d, f32x4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv});
}

struct AppendArgs {
  const void *k, *v;
  void *k_pages, *v_pages;
  Index cu, kv_lens;
  const int32_t* table;
  int64_t table_stride, total, N, k_t, k_h, v_t, v_h, num_pages, max_keys, chunks;
  int32_t page_shift, Hkv, head_chunks, elems;  // 16-byte chunks of a head, elements of a chunk
  int32_t elem_bytes;
};

// one 16-byte chunk of a new token's keys and of its values per thread; the token's sequence by
// bisection over the starts
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  const int per = a.Hkv * a.head_chunks;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.chunks) return;
  const int64_t tok = i / per;
  const int at = (int)(i - tok * per), h = at / a.head_chunks, c = at - h * a.head_chunks;
  int64_t lo = 0, hi = a.N;  // the last sequence that starts at or before the token
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (a.cu.at(mid) <= tok) lo = mid;
    else hi = mid;
  }
  int start, end;
  seq_range(a.cu, lo, a.total, start, end);
  if (tok < start || tok >= end) return;
  const int64_t pos = (int64_t)first_position(a.kv_lens, lo, end - start, a.max_keys) + (tok - start);
  if (pos < 0 || pos >= a.max_keys) return;
  const int32_t p = a.table[lo * a.table_stride + (pos >> a.page_shift)];
  if (p < 0 || p >= a.num_pages) return;
  const int64_t slot = ((int64_t)p << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
  const int64_t to = (slot * per + at) * 16;
  const char* k = static_cast<const char*>(a.k) + (tok * a.k_t + h * a.k_h + c * a.elems) * a.elem_bytes;
  const char* v = static_cast<const char*>(a.v) + (tok * a.v_t + h * a.v_h + c * a.elems) * a.elem_bytes;
  *reinterpret_cast<u32x4*>(static_cast<char*>(a.k_pages) + to) = *reinterpret_cast<const u32x4*>(k);
  *reinterpret_cast<u32x4*>(static_cast<char*>(a.v_pages) + to) = *reinterpret_cast<const u32x4*>(v);
}

// Which kernel and how many splits, from what the host knows (the lengths themselves are on the
// device): form 1 / 2 = decode tiles of 16 / 32 rows, 0 = 128-row tiles; one for the whole call, the same for every
// type.
struct PagedPlan { int form; int64_t tiles; int splits; };

static PagedPlan paged_plan(int64_t total, int64_t N, int64_t G, int64_t Hkv, int64_t max_keys) {
  PagedPlan p;
  const int64_t mean = (total * G + N - 1) / N;  // rows of a sequence and key head
  // (16 x 2 000 keys, rows of 128: 32 rows of bf16 / f32 take 16 / 28 us in decode tiles and 20 / 42 in 128-row
  // tiles; 64 rows over 4 000 keys of 64: 48 / 147 us against 44 / 118)
  p.form = mean <= 16 ? 1 : (mean <= 32 ? 2 : 0);
  const int64_t tile = p.form == 1 ? 16 : (p.form == 2 ? 32 : kRowTile);
  p.tiles = (total * G + tile - 1) / tile + N + 1;
  const int64_t busy = ((total * G + tile - 1) / tile > N ? (total * G + tile - 1) / tile : N) * Hkv;
  // Workgroups to aim for.  Decode: the lengths differ, so twice what the chip holds evens them out (16 contexts of
  // 1 367 - 16 000 keys, 8 key heads of 128, bf16: 131 us with 1 024, 126 with 2 048, 125 with 4 096 and 4 us
  // more in the second launch).  128-row tiles: 1 024 (8 chunks over up to 4 096 keys: 68 us with 256).
  const int64_t target = p.form ? 2048 : 1024;
  const int64_t least = p.form ? kDecodeChunk * kDecodeLeast : 256;
  int64_t s = (target + busy - 1) / busy, most = (max_keys + least - 1) / least;
  if (s > most) s = most;
  p.splits = (int)(s < 1 ? 1 : (s > 128 ? 128 : s));
  return p;
}

template <typename T, int D>
static void launch_paged(const RowsArgs& a, const PagedPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.tiles * a.Hkv), (unsigned)p.splits);
  if (p.form == 1)
    hipLaunchKernelGGL((attention_decode_kernel<T, D, 1>), grid, dim3(256), 0, st, a);
  else if (p.form == 2)
    hipLaunchKernelGGL((attention_decode_kernel<T, D, 2>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attention_rows_kernel<T, D, true>), grid, dim3(256), 0, st, a);
  if (p.splits > 1) {
    constexpr int per = 256 / (D / 4);
    const int64_t blocks = (a.total * a.Hkv * a.G + per - 1) / per;
    hipLaunchKernelGGL((attention_combine_kernel<T, D>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  }
}

}  // namespace att
}  // namespace aps

using namespace aps;
using namespace aps::att;

static bool paged_sizes_fit(int64_t total, int64_t N, int64_t Hq, int64_t Hkv, int64_t num_pages, int64_t page,
                            int64_t width) {
  return sizes_fit(total, N, Hq, Hkv) && total * Hq < (int64_t)0x7fffffff * 8 && page >= 1 && page <= 65536 &&
         (page & (page - 1)) == 0 && num_pages >= 1 && num_pages <= (int64_t)0x7fff0000 / page && width >= 1 && width <= (int64_t)0x7fff0000 / page;
}

static inline bool apart(const void* p, int64_t p_bytes, const void* q, int64_t q_bytes) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return a + (uint64_t)p_bytes <= b || b + (uint64_t)q_bytes <= a;
}

extern "C" int64_t aps_attention_paged_workspace(int64_t total, int64_t N, int64_t Hq, int64_t Hkv,
                                                 int64_t head_dim, int64_t page, int64_t width, int32_t) {
  if (!paged_sizes_fit(total, N, Hq, Hkv, 1, page, width)) return -1;
  const PagedPlan p = paged_plan(total, N, Hq / Hkv, Hkv, width * page);
  return p.splits > 1 ? p.splits * total * Hq * (head_dim + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int aps_attention_paged(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                                   const void* cu_seqlens, int32_t cu_wide, const void* kv_lens, int32_t kv_wide,
                                   void* out, int64_t total, int64_t N, int64_t Hq, int64_t Hkv, int64_t head_dim,
                                   int64_t num_pages, int64_t page, int64_t width, int64_t table_stride, int64_t q_t,
                                   int64_t q_h, int32_t dtype, float scale, int32_t keep_tail, void* workspace,
                                   void* stream) {
  if (total == 0) return APS_OK;
  APS_CHECK_ARG(q && k_pages && v_pages && page_table && cu_seqlens && kv_lens && out && scale_fits(scale));
  APS_CHECK_ARG(paged_sizes_fit(total, N, Hq, Hkv, num_pages, page, width) && table_stride >= width);
  const int64_t e = dtype == kTypeF32 ? 4 : 8;
  APS_CHECK_ARG(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out));
  APS_CHECK_ARG(strides_fit(q_t, q_h, e));
  RowsArgs a{};
  a.q = q, a.k = k_pages, a.v = v_pages, a.out = out;
  a.cu = Index{cu_seqlens, cu_wide}, a.kv_lens = Index{kv_lens, kv_wide};
  a.table = page_table, a.table_stride = table_stride;
  a.total = total, a.N = N;
  a.G = (int32_t)(Hq / Hkv), a.Hkv = (int32_t)Hkv;
  a.q_t = q_t, a.q_h = q_h;
  a.k_t = a.v_t = Hkv * head_dim, a.k_h = a.v_h = head_dim;
  a.num_pages = num_pages, a.max_keys = width * page, a.page_shift = __builtin_ctzll((uint64_t)page);
  a.causal = 1, a.zero_tail = keep_tail == 0, a.c = scale * kLog2e;
  const PagedPlan p = paged_plan(total, N, a.G, Hkv, a.max_keys);
  APS_CHECK_ARG(p.tiles * Hkv < 0x7fffffff);
  a.tiles = p.tiles, a.splits = p.splits;
  if (p.splits > 1) {
    APS_CHECK_ARG(workspace && aligned16(workspace));
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (int64_t)p.splits * total * Hq * head_dim;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  APS_ATT_DISPATCH(launch_paged, a, p, st);
  return aps_launch_status();
}

extern "C" int aps_paged_append(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* page_table,
                                const void* cu_seqlens, int32_t cu_wide, const void* kv_lens, int32_t kv_wide,
                                int64_t total, int64_t N, int64_t Hkv, int64_t head_dim, int64_t num_pages,
                                int64_t page, int64_t width, int64_t table_stride, int64_t k_t, int64_t k_h,
                                int64_t v_t, int64_t v_h, int32_t dtype, void* stream) {
  if (total == 0) return APS_OK;
  APS_CHECK_ARG(k && v && k_pages && v_pages && page_table && cu_seqlens && kv_lens);
  APS_CHECK_ARG(paged_sizes_fit(total, N, Hkv, Hkv, num_pages, page, width) && table_stride >= width);
  if (dtype < kTypeF32 || dtype > kTypeF16 || (head_dim != 32 && head_dim != 64 && head_dim != 128))
    return APS_ERR_UNSUPPORTED;
  const int64_t e = dtype == kTypeF32 ? 4 : 8;
  APS_CHECK_ARG(aligned16(k) && aligned16(v) && aligned16(k_pages) && aligned16(v_pages));
  APS_CHECK_ARG(strides_fit(k_t, k_h, e) && strides_fit(v_t, v_h, e));
  // (slots that one launch reads and writes, or writes twice, would hold what came last)
  const int64_t bytes = 16 / e, held = num_pages * page * Hkv * head_dim * bytes;
  const int64_t of_k = ((total - 1) * k_t + (Hkv - 1) * k_h + head_dim) * bytes;
  const int64_t of_v = ((total - 1) * v_t + (Hkv - 1) * v_h + head_dim) * bytes;
  APS_CHECK_ARG(apart(k_pages, held, v_pages, held));
  APS_CHECK_ARG(apart(k, of_k, k_pages, held) && apart(k, of_k, v_pages, held));
  APS_CHECK_ARG(apart(v, of_v, k_pages, held) && apart(v, of_v, v_pages, held));
  AppendArgs a{};
  a.k = k, a.v = v, a.k_pages = k_pages, a.v_pages = v_pages;
  a.cu = Index{cu_seqlens, cu_wide}, a.kv_lens = Index{kv_lens, kv_wide};
  a.table = page_table, a.table_stride = table_stride, a.total = total, a.N = N;
  a.k_t = k_t, a.k_h = k_h, a.v_t = v_t, a.v_h = v_h, a.num_pages = num_pages, a.max_keys = width * page;
  a.page_shift = __builtin_ctzll((uint64_t)page), a.Hkv = (int32_t)Hkv;
  a.head_chunks = (int32_t)(head_dim / e), a.elems = (int32_t)e, a.elem_bytes = (int32_t)(16 / e);
  a.chunks = total * Hkv * a.head_chunks;
  const int64_t blocks = (a.chunks + 255) / 256;
  APS_CHECK_ARG(blocks < 0x7fffffff);
  hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return aps_launch_status();
}
