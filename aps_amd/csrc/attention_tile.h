// Pieces shared by the packed and the paged attention kernels (attention_packed.hip,
// attention_paged.hip): matrix fragments of 16-byte chunks, the swizzled LDS tile they are read from,
// and the search of a workgroup's tile in a batch of sequences packed end to end.
//
// One formulation serves bf16, f16 and f32.  A tile in LDS is row-major with rows of D 16-bit elements cut
// into chunks of 8 (16 bytes); a matrix step contracts over two chunks: lanes 0-31 of the 32x32x16 MFMA hold
// the even one, lanes 32-63 the odd one.  The 32x32 result holds column = lane % 32 and rows
// (i / 4) * 8 + (lane / 32) * 4 + i % 4 in register i; registers 8 s .. 8 s + 7 are therefore the B operand of
// the s-th step of a product that contracts over those rows, provided the A operand takes its contraction
// index in the same order (`LaneAt::frag_t`): no lane exchange lies between the two products of a tile.
//
// f32 runs on the same pipe as three bf16 planes, x = h + m + l: h the upper 16 bits (finite for every finite
// x), m and l what is left, each rounded to bf16, the sum exact to 2^-25 |x|.  Of the nine plane products six
// are formed, h h + (h m + m h) + (h l + l h + m m), smallest first, in f32; the three left out are below
// 2^-22 |x y| together, as is usual of an f32 product sum.  Any exponent is kept (no scaling); an infinity
// makes what it is multiplied into NaN.  Six 16-bit MFMAs of 32 cycles stand for eight f32 ones of 64 (32x32x2,
// 16 deep): 8 sequences of 1 400 - 1 500 tokens, 8 heads of 64, causal, forward and gradients 775 us where the f32
// instructions took 1 160 (head size 128: 1 640 against 2 566).  Now 614 (1 166), the forward pass 140 (265): 122 - 129
// TFLOP/s, where a sixth of the library's large bf16 product is 193 - 216; the rest is splitting P and the softmax.
#ifndef APS_AMD_ATTENTION_TILE_H_
#define APS_AMD_ATTENTION_TILE_H_

#include "common.h"

#include <type_traits>

namespace aps {
namespace att {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

enum { kTypeF32 = 0, kTypeBf16 = 1, kTypeF16 = 2 };

template <typename T>
constexpr int vec_elems() { return 16 / (int)sizeof(T); }  // elements of 16 bytes in memory
constexpr int kChunk = 8;                                   // elements of a chunk of a tile
template <typename T>
constexpr int planes() { return sizeof(T) == 4 ? 3 : 1; }

template <typename T>
struct Vec;
template <>
struct Vec<__bf16> { typedef bf16x4 v4; typedef bf16x8 v8; };
template <>
struct Vec<_Float16> { typedef f16x4 v4; typedef f16x8 v8; };

// 8 elements as they lie in memory / as matrix operand
template <typename T>
struct Raw { u32x4 v[sizeof(T) / 2]; };
template <typename T>
struct Frag { u32x4 p[planes<T>()]; };

template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const char* at) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const u32x4*>(at)[i];
  return r;
}
template <typename T>
__device__ __forceinline__ Raw<T> zero_raw() {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = u32x4{0, 0, 0, 0};
  return r;
}

// 8 floats as three planes
__device__ __forceinline__ Frag<float> split8(const float* x) {
  bf16x8 m, l;
  u32x4 h;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = __float_as_uint(x[2 * i]), b = __float_as_uint(x[2 * i + 1]);
    h[i] = __builtin_amdgcn_perm(b, a, 0x07060302);
    const float ra = x[2 * i] - __uint_as_float(a & 0xffff0000u), rb = x[2 * i + 1] - __uint_as_float(b & 0xffff0000u);
    m[2 * i] = (__bf16)ra, m[2 * i + 1] = (__bf16)rb;
    l[2 * i] = (__bf16)(ra - (float)m[2 * i]), l[2 * i + 1] = (__bf16)(rb - (float)m[2 * i + 1]);
  }
  return Frag<float>{{h, __builtin_bit_cast(u32x4, m), __builtin_bit_cast(u32x4, l)}};
}

template <typename T>
__device__ __forceinline__ Frag<T> operand(const Raw<T>& r) {
  if constexpr (sizeof(T) == 2) {
    return Frag<T>{{r.v[0]}};
  } else {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r.v[i >> 2][i & 3]);
    return split8(x);
  }
}

__device__ __forceinline__ f32x16 mma_bf16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ f32x16 mma(const Frag<T>& a, const Frag<T>& b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 mma<__bf16>(const Frag<__bf16>& a, const Frag<__bf16>& b, f32x16 c) {
  return mma_bf16(a.p[0], b.p[0], c);
}
template <>
__device__ __forceinline__ f32x16 mma<_Float16>(const Frag<_Float16>& a, const Frag<_Float16>& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a.p[0]), __builtin_bit_cast(f16x8, b.p[0]), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mma<float>(const Frag<float>& a, const Frag<float>& b, f32x16 c) {
  c = mma_bf16(a.p[0], b.p[2], c);
  c = mma_bf16(a.p[2], b.p[0], c);
  c = mma_bf16(a.p[1], b.p[1], c);
  c = mma_bf16(a.p[0], b.p[1], c);
  c = mma_bf16(a.p[1], b.p[0], c);
  return mma_bf16(a.p[0], b.p[0], c);
}

// 8 registers of a result as an operand.  16-bit types: one rounding, of at most 2^-8 (bf16) / 2^-11 (f16) of each number, as
// the result's own.  A second plane for what it takes away would cost half as many products again.  The weights lie
// in [0, 1] up to a common factor and their sum is kept from the unrounded values; over many keys the roundings average
// out, but a result that one rounding alone would leave 1.7e-3 off (bf16, norm) is 2.0e-3 - 2.4e-3 off, and 2.1e-4
// becomes 2.8e-4 - 3.0e-4 in f16.  f16 weights below 2^-14 of the reference (at most the row's largest) keep 2^-25 of it;
// the gradients, whose size is the caller's, are scaled first (attention_packed.hip).
template <typename T>
__device__ __forceinline__ Frag<T> pack(const float* p) {
  if constexpr (sizeof(T) == 2) {
    typename Vec<T>::v8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)p[e];
    return Frag<T>{{__builtin_bit_cast(u32x4, v)}};
  } else {
    return split8(p);
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 v) {
  if constexpr (sizeof(T) == 2) {
    typename Vec<T>::v4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
    *reinterpret_cast<u32x2*>(p) = __builtin_bit_cast(u32x2, o);
  } else {
    *reinterpret_cast<f32x4*>(p) = v;
  }
}

// sum of the products of 8 elements
template <typename T>
__device__ __forceinline__ float dot_raw(const Raw<T>& a, const Raw<T>& b) {
  float s = 0.f;
  if constexpr (sizeof(T) == 2) {
    const typename Vec<T>::v8 x = __builtin_bit_cast(typename Vec<T>::v8, a.v[0]);
    const typename Vec<T>::v8 y = __builtin_bit_cast(typename Vec<T>::v8, b.v[0]);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (float)x[e] * (float)y[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) s += __uint_as_float(a.v[e >> 2][e & 3]) * __uint_as_float(b.v[e >> 2][e & 3]);
  }
  return s;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028234663852886e38f; }

// 8 elements with the non-finite ones zeroed (`any` set if there were some)
template <typename T>
__device__ __forceinline__ Raw<T> only_finite(Raw<T> r, bool& any) {
  // an exponent of ones: infinity or NaN
  constexpr uint32_t one = sizeof(T) == 4 ? 0x7f800000u : (__is_same(T, __bf16) ? 0x7f80u : 0x7c00u);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t v = r.v[i][w];
      if constexpr (sizeof(T) == 4) {
        if ((v & one) == one) v = 0, any = true;
      } else {
        if ((v & one) == one) v &= 0xffff0000u, any = true;
        if ((v & (one << 16)) == one << 16) v &= 0xffffu, any = true;
      }
      r.v[i][w] = v;
    }
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

// Chunk c of row r lies at chunk position c ^ swizzle(r).  The masks make both reads of a tile touch
// every LDS bank once: 16 lanes reading one chunk of 16 rows (row fragments), and 16 lanes reading 32
// bytes of 4 rows (transposing read).
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (D >= 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  if constexpr (D == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  return (r >> 2) & 3;
}

// byte offset of chunk c of row r
template <int D>
__device__ __forceinline__ int tile_at(int r, int c) {
  return r * (D * 2) + ((c ^ swizzle<D>(r)) << 4);
}

// Where a lane's fragments lie, from a tile's first byte (planes PLANE bytes apart).  The swizzle depends on a
// row's last four bits, so 32 rows (16 for the transposing read) further on is a constant to the instruction's
// offset, and so is another plane.
//   row fragment, step s: row lane % 32, chunk 2 s + lane / 32
//   transposed fragment:  ds_read_b64_tr_b16: within 16 lanes, lane j points at 4 elements of row j / 4 and
//                         receives column j of the 4 x 16 block
template <typename T, int D, int PLANE>
struct LaneAt {
  static constexpr int NS = D / 16, NDB = D / 32, PITCH = D * 2;
  int f[NS], t[NDB][2];

  __device__ __forceinline__ explicit LaneAt(int l) {
    const int half = l >> 5;
#pragma unroll
    for (int s = 0; s < NS; ++s) f[s] = tile_at<D>(l & 31, 2 * s + half);
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int hi = 0; hi < 2; ++hi)
        t[db][hi] = tile_at<D>(half * 4 + ((l & 15) >> 2) + hi * 8, db * 4 + ((l >> 4) & 1) * 2 + ((l & 3) >> 1)) +
                    (l & 1) * 8;
  }
  // rows row0 .. row0 + 31 (a multiple of 32)
  __device__ __forceinline__ Frag<T> frag(const char* tile, int row0, int s) const {
    Frag<T> r;
#pragma unroll
    for (int p = 0; p < planes<T>(); ++p)
      r.p[p] = *reinterpret_cast<const u32x4*>(tile + p * PLANE + row0 * PITCH + f[s]);
    return r;
  }
  // column db * 32 + lane % 32 of the 16 rows that registers 8 s .. 8 s + 7 of a 32x32 result stand for
  __device__ __forceinline__ Frag<T> frag_t(const char* tile, int row0, int s, int db) const {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    Frag<T> r;
#pragma unroll
    for (int p = 0; p < planes<T>(); ++p) {
      const char* at = tile + p * PLANE + (row0 + s * 16) * PITCH;
      const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + t[db][0])));
      const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + t[db][1])));
      r.p[p] = u32x4{a.x, a.y, b.x, b.y};
    }
    return r;
  }
};

// 8 elements to a tile
template <typename T, int D, int PLANE>
__device__ __forceinline__ void store_chunk(char* tile, int row, int c, const Raw<T>& r) {
  const Frag<T> f = operand<T>(r);
#pragma unroll
  for (int p = 0; p < planes<T>(); ++p) *reinterpret_cast<u32x4*>(tile + p * PLANE + tile_at<D>(row, c)) = f.p[p];
}

// Wait for every global load.  Said before a loop where its operands have arrived anyway on the way that is
// taken: the compiler, which sees another way, else waits in the loop, for the loop's own loads too.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// In a branch that is seldom taken: keeps the compiler from turning it into selects that every tile pays for
__device__ __forceinline__ void rare() { asm volatile(""); }

// A chunk at a byte offset from a base that is the same for the whole wavefront: the load takes the base
// from scalar registers, and a loop that steps the base adds nothing per lane.  (Strides are at most
// kMaxStride bytes, so 128 rows stay within the 32-bit offset.)
constexpr int64_t kMaxStride = 1 << 23;
template <typename T>
__device__ __forceinline__ Raw<T> load_chunk(const char* base, uint32_t offset) { return load_raw<T>(base + offset); }

// row of a 32x32 result that register i of a lane holds
__device__ __forceinline__ int result_row(int i, int half) { return (i >> 2) * 8 + half * 4 + (i & 3); }

// int32 or int64 index arrays (cu_seqlens, kv_lens)
struct Index {
  const void* p;
  int32_t wide;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return wide ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
  }
};

struct SeqTile {
  int seq;        // -1: no tile of this number
  int tile;       // tile within the sequence
  int64_t start;  // first token of the sequence
  int len;        // its tokens
  int64_t used;   // seq == -1: tiles there are in all
};

// tokens [start, end) of sequence n, whatever the array holds: inside [0, total), never negative (token
// numbers fit 31 bits: sizes_fit)
__device__ __forceinline__ void seq_range(const Index& cu, int64_t n, int64_t total, int& start, int& end) {
  const int64_t a = cu.at(n), b = cu.at(n + 1);
  start = (int)(a < 0 ? 0 : (a > total ? total : a));
  end = b < start ? start : (int)(b > total ? total : b);
}

// Tile number `want` of the batch: every sequence of L tokens has ceil(L * per / rows) tiles.  Each
// wavefront scans the lengths 64 at a time (no shared memory, no barrier); the whole block gets the
// same answer.
__device__ __forceinline__ SeqTile find_tile(const Index& cu, int64_t N, int64_t total, int per, int rows,
                                             int want, int lane) {
  int64_t base = 0;  // (64 bits: sequences that overlap, which they must not, count more tiles than there are)
  for (int64_t n0 = 0; n0 < N; n0 += 64) {
    int s = 0, e = 0;
    if (n0 + lane < N) seq_range(cu, n0 + lane, total, s, e);
    const int len = e - s, tiles = (int)(((uint32_t)len * (uint32_t)per + rows - 1) / (uint32_t)rows);
    int upto = tiles;
    const int most = N - n0 < 64 ? (int)(N - n0) : 64;
    for (int o = 1; o < most; o <<= 1) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    const uint64_t beyond = __ballot(base + upto > want && tiles > 0);
    if (beyond) {
      const int at = __builtin_ctzll(beyond);
      SeqTile t;
      t.seq = (int)n0 + at;
      t.tile = (int)(want - base) - __builtin_amdgcn_readlane(upto - tiles, at);
      t.len = __builtin_amdgcn_readlane(len, at);
      t.start = __builtin_amdgcn_readlane(s, at);
      t.used = 0;
      return t;
    }
    base += __builtin_amdgcn_readlane(upto, 63 < most - 1 ? 63 : most - 1);
  }
  return SeqTile{-1, 0, 0, 0, base};
}

// The sum over the wavefront of numbers 0 <= v < 2^bits, by one ballot a bit
__device__ __forceinline__ int sum_by_bits(int v, int bits) {
  int sum = 0;
  for (int b = 0; b < bits; ++b) sum += __builtin_popcountll(__ballot((v >> b) & 1)) << b;
  return sum;
}

// The same tiles, those with the highest number within their sequence first: tile i of a causal sequence sees the keys
// up to its own, so that is the order of their cost, and the launch does not end on a long one.  N <= 64.
__device__ __forceinline__ SeqTile find_tile_by_cost(const Index& cu, int N, int64_t total, int per, int rows, int want,
                                                     int lane) {
  int s = 0, e = 0;
  if (lane < N) seq_range(cu, lane, total, s, e);
  const int len = e - s, tiles = (int)(((uint32_t)len * (uint32_t)per + rows - 1) / (uint32_t)rows);
  int most = 1;  // 2^bits > tiles of any sequence
  int bits = 0;
  while (__ballot(tiles >= most)) most <<= 1, ++bits;
  const int all = sum_by_bits(tiles, bits);
  if (want >= all) return SeqTile{-1, 0, 0, 0, all};
  // the largest number `lo` such that more than `want` tiles have it or a higher one
  int lo = 0, hi = most, above = 0;  // above: tiles numbered `hi` or higher
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, n = sum_by_bits(max(tiles - mid, 0), bits);
    if (n > want) lo = mid;
    else hi = mid, above = n;
  }
  const uint64_t have = __ballot(tiles > lo);
  const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0));
  const int at = __builtin_ctzll(__ballot(tiles > lo && before == want - above));
  SeqTile t;
  t.seq = at, t.tile = lo, t.used = 0;
  t.len = __builtin_amdgcn_readlane(len, at);
  t.start = __builtin_amdgcn_readlane(s, at);
  return t;
}

// first token behind the last sequence
__device__ __forceinline__ int64_t tail_of(const Index& cu, int64_t N, int64_t total) {
  const int64_t e = cu.at(N);
  return e < 0 ? 0 : (e > total ? total : e);
}

}  // namespace att
}  // namespace aps
#endif  // APS_AMD_ATTENTION_TILE_H_
