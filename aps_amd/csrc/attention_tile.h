// Pieces shared by the packed and the paged attention kernels (attention_packed.hip,
// attention_paged.hip): matrix fragments of 16-byte chunks, the swizzled LDS tile they are read from,
// and the search of a workgroup's tile in a batch of sequences packed end to end.
//
// One formulation serves bf16, f16 and f32.  A tile in LDS is row-major with rows of D elements cut
// into 16-byte chunks (8 or 4 elements); a matrix step contracts over KS = two chunks (16 or 8
// elements): lanes 0-31 hold the even chunk, lanes 32-63 the odd one.  16-bit types: one 32x32x16
// MFMA; f32: four 32x32x2 MFMAs, element e of both chunks in the e-th (exact fp32 products).
// The 32x32 result holds column = lane % 32 and rows (i / 4) * 8 + (lane / 32) * 4 + i % 4 in register
// i; registers s * KS / 2 .. (s + 1) * KS / 2 - 1 are therefore the B operand of the s-th step of a
// product that contracts over those rows, provided the A operand takes its contraction index in the
// same order (`frag_t`): no lane exchange lies between the two products of an attention tile.
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
constexpr int chunk_elems() { return 16 / (int)sizeof(T); }

template <typename T>
struct Vec;
template <>
struct Vec<__bf16> { typedef bf16x4 v4; typedef bf16x8 v8; };
template <>
struct Vec<_Float16> { typedef f16x4 v4; typedef f16x8 v8; };

template <typename T>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 mma<__bf16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mma<_Float16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mma<float>(u32x4 a, u32x4 b, f32x16 c) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
  return c;
}

// registers p[0 .. KS/2) of a result as an operand chunk (one rounding to the 16-bit type: the weights
// lie in [0, 1] up to a common factor, so the rounding is 2^-9 / 2^-12 of each weight; sums over
// many keys average it out, and the softmax's own sum is kept from the unrounded values)
template <typename T>
__device__ __forceinline__ u32x4 pack(const float* p) {
  if constexpr (sizeof(T) == 2) {
    typename Vec<T>::v8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)p[e];
    return __builtin_bit_cast(u32x4, v);
  } else {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = p[e];
    return __builtin_bit_cast(u32x4, v);
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

// sum of the products of two chunks
template <typename T>
__device__ __forceinline__ float dot_chunk(u32x4 a, u32x4 b) {
  float s = 0.f;
  if constexpr (sizeof(T) == 2) {
    const typename Vec<T>::v8 x = __builtin_bit_cast(typename Vec<T>::v8, a);
    const typename Vec<T>::v8 y = __builtin_bit_cast(typename Vec<T>::v8, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (float)x[e] * (float)y[e];
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) s += x[e] * y[e];
  }
  return s;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028234663852886e38f; }

// element e of a chunk / the chunk with its non-finite elements zeroed (`any` set if there were some)
template <typename T>
__device__ __forceinline__ float chunk_at(u32x4 v, int e) {
  if constexpr (sizeof(T) == 2) return (float)__builtin_bit_cast(typename Vec<T>::v8, v)[e];
  else return __builtin_bit_cast(f32x4, v)[e];
}
template <typename T>
__device__ __forceinline__ u32x4 only_finite(u32x4 v, bool& any) {
  // an exponent of ones: infinity or NaN
  constexpr uint32_t one = sizeof(T) == 4 ? 0x7f800000u : (__is_same(T, __bf16) ? 0x7f80u : 0x7c00u);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (sizeof(T) == 4) {
      if ((v[w] & one) == one) v[w] = 0, any = true;
    } else {
      if ((v[w] & one) == one) v[w] &= 0xffff0000u, any = true;
      if ((v[w] & (one << 16)) == one << 16) v[w] &= 0xffffu, any = true;
    }
  }
  return v;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

// Chunk c of row r lies at chunk position c ^ swizzle(r).  The masks make both reads of a tile touch
// every LDS bank once: 16 lanes reading one chunk of 16 rows (row fragments), and 16 lanes reading 32
// bytes of 4 rows for the transposing read (16-bit) / rows r and r + 4 of one 128-byte run (f32).
template <typename T, int D>
__device__ __forceinline__ int swizzle(int r) {
  constexpr int CH = D / chunk_elems<T>();
  if constexpr (sizeof(T) == 2) {
    if constexpr (CH >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    if constexpr (CH == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    return (r >> 2) & 3;
  } else {
    if constexpr (CH >= 16) return (r & 3) | (((r >> 2) & 1) << 3) | (((r >> 3) & 1) << 2);
    return (r >> 1) & 7;
  }
}

// byte offset of chunk c of row r
template <typename T, int D>
__device__ __forceinline__ int tile_at(int r, int c) {
  return r * (D * (int)sizeof(T)) + ((c ^ swizzle<T, D>(r)) << 4);
}

// Where a lane's fragments lie, from a tile's first byte.  The swizzle depends on a row's last four bits, so
// 32 rows (16 for the 16-bit transposing read) further on is a constant to the instruction's offset, and so
// is the other buffer: the loops below run over both buffers in turn, unrolled, and add nothing per read.
//   row fragment, step s:         row lane % 32, chunk 2 s + lane / 32
//   transposed fragment (16-bit): ds_read_b64_tr_b16: within 16 lanes, lane j points at 4 elements of row
//                                 j / 4 and receives column j of the 4 x 16 block
template <typename T, int D>
struct LaneAt {
  static constexpr int NS = D / (2 * chunk_elems<T>()), NDB = D / 32, PITCH = D * (int)sizeof(T);
  int f[NS], t[sizeof(T) == 2 ? NDB : 1][2], lane;

  __device__ __forceinline__ explicit LaneAt(int l) : lane(l) {
    const int half = l >> 5;
#pragma unroll
    for (int s = 0; s < NS; ++s) f[s] = tile_at<T, D>(l & 31, 2 * s + half);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int hi = 0; hi < 2; ++hi)
          t[db][hi] = tile_at<T, D>(half * 4 + ((l & 15) >> 2) + hi * 8, db * 4 + ((l >> 4) & 1) * 2 + ((l & 3) >> 1)) +
                      (l & 1) * 8;
    }
  }
  // rows row0 .. row0 + 31 (a multiple of 32)
  __device__ __forceinline__ u32x4 frag(const char* tile, int row0, int s) const {
    return *reinterpret_cast<const u32x4*>(tile + row0 * PITCH + f[s]);
  }
  // column db * 32 + lane % 32 of the KS rows that registers s * KS / 2 .. of a 32x32 result stand for
  __device__ __forceinline__ u32x4 frag_t(const char* tile, int row0, int s, int db) const {
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4* lds_ptr;
      const char* p = tile + (row0 + s * 16) * PITCH;
      const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + t[db][0])));
      const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + t[db][1])));
      return u32x4{a.x, a.y, b.x, b.y};
    } else {
      const int d = db * 32 + (lane & 31);
      u32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = row0 + s * 8 + (lane >> 5) * 4 + e;
        v[e] = *reinterpret_cast<const uint32_t*>(tile + tile_at<T, D>(r, d >> 2) + (d & 3) * 4);
      }
      return v;
    }
  }
};

// In a branch that is seldom taken: keeps the compiler from turning it into selects that every tile pays for
__device__ __forceinline__ void rare() { asm volatile(""); }

// A chunk at a byte offset from a base that is the same for the whole wavefront: the load takes the base
// from scalar registers, and a loop that steps the base adds nothing per lane.  (Strides are at most
// kMaxStride bytes, so 128 rows stay within the 32-bit offset.)
constexpr int64_t kMaxStride = 1 << 23;
__device__ __forceinline__ u32x4 load_chunk(const char* base, uint32_t offset) {
  return *reinterpret_cast<const u32x4*>(base + offset);
}

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
  int used;       // seq == -1: tiles there are in all
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
  int base = 0;
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
      t.tile = want - base - __builtin_amdgcn_readlane(upto - tiles, at);
      t.len = __builtin_amdgcn_readlane(len, at);
      t.start = __builtin_amdgcn_readlane(s, at);
      t.used = 0;
      return t;
    }
    base += __builtin_amdgcn_readlane(upto, 63 < most - 1 ? 63 : most - 1);
  }
  return SeqTile{-1, 0, 0, 0, base};
}

// first token behind the last sequence
__device__ __forceinline__ int64_t tail_of(const Index& cu, int64_t N, int64_t total) {
  const int64_t e = cu.at(N);
  return e < 0 ? 0 : (e > total ? total : e);
}

}  // namespace att
}  // namespace aps
#endif  // APS_AMD_ATTENTION_TILE_H_
