// Element types, 16-byte row pieces and the 8-bit checkpoint format, shared by the kernels of
// norm_fwd.hip and norm_bwd.hip (group norm), ckpt8.hip (checkpoint write / read) and wgrad8.hip (weight gradients).
//
// Checkpoint format.  A row of C values is cut into blocks of 32 consecutive channels.  A block
// holds one byte s and a signed code per value, value = code * 2^(s - 127), where e = s - 127 is the
// least integer >= -126 with max|x| <= 127 * 2^e and code = x / 2^e rounded to nearest, ties to
// even: off by at most 2^(e-1), which is under max|x| / 127 unless e = -126.  At e = 122 (max|x| over
// 127 * 2^121, within 1 % of the largest float) codes end at 63, since 64 * 2^122 is no float: off by at most
// 2^122.  A power of two as the scale keeps every step exact: x / 2^e is an exponent shift, and code * 2^e
// has at most 7 significant bits and is a value of bfloat16, of float and (inside its range) of half.  A block
// with an infinity or a NaN has s = 255 and codes 0 and reads as NaN throughout; s = 0, never written, reads as 0.
// Codes of a row take ld = 16 * ceil(C / 16) bytes (the tail is zero) so that every row can be read
// in 16-byte pieces; scales take ceil(C / 32) bytes.
#pragma once
#include "gvae_common.h"

namespace gvae {

constexpr int kBlock8 = 32;
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
inline int ckpt8_ld(int C) { return (C + 15) / 16 * 16; }
inline int ckpt8_blocks(int C) { return (C + kBlock8 - 1) / kBlock8; }

// Consecutive work-groups are handed to the eight XCDs in turn.  This numbers them so that each XCD takes a
// run of neighbours, which then share what they read (and lines that they write parts of) in its L2.
__device__ __forceinline__ int xcd_run(unsigned id, unsigned total) {
  const unsigned xcd = id & 7, q = total >> 3, r = total & 7;
  return (int)(xcd * q + (xcd < r ? xcd : r) + (id >> 3));
}

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// a 16-byte piece of a row, at the alignment of its element (the hardware takes any)
template <class T>
struct Piece {
  static constexpr int V = 16 / (int)sizeof(T);
  typedef T raw __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef raw mem __attribute__((aligned(sizeof(T))));
};

// The elements [c0, c0 + nv) of rows of C, zero behind them, nv in 1..V.  Fewer than V are cut out of a
// whole piece that lies in the row, in two steps: every load of a thread can be on its way before the
// first is cut (a cut beside its load waits for it).  Against elements one by one, group norm backward:
// 300 graphs of 50 rows, 60 channels in groups of 3, bf16 19.0 -> 15.1 us; 37 graphs of 777 rows, 45 channels
// in groups of 5, half 18.8 -> 16.6.
typedef unsigned __int128 bits128;
template <class T>
struct Cut {
  typedef typename Piece<T>::raw raw;
  static constexpr int V = Piece<T>::V, kBits = 8 * (int)sizeof(T);
  int c0, nv, C, off;
  __device__ __forceinline__ Cut(int c0, int nv, int C) : c0(c0), nv(nv), C(C), off(c0 < C - V ? c0 : C - V) {}
  __device__ __forceinline__ raw load(const T *row) const {
    if (C >= V) return *reinterpret_cast<const typename Piece<T>::mem *>(row + off);
    raw r;
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = v < nv ? row[c0 + v] : (T)0.0f;
    return r;
  }
  __device__ __forceinline__ void cut(raw &r) const {
    if (nv == V || C < V) return;
    r = __builtin_bit_cast(raw, (__builtin_bit_cast(bits128, r) >> (kBits * (c0 - off))) &
                                    (~(bits128)0 >> (kBits * (V - nv))));
  }
};
// A piece held over several passes of a kernel: between two passes the compiler must not keep its
// values converted to float (twice the registers for 16-bit types) instead of converting again.
template <class T>
__device__ __forceinline__ void keep_raw(typename Piece<T>::raw &r) {
  if (sizeof(T) == 4) return;
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  words w = __builtin_bit_cast(words, r);
  asm volatile("" : "+v"(w));
  r = __builtin_bit_cast(typename Piece<T>::raw, w);
}

// Results of this size or more are stored past the caches (nontemporal): they would not stay there for
// their reader, and what is still to be read would make room for them.  Measured: group norm of 192 graphs of
// 1000 rows, 512 channels, bf16 (197 MB) 111 -> 104 us, its backward 215 -> 203; 4 graphs of 65536 rows,
// 320 channels 111 -> 99; a few MB are the same or 5 % slower.
constexpr int64_t kPastCaches = 64LL << 20;

template <bool PAST, class T>
__device__ __forceinline__ void store_piece(T *p, const float *f, int nv) {
  constexpr int V = Piece<T>::V;
  typename Piece<T>::raw r;
#pragma unroll
  for (int v = 0; v < V; ++v) r[v] = (T)f[v];
  if (nv == V) {
    if (PAST) __builtin_nontemporal_store(r, reinterpret_cast<typename Piece<T>::mem *>(p));
    else *reinterpret_cast<typename Piece<T>::mem *>(p) = r;
    return;
  }
  // (nv in binary: up to three stores)
  bits128 w = __builtin_bit_cast(bits128, r);
  auto part = [&](auto kind) {
    typedef decltype(kind) word __attribute__((aligned(sizeof(T))));
    *reinterpret_cast<word *>(p) = (word)w;
    p += sizeof(word) / sizeof(T);
    w >>= 8 * sizeof(word);
  };
  if (sizeof(T) == 2) {
    if (nv & 4) part((uint64_t)0);
    if (nv & 2) part((uint32_t)0);
    if (nv & 1) part((uint16_t)0);
  } else {
    if (nv & 2) part((uint64_t)0);
    if (nv & 1) part((uint32_t)0);
  }
}

// the values as they are stored
template <class T>
struct rounded {
  float f[Piece<T>::V];
  __device__ __forceinline__ explicit rounded(const float *y) {
#pragma unroll
    for (int v = 0; v < Piece<T>::V; ++v) f[v] = (float)(T)y[v];
  }
  __device__ __forceinline__ operator const float *() const { return f; }
};

__device__ __forceinline__ float pow2_field(uint32_t field) { return __uint_as_float(field << 23); }

// max over the 2, 4 or 8 neighbouring lanes that share a block (lane groups aligned to their size)
template <int W>
__device__ __forceinline__ uint32_t lanes_max(uint32_t m) {
  static_assert(W == 1 || W == 2 || W == 4 || W == 8, "lanes of a block");
  if (W >= 2) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));
  if (W >= 4) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));
  // (mirror within 8 lanes: by now each half of four holds one value)
  if (W >= 8) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, false));
  return m;
}

// The scale byte of a block from the largest bit pattern of |x| in it: with |x| = 1.M * 2^(E-127),
// 127 * 2^e reaches it for e = E - 133 as long as 1.M <= 127/64, and for e = E - 132 always.
__device__ __forceinline__ uint32_t scale_byte(uint32_t absmax) {
  if (absmax >= 0x7f800000u) return 255u;
  const int s = (int)(absmax >> 23) - 6 + ((absmax & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return (uint32_t)(s < 1 ? 1 : s);
}

// V codes to their place (of the nc left in the row)
template <bool PAST, int V>
__device__ __forceinline__ void put_codes(const uint32_t *w, int8_t *codes, int nc) {
  if (nc < V) return;
  typedef uint32_t words __attribute__((ext_vector_type(V / 4)));
  words x;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) x[q] = w[q];
  if (PAST) __builtin_nontemporal_store(x, reinterpret_cast<words *>(codes));
  else *reinterpret_cast<words *>(codes) = x;
}
// V values of a row's block, spread over W = 32 / V neighbouring lanes that all make this call:
// codes to `codes` (ld bytes a row, nc of this lane's places inside it) and the block's byte.
// Places behind the last channel are given as 0.  Five instructions a value (ten with a rounding, two
// limits and a shift of its own each): group norm of 192 ragged graphs of 1000 rows, 512 channels, bf16, with
// two checkpoints, second pass 114 -> 101 us.
template <bool PAST, int V>
__device__ __forceinline__ void emit8(const float *f, int8_t *codes, int nc, uint8_t *scale, bool first) {
  uint32_t m = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) m = max(m, __float_as_uint(f[v]) & 0x7fffffffu);
  m = lanes_max<kBlock8 / V>(m);
  const uint32_t s = scale_byte(m);
  // Adding 1.5 * 2^23 rounds to an integer, ties to even, whose low byte is the code's; the product before it
  // is exact.  (|x| / 2^e is at most 127; at 2^122, where 64 steps are no float any more, at most 63)
  constexpr float kShift = 12582912.0f;
  const float lim = s == 249u ? 63.0f : 127.0f;
  const float inv = s == 255u ? 0.0f : pow2_field(254u - s);
  uint32_t w[V / 4];
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    uint32_t c[4];
#pragma unroll
    for (int v = 0; v < 4; ++v)
      c[v] = __float_as_uint(__builtin_amdgcn_fmed3f(__fmaf_rn(f[4 * q + v], inv, kShift), kShift - lim, kShift + lim));
    const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
    w[q] = s == 255u ? 0u : lo | hi;
  }
  put_codes<PAST, V>(w, codes, nc);
  if (first) *scale = (uint8_t)s;
}
// the same for values that are all 0
template <bool PAST, int V>
__device__ __forceinline__ void emit8_zeros(int8_t *codes, int nc, uint8_t *scale, bool first) {
  const uint32_t w[V / 4] = {};
  put_codes<PAST, V>(w, codes, nc);
  if (first) *scale = (uint8_t)scale_byte(0);
}

// V codes at `codes` (aligned to V bytes) times their block's power of two
template <int V>
struct Codes {
  uint32_t w[V / 4];
};
template <int V>
__device__ __forceinline__ Codes<V> load_codes(const int8_t *codes) {
  Codes<V> r;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) r.w[q] = reinterpret_cast<const uint32_t *>(codes)[q];
  return r;
}
template <int V>
__device__ __forceinline__ void decode8(const Codes<V> &c, float p, float *f) {
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = (float)(int8_t)(c.w[v >> 2] >> (8 * (v & 3))) * p;
}

#define GVAE_DTYPE_SWITCH(dtype, T, ...)                                  \
  switch (dtype) {                                                       \
    case GVAE_F32: { typedef float T; __VA_ARGS__; } break;              \
    case GVAE_BF16: { typedef gvae::bf16_t T; __VA_ARGS__; } break;      \
    default: { typedef gvae::f16_t T; __VA_ARGS__; } break;              \
  }

inline int dtype_bytes(int dtype) { return dtype == GVAE_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype >= GVAE_F32 && dtype <= GVAE_F16; }

}  // namespace gvae
