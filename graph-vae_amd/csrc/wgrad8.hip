// Weight and bias gradient of a linear layer y = x W^T + b from the 8-bit checkpoint of its input:
//   dW[o,i] = sum_t dY[t,o] * code[t,i] * 2^(s[t,i/32] - 127),   db[o] = sum_t dY[t,o]
//
// On the matrix cores in bf16 without a rounding of either factor: code * 2^e has 7 significant bits
// and is a bf16 value as it stands; a gradient is cut into bf16 pieces that add up to it, one for bf16 (8
// significant bits), two for half (11), three for float (24), each multiplied in turn.  The matrix cores keep
// subnormal pieces, so that bf16 and half enter exactly throughout and float from 2^-110 on; of a smaller
// float what lies below 2^-133, the least bf16 number, is dropped.  Sums are fp32 (v_mfma_f32_32x32x16_bf16).
//
// Both factors lie with the summed axis outermost in memory, so a lane's eight consecutive rows of
// one column are a column of the tile: tiles are staged row by row in LDS and read through
// the transposing ds_read_b64_tr_b16 (a group of 16 lanes reads 4 rows x 16 columns and gets 4 rows
// of one column each).  Those 4 rows are brought to different banks by XORing the 64-byte piece of a
// row with bits of its row number.
//
// 65536 rows, 2048 x 2048, bf16: 468 us on one card, 498 on another (medians of 400 calls) and 13 for the sums
// of its parts, 1080 to 1140 TFLOP/s.  The products and their reads from LDS alone take 390 us of it on random
// numbers (less on zeros: the clock gives way to the power drawn), conversions and stores to LDS the rest.
// Half and float pay for each piece of a gradient with a whole product: 50001 rows, 515 x 387, half 75 us (and
// 10 for its sums) in 128 x 256 tiles that cover 1.64 times dW.
//
// A work-group owns a tile of dW and a range of rows; the parts are summed in their order by a second
// launch.  Column sums of dY ride along: among the work-groups that share a dY tile, each adds up its
// share of the row steps.
#include "gvae_ckpt8.h"

namespace gvae {

struct WgradArgs {
  const void *dy;
  const int8_t *codes;
  const uint8_t *scales;
  void *dw, *db;
  float *part, *part_b;       // (splits, O, ldp) and (splits * tx, O)
  int64_t rows, ldy;
  int O, I, ldp, ld8, nb8, splits, tx, ty;
  int64_t split_rows;
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <class T> struct Pieces;
template <> struct Pieces<bf16_t> { static constexpr int P = 1; };
template <> struct Pieces<f16_t> { static constexpr int P = 2; };
template <> struct Pieces<float> { static constexpr int P = 3; };

// A finite value into P > 1 bf16 pieces that add up to it (to its multiple of 2^-133), each the upper half of a
// float.  An infinity stays in the first; a NaN may lie in the second alone (the first is then an infinity).
template <int P>
__device__ __forceinline__ void cut(float x, uint32_t *out) {
  out[0] = __float_as_uint(x);
  float r = x - __uint_as_float(out[0] & 0xffff0000u);
  r = fabsf(x) == __builtin_inff() ? 0.0f : r;
#pragma unroll
  for (int p = 1; p < P; ++p) {
    out[p] = __float_as_uint(r);
    r -= __uint_as_float(out[p] & 0xffff0000u);
  }
}
// the upper halves of two floats
__device__ __forceinline__ uint32_t upper_halves(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}

// What the 64-byte piece of a row is XORed with in a tile of W columns: four rows that are read together
// then lie in different banks (256 bytes of them; two rows of 64 columns fill those already).
template <int W>
__device__ __forceinline__ int swizzle(int k) {
  static_assert(W == 64 || W % 128 == 0, "pieces of a row");
  return W == 64 ? (k >> 1) & 1 : k & 3;
}
// byte offset of column c (a multiple of 8) of row k
template <int W>
__device__ __forceinline__ int tile_at(int k, int c) {
  return k * (2 * W) + (((c >> 5) ^ swizzle<W>(k)) << 6) + 2 * (c & 31);
}

// FM x FN matrix-core tiles of 32 x 32 per wavefront, WM x WN wavefronts, KT rows per step
template <class T, int FM, int FN, int WM, int WN, int KT>
struct Wgrad {
  static constexpr int P = Pieces<T>::P, V = Piece<T>::V;
  static constexpr int TM = 32 * FM * WM, TN = 32 * FN * WN, NT = 64 * WM * WN;
  static constexpr int kBytesA = KT * TM * 2, kBytesB = KT * TN * 2;
  static constexpr int kStage = P * kBytesA + kBytesB;
  static constexpr int NA = KT * TM / (V * NT), NB = KT * TN / (16 * NT);   // pieces of a thread per step
  static_assert(NA * V * NT == KT * TM && NB * 16 * NT == KT * TN && NB >= 1, "tile and threads");
};

template <class T, int FM, int FN, int WM, int WN, int KT>
__global__ __launch_bounds__(64 * WM * WN, 2) void wgrad8_kernel(WgradArgs a) {
  using S = Wgrad<T, FM, FN, WM, WN, KT>;
  constexpr int P = S::P, V = S::V, TM = S::TM, TN = S::TN, NT = S::NT;
  extern __shared__ __align__(16) char lds[];
  // (the tiles of one row range are neighbours: they share that range in an XCD's L2)
  const int id = xcd_run(blockIdx.x, gridDim.x);
  const int tiles = a.tx * a.ty, split = id / tiles, tile = id - split * tiles;
  const int ix = tile % a.tx, i0 = ix * TN, o0 = (tile / a.tx) * TM;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
  const int64_t t0 = (int64_t)split * a.split_rows;
  const int64_t t1 = t0 + a.split_rows < a.rows ? t0 + a.split_rows : a.rows;

  typename Piece<T>::raw ra[S::NA];
  uint4 rb[S::NB];
  uint32_t rs[S::NB];
  float bias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = 0.0f;

  // A thread's pieces: always the same columns, rows k = first + j * step.  Columns behind the last are
  // read from the first one instead: they end up in columns of the tile that are not stored.
  constexpr int CA = TM / V, CB = TN / 16;
  const int ca = (tid % CA) * V, ka = tid / CA, cb = (tid % CB) * 16, kb = tid / CB;
  const int nva = a.O - (o0 + ca) < V ? a.O - (o0 + ca) : V;
  const int cola = nva > 0 ? o0 + ca : 0, colb = i0 + cb < a.ld8 ? i0 + cb : 0;
  const T *dy = (const T *)a.dy + t0 * a.ldy;
  const int8_t *codes = a.codes + t0 * a.ld8;
  const uint8_t *scales = a.scales + t0 * a.nb8;
  // 32-bit offsets from the step's first row; a piece's distance from the first is the same for all threads
  const uint32_t va = (uint32_t)ka * (uint32_t)a.ldy + cola, vb = (uint32_t)kb * (uint32_t)a.ld8 + colb;
  const uint32_t vs = (uint32_t)kb * (uint32_t)a.nb8 + colb / kBlock8;
  // Steps of whole rows run with unconditional loads (their waits then count loads and not worst cases).  A
  // last piece of a row may run into the row behind it; the steps with the last row of all, and those
  // that are not full, take guarded loads.
  const int64_t own_rows = t1 - t0;
  const int all = (int)((own_rows + KT - 1) / KT);
  int fast = (int)(own_rows / KT);
  if (a.O % V != 0 && (a.ldy < V || (t1 == a.rows && own_rows % KT == 0))) fast = a.ldy < V ? 0 : fast - 1;
  auto load_a = [&](int j, int step) {
    const T *d = dy + ((int64_t)step * KT + j * (NT / CA)) * a.ldy;
    ra[j] = *reinterpret_cast<const typename Piece<T>::mem *>(d + va);
  };
  auto load_b = [&](int j, int step) {
    const int64_t row = (int64_t)step * KT + j * (NT / CB);
    rb[j] = *reinterpret_cast<const uint4 *>(codes + row * a.ld8 + vb);
    rs[j] = (scales + row * a.nb8)[vs];
  };
  auto load_guarded = [&](int step) {
    const int left = (int)(own_rows - (int64_t)step * KT < KT ? own_rows - (int64_t)step * KT : KT);
#pragma unroll
    for (int j = 0; j < S::NA; ++j) {
      ra[j] = typename Piece<T>::raw{};
      if (ka + j * (NT / CA) < left && nva > 0) {
        const Cut<T> cut(cola, nva, a.O);
        ra[j] = cut.load(dy + ((int64_t)step * KT + j * (NT / CA) + ka) * a.ldy);
        cut.cut(ra[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < S::NB; ++j) {
      rb[j] = make_uint4(0, 0, 0, 0);
      rs[j] = 0;
      if (kb + j * (NT / CB) < left) load_b(j, step);
    }
  };
  auto add_bias = [&](int j) {
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] += (float)ra[j][v];
  };
  auto stage_a = [&](int j, char *buf) {
    const int k = ka + j * (NT / CA);
    char *dst = buf + tile_at<TM>(k, ca & ~7) + 2 * (ca & 7);
    if constexpr (P == 1) {
      *reinterpret_cast<typename Piece<T>::raw *>(dst) = ra[j];
    } else {
      uint32_t out[V][P];
#pragma unroll
      for (int v = 0; v < V; ++v) cut<P>((float)ra[j][v], out[v]);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        uint32_t w[V / 2];
#pragma unroll
        for (int v = 0; v < V / 2; ++v) w[v] = upper_halves(out[2 * v][p], out[2 * v + 1][p]);
        if constexpr (V == 8) *reinterpret_cast<uint4 *>(dst + p * S::kBytesA) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2 *>(dst + p * S::kBytesA) = make_uint2(w[0], w[1]);
      }
    }
  };
  auto stage_b = [&](int j, char *buf) {
    char *bb = buf + P * S::kBytesA;
    const int k = kb + j * (NT / CB);
    const float p = pow2_field(rs[j]);
    const uint32_t src[4] = {rb[j].x, rb[j].y, rb[j].z, rb[j].w};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        // (exact in bf16: the upper half of the float is all of it)
        const uint32_t c = src[2 * h + (v >> 1)] >> (16 * (v & 1));
        const uint32_t lo = __float_as_uint((float)(int8_t)c * p), hi = __float_as_uint((float)(int8_t)(c >> 8) * p);
        w[v] = upper_halves(lo, hi);
      }
      *reinterpret_cast<uint4 *>(bb + tile_at<TN>(k, cb + 8 * h)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  };

  f32x16 acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[m][n][q] = 0.0f;

  // transposed read: this lane's row within a group of four, its 16 columns and 4 of them
  const int kr = 8 * (lane >> 5) + ((lane >> 2) & 3), swa = swizzle<TM>(kr), swb = swizzle<TN>(kr);
  const int off = 2 * (16 * ((lane >> 4) & 1) + 4 * (lane & 3));
  typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
  auto frag = [&](char *base, int rowbytes, int k0, int blk, int sw) -> bf16x8 {
    char *p = base + (k0 + kr) * rowbytes + ((blk ^ sw) << 6) + off;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * rowbytes));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // A step is a run of items: one fragment of dY (32 columns, 16 rows, one piece) against the FN fragments
  // of x.  Fragments are read from LDS two items ahead, those of x a 16-row chunk ahead.  Between the
  // items the next step's rows, which arrived during the last step, are converted and written to LDS part by
  // part, and a part's registers at once take the rows of the step after: every load has a whole step.
  constexpr int kChunks = KT / 16, kPer = P * FM, kItems = kChunks * kPer, kParts = S::NA + S::NB;
  auto frag_a = [&](char *buf, int t) {
    const int c = t / kPer, p = (t % kPer) / FM, m = t % FM;
    return frag(buf + p * S::kBytesA, 2 * TM, 16 * c, wm * FM + m, swa);
  };
  auto frag_b = [&](char *buf, int c, int n) { return frag(buf + P * S::kBytesA, 2 * TN, 16 * c, wn * FN + n, swb); };
  // part j of the rows of `step` to buf
  auto stage_part = [&](int j, bool sums, char *buf) {
    if (j < S::NB) {
      stage_b(j, buf);
    } else {
      if (sums) add_bias(j - S::NB);
      stage_a(j - S::NB, buf);
    }
  };
  // the items of the step in buf; `between(t)` after item t
  auto multiply = [&](char *buf, auto between) {
    bf16x8 fa[3], fb[2][FN];
#pragma unroll
    for (int n = 0; n < FN; ++n) fb[0][n] = frag_b(buf, 0, n);
    fa[0] = frag_a(buf, 0);
    fa[1] = frag_a(buf, 1);
#pragma unroll
    for (int t = 0; t < kItems; ++t) {
      const int c = t / kPer;
      if (t + 2 < kItems) fa[(t + 2) % 3] = frag_a(buf, t + 2);
      if (t % kPer == 0 && c + 1 < kChunks)
#pragma unroll
        for (int n = 0; n < FN; ++n) fb[(c + 1) & 1][n] = frag_b(buf, c + 1, n);
#pragma unroll
      for (int n = 0; n < FN; ++n)
        acc[t % FM][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[t % 3], fb[c & 1][n], acc[t % FM][n], 0, 0, 0);
      between(t);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (fast > 0) {
    const int last = fast - 1;      // (loads behind it repeat its rows, which are staged and not read)
#pragma unroll
    for (int j = 0; j < kParts; ++j) j < S::NB ? load_b(j, 0) : load_a(j - S::NB, 0);
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      stage_part(j, ix == 0, lds);
      j < S::NB ? load_b(j, last < 1 ? last : 1) : load_a(j - S::NB, last < 1 ? last : 1);
    }
    __syncthreads();
    for (int s = 0; s < fast; ++s) {
      char *cur = lds + (s & 1) * S::kStage, *nxt = lds + ((s & 1) ^ 1) * S::kStage;
      const bool sums = (s + 1) % a.tx == ix && s + 1 < fast;
      const int ahead = s + 2 < last ? s + 2 : last;
      multiply(cur, [&](int t) {
#pragma unroll
        for (int j = 0; j < kParts; ++j)
          if (t == j * kItems / kParts) {
            stage_part(j, sums, nxt);
            j < S::NB ? load_b(j, ahead) : load_a(j - S::NB, ahead);
          }
      });
      __syncthreads();
    }
  }
  for (int s = fast; s < all; ++s) {
    load_guarded(s);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kParts; ++j) stage_part(j, s % a.tx == ix, lds);
    __syncthreads();
    multiply(lds, [](int) {});
  }
  __syncthreads();

  const bool whole = a.splits == 1;
  float *part = a.part + (int64_t)split * a.O * a.ldp;
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n) {
      const int i = i0 + (wn * FN + n) * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const int o = o0 + (wm * FM + m) * 32 + (q & 3) + 8 * (q >> 2) + 4 * (lane >> 5);
        if (o < a.O && i < a.I) {
          if (whole) ((T *)a.dw)[(int64_t)o * a.I + i] = (T)acc[m][n][q];
          else part[(int64_t)o * a.ldp + i] = acc[m][n][q];
        }
      }
    }
  // column sums over this work-group's share of the steps: its row lanes in order
  if (!a.db) return;
  float *sb = reinterpret_cast<float *>(lds);   // (all reads of the tiles are behind the last barrier)
#pragma unroll
  for (int v = 0; v < V; ++v) sb[ka * TM + ca + v] = bias[v];
  __syncthreads();
  for (int c = tid; c < TM; c += NT) {
    float s = 0.0f;
    for (int k = 0; k < NT / CA; ++k) s += sb[k * TM + c];
    if (o0 + c < a.O) a.part_b[((int64_t)split * a.tx + ix) * a.O + o0 + c] = s;
  }
}

// The parts of dW (if there is more than one) and of db, in a fixed order: a work-group's 256 threads are
// PL lanes to a value's parts times lanes of four neighbouring values (rows of a part are whole
// vectors).  The first `wide_groups` work-groups sum dW, the others db.
template <class T, int PL>
__global__ __launch_bounds__(256) void wgrad8_sum_kernel(WgradArgs a, unsigned wide_groups) {
  typedef float vec __attribute__((ext_vector_type(4)));
  constexpr int L = 256 / PL;
  __shared__ vec sh[PL][L];
  const int lane = threadIdx.x % L, part = threadIdx.x / L;
  if (blockIdx.x < wide_groups) {
    const int64_t n = (int64_t)a.O * a.ldp, e = ((int64_t)blockIdx.x * L + lane) * 4;
    vec s[4] = {};
    if (e < n) {
      int k = part;
      for (; k + 3 * PL < a.splits; k += 4 * PL)
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] += *reinterpret_cast<const vec *>(a.part + (k + PL * u) * n + e);
      for (; k < a.splits; k += PL) s[0] += *reinterpret_cast<const vec *>(a.part + k * n + e);
    }
    s[0] = (s[0] + s[1]) + (s[2] + s[3]);
    if (PL > 1) {
      sh[part][lane] = s[0];
      __syncthreads();
      if (part != 0) return;
#pragma unroll
      for (int k = 1; k < PL; ++k) s[0] += sh[k][lane];
    }
    if (e >= n) return;
    // (values behind a row's last are whatever the workspace held)
    const unsigned o = (unsigned)e / (unsigned)a.ldp, i = (unsigned)e - o * (unsigned)a.ldp;
    T *out = (T *)a.dw + (int64_t)o * a.I + i;
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (i + v < (unsigned)a.I) out[v] = (T)s[0][v];
    return;
  }
  const int o = (blockIdx.x - wide_groups) * 16 + (threadIdx.x & 15), p0 = threadIdx.x >> 4, parts = a.splits * a.tx;
  float s = 0.0f;
  if (o < a.O)
    for (int k = p0; k < parts; k += 16) s += a.part_b[(int64_t)k * a.O + o];
  float *f = reinterpret_cast<float *>(sh);
  f[threadIdx.x] = s;
  __syncthreads();
  if (p0 == 0 && o < a.O) {
    for (int k = 1; k < 16; ++k) s += f[16 * k + threadIdx.x];
    ((T *)a.db)[o] = (T)s;
  }
}

struct WgradShape {
  int tm, tn, tx, ty, splits;
  int64_t split_rows;
};
// Larger tiles need fewer bytes and conversions per product, smaller ones fill the chip sooner.  Measured
// (us, tiles of 64 x 64 / 128 x 128 / 128 x 256 / 256 x 256): 8192 rows of 256 x 256 float 18 / 23 / 26 / 30;
// 100000 x 64 x 64 float 19 / 27 / 35 / 44; 4096 x 1024 x 1024 bf16 38 / 30 / 36 / 35; 50001 x 515 x 387 half
// 108 / 92 / 82 / 87; 100000 x 640 x 640 half 310 / 201 / 193 / 211; 65536 x 1024 x 1024 bf16 473 / 180 / 175
// / 140.  So: 256 x 256 from 200000 rows times tiles on, or 128 x 256 where that covers dW with 10 % less;
// 64 x 64 below 100000 or where a side has no more than 64.  Rows are split until there is a work-group
// for each CU (two of the smaller ones; one range where that makes half of them already), no range shorter
// than 128 rows.
static WgradShape wgrad_shape(int64_t rows, int O, int I) {
  WgradShape s;
  auto tiles_of = [&](int tm, int tn) { return (int64_t)ceil_div(I, tn) * ceil_div(O, tm); };
  s.tm = s.tn = 128;
  if (O >= 256 && I >= 256 && tiles_of(256, 256) * rows >= 200000) {
    s.tn = 256;
    s.tm = 10 * tiles_of(128, 256) < 9 * 2 * tiles_of(256, 256) ? 128 : 256;
  } else if (O <= 64 || I <= 64 || tiles_of(128, 128) * rows < 100000) {
    s.tm = s.tn = 64;
  }
  s.tx = ceil_div(I, s.tn);
  s.ty = ceil_div(O, s.tm);
  const int64_t tiles = (int64_t)s.tx * s.ty, fill = s.tm == 256 ? 256 : 512;
  int64_t want = tiles >= fill / 2 ? 1 : fill / tiles;
  const int64_t most = (rows + 127) / 128;
  if (want > most) want = most;
  s.split_rows = ((rows + want - 1) / want + 63) / 64 * 64;
  s.splits = (int)((rows + s.split_rows - 1) / s.split_rows);
  return s;
}
static int wgrad_ldp(int I) { return (I + 3) / 4 * 4; }
static int64_t wgrad_bias_floats(const WgradShape &s, int O) { return ((int64_t)s.splits * s.tx * O + 3) / 4 * 4; }

template <class T, int FM, int FN, int WM, int WN, int KT>
static int wgrad_launch(const WgradArgs &a, hipStream_t s) {
  using S = Wgrad<T, FM, FN, WM, WN, KT>;
  const size_t lds = 2 * S::kStage;
  static_assert(2 * S::kStage <= (int)kMaxDynLds && S::NT * S::V * 4 <= 2 * S::kStage, "LDS");
  auto kernel = wgrad8_kernel<T, FM, FN, WM, WN, KT>;
  hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  GVAE_REQUIRE(e == hipSuccess, GVAE_ELAUNCH, "linear_wgrad8: %s", hipGetErrorString(e));
  hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)a.tx * a.ty * a.splits)), dim3(S::NT), lds, s, a);
  return GVAE_OK;
}

// many parts: 16 lanes to a value's parts; few: one
template <class T>
static void sum_launch(const WgradArgs &a, hipStream_t s) {
  const int64_t n = a.splits > 1 ? (int64_t)a.O * a.ldp : 0;
  const unsigned bias_groups = a.db ? ceil_div(a.O, 16) : 0;
  auto run = [&](auto kernel, int values) {
    const unsigned wide = (unsigned)((n + values - 1) / values);
    if (wide + bias_groups > 0) hipLaunchKernelGGL(kernel, dim3(wide + bias_groups), dim3(256), 0, s, a, wide);
  };
  if (a.splits <= 8) run(wgrad8_sum_kernel<T, 1>, 1024);
  else run(wgrad8_sum_kernel<T, 16>, 64);
}

}  // namespace gvae

using namespace gvae;

extern "C" {

int64_t gvae_linear_wgrad8_ws_bytes(int64_t rows, int O, int I) {
  if (rows <= 0 || O <= 0 || I <= 0) return 0;
  const WgradShape s = wgrad_shape(rows, O, I);
  return 4 * (wgrad_bias_floats(s, O) + (s.splits > 1 ? (int64_t)s.splits * O * wgrad_ldp(I) : 0));
}

int gvae_linear_wgrad8(const void *d_dy, int dtype, int64_t row_stride, const int8_t *d_codes, const uint8_t *d_scales,
                       int64_t rows, int O, int I, void *d_dw, void *d_db, void *d_ws, void *stream) {
  GVAE_REQUIRE(d_dy && d_codes && d_scales && d_dw && d_ws, GVAE_EINVAL, "linear_wgrad8: null pointer");
  GVAE_REQUIRE(aligned16(d_codes) && aligned16(d_ws), GVAE_EINVAL,
               "linear_wgrad8: codes or workspace not 16-byte aligned");
  GVAE_REQUIRE(dtype_known(dtype), GVAE_EINVAL, "linear_wgrad8: unknown element type %d", dtype);
  GVAE_REQUIRE(rows > 0 && O > 0 && I > 0 && row_stride >= O, GVAE_EINVAL,
               "linear_wgrad8: bad sizes (rows=%lld out=%d in=%d stride=%lld)", (long long)rows, O, I,
               (long long)row_stride);
  const WgradShape sh = wgrad_shape(rows, O, I);
  // (grids under 2^32 threads, offsets within a step under 2^32)
  GVAE_REQUIRE(O <= (1 << 20) && I <= (1 << 20) && (int64_t)O * I < (1LL << 31) &&
                   (int64_t)sh.tx * sh.ty * sh.splits < (1LL << 22) && row_stride < (1LL << 26) &&
                   sh.split_rows < (1LL << 31), GVAE_ELIMIT,
               "linear_wgrad8: %lld rows, %d x %d weights, stride %lld", (long long)rows, O, I, (long long)row_stride);
  WgradArgs a;
  a.dy = d_dy; a.codes = d_codes; a.scales = d_scales; a.dw = d_dw; a.db = d_db;
  a.rows = rows; a.ldy = row_stride; a.O = O; a.I = I; a.ldp = wgrad_ldp(I); a.ld8 = ckpt8_ld(I); a.nb8 = ckpt8_blocks(I);
  a.splits = sh.splits; a.split_rows = sh.split_rows; a.tx = sh.tx; a.ty = sh.ty;
  a.part_b = (float *)d_ws;
  a.part = a.part_b + wgrad_bias_floats(sh, O);
  hipStream_t s = (hipStream_t)stream;
  int rc = GVAE_OK;
  GVAE_DTYPE_SWITCH(dtype, T, {
    constexpr int kDeep = Pieces<T>::P == 1 ? 64 : 32;
    rc = sh.tm != sh.tn ? wgrad_launch<T, 4, 2, 1, 4, 32>(a, s)
         : sh.tm == 256 ? wgrad_launch<T, 4, 2, 2, 4, kDeep>(a, s)
         : sh.tm == 128 ? wgrad_launch<T, 2, 2, 2, 2, kDeep>(a, s) : wgrad_launch<T, 1, 1, 2, 2, 64>(a, s);
    if (rc == GVAE_OK) sum_launch<T>(a, s);
  });
  if (rc) return rc;
  return check_launch("linear_wgrad8");
}

}  // extern "C"
