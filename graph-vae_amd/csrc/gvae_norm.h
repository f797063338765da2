// Group norm over each graph's live rows, channels last, with an activation: what the forward
// (norm_fwd.hip) and the backward (norm_bwd.hip) share.
//
//   graph b, group q of C/G channels, live rows i < rows[b], m = rows[b] * C/G:
//   mean = sum x / m,  var = sum (x - mean)^2 / m,  r = 1 / sqrt(var + eps)
//   h = (x - mean) r,  z = h w_c + b_c,  y = act(z);  rows behind the last live one: y = 0
//   dz = dy act'(z);  dw_c = sum dz h,  db_c = sum dz  (over graphs and rows)
//   dx = r (w dz - (A1 + h A2)),  A1 = sum_group w dz / m,  A2 = sum_group w dz h / m
//
// For a ReLU z is formed by a subtraction, two products and a sum, each rounded, in the forward and in the
// backward alike: its branch is the same in both.  The other activations add b in the same step as the
// product (one rounding less); for 16-bit types the split form also centres and scales in one step, by a power
// of two (`Scale`: as exact, an instruction less).
//
// The split kernels come near the rate of the vector units before that of memory: a SiLU's slope is 13
// instructions a value, two of them at a quarter of the rate.
//
// All of it is bound by memory.  Two forms each:
//   resident   a work-group holds a graph's live rows of a run of groups (a slab) in registers: one
//              read, the sums through LDS, one write.  The slab is as narrow as fills the chip, but
//              no row segment is under 64 bytes.
//   split      a group too long for that is summed in chunks of rows by as many work-groups, joined
//              by one wavefront (few chunks) or work-group (many) per group, and read again to be written.
#pragma once
#include "gvae_ckpt8.h"

#include <cmath>
#include <type_traits>

namespace gvae {

constexpr int kThreads = 256;
constexpr int kBatch = 8;     // rows of a thread in registers at a time (statistics of the split form)
constexpr int kLeast = 4;     // rows of a thread in a chunk, at least

struct NormArgs {
  const void *x;              // input, or null if the codes are given (backward)
  const int8_t *codes;
  const uint8_t *scales;
  const void *dy;
  void *out;                  // y or dx, contiguous
  const float *w, *b;
  float *mean, *rstd;         // (B, G)
  const int32_t *rows;
  int8_t *x8, *y8;
  uint8_t *x8s, *y8s;
  float *part1, *part2;       // split: (B * chunks, C), mean and M2 or the two sums of the backward;
                              // resident backward: (graph lanes, C), the two sums
  float *A;                   // (B, G, 2)
  int64_t xb, xr, dyb, dyr;   // strides of x and dy in elements
  float eps;
  int act;
  int B, N, C, G, cpg;
  int lanes;                  // pieces per row (split: in one column tile, resident: in a slab)
  int rp;                     // rows side by side in a work-group
  int chunk_rows, chunks;     // split
  int slab, nslab;            // resident: channels of a slab
  int graph_step;             // resident backward: graphs walked in steps of this
  int join;                   // resident: lanes (a power of two) that add up one group
  int ld8, nb8;
  bool past;                  // large results: nontemporal stores
};

__device__ __forceinline__ int live_rows(const NormArgs &a, int b) {
  if (!a.rows) return a.N;
  const int r = a.rows[b];
  return r < 0 ? 0 : (r > a.N ? a.N : r);
}

// 1 / (1 + exp(-z)) from the hardware's exp2 and reciprocal (one unit in the last place each): the
// argument's rounding makes it |z| u relative, under the rounding of z that it is computed from.
__device__ __forceinline__ float sigmoid_fast(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}
// Phi(z) = (1 + erf(z / sqrt 2)) / 2 and *e = exp(-z^2 / 2).  FULL (fp32 tensors): with erff.  Else by
// formula 7.1.26 of Abramowitz and Stegun (Hastings): 1 - erf(x) = (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 + p x),
// |error| <= 1.5e-7, in half the instructions: under the rounding of 16-bit values, over that of fp32 (GELU of
// normal values off by 5.6e-8 rms, 2.4e-8 with erff).
template <bool FULL>
__device__ __forceinline__ float normal_cdf(float z, float *e) {
  *e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  if (FULL) return __fmaf_rn(0.5f, erff(z * 0.70710678118654752f), 0.5f);
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(__fmaf_rn(0.3275911f, x, 1.0f));
  float p = __fmaf_rn(1.061405429f, t, -1.453152027f);
  p = __fmaf_rn(p, t, 1.421413741f);
  p = __fmaf_rn(p, t, -0.284496736f);
  p = __fmaf_rn(p, t, 0.254829592f);
  const float tail = 0.5f * p * t * *e;                  // 1 - Phi(|z|)
  return z < 0.0f ? tail : 1.0f - tail;
}
template <int ACT, bool FULL>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == GVAE_ACT_RELU) return z < 0.0f ? 0.0f : z;   // (keeps a NaN)
  if (ACT == GVAE_ACT_SILU) return z * sigmoid_fast(z);
  if (ACT == GVAE_ACT_GELU) {
    float e;
    return z * normal_cdf<FULL>(z, &e);
  }
  return z;
}
template <int ACT, bool FULL>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == GVAE_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (ACT == GVAE_ACT_SILU) {
    const float s = sigmoid_fast(z);      // s + s z (1 - s)
    return __fmaf_rn(s, __fmaf_rn(-z, s, z), s);
  }
  if (ACT == GVAE_ACT_GELU) {
    float e;
    const float c = normal_cdf<FULL>(z, &e);
    return __fmaf_rn(z * 0.39894228040143268f, e, c);
  }
  return 1.0f;
}
template <int ACT>
__device__ __forceinline__ float pre_act(float h, float w, float b) {
  return ACT == GVAE_ACT_RELU ? h * w + b : __fmaf_rn(h, w, b);
}
// the same for a piece, with the activation chosen at run time (uniform over the launch)
template <int V, bool FULL>
__device__ __forceinline__ void act_values(int act, const float *h, const float *w, const float *b, float *y) {
  auto all = [&](auto tag) {
    constexpr int ACT = decltype(tag)::value;
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = act_value<ACT, FULL>(pre_act<ACT>(h[v], w[v], b[v]));
  };
  switch (act) {
    case GVAE_ACT_RELU: all(std::integral_constant<int, GVAE_ACT_RELU>{}); break;
    case GVAE_ACT_SILU: all(std::integral_constant<int, GVAE_ACT_SILU>{}); break;
    case GVAE_ACT_GELU: all(std::integral_constant<int, GVAE_ACT_GELU>{}); break;
    default: all(std::integral_constant<int, GVAE_ACT_NONE>{}); break;
  }
}
template <int V, bool FULL>
__device__ __forceinline__ void act_slopes(int act, const float *h, const float *w, const float *b, float *s) {
  auto all = [&](auto tag) {
    constexpr int ACT = decltype(tag)::value;
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = act_slope<ACT, FULL>(pre_act<ACT>(h[v], w[v], b[v]));
  };
  switch (act) {
    case GVAE_ACT_RELU: all(std::integral_constant<int, GVAE_ACT_RELU>{}); break;
    case GVAE_ACT_SILU: all(std::integral_constant<int, GVAE_ACT_SILU>{}); break;
    case GVAE_ACT_GELU: all(std::integral_constant<int, GVAE_ACT_GELU>{}); break;
    default: all(std::integral_constant<int, GVAE_ACT_NONE>{}); break;
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// the same over a work-group of NT threads (every thread gets the sum)
template <int NT>
__device__ __forceinline__ float group_sum(float v, float *sh) {
  v = wave_sum(v);
  if (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int k = 0; k < NT / 64; ++k) v += sh[k];
  return v;
}

// a (graphs, groups) table at the channels of a piece, 0 behind the last channel
template <int V>
__device__ __forceinline__ void per_group(const NormArgs &a, const float *table, int g, int c0, int nv, float *f) {
  const float *row = table + (int64_t)g * a.G;
  if (a.cpg % V == 0) {          // (uniform: a piece then lies inside one group)
    const float one = nv > 0 ? row[c0 / a.cpg] : 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = one;
    return;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = v < nv ? row[(c0 + v) / a.cpg] : 0.0f;
}

// V floats of a per-channel parameter (`none` where there is no parameter), 0 behind the last channel
template <int V>
__device__ __forceinline__ void load_params(const float *p, int c0, int nv, float none, float *f) {
  typedef float four __attribute__((ext_vector_type(4), aligned(4)));
  if (p && nv == V) {
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
      const four q = *reinterpret_cast<const four *>(p + c0 + 4 * h);
#pragma unroll
      for (int v = 0; v < 4; ++v) f[4 * h + v] = q[v];
    }
    return;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = v < nv ? (p ? p[c0 + v] : none) : 0.0f;
}

// What the channels of a piece are scaled and shifted by: centred(x) * unit is h, and pre<ACT>(centred(x)) the
// value before the activation.
//   POW2: centred(x) = x p - mean p in one step, p the power of two at or under rstd, at most 1: both products
//         are exact, so it is (x - mean) p rounded once; unit = rstd / p is left in the weight.
//   else: centred(x) = (x - mean) rstd, unit = 1.
template <int V, bool POW2>
struct Scale {
  float mean[V], rstd[V], w[V], b[V], unit[V];      // POW2: -mean p, p, w unit
  static __device__ __forceinline__ float pow2_of(float rstd) {
    const float p = __uint_as_float(__float_as_uint(rstd) & 0x7f800000u);
    return fminf(fmaxf(p, 0x1p-126f), 1.0f);
  }
  // (rstd / p by an exponent's subtraction: exact)
  static __device__ __forceinline__ float unit_of(float rstd) {
    return POW2 ? rstd * __uint_as_float(0x7f000000u - __float_as_uint(pow2_of(rstd))) : 1.0f;
  }
  __device__ __forceinline__ float centred(int v, float x) const {
    return POW2 ? __fmaf_rn(x, rstd[v], mean[v]) : (x - mean[v]) * rstd[v];
  }
  template <int ACT>
  __device__ __forceinline__ float pre(int v, float c) const { return pre_act<ACT>(c, w[v], b[v]); }
  __device__ Scale(const NormArgs &a, int g, int c0, int nv) {
    load_params<V>(a.w, c0, nv, 1.0f, w);
    load_params<V>(a.b, c0, nv, 0.0f, b);
    per_group<V>(a, a.mean, g, c0, nv, mean);
    per_group<V>(a, a.rstd, g, c0, nv, rstd);
#pragma unroll
    for (int v = 0; v < V; ++v) unit[v] = 1.0f;
    if (!POW2) return;
    auto split = [&](int from, int v) {
      unit[v] = unit_of(rstd[from]);
      w[v] *= unit[v];
      mean[v] *= -pow2_of(rstd[from]);
    };
    if (a.cpg % V == 0) {          // (uniform: one group, as in per_group)
      const float p = pow2_of(rstd[0]);
#pragma unroll
      for (int v = 0; v < V; ++v) split(0, v);
#pragma unroll
      for (int v = 0; v < V; ++v) rstd[v] = p;
      return;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      split(v, v);
      rstd[v] = pow2_of(rstd[v]);
    }
  }
};

// ---- split form: where a thread of a chunk work-group stands
template <int V>
struct Place {
  int b, chunk, c0, nv, r, row_end;   // first channel, channels of the piece, first row lane
  bool on;
  __device__ Place(const NormArgs &a, bool live_only, bool backwards) {
    const int id = backwards ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x;
    b = id / a.chunks;
    chunk = id - b * a.chunks;
    const int col = threadIdx.x % a.lanes;
    r = threadIdx.x / a.lanes;
    c0 = (blockIdx.y * a.lanes + col) * V;
    nv = a.C - c0 < V ? a.C - c0 : V;
    on = r < a.rp;
    const int stop = live_only ? live_rows(a, b) : a.N;
    row_end = (chunk + 1) * a.chunk_rows < stop ? (chunk + 1) * a.chunk_rows : stop;
  }
};

// ---- resident form: sums over the groups of a slab.  Every thread has left E entries of its piece in
// LDS (thread order, which is row-major: rp rows of row_entries); a group is ge neighbouring entries of
// each row.  `join` lanes add up a group, in a fixed order.
// Sums over the row lanes of a work-group: NS tables of rp rows of `wide` columns in LDS, the sum of a
// column by as many lanes (a power of two, at most 64) as there are threads for, in a fixed order;
// done(column, sums) once per column.
template <int NS, int NT, int LEN, class F>
__device__ __forceinline__ void column_sums(const float (*tab)[LEN], int wide, int rp, F done) {
  int lanes = 1;
  while (lanes < 64 && 2 * lanes * wide <= NT && lanes < rp) lanes *= 2;
  const int lane = threadIdx.x & (lanes - 1);
  for (int c = threadIdx.x / lanes; c < wide; c += NT / lanes) {
    float s[NS];
#pragma unroll
    for (int k = 0; k < NS; ++k) s[k] = 0.0f;
    for (int r = lane; r < rp; r += lanes)
#pragma unroll
      for (int k = 0; k < NS; ++k) s[k] += tab[k][r * wide + c];
    for (int off = lanes >> 1; off > 0; off >>= 1)
#pragma unroll
      for (int k = 0; k < NS; ++k) s[k] += __shfl_xor(s[k], off, 64);
    if (lane == 0) done(c, s);
  }
}

template <int NS, int LA, int LB>
__device__ __forceinline__ void join_groups(const float (*ent)[LA], int row_entries, int ge, int ng, int rp, int join,
                                            int threads, float (*out)[LB]) {
  const int lane = threadIdx.x & (join - 1);
  const int dr = join / ge, dq = join - dr * ge;
  for (int g = threadIdx.x / join; g < ng; g += threads / join) {
    float s[NS];
#pragma unroll
    for (int k = 0; k < NS; ++k) s[k] = 0.0f;
    int r = lane / ge, q = lane - r * ge;
    while (r < rp) {
      const int e = r * row_entries + g * ge + q;
#pragma unroll
      for (int k = 0; k < NS; ++k) s[k] += ent[k][e];
      r += dr;
      q += dq;
      if (q >= ge) { q -= ge; ++r; }
    }
    for (int off = join >> 1; off > 0; off >>= 1)
#pragma unroll
      for (int k = 0; k < NS; ++k) s[k] += __shfl_xor(s[k], off, 64);
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < NS; ++k) out[k][g] = s[k];
  }
}

// The group of a slab's channel c (one after the last channel of group g or one of its own), the last
// group behind the slab
__device__ __forceinline__ int group_after(int g, int c, int cpg, int ng) {
  return c >= (g + 1) * cpg && g + 1 < ng ? g + 1 : g;
}

// Column tiles, row lanes and row chunks of the split form: a row is cut into tiles of at most 256
// pieces; the rows of a graph are cut so that about 2048 work-groups (eight per CU) share the
// batch, each with at least kLeast rows per row lane.
struct SplitShape {
  int lanes, tiles, rp, chunk_rows, chunks;
};
inline SplitShape split_shape(int B, int N, int C, int V, bool whole_blocks) {
  SplitShape s;
  int pieces = ceil_div(C, V);
  if (whole_blocks) pieces = ceil_div(C, kBlock8) * (kBlock8 / V);
  s.lanes = pieces < kThreads ? pieces : kThreads;
  s.tiles = ceil_div(pieces, s.lanes);
  s.rp = kThreads / s.lanes;
  const int64_t have = (int64_t)B * s.tiles;
  const int want = (int)(have >= 2048 ? 1 : (2048 + have - 1) / have);
  int rows = ceil_div(N, want), least = kLeast * s.rp;
  if (rows < least) rows = least;
  s.chunk_rows = ceil_div(rows, s.rp) * s.rp;
  s.chunks = ceil_div(N, s.chunk_rows);
  return s;
}

// Slab of the resident form.  `align`: channels a slab has to start at a multiple of (32 where
// checkpoints are written, the piece where one is read); `least`: pieces of a row segment that are worth a
// memory transaction (4 of 16 bytes; 8 where checkpoints are written, whose segments are half as long; 1
// where everything is a few MB and stays in the caches: there a slab may end inside its one piece);
// `threads` and `held`: the largest work-group and the pieces a thread holds in it.  The slab is the
// widest that leaves 1024 work-groups and has at most `most` pieces, so that several work-groups share a CU
// and one's loads run beside another's sums; the narrowest may have `last_most`.  false: no slab of whole
// groups is that small, or the batch would leave most of the chip idle that the split form fills.
// Measured, forward, bf16, SiLU, 512 channels: 256 graphs of 250 rows 34 us (42 with slabs of up to 4096
// pieces, 53 split); 192 graphs of 1000 rows 107 us (127 split), but 180 (162 split) with checkpoints
// in 64-byte segments; 256 graphs of 2000 rows, 320 channels: 339 us in slabs of 8000 pieces, 205 split.
struct ResidentShape {
  int slab, nslab, lanes;
};
inline bool resident_shape(int B, int N, int C, int cpg, int V, int align, int least, int threads, int held, int most,
                           int last_most, ResidentShape *s) {
  int64_t unit = cpg;
  while (unit % align && unit < C) unit += cpg;
  if (unit > C) unit = C;
  auto lanes_of = [&](int64_t slab) { return (int)(((slab + align - 1) / align * align + V - 1) / V); };
  const int64_t want = B >= 1024 ? 1 : (1024 + B - 1) / B;
  int64_t units = ((C + unit - 1) / unit + want - 1) / want;
  const int64_t fewest = least > 1 ? (least * V + unit - 1) / unit : unit < V ? V / unit : 1;
  if (units < fewest) units = fewest;
  for (;; --units) {
    const int64_t slab = units * unit < C ? units * unit : C;
    const int lanes = lanes_of(slab);
    const int64_t pieces = (int64_t)N * lanes;
    const bool last = units <= fewest || units <= 1;
    if (pieces <= (last ? last_most : most) && lanes <= threads && (int64_t)(threads / lanes) * held >= N) {
      s->slab = (int)slab; s->lanes = lanes; s->nslab = ceil_div(C, (int)slab);
      return (int64_t)B * s->nslab >= 128 || pieces <= 2048;
    }
    if (last) return false;
  }
}
// lanes that add up one of `groups` groups with `threads` threads
inline int join_lanes(int groups, int threads) {
  int j = 64;
  while (j > 1 && (int64_t)j * groups > threads) j >>= 1;
  return j;
}

// which form a call takes, and the workspace it needs (floats): resident forward none; resident backward
// a row of partial sums per graph lane; split the chunks' partial rows and A1, A2
struct NormPlan {
  bool resident;
  ResidentShape rs;
  SplitShape sp;
  int graph_step;
  int64_t floats;
};
inline NormPlan norm_plan(bool backward, int dtype, int B, int N, int C, int G, bool checkpoints) {
  NormPlan p{};
  const int V = dtype == GVAE_F32 ? 4 : 8, cpg = C / G;
  const int least = (int64_t)B * N * C * (16 / V) <= (8 << 20) ? 1 : 4;
  // The backward holds two to three times the registers a piece, hence smaller work-groups.  Measured, SiLU,
  // bf16, slabs of up to 512 / 2048 pieces: 256 graphs of 250 rows, 512 channels 56 / 64 us, from the
  // checkpoint 54 / 68; 512 graphs of 128 rows, 128 channels, float 25 / 36.  Split / narrowest slab: 192
  // graphs of 500 rows, 512 channels (2000 pieces) 99 / 107, of 400 rows 85 / 79; 300 graphs of 300 rows,
  // 320 channels in groups of ten (1500) 80 / 88.
  p.resident = backward ? resident_shape(B, N, C, cpg, V, checkpoints ? V : 1, least, 512, 4, 512,
                                         cpg % V == 0 ? 1600 : 1024, &p.rs)
                        : resident_shape(B, N, C, cpg, V, checkpoints ? kBlock8 : 1, checkpoints ? 8 : least, 1024, 8,
                                         2048, 4096, &p.rs);
  if (p.resident) {
    // about 1024 work-groups walk the graphs of the backward
    p.graph_step = p.rs.nslab >= 1024 ? 1 : 1024 / p.rs.nslab;
    if (p.graph_step > B) p.graph_step = B;
    p.floats = backward ? 2 * (int64_t)p.graph_step * C : 0;
    return p;
  }
  p.sp = split_shape(B, N, C, V, !backward && checkpoints);
  p.floats = 2 * (int64_t)B * p.sp.chunks * C + (backward ? 2 * (int64_t)B * G : 0);
  return p;
}

int norm_check(const char *who, int dtype, int B, int N, int C, int G, int act, int64_t ld);

}  // namespace gvae
