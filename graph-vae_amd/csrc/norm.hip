// Group norm over each graph's live rows, channels last, with an activation: forward, statistics,
// 8-bit checkpoints of its input and output, and backward (from the input or its checkpoint).
//
//   graph b, group q of C/G channels, live rows i < rows[b], m = rows[b] * C/G:
//   mean = sum x / m,  var = sum (x - mean)^2 / m,  r = 1 / sqrt(var + eps)
//   h = (x - mean) r,  z = h w_c + b_c,  y = act(z);  rows behind the last live one: y = 0
//   dz = dy act'(z);  dw_c = sum dz h,  db_c = sum dz  (over graphs and rows)
//   dx = r (w dz - (A1 + h A2)),  A1 = sum_group w dz / m,  A2 = sum_group w dz h / m
//
// z is formed by a subtraction, two products and a sum, each rounded (no contraction), in the
// forward and in the backward alike: the branch of a ReLU is the same in both.
//
// A sum over rows is split over work-groups by chunks of rows; what a chunk leaves is one pair per
// channel (count-weighted mean and centred square sum, combined as n, mean, M2 with
// M2 = M2a + M2b + d^2 na nb / n), so no square of an uncentred value is ever summed.
#include "gvae_ckpt8.h"

#include <cmath>

namespace gvae {

constexpr int kThreads = 256;
constexpr int kBatch = 8;     // rows of a thread in registers at a time

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
  float *part1, *part2;       // (B * chunks, C): mean and M2, or the two sums of the backward
  float *A;                   // (B, G, 2)
  int64_t xb, xr, dyb, dyr;   // strides of x and dy in elements
  float eps;
  int B, N, C, G, cpg;
  int lanes;                  // pieces per row in one column tile
  int rp;                     // rows side by side in a work-group
  int chunk_rows, chunks;
  int ld8, nb8;
};

__device__ __forceinline__ int live_rows(const NormArgs &a, int b) {
  if (!a.rows) return a.N;
  const int r = a.rows[b];
  return r < 0 ? 0 : (r > a.N ? a.N : r);
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == GVAE_ACT_RELU) return z < 0.0f ? 0.0f : z;   // (keeps a NaN)
  if (ACT == GVAE_ACT_SILU) return z / (1.0f + expf(-z));
  if (ACT == GVAE_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == GVAE_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (ACT == GVAE_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  if (ACT == GVAE_ACT_GELU)
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
  return 1.0f;
}

// Where a thread of a chunk work-group stands: its piece of V channels and its rows.
template <int V>
struct Place {
  int b, chunk, c0, nv, r, row_end;   // first channel, channels of the piece, first row lane
  bool on;
  __device__ Place(const NormArgs &a, bool live_only) {
    b = blockIdx.x / a.chunks;
    chunk = blockIdx.x - b * a.chunks;
    const int col = threadIdx.x % a.lanes;
    r = threadIdx.x / a.lanes;
    c0 = (blockIdx.y * a.lanes + col) * V;
    nv = a.C - c0 < V ? a.C - c0 : V;
    on = r < a.rp;
    const int stop = live_only ? live_rows(a, b) : a.N;
    row_end = (chunk + 1) * a.chunk_rows < stop ? (chunk + 1) * a.chunk_rows : stop;
  }
};

// --------------------------------------------------------------------------- forward
// (n, mean, M2) of every channel over a chunk's live rows
template <class T>
__global__ __launch_bounds__(kThreads) void norm_stats_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V;
  __shared__ float sh_mean[kThreads * V], sh_m2[kThreads * V];
  __shared__ int sh_n[kThreads];
  const Place<V> p(a, true);
  const int row0 = p.chunk * a.chunk_rows;
  float mean[V], m2[V];
  int n = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) mean[v] = m2[v] = 0.0f;
  if (p.on && p.nv > 0) {
    const T *x = (const T *)a.x + p.b * a.xb + p.c0;
    for (int i = row0 + p.r; i < p.row_end; i += kBatch * a.rp) {
      typename Piece<T>::raw k[kBatch];
      int cnt = 0;
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + u * a.rp < p.row_end) {
          k[u] = load_piece<T>(x + (int64_t)(i + u * a.rp) * a.xr, p.nv);
          ++cnt;
        }
      const float inv = 1.0f / (float)cnt;
      const float share = (float)cnt / (float)(n + cnt), cross = (float)n * share;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) if (u < cnt) s += (float)k[u][v];
        const float mb = s * inv;
        float q = 0.0f;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) if (u < cnt) {
          const float d = (float)k[u][v] - mb;
          q = __fmaf_rn(d, d, q);
        }
        const float d = mb - mean[v];
        mean[v] = __fmaf_rn(d, share, mean[v]);
        m2[v] += __fmaf_rn(d * d, cross, q);
      }
      n += cnt;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sh_mean[threadIdx.x * V + v] = mean[v];
    sh_m2[threadIdx.x * V + v] = m2[v];
  }
  sh_n[threadIdx.x] = n;
  __syncthreads();
  // the row lanes of a channel, in their order
  const int wide = a.lanes * V;
  for (int c = threadIdx.x; c < wide; c += kThreads) {
    const int gc = blockIdx.y * wide + c;
    if (gc >= a.C) continue;
    const int col = c / V;
    float tot = 0.0f, s = 0.0f;
    for (int r = 0; r < a.rp; ++r) {
      const float nr = (float)sh_n[r * a.lanes + col];
      tot += nr;
      s = __fmaf_rn(nr, sh_mean[r * wide + c], s);
    }
    const float mu = tot > 0.0f ? s / tot : 0.0f;
    float q = 0.0f;
    for (int r = 0; r < a.rp; ++r) {
      const float d = sh_mean[r * wide + c] - mu;
      q += sh_m2[r * wide + c] + (float)sh_n[r * a.lanes + col] * d * d;
    }
    const int64_t o = (int64_t)blockIdx.x * a.C + gc;
    a.part1[o] = mu;
    a.part2[o] = q;
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// mean and 1/sqrt(var + eps) of a group from its chunks' channels, one wavefront per group
__global__ __launch_bounds__(kThreads) void norm_stats_join_kernel(NormArgs a) {
  const int64_t q = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (q >= (int64_t)a.B * a.G) return;
  const int b = (int)(q / a.G), g = (int)(q - (int64_t)b * a.G), lane = threadIdx.x & 63;
  const int live = live_rows(a, b), total = a.chunks * a.cpg;
  auto rows_of = [&](int k) {
    const int n = live - k * a.chunk_rows;
    return (float)(n < 0 ? 0 : (n > a.chunk_rows ? a.chunk_rows : n));
  };
  const int64_t base = (int64_t)b * a.chunks * a.C + g * a.cpg;
  float s = 0.0f;
  for (int e = lane; e < total; e += 64) {
    const int k = e / a.cpg, c = e - k * a.cpg;
    s = __fmaf_rn(rows_of(k), a.part1[base + (int64_t)k * a.C + c], s);
  }
  s = wave_sum(s);
  const float m = (float)live * (float)a.cpg;
  const float mu = live > 0 ? s / m : 0.0f;
  float v = 0.0f;
  for (int e = lane; e < total; e += 64) {
    const int k = e / a.cpg, c = e - k * a.cpg;
    const float d = a.part1[base + (int64_t)k * a.C + c] - mu;
    v += __fmaf_rn(rows_of(k) * d, d, a.part2[base + (int64_t)k * a.C + c]);
  }
  v = wave_sum(v);
  if (lane == 0) {
    a.mean[q] = mu;
    a.rstd[q] = 1.0f / sqrtf((live > 0 ? v / m : 0.0f) + a.eps);
  }
}

// what a channel of a piece is scaled and shifted by
template <int V>
struct Scale {
  float mean[V], rstd[V], w[V], b[V];
  __device__ Scale(const NormArgs &a, int g, int c0, int nv) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool in = v < nv;
      const int c = in ? c0 + v : 0;
      const int64_t q = (int64_t)g * a.G + c / a.cpg;
      mean[v] = in ? a.mean[q] : 0.0f;
      rstd[v] = in ? a.rstd[q] : 0.0f;
      w[v] = in && a.w ? a.w[c] : (in ? 1.0f : 0.0f);
      b[v] = in && a.b ? a.b[c] : 0.0f;
    }
  }
};

template <class T, int ACT>
__global__ __launch_bounds__(kThreads) void norm_apply_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V;
  const Place<V> p(a, false);
  if (!p.on) return;
  const int live = live_rows(a, p.b);
  const Scale<V> k(a, p.b, p.c0, p.nv);
  const T *x = (const T *)a.x + p.b * a.xb + p.c0;
  for (int i = p.chunk * a.chunk_rows + p.r; i < p.row_end; i += a.rp) {
    float xf[V], y[V];
#pragma unroll
    for (int v = 0; v < V; ++v) xf[v] = y[v] = 0.0f;
    if (i < live && p.nv > 0) {
      const typename Piece<T>::raw r = load_piece<T>(x + (int64_t)i * a.xr, p.nv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (v < p.nv) {
          xf[v] = (float)r[v];
          y[v] = (float)(T)act_value<ACT>((xf[v] - k.mean[v]) * k.rstd[v] * k.w[v] + k.b[v]);
        }
      }
    }
    const int64_t row = (int64_t)p.b * a.N + i;
    if (p.nv > 0) store_piece<T>((T *)a.out + row * a.C + p.c0, y, p.nv);
    // (the lanes of a block share a row: with checkpoints kept, `lanes` is a whole number of blocks)
    const int nc = a.ld8 - p.c0;
    const bool first = p.c0 % kBlock8 == 0 && p.nv > 0;
    if (a.x8) emit8<V>(xf, a.x8 + row * a.ld8 + p.c0, nc, a.x8s + row * a.nb8 + p.c0 / kBlock8, first);
    if (a.y8) emit8<V>(y, a.y8 + row * a.ld8 + p.c0, nc, a.y8s + row * a.nb8 + p.c0 / kBlock8, first);
  }
}

// --------------------------------------------------------------------------- backward
// V values of x at row `row` of the whole batch, from the tensor or from the checkpoint
template <class T, bool KEPT>
__device__ __forceinline__ void load_x(const NormArgs &a, int b, int i, int c0, int nv, float *f) {
  constexpr int V = Piece<T>::V;
  if (KEPT) {
    const int64_t row = (int64_t)b * a.N + i;
    decode8<V>(load_codes<V>(a.codes + row * a.ld8 + c0), pow2_field(a.scales[row * a.nb8 + c0 / kBlock8]), f);
  } else {
    const typename Piece<T>::raw r = load_piece<T>((const T *)a.x + b * a.xb + (int64_t)i * a.xr + c0, nv);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = (float)r[v];
  }
}

template <class T, int ACT, bool KEPT>
__global__ __launch_bounds__(kThreads) void norm_bwd_sums_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V;
  __shared__ float sh1[kThreads * V], sh2[kThreads * V];
  const Place<V> p(a, true);
  float s1[V], s2[V];
#pragma unroll
  for (int v = 0; v < V; ++v) s1[v] = s2[v] = 0.0f;
  if (p.on && p.nv > 0) {
    const Scale<V> k(a, p.b, p.c0, p.nv);
    const T *dy = (const T *)a.dy + p.b * a.dyb + p.c0;
    for (int i = p.chunk * a.chunk_rows + p.r; i < p.row_end; i += a.rp) {
      const typename Piece<T>::raw g = load_piece<T>(dy + (int64_t)i * a.dyr, p.nv);
      float x[V];
      load_x<T, KEPT>(a, p.b, i, p.c0, p.nv, x);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float h = (x[v] - k.mean[v]) * k.rstd[v];
        const float dz = (float)g[v] * act_slope<ACT>(h * k.w[v] + k.b[v]);
        s1[v] += dz;
        s2[v] = __fmaf_rn(dz, h, s2[v]);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sh1[threadIdx.x * V + v] = s1[v];
    sh2[threadIdx.x * V + v] = s2[v];
  }
  __syncthreads();
  const int wide = a.lanes * V;
  for (int c = threadIdx.x; c < wide; c += kThreads) {
    const int gc = blockIdx.y * wide + c;
    if (gc >= a.C) continue;
    float t1 = 0.0f, t2 = 0.0f;
    for (int r = 0; r < a.rp; ++r) {
      t1 += sh1[r * wide + c];
      t2 += sh2[r * wide + c];
    }
    a.part1[(int64_t)blockIdx.x * a.C + gc] = t1;
    a.part2[(int64_t)blockIdx.x * a.C + gc] = t2;
  }
}

// A1 and A2 of a group, one wavefront per group
__global__ __launch_bounds__(kThreads) void norm_bwd_join_kernel(NormArgs a) {
  const int64_t q = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (q >= (int64_t)a.B * a.G) return;
  const int b = (int)(q / a.G), g = (int)(q - (int64_t)b * a.G), lane = threadIdx.x & 63;
  const int64_t base = (int64_t)b * a.chunks * a.C + g * a.cpg;
  float s1 = 0.0f, s2 = 0.0f;
  for (int e = lane; e < a.chunks * a.cpg; e += 64) {
    const int k = e / a.cpg, c = e - k * a.cpg;
    const float w = a.w ? a.w[g * a.cpg + c] : 1.0f;
    s1 = __fmaf_rn(w, a.part1[base + (int64_t)k * a.C + c], s1);
    s2 = __fmaf_rn(w, a.part2[base + (int64_t)k * a.C + c], s2);
  }
  s1 = wave_sum(s1);
  s2 = wave_sum(s2);
  if (lane == 0) {
    const int live = live_rows(a, b);
    const float m = (float)(live > 0 ? live : 1) * (float)a.cpg;
    a.A[2 * q] = s1 / m;
    a.A[2 * q + 1] = s2 / m;
  }
}

// dw and db: the partial rows summed, 16 channels x 64 row lanes per work-group
__global__ __launch_bounds__(1024) void norm_bwd_params_kernel(const float *__restrict__ part1,
                                                               const float *__restrict__ part2, int64_t n,
                                                               int C, float *__restrict__ db,
                                                               float *__restrict__ dw) {
  __shared__ float sh[64][17];
  const float *p = blockIdx.y ? part2 : part1;
  float *out = blockIdx.y ? dw : db;
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < C) {
    int64_t r = rl;
    for (; r + 192 < n; r += 256)
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += p[(r + 64 * u) * C + c];
    for (; r < n; r += 64) s[0] += p[r * C + c];
  }
  sh[rl][cl] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (rl == 0 && c < C) {
    float t = 0.0f;
    for (int k = 0; k < 64; ++k) t += sh[k][cl];
    out[c] = t;
  }
}

template <class T, int ACT, bool KEPT>
__global__ __launch_bounds__(kThreads) void norm_bwd_apply_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V;
  const Place<V> p(a, false);
  if (!p.on || p.nv <= 0) return;
  const int live = live_rows(a, p.b);
  const Scale<V> k(a, p.b, p.c0, p.nv);
  float a1[V], a2[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int64_t q = (int64_t)p.b * a.G + (p.c0 + (v < p.nv ? v : 0)) / a.cpg;
    a1[v] = a.A[2 * q];
    a2[v] = a.A[2 * q + 1];
  }
  const T *dy = (const T *)a.dy + p.b * a.dyb + p.c0;
  for (int i = p.chunk * a.chunk_rows + p.r; i < p.row_end; i += a.rp) {
    float dx[V];
#pragma unroll
    for (int v = 0; v < V; ++v) dx[v] = 0.0f;
    if (i < live) {
      const typename Piece<T>::raw g = load_piece<T>(dy + (int64_t)i * a.dyr, p.nv);
      float x[V];
      load_x<T, KEPT>(a, p.b, i, p.c0, p.nv, x);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float h = (x[v] - k.mean[v]) * k.rstd[v];
        const float dz = (float)g[v] * act_slope<ACT>(h * k.w[v] + k.b[v]);
        dx[v] = k.rstd[v] * (dz * k.w[v] - __fmaf_rn(h, a2[v], a1[v]));
      }
    }
    store_piece<T>((T *)a.out + ((int64_t)p.b * a.N + i) * a.C + p.c0, dx, p.nv);
  }
}

// --------------------------------------------------------------------------- host side
// Column tiles, row lanes and row chunks: a row is cut into tiles of at most 256 pieces; the
// rows of a graph are cut so that about 2048 work-groups (eight per CU) share the batch, each
// with at least eight rows per row lane.
struct Shape {
  int lanes, tiles, rp, chunk_rows, chunks;
};
static Shape norm_shape(int B, int N, int C, int V, bool whole_blocks) {
  Shape s;
  int pieces = ceil_div(C, V);
  if (whole_blocks) pieces = ceil_div(C, kBlock8) * (kBlock8 / V);
  s.lanes = pieces < kThreads ? pieces : kThreads;
  s.tiles = ceil_div(pieces, s.lanes);
  s.rp = kThreads / s.lanes;
  const int64_t have = (int64_t)B * s.tiles;
  const int want = (int)(have >= 2048 ? 1 : (2048 + have - 1) / have);
  int rows = ceil_div(N, want), least = kBatch * s.rp;
  if (rows < least) rows = least;
  s.chunk_rows = ceil_div(rows, s.rp) * s.rp;
  s.chunks = ceil_div(N, s.chunk_rows);
  return s;
}

static int64_t norm_ws_floats(int B, int N, int C, int G) {
  // the most chunks any element type and tiling leads to: 2048 work-groups, or one per graph
  const int64_t chunks = (int64_t)2048 + B;
  return 2 * chunks * C + 2 * (int64_t)B * G;
}

}  // namespace gvae

using namespace gvae;

extern "C" {

int64_t gvae_group_norm_ws_bytes(int B, int N, int C, int G) {
  if (B <= 0 || N <= 0 || C <= 0 || G <= 0) return 0;
  return norm_ws_floats(B, N, C, G) * 4;
}


static int norm_check(const char *who, int dtype, int B, int N, int C, int G, int act, int64_t ld) {
  GVAE_REQUIRE(dtype_known(dtype), GVAE_EINVAL, "%s: unknown element type %d", who, dtype);
  GVAE_REQUIRE(B > 0 && N > 0 && C > 0 && G > 0 && C % G == 0, GVAE_EINVAL,
               "%s: bad sizes (graphs=%d rows=%d channels=%d groups=%d)", who, B, N, C, G);
  GVAE_REQUIRE(act >= GVAE_ACT_NONE && act <= GVAE_ACT_GELU, GVAE_EINVAL, "%s: unknown activation %d", who, act);
  GVAE_REQUIRE(ld >= C, GVAE_EINVAL, "%s: rows overlap (stride %lld for %d channels)", who, (long long)ld, C);
  GVAE_REQUIRE((int64_t)B * G < (1LL << 31) && (int64_t)N * (C / G) < (1LL << 31) && C <= 65535 * 32 &&
                   (int64_t)B + 2048 < (1LL << 31), GVAE_ELIMIT,
               "%s: too many groups or values per group (graphs=%d rows=%d channels=%d groups=%d)", who, B, N, C, G);
  return GVAE_OK;
}

int gvae_group_norm_fwd(const void *d_x, int dtype, int64_t batch_stride, int64_t row_stride, const int32_t *d_rows,
                        int B, int N, int C, int G, const float *d_weight, const float *d_bias, float eps, int act,
                        void *d_y, float *d_mean, float *d_rstd, int8_t *d_x8, uint8_t *d_x8_scales, int8_t *d_y8,
                        uint8_t *d_y8_scales, void *d_ws, void *stream) {
  GVAE_REQUIRE(d_x && d_y && d_mean && d_rstd && d_ws, GVAE_EINVAL, "group_norm_fwd: null pointer");
  GVAE_REQUIRE(!d_x8 == !d_x8_scales && !d_y8 == !d_y8_scales, GVAE_EINVAL,
               "group_norm_fwd: a checkpoint needs both its codes and its scales");
  GVAE_REQUIRE(eps > 0.0f && std::isfinite(eps), GVAE_EINVAL, "group_norm_fwd: eps must be positive");
  if (int rc = norm_check("group_norm_fwd", dtype, B, N, C, G, act, row_stride)) return rc;
  GVAE_REQUIRE(batch_stride >= 0, GVAE_EINVAL, "group_norm_fwd: negative stride");
  hipStream_t s = (hipStream_t)stream;
  NormArgs a{};
  a.x = d_x; a.xb = batch_stride; a.xr = row_stride; a.rows = d_rows;
  a.w = d_weight; a.b = d_bias; a.eps = eps; a.out = d_y; a.mean = d_mean; a.rstd = d_rstd;
  a.x8 = d_x8; a.x8s = d_x8_scales; a.y8 = d_y8; a.y8s = d_y8_scales;
  a.B = B; a.N = N; a.C = C; a.G = G; a.cpg = C / G;
  a.ld8 = ckpt8_ld(C); a.nb8 = ckpt8_blocks(C);
  const Shape sh = norm_shape(B, N, C, 16 / dtype_bytes(dtype), d_x8 || d_y8);
  a.lanes = sh.lanes; a.rp = sh.rp; a.chunk_rows = sh.chunk_rows; a.chunks = sh.chunks;
  a.part1 = (float *)d_ws;
  a.part2 = a.part1 + (int64_t)B * sh.chunks * C;
  const dim3 grid((unsigned)(B * sh.chunks), sh.tiles), joins((unsigned)(((int64_t)B * G + 3) / 4));
  GVAE_DTYPE_SWITCH(dtype, T, {
    hipLaunchKernelGGL((norm_stats_kernel<T>), grid, dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(norm_stats_join_kernel, joins, dim3(kThreads), 0, s, a);
    switch (act) {
      case GVAE_ACT_NONE: hipLaunchKernelGGL((norm_apply_kernel<T, GVAE_ACT_NONE>), grid, dim3(kThreads), 0, s, a); break;
      case GVAE_ACT_RELU: hipLaunchKernelGGL((norm_apply_kernel<T, GVAE_ACT_RELU>), grid, dim3(kThreads), 0, s, a); break;
      case GVAE_ACT_SILU: hipLaunchKernelGGL((norm_apply_kernel<T, GVAE_ACT_SILU>), grid, dim3(kThreads), 0, s, a); break;
      default: hipLaunchKernelGGL((norm_apply_kernel<T, GVAE_ACT_GELU>), grid, dim3(kThreads), 0, s, a); break;
    }
  });
  return check_launch("group_norm_fwd");
}

}  // extern "C"

template <class T, int ACT, bool KEPT>
static void norm_bwd_launch(const NormArgs &a, const Shape &sh, float *dw, float *db, hipStream_t s) {
  const dim3 grid((unsigned)(a.B * sh.chunks), sh.tiles), joins((unsigned)(((int64_t)a.B * a.G + 3) / 4));
  hipLaunchKernelGGL((norm_bwd_sums_kernel<T, ACT, KEPT>), grid, dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL(norm_bwd_join_kernel, joins, dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL((norm_bwd_apply_kernel<T, ACT, KEPT>), grid, dim3(kThreads), 0, s, a);
  if (dw || db)
    hipLaunchKernelGGL(norm_bwd_params_kernel, dim3(ceil_div(a.C, 16), 2), dim3(1024), 0, s, a.part1, a.part2,
                       (int64_t)a.B * sh.chunks, a.C, db, dw);
}
template <class T, bool KEPT>
static void norm_bwd_act(const NormArgs &a, const Shape &sh, int act, float *dw, float *db, hipStream_t s) {
  switch (act) {
    case GVAE_ACT_NONE: norm_bwd_launch<T, GVAE_ACT_NONE, KEPT>(a, sh, dw, db, s); break;
    case GVAE_ACT_RELU: norm_bwd_launch<T, GVAE_ACT_RELU, KEPT>(a, sh, dw, db, s); break;
    case GVAE_ACT_SILU: norm_bwd_launch<T, GVAE_ACT_SILU, KEPT>(a, sh, dw, db, s); break;
    default: norm_bwd_launch<T, GVAE_ACT_GELU, KEPT>(a, sh, dw, db, s); break;
  }
}

extern "C" {

int gvae_group_norm_bwd(const void *d_dy, int dtype, int64_t dy_batch_stride, int64_t dy_row_stride, const void *d_x,
                        int64_t batch_stride, int64_t row_stride, const int8_t *d_x8, const uint8_t *d_x8_scales,
                        const int32_t *d_rows, int B, int N, int C, int G, const float *d_weight,
                        const float *d_bias, const float *d_mean, const float *d_rstd, int act, void *d_dx,
                        float *d_dweight, float *d_dbias, void *d_ws, void *stream) {
  GVAE_REQUIRE(d_dy && d_dx && d_mean && d_rstd && d_ws, GVAE_EINVAL, "group_norm_bwd: null pointer");
  GVAE_REQUIRE(!d_dweight == !d_dbias, GVAE_EINVAL, "group_norm_bwd: weight and bias gradients come together");
  GVAE_REQUIRE(!d_x == (d_x8 && d_x8_scales) && !d_x8 == !d_x8_scales, GVAE_EINVAL,
               "group_norm_bwd: give either the input or its checkpoint (codes and scales)");
  if (int rc = norm_check("group_norm_bwd", dtype, B, N, C, G, act, dy_row_stride)) return rc;
  GVAE_REQUIRE(d_x8 || row_stride >= C, GVAE_EINVAL, "group_norm_bwd: rows of x overlap");
  GVAE_REQUIRE(dy_batch_stride >= 0 && batch_stride >= 0, GVAE_EINVAL, "group_norm_bwd: negative stride");
  NormArgs a{};
  a.dy = d_dy; a.dyb = dy_batch_stride; a.dyr = dy_row_stride;
  a.x = d_x; a.xb = batch_stride; a.xr = row_stride; a.codes = d_x8; a.scales = d_x8_scales; a.rows = d_rows;
  a.w = d_weight; a.b = d_bias; a.out = d_dx;
  a.mean = const_cast<float *>(d_mean); a.rstd = const_cast<float *>(d_rstd);   // (read only in the backward)
  a.B = B; a.N = N; a.C = C; a.G = G; a.cpg = C / G;
  a.ld8 = ckpt8_ld(C); a.nb8 = ckpt8_blocks(C);
  const Shape sh = norm_shape(B, N, C, 16 / dtype_bytes(dtype), false);
  a.lanes = sh.lanes; a.rp = sh.rp; a.chunk_rows = sh.chunk_rows; a.chunks = sh.chunks;
  a.part1 = (float *)d_ws;
  a.part2 = a.part1 + (int64_t)B * sh.chunks * C;
  a.A = a.part2 + (int64_t)B * sh.chunks * C;
  hipStream_t s = (hipStream_t)stream;
  GVAE_DTYPE_SWITCH(dtype, T, {
    if (d_x8) norm_bwd_act<T, true>(a, sh, act, d_dweight, d_dbias, s);
    else norm_bwd_act<T, false>(a, sh, act, d_dweight, d_dbias, s);
  });
  return check_launch("group_norm_bwd");
}

}  // extern "C"
