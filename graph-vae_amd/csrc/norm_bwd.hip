// Group norm with an activation: gradients (gvae_norm.h has the mathematics and the two forms).
#include "gvae_norm.h"

namespace gvae {

// --------------------------------------------------------------------------- resident form
// A slab per work-group, graph after graph (graph_step apart): K pieces of dy and of x a thread, kept as
// they were loaded between the pass that sums and the pass that writes.  Every thread keeps its
// channels' share of dw and db over all its graphs; the work-group writes one row of partial sums.
template <class T, bool KEPT>
struct XPiece {
  typename Piece<T>::raw r;
  __device__ __forceinline__ void load(const NormArgs &a, int b, int i, int c0, int nv) {
    r = load_piece<T>((const T *)a.x + b * a.xb + (int64_t)i * a.xr + c0, nv);
  }
  __device__ __forceinline__ float at(int v) const { return (float)r[v]; }
  __device__ __forceinline__ void keep() { keep_raw<T>(r); }
};
template <class T>
struct XPiece<T, true> {
  static constexpr int V = Piece<T>::V;
  Codes<V> c;
  float p;
  __device__ __forceinline__ void load(const NormArgs &a, int b, int i, int c0, int) {
    const int64_t row = (int64_t)b * a.N + i;
    c = load_codes<V>(a.codes + row * a.ld8 + c0);
    p = pow2_field(a.scales[row * a.nb8 + c0 / kBlock8]);
  }
  __device__ __forceinline__ float at(int v) const { return (float)(int8_t)(c.w[v >> 2] >> (8 * (v & 3))) * p; }
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) asm volatile("" : "+v"(c.w[q]));
  }
};

template <class T, bool KEPT, bool IN, int NT, int K>
__global__ __launch_bounds__(NT) void norm_bwd_resident_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V, E = IN ? 1 : V;
  __shared__ float ent[2][NT * E], grp[2][NT * E];
  const int lane_b = blockIdx.x / a.nslab, s0 = (blockIdx.x - lane_b * a.nslab) * a.slab;
  const int s1 = s0 + a.slab < a.C ? s0 + a.slab : a.C;
  const int col = threadIdx.x % a.lanes, r0 = threadIdx.x / a.lanes;
  const int c0 = s0 + col * V, nv = s1 - c0 < V ? s1 - c0 : V;
  const bool on = r0 < a.rp && nv > 0;
  const int ng = (s1 - s0) / a.cpg, ge = IN ? a.cpg / V : a.cpg;
  const int mine = (threadIdx.x < a.rp * a.lanes) ? (int)threadIdx.x * E : -1;
  float w[V], bias[V], t1[V], t2[V];
  int group[E];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    w[v] = v < nv ? (a.w ? a.w[c0 + v] : 1.0f) : 0.0f;
    bias[v] = v < nv && a.b ? a.b[c0 + v] : 0.0f;
    t1[v] = t2[v] = 0.0f;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) group[e] = ((c0 + e < s1 ? c0 + e : s1 - 1) - s0) / a.cpg;
  for (int b = lane_b; b < a.B; b += a.graph_step) {
    const int live = live_rows(a, b);
    const T *dy = (const T *)a.dy + b * a.dyb + c0;
    typename Piece<T>::raw g[K];
    XPiece<T, KEPT> x[K];
#pragma unroll
    for (int u = 0; u < K; ++u) {
      const int i = r0 + u * a.rp;
      if (on && i < live) {
        g[u] = load_piece<T>(dy + (int64_t)i * a.dyr, nv);
        x[u].load(a, b, i, c0, nv);
      }
    }
    float mean[E], rstd[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int64_t q = (int64_t)b * a.G + s0 / a.cpg + group[e];
      mean[e] = a.mean[q];
      rstd[e] = a.rstd[q];
    }
    float p1[V], p2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) p1[v] = p2[v] = 0.0f;
#pragma unroll
    for (int u = 0; u < K; ++u)
      if (on && r0 + u * a.rp < live) {
        float h[V], dz[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[v] = (x[u].at(v) - mean[IN ? 0 : v]) * rstd[IN ? 0 : v];
          dz[v] = h[v] * w[v] + bias[v];
        }
        act_slopes<V>(a.act, dz);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = v < nv ? (float)g[u][v] * dz[v] : 0.0f;
          p1[v] += d;
          p2[v] += v < nv ? d * h[v] : 0.0f;
        }
      }
    {
      float e1[E], e2[E];
#pragma unroll
      for (int e = 0; e < E; ++e) e1[e] = e2[e] = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        e1[IN ? 0 : v] = __fmaf_rn(w[v], p1[v], e1[IN ? 0 : v]);
        e2[IN ? 0 : v] = __fmaf_rn(w[v], p2[v], e2[IN ? 0 : v]);
        t1[v] += p1[v];
        t2[v] += p2[v];
      }
      if (mine >= 0)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          ent[0][mine + e] = e1[e];
          ent[1][mine + e] = e2[e];
        }
    }
#pragma unroll
    for (int u = 0; u < K; ++u) {
      keep_raw<T>(g[u]);
      x[u].keep();
    }
    __syncthreads();
    join_groups<2, NT * E>(ent, a.lanes * E, ge, ng, a.rp, a.join, NT, grp);
    __syncthreads();
    const float inv = 1.0f / ((float)(live > 0 ? live : 1) * (float)a.cpg);
    float a1[E], a2[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      a1[e] = grp[0][group[e]] * inv;
      a2[e] = grp[1][group[e]] * inv;
    }
    if (!on) continue;
#pragma unroll
    for (int u = 0; u < K; ++u) {
      const int i = r0 + u * a.rp;
      if (i >= a.N) break;
      float h[V], dx[V];
      if (i < live) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[v] = (x[u].at(v) - mean[IN ? 0 : v]) * rstd[IN ? 0 : v];
          dx[v] = h[v] * w[v] + bias[v];
        }
        act_slopes<V>(a.act, dx);
#pragma unroll
        for (int v = 0; v < V; ++v)
          dx[v] = rstd[IN ? 0 : v] * ((float)g[u][v] * dx[v] * w[v] - __fmaf_rn(h[v], a2[IN ? 0 : v], a1[IN ? 0 : v]));
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) dx[v] = 0.0f;
      }
      store_piece<T>((T *)a.out + ((int64_t)b * a.N + i) * a.C + c0, dx, nv);
    }
  }
  // the row lanes of a channel, in their order, one channel of every piece at a time
#pragma unroll
  for (int v = 0; v < V; ++v) {
    __syncthreads();
    ent[0][threadIdx.x] = t1[v];
    ent[1][threadIdx.x] = t2[v];
    __syncthreads();
    if (threadIdx.x < a.lanes && v < nv) {
      float u1 = 0.0f, u2 = 0.0f;
      for (int r = 0; r < a.rp; ++r) {
        u1 += ent[0][r * a.lanes + threadIdx.x];
        u2 += ent[1][r * a.lanes + threadIdx.x];
      }
      a.part1[(int64_t)lane_b * a.C + c0 + v] = u1;
      a.part2[(int64_t)lane_b * a.C + c0 + v] = u2;
    }
  }
}

// --------------------------------------------------------------------------- split form
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

// A1 and A2 of a group, a work-group per group
template <int NT>
__global__ __launch_bounds__(NT) void norm_bwd_join_kernel(NormArgs a) {
  __shared__ float sh[NT / 64];
  const int64_t q = blockIdx.x;
  const int b = (int)(q / a.G), g = (int)(q - (int64_t)b * a.G);
  const int64_t base = (int64_t)b * a.chunks * a.C + g * a.cpg;
  float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 4
  for (int e = threadIdx.x; e < a.chunks * a.cpg; e += NT) {
    const int k = e / a.cpg, c = e - k * a.cpg;
    const float w = a.w ? a.w[g * a.cpg + c] : 1.0f;
    s1 = __fmaf_rn(w, a.part1[base + (int64_t)k * a.C + c], s1);
    s2 = __fmaf_rn(w, a.part2[base + (int64_t)k * a.C + c], s2);
  }
  s1 = group_sum<NT>(s1, sh);
  s2 = group_sum<NT>(s2, sh);
  if (threadIdx.x == 0) {
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


}  // namespace gvae

using namespace gvae;

static void params_launch(const NormArgs &a, int64_t rows, float *dw, float *db, hipStream_t s) {
  hipLaunchKernelGGL(norm_bwd_params_kernel, dim3(ceil_div(a.C, 16), 2), dim3(1024), 0, s, a.part1, a.part2, rows, a.C,
                     db, dw);
}

template <class T, bool KEPT, bool IN>
static void resident_launch(NormArgs &a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.graph_step * a.nslab));
  const int groups = a.slab / a.cpg;
#define RUN(NT, K)                                                                                  \
  do {                                                                                              \
    a.rp = NT / a.lanes;                                                                            \
    a.join = join_lanes(groups, NT);                                                                \
    if ((int64_t)a.rp * K >= a.N) {                                                                 \
      hipLaunchKernelGGL((norm_bwd_resident_kernel<T, KEPT, IN, NT, K>), grid, dim3(NT), 0, s, a);  \
      return;                                                                                       \
    }                                                                                               \
  } while (0)
  if (a.lanes <= 64) RUN(64, 4);
  if (a.lanes <= 256) {
    RUN(256, 2);
    RUN(256, 4);
  }
  RUN(512, 4);
  RUN(512, 8);
#undef RUN
}
static bool resident_fits(int N, int lanes) { return lanes <= 512 && (int64_t)(512 / lanes) * 8 >= N; }

template <class T, int ACT, bool KEPT>
static void norm_bwd_launch(const NormArgs &a, const SplitShape &sh, float *dw, float *db, hipStream_t s) {
  const dim3 grid((unsigned)(a.B * sh.chunks), sh.tiles), joins((unsigned)((int64_t)a.B * a.G));
  hipLaunchKernelGGL((norm_bwd_sums_kernel<T, ACT, KEPT>), grid, dim3(kThreads), 0, s, a);
  if ((int64_t)sh.chunks * a.cpg <= 256) hipLaunchKernelGGL((norm_bwd_join_kernel<64>), joins, dim3(64), 0, s, a);
  else hipLaunchKernelGGL((norm_bwd_join_kernel<512>), joins, dim3(512), 0, s, a);
  hipLaunchKernelGGL((norm_bwd_apply_kernel<T, ACT, KEPT>), grid, dim3(kThreads), 0, s, a);
  if (dw) params_launch(a, (int64_t)a.B * sh.chunks, dw, db, s);
}
template <class T, bool KEPT>
static void norm_bwd_act(const NormArgs &a, const SplitShape &sh, int act, float *dw, float *db, hipStream_t s) {
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
  a.act = act;
  hipStream_t s = (hipStream_t)stream;
  const int V = 16 / dtype_bytes(dtype);
  ResidentShape rs;
  if (resident_shape(B, N, C, a.cpg, V, d_x8 ? V : 1, 4096, 512, &rs) && resident_fits(N, rs.lanes)) {
    a.slab = rs.slab; a.nslab = rs.nslab; a.lanes = rs.lanes;
    // about 1024 work-groups, each with a row of partial sums; a single row is the result
    a.graph_step = rs.nslab >= 1024 ? 1 : 1024 / rs.nslab;
    if (a.graph_step > B) a.graph_step = B;
    const bool direct = a.graph_step == 1 && d_dweight;
    a.part1 = direct ? d_dbias : (float *)d_ws;
    a.part2 = direct ? d_dweight : a.part1 + (int64_t)a.graph_step * C;
    const bool in = a.cpg % V == 0;
    GVAE_DTYPE_SWITCH(dtype, T, {
      if (d_x8 && in) resident_launch<T, true, true>(a, s);
      else if (d_x8) resident_launch<T, true, false>(a, s);
      else if (in) resident_launch<T, false, true>(a, s);
      else resident_launch<T, false, false>(a, s);
    });
    if (d_dweight && !direct) params_launch(a, a.graph_step, d_dweight, d_dbias, s);
    return check_launch("group_norm_bwd");
  }
  const SplitShape sh = split_shape(B, N, C, V, false);
  a.lanes = sh.lanes; a.rp = sh.rp; a.chunk_rows = sh.chunk_rows; a.chunks = sh.chunks;
  a.part1 = (float *)d_ws;
  a.part2 = a.part1 + (int64_t)B * sh.chunks * C;
  a.A = a.part2 + (int64_t)B * sh.chunks * C;
  GVAE_DTYPE_SWITCH(dtype, T, {
    if (d_x8) norm_bwd_act<T, true>(a, sh, act, d_dweight, d_dbias, s);
    else norm_bwd_act<T, false>(a, sh, act, d_dweight, d_dbias, s);
  });
  return check_launch("group_norm_bwd");
}

}  // extern "C"
