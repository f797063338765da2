// Group norm with an activation: gradients (gvae_norm.h has the mathematics and the two forms).
//
// Measured (medians of 400 calls).  Resident: 256 graphs of 250 rows, 512 channels, bf16, SiLU 51 us and 5 for
// dw and db (197 MB, 3.9 TB/s: loads, sums and writes of a slab follow one another, and registers leave few
// work-groups to a CU); 64 ragged graphs of at most 126 rows, 128 channels, float, from the checkpoint 7.2 us
// and 2.9.  Split: 16 graphs of 16384 rows, 512 channels, bf16, SiLU, from the checkpoint: sums 80 to 82 us
// (406 MB, 5 TB/s, bound by the vector units as much), join 6, second pass 120 (675 MB, 5.6 TB/s).
#include "gvae_norm.h"

namespace gvae {

// --------------------------------------------------------------------------- resident form
// A slab per work-group, graph after graph (graph_step apart): K pieces of dy and of x a thread, kept as
// they were loaded between the pass that sums and the pass that writes.  Every thread keeps its
// channels' share of dw and db over all its graphs; the work-group writes one row of partial sums.
template <class T, bool KEPT>
struct XPiece {
  typename Piece<T>::raw r;
  __device__ __forceinline__ void load(const NormArgs &a, int b, int i, int c0, const Cut<T> &cut) {
    r = cut.load((const T *)a.x + b * a.xb + (int64_t)i * a.xr);
  }
  __device__ __forceinline__ void cut(const Cut<T> &cut) { cut.cut(r); }
  __device__ __forceinline__ float at(int v) const { return (float)r[v]; }
  __device__ __forceinline__ void keep() { keep_raw<T>(r); }
};
template <class T>
struct XPiece<T, true> {
  static constexpr int V = Piece<T>::V;
  Codes<V> c;
  float p;
  __device__ __forceinline__ void load(const NormArgs &a, int b, int i, int c0, const Cut<T> &) {
    const int64_t row = (int64_t)b * a.N + i;
    c = load_codes<V>(a.codes + row * a.ld8 + c0);
    p = pow2_field(a.scales[row * a.nb8 + c0 / kBlock8]);
  }
  __device__ __forceinline__ void cut(const Cut<T> &) {}
  __device__ __forceinline__ float at(int v) const { return (float)(int8_t)(c.w[v >> 2] >> (8 * (v & 3))) * p; }
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) asm volatile("" : "+v"(c.w[q]));
  }
};

template <class T, bool KEPT, bool IN, int NT, int K>
__global__ __launch_bounds__(NT) void norm_bwd_resident_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V, E = IN ? 1 : V;
  __shared__ float ent[2][NT * V], grp[2][NT * E];
  const int id = xcd_run(blockIdx.x, gridDim.x), lane_b = id / a.nslab, s0 = (id - lane_b * a.nslab) * a.slab;
  const int s1 = s0 + a.slab < a.C ? s0 + a.slab : a.C;
  const int col = threadIdx.x % a.lanes, r0 = threadIdx.x / a.lanes;
  const int c0 = s0 + col * V, nv = s1 - c0 < V ? s1 - c0 : V;
  const bool on = r0 < a.rp && nv > 0;
  const int ng = (s1 - s0) / a.cpg, ge = IN ? a.cpg / V : a.cpg;
  const int mine = (threadIdx.x < a.rp * a.lanes) ? (int)threadIdx.x * E : -1;
  const Cut<T> cut(c0, nv, a.C);
  float w[V], bias[V], t1[V], t2[V];
  int group[E];
  load_params<V>(a.w, c0, nv, 1.0f, w);
  load_params<V>(a.b, c0, nv, 0.0f, bias);
#pragma unroll
  for (int v = 0; v < V; ++v) t1[v] = t2[v] = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e)
    group[e] = e == 0 ? (c0 < s1 ? c0 - s0 : 0) / a.cpg : group_after(group[e - 1], c0 + e - s0, a.cpg, ng);
  for (int b = lane_b; b < a.B; b += a.graph_step) {
    const int live = live_rows(a, b);
    const T *dy = (const T *)a.dy + b * a.dyb;
    typename Piece<T>::raw g[K];
    XPiece<T, KEPT> x[K];
#pragma unroll
    for (int u = 0; u < K; ++u) {
      const int i = r0 + u * a.rp;
      if (on && i < live) {
        g[u] = cut.load(dy + (int64_t)i * a.dyr);
        x[u].load(a, b, i, c0, cut);
      }
    }
    float mean[E], rstd[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int64_t q = (int64_t)b * a.G + s0 / a.cpg + group[e];
      mean[e] = a.mean[q];
      rstd[e] = a.rstd[q];
    }
    // (dz stays in fp32: the slope costs more than the registers)
    float p1[V], p2[V], dz[K][V];
#pragma unroll
    for (int v = 0; v < V; ++v) p1[v] = p2[v] = 0.0f;
#pragma unroll
    for (int u = 0; u < K; ++u)
      if (on && r0 + u * a.rp < live) {
        float h[V], s[V];
        cut.cut(g[u]);
        x[u].cut(cut);
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = (x[u].at(v) - mean[IN ? 0 : v]) * rstd[IN ? 0 : v];
        act_slopes<V, sizeof(T) == 4>(a.act, h, w, bias, s);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          dz[u][v] = (float)g[u][v] * s[v];
          p1[v] += dz[u][v];
          p2[v] = __fmaf_rn(dz[u][v], h[v], p2[v]);
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
    for (int u = 0; u < K; ++u) x[u].keep();
    __syncthreads();
    join_groups<2, NT * V, NT * E>(ent, a.lanes * E, ge, ng, a.rp, a.join, NT, grp);
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
      float dx[V];
#pragma unroll
      for (int v = 0; v < V; ++v) dx[v] = 0.0f;
      if (i < live)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int e = IN ? 0 : v;
          const float h = (x[u].at(v) - mean[e]) * rstd[e];
          dx[v] = rstd[e] * __fmaf_rn(dz[u][v], w[v], -__fmaf_rn(h, a2[e], a1[e]));
        }
      store_piece<false, T>((T *)a.out + ((int64_t)b * a.N + i) * a.C + c0, dx, nv);
    }
  }
  // this work-group's row of partial sums
  __syncthreads();
  if (mine >= 0)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      ent[0][threadIdx.x * V + v] = t1[v];
      ent[1][threadIdx.x * V + v] = t2[v];
    }
  __syncthreads();
  column_sums<2, NT>(ent, a.lanes * V, a.rp, [&](int c, const float *s) {
    if (s0 + c < s1) {
      a.part1[(int64_t)lane_b * a.C + s0 + c] = s[0];
      a.part2[(int64_t)lane_b * a.C + s0 + c] = s[1];
    }
  });
}

// --------------------------------------------------------------------------- split form
constexpr int kAhead = 4;   // rows of a thread requested at a time
template <class T, int ACT, bool KEPT>
__global__ __launch_bounds__(kThreads) void norm_bwd_sums_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V;
  __shared__ float sh[2][kThreads * V];
  const Place<V> p(a, true, false);
  float s1[V], s2[V];
#pragma unroll
  for (int v = 0; v < V; ++v) s1[v] = s2[v] = 0.0f;
  if (p.on && p.nv > 0) {
    const Scale<V, sizeof(T) == 2 && ACT != GVAE_ACT_RELU> k(a, p.b, p.c0, p.nv);
    const T *dy = (const T *)a.dy + p.b * a.dyb;
    const Cut<T> cut(p.c0, p.nv, a.C);
    for (int i0 = p.chunk * a.chunk_rows + p.r; i0 < p.row_end; i0 += kAhead * a.rp) {
      typename Piece<T>::raw g[kAhead];
      XPiece<T, KEPT> x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * a.rp;
        if (i >= p.row_end) break;
        g[u] = cut.load(dy + (int64_t)i * a.dyr);
        x[u].load(a, p.b, i, p.c0, cut);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (i0 + u * a.rp >= p.row_end) break;
        cut.cut(g[u]);
        x[u].cut(cut);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float c = k.centred(v, x[u].at(v));
          const float dz = (float)g[u][v] * act_slope<ACT, sizeof(T) == 4>(k.template pre<ACT>(v, c));
          s1[v] += dz;
          s2[v] = __fmaf_rn(dz, c, s2[v]);
        }
      }
    }
    float rstd[V];
    per_group<V>(a, a.rstd, p.b, p.c0, p.nv, rstd);
#pragma unroll
    for (int v = 0; v < V; ++v) s2[v] *= k.unit_of(rstd[v]);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sh[0][threadIdx.x * V + v] = s1[v];
    sh[1][threadIdx.x * V + v] = s2[v];
  }
  __syncthreads();
  const int wide = a.lanes * V;
  column_sums<2, kThreads>(sh, wide, a.rp, [&](int c, const float *s) {
    const int gc = blockIdx.y * wide + c;
    if (gc >= a.C) return;
    a.part1[(int64_t)blockIdx.x * a.C + gc] = s[0];
    a.part2[(int64_t)blockIdx.x * a.C + gc] = s[1];
  });
}

// A row of 16 channels of dw or db: the partial rows summed by NT / 16 row lanes, in their order
template <int NT>
__device__ __forceinline__ void param_sums(const float *__restrict__ p, int64_t n, int C, int c,
                                           float *__restrict__ out, float (*sh)[17]) {
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
  constexpr int L = NT / 16;
  c += cl;
  float s[8] = {};
  if (c < C) {
    int64_t r = rl;
    for (; r + 7 * L < n; r += 8 * L)
#pragma unroll
      for (int u = 0; u < 8; ++u) s[u] += p[(r + u * L) * C + c];
    for (; r < n; r += L) s[0] += p[r * C + c];
  }
  sh[rl][cl] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (rl == 0 && c < C) {
    float t = 0.0f;
    for (int k = 0; k < L; ++k) t += sh[k][cl];
    out[c] = t;
  }
}
__global__ __launch_bounds__(1024) void norm_bwd_params_kernel(NormArgs a, int64_t n, float *dw, float *db) {
  __shared__ float sh[64][17];
  param_sums<1024>(blockIdx.y ? a.part2 : a.part1, n, a.C, blockIdx.x * 16, blockIdx.y ? dw : db, sh);
}

// A1 and A2 of a group, a work-group per group, and behind the B * G groups the sums for dw and db
// (both read the partial rows, neither waits for the other)
template <int NT>
__global__ __launch_bounds__(NT) void norm_bwd_join_kernel(NormArgs a, float *dw, float *db) {
  __shared__ float sh[NT / 16][17];
  const int64_t q = blockIdx.x, groups = (int64_t)a.B * a.G;
  if (q >= groups) {
    const int k = (int)(q - groups), tiles = (a.C + 15) / 16;
    const bool second = k >= tiles;
    param_sums<NT>(second ? a.part2 : a.part1, (int64_t)a.B * a.chunks, a.C, (second ? k - tiles : k) * 16,
                   second ? dw : db, sh);
    return;
  }
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
  s1 = group_sum<NT>(s1, &sh[0][0]);
  s2 = group_sum<NT>(s2, &sh[0][0]);
  if (threadIdx.x == 0) {
    const int live = live_rows(a, b);
    const float m = (float)(live > 0 ? live : 1) * (float)a.cpg;
    a.A[2 * q] = s1 / m;
    a.A[2 * q + 1] = s2 / m;
  }
}

// (walked from the last graph to the first: what the sums read last may still be in the caches)
template <class T, int ACT, bool KEPT, bool PAST>
__global__ __launch_bounds__(kThreads) void norm_bwd_apply_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V;
  const Place<V> p(a, false, true);
  if (!p.on || p.nv <= 0) return;
  const int live = live_rows(a, p.b);
  const Scale<V, sizeof(T) == 2 && ACT != GVAE_ACT_RELU> k(a, p.b, p.c0, p.nv);
  float a1[V], a2[V], wr[V];       // dx = dz (w r) - (A1 r + h (A2 r))
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int64_t q = (int64_t)p.b * a.G + (p.c0 + (v < p.nv ? v : 0)) / a.cpg;
    const float r = k.rstd[v] * k.unit[v];
    a1[v] = a.A[2 * q] * r;
    a2[v] = a.A[2 * q + 1] * r;
    wr[v] = k.w[v] * k.rstd[v];
  }
  const T *dy = (const T *)a.dy + p.b * a.dyb;
  const Cut<T> cut(p.c0, p.nv, a.C);
  for (int i0 = p.chunk * a.chunk_rows + p.r; i0 < p.row_end; i0 += kAhead * a.rp) {
    typename Piece<T>::raw g[kAhead];
    XPiece<T, KEPT> x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * a.rp;
      if (i >= p.row_end || i >= live) break;
      g[u] = cut.load(dy + (int64_t)i * a.dyr);
      x[u].load(a, p.b, i, p.c0, cut);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * a.rp;
      if (i >= p.row_end) break;
      float dx[V];
#pragma unroll
      for (int v = 0; v < V; ++v) dx[v] = 0.0f;
      if (i < live) {
        cut.cut(g[u]);
        x[u].cut(cut);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float c = k.centred(v, x[u].at(v));
          const float dz = (float)g[u][v] * act_slope<ACT, sizeof(T) == 4>(k.template pre<ACT>(v, c));
          dx[v] = __fmaf_rn(dz, wr[v], -__fmaf_rn(c * k.unit[v], a2[v], a1[v]));
        }
      }
      store_piece<PAST, T>((T *)a.out + ((int64_t)p.b * a.N + i) * a.C + p.c0, dx, p.nv);
    }
  }
}

}  // namespace gvae

using namespace gvae;

static void params_launch(const NormArgs &a, int64_t rows, float *dw, float *db, hipStream_t s) {
  hipLaunchKernelGGL(norm_bwd_params_kernel, dim3(ceil_div(a.C, 16), 2), dim3(1024), 0, s, a, rows, dw, db);
}

template <class T, bool KEPT, bool IN>
static bool resident_launch(NormArgs &a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.graph_step * a.nslab));
  const int groups = a.slab / a.cpg;
#define RUN(NT, K)                                                                                  \
  do {                                                                                              \
    a.rp = NT / a.lanes;                                                                            \
    a.join = join_lanes(groups, NT);                                                                \
    if ((int64_t)a.rp * K >= a.N) {                                                                 \
      hipLaunchKernelGGL((norm_bwd_resident_kernel<T, KEPT, IN, NT, K>), grid, dim3(NT), 0, s, a);  \
      return true;                                                                                  \
    }                                                                                               \
  } while (0)
  if (a.lanes <= 64) RUN(64, 4);
  if (a.lanes <= 256) {
    RUN(256, 2);
    RUN(256, 4);
  }
  RUN(512, 4);
#undef RUN
  return false;
}
template <class T, int ACT, bool KEPT>
static void norm_bwd_launch(const NormArgs &a, const SplitShape &sh, float *dw, float *db, hipStream_t s) {
  const dim3 grid((unsigned)(a.B * sh.chunks), sh.tiles);
  const dim3 joins((unsigned)((int64_t)a.B * a.G + (dw ? 2 * ceil_div(a.C, 16) : 0)));
  hipLaunchKernelGGL((norm_bwd_sums_kernel<T, ACT, KEPT>), grid, dim3(kThreads), 0, s, a);
  if ((int64_t)sh.chunks * a.cpg <= 256 && (int64_t)a.B * sh.chunks <= 64)
    hipLaunchKernelGGL((norm_bwd_join_kernel<64>), joins, dim3(64), 0, s, a, dw, db);
  else
    hipLaunchKernelGGL((norm_bwd_join_kernel<512>), joins, dim3(512), 0, s, a, dw, db);
  auto kernel = a.past ? norm_bwd_apply_kernel<T, ACT, KEPT, true> : norm_bwd_apply_kernel<T, ACT, KEPT, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, a);
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
  GVAE_REQUIRE(d_dy && d_dx && d_mean && d_rstd, GVAE_EINVAL, "group_norm_bwd: null pointer");
  GVAE_REQUIRE(!d_dweight == !d_dbias, GVAE_EINVAL, "group_norm_bwd: weight and bias gradients come together");
  GVAE_REQUIRE(!d_x == (d_x8 && d_x8_scales) && !d_x8 == !d_x8_scales, GVAE_EINVAL,
               "group_norm_bwd: give either the input or its checkpoint (codes and scales)");
  GVAE_REQUIRE(aligned16(d_x8) && aligned16(d_ws), GVAE_EINVAL,
               "group_norm_bwd: codes or workspace not 16-byte aligned");
  if (int rc = norm_check("group_norm_bwd", dtype, B, N, C, G, act, dy_row_stride)) return rc;
  GVAE_REQUIRE(dy_batch_stride >= 0 && batch_stride >= 0 && row_stride >= 0, GVAE_EINVAL,
               "group_norm_bwd: negative stride");
  NormArgs a{};
  a.dy = d_dy; a.dyb = dy_batch_stride; a.dyr = dy_row_stride;
  a.x = d_x; a.xb = batch_stride; a.xr = row_stride; a.codes = d_x8; a.scales = d_x8_scales; a.rows = d_rows;
  a.w = d_weight; a.b = d_bias; a.out = d_dx;
  a.mean = const_cast<float *>(d_mean); a.rstd = const_cast<float *>(d_rstd);   // (read only in the backward)
  a.B = B; a.N = N; a.C = C; a.G = G; a.cpg = C / G;
  a.ld8 = ckpt8_ld(C); a.nb8 = ckpt8_blocks(C);
  a.past = (int64_t)B * N * C * dtype_bytes(dtype) >= kPastCaches;
  a.act = act;
  hipStream_t s = (hipStream_t)stream;
  const int V = 16 / dtype_bytes(dtype);
  const NormPlan plan = norm_plan(true, dtype, B, N, C, G, d_x8 != nullptr);
  GVAE_REQUIRE(d_ws, GVAE_EINVAL, "group_norm_bwd: null pointer");
  if (plan.resident) {
    a.slab = plan.rs.slab; a.nslab = plan.rs.nslab; a.lanes = plan.rs.lanes; a.graph_step = plan.graph_step;
    // (a single row of sums is the result)
    const bool direct = a.graph_step == 1 && d_dweight;
    a.part1 = direct ? d_dbias : (float *)d_ws;
    a.part2 = direct ? d_dweight : a.part1 + (int64_t)a.graph_step * C;
    const bool in = a.cpg % V == 0;
    bool ran = false;
    GVAE_DTYPE_SWITCH(dtype, T, {
      if (d_x8) ran = in ? resident_launch<T, true, true>(a, s) : resident_launch<T, true, false>(a, s);
      else ran = in ? resident_launch<T, false, true>(a, s) : resident_launch<T, false, false>(a, s);
    });
    GVAE_REQUIRE(ran, GVAE_ELIMIT, "group_norm_bwd: no kernel holds %d rows of %d pieces", N, a.lanes);
    if (d_dweight && !direct) params_launch(a, a.graph_step, d_dweight, d_dbias, s);
    return check_launch("group_norm_bwd");
  }
  const SplitShape &sh = plan.sp;
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
