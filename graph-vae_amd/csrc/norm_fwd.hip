// Group norm with an activation: forward (gvae_norm.h has the mathematics and the two forms).
//
// Split form: what a chunk leaves is one (mean, M2) pair per channel, combined as n, mean, M2 with
// M2 = M2a + M2b + d^2 na nb / n, so no square of an uncentred value is ever summed.
//
// Measured (bf16, SiLU; medians of 400 calls).  Resident: 256 graphs of 250 rows, 512 channels 32 us (131 MB,
// 4.1 TB/s); in a few MB the latency of one work-group remains: 256 graphs of 32 rows, 128 channels, float,
// with both checkpoints 9.0 us, a graph of 20 rows 5.3.  Split: 4 graphs of 65536 rows, 320 channels: sums 33 us
// (5.1 TB/s), join 6, second pass 57 (336 MB, 5.9 TB/s); 192 ragged graphs of 1000 rows, 512 channels, with
// both checkpoints: 25 + 6 + 93.
#include "gvae_norm.h"

namespace gvae {

// --------------------------------------------------------------------------- resident form
// One graph and one slab per work-group; K pieces a thread, kept as they were loaded.  Two passes over
// the registers (mean, then centred squares).  IN: a piece lies inside one group (one entry per
// thread in LDS), else every channel has its own.
template <class T, bool IN, int NT, int K, bool PAST>
__global__ __launch_bounds__(NT) void norm_resident_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V, E = IN ? 1 : V;
  __shared__ float ent[1][NT * E], grp[2][NT * E];
  const int id = xcd_run(blockIdx.x, gridDim.x), b = id / a.nslab, s0 = (id - b * a.nslab) * a.slab;
  const int s1 = s0 + a.slab < a.C ? s0 + a.slab : a.C;
  const int col = threadIdx.x % a.lanes, r0 = threadIdx.x / a.lanes;
  const int c0 = s0 + col * V, nv = s1 - c0 < V ? s1 - c0 : V;
  const bool on = r0 < a.rp && nv > 0;
  const int live = live_rows(a, b), ng = (s1 - s0) / a.cpg, g0 = s0 / a.cpg;
  const T *x = (const T *)a.x + b * a.xb;
  const Cut<T> cut(c0, nv, a.C);
  typename Piece<T>::raw k[K];
#pragma unroll
  for (int u = 0; u < K; ++u) {
    const int i = r0 + u * a.rp;
    k[u] = typename Piece<T>::raw{};
    if (on && i < live) k[u] = cut.load(x + (int64_t)i * a.xr);
  }
  float w[V], bias[V];
  load_params<V>(a.w, c0, nv, 1.0f, w);
  load_params<V>(a.b, c0, nv, 0.0f, bias);
  // this thread's entry e of group entries starts at the piece's own group
  const int mine = (threadIdx.x < a.rp * a.lanes) ? (int)threadIdx.x * E : -1;
  const int ge = IN ? a.cpg / V : a.cpg;
  const float inv = 1.0f / ((float)(live > 0 ? live : 1) * (float)a.cpg);
  float mean[E], rstd[E];
  {
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = 0.0f;
#pragma unroll
    for (int u = 0; u < K; ++u) {
      if (on) cut.cut(k[u]);
#pragma unroll
      for (int v = 0; v < V; ++v) s[IN ? 0 : v] += (float)k[u][v];
    }
    if (mine >= 0)
#pragma unroll
      for (int e = 0; e < E; ++e) ent[0][mine + e] = s[e];
  }
#pragma unroll
  for (int u = 0; u < K; ++u) keep_raw<T>(k[u]);
  __syncthreads();
  join_groups<1, NT * E, NT * E>(ent, a.lanes * E, ge, ng, a.rp, a.join, NT, grp);
  __syncthreads();
  int group[E];
#pragma unroll
  for (int e = 0; e < E; ++e)
    group[e] = e == 0 ? (c0 < s1 ? c0 - s0 : 0) / a.cpg : group_after(group[e - 1], c0 + e - s0, a.cpg, ng);
  // (0 behind the slab's last channel, as rstd below: what a lane there adds to a block's checkpoint must not
  // come from another group, whose mean may be large or not finite)
#pragma unroll
  for (int e = 0; e < E; ++e) mean[e] = c0 + e < s1 ? grp[0][group[e]] * inv : 0.0f;
  {
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = 0.0f;
#pragma unroll
    for (int u = 0; u < K; ++u)
      if (on && r0 + u * a.rp < live)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = (float)k[u][v] - mean[IN ? 0 : v];
          s[IN ? 0 : v] = __fmaf_rn(d, d, s[IN ? 0 : v]);
        }
    if (mine >= 0)
#pragma unroll
      for (int e = 0; e < E; ++e) ent[0][mine + e] = s[e];
  }
#pragma unroll
  for (int u = 0; u < K; ++u) keep_raw<T>(k[u]);
  __syncthreads();
  join_groups<1, NT * E, NT * E>(ent, a.lanes * E, ge, ng, a.rp, a.join, NT, grp + 1);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) rstd[e] = c0 + e < s1 ? 1.0f / sqrtf(grp[1][group[e]] * inv + a.eps) : 0.0f;
  for (int g = threadIdx.x; g < ng; g += NT) {
    const int64_t q = (int64_t)b * a.G + g0 + g;
    a.mean[q] = grp[0][g] * inv;
    a.rstd[q] = 1.0f / sqrtf(grp[1][g] * inv + a.eps);
  }
  if (r0 >= a.rp) return;
#pragma unroll
  for (int u = 0; u < K; ++u) {
    const int i = r0 + u * a.rp;
    if (i >= a.N) break;
    float xf[V], y[V];
#pragma unroll
    for (int v = 0; v < V; ++v) xf[v] = y[v] = 0.0f;
    if (i < live) {      // (channels behind the last: weight and bias 0, and every activation of 0 is 0)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        xf[v] = (float)k[u][v];
        y[v] = (xf[v] - mean[IN ? 0 : v]) * rstd[IN ? 0 : v];
      }
      act_values<V, sizeof(T) == 4>(a.act, y, w, bias, y);
    }
    const int64_t row = (int64_t)b * a.N + i;
    if (nv > 0) store_piece<PAST, T>((T *)a.out + row * a.C + c0, y, nv);
    // (the lanes of a block share a row: with checkpoints kept, `lanes` is a whole number of blocks)
    const int nc = a.ld8 - c0;
    const bool first = c0 % kBlock8 == 0 && nv > 0;
    auto leave = [&](const float *f, int8_t *codes, uint8_t *scales) {
      codes += row * a.ld8 + c0;
      scales += row * a.nb8 + c0 / kBlock8;
      if (i < live) emit8<PAST, V>(f, codes, nc, scales, first);
      else emit8_zeros<PAST, V>(codes, nc, scales, first);
    };
    if (a.x8) leave(xf, a.x8, a.x8s);
    if (a.y8) leave(rounded<T>(y), a.y8, a.y8s);
  }
}

// --------------------------------------------------------------------------- split form
// (n, mean, M2) of every channel over a chunk's live rows
template <class T>
__global__ __launch_bounds__(kThreads) void norm_stats_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V;
  __shared__ float sh_mean[kThreads * V], sh_m2[kThreads * V];
  __shared__ int sh_n[kThreads];
  const Place<V> p(a, true, false);
  const int row0 = p.chunk * a.chunk_rows;
  float mean[V], m2[V];
  int n = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) mean[v] = m2[v] = 0.0f;
  if (p.on && p.nv > 0) {
    const T *x = (const T *)a.x + p.b * a.xb;
    const Cut<T> cut(p.c0, p.nv, a.C);
    typename Piece<T>::raw k[kBatch], ahead[kBatch];
    auto request = [&](int i, typename Piece<T>::raw *to) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + u * a.rp < p.row_end) to[u] = cut.load(x + (int64_t)(i + u * a.rp) * a.xr);
    };
    request(row0 + p.r, ahead);
    for (int i = row0 + p.r; i < p.row_end; i += kBatch * a.rp) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        k[u] = ahead[u];
        cut.cut(k[u]);
      }
      request(i + kBatch * a.rp, ahead);
      const int left = (p.row_end - i + a.rp - 1) / a.rp, cnt = left < kBatch ? left : kBatch;
      const float inv = 1.0f / (float)cnt;
      const float share = (float)cnt / (float)(n + cnt), cross = (float)n * share;
      auto batch = [&](auto whole) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float s = 0.0f;
#pragma unroll
          for (int u = 0; u < kBatch; ++u) if (whole || u < cnt) s += (float)k[u][v];
          const float mb = s * inv;
          float q = 0.0f;
#pragma unroll
          for (int u = 0; u < kBatch; ++u) if (whole || u < cnt) {
            const float d = (float)k[u][v] - mb;
            q = __fmaf_rn(d, d, q);
          }
          const float d = mb - mean[v];
          mean[v] = __fmaf_rn(d, share, mean[v]);
          m2[v] += __fmaf_rn(d * cross, d, q);   // (first batch: cross is 0, and d * d alone may overflow)
        }
      };
      if (cnt == kBatch) batch(std::true_type{});
      else batch(std::false_type{});
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

// mean and 1/sqrt(var + eps) of a group from its chunks' channels, a work-group per group.  One pass in
// fp64: sum n mean and sum (M2 + n mean^2), whose difference keeps 2^-53 (mean / deviation)^2.
template <int NT>
__global__ __launch_bounds__(NT) void norm_stats_join_kernel(NormArgs a) {
  __shared__ double sh[2][NT / 64];
  const int64_t q = blockIdx.x;
  const int b = (int)(q / a.G), g = (int)(q - (int64_t)b * a.G);
  const int live = live_rows(a, b), total = a.chunks * a.cpg;
  const float *p1 = a.part1 + (int64_t)b * a.chunks * a.C + g * a.cpg;
  const float *p2 = a.part2 + (int64_t)b * a.chunks * a.C + g * a.cpg;
  double s = 0.0, v = 0.0;
#pragma unroll 4
  for (int e = threadIdx.x; e < total; e += NT) {
    const int k = e / a.cpg, c = e - k * a.cpg;
    const int n = live - k * a.chunk_rows;
    const double rows = (double)(n < 0 ? 0 : (n > a.chunk_rows ? a.chunk_rows : n));
    const double mu = (double)p1[(int64_t)k * a.C + c];
    s = fma(rows, mu, s);
    v += fma(rows * mu, mu, (double)p2[(int64_t)k * a.C + c]);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    s += __shfl_xor(s, off, 64);
    v += __shfl_xor(v, off, 64);
  }
  if (NT > 64) {
    if ((threadIdx.x & 63) == 0) {
      sh[0][threadIdx.x >> 6] = s;
      sh[1][threadIdx.x >> 6] = v;
    }
    __syncthreads();
    s = v = 0.0;
    for (int k = 0; k < NT / 64; ++k) {
      s += sh[0][k];
      v += sh[1][k];
    }
  }
  if (threadIdx.x == 0) {
    const double m = (double)(live > 0 ? live : 1) * (double)a.cpg;
    const double mu = s / m, var = v / m - mu * mu;
    a.mean[q] = (float)mu;
    // (an infinity or a NaN in the group: var is NaN and stays one)
    a.rstd[q] = 1.0f / sqrtf((float)(var < 0.0 ? 0.0 : var) + a.eps);
  }
}

// Rows of a thread are requested kAhead at a time.  The graphs are walked from the last to the first: what
// the statistics read last may still be in the caches.
constexpr int kAhead = 4;
template <class T, int ACT, bool PAST>
__global__ __launch_bounds__(kThreads) void norm_apply_kernel(NormArgs a) {
  constexpr int V = Piece<T>::V;
  const Place<V> p(a, false, true);
  if (!p.on) return;
  const int live = live_rows(a, p.b);
  const Scale<V, sizeof(T) == 2 && ACT != GVAE_ACT_RELU> k(a, p.b, p.c0, p.nv);
  const T *x = (const T *)a.x + p.b * a.xb;
  const Cut<T> cut(p.c0, p.nv, a.C);
  for (int i0 = p.chunk * a.chunk_rows + p.r; i0 < p.row_end; i0 += kAhead * a.rp) {
    typename Piece<T>::raw r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * a.rp;
      r[u] = typename Piece<T>::raw{};
      if (i < p.row_end && i < live && p.nv > 0) r[u] = cut.load(x + (int64_t)i * a.xr);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * a.rp;
      if (i >= p.row_end) break;
      float xf[V], y[V];
#pragma unroll
      for (int v = 0; v < V; ++v) xf[v] = y[v] = 0.0f;
      if (p.nv > 0) cut.cut(r[u]);
      if (i < live) {    // (channels behind the last: weight and bias 0, and every activation of 0 is 0)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          xf[v] = (float)r[u][v];
          y[v] = act_value<ACT, sizeof(T) == 4>(k.template pre<ACT>(v, k.centred(v, xf[v])));
        }
      }
      const int64_t row = (int64_t)p.b * a.N + i;
      if (p.nv > 0) store_piece<PAST, T>((T *)a.out + row * a.C + p.c0, y, p.nv);
      // (the lanes of a block share a row: with checkpoints kept, `lanes` is a whole number of blocks)
      const int nc = a.ld8 - p.c0;
      const bool first = p.c0 % kBlock8 == 0 && p.nv > 0;
      auto leave = [&](const float *f, int8_t *codes, uint8_t *scales) {
        codes += row * a.ld8 + p.c0;
        scales += row * a.nb8 + p.c0 / kBlock8;
        if (i < live) emit8<PAST, V>(f, codes, nc, scales, first);
        else emit8_zeros<PAST, V>(codes, nc, scales, first);
      };
      if (a.x8) leave(xf, a.x8, a.x8s);
      if (a.y8) leave(rounded<T>(y), a.y8, a.y8s);
    }
  }
}

template <class T, int ACT>
static void apply_launch(const NormArgs &a, dim3 grid, hipStream_t s) {
  auto kernel = a.past ? norm_apply_kernel<T, ACT, true> : norm_apply_kernel<T, ACT, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, a);
}

template <class T, bool IN>
static bool resident_launch(NormArgs &a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.B * a.nslab));
  const int groups = a.slab / a.cpg;
#define RUN(NT, K)                                                                        \
  do {                                                                                    \
    a.rp = NT / a.lanes;                                                                  \
    a.join = join_lanes(groups, NT);                                                      \
    if ((int64_t)a.rp * K >= a.N) {                                                       \
      auto kernel = a.past ? norm_resident_kernel<T, IN, NT, K, true> : norm_resident_kernel<T, IN, NT, K, false>; \
      hipLaunchKernelGGL(kernel, grid, dim3(NT), 0, s, a);                                \
      return true;                                                                        \
    }                                                                                     \
  } while (0)
  if (a.lanes <= 64) RUN(64, 4);
  if (a.lanes <= 256) {
    RUN(256, 2);
    RUN(256, 4);
    RUN(256, 8);
    RUN(256, 16);
  }
  RUN(1024, 8);
#undef RUN
  return false;
}

}  // namespace gvae

using namespace gvae;

extern "C" {

int64_t gvae_group_norm_ws_bytes(int backward, int dtype, int B, int N, int C, int G, int checkpoints) {
  if (!dtype_known(dtype) || B <= 0 || N <= 0 || C <= 0 || G <= 0 || C % G) return 0;
  return 4 * norm_plan(backward != 0, dtype, B, N, C, G, checkpoints != 0).floats;
}

}  // extern "C"

int gvae::norm_check(const char *who, int dtype, int B, int N, int C, int G, int act, int64_t ld) {
  GVAE_REQUIRE(dtype_known(dtype), GVAE_EINVAL, "%s: unknown element type %d", who, dtype);
  GVAE_REQUIRE(B > 0 && N > 0 && C > 0 && G > 0 && C % G == 0, GVAE_EINVAL,
               "%s: bad sizes (graphs=%d rows=%d channels=%d groups=%d)", who, B, N, C, G);
  GVAE_REQUIRE(act >= GVAE_ACT_NONE && act <= GVAE_ACT_GELU, GVAE_EINVAL, "%s: unknown activation %d", who, act);
  GVAE_REQUIRE(ld >= 0, GVAE_EINVAL, "%s: negative stride", who);
  // (grids of up to 1024 threads a group or slab stay under 2^32 threads; row numbers and the values of a
  // group stay under 2^30)
  GVAE_REQUIRE((int64_t)B * G < (1LL << 22) && (int64_t)N * (C / G) < (1LL << 30) && C <= (1 << 20), GVAE_ELIMIT,
               "%s: too many groups or values per group (graphs=%d rows=%d channels=%d groups=%d)", who, B, N, C, G);
  return GVAE_OK;
}


extern "C" {

int gvae_group_norm_fwd(const void *d_x, int dtype, int64_t batch_stride, int64_t row_stride, const int32_t *d_rows,
                        int B, int N, int C, int G, const float *d_weight, const float *d_bias, float eps, int act,
                        void *d_y, float *d_mean, float *d_rstd, int8_t *d_x8, uint8_t *d_x8_scales, int8_t *d_y8,
                        uint8_t *d_y8_scales, void *d_ws, void *stream) {
  GVAE_REQUIRE(d_x && d_y && d_mean && d_rstd, GVAE_EINVAL, "group_norm_fwd: null pointer");
  GVAE_REQUIRE(!d_x8 == !d_x8_scales && !d_y8 == !d_y8_scales, GVAE_EINVAL,
               "group_norm_fwd: a checkpoint needs both its codes and its scales");
  GVAE_REQUIRE(aligned16(d_x8) && aligned16(d_y8) && aligned16(d_ws), GVAE_EINVAL,
               "group_norm_fwd: codes or workspace not 16-byte aligned");
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
  a.past = (int64_t)B * N * C * dtype_bytes(dtype) >= kPastCaches;
  a.act = act;
  const int V = 16 / dtype_bytes(dtype);
  const NormPlan plan = norm_plan(false, dtype, B, N, C, G, d_x8 || d_y8);
  GVAE_REQUIRE(d_ws || !plan.floats, GVAE_EINVAL, "group_norm_fwd: null pointer");
  if (plan.resident) {
    const ResidentShape &rs = plan.rs;
    a.slab = rs.slab; a.nslab = rs.nslab; a.lanes = rs.lanes;
    bool ran = false;
    GVAE_DTYPE_SWITCH(dtype, T, ran = a.cpg % V == 0 ? resident_launch<T, true>(a, s) : resident_launch<T, false>(a, s));
    GVAE_REQUIRE(ran, GVAE_ELIMIT, "group_norm_fwd: no kernel holds %d rows of %d pieces", N, a.lanes);
    return check_launch("group_norm_fwd");
  }
  const SplitShape &sh = plan.sp;
  a.lanes = sh.lanes; a.rp = sh.rp; a.chunk_rows = sh.chunk_rows; a.chunks = sh.chunks;
  a.part1 = (float *)d_ws;
  a.part2 = a.part1 + (int64_t)B * sh.chunks * C;
  const dim3 grid((unsigned)(B * sh.chunks), sh.tiles), joins((unsigned)((int64_t)B * G));
  GVAE_DTYPE_SWITCH(dtype, T, {
    hipLaunchKernelGGL((norm_stats_kernel<T>), grid, dim3(kThreads), 0, s, a);
    if ((int64_t)sh.chunks * a.cpg <= 256) hipLaunchKernelGGL((norm_stats_join_kernel<64>), joins, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((norm_stats_join_kernel<512>), joins, dim3(512), 0, s, a);
    switch (act) {
      case GVAE_ACT_NONE: apply_launch<T, GVAE_ACT_NONE>(a, grid, s); break;
      case GVAE_ACT_RELU: apply_launch<T, GVAE_ACT_RELU>(a, grid, s); break;
      case GVAE_ACT_SILU: apply_launch<T, GVAE_ACT_SILU>(a, grid, s); break;
      default: apply_launch<T, GVAE_ACT_GELU>(a, grid, s); break;
    }
  });
  return check_launch("group_norm_fwd");
}

}  // extern "C"

