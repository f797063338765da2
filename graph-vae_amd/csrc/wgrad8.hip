// Weight and bias gradient of a linear layer y = x W^T + b from the 8-bit checkpoint of its input:
//   dW[o,i] = sum_t dY[t,o] * code[t,i] * 2^(s[t,i/32] - 127),   db[o] = sum_t dY[t,o]
// Rows are split over work-groups; the parts are summed in their order by a second launch.
#include "gvae_ckpt8.h"

namespace gvae {

struct WgradArgs {
  const void *dy;
  const int8_t *codes;
  const uint8_t *scales;
  void *dw, *db;
  float *part, *part_b;       // (splits, O, I) and (splits, O)
  int64_t rows, ldy;
  int O, I, ld8, nb8, splits;
  int64_t split_rows;
};

constexpr int kTile = 64, kDepth = 16;

template <class T>
__global__ __launch_bounds__(256) void wgrad8_kernel(WgradArgs a) {
  __shared__ float sa[kDepth][kTile], sb[kDepth][kTile + 4];
  const int i0 = blockIdx.x * kTile, o0 = blockIdx.y * kTile, tid = threadIdx.x;
  const int tx = tid & 15, ty = tid >> 4;
  const int64_t t0 = (int64_t)blockIdx.z * a.split_rows;
  const int64_t t1 = t0 + a.split_rows < a.rows ? t0 + a.split_rows : a.rows;
  float acc[4][4] = {}, bias[4] = {};
  for (int64_t t = t0; t < t1; t += kDepth) {
    for (int e = tid; e < kDepth * kTile; e += 256) {
      const int k = e / kTile, c = e % kTile;
      const bool row = t + k < t1;
      sa[k][c] = row && o0 + c < a.O ? (float)((const T *)a.dy)[(t + k) * a.ldy + o0 + c] : 0.0f;
      float x = 0.0f;
      if (row && i0 + c < a.I)
        x = (float)a.codes[(t + k) * a.ld8 + i0 + c] * pow2_field(a.scales[(t + k) * a.nb8 + (i0 + c) / kBlock8]);
      sb[k][c] = x;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float av = sa[k][ty * 4 + u];
        bias[u] += av;
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[u][v] = __fmaf_rn(av, sb[k][tx * 4 + v], acc[u][v]);
      }
    __syncthreads();
  }
  float *p = a.part + (int64_t)blockIdx.z * a.O * a.I;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int o = o0 + ty * 4 + u;
    if (o >= a.O) continue;
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (i0 + tx * 4 + v < a.I) p[(int64_t)o * a.I + i0 + tx * 4 + v] = acc[u][v];
    if (blockIdx.x == 0 && tx == 0) a.part_b[(int64_t)blockIdx.z * a.O + o] = bias[u];
  }
}

template <class T>
__global__ __launch_bounds__(256) void wgrad8_sum_kernel(WgradArgs a) {
  const int64_t n = (int64_t)a.O * a.I, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e < n) {
    float s = 0.0f;
    for (int k = 0; k < a.splits; ++k) s += a.part[k * n + e];
    ((T *)a.dw)[e] = (T)s;
  } else if (e < n + a.O && a.db) {
    float s = 0.0f;
    for (int k = 0; k < a.splits; ++k) s += a.part_b[(int64_t)k * a.O + (e - n)];
    ((T *)a.db)[e - n] = (T)s;
  }
}

struct WgradShape {
  int tx, ty, splits;
  int64_t split_rows;
};
static WgradShape wgrad_shape(int64_t rows, int O, int I) {
  WgradShape s;
  s.tx = ceil_div(I, kTile);
  s.ty = ceil_div(O, kTile);
  const int64_t tiles = (int64_t)s.tx * s.ty;
  int64_t want = tiles >= 1024 ? 1 : 1024 / tiles;
  const int64_t most = (rows + 127) / 128;
  if (want > most) want = most;
  s.split_rows = ((rows + want - 1) / want + kDepth - 1) / kDepth * kDepth;
  s.splits = (int)((rows + s.split_rows - 1) / s.split_rows);
  return s;
}

}  // namespace gvae

using namespace gvae;

extern "C" {

int64_t gvae_linear_wgrad8_ws_bytes(int64_t rows, int O, int I) {
  if (rows <= 0 || O <= 0 || I <= 0) return 0;
  return 4 * (int64_t)wgrad_shape(rows, O, I).splits * ((int64_t)O * I + O);
}

int gvae_linear_wgrad8(const void *d_dy, int dtype, int64_t row_stride, const int8_t *d_codes, const uint8_t *d_scales,
                       int64_t rows, int O, int I, void *d_dw, void *d_db, void *d_ws, void *stream) {
  GVAE_REQUIRE(d_dy && d_codes && d_scales && d_dw && d_ws, GVAE_EINVAL, "linear_wgrad8: null pointer");
  GVAE_REQUIRE(dtype_known(dtype), GVAE_EINVAL, "linear_wgrad8: unknown element type %d", dtype);
  GVAE_REQUIRE(rows > 0 && O > 0 && I > 0 && row_stride >= O, GVAE_EINVAL,
               "linear_wgrad8: bad sizes (rows=%lld out=%d in=%d stride=%lld)", (long long)rows, O, I,
               (long long)row_stride);
  GVAE_REQUIRE((int64_t)O * I < (1LL << 38) && O <= (1 << 20) && I <= (1 << 20), GVAE_ELIMIT,
               "linear_wgrad8: %d x %d weights", O, I);
  const WgradShape sh = wgrad_shape(rows, O, I);
  WgradArgs a;
  a.dy = d_dy; a.codes = d_codes; a.scales = d_scales; a.dw = d_dw; a.db = d_db;
  a.rows = rows; a.ldy = row_stride; a.O = O; a.I = I; a.ld8 = ckpt8_ld(I); a.nb8 = ckpt8_blocks(I);
  a.splits = sh.splits; a.split_rows = sh.split_rows;
  a.part = (float *)d_ws;
  a.part_b = a.part + (int64_t)sh.splits * O * I;
  hipStream_t s = (hipStream_t)stream;
  const int64_t n = (int64_t)O * I + O;
  GVAE_DTYPE_SWITCH(dtype, T, {
    hipLaunchKernelGGL((wgrad8_kernel<T>), dim3(sh.tx, sh.ty, sh.splits), dim3(256), 0, s, a);
    hipLaunchKernelGGL((wgrad8_sum_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
  });
  return check_launch("linear_wgrad8");
}

}  // extern "C"
