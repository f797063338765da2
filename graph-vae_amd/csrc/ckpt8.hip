// Activations into 8-bit checkpoints and back (the format: gvae_ckpt8.h).  Bound by memory: a value
// is read once and a byte written, or the other way round.  A lane holds 16 bytes of a row, four (16-bit
// types) or eight neighbouring lanes a block; the block's largest magnitude is an integer maximum of
// bit patterns over its lanes.  262144 rows of 1024, bf16 (537 MB and 277 MB): written in 145 us, read
// in 137 (5.6 and 5.9 TB/s; medians of 400 calls); four pieces of a lane in flight instead of one were slower.
#include "gvae_ckpt8.h"

#include <type_traits>

namespace gvae {

struct Ckpt8Args {
  void *x;
  int8_t *codes;
  uint8_t *scales;
  int64_t rows, ld;
  int C, ld8, nb8, lanes;   // lanes: pieces of a row, whole blocks
  int group_rows;           // rows of a work-group
};

template <class T, bool PAST>
__global__ __launch_bounds__(256) void ckpt8_write_kernel(Ckpt8Args a) {
  constexpr int V = Piece<T>::V;
  const int64_t row0 = (int64_t)blockIdx.x * a.group_rows;
  const int rows = (int)(a.rows - row0 < a.group_rows ? a.rows - row0 : a.group_rows);
  for (int e = threadIdx.x; e < rows * a.lanes; e += 256) {
    const int i = e / a.lanes, c0 = (e - i * a.lanes) * V;
    const int64_t row = row0 + i;
    const int nv = a.C - c0 < V ? a.C - c0 : V;
    typename Piece<T>::raw r{};
    if (nv > 0) {
      const Cut<T> cut(c0, nv, a.C);
      r = cut.load((const T *)a.x + row * a.ld);
      cut.cut(r);
    }
    float f[V];
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = (float)r[v];
    emit8<PAST, V>(f, a.codes + row * a.ld8 + c0, a.ld8 - c0, a.scales + row * a.nb8 + c0 / kBlock8, c0 % kBlock8 == 0);
  }
}

template <class T, bool PAST>
__global__ __launch_bounds__(256) void ckpt8_read_kernel(Ckpt8Args a) {
  constexpr int V = Piece<T>::V;
  const int64_t row0 = (int64_t)blockIdx.x * a.group_rows;
  const int rows = (int)(a.rows - row0 < a.group_rows ? a.rows - row0 : a.group_rows);
  for (int e = threadIdx.x; e < rows * a.lanes; e += 256) {
    const int i = e / a.lanes, c0 = (e - i * a.lanes) * V;
    const int64_t row = row0 + i;
    const int nv = a.C - c0 < V ? a.C - c0 : V;
    if (nv <= 0) continue;
    float f[V];
    decode8<V>(load_codes<V>(a.codes + row * a.ld8 + c0), pow2_field(a.scales[row * a.nb8 + c0 / kBlock8]), f);
    // (64 * 2^10 stands for the largest halves and is itself none: the nearest half is taken)
    if (std::is_same<T, f16_t>::value)
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = f[v] == f[v] ? fminf(fmaxf(f[v], -65504.0f), 65504.0f) : f[v];
    store_piece<PAST, T>((T *)a.x + row * a.ld + c0, f, nv);
  }
}

}  // namespace gvae

using namespace gvae;

static int ckpt8_args(const char *who, void *x, int dtype, int64_t rows, int C, int64_t ld, int8_t *codes,
                      uint8_t *scales, Ckpt8Args *a) {
  GVAE_REQUIRE(x && codes && scales, GVAE_EINVAL, "%s: null pointer", who);
  GVAE_REQUIRE(dtype_known(dtype), GVAE_EINVAL, "%s: unknown element type %d", who, dtype);
  GVAE_REQUIRE(rows > 0 && C > 0 && ld >= C, GVAE_EINVAL, "%s: bad sizes (rows=%lld channels=%d stride=%lld)", who,
               (long long)rows, C, (long long)ld);
  GVAE_REQUIRE(aligned16(codes), GVAE_EINVAL, "%s: codes are not 16-byte aligned", who);
  GVAE_REQUIRE(C <= (1 << 24), GVAE_ELIMIT, "%s: %d channels", who, C);
  a->x = x; a->codes = codes; a->scales = scales; a->rows = rows; a->ld = ld;
  a->C = C; a->ld8 = ckpt8_ld(C); a->nb8 = ckpt8_blocks(C); a->lanes = a->nb8 * (kBlock8 * dtype_bytes(dtype) / 16);
  // about four pieces a thread, at least one row
  a->group_rows = a->lanes >= 1024 ? 1 : 1024 / a->lanes;
  GVAE_REQUIRE((rows + a->group_rows - 1) / a->group_rows < (1LL << 24), GVAE_ELIMIT, "%s: %lld rows", who,
               (long long)rows);
  return GVAE_OK;
}

extern "C" {

int gvae_ckpt8_row_bytes(int C) { return C > 0 ? ckpt8_ld(C) : 0; }
int gvae_ckpt8_row_scales(int C) { return C > 0 ? ckpt8_blocks(C) : 0; }

int gvae_ckpt8_write(const void *d_x, int dtype, int64_t rows, int C, int64_t row_stride, int8_t *d_codes,
                     uint8_t *d_scales, void *stream) {
  Ckpt8Args a;
  if (int rc = ckpt8_args("ckpt8_write", const_cast<void *>(d_x), dtype, rows, C, row_stride, d_codes, d_scales, &a))
    return rc;
  const dim3 grid((unsigned)((rows + a.group_rows - 1) / a.group_rows));
  GVAE_DTYPE_SWITCH(dtype, T, {
    auto kernel = rows * C >= kPastCaches ? ckpt8_write_kernel<T, true> : ckpt8_write_kernel<T, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, a);
  });
  return check_launch("ckpt8_write");
}

int gvae_ckpt8_read(const int8_t *d_codes, const uint8_t *d_scales, int64_t rows, int C, void *d_x, int dtype,
                    int64_t row_stride, void *stream) {
  Ckpt8Args a;
  if (int rc = ckpt8_args("ckpt8_read", d_x, dtype, rows, C, row_stride, const_cast<int8_t *>(d_codes),
                          const_cast<uint8_t *>(d_scales), &a))
    return rc;
  const dim3 grid((unsigned)((rows + a.group_rows - 1) / a.group_rows));
  GVAE_DTYPE_SWITCH(dtype, T, {
    auto kernel = rows * C * (int64_t)sizeof(T) >= kPastCaches ? ckpt8_read_kernel<T, true> : ckpt8_read_kernel<T, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, a);
  });
  return check_launch("ckpt8_read");
}

}  // extern "C"
