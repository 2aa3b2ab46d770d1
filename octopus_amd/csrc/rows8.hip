// Rows held as 8-bit integers with fp32 scales (octo_quantise_i8_rows, octo_widen_i8_rows), and the copies that the
// gradients of the 8-bit head multiply with (launch_widen_t, launch_stage_rows).
//
//   a = max |x| of a group of a row's values (the whole row, or 32 to 256 of them), scale = a times 1/127, both in fp32,
//   q = the exact quotient x / scale to the nearest integer, ties to even;   x^ = q scale, rounded once
//
// A group below 2^-119 (its scale would not be a normal number) is held as zeros, one with a NaN or an infinity as NaN
// (scale NaN, q 0).
//
// Bound by memory: a wave per row, 16-byte loads of 8 values (fp32: two), a row of up to 4,096 values in registers
// between its maximum and its quotients.
#include "octo_internal.h"
#include "row_values.h"
#include "rows8.h"

namespace octo {


// GL: lanes of a group (8 values each); 0: the group is the row. Zeros behind the row, up to its next 16 bytes.
template <int DT, int GL>
__global__ __launch_bounds__(256) void quantise_i8_kernel(const typename Elem<DT>::T *x, int64_t ldx, int64_t rows,
                                                          int d, int8_t *q, int64_t ldq, float *scale) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const typename Elem<DT>::T *row = x + r * ldx;
  int8_t *out = q + r * ldq;
  const int chunks = (d + 7) >> 3, padded = ((d + 15) >> 4) << 1;
  if constexpr (GL == 0) {
    const float s = quantise_row<DT, 8>(row, d, padded, [&](int c, i32x2 v) { *(i32x2 *)(out + 8 * c) = v; });
    if (lane == 0) scale[r] = s;
  } else {
    const int groups = (chunks + GL - 1) / GL;
    for (int c0 = 0; c0 < padded; c0 += 64 * 4) {  // 4 chunks in flight
      Raw8<DT> v[4];
      load_chunks<DT, 4>(row, d, c0, v);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = c0 + 64 * u + lane;
        float x[8];
        values8<DT>(v[u], x);
        const float s = scale_of(lanes_max<GL>(max_bits(x, 0)));
        if (lane % GL == 0 && c < chunks) scale[r * groups + c / GL] = s;
        if (c < padded) *(i32x2 *)(out + 8 * c) = quotients(x, s, 1.f / s);
      }
    }
  }
}

__device__ __forceinline__ void unpack_i8(const i32x2 v, float s, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)((uint32_t)v[e >> 2] >> (8 * (e & 3))) * s;
}

// out[r, c] = q scale for r < rows, c < d; zeros for the other r < rows_pad and c < cols_pad. 8 columns a thread.
template <int DT>
__global__ __launch_bounds__(256) void widen_i8_kernel(const int8_t *q, int64_t ldq, const float *scale, int64_t rows,
                                                       int d, int group, typename Elem<DT>::T *out, int64_t ldo,
                                                       int64_t rows_pad, int cols_pad) {
  const int64_t chunks = (cols_pad + 7) >> 3, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = i / chunks;
  const int c = (int)(i - r * chunks) * 8;
  if (r >= rows_pad) return;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (r < rows && c < d) {
    const int groups = group ? (d + group - 1) / group : 1;
    i32x2 v = {0, 0};
    if (c + 8 <= d) {
      v = *(const i32x2 *)(q + r * ldq + c);
    } else {
      for (int e = 0; c + e < d; ++e) v[e >> 2] |= (q[r * ldq + c + e] & 0xff) << (8 * (e & 3));
    }
    unpack_i8(v, scale[r * groups + (group ? c / group : 0)], x);
  }
  typename Elem<DT>::T *o = out + r * ldo + c;
  if (c + 8 <= cols_pad) {
    if constexpr (DT == OCTO_F32) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *((i32x4_any4 *)o + h) = i32x4{__float_as_int(x[4 * h]), __float_as_int(x[4 * h + 1]),
                                       __float_as_int(x[4 * h + 2]), __float_as_int(x[4 * h + 3])};
    } else {
      *(i32x4_any *)o = pack8(x, DT == OCTO_F16);
    }
  } else {
    for (int e = 0; c + e < cols_pad; ++e) o[e] = from_f32<DT>(x[e]);
  }
}

// out[c, r] = q[r, c] scale[r] for c < d; zeros for rows <= r < rows_pad (a multiple of 64). One 64 x 64 tile a
// workgroup, through the LDS.
template <int DT>
__global__ __launch_bounds__(256) void widen_t_kernel(const int8_t *q, int64_t ldq, const float *scale, int64_t rows,
                                                      int d, typename Elem<DT>::T *out, int64_t ldo) {
  typedef typename Elem<DT>::T T;
  constexpr int PAD = 16 / sizeof(T), PER = 16 / sizeof(T);
  __shared__ __attribute__((aligned(16))) T tile[64][64 + PAD];
  const int64_t r0 = (int64_t)blockIdx.x * 64;
  const int c0 = blockIdx.y * 64, t = threadIdx.x;
  {
    const int row = t & 63, c = (t >> 6) * 16;  // a wave's lanes: one 16-byte chunk of 64 rows
    const int64_t r = r0 + row;
    i32x4 v = {0, 0, 0, 0};
    float s = 0.f;
    if (r < rows && c0 + c < d) {
      const int8_t *p = q + r * ldq + c0 + c;
      s = scale[r];
      if (c0 + c + 16 <= d) v = *(const i32x4 *)p;
      else
        for (int e = 0; c0 + c + e < d; ++e) v[e >> 2] |= (p[e] & 0xff) << (8 * (e & 3));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[8];
      unpack_i8(i32x2{v[2 * h], v[2 * h + 1]}, s, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) tile[c + 8 * h + e][row] = from_f32<DT>(x[e]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 64 * 64 / PER / 256; ++k) {
    const int i = t + 256 * k, c = i / (64 / PER), r = (i % (64 / PER)) * PER;
    if (c0 + c < d) *(i32x4 *)(out + (int64_t)(c0 + c) * ldo + r0 + r) = *(const i32x4 *)&tile[c][r];
  }
}

// A copy of g [n, V] whose rows start on 16 bytes, zeros behind it up to rows_pad and cols_pad (a multiple of 8).
template <int DT>
__global__ __launch_bounds__(256) void stage_rows_kernel(const typename Elem<DT>::T *g, int64_t ldg, int64_t n, int V,
                                                         typename Elem<DT>::T *out, int64_t ldo, int cols_pad) {
  constexpr int PER = 16 / Elem<DT>::bytes;
  const int64_t r = blockIdx.y;
  const int c = (blockIdx.x * 256 + threadIdx.x) * PER;
  if (c >= cols_pad) return;
  i32x4 v = {0, 0, 0, 0};
  if (r < n && c < V) {
    const typename Elem<DT>::T *p = g + r * ldg + c;
    if (c + PER <= V) {
      if constexpr (DT == OCTO_F32) v = *(const i32x4_any4 *)p;
      else v = *(const i32x4_any *)p;
    } else {
      typename Elem<DT>::T x[PER] = {};
      for (int e = 0; c + e < V; ++e) x[e] = p[e];
      v = __builtin_bit_cast(i32x4, x);
    }
  }
  *(i32x4 *)(out + r * ldo + c) = v;
}

int launch_widen_rows(const int8_t *q, int64_t ldq, const float *scale, int64_t rows, int d, int group, void *out,
                      int64_t ldo, int dtype, int64_t rows_pad, int cols_pad, hipStream_t st) {
  const int64_t chunks = (cols_pad + 7) / 8;
  const int64_t step = ((int64_t)1 << 31) / chunks;  // rows a launch: fewer than 2^32 threads
  for (int64_t r0 = 0; r0 < rows_pad; r0 += step) {
    const int64_t part = rows_pad - r0 < step ? rows_pad - r0 : step;
    const int64_t have = rows - r0 < 0 ? 0 : (rows - r0 < part ? rows - r0 : part);
    const int64_t groups = group ? cdiv(d, group) : 1;
    const dim3 grid((unsigned)cdiv(part * chunks, 256));
    const int8_t *qr = q + r0 * ldq;
    const float *sr = scale + r0 * groups;
    switch (dtype) {
      case OCTO_BF16:
        hipLaunchKernelGGL(widen_i8_kernel<OCTO_BF16>, grid, dim3(256), 0, st, qr, ldq, sr, have, d, group,
                           (__bf16 *)out + r0 * ldo, ldo, part, cols_pad);
        break;
      case OCTO_F16:
        hipLaunchKernelGGL(widen_i8_kernel<OCTO_F16>, grid, dim3(256), 0, st, qr, ldq, sr, have, d, group,
                           (_Float16 *)out + r0 * ldo, ldo, part, cols_pad);
        break;
      default:
        hipLaunchKernelGGL(widen_i8_kernel<OCTO_F32>, grid, dim3(256), 0, st, qr, ldq, sr, have, d, group,
                           (float *)out + r0 * ldo, ldo, part, cols_pad);
        break;
    }
    OCTO_CHECK_LAUNCH("widen_i8");
  }
  return OCTO_OK;
}

int launch_widen_t(const int8_t *q, int64_t ldq, const float *scale, int64_t rows, int d, void *out, int64_t ldo,
                   int dtype, hipStream_t st) {
  const dim3 grid((unsigned)(ldo / 64), (unsigned)cdiv(d, 64));
  switch (dtype) {
    case OCTO_BF16: hipLaunchKernelGGL(widen_t_kernel<OCTO_BF16>, grid, dim3(256), 0, st, q, ldq, scale, rows, d, (__bf16 *)out, ldo); break;
    case OCTO_F16: hipLaunchKernelGGL(widen_t_kernel<OCTO_F16>, grid, dim3(256), 0, st, q, ldq, scale, rows, d, (_Float16 *)out, ldo); break;
    default: hipLaunchKernelGGL(widen_t_kernel<OCTO_F32>, grid, dim3(256), 0, st, q, ldq, scale, rows, d, (float *)out, ldo); break;
  }
  OCTO_CHECK_LAUNCH("widen_t");
  return OCTO_OK;
}

int launch_stage_rows(const void *g, int64_t ldg, int dtype, int64_t n, int V, void *out, int64_t ldo, int64_t rows_pad,
                      int cols_pad, hipStream_t st) {
  const int per = 16 / float_bytes(dtype);
  for (int64_t r0 = 0; r0 < rows_pad; r0 += 65535) {  // a grid's second dimension
    const int64_t part = rows_pad - r0 < 65535 ? rows_pad - r0 : 65535, have = n - r0 < 0 ? 0 : n - r0;
    const dim3 grid((unsigned)cdiv(cols_pad, 256 * per), (unsigned)part);
    switch (dtype) {
      case OCTO_BF16: hipLaunchKernelGGL(stage_rows_kernel<OCTO_BF16>, grid, dim3(256), 0, st, (const __bf16 *)g + r0 * ldg, ldg, have, V, (__bf16 *)out + r0 * ldo, ldo, cols_pad); break;
      case OCTO_F16: hipLaunchKernelGGL(stage_rows_kernel<OCTO_F16>, grid, dim3(256), 0, st, (const _Float16 *)g + r0 * ldg, ldg, have, V, (_Float16 *)out + r0 * ldo, ldo, cols_pad); break;
      default: hipLaunchKernelGGL(stage_rows_kernel<OCTO_F32>, grid, dim3(256), 0, st, (const float *)g + r0 * ldg, ldg, have, V, (float *)out + r0 * ldo, ldo, cols_pad); break;
    }
    OCTO_CHECK_LAUNCH("stage_rows");
  }
  return OCTO_OK;
}

template <int DT>
static void go_quantise(const void *x, int64_t ldx, int64_t rows, int d, int group, int8_t *q, int64_t ldq,
                        float *scale, hipStream_t st) {
  typedef typename Elem<DT>::T T;
  const dim3 grid((unsigned)cdiv(rows, 4));
#define OCTO_GO(GL)                                                                                                  \
  hipLaunchKernelGGL((quantise_i8_kernel<DT, GL>), grid, dim3(256), 0, st, (const T *)x, ldx, rows, d, q, ldq, scale)
  switch (group) {
    case 0: OCTO_GO(0); break;
    case 32: OCTO_GO(4); break;
    case 64: OCTO_GO(8); break;
    case 128: OCTO_GO(16); break;
    default: OCTO_GO(32); break;
  }
#undef OCTO_GO
}

}  // namespace octo

using namespace octo;

static int rows8_checks(const char *what, int64_t rows, int d, int group, int64_t ld, int64_t ldq, int dtype) {
  OCTO_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff && d > 0 && d <= OCTO_ROW_MAX, "%s: bad shape rows=%lld d=%d", what,
                 (long long)rows, d);
  OCTO_CHECK_ARG(group == 0 || group == 32 || group == 64 || group == 128 || group == 256,
                 "%s: group %d (0, 32, 64, 128 or 256)", what, group);
  OCTO_CHECK_ARG(ld >= d, "%s: row stride %lld below d=%d", what, (long long)ld, d);
  OCTO_CHECK_ARG(ldq >= round_up(d, 16) && ldq % 16 == 0,
                 "%s: 8-bit rows of stride %lld (a multiple of 16, at least d=%d)", what, (long long)ldq, d);
  if (!is_float(dtype)) return octo_fail(OCTO_EUNSUPPORTED, "%s: dtype %d", what, dtype);
  return OCTO_OK;
}

extern "C" {

int octo_quantise_i8_rows(const void *x, int64_t ldx, int x_dtype, int64_t rows, int d, int group, int8_t *q,
                          int64_t ldq, float *scale, void *stream) {
  const int rc = rows8_checks("quantise_i8", rows, d, group, ldx, ldq, x_dtype);
  if (rc) return rc;
  if (rows == 0) return OCTO_OK;
  OCTO_CHECK_ARG(x && q && scale, "quantise_i8: null pointer");
  OCTO_CHECK_ARG((uintptr_t)x % float_bytes(x_dtype) == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)scale % 4 == 0,
                 "quantise_i8: misaligned pointer");
  const int64_t groups = group ? cdiv(d, group) : 1;
  for (int64_t r0 = 0; r0 < rows; r0 += kLaunchRows) {
    const int64_t n = rows - r0 < kLaunchRows ? rows - r0 : kLaunchRows;
    const char *xr = (const char *)x + r0 * ldx * float_bytes(x_dtype);
    switch (x_dtype) {
      case OCTO_BF16: go_quantise<OCTO_BF16>(xr, ldx, n, d, group, q + r0 * ldq, ldq, scale + r0 * groups, (hipStream_t)stream); break;
      case OCTO_F16: go_quantise<OCTO_F16>(xr, ldx, n, d, group, q + r0 * ldq, ldq, scale + r0 * groups, (hipStream_t)stream); break;
      default: go_quantise<OCTO_F32>(xr, ldx, n, d, group, q + r0 * ldq, ldq, scale + r0 * groups, (hipStream_t)stream); break;
    }
    OCTO_CHECK_LAUNCH("quantise_i8");
  }
  return OCTO_OK;
}

int octo_widen_i8_rows(const int8_t *q, int64_t ldq, const float *scale, int64_t rows, int d, int group, void *out,
                       int64_t ldo, int out_dtype, void *stream) {
  const int rc = rows8_checks("widen_i8", rows, d, group, ldo, ldq, out_dtype);
  if (rc) return rc;
  if (rows == 0) return OCTO_OK;
  OCTO_CHECK_ARG(q && scale && out, "widen_i8: null pointer");
  OCTO_CHECK_ARG((uintptr_t)out % float_bytes(out_dtype) == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)scale % 4 == 0,
                 "widen_i8: misaligned pointer");
  return launch_widen_rows(q, ldq, scale, rows, d, group, out, ldo, out_dtype, rows, d, (hipStream_t)stream);
}

}  // extern "C"
