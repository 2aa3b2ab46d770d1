// Rows held as 8-bit integers with fp32 scales (octo_quantise_i8_rows, octo_widen_i8_rows), and the copies that the
// gradients of the 8-bit head multiply with (launch_prepare8).
//
//   a = max |x| of a group of a row's values (the whole row, or 32 to 256 of them), scale = a times 1/127 in fp32,
//   q = the exact quotient x / scale to the nearest integer, ties to even;   x^ = q scale in fp32, then in x's type
//
// A group below 2^-119 (its scale would not be a normal number) is held as zeros, one with a NaN or an infinity as NaN
// (scale NaN, q 0).
//
// Bound by memory: a wave per row, 16-byte loads of 8 values (fp32: two), a row of up to 4,096 values in registers
// between its maximum and its quotients. 32,768 x 2,560 bf16: quantised 48 us (5.3 TB/s; groups of 128 54 to 62),
// widened 40 us (6.3 TB/s, part of it from the caches); a copy of such rows takes 63.
#include "octo_internal.h"
#include "row_values.h"
#include "rows8.h"

namespace octo {

constexpr int64_t kFewHeld = 2048;  // quantise_i8_row_kernel up to here

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

// Few rows, a scale each: a workgroup per row, whose chain of instructions is the time. 320 rows of 4,096 bf16 values
// 4.0 us so, 7.2 by a wave each; 2,048 of 2,560 6.6 and 7.4; 8,192 17.2 and 16.7.
template <int DT>
__global__ __launch_bounds__(256) void quantise_i8_row_kernel(const typename Elem<DT>::T *x, int64_t ldx, int d,
                                                              int8_t *q, int64_t ldq, float *scale) {
  constexpr int N = 2;  // chunks of 8 values a thread keeps
  __shared__ uint32_t top[4];
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, chunks = (d + 7) >> 3, padded = ((d + 15) >> 4) << 1;
  const typename Elem<DT>::T *row = x + r * ldx;
  int8_t *out = q + r * ldq;
  Raw8<DT> v[N];
  float f[8];
  uint32_t m = 0;
  for (int c0 = 0; c0 < chunks; c0 += 256 * N) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int c = c0 + 256 * u + t;
      v[u] = load_raw8<DT>(row + 8 * (c < chunks ? c : 0), c < chunks ? d - 8 * c : 0);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      values8<DT>(v[u], f);
      m = max_bits(f, m);
    }
  }
  m = lanes_max<64>(m);
  if (lane == 0) top[w] = m;
  __syncthreads();
  const float s = scale_of(max(max(top[0], top[1]), max(top[2], top[3]))), inv = 1.f / s;
  if (t == 0) scale[r] = s;
  for (int c0 = 0; c0 < padded; c0 += 256 * N) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int c = c0 + 256 * u + t;
      if (chunks > 256 * N) v[u] = load_raw8<DT>(row + 8 * (c < chunks ? c : 0), c < chunks ? d - 8 * c : 0);
      values8<DT>(v[u], f);
      if (c < padded) *(i32x2 *)(out + 8 * c) = quotients(f, s, inv);
    }
  }
}

__device__ __forceinline__ void unpack_i8(const i32x2 v, float s, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)((uint32_t)v[e >> 2] >> (8 * (e & 3))) * s;
}

// Row r of out = q scale for the columns c < d, zeros up to cols_pad (and for all of a row past `rows`), by one wave, 4
// chunks of 8 columns a lane in flight. gshift: log2 of the group, or -1. The bytes of q behind d are readable up to
// the next multiple of 16. UNIT: the integers themselves (exact in every type). times(): a power of two for all scales,
// asked for with the loads in flight.
struct TimesOne {
  __device__ __forceinline__ float operator()() const { return 1.f; }
};
template <int DT, bool UNIT = false, class F = TimesOne>
__device__ __forceinline__ void widen_row(const int8_t *q, const float *scale, bool there, int d, int gshift,
                                          typename Elem<DT>::T *out, int cols_pad, F times = F{}) {
  for (int start = 0; start < cols_pad; start += 512 * 4) {  // the whole wave: times() may join its lanes
    const int c0 = start + 8 * (int)(threadIdx.x & 63);
    i32x2 v[4];
    float s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + 512 * u, at = there && c < d ? c : 0;
      v[u] = there ? *(const i32x2 *)(q + at) : i32x2{0, 0};
      s[u] = !there || c >= d ? 0.f : (UNIT ? 1.f : scale[gshift < 0 ? 0 : at >> gshift]);
    }
    const float by = UNIT ? 1.f : times();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + 512 * u;
      float x[8];
      unpack_i8(v[u], s[u] * by, x);
      if (c + 8 <= cols_pad) {
        if constexpr (DT == OCTO_F32) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            ((i32x4_any4 *)(out + c))[h] = i32x4{__float_as_int(x[4 * h]), __float_as_int(x[4 * h + 1]),
                                                 __float_as_int(x[4 * h + 2]), __float_as_int(x[4 * h + 3])};
        } else {
          *(i32x4_any *)(out + c) = pack8(x, DT == OCTO_F16);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < cols_pad) out[c + e] = from_f32<DT>(x[e]);
      }
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void widen_i8_kernel(const int8_t *q, int64_t ldq, const float *scale, int64_t rows,
                                                       int d, int gshift, int groups, typename Elem<DT>::T *out,
                                                       int64_t ldo) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r < rows) widen_row<DT>(q + r * ldq, scale + r * groups, true, d, gshift, out + r * ldo, d);
}

// f16_range of the weights' scales (k 0) or the rows', its inverse left to the product by one workgroup.
template <int DT> struct RangeTimes {
  Norm8 *norm;
  int k;
  bool leave;
  __device__ __forceinline__ float operator()() const {
    float times = 1.f, back;
    if constexpr (DT == OCTO_F16) {
      f16_range(lanes_max<64>(norm->top[k][threadIdx.x & 63]), times, back);
      if (leave && threadIdx.x == 0) norm->back[k] = back;
    }
    return times;
  }
};

// xt[c, r] = q[r, c] scale[r] for c < d, r0 <= r < r0 + 64; zeros from n on; `repeats` of it np columns apart. A 64 x
// 64 tile through the LDS.
template <int DT, bool UNIT = false, class F>
__device__ __forceinline__ void widen_t_tile(const Prepare8 &a, int64_t r0, int c0, int repeats,
                                             typename Elem<DT>::T (*tile)[64 + 16 / Elem<DT>::bytes], F times) {
  typedef typename Elem<DT>::T T;
  constexpr int PER = 16 / sizeof(T);
  const int t = threadIdx.x;
  {
    const int row = t & 63, c = (t >> 6) * 16;  // a wave's lanes: one 16-byte chunk of 64 rows
    const int64_t r = r0 + row;
    i32x4 v = {0, 0, 0, 0};
    float s = 0.f;
    if (r < a.n && c0 + c < a.d) {
      s = UNIT ? 1.f : a.xs[r];
      v = *(const i32x4 *)(a.xq + r * a.ldxq + c0 + c);
    }
    if (!UNIT) s *= times();
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
    if (c0 + c >= a.d) continue;
    const i32x4 v = *(const i32x4 *)&tile[c][r];
    for (int p = 0; p < repeats; ++p) *(i32x4 *)((T *)a.xt + (int64_t)(c0 + c) * a.ldt + p * a.np + r0 + r) = v;
  }
}

// 8,192 bytes of row r of the copy of g, zeros behind it.
template <int DT>
__device__ __forceinline__ void stage_part(const Prepare8 &a, int64_t r, int part) {
  typedef typename Elem<DT>::T T;
  constexpr int PER = 16 / sizeof(T);
  const T *g = (const T *)a.g + r * a.ldg;
  i32x4 v[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int c = ((2 * part + u) * 256 + (int)threadIdx.x) * PER;
    v[u] = i32x4{0, 0, 0, 0};
    if (r >= a.n || c >= a.V) continue;
    if (c + PER <= a.V) {
      v[u] = *(const i32x4_any *)(g + c);
    } else {
      T x[PER] = {};
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (c + e < a.V) x[e] = g[c + e];
      v[u] = __builtin_bit_cast(i32x4, x);
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int c = ((2 * part + u) * 256 + (int)threadIdx.x) * PER;
    if (c < a.Vp) *(i32x4 *)((T *)a.gs + r * a.Vp + c) = v[u];
  }
}

// fp32 g: 8 values of a row times their weights' scales, and times the row's, in three parts each.
__device__ __forceinline__ void stage_f32(const Prepare8 &a, int64_t r, int part) {
  const int c = (part * 256 + (int)threadIdx.x) * 8;
  float x[8], y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  if (r < a.n && c < a.V) values8<OCTO_F32>(load_raw8<OCTO_F32>((const float *)a.g + r * a.ldg + c, a.V - c), x);
  i32x4 v[3];
  if (a.gh && r < a.n && c < a.Vr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = c + e < a.V ? x[e] * a.ws[c + e] : 0.f;
    split_parts(y, v);
#pragma unroll
    for (int p = 0; p < 3; ++p) *(i32x4 *)((__bf16 *)a.gh + r * 3 * a.Vr + p * a.Vr + c) = v[p];
  }
  if (a.gs && c < a.Vp) {
    const float s = r < a.n ? a.xs[r] : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = r < a.n ? x[e] * s : 0.f;
    split_parts(y, v);
#pragma unroll
    for (int p = 0; p < 3; ++p) *(i32x4 *)((__bf16 *)a.gs + (p * a.np + r) * a.Vp + c) = v[p];
  }
}

// The copies that the gradients' products read, in one launch: blocks of 4 weight rows, of 64 x 64 tiles of the
// transposed rows, of parts of g's rows.
template <int DT>
__global__ __launch_bounds__(256) void prepare8_kernel(Prepare8 a) {
  constexpr bool F32 = DT == OCTO_F32;
  constexpr int WT = F32 ? OCTO_BF16 : DT;  // fp32 g: the integers in bf16, the scales in g's parts
  typedef typename Elem<WT>::T T;
  __shared__ __attribute__((aligned(16))) T tile[64][64 + 16 / sizeof(T)];
  unsigned b = a.first + blockIdx.x;
  if (b < a.wide_blocks) {
    const int64_t r = (int64_t)b * 4 + (threadIdx.x >> 6);  // Vr is a multiple of 64
    const RangeTimes<DT> times{a.norm, 0, b == 0};
    widen_row<WT, F32>(a.wq + r * a.ldw, a.ws + r, r < a.V, a.d, -1, (T *)a.wide + r * a.dp, a.dp, times);
    return;
  }
  b -= a.wide_blocks;
  if (b < a.t_blocks) {
    const unsigned tiles = (unsigned)(a.np / 64);
    const RangeTimes<DT> times{a.norm, 1, b == 0};
    widen_t_tile<WT, F32>(a, (int64_t)(b % tiles) * 64, (int)(b / tiles) * 64, F32 ? 3 : 1, tile, times);
    return;
  }
  b -= a.t_blocks;
  if constexpr (F32) stage_f32(a, b / a.g_parts, (int)(b % a.g_parts));
  else stage_part<DT>(a, b / a.g_parts, (int)(b % a.g_parts));
}

// The largest finite scales of 64 shares of the weights (blocks 0 .. 63) and of the rows, for f16_range.
__global__ __launch_bounds__(256) void norm8_kernel(const float *ws, int64_t V, const float *xs, int64_t n,
                                                    Norm8 *norm) {
  __shared__ uint32_t top[4];
  const int k = blockIdx.x >> 6, part = blockIdx.x & 63, t = threadIdx.x;
  const float *s = k ? xs : ws;
  const int64_t count = k ? n : V;
  uint32_t m = 0;
#pragma unroll 4
  for (int64_t i = part * 256 + t; i < count; i += 64 * 256) m = max(m, finite_bits(s[i]));
  m = lanes_max<64>(m);
  if ((t & 63) == 0) top[t >> 6] = m;
  __syncthreads();
  if (t == 0) norm->top[k][part] = max(max(top[0], top[1]), max(top[2], top[3]));
}

// Blocks a launch: 2^24 of 256 threads are more threads than one can have. At most 2^31 in all (2^21 rows and columns).
constexpr int64_t kPrepareBlocks = 1 << 22;
int launch_prepare8(Prepare8 a, int dtype, hipStream_t st) {
  const bool f32 = dtype == OCTO_F32;
  const int64_t per = f32 ? 256 * 8 : 512 * 8;  // values of a part of g
  const int64_t wide = a.wide ? a.Vr / 4 : 0, t = a.xt ? a.np / 64 * cdiv(a.d, 64) : 0;
  a.g_parts = (unsigned)cdiv(a.Vp, per);
  const int64_t staged = a.gs || a.gh ? a.np * a.g_parts : 0, blocks = wide + t + staged;
  if (blocks == 0) return OCTO_OK;
  a.wide_blocks = (unsigned)wide;
  a.t_blocks = (unsigned)t;
  if (a.norm) {
    hipLaunchKernelGGL(norm8_kernel, dim3(128), dim3(256), 0, st, a.ws, a.wide ? a.V : 0, a.xs, a.xt ? a.n : 0, a.norm);
    OCTO_CHECK_LAUNCH("norm8");
  }
  for (int64_t first = 0; first < blocks; first += kPrepareBlocks) {
    const dim3 grid((unsigned)(blocks - first < kPrepareBlocks ? blocks - first : kPrepareBlocks));
    a.first = (unsigned)first;
    switch (dtype) {
      case OCTO_BF16: hipLaunchKernelGGL(prepare8_kernel<OCTO_BF16>, grid, dim3(256), 0, st, a); break;
      case OCTO_F16: hipLaunchKernelGGL(prepare8_kernel<OCTO_F16>, grid, dim3(256), 0, st, a); break;
      default: hipLaunchKernelGGL(prepare8_kernel<OCTO_F32>, grid, dim3(256), 0, st, a); break;
    }
    OCTO_CHECK_LAUNCH("prepare8");
  }
  return OCTO_OK;
}

template <int DT>
static void go_widen(const int8_t *q, int64_t ldq, const float *scale, int64_t rows, int d, int group, void *out,
                     int64_t ldo, hipStream_t st) {
  const int gshift = group ? __builtin_ctz((unsigned)group) : -1, groups = group ? (int)cdiv(d, group) : 1;
  hipLaunchKernelGGL(widen_i8_kernel<DT>, dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, st, q, ldq, scale, rows, d,
                     gshift, groups, (typename Elem<DT>::T *)out, ldo);
}

template <int DT>
static void go_quantise(const void *x, int64_t ldx, int64_t rows, int d, int group, int8_t *q, int64_t ldq,
                        float *scale, hipStream_t st) {
  typedef typename Elem<DT>::T T;
  if (group == 0 && rows <= kFewHeld) {
    hipLaunchKernelGGL(quantise_i8_row_kernel<DT>, dim3((unsigned)rows), dim3(256), 0, st, (const T *)x, ldx, d, q, ldq,
                       scale);
    return;
  }
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
    int8_t *qr = q + r0 * ldq;
    float *sr = scale + r0 * groups;
    hipStream_t st = (hipStream_t)stream;
    switch (x_dtype) {
      case OCTO_BF16: go_quantise<OCTO_BF16>(xr, ldx, n, d, group, qr, ldq, sr, st); break;
      case OCTO_F16: go_quantise<OCTO_F16>(xr, ldx, n, d, group, qr, ldq, sr, st); break;
      default: go_quantise<OCTO_F32>(xr, ldx, n, d, group, qr, ldq, sr, st); break;
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
  const int64_t groups = group ? cdiv(d, group) : 1;
  for (int64_t r0 = 0; r0 < rows; r0 += kLaunchRows) {
    const int64_t n = rows - r0 < kLaunchRows ? rows - r0 : kLaunchRows;
    char *o = (char *)out + r0 * ldo * float_bytes(out_dtype);
    const int8_t *qr = q + r0 * ldq;
    const float *sr = scale + r0 * groups;
    hipStream_t st = (hipStream_t)stream;
    switch (out_dtype) {
      case OCTO_BF16: go_widen<OCTO_BF16>(qr, ldq, sr, n, d, group, o, ldo, st); break;
      case OCTO_F16: go_widen<OCTO_F16>(qr, ldq, sr, n, d, group, o, ldo, st); break;
      default: go_widen<OCTO_F32>(qr, ldq, sr, n, d, group, o, ldo, st); break;
    }
    OCTO_CHECK_LAUNCH("widen_i8");
  }
  return OCTO_OK;
}

}  // extern "C"
