// A row's values as 8-bit integers: the loads, the scale and the quotients (rows8.hip, int8_head.hip).
#pragma once

#include "row_values.h"

namespace octo {

constexpr float kLeastMax = 0x1p-119f;

// 8 consecutive values as they lie, from an address of any element alignment (global loads of 16 bytes need none);
// zeros from `valid` on.
typedef i32x4 i32x4_any __attribute__((aligned(2)));
typedef i32x4 i32x4_any4 __attribute__((aligned(4)));
template <int DT> struct Raw8 {
  i32x4 v[DT == OCTO_F32 ? 2 : 1];
};
template <int DT> __device__ __forceinline__ Raw8<DT> load_raw8(const typename Elem<DT>::T *p) {
  Raw8<DT> r;
  if constexpr (DT == OCTO_F32) {
    r.v[0] = ((const i32x4_any4 *)p)[0];
    r.v[1] = ((const i32x4_any4 *)p)[1];
  } else {
    r.v[0] = *(const i32x4_any *)p;
  }
  return r;
}
template <int DT> __device__ __forceinline__ Raw8<DT> load_raw8(const typename Elem<DT>::T *p, int valid) {
  if (valid >= 8) return load_raw8<DT>(p);
  typedef typename Elem<DT>::T T;
  T x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = e < valid ? p[e] : (T)0.f;
  return __builtin_bit_cast(Raw8<DT>, x);
}
template <int DT> __device__ __forceinline__ void values8(const Raw8<DT> &r, float (&x)[8]) {
  if constexpr (DT == OCTO_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __int_as_float(r.v[e >> 2][e & 3]);
  } else {
    unpack8(r.v[0], DT == OCTO_F16, x);
  }
}
// Chunks c0 + lane, c0 + 64 + lane, ... of a row; without a branch a chunk (which makes each load wait for the one
// before) where all of them are whole.
template <int DT, int N>
__device__ __forceinline__ void load_chunks(const typename Elem<DT>::T *row, int d, int c0, Raw8<DT> (&v)[N]) {
  const int lane = threadIdx.x & 63;
  if (8 * (c0 + 64 * N) <= d) {
#pragma unroll
    for (int u = 0; u < N; ++u) v[u] = load_raw8<DT>(row + 8 * (c0 + 64 * u + lane));
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int c = c0 + 64 * u;
      if (8 * (c + 64) <= d) v[u] = load_raw8<DT>(row + 8 * (c + lane));
      else if (8 * c < d) v[u] = load_raw8<DT>(row + 8 * (c + lane), d - 8 * (c + lane));
      else v[u] = Raw8<DT>{};
    }
  }
}

// The magnitudes' bits compare as the magnitudes do, NaN above all.
__device__ __forceinline__ uint32_t max_bits(const float (&x)[8], uint32_t m) {
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
  return m;
}
template <int LANES> __device__ __forceinline__ uint32_t lanes_max(uint32_t m) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  return m;
}
__device__ __forceinline__ float scale_of(uint32_t maxbits) {
  if (maxbits >= 0x7f800000u) return __builtin_nanf("");
  const float a = __uint_as_float(maxbits);
  return a < kLeastMax ? 0.f : a * (1.f / 127.f);
}
// 8 quotients as bytes. x inv is within an integer of x / s and the remainder x - q s is exact in one fma (at most 7
// bits of q times 24 of s, less x: within fp32's 24 bits above the finer of the two last places), so comparing twice it
// with s gives the quotient's rounding exactly (half of an s below 2^-125 is not always a number of fp32).
__device__ __forceinline__ i32x2 quotients(const float (&x)[8], float s, float inv) {
  i32x2 out = {0, 0};
  if (!(s > 0.f)) return out;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float q = __builtin_rintf(x[e] * inv);
    const float r = __builtin_fmaf(-q, s, x[e]), twice = 2.f * fabsf(r);
    const int odd = (int)q & 1;
    if (twice > s || (twice == s && odd)) q += __builtin_copysignf(1.f, r);
    out[e >> 2] |= ((int)q & 0xff) << (8 * (e & 3));
  }
  return out;
}

// A row's scale and quotients by one wave, N chunks a lane at a time: put(chunk, bytes) for every chunk of 8 up to
// `padded` of them (zeros past the row), each by one lane. A row of up to 512 N values is read once, a longer one
// twice.
template <int DT, int N, class F>
__device__ __forceinline__ float quantise_row(const typename Elem<DT>::T *row, int d, int padded, F put) {
  const int lane = threadIdx.x & 63, chunks = (d + 7) >> 3;
  Raw8<DT> v[N];
  float x[8];
  uint32_t m = 0;
  for (int c0 = 0; c0 < chunks; c0 += 64 * N) {
    load_chunks<DT, N>(row, d, c0, v);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      values8<DT>(v[u], x);
      m = max_bits(x, m);
    }
  }
  const float s = scale_of(lanes_max<64>(m)), inv = 1.f / s;
  for (int c0 = 0; c0 < padded; c0 += 64 * N) {
    if (c0 > 0 || chunks > 64 * N) load_chunks<DT, N>(row, d, c0, v);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int c = c0 + 64 * u + lane;
      values8<DT>(v[u], x);
      if (c < padded) put(c, quotients(x, s, inv));
    }
  }
  return s;
}

// 8 fp32 values as three bf16 parts each, whose sum they are (24 bits; one that bf16 cannot hold stays in the first
// part alone).
__device__ __forceinline__ void split_parts(const float (&x)[8], i32x4 (&part)[3]) {
  float p0[8], p1[8], p2[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    p0[e] = (float)(__bf16)x[e];
    const bool fine = fabsf(p0[e]) < INFINITY;
    p1[e] = fine ? (float)(__bf16)(x[e] - p0[e]) : 0.f;
    p2[e] = fine ? x[e] - p0[e] - p1[e] : 0.f;
  }
  part[0] = pack8(p0, false);
  part[1] = pack8(p1, false);
  part[2] = pack8(p2, false);
}

// Integers times scales as f16 numbers: bf16 and fp32 rows, and scales as a caller gives them, may lie outside f16's
// range. times: the power of two that brings the largest finite scale to [2^7, 2^8), so that 128 of it stays short of
// f16's infinity and its 11 bits reach down to 2^-29 of it; back: the inverse, for the sum. maxbits: that scale's.
__device__ __forceinline__ uint32_t finite_bits(float s) {
  const uint32_t b = __float_as_uint(s) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0;
}
__device__ __forceinline__ void f16_range(uint32_t maxbits, float &times, float &back) {
  const int by = min(7 - ((int)(maxbits >> 23) - 127), 120);  // the scale is below 2^(8 - by)
  times = __uint_as_float((uint32_t)(127 + by) << 23);
  back = __uint_as_float((uint32_t)(127 - by) << 23);
}

}  // namespace octo
