// Rows of values read in 16-byte chunks: their values as fp32 and back, dot products of two rows, the online softmax
// statistics of a row of logits.
#pragma once

#include "octo_common.h"

namespace octo {

// Rows per launch of the kernels with a workgroup a row: a launch has fewer than 2^32 threads.
constexpr int64_t kLaunchRows = 1 << 21;

// 8 consecutive 16-bit values (one 16-byte chunk) as fp32, and back (round to nearest even).
__device__ __forceinline__ void unpack8(const i32x4 v, bool f16, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = ((uint32_t)v[e >> 1] >> (16 * (e & 1))) & 0xffffu;
    x[e] = f16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)b) : __uint_as_float(b << 16);
  }
}
__device__ __forceinline__ i32x4 pack8(const float (&x)[8], bool f16) {
  i32x4 v;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uint32_t lo, hi;
    if (f16) {
      lo = __builtin_bit_cast(uint16_t, (_Float16)x[2 * h]);
      hi = __builtin_bit_cast(uint16_t, (_Float16)x[2 * h + 1]);
    } else {
      lo = __builtin_bit_cast(uint16_t, (__bf16)x[2 * h]);
      hi = __builtin_bit_cast(uint16_t, (__bf16)x[2 * h + 1]);
    }
    v[h] = (int)(lo | (hi << 16));
  }
  return v;
}

// 16-byte loads a lane of the merge keeps in flight per operand: a row of d 2560 at once, 320 vocabulary tiles. With
// few rows the merge is a chain of loads (57 rows, d 2560, V 151,936: 14.9 us one at a time, 11.0 now; the sums keep
// their order).
constexpr int kRowLoads = 5;

// This lane's part of the fp32 dot product of hidden row hrow and weight row y (the target logit before any scale):
// 16-byte chunks when both are the same 16-bit type, element by element otherwise.
__device__ __forceinline__ float row_dot(const void *h, int h_dtype, int64_t hoff, const void *w, int w_dtype,
                                         int64_t woff, int d, int lane) {
  float dot = 0.f;
  if (h_dtype == w_dtype && (h_dtype == OCTO_BF16 || h_dtype == OCTO_F16) && d % 8 == 0) {
    const bool f16 = h_dtype == OCTO_F16;
    const char *hp = (const char *)h + hoff * 2, *wp = (const char *)w + woff * 2;
    for (int k0 = lane; k0 < d / 8; k0 += 64 * kRowLoads) {  // loads of kRowLoads chunks in flight, summed in order
      i32x4 hv[kRowLoads], wv[kRowLoads];
#pragma unroll
      for (int u = 0; u < kRowLoads; ++u) {
        const int k = min(k0 + 64 * u, d / 8 - 1);  // past the end: the last chunk again, left out below
        hv[u] = *(const i32x4 *)(hp + k * 16);
        wv[u] = *(const i32x4 *)(wp + k * 16);
      }
#pragma unroll
      for (int u = 0; u < kRowLoads; ++u) {
        if (k0 + 64 * u >= d / 8) break;
        float a[8], b[8];
        unpack8(hv[u], f16, a);
        unpack8(wv[u], f16, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = __builtin_fmaf(a[e], b[e], dot);
      }
    }
    return dot;
  }
  if (h_dtype == OCTO_BF16 && w_dtype == OCTO_FP8E4M3 && d % 16 == 0) {
    // 16 e4m3 weights per 16-byte load against 16 bf16 hidden values (rows are 16-byte aligned: the head's checks);
    // byte-wise loads made the merge 0.75 ms at 114,688 rows, d 2560
    const char *hp = (const char *)h + hoff * 2;
    const uint8_t *wp = (const uint8_t *)w + woff;
    for (int k = lane; k < d / 16; k += 64) {
      const i32x4 wv = *(const i32x4 *)(wp + k * 16);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float a[8];
        unpack8(*(const i32x4 *)(hp + k * 32 + half * 16), false, a);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t byte = ((uint32_t)wv[2 * half + (e >> 2)] >> (8 * (e & 3))) & 0xffu;
          dot = __builtin_fmaf(a[e], e4m3_to_f32(byte), dot);
        }
      }
    }
    return dot;
  }
  for (int k = lane; k < d; k += 64) {
    const float hv = load_as_f32(h, h_dtype, hoff + k);
    const float wv = w_dtype == OCTO_FP8E4M3 ? e4m3_to_f32(((const uint8_t *)w)[woff + k])
                                             : load_as_f32(w, w_dtype, woff + k);
    dot = __builtin_fmaf(hv, wv, dot);
  }
  return dot;
}

// The 16-byte chunks of a row of V values at p: `head` values before the first chunk, `chunks` of PER, then the rest.
struct RowChunks {
  int head, chunks;
};
template <int DT> __device__ __forceinline__ RowChunks row_chunks(const void *p, int V) {
  constexpr int PER = 16 / Elem<DT>::bytes;
  RowChunks c;
  c.head = min(V, (int)((16 - ((uintptr_t)p & 15)) & 15) / Elem<DT>::bytes);
  c.chunks = (V - c.head) / PER;
  return c;
}
// A chunk's values as fp32 (4 of fp32, 8 of 16 bits) and back.
template <int DT> __device__ __forceinline__ void unpack_chunk(const i32x4 v, float (&x)[16 / Elem<DT>::bytes]) {
  if constexpr (DT == OCTO_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __int_as_float(v[e]);
  } else {
    unpack8(v, DT == OCTO_F16, x);
  }
}
template <int DT> __device__ __forceinline__ i32x4 pack_chunk(const float (&x)[16 / Elem<DT>::bytes]) {
  if constexpr (DT == OCTO_F32) {
    i32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __float_as_int(x[e]);
    return v;
  } else {
    return pack8(x, DT == OCTO_F16);
  }
}

// One thread's online statistics: m the running base-2 maximum (-inf before any finite value), S and U the sums of e =
// exp2(t - m) and e (t - m). A logit of -inf adds 0 to S and, as 0 x -inf, NaN to U: its row's entropy is NaN, its
// logprob is not.
struct ColStat {
  float m = -INFINITY, S = 0.f, U = 0.f;
  // S and U relative to a maximum -d above m. Far below it they count for nothing, and what they hold may be no number:
  // a thread that has only seen logits masked with a finite -1e38 or lower has m = x c rounded by up to 2^103, and its
  // e are exp2 of that. (A NaN stays: it came from a NaN or infinite logit.)
  __device__ __forceinline__ void shift(float d) {
    if (d < -256.f) {
      S = S == S ? 0.f : S;
      U = U == U ? 0.f : U;
    } else {
      const float f = fexp2(d);
      U = f * __builtin_fmaf(d, S, U);
      S *= f;
    }
  }
  __device__ __forceinline__ void raise(float mx) {
    if (mx > m) {
      if (m != -INFINITY) shift(m - mx);
      m = mx;
    }
  }
  __device__ __forceinline__ void add(float x, float c) {  // after raise() to at least x c
    const float t = __builtin_fmaf(x, c, m == -INFINITY ? 0.f : -m);
    const float e = fexp2(t);
    S += e;
    U = __builtin_fmaf(e, t, U);
  }
};

// One thread's part of a row's logsumexp at c = log2(e) / T: m the running maximum of the logits themselves (-inf
// before any above it), S the sum of exp2((x - m) c). Against m and not m c: logits masked with the type's lowest value
// times c overflow, and a row of nothing else still has its logsumexp. -inf adds nothing; a NaN or +inf makes S NaN for
// good.
struct RowSum {
  float m = -INFINITY, S = 0.f;
  // S against a maximum raised by -d / c; far below the new one it counts for nothing
  __device__ __forceinline__ void shift(float d) { S = d < -256.f ? (S == S ? 0.f : S) : S * fexp2(d); }
  __device__ __forceinline__ void raise(float mx, float c) {
    if (mx > m) {
      shift((m - mx) * c);
      m = mx;
    }
  }
  __device__ __forceinline__ void add(float x, float c) {  // after raise() to at least x
    S += fexp2((x - (m == -INFINITY ? 0.f : m)) * c);
  }
};

// A workgroup's logsumexp from its threads' parts: (m, S) in every thread. red: 2 x NW floats of shared memory.
template <int NW>
__device__ __forceinline__ void block_row_sum(RowSum st, float c, float (*red)[NW], float &m, float &S) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  m = wave_max(st.m);
  if (lane == 0) red[0][w] = m;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NW; ++k) m = fmaxf(m, red[0][k]);
  if (st.m != -INFINITY) st.shift((st.m - m) * c);  // else S is 0, or NaN
  const float s = wave_sum(st.S);
  if (lane == 0) red[1][w] = s;
  __syncthreads();
  S = 0.f;
#pragma unroll
  for (int k = 0; k < NW; ++k) S += red[1][k];
}

inline int float_bytes(int dtype) { return dtype == OCTO_F32 ? 4 : 2; }
inline bool is_float(int dtype) { return dtype == OCTO_BF16 || dtype == OCTO_F16 || dtype == OCTO_F32; }

}  // namespace octo
