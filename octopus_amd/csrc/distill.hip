// The divergence of a student's logits from a teacher's lists (octo_distill_columns_fwd / _bwd). A row's list holds K
// slots (id, t): t the teacher's logit or log-probability of token id. A slot whose id lies outside [0, V), or whose t
// is -inf, is empty.
//
//   q = softmax of t over the row's slots (OCTO_LIST_RAW: exp(t)),  Q = sum q,  p = softmax(z / T)
//   kl = sum_k q_k (log q_k - log p_id_k)        a row without a slot: 0
//   dL/dz_v = g (Q p_v - sum of q_k over the slots with id_k = v) / T,   g = dL/dkl
//
// Both directions are bound by memory: the forward reads each logit once, the backward reads it once more and writes
// its gradient. The forward leaves q, and the row's (maximum, log2 S, Q), for the backward. [2048, 151,936] bf16, K 64:
// forward 125 to 144 us (4.3 to 5.0 TB/s), backward 217 (5.7).
#include "octo_internal.h"
#include "row_values.h"

namespace octo {

constexpr int kDistThreads = 1024;
constexpr int kDistLoads = 4;  // 16-byte chunks in flight per thread

// The teacher's probabilities of a row's slots, by the first wave: lane l holds slots l + 64 i. q and lq = log q of an
// empty slot: 0 and 0.
constexpr int kSlots = OCTO_LIST_MAX / 64;
__device__ __forceinline__ void teacher_slots(const int64_t *ids, const float *t, int K, int64_t V, bool raw, int lane,
                                              int64_t (&id)[kSlots], float (&q)[kSlots], float (&lq)[kSlots],
                                              float &Q) {
  float m = -INFINITY, x[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int k = lane + 64 * i;
    id[i] = -1;
    x[i] = -INFINITY;
    if (k < K) {
      const int64_t y = ids[k];
      if (y >= 0 && y < V && t[k] != -INFINITY) {
        id[i] = y;
        x[i] = t[k];
        m = fmaxf(m, x[i]);
      }
    }
  }
  m = wave_max(m);
  if (raw || m == -INFINITY) m = 0.f;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    q[i] = id[i] >= 0 ? expf(x[i] - m) : 0.f;
    s += q[i];
  }
  s = wave_sum(s);
  const float inv = raw ? 1.f : 1.f / s, ls = raw ? 0.f : logf(s);
  Q = 0.f;
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    if (id[i] >= 0) {
      q[i] *= inv;
      lq[i] = x[i] - m - ls;
    } else {
      q[i] = lq[i] = 0.f;
    }
    Q += q[i];
  }
  Q = wave_sum(Q);
}

template <int DT>
__global__ __launch_bounds__(kDistThreads, 8) void distill_columns_fwd_kernel(const void *logits, int64_t ld,
                                                                           const int64_t *ids, const float *teacher,
                                                                           int V, int K, float inv_T, int raw,
                                                                           float *kl, float *state, float *q_out) {
  constexpr int PER = 16 / Elem<DT>::bytes, NW = kDistThreads / 64;
  typedef typename Elem<DT>::T T;
  __shared__ float red[2][NW];
  __shared__ float slot_q[OCTO_LIST_MAX], slot_lq[OCTO_LIST_MAX], slot_z[OCTO_LIST_MAX];
  const int64_t r = blockIdx.x;
  const T *row = (const T *)logits + r * ld;
  const float c = inv_T * OCTO_LOG2E;
  // the first wave reads the list, and its logits, ahead of the sweep
  const int lane = threadIdx.x & 63;
  float Q = 0.f;
  if (threadIdx.x < 64) {
    int64_t id[kSlots];
    float q[kSlots], lq[kSlots];
    teacher_slots(ids + r * K, teacher + r * K, K, V, raw != 0, lane, id, q, lq, Q);
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int k = lane + 64 * i;
      if (k < K) {
        q_out[r * K + k] = q[i];
        slot_q[k] = q[i];
        slot_lq[k] = lq[i];
        slot_z[k] = id[i] >= 0 ? (float)row[id[i]] : 0.f;
      }
    }
  }
  const RowChunks rc = row_chunks<DT>(row, V);
  const i32x4 *vec = (const i32x4 *)(row + rc.head);
  RowSum st;
  for (int k0 = threadIdx.x; k0 < rc.chunks; k0 += kDistLoads * kDistThreads) {
    i32x4 v[kDistLoads];
#pragma unroll
    for (int u = 0; u < kDistLoads; ++u)  // past the end: the last chunk again, left out below
      v[u] = vec[min(k0 + u * kDistThreads, rc.chunks - 1)];
    float x[kDistLoads][PER], mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kDistLoads; ++u) {
      unpack_chunk<DT>(v[u], x[u]);
#pragma unroll
      for (int e = 0; e < PER; ++e) mx = fmaxf(mx, x[u][e]);
    }
    st.raise(mx, c);
#pragma unroll
    for (int u = 0; u < kDistLoads; ++u)
      if (k0 + u * kDistThreads < rc.chunks)
#pragma unroll
        for (int e = 0; e < PER; ++e) st.add(x[u][e], c);
  }
  const int tail = rc.head + rc.chunks * PER;
  const int j = (int)threadIdx.x < rc.head ? (int)threadIdx.x : (int)threadIdx.x - rc.head + tail;
  if (j < rc.head || (j >= tail && j < V)) {
    const float x = (float)row[j];
    st.raise(x, c);
    st.add(x, c);
  }
  float m, S;
  block_row_sum<NW>(st, c, red, m, S);
  if (threadIdx.x >= 64) return;
  const float lnS = flog2(S) * OCTO_LN2;
  float sum = 0.f;
  // q 0 (an empty slot, or an exp that underflows): its term's limit, 0, whatever log p is
  for (int k = lane; k < K; k += 64)
    if (slot_q[k] != 0.f) sum += slot_q[k] * (slot_lq[k] - ((slot_z[k] - m) * inv_T - lnS));
  sum = wave_sum(sum);
  if (lane == 0) {
    kl[r] = sum;
    state[4 * r] = m;
    state[4 * r + 1] = flog2(S);
    state[4 * r + 2] = Q;
    state[4 * r + 3] = 0.f;
  }
}

// One workgroup per kDistLoads x 256 chunks of a row. Its first wave picks the slots that lie in its columns, in the
// list's order, and marks their chunks in a bit map; a thread with a marked chunk goes through the picked ones (3 of 64
// on average at V 151,936; each thread through the whole list, and per value, made the kernel 680 us at [2048,
// 151,936]).
constexpr int kMarkWords = 256 * kDistLoads / 32;
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void distill_columns_bwd_kernel(const void *logits, int64_t ld, const int64_t *ids,
                                                                  const float *q, int V, int K, float inv_T,
                                                                  const float *state, const float *g, void *dl,
                                                                  int64_t ld_d) {
  constexpr int PER = 16 / Elem<DT>::bytes;
  typedef typename Elem<DT>::T T;
  __shared__ int slot_col[OCTO_LIST_MAX];
  __shared__ float slot_q[OCTO_LIST_MAX];
  __shared__ uint32_t marks[kMarkWords];
  __shared__ int picked;
  const int64_t r = blockIdx.y;
  const T *row = (const T *)logits + r * ld;
  T *drow = (T *)dl + r * ld_d;
  const float c = inv_T * OCTO_LOG2E, m = state[4 * r], l2S = state[4 * r + 1], Q = state[4 * r + 2];
  const float gs = g[r] * inv_T;
  const RowChunks rc = VEC ? row_chunks<DT>(row, V) : RowChunks{0, V / PER};
  const int k0 = blockIdx.x * (256 * kDistLoads);  // this workgroup's first chunk
  // the values before the first and after the last chunk belong to workgroup 0, as columns of its own
  const int tail = rc.head + rc.chunks * PER;
  const int je = (int)threadIdx.x < rc.head ? (int)threadIdx.x : (int)threadIdx.x - rc.head + tail;
  const bool edge = blockIdx.x == 0 && (je < rc.head || (je >= tail && je < V));
  if (Q == 0.f) {  // a row without a slot: its logits are not looked at
    for (int u = 0; u < kDistLoads; ++u) {
      const int k = k0 + u * 256 + threadIdx.x;
      if (k >= rc.chunks) break;
      if constexpr (VEC) *(i32x4 *)(drow + rc.head + k * PER) = i32x4{0, 0, 0, 0};
      else
        for (int e = 0; e < PER; ++e) drow[k * PER + e] = (T)0.f;
    }
    if (edge) drow[je] = (T)0.f;
    return;
  }
  i32x4 v[kDistLoads];
  if constexpr (VEC) {
#pragma unroll
    for (int u = 0; u < kDistLoads; ++u)  // past the end: the last chunk again, not stored below
      if (rc.chunks) v[u] = *(const i32x4 *)(row + rc.head + min(k0 + u * 256 + (int)threadIdx.x, rc.chunks - 1) * PER);
  }
  if (threadIdx.x < 64) {
    if (threadIdx.x < kMarkWords) marks[threadIdx.x] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int c0 = rc.head + k0 * PER, c1 = min(tail, c0 + 256 * kDistLoads * PER);
    int n = 0;
    for (int s0 = 0; s0 < K; s0 += 64) {
      const int k = s0 + threadIdx.x;
      float qk = 0.f;
      int64_t y = -1;
      if (k < K) {
        qk = q[r * K + k];
        y = ids[r * K + k];
      }
      const bool inside = y >= c0 && y < c1;
      const bool mine = qk != 0.f && y >= 0 && y < V &&
                        (inside || (blockIdx.x == 0 && (y < rc.head || y >= tail)));
      const uint64_t all = __ballot(mine);
      if (mine) {
        const int at = n + __popcll(all & ((1ull << threadIdx.x) - 1ull));
        slot_col[at] = (int)y;
        slot_q[at] = qk;
        if (inside) {
          const int chunk = ((int)y - c0) / PER;
          atomicOr(&marks[chunk >> 5], 1u << (chunk & 31));
        }
      }
      n += __popcll(all);
    }
    if (threadIdx.x == 0) picked = n;
  }
  __syncthreads();
  auto dense = [&](float x) { return Q * fexp2((x - m) * c - l2S); };
#pragma unroll
  for (int u = 0; u < kDistLoads; ++u) {
    const int at = u * 256 + threadIdx.x, k = k0 + at;
    if (k >= rc.chunks) break;
    const int j0 = rc.head + k * PER;
    float x[PER];
    if constexpr (VEC) unpack_chunk<DT>(v[u], x);
    else
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] = (float)row[j0 + e];
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] = dense(x[e]);
    if (marks[at >> 5] >> (at & 31) & 1)
      for (int s = 0; s < picked; ++s) {
        const uint32_t o = (uint32_t)(slot_col[s] - j0);
        if (o < (uint32_t)PER)
#pragma unroll
          for (int e = 0; e < PER; ++e) x[e] -= (int)o == e ? slot_q[s] : 0.f;
      }
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] *= gs;
    if constexpr (VEC) *(i32x4 *)(drow + j0) = pack_chunk<DT>(x);
    else
#pragma unroll
      for (int e = 0; e < PER; ++e) drow[j0 + e] = (T)x[e];
  }
  if (edge) {
    float x = dense((float)row[je]);
    for (int s = 0; s < picked; ++s) x -= slot_col[s] == je ? slot_q[s] : 0.f;
    drow[je] = (T)(gs * x);
  }
}

template <int DT>
static void go_fwd(const void *logits, int64_t ld, const int64_t *ids, const float *teacher, int64_t n, int V, int K,
                   float inv_T, int raw, float *kl, float *state, float *q, hipStream_t st) {
  for (int64_t r0 = 0; r0 < n; r0 += kLaunchRows)
    hipLaunchKernelGGL(distill_columns_fwd_kernel<DT>, dim3((unsigned)(n - r0 < kLaunchRows ? n - r0 : kLaunchRows)),
                       dim3(kDistThreads), 0, st, (const char *)logits + r0 * ld * Elem<DT>::bytes, ld, ids + r0 * K,
                       teacher + r0 * K, V, K, inv_T, raw, kl + r0, state + 4 * r0, q + r0 * K);
}

template <int DT>
static void go_bwd(const void *logits, int64_t ld, const int64_t *ids, const float *q, int64_t n, int V, int K,
                   float inv_T, const float *state, const float *g, void *dl, int64_t ld_d, hipStream_t st) {
  constexpr int B = Elem<DT>::bytes, PER = 16 / B;
  const int64_t chunks = V / PER > 0 ? V / PER : 1;
  // rows whose logits and gradients start at the same offset from a 16-byte boundary; others go value by value
  const bool vec = ((uintptr_t)logits - (uintptr_t)dl) % 16 == 0 && ((ld - ld_d) * B) % 16 == 0;
  for (int64_t r0 = 0; r0 < n; r0 += 65535) {  // rows per launch: the grid's y
    const int64_t rows = n - r0 < 65535 ? n - r0 : 65535;
    const dim3 grid((unsigned)cdiv(chunks, 256 * kDistLoads), (unsigned)rows);
    const char *z = (const char *)logits + r0 * ld * B;
    char *d = (char *)dl + r0 * ld_d * B;
    if (vec)
      hipLaunchKernelGGL((distill_columns_bwd_kernel<DT, true>), grid, dim3(256), 0, st, z, ld, ids + r0 * K,
                         q + r0 * K, V, K, inv_T, state + 4 * r0, g + r0, d, ld_d);
    else
      hipLaunchKernelGGL((distill_columns_bwd_kernel<DT, false>), grid, dim3(256), 0, st, z, ld, ids + r0 * K,
                         q + r0 * K, V, K, inv_T, state + 4 * r0, g + r0, d, ld_d);
  }
}

// ---- the distillation step over hidden rows -------------------------------------------------------------------------
// A listed logit in the softmax's base-2 units before the row's maximum is taken off: x c, x the (soft-capped) logit.
__device__ __forceinline__ float listed_x(const DistillArgs &a, float dot, int64_t y, bool exact_tanh) {
  const float x = a.w_dtype == OCTO_FP8E4M3 ? dot * a.wscale[y] : dot;
  return a.use_tanh ? (exact_tanh ? tanhf(a.pre * x) : ftanh(a.pre * x)) : x;
}

// One workgroup per compact row. A wave takes kDotSlots slots at a time, so that a part of the hidden row is read once
// for all of them and their loads are in flight together; the lanes' sums are exchanged and halved together. fp8
// weights are read from their widened copy. Bound by the gathered weight rows, n K d x 2 bytes out of the caches: 8,192
// rows, K 64, d 2560 (2.7 GB) 365 us, 7.4 TB/s (8 waves a row 413; a slot at a time 504).
constexpr int kDotWaves = 4, kDotSlots = 8;
template <int DT>
__device__ __forceinline__ float dot_slots(const char *h, const char *const (&w)[kDotSlots], int d, int lane) {
  constexpr int PER = 16 / Elem<DT>::bytes;
  float s[kDotSlots] = {};
#pragma unroll 1
  for (int k = lane; k < d / PER; k += 64) {
    i32x4 wv[kDotSlots];
    const i32x4 hv = *(const i32x4 *)(h + k * 16);
#pragma unroll
    for (int j = 0; j < kDotSlots; ++j) wv[j] = *(const i32x4 *)(w[j] + k * 16);
    float a[PER], b[PER];
    unpack_chunk<DT>(hv, a);
#pragma unroll
    for (int j = 0; j < kDotSlots; ++j) {
      unpack_chunk<DT>(wv[j], b);
#pragma unroll
      for (int e = 0; e < PER; ++e) s[j] = __builtin_fmaf(a[e], b[e], s[j]);
    }
  }
  // lane l ends with the sum of slot (l >> 3) & 7
#pragma unroll
  for (int half = kDotSlots / 2, o = 32; half >= 1; half >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < kDotSlots / 2; ++j)
      if (j < half) {
        const float keep = up ? s[j + half] : s[j], give = up ? s[j] : s[j + half];
        s[j] = keep + __shfl_xor(give, o, 64);
      }
  }
  float t = s[0];
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  return t;
}

template <int DT>
__global__ __launch_bounds__(64 * kDotWaves) void distill_dots_kernel(DistillArgs a) {
  __shared__ float best[kDotWaves];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t r = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (r == 0)
    for (int k = threadIdx.x; k < a.nflag; k += 64 * waves) a.flag_cnt[k] = 0;
  const int64_t cnt = a.count ? min((int64_t)(*a.count), a.n_max) : a.n_max;
  if (r >= cnt) return;
  const int64_t hrow = a.idx ? a.idx[r] : r;
  const int64_t *ids = a.ids + hrow * a.K;
  const float *teacher = a.teacher + hrow * a.K;
  auto token = [&](int k) {  // -1 for an empty slot
    if (k >= a.K) return (int64_t)-1;
    const int64_t y = ids[k];
    return y >= 0 && y < a.V && teacher[k] != -INFINITY ? y : (int64_t)-1;
  };
  float top = -INFINITY;
  for (int k0 = w * kDotSlots; k0 < a.K; k0 += waves * kDotSlots) {
    const int64_t mine = token(k0 + (lane >> 3));  // the slot whose sum this lane ends with
    const uint64_t used = __ballot(mine >= 0);
    float dot = 0.f;
    if (used) {
      const int64_t any = __shfl(mine, __ffsll((unsigned long long)used) - 1, 64);
      const char *rows[kDotSlots];
#pragma unroll
      for (int j = 0; j < kDotSlots; ++j) {  // an empty slot reads another's row
        const int64_t y = __shfl(mine, 8 * j, 64);
        rows[j] = (const char *)a.wm + (y >= 0 ? y : any) * a.ldm * Elem<DT>::bytes;
      }
      dot = dot_slots<DT>((const char *)a.h + hrow * a.ldh * Elem<DT>::bytes, rows, a.d, lane);
      if (mine >= 0) top = fmaxf(top, listed_x(a, dot, mine, false));
      else dot = 0.f;
    }
    if ((lane & 7) == 0 && k0 + (lane >> 3) < a.K) a.dots[r * a.K + k0 + (lane >> 3)] = dot;
  }
  top = wave_max(top);
  if (lane == 0) best[w] = top;
  __syncthreads();
  if (threadIdx.x == 0 && a.xoff) {
    for (int k = 0; k < waves; ++k) top = fmaxf(top, best[k]);
    a.xoff[r] = top == -INFINITY ? -INFINITY : __builtin_fmaf(top, a.c, kExAbove);
  }
}

// One wave per row: merges the row's partials as merge_kernel does, then lane l takes slots l + 64 i.
constexpr int kDistMergeRows = 4;
__global__ __launch_bounds__(64 * kDistMergeRows) void distill_merge_kernel(DistillArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kDistMergeRows + (threadIdx.x >> 6);
  const int64_t r = a.r0 + i;
  const int lane = threadIdx.x & 63;
  const int64_t cnt = a.count ? min((int64_t)(*a.count), a.n_max) : a.n_max;
  if (i >= a.rows || r >= cnt) return;
  const int64_t hrow = a.idx ? a.idx[r] : r;
  Stat3 st{-INFINITY, 0.f, 0.f};
  const f32x4 *pr = a.part + i * a.mtiles;
  for (int64_t k0 = lane; k0 < a.mtiles; k0 += 64 * kRowLoads) {
    f32x4 p[kRowLoads];
#pragma unroll
    for (int u = 0; u < kRowLoads; ++u) p[u] = pr[min(k0 + 64 * u, a.mtiles - 1)];
#pragma unroll
    for (int u = 0; u < kRowLoads; ++u) {
      if (k0 + 64 * u >= a.mtiles) break;
      st = stat_merge(st, Stat3{fmaxf(p[u][0], p[u][3]), p[u][1], p[u][2]});
    }
  }
  st = wave_stat_merge(st);
  const float l2S = flog2(st.S);
  int64_t id[kSlots];
  float q[kSlots], lq[kSlots], Q, sum = 0.f;
  teacher_slots(a.ids + hrow * a.K, a.teacher + hrow * a.K, a.K, a.V, a.raw != 0, lane, id, q, lq, Q);
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    const int k = lane + 64 * s;
    if (k >= a.K) break;
    if (id[s] >= 0 && q[s] != 0.f) {
      const float x = listed_x(a, a.dots[r * a.K + k], id[s], true);
      sum += q[s] * (lq[s] - (__builtin_fmaf(x, a.c, -st.m) - l2S) * OCTO_LN2);
    }
    a.q[r * a.K + k] = q[s];
  }
  sum = wave_sum(sum);
  if (lane != 0) return;
  const float wt = a.weight ? a.weight[hrow] : 1.f, g = -wt * Q;
  a.kl[hrow] = sum;
  a.g[r] = g;
  a.lse[2 * r] = st.m;
  a.lse[2 * r + 1] = l2S;
  if (a.rowoff) {
    const float xo = a.xoff[r];
    const bool low = !(st.m - xo <= kExClamp);  // the offset lies too low, or there is none
    float xn = low ? st.m : xo;
    if (a.even) {  // the dz scale |g gmul| exp2(xn - m2 - l2S) a power of two (not of a weight of 0 or inf)
      const float ls = flog2(fabsf(g * a.gmul)) + (xn - st.m - l2S);  // gmul < 0: a soft-cap with pre < 0
      if (fabsf(ls) < 1024.f) xn += rintf(ls) - ls;
    } else if (low && g != 0.f) {  // a row without weight needs no rescale, its scale is 0
      a.flag_rows[atomicAdd(a.flag_cnt, 1)] = (int32_t)i;
    }
    a.xuse[i] = xn;
  }
}

// The maximum of a half tile's 128 exponentials, whose value is known in fp32, before it was rounded to 16 bits. 16
// neighbouring lanes, all active, hold 8 of them each: v as stored, x as fp32. Where one value of them all has the
// maximum's bits `top`, its x becomes `exact`; where more do, which of them is the maximum cannot be told.
__device__ __forceinline__ void unround_max(const i32x4 v, uint32_t top, float exact, float (&x)[8]) {
  uint32_t hit = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) hit |= (((uint32_t)v[e >> 1] >> (16 * (e & 1))) & 0xffffu) == top ? 1u << e : 0u;
  const uint64_t lanes = __ballot(hit != 0) >> (threadIdx.x & 48) & 0xffffu;
  if ((hit & (hit - 1)) || __popcll(lanes) != 1) hit = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = hit >> e & 1 ? exact : x[e];
}

// Every row's exponentials from the offset they were stored at to xuse, and its dz scale: launch_ex_fix's work for all
// rows, where grad_W is asked for. h^T times the row's scale is rounded to bf16 there; at a scale of 2^k (1 + 2^-17 or
// so, from xuse's own rounding) that product is h's own bits, and what is rounded a second time are the dense entries.
// The ones that weigh, a student's own likely tokens, are nearly always their half tile's maximum, which the statistics
// keep in fp32: they are made of that and rounded once. So are the listed ones, and grad_W's error falls from 2.9e-3 to
// 2.35e-3 (one rounding of the result alone is 1.7e-3); a student certain of tokens off its list (0.3 of the norm's
// square) 2.54e-3 with the maxima rounded twice, 2.4e-3 now. Bound by memory, 4 bytes an element: [8,192, 151,936] 790
// us (6.3 TB/s), 5% of the call.
constexpr int kEvenChunks = 2;  // 16-byte chunks per thread
__global__ __launch_bounds__(256) void distill_even_kernel(DistillArgs a, float *scale) {
  const int64_t cnt = a.count ? min((int64_t)(*a.count), a.n_max) : a.n_max;
  const int64_t chunk0 = (int64_t)blockIdx.x * (256 * kEvenChunks) + threadIdx.x;
  const float inv_c = 1.f / a.c;
  for (int64_t i = blockIdx.y; i < a.rows; i += gridDim.y) {
    const int64_t r = a.r0 + i;
    const bool in = r < cnt;
    const float g = in ? a.g[r] : 0.f;
    if (g == 0.f) {  // also past the count: the scale of 0 leaves the row out
      if (blockIdx.x == 0 && threadIdx.x == 0) scale[i] = 0.f;
      continue;
    }
    const float xo = a.xoff[r], xn = a.xuse[i];
    if (blockIdx.x == 0 && threadIdx.x == 0)
      scale[i] = -(g * a.gmul) * fexp2(xn - a.lse[2 * r] - a.lse[2 * r + 1]);
    const f32x4 *pr = a.part + i * a.mtiles;
    __bf16 *row = (__bf16 *)a.dz + i * a.ldx;
    i32x4 v[kEvenChunks];
#pragma unroll
    for (int u = 0; u < kEvenChunks; ++u) {
      const int64_t c0 = (chunk0 + 256 * u) * 8;
      if (c0 < a.ldx) v[u] = __builtin_nontemporal_load((const i32x4 *)(row + c0));
    }
#pragma unroll
    for (int u = 0; u < kEvenChunks; ++u) {
      const int64_t c0 = (chunk0 + 256 * u) * 8;
      if (c0 >= a.ldx) continue;
      const f32x4 q = pr[c0 >> 8];  // 8 columns never straddle a 128-column half tile
      const float mh = (c0 & 128) ? q[3] : q[0];  // -inf: no column of the half lies below V (stored zeros)
      const float above = fminf(mh - xo, kExClamp), fac = mh == -INFINITY ? 0.f : fexp2(mh - xn - above);
      float x[8];
      unpack8(v[u], false, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= fac;
      const float th = a.use_tanh ? mh * inv_c : 0.f, slope = 1.f - th * th;  // as the epilogue stored it
      unround_max(v[u], __builtin_bit_cast(uint16_t, (__bf16)(slope * fexp2(above))), slope * fexp2(mh - xn), x);
      __builtin_nontemporal_store(pack8(x, false), (i32x4 *)(row + c0));
    }
  }
}

// A workgroup's sum of the loss: every thread's rows in order, in 64 bits, then a tree.
constexpr int kLossThreads = 256;
__device__ __forceinline__ void loss_sum(const DistillArgs &a, double *part) {
  const int64_t cnt = a.count ? min((int64_t)(*a.count), a.n_max) : a.n_max;
  double s = 0.0;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < cnt; r += kLossThreads) {
    const int64_t hrow = a.idx ? a.idx[r] : r;
    const float wt = a.weight ? a.weight[hrow] : 1.f, kl = a.kl[hrow];
    s += wt != 0.f ? (double)wt * (double)kl : 0.0;  // a row without weight, whatever its divergence is
  }
  part[threadIdx.x] = s;
  __syncthreads();
  for (int k = kLossThreads / 2; k > 0; k >>= 1) {
    if ((int)threadIdx.x < k) part[threadIdx.x] += part[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) *a.loss = (float)part[0];
}

// One wave per row. Slots of one token all write the sum of their weights, taken in the list's order. The last pass's
// launch has a workgroup more, the loss's: every row's kl is there by then (a launch of its own: 4 us of a call's 130
// at 225 rows, V 32,000).
constexpr int kEntryRows = 4;
static_assert(64 * kEntryRows == kLossThreads, "the loss's workgroup");
__global__ __launch_bounds__(64 * kEntryRows) void distill_entries_kernel(DistillArgs a) {
  __shared__ int64_t slot_id[kEntryRows][OCTO_LIST_MAX];
  __shared__ float slot_q[kEntryRows][OCTO_LIST_MAX];
  if ((int64_t)blockIdx.x * kEntryRows >= a.rows) {
    loss_sum(a, (double *)slot_id);
    return;
  }
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * kEntryRows + w, r = a.r0 + i;
  const int64_t cnt = a.count ? min((int64_t)(*a.count), a.n_max) : a.n_max;
  const bool in = i < a.rows && r < cnt;
  const int64_t hrow = in ? (a.idx ? a.idx[r] : r) : 0;
  float Q = 0.f;
  if (in) {
    for (int k = lane; k < a.K; k += 64) {
      const float q = a.q[r * a.K + k];
      slot_q[w][k] = q;
      const int64_t y = a.ids[hrow * a.K + k] - a.v0;
      slot_id[w][k] = q != 0.f && y >= 0 && y < a.cols ? y : -1;  // an empty slot has q 0
      Q += q;
    }
    Q = wave_sum(Q);
  }
  __syncthreads();
  if (!in) return;
  const float g = a.g[r];
  if (g == 0.f) return;
  const float m2 = a.lse[2 * r], l2S = a.lse[2 * r + 1];
  for (int k = lane; k < a.K; k += 64) {
    const int64_t col = slot_id[w][k], y = col + a.v0;
    if (col < 0) continue;
    float share = 0.f;
    for (int j = 0; j < a.K; ++j) share += slot_id[w][j] == col ? slot_q[w][j] : 0.f;
    const float x = listed_x(a, a.dots[r * a.K + k], y, false);
    float v = share / Q - fexp2(__builtin_fmaf(x, a.c, -m2) - l2S);
    if (a.use_tanh) v *= 1.f - x * x;
    if (a.w_dtype == OCTO_FP8E4M3) v *= a.wscale[y];
    if (a.rowoff) ((__bf16 *)a.dz)[i * a.ldx + col] = (__bf16)(-v * fexp2(m2 - a.xuse[i] + l2S));
    else store_from_f32(a.dz, a.dt, i * a.ldx + col, g * a.gmul * v);
  }
}

__global__ __launch_bounds__(kLossThreads) void distill_loss_kernel(DistillArgs a) {
  __shared__ double part[kLossThreads];
  loss_sum(a, part);
}

int launch_distill_dots(const DistillArgs &a, hipStream_t st) {
  if (a.n_max == 0) return OCTO_OK;
  // no more waves than have slots: 4,000 rows of K 20, 149 us with 8 each, 95 with 3
  const int waves = (int)cdiv(a.K, kDotSlots);
  const dim3 g((unsigned)(a.n_max < kLaunchRows ? a.n_max : kLaunchRows), (unsigned)cdiv(a.n_max, kLaunchRows));
  const dim3 b(64 * (waves < kDotWaves ? waves : kDotWaves));
  if (a.dt == OCTO_BF16) hipLaunchKernelGGL(distill_dots_kernel<OCTO_BF16>, g, b, 0, st, a);
  else if (a.dt == OCTO_F16) hipLaunchKernelGGL(distill_dots_kernel<OCTO_F16>, g, b, 0, st, a);
  else hipLaunchKernelGGL(distill_dots_kernel<OCTO_F32>, g, b, 0, st, a);
  OCTO_CHECK_LAUNCH("distill_dots");
  return OCTO_OK;
}
int launch_distill_merge(const DistillArgs &a, hipStream_t st) {
  if (a.rows == 0) return OCTO_OK;
  hipLaunchKernelGGL(distill_merge_kernel, dim3((unsigned)cdiv(a.rows, kDistMergeRows)), dim3(64 * kDistMergeRows), 0,
                     st, a);
  OCTO_CHECK_LAUNCH("distill_merge");
  return OCTO_OK;
}
int launch_distill_even(const DistillArgs &a, float *scale, hipStream_t st) {
  if (a.rows == 0) return OCTO_OK;
  OCTO_CHECK_ARG(a.ldx % 256 == 0 && (uintptr_t)a.dz % 16 == 0, "distill_even: rows of whole 256-column tiles");
  const dim3 g((unsigned)cdiv(a.ldx / 8, 256 * kEvenChunks), (unsigned)(a.rows < 65535 ? a.rows : 65535));
  hipLaunchKernelGGL(distill_even_kernel, g, dim3(256), 0, st, a, scale);
  OCTO_CHECK_LAUNCH("distill_even");
  return OCTO_OK;
}
int launch_distill_entries(const DistillArgs &a, hipStream_t st) {
  if (a.rows == 0) return OCTO_OK;
  const int64_t blocks = cdiv(a.rows, kEntryRows) + (a.loss ? 1 : 0);
  hipLaunchKernelGGL(distill_entries_kernel, dim3((unsigned)blocks), dim3(64 * kEntryRows), 0, st, a);
  OCTO_CHECK_LAUNCH("distill_entries");
  return OCTO_OK;
}
int launch_distill_loss(const DistillArgs &a, float *loss, hipStream_t st) {
  DistillArgs b = a;
  b.loss = loss;
  hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(kLossThreads), 0, st, b);
  OCTO_CHECK_LAUNCH("distill_loss");
  return OCTO_OK;
}

}  // namespace octo

using namespace octo;

extern "C" {

int octo_distill_columns_fwd(const void *logits, int64_t ld, int dtype, const int64_t *ids, const float *teacher,
                             int64_t n, int V, int K, float inv_T, int flags, float *kl, float *state, float *q,
                             void *stream) {
  OCTO_CHECK_ARG(n >= 0 && n <= 0x7fffffff && V > 0 && V <= OCTO_ROW_MAX && ld >= V,
                 "distill_columns_fwd: bad shape n=%lld V=%d ld=%lld", (long long)n, V, (long long)ld);
  OCTO_CHECK_ARG(K >= 1 && K <= OCTO_LIST_MAX, "distill_columns_fwd: K=%d outside [1, %d]", K, OCTO_LIST_MAX);
  OCTO_CHECK_ARG(is_float(dtype), "distill_columns_fwd: dtype %d", dtype);
  OCTO_CHECK_ARG((flags & ~OCTO_LIST_RAW) == 0, "distill_columns_fwd: unknown flags %d", flags);
  OCTO_CHECK_ARG(inv_T > 0.f, "distill_columns_fwd: temperature must be positive");
  if (n == 0) return OCTO_OK;
  OCTO_CHECK_ARG(logits && ids && teacher && kl && state && q, "distill_columns_fwd: null pointer");
  OCTO_CHECK_ARG((uintptr_t)logits % float_bytes(dtype) == 0, "distill_columns_fwd: misaligned logits");
  hipStream_t st = (hipStream_t)stream;
  const int raw = (flags & OCTO_LIST_RAW) != 0;
  if (dtype == OCTO_BF16) go_fwd<OCTO_BF16>(logits, ld, ids, teacher, n, V, K, inv_T, raw, kl, state, q, st);
  else if (dtype == OCTO_F16) go_fwd<OCTO_F16>(logits, ld, ids, teacher, n, V, K, inv_T, raw, kl, state, q, st);
  else go_fwd<OCTO_F32>(logits, ld, ids, teacher, n, V, K, inv_T, raw, kl, state, q, st);
  OCTO_CHECK_LAUNCH("distill_columns_fwd");
  return OCTO_OK;
}

int octo_distill_columns_bwd(const void *logits, int64_t ld, int dtype, const int64_t *ids, const float *q, int64_t n,
                             int V, int K, float inv_T, const float *state, const float *g, void *dlogits,
                             int64_t ld_d, void *stream) {
  OCTO_CHECK_ARG(n >= 0 && n <= 0x7fffffff && V > 0 && V <= OCTO_ROW_MAX && ld >= V && ld_d >= V,
                 "distill_columns_bwd: bad shape");
  OCTO_CHECK_ARG(K >= 1 && K <= OCTO_LIST_MAX, "distill_columns_bwd: K=%d outside [1, %d]", K, OCTO_LIST_MAX);
  OCTO_CHECK_ARG(is_float(dtype), "distill_columns_bwd: dtype %d", dtype);
  OCTO_CHECK_ARG(inv_T > 0.f, "distill_columns_bwd: temperature must be positive");
  if (n == 0) return OCTO_OK;
  OCTO_CHECK_ARG(logits && ids && q && state && g && dlogits, "distill_columns_bwd: null pointer");
  OCTO_CHECK_ARG((uintptr_t)logits % float_bytes(dtype) == 0 && (uintptr_t)dlogits % float_bytes(dtype) == 0,
                 "distill_columns_bwd: misaligned logits");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == OCTO_BF16) go_bwd<OCTO_BF16>(logits, ld, ids, q, n, V, K, inv_T, state, g, dlogits, ld_d, st);
  else if (dtype == OCTO_F16) go_bwd<OCTO_F16>(logits, ld, ids, q, n, V, K, inv_T, state, g, dlogits, ld_d, st);
  else go_bwd<OCTO_F32>(logits, ld, ids, q, n, V, K, inv_T, state, g, dlogits, ld_d, st);
  OCTO_CHECK_LAUNCH("distill_columns_bwd");
  return OCTO_OK;
}

}  // extern "C"
