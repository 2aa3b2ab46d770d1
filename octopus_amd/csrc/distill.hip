// The divergence of a student's logits from a teacher's lists (octo_distill_columns_fwd / _bwd). A row's list holds K
// slots (id, t): t the teacher's logit or log-probability of token id. A slot whose id lies outside [0, V), or whose t
// is -inf, is empty.
//
//   q = softmax of t over the row's slots (OCTO_LIST_RAW: exp(t)),  Q = sum q,  p = softmax(z / T)
//   kl = sum_k q_k (log q_k - log p_id_k)        a row without a slot: 0
//   dL/dz_v = g (Q p_v - sum of q_k over the slots with id_k = v) / T,   g = dL/dkl
//
// Both directions are bound by memory: the forward reads each logit once, the backward reads it once more and writes
// its gradient. The forward leaves q, and the row's (maximum, ln S), for the backward.
#include "octo_common.h"
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
__global__ __launch_bounds__(kDistThreads) void distill_columns_fwd_kernel(const void *logits, int64_t ld,
                                                                           const int64_t *ids, const float *teacher,
                                                                           int V, int K, float inv_T, int raw,
                                                                           float *kl, float *state, float *q_out) {
  constexpr int PER = 16 / Elem<DT>::bytes, NW = kDistThreads / 64;
  typedef typename Elem<DT>::T T;
  __shared__ float red[2][NW];
  const int64_t r = blockIdx.x;
  const T *row = (const T *)logits + r * ld;
  const float c = inv_T * OCTO_LOG2E;
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
  const int lane = threadIdx.x;
  const float lnS = flog2(S) * OCTO_LN2;
  int64_t id[kSlots];
  float q[kSlots], lq[kSlots], Q, sum = 0.f;
  teacher_slots(ids + r * K, teacher + r * K, K, V, raw != 0, lane, id, q, lq, Q);
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int k = lane + 64 * i;
    // q 0 (an exp that underflows): its term's limit, 0, whatever log p is
    if (id[i] >= 0 && q[i] != 0.f) sum += q[i] * (lq[i] - (((float)row[id[i]] - m) * inv_T - lnS));
    if (k < K) q_out[r * K + k] = q[i];
  }
  sum = wave_sum(sum);
  if (lane == 0) {
    kl[r] = sum;
    state[4 * r] = m;
    state[4 * r + 1] = flog2(S);
    state[4 * r + 2] = Q;
    state[4 * r + 3] = 0.f;
  }
}

// One workgroup per kDistLoads x 256 chunks of a row. The slots that lie in its columns are marked by chunk in a bit
// map; a thread with a marked chunk looks through the list.
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
  for (int i = threadIdx.x; i < kMarkWords; i += 256) marks[i] = 0;
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += 256) {
    const float qk = q[r * K + k];
    const int64_t y = ids[r * K + k];
    const int col = qk != 0.f && y >= 0 && y < V ? (int)y : -1;
    slot_col[k] = col;
    slot_q[k] = qk;
    if (col >= rc.head && col < tail) {
      const int at = (col - rc.head) / PER - k0;
      if (at >= 0 && at < 256 * kDistLoads) atomicOr(&marks[at >> 5], 1u << (at & 31));
    }
  }
  __syncthreads();
  // the slots of column j, in the order of the list
  auto listed = [&](int j) {
    float s = 0.f;
    for (int k = 0; k < K; ++k) s += slot_col[k] == j ? slot_q[k] : 0.f;
    return s;
  };
  auto dense = [&](float x) { return Q * fexp2((x - m) * c - l2S); };
  i32x4 v[kDistLoads];
  if constexpr (VEC) {
#pragma unroll
    for (int u = 0; u < kDistLoads; ++u) {
      const int k = k0 + u * 256 + threadIdx.x;
      if (k < rc.chunks) v[u] = *(const i32x4 *)(row + rc.head + k * PER);
    }
  }
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
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] -= listed(j0 + e);
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] *= gs;
    if constexpr (VEC) *(i32x4 *)(drow + j0) = pack_chunk<DT>(x);
    else
#pragma unroll
      for (int e = 0; e < PER; ++e) drow[j0 + e] = (T)x[e];
  }
  if (edge) drow[je] = (T)(gs * (dense((float)row[je]) - listed(je)));
}

template <int DT>
static void go_fwd(const void *logits, int64_t ld, const int64_t *ids, const float *teacher, int64_t n, int V, int K,
                   float inv_T, int raw, float *kl, float *state, float *q, hipStream_t st) {
  hipLaunchKernelGGL(distill_columns_fwd_kernel<DT>, dim3((unsigned)n), dim3(kDistThreads), 0, st, logits, ld, ids,
                     teacher, V, K, inv_T, raw, kl, state, q);
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

}  // namespace octo

using namespace octo;

extern "C" {

int octo_distill_columns_fwd(const void *logits, int64_t ld, int dtype, const int64_t *ids, const float *teacher,
                             int64_t n, int V, int K, float inv_T, int flags, float *kl, float *state, float *q,
                             void *stream) {
  OCTO_CHECK_ARG(n >= 0 && n <= 0x7fffffff && V > 0 && ld >= V, "distill_columns_fwd: bad shape n=%lld V=%d ld=%lld",
                 (long long)n, V, (long long)ld);
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
  OCTO_CHECK_ARG(n >= 0 && n <= 0x7fffffff && V > 0 && ld >= V && ld_d >= V, "distill_columns_bwd: bad shape");
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
