// The teacher's list of a row of logits: its k largest values, their columns and log-probabilities (octo_topk).
//
//   ids[r] = the columns of the k largest z_rv, by value descending, equal values by column ascending
//   logp[r][j] = z_r,ids[j] / T - logsumexp_v(z_rv / T)
//
// One workgroup per row. The first sweep takes the row's logsumexp and each thread's largest value. At least k values of
// the row are no smaller than the k-th largest of the threads' maxima, so that one is a lower bound of the list, and a
// close one: 1,024 threads of 148 values each hold two of the 64 largest now and then. The second sweep collects what
// reaches the bound; every collected value is ranked against the others by (value, column) and the first k ranks are
// the list. Rows with more than kCand such values (long runs of equal ones) or with a NaN or +inf are done by a radix
// select over the values' 32-bit keys instead, any row correctly.
#include "octo_common.h"
#include "row_values.h"

namespace octo {

constexpr int kTopThreads = 1024;
constexpr int kTopLoads = 4;   // 16-byte chunks in flight per thread
constexpr int kCand = 2048;    // values that may reach the bound

// The order of the list as unsigned numbers: NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// larger is earlier in the list
__device__ __forceinline__ uint64_t list_entry(float x, int col) {
  return ((uint64_t)order_key(x) << 32) | (uint32_t)~col;
}

// f(x, column) for every value of the row that this thread takes, each value once over the workgroup; pre(chunk
// maximum) says whether any value of a chunk is wanted.
template <int DT, class Pre, class F>
__device__ __forceinline__ void sweep_row(const typename Elem<DT>::T *row, int V, Pre pre, F f) {
  constexpr int PER = 16 / Elem<DT>::bytes;
  const RowChunks rc = row_chunks<DT>(row, V);
  const i32x4 *vec = (const i32x4 *)(row + rc.head);
  for (int k0 = threadIdx.x; k0 < rc.chunks; k0 += kTopLoads * kTopThreads) {
    i32x4 v[kTopLoads];
#pragma unroll
    for (int u = 0; u < kTopLoads; ++u) v[u] = vec[min(k0 + u * kTopThreads, rc.chunks - 1)];
#pragma unroll
    for (int u = 0; u < kTopLoads; ++u) {
      const int k = k0 + u * kTopThreads;
      if (k >= rc.chunks) break;
      float x[PER], mx = -INFINITY;
      unpack_chunk<DT>(v[u], x);
#pragma unroll
      for (int e = 0; e < PER; ++e) mx = fmaxf(mx, x[e]);
      if (pre(mx)) {
#pragma unroll
        for (int e = 0; e < PER; ++e) f(x[e], rc.head + k * PER + e);
      }
    }
  }
  const int tail = rc.head + rc.chunks * PER;
  const int j = (int)threadIdx.x < rc.head ? (int)threadIdx.x : (int)threadIdx.x - rc.head + tail;
  if (j < rc.head || (j >= tail && j < V)) f((float)row[j], j);
}

template <int DT>
__global__ __launch_bounds__(kTopThreads) void topk_kernel(const void *logits, int64_t ld, int V, float inv_T, int k,
                                                           int64_t *ids, float *logp) {
  constexpr int PER = 16 / Elem<DT>::bytes, NW = kTopThreads / 64;
  typedef typename Elem<DT>::T T;
  __shared__ float red[2][NW];
  __shared__ int cnts[2][NW];
  __shared__ uint64_t cand[kCand];
  __shared__ int hist[256];
  __shared__ int ncand, sel_bin, sel_above;
  const int64_t r = blockIdx.x;
  const T *row = (const T *)logits + r * ld;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const float c = inv_T * OCTO_LOG2E;

  // ---- the row's logsumexp and this thread's largest value
  RowSum st;
  float top = -INFINITY;
  {
    const RowChunks rc = row_chunks<DT>(row, V);
    const i32x4 *vec = (const i32x4 *)(row + rc.head);
    for (int k0 = threadIdx.x; k0 < rc.chunks; k0 += kTopLoads * kTopThreads) {
      i32x4 v[kTopLoads];
#pragma unroll
      for (int u = 0; u < kTopLoads; ++u)  // past the end: the last chunk again, left out below
        v[u] = vec[min(k0 + u * kTopThreads, rc.chunks - 1)];
      float x[kTopLoads][PER], mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < kTopLoads; ++u) {
        unpack_chunk<DT>(v[u], x[u]);
        if (k0 + u * kTopThreads < rc.chunks)
#pragma unroll
          for (int e = 0; e < PER; ++e) mx = fmaxf(mx, x[u][e]);
      }
      top = fmaxf(top, mx);
      st.raise(mx, c);
#pragma unroll
      for (int u = 0; u < kTopLoads; ++u)
        if (k0 + u * kTopThreads < rc.chunks)
#pragma unroll
          for (int e = 0; e < PER; ++e) st.add(x[u][e], c);
    }
    const int tail = rc.head + rc.chunks * PER;
    const int j = (int)threadIdx.x < rc.head ? (int)threadIdx.x : (int)threadIdx.x - rc.head + tail;
    if (j < rc.head || (j >= tail && j < V)) {
      const float x = (float)row[j];
      top = fmaxf(top, x);
      st.raise(x, c);
      st.add(x, c);
    }
  }
  float m, S;
  if (threadIdx.x == 0) ncand = 0;
  block_row_sum<NW>(st, c, red, m, S);
  const float lnS = flog2(S) * OCTO_LN2;
  bool listed = S == S;  // no NaN, no +inf

  if (listed) {
    // ---- the bound: the k-th largest of the threads' maxima, to its upper 16 bits (rounded down)
    const uint32_t key = order_key(top) >> 16;
    uint32_t bound = 0;
    for (int b = 15, it = 0; b >= 0; --b, ++it) {
      const uint32_t test = bound | (1u << b);
      const int have = __popcll(__ballot(key >= test));
      if (lane == 0) cnts[it & 1][w] = have;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int q = 0; q < NW; ++q) all += cnts[it & 1][q];
      if (all >= k) bound = test;
    }
    const float least = bound <= 0x007fu ? -INFINITY : key_value(bound << 16);
    // ---- what reaches it
    sweep_row<DT>(row, V, [&](float mx) { return mx >= least; },
                  [&](float x, int j) {
                    if (x >= least) {
                      const int at = atomicAdd(&ncand, 1);
                      if (at < kCand) cand[at] = list_entry(x, j);
                    }
                  });
    __syncthreads();
    listed = ncand <= kCand;
  }
  if (!listed) {
    // ---- radix select: the key of the k-th value, 8 bits at a time
    uint32_t prefix = 0;
    int above = 0;  // values whose key is larger than every key that starts with prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (threadIdx.x < 256) hist[threadIdx.x] = 0;
      __syncthreads();
      const uint32_t high = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      sweep_row<DT>(row, V, [](float) { return true; },
                    [&](float x, int) {
                      const uint32_t q = order_key(x);
                      if ((q & high) == prefix) atomicAdd(&hist[(q >> shift) & 255], 1);
                    });
      __syncthreads();
      if (threadIdx.x == 0) {
        int a = above, b = 255;
        while (b > 0 && a + hist[b] < k) a += hist[b--];
        sel_bin = b;
        sel_above = a;
      }
      __syncthreads();
      prefix |= (uint32_t)sel_bin << shift;
      above = sel_above;
    }
    // the values above it, and of its equals the first k - above columns
    if (threadIdx.x == 0) ncand = 0;
    __syncthreads();
    int equals = 0;
    for (int s0 = 0, it = 0; s0 < V; s0 += kTopThreads, ++it) {
      const int j = s0 + (int)threadIdx.x;
      const float x = j < V ? (float)row[j] : 0.f;
      const uint32_t q = order_key(x);
      const bool eq = j < V && q == prefix;
      if (j < V && q > prefix) cand[atomicAdd(&ncand, 1)] = list_entry(x, j);  // fewer than k of them
      const uint64_t bal = __ballot(eq);
      if (lane == 0) cnts[it & 1][w] = __popcll(bal);
      __syncthreads();
      int off = equals;
#pragma unroll
      for (int u = 0; u < NW; ++u) {
        off += u < w ? cnts[it & 1][u] : 0;
        equals += cnts[it & 1][u];
      }
      off += __popcll(bal & ((1ull << lane) - 1ull));
      if (eq && off < k - above) cand[k - 1 - off] = list_entry(x, j);  // from the other end: above + equals = k
    }
    __syncthreads();
    if (threadIdx.x == 0) ncand = k;
    __syncthreads();
  }

  // ---- rank and write
  const int n = ncand;
  for (int i = threadIdx.x; i < n; i += kTopThreads) {
    const uint64_t mine = cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += cand[j] > mine ? 1 : 0;
    if (rank < k) {
      const int col = (int)~(uint32_t)mine;
      ids[r * k + rank] = col;
      logp[r * k + rank] = ((float)row[col] - m) * inv_T - lnS;
    }
  }
}

}  // namespace octo

using namespace octo;

extern "C" {

int octo_topk(const void *logits, int64_t ld, int dtype, int64_t n, int V, float inv_T, int k, int64_t *ids,
              float *logp, void *stream) {
  OCTO_CHECK_ARG(n >= 0 && n <= 0x7fffffff && V > 0 && ld >= V, "topk: bad shape n=%lld V=%d ld=%lld", (long long)n, V,
                 (long long)ld);
  OCTO_CHECK_ARG(is_float(dtype), "topk: dtype %d", dtype);
  OCTO_CHECK_ARG(inv_T > 0.f, "topk: temperature must be positive");
  OCTO_CHECK_ARG(k >= 1 && k <= V && k <= OCTO_LIST_MAX, "topk: k=%d outside [1, min(V, %d)]", k, OCTO_LIST_MAX);
  if (n == 0) return OCTO_OK;
  OCTO_CHECK_ARG(logits && ids && logp, "topk: null pointer");
  OCTO_CHECK_ARG((uintptr_t)logits % float_bytes(dtype) == 0, "topk: misaligned logits");
  hipStream_t st = (hipStream_t)stream;
  const dim3 g((unsigned)n), b(kTopThreads);
  if (dtype == OCTO_BF16) hipLaunchKernelGGL(topk_kernel<OCTO_BF16>, g, b, 0, st, logits, ld, V, inv_T, k, ids, logp);
  else if (dtype == OCTO_F16) hipLaunchKernelGGL(topk_kernel<OCTO_F16>, g, b, 0, st, logits, ld, V, inv_T, k, ids, logp);
  else hipLaunchKernelGGL(topk_kernel<OCTO_F32>, g, b, 0, st, logits, ld, V, inv_T, k, ids, logp);
  OCTO_CHECK_LAUNCH("topk");
  return OCTO_OK;
}

}  // extern "C"
