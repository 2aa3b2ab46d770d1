// The teacher's list of a row of logits: its k largest values, their columns and log-probabilities (octo_topk).
//
//   ids[r] = the columns of the k largest z_rv, by value descending, equal values by column ascending
//   logp[r][j] = z_r,ids[j] / T - logsumexp_v(z_rv / T)
//
// One workgroup per row, one sweep over it. Of the values a workgroup has seen, at least k are no smaller than the k-th
// largest of its threads' maxima, so that one is a lower bound of the list. It is taken after the first kTopLoads chunks
// of every thread (32,768 values of 16 bits); from there on the sweep collects what reaches it (300 of 151,936 values at k
// 64), and sums the row's exponentials as it goes. Every collected value is ranked against the others by (value, column),
// and the first k ranks are the list. Where more than kCand values reach the bound, a second sweep uses the bound of the
// whole row; a row with more than kCand even so (runs of equal values), or with a NaN or +inf, is done by a radix select
// over the values' 32-bit keys.
#include "octo_common.h"
#include "row_values.h"

namespace octo {

constexpr int kTopThreads = 512;
constexpr int kTopLoads = 8;   // 16-byte chunks in flight per thread
constexpr int kCand = 2048;    // values that may reach the bound
constexpr int kHits = 1536;    // chunks that may hold them
constexpr int kTighten = 256;  // chunks from which on the whole row's bound is taken before they are looked through

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

// The k-th largest of the threads' values to its upper 16 bits, rounded down, as a value: four bits a step, the threads
// that reach each of 15 tests counted in cnt (4 x 15, zero at the start).
__device__ __forceinline__ float kth_bound(float top, int k, int (*cnt)[15]) {
  const uint32_t key = order_key(top) >> 16;
  const int lane = threadIdx.x & 63;
  uint32_t bound = 0;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int sh = 12 - 4 * s;
    int n = 0;
#pragma unroll
    for (int q = 0; q < 15; ++q) {
      const int have = __popcll(__ballot(key >= (bound | ((uint32_t)(q + 1) << sh))));
      n = lane == q ? have : n;
    }
    if (n) atomicAdd(&cnt[s][lane], n);
    __syncthreads();
    // the largest test that k threads reach: the counts fall from test to test
    const uint32_t step = __popcll(__ballot(lane < 15 && cnt[s][min(lane, 14)] >= k));
    bound |= step << sh;
  }
  return bound <= 0x007fu ? -INFINITY : key_value(bound << 16);  // 0x007f: the key of -inf, and below
}

template <int DT>
__global__ __launch_bounds__(kTopThreads, 6) void topk_kernel(const void *logits, int64_t ld, int V, float inv_T, int k,
                                                           int64_t *ids, float *logp) {
  constexpr int PER = 16 / Elem<DT>::bytes, NW = kTopThreads / 64;
  typedef typename Elem<DT>::T T;
  __shared__ float red[2][NW];
  __shared__ int cnts[2][NW];
  __shared__ __attribute__((aligned(16))) uint64_t cand[kCand];
  __shared__ i32x4 hit[kHits];    // chunks with a value that reaches the bound, as they were loaded
  __shared__ int hit_at[kHits];   // and their place in the row
  __shared__ int bits[2][4][15];
  __shared__ int nhit, ncand, sel_bin, sel_above;
  static_assert(sizeof hit >= kCand * sizeof(int), "room for the ranks");
  int *ranks = (int *)hit, *hist = (int *)hit;  // where the chunks were, once they are looked through
  const int64_t r = blockIdx.x;
  const T *row = (const T *)logits + r * ld;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const float c = inv_T * OCTO_LOG2E;
  for (int i = threadIdx.x; i < 2 * 4 * 15; i += kTopThreads) (&bits[0][0][0])[i] = 0;
  if (threadIdx.x == 0) nhit = ncand = 0;

  // ---- the sweep
  RowSum st;
  float top = -INFINITY, least = INFINITY;
  const RowChunks rc = row_chunks<DT>(row, V);
  const i32x4 *vec = (const i32x4 *)(row + rc.head);
  const int tail = rc.head + rc.chunks * PER;
  const int je = (int)threadIdx.x < rc.head ? (int)threadIdx.x : (int)threadIdx.x - rc.head + tail;
  const bool edge = je < rc.head || (je >= tail && je < V);
  const float xe = edge ? (float)row[je] : -INFINITY;
  if (edge) {
    top = xe;
    st.raise(xe, c);
    st.add(xe, c);
  }
  for (int b = 0; b == 0 || b < rc.chunks; b += kTopLoads * kTopThreads) {  // the first step also without a chunk
    const int k0 = b + threadIdx.x;
    i32x4 v[kTopLoads];
#pragma unroll
    for (int u = 0; u < kTopLoads; ++u) {  // past the end: the last chunk again, left out below
      v[u] = i32x4{0, 0, 0, 0};
      if (rc.chunks) v[u] = vec[min(k0 + u * kTopThreads, rc.chunks - 1)];
    }
    float mxs[kTopLoads], mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kTopLoads; ++u) {
      float x[PER];
      unpack_chunk<DT>(v[u], x);
      mxs[u] = -INFINITY;
      if (k0 + u * kTopThreads < rc.chunks)
#pragma unroll
        for (int e = 0; e < PER; ++e) mxs[u] = fmaxf(mxs[u], x[e]);
      mx = fmaxf(mx, mxs[u]);
    }
    top = fmaxf(top, mx);
    st.raise(mx, c);
#pragma unroll
    for (int u = 0; u < kTopLoads; ++u)
      if (k0 + u * kTopThreads < rc.chunks) {
        float x[PER];
        asm("" : "+v"(v[u]));  // unpacked again: 32 values held from above would not fit the registers of two rows a CU
        unpack_chunk<DT>(v[u], x);
#pragma unroll
        for (int e = 0; e < PER; ++e) st.add(x[e], c);
      }
    if (b == 0) {
      __syncthreads();
      least = kth_bound(top, k, bits[0]);
    }
#pragma unroll
    for (int u = 0; u < kTopLoads; ++u)
      if (k0 + u * kTopThreads < rc.chunks && mxs[u] >= least) {
        const int at = atomicAdd(&nhit, 1);
        if (at < kHits) {
          hit[at] = v[u];
          hit_at[at] = k0 + u * kTopThreads;
        }
      }
  }
  float m, S;
  block_row_sum<NW>(st, c, red, m, S);
  const float lnS = flog2(S) * OCTO_LN2;
  bool listed = S == S;  // no NaN, no +inf
  // ---- the values that reach the bound
  auto take = [&](float x, int j) {
    if (x >= least) {
      const int at = atomicAdd(&ncand, 1);
      if (at < kCand) cand[at] = list_entry(x, j);
    }
  };
  int n = nhit;
  if (listed && n > kTighten) least = kth_bound(top, k, bits[1]);  // of the whole row
  if (listed && n <= kHits) {
    if (edge) take(xe, je);
    for (int i = threadIdx.x; i < n; i += kTopThreads) {
      float x[PER];
      unpack_chunk<DT>(hit[i], x);
#pragma unroll
      for (int e = 0; e < PER; ++e) take(x[e], rc.head + hit_at[i] * PER + e);
    }
  } else if (listed) {
    sweep_row<DT>(row, V, [&](float mx) { return mx >= least; }, take);
  }
  __syncthreads();
  n = ncand;
  listed = listed && n <= kCand;
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
    n = k;
  }

  // ---- ranks: each value against a share of the others, four at a time; the list behind them filled up with 0, which is
  // behind every value
  const int span = (n + 63) & ~63, groups = max(1, min(16, kTopThreads / span)), full = (n + 3) & ~3;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kTopThreads) ranks[i] = 0;
  if (threadIdx.x < full - n) cand[n + threadIdx.x] = 0;
  __syncthreads();
  const int g = groups > 1 ? (int)threadIdx.x / span : 0;
  for (int i = (int)threadIdx.x - g * span; i < n && g < groups; i += kTopThreads) {
    const uint64_t mine = cand[i];
    int before = 0;
#pragma unroll 2
    for (int j = 4 * g; j < full; j += 4 * groups) {
      uint64_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = cand[j + e];
#pragma unroll
      for (int e = 0; e < 4; ++e) before += o[e] > mine ? 1 : 0;
    }
    if (groups > 1) atomicAdd(&ranks[i], before);
    else ranks[i] = before;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kTopThreads) {
    const int at = ranks[i];
    if (at < k) {
      const uint64_t e = cand[i];
      ids[r * k + at] = (int)~(uint32_t)e;
      logp[r * k + at] = (key_value((uint32_t)(e >> 32)) - m) * inv_T - lnS;
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
