// The teacher's list of a row of logits: its k largest values, their columns and log-probabilities (octo_topk).
//
//   ids[r] = the columns of the k largest z_rv, by value descending, equal values by column ascending
//   logp[r][j] = z_r,ids[j] / T - logsumexp_v(z_rv / T)
//
// One workgroup per row, one sweep over it. Of the values a workgroup has seen, at least k are no smaller than the k-th
// largest of its threads' maxima, so that one is a lower bound of the list. It is taken after the first kTopLoads
// chunks of every thread (32,768 values of 16 bits); from there on the sweep collects what reaches it (300 of 151,936
// values at k 64), and sums the row's exponentials as it goes. Every collected value is ranked against the others by
// (value, column), and the first k ranks are the list. Where more than kCand values reach the bound (runs of equal
// values: rows with fewer than k unmasked logits), a second sweep takes those above the bound of the whole row, and the
// rest of the list are the first columns that equal it. A row with more than kCand even so, or with a NaN or +inf, is
// done by a radix select over the values' 32-bit keys.
//
// Few rows: a row is cut into slices of a workgroup each (topk_slices), whose lists and sums a second launch joins the
// same way.
//
// Bound by memory, 2 bytes a value at 16 bits: [2048, 151,936] bf16 at k 64 118 to 131 us (4.8 to 5.3 TB/s; a 4 GiB
// copy moves 5.0), fp32 214 (5.8). Rows with 10 unmasked values 189 and 395 (by the radix select, whose counts of one
// value wait for each other, 4,560 and 4,640).
#include "octo_common.h"
#include "row_values.h"

namespace octo {

constexpr int kTopThreads = 512;
constexpr int kTopLoads = 8;   // 16-byte chunks in flight per thread
constexpr int kCand = 2048;    // values that may reach the bound
constexpr int kHits = 1536;    // chunks that may hold them
constexpr int kJoin = 2048;    // entries a row's join takes from its slices
constexpr int kTighten = 254;  // chunks from which on the whole row's bound is taken before they are looked through
static_assert(kTighten * 8 + 2 * 7 <= kCand, "room for so many chunks' values, and those before and behind the chunks");

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

// put(u, place) for the lanes whose wanted[u] is set, places counted on in *count: one atomic a wave for all of them,
// where one per value waited for each in turn.
template <int N, class F> __device__ __forceinline__ void append(const bool (&wanted)[N], int *count, F put) {
  uint64_t bal[N];
  int all = 0;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    bal[u] = __ballot(wanted[u]);
    all += __popcll(bal[u]);
  }
  if (all == 0) return;
  const int lane = threadIdx.x & 63;
  int base = 0;
  if (lane == 0) base = atomicAdd(count, all);
  base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
  for (int u = 0; u < N; ++u) {
    if (wanted[u]) put(u, base + __popcll(bal[u] & ((1ull << lane) - 1ull)));
    base += __popcll(bal[u]);
  }
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

// The k-th largest of the threads' keys, its upper 16 bits: four bits a step, the threads that reach each of 15 tests
// counted in cnt (4 x 15, zero at the start). With N keys a thread, the k-th largest of all of them.
template <int N> __device__ __forceinline__ uint32_t kth_key(const uint32_t (&top)[N], int k, int (*cnt)[15]) {
  const int lane = threadIdx.x & 63;
  uint32_t bound = 0;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int sh = 12 - 4 * s;
    int n = 0;
#pragma unroll
    for (int q = 0; q < 15; ++q) {
      int have = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) have += __popcll(__ballot(top[i] >> 16 >= (bound | ((uint32_t)(q + 1) << sh))));
      n = lane == q ? have : n;
    }
    if (n) atomicAdd(&cnt[s][lane], n);
    __syncthreads();
    // the largest test that k threads reach: the counts fall from test to test
    const uint32_t step = __popcll(__ballot(lane < 15 && cnt[s][min(lane, 14)] >= k));
    bound |= step << sh;
  }
  return bound;
}
// As a value. Up to kOneTop entries a thread's one maximum will do; for longer lists the maxima of its even and odd
// chunks count each by itself, or k would be half the threads and the bound far below the k-th value (k 256 of 512
// maxima: 1,640 chunks of a row of 151,936 collected, of 1,024 maxima 1,370).
constexpr int kOneTop = 64;
__device__ __forceinline__ uint32_t kth_bound(const float (&top)[2], int k, int (*cnt)[15]) {
  if (k <= kOneTop) {
    const uint32_t one[1] = {order_key(fmaxf(top[0], top[1]))};
    return kth_key(one, k, cnt);
  }
  const uint32_t two[2] = {order_key(top[0]), order_key(top[1])};
  return kth_key(two, k, cnt);
}
__device__ __forceinline__ float bound_value(uint32_t bound) {
  return bound <= 0x007fu ? -INFINITY : key_value(bound << 16);  // 0x007f: the key of -inf, and below
}
// The lower 16 bits too: the k-th largest itself.
__device__ __forceinline__ float kth_value(const float (&top)[2], int k, uint32_t bound, int (*cnt)[15]) {
  const uint32_t keys[2] = {order_key(k <= kOneTop ? fmaxf(top[0], top[1]) : top[0]),
                            k <= kOneTop ? 0u : order_key(top[1])};
  uint32_t rest[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    rest[i] = keys[i] >> 16 == bound ? keys[i] << 16 : keys[i] >> 16 > bound ? 0xffffffffu : 0u;
  return key_value(bound << 16 | kth_key(rest, k, cnt));
}

// A ranked value's place in the row's list, if it has one.
__device__ __forceinline__ void write_value(uint64_t e, int rank, int64_t r, int k, float m, float lnS, float inv_T,
                                            int64_t *ids, float *logp) {
  if (rank >= k) return;
  ids[r * k + rank] = (int)~(uint32_t)e;
  logp[r * k + rank] = (key_value((uint32_t)(e >> 32)) - m) * inv_T - lnS;
}

// Ranks of the n collected values in cand (n <= kCand, room up to a multiple of 4): each against a share of the others,
// four at a time, the list behind them filled up with 0, which is behind every value.
__device__ __forceinline__ void rank_values(uint64_t *cand, int n, int *ranks) {
  const int span = (n + 63) & ~63, groups = max(1, min(16, kTopThreads / max(span, 64))), full = (n + 3) & ~3;
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
}

// SLICED: workgroup (r, s) takes the values s per .. s per + per of row r, and leaves its list as entries [r][s][k] (0
// where the slice has fewer values) and its (maximum, sum) as sums [r][s].
template <int DT, bool SLICED>
__global__ __launch_bounds__(kTopThreads, 6) void topk_kernel(const void *logits, int64_t ld, int V_, float inv_T,
                                                              int k_, int64_t *ids, float *logp, int per,
                                                              uint64_t *entries, float *sums) {
  constexpr int PER = 16 / Elem<DT>::bytes, NW = kTopThreads / 64;
  typedef typename Elem<DT>::T T;
  __shared__ float red[2][NW];
  __shared__ int cnts[2][NW];
  __shared__ __attribute__((aligned(16))) uint64_t cand[kCand];
  __shared__ i32x4 hit[kHits];    // chunks with a value that reaches the bound, as they were loaded
  __shared__ int hit_at[kHits];   // and their place in the row
  __shared__ int bits[3][4][15];
  __shared__ int nhit, ncand, sel_bin, sel_above;
  static_assert(sizeof hit >= kCand * sizeof(int), "room for the ranks");
  int *ranks = (int *)hit, *hist = (int *)hit;  // where the chunks were, once they are looked through
  const int64_t r = blockIdx.x;
  const int first = SLICED ? (int)blockIdx.y * per : 0, V = SLICED ? min(per, V_ - first) : V_, k = min(k_, V);
  const T *row = (const T *)logits + r * ld + first;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const float c = inv_T * OCTO_LOG2E;
  for (int i = threadIdx.x; i < 3 * 4 * 15; i += kTopThreads) (&bits[0][0][0])[i] = 0;
  if (threadIdx.x == 0) nhit = ncand = 0;

  // ---- the sweep
  RowSum st;
  float top[2] = {-INFINITY, -INFINITY}, least = INFINITY;
  const RowChunks rc = row_chunks<DT>(row, V);
  const i32x4 *vec = (const i32x4 *)(row + rc.head);
  const int tail = rc.head + rc.chunks * PER;
  const int je = (int)threadIdx.x < rc.head ? (int)threadIdx.x : (int)threadIdx.x - rc.head + tail;
  const bool edge = je < rc.head || (je >= tail && je < V);
  const float xe = edge ? (float)row[je] : -INFINITY;
  if (edge) {
    top[0] = xe;
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
#pragma unroll
    for (int u = 0; u < kTopLoads; ++u) top[u & 1] = fmaxf(top[u & 1], mxs[u]);
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
      least = bound_value(kth_bound(top, k, bits[0]));
    }
    bool wanted[kTopLoads];
#pragma unroll
    for (int u = 0; u < kTopLoads; ++u) wanted[u] = k0 + u * kTopThreads < rc.chunks && mxs[u] >= least;
    append(wanted, &nhit, [&](int u, int at) {
      if (at < kHits) {
        hit[at] = v[u];
        hit_at[at] = k0 + u * kTopThreads;
      }
    });
  }
  float m, S;
  block_row_sum<NW>(st, c, red, m, S);
  const float lnS = flog2(S) * OCTO_LN2;
  bool listed = S == S;  // no NaN, no +inf
  // ---- the values that reach the bound
  int n = nhit;
  bool more = n > kHits;
  uint32_t bound = 0;
  if (listed && n > kTighten) {  // of the whole row
    bound = kth_bound(top, k, bits[1]);
    least = bound_value(bound);
  }
  if (listed && !more) {
    if (edge && xe >= least) {
      const int at = atomicAdd(&ncand, 1);
      if (at < kCand) cand[at] = list_entry(xe, je);
    }
    for (int i0 = 0; i0 < n; i0 += kTopThreads) {  // whole waves: append counts over them
      const int i = i0 + threadIdx.x, at0 = i < n ? hit_at[i] : 0;
      float x[PER];
      bool wanted[PER];
      unpack_chunk<DT>(i < n ? hit[i] : i32x4{0, 0, 0, 0}, x);
#pragma unroll
      for (int e = 0; e < PER; ++e) wanted[e] = i < n && x[e] >= least;
      append(wanted, &ncand, [&](int e, int at) {
        if (at < kCand) cand[at] = list_entry(x[e], rc.head + at0 * PER + e);
      });
    }
    __syncthreads();
    n = ncand;
    more = n > kCand;
  }
  // put(place, x, column) for the first `need` columns whose value is wanted
  auto first_of = [&](int need, auto wanted, auto put) {
    int seen = 0;
    for (int s0 = 0, it = 0; s0 < V && seen < need; s0 += kTopThreads, ++it) {
      const int j = s0 + (int)threadIdx.x;
      const float x = j < V ? (float)row[j] : 0.f;
      const bool mine = j < V && wanted(x);
      const uint64_t bal = __ballot(mine);
      if (lane == 0) cnts[it & 1][w] = __popcll(bal);
      __syncthreads();
      int off = seen;
#pragma unroll
      for (int u = 0; u < NW; ++u) {
        off += u < w ? cnts[it & 1][u] : 0;
        seen += cnts[it & 1][u];
      }
      off += __popcll(bal & ((1ull << lane) - 1ull));
      if (mine && off < need) put(off, x, j);
    }
  };
  if (__builtin_expect(listed && more, 0)) {
    // ---- runs of equal values at the bound (fewer than k unmasked logits, say): those above it, then its first
    // columns
    least = kth_value(top, k, bound, bits[2]);
    if (threadIdx.x == 0) ncand = 0;  // read by all before the barriers of kth_value
    __syncthreads();
    sweep_row<DT>(row, V, [&](float mx) { return mx > least; }, [&](float x, int j) {
      if (x > least) {
        const int at = atomicAdd(&ncand, 1);
        if (at < kCand) cand[at] = list_entry(x, j);
      }
    });
    __syncthreads();
    n = ncand;
    if (n < k) {  // k values at least are no smaller than `least`
      first_of(k - n, [&](float x) { return x == least; },
               [&](int at, float x, int j) { cand[n + at] = list_entry(x, j); });
      n = k;
    }
  }
  listed = listed && n <= kCand;
  if (__builtin_expect(!listed, 0)) {
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
    sweep_row<DT>(row, V, [](float) { return true; }, [&](float x, int j) {
      if (order_key(x) > prefix) cand[atomicAdd(&ncand, 1)] = list_entry(x, j);  // `above` of them, fewer than k
    });
    first_of(k - above, [&](float x) { return order_key(x) == prefix; },
             [&](int at, float x, int j) { cand[above + at] = list_entry(x, j); });
    n = k;
  }

  rank_values(cand, n, ranks);
  if constexpr (SLICED) {
    const int64_t slice = r * gridDim.y + blockIdx.y;
    for (int i = threadIdx.x; i < n; i += kTopThreads)
      if (ranks[i] < k) entries[slice * k_ + ranks[i]] = cand[i] - (uint32_t)first;  // ~(column + first)
    for (int i = k + threadIdx.x; i < k_; i += kTopThreads) entries[slice * k_ + i] = 0;
    if (threadIdx.x == 0) {
      sums[2 * slice] = m;
      sums[2 * slice + 1] = S;
    }
  } else {
    for (int i = threadIdx.x; i < n; i += kTopThreads) write_value(cand[i], ranks[i], r, k, m, lnS, inv_T, ids, logp);
  }
}

// A row's list from its slices': n = slices x k entries, at least k of them values.
__global__ __launch_bounds__(kTopThreads) void topk_join_kernel(const uint64_t *entries, const float *sums, int slices,
                                                                int k, float inv_T, int64_t *ids, float *logp) {
  __shared__ __attribute__((aligned(16))) uint64_t cand[kCand];
  __shared__ int ranks[kCand];
  __shared__ int bits[4][15];
  __shared__ int ncand;
  const int64_t r = blockIdx.x;
  const int n = slices * k;  // at most kJoin
  const uint64_t *e = entries + r * n;
  for (int i = threadIdx.x; i < 4 * 15; i += kTopThreads) (&bits[0][0])[i] = 0;
  if (threadIdx.x == 0) ncand = 0;
  constexpr int PER = kJoin / kTopThreads;
  uint64_t mine[PER], top = 0;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = u * kTopThreads + threadIdx.x;
    mine[u] = i < n ? e[i] : 0;
    top = max(top, mine[u]);
  }
  RowSum st;
  const float c = inv_T * OCTO_LOG2E;
  for (int s = 0; s < slices; ++s) st.raise(sums[(r * slices + s) * 2], c);
  for (int s = 0; s < slices; ++s) {  // a slice of -inf alone adds its sum, 0 or NaN
    const float m = sums[(r * slices + s) * 2], S = sums[(r * slices + s) * 2 + 1];
    st.S += m == -INFINITY ? S : S * fexp2((m - st.m) * c);
  }
  const float lnS = flog2(st.S) * OCTO_LN2;
  __syncthreads();
  // two of a slice's entries may lie with one thread: the bound is that of the threads' largest, as the sweep's
  const uint32_t largest[1] = {(uint32_t)(top >> 32)}, bound = kth_key(largest, k, bits);
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (mine[u] && (uint32_t)(mine[u] >> 48) >= bound) cand[atomicAdd(&ncand, 1)] = mine[u];
  __syncthreads();
  const int got = ncand;
  rank_values(cand, got, ranks);
  for (int i = threadIdx.x; i < got; i += kTopThreads)
    write_value(cand[i], ranks[i], r, k, st.m, lnS, inv_T, ids, logp);
}

// Slices a row of V values is cut into for n rows: rows of 192 KB and of 60,000 values and more, up to 128 of them,
// four slices at least. us a call in a captured graph at k 64, whole and sliced, for 1, 16 and 128 rows. bf16, V
// 151,936: 21.0 and 15.5, 21.7 and 15.5, 23.0 and 21.8; 100,000 (195 KB): 17.0 and 15.3, 17.6 and 15.4, 19.1 and 17.8;
// 64,000 (125 KB): 12.9 and 15.2, 13.7 and 15.2, 13.6 and 16.3. fp32, V 64,000 (250 KB): 15.0 and 14.7, 15.8 and 14.9,
// 17.0 and 16.5; 49,152 (192 KB): 13.5 and 14.8, 13.6 and 14.8, 14.2 and 15.8. More rows or longer lists lose by it:
// 256 rows 25.2 and 28.2, k 256 28 and 50.
constexpr int kMaxSlices = 16, kSliceK = 128;
static int topk_slices(int64_t n, int V, int k, int dtype) {
  if (n < 1 || n > 128 || k > kSliceK || V < 60000 || (int64_t)V * float_bytes(dtype) < 192 * 1024) return 1;
  const int s = (int)(512 / n);
  return s < kMaxSlices ? s : kMaxSlices;
}
static_assert(kMaxSlices * kSliceK <= kJoin, "the join's entries");

template <bool SLICED>
static void go_topk(const void *logits, int64_t ld, int dtype, int64_t n, int V, float inv_T, int k, int64_t *ids,
                    float *logp, int slices, int per, uint64_t *entries, float *sums, hipStream_t st) {
  const dim3 g((unsigned)n, (unsigned)slices), b(kTopThreads);
  if (dtype == OCTO_BF16)
    hipLaunchKernelGGL((topk_kernel<OCTO_BF16, SLICED>), g, b, 0, st, logits, ld, V, inv_T, k, ids, logp, per, entries,
                       sums);
  else if (dtype == OCTO_F16)
    hipLaunchKernelGGL((topk_kernel<OCTO_F16, SLICED>), g, b, 0, st, logits, ld, V, inv_T, k, ids, logp, per, entries,
                       sums);
  else
    hipLaunchKernelGGL((topk_kernel<OCTO_F32, SLICED>), g, b, 0, st, logits, ld, V, inv_T, k, ids, logp, per, entries,
                       sums);
}

}  // namespace octo

using namespace octo;

extern "C" {

int octo_topk_workspace_bytes(int64_t n, int V, int dtype, int k, size_t *bytes) {
  OCTO_CHECK_ARG(bytes != nullptr, "topk_workspace_bytes: null pointer");
  OCTO_CHECK_ARG(n >= 0 && n <= 0x7fffffff && V > 0 && V <= OCTO_ROW_MAX, "topk: bad shape n=%lld V=%d", (long long)n,
                 V);
  OCTO_CHECK_ARG(k >= 1 && k <= V && k <= OCTO_LIST_MAX, "topk: k=%d outside [1, min(V, %d)]", k, OCTO_LIST_MAX);
  OCTO_CHECK_ARG(is_float(dtype), "topk: dtype %d", dtype);
  const int slices = topk_slices(n, V, k, dtype);
  *bytes = slices > 1 ? (size_t)n * slices * (k * 8 + 8) : 0;
  return OCTO_OK;
}

int octo_topk(const void *logits, int64_t ld, int dtype, int64_t n, int V, float inv_T, int k, int64_t *ids,
              float *logp, void *ws, size_t ws_bytes, void *stream) {
  size_t need = 0;
  const int rc = octo_topk_workspace_bytes(n, V, dtype, k, &need);
  if (rc) return rc;
  OCTO_CHECK_ARG(ld >= V, "topk: row stride %lld below V=%d", (long long)ld, V);
  OCTO_CHECK_ARG(inv_T > 0.f, "topk: temperature must be positive");
  if (n == 0) return OCTO_OK;
  OCTO_CHECK_ARG(logits && ids && logp, "topk: null pointer");
  OCTO_CHECK_ARG((uintptr_t)logits % float_bytes(dtype) == 0, "topk: misaligned logits");
  if (need && (!ws || ws_bytes < need))
    return octo_fail(OCTO_EWORKSPACE, "topk: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
  OCTO_CHECK_ARG((uintptr_t)ws % 8 == 0, "topk: misaligned workspace");
  hipStream_t st = (hipStream_t)stream;
  const int slices = topk_slices(n, V, k, dtype);
  if (slices == 1) {
    for (int64_t r0 = 0; r0 < n; r0 += kLaunchRows)
      go_topk<false>((const char *)logits + r0 * ld * float_bytes(dtype), ld, dtype,
                     n - r0 < kLaunchRows ? n - r0 : kLaunchRows, V, inv_T, k, ids + r0 * k, logp + r0 * k, 1, 0,
                     nullptr, nullptr, st);
  } else {
    const int per = (int)round_up(cdiv(V, slices), 64);  // the last slice has the rest, at least one value
    uint64_t *entries = (uint64_t *)ws;
    float *sums = (float *)(entries + n * slices * k);
    go_topk<true>(logits, ld, dtype, n, V, inv_T, k, ids, logp, slices, per, entries, sums, st);
    OCTO_CHECK_LAUNCH("topk");
    hipLaunchKernelGGL(topk_join_kernel, dim3((unsigned)n), dim3(kTopThreads), 0, st, entries, sums, slices, k, inv_T,
                       ids, logp);
  }
  OCTO_CHECK_LAUNCH("topk");
  return OCTO_OK;
}

}  // extern "C"
