// Embedding lookup with scaling, and its gradient by sorted tokens (octo_embed_fwd, octo_embed_bwd).
//
//   out[t] = scale W[ids[t]]              (zeros for an id outside [0, V))
//   grad_W[v] = scale sum of grad[t] over the tokens with ids[t] = v, t ascending; no token of padding_idx
//
// Both are bound by memory: the lookup reads and writes a row per token; the gradient reads a row per token and writes
// one per vocabulary entry (or adds to the entries that occur). A gradient row's sum is taken in fp32 in an order that
// the tokens alone decide, and rounded once, so equal inputs give equal bits.
//
// The gradient takes three launches:
//   sort   a workgroup per range of kBins vocabulary entries: it reads all ids, counts those below its range (the place
//          of its first token) and those of each entry by wave (a wave takes a contiguous part of the tokens), and
//          places its tokens, so that sorted tokens of one entry keep their order. No workgroup waits for another.
//          Behind them, in the same launch, workgroups that write the zeros of the whole gradient while the sort waits
//          for its loads: the rows that tokens name are written twice, 9,000 of 151,936 for 32,768 tokens of text.
//   sum    a wave per kRun sorted tokens x 512 columns: the sum of every entry whose tokens all lie in the piece goes
//          to grad_W, that of an entry that crosses a piece's border to the piece's two fp32 partial rows (its first
//          and its last entry). Frequent tokens are so shared out evenly.
//   join   a workgroup per piece in which a crossing entry starts: its partial rows summed in order.
// 32,768 tokens of text, d 2560, V 151,936, bf16: 207 us (0.95 GB at 4.6 TB/s: sort and zeros 115, sum 75, of which
// half is the zeros' way out of the caches, join 13); added in place 80 (sort 18, sum 27 to 50). One entry alone: 112
// in place.
#include "octo_common.h"
#include "row_values.h"

namespace octo {

constexpr int kBins = 512;    // vocabulary entries per sort workgroup
constexpr int kRun = 32;      // sorted tokens per piece
constexpr int kCols = 512;    // columns per wave of the sum
constexpr int kSumLoads = 8;  // rows in flight per wave

// ---- lookup ---------------------------------------------------------------------------------------------------------
// A wave per token and 4 KB of its row: 32,768 tokens of d 2560, V 151,936 in bf16 38 us (8,200 distinct rows).
constexpr int kRowLoadsF = 4;
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void *w, int64_t ldw, int64_t V, int d,
                                                        const int64_t *ids, int64_t n, float scale, void *out,
                                                        int64_t ldo) {
  constexpr int PER = 16 / Elem<DT>::bytes;
  typedef typename Elem<DT>::T T;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (t >= n) return;
  const int64_t id = ids[t];
  const bool ok = id >= 0 && id < V;
  const T *src = (const T *)w + (ok ? id : 0) * ldw;
  T *dst = (T *)out + t * ldo;
  if constexpr (VEC) {
    const int chunks = d / PER;
    const int c0 = blockIdx.y * (64 * kRowLoadsF) + lane;
    i32x4 v[kRowLoadsF];
#pragma unroll
    for (int u = 0; u < kRowLoadsF; ++u) {
      v[u] = i32x4{0, 0, 0, 0};
      if (ok && c0 + 64 * u < chunks) v[u] = ((const i32x4 *)src)[c0 + 64 * u];
    }
#pragma unroll
    for (int u = 0; u < kRowLoadsF; ++u) {
      if (c0 + 64 * u >= chunks) break;
      float x[PER];
      unpack_chunk<DT>(v[u], x);
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] = ok ? x[e] * scale : 0.f;
      ((i32x4 *)dst)[c0 + 64 * u] = pack_chunk<DT>(x);
    }
  } else {
    const int j0 = blockIdx.y * (64 * kRowLoadsF * PER), j1 = min(d, j0 + 64 * kRowLoadsF * PER);
    for (int j = j0 + lane; j < j1; j += 64) dst[j] = ok ? (T)((float)src[j] * scale) : (T)0.f;
  }
}

// ---- sort -----------------------------------------------------------------------------------------------------------
struct SortOut {
  int32_t *order;  // [n] token positions by (entry, position)
  int32_t *entry;  // [n] the entries of them
  int32_t *start;  // [V + 1] first place of each entry's tokens; start[V]: how many tokens there are
};

constexpr int kSortWaves = 16, kSortLoads = 8;
constexpr int kListed = 1024;  // tokens of its range that a wave notes on its first sweep
// The zeros: `rows` runs of `bytes` bytes, `stride` apart. A gradient without gaps is one run.
struct ZeroFill {
  char *at;
  int64_t stride, bytes, rows;
  int blocks;
};
// A workgroup's first kZeroThreads threads write one chunk each, or two of a gradient below kZeroTwo bytes: memory
// takes stores best from few waves at a time that move through it as one front, and a small gradient is bound by the
// launching of the workgroups. us of embed_bwd, one and two: fp32, 8 tokens, [151,936, 2560] (1.56 GB) 230 and 242,
// [64,000, 2304] (590 MB) 93 and 99; bf16, 8 tokens, [151,936, 2560] (778 MB) 121 and 126; 1,501 tokens, f16 [64,000,
// 2304] (295 MB) 63 and 60, bf16 [32,000, 1024] (66 MB) 28 and 26. All 1,024 threads, four each, a quarter of the
// gradient apart: 274, 111, 141, 61, 26; a fill and an index_add_ in fp32: 261, 119.
constexpr int kZeroThreads = 512;
constexpr int64_t kZeroTwo = 512 << 20;
// Thread t of T: the 16-byte chunks t, t + T, .. of the run at p, and the 2-byte values before the first and after the
// last.
__device__ __forceinline__ void zero_run(char *p, int64_t bytes, int64_t t, int64_t T) {
  const int64_t head = min(bytes, (int64_t)((16 - ((uintptr_t)p & 15)) & 15)), chunks = (bytes - head) / 16;
  for (int64_t k = t; k < chunks; k += T) ((i32x4 *)(p + head))[k] = i32x4{0, 0, 0, 0};
  const int64_t tail = head + 16 * chunks;
  if (t < head / 2) ((uint16_t *)p)[t] = 0;
  if (t < (bytes - tail) / 2) ((uint16_t *)(p + tail))[t] = 0;
}
__device__ __forceinline__ void zero_rows(const ZeroFill &z, int block) {
  if (z.rows == 1) {
    if ((int)threadIdx.x < kZeroThreads)
      zero_run(z.at, z.bytes, (int64_t)block * kZeroThreads + threadIdx.x, (int64_t)z.blocks * kZeroThreads);
    return;
  }
  for (int64_t r = (int64_t)block * kSortWaves + (threadIdx.x >> 6); r < z.rows; r += (int64_t)z.blocks * kSortWaves)
    zero_run(z.at + r * z.stride, z.bytes, threadIdx.x & 63, 64);
}

__global__ __launch_bounds__(1024) void embed_sort_kernel(const int64_t *ids, int n, int V, int64_t padding, SortOut o,
                                                          int ranges, ZeroFill z) {
  __shared__ int hist[kSortWaves][kBins];
  __shared__ uint16_t list[kSortWaves][kListed];
  __shared__ int part[2][kSortWaves];
  if ((int)blockIdx.x >= ranges) {
    zero_rows(z, (int)blockIdx.x - ranges);
    return;
  }
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int lo = blockIdx.x * kBins, hi = min(V, lo + kBins);
  for (int i = threadIdx.x; i < kSortWaves * kBins; i += 1024) ((int *)hist)[i] = 0;
  __syncthreads();
  const int seg = (int)round_up(cdiv(n, kSortWaves), 64);
  const int t0 = min(n, w * seg), t1 = min(n, t0 + seg);
  // an entry in [0, V), -1 for a token that has none
  auto entry = [&](int64_t v) { return v >= 0 && v < V && v != padding ? (int)v : -1; };
  int below = 0, noted = 0, resume = t1;  // the wave's tokens from `resume` on are not noted: too many, or too far
  for (int s = t0; s < t1; s += 64 * kSortLoads) {
    int64_t v[kSortLoads];
#pragma unroll
    for (int u = 0; u < kSortLoads; ++u) {
      const int t = s + 64 * u + lane;
      v[u] = t < t1 ? ids[t] : -1;
    }
#pragma unroll
    for (int u = 0; u < kSortLoads; ++u) {
      const int y = entry(v[u]), g = s + 64 * u;
      const bool in = y >= lo && y < hi;
      if (y >= 0 && y < lo) ++below;
      const uint64_t bal = __ballot(in);
      if (!bal) continue;
      if (in) atomicAdd(&hist[w][y - lo], 1);
      if (resume < t1) continue;
      if (noted + __popcll(bal) <= kListed && g - t0 < 65536 - 64) {
        if (in) list[w][noted + __popcll(bal & ((1ull << lane) - 1ull))] = (uint16_t)(g - t0 + lane);
        noted += __popcll(bal);
      } else {
        resume = g;
      }
    }
  }
  below = wave_sum(below);
  if (lane == 0) part[0][w] = below;
  __syncthreads();
  int first = 0;
#pragma unroll
  for (int k = 0; k < kSortWaves; ++k) first += part[0][k];
  // places by entry, then by wave
  int total = 0;
  if (threadIdx.x < kBins)
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) total += hist[k][threadIdx.x];
  int x = total;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int y = __shfl_up(x, s, 64);
    if (lane >= s) x += y;
  }
  if (lane == 63) part[1][w] = x;
  __syncthreads();
  for (int k = 0; k < w; ++k) x += part[1][k];
  if (threadIdx.x < kBins) {
    int at = first + x - total;
    if (lo + (int)threadIdx.x < hi) o.start[lo + threadIdx.x] = at;
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) {
      const int h = hist[k][threadIdx.x];
      hist[k][threadIdx.x] = at;
      at += h;
    }
    if (hi == V && threadIdx.x == kBins - 1) o.start[V] = at;
  }
  __syncthreads();
  // each wave places its tokens in their order: 64 at a time, those of one entry by lane
  auto place = [&](int t, int y) {
    const bool in = y >= lo && y < hi;
    uint64_t same = __ballot(in);
    if (!same) return;
    const int bin = in ? y - lo : 0;
#pragma unroll
    for (int b = 1; b < kBins; b <<= 1) {
      const uint64_t on = __ballot(bin & b);
      same &= bin & b ? on : ~on;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1ull));
    int base = 0;
    if (in) base = hist[w][bin];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) {
      o.order[base + rank] = t;
      o.entry[base + rank] = y;
      if (rank == 0) hist[w][bin] = base + __popcll(same);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  for (int q = 0; q < noted; q += 256) {
    int t[4], y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = q + 64 * u + lane;
      t[u] = k < noted ? t0 + list[w][k] : -1;
      y[u] = t[u] >= 0 ? entry(ids[t[u]]) : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) place(t[u], y[u]);
  }
  for (int s = resume; s < t1; s += 64 * 4) {
    int y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) y[u] = s + 64 * u + lane < t1 ? entry(ids[s + 64 * u + lane]) : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) place(s + 64 * u + lane, y[u]);
  }
}

// ---- sum ------------------------------------------------------------------------------------------------------------
struct SumArgs {
  const void *grad;
  int64_t ldg;
  int d, V;
  int n;  // tokens; as many of them as start[V] says are sorted
  SortOut s;
  float scale;
  void *gw;
  int64_t ldw;
  int accumulate;
  float *part;  // [pieces][2][d]
  int pieces, colblocks;
};

// 8 columns of a row per lane: c0 + 8 lane .. + 8 (VEC), or c0 + lane + 64 e. As loaded, so that a wave's loads are all
// under way before the first is used.
template <int DT, bool VEC> struct Cols {
  typedef typename Elem<DT>::T T;
  static constexpr int PER = 16 / Elem<DT>::bytes;
  i32x4 v[8 / PER];
  uint32_t s[8];  // bits, 16 of them by themselves: two loads into one register would wait for each other
  __device__ __forceinline__ void load(const void *base, int64_t off, int c0, int lane, int d) {
    const T *p = (const T *)base + off;
    if constexpr (VEC) {
      const int c = c0 + 8 * lane;
#pragma unroll
      for (int h = 0; h < 8 / PER; ++h) {
        v[h] = i32x4{0, 0, 0, 0};
        if (c < d) v[h] = *(const i32x4 *)(p + c + h * PER);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // past the end: the last column, not stored
        const int c = min(c0 + lane + 64 * e, d - 1);
        if constexpr (DT == OCTO_F32) s[e] = ((const uint32_t *)p)[c];
        else s[e] = ((const uint16_t *)p)[c];
      }
    }
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (VEC) {
#pragma unroll
      for (int h = 0; h < 8 / PER; ++h) {
        float y[PER];
        unpack_chunk<DT>(v[h], y);
#pragma unroll
        for (int e = 0; e < PER; ++e) x[h * PER + e] = y[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (DT == OCTO_F32) x[e] = __uint_as_float(s[e]);
        else if constexpr (DT == OCTO_F16) x[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)s[e]);
        else x[e] = __uint_as_float(s[e] << 16);
      }
    }
  }
  static __device__ __forceinline__ void store(const float (&x)[8], void *base, int64_t off, int c0, int lane, int d) {
    T *p = (T *)base + off;
    if constexpr (VEC) {
      const int c = c0 + 8 * lane;
      if (c < d)
#pragma unroll
        for (int h = 0; h < 8 / PER; ++h) {
          float y[PER];
#pragma unroll
          for (int e = 0; e < PER; ++e) y[e] = x[h * PER + e];
          *(i32x4 *)(p + c + h * PER) = pack_chunk<DT>(y);
        }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = c0 + lane + 64 * e;
        if (c < d) p[c] = (T)x[e];
      }
    }
  }
};

// grad_W's row v: scale x the sum, rounded once; added to what it holds where asked for.
template <int WT, bool VEC, bool ACC>
__device__ __forceinline__ void store_entry(const SumArgs &a, int v, const float (&sum)[8], int c0, int lane) {
  const int64_t off = (int64_t)v * a.ldw;
  float x[8];
  if constexpr (ACC) {
    Cols<WT, VEC> o;
    o.load(a.gw, off, c0, lane, a.d);
    o.get(x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(a.scale, sum[e], x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = a.scale * sum[e];
  }
  Cols<WT, VEC>::store(x, a.gw, off, c0, lane, a.d);
}

template <int GT, int WT, bool VEC, bool ACC>
__global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int items = a.pieces * a.colblocks;
  if (wave >= items) return;
  const int piece = wave / a.colblocks, c0 = (wave - piece * a.colblocks) * kCols;
  // this piece's tokens and entries, one per lane; lanes kRun and kRun + 1 hold the entries before and behind it. What
  // lies at or past start[V] is not there (and was not written).
  const int m = a.s.start[a.V], i0 = piece * kRun, i1 = min(m, i0 + kRun);
  const int at = lane < kRun ? i0 + lane : lane == kRun ? i0 - 1 : i0 + kRun;
  const bool there = at >= 0 && at < a.n;
  const int tok = there ? a.s.order[at] : 0, ent_ = there ? a.s.entry[at] : -1;
  if (i0 >= m) return;
  const int ent = at < m ? ent_ : -1;
  auto entry_of = [&](int k) { return __builtin_amdgcn_readlane(ent, k); };
  const int first = entry_of(0), last = entry_of(i1 - i0 - 1);
  const bool head = entry_of(kRun) == first;      // the first entry began before the piece
  const bool tail = entry_of(kRun + 1) == last;   // the last one goes on behind it
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int cur = first;
  auto flush = [&](int v) {
    if ((head && v == first) || (tail && v == last)) {
      // the piece's partial rows: 0 of its first entry where that began before it, else 1 of its last
      float *p = a.part + ((int64_t)piece * 2 + (head && v == first ? 0 : 1)) * a.d;
      Cols<OCTO_F32, VEC>::store(sum, p, 0, c0, lane, a.d);
    } else {
      store_entry<WT, VEC, ACC>(a, v, sum, c0, lane);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  };
  for (int i = 0; i < i1 - i0; i += kSumLoads) {
    Cols<GT, VEC> g[kSumLoads];
#pragma unroll
    for (int u = 0; u < kSumLoads; ++u) {
      const int k = min(i + u, i1 - i0 - 1);  // past the end: the last token again, left out below
      g[u].load(a.grad, (int64_t)__builtin_amdgcn_readlane(tok, k) * a.ldg, c0, lane, a.d);
    }
#pragma unroll
    for (int u = 0; u < kSumLoads; ++u) {
      if (i + u >= i1 - i0) break;
      const int v = entry_of(i + u);
      if (v != cur) {
        flush(cur);
        cur = v;
      }
      float x[8];
      g[u].get(x);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += x[e];
    }
  }
  flush(cur);
}

// ---- join -----------------------------------------------------------------------------------------------------------
// The entry that starts in piece p and goes on behind it: its partial rows are row 1 of p and row 0 of the pieces up to
// the one that holds its last token. The waves take them in turn, each in order, and are added in order.
constexpr int kJoinWaves = 8, kJoinLoads = 8;
template <int WT, bool VEC, bool ACC>
__global__ __launch_bounds__(64 * kJoinWaves) void embed_join_kernel(SumArgs a) {
  __shared__ float sums[kJoinWaves][64][8];
  const int p = blockIdx.x, c0 = blockIdx.y * kCols;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int m = a.s.start[a.V], i1 = (p + 1) * kRun;
  if (i1 >= m) return;
  const int v = a.s.entry[i1 - 1];
  if (a.s.entry[i1] != v) return;
  const int s0 = a.s.start[v], s1 = a.s.start[v + 1];
  if (s0 < p * kRun) return;  // it began before: another workgroup's
  const int parts = (s1 - 1) / kRun - p + 1;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int k = w; k < parts; k += kJoinWaves * kJoinLoads) {
    Cols<OCTO_F32, VEC> x[kJoinLoads];
#pragma unroll
    for (int u = 0; u < kJoinLoads; ++u) {
      const int q = min(k + kJoinWaves * u, parts - 1);
      x[u].load(a.part, ((int64_t)(p + q) * 2 + (q == 0 ? 1 : 0)) * a.d, c0, lane, a.d);
    }
#pragma unroll
    for (int u = 0; u < kJoinLoads; ++u)
      if (k + kJoinWaves * u < parts) {
        float y[8];
        x[u].get(y);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += y[e];
      }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[w][lane][e] = sum[e];
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int k = 1; k < kJoinWaves; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += sums[k][lane][e];
  store_entry<WT, VEC, ACC>(a, v, sum, c0, lane);
}

// ---- workspace ------------------------------------------------------------------------------------------------------
static size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
static size_t embed_ws(int64_t n, int64_t V, int64_t d, char *ws, SumArgs *a) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char *p = ws ? ws + off : nullptr;
    off += align256(bytes);
    return p;
  };
  char *order = take((size_t)n * 4), *entry = take((size_t)n * 4), *start = take((size_t)(V + 1) * 4);
  const int64_t pieces = cdiv(n, kRun);
  char *part = take((size_t)pieces * 2 * d * 4);
  if (a) {
    a->s.order = (int32_t *)order;
    a->s.entry = (int32_t *)entry;
    a->s.start = (int32_t *)start;
    a->part = (float *)part;
    a->pieces = (int)pieces;
  }
  return off;
}

template <int GT, int WT, bool VEC, bool ACC> static int go_bwd(const SumArgs &a, hipStream_t st) {
  if (a.pieces == 0) return OCTO_OK;
  const int64_t items = cdiv((int64_t)a.pieces * a.colblocks, 4);
  hipLaunchKernelGGL((embed_sum_kernel<GT, WT, VEC, ACC>), dim3((unsigned)items), dim3(256), 0, st, a);
  OCTO_CHECK_LAUNCH("embed_sum");
  if (a.pieces > 1) {
    hipLaunchKernelGGL((embed_join_kernel<WT, VEC, ACC>), dim3((unsigned)(a.pieces - 1), (unsigned)a.colblocks),
                       dim3(64 * kJoinWaves), 0, st, a);
    OCTO_CHECK_LAUNCH("embed_join");
  }
  return OCTO_OK;
}
template <int GT, int WT> static int pick_bwd(const SumArgs &a, bool vec, hipStream_t st) {
  if (a.accumulate) return vec ? go_bwd<GT, WT, true, true>(a, st) : go_bwd<GT, WT, false, true>(a, st);
  return vec ? go_bwd<GT, WT, true, false>(a, st) : go_bwd<GT, WT, false, false>(a, st);
}
template <int GT> static int pick_bwd(const SumArgs &a, int wt, bool vec, hipStream_t st) {
  if (wt == OCTO_BF16) return pick_bwd<GT, OCTO_BF16>(a, vec, st);
  if (wt == OCTO_F16) return pick_bwd<GT, OCTO_F16>(a, vec, st);
  return pick_bwd<GT, OCTO_F32>(a, vec, st);
}

template <int DT>
static void go_fwd(const void *w, int64_t ldw, int64_t V, int d, const int64_t *ids, int64_t n, float scale, void *out,
                   int64_t ldo, hipStream_t st) {
  constexpr int B = Elem<DT>::bytes, PER = 16 / B;
  const bool vec = d % PER == 0 && ldw % PER == 0 && ldo % PER == 0 && (uintptr_t)w % 16 == 0 &&
                   (uintptr_t)out % 16 == 0;
  constexpr int64_t kTokens = 4 * kLaunchRows;
  for (int64_t t0 = 0; t0 < n; t0 += kTokens) {
    const int64_t m = n - t0 < kTokens ? n - t0 : kTokens;
    const dim3 grid((unsigned)cdiv(m, 4), (unsigned)cdiv(d, 64 * kRowLoadsF * PER));
    char *o = (char *)out + t0 * ldo * B;
    if (vec)
      hipLaunchKernelGGL((embed_fwd_kernel<DT, true>), grid, dim3(256), 0, st, w, ldw, V, d, ids + t0, m, scale, o,
                         ldo);
    else
      hipLaunchKernelGGL((embed_fwd_kernel<DT, false>), grid, dim3(256), 0, st, w, ldw, V, d, ids + t0, m, scale, o,
                         ldo);
  }
}

}  // namespace octo

using namespace octo;

extern "C" {

int octo_embed_fwd(const void *w, int64_t ldw, int dtype, int64_t V, int d, const int64_t *ids, int64_t n, float scale,
                   void *out, int64_t ldo, void *stream) {
  OCTO_CHECK_ARG(V > 0 && V <= OCTO_ROW_MAX && d > 0 && ldw >= d && ldo >= d && n >= 0 && n < 0x7fffffff,
                 "embed_fwd: bad shape V=%lld d=%d n=%lld", (long long)V, d, (long long)n);
  if (!is_float(dtype)) return octo_fail(OCTO_EUNSUPPORTED, "embed_fwd: dtype %d", dtype);
  if (n == 0) return OCTO_OK;
  OCTO_CHECK_ARG(w && ids && out, "embed_fwd: null pointer");
  OCTO_CHECK_ARG((uintptr_t)w % float_bytes(dtype) == 0 && (uintptr_t)out % float_bytes(dtype) == 0,
                 "embed_fwd: misaligned rows");
  OCTO_CHECK_ARG(d <= 65535 * 1024, "embed_fwd: d=%d", d);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == OCTO_BF16) go_fwd<OCTO_BF16>(w, ldw, V, d, ids, n, scale, out, ldo, st);
  else if (dtype == OCTO_F16) go_fwd<OCTO_F16>(w, ldw, V, d, ids, n, scale, out, ldo, st);
  else go_fwd<OCTO_F32>(w, ldw, V, d, ids, n, scale, out, ldo, st);
  OCTO_CHECK_LAUNCH("embed_fwd");
  return OCTO_OK;
}

int octo_embed_bwd_workspace_bytes(int64_t n, int64_t V, int d, size_t *bytes) {
  OCTO_CHECK_ARG(bytes != nullptr, "embed_bwd_workspace_bytes: null pointer");
  OCTO_CHECK_ARG(V > 0 && V <= OCTO_ROW_MAX && d > 0 && d <= 65535 * kCols && n >= 0 && n <= (int64_t)1 << 27,
                 "embed_bwd: bad shape V=%lld d=%d n=%lld", (long long)V, d, (long long)n);
  *bytes = embed_ws(n, V, d, nullptr, nullptr);
  return OCTO_OK;
}

int octo_embed_bwd(const void *grad, int64_t ldg, int g_dtype, const int64_t *ids, int64_t n, int64_t V, int d,
                   int64_t padding_idx, float scale, void *grad_w, int64_t ldw, int w_dtype, int accumulate, void *ws,
                   size_t ws_bytes, void *stream) {
  size_t need = 0;
  const int rc = octo_embed_bwd_workspace_bytes(n, V, d, &need);
  if (rc) return rc;
  OCTO_CHECK_ARG(ldg >= d && ldw >= d, "embed_bwd: row strides below d");
  if (!is_float(g_dtype) || !is_float(w_dtype))
    return octo_fail(OCTO_EUNSUPPORTED, "embed_bwd: dtypes %d, %d", g_dtype, w_dtype);
  OCTO_CHECK_ARG(grad_w && (n == 0 || (grad && ids)), "embed_bwd: null pointer");
  OCTO_CHECK_ARG((uintptr_t)grad % float_bytes(g_dtype) == 0 && (uintptr_t)grad_w % float_bytes(w_dtype) == 0,
                 "embed_bwd: misaligned rows");
  SumArgs a{};
  if (!ws || ws_bytes < need)
    return octo_fail(OCTO_EWORKSPACE, "embed_bwd: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
  OCTO_CHECK_ARG((uintptr_t)ws % 16 == 0, "embed_bwd: misaligned workspace");
  if (n == 0 && accumulate) return OCTO_OK;
  embed_ws(n, V, d, (char *)ws, &a);
  a.grad = grad;
  a.ldg = ldg;
  a.d = d;
  a.V = (int)V;
  a.n = (int)n;
  a.scale = scale;
  a.gw = grad_w;
  a.ldw = ldw;
  a.accumulate = accumulate != 0;
  a.colblocks = (int)cdiv(d, kCols);
  OCTO_CHECK_ARG((int64_t)a.pieces * a.colblocks < (int64_t)1 << 26, "embed_bwd: %lld tokens of width %d", (long long)n,
                 d);
  ZeroFill z{};
  if (!accumulate) {
    const int64_t row = (int64_t)d * float_bytes(w_dtype);
    const bool one = ldw == d || V == 1;
    z.at = (char *)grad_w;
    z.stride = ldw * float_bytes(w_dtype);
    z.bytes = one ? V * row : row;
    z.rows = one ? 1 : V;
    // rows apart: 64 KB of them a workgroup
    const int64_t work = one ? cdiv(z.bytes, kZeroThreads * 16 * (z.bytes < kZeroTwo ? 2 : 1)) : cdiv(V * row, 65536);
    z.blocks = (int)(work < (1 << 20) ? work : 1 << 20);
  }
  const int ranges = (int)cdiv(V, kBins);
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(embed_sort_kernel, dim3((unsigned)(ranges + z.blocks)), dim3(1024), 0, st, ids, (int)n, (int)V,
                     padding_idx, a.s, ranges, z);
  OCTO_CHECK_LAUNCH("embed_sort");
  const auto whole = [&](const void *p, int64_t ld, int dt) {
    return (uintptr_t)p % 16 == 0 && ld * float_bytes(dt) % 16 == 0;
  };
  const bool vec = d % 8 == 0 && whole(grad, ldg, g_dtype) && whole(grad_w, ldw, w_dtype);
  if (g_dtype == OCTO_BF16) return pick_bwd<OCTO_BF16>(a, w_dtype, vec, st);
  if (g_dtype == OCTO_F16) return pick_bwd<OCTO_F16>(a, w_dtype, vec, st);
  return pick_bwd<OCTO_F32>(a, w_dtype, vec, st);
}

}  // extern "C"
