// Drafted tokens checked against the target's probabilities (octo_verify_drafts).
//
//   p_i = softmax(z_i / T), q_i = softmax(z'_i / T), or all of it at the draft where the drafts come without logits.
//   Draft i is accepted when u_i q_i(x_i) < p_i(x_i); the first that is not ends the sequence at a. The next token is
//   the lowest v whose running sum of r_w = max(p_a(w) - q_a(w), 0) exceeds u_K sum r, and r = p_a after the last draft.
//
// Which token that is has to be the definition's, not one beside it: of 150,000 running sums some lie within fp32's
// rounding of any number, and then another token is answered. So the exponentials and sums are taken in 64 bits (exp64
// below, 6e-15 relative), and a draw differs from the exact one with a probability of about V times that.
//
// Three launches. stats: a workgroup per slice of a row, the slice's maximum and its sum of exponentials against it.
// residual: a workgroup per slice of a sequence's row a; each joins the rows' slices and finds a by itself, and sums
// its slice's r. pick: a workgroup per sequence finds the slice in which the running sum passes u_K sum r, and in it the
// token. All sums are in an order that the sizes alone decide.
#include "octo_common.h"
#include "row_values.h"

namespace octo {

constexpr int kVThreads = 256, kVWaves = kVThreads / 64;
constexpr int kVDrafts = OCTO_DRAFTS_MAX;
constexpr int kVSlices = 1024;  // slices of a row, at most

// 2^(y) for y = x log2(e): the nearest integer's power by the exponent, the rest, within 1/2, by exp's series in
// f ln 2: the first term left out is (ln 2 / 2)^12 / 12! = 6e-15.
__device__ __forceinline__ double exp64(double x) {  // x <= 0 or -inf; below -760 it gives 0
  const double y = fmax(x, -800.0) * 1.4426950408889634074;
  const double n = __builtin_rint(y);
  const double f = __builtin_fma(n, -0.69314718055994530942, fmax(x, -800.0));
  const double g = __builtin_fma(n, -2.3190468138462996e-17, f);  // ln 2's rest below its 53 bits
  double e = 1.0 / 39916800.0;
  e = __builtin_fma(e, g, 1.0 / 3628800.0);
  e = __builtin_fma(e, g, 1.0 / 362880.0);
  e = __builtin_fma(e, g, 1.0 / 40320.0);
  e = __builtin_fma(e, g, 1.0 / 5040.0);
  e = __builtin_fma(e, g, 1.0 / 720.0);
  e = __builtin_fma(e, g, 1.0 / 120.0);
  e = __builtin_fma(e, g, 1.0 / 24.0);
  e = __builtin_fma(e, g, 1.0 / 6.0);
  e = __builtin_fma(e, g, 0.5);
  e = __builtin_fma(e, g, 1.0);
  e = __builtin_fma(e, g, 1.0);
  return ldexp(e, (int)n);
}

struct SliceStat {
  double S;   // sum of exp((z - m) / T); NaN where the slice has a NaN or +inf
  float m;    // maximum
  int first;  // its first column
};
struct RowStat {
  double inv;  // 1 / sum over the row; 0 where the row has no distribution
  float m;
  int first;
};

struct VerifyArgs {
  const void *z, *zd;  // target and draft logits; row i of sequence s at s ls + i lr elements
  int64_t ls, lr, ls_d, lr_d;
  const int64_t *drafts;   // [S, K]
  const int64_t *lengths;  // [S] or NULL
  const float *u;          // [S, K + 1] (NULL: greedy)
  int64_t S;
  int K, V;
  double inv_T;
  int greedy;
  int slices, per;   // per: values of a slice, a multiple of 64
  SliceStat *stats;  // [S, 2 K + 1, slices]: target rows, then draft rows
  double *sums;      // [S, slices]: r's
  struct Decision {
    RowStat p, q;
    int a, residual, x, pad;  // residual: 0 r = p, 1 r = p - q, 2 r = p without x
  } *dec;  // [S]
  int64_t *tokens, *accepted;  // [S, K + 1], [S]
  float *logp;                 // [S, K + 1]
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

__device__ __forceinline__ int drafts_of(const VerifyArgs &a, int64_t s) {
  if (!a.lengths) return a.K;
  const int64_t n = a.lengths[s];
  return (int)(n < 0 ? 0 : (n > a.K ? a.K : n));
}

template <int DT>
__device__ __forceinline__ const typename Elem<DT>::T *row_of(const void *z, int64_t ls, int64_t lr, int64_t s, int i) {
  return (const typename Elem<DT>::T *)z + s * ls + i * lr;
}

// f(value, column) for the columns [c0, c1) that this thread takes, 16-byte loads where the row's alignment allows.
template <int DT, class F>
__device__ __forceinline__ void sweep_slice(const typename Elem<DT>::T *row, int c0, int c1, F f) {
  constexpr int PER = 16 / Elem<DT>::bytes;
  const int head = min(c1 - c0, (int)((16 - ((uintptr_t)(row + c0) & 15)) & 15) / Elem<DT>::bytes);
  const int chunks = (c1 - c0 - head) / PER;
  const i32x4 *vec = (const i32x4 *)(row + c0 + head);
  for (int k0 = threadIdx.x; k0 < chunks; k0 += 4 * kVThreads) {
    i32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = vec[min(k0 + u * kVThreads, chunks - 1)];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + u * kVThreads;
      if (k >= chunks) break;
      float x[PER];
      unpack_chunk<DT>(v[u], x);
#pragma unroll
      for (int e = 0; e < PER; ++e) f(x[e], c0 + head + k * PER + e);
    }
  }
  const int tail = c0 + head + chunks * PER, t = threadIdx.x;
  const int j = t < head ? c0 + t : tail + t - head;
  if (j < c1) f((float)row[j], j);
}

template <int DT>
__global__ __launch_bounds__(kVThreads) void verify_stats_kernel(VerifyArgs a) {
  const int64_t s = blockIdx.y / (2 * a.K + 1);
  const int i = (int)(blockIdx.y - s * (2 * a.K + 1)), len = drafts_of(a, s);
  const bool draft = i > a.K;
  if (draft ? (!a.zd || i - a.K - 1 >= len) : i > len) return;  // nobody asks for the row
  const typename Elem<DT>::T *row = draft ? row_of<DT>(a.zd, a.ls_d, a.lr_d, s, i - a.K - 1)
                                          : row_of<DT>(a.z, a.ls, a.lr, s, i);
  const int c0 = blockIdx.x * a.per, c1 = min(a.V, c0 + a.per);
  __shared__ float sm[kVWaves];
  __shared__ int si[kVWaves];
  __shared__ double ss[kVWaves];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float m = -INFINITY;
  bool bad = false;
  sweep_slice<DT>(row, c0, c1, [&](float x, int) {
    m = fmaxf(m, x);
    bad |= !(x < INFINITY);
  });
  m = wave_max(m);
  if (lane == 0) sm[w] = m;
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int k = 0; k < kVWaves; ++k) m = fmaxf(m, sm[k]);
  double S = 0.0;
  int first = 0x7fffffff;
  const double md = m == -INFINITY ? 0.0 : (double)m;
  sweep_slice<DT>(row, c0, c1, [&](float x, int c) {
    S += exp64(((double)x - md) * a.inv_T);
    if (x == m) first = min(first, c);
  });
  S = wave_sum64(S);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
  if (lane == 0) {
    ss[w] = S;
    si[w] = first;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    SliceStat out;
    out.S = 0.0;
    out.first = 0x7fffffff;
    for (int k = 0; k < kVWaves; ++k) {
      out.S += ss[k];
      out.first = min(out.first, si[k]);
    }
    out.m = m;
    if (bad) out.S = __builtin_nan("");
    a.stats[(s * (2 * a.K + 1) + i) * a.slices + blockIdx.x] = out;
  }
}

// Row i's statistics from its slices, by one wave; the same in every lane.
__device__ __forceinline__ RowStat join_row(const VerifyArgs &a, int64_t s, int i) {
  const SliceStat *p = a.stats + (s * (2 * a.K + 1) + i) * a.slices;
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  for (int k = lane; k < a.slices; k += 64) m = fmaxf(m, p[k].m);
  m = wave_max(m);
  double S = 0.0;
  int first = 0x7fffffff;
  for (int k = lane; k < a.slices; k += 64) {
    const SliceStat t = p[k];
    if (t.m != -INFINITY || !(t.S == 0.0)) S += t.S * exp64(((double)t.m - (double)m) * a.inv_T);
    if (t.m == m) first = min(first, t.first);
  }
  S = wave_sum64(S);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
  RowStat r;
  r.inv = S > 0.0 && m != -INFINITY ? 1.0 / S : 0.0;  // NaN: no distribution
  r.m = m;
  r.first = first;
  return r;
}

__device__ __forceinline__ double prob(float x, const RowStat &r, double inv_T) {
  return exp64(((double)x - (double)r.m) * inv_T) * r.inv;
}

// The sequence's rows joined, the first draft that is not accepted found; tokens and log-probabilities of the accepted
// ones written by the workgroup that is told to.
template <int DT>
__device__ void decide(const VerifyArgs &a, int64_t s, bool write, VerifyArgs::Decision &dec) {
  __shared__ RowStat rows[2 * kVDrafts + 1];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, len = drafts_of(a, s);
  for (int i = w; i < 2 * a.K + 1; i += kVWaves) {
    const bool draft = i > a.K;
    if (draft ? (!a.zd || i - a.K - 1 >= len) : i > len) continue;
    const RowStat r = join_row(a, s, i);
    if (lane == 0) rows[i] = r;
  }
  __syncthreads();
  __shared__ VerifyArgs::Decision found;
  if (w == 0) {
    int64_t x = -1;
    bool ok = false, token = false;
    double lp = 0.0;
    RowStat p{}, q{};
    if (lane < len) {
      x = a.drafts[s * a.K + lane];
      p = rows[lane];
      token = x >= 0 && x < a.V;
      if (a.greedy) {
        ok = p.inv > 0.0 && x == p.first;
      } else if (token && p.inv > 0.0) {
        double qx = 1.0;
        if (a.zd) {
          q = rows[a.K + 1 + lane];
          qx = q.inv > 0.0 ? prob((float)row_of<DT>(a.zd, a.ls_d, a.lr_d, s, lane)[x], q, a.inv_T) : __builtin_nan("");
        }
        ok = (double)a.u[s * (a.K + 1) + lane] * qx < prob((float)row_of<DT>(a.z, a.ls, a.lr, s, lane)[x], p, a.inv_T);
      }
      if (ok && write)
        lp = ((double)(float)row_of<DT>(a.z, a.ls, a.lr, s, lane)[x] - (double)p.m) * a.inv_T + log(p.inv);
    }
    const uint64_t no = __ballot(!ok);  // lanes from len on are among them; K < 64
    const int at = __ffsll((long long)no) - 1;
    if (write && lane <= a.K) {
      a.tokens[s * (a.K + 1) + lane] = lane < at ? x : -1;
      a.logp[s * (a.K + 1) + lane] = lane < at ? (float)lp : 0.f;
      if (lane == 0) a.accepted[s] = at;
    }
    if (lane == at) {  // at <= len <= K
      found.p = rows[at];
      found.a = at;
      found.residual = 0;
      found.x = (int)x;
      if (at < len && token && !a.greedy) {
        if (!a.zd) found.residual = 2;
        else if (q.inv > 0.0) found.residual = 1;
      }
      found.q = found.residual == 1 ? q : RowStat{0.0, 0.f, 0};
    }
  }
  __syncthreads();
  dec = found;
}

// r of one column.
__device__ __forceinline__ double mass(const VerifyArgs &a, const VerifyArgs::Decision &d, float x, float y, int c) {
  const double p = prob(x, d.p, a.inv_T);
  if (d.residual == 1) return fmax(p - prob(y, d.q, a.inv_T), 0.0);
  return d.residual == 2 && c == d.x ? 0.0 : p;
}

template <int DT>
__global__ __launch_bounds__(kVThreads) void verify_residual_kernel(VerifyArgs a) {
  const int64_t s = blockIdx.y;
  VerifyArgs::Decision d;
  decide<DT>(a, s, blockIdx.x == 0, d);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.dec[s] = d;
  if (d.residual == 0 || !(d.p.inv > 0.0)) return;
  const int c0 = blockIdx.x * a.per, c1 = min(a.V, c0 + a.per);
  const typename Elem<DT>::T *row = row_of<DT>(a.z, a.ls, a.lr, s, d.a);
  const typename Elem<DT>::T *rowd = d.residual == 1 ? row_of<DT>(a.zd, a.ls_d, a.lr_d, s, d.a) : row;
  double sum = 0.0;
  sweep_slice<DT>(row, c0, c1, [&](float x, int c) { sum += mass(a, d, x, d.residual == 1 ? (float)rowd[c] : 0.f, c); });
  __shared__ double ss[kVWaves];
  sum = wave_sum64(sum);
  if ((threadIdx.x & 63) == 0) ss[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int k = 0; k < kVWaves; ++k) sum += ss[k];
    a.sums[s * a.slices + blockIdx.x] = sum;
  }
}

// Of values that the threads hold in order (v, no less than 0): the first whose running sum, from `base` on, exceeds t,
// else the last above 0; -1 without one. before: the running sum ahead of it. buf: kVThreads doubles.
__device__ __forceinline__ int find_passing(double v, int n, double base, double t, double *buf, double &before) {
  buf[threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.x < 64) {  // each lane a run of the values, the runs' sums scanned
    const int run = (n + 63) / 64, lo = min(n, (int)threadIdx.x * run), hi = min(n, lo + run);
    double mine = 0.0;
    for (int k = lo; k < hi; ++k) mine += buf[k];
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(incl, o, 64);
      if ((int)threadIdx.x >= o) incl += up;
    }
    double cum = base + (incl - mine);
    int at = -1, last = -1;
    double ahead = 0.0, ahead_last = 0.0;
    for (int k = lo; k < hi; ++k) {
      const double x = buf[k];
      if (x > 0.0) {
        last = k;
        ahead_last = cum;
        if (at < 0 && cum + x > t) {
          at = k;
          ahead = cum;
        }
      }
      cum += x;
    }
    const uint64_t hit = __ballot(at >= 0), some = __ballot(last >= 0);
    int got = -1;
    double b = 0.0;
    if (hit) {
      const int l = __ffsll((long long)hit) - 1;
      got = __shfl(at, l, 64);
      b = __shfl(ahead, l, 64);
    } else if (some) {
      const int l = 63 - __clzll((long long)some);
      got = __shfl(last, l, 64);
      b = __shfl(ahead_last, l, 64);
    }
    if (threadIdx.x == 0) {
      buf[kVThreads] = b;
      buf[kVThreads + 1] = (double)got;
    }
  }
  __syncthreads();
  before = buf[kVThreads];
  const int got = (int)buf[kVThreads + 1];
  __syncthreads();
  return got;
}

template <int DT>
__global__ __launch_bounds__(kVThreads) void verify_pick_kernel(VerifyArgs a) {
  __shared__ double part[kVSlices];
  __shared__ double buf[kVThreads + 2];
  __shared__ int token;
  const int64_t s = blockIdx.x;
  VerifyArgs::Decision d;
  if (a.greedy) decide<DT>(a, s, true, d);
  else d = a.dec[s];
  const int64_t out = s * (a.K + 1) + d.a;
  if (!(d.p.inv > 0.0)) {  // the target's row has no distribution: no token
    if (threadIdx.x == 0) a.logp[out] = __builtin_nanf("");
    return;
  }
  const typename Elem<DT>::T *row = row_of<DT>(a.z, a.ls, a.lr, s, d.a);
  if (a.greedy) {
    if (threadIdx.x == 0) {
      a.tokens[out] = d.p.first;
      a.logp[out] = (float)log(d.p.inv);
    }
    return;
  }
  const typename Elem<DT>::T *rowd = d.residual == 1 ? row_of<DT>(a.zd, a.ls_d, a.lr_d, s, d.a) : row;
  // the slices' sums; where p - q leaves nothing (p = q up to rounding), p itself
  double all = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    const bool res = d.residual != 0;
    double mine = 0.0;
    for (int k = threadIdx.x; k < a.slices; k += kVThreads) {
      double x;
      if (res) {
        x = a.sums[s * a.slices + k];
      } else {
        const SliceStat t = a.stats[(s * (2 * a.K + 1) + d.a) * a.slices + k];
        x = t.m == -INFINITY ? 0.0 : t.S * exp64(((double)t.m - (double)d.p.m) * a.inv_T) * d.p.inv;
      }
      part[k] = x;
      mine += x;
    }
    mine = wave_sum64(mine);
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = mine;
    __syncthreads();
    all = 0.0;
    for (int k = 0; k < kVWaves; ++k) all += buf[k];
    __syncthreads();
    if (all > 0.0 || !res) break;
    d.residual = 0;
  }
  const double t = (double)a.u[s * (a.K + 1) + a.K] * all;
  // the slice: each thread a run of slices
  const int srun = (a.slices + kVThreads - 1) / kVThreads;
  double mine = 0.0;
  for (int k = threadIdx.x * srun; k < min(a.slices, (int)(threadIdx.x + 1) * srun); ++k) mine += part[k];
  double base;
  const int owner = find_passing(mine, kVThreads, 0.0, t, buf, base);
  if (owner < 0) {  // u is no number, or nothing is left
    if (threadIdx.x == 0) a.logp[out] = __builtin_nanf("");
    return;
  }
  int slice = owner * srun, last = slice;
  double cum = base, cum_last = base;
  for (int k = slice, done = 0; k < min(a.slices, (owner + 1) * srun) && !done; ++k) {
    if (part[k] > 0.0) {
      last = k;
      cum_last = cum;
      done = cum + part[k] > t;
    }
    cum += part[k];
  }
  slice = last;
  base = cum_last;
  // the token: each thread a run of the slice's columns
  const int c0 = slice * a.per, c1 = min(a.V, c0 + a.per), run = a.per / kVThreads;
  const int lo = min(c1, c0 + (int)threadIdx.x * run), hi = min(c1, lo + run);
  mine = 0.0;
  for (int c = lo; c < hi; ++c) mine += mass(a, d, (float)row[c], d.residual == 1 ? (float)rowd[c] : 0.f, c);
  const int who = find_passing(mine, kVThreads, base, t, buf, base);
  if (threadIdx.x == 0) token = -1;
  __syncthreads();
  if ((int)threadIdx.x == who) {
    int got = -1;
    double run_sum = base;
    for (int c = lo; c < hi; ++c) {
      const double x = mass(a, d, (float)row[c], d.residual == 1 ? (float)rowd[c] : 0.f, c);
      if (x > 0.0) {
        got = c;
        if (run_sum + x > t) break;
      }
      run_sum += x;
    }
    token = got;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.tokens[out] = token;
    a.logp[out] = token < 0 ? __builtin_nanf("") : (float)(((double)(float)row[token] - (double)d.p.m) * a.inv_T + log(d.p.inv));
  }
}

// Values of a slice: 4,096, and as many times 1,024 more as keep a row within kVSlices slices.
static int slice_values(int V) {
  const int64_t least = round_up(cdiv(V, kVSlices), 1024);
  return (int)(least > 4096 ? least : 4096);
}

struct VerifyLayout {
  int slices, per;
  size_t stats, sums, dec, total;
};
static VerifyLayout verify_layout(int64_t S, int K, int V) {
  VerifyLayout L;
  L.per = slice_values(V);
  L.slices = (int)cdiv(V, L.per);
  L.stats = 0;
  L.sums = (size_t)S * (2 * K + 1) * L.slices * sizeof(SliceStat);
  L.dec = L.sums + (size_t)round_up(S * L.slices * 8, 16);
  L.total = L.dec + (size_t)S * sizeof(VerifyArgs::Decision);
  return L;
}

template <int DT> static int go_verify(const VerifyArgs &a, hipStream_t st) {
  const int rows = 2 * a.K + 1;
  VerifyArgs b = a;
  const int64_t step = 65535 / rows;  // sequences a launch: a grid's second dimension
  for (int64_t s0 = 0; s0 < a.S; s0 += step) {
    const int64_t n = a.S - s0 < step ? a.S - s0 : step;
    b.S = n;
    b.z = (const typename Elem<DT>::T *)a.z + s0 * a.ls;
    b.zd = a.zd ? (const typename Elem<DT>::T *)a.zd + s0 * a.ls_d : nullptr;
    b.drafts = a.drafts + s0 * a.K;
    b.lengths = a.lengths ? a.lengths + s0 : nullptr;
    b.u = a.u ? a.u + s0 * (a.K + 1) : nullptr;
    b.stats = a.stats + s0 * rows * a.slices;
    b.sums = a.sums + s0 * a.slices;
    b.dec = a.dec + s0;
    b.tokens = a.tokens + s0 * (a.K + 1);
    b.accepted = a.accepted + s0;
    b.logp = a.logp + s0 * (a.K + 1);
    hipLaunchKernelGGL(verify_stats_kernel<DT>, dim3((unsigned)a.slices, (unsigned)(n * rows)), dim3(kVThreads), 0, st, b);
    OCTO_CHECK_LAUNCH("verify_stats");
    if (!a.greedy) {
      hipLaunchKernelGGL(verify_residual_kernel<DT>, dim3((unsigned)a.slices, (unsigned)n), dim3(kVThreads), 0, st, b);
      OCTO_CHECK_LAUNCH("verify_residual");
    }
    hipLaunchKernelGGL(verify_pick_kernel<DT>, dim3((unsigned)n), dim3(kVThreads), 0, st, b);
    OCTO_CHECK_LAUNCH("verify_pick");
  }
  return OCTO_OK;
}

}  // namespace octo

using namespace octo;

extern "C" {

int octo_verify_workspace_bytes(int64_t S, int K, int V, size_t *bytes) {
  OCTO_CHECK_ARG(bytes != nullptr, "verify_workspace_bytes: null pointer");
  OCTO_CHECK_ARG(S >= 0 && S <= (1 << 20) && K >= 0 && K <= kVDrafts && V > 0 && V <= OCTO_ROW_MAX,
                 "verify: bad shape S=%lld K=%d V=%d (at most %d drafts)", (long long)S, K, V, kVDrafts);
  *bytes = verify_layout(S, K, V).total;
  return OCTO_OK;
}

int octo_verify_drafts(const void *logits, int64_t ld_seq, int64_t ld_row, const void *draft_logits, int64_t ld_seq_d,
                       int64_t ld_row_d, int dtype, const int64_t *drafts, const int64_t *lengths, const float *uniform,
                       int64_t S, int K, int V, double inv_T, int greedy, int64_t *tokens, int64_t *accepted,
                       float *logp, void *ws, size_t ws_bytes, void *stream) {
  size_t need = 0;
  const int rc = octo_verify_workspace_bytes(S, K, V, &need);
  if (rc) return rc;
  if (!is_float(dtype)) return octo_fail(OCTO_EUNSUPPORTED, "verify: dtype %d", dtype);
  OCTO_CHECK_ARG(ld_row >= 0 && ld_seq >= 0 && (!draft_logits || (ld_row_d >= 0 && ld_seq_d >= 0)), "verify: strides");
  OCTO_CHECK_ARG(inv_T > 0.0 && inv_T < 1e38, "verify: temperature must be positive");
  if (S == 0) return OCTO_OK;
  OCTO_CHECK_ARG(logits && (drafts || K == 0) && (uniform || greedy) && tokens && accepted && logp,
                 "verify: null pointer");
  OCTO_CHECK_ARG((uintptr_t)logits % float_bytes(dtype) == 0 && (uintptr_t)draft_logits % float_bytes(dtype) == 0,
                 "verify: misaligned logits");
  OCTO_CHECK_ARG((uintptr_t)ws % 16 == 0, "verify: misaligned workspace");
  if (!ws || ws_bytes < need)
    return octo_fail(OCTO_EWORKSPACE, "verify: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
  const VerifyLayout L = verify_layout(S, K, V);
  VerifyArgs a;
  a.z = logits;
  a.zd = greedy || K == 0 ? nullptr : draft_logits;
  a.ls = ld_seq;
  a.lr = ld_row;
  a.ls_d = ld_seq_d;
  a.lr_d = ld_row_d;
  a.drafts = drafts;
  a.lengths = lengths;
  a.u = uniform;
  a.S = S;
  a.K = K;
  a.V = V;
  a.inv_T = inv_T;
  a.greedy = greedy != 0;
  a.slices = L.slices;
  a.per = L.per;
  a.stats = (SliceStat *)((char *)ws + L.stats);
  a.sums = (double *)((char *)ws + L.sums);
  a.dec = (VerifyArgs::Decision *)((char *)ws + L.dec);
  a.tokens = tokens;
  a.accepted = accepted;
  a.logp = logp;
  switch (dtype) {
    case OCTO_BF16: return go_verify<OCTO_BF16>(a, (hipStream_t)stream);
    case OCTO_F16: return go_verify<OCTO_F16>(a, (hipStream_t)stream);
    default: return go_verify<OCTO_F32>(a, (hipStream_t)stream);
  }
}

}  // extern "C"
