// Drafted tokens checked against the target's probabilities (octo_verify_drafts).
//
//   p_i = softmax(z_i / T), q_i = softmax(z'_i / T), or all of it at the draft where the drafts come without logits.
//   Draft i is accepted when u_i q_i(x_i) < p_i(x_i); the first that is not ends the sequence at a. The next token is
//   the lowest v whose running sum of r_w = max(p_a(w) - q_a(w), 0) exceeds u_K sum r; r = p_a after the last draft.
//
// Which token that is has to be the definition's, not one beside it: of 150,000 running sums some lie within fp32's
// rounding of any number, and then another token is answered. So the exponentials and sums are taken in 64 bits
// (exp2_64 below, 4e-16 relative; some 1e-15 with its argument's rounding), and a draw differs from the exact one with
// a probability of about V times that.
//
// Rows are summed by waves, a part of a row each, in an order that the sizes alone decide. Few logits take three
// launches, all in 64 bits:
//   stats     each part's maximum and its sum of exponentials against it, every row that a sequence may need
//   residual  each workgroup joins its sequence's rows, finds a by itself, and its waves sum their parts' r
//   pick      a workgroup per sequence finds the part in which the running sum passes u_K sum r, and in it the token
// Many take the exponentials of stats in 32 bits (64-bit ones are 20 instructions each with their argument, and stats
// is most of the work), which leave each row's sum within 5e-6 (see fast_spread). That decides a draft unless u q and p
// are closer than 2^-15; then the row and its draft's are summed again in 64 bits there. Accepted drafts' and greedy's
// log-probabilities keep those sums, and with them the 5e-6. decide, sums and rest take residual's place: a is found
// once a sequence, and one sweep over row a of both models finds in 64 bits their sums and those of r (part_sums).
//
// Few logits are bound by the launches' latency (one sequence, 4 drafts, V 151,936: 6 + 8 + 6 us), many by memory and
// by 64-bit arithmetic: 256 sequences of up to 7 drafts, bf16, statistics 175 us for 1.1 GB, sums 79 us for 2 x 39
// million exponentials, the other three 33 us.
#include "octo_common.h"
#include "row_values.h"
#include "rows8.h"

namespace octo {

constexpr int kVThreads = 256, kVWaves = kVThreads / 64;
constexpr int kVDrafts = OCTO_DRAFTS_MAX;
constexpr int kVParts = 1024;   // parts of a row, at most
constexpr int kVBlock = 2048;   // values that a wave holds at a time: 4 chunks of 8 a lane
constexpr double kVClose = 1.0 / 32768;
constexpr double kVLn2 = 0.69314718055994530942;

// 2^t for t <= 0, -inf included (below -1000: 0), within 4e-16 of its value: t = n + f, |f| <= 1/2, n from the last
// bits of t + 1.5 x 2^52, and 2^f by the polynomial of degree 10 through it at the 11 Chebyshev nodes of [-1/2, 1/2]:
// 17 instructions, no conversion, rounding or ldexp of 64 bits.
__device__ __forceinline__ double exp2_64(double t) {
  const double shift = 6755399441055744.0, b = t + shift, f = t - (b - shift);
  double e = 7.072585949269223e-09;
  e = __builtin_fma(e, f, 1.0208690299958306e-07);
  e = __builtin_fma(e, f, 1.321544258792169e-06);
  e = __builtin_fma(e, f, 1.5252657260200837e-05);
  e = __builtin_fma(e, f, 0.0001540353044173605);
  e = __builtin_fma(e, f, 0.0013333558230164974);
  e = __builtin_fma(e, f, 0.009618129107606888);
  e = __builtin_fma(e, f, 0.05550410866444772);
  e = __builtin_fma(e, f, 0.24022650695910097);
  e = __builtin_fma(e, f, 0.69314718055995);
  e = __builtin_fma(e, f, 1.0);
  const uint64_t bits = __builtin_bit_cast(uint64_t, e) + ((uint64_t)(uint32_t)__builtin_bit_cast(uint64_t, b) << 52);
  return t < -1000.0 ? 0.0 : __builtin_bit_cast(double, bits);
}

struct PartStat {
  double S;   // sum of exp((z - m) / T); NaN where the part has a NaN or +inf
  float m;    // maximum
  int first;  // its first column (greedy)
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
  double c;                   // log2(e) / T
  float cf;                   // the same in 32 bits
  int greedy;
  int parts, part;      // parts of a row, values of each (a multiple of kVBlock)
  int sparts, spart;    // the same of stats (EXACT: as these)
  PartStat *stats;      // [S, 2 K + 1, sparts]: target rows, then draft rows
  // [S, parts]: of e = exp((z - m) / T) of row a, of its draft row's; of both over the columns with r > 0 (sum_a NaN:
  // not known yet). Few logits: sum_a holds the sums of r.
  double *sum_p, *sum_q, *sum_a, *sum_b;
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
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
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

// Chunk u of a lane of the kVBlock values from column c on: columns c + 512 u + 8 lane .. + 7, -inf from c1 on. Rows
// may start at any element (16-byte global loads need no alignment).
typedef i32x4 i32x4_any2 __attribute__((aligned(2)));
typedef i32x4 i32x4_any4 __attribute__((aligned(4)));
template <int DT>
__device__ __forceinline__ void load_whole(const typename Elem<DT>::T *p, float (&x)[8]) {
  if constexpr (DT == OCTO_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const i32x4 v = ((const i32x4_any4 *)p)[h];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * h + e] = __int_as_float(v[e]);
    }
  } else {
    unpack8(*(const i32x4_any2 *)p, DT == OCTO_F16, x);
  }
}
template <int DT>
__device__ __forceinline__ void load_values(const typename Elem<DT>::T *row, int c, int c1, float (&x)[8]) {
  if (c + 8 <= c1) {
    load_whole<DT>(row + c, x);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = c + e < c1 ? (float)row[c + e] : -INFINITY;
  }
}
// All of them at once but for a row's last block: a branch a chunk makes each load wait for the one before.
template <int DT>
__device__ __forceinline__ void load_block(const typename Elem<DT>::T *row, int c, int c1, float (&x)[4][8]) {
  const int lane = threadIdx.x & 63;
  if (c + kVBlock <= c1) {
#pragma unroll
    for (int u = 0; u < 4; ++u) load_whole<DT>(row + c + 512 * u + 8 * lane, x[u]);
  } else {
#pragma unroll
    for (int u = 0; u < 4; ++u) load_values<DT>(row, c + 512 * u + 8 * lane, c1, x[u]);
  }
}

// The same as they lie, for sweeps over two rows: half the registers until each chunk's turn.
template <int DT>
__device__ __forceinline__ void load_raw_block(const typename Elem<DT>::T *row, int c, int c1, Raw8<DT> (&v)[4]) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x & 63;
  if (c + kVBlock <= c1) {
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = load_raw8<DT>(row + c + 512 * u + 8 * lane);
  } else {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = c + 512 * u + 8 * lane;
      T x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = at + e < c1 ? row[at + e] : (T)-INFINITY;
      v[u] = __builtin_bit_cast(Raw8<DT>, x);
    }
  }
}

// A wave's part in 64 bits.
template <int DT>
__device__ __forceinline__ PartStat exact_part(const VerifyArgs &a, const typename Elem<DT>::T *row, int c0, int c1) {
  float m = -INFINITY;
  double S = 0.0;
  int first = 0x7fffffff;
  bool bad = false;
  for (int c = c0; c < c1; c += kVBlock) {
    float x[4][8], mx = m;
    load_block<DT>(row, c, c1, x);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        mx = fmaxf(mx, x[u][e]);
        bad |= !(x[u][e] < INFINITY);
      }
    if (mx > m) {
      S *= exp2_64(((double)m - (double)mx) * a.c);
      first = 0x7fffffff;
      m = mx;
    }
    const double md = m == -INFINITY ? 0.0 : (double)m;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) S += exp2_64(((double)x[u][e] - md) * a.c);
    if (a.greedy) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (x[u][e] == m) first = min(first, c + 512 * u + 8 * (int)(threadIdx.x & 63) + e);
    }
  }
  PartStat r;
  r.m = wave_max(m);
  r.S = wave_sum64(m == -INFINITY ? 0.0 : S * exp2_64(((double)m - (double)r.m) * a.c));
  if (__any(bad)) r.S = __builtin_nan("");
  r.first = wave_min(m == r.m ? first : 0x7fffffff);
  return r;
}

// A wave's run of blocks with exponentials in 32 bits, the next block's loads in flight. exp2 is within 2^-23 of its
// value, and its argument (z - m) c, c rounded to 32 bits, off by at most 1.5 x 2^-23 of itself (d, c and the product),
// which makes ln 2 times that of the value: over a row at most 2^-23 (1 + 1.04 x 30), as the mean of |d c| under the
// softmax is at most log2 V. Eight values are summed in 32 bits (3 x 2^-24), all else in 64. Together below 5e-6 of the
// row's sum. A NaN stays one through difference, product and exponential, and +inf makes one (inf - inf): S shows both.
template <int DT>
__device__ __forceinline__ PartStat fast_spread(const VerifyArgs &a, const typename Elem<DT>::T *row, int c0, int c1) {
  float m = -INFINITY;
  double S = 0.0;
  int first = 0x7fffffff;
  Raw8<DT> v[2][4];
  auto take = [&](const Raw8<DT>(&r)[4], int c) {
    float x[4][8], mx = m;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      values8<DT>(r[u], x[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, x[u][e]);
    }
    if (mx > m) {
      S *= exp2_64(((double)m - (double)mx) * a.c);
      first = 0x7fffffff;
      m = mx;
    }
    const float mf = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = fexp2((x[u][e] - mf) * a.cf);
      S += (double)(((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7])));
    }
    if (a.greedy) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (x[u][e] == m) first = min(first, c + 512 * u + 8 * (int)(threadIdx.x & 63) + e);
    }
  };
  load_raw_block<DT>(row, c0, c1, v[0]);
  for (int c = c0;;) {
    if (c + kVBlock < c1) load_raw_block<DT>(row, c + kVBlock, c1, v[1]);
    take(v[0], c);
    if ((c += kVBlock) >= c1) break;
    if (c + kVBlock < c1) load_raw_block<DT>(row, c + kVBlock, c1, v[0]);
    take(v[1], c);
    if ((c += kVBlock) >= c1) break;
  }
  PartStat r;
  r.m = wave_max(m);
  r.S = wave_sum64(m == -INFINITY ? S : S * exp2_64(((double)m - (double)r.m) * a.c));  // m -inf: S is 0 or NaN
  r.first = wave_min(m == r.m ? first : 0x7fffffff);
  return r;
}

template <int DT, bool EXACT>
__global__ __launch_bounds__(kVThreads) void verify_stats_kernel(VerifyArgs a) {
  const int rows = 2 * a.K + 1;
  const int64_t s = blockIdx.y / rows;
  const int i = (int)(blockIdx.y - s * rows), len = drafts_of(a, s);
  const int k = __builtin_amdgcn_readfirstlane(blockIdx.x * kVWaves + (threadIdx.x >> 6));
  const bool draft = i > a.K;
  if (draft ? (!a.zd || i - a.K - 1 >= len) : i > len) return;  // nobody asks for the row
  if (k >= a.sparts) return;
  const typename Elem<DT>::T *row = draft ? row_of<DT>(a.zd, a.ls_d, a.lr_d, s, i - a.K - 1)
                                          : row_of<DT>(a.z, a.ls, a.lr, s, i);
  const int c0 = k * a.spart, c1 = (int)min((int64_t)a.V, (int64_t)c0 + a.spart);
  const PartStat r = EXACT ? exact_part<DT>(a, row, c0, c1) : fast_spread<DT>(a, row, c0, c1);
  if ((threadIdx.x & 63) == 0) a.stats[(int64_t)blockIdx.y * a.sparts + k] = r;
}

// Row i's statistics from its parts, by one wave; the same in every lane.
__device__ __forceinline__ RowStat join_row(const VerifyArgs &a, int64_t s, int i) {
  const PartStat *p = a.stats + (s * (2 * a.K + 1) + i) * a.sparts;
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  double S = 0.0;
  int first = 0x7fffffff;
  for (int k = lane; k < a.sparts; k += 64) {
    const PartStat t = p[k];
    const float mx = fmaxf(m, t.m);
    if (mx > m) {
      S = m == -INFINITY ? S : S * exp2_64(((double)m - (double)mx) * a.c);
      first = 0x7fffffff;
      m = mx;
    }
    S += t.m == -INFINITY ? t.S : t.S * exp2_64(((double)t.m - (double)m) * a.c);
    if (t.m == m) first = min(first, t.first);
  }
  RowStat r;
  r.m = wave_max(m);
  S = wave_sum64(m == -INFINITY ? S : S * exp2_64(((double)m - (double)r.m) * a.c));
  r.first = wave_min(m == r.m ? first : 0x7fffffff);
  r.inv = S > 0.0 && r.m != -INFINITY && r.m != INFINITY ? 1.0 / S : 0.0;  // NaN: no distribution
  return r;
}

__device__ __forceinline__ double prob(float x, const RowStat &r, double c) {
  return exp2_64(((double)x - (double)r.m) * c) * r.inv;
}

// 1 / the sum of a whole row in 64 bits, by the workgroup.
template <int DT, int NW>
__device__ double exact_inv(const VerifyArgs &a, const typename Elem<DT>::T *row, float m, double *red) {
  double S = 0.0;
  for (int64_t c = (int64_t)(threadIdx.x >> 6) * kVBlock; c < a.V; c += NW * kVBlock) {
    float x[4][8];
    load_block<DT>(row, (int)c, a.V, x);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) S += exp2_64(((double)x[u][e] - (double)m) * a.c);
  }
  S = wave_sum64(S);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = S;
  __syncthreads();
  S = 0.0;
  for (int k = 0; k < NW; ++k) S += red[k];
  return 1.0 / S;
}

// The sequence's rows joined, the first draft that is not accepted found; tokens and log-probabilities of the accepted
// ones written by the workgroup that is told to.
template <int DT, bool EXACT, int NW>
__device__ void decide(const VerifyArgs &a, int64_t s, bool write, VerifyArgs::Decision &dec) {
  __shared__ RowStat rows[2 * kVDrafts + 1];
  __shared__ VerifyArgs::Decision found;
  __shared__ double red[NW];
  __shared__ int again;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, len = drafts_of(a, s);
  for (int i = w; i < 2 * a.K + 1; i += NW) {
    const bool draft = i > a.K;
    if (draft ? (!a.zd || i - a.K - 1 >= len) : i > len) continue;
    const RowStat r = join_row(a, s, i);
    if (lane == 0) rows[i] = r;
  }
  __syncthreads();
  int64_t x = -1;
  bool ok = false, token = false, close = false;
  float zp = 0.f, zq = 0.f, u = 0.f;
  RowStat p{}, q{};
  if (w == 0 && lane < len) {
    x = a.drafts[s * a.K + lane];
    token = x >= 0 && x < a.V;
    if (!a.greedy) u = a.u[s * (a.K + 1) + lane];
    if (token) {
      zp = (float)row_of<DT>(a.z, a.ls, a.lr, s, lane)[x];
      if (a.zd) zq = (float)row_of<DT>(a.zd, a.ls_d, a.lr_d, s, lane)[x];
    }
  }
  for (int32_t known = -1;;) {  // once, and again for every draft whose rows have to be summed in 64 bits
    if (w == 0) {
      if (lane < len) {
        p = rows[lane];
        if (a.zd) q = rows[a.K + 1 + lane];
        if (a.greedy) {
          ok = p.inv > 0.0 && x == p.first;
        } else if (token && p.inv > 0.0 && !(a.zd && !(q.inv > 0.0))) {
          const double lhs = (double)u * (a.zd ? prob(zq, q, a.c) : 1.0), rhs = prob(zp, p, a.c);
          ok = lhs < rhs;
          close = !EXACT && lane > known && fabs(lhs - rhs) <= kVClose * rhs;
        }
      }
      const uint64_t no = __ballot(!ok), near = __ballot(close);  // lanes from len on are in `no`; K < 64
      const int at = __ffsll((long long)no) - 1, first_near = near ? __ffsll((long long)near) - 1 : 64;
      if (first_near <= at && first_near < len) {
        if (lane == 0) again = first_near;
      } else {
        if (lane == 0) again = -1;
        if (write && lane <= a.K) {
          a.tokens[s * (a.K + 1) + lane] = lane < at ? x : -1;
          a.logp[s * (a.K + 1) + lane] =
              lane < at ? (float)(((double)zp - (double)p.m) * a.c * kVLn2 + log(p.inv)) : 0.f;
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
    }
    __syncthreads();
    const int i = again;
    if (EXACT || i < 0) break;
    const double inv_p = exact_inv<DT, NW>(a, row_of<DT>(a.z, a.ls, a.lr, s, i), rows[i].m, red);
    double inv_q = 0.0;
    if (a.zd) inv_q = exact_inv<DT, NW>(a, row_of<DT>(a.zd, a.ls_d, a.lr_d, s, i), rows[a.K + 1 + i].m, red);
    __syncthreads();
    if (threadIdx.x == 0) {
      rows[i].inv = inv_p;
      if (a.zd) rows[a.K + 1 + i].inv = inv_q;
    }
    __syncthreads();
    known = i;
    close = false;
  }
  dec = found;
}

// r of one column. MODE: Decision::residual.
template <int MODE>
__device__ __forceinline__ double mass(const VerifyArgs &a, const VerifyArgs::Decision &d, float x, float y, int c) {
  const double p = prob(x, d.p, a.c);
  if (MODE == 1) return fmax(p - prob(y, d.q, a.c), 0.0);
  return MODE == 2 && c == d.x ? 0.0 : p;
}

__device__ __forceinline__ double sum_parts(const double *v, int n) {  // by each wave; the same in every lane
  double S = 0.0;
  for (int k = threadIdx.x & 63; k < n; k += 64) S += v[k];
  return wave_sum64(S);
}
// Row a's statistics with the sums of the sums launch.
__device__ __forceinline__ void exact_rows(const VerifyArgs &a, int64_t s, VerifyArgs::Decision &d) {
  if (d.p.inv > 0.0) d.p.inv = 1.0 / sum_parts(a.sum_p + s * a.parts, a.parts);
  if (d.residual == 1) d.q.inv = 1.0 / sum_parts(a.sum_q + s * a.parts, a.parts);
}

// A row a wave, for up to 8 drafts: 64 sequences of 4 drafts 6 us. Once a sequence: in sums each of some 20 workgroups
// would join the same rows.
constexpr int kVDecide = 1024;
template <int DT>
__global__ __launch_bounds__(kVDecide) void verify_decide_kernel(VerifyArgs a) {
  VerifyArgs::Decision d;
  decide<DT, false, kVDecide / 64>(a, blockIdx.x, true, d);
  if (threadIdx.x == 0) a.dec[blockIdx.x] = d;
}

// With S_p and S_q the rows' sums, r > 0 where e_p > rho e_q, rho = S_p / S_q, and there r = e_p / S_p - e_q / S_q: one
// sweep finds the sums of e_p and e_q over all columns and over those, for which it is enough to know rho within 2^-15
// (the statistics give it within 1e-5), unless a column's e_p lies that close to rho e_q. A part with such a column
// (one in fifty where the models differ) is left to the next launch. 256 sequences of V 151,936: the call 358 us in
// kernels so, 388 with a sweep for S_p and S_q and another for r.
template <int DT, int MODE>
__device__ __forceinline__ void part_sums(const VerifyArgs &a, const VerifyArgs::Decision &d, int64_t s, int k, int c0,
                                          int c1) {
  const int lane = threadIdx.x & 63;
  const typename Elem<DT>::T *row = row_of<DT>(a.z, a.ls, a.lr, s, d.a);
  const typename Elem<DT>::T *rowd = MODE == 1 ? row_of<DT>(a.zd, a.ls_d, a.lr_d, s, d.a) : row;
  const double mp = d.p.m, mq = d.q.m, rho = MODE == 1 ? d.q.inv / d.p.inv : 0.0;
  double P = 0.0, Q = 0.0, A = 0.0, B = 0.0;
  bool near = false;
  for (int c = c0; c < c1; c += kVBlock) {
    Raw8<DT> xr[4], yr[4];
    load_raw_block<DT>(row, c, c1, xr);
    if (MODE == 1) load_raw_block<DT>(rowd, c, c1, yr);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float x[8], y[8];
      values8<DT>(xr[u], x);
      if (MODE == 1) values8<DT>(yr[u], y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double ep = exp2_64(((double)x[e] - mp) * a.c);
        P += ep;
        if (MODE == 1) {
          const double eq = exp2_64(((double)y[e] - mq) * a.c), over = __builtin_fma(-rho, eq, ep);
          Q += eq;
          A += over > 0.0 ? ep : 0.0;
          B += over > 0.0 ? eq : 0.0;
          near |= fabs(over) < kVClose * ep;
        } else if (MODE == 2) {
          A += c + 512 * u + 8 * lane + e == d.x ? 0.0 : ep;
        }
      }
    }
  }
  P = wave_sum64(P);
  if (MODE) A = wave_sum64(A);
  if (MODE == 1) {
    Q = wave_sum64(Q);
    B = wave_sum64(B);
    if (__any(near)) A = __builtin_nan("");
  }
  if (lane == 0) {
    a.sum_p[s * a.parts + k] = P;
    if (MODE) a.sum_a[s * a.parts + k] = A;
    if (MODE) a.sum_b[s * a.parts + k] = B;
    if (MODE == 1) a.sum_q[s * a.parts + k] = Q;
  }
}

template <int DT>
__global__ __launch_bounds__(kVThreads) void verify_sums_kernel(VerifyArgs a) {
  const int64_t s = blockIdx.y;
  const VerifyArgs::Decision d = a.dec[s];
  if (!(d.p.inv > 0.0)) return;
  const int k = __builtin_amdgcn_readfirstlane(blockIdx.x * kVWaves + (threadIdx.x >> 6));
  if (k >= a.parts) return;
  const int c0 = k * a.part, c1 = (int)min((int64_t)a.V, (int64_t)c0 + a.part);
  if (d.residual == 1) part_sums<DT, 1>(a, d, s, k, c0, c1);
  else if (d.residual == 2) part_sums<DT, 2>(a, d, s, k, c0, c1);
  else part_sums<DT, 0>(a, d, s, k, c0, c1);
}

template <int DT, int MODE>
__device__ __forceinline__ double part_mass(const VerifyArgs &a, const VerifyArgs::Decision &d,
                                            const typename Elem<DT>::T *row, const typename Elem<DT>::T *rowd, int c0,
                                            int c1) {
  const int lane = threadIdx.x & 63;
  double S = 0.0;
  for (int c = c0; c < c1; c += kVBlock) {
    Raw8<DT> xr[4], yr[4];
    load_raw_block<DT>(row, c, c1, xr);
    if (MODE == 1) load_raw_block<DT>(rowd, c, c1, yr);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float x[8], y[8];
      values8<DT>(xr[u], x);
      if (MODE == 1) values8<DT>(yr[u], y);
#pragma unroll
      for (int e = 0; e < 8; ++e) S += mass<MODE>(a, d, x[e], MODE == 1 ? y[e] : 0.f, c + 512 * u + 8 * lane + e);
    }
  }
  return wave_sum64(S);
}

template <int DT>
__global__ __launch_bounds__(kVThreads) void verify_residual_kernel(VerifyArgs a) {
  const int64_t s = blockIdx.y;
  VerifyArgs::Decision d;
  decide<DT, true, kVWaves>(a, s, blockIdx.x == 0, d);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.dec[s] = d;
  if (d.residual == 0 || !(d.p.inv > 0.0)) return;
  const typename Elem<DT>::T *row = row_of<DT>(a.z, a.ls, a.lr, s, d.a);
  const typename Elem<DT>::T *rowd = d.residual == 1 ? row_of<DT>(a.zd, a.ls_d, a.lr_d, s, d.a) : row;
  const int k = __builtin_amdgcn_readfirstlane(blockIdx.x * kVWaves + (threadIdx.x >> 6));
  if (k >= a.parts) return;
  const int c0 = k * a.part, c1 = (int)min((int64_t)a.V, (int64_t)c0 + a.part);
  const double S =
      d.residual == 1 ? part_mass<DT, 1>(a, d, row, rowd, c0, c1) : part_mass<DT, 2>(a, d, row, rowd, c0, c1);
  if ((threadIdx.x & 63) == 0) a.sum_a[s * a.parts + k] = S;
}

// The parts that verify_sums_kernel left: their sum of r, in the form of the others (sum_a / S_p - sum_b / S_q).
template <int DT>
__global__ __launch_bounds__(kVThreads) void verify_rest_kernel(VerifyArgs a) {
  const int64_t s = blockIdx.y;
  if (a.dec[s].residual != 1) return;
  const int k = __builtin_amdgcn_readfirstlane(blockIdx.x * kVWaves + (threadIdx.x >> 6));
  if (k >= a.parts || a.sum_a[s * a.parts + k] == a.sum_a[s * a.parts + k]) return;
  VerifyArgs::Decision d = a.dec[s];
  if (!(d.p.inv > 0.0)) return;
  exact_rows(a, s, d);
  const int c0 = k * a.part, c1 = (int)min((int64_t)a.V, (int64_t)c0 + a.part);
  const double S = part_mass<DT, 1>(a, d, row_of<DT>(a.z, a.ls, a.lr, s, d.a),
                                    row_of<DT>(a.zd, a.ls_d, a.lr_d, s, d.a), c0, c1);
  if ((threadIdx.x & 63) == 0) {
    a.sum_a[s * a.parts + k] = S / d.p.inv;
    a.sum_b[s * a.parts + k] = 0.0;
  }
}

// Of values that the threads hold in order (v, no less than 0): the first whose running sum, from `base` on, exceeds t,
// else the last above 0; -1 without one. before: the running sum ahead of it. buf: kVThreads + 2 doubles.
__device__ __forceinline__ int find_passing(double v, double base, double t, double *buf, double &before) {
  constexpr int RUN = kVThreads / 64;
  buf[threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.x < 64) {  // each lane a run of the values, the runs' sums scanned
    const int lo = (int)threadIdx.x * RUN;
    double mine = 0.0;
#pragma unroll
    for (int k = 0; k < RUN; ++k) mine += buf[lo + k];
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(incl, o, 64);
      if ((int)threadIdx.x >= o) incl += up;
    }
    double cum = base + (incl - mine);
    int at = -1, last = -1;
    double ahead = 0.0, ahead_last = 0.0;
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      const double x = buf[lo + k];
      if (x > 0.0) {
        last = lo + k;
        ahead_last = cum;
        if (at < 0 && cum + x > t) {
          at = lo + k;
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

// A thread's run of columns.
template <int DT, int MODE>
__device__ __forceinline__ double run_mass(const VerifyArgs &a, const VerifyArgs::Decision &d,
                                           const typename Elem<DT>::T *row, const typename Elem<DT>::T *rowd, int lo,
                                           int hi) {
  double S = 0.0;
  for (int c = lo; c < hi; c += 8) {
    float x[8], y[8];
    load_values<DT>(row, c, hi, x);
    if (MODE == 1) load_values<DT>(rowd, c, hi, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) S += mass<MODE>(a, d, x[e], MODE == 1 ? y[e] : 0.f, c + e);
  }
  return S;
}

template <int DT, bool EXACT>
__global__ __launch_bounds__(kVThreads) void verify_pick_kernel(VerifyArgs a) {
  __shared__ double part[kVParts];
  __shared__ double buf[kVThreads + 2];
  __shared__ int token;
  const int64_t s = blockIdx.x;
  VerifyArgs::Decision d;
  if (a.greedy) decide<DT, EXACT, kVWaves>(a, s, true, d);
  else d = a.dec[s];
  const int64_t out = s * (a.K + 1) + d.a;
  if (!(d.p.inv > 0.0)) {  // the target's row has no distribution: no token
    if (threadIdx.x == 0) a.logp[out] = __builtin_nanf("");
    return;
  }
  if (a.greedy) {
    if (threadIdx.x == 0) {
      a.tokens[out] = d.p.first;
      a.logp[out] = (float)log(d.p.inv);
    }
    return;
  }
  if constexpr (!EXACT) exact_rows(a, s, d);
  const typename Elem<DT>::T *row = row_of<DT>(a.z, a.ls, a.lr, s, d.a);
  const typename Elem<DT>::T *rowd = d.residual == 1 ? row_of<DT>(a.zd, a.ls_d, a.lr_d, s, d.a) : row;
  // the parts' sums; where p - q leaves nothing (p = q up to rounding), p itself
  double all = 0.0;
  for (;;) {
    const bool res = d.residual != 0;
    double mine = 0.0;
    for (int k = threadIdx.x; k < a.parts; k += kVThreads) {
      double x;
      if (res) {
        x = a.sum_a[s * a.parts + k];
        if constexpr (!EXACT) x = fmax(x * d.p.inv - a.sum_b[s * a.parts + k] * d.q.inv, 0.0);
      } else if constexpr (EXACT) {
        const PartStat t = a.stats[(s * (2 * a.K + 1) + d.a) * a.parts + k];
        x = t.m == -INFINITY ? 0.0 : t.S * exp2_64(((double)t.m - (double)d.p.m) * a.c) * d.p.inv;
      } else {
        x = a.sum_p[s * a.parts + k] * d.p.inv;
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
  // the part: each thread a run of them
  const int run = (a.parts + kVThreads - 1) / kVThreads;
  double mine = 0.0;
  for (int k = threadIdx.x * run; k < min(a.parts, (int)(threadIdx.x + 1) * run); ++k) mine += part[k];
  double base;
  const int owner = find_passing(mine, 0.0, t, buf, base);
  if (owner < 0) {  // nothing is left
    if (threadIdx.x == 0) a.logp[out] = __builtin_nanf("");
    return;
  }
  int got = owner * run;
  double cum = base;
  for (int k = got, done = 0; k < min(a.parts, (owner + 1) * run) && !done; ++k) {
    if (part[k] > 0.0) {
      got = k;
      base = cum;
      done = cum + part[k] > t;
    }
    cum += part[k];
  }
  // the token: each thread a run of the part's columns, 8 at a time
  const int c0 = got * a.part, c1 = (int)min((int64_t)a.V, (int64_t)c0 + a.part), width = a.part / kVThreads;
  const int lo = min(c1, c0 + (int)threadIdx.x * width), hi = min(c1, lo + width);
  mine = d.residual == 1 ? run_mass<DT, 1>(a, d, row, rowd, lo, hi)
         : d.residual == 2 ? run_mass<DT, 2>(a, d, row, rowd, lo, hi)
                           : run_mass<DT, 0>(a, d, row, rowd, lo, hi);
  const int who = find_passing(mine, base, t, buf, base);
  if (threadIdx.x == 0) token = -1;
  __syncthreads();
  if ((int)threadIdx.x == who) {
    int v = -1;
    double sum = base;
    for (int c = lo; c < hi; ++c) {
      const float z = (float)row[c];
      const double x = d.residual == 1 ? mass<1>(a, d, z, (float)rowd[c], c)
                       : d.residual == 2 ? mass<2>(a, d, z, z, c) : mass<0>(a, d, z, z, c);
      if (x > 0.0) {
        v = c;
        if (sum + x > t) break;
      }
      sum += x;
    }
    token = v;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.tokens[out] = token;
    a.logp[out] = token < 0 ? __builtin_nanf("")
                            : (float)(((double)(float)row[token] - (double)d.p.m) * a.c * kVLn2 + log(d.p.inv));
  }
}

// Parts of one block, and as many blocks more as keep a row within kVParts parts: pick scans a row's parts in the LDS
// and sweeps one again. A wave that takes several of them in sums measured the same.
static int part_values(int V) { return (int)round_up(cdiv(V, kVParts), kVBlock); }

// Rows that are summed with 32-bit exponentials, from this many logits on. V 128,256, 4 drafts with logits, us a call
// without and with: 9.2M logits 32.3 and 37.0, 18.5M 40.9 and 41.4, 36.9M 56.0 and 50.5, 73.9M 89.5 and 74.5. V
// 151,936: 128 sequences of one draft without logits 74.1 and 54.6, with them 82.2 and 74.6; 256 of 4 drafts 377 and
// 209, of 7 599 and 292; greedy, no draft, 42 and 24. A draw without drafts is summed in 64 bits on either route and
// gains nothing: 128 sequences 33.2 and 38.8, 256 56.6 and 63.9, 512 91.7 and 97.3.
constexpr int64_t kVMany = (int64_t)1 << 24;
// Their statistics by runs of up to 4 parts a wave, whose next loads are in flight during a part's arithmetic and whose
// reductions across lanes come once, as long as that leaves this many waves. 256 x 9 rows of 151,936 bf16 values, us a
// call: runs of 2 238, 4 222, 8 225; 512 x 15 rows 545, 519, 529. 256 x 15, statistics alone: runs of 1 240, 4 175.
constexpr int64_t kVSpread = 16384;

struct VerifyLayout {
  int parts, part;
  size_t stats, sums, dec, total;
};
static VerifyLayout verify_layout(int64_t S, int K, int V) {
  VerifyLayout L;
  L.part = part_values(V);
  L.parts = (int)cdiv(V, L.part);
  L.stats = 0;
  L.sums = (size_t)S * (2 * K + 1) * L.parts * sizeof(PartStat);
  L.dec = L.sums + (size_t)(4 * S * L.parts * 8);
  L.total = L.dec + (size_t)S * sizeof(VerifyArgs::Decision);
  return L;
}

template <int DT, bool EXACT> static int go_launches(const VerifyArgs &a, hipStream_t st) {
  const dim3 spread((unsigned)cdiv(a.sparts, kVWaves), (unsigned)(a.S * (2 * a.K + 1)));
  const dim3 parts((unsigned)cdiv(a.parts, kVWaves), (unsigned)a.S);
  hipLaunchKernelGGL((verify_stats_kernel<DT, EXACT>), spread, dim3(kVThreads), 0, st, a);
  OCTO_CHECK_LAUNCH("verify_stats");
  if (!a.greedy && !EXACT) {
    hipLaunchKernelGGL(verify_decide_kernel<DT>, dim3((unsigned)a.S), dim3(kVDecide), 0, st, a);
    OCTO_CHECK_LAUNCH("verify_decide");
    hipLaunchKernelGGL(verify_sums_kernel<DT>, parts, dim3(kVThreads), 0, st, a);
    OCTO_CHECK_LAUNCH("verify_sums");
  }
  if (!a.greedy && !EXACT && a.zd) {
    hipLaunchKernelGGL(verify_rest_kernel<DT>, parts, dim3(kVThreads), 0, st, a);
    OCTO_CHECK_LAUNCH("verify_rest");
  }
  if (!a.greedy && EXACT) {
    hipLaunchKernelGGL(verify_residual_kernel<DT>, parts, dim3(kVThreads), 0, st, a);
    OCTO_CHECK_LAUNCH("verify_residual");
  }
  hipLaunchKernelGGL((verify_pick_kernel<DT, EXACT>), dim3((unsigned)a.S), dim3(kVThreads), 0, st, a);
  OCTO_CHECK_LAUNCH("verify_pick");
  return OCTO_OK;
}

template <int DT> static int go_verify(const VerifyArgs &a, bool exact, hipStream_t st) {
  const int rows = 2 * a.K + 1;
  const int64_t step = 65535 / rows;  // sequences a launch: a grid's second dimension
  for (int64_t s0 = 0; s0 < a.S; s0 += step) {
    VerifyArgs b = a;
    b.S = a.S - s0 < step ? a.S - s0 : step;
    b.z = (const typename Elem<DT>::T *)a.z + s0 * a.ls;
    b.zd = a.zd ? (const typename Elem<DT>::T *)a.zd + s0 * a.ls_d : nullptr;
    b.drafts = a.drafts + s0 * a.K;
    b.lengths = a.lengths ? a.lengths + s0 : nullptr;
    b.u = a.u ? a.u + s0 * (a.K + 1) : nullptr;
    b.stats = a.stats + s0 * rows * a.sparts;
    b.sum_p = a.sum_p + s0 * a.parts;
    b.sum_q = a.sum_q + s0 * a.parts;
    b.sum_a = a.sum_a + s0 * a.parts;
    b.sum_b = a.sum_b + s0 * a.parts;
    b.dec = a.dec + s0;
    b.tokens = a.tokens + s0 * (a.K + 1);
    b.accepted = a.accepted + s0;
    b.logp = a.logp + s0 * (a.K + 1);
    const int rc = exact ? go_launches<DT, true>(b, st) : go_launches<DT, false>(b, st);
    if (rc) return rc;
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
  a.greedy = greedy != 0;
  const double c = inv_T * 1.4426950408889634074;
  a.c = c;
  a.cf = (float)c;
  a.parts = L.parts;
  a.part = L.part;
  a.stats = (PartStat *)((char *)ws + L.stats);
  a.sum_p = (double *)((char *)ws + L.sums);
  a.sum_q = a.sum_p + S * L.parts;
  a.sum_a = a.sum_q + S * L.parts;
  a.sum_b = a.sum_a + S * L.parts;
  a.dec = (VerifyArgs::Decision *)((char *)ws + L.dec);
  a.tokens = tokens;
  a.accepted = accepted;
  a.logp = logp;
  const int64_t rows = S * (a.zd ? 2 * K + 1 : K + 1);
  const bool exact = rows * V < kVMany || !(c >= 0x1p-40 && c <= 0x1p40);
  const int64_t run = exact ? 1 : rows * L.parts / kVSpread;
  a.spart = L.part * (int)(run < 1 ? 1 : (run > 4 ? 4 : run));
  a.sparts = (int)cdiv(V, a.spart);
  switch (dtype) {
    case OCTO_BF16: return go_verify<OCTO_BF16>(a, exact, (hipStream_t)stream);
    case OCTO_F16: return go_verify<OCTO_F16>(a, exact, (hipStream_t)stream);
    default: return go_verify<OCTO_F32>(a, exact, (hipStream_t)stream);
  }
}

}  // extern "C"
