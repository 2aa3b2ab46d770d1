// The head's logits from 8-bit integers, and their gradients (octo_head_logits_i8, octo_head_grads_i8).
//
//   z[r, v] = sx[r] sw[v] sum_k qx[r, k] qw[v, k]          (the sum exact in 32 bits: d <= 131,072)
//   dx[r, k] = sum_v g[r, v] sw[v] qw[v, k]                (straight through the rounding of rows and weights)
//   dW[v, k] = sum_r g[r, v] sx[r] qx[r, k]
//
// Three routes for the logits, by the rows. Up to 32 read the weight's bytes once and are bound by them (few_i8_kernel:
// 1 row of d 2560, V 151,936 74 us, 5.2 TB/s). Up to 128, and more of a small vocabulary, the same in tiles, two
// workgroups a CU (64 rows 95 us, 4.3 TB/s with the logits). More are bound by the matrix rate: 8,192 rows 2,740 us,
// 2.33 POP/s with the logits' 2.5 GB written beside it (without them 2,614; a library product of these integers, which
// writes 32-bit sums, reaches 1.82).
//
// The gradients are 16-bit products of the widened operands (prepare8_kernel: 190 us at that weight, a write of 778
// MB), at the rate of the head's other gradients: 2,048 rows 2,480 us for both, 1.29 PFLOP/s. The rows' gradient of up
// to 128 reads the 8-bit weight itself (few_dx_kernel). f16 operands are widened times a power of two (f16_range), for
// which a launch finds the largest scale: 225 rows of d 1024, V 32,000 80.7 us, 76.3 without, where rows of 1e5 gave
// NaN.
#include <type_traits>

#include "gemm_nt.h"
#include "octo_internal.h"
#include "row_values.h"
#include "rows8.h"

namespace octo {

constexpr int kMaxD8 = 131072;       // 127^2 d < 2^31
constexpr int kMaxV8 = 1 << 21;      // a tile's 256 rows of g within 32-bit offsets
constexpr int64_t kMaxN8 = 1 << 21;  // the same of the transposed rows
// M-tiles that an XCD walks the tokens with: 2,048 rows at d 2560, V 151,936 795 us in fours, 749 in eights, the same
// in sixteens, more in thirty-twos.
constexpr int kGroup8 = 8;
// Tiles of 128 x 128 up to this many rows. The same weight, us with them and with wide ones: 64 rows 95 and 118, 128
// 104 and 119, 192 147 and 126, 256 157 and 133. (Eight waves on the small tile: 128 rows 111.) And where the card
// holds all of them at once, two a CU: 256 rows of d 1024 V 32,000 20.0 and 22.8, 512 of V 16,000 19.9 and 27.3, 256 of
// d 4096 V 32,000 41.6 and 46.1; beyond, 512 of V 32,000 31.2 and 27.7, 256 of d 2304 V 64,000 48.8 and 43.2.
constexpr int64_t kSmallRows = 128;
static bool small_tiles(int64_t n, int V) {
  return n <= kSmallRows || cdiv(n, 128) * cdiv(V, 128) <= 2 * octo_tiles::kCus;
}

typedef i32x4 i32x4_el __attribute__((aligned(2)));
typedef i32x4 i32x4_el4 __attribute__((aligned(4)));
typedef i32x2 i32x2_el __attribute__((aligned(2)));

struct Logits8 {
  const float *sx, *sw;
  void *z;
  int64_t ldz;
};

// The product over tiles of VM vocabulary rows x TN tokens, weights as the MFMA's first operand: a lane's 4 sums of a
// block are 4 neighbouring logits of one token. NW waves, 2 along the vocabulary.
template <int VM, int TOK, int NW_> struct Tile8 {
  static constexpr int NW = NW_, NWN = NW / 2, ROWS = VM, TOKENS = TOK;
  typedef OpRowsN<NW, VM / 2, VM> A;
  typedef OpRowsN<NW, TOK / NWN, TOK> B;
  static constexpr int NA = A::NB, NB = B::NB, LDS = ENSLOT * ring5_slot<A, B>();
  static __device__ __forceinline__ int row(int w, int i, int lane) {
    return w / NWN * (VM / 2) + i * 16 + 4 * (lane >> 4);
  }
  static __device__ __forceinline__ int col(int w, int j, int lane) {
    return w % NWN * (TOK / NWN) + j * 16 + (lane & 15);
  }
};
typedef Tile8<256, 256, 8> TileWide;   // one workgroup a CU
typedef Tile8<256, 192, 8> Tile192;    // the last tokens of a wide grid: 320 rows of d 4096 228 us without, 209 with
typedef Tile8<256, 128, 8> Tile128;
typedef Tile8<128, 128, 4> TileSmall;  // half the LDS: two workgroups a CU, one loading and multiplying while the other
                                       // begins or stores

// Scaled in fp32 (the sum, times the token's scale, times the weight's), rounded to the logits' type, and out through
// the LDS in rows of the tile's logits. A slot holds 4 logits; slot s of token t sits at s ^ 4 (t & 15) (128 logits: t
// & 7): a write's 16 tokens x 4 slots cover all banks.
template <class L, typename OT>
__device__ __forceinline__ void store_logits8(const f32x4 (&acc)[L::NA][L::NB], const Logits8 &e, int64_t v0,
                                              int64_t n0, int V, int64_t nvalid, lds_char *smem) {
  constexpr int SLOT = 4 * sizeof(OT), ROW = L::ROWS / 4 * SLOT, HALVES = L::TOKENS * ROW > L::LDS ? 2 : 1;
  constexpr int TOK = L::TOKENS / HALVES;
  constexpr int LPR = ROW / 16, PER = 16 / sizeof(OT), SWZ = L::ROWS / 16 - 1;  // lanes of a row, logits of a lane
  static_assert(TOK * ROW <= L::LDS && L::NWN % HALVES == 0, "staged in the ring");
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int vvalid = (int)min((int64_t)L::ROWS, V - v0);
  float sx[L::NB];
#pragma unroll
  for (int j = 0; j < L::NB; ++j) {
    const int t = L::col(w, j, lane);
    sx[j] = t < nvalid ? e.sx[n0 + t] : 0.f;
  }
  OT *out = (OT *)e.z + n0 * e.ldz + v0;
  for (int h = 0; h < HALVES; ++h) {
    if (h) __syncthreads();
    if (w % L::NWN / (L::NWN / HALVES) == h) {
#pragma unroll
      for (int i = 0; i < L::NA; ++i) {
        const int m = L::row(w, i, lane);
        float sw[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) sw[v] = m + v < vvalid ? e.sw[v0 + m + v] : 0.f;
#pragma unroll
        for (int j = 0; j < L::NB; ++j) {
          const i32x4 q = __builtin_bit_cast(i32x4, acc[i][j]);
          const int t = L::col(w, j, lane) - h * TOK;
          OT o[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = (OT)((float)q[v] * sx[j] * sw[v]);
          lds_char *at = smem + t * ROW + (((m >> 2) ^ ((t & SWZ) << 2)) * SLOT);
          if constexpr (sizeof(OT) == 4) *(lds_i32x4 *)at = __builtin_bit_cast(i32x4, o);
          else *(__attribute__((address_space(3))) i32x2 *)at = __builtin_bit_cast(i32x2, o);
        }
      }
    }
    __syncthreads();
    const int c = threadIdx.x % LPR, c0 = c * PER;
    for (int t = threadIdx.x / LPR; t < TOK && h * TOK + t < nvalid; t += 64 * L::NW / LPR) {
      const i32x4 v = *(const lds_i32x4 *)(smem + t * ROW + (c * 16 ^ (((t & SWZ) << 2) * SLOT)));
      OT *o = out + (h * TOK + t) * e.ldz + c0;
      if (vvalid == L::ROWS) {
        if constexpr (sizeof(OT) == 4) __builtin_nontemporal_store(v, (i32x4_el4 *)o);
        else __builtin_nontemporal_store(v, (i32x4_el *)o);
      } else {
        OT x[PER];
        __builtin_memcpy(x, &v, 16);
#pragma unroll
        for (int u = 0; u < PER; ++u)
          if (c0 + u < vvalid) o[u] = x[u];
      }
    }
  }
}

template <class L, typename OT>
__device__ __forceinline__ void gemm_i8_tile(const Operand &A, const Operand &B, const GemmShape &s, const Logits8 &e,
                                             int64_t m0, int64_t n0, lds_char *smem) {
  f32x4 acc[L::NA][L::NB];
  mainloop_ring5<DT_I8, typename L::A, typename L::B, true>(A, B, m0, n0, s.K, smem, acc);
  store_logits8<L, OT>(acc, e, m0, n0, (int)s.M, min(s.N - n0, (int64_t)L::TOKENS), smem);
}
template <typename OT>
__global__ __launch_bounds__(512, 1) __attribute__((amdgpu_waves_per_eu(2, 2)))
void gemm_i8_kernel(Operand A, Operand B, GemmShape s, Logits8 e) {
  __shared__ __attribute__((aligned(16))) char smem_[TileWide::LDS];
  int mt, nt;
  if (!tile_of(s, mt, nt)) return;
  const int64_t m0 = (int64_t)mt * 256, n0 = (int64_t)nt * 256, left = s.N - n0;
  if (left <= 128) gemm_i8_tile<Tile128, OT>(A, B, s, e, m0, n0, (lds_char *)smem_);
  else if (left <= 192) gemm_i8_tile<Tile192, OT>(A, B, s, e, m0, n0, (lds_char *)smem_);
  else gemm_i8_tile<TileWide, OT>(A, B, s, e, m0, n0, (lds_char *)smem_);
}
template <typename OT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void gemm_i8_small_kernel(Operand A, Operand B, GemmShape s, Logits8 e) {
  __shared__ __attribute__((aligned(16))) char smem_[TileSmall::LDS];
  int mt, nt;
  if (!tile_of(s, mt, nt)) return;
  gemm_i8_tile<TileSmall, OT>(A, B, s, e, (int64_t)mt * 128, (int64_t)nt * 128, (lds_char *)smem_);
}

// ---- few rows -------------------------------------------------------------------------------------------------------
//
// Up to 32 rows the weight's bytes set the time. The rows, quantised by every workgroup for itself (which saves a
// launch; workgroup 0 leaves them to the caller), stay in the LDS, and each wave runs through a share of the weight
// rows of its own, 16 at a time: the MFMA's first operand comes from global memory as it lies (lane l: row l & 15, 16
// bytes at 16 (l >> 4) of each 64), kFewSteps loads ahead, also into the next 16 rows, and no wave waits for another.
// The shares are equal to 4 rows, so that all waves end together: of 16 rows each, 9,496 blocks would take the 4,096
// waves of 16 a CU three rounds, as long as 12,288. A share's last block repeats its last row (no bytes of its own, and
// its MFMAs are idle time).
//
// us so and in the small tiles: d 2560, V 151,936, bf16 1 row 74 and 90, 8 80 and 91, 16 87 and 91, 24 94 and 92, 32 96
// and 92, fp32 1 row 75 and 91, 16 91 and 91, 32 102 and 92; d 4096, V 128,256, bf16 1 row 109 and 121, 17 125 and 124,
// 32 125 and 126; d 1024, V 32,000, bf16 1 row 8.6 and 12.2, 8 9.5 and 12.5, 16 13.3 and 12.5, 32 18.7 and 12.5. So the
// crossing lies at 12 to 24 rows, below the limit. Weight loads past the caches (nontemporal) take a quarter longer for
// 1 row.
constexpr int kFewSteps = 8;
constexpr int kFewLds = 156 * 1024;  // with the scales, what a workgroup can have
constexpr int64_t kFewRows = 32;

struct Few8 {
  const void *x;
  int64_t ldx;
  const int8_t *wq;
  int64_t ldw;
  const float *sw;
  int n, d, V, share;  // share: weight rows a wave takes
  int8_t *xq;
  int64_t ldxq;
  float *sx;
  void *z;
  int64_t ldz;
};

// LDS bytes between rows: the next multiple of 64 (a step), and 16 so that rows start on different banks.
__host__ __device__ constexpr int few_ld(int d) { return (d + 63) / 64 * 64 + 16; }

template <int DT, typename OT, int NB, int NW>
__global__ __launch_bounds__(64 * NW) void few_i8_kernel(Few8 a) {
  extern __shared__ __attribute__((aligned(16))) char few_smem[];
  __shared__ float scales[16 * NB];
  lds_char *smem = (lds_char *)few_smem;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qd = lane >> 4;
  const int chunks = (a.d + 15) >> 4, steps = (chunks + 3) >> 2, ld = few_ld(a.d);
  const int first = (blockIdx.x * NW + w) * a.share, last = min(first + a.share, a.V);
  i32x4 cur[kFewSteps], nxt[kFewSteps];
  // steps s0 .. of the 16 rows from m0; chunks past a row's end: its last one, times the zeros of x there
  auto load = [&](i32x4(&v)[kFewSteps], int m0, int s0) {
    const i32x4 *p = (const i32x4 *)(a.wq + (int64_t)min(m0 + (lane & 15), last - 1) * a.ldw);
#pragma unroll
    for (int u = 0; u < kFewSteps; ++u) v[u] = p[min(4 * (s0 + u) + qd, chunks - 1)];
  };
  if (first < last) load(cur, first, 0);
  for (int r = w; r < a.n; r += NW) {
    lds_char *row = smem + r * ld;
    int8_t *kept = blockIdx.x == 0 ? a.xq + r * a.ldxq : nullptr;
    const auto *x = (const typename Elem<DT>::T *)a.x + r * a.ldx;
    auto put = [&](int c, i32x2 v) {
      *(__attribute__((address_space(3))) i32x2 *)(row + 8 * c) = v;
      if (kept && c < 2 * chunks) *(i32x2 *)(kept + 8 * c) = v;
    };
    const float s = quantise_row<DT, (DT == OCTO_F32 ? 2 : 4)>(x, a.d, (a.d + 63) / 64 * 8, put);
    if (lane == 0) {
      scales[r] = s;
      if (kept) a.sx[r] = s;
    }
  }
  __syncthreads();
  if (first >= last) return;
  const lds_char *xl[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) xl[b] = smem + min(16 * b + (lane & 15), a.n - 1) * ld + 16 * qd;
  for (int m0 = first; m0 < last; m0 += 16) {
    i32x4 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = i32x4{0, 0, 0, 0};
    for (int s0 = 0; s0 < steps; s0 += kFewSteps) {
      const bool more = s0 + kFewSteps < steps;
      if (more || m0 + 16 < last) load(nxt, more ? m0 : m0 + 16, more ? s0 + kFewSteps : 0);
#pragma unroll
      for (int u = 0; u < kFewSteps; ++u) {
        if (s0 + u >= steps) break;
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(cur[u], *(const lds_i32x4 *)(xl[b] + 64 * (s0 + u)), acc[b], 0,
                                                         0, 0);
      }
#pragma unroll
      for (int u = 0; u < kFewSteps; ++u) cur[u] = nxt[u];
    }
    const int v0 = m0 + 4 * qd;
    if (v0 < last) {
      float sw[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) sw[e] = a.sw[min(v0 + e, a.V - 1)];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int t = 16 * b + (lane & 15);
        if (t >= a.n) continue;
        OT o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (OT)((float)acc[b][e] * scales[t] * sw[e]);
        OT *out = (OT *)a.z + t * a.ldz + v0;
        if (v0 + 4 <= a.V) {
          if constexpr (sizeof(OT) == 2) *(i32x2_el *)out = __builtin_bit_cast(i32x2, o);
          else *(i32x4_el4 *)out = __builtin_bit_cast(i32x4, o);
        } else {
          for (int e = 0; v0 + e < a.V; ++e) out[e] = o[e];
        }
      }
    }
  }
}

// Whether the rows fit.
static bool few_fits(int64_t n, int d) { return n <= kFewRows && n * few_ld(d) <= kFewLds; }

template <int DT, typename OT, int NB> static int go_few(Few8 a, hipStream_t st) {
  const int lds = a.n * few_ld(a.d);
  // 16 waves a CU: two workgroups of 8 where two fit, else one of 16
  const int wgs = lds <= 78 * 1024 ? 2 : 1, NW = 16 / wgs;
  const int64_t waves = (int64_t)octo_tiles::kCus * wgs * NW;
  a.share = (int)round_up(cdiv(a.V, waves), 4);
  const dim3 grid((unsigned)cdiv(a.V, (int64_t)a.share * NW));
  if (wgs > 1) hipLaunchKernelGGL((few_i8_kernel<DT, OT, NB, 8>), grid, dim3(512), lds, st, a);
  else hipLaunchKernelGGL((few_i8_kernel<DT, OT, NB, 16>), grid, dim3(1024), lds, st, a);
  OCTO_CHECK_LAUNCH("few_i8");
  return OCTO_OK;
}
template <int DT, typename OT> static int go_few(const Few8 &a, hipStream_t st) {
  return a.n <= 16 ? go_few<DT, OT, 1>(a, st) : go_few<DT, OT, 2>(a, st);
}
template <typename OT> static int go_few(const Few8 &a, int x_dtype, hipStream_t st) {
  switch (x_dtype) {
    case OCTO_BF16: return go_few<OCTO_BF16, OT>(a, st);
    case OCTO_F16: return go_few<OCTO_F16, OT>(a, st);
    default: return go_few<OCTO_F32, OT>(a, st);
  }
}

// ---- few rows' gradient --------------------------------------------------------------------------------------------
//
// dx of few rows is the weight's bytes too, which a widened copy multiplies by five. Here a wave takes a share of the
// vocabulary and 256 columns: lane l holds 16 columns (16 bytes at 16 (l & 15)) of 8 rows (8 (l >> 4) ..) of each 32,
// so that its 8 bytes of a column are 8 neighbours along K, and product j of 16 takes column j of every lane: widened,
// rounded to g's type and fed without an exchange between lanes. f16: each wave widens by the power of two of its own
// share's scales (f16_range) and takes it back before the sums are joined. fp32 g: the integers and g's three parts, as
// in the large products. A workgroup's waves join their sums in the LDS, a second launch the workgroups', both in
// order.
//
// us so and by the widened copy: d 2560, V 151,936, bf16 8 rows 80 (4.9 TB/s) and 404, 32 89 and 403, 64 145 and 404,
// 128 270 and 408, 160 326 and 409, 192 391 and 412, 225 510 and 413 (blocks of 32 tokens run side by side and share
// some of their reads); fp32 8 rows 88 and 687, 128 574 and 761, 160 865 and 793; d 1024, V 32,000, bf16 128 rows 34
// and 57, 225 50 and 58, 384 72 and 64, fp32 128 53 and 92, 256 98 and 108, 384 183 and 136. So the crossing lies
// between 129 rows (fp32, large) and some 300 (small), at or above the limit.
//
// g times the scale in two bf16 parts against the integers, which rounds no operand to g's type, takes twice the
// products: 16 rows 82 us, but 32 138 and 128 426.
constexpr int kDxCols = 256, kDxWaves = 8;
constexpr int64_t kFewDx = 128;

struct FewDx {
  const void *g;
  int64_t ldg;
  const int8_t *wq;
  int64_t ldw;
  const float *sw;
  int n, d, V;
  int strips, groups, share;  // columns / 256; workgroups along the vocabulary; rows of one of their waves (32 k)
  f32x4 *part;                // [token blocks, strips, groups, 16 NB, 64]
  void *out;
  int64_t ldo;
};

template <int DT, int NB>
__global__ __launch_bounds__(64 * kDxWaves) void few_dx_kernel(FewDx a) {
  constexpr bool F32 = DT == OCTO_F32;
  constexpr int WT = F32 ? OCTO_BF16 : DT, NP = F32 ? 3 : 1, R = 16 * NB;
  typedef typename Elem<DT>::T T;
  __shared__ f32x4 smem[kDxWaves / 2][R][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qd = lane >> 4;
  const int strip = blockIdx.x % a.strips, group = blockIdx.x / a.strips;
  const int c = strip * kDxCols + 16 * (lane & 15);
  const int first = (group * kDxWaves + w) * a.share, last = min(first + a.share, a.V);
  const int8_t *col = a.wq + (c < a.d ? c : 0);
  const T *grow[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
    grow[b] = (const T *)a.g + min((int)blockIdx.y * 16 * NB + 16 * b + (lane & 15), a.n - 1) * a.ldg;
  f32x4 acc[NB][16];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Step {
    i32x4 q[8];
    Raw8<DT> g[NB];
    float s[8];
  };
  // rows past the share's end: its last one, times the zeros of g there
  auto load = [&](Step &t, int v0) {
    const int v = v0 + 8 * qd;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t r = min(v + e, last - 1);
      t.q[e] = *(const i32x4 *)(col + r * a.ldw);
      t.s[e] = a.sw[r];
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
      t.g[b] = v0 + 32 <= last ? load_raw8<DT>(grow[b] + v) : load_raw8<DT>(grow[b] + v, last - v);
  };
  float times = 1.f, back = 1.f;  // f16: f16_range of the share's scales
  auto take = [&](Step &t) {
    i32x4 gop[NB][NP];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if constexpr (F32) {
        float x[8];
        values8<DT>(t.g[b], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= t.s[e];
        split_parts(x, gop[b]);
      } else {
        gop[b][0] = t.g[b].v[0];
      }
    }
    if constexpr (DT == OCTO_F16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) t.s[e] *= times;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = (float)(int8_t)((uint32_t)t.q[e][j >> 2] >> (8 * (j & 3)));
        if constexpr (!F32) x[e] *= t.s[e];
      }
      const i32x4 op = pack8(x, WT == OCTO_F16);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int p = 0; p < NP; ++p) Mfma16<WT>::run(op, gop[b][p], acc[b][j]);
    }
  };
  if (first < last) {
    Step t[2];
    if constexpr (DT == OCTO_F16) {
      uint32_t m = 0;
#pragma unroll 4
      for (int v = first + lane; v < last; v += 64) m = max(m, finite_bits(a.sw[v]));
      f16_range((uint32_t)__builtin_amdgcn_readfirstlane((int)lanes_max<64>(m)), times, back);
    }
    load(t[0], first);
    for (int v = first;;) {
      if (v + 32 < last) load(t[1], v + 32);
      take(t[0]);
      if ((v += 32) >= last) break;
      if (v + 32 < last) load(t[0], v + 32);
      take(t[1]);
      if ((v += 32) >= last) break;
    }
  }
#pragma unroll
  for (int half = kDxWaves / 2; half > 0; half >>= 1) {
    const float own = DT == OCTO_F16 && half == kDxWaves / 2 ? back : 1.f;
    if (w >= half && w < 2 * half) {
#pragma unroll
      for (int r = 0; r < R; ++r) smem[w - half][r][lane] = acc[r >> 4][r & 15] * own;
    }
    __syncthreads();
    if (w < half) {
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r >> 4][r & 15] = acc[r >> 4][r & 15] * own + smem[w][r][lane];
    }
    __syncthreads();
  }
  if (w == 0) {
    f32x4 *out = a.part + (((int64_t)blockIdx.y * a.strips + strip) * a.groups + group) * R * 64;
#pragma unroll
    for (int r = 0; r < R; ++r) out[r * 64 + lane] = acc[r >> 4][r & 15];
  }
}

// The workgroups' sums joined: register r = 16 b + j of lane l holds token 16 b + (l & 15), columns 64 (l >> 4) + 16 e
// + j.
template <typename OT, int NB>
__global__ __launch_bounds__(256) void few_dx_sum_kernel(FewDx a) {
  constexpr int R = 16 * NB;
  const int strip = blockIdx.x / (R / 4), r = blockIdx.x % (R / 4) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const f32x4 *p = a.part + ((int64_t)blockIdx.y * a.strips + strip) * a.groups * R * 64 + r * 64 + lane;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = 0; k < a.groups; ++k) sum += p[(int64_t)k * R * 64];
  const int t = (int)blockIdx.y * 16 * NB + (r & ~15) + (lane & 15);
  const int c = strip * kDxCols + 64 * (lane >> 4) + (r & 15);
  if (t >= a.n) return;
  OT *out = (OT *)a.out + t * a.ldo;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + 16 * e < a.d) out[c + 16 * e] = (OT)sum[e];
}

struct DxSplit {
  int nb, blocks, strips, groups, share;
  size_t bytes;
};
// A workgroup a CU (its registers fill one).
static DxSplit dx_split(int64_t n, int d, int V, int dtype) {
  DxSplit s;
  s.nb = n <= 16 || dtype == OCTO_F32 ? 1 : 2;  // fp32's parts of 32 rows do not fit the registers
  s.blocks = (int)cdiv(n, 16 * s.nb);
  s.strips = (int)cdiv(d, kDxCols);
  const int64_t most = cdiv(V, 32 * kDxWaves), want = octo_tiles::kCus / ((int64_t)s.strips * s.blocks);
  const int64_t groups = want < 1 ? 1 : (want < most ? want : most);
  s.share = (int)round_up(cdiv(V, groups * kDxWaves), 32);
  s.groups = (int)cdiv(V, (int64_t)s.share * kDxWaves);
  s.bytes = (size_t)s.blocks * s.strips * s.groups * 16 * s.nb * 64 * sizeof(f32x4);
  return s;
}

template <int DT, int NB> static int go_few_dx(const FewDx &a, const DxSplit &s, int out_dtype, hipStream_t st) {
  hipLaunchKernelGGL((few_dx_kernel<DT, NB>), dim3((unsigned)(s.strips * s.groups), (unsigned)s.blocks),
                     dim3(64 * kDxWaves), 0, st, a);
  OCTO_CHECK_LAUNCH("few_dx");
  const dim3 grid((unsigned)(s.strips * 4 * NB), (unsigned)s.blocks);
  switch (out_dtype) {
    case OCTO_BF16: hipLaunchKernelGGL((few_dx_sum_kernel<__bf16, NB>), grid, dim3(256), 0, st, a); break;
    case OCTO_F16: hipLaunchKernelGGL((few_dx_sum_kernel<_Float16, NB>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((few_dx_sum_kernel<float, NB>), grid, dim3(256), 0, st, a); break;
  }
  OCTO_CHECK_LAUNCH("few_dx_sum");
  return OCTO_OK;
}
static int go_few_dx(const FewDx &a, const DxSplit &s, int dtype, int out_dtype, hipStream_t st) {
  switch (dtype) {
    case OCTO_BF16:
      return s.nb == 1 ? go_few_dx<OCTO_BF16, 1>(a, s, out_dtype, st) : go_few_dx<OCTO_BF16, 2>(a, s, out_dtype, st);
    case OCTO_F16:
      return s.nb == 1 ? go_few_dx<OCTO_F16, 1>(a, s, out_dtype, st) : go_few_dx<OCTO_F16, 2>(a, s, out_dtype, st);
    default: return go_few_dx<OCTO_F32, 1>(a, s, out_dtype, st);
  }
}

static Operand operand8(const void *base, int64_t ld_bytes, int64_t rows) {
  Operand X;
  X.base = (const char *)base;
  X.ld = ld_bytes;
  X.map = nullptr;
  X.rows = rows;
  X.count = nullptr;
  X.count_off = 0;
  X.extent = 0;
  return X;
}

static GemmShape shape8(int64_t M, int64_t N, int64_t K, int tile = TM) {
  GemmShape s;
  s.M = M;
  s.N = N;
  s.K = K;
  s.mtiles = (int)cdiv(M, tile);
  s.ntiles = (int)cdiv(N, tile);
  s.group_m = kGroup8;
  s.count_on = 0;
  s.count = nullptr;
  s.count_off = 0;
  return s;
}

// Workspace of the gradients: the widened weight [V, d] (K-major for dx) and the partial tiles of its split; the
// transposed rows [d, n]; g where its rows cannot be read as they are (g_as_is). Sizes padded as the K-major loads
// read.
//
// 16-bit g: the widened operand is rounded to its type, as the head's other gradients take their operands: 2.4e-3 from
// 64 bits in bf16, sqrt(2) times one rounding of an exact result. Two parts of g times the scale against the exact
// integers would double the products, which are most of the time; fp32 logits have gradients within 1e-6.
//
// fp32 g is not multiplied in fp32: an 8-bit integer is a bf16 number as it stands, so g times the scale that its
// product sums over, in three bf16 parts, times the integers is exact but for the sum: three bf16 products, where two
// fp32 operands take six. dx: the parts beside each other, K = 3 Vr through the weight's rows three times. dW: the
// parts below each other, K = 3 np against the rows' integers three times. d 2560, V 151,936, both gradients of 512
// rows 2,500 us, 4,700 as fp32 products (a library's 6,700).
struct Grads8Layout {
  int64_t Vr, dp, np, Vp;  // rows and columns of the copies
  int64_t Kh;              // dx's K
  int parts;               // of g
  size_t norm, wide, xt, g, gh, split, total;
  int64_t split_items;
  bool few;  // dx by few_dx_kernel, its partial sums in split
};

static Grads8Layout grads8_layout(int64_t n, int d, int V, int dtype, bool need_rows, bool need_w, bool as_is) {
  Grads8Layout L;
  L.parts = dtype == OCTO_F32 ? 3 : 1;
  L.Vr = round_up(V, 64);
  L.dp = round_up(d, TN);
  L.np = round_up(n, 64);
  L.Vp = round_up(V, TM);
  L.Kh = L.parts == 1 ? V : 3 * L.Vr;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (size_t)round_up((int64_t)bytes, 256);
    return p;
  };
  L.split_items = 0;
  L.few = need_rows && n <= kFewDx;
  if (L.few) need_rows = false;  // none of the copies for it
  if (need_rows) {
    const int64_t tiles = cdiv(n, TM) * cdiv(d, TN);
    if (tiles < octo_tiles::kSplitItemsMax) {
      const int S = octo_tiles::k_splits((int)tiles, (int)cdiv(L.Kh, 64), true, octo_tiles::kSplitItemsMax);
      if (S > 1) L.split_items = tiles * S;
    }
  }
  L.wide = take(need_rows ? (size_t)L.Vr * L.dp * 2 : 0);
  L.xt = take(need_w ? (size_t)d * L.parts * L.np * 2 : 0);
  const bool copied = L.parts == 3 ? need_w : !as_is && (need_rows || need_w);
  L.g = take(copied ? (size_t)L.parts * L.np * L.Vp * 2 : 0);
  L.gh = take(L.parts == 3 && need_rows ? (size_t)n * L.Kh * 2 : 0);
  L.split = take(L.few ? dx_split(n, d, V, dtype).bytes : (size_t)L.split_items * TM * TN * 4);
  L.norm = take(dtype == OCTO_F16 && (need_rows || need_w) ? sizeof(Norm8) : 0);
  L.total = at;
  return L;
}

// Whether the products can read g where it lies (2,048 rows of V 151,936: 2,728 us, 2,850 with a copy): 16-bit values
// in whole 16-byte chunks, a tile's rows and a stage's within 32-bit offsets.
static bool g_as_is(const void *g, int64_t ldg, int dtype, int V) {
  return dtype != OCTO_F32 && V % 8 == 0 && V >= TM && ldg % 8 == 0 && ldg <= kMaxV8 && (uintptr_t)g % 16 == 0;
}

static int head8_checks(const char *what, int64_t n, int d, int V, int64_t ldxq, int64_t ldw) {
  OCTO_CHECK_ARG(n >= 0 && n <= kMaxN8, "%s: n=%lld outside [0, %lld]", what, (long long)n, (long long)kMaxN8);
  OCTO_CHECK_ARG(d > 0 && d <= kMaxD8, "%s: d=%d outside [1, %d]", what, d, kMaxD8);
  OCTO_CHECK_ARG(V > 0 && V <= kMaxV8, "%s: V=%d outside [1, %d]", what, V, kMaxV8);
  for (int64_t ld : {ldxq, ldw})
    OCTO_CHECK_ARG(ld >= round_up(d, 16) && ld % 16 == 0 && ld <= 2 * kMaxD8,
                   "%s: 8-bit rows of stride %lld (a multiple of 16, at least d=%d)", what, (long long)ld, d);
  return OCTO_OK;
}

}  // namespace octo

using namespace octo;

extern "C" {

int octo_head_logits_i8(const void *rows, int64_t ldx, int x_dtype, const int8_t *wq, int64_t ldw, const float *w_scale,
                        int64_t n, int d, int V, int8_t *xq, int64_t ldxq, float *x_scale, void *logits, int64_t ldz,
                        int z_dtype, void *stream) {
  int rc = head8_checks("head_logits_i8", n, d, V, ldxq, ldw);
  if (rc) return rc;
  if (rows && !is_float(x_dtype)) return octo_fail(OCTO_EUNSUPPORTED, "head_logits_i8: dtype %d", x_dtype);
  OCTO_CHECK_ARG(ldz >= V, "head_logits_i8: row stride %lld below V=%d", (long long)ldz, V);
  if (!is_float(z_dtype)) return octo_fail(OCTO_EUNSUPPORTED, "head_logits_i8: dtype %d", z_dtype);
  if (n == 0) return OCTO_OK;
  OCTO_CHECK_ARG(wq && w_scale && xq && x_scale && logits, "head_logits_i8: null pointer");
  OCTO_CHECK_ARG((uintptr_t)wq % 16 == 0 && (uintptr_t)xq % 16 == 0 && (uintptr_t)w_scale % 4 == 0 &&
                     (uintptr_t)x_scale % 4 == 0 && (uintptr_t)logits % float_bytes(z_dtype) == 0,
                 "head_logits_i8: misaligned pointer");
  hipStream_t st = (hipStream_t)stream;
  if (rows && few_fits(n, d)) {
    OCTO_CHECK_ARG(ldx >= d && (uintptr_t)rows % float_bytes(x_dtype) == 0, "head_logits_i8: row stride or alignment");
    const Few8 a{rows, ldx, wq, ldw, w_scale, (int)n, d, V, 0, xq, ldxq, x_scale, logits, ldz};
    switch (z_dtype) {
      case OCTO_BF16: return go_few<__bf16>(a, x_dtype, st);
      case OCTO_F16: return go_few<_Float16>(a, x_dtype, st);
      default: return go_few<float>(a, x_dtype, st);
    }
  }
  if (rows) {
    rc = octo_quantise_i8_rows(rows, ldx, x_dtype, n, d, 0, xq, ldxq, x_scale, stream);
    if (rc) return rc;
  }
  const Logits8 e{x_scale, w_scale, logits, ldz};
  const Operand A = operand8(wq, ldw, V), B = operand8(xq, ldxq, n);
  const bool small = small_tiles(n, V);
  const GemmShape s = shape8(V, n, round_up(d, 16), small ? 128 : 256);
  const dim3 grid((unsigned)tile_grid(s.mtiles, s.ntiles)), block(small ? 256 : 512);
#define OCTO_GO(OT)                                                                                \
  if (small) hipLaunchKernelGGL(gemm_i8_small_kernel<OT>, grid, block, 0, st, A, B, s, e);         \
  else hipLaunchKernelGGL(gemm_i8_kernel<OT>, grid, block, 0, st, A, B, s, e)
  switch (z_dtype) {
    case OCTO_BF16: OCTO_GO(__bf16); break;
    case OCTO_F16: OCTO_GO(_Float16); break;
    default: OCTO_GO(float); break;
  }
#undef OCTO_GO
  OCTO_CHECK_LAUNCH("gemm_i8");
  return OCTO_OK;
}

int octo_head_grads_i8_workspace_bytes(const void *g, int64_t ldg, int dtype, int64_t n, int d, int V, int need_rows,
                                       int need_w, size_t *bytes) {
  OCTO_CHECK_ARG(bytes != nullptr, "head_grads_i8_workspace_bytes: null pointer");
  const int rc = head8_checks("head_grads_i8", n, d, V, round_up(d < 1 ? 1 : d, 16), round_up(d < 1 ? 1 : d, 16));
  if (rc) return rc;
  if (!is_float(dtype)) return octo_fail(OCTO_EUNSUPPORTED, "head_grads_i8: dtype %d", dtype);
  *bytes = grads8_layout(n, d, V, dtype, need_rows != 0, need_w != 0, g_as_is(g, ldg, dtype, V)).total;
  return OCTO_OK;
}

int octo_head_grads_i8(const void *g, int64_t ldg, int g_dtype, const int8_t *xq, int64_t ldxq, const float *x_scale,
                       const int8_t *wq, int64_t ldw, const float *w_scale, int64_t n, int d, int V, void *grad_rows,
                       int64_t ld_gr, int gr_dtype, void *grad_w, int64_t ld_gw, int gw_dtype, void *ws,
                       size_t ws_bytes, void *stream) {
  int rc = head8_checks("head_grads_i8", n, d, V, ldxq, ldw);
  if (rc) return rc;
  for (int t : {g_dtype, grad_rows ? gr_dtype : OCTO_F32, grad_w ? gw_dtype : OCTO_F32})
    if (!is_float(t)) return octo_fail(OCTO_EUNSUPPORTED, "head_grads_i8: dtype %d", t);
  OCTO_CHECK_ARG(n > 0, "head_grads_i8: no rows");
  OCTO_CHECK_ARG(g_dtype != OCTO_F32 || (V <= kMaxV8 / 2 && n <= kMaxN8 / 2),  // three parts within 32-bit offsets
                 "head_grads_i8: n=%lld, V=%d with fp32 gradients", (long long)n, V);
  OCTO_CHECK_ARG(ldg >= V && (!grad_rows || ld_gr >= d) && (!grad_w || ld_gw >= d), "head_grads_i8: row strides");
  if (!grad_rows && !grad_w) return OCTO_OK;
  OCTO_CHECK_ARG(g && (!grad_rows || (wq && w_scale)) && (!grad_w || (xq && x_scale)), "head_grads_i8: null pointer");
  OCTO_CHECK_ARG((uintptr_t)wq % 16 == 0 && (uintptr_t)xq % 16 == 0 && (uintptr_t)w_scale % 4 == 0 &&
                     (uintptr_t)x_scale % 4 == 0 && (uintptr_t)g % float_bytes(g_dtype) == 0 &&
                     (uintptr_t)grad_rows % float_bytes(gr_dtype) == 0 &&
                     (uintptr_t)grad_w % float_bytes(gw_dtype) == 0 && (uintptr_t)ws % 256 == 0,
                 "head_grads_i8: misaligned pointer");
  const bool as_is = g_as_is(g, ldg, g_dtype, V);
  const Grads8Layout L = grads8_layout(n, d, V, g_dtype, grad_rows != nullptr, grad_w != nullptr, as_is);
  if (!ws || ws_bytes < L.total)
    return octo_fail(OCTO_EWORKSPACE, "head_grads_i8: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, L.total);
  hipStream_t st = (hipStream_t)stream;
  char *wsb = (char *)ws;
  const bool f32 = g_dtype == OCTO_F32;
  Prepare8 p{};
  p.wq = wq;
  p.ldw = ldw;
  p.ws = w_scale;
  const bool wide = grad_rows && !L.few;
  p.wide = wide ? wsb + L.wide : nullptr;
  p.Vr = L.Vr;
  p.dp = (int)L.dp;
  p.xq = xq;
  p.ldxq = ldxq;
  p.xs = x_scale;
  p.xt = grad_w ? wsb + L.xt : nullptr;
  p.ldt = L.parts * L.np;
  p.g = g;
  p.ldg = ldg;
  p.gs = as_is || (!grad_w && (f32 || !wide)) ? nullptr : wsb + L.g;
  p.gh = f32 && wide ? wsb + L.gh : nullptr;
  p.norm = g_dtype == OCTO_F16 && (wide || grad_w) ? (Norm8 *)(wsb + L.norm) : nullptr;
  p.np = L.np;
  p.Vp = L.Vp;
  p.n = n;
  p.d = d;
  p.V = V;
  rc = launch_prepare8(p, g_dtype, st);
  if (rc) return rc;
  if (L.few) {
    const DxSplit s = dx_split(n, d, V, g_dtype);
    const FewDx a{g,        ldg,      wq,      ldw,                      w_scale,   (int)n, d, V,
                  s.strips, s.groups, s.share, (f32x4 *)(wsb + L.split), grad_rows, ld_gr};
    rc = go_few_dx(a, s, g_dtype, gr_dtype, st);
    if (rc) return rc;
  }

  const int dt = f32 ? OCTO_BF16 : g_dtype;
  const char *gs = as_is ? (const char *)g : wsb + L.g;
  const int64_t lds = (as_is ? ldg : L.Vp) * 2;
  StoreArgs oh, ow;
  const Operand Ah = f32 ? operand8(wsb + L.gh, L.Kh * 2, n) : operand8(gs, lds, n);
  const Operand Bh = operand8(wsb + L.wide, L.dp * 2, f32 ? L.Vr : d);
  const GemmShape sh = shape8(n, d, L.Kh), sw = shape8(V, d, f32 ? 3 * L.np : n);
  Operand Aw = operand8(gs, lds, as_is ? n : V);
  const Operand Bw = operand8(wsb + L.xt, L.parts * L.np * 2, d);
  const int kma = as_is ? KM_EDGE : KM_A;
  if (as_is) Aw.extent = (uint32_t)V;
  if (wide) {
    oh.C = grad_rows;
    oh.ldc = ld_gr;
    oh.dtype = gr_dtype;
    oh.alpha = p.norm ? &p.norm->back[0] : nullptr;
    if (L.split_items) {
      oh.split = (float *)(wsb + L.split);
      oh.split_cap = (int)L.split_items;
      oh.split_alone = 1;
    }
  }
  if (grad_w) {
    ow.C = grad_w;
    ow.ldc = ld_gw;
    ow.dtype = gw_dtype;
    ow.alpha = p.norm ? &p.norm->back[1] : nullptr;
  }
  // Both in one launch, dx's runs as long as if it had the card to itself: dW's short tiles follow them on every CU.
  // Two launches take 20 us more up to 700 rows of d 2560, V 151,936 and as long from 1,024 on; runs cut for sharing
  // the card (fewer, longer ones) 949 us for 300 rows against 835.
  const bool both = wide && grad_w && !f32;
  if (both) rc = launch_gemm_grads(dt, Ah, Bh, sh, oh, true, Aw, Bw, sw, ow, st, kma);
  else if (wide) rc = launch_gemm_store(dt, Ah, Bh, sh, oh, st, f32 ? KM_WRAP : KM_B);
  if (!rc && wide) rc = launch_split_sum(sh, oh, false, st);
  if (!rc && grad_w && !both) rc = launch_gemm_store(dt, Aw, Bw, sw, ow, st, kma);
  return rc;
}

}  // extern "C"
