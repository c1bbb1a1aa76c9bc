// kh_paged_attn.cu -- decode attention over a paged packed cache.
//
// Per query row (sequence b, head hq, KV head h = hq / n_q), with
// q~ = H (d_k . q) / sqrt(D) and g = sqrt(2 / pi):
//   s_j = norm_j <q~, c[code_j]> + rnorm_j / sqrt(D) <q~, sign_j>
//   t_j = cap tanh(s_j scale / cap) - slope (len - 1 - j)
//   j in [max(start, len - window), len)
//   out = d_v . H (sum_j p_j (norm'_j / sqrt(D) c[code'_j] + g rnorm'_j / D sign'_j)),
//   p = softmax(t); no row attended: zeros, lse = -inf.
//
// paged_prepare_kernel cuts a call's rows into units of equal length, those of
// the shared prefix (read once for every sequence's queries) before each
// sequence's own; a warp of paged_rows_kernel takes a unit, which may hold pieces
// of several sequences or KV heads.  A piece leaves a record (reference exponent
// m in log2 units, l = sum 2^(t' - m), acc = sum 2^(t' - m) v~ with
// t' = t log2 e) per query row; paged_combine_kernel merges them and leaves the
// transformed domain.  A prefix with many bf16 queries goes to kh_paged_prefix.cu
// instead, a record per query row and chunk.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "kh_common.cuh"
#include "kh_paged_attn.cuh"

namespace kh {
namespace {

// ------------------------------------------------------------------ rows
//
// paged_rows_kernel: both products on mma.sync with 8-bit integers, fed from
// registers, so that a row's bits are never written out as elements.  A packed
// word masked to one bit a byte IS a register of four matrix elements, each 2^b
// or zero; the factor 2^b goes into the other operand or into the
// accumulator's scale.  What bit belongs to what index of the product is free,
// as long as both operands agree:
//   scores  A = 16 rows: lane (g, t) holds word t of rows pi(g) and pi(g) + 8
//           (words 2 t, 2 t + 1 at D = 256).  B = q~.
//   values  A = 16 elements of lane g's halfword (word at D = 256), of rows
//           t, t + 8, t + 4, t + 12 (and 16 more).  B = the weights p norm' and
//           p rnorm', which movmatrix turns from the scores' accumulator
//           layout into the operand's.
// Queries and weights are fixed point, PARTS bytes of them a column each, and
// sums are exact in 32 bits.  Bits count as 0 / 1: sum w sign = 2 sum w bit -
// sum w, whose second sum is a product with ones, exact too (as a float sum of
// 1800 weights it cost fp32 results 2.5e-6 of their norm, now 2.6e-7).
//   PARTS = 2 (16-bit queries, 4 a block of 8 columns): q~ in steps of 2^-15 of
//     its largest element (2^-14 for bits that count twice), weights in steps of
//     2^-16 to 2^-14 (bf16: 2^-12) of the largest of the 128 rows around them.
//   PARTS = 4 (32-bit queries, 2 a block): q~ of 2^-31 to 2^-28, weights of 2^-31 to
//     2^-22.
// A long tail of rows far below a step would count in the softmax's
// denominator and not in its values (a first row with half of the weight before
// 32767 alike ones: 2% off), so
//   - the step follows the weights: every kSpan tiles it comes down to them where
//     they have become small, so that a heavy row costs the 256 rows around it
//     their low bits and no more; and
//   - a lane of 16-bit queries carries what each rounding left into its next
//     row's weight, so that rounded weights sum to the true ones.
// What remains is 0.41 of a step a row, of either sign: 2^-12 of one heavy row.
// Both cost the ragged batch below 3 us.
// What bounds it is the latency of dependent instructions: a 32-row tile takes
// some 730, 340 of them on the ALU at half rate, and 32 products of 7.5 cycles, and
// three warps a scheduler issue on 55% of the cycles.  On a ragged
// batch (32 sequences up to 8192 rows, 8 KV heads x 4, D 128, bf16) the kernel
// takes 44.7 us; as fp16 products, two elements a logic operation, it took 63 us
// when these took 41.  Two column blocks, where a KV head has queries for them,
// take the same masked bits: 16 sequences of 4096 rows, 8 KV heads x 5 bf16
// queries 36.4 us (one block at a time 40.4), x 16 61.9 (72.4), x 3 fp32 queries
// 36.3 (40.2); at D 256 two blocks' sums do not fit the registers.
//
// A warp runs on its own: 32-row tiles in a ring of cp.async stages, one lane
// fetching one row (so pages may end anywhere).  The reference exponent of a
// column moves up when a weight would leave its range, and down as above; the
// sums so far are then folded into floats in shared memory, so that most tiles
// rescale nothing.
// A piece of a unit is at most 16384 rows: 32-bit sums hold those (weights up
// to 255 x 128 each), and what is summed as floats keeps its bits; the next
// piece's record joins in.
constexpr int kWarps = 4;
constexpr int64_t kPieceTiles = 512;
constexpr int kSpan = 4;  // tiles (a power of two)

template <int D>
struct RowsCfg {
  static constexpr int W = D / 32;
  static constexpr int kStages = D == 128 ? 4 : 3;
  static constexpr int kPlane = 32 * W * 4;             // one plane of a tile
  static constexpr int kStage = 4 * kPlane + 512 + 16;  // + norms by row + valid mask
  static constexpr int kRing = kWarps * kStages * kStage;
  // a warp's folded sums: a lane's elements of each block of columns, and
  // {reference, l, sum of the code plane's weights, -}, {that since the last fold, -}
  // and, by column, constants that would take 7 registers a block
  template <int PARTS, int NB>
  static constexpr int kFold = NB * ((W * 4 / (PARTS / 2) + 8) * 32 * 4 + 4 * 32);
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// ---- how a call's rows are split
//
// The tiles of 32 rows of all groups of the call lie one after another: first
// those of the prefix's groups (KV head, block of NQ of every sequence's query
// rows), then for each sequence those of its groups (KV head, block of NQ of
// its own).  They are cut into units of equal length, one for every warp that
// the GPU holds (two to four a warp made more records and measured the same, or
// 119 us instead of 110 on 8 sequences up to 40000 rows).  Lengths live on the
// device, so the cut is made there: units from what max_len allows left a
// quarter of the SM time idle on the ragged batch, CTAs with a chunk of a fixed
// length more.  Tiles and not rows are counted, as a group of one row costs its
// tile (counted by rows, 17 x 4 x 5 queries with one own row each took 560 us),
// and kGap more places a group without anything in them, as starting a piece
// takes a warp about as long as three tiles (without them a warp was left with
// 37 short pieces: 64 x 32 fp16 queries over a prefix of 8192 rows and 32 own
// rows each took 175 us, and 94 with them).
// A unit may hold pieces of several groups; piece (unit u, group G) has record
// u + G, as a unit's or a group's begin starts a new piece.
//
// What the warps need is prepared by a launch before: where each sequence's
// tiles start, its rows, the units, through which sequence the prefix is read,
// and each group's queries as operand fragments.
constexpr int64_t kGap = 3;

// Keys' bits are masked in places 0 .. kPlaces - 1 of each byte, by moving the word
// down: more places save moves and cost the queries bits.  Of 16-bit queries four
// places left fp16 results 2.4e-4 to 2.7e-4 off (of which 2.1e-4 is their own
// rounding), two leave 2.2e-4 to 2.4e-4 for 1 to 4% more time.
template <int PARTS>
constexpr int kPlaces = PARTS == 2 ? 2 : 4;

template <int D, int NB>
struct Frags {  // of a group
  static constexpr int kSteps = D / 32;
  uint2 q[NB * kSteps][32];
  float sum[NB * 4], scale[NB * 4];  // per query: sum of q~ and the exponent's scale
};

// Groups: [0, n_pre) the prefix's, then those of each sequence.
struct Group {
  bool pre;
  int h, z;
  int64_t b;  // sequence (0 for the prefix)
};
__device__ __forceinline__ Group group_of(const AttnParams& P, int64_t i) {
  Group g;
  const int64_t n_pre = (int64_t)P.r.n_kv_heads * P.plan.pre_blocks;
  g.pre = i < n_pre;
  const int blocks = g.pre ? P.plan.pre_blocks : P.plan.own_blocks;
  const int64_t per = (int64_t)P.r.n_kv_heads * blocks, x = g.pre ? i : i - n_pre;
  g.b = g.pre ? 0 : x / per;
  const int hz = (int)(x - g.b * per);
  g.h = hz / blocks;
  g.z = hz - g.h * blocks;
  return g;
}

__device__ __forceinline__ void mma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {  // u8 x s8
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16832_0(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                           uint32_t a3, uint32_t b0, uint32_t b1) {  // from zero
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma16832u(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {  // u8 x u8
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int64_t kFragBytes = 2176;  // of a group's Frags, at most


// Sixteen query rows of a KV head as the tensor-core prefix's operand: element
// e at position 2 (e & 15) + (e >> 4 & 1) of its block of 32, 128-byte blocks
// swizzled; times log_scale and a power of two that brings the row's largest
// under 2^14 (fp16 holds elements 2^28 below that with full steps).
template <int D>
__device__ __forceinline__ void write_query_tiles(const AttnParams& P, int64_t block, int lane,
                                                  int warp) {
  using Q = QueryTiles<D>;
  constexpr int W = D / 32, GROUP = Q::MT * 128;
  const PagedAttnRequest& r = P.r;
  const int64_t n_rows = r.n_seqs * r.n_q, per = (n_rows + GROUP - 1) / GROUP * (GROUP / 16);
  const int h = (int)(block / per);
  const int64_t first = (block - h * per) * 16 + warp * 4;
  uint8_t* group = reinterpret_cast<uint8_t*>(P.queries) +
                   (h * (per / (GROUP / 16)) + first / GROUP) * (int64_t)Q::kGroup;
  float x[4][W];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t i = first + k, b = i / r.n_q;
    const int64_t row = (b * r.n_kv_heads + h) * r.n_q + (i - b * r.n_q);
#pragma unroll
    for (int j = 0; j < W; ++j)
      x[k][j] = i < n_rows ? ld_any(r.q, r.dtype, row * D + 32 * j + lane) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int y = (int)((first + k) % GROUP);
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j)
      if ((r.dk_neg[j] >> lane) & 1) x[k][j] = -x[k][j];
    fwht_lanes<W>(x[k], lane);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      x[k][j] *= P.log_scale;
      mx = fmaxf(mx, fabsf(x[k][j]));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    int e = 14;
    if (mx > 0.f && mx < INFINITY) frexpf(mx, &e);
    const float up = ldexpf(1.f, max(-120, min(120, 14 - e)));
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const int pos = 32 * j + 2 * (lane & 15) + (lane >> 4);
      const int c = (pos & 63) >> 3;
      *reinterpret_cast<__half*>(group + (y >> 7) * Q::kTile + (pos >> 6) * (128 * 128) +
                                 (y & 127) * 128 + ((c ^ (y & 7)) << 4) + (pos & 7) * 2) =
          __float2half_rn(x[k][j] * up);
    }
    if (lane == 0) reinterpret_cast<float*>(group + Q::MT * Q::kTile)[y] = up;
  }
}

// Block 0: starts, own rows, the units.  Then a group each; then, where the
// prefix goes to the tensor cores, sixteen rows of its operand each.
template <int D, int PARTS, int NB>
__global__ void __launch_bounds__(128) paged_prepare_kernel(const __grid_constant__ AttnParams P) {
  using F = Frags<D, NB>;
  constexpr int W = D / 32, KS = F::kSteps, QB = 8 / PARTS, NQ = NB * QB;
  const PagedAttnRequest& r = P.r;
  __shared__ float qs[NQ][D];
  __shared__ int64_t part[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dependency_wait();
  grid_dependents_launch();
  if (blockIdx.x == 0) {
    int64_t base = 0;
    uint64_t best = 0;  // (rows of the prefix, the lower of two sequences) as one number
    for (int64_t b0 = 0; b0 < r.n_seqs; b0 += 128) {
      const int64_t b = b0 + threadIdx.x;
      int64_t n = 0;
      if (b < r.n_seqs) {
        const int64_t len = length_of(P, b), first = own_first(P, b, len);
        best = max(best, (uint64_t)min(len, r.prefix_len) << 32 | (uint64_t)(0xffffffffll - b));
        n = first < len ? (len - first + 31) / 32 + kGap : 0;
        P.own[b] = make_int2((int)min(first, len), (int)len);
      }
      int64_t upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      __syncthreads();
      if (lane == 31) part[warp] = upto;
      __syncthreads();
      int64_t before = base;
      for (int w = 0; w < 4; ++w) {
        if (w < warp) before += part[w];
        base += part[w];
      }
      if (b < r.n_seqs) P.starts[b] = before + upto - n;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
      best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) part[warp] = (int64_t)best;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 4; ++w) best = max(best, (uint64_t)part[w]);
      Units u;
      u.source = 0xffffffffll - (int64_t)(best & 0xffffffffu);
      u.pre_end = (int64_t)(best >> 32);
      P.starts[r.n_seqs] = base;
      const int64_t total =
          r.n_kv_heads * (P.plan.pre_blocks * ((u.pre_end + 31) / 32 + kGap) +
                          base * P.plan.own_blocks);
      u.size = max((int64_t)2, (total + P.n_warps - 1) / P.n_warps);
      u.mul = ~uint64_t(0) / (uint64_t)u.size + 1;
      *P.units = u;
    }
    return;
  }
  const int64_t gi = blockIdx.x - 1;
  if (gi >= P.plan.groups) {
    write_query_tiles<D>(P, gi - P.plan.groups, lane, warp);
    return;
  }
  const Group grp = group_of(P, gi);
  const int64_t y0 = (int64_t)grp.z * NQ;
  const int nq = (int)min((int64_t)NQ, (grp.pre ? r.n_seqs * r.n_q : (int64_t)r.n_q) - y0);
  F* out = reinterpret_cast<F*>(P.frags) + gi;
  for (int y = warp; y < NQ; y += 4) {
    float x[W], mx = 0.f, sum = 0.f;
    const int64_t i = y0 + y, b = grp.pre ? i / r.n_q : grp.b;
    const int64_t row = (b * r.n_kv_heads + grp.h) * r.n_q + (grp.pre ? i - b * r.n_q : i);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float v = y < nq ? ld_any(r.q, r.dtype, row * D + 32 * j + lane) : 0.f;
      x[j] = (r.dk_neg[j] >> lane) & 1 ? -v : v;
    }
    fwht_lanes<W>(x, lane);
#pragma unroll
    for (int j = 0; j < W; ++j) mx = fmaxf(mx, fabsf(x[j]));
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    // whole numbers that PARTS signed bytes hold: 127 x 256 + 127, or 127 x 2^24
    constexpr float kLargest = PARTS == 2 ? 32639.f : 2130706432.f;
    // (at most 2^110, so that its inverse keeps its bits: smaller queries' scores are 0)
    const float up = mx > 0.f && mx < INFINITY ? fminf(kLargest / mx, 0x1p110f) : 1.f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      // element 32 j + lane: its bit counts 2^place times
      const float times = (float)(1 << (lane & (kPlaces<PARTS> - 1)));
      const float v = rintf(x[j] * up / times) * times;
      sum += v;
      qs[y][32 * j + lane] = v;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      out->sum[y] = mx < INFINITY ? sum : NAN;
      out->scale[y] = P.log_scale / up;  // sm_scale log2(e) / sqrt(D) and the scale above
    }
  }
  __syncthreads();
  // column g: byte PARTS - 1 - g % PARTS of query g / PARTS; k = 4 t + j is bit
  // 2 i of byte j of the lane's word, k = 4 t + 16 + j bit 2 i + 1
  const int g = lane >> 2, t = lane & 3;
  for (int k = warp; k < NB * KS; k += 4) {
    const int i = k % KS, y = k / KS * QB + g / PARTS;
    const int word = D == 128 ? t : 2 * t + (i >> 2);
    uint32_t f[2] = {0, 0};
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int bit = 2 * (i & 3) + o;
        int v = (int)qs[y][32 * word + 8 * j + bit] >> (bit & (kPlaces<PARTS> - 1));
        for (int d = PARTS - 1 - g % PARTS; d > 0; --d) v = (v - (((v + 128) & 255) - 128)) >> 8;
        f[o] |= (uint32_t)(v & 255) << (8 * j);
      }
    out->q[k][lane] = make_uint2(f[0], f[1]);
  }
}

// Sequence b with starts[b] * per <= x < starts[b + 1] * per: a warp looks at
// 128 places at once.
__device__ __forceinline__ int64_t find_sequence(const AttnParams& P, int64_t x, int64_t per,
                                                 int lane) {
  int64_t lo = 0, n = P.r.n_seqs;  // it is among [lo, lo + n)
  while (n > 1) {
    const int64_t step = (n + 127) / 128;
    int64_t start[4];
    int below = 0;  // of the places lo + step, lo + 2 step, ... those that are not after x
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t i = lo + (32 * k + lane + 1) * step;
      start[k] = i < lo + n ? P.starts[i] : -1;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      below += __popc(__ballot_sync(0xffffffffu, start[k] >= 0 && start[k] * per <= x));
    lo += below * step;
    n = min(step, n - below * step);
  }
  return lo;
}

// CTAs an SM that the registers are bounded for: three (168 registers), or two where
// a warp's sums would spill then: 16 sequences of 4096 rows, 8 KV heads x 16 bf16
// queries 62.0 us (three: 63.3), 13 x 28 fp16 queries of D 256 over a prefix of 5001 rows
// 44.8 (46.3).  Two elsewhere: ragged batch 48.9 (46.7), long fp32 contexts 131 (112).
constexpr int kMostCtas = 3;
template <int D, int NB>
constexpr int kRowsCtas = D == 128 && NB == 1 ? kMostCtas : 2;

template <int D, int PARTS, bool EXTRA, int NB>
__global__ void __launch_bounds__(32 * kWarps, kRowsCtas<D, NB>)
    paged_rows_kernel(const __grid_constant__ AttnParams P) {
  using C = RowsCfg<D>;
  using F = Frags<D, NB>;
  constexpr int W = C::W;
  constexpr int kStages = C::kStages;
  constexpr int KS = F::kSteps;         // steps of the score product
  constexpr int MT = D / 16;            // element tiles of the value product
  constexpr int QB = 8 / PARTS;         // queries a column block
  constexpr int NQ = NB * QB;
  const PagedAttnRequest& r = P.r;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int mine = PARTS == 2 ? t : t >> 1;   // this lane's query of a block
  const bool low = PARTS == 4 && (t & 1);     // it holds the query's low bytes
  uint8_t* ring = smem + warp * kStages * C::kStage;
  // element x of block nb at [nb * kOwn / 4 + x / 4][lane], then the block's statistics
  constexpr int kOwn = 2 * MT / (PARTS / 2);
  float4* fold4 = reinterpret_cast<float4*>(smem + C::kRing +
                                            warp * C::template kFold<PARTS, NB>) + lane;
  float4* stat4 = fold4 + NB * (kOwn / 4) * 32;
  // {a1, b1, a2, b2}, {slope, first and last row} of the query in block nb's column t
  float4* col4 = stat4 - lane + NB * 64 + 2 * t;
  // Also behind a tensor-core prefix, which starts only when the preparing launch
  // is done: that orders the launches, but only a grid's own wait makes what came
  // before visible to it.  (Own rows beside the prefix's last CTAs without the wait: 64 x 32
  // queries behind a prompt of 8192 rows 42.8 us, with it 44.3.)
  grid_dependency_wait();
  const int64_t pre_end = P.units->pre_end, pre_tiles = (pre_end + 31) / 32;
  const int64_t n_pre = r.n_kv_heads * P.plan.pre_blocks * (pre_tiles + kGap);
  const int64_t per = (int64_t)r.n_kv_heads * P.plan.own_blocks, size = P.units->size;
  const int64_t total = n_pre + P.starts[r.n_seqs] * per;
  const int64_t unit = (int64_t)blockIdx.x * kWarps + warp;
  int64_t at = unit * size;
  const int64_t end = min(at + size, total);
#pragma unroll 1
  while (at < end) {
  // ---- the piece: rows [lo, hi) of a sequence (or of the prefix, for every
  // sequence's queries) for query rows y0 .. y0 + nq of KV head h
  const bool pre = at < n_pre;
  const int64_t b = pre ? P.units->source : find_sequence(P, at - n_pre, per, lane);
  const int64_t start = pre ? 0 : n_pre + P.starts[b] * per;
  const int64_t places = pre ? pre_tiles + kGap : P.starts[b + 1] - P.starts[b];
  const int64_t tiles = places - kGap;
  const int2 all = pre ? make_int2(0, (int)pre_end) : P.own[b];
  const int hz = (int)((at - start) / places);
  const int64_t begin = start + hz * places;
  if (at - begin >= tiles) {  // the gap
    at = begin + places;
    continue;
  }
  const int n_tiles = (int)min(min(tiles - (at - begin), end - at), kPieceTiles);
  const int lo = all.x + 32 * (int)(at - begin);
  const int hi = n_tiles < tiles - (at - begin) ? lo + 32 * n_tiles : all.y;
  const bool more = at > begin && at > unit * size;  // the record holds rows already
  at += n_tiles;
  const int blocks = pre ? P.plan.pre_blocks : P.plan.own_blocks;
  const int h = hz / blocks;
  const int64_t y0 = (int64_t)(hz - h * blocks) * NQ;
  const int nq = (int)min((int64_t)NQ, (pre ? r.n_seqs * r.n_q : (int64_t)r.n_q) - y0);
  const int64_t group = pre ? hz : r.n_kv_heads * P.plan.pre_blocks + b * per + hz;
  const F* frags = reinterpret_cast<const F*>(P.frags) + group;
  auto seq_of = [&](int y) { return pre ? (y0 + y) / r.n_q : b; };
  auto head_of = [&](int y) { return h * r.n_q + (int)(pre ? (y0 + y) % r.n_q : y0 + y); };

  // ---- tiles of 32 rows: lane = row.  Its place in the table and in the page
  // moves on by 32 rows a tile; pages are read a tile before they are used.
  const int32_t* tab = r.table + b * r.table_stride;
  uint32_t block = P.page_div(lo + lane), off = lo + lane - block * r.page_size;
  int left = hi - lo - lane;
  auto take = [&](int& page, uint32_t& place) {
    page = left > 0 ? tab[block] : -1;
    place = off;
    left -= 32;
    block += P.step_blocks;
    off += P.step_off;
    if (off >= (uint32_t)r.page_size) {
      off -= r.page_size;
      ++block;
    }
  };
  auto issue = [&](int tile, int stage, int page, uint32_t place) {
    if (tile < n_tiles) {
      const bool on = (uint32_t)page < (uint32_t)r.n_pages;
      const int64_t row = on ? ((int64_t)page * r.n_kv_heads + h) * r.page_size + place : 0;
      uint8_t* st = ring + stage * C::kStage;
      const uint32_t s = smem_u32(st);
#pragma unroll
      for (int v = 0; v < W / 4; ++v) {
        const uint32_t d = s + lane * W * 4 + v * 16;
        cp_async16(d, r.kp.code + row * W + 4 * v, on);
        cp_async16(d + C::kPlane, r.kp.res + row * W + 4 * v, on);
        cp_async16(d + 2 * C::kPlane, r.vp.code + row * W + 4 * v, on);
        cp_async16(d + 3 * C::kPlane, r.vp.res + row * W + 4 * v, on);
      }
      const uint32_t n = s + 4 * C::kPlane + lane * 16;
      cp_async4(n, r.kp.norms + row, on);
      cp_async4(n + 4, r.kp.rnorms + row, on);
      cp_async4(n + 8, r.vp.norms + row, on);
      cp_async4(n + 12, r.vp.rnorms + row, on);
      const uint32_t mask = __ballot_sync(0xffffffffu, on);
      if (lane == 0) *reinterpret_cast<uint32_t*>(st + 4 * C::kPlane + 512) = mask;
      // rows that there are, and pages that there are not
      const int n_rows = hi - lo - 32 * tile;
      if (mask != (n_rows >= 32 ? 0xffffffffu : (1u << n_rows) - 1u))
        flag_error(P.err, kErrBadIndex);
    }
    cp_commit();
  };
  int next_page;
  uint32_t next_place;
  {
    int pages[kStages - 1];
    uint32_t places[kStages - 1];
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) take(pages[s], places[s]);
    take(next_page, next_place);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s, s, pages[s], places[s]);
  }

  uint2 qf[NB * KS];
#pragma unroll
  for (int i = 0; i < NB * KS; ++i) qf[i] = frags->q[i][lane];

  // ---- constants of this thread's query of each block
  //   t2 = norm (a1 M1 + b1) + rnorm (a2 M2 + b2), M the masked sums
  const float ch = 0.5f * (r.c1 - r.c0), cm = 0.5f * (r.c1 + r.c0);
  const float inv_sd = P.inv_sd;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int y = nb * QB + mine;
    const float k = frags->scale[y], sum = frags->sum[y] * k;
    float slope = 0.f;
    int q_lo = 0, q_hi = 0x7fffffff;
    if (y < nq) {
      if (pre || (EXTRA && r.slopes)) {
        const int64_t len = length_of(P, seq_of(y));
        q_hi = (int)len;
        if (pre) q_lo = (int)min(first_of(P, seq_of(y), len), (int64_t)0x7fffffff);
      }
      if (EXTRA && r.slopes) slope = r.slopes[head_of(y)] * kLog2e;
    }
    if (g == 0) {
      col4[nb * 8] = make_float4(2.f * ch * k, (cm - ch) * sum, 2.f * inv_sd * k, -inv_sd * sum);
      col4[nb * 8 + 1] = make_float4(slope, __int_as_float(q_lo), __int_as_float(q_hi), 0.f);
    }
  }
  // weight 1 as a whole number, and the most one may be
  constexpr float kOne = PARTS == 2 ? 32768.f : 1073741824.f;
  constexpr float kMost = PARTS == 2 ? 65534.f : 4294967040.f;  // and a remainder
  // A span's largest weight that lets the step come down: what that costs is sums
  // being folded, what it saves is noise of 0.41 of a step a row.  fp16 results have
  // no room for it, bf16's own rounding is eight times as large; 32-bit queries'
  // weights are that far from their steps.
  const float fall = kOne * (PARTS == 4 ? 0x1p-8f : r.dtype == KH_BF16 ? 0.125f : 0.5f);
  const float va = ch * inv_sd * kOne;
  const float vb = 0.7978845608028654f * inv_sd * inv_sd * kOne;
  const float cap = r.softcap * kLog2e, inv_cap = r.softcap > 0.f ? 1.f / cap : 0.f;

  // the last tile's rows are all ones: sums of the weights themselves
  float ref[NB];
  float2 l[NB];     // and what its last addition lost (of 32-bit queries)
  float top[NB];    // largest weight since the reference moved, or of the last kSpan tiles
  float2 over[NB];  // what the last roundings left, of either plane
  int acc[NB][MT + 1][4];
  uint32_t folded = 0;  // blocks with sums in shared memory
  const bool uneven = cm != 0.f;  // the levels' middle adds a part of the weights' sum
  // lanes start with remainders spread over a step: what they end with does too
  const float2 over0 = make_float2((2 * g - 7) * 0.0625f, (7 - 2 * g) * 0.0625f);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    ref[nb] = kNoRef;
    l[nb] = make_float2(0.f, 0.f);
    top[nb] = 0.f;
    over[nb] = over0;
    if (uneven) stat4[nb * 64 + 32] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i <= MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[nb][i][k] = 0;
  }
  const int pg = (g >> 1) + 4 * (g & 1);  // pi(g)

  // A tile's scores and a tile's values are independent: in the loop the next
  // tile's scores and exponents run between this tile's value products.
  int s1[2][NB][4], s2[2][NB][4];
  float tt[2][2][NB], ra[2][2], rb[2][2], ee[2][2][NB];
  uint32_t p1[2][NB], p2[2][NB];
  bool full;
  // scores of a tile's two 16-row halves, both planes
  auto scores = [&](const uint8_t* st) {
#pragma unroll
    for (int v = 0; v < W / 4; ++v) {
      uint32_t w[2][2][2];  // half, plane, row
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int rr = 0; rr < 2; ++rr)
            w[hf][p][rr] = reinterpret_cast<const uint32_t*>(
                st + p * C::kPlane)[(16 * hf + pg + 8 * rr) * W + (D == 128 ? t : 2 * t + v)];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        constexpr int kMove = kPlaces<PARTS>;
        if (i && 2 * i % kMove == 0)
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k >> 2][(k >> 1) & 1][k & 1] >>= kMove;
        const uint32_t m0 = 0x01010101u << (2 * i % kMove), m1 = m0 << 1;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const uint2 f = qf[nb * KS + v * 4 + i];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              auto& c = p == 0 ? s1[hf][nb] : s2[hf][nb];
              const uint32_t x0 = w[hf][p][0], x1 = w[hf][p][1];
              if (v == 0 && i == 0) mma16832_0(c, x0 & m0, x1 & m0, x0 & m1, x1 & m1, f.x, f.y);
              else mma16832(c, x0 & m0, x1 & m0, x0 & m1, x1 & m1, f.x, f.y);
            }
        }
      }
    }

  };
  // their exponents without the reference, -inf where nothing is attended
  auto exponents = [&](const uint8_t* st, int j0) {
    const float4* nrm = reinterpret_cast<const float4*>(st + 4 * C::kPlane);
    const uint32_t valid = *reinterpret_cast<const uint32_t*>(st + 4 * C::kPlane + 512);
    full = valid == 0xffffffffu;
    if (pre) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float4 col = col4[nb * 8 + 1];
        full = full && j0 >= __float_as_int(col.y) && j0 + 32 <= __float_as_int(col.z);
      }
      full = __all_sync(0xffffffffu, full);
    }
    // a query's masked sum from its columns' (2 PARTS bytes of them)
    auto joined = [&](const int(&s)[4], int rr) {
      const float x = (float)(s[2 * rr] * 256 + s[2 * rr + 1]);
      if constexpr (PARTS == 2) return x;
      const float y = __shfl_xor_sync(0xffffffffu, x, 1);
      return low ? fmaf(y, 65536.f, x) : fmaf(x, 65536.f, y);
    };
    float4 ab[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) ab[nb] = col4[nb * 8];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        const int row = 16 * hf + pg + 8 * rr;
        const float4 n = nrm[row];
        // NaN for an infinite norm too, whose products with bits of either sign have
        // no sum: a score of minus infinity would count as not attended
        const float nil = fmaf(n.y, 0.f, n.x * 0.f);
        ra[hf][rr] = n.z * va;
        rb[hf][rr] = n.w * vb;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float x = fmaf(n.x, fmaf(ab[nb].x, joined(s1[hf][nb], rr), ab[nb].y), nil);
          x = fmaf(n.y, fmaf(ab[nb].z, joined(s2[hf][nb], rr), ab[nb].w), x);
          if (EXTRA && r.softcap > 0.f)
            x = PARTS == 2 ? soft_cap_16(x, cap, inv_cap) : soft_cap(x, cap, inv_cap);
          if (EXTRA && r.slopes) {
            const float4 col = col4[nb * 8 + 1];
            x = fmaf(col.x, (float)(j0 + row + 1 - __float_as_int(col.z)), x);
          }
          tt[hf][rr][nb] = x;
        }
      }
    if (!full) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int row = 16 * (k >> 1) + pg + 8 * (k & 1), j = j0 + row;
          const float4 col = col4[nb * 8 + 1];
          const bool on = ((valid >> row) & 1) && j >= __float_as_int(col.y) &&
                          j < __float_as_int(col.z);
          if (!on) tt[k >> 1][k & 1][nb] = -INFINITY;
        }
    }
  };
  // weights e = 2^(t2 - ref); true where they fit: a row's larger one decides
  // (and a NaN among the attended, which whole numbers would lose)
  auto weigh = [&](int nb) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = tt[k >> 1][k & 1][nb], e = ex2(x - ref[nb]);
      ee[k >> 1][k & 1][nb] = e;
      const float most = max_nan(max_nan(ra[k >> 1][k & 1], rb[k >> 1][k & 1]), kOne * kLeastNorm);
      // nothing attended: 0 whatever the row's norms hold (but a weight that is
      // only too small to tell from 0 makes NaN of an infinite one)
      top[nb] = max_nan(top[nb], x == -INFINITY ? 0.f : e * most);
    }
    return top[nb] <= kMost;
  };
  // Four elements of a lane's sums, in the order i, k (a lane of 32-bit queries has
  // its k), times `is`.  2 sum w bit - sum w, bit i counting 2^(i & 7) times: the
  // difference is taken in whole numbers, it is small beside its parts.
  auto sums = [&](int nb, int x, float is, float (&v)[4]) {
    const int c0 = acc[nb][MT][0], c1 = acc[nb][MT][1];
    auto element = [&](int i, int k) {
      const int h = acc[nb][i][2 * k], o = acc[nb][i][2 * k + 1];
      const float fh = (float)(2 * h - (c0 << (i & 7))), fo = (float)(2 * o - (c1 << (i & 7)));
      float x = PARTS == 2 || low ? fmaf(fh, 256.f, fo) : fmaf(fh, 16777216.f, fo * 65536.f);
      if (PARTS == 4) x += __shfl_xor_sync(0xffffffffu, x, 1);
      return x * (is * (1.f / (float)(1 << (i & 7))));
    };
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      if constexpr (PARTS == 2) {
        v[y] = element((x + y) >> 1, y & 1);
      } else {
        const float v0 = element(x + y, 0), v1 = element(x + y, 1);
        v[y] = t & 1 ? v1 : v0;
      }
    }
  };
  // A block's reference, l and sum of the code plane's weights, with what is in
  // shared memory; `was` and `is` scale that and the sums in registers.
  auto totals = [&](int nb, float& was, float& is) {
    float4 now = make_float4(ref[nb], l[nb].x + l[nb].y, uneven ? stat4[nb * 64 + 32].x : 0.f, 0.f);
    was = 0.f;
    is = 1.f;
    if ((folded >> nb) & 1) {
      const float4 old = stat4[nb * 64];
      now.x = fmaxf(old.x, ref[nb]);
      was = ex2(old.x - now.x);
      is = ex2(ref[nb] - now.x);
      now.y = fmaf(old.y, was, now.y * is);
      now.z = fmaf(old.z, was, now.z * is);
    }
    return now;
  };
  // What has been summed joins the sums in shared memory.
  auto fold = [&](int nb) {
    float was, is;
    stat4[nb * 64] = totals(nb, was, is);
    if (uneven) stat4[nb * 64 + 32] = make_float4(0.f, 0.f, 0.f, 0.f);
    l[nb] = make_float2(0.f, 0.f);
#pragma unroll
    for (int x = 0; x < kOwn; x += 4) {
      float v[4];
      sums(nb, x, is, v);
      float4* to = fold4 + (nb * (kOwn / 4) + x / 4) * 32;
      if ((folded >> nb) & 1) {
        const float4 sum = *to;
        v[0] = fmaf(sum.x, was, v[0]);
        v[1] = fmaf(sum.y, was, v[1]);
        v[2] = fmaf(sum.z, was, v[2]);
        v[3] = fmaf(sum.w, was, v[3]);
      }
      *to = make_float4(v[0], v[1], v[2], v[3]);
    }
    folded |= 1u << nb;
#pragma unroll
    for (int i = 0; i <= MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[nb][i][k] = 0;
  };
  // the reference moves down by as much, or up to the tile's largest
  auto refer = [&](int nb, float down) {
    float mx = kNoRef;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float most = max_nan(max_nan(ra[k >> 1][k & 1], rb[k >> 1][k & 1]), kOne * kLeastNorm);
      const float x = tt[k >> 1][k & 1][nb];
      if (x > -INFINITY) mx = max_nan(mx, x + lg2(most * (1.f / kOne)));
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (!(mx < INFINITY)) l[nb].x = NAN;  // a norm that is not finite has no average
    ref[nb] = fmaxf(ref[nb] - down, mx);
    if (PARTS == 4) ref[nb] = ceilf(ref[nb]);  // then factors between references are exact
    over[nb] = over0;
    top[nb] = 0.f;
  };
  // sum + x, its rounding in the next one: thousands of alike small weights
  // behind a large one lose the same part of each, 1e-5 of fp32 results (of a piece
  // of 16384 rows 2^-15 at most, which 16-bit results are left with)
  auto add = [](float2& sum, float x) {
    const float y = x + sum.y, to = sum.x + y;
    sum = make_float2(to, y - (to - sum.x));
  };
  auto pack = [&] {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float sum = (ee[0][0][nb] + ee[0][1][nb]) + (ee[1][0][nb] + ee[1][1][nb]);
      if (PARTS == 4) add(l[nb], sum);
      else l[nb].x += sum;
      float w1s = 0.f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t u1[2], u2[2];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const float e = ee[hf][rr][nb];
          const bool none = !full && tt[hf][rr][nb] == -INFINITY;
          if constexpr (PARTS == 2) {
            // 1.5 2^23 + w: the low bits are w as a whole number
            const float2 big = make_float2(12582912.f, 12582912.f);
            float2 x = __ffma2_rn(make_float2(e, e), make_float2(ra[hf][rr], rb[hf][rr]), over[nb]);
            if (none) x = over[nb];  // rounds to 0, as it is half a step at most
            const float2 w = __fadd2_rn(x, big);
            over[nb] = __fadd2_rn(__fadd2_rn(big, make_float2(-w.x, -w.y)), x);
            if (uneven) w1s += w.x - big.x;
            u1[rr] = __float_as_uint(w.x);
            u2[rr] = __float_as_uint(w.y);
          } else {
            const float x1 = none ? 0.f : e * ra[hf][rr], x2 = none ? 0.f : e * rb[hf][rr];
            w1s += x1;
            u1[rr] = __float2uint_rn(x1);
            u2[rr] = __float2uint_rn(x2);
          }
        }
        // this lane's two columns, high byte first, of both rows
        const uint32_t sel = PARTS == 2 || low ? 0x4051u : 0x6273u;
        p1[hf][nb] = transpose8(__byte_perm(u1[0], u1[1], sel));
        p2[hf][nb] = transpose8(__byte_perm(u2[0], u2[1], sel));
      }
      if (uneven) {
        float4 sum = stat4[nb * 64 + 32];
        float2 two = make_float2(sum.x, sum.y);
        add(two, w1s);
        stat4[nb * 64 + 32] = make_float4(two.x, two.y, 0.f, 0.f);
      }
    }
  };
  auto values = [&](const uint8_t* st, int p) {
    const auto& ones = p == 0 ? p1 : p2;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      mma16832u(acc[nb][MT], 0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u, ones[0][nb],
                ones[1][nb]);
    uint32_t x[2][W / 4], y[2][W / 4];  // even and odd bytes of four rows, by half
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint32_t* pl = reinterpret_cast<const uint32_t*>(st + (2 + p) * C::kPlane) +
                           (16 * hf + t) * W + (D == 128 ? g >> 1 : g);
      const uint32_t r0 = pl[0], r1 = pl[8 * W], r2 = pl[4 * W], r3 = pl[12 * W];
#pragma unroll
      for (int v = 0; v < W / 4; ++v) {
        const uint32_t sel = (D == 128 ? (g & 1) : v) ? 0x7362u : 0x5140u;
        const uint32_t a = __byte_perm(r0, r1, sel), b = __byte_perm(r2, r3, sel);
        x[hf][v] = __byte_perm(a, b, 0x5410);
        y[hf][v] = __byte_perm(a, b, 0x7632);
      }
    }
#pragma unroll
    for (int v = 0; v < W / 4; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t m = 0x01010101u << i;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const auto& f = p == 0 ? p1 : p2;
          mma16832u(acc[nb][8 * v + i], x[0][v] & m, y[0][v] & m, x[1][v] & m, y[1][v] & m,
                    f[0][nb], f[1][nb]);
        }
      }
  };
  // weights of tile i, with the reference where it should be
  auto settle = [&](int i) {
    float down[NB] = {};
    uint32_t move = 0;  // blocks of which one does
    if (i != 0 && (i & (kSpan - 1)) == 0) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
          top[nb] = max_nan(top[nb], __shfl_xor_sync(0xffffffffu, top[nb], o));
        // weights like the last ones leave a bit, and one more that kMost has
        if (top[nb] <= fall && top[nb] > 0.f) {
          down[nb] = -1.f - lg2(top[nb] * (1.f / kOne));
          move |= 1u << nb;
        }
        top[nb] = 0.f;
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      if (!weigh(nb)) move |= 1u << nb;
    move = __reduce_or_sync(0xffffffffu, move);
    if (move) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        if ((move >> nb) & 1) {
          if (i != 0) fold(nb);
          refer(nb, down[nb]);
          weigh(nb);
        }
    }
    pack();
  };

  cp_wait<kStages - 2>();
  __syncwarp();
  scores(ring);
  exponents(ring, lo);
  settle(0);
  int stage = 0;
#pragma unroll 1
  for (int tile = 0; tile + 1 < n_tiles; ++tile) {
    const uint8_t* st = ring + stage * C::kStage;
    issue(tile + kStages - 1, stage == 0 ? kStages - 1 : stage - 1, next_page, next_place);
    take(next_page, next_place);
    stage = stage == kStages - 1 ? 0 : stage + 1;
    cp_wait<kStages - 2>();
    __syncwarp();
    const uint8_t* next = ring + stage * C::kStage;
    scores(next);
    values(st, 0);
    exponents(next, lo + (tile + 1) * 32);
    values(st, 1);
    settle(tile + 1);
    __syncwarp();
  }
  values(ring + stage * C::kStage, 0);
  values(ring + stage * C::kStage, 1);
  cp_wait<0>();
  __syncwarp();

  // ---- the record: 16 consecutive elements a lane (32 at D = 256), tile i's
  // parts elements i and 8 + i of each 16
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float fold_was, fold_is;
    float4 now = totals(nb, fold_was, fold_is);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      now.y += __shfl_xor_sync(0xffffffffu, now.y, o);
      now.z += __shfl_xor_sync(0xffffffffu, now.z, o);
    }
    const int y = nb * QB + mine;
    float* rec = P.records + ((unit + group) * NQ + y) * (int64_t)(D + 2);
    float is = 1.f / kOne, was = 0.f;
    if (more && y < nq) {  // joins the record
      const float2 old = *reinterpret_cast<const float2*>(rec);
      const float to = fmaxf(old.x, now.x), f = ex2(now.x - to);
      now.x = to;
      is *= f;
      was = ex2(old.x - to);
      now.y = fmaf(now.y, f, old.y * was);
    }
    __syncwarp();
    if (y < nq && g == 0 && !low) *reinterpret_cast<float2*>(rec) = make_float2(now.x, now.y);
    const float base = (cm / ch) * now.z;
    const int e0 = 2 + (D == 128 ? 16 : 32) * g;
    auto put = [&](int i, int k, float v0, float v1) {  // elements i and i + 1
      float2 v = make_float2((v0 + base) * is, (v1 + base) * is);
      float2* at2 = reinterpret_cast<float2*>(rec + e0 + 16 * (i >> 3) + 8 * k + (i & 7));
      if (more) v = make_float2(fmaf(at2->x, was, v.x), fmaf(at2->y, was, v.y));
      *at2 = v;
    };
#pragma unroll
    for (int x = 0; x < kOwn; x += 4) {
      float v[4];
      sums(nb, x, fold_is, v);
      if ((folded >> nb) & 1) {
        const float4 sum = fold4[(nb * (kOwn / 4) + x / 4) * 32];
        v[0] = fmaf(sum.x, fold_was, v[0]);
        v[1] = fmaf(sum.y, fold_was, v[1]);
        v[2] = fmaf(sum.z, fold_was, v[2]);
        v[3] = fmaf(sum.w, fold_was, v[3]);
      }
      if (y >= nq) continue;
      if constexpr (PARTS == 2) {
        put(x >> 1, 0, v[0], v[2]);
        put(x >> 1, 1, v[1], v[3]);
      } else {
        put(x, t & 1, v[0], v[1]);
        put(x + 2, t & 1, v[2], v[3]);
      }
    }
  }
  __syncwarp();
  }
  grid_dependents_launch();
}

// A block per query row: its records merged, back from the transformed
// domain, divided by l, in the query's type.  What it takes is the time of a
// few dependent steps, so that a warp takes four records at once.  4 warps; 8 or
// 16 where there are so few query rows that the GPU holds them (a row of a long
// cache has a hundred records).
constexpr int kMostJoin = 16;
template <int D>
__global__ void __launch_bounds__(32 * kMostJoin, D == 128 ? 3 : 2)
    paged_combine_kernel(const __grid_constant__ AttnParams P) {
  constexpr int J = D / 32, U = 4;
  const PagedAttnRequest& r = P.r;
  __shared__ float sums[kMostJoin][D], tops[kMostJoin], ls[kMostJoin];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int hq_all = r.n_kv_heads * r.n_q;
  const uint32_t row = blockIdx.x;
  const uint32_t b = row / hq_all;
  const int hq = (int)(row - b * hq_all), h = hq / r.n_q, y = hq - h * r.n_q;
  constexpr int64_t kRec = D + 2;
  const int64_t stride = P.plan.block * kRec;
  grid_dependency_wait();
  // record 0 and how many there are of the prefix, and of the sequence's own rows
  struct Run {
    const float* at;
    int n;
  };
  auto run = [&](int64_t begin, int64_t tiles, int64_t group, int place) {
    if (tiles <= 0) return Run{P.records, 0};
    const int64_t u = P.units->of(begin);
    return Run{P.records + (u + group) * stride + place * kRec,
               (int)(P.units->of(begin + tiles - 1) - u) + 1};
  };
  Run pre{P.records, 0}, own{P.records, 0};
  int64_t pre_stride = stride;
  const int64_t pre_tiles = P.plan.groups > 0 ? (P.units->pre_end + 31) / 32 : 0;
  if (P.plan.pre_chunks) {
    pre = Run{r.workspace + (int64_t)row * P.plan.pre_chunks * kRec, P.plan.pre_chunks};
    pre_stride = kRec;
  } else if (P.plan.pre_blocks) {
    const uint32_t i = b * r.n_q + y, z = i / P.plan.block;
    const int64_t group = (int64_t)h * P.plan.pre_blocks + z;
    pre = run(group * (pre_tiles + kGap), pre_tiles, group, i - z * P.plan.block);
  }
  if (P.plan.own_blocks) {
    const int64_t first = P.starts[b], places = P.starts[b + 1] - first;
    const int z = y / P.plan.block, hz = h * P.plan.own_blocks + z;
    const int64_t per = (int64_t)r.n_kv_heads * P.plan.own_blocks;
    own = run(r.n_kv_heads * P.plan.pre_blocks * (pre_tiles + kGap) + first * per + hz * places,
              places - kGap, r.n_kv_heads * P.plan.pre_blocks + b * per + hz, y - z * P.plan.block);
  }
  const int n = pre.n + own.n;
  float mx = -INFINITY, l = 0.f, a[J];
#pragma unroll
  for (int j = 0; j < J; ++j) a[j] = 0.f;
  for (int p0 = warp; p0 < n; p0 += warps * U) {
    float2 ml[U];
    float v[U][J];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(p0 + warps * u, n - 1);
      const float* q = i < pre.n ? pre.at + i * pre_stride : own.at + (i - pre.n) * stride;
      ml[u] = *reinterpret_cast<const float2*>(q);
#pragma unroll
      for (int j = 0; j < J; j += 2) {  // elements 32 j + 2 lane and the next
        const float2 two = *reinterpret_cast<const float2*>(q + 2 + 32 * j + 2 * lane);
        v[u][j] = two.x;
        v[u][j + 1] = two.y;
      }
    }
    float top = mx;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p0 + warps * u >= n) ml[u].y = 0.f;
      if (ml[u].y != 0.f) top = fmaxf(top, ml[u].x);  // else nothing was attended there
    }
    if (top == -INFINITY) continue;
    const float old = ex2(mx - top);
    mx = top;
    l *= old;
#pragma unroll
    for (int j = 0; j < J; ++j) a[j] *= old;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ml[u].y != 0.f) {
        const float f = ex2(ml[u].x - top);
        l = fmaf(ml[u].y, f, l);
#pragma unroll
        for (int j = 0; j < J; ++j) a[j] = fmaf(v[u][j], f, a[j]);
      }
  }
#pragma unroll
  for (int j = 0; j < J; ++j) sums[warp][32 * j + lane] = a[j];
  if (lane == 0) {
    tops[warp] = mx;
    ls[warp] = l;
  }
  __syncthreads();
  if (warp) return;
  float top = tops[0];
  for (int w = 1; w < warps; ++w) top = fmaxf(top, tops[w]);
  l = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) a[j] = 0.f;
#pragma unroll 4
  for (int w = 0; w < warps; ++w) {
    if (tops[w] == -INFINITY) continue;
    const float f = ex2(tops[w] - top);
    l = fmaf(ls[w], f, l);
#pragma unroll
    for (int j = 0; j < J; ++j) a[j] = fmaf(sums[w][32 * j + lane], f, a[j]);
  }
  fwht_lanes<J>(a, lane);
  const float inv = 1.f / l;
  char* out = static_cast<char*>(r.out) + (int64_t)row * D * (r.dtype == KH_F32 ? 4 : 2);
#pragma unroll
  for (int j = 0; j < J; j += 2) {
    const int e = 32 * j + 2 * lane;
    const uint32_t neg = r.dv_neg[e >> 5] >> (e & 31);
    float2 v = l == 0.f ? make_float2(0.f, 0.f) : make_float2(a[j] * inv, a[j + 1] * inv);
    if (neg & 1) v.x = -v.x;
    if (neg & 2) v.y = -v.y;
    st_any(out, r.dtype, e, v.x);
    st_any(out, r.dtype, e + 1, v.y);
  }
  if (r.lse && lane == 0) r.lse[row] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
}

template <int D, int PARTS, bool EXTRA, int NB>
kh_status launch_rows(AttnParams P, cudaStream_t stream) {
  const PagedAttnRequest& r = P.r;
  constexpr int NQ = NB * 8 / PARTS;
  constexpr int kSmem = RowsCfg<D>::kRing + kWarps * RowsCfg<D>::template kFold<PARTS, NB>;
  static_assert(kRowsCtas<D, NB> * (kSmem + 1024) <= 233472, "shared memory of an SM");
  auto kern = paged_rows_kernel<D, PARTS, EXTRA, NB>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KH_ECUDA;
  static std::once_flag once[64];
  static int ctas[64];  // that fit an SM
  std::call_once(once[dev & 63], [&] {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas[dev & 63], kern, 32 * kWarps, kSmem) !=
        cudaSuccess)
      ctas[dev & 63] = 0;
  });
  constexpr int kGroup = 128 * QueryTiles<D>::MT;
  // the preparing launch's blocks, and the rows launch's
  const int64_t operand =
      P.pre_tensor ? r.n_kv_heads * ((r.n_seqs * r.n_q + kGroup - 1) / kGroup) * (kGroup / 16) : 0;
  const int64_t groups = P.plan.groups;
  if (P.plan.block != NQ || groups + operand > 0x7ffffff0ll || P.plan.tiles >= int64_t(1) << 36)
    return KH_EINVAL;
  const int64_t grid = std::min<int64_t>(
      (int64_t)std::min(std::max(1, ctas[dev & 63]), kRowsCtas<D, NB>) * sm_count(),
      (P.plan.tiles / 2 + kWarps) / kWarps);
  P.n_warps = grid * kWarps;
  static_assert(sizeof(Frags<D, NB>) <= kFragBytes, "workspace of the fragments");
  if (groups + operand > 0 &&
      launch_programmatic(paged_prepare_kernel<D, PARTS, NB>, dim3((unsigned)(groups + operand + 1)),
                          dim3(128), 0, stream, P) != cudaSuccess)
    return KH_ELAUNCH;
  if (P.pre_tensor) {
    const kh_status st = launch_paged_prefix(P, stream);
    if (st != KH_OK) return st;
  }
  if (P.plan.tiles > 0) {
    if (launch_programmatic(kern, dim3((unsigned)grid), dim3(32 * kWarps), kSmem, stream, P) !=
        cudaSuccess)
      return KH_ELAUNCH;
  }
  const int64_t rows = r.n_seqs * r.n_kv_heads * r.n_q;
  if (rows > 0x7fffffffll) return KH_EINVAL;
  const int join = rows <= sm_count() ? kMostJoin : rows <= 4 * sm_count() ? 8 : 4;
  return launch_programmatic(paged_combine_kernel<D>, dim3((unsigned)rows), dim3(32 * join), 0,
                             stream, P) == cudaSuccess
             ? KH_OK
             : KH_ELAUNCH;
}

template <int D>
kh_status launch_dim(const AttnParams& P, cudaStream_t stream) {
  const PagedAttnRequest& r = P.r;
  constexpr int kTwo = D == 128 ? 2 : 1;
  const bool extra = r.softcap > 0.f || r.slopes;
  auto go = [&](auto parts, auto with) {
    constexpr int kParts = decltype(parts)::value;
    return P.plan.block > 8 / kParts ? launch_rows<D, kParts, decltype(with)::value, kTwo>(P, stream)
                           : launch_rows<D, kParts, decltype(with)::value, 1>(P, stream);
  };
  using std::integral_constant;
  const kh_status st =
      r.dtype == KH_F32
          ? (extra ? go(integral_constant<int, 4>{}, std::true_type{})
                   : go(integral_constant<int, 4>{}, std::false_type{}))
          : (extra ? go(integral_constant<int, 2>{}, std::true_type{})
                   : go(integral_constant<int, 2>{}, std::false_type{}));
  if (st != KH_OK) return st;
  return cudaGetLastError() == cudaSuccess ? KH_OK : KH_ELAUNCH;
}

}  // namespace

// Above how many query rows a KV head's prefix goes to the tensor cores: their
// products have 128 query rows whatever there are, the rows kernel's time grows
// with them.  Measured (us, rows kernel / tensor cores, 8 KV heads, bf16):
//                 16 rows      32           48           64           128
//   D 128, 1024   14.7 / 17.4  15.8 / 17.6  16.8 / 18.7  17.8 / 18.6  20.9 / 18.4
//   D 128, 8192   21.8 / 31.8  26.7 / 30.7  32.4 / 31.7  37.7 / 30.8  59.4 / 30.5
//   D 256, 1024   16.5 / 19.9  17.3 / 20.1  19.1 / 21.0  21.3 / 20.5  28.1 / 20.6
//   D 256, 8192   26.3 / 34.4  37.5 / 34.2  49.6 / 35.5  61.8 / 34.5   109 / 33.1
// (Of one KV head and 1024 rows the rows kernel stays ahead up to 128 query
// rows, by 2 us at D 128 and 2 to 5 us at D 256.)
int64_t prefix_tensor_rows(int D) { return D == 128 ? 32 : 16; }

// The workspace, each part 16-byte aligned: a tensor-core prefix's records, by
// query row and chunk; the other records; the sequences' starts and own rows;
// the units; the groups' fragments; a tensor-core prefix's queries.
struct Layout {
  int64_t records, starts, own, units, frags, queries, bytes;
};
Layout layout_of(const PagedPlan& p, int64_t n_seqs, int n_q, int n_kv_heads, int D) {
  auto up = [](int64_t x) { return (x + 15) / 16 * 16; };
  const int64_t nq = n_seqs * n_q, record = (D + 2) * 4;
  Layout l;
  l.records = up(nq * n_kv_heads * p.pre_chunks * record);
  l.starts = l.records + up((p.max_units + p.groups) * p.block * record);
  l.own = l.starts + up((n_seqs + 1) * 8);
  l.units = l.own + up(n_seqs * 8);
  l.frags = l.units + up(sizeof(Units));
  l.queries = l.frags + p.groups * kFragBytes;
  l.bytes = l.queries;
  if (p.pre_chunks > 0)
    l.bytes += D == 128 ? (nq + 255) / 256 * n_kv_heads * QueryTiles<128>::kGroup
                        : (nq + 127) / 128 * n_kv_heads * QueryTiles<256>::kGroup;
  return l;
}
int64_t paged_workspace_bytes(const PagedPlan& p, int64_t n_seqs, int n_q, int n_kv_heads, int D) {
  return p.pre_chunks || p.groups ? layout_of(p, n_seqs, n_q, n_kv_heads, D).bytes : 0;
}

PagedPlan paged_plan(int64_t n_seqs, int n_q, int n_kv_heads, int D, int64_t max_len,
                     int64_t prefix_len, int64_t window, int dtype, int n_sms) {
  PagedPlan p;
  const int64_t pre = std::min(prefix_len, max_len), nq = n_seqs * n_q;
  p.own_rows = max_len - pre;
  if (window > 0) p.own_rows = std::min(p.own_rows, window);
  // the prefix's chunks on the tensor cores: one round of CTAs, one an SM, in
  // whole tiles; more where they would be long, as every 16 rows' sum is truncated
  // to the sums so far: beside a heavy row 131072 alike ones came out 0.6% short,
  // 16384 cost 2^-13 of the result at most (256 such chunks, so that records stay
  // a small part of what a prefix of millions of rows takes)
  if (pre > 0 && nq > prefix_tensor_rows(D) && dtype == KH_BF16) {
    const int64_t each = D == 128 ? 256 : 128, tile = D == 128 ? 128 : 64;
    const int64_t ctas = std::max<int64_t>(std::min<int64_t>((pre + 16383) / 16384, 256),
                                           n_sms / (n_kv_heads * ((nq + each - 1) / each)));
    p.chunk_rows = ((pre + ctas - 1) / ctas + tile - 1) / tile * tile;
    p.pre_chunks = (int)((pre + p.chunk_rows - 1) / p.chunk_rows);
  } else {
    p.pre_rows = pre;
  }
  // a column block's queries, or two blocks' where there are queries for them
  const int64_t most = p.pre_rows > 0 ? nq : n_q, one = dtype == KH_F32 ? 2 : 4;
  p.block = (int)(D == 128 && most > one ? 2 * one : one);
  if (p.pre_rows > 0) p.pre_blocks = (int)((nq + p.block - 1) / p.block);
  if (p.own_rows > 0) p.own_blocks = (n_q + p.block - 1) / p.block;
  p.groups = n_kv_heads * (p.pre_blocks + n_seqs * p.own_blocks);
  p.tiles = n_kv_heads * (p.pre_blocks * ((p.pre_rows + 31) / 32 + kGap) +
                          n_seqs * p.own_blocks * ((p.own_rows + 31) / 32 + kGap));
  p.max_units = std::min<int64_t>((int64_t)kMostCtas * kWarps * n_sms, p.tiles / 2 + 1);
  return p;
}

kh_status launch_paged_attn(const PagedAttnRequest& r, cudaStream_t stream) {
  AttnParams P{};
  P.r = r;
  P.plan = paged_plan(r.n_seqs, r.n_q, r.n_kv_heads, r.D, r.max_len, r.prefix_len, r.window,
                      r.dtype, sm_count());
  const double sd = std::sqrt((double)r.D);
  P.log_scale = (float)(r.sm_scale * 1.4426950408889634 / sd);
  P.inv_sd = (float)(1.0 / sd);
  int bits = 0;
  while ((int64_t(1) << bits) < r.page_size) ++bits;
  P.div_shift = 31 + bits;
  P.div_mul = ((uint64_t(1) << P.div_shift) + r.page_size - 1) / r.page_size;
  P.step_blocks = 32 / r.page_size;
  P.step_off = 32 % r.page_size;
  P.pre_tensor = P.plan.pre_chunks > 0;
  const Layout l = layout_of(P.plan, r.n_seqs, r.n_q, r.n_kv_heads, r.D);
  uint8_t* ws = reinterpret_cast<uint8_t*>(r.workspace);
  P.starts = reinterpret_cast<int64_t*>(ws + l.starts);
  P.own = reinterpret_cast<int2*>(ws + l.own);
  P.units = reinterpret_cast<Units*>(ws + l.units);
  P.records = reinterpret_cast<float*>(ws + l.records);
  P.frags = ws + l.frags;
  P.queries = reinterpret_cast<uint16_t*>(ws + l.queries);
  P.err = device_error_ptr();
  return r.D == 128 ? launch_dim<128>(P, stream) : launch_dim<256>(P, stream);
}

}  // namespace kh
