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
// The rows of a call are cut into chunks of equal length: first those of the
// shared prefix, which one CTA reads for every sequence, then each sequence's
// own.  A chunk leaves a record (reference exponent m in log2 units,
// l = sum 2^(t' - m), acc = sum 2^(t' - m) v~ with t' = t log2 e) per query
// row; paged_combine_kernel merges them and leaves the transformed domain.
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
// paged_rows_kernel: both products on mma.sync, fed from registers, so that a
// row's bits are never written out as elements.  A packed word masked to one
// bit a byte (or halfword) IS a register of matrix elements, each 2^b or zero
// (8-bit integers), or 2^(b - 24) or zero (fp16, subnormal): one logic
// operation makes four elements, or two.  The factor 2^b goes into the other
// operand or into the accumulator's scale.  What bit belongs to what index of
// the product is free, as long as both operands agree:
//   scores  A = 16 rows: lane (g, t) holds word t of rows pi(g) and pi(g) + 8
//           (words 2 t, 2 t + 1 at D = 256).  B = q~, a query in two columns.
//   values  A = 16 elements of lane g's halfword (word at D = 256), of rows
//           t, t + 4, t + 8, t + 12 (and 16 more).  B = the weights p norm' and
//           p rnorm', which movmatrix turns from the scores' accumulator
//           layout into the operand's.
// A query's (and a weight's) two columns are its high and low part:
//   I8    (16-bit queries) 16-bit fixed point in two bytes, sums exact in 32-bit
//         integers.  q~ keeps 2^-13 of its largest element (2^-16 for three
//         bits of four), a weight 2^-16 of the largest of its unit, whose
//         rounding errors average out; together under a tenth of a bf16 step.
//         Bits count as 0 / 1: sum w sign = 2 sum w bit - sum w, exactly.
//   else  (32-bit queries) two fp16 parts of 11 bits, the second times 2^11.
//         There the difference would cost bits, so values move their bits
//         to the sign of +-1, one more shift each.
// Measured on the ragged batch (32 sequences up to 8192, 8 x 4 heads): fp16
// parts for bf16 queries 25 instructions a row, 63 us.
//
// A warp runs on its own: 32-row tiles in a ring of cp.async stages, one lane
// fetching one row (so pages may end anywhere).  The reference exponent of a
// column moves only when a weight would leave its type's range, so most tiles
// rescale nothing.
constexpr int kWarps = 4;

template <int D>
struct RowsCfg {
  static constexpr int W = D / 32;
  static constexpr int kStages = D == 128 ? 4 : 3;
  static constexpr int kPlane = 32 * W * 4;             // one plane of a tile
  static constexpr int kStage = 4 * kPlane + 512 + 16;  // + norms by row + valid mask
  static constexpr int kRing = kWarps * kStages * kStage;
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
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- how a call's rows are split
//
// All (group, row) pairs of the call lie one after another: first the prefix's
// groups (KV head, block of NQ of every sequence's query rows), then for each
// sequence its groups (KV head, block of NQ of its own).  They are cut into
// units of equal length, which the warps claim one by one: lengths live on the
// device, and neither CTAs with a chunk of a fixed length nor equal ranges per
// CTA kept the GPU busy to the end (an SM's CTAs progress unevenly, and one
// left alone runs at a third of the SM's rate).  A unit may hold pieces of
// several groups; a group has a record slot for every unit it touches.
//
// What the claims need is prepared by a launch before: where each sequence's
// pairs start, its first row, the claim counter, and each group's queries as
// operand fragments.
template <int D, bool I8, int NB>
struct Frags {  // of a group
  static constexpr int kSteps = D / (I8 ? 32 : 16);
  uint2 q[NB * kSteps][32];
  float sum[NB * 4], scale[NB * 4];  // per query: sum of q~ and the exponent's scale
};

// Groups: [0, n_pre) the prefix's, then those of each sequence.
struct Group {
  bool pre;
  int h, z;
  int64_t b;  // sequence whose table is read
};
__device__ __forceinline__ Group group_of(const AttnParams& P, int64_t i) {
  Group g;
  const int64_t n_pre = (int64_t)P.r.n_kv_heads * P.pre_blocks;
  g.pre = i < n_pre;
  const int blocks = g.pre ? P.pre_blocks : P.own_blocks;
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

constexpr int64_t kFragBytes = 4352;  // of a group's Frags, at most

constexpr float kPart = 2048.f;      // second fp16 parts are stored times 2^11

// Block 0: starts, first rows, the counter.  The others: a group each.
template <int D, bool I8, int NB>
__global__ void __launch_bounds__(128) paged_prepare_kernel(const __grid_constant__ AttnParams P) {
  using F = Frags<D, I8, NB>;
  constexpr int W = D / 32, KS = F::kSteps, NQ = NB * 4;
  const PagedAttnRequest& r = P.r;
  __shared__ float qs[NQ][D];
  __shared__ int64_t part[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dependency_wait();
  grid_dependents_launch();
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *P.next_unit = 0u;
    int64_t base = 0;
    for (int64_t b0 = 0; b0 < r.n_seqs; b0 += 128) {
      const int64_t b = b0 + threadIdx.x;
      int64_t n = 0;
      if (b < r.n_seqs) {
        const int64_t len = length_of(P, b), first = own_first(P, b, len);
        n = max((int64_t)0, len - first);
        P.first_row[b] = (int32_t)min(first, (int64_t)0x7fffffff);
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
    if (threadIdx.x == 0) P.starts[r.n_seqs] = base;
    return;
  }
  const int64_t gi = blockIdx.x - 1;
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
    float up;
    if constexpr (I8) {
      // whole numbers up to 32639 = 127 x 256 + 127 where a bit counts once
      up = mx > 0.f && mx < INFINITY ? 32639.f / mx : 1.f;
    } else {
      // the largest element into [2^-10, 2^-9): q~ 2^(24 - b) stays inside fp16
      int e = 0;
      if (mx > 0.f && mx < INFINITY) frexpf(mx, &e);
      up = ldexpf(1.f, max(-120, min(-9 - e, 120)));
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float v = x[j] * up;
      if constexpr (I8) {  // element 32 j + lane counts 2^(bit & 3) times
        const float times = (float)(1 << (lane & 3));
        v = rintf(v / times) * times;
      }
      sum += v;
      qs[y][32 * j + lane] = v;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      out->sum[y] = sum;
      out->scale[y] = P.log_scale / up;  // sm_scale log2(e) / sqrt(D) and the scale above
    }
  }
  __syncthreads();
  // column g: query g / 2, its high part (even) or low part
  const int g = lane >> 2, t = lane & 3;
  for (int k = warp; k < NB * KS; k += 4) {
    const int i = k % KS, y = k / KS * 4 + (g >> 1);
    if constexpr (I8) {
      // k = 4 t + j is bit 2 i of byte j of the lane's word, k = 4 t + 16 + j bit 2 i + 1
      const int word = D == 128 ? t : 2 * t + (i >> 2);
      uint32_t f[2] = {0, 0};
#pragma unroll
      for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int bit = 2 * (i & 3) + o;
          const int v = (int)qs[y][32 * word + 8 * j + bit] >> (bit & 3);
          const int low = ((v + 128) & 255) - 128;
          f[o] |= (uint32_t)((g & 1 ? low : (v - low) >> 8) & 255) << (8 * j);
        }
      out->q[k][lane] = make_uint2(f[0], f[1]);
    } else {
      // k = 2 t, 2 t + 1 are bit 2 i of the two halves of the lane's word,
      // k = 2 t + 8, 2 t + 9 bit 2 i + 1
      auto value = [&](int e, int bit) {
        const float v = qs[y][e] * (float)(1 << (24 - (bit & 7)));
        const float hi_part = round_h(v);
        return g & 1 ? (v - hi_part) * kPart : hi_part;
      };
      const int e = (D == 128 ? 32 * t : 64 * t + 32 * (i >> 3)), bit = 2 * (i & 7);
      out->q[k][lane] =
          make_uint2(pack_h2(value(e + bit, bit), value(e + 16 + bit, bit)),
                     pack_h2(value(e + bit + 1, bit + 1), value(e + 17 + bit, bit + 1)));
    }
  }
}

// Sequence b with starts[b] * per <= x < starts[b + 1] * per: a warp looks at
// 32 places at once.
__device__ __forceinline__ int64_t find_sequence(const AttnParams& P, int64_t x, int64_t per,
                                                 int lane) {
  int64_t lo = 0, n = P.r.n_seqs;  // it is among [lo, lo + n)
  while (n > 1) {
    const int64_t step = (n + 31) / 32, i = min(lo + (lane + 1) * step, lo + n);
    const int below = __popc(__ballot_sync(0xffffffffu, i < lo + n && P.starts[i] * per <= x));
    lo += below * step;
    n = min(step, n - below * step);
  }
  return lo;
}

// CTAs an SM that the registers are bounded for.
template <int D, bool I8, int NB>
constexpr int rows_ctas() {
  return D == 256 || NB == 2 ? 3 : I8 ? 5 : 4;
}

template <int D, bool I8, bool EXTRA, int NB>
__global__ void __launch_bounds__(32 * kWarps, rows_ctas<D, I8, NB>())
    paged_rows_kernel(const __grid_constant__ AttnParams P) {
  using C = RowsCfg<D>;
  using F = Frags<D, I8, NB>;
  using Acc = std::conditional_t<I8, int, float>;
  constexpr int W = C::W;
  constexpr int kStages = C::kStages;
  constexpr int KS = F::kSteps;         // steps of the score product
  constexpr int MT = D / 16;            // element tiles of the value product
  constexpr int NQ = NB * 4;
  constexpr bool kRegs = NB * KS <= 8;  // query fragments in registers
  const PagedAttnRequest& r = P.r;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int hq_all = r.n_kv_heads * r.n_q;
  uint8_t* ring = smem + warp * kStages * C::kStage;
  uint2(*q_frag)[32] = reinterpret_cast<uint2(*)[32]>(smem + C::kRing + warp * NB * KS * 256);
  // After a prefix launch this grid may run beside it: that one signals its
  // dependents once all earlier work is done, and nothing here reads its
  // records.  The wait then comes at the end, so that this grid's completion
  // implies the prefix's.
  if (!P.pre_tensor) grid_dependency_wait();
  const int64_t n_pre = (int64_t)r.n_kv_heads * P.pre_blocks * r.prefix_len;
  const int64_t per = (int64_t)r.n_kv_heads * P.own_blocks;
  const int64_t total = n_pre + P.starts[r.n_seqs] * per;

#pragma unroll 1
  for (;;) {
  uint32_t unit = 0;
  if (lane == 0) unit = atomicAdd(P.next_unit, 1u);
  unit = __shfl_sync(0xffffffffu, unit, 0);
  int64_t at = (int64_t)unit * P.unit;
  if (at >= total) break;
  const int64_t end = min(at + P.unit, total);
#pragma unroll 1
  while (at < end) {
  // ---- the piece: rows [lo, hi) of a sequence (or of the prefix, for every
  // sequence's queries) for query rows y0 .. y0 + nq of KV head h
  const bool pre = at < n_pre;
  const int64_t b = pre ? 0 : find_sequence(P, at - n_pre, per, lane);
  const int64_t start = pre ? 0 : n_pre + P.starts[b] * per;
  const int64_t rows = pre ? r.prefix_len : P.starts[b + 1] - P.starts[b];
  const int hz = (int)((at - start) / rows);
  const int64_t begin = start + hz * rows;
  const int lo = (pre ? 0 : P.first_row[b]) + (int)(at - begin);
  const int hi = lo + (int)min(rows - (at - begin), end - at);
  at += hi - lo;
  const int blocks = pre ? P.pre_blocks : P.own_blocks;
  const int h = hz / blocks;
  const int64_t y0 = (int64_t)(hz - h * blocks) * NQ;
  const int nq = (int)min((int64_t)NQ, (pre ? r.n_seqs * r.n_q : (int64_t)r.n_q) - y0);
  const int part = (int)(unit - begin / P.unit) + (pre ? 0 : P.plan.pre_parts);
  const F* frags = reinterpret_cast<const F*>(P.frags) +
                              (pre ? hz : r.n_kv_heads * P.pre_blocks + b * per + hz);
  auto seq_of = [&](int y) { return pre ? (y0 + y) / r.n_q : b; };
  auto head_of = [&](int y) { return h * r.n_q + (int)(pre ? (y0 + y) % r.n_q : y0 + y); };

  // ---- tiles of 32 rows: lane = row
  const int n_tiles = (hi - lo + 31) >> 5;
  const int32_t* tab = r.table + b * r.table_stride;
  auto page_of = [&](int tile) {
    const uint32_t j = lo + tile * 32 + lane;
    return (tile < n_tiles && (int)j < hi) ? tab[P.page_div(j)] : -1;
  };
  auto issue = [&](int tile, int stage, int page) {
    if (tile < n_tiles) {
      const uint32_t j = lo + tile * 32 + lane;
      const bool in = (int)j < hi;
      const bool on = in && (uint32_t)page < (uint32_t)r.n_pages;
      if (in && !on) flag_error(P.err, kErrBadIndex);
      const uint32_t off = j - P.page_div(j) * r.page_size;
      const int64_t row = on ? ((int64_t)page * r.n_kv_heads + h) * r.page_size + off : 0;
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
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s, s, page_of(s));
  int next_page = page_of(kStages - 1);

  uint2 qf[kRegs ? NB * KS : 1];
#pragma unroll
  for (int i = 0; i < NB * KS; ++i) {
    const uint2 f = frags->q[i][lane];
    if constexpr (kRegs) qf[i] = f;
    else q_frag[i][lane] = f;
  }

  // ---- constants of this thread's query of each block
  //   t2 = norm (a1 M1 + b1) + rnorm (a2 M2 + b2), M the masked sums
  const float ch = 0.5f * (r.c1 - r.c0), cm = 0.5f * (r.c1 + r.c0);
  const float inv_sd = P.inv_sd;
  float a1[NB], b1[NB], a2[NB], b2[NB], slope[NB];
  int q_lo[NB], q_hi[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int y = nb * 4 + t;
    const float k = frags->scale[y], sum = frags->sum[y] * k;
    a1[nb] = 2.f * ch * k;
    b1[nb] = (cm - ch) * sum;
    a2[nb] = 2.f * inv_sd * k;
    b2[nb] = -inv_sd * sum;
    slope[nb] = 0.f;
    q_lo[nb] = 0;
    q_hi[nb] = 0x7fffffff;
    if (y < nq) {
      if (pre || (EXTRA && r.slopes)) {
        const int64_t len = length_of(P, seq_of(y));
        q_hi[nb] = (int)len;
        if (pre) q_lo[nb] = (int)min(first_of(P, seq_of(y), len), (int64_t)0x7fffffff);
      }
      if (EXTRA && r.slopes) slope[nb] = r.slopes[head_of(y)] * kLog2e;
    }
  }
  constexpr float kUnitWeight = I8 ? 32768.f : 1.f;  // how weight 1 is stored
  constexpr float kMost = I8 ? 65535.f : kMaxWeight;
  const float va = ch * inv_sd * kUnitWeight;
  const float vb = 0.7978845608028654f * inv_sd * inv_sd * kUnitWeight;
  const float cap = r.softcap * kLog2e, inv_cap = r.softcap > 0.f ? 1.f / cap : 0.f;

  // w1s, w2s: sums of weights; in i1, i2 those since the reference last moved
  float ref[NB], l[NB], w1s[NB], w2s[NB];
  uint32_t i1[NB], i2[NB];
  Acc acc[NB][MT][4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    ref[nb] = kNoRef;
    l[nb] = w1s[nb] = w2s[nb] = 0.f;
    i1[nb] = i2[nb] = 0u;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[nb][i][k] = 0;
  }
  const int pg = (g >> 1) + 4 * (g & 1);  // pi(g)

#pragma unroll 1
  for (int tile = 0; tile < n_tiles; ++tile) {
    cp_wait<kStages - 2>();
    __syncwarp();
    const uint8_t* st = ring + (tile % kStages) * C::kStage;
    const float4* nrm = reinterpret_cast<const float4*>(st + 4 * C::kPlane);
    const uint32_t valid = *reinterpret_cast<const uint32_t*>(st + 4 * C::kPlane + 512);
    const int j0 = lo + tile * 32;

    // scores of the tile's two 16-row halves, both planes
    Acc s1[2][NB][4], s2[2][NB][4];
    if constexpr (!I8) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int k = 0; k < 4; ++k) s1[hf][nb][k] = s2[hf][nb][k] = 0;
    }
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
      constexpr int kPer = KS / (W / 4);  // steps of a word
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (i == kPer / 2)
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k >> 2][(k >> 1) & 1][k & 1] >>= kPer;
        const uint32_t m0 = (I8 ? 0x01010101u : 0x00010001u) << ((2 * i) % kPer), m1 = m0 << 1;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          uint2 f;
          if constexpr (kRegs) f = qf[nb * KS + v * kPer + i];
          else f = q_frag[nb * KS + v * kPer + i][lane];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              auto& c = p == 0 ? s1[hf][nb] : s2[hf][nb];
              const uint32_t x0 = w[hf][p][0], x1 = w[hf][p][1];
              if constexpr (I8) {
                if (v == 0 && i == 0) mma16832_0(c, x0 & m0, x1 & m0, x0 & m1, x1 & m1, f.x, f.y);
                else mma16832(c, x0 & m0, x1 & m0, x0 & m1, x1 & m1, f.x, f.y);
              } else mma16816(c, x0 & m0, x1 & m0, x0 & m1, x1 & m1, f.x, f.y);
            }
        }
      }
    }

    // exponents
    bool full = valid == 0xffffffffu;
    if (pre) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) full = full && j0 >= q_lo[nb] && j0 + 32 <= q_hi[nb];
      full = __all_sync(0xffffffffu, full);
    }
    float tt[2][2][NB], ra[2][2], rb[2][2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        const int row = 16 * hf + pg + 8 * rr;
        const float4 n = nrm[row];
        ra[hf][rr] = n.z * va;
        rb[hf][rr] = n.w * vb;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float m1, m2;
          if constexpr (I8) {
            m1 = (float)(s1[hf][nb][2 * rr] * 256 + s1[hf][nb][2 * rr + 1]);
            m2 = (float)(s2[hf][nb][2 * rr] * 256 + s2[hf][nb][2 * rr + 1]);
          } else {
            m1 = fmaf(s1[hf][nb][2 * rr + 1], 1.f / kPart, s1[hf][nb][2 * rr]);
            m2 = fmaf(s2[hf][nb][2 * rr + 1], 1.f / kPart, s2[hf][nb][2 * rr]);
          }
          float x = n.x * fmaf(a1[nb], m1, b1[nb]);
          x = fmaf(n.y, fmaf(a2[nb], m2, b2[nb]), x);
          if (EXTRA && r.softcap > 0.f) x = soft_cap(x, cap, inv_cap);
          if (EXTRA && r.slopes) x = fmaf(slope[nb], (float)(j0 + row + 1 - q_hi[nb]), x);
          tt[hf][rr][nb] = x;
        }
      }
    if (!full) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int row = 16 * (k >> 1) + pg + 8 * (k & 1), j = j0 + row;
          const bool on = ((valid >> row) & 1) && j >= q_lo[nb] && j < q_hi[nb];
          if (!on) tt[k >> 1][k & 1][nb] = -INFINITY;
        }
    }
    // weights: e = 2^(t2 - ref); a row's larger weight decides whether they fit
    float ee[2][2][NB];
#pragma unroll 1
    for (bool again = false;; again = true) {
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float e = ex2(tt[k >> 1][k & 1][nb] - ref[nb]);
          ee[k >> 1][k & 1][nb] = e;
          const float most =
              fmaxf(fmaxf(ra[k >> 1][k & 1], rb[k >> 1][k & 1]), kUnitWeight * 0x1p-40f);
          // nothing attended: 0 times whatever the row's norms hold
          top = fmaxf(top, e == 0.f ? 0.f : e * most);
        }
      if (again || !__any_sync(0xffffffffu, !(top <= kMost))) break;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float mx = kNoRef;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float most =
              fmaxf(fmaxf(ra[k >> 1][k & 1], rb[k >> 1][k & 1]), kUnitWeight * 0x1p-40f);
          const float x = tt[k >> 1][k & 1][nb];
          if (x > -INFINITY) mx = fmaxf(mx, x + lg2(most * (1.f / kUnitWeight)));
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (mx == INFINITY) l[nb] = NAN;  // an infinite norm has no average
        // whole exponents: integer sums move by shifts
        const float to = fmaxf(ref[nb], I8 ? ceilf(mx) : mx), f = ex2(ref[nb] - to);
        const int shift = (int)fminf(to - ref[nb], 31.f);
        if constexpr (I8) {
          w1s[nb] += (float)i1[nb];
          w2s[nb] += (float)i2[nb];
          i1[nb] = i2[nb] = 0u;
        }
        ref[nb] = to;
        if (tile == 0) continue;  // nothing summed yet
        l[nb] *= f;
        w1s[nb] *= f;
        w2s[nb] *= f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (I8) acc[nb][i][k] = (acc[nb][i][k] + (int)((1u << shift) >> 1)) >> shift;
            else acc[nb][i][k] *= f;
          }
      }
    }
    uint32_t p1[2][NB][2], p2[2][NB][2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        uint32_t u1[2], u2[2];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const float e = ee[hf][rr][nb];
          l[nb] += e;
          float x1, x2;
          if constexpr (I8) {
            // 2^23 + w: the low bits are w as a whole number
            x1 = fmaf(e, ra[hf][rr], 8388608.f);
            x2 = fmaf(e, rb[hf][rr], 8388608.f);
          } else {
            x1 = e * ra[hf][rr];
            x2 = e * rb[hf][rr];
          }
          if (!full && tt[hf][rr][nb] == -INFINITY) x1 = x2 = I8 ? 8388608.f : 0.f;
          if constexpr (I8) {
            u1[rr] = __float_as_uint(x1);
            u2[rr] = __float_as_uint(x2);
          } else {
            w1s[nb] += x1;
            w2s[nb] += x2;
            p1[hf][nb][rr] = transpose8(pack_h2(x1, (x1 - round_h(x1)) * kPart));
            p2[hf][nb][rr] = transpose8(pack_h2(x2, (x2 - round_h(x2)) * kPart));
          }
        }
        if constexpr (I8) {
          i1[nb] += u1[0] + u1[1];
          i2[nb] += u2[0] + u2[1];
          // columns 2 t, 2 t + 1: high and low bytes, of both rows
          p1[hf][nb][0] = transpose8(__byte_perm(u1[0], u1[1], 0x4051));
          p2[hf][nb][0] = transpose8(__byte_perm(u2[0], u2[1], 0x4051));
        }
      }

    // values
    if constexpr (I8) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {  // without the four exponent fields of 2^23
        i1[nb] -= 4u * 0x4B000000u;
        i2[nb] -= 4u * 0x4B000000u;
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
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
                        f[0][nb][0], f[1][nb][0]);
            }
          }
      }
    } else {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint32_t* pl = reinterpret_cast<const uint32_t*>(st + (2 + p) * C::kPlane) +
                               (16 * hf + t) * W + (D == 128 ? g >> 1 : g);
          const uint32_t r0 = pl[0], r1 = pl[4 * W], r2 = pl[8 * W], r3 = pl[12 * W];
#pragma unroll
          for (int v = 0; v < W / 4; ++v) {
            const uint32_t sel = (D == 128 ? (g & 1) : v) ? 0x7632u : 0x5410u;
            const uint32_t x0 = __byte_perm(r0, r1, sel), x1 = __byte_perm(r2, r3, sel);
            auto sign = [](uint32_t x, int bit) {
              return ((x << (15 - bit)) & 0x80008000u) ^ 0xBC00BC00u;
            };
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t a0 = sign(x0, 2 * i), b0 = sign(x0, 2 * i + 1);
              const uint32_t a1 = sign(x1, 2 * i), b1 = sign(x1, 2 * i + 1);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                const uint32_t(&f)[2] = p == 0 ? p1[hf][nb] : p2[hf][nb];
                mma16816(acc[nb][8 * v + i], a0, b0, a1, b1, f[0], f[1]);
              }
            }
          }
        }
    }
    __syncwarp();
    issue(tile + kStages - 1, (tile + kStages - 1) % kStages, next_page);
    next_page = page_of(tile + kStages);
  }
  cp_wait<0>();
  __syncwarp();

  // ---- the record: 16 consecutive elements a lane (32 at D = 256)
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    if constexpr (I8) {
      w1s[nb] += (float)i1[nb];
      w2s[nb] += (float)i2[nb];
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l[nb] += __shfl_xor_sync(0xffffffffu, l[nb], o);
      w1s[nb] += __shfl_xor_sync(0xffffffffu, w1s[nb], o);
      w2s[nb] += __shfl_xor_sync(0xffffffffu, w2s[nb], o);
    }
    const int y = nb * 4 + t;
    if (y < nq) {
      float* rec = r.workspace +
                   ((seq_of(y) * hq_all + head_of(y)) * P.plan.parts() + part) * (int64_t)(D + 2);
      if (g == 0) *reinterpret_cast<float2*>(rec) = make_float2(ref[nb], l[nb]);
      const float base = (I8 ? -w1s[nb] - w2s[nb] : 0.f) + (cm / ch) * w1s[nb];
      // element i of part k of the lane's 16 (or 32)
      auto element = [&](int i, int k) {
        if constexpr (I8) {  // 2 sum w bit, bit i counting 2^(i & 7) times
          const float x = fmaf((float)acc[nb][i][2 * k], 256.f, (float)acc[nb][i][2 * k + 1]);
          return (fmaf(x, 2.f / (float)(1 << (i & 7)), base)) * (1.f / kUnitWeight);
        } else {
          return fmaf(acc[nb][i][2 * k + 1], 1.f / kPart, acc[nb][i][2 * k]) + base;
        }
      };
      const int e0 = 2 + (D == 128 ? 16 : 32) * g;
#pragma unroll
      for (int i = 0; i < MT; i += 2) {
        if constexpr (I8) {  // tile i: elements i and 8 + i of each 16
#pragma unroll
          for (int k = 0; k < 2; ++k)
            *reinterpret_cast<float2*>(rec + e0 + 16 * (i >> 3) + 8 * k + (i & 7)) =
                make_float2(element(i, k), element(i + 1, k));
        } else {  // tile i: elements 2 i and 2 i + 1
#pragma unroll
          for (int k = 0; k < 2; ++k)
            *reinterpret_cast<float2*>(rec + e0 + 2 * (i + k)) =
                make_float2(element(i + k, 0), element(i + k, 1));
        }
      }
    }
  }
  }
  }
  if (P.pre_tensor) grid_dependency_wait();
  else grid_dependents_launch();
}

// A block per query row: its records merged, back from the transformed
// domain, divided by l, in the query's type.  What it takes is the time of a
// few dependent loads, so each warp takes every fourth record and loads four
// of them at once.
template <int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const __grid_constant__ AttnParams P) {
  constexpr int J = D / 32, U = 4;
  const PagedAttnRequest& r = P.r;
  __shared__ float sums[4][D], tops[4], ls[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int hq_all = r.n_kv_heads * r.n_q;
  const uint32_t row = blockIdx.x;
  const uint32_t b = row / hq_all;
  const float* rec = r.workspace + (int64_t)row * P.plan.parts() * (D + 2);
  grid_dependency_wait();
  // slots of the units that the row's groups touch
  const int hq = (int)(row - b * hq_all), h = hq / r.n_q, y = hq - h * r.n_q;
  auto slots = [&](int64_t begin, int64_t rows) {
    return rows > 0 ? (int)((begin + rows - 1) / P.unit - begin / P.unit) + 1 : 0;
  };
  const int n_pre = P.pre_tensor ? P.plan.pre_chunks
                    : P.pre_blocks
                        ? slots((int64_t)(h * P.pre_blocks + (b * r.n_q + y) / P.block) * r.prefix_len,
                                r.prefix_len)
                        : 0;
  int n = n_pre;
  if (P.plan.own_parts) {
    const int64_t first = P.starts[b], rows = P.starts[b + 1] - first;
    n += slots(((int64_t)P.pre_blocks * r.prefix_len + first * P.own_blocks) * r.n_kv_heads +
                   (int64_t)(h * P.own_blocks + y / P.block) * rows,
               rows);
  }
  float mx = -INFINITY, l = 0.f, a[J];
#pragma unroll
  for (int j = 0; j < J; ++j) a[j] = 0.f;
  // 32 slots at a time: a lane each for m and l (0 where nothing was attended)
  for (int p0 = 0; p0 < n; p0 += 32) {
    const int i = p0 + lane, slot = i < n_pre ? i : i - n_pre + P.plan.pre_parts;
    const float* mine = rec + (int64_t)(i < n ? slot : 0) * (D + 2);
    const float mp = mine[0], lp = i < n ? mine[1] : 0.f;
    uint32_t live = __ballot_sync(0xffffffffu, lp != 0.f);
    if (!live) continue;
    float top = lp != 0.f ? mp : -INFINITY;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = fmaxf(top, mx);
    const float old = mx == -INFINITY ? 0.f : ex2(mx - top), f = lp != 0.f ? ex2(mp - top) : 0.f;
    mx = top;
    l *= old;
#pragma unroll
    for (int j = 0; j < J; ++j) a[j] *= old;
    // this warp's share of them: every fourth
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < warp) live &= live - 1;
    while (live) {
      int q[U];
      float v[U][J];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        q[u] = live ? __ffs(live) - 1 : -1;
        live &= live - 1;
        live &= live - 1;
        live &= live - 1;
        live &= live - 1;
        const int at = __shfl_sync(0xffffffffu, slot, max(q[u], 0));
#pragma unroll
        for (int j = 0; j < J; ++j)
          v[u][j] = q[u] >= 0 ? rec[(int64_t)at * (D + 2) + 2 + 32 * j + lane] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float fu = __shfl_sync(0xffffffffu, f, max(q[u], 0));
        const float lu = __shfl_sync(0xffffffffu, lp, max(q[u], 0));
        if (q[u] >= 0) {
          l = fmaf(lu, fu, l);
#pragma unroll
          for (int j = 0; j < J; ++j) a[j] = fmaf(v[u][j], fu, a[j]);
        }
      }
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
  const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  l = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) a[j] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (tops[w] == -INFINITY) continue;
    const float f = ex2(tops[w] - top);
    l = fmaf(ls[w], f, l);
#pragma unroll
    for (int j = 0; j < J; ++j) a[j] = fmaf(sums[w][32 * j + lane], f, a[j]);
  }
  fwht_lanes<J>(a, lane);
  const float inv = 1.f / l;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const float v = l == 0.f ? 0.f : a[j] * inv;
    st_any(r.out, r.dtype, (int64_t)row * D + 32 * j + lane, (r.dv_neg[j] >> lane) & 1 ? -v : v);
  }
  if (r.lse && lane == 0) r.lse[row] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
}

template <int D, bool I8, bool EXTRA, int NB>
kh_status launch_rows(AttnParams P, cudaStream_t stream) {
  const PagedAttnRequest& r = P.r;
  constexpr int NQ = NB * 4, KS = Frags<D, I8, NB>::kSteps;
  using C = RowsCfg<D>;
  auto kern = paged_rows_kernel<D, I8, EXTRA, NB>;
  constexpr int kSmem = C::kRing + (NB * KS <= 8 ? 0 : kWarps * NB * KS * 256);
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
  P.block = NQ;
  P.own_blocks = P.plan.own_parts > 0 ? (r.n_q + NQ - 1) / NQ : 0;
  P.pre_blocks =
      P.plan.pre_parts > 0 && !P.pre_tensor ? (int)((r.n_seqs * r.n_q + NQ - 1) / NQ) : 0;
  const int64_t groups = (int64_t)r.n_kv_heads * (P.pre_blocks + r.n_seqs * P.own_blocks);
  const int64_t pairs = (int64_t)r.n_kv_heads * (P.pre_blocks * r.prefix_len +
                                                 r.n_seqs * P.own_blocks * P.plan.own_rows);
  if (groups > 0x7ffffff0ll || pairs / P.unit > 0x7ffffff0ll) return KH_EINVAL;
  static_assert(sizeof(Frags<D, I8, NB>) <= kFragBytes, "workspace of the fragments");
  if (P.plan.parts() > 0 &&
      launch_programmatic(paged_prepare_kernel<D, I8, NB>, dim3((unsigned)(groups + 1)),
                          dim3(128), 0, stream, P) != cudaSuccess)
    return KH_ELAUNCH;
  if (P.pre_tensor) {
    const kh_status st = launch_paged_prefix(P, stream);
    if (st != KH_OK) return st;
  }
  if (pairs > 0) {
    const int64_t units = (pairs + P.unit - 1) / P.unit;
    const int64_t grid = std::min<int64_t>((int64_t)std::max(1, ctas[dev & 63]) * sm_count(),
                                           (units + kWarps - 1) / kWarps);
    if (launch_programmatic(kern, dim3((unsigned)grid), dim3(32 * kWarps), kSmem, stream, P) !=
        cudaSuccess)
      return KH_ELAUNCH;
  }
  const int64_t rows = r.n_seqs * r.n_kv_heads * r.n_q;
  if (rows > 0x7fffffffll) return KH_EINVAL;
  return launch_programmatic(paged_combine_kernel<D>, dim3((unsigned)rows), dim3(128), 0, stream,
                             P) == cudaSuccess
             ? KH_OK
             : KH_ELAUNCH;
}

template <int D>
kh_status launch_dim(const AttnParams& P, cudaStream_t stream) {
  const PagedAttnRequest& r = P.r;
  const int64_t nq = P.plan.pre_parts > 0 && !P.pre_tensor ? r.n_seqs * r.n_q : r.n_q;
  constexpr int kTwo = D == 128 ? 2 : 1;  // column blocks a pass, where there are queries for two
  // 32-bit queries need more than 16-bit parts, and so do units so long that
  // a 32-bit integer could not hold a column's sum (255 x 128 a row)
  const bool i8 = r.dtype != KH_F32 && P.unit <= 32768;
  const bool extra = r.softcap > 0.f || r.slopes;
  auto go = [&](auto i8c, auto extrac) {
    return nq > 4 ? launch_rows<D, decltype(i8c)::value, decltype(extrac)::value, kTwo>(P, stream)
                  : launch_rows<D, decltype(i8c)::value, decltype(extrac)::value, 1>(P, stream);
  };
  const kh_status st = i8 ? (extra ? go(std::true_type{}, std::true_type{})
                                   : go(std::true_type{}, std::false_type{}))
                          : (extra ? go(std::false_type{}, std::true_type{})
                                   : go(std::false_type{}, std::false_type{}));
  if (st != KH_OK) return st;
  return cudaGetLastError() == cudaSuccess ? KH_OK : KH_ELAUNCH;
}

}  // namespace

// From how many query rows a KV head's prefix is worth 128-row products.
constexpr int64_t kPrefixTensorRows = 33;

// The workspace: the records; then, each 16-byte aligned, the sequences'
// starts and first rows, the claim counter, the queries' fragments (blocks of
// 4 queries at least, so n_q / 4 of them at most) and, of a tensor-core
// prefix, its transformed queries.
struct Layout {
  int64_t starts, first, next, frags, queries, bytes;
};
Layout layout_of(const PagedPlan& p, int64_t n_seqs, int n_q, int n_kv_heads, int D) {
  auto up = [](int64_t x) { return (x + 15) / 16 * 16; };
  const int64_t nq = n_seqs * n_q, blocks = (n_q + 3) / 4;
  Layout l;
  l.starts = up(nq * n_kv_heads * p.parts() * (int64_t)(D + 2) * 4);
  l.first = l.starts + up((n_seqs + 1) * 8);
  l.next = l.first + up(n_seqs * 4);
  l.frags = l.next + 16;
  int64_t groups = p.own_parts > 0 ? n_seqs * blocks : 0;
  if (p.pre_parts > 0) groups += (nq + 3) / 4;
  l.queries = l.frags + groups * n_kv_heads * kFragBytes;
  l.bytes = l.queries;
  if (p.pre_chunks > 0) l.bytes += paged_queries_bytes(nq, n_kv_heads, D);
  return l;
}
int64_t paged_workspace_bytes(const PagedPlan& p, int64_t n_seqs, int n_q, int n_kv_heads, int D) {
  return p.parts() > 0 ? layout_of(p, n_seqs, n_q, n_kv_heads, D).bytes : 0;
}

PagedPlan paged_plan(int64_t n_seqs, int n_q, int n_kv_heads, int D, int64_t max_len,
                     int64_t prefix_len, int64_t window, int dtype, int n_sms) {
  PagedPlan p;
  const int64_t rows = n_seqs * n_q * n_kv_heads, record = (D + 2) * 4;
  const int64_t pre = std::min(prefix_len, max_len), nq = n_seqs * n_q;
  int64_t own = max_len - pre;
  if (window > 0) own = std::min(own, window);
  // the prefix's chunks on the tensor cores: one round of CTAs, one an SM, in
  // whole tiles
  if (pre > 0 && nq >= kPrefixTensorRows && dtype == KH_BF16) {
    const int64_t each = D == 128 ? 256 : 128, tile = D == 128 ? 128 : 64;
    const int64_t ctas = std::max<int64_t>(1, n_sms / (n_kv_heads * ((nq + each - 1) / each)));
    p.pre_rows = ((pre + ctas - 1) / ctas + tile - 1) / tile * tile;
    p.pre_chunks = (int)((pre + p.pre_rows - 1) / p.pre_rows);
  }
  // Units: three for every two warps (20 an SM) where the longest sequences
  // give that many, so that the last ones end together; not under two tiles
  // (a unit's fixed cost is about one tile's) nor over 64, and not so short
  // that the records take over 64 MB (at least 6 slots a row).
  const int64_t blocks = (n_q + 3) / 4;
  const int64_t pairs = n_kv_heads * (n_seqs * blocks * own + (p.pre_chunks ? 0 : (nq + 3) / 4 * pre));
  const int64_t room =
      rows > 0 ? std::max<int64_t>(6, (int64_t(64) << 20) / (rows * record)) - 4 : 2;
  int64_t unit = std::max<int64_t>(64, std::min<int64_t>(2048, pairs / (32 * (int64_t)n_sms)));
  unit = std::max(unit, (own + (p.pre_chunks ? 0 : pre) + room - 1) / room);
  p.unit = (unit + 31) / 32 * 32;
  // a group touches at most this many units
  if (pre > 0) p.pre_parts = p.pre_chunks ? p.pre_chunks : (int)(pre / p.unit + 2);
  if (own > 0) p.own_parts = (int)(own / p.unit + 2);
  p.own_rows = own;
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
  P.pre_tensor = P.plan.pre_chunks > 0;
  P.unit = P.plan.unit;
  const Layout l = layout_of(P.plan, r.n_seqs, r.n_q, r.n_kv_heads, r.D);
  uint8_t* ws = reinterpret_cast<uint8_t*>(r.workspace);
  P.starts = reinterpret_cast<int64_t*>(ws + l.starts);
  P.first_row = reinterpret_cast<int32_t*>(ws + l.first);
  P.next_unit = reinterpret_cast<uint32_t*>(ws + l.next);
  P.frags = ws + l.frags;
  P.queries = reinterpret_cast<uint16_t*>(ws + l.queries);
  P.err = device_error_ptr();
  return r.D == 128 ? launch_dim<128>(P, stream) : launch_dim<256>(P, stream);
}

}  // namespace kh
