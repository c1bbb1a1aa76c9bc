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

#include "kh_common.cuh"
#include "kh_paged_attn.cuh"

namespace kh {
namespace {

// ------------------------------------------------------------------ rows
//
// paged_rows_kernel: the two products of a chunk on mma.sync, fed from
// registers.  A row's bits need no shared-memory expansion: a 16-bit lane of
// a packed word, masked to bit b, IS the fp16 number 2^(b - 24) (a
// subnormal) or zero, exactly, so one LOP3 makes two matrix elements and
// the factor goes into the other operand (q~ 2^(24 - b)) or into the
// accumulator's scale.  What bit belongs to what index of the product is
// free, as long as both operands agree:
//   scores  A = 16 rows x 16 elements: lane (g, t) holds word t of rows
//           pi(g) and pi(g) + 8; step i takes its bits 2 i and 2 i + 1 in
//           both halves.  B = q~ of 8 columns.
//   values  A = 16 elements x 16 rows: lane (g, t) holds halfword g (word g
//           at D = 256) of rows t, t + 4, t + 8, t + 12.  B = the weights
//           p norm' and p rnorm', which movmatrix turns from the scores'
//           accumulator layout into the operand's.
// With bits as 0 / 1, sum w sign = 2 sum w bit - sum w.  That difference
// costs the values a few bits of 24, nothing next to a 16-bit result's
// rounding; for fp32 results (EXACT) the bits are moved to the sign
// of +-1 instead, one more shift each.
//
// Columns: HILO splits a query (and its weights) into two fp16 parts, the
// second times 2^11: 22 bits from 4 queries a block of 8 columns.  Without,
// 8 queries of 11 bits: for bf16 results of groups over 4.
//
// A warp runs on its own: 32-row tiles in a ring of cp.async stages, one lane
// fetching one row (so pages may end anywhere), no block barrier until the
// warps' sums are joined.  The reference exponent of a column moves only when
// a weight would leave fp16's upper range (2^12), so most tiles rescale
// nothing.
constexpr int kWarps = 4;

template <int D>
struct RowsCfg {
  static constexpr int W = D / 32;
  static constexpr int kStages = D == 128 ? 4 : 3;
  static constexpr int kPlane = 32 * W * 4;             // one plane of a tile
  static constexpr int kStage = 4 * kPlane + 4 * 128 + 16;  // + norms + valid mask
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

constexpr float kPart = 2048.f;      // second fp16 parts are stored times 2^11

template <int D, bool HILO, bool EXACT, int NB>
__global__ void __launch_bounds__(32 * kWarps, D == 128 ? (NB == 1 ? 4 : 3) : 3)
    paged_rows_kernel(const __grid_constant__ AttnParams P) {
  using C = RowsCfg<D>;
  constexpr int W = C::W;
  constexpr int kStages = C::kStages;
  constexpr int KS = D / 16;            // steps of the score product
  constexpr int MT = D / 16;            // element tiles of the value product
  constexpr int QB = HILO ? 4 : 8;      // queries a column block
  constexpr int QT = HILO ? 1 : 2;      // of them this thread's
  constexpr int NQ = NB * QB;
  const PagedAttnRequest& r = P.r;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float qs[NQ][D];
  __shared__ float q_sum[NQ], q_scale[NQ];
  __shared__ float rec_m[kWarps][NQ], rec_l[kWarps][NQ];
  __shared__ uint2 q_frag[(D == 128 && NB == 1) ? 1 : NB * KS][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;

  // ---- the work item
  const int h = blockIdx.y % r.n_kv_heads;
  const int64_t item = blockIdx.y / r.n_kv_heads;  // 0: the prefix when there is one
  const bool has_pre = P.plan.pre_chunks > 0 && !P.pre_tensor;
  const bool pre = has_pre && item == 0;
  const int64_t b = pre ? 0 : item - has_pre;
  const int chunk = blockIdx.x;
  if (chunk >= (pre ? P.plan.pre_chunks : P.plan.own_chunks)) return;
  const int64_t n_rows = pre ? r.n_seqs * r.n_q : r.n_q;
  const int64_t y0 = (int64_t)blockIdx.z * NQ;
  if (y0 >= n_rows) return;
  const int nq = (int)min((int64_t)NQ, n_rows - y0);
  // After a prefix launch this grid may run beside it: that one signals its
  // dependents once all earlier work is done, and nothing here reads its
  // records.  The wait then comes at the end, so that this grid's completion
  // implies the prefix's.
  if (!P.pre_tensor) grid_dependency_wait();
  int lo, hi;
  if (pre) {
    lo = (int)(chunk * P.plan.pre_rows);
    hi = (int)min(lo + P.plan.pre_rows, r.prefix_len);
  } else {
    const int64_t len = length_of(P, b);
    const int64_t first = own_first(P, b, len) + chunk * P.plan.own_rows;
    if (first >= len) {
      if (P.pre_tensor) grid_dependency_wait();
      return;
    }
    lo = (int)first;
    hi = (int)min(first + P.plan.own_rows, len);
  }
  const int hq_all = r.n_kv_heads * r.n_q;
  auto seq_of = [&](int y) { return pre ? (y0 + y) / r.n_q : b; };
  auto head_of = [&](int y) { return h * r.n_q + (int)(pre ? (y0 + y) % r.n_q : y0 + y); };

  // ---- tiles: lane = row
  uint8_t* ring = smem + warp * kStages * C::kStage;
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
      const uint32_t n = s + 4 * C::kPlane + lane * 4;
      cp_async4(n, r.kp.norms + row, on);
      cp_async4(n + 128, r.kp.rnorms + row, on);
      cp_async4(n + 256, r.vp.norms + row, on);
      cp_async4(n + 384, r.vp.rnorms + row, on);
      const uint32_t mask = __ballot_sync(0xffffffffu, on);
      if (lane == 0) *reinterpret_cast<uint32_t*>(st + 4 * C::kPlane + 512) = mask;
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(warp + s * kWarps, s, page_of(warp + s * kWarps));
  int next_page = page_of(warp + (kStages - 1) * kWarps);

  // ---- queries: q~ times a power of two that brings its largest element to
  // [2^-10, 2^-9), so that q~ 2^(24 - b) stays inside fp16 for b = 0 .. 7
  for (int y = warp; y < NQ; y += kWarps) {
    float x[W], mx = 0.f, sum = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float v = 0.f;
      if (y < nq) v = ld_any(r.q, r.dtype, (seq_of(y) * hq_all + head_of(y)) * D + 32 * j + lane);
      x[j] = (r.dk_neg[j] >> lane) & 1 ? -v : v;
    }
    fwht_lanes<W>(x, lane);
#pragma unroll
    for (int j = 0; j < W; ++j) mx = fmaxf(mx, fabsf(x[j]));
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    int e = 0;
    if (mx > 0.f && mx < INFINITY) frexpf(mx, &e);
    const float up = ldexpf(1.f, min(-9 - e, 120));
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float v = x[j] * up;
      if (!HILO) v = round_h(v * 16777216.f) * (1.f / 16777216.f);
      sum += v;
      qs[y][32 * j + lane] = v;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      q_sum[y] = sum;
      q_scale[y] = P.log_scale / up;  // sm_scale log2(e) / sqrt(D) and the power of two
    }
  }
  __syncthreads();
  // B fragments: column g; k = 2 t, 2 t + 1 are bit 2 i of the two halves of
  // the lane's word, k = 2 t + 8, 2 t + 9 bit 2 i + 1
  uint2 qf[(D == 128 && NB == 1) ? KS : 1];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int y = nb * QB + (HILO ? g >> 1 : g);
    auto part = [&](int e, int bit) {
      const float v = qs[y][e] * (float)(1 << (24 - (bit & 7)));
      const float hi_part = round_h(v);
      return HILO && (g & 1) ? (v - hi_part) * kPart : hi_part;
    };
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int e = (D == 128 ? 32 * t : 64 * t + 32 * (i >> 3)), bit = 2 * (i & 7);
      if ((D != 128 || NB != 1) && (i & 3) != warp) continue;
      const uint2 f = make_uint2(pack_h2(part(e + bit, bit), part(e + 16 + bit, bit)),
                                 pack_h2(part(e + bit + 1, bit + 1), part(e + 17 + bit, bit + 1)));
      if constexpr (D == 128 && NB == 1) qf[i] = f;
      else q_frag[nb * KS + i][lane] = f;
    }
  }
  if (D != 128 || NB != 1) __syncthreads();

  // ---- per-thread constants of its queries
  //   t2 = norm (a1 M1 + b1) + rnorm (a2 M2 + b2), M the masked sums
  const float ch = 0.5f * (r.c1 - r.c0), cm = 0.5f * (r.c1 + r.c0);
  const float inv_sd = P.inv_sd;
  float a1[NB][QT], b1[NB][QT], a2[NB][QT], b2[NB][QT], slope[NB][QT];
  int q_lo[NB][QT], q_hi[NB][QT];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int qq = 0; qq < QT; ++qq) {
      const int y = nb * QB + (HILO ? t : 2 * t + qq);
      const float k = q_scale[y], sum = q_sum[y] * k;
      a1[nb][qq] = 2.f * ch * k;
      b1[nb][qq] = (cm - ch) * sum;
      a2[nb][qq] = 2.f * inv_sd * k;
      b2[nb][qq] = -inv_sd * sum;
      slope[nb][qq] = 0.f;
      q_lo[nb][qq] = 0;
      q_hi[nb][qq] = 0x7fffffff;
      if (y < nq) {
        if (pre || r.slopes) {
          const int64_t len = length_of(P, seq_of(y));
          q_hi[nb][qq] = (int)len;
          if (pre) q_lo[nb][qq] = (int)min(first_of(P, seq_of(y), len), (int64_t)0x7fffffff);
        }
        if (r.slopes) slope[nb][qq] = r.slopes[head_of(y)] * kLog2e;
      }
    }
  const float va = ch * inv_sd, vb = 0.7978845608028654f * inv_sd * inv_sd;
  const float cap = r.softcap * kLog2e, inv_cap = r.softcap > 0.f ? 1.f / cap : 0.f;

  float ref[NB][QT], l[NB][QT], w1s[NB][QT], w2s[NB][QT], acc[NB][MT][4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int qq = 0; qq < QT; ++qq) {
      ref[nb][qq] = kNoRef;
      l[nb][qq] = w1s[nb][qq] = w2s[nb][qq] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[nb][i][k] = 0.f;
  }
  const int pg = (g >> 1) + 4 * (g & 1);  // pi(g)

#pragma unroll 1
  for (int n = 0, tile = warp; tile < n_tiles; ++n, tile += kWarps) {
    cp_wait<kStages - 2>();
    __syncwarp();
    const uint8_t* st = ring + (n % kStages) * C::kStage;
    const float* nrm = reinterpret_cast<const float*>(st + 4 * C::kPlane);
    const uint32_t valid = *reinterpret_cast<const uint32_t*>(st + 4 * C::kPlane + 512);
    const int j0 = lo + tile * 32;

    // scores of the tile's two 16-row halves
    float s1[2][NB][4], s2[2][NB][4];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int k = 0; k < 4; ++k) s1[hf][nb][k] = s2[hf][nb][k] = 0.f;
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
      for (int i = 0; i < 8; ++i) {
        if (i == 4)
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k >> 2][(k >> 1) & 1][k & 1] >>= 8;
        const uint32_t m0 = 0x00010001u << ((2 * i) & 7), m1 = m0 << 1;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          uint2 f;
          if constexpr (D == 128 && NB == 1) f = qf[i];
          else f = q_frag[nb * KS + v * 8 + i][lane];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            mma16816(s1[hf][nb], w[hf][0][0] & m0, w[hf][0][1] & m0, w[hf][0][0] & m1,
                     w[hf][0][1] & m1, f.x, f.y);
            mma16816(s2[hf][nb], w[hf][1][0] & m0, w[hf][1][1] & m0, w[hf][1][0] & m1,
                     w[hf][1][1] & m1, f.x, f.y);
          }
        }
      }
    }

    // exponents and weights
    bool full = valid == 0xffffffffu;
    if (pre) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int qq = 0; qq < QT; ++qq)
          full = full && j0 >= q_lo[nb][qq] && j0 + 32 <= q_hi[nb][qq];
      full = __all_sync(0xffffffffu, full);
    }
    float tt[2][2][NB][QT], ra[2][2], rb[2][2];
    float w1[2][2][NB][QT], w2[2][2][NB][QT];
    bool over = false;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        const int row = 16 * hf + pg + 8 * rr;
        const float kn = nrm[row], krn = nrm[32 + row];
        ra[hf][rr] = nrm[64 + row] * va;
        rb[hf][rr] = nrm[96 + row] * vb;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int qq = 0; qq < QT; ++qq) {
            const float m1 = HILO ? fmaf(s1[hf][nb][2 * rr + 1], 1.f / kPart, s1[hf][nb][2 * rr])
                                  : s1[hf][nb][2 * rr + qq];
            const float m2 = HILO ? fmaf(s2[hf][nb][2 * rr + 1], 1.f / kPart, s2[hf][nb][2 * rr])
                                  : s2[hf][nb][2 * rr + qq];
            float x = kn * fmaf(a1[nb][qq], m1, b1[nb][qq]);
            x = fmaf(krn, fmaf(a2[nb][qq], m2, b2[nb][qq]), x);
            if (r.softcap > 0.f) x = soft_cap(x, cap, inv_cap);
            if (r.slopes) x = fmaf(slope[nb][qq], (float)(j0 + row + 1 - q_hi[nb][qq]), x);
            if (!full) {
              const int j = j0 + row;
              const bool on = ((valid >> row) & 1) && j >= q_lo[nb][qq] && j < q_hi[nb][qq];
              x = on ? x : -INFINITY;
            }
            tt[hf][rr][nb][qq] = x;
            const float e = ex2(x - ref[nb][qq]);
            w1[hf][rr][nb][qq] = e * ra[hf][rr];
            w2[hf][rr][nb][qq] = e * rb[hf][rr];
            // not <=: a NaN of 0 * infinity has to go the long way too
            over |= !(fmaxf(fmaxf(w1[hf][rr][nb][qq], w2[hf][rr][nb][qq]), e * 0x1p-40f) <=
                      kMaxWeight);
          }
      }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float f[QT];
#pragma unroll
        for (int qq = 0; qq < QT; ++qq) {
          float mx = kNoRef;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = tt[k >> 1][k & 1][nb][qq];
            const float a = lg2(fmaxf(fmaxf(ra[k >> 1][k & 1], rb[k >> 1][k & 1]), 0x1p-40f));
            if (x > -INFINITY) mx = fmaxf(mx, x + a);
          }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          const float to = fmaxf(ref[nb][qq], mx);
          f[qq] = ex2(ref[nb][qq] - to);
          ref[nb][qq] = to;
          l[nb][qq] *= f[qq];
          w1s[nb][qq] *= f[qq];
          w2s[nb][qq] *= f[qq];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[nb][i][k] *= f[HILO ? 0 : k & 1];
      }
    }
    uint32_t p1[2][NB][2], p2[2][NB][2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int rr = 0; rr < 2; ++rr)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float u1[2], u2[2];
#pragma unroll
          for (int qq = 0; qq < QT; ++qq) {
            const float x = tt[hf][rr][nb][qq];
            const float e = ex2(x - ref[nb][qq]);
            l[nb][qq] += e;
            float v1 = e * ra[hf][rr], v2 = e * rb[hf][rr];
            if (!full && x == -INFINITY) v1 = v2 = 0.f;  // whatever the row's norms hold
            if constexpr (HILO) {
              w1s[nb][0] += v1;
              w2s[nb][0] += v2;
              u1[0] = v1;
              u2[0] = v2;
              u1[1] = (v1 - round_h(v1)) * kPart;
              u2[1] = (v2 - round_h(v2)) * kPart;
            } else {
              u1[qq] = round_h(v1);
              u2[qq] = round_h(v2);
              w1s[nb][qq] += u1[qq];
              w2s[nb][qq] += u2[qq];
            }
          }
          p1[hf][nb][rr] = transpose8(pack_h2(u1[0], u1[1]));
          p2[hf][nb][rr] = transpose8(pack_h2(u2[0], u2[1]));
        }

    // values
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
          uint32_t x0 = __byte_perm(r0, r1, sel), x1 = __byte_perm(r2, r3, sel);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t a[4];
            if constexpr (EXACT) {
              const int s0 = 15 - 2 * i, s1x = 14 - 2 * i;
              a[0] = ((x0 << s0) & 0x80008000u) ^ 0xBC00BC00u;
              a[1] = ((x0 << s1x) & 0x80008000u) ^ 0xBC00BC00u;
              a[2] = ((x1 << s0) & 0x80008000u) ^ 0xBC00BC00u;
              a[3] = ((x1 << s1x) & 0x80008000u) ^ 0xBC00BC00u;
            } else {
              if (i == 4) {
                x0 >>= 8;
                x1 >>= 8;
              }
              const uint32_t m0 = 0x00010001u << ((2 * i) & 7), m1 = m0 << 1;
              a[0] = x0 & m0;
              a[1] = x0 & m1;
              a[2] = x1 & m0;
              a[3] = x1 & m1;
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              const uint32_t(&f)[2] = p == 0 ? p1[hf][nb] : p2[hf][nb];
              mma16816(acc[nb][8 * v + i], a[0], a[1], a[2], a[3], f[0], f[1]);
            }
          }
        }
      }
    __syncwarp();
    issue(tile + (kStages - 1) * kWarps, (n + kStages - 1) % kStages, next_page);
    next_page = page_of(tile + kStages * kWarps);
  }
  if (!P.pre_tensor) grid_dependents_launch();
  cp_wait<0>();
  __syncthreads();

  // ---- the warps' sums: element e of query y of warp w in out[w][y][e]
  float* out = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int qq = 0; qq < QT; ++qq) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[nb][qq] += __shfl_xor_sync(0xffffffffu, l[nb][qq], o);
        w1s[nb][qq] += __shfl_xor_sync(0xffffffffu, w1s[nb][qq], o);
        w2s[nb][qq] += __shfl_xor_sync(0xffffffffu, w2s[nb][qq], o);
      }
      const int y = nb * QB + (HILO ? t : 2 * t + qq);
      if (g == 0) {
        rec_m[warp][y] = ref[nb][qq];
        rec_l[warp][y] = l[nb][qq];
      }
      const float base = (EXACT ? 0.f : -w1s[nb][qq] - w2s[nb][qq]) + (cm / ch) * w1s[nb][qq];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int bit = 2 * (i & 7) + k;
          const int e = (D == 128 ? 16 * g : 32 * g + 16 * (i >> 3)) + bit;
          float v = HILO ? fmaf(acc[nb][i][2 * k + 1], 1.f / kPart, acc[nb][i][2 * k])
                         : acc[nb][i][2 * k + qq];
          if (!EXACT) v *= (float)(1 << (25 - (bit & 7)));  // 2 sum w bit
          out[(warp * NQ + y) * D + e] = v + base;
        }
    }
  }
  __syncthreads();
  const int part = pre ? chunk : P.plan.pre_chunks + chunk;
  for (int y = warp; y < nq; y += kWarps) {
    float mx = rec_m[0][y];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, rec_m[w][y]);
    float f[kWarps], sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      f[w] = ex2(rec_m[w][y] - mx);
      sum = fmaf(rec_l[w][y], f[w], sum);
    }
    float* rec = r.workspace +
                 ((seq_of(y) * hq_all + head_of(y)) * P.plan.parts() + part) * (int64_t)(D + 2);
    if (lane == 0) {
      rec[0] = mx;
      rec[1] = sum;
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v = fmaf(out[(w * NQ + y) * D + 32 * j + lane], f[w], v);
      rec[2 + 32 * j + lane] = v;
    }
  }
  if (P.pre_tensor) grid_dependency_wait();
}

// A block per query row: its records merged, back from the transformed
// domain, divided by l, in the query's type.  What it takes is the time of a
// few dependent loads, so each warp takes every fourth record and loads eight
// of them at once.
template <int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const __grid_constant__ AttnParams P) {
  constexpr int J = D / 32, U = 8;
  const PagedAttnRequest& r = P.r;
  __shared__ float sums[4][D], tops[4], ls[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int hq_all = r.n_kv_heads * r.n_q;
  const uint32_t row = blockIdx.x;
  const uint32_t b = row / hq_all;
  const float* rec = r.workspace + (int64_t)row * P.plan.parts() * (D + 2);
  grid_dependency_wait();
  const int64_t len = length_of(P, b);
  const int64_t own = max((int64_t)0, len - own_first(P, b, len));
  const int n = P.plan.pre_chunks +
                (P.plan.own_rows ? (int)min((own + P.plan.own_rows - 1) / P.plan.own_rows,
                                            (int64_t)P.plan.own_chunks)
                                 : 0);
  float mx = -INFINITY, l = 0.f, a[J];
#pragma unroll
  for (int j = 0; j < J; ++j) a[j] = 0.f;
  for (int p0 = warp; p0 < n; p0 += 4 * U) {
    float mp[U], lp[U], v[U][J], top = mx;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = min(p0 + 4 * u, n - 1);
      const float* q = rec + (int64_t)p * (D + 2);
      mp[u] = q[0];
      lp[u] = p0 + 4 * u < n ? q[1] : 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) v[u][j] = q[2 + 32 * j + lane];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (lp[u] != 0.f) top = fmaxf(top, mp[u]);  // else nothing was attended there
    if (top == -INFINITY) continue;
    const float old = ex2(mx - top);
    l *= old;
#pragma unroll
    for (int j = 0; j < J; ++j) a[j] *= old;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (lp[u] != 0.f) {
        const float f = ex2(mp[u] - top);
        l = fmaf(lp[u], f, l);
#pragma unroll
        for (int j = 0; j < J; ++j) a[j] = fmaf(v[u][j], f, a[j]);
      }
    mx = top;
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

template <int D, bool HILO, bool EXACT, int NB>
kh_status launch_rows(const AttnParams& P, cudaStream_t stream) {
  const PagedAttnRequest& r = P.r;
  constexpr int NQ = NB * (HILO ? 4 : 8);
  using C = RowsCfg<D>;
  auto kern = paged_rows_kernel<D, HILO, EXACT, NB>;
  static_assert(kWarps * NQ * D * 4 <= C::kRing, "the warps' sums take the ring's place");
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KH_ECUDA;
  static std::once_flag once[64];
  std::call_once(once[dev & 63], [&] {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kRing);
  });
  const bool pre = P.plan.pre_chunks > 0 && !P.pre_tensor;
  const int64_t gy = (r.n_seqs + pre) * r.n_kv_heads;
  const int64_t nq = pre ? r.n_seqs * r.n_q : r.n_q;
  const int64_t gz = (nq + NQ - 1) / NQ;
  if (gy > 65535 || gz > 65535) return KH_EINVAL;
  const dim3 grid((unsigned)std::max(pre ? P.plan.pre_chunks : 0, P.plan.own_chunks),
                  (unsigned)gy, (unsigned)gz);
  return launch_programmatic(kern, grid, dim3(32 * kWarps), C::kRing, stream, P) == cudaSuccess
             ? KH_OK
             : KH_ELAUNCH;
}

template <int D>
kh_status launch_dim(const AttnParams& P, cudaStream_t stream) {
  const PagedAttnRequest& r = P.r;
  const int64_t rows = r.n_seqs * r.n_kv_heads * r.n_q;
  if (P.plan.pre_chunks > 0 && P.pre_tensor) {
    const kh_status st = launch_paged_prefix(P, stream);
    if (st != KH_OK) return st;
  }
  if (P.plan.own_chunks > 0 || (P.plan.pre_chunks > 0 && !P.pre_tensor)) {
    const int64_t nq = P.plan.pre_chunks > 0 && !P.pre_tensor ? r.n_seqs * r.n_q : r.n_q;
    kh_status st;
    if (r.dtype == KH_F32)
      st = nq > 4 && D == 128 ? launch_rows<D, true, true, D == 128 ? 2 : 1>(P, stream)
                              : launch_rows<D, true, true, 1>(P, stream);
    else if (nq <= 4 || r.dtype == KH_F16)
      st = nq > 4 && D == 128 ? launch_rows<D, true, false, D == 128 ? 2 : 1>(P, stream)
                              : launch_rows<D, true, false, 1>(P, stream);
    else
      st = nq > 8 && D == 128 ? launch_rows<D, false, false, D == 128 ? 2 : 1>(P, stream)
                              : launch_rows<D, false, false, 1>(P, stream);
    if (st != KH_OK) return st;
  }
  if (launch_programmatic(paged_combine_kernel<D>, dim3((unsigned)rows), dim3(128), 0,
                          stream, P) != cudaSuccess)
    return KH_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? KH_OK : KH_ELAUNCH;
}

}  // namespace

// From how many query rows a KV head's prefix is worth 128-row products.
constexpr int64_t kPrefixTensorRows = 33;

// The workspace: the records, then (16-byte aligned) the transformed queries
// of a tensor-core prefix.
int64_t paged_records_bytes(const PagedPlan& p, int64_t rows, int D) {
  return (rows * p.parts() * (int64_t)(D + 2) * 4 + 15) / 16 * 16;
}
int64_t paged_workspace_bytes(const PagedPlan& p, int64_t n_seqs, int n_q, int n_kv_heads, int D) {
  const int64_t nq = n_seqs * n_q;
  int64_t n = paged_records_bytes(p, nq * n_kv_heads, D);
  if (p.pre_chunks > 0 && nq >= kPrefixTensorRows) n += paged_queries_bytes(nq, n_kv_heads, D);
  return n;
}

PagedPlan paged_plan(int64_t n_seqs, int n_q, int n_kv_heads, int D, int64_t max_len,
                     int64_t prefix_len, int64_t window, int n_sms) {
  PagedPlan p;
  // Two rounds of the CTAs that fit (4 an SM), so that uneven sequences even
  // out, but at least a tile for each warp of a CTA and at most 16.
  const int64_t qb = (n_q + 3) / 4;
  auto chunk_of = [&](int64_t rows) {
    const int64_t even = (rows / (8 * (int64_t)n_sms) + 127) / 128 * 128;
    return std::max<int64_t>(128, std::min<int64_t>(2048, even));
  };
  const int64_t pre = std::min(prefix_len, max_len);
  int64_t own = max_len - pre;
  if (window > 0) own = std::min(own, window);
  if (pre > 0) {
    const int64_t nq = n_seqs * n_q;
    if (nq >= kPrefixTensorRows) {
      // one round of CTAs, one an SM, in whole tiles
      const int64_t per = D == 128 ? 256 : 128, tile = D == 128 ? 128 : 64;
      const int64_t ctas = std::max<int64_t>(1, n_sms / (n_kv_heads * ((nq + per - 1) / per)));
      p.pre_rows = ((pre + ctas - 1) / ctas + tile - 1) / tile * tile;
    } else {
      p.pre_rows = chunk_of(pre * n_kv_heads * ((nq + 7) / 8));
    }
    p.pre_chunks = (int)((pre + p.pre_rows - 1) / p.pre_rows);
  }
  if (own > 0) {
    p.own_rows = chunk_of(n_seqs * n_kv_heads * qb * own);
    p.own_chunks = (int)((own + p.own_rows - 1) / p.own_rows);
  }
  return p;
}

kh_status launch_paged_attn(const PagedAttnRequest& r, cudaStream_t stream) {
  AttnParams P;
  P.r = r;
  P.plan = paged_plan(r.n_seqs, r.n_q, r.n_kv_heads, r.D, r.max_len, r.prefix_len, r.window,
                      sm_count());
  const double sd = std::sqrt((double)r.D);
  P.log_scale = (float)(r.sm_scale * 1.4426950408889634 / sd);
  P.inv_sd = (float)(1.0 / sd);
  int bits = 0;
  while ((int64_t(1) << bits) < r.page_size) ++bits;
  P.pre_tensor = P.plan.pre_chunks > 0 && r.dtype == KH_BF16 && r.c0 == -r.c1 &&
                 r.n_seqs * r.n_q >= kPrefixTensorRows;
  P.queries = reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(r.workspace) +
                                          paged_records_bytes(P.plan, r.n_seqs * r.n_q * r.n_kv_heads, r.D));
  P.div_shift = 31 + bits;
  P.div_mul = ((uint64_t(1) << P.div_shift) + r.page_size - 1) / r.page_size;
  P.err = device_error_ptr();
  return r.D == 128 ? launch_dim<128>(P, stream) : launch_dim<256>(P, stream);
}

}  // namespace kh
