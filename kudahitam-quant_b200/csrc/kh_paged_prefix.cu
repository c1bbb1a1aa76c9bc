// kh_paged_prefix.cu -- attention of many query rows over the shared prefix of
// a paged packed cache, on the 5th-generation tensor cores.
//
// One CTA takes a chunk of the prefix, one KV head and up to 256 query rows
// (128 at D = 256): every sequence's queries of that head.  With that many
// queries a row is worth decoding into fp16 once, and both products are
// 128-row tiles of tcgen05.mma:
//   S = Q~ K^      (queries x rows, accumulator in tensor memory)
//   O += W V^      (W = weights, fp16, back in S's columns as the operand)
// Row scales stay out of the tiles: K^ and V^ rows are divided by their
// largest possible element (so any norm fits fp16), the scale multiplies the
// column of S, or the weight, in 32 bits.  Each element is the sum of two
// signed constants: a shift, a logic operation per plane and one packed add
// for two elements, since elements 32 w + e and 32 w + e + 16 are neighbours
// in the tile (the order of elements is free as long as Q~ and the output
// follow it) and so move to the sign positions of one register together.
//
// Roles: 4 warps a query tile for the softmax, a thread per query row; 4 warps
// that decode, a thread per cached row; 1 warp whose first lane issues the
// products.  At D = 128 two query tiles alternate, so that one's exponentials
// run beside the other's products; at D = 256 one tile alternates between two
// score buffers.  The reference exponent of a row moves only when a weight
// would pass 2^12: then the tile's weights are taken again and O rescaled.
//
// Rounding to 16 bits: q~, K^, the weights and V^ to fp16 (half a step 2^-12
// each); sums, exponents and l in 32 bits.  That is under a result of
// bf16's own half step (2^-9), so only bf16 queries take this path.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "kh_paged_attn.cuh"
#include "kh_tcgen05.cuh"

namespace kh {
namespace {

template <int D>
struct PreCfg {
  static constexpr int MT = D == 128 ? 2 : 1;          // query tiles
  static constexpr int ROWS = D == 128 ? 128 : 64;     // cached rows a tile
  static constexpr int kBoxes = D / 64;                // 64-element blocks of a row
  static constexpr int kQTile = kBoxes * 128 * 128;    // bytes
  static constexpr int kKvBox = ROWS * 128;
  static constexpr int kKvTile = kBoxes * kKvBox;
  static constexpr int kGroup = MT * kQTile + 16;      // a CTA's queries in the workspace
  static constexpr int kOffK = MT * kQTile;
  static constexpr int kOffV = kOffK + 2 * kKvTile;
  static constexpr int kOffScale = kOffV + 2 * kKvTile;  // [2][kappa ROWS, r ROWS] floats
  static constexpr int kOffValid = kOffScale + 2 * 2 * ROWS * 4;  // [2][4] masks
  static constexpr int kOffBar = kOffValid + 32;
  static constexpr int kOffMisc = kOffBar + 16 * 8;
  static constexpr int kSmem = 1024 + kOffMisc + 16;
  static constexpr int kSoftWarps = 4 * MT;
  static constexpr int kThreads = 32 * (kSoftWarps + 4 + 1);
  static constexpr uint32_t kTmemCols = 512;
  static constexpr uint32_t kColO = D == 128 ? 256 : 128;  // O's first column
  static constexpr uint32_t kColS = D == 128 ? 128 : 64;   // S buffers apart
  static_assert(kSmem <= 232448, "exceeds the shared memory of a CTA");
  // the sums of 128 queries leave through the tiles' place
  static_assert(MT * 128 * (D + 1) * 4 <= kOffScale, "staging of the sums");
};

// Queries are stored times a power of two that keeps the largest |q~| of the
// CTA under 2^14: fp16 holds elements 2^28 below that with full steps.
__device__ __forceinline__ float query_scale(float bound) {
  int e = 0;
  if (bound > 0.f && bound < INFINITY) frexpf(bound, &e);
  return ldexpf(1.f, max(-120, min(120, 14 - e)));
}

// Q~ of 128 MT query rows of one KV head, as the products' operand: tiles of
// 128 rows, element e at position 2 (e & 15) + (e >> 4 & 1) of its block of
// 32, 128-byte blocks swizzled; times log_scale and the power of two that the
// last 4 bytes of the group hold.  Once per call, not per chunk: a warp's
// transforms cost 4 us for 256 rows, as much as a chunk's products.
template <int D>
__global__ void __launch_bounds__(1024) paged_queries_kernel(const __grid_constant__ AttnParams P) {
  using C = PreCfg<D>;
  constexpr int W = D / 32, PER = C::MT * 4;  // query rows a warp
  const PagedAttnRequest& r = P.r;
  __shared__ uint32_t bound;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y;
  const int n_rows = (int)(r.n_seqs * r.n_q);
  const int y0 = blockIdx.x * (C::MT * 128);
  const uint16_t* q16 = static_cast<const uint16_t*>(r.q);
  if (threadIdx.x == 0) bound = 0u;
  __syncthreads();
  grid_dependency_wait();
  grid_dependents_launch();
  float x[PER][W], mx = 0.f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = y0 + warp * PER + k;
    const int b = i / r.n_q;
    const int64_t row = (int64_t)b * r.n_kv_heads * r.n_q + h * r.n_q + (i - b * r.n_q);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      x[k][j] = i < n_rows ? __uint_as_float((uint32_t)q16[row * D + 32 * j + lane] << 16) : 0.f;
      mx = fmaxf(mx, fabsf(x[k][j]));
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) atomicMax(&bound, __float_as_uint(mx));
  __syncthreads();
  const float up = query_scale(__uint_as_float(bound) * (float)D * fabsf(P.log_scale));
  uint8_t* group = reinterpret_cast<uint8_t*>(P.queries) +
                   (int64_t)(h * gridDim.x + blockIdx.x) * C::kGroup;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int y = warp * PER + k, row = y & 127;
#pragma unroll
    for (int j = 0; j < W; ++j)
      if ((r.dk_neg[j] >> lane) & 1) x[k][j] = -x[k][j];
    fwht_lanes<W>(x[k], lane);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const int pos = 32 * j + 2 * (lane & 15) + (lane >> 4);
      const int c = (pos & 63) >> 3;
      *reinterpret_cast<__half*>(group + (y >> 7) * C::kQTile + (pos >> 6) * (128 * 128) +
                                 row * 128 + ((c ^ (row & 7)) << 4) + (pos & 7) * 2) =
          __float2half_rn(x[k][j] * (P.log_scale * up));
    }
  }
  if (threadIdx.x == 0) *reinterpret_cast<float*>(group + C::MT * C::kQTile) = up;
}

template <int D, bool EXTRA>
__global__ void __launch_bounds__(PreCfg<D>::kThreads, 1)
    paged_prefix_kernel(const __grid_constant__ AttnParams P) {
  using C = PreCfg<D>;
  constexpr int W = D / 32, ROWS = C::ROWS, MT = C::MT;
  constexpr uint32_t kIdescS = make_idesc(false, 128, ROWS);
  constexpr uint32_t kIdescO = make_idesc(false, 128, D) | kIdescTransposeB;
  const PagedAttnRequest& r = P.r;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::kOffBar);
  uint64_t *kfull = bars, *kempty = bars + 2, *vfull = bars + 4, *vempty = bars + 6,
           *sfull = bars + 8, *pfull = bars + 10, *odone = bars + 12, *qfull = bars + 14;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::kOffMisc);
  const uint8_t* group = reinterpret_cast<const uint8_t*>(P.queries) +
                         (int64_t)(blockIdx.y * gridDim.z + blockIdx.z) * C::kGroup;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int h = blockIdx.y;
  const int64_t n_rows = r.n_seqs * r.n_q;
  const int64_t y0 = (int64_t)blockIdx.z * (MT * 128);
  const int nq = (int)min((int64_t)(MT * 128), n_rows - y0);
  const int lo = (int)(blockIdx.x * P.plan.pre_rows);
  const int hi = (int)min(lo + P.plan.pre_rows, r.prefix_len);
  const int n_tiles = (hi - lo + ROWS - 1) / ROWS;
  const int hq_all = r.n_kv_heads * r.n_q;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kfull[i], 4);
      mbar_init(&kempty[i], 1);
      mbar_init(&vfull[i], 4);
      mbar_init(&vempty[i], 1);
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 4);
      mbar_init(&odone[i], 1);
    }
    mbar_init(qfull, 32 * C::kSoftWarps);
    fence_mbar_init();
  }
  if (warp == C::kSoftWarps + 4) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto query_row = [&](int y) {
    const int64_t i = y0 + y;
    const int64_t b = i / r.n_q;
    return b * hq_all + h * r.n_q + (int)(i - b * r.n_q);
  };

  if (warp >= C::kSoftWarps && warp < C::kSoftWarps + 4) {
    // ------------------------------------------------------------ decoding
    const int i = threadIdx.x - 32 * C::kSoftWarps;  // row of the tile
    // at D = 256 a row is two threads', half its words each
    constexpr int kSplit = 128 / ROWS;
    constexpr int WT = W / kSplit;
    const int row = i % ROWS, part = i / ROWS;
    struct Row {
      uint32_t kc[WT], kr[WT], vc[WT], vr[WT];
      float kn, krn, vn, vrn;
      bool on;
    };
    auto page_of = [&](int t) {
      const uint32_t j = lo + t * ROWS + row;
      return (t < n_tiles && (int)j < hi) ? r.table[P.page_div(j)] : -1;
    };
    auto fetch = [&](int t, int page) {
      Row x;
      const uint32_t j = lo + t * ROWS + row;
      const bool in = t < n_tiles && (int)j < hi;
      x.on = in && (uint32_t)page < (uint32_t)r.n_pages;
      if (in && !x.on) flag_error(P.err, kErrBadIndex);
      x.kn = x.krn = x.vn = x.vrn = 0.f;
#pragma unroll
      for (int w = 0; w < WT; ++w) x.kc[w] = x.kr[w] = x.vc[w] = x.vr[w] = 0u;
      if (x.on) {
        const uint32_t off = j - P.page_div(j) * r.page_size;
        const int64_t at = ((int64_t)page * r.n_kv_heads + h) * r.page_size + off;
        auto take = [&](const uint32_t* plane, uint32_t(&to)[WT]) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(plane + at * W) + part);
          to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
        };
        static_assert(WT == 4, "a thread decodes 128 elements");
        take(r.kp.code, x.kc);
        take(r.kp.res, x.kr);
        take(r.vp.code, x.vc);
        take(r.vp.res, x.vr);
        x.kn = __ldg(r.kp.norms + at);
        x.krn = __ldg(r.kp.rnorms + at);
        x.vn = __ldg(r.vp.norms + at);
        x.vrn = __ldg(r.vp.rnorms + at);
      }
      return x;
    };
    // +-a +-b for 128 elements, divided by what the row's scale takes out
    auto write = [&](uint8_t* tile, const uint32_t(&code)[WT], const uint32_t(&res)[WT], float a,
                     float b) {
      constexpr uint32_t M = 0x80008000u;
      const uint32_t pa = pack_h2(a, a) ^ M, pb = pack_h2(b, b) ^ M;
#pragma unroll
      for (int w = 0; w < WT; ++w) {
        const int word = part * WT + w;
        uint32_t v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t t0 = ((code[w] << (15 - e)) & M) ^ pa;
          const uint32_t t1 = ((res[w] << (15 - e)) & M) ^ pb;
          asm("add.rn.f16x2 %0, %1, %2;" : "=r"(v[e]) : "r"(t0), "r"(t1));
        }
        uint8_t* at = tile + (word >> 1) * C::kKvBox + row * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<uint4*>(at + ((((word & 1) * 4 + c) ^ (row & 7)) << 4)) =
              make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
      }
    };
    // A row's two constants divided by the larger, which is returned: any two
    // norms fit fp16.  Norms that are not finite give a row of zeros and
    // leave through the scale, which masked places do not take.
    auto scaled = [&](float& a, float& b) {
      const float m = fmaxf(fabsf(a), fabsf(b));
      if (!(m > 1e-35f && m < INFINITY) || a != a || b != b) {
        const bool none = fabsf(a) <= 1e-35f && fabsf(b) <= 1e-35f;
        a = b = 0.f;
        return none ? 0.f : NAN;
      }
      const float inv = 1.f / m;
      a *= inv;
      b *= inv;
      return m;
    };
    const float inv_sd = P.inv_sd;
    float down = 1.f;
    int page = page_of(0);
    Row x = fetch(0, page);
    page = page_of(1);
    for (int t = 0; t < n_tiles; ++t) {
      const int s = t & 1;
      const uint32_t ph = (uint32_t)((t >> 1) & 1);
      float ka = x.kn * r.c1, kb = x.krn * inv_sd;
      float va = x.vn * r.c1 * inv_sd, vb = x.vrn * (0.7978845608028654f * inv_sd * inv_sd);
      const float kappa = scaled(ka, kb), rv = scaled(va, vb);
      if (!__all_sync(0xffffffffu, mbar_wait(&kempty[s], ph ^ 1u, P.err))) break;
      write(sm + C::kOffK + s * C::kKvTile, x.kc, x.kr, ka, kb);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kfull[s]);
      if (t == 0) {
        // everything before the queries' launch was done when this grid could
        // start, so only their scale has to be waited for
        grid_dependency_wait();
        down = 1.f / *reinterpret_cast<const float*>(group + MT * C::kQTile);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&vempty[s], ph ^ 1u, P.err))) break;
      write(sm + C::kOffV + s * C::kKvTile, x.vc, x.vr, va, vb);
      if (part == 0) {
        float* sc = reinterpret_cast<float*>(sm + C::kOffScale) + s * 2 * ROWS;
        sc[row] = kappa * down;
        sc[ROWS + row] = rv;
        const uint32_t mask = __ballot_sync(0xffffffffu, x.on);
        if (lane == 0)
          reinterpret_cast<uint32_t*>(sm + C::kOffValid)[s * 4 + (row >> 5)] = mask;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&vfull[s]);
      x = fetch(t + 1, page);
      page = page_of(t + 2);
    }
  } else if (warp == C::kSoftWarps + 4) {
    // ------------------------------------------------------------ products
    grid_dependency_wait();
    grid_dependents_launch();
    if (lane == 0) {
      auto scores = [&](int m, int s, int buf) {
        const uint32_t d = tmem + buf * C::kColS;
        const uint32_t qa = base + m * C::kQTile, ka = base + C::kOffK + s * C::kKvTile;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t ad = sw128_desc(qa + (k >> 2) * (128 * 128)) + 2 * (k & 3);
          const uint64_t bd = sw128_desc(ka + (k >> 2) * C::kKvBox) + 2 * (k & 3);
          umma_f16(d, ad, bd, kIdescS, k != 0);
        }
      };
      auto values = [&](int m, int s, int buf, bool more) {
        const uint32_t d = tmem + C::kColO + m * 128;
        const uint32_t pa = tmem + buf * C::kColS, va = base + C::kOffV + s * C::kKvTile;
#pragma unroll
        for (int k = 0; k < ROWS / 16; ++k)
          umma_f16_ta(d, pa + 8 * k, sw128_desc_mn(va + k * 2048, C::kKvBox), kIdescO,
                      more || k != 0);
      };
      bool ok = mbar_wait(qfull, 0, P.err) && mbar_wait(&kfull[0], 0, P.err);
      if (ok) {
        tc_fence_after();
        for (int m = 0; m < MT; ++m) {
          scores(m, 0, m);
          umma_commit(&sfull[m]);
        }
        umma_commit(&kempty[0]);
      }
      for (int t = 0; ok && t < n_tiles; ++t) {
        const int s = t & 1, s1 = s ^ 1;
        const uint32_t ph = (uint32_t)((t >> 1) & 1), ph1 = (uint32_t)(((t + 1) >> 1) & 1);
        const bool next = t + 1 < n_tiles;
        if (MT == 1 && next) {  // the other buffer's scores run beside this tile's softmax
          if (!(ok = mbar_wait(&kfull[s1], ph1, P.err))) break;
          tc_fence_after();
          scores(0, s1, s1);
          umma_commit(&sfull[s1]);
          umma_commit(&kempty[s1]);
        }
        if (!(ok = mbar_wait(&vfull[s], ph, P.err))) break;
        for (int m = 0; m < MT; ++m) {
          const int buf = MT == 2 ? m : s;
          if (!(ok = mbar_wait(&pfull[MT == 2 ? m : 0], (uint32_t)(t & 1), P.err))) break;
          tc_fence_after();
          values(m, s, buf, t != 0);
          umma_commit(&odone[m]);
          if (m == MT - 1) umma_commit(&vempty[s]);
          if (MT == 2 && next) {
            // the products run in order: the weights have been read when the
            // scores that take their columns are written
            if (m == 0 && !(ok = mbar_wait(&kfull[s1], ph1, P.err))) break;
            tc_fence_after();
            scores(m, s1, m);
            umma_commit(&sfull[m]);
            if (m == 1) umma_commit(&kempty[s1]);
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int m = warp >> 2, quarter = warp & 3;
    const int y = m * 128 + quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    // the queries, transformed by the launch before this one
    grid_dependency_wait();
    for (int k = threadIdx.x; k < MT * C::kQTile / 16; k += 32 * C::kSoftWarps)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + 16 * k),
                   "l"(group + 16 * k)
                   : "memory");
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_proxy_async_smem();
    mbar_arrive(qfull);
    int q_lo = 0, q_hi = 0;
    float slope = 0.f;
    if (y < nq) {
      const int64_t b = (y0 + y) / r.n_q;
      const int64_t len = length_of(P, b);
      q_hi = (int)len;
      q_lo = (int)min(first_of(P, b, len), (int64_t)0x7fffffff);
      if (EXTRA && r.slopes) slope = r.slopes[h * r.n_q + (int)((y0 + y) - b * r.n_q)] * kLog2e;
    }
    const float cap = r.softcap * kLog2e, inv_cap = r.softcap > 0.f ? 1.f / cap : 0.f;
    float ref = kNoRef, l = 0.f;
    bool ok = true;
    for (int t = 0; ok && t < n_tiles; ++t) {
      const int s = t & 1, buf = MT == 2 ? m : s;
      const int j0 = lo + t * ROWS;
      ok = mbar_wait(&vfull[s], (uint32_t)((t >> 1) & 1), P.err);
      ok = ok && mbar_wait(&sfull[buf], (uint32_t)(MT == 2 ? t & 1 : (t >> 1) & 1), P.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const float* kap = reinterpret_cast<const float*>(sm + C::kOffScale) + s * 2 * ROWS;
      const float* rv = kap + ROWS;
      const uint32_t* valid = reinterpret_cast<const uint32_t*>(sm + C::kOffValid) + s * 4;
      bool whole = j0 >= q_lo && j0 + ROWS <= q_hi;
#pragma unroll
      for (int c = 0; c < ROWS / 32; ++c) whole = whole && valid[c] == 0xffffffffu;
      // places of chunk c that this query attends
      auto places = [&](int c) {
        const int a = max(q_lo - (j0 + 32 * c), 0), z = min(q_hi - (j0 + 32 * c), 32);
        if (a >= z) return 0u;
        const uint32_t below = z == 32 ? 0xffffffffu : (1u << z) - 1u;
        return valid[c] & below & (0xffffffffu << a);
      };
      // exponents of chunk c, without the reference
      auto exponents = [&](int c, float (&v)[32]) {
        tmem_ld32(tmem + lanes + buf * C::kColS + 32 * c, v);
        tmem_wait_ld();
        if constexpr (EXTRA) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float x = v[i] * kap[32 * c + i];
            if (r.softcap > 0.f) x = soft_cap(x, cap, inv_cap);
            if (r.slopes) x = fmaf(slope, (float)(j0 + 32 * c + i + 1 - q_hi), x);
            v[i] = x;
          }
        }
      };
      uint32_t p[ROWS / 32][16];
      float lt;
      const bool all_whole = __all_sync(0xffffffffu, whole);
      auto pass = [&](auto masked) {
        float2 sum = make_float2(0.f, 0.f);
        float top = 0.f;
        const float2 nref = make_float2(-ref, -ref);
#pragma unroll
        for (int c = 0; c < ROWS / 32; ++c) {
          float v[32];
          exponents(c, v);
          const uint32_t on = decltype(masked)::value ? places(c) : 0u;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 k4 = EXTRA ? make_float4(1.f, 1.f, 1.f, 1.f)
                                    : *reinterpret_cast<const float4*>(kap + 32 * c + i);
            const float4 r4 = *reinterpret_cast<const float4*>(rv + 32 * c + i);
#pragma unroll
            for (int o = 0; o < 4; o += 2) {
              const float2 kk = o ? make_float2(k4.z, k4.w) : make_float2(k4.x, k4.y);
              const float2 rr = o ? make_float2(r4.z, r4.w) : make_float2(r4.x, r4.y);
              float2 x = __ffma2_rn(make_float2(v[i + o], v[i + o + 1]), kk, nref);
              if constexpr (decltype(masked)::value) {
                if (!(on >> (i + o) & 1)) x.x = -INFINITY;
                if (!(on >> (i + o + 1) & 1)) x.y = -INFINITY;
              }
              const float2 e = make_float2(ex2(x.x), ex2(x.y));
              sum = __fadd2_rn(sum, e);
              float2 w = __fmul2_rn(e, rr);
              if constexpr (decltype(masked)::value) {
                if (!(on >> (i + o) & 1)) w.x = 0.f;  // whatever the row's norms hold
                if (!(on >> (i + o + 1) & 1)) w.y = 0.f;
              }
              top = fmaxf(fmaxf(top, w.x), w.y);
              p[c][(i + o) >> 1] = pack_h2(w.x, w.y);
            }
          }
        }
        lt = sum.x + sum.y;
        return !(top <= kMaxWeight && lt < 0x1p60f);
      };
      auto weigh = [&] {
        return all_whole ? pass(std::false_type{}) : pass(std::true_type{});
      };
      bool over = weigh();
      if (__any_sync(0xffffffffu, over)) {
        float top = kNoRef;
#pragma unroll 1
        for (int c = 0; c < ROWS / 32; ++c) {
          float v[32];
          exponents(c, v);
          const uint32_t on = places(c);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float x = EXTRA ? v[i] : v[i] * kap[32 * c + i];
            if (on >> i & 1) top = fmaxf(top, x + lg2(fmaxf(rv[32 * c + i], 0x1p-40f)));
          }
        }
        const float to = fmaxf(ref, top), f = ex2(ref - to);
        ref = to;
        l *= f;
        if (t > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(&odone[m], (uint32_t)((t - 1) & 1), P.err));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            const uint32_t at = tmem + lanes + C::kColO + m * 128 + 32 * c;
            float v[32];
            uint32_t u[32];
            tmem_ld32(at, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(v[i] * f);
            tmem_st32(at, u);
          }
          tmem_wait_st();
        }
        weigh();
      }
      l += lt;
#pragma unroll
      for (int c = 0; c < ROWS / 64; ++c) {
        uint32_t u[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) u[i] = p[2 * c + (i >> 4)][i & 15];
        tmem_st32(tmem + lanes + buf * C::kColS + 32 * c, u);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[m]);
    }
    // ---- the sums leave through the tiles' shared memory
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&odone[m], (uint32_t)((n_tiles - 1) & 1), P.err));
    if (MT == 2) {
      // both query tiles have read Q~, K^ and V^ for the last time
      ok = __all_sync(0xffffffffu, mbar_wait(&odone[m ^ 1], (uint32_t)((n_tiles - 1) & 1), P.err)) && ok;
    }
    tc_fence_after();
    float* out = reinterpret_cast<float*>(sm) + (m * 128 + quarter * 32) * (D + 1);
    if (ok) {
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float v[32];
        tmem_ld32(tmem + lanes + C::kColO + m * 128 + 32 * c, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) out[lane * (D + 1) + 32 * c + (i >> 1) + 16 * (i & 1)] = v[i];
      }
    }
    __syncwarp();
    for (int k = 0; k < 32; ++k) {
      const int yk = m * 128 + quarter * 32 + k;
      if (yk >= nq) break;
      float* rec = r.workspace + (query_row(yk) * P.plan.parts() + blockIdx.x) * (int64_t)(D + 2);
      const float mk = __shfl_sync(0xffffffffu, ref, k), lk = __shfl_sync(0xffffffffu, l, k);
      if (lane == 0) {
        rec[0] = mk;
        rec[1] = ok ? lk : 0.f;
      }
#pragma unroll
      for (int j = 0; j < W; ++j) rec[2 + 32 * j + lane] = out[k * (D + 1) + 32 * j + lane];
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kSoftWarps + 4) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

template <int D>
int64_t queries_bytes(int64_t nq, int n_kv_heads) {
  using C = PreCfg<D>;
  return (nq + 128 * C::MT - 1) / (128 * C::MT) * n_kv_heads * C::kGroup;
}

template <int D, bool EXTRA>
kh_status launch_typed(const AttnParams& P, cudaStream_t stream) {
  using C = PreCfg<D>;
  auto kern = paged_prefix_kernel<D, EXTRA>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KH_ECUDA;
  static std::once_flag once[64];
  std::call_once(once[dev & 63], [&] {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  const int64_t nq = P.r.n_seqs * P.r.n_q, per = 128 * C::MT;
  const dim3 grid((unsigned)P.plan.pre_chunks, (unsigned)P.r.n_kv_heads,
                  (unsigned)((nq + per - 1) / per));
  if (grid.y > 65535 || (nq + per - 1) / per > 65535) return KH_EINVAL;
  if (launch_programmatic(paged_queries_kernel<D>, dim3(grid.z, grid.y), dim3(1024), 0, stream,
                          P) != cudaSuccess)
    return KH_ELAUNCH;
  return launch_programmatic(kern, grid, dim3(C::kThreads), C::kSmem, stream, P) == cudaSuccess
             ? KH_OK
             : KH_ELAUNCH;
}

}  // namespace

int64_t paged_queries_bytes(int64_t nq, int n_kv_heads, int D) {
  return D == 128 ? queries_bytes<128>(nq, n_kv_heads) : queries_bytes<256>(nq, n_kv_heads);
}

kh_status launch_paged_prefix(const AttnParams& P, cudaStream_t stream) {
  const bool extra = P.r.softcap > 0.f || P.r.slopes;
  if (P.r.D == 128)
    return extra ? launch_typed<128, true>(P, stream) : launch_typed<128, false>(P, stream);
  return extra ? launch_typed<256, true>(P, stream) : launch_typed<256, false>(P, stream);
}

}  // namespace kh
