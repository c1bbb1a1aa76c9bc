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
// largest constant or, where a tile's rows are alike, all by one power of two
// (so any norm fits fp16); the scale multiplies the score, or the weight, in
// 32 bits.  Elements 32 w + e and 32 w + e + 16 are neighbours in the tile (the
// order of elements is free as long as Q~ and the output follow it), so that
// one mask serves both.
//
// Roles: 4 warps a query tile for the softmax, a thread per query row; 4 warps
// that decode; 1 thread that issues the products.  At D = 128 two query tiles
// alternate, so that one's exponentials run beside the other's products (two
// buffers of 64 rows each instead of one of 128 measured slower: a product
// 64 wide takes as long as one of 128, both read 4 KB of Q~ a step); at
// D = 256 one tile alternates between two score buffers.  The reference exponent of
// a row moves only when a weight would leave fp16: then the chunk's weights
// are taken again, O and the weights before it rescaled.
//
// What bounds it is that turn-taking: of a tile's 5500 cycles (256 queries x 128
// rows, D = 128) the products take 2600, and tensor memory has no columns left
// for a second set of scores.  128 x 32 bf16 queries over 32768 rows of 8 KV heads
// take 96 us, 715 TFLOP/s.
//
// Rounding to 16 bits: q~, K^, the weights and V^ to fp16 (half a step 2^-11
// each); sums, exponents and l in 32 bits.  That is under a bf16 result's own
// half step (2^-8), so only bf16 queries take this path: results are 1.86e-3 to
// 1.89e-3 off, of which their own rounding is 1.66e-3.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "kh_paged_attn.cuh"
#include "kh_tcgen05.cuh"

namespace kh {
namespace {

// D = 128: the block launches with 4 x 128 registers a lane = 2 x 176 + 112 + 48.
constexpr int kRegsSoft = 176, kRegsDecode = 112, kRegsIssue = 48;

template <int D>
struct PreCfg {
  static constexpr int MT = QueryTiles<D>::MT;         // query tiles
  static constexpr int ROWS = D == 128 ? 128 : 64;     // cached rows a tile
  static constexpr int SB = D == 128 ? 1 : 2;          // score buffers of a query tile
  static constexpr int kBoxes = D / 64;                // 64-element blocks of a row
  static constexpr int kQTile = QueryTiles<D>::kTile;  // bytes
  static constexpr int kKvBox = ROWS * 128;
  static constexpr int kKvTile = kBoxes * kKvBox;
  static constexpr int kStages = 2;                    // of K^ and of V^
  static constexpr int kGroup = QueryTiles<D>::kGroup; // a CTA's queries in the workspace
  static constexpr int kOffK = MT * kQTile;
  static constexpr int kOffV = kOffK + kStages * kKvTile;
  static constexpr int kOffScale = kOffV + kStages * kKvTile;  // {kappa, r} of ROWS columns
  static constexpr int kOffValid = kOffScale + kStages * 2 * ROWS * 4;  // masks of 32 rows
  static constexpr int kOffEven = kOffValid + kStages * 16;  // {kappa, 1 / r, log2 r, even}
  static constexpr int kOffRange = kOffEven + kStages * 16;  // 4 warps' extremes
  static constexpr int kOffBar = kOffRange + kStages * 64;
  static constexpr int kBars = 4 * kStages + 4 + 4 + 2 + 1;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kSmem = 1024 + kOffMisc + 16;
  static constexpr int kSoftWarps = 4 * MT;
  // whole warpgroups, so that the softmax can take registers from the others
  static constexpr int kThreads = 32 * (kSoftWarps + 4 + 4);
  static constexpr uint32_t kTmemCols = 512;
  // tensor memory: the score buffers of ROWS columns, then the sums
  static constexpr uint32_t kColO = SB * MT * ROWS;
  static_assert(kColO + MT * D <= kTmemCols, "tensor memory");
  static_assert(kSmem <= 232448, "exceeds the shared memory of a CTA");
  static_assert(MT * 128 * (D + 1) * 4 <= kOffScale, "the sums leave through the tiles' place");
};

// 2^y for two y: y = n + f with n whole (the sum with 1.5 2^23 rounds to it),
// 2^f on [-1/2, 1/2] by the cubic of least relative error (2^-13.7, found by
// exchange), n added to the exponent.  A quarter of the exponentials go this way: the
// special-function pipe takes 8 cycles for a warp's 32, and two warps' 32
// columns measured 531 cycles with none, 446 with a quarter, 489 with half.
constexpr float kE0 = 0.999928074f, kE1 = 0.693260985f, kE2 = 0.242611122f, kE3 = 0.0551716691f;
__device__ __forceinline__ float2 ex2_poly(float2 y) {
  y = make_float2(fminf(fmaxf(y.x, -126.f), 127.f), fminf(fmaxf(y.y, -126.f), 127.f));
  const float2 big = make_float2(12582912.f, 12582912.f);
  const float2 n = __fadd2_rn(y, big);
  const float2 f = __fadd2_rn(y, __ffma2_rn(n, make_float2(-1.f, -1.f), big));
  float2 p = __ffma2_rn(f, make_float2(kE3, kE3), make_float2(kE2, kE2));
  p = __ffma2_rn(p, f, make_float2(kE1, kE1));
  p = __ffma2_rn(p, f, make_float2(kE0, kE0));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(n.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(n.y) << 23)));
}

// Rows are decoded so that their largest constant becomes this or less: then
// 2^25 times it is in fp16's range.
constexpr float kTileScale = 0x1p-11f;

// fp16 ends at 65504; 32 weights with this sum are all below it.
constexpr float kMostSum = 32768.f;

// A moved reference puts the largest weight just under 2^kLift: fp16's fixed steps
// (2^-24, below 2^-14) are then 2^-32 of it, so that a long tail of small weights
// is not rounded to one side by much of itself (from 2^0, 131072 alike rows with 0.13
// of the weight were 2.5% off), and 32 as large ones still fit kMostSum four times.
constexpr float kLift = 8.f;

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Barrier of the four decoding warps, true where `in` is for all of them.
__device__ __forceinline__ bool decoders_agree(bool in) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "barrier.cta.red.and.pred p, 1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)in)
      : "memory");
  return all != 0;
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
  constexpr int NS = C::kStages;
  // sfull and pfull by score buffer: SB m + t % SB
  uint64_t *kfull = bars, *kempty = kfull + NS, *vfull = kempty + NS, *vempty = vfull + NS,
           *sfull = vempty + NS, *pfull = sfull + 4, *odone = pfull + 4, *qfull = odone + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::kOffMisc);
  const uint8_t* group = reinterpret_cast<const uint8_t*>(P.queries) +
                         (int64_t)(blockIdx.y * gridDim.z + blockIdx.z) * C::kGroup;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int h = blockIdx.y;
  const int64_t n_rows = r.n_seqs * r.n_q;
  const int64_t y0 = (int64_t)blockIdx.z * (MT * 128);
  const int nq = (int)min((int64_t)(MT * 128), n_rows - y0);
  const int lo = (int)(blockIdx.x * P.plan.chunk_rows);
  const int hi = (int)min(lo + P.plan.chunk_rows, r.prefix_len);
  const int n_tiles = (hi - lo + ROWS - 1) / ROWS;
  const int hq_all = r.n_kv_heads * r.n_q;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kfull[i], 4);
      mbar_init(&kempty[i], 1);
      mbar_init(&vfull[i], 4);
      mbar_init(&vempty[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 4);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&odone[i], 1);
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
    if constexpr (D == 128) fewer_registers<kRegsDecode>();
    grid_dependency_wait();
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
    const int32_t* table = r.table + P.units->source * r.table_stride;
    const int end = (int)min((int64_t)hi, P.units->pre_end);
    auto page_of = [&](int t) {
      const uint32_t j = lo + t * ROWS + row;
      return (t < n_tiles && (int)j < end) ? table[P.page_div(j)] : -1;
    };
    auto fetch = [&](int t, int page) {
      Row x;
      const uint32_t j = lo + t * ROWS + row;
      const bool in = t < n_tiles && (int)j < end;
      x.on = in && (uint32_t)page < (uint32_t)r.n_pages;
      if (in && !x.on) flag_error(P.err, kErrBadIndex);
      x.kn = x.krn = x.vn = x.vrn = 0.f;
#pragma unroll
      for (int w = 0; w < WT; ++w) x.kc[w] = x.kr[w] = x.vc[w] = x.vr[w] = 0u;
      if (x.on) {
        const uint32_t off = j - P.page_div(j) * r.page_size;
        const int64_t at = ((int64_t)page * r.n_kv_heads + h) * r.page_size + off;
        auto take = [&](const uint32_t* plane, uint32_t(&to)[WT]) {
          if constexpr (WT == 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(plane + at * W) + part);
            to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
          } else {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(plane + at * W) + part);
            to[0] = v.x; to[1] = v.y;
          }
        };
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
    // The thread's words decoded: the bits masked to b = 0 .. 7 are fp16
    // numbers 2^(b - 24), exact factors of 2 a 2^(24 - b); what both planes'
    // zeros stand for is added.
    // A logic operation and a multiply-add for two elements of a plane, where
    // moving bits to the sign took a shift and a logic operation, both on the
    // pipe that the softmax's conversions need.
    auto write = [&](uint8_t* tile, const uint32_t(&code)[WT], const uint32_t(&res)[WT], float a,
                     float b, float least) {
      uint32_t fa[8], fb[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float up = (float)(1 << (25 - k));
        fa[k] = pack_h2(a * up, a * up);
        fb[k] = pack_h2(b * up, b * up);
      }
      const uint32_t low = pack_h2(least, least);
#pragma unroll
      for (int w = 0; w < WT; ++w) {
        const int word = part * WT + w;
        uint32_t v[16], c = code[w], s = res[w];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (e == 8) {
            c >>= 8;
            s >>= 8;
          }
          const uint32_t m = 0x00010001u << (e & 7);
          asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v[e]) : "r"(c & m), "r"(fa[e & 7]), "r"(low));
          asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(v[e]) : "r"(s & m), "r"(fb[e & 7]));
        }
        uint8_t* at = tile + (word >> 1) * C::kKvBox + row * 128;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<uint4*>(at + ((((word & 1) * 4 + k) ^ (row & 7)) << 4)) =
              make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
      }
    };
    // The larger of a row's two constants, a times a level and b: what it is
    // divided by, so that any two norms fit
    // fp16.  Norms that are not finite give a row of zeros and leave through
    // the scale, which masked places do not take.
    const float c_most = fmaxf(fabsf(r.c0), fabsf(r.c1)), c_half = 0.5f * (r.c1 - r.c0);
    auto largest = [&](float& a, float& b) {
      const float m = fmaxf(fabsf(a) * c_most, fabsf(b));
      if (!(m > 1e-35f && m < 1e35f) || a != a || b != b) {
        const bool none = m <= 1e-35f && a == a && b == b;
        a = b = 0.f;
        return none ? 0.f : NAN;
      }
      return m;
    };
    const float inv_sd = P.inv_sd;
    // two tiles' rows on their way while one is decoded, their pages one ahead
    Row now = fetch(0, page_of(0)), next = fetch(1, page_of(1));
    int page = page_of(2);
    bool in = true;  // no wait has given up
#pragma unroll 1
    for (int t = 0; t < n_tiles; ++t) {
      const int s = t % NS;
      const uint32_t ph = (uint32_t)((t / NS) & 1);
      Row x = now;
      now = next;
      next = fetch(t + 2, page);
      page = page_of(t + 3);
      float ka = x.kn, kb = x.krn * inv_sd;
      float va = x.vn * inv_sd, vb = x.vrn * (0.7978845608028654f * inv_sd * inv_sd);
      float kappa = largest(ka, kb), rv = largest(va, vb);
      // Where the tile's rows are all there and their scales lie within 2^10 of
      // one another, one power of two serves them all: fp16 still gives every
      // row its full steps, and the softmax needs no scale per column.
      float* range = reinterpret_cast<float*>(sm + C::kOffRange) + s * 16;
      {
        const float k0 = x.on ? kappa : NAN, v0 = x.on ? rv : NAN;
        float most[2] = {k0, v0}, least[2] = {k0, v0};
        const bool odd = __any_sync(0xffffffffu, !(k0 > 0.f) || !(v0 > 0.f));
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int o = 16; o; o >>= 1) {
            most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], o));
            least[i] = fminf(least[i], __shfl_xor_sync(0xffffffffu, least[i], o));
          }
        if (lane == 0)
          *reinterpret_cast<float4*>(range + 4 * (warp - C::kSoftWarps)) =
              make_float4(odd ? INFINITY : most[0], least[0], most[1], least[1]);
      }
      // a warp whose wait gave up comes here too, so that the four leave together
      if (!decoders_agree(in)) break;
      float4 all = *reinterpret_cast<const float4*>(range);
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float4 q = *reinterpret_cast<const float4*>(range + 4 * w);
        all = make_float4(fmaxf(all.x, q.x), fminf(all.y, q.y), fmaxf(all.z, q.z), fminf(all.w, q.w));
      }
      const bool even = all.x <= 1024.f * all.y && all.z <= 1024.f * all.w;
      int ve = 0;
      float ki, vi;
      if (even) {
        // the power of two above the largest, its inverse and its exponent
        const uint32_t kx = (__float_as_uint(all.x) & 0x7f800000u) + 0x00800000u;
        const uint32_t vx = (__float_as_uint(all.z) & 0x7f800000u) + 0x00800000u;
        kappa = __uint_as_float(kx);
        rv = __uint_as_float(vx);
        ki = __uint_as_float(0x7f000000u - kx);
        vi = __uint_as_float(0x7f000000u - vx);
        ve = (int)(vx >> 23) - 127;
      } else {
        ki = kappa > 0.f ? 1.f / kappa : 0.f;
        vi = rv > 0.f ? 1.f / rv : 0.f;
      }
      ka *= ki * kTileScale;
      kb *= ki * kTileScale;
      va *= vi * kTileScale;
      vb *= vi * kTileScale;
      // Keys, then values, through the same code: written out twice (and for
      // two tiles) it did not stay in the instruction cache beside the softmax.
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        in = __all_sync(0xffffffffu, mbar_wait(kv ? &vempty[s] : &kempty[s], ph ^ 1u, P.err));
        if (!in) break;
        write(sm + (kv ? C::kOffV : C::kOffK) + s * C::kKvTile, x.kc, x.kr, ka * c_half, kb,
              ka * r.c0 - kb);
        if (kv == 1 && part == 0) {
          float* sc = reinterpret_cast<float*>(sm + C::kOffScale) + s * 2 * ROWS;
          sc[row] = kappa * (1.f / kTileScale);
          sc[ROWS + row] = rv;
          const uint32_t mask = __ballot_sync(0xffffffffu, x.on);
          if (lane == 0)
            reinterpret_cast<uint32_t*>(sm + C::kOffValid)[s * 4 + (row >> 5)] = mask;
          if (i == 0)
            *reinterpret_cast<float4*>(sm + C::kOffEven + 16 * s) =
                make_float4(kappa * (1.f / kTileScale), vi, (float)ve, even ? 1.f : 0.f);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(kv ? &vfull[s] : &kfull[s]);
        ka = va;
        kb = vb;
#pragma unroll
        for (int w = 0; w < WT; ++w) {
          x.kc[w] = x.vc[w];
          x.kr[w] = x.vr[w];
        }
      }
    }
  } else if (warp >= C::kSoftWarps + 4) {
    // ------------------------------------------------------------ products
    if constexpr (D == 128) fewer_registers<kRegsIssue>();
    grid_dependency_wait();
    grid_dependents_launch();
    if (warp == C::kSoftWarps + 4 && lane == 0) {
      auto scores = [&](int m, int t) {  // of tile t and query tile m
        const uint32_t ka = base + C::kOffK + (t % NS) * C::kKvTile;
        const int i = C::SB * m + t % C::SB;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16(tmem + i * ROWS, sw128_desc(base + m * C::kQTile + (k >> 2) * (128 * 128)) + 2 * (k & 3),
                   sw128_desc(ka + (k >> 2) * C::kKvBox) + 2 * (k & 3), kIdescS, k != 0);
        umma_commit(&sfull[i]);
        if (m == MT - 1) umma_commit(&kempty[t % NS]);
      };
      auto keys = [&](int t) {
        const bool in = mbar_wait(&kfull[t % NS], (uint32_t)((t / NS) & 1), P.err);
        tc_fence_after();
        return in;
      };
      bool ok = mbar_wait(qfull, 0, P.err) && keys(0);
      for (int m = 0; ok && m < MT; ++m) scores(m, 0);
#pragma unroll 1
      for (int t = 0; ok && t < n_tiles; ++t) {
        // The next tile's scores: beside this tile's softmax into the other
        // buffer, or else right after its weights have been used.  Either way
        // they take columns that held weights; the products run in the order
        // of issue, so those have been read.
        const bool more = t + 1 < n_tiles;
        if (C::SB == 2 && more) {
          if (!(ok = keys(t + 1))) break;
          scores(0, t + 1);
        }
        if (!(ok = mbar_wait(&vfull[t % NS], (uint32_t)((t / NS) & 1), P.err))) break;
        const uint32_t va = base + C::kOffV + (t % NS) * C::kKvTile;
#pragma unroll 1
        for (int m = 0; m < MT; ++m) {
          const int i = C::SB * m + t % C::SB;
          if (!(ok = mbar_wait(&pfull[i], (uint32_t)((t / C::SB) & 1), P.err))) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < ROWS / 16; ++k)
            umma_f16_ta(tmem + C::kColO + m * D, tmem + i * ROWS + 8 * k,
                        sw128_desc_mn(va + k * 2048, C::kKvBox), kIdescO, t != 0 || k != 0);
          umma_commit(&odone[m]);
          if (m == MT - 1) umma_commit(&vempty[t % NS]);
          if (C::SB == 1 && more) {
            if (m == 0 && !(ok = keys(t + 1))) break;
            scores(m, t + 1);
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    if constexpr (D == 128) more_registers<kRegsSoft>();
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
    // q~ is stored times log_scale and a power of two
    const float down = 1.f / reinterpret_cast<const float*>(group + MT * C::kQTile)[y];
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
      const int s = t % NS, i = C::SB * m + t % C::SB;
      const int j0 = lo + t * ROWS;
      const uint32_t scores = tmem + lanes + i * ROWS;  // and the weights
      ok = mbar_wait(&vfull[s], (uint32_t)((t / NS) & 1), P.err);
      ok = ok && mbar_wait(&sfull[i], (uint32_t)((t / C::SB) & 1), P.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const float* kap = reinterpret_cast<const float*>(sm + C::kOffScale) + s * 2 * ROWS;
      const float* rv = kap + ROWS;
      const uint32_t* valid = reinterpret_cast<const uint32_t*>(sm + C::kOffValid) + s * 4;
      const float4 tile = *reinterpret_cast<const float4*>(sm + C::kOffEven + 16 * s);
      const bool whole = j0 >= q_lo && j0 + ROWS <= q_hi && tile.w != 0.f;
      // places of chunk c that this query attends
      auto places = [&](int c) {
        const int a = max(q_lo - (j0 + 32 * c), 0), z = min(q_hi - (j0 + 32 * c), 32);
        if (a >= z) return 0u;
        const uint32_t below = z == 32 ? 0xffffffffu : (1u << z) - 1u;
        return valid[c] & below & (0xffffffffu << a);
      };
      // 32 columns at a time; their weights take the columns of scores already
      // read (half as many), so a chunk's own scores stay until it is settled
      // a score as an exponent of two, without the reference
      auto exponent = [&](int j, float x, float k) {
        x *= k;
        if (EXTRA && r.softcap > 0.f) x = soft_cap_16(x, cap, inv_cap);
        if (EXTRA && r.slopes) x = fmaf(slope, (float)(j0 + j + 1 - q_hi), x);
        return x;
      };
      uint32_t p[16];
      float lt;
      // Weights of chunk c into p, their sum (without the rows' scale) into lt;
      // false when one may pass fp16: none does while 32 sum to less.
      // A whole, even tile: w = 2^(x kappa - ref + log2 r).
      auto weigh_even = [&](int c, const float (&x)[32]) {
        float2 sum = make_float2(0.f, 0.f);
        const float shift = tile.z - ref;
        const float k = tile.x * down;
        const float2 kk = make_float2(k, k), sh = make_float2(shift, shift);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float2 y;
          if constexpr (EXTRA)
            y = __fadd2_rn(make_float2(exponent(32 * c + i, x[i], k),
                                       exponent(32 * c + i + 1, x[i + 1], k)), sh);
          else
            y = __ffma2_rn(make_float2(x[i], x[i + 1]), kk, sh);
          const float2 w = (i & 6) == 2 ? ex2_poly(y) : make_float2(ex2(y.x), ex2(y.y));
          sum = __fadd2_rn(sum, w);
          p[i >> 1] = pack_h2(w.x, w.y);
        }
        const float s0 = sum.x + sum.y;
        lt = s0 * tile.y;
        return s0 <= kMostSum && lt < 0x1p110f;
      };
      // Any tile: scales and places by column.
      auto weigh_any = [&](int c, const float (&x)[32], uint32_t on) {
        float sum = 0.f, total = 0.f;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float w[2];
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const int j = 32 * c + i + o;
            const float e = on >> (i + o) & 1 ? ex2(exponent(j, x[i + o], kap[j] * down) - ref) : 0.f;
            w[o] = on >> (i + o) & 1 ? e * rv[j] : 0.f;  // whatever the row's norms hold
            sum += e;
            total += w[o];
          }
          p[i >> 1] = pack_h2(w[0], w[1]);
        }
        lt = sum;
        return total <= kMostSum && sum < 0x1p110f;
      };
      const bool all_whole = __all_sync(0xffffffffu, whole);
#pragma unroll 1
      for (int c = 0; c < ROWS / 32; ++c) {
        float x[32];
        tmem_ld32(scores + 32 * c, x);
        tmem_wait_ld();
        tmem_pin(x);
        const uint32_t on = all_whole ? 0xffffffffu : places(c);
#pragma unroll 1
        for (bool again = false;; again = true) {
          const bool fits = all_whole ? weigh_even(c, x) : weigh_any(c, x, on);
          if (again || __all_sync(0xffffffffu, fits)) break;
          // a weight would leave fp16: the reference moves up to this chunk's
          // largest, what has been summed and stored so far follows.  It moves by
          // whole numbers, and weights take their factor in two parts that fp16
          // holds, so that the weights and l stay of one scale.
          float top = kNoRef;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int j = 32 * c + i;
            const float y = exponent(j, x[i], kap[j] * down) + lg2(fmaxf(rv[j], kLeastNorm));
            if (on >> i & 1) top = fmaxf(top, y);
          }
          const float to = fmaxf(ref, ceilf(top) - kLift), f = ex2(ref - to);
          const float fa = ex2(fmaxf(ref - to, -14.f)), fb = ex2(fminf(ref - to + 14.f, 0.f));
          ref = to;
          l *= f;
          const uint32_t fa2 = pack_h2(fa, fa), fb2 = pack_h2(fb, fb);
#pragma unroll 1
          for (int k = 0; k < c; ++k) {
            const uint32_t at = scores + 16 * k;
            tmem_ld16(at, p);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i)
              asm volatile("mul.rn.f16x2 %0, %0, %1;\n\tmul.rn.f16x2 %0, %0, %2;"
                           : "+r"(p[i]) : "r"(fa2), "r"(fb2));
            tmem_st16(at, p);
          }
          if (t > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(&odone[m], (uint32_t)((t - 1) & 1), P.err)) && ok;
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t at = tmem + lanes + C::kColO + m * D + 16 * k;
              tmem_ld16(at, p);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                asm volatile("mul.rn.f32 %0, %0, %1;" : "+r"(p[i]) : "r"(__float_as_uint(f)));
              tmem_st16(at, p);
            }
          }
          tmem_wait_st();
        }
        l += lt;
        tmem_st16(scores + 16 * c, p);
      }
      if (!ok) break;
      tmem_wait_st();
      // With two score buffers the softmax may be a tile ahead of the products,
      // and the wait for the last of them below would return at once while the
      // one before it runs: that one is waited for here, while it can only be the
      // latest or the one before.
      if (C::SB == 2 && t > 0 && t == n_tiles - 1)
        ok = __all_sync(0xffffffffu, mbar_wait(&odone[m], (uint32_t)((t - 1) & 1), P.err));
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[i]);
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
        tmem_ld32(tmem + lanes + C::kColO + m * D + 32 * c, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) 
          out[lane * (D + 1) + 32 * c + (i >> 1) + 16 * (i & 1)] = v[i] * (1.f / kTileScale);
      }
    }
    __syncwarp();
    const int64_t mine = y < nq ? (query_row(y) * P.plan.pre_chunks + blockIdx.x) * (int64_t)(D + 2) : -1;
    if (!ok) l = 0.f;
#pragma unroll 4
    for (int k = 0; k < 32; ++k) {
      const int64_t at = __shfl_sync(0xffffffffu, mine, k);
      const float mk = __shfl_sync(0xffffffffu, ref, k), lk = __shfl_sync(0xffffffffu, l, k);
      if (at < 0) break;
      float* rec = r.workspace + at;
      if (lane < 2) rec[lane] = lane ? lk : mk;
#pragma unroll
      for (int j = 0; j < W; ++j)
        rec[2 + 32 * j + lane] = ok ? out[k * (D + 1) + 32 * j + lane] : 0.f;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kSoftWarps + 4) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
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
  return launch_programmatic(kern, grid, dim3(C::kThreads), C::kSmem, stream, P) == cudaSuccess
             ? KH_OK
             : KH_ELAUNCH;
}

}  // namespace

kh_status launch_paged_prefix(const AttnParams& P, cudaStream_t stream) {
  const bool extra = P.r.softcap > 0.f || P.r.slopes;
  if (P.r.D == 128)
    return extra ? launch_typed<128, true>(P, stream) : launch_typed<128, false>(P, stream);
  return extra ? launch_typed<256, true>(P, stream) : launch_typed<256, false>(P, stream);
}

}  // namespace kh
