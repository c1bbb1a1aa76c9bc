// kh_paged_append.cu -- new keys and values into a paged packed cache, the
// position rotation of the keys applied on the way: one launch per layer and
// step instead of a rotation, two compressions and eight copies.
//
//   x    = rotate(k, position) (keys) or v (values), in 32 bits
//   u    = H (d . x),  norm = |x|,  y = u / (sqrt(D) norm)
//   bit  = [y > (c0 + c1) / 2],  res = [y - c[bit] >= 0],
//   rnorm = norm |y - c[bit]|
// (H carries the residual's transform too: H (d . (x - k_mse)) =
// sqrt(D) norm (y - c[bit]), so one transform serves both planes.)
//
// The planes are decisions, and a cache shared between runs should not depend
// on the order of a sum: a row with an element so near a border that 32-bit
// rounding could decide it is transformed again in 64 bits (one row in 600
// at D = 128).  The band is the a-priori error of the 32-bit transform,
//   |du| <= 2^-24 (log2 D + 3) sqrt(D) norm
// (log2 D butterfly stages, two roundings of the rotation, each at most
// 2^-24 of a partial sum that |x|_1 <= sqrt(D) norm bounds), plus 16 ulps for
// the division by the norm.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "kh_common.cuh"
#include "kh_paged.h"

namespace kh {
namespace {

struct AppendParams {
  PagedAppendRequest r;
  float mid, c0, c1;   // levels and border of u / norm (times sqrt(D))
  double midd, c0d, c1d;
  float band;
  uint32_t* err;
};

constexpr float kMinSquares = 1e-30f, kMaxSquares = 1e37f;

template <typename T>
__device__ __forceinline__ float ld_elt(const T* p) { return static_cast<float>(*p); }
template <>
__device__ __forceinline__ float ld_elt<__half>(const __half* p) { return __half2float(*p); }
template <>
__device__ __forceinline__ float ld_elt<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}

template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Walsh-Hadamard sums of the warp's row: element 32 j + lane in x[j].
template <int J, typename F>
__device__ __forceinline__ void fwht_warp(F (&x)[J], int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const F y = __shfl_xor_sync(0xffffffffu, x[j], o);
      x[j] = up ? y - x[j] : x[j] + y;
    }
  }
#pragma unroll
  for (int h = 1; h < J; h <<= 1)
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (!(j & h)) {
        const F a = x[j], b = x[j + h];
        x[j] = a + b;
        x[j + h] = a - b;
      }
}

// Element e of the row at src, rotated when rot_dim > 0, times d.
template <typename F, typename T>
__device__ __forceinline__ F element(const T* src, int e, int rot, bool inter, const float* cs,
                                     const float* sn, bool neg) {
  F x = (F)ld_elt(src + e);
  if (e < rot) {
    const int half = rot >> 1;
    const int i = inter ? e >> 1 : (e < half ? e : e - half);
    const bool second = inter ? (e & 1) : (e >= half);
    const int other = inter ? e ^ 1 : (second ? e - half : e + half);
    const F z = (F)ld_elt(src + other);
    const F c = (F)cs[i], s = (F)sn[i];
    const F zs = z * s;
    x = second ? fma(x, c, zs) : fma(x, c, -zs);
  }
  return neg ? -x : x;
}

// One row transformed by a warp in 64 bits: words and norms for lane 0 .. J-1.
struct Coded {
  uint32_t code, res;  // lane j < J: word j
  float norm, rnorm;
};
template <typename T, int J>
__device__ __noinline__ Coded encode_row_64(const AppendParams& P, const T* src, bool is_v, int rot,
                                            const float* cs, const float* sn, int lane) {
  const PagedAppendRequest& r = P.r;
  double x[J], sd = 0.0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint32_t neg = is_v ? r.dv_neg[j] : r.dk_neg[j];
    x[j] = element<double>(src, 32 * j + lane, rot, r.interleaved, cs, sn, (neg >> lane) & 1);
    sd = fma(x[j], x[j], sd);
  }
  sd = warp_sum(sd);
  const double norm = sd == 0.0 ? 1e-8 : sqrt(sd);
  fwht_warp<J>(x, lane);
  Coded o{};
  double vd = 0.0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const bool bit = x[j] > P.midd * norm;
    const double v = x[j] - (bit ? P.c1d : P.c0d) * norm;
    vd = fma(v, v, vd);
    const uint32_t c = __ballot_sync(0xffffffffu, bit);
    const uint32_t s = __ballot_sync(0xffffffffu, v >= 0.0);
    if (lane == j) {
      o.code = c;
      o.res = s;
    }
  }
  vd = warp_sum(vd);
  o.norm = (float)norm;
  o.rnorm = (float)sqrt(vd * (1.0 / (32 * J)));
  return o;
}

// Where token t's rows of head h go and how a key turns; row < 0: nowhere.
struct Place {
  int64_t row;
  const float *cs, *sn;
};
__device__ __forceinline__ Place place_of(const AppendParams& P, int64_t t, int h, bool report) {
  const PagedAppendRequest& r = P.r;
  Place p{-1, nullptr, nullptr};
  const int64_t slot = r.slots[t];
  if (slot == -1) return p;  // a padding token
  const int64_t pos = r.positions ? r.positions[t] : 0;
  if (slot < 0 || slot >= r.n_pages * r.page_size ||
      (r.positions && (pos < 0 || pos >= r.n_positions))) {
    if (report) flag_error(P.err, kErrBadIndex);
    return p;
  }
  p.cs = r.cos + pos * (r.rot_dim >> 1);
  p.sn = r.sin + pos * (r.rot_dim >> 1);
  const int64_t page = slot / r.page_size;
  p.row = (page * r.n_kv_heads + h) * r.page_size + (slot - page * r.page_size);
  return p;
}

// Few rows, or layouts that the tiled kernel does not take: a warp per row,
// which ends soonest when there is little to do.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_append_kernel(const __grid_constant__ AppendParams P) {
  constexpr int J = D / 32;
  const PagedAppendRequest& r = P.r;
  const int lane = threadIdx.x & 31;
  const int64_t n_items = r.n_tokens * r.n_kv_heads * 2;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  grid_dependency_wait();
  if (item >= n_items) return;
  const int64_t t = item / (2 * r.n_kv_heads);
  const int hv = (int)(item - t * 2 * r.n_kv_heads);
  const bool is_v = hv >= r.n_kv_heads;
  const int h = is_v ? hv - r.n_kv_heads : hv;
  const Place at = place_of(P, t, h, lane == 0);
  if (at.row < 0) return;
  const T* src = is_v ? static_cast<const T*>(r.v) + t * r.v_stride_t + h * r.v_stride_h
                      : static_cast<const T*>(r.k) + t * r.k_stride_t + h * r.k_stride_h;
  const int rot = is_v ? 0 : r.rot_dim;
  float x[J], ss = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint32_t neg = is_v ? r.dv_neg[j] : r.dk_neg[j];
    x[j] = element<float>(src, 32 * j + lane, rot, r.interleaved, at.cs, at.sn, (neg >> lane) & 1);
    ss = fmaf(x[j], x[j], ss);
  }
  ss = warp_sum(ss);
  Coded o{};
  o.norm = sqrtf(ss);
  const float inv = 1.f / o.norm;
  fwht_warp<J>(x, lane);
  // squares that leave the 32-bit range (rows of zeros among them) go the
  // 64-bit way as well
  bool near = !(ss > kMinSquares && ss < kMaxSquares);
  float vv = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const float y = x[j] * inv;
    const bool bit = y > P.mid;
    const float v = y - (bit ? P.c1 : P.c0);
    near |= fabsf(y - P.mid) < P.band || fabsf(v) < P.band;
    vv = fmaf(v, v, vv);
    const uint32_t c = __ballot_sync(0xffffffffu, bit);
    const uint32_t s = __ballot_sync(0xffffffffu, v >= 0.f);
    if (lane == j) {
      o.code = c;
      o.res = s;
    }
  }
  o.rnorm = o.norm * sqrtf(warp_sum(vv) * (1.f / D));
  if (__any_sync(0xffffffffu, near))
    o = encode_row_64<T, J>(P, src, is_v, rot, at.cs, at.sn, lane);
  const PagedPool& pool = is_v ? r.vp : r.kp;
  if (lane < J) {
    pool.code[at.row * J + lane] = o.code;
    pool.res[at.row * J + lane] = o.res;
  }
  if (lane == 0) {
    pool.norms[at.row] = o.norm;
    pool.rnorms[at.row] = o.rnorm == 0.f ? 1e-8f : o.rnorm;
  }
}

// ------------------------------------------------------------------ tiles
//
// Many rows: a lane owns 64 elements of a row, so that six stages of the
// transform stay in registers on packed adds and only the last one (two at
// D = 256) crosses lanes, while 16 warps fit an SM (20, with 96 registers,
// spilled and measured 82 us where 16 measure 74: 32768 tokens of 8 heads, D 128,
// bf16, all rotated).  A warp's tile is 2048 elements, 32 "slots" of 64: 16 or 8
// rows in (token, head) order, so that a token's angles serve its heads from
// L1.  Slots come by cp.async, 16 bytes a lane, into a private double buffer;
// each is 16 bytes longer than it needs to be, so that the lanes' 16-byte reads
// hit different banks.  What bounds it is latency: a warp's 64-element chain at 16
// warps an SM uses 58% of the issue slots (82 instructions a row; the widest parts:
// two shifts an element for its bits, a third of one for the borders).
constexpr int kTileWarps = 4;
constexpr int kTileCtas = 4;
// From how many keys (tokens x heads) they come in tiles: of fewer, most warps
// have no tile and the others' chain of 64 elements a lane is the time.  Measured (us,
// a warp per row / tiles, bf16, whole keys rotated), D 128: 4096 keys 6.9 / 10.1,
// 8192 11.2 / 9.4, 32768 36.1 / 14.0; D 256: 4096 9.9 / 13.5, 8192 16.3 / 14.2, 32768
// 53.5 / 30.1.  Straight lines between the first two cross at 6700 keys.
constexpr int64_t kTileRows = 6656;

template <typename T>
struct TileCfg {
  static constexpr int N = 16 / (int)sizeof(T);           // elements of a 16-byte piece
  static constexpr int kPieces = 64 / N;                  // of a slot
  static constexpr int kSlot = 64 * (int)sizeof(T) + 16;  // bytes, with the pad
  static constexpr int kStage = 32 * kSlot;
  static constexpr int kFlips = 3 * 4 * kSlot;            // sign bits: see the kernel
  static constexpr int kSmem = kFlips + kTileWarps * 2 * kStage;
};

// j / n for j < 2^31 by a multiplication: mul = ceil(2^shift / n) with
// shift = 31 + ceil(log2 n), so that the error j (mul n - 2^shift) / (n 2^shift)
// stays under 1 / n.
struct FastDiv {
  uint64_t mul;
  int shift;
  __device__ __forceinline__ uint32_t operator()(uint32_t j) const {
    return (uint32_t)((j * mul) >> shift);
  }
};
FastDiv fast_div(uint32_t n) {
  int bits = 0;
  while ((uint64_t(1) << bits) < n) ++bits;
  return FastDiv{((uint64_t(1) << (31 + bits)) + n - 1) / n, 31 + bits};
}

struct TileParams {
  AppendParams a;
  FastDiv by_heads, by_page;
  int contiguous;  // k's and v's rows follow one another
};

template <typename T>
__device__ __forceinline__ void widen(const uint4& v, const uint4& flip, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {v.x ^ flip.x, v.y ^ flip.y, v.z ^ flip.z, v.w ^ flip.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      __half2 h;
      memcpy(&h, &w[i], 4);
      const float2 p = __half22float2(h);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}

// How the keys of a launch turn.
enum Turn { kNone, kWhole, kPairs, kPart };  // kWhole: (i, i + D / 2); kPart: rot < D

// x = slot p of the row whose slots begin at `row`, d applied, rotated.
template <typename T, int D, int TURN>
__device__ __forceinline__ void load_slot(const uint8_t* row, const uint8_t* flips, int p, int rot,
                                          bool pairs, const float* cs, const float* sn,
                                          float (&x)[64]) {
  using C = TileCfg<T>;
  constexpr int N = C::N, S = D / 64;
#pragma unroll
  for (int c = 0; c < C::kPieces; ++c) {
    const uint4 fl = *reinterpret_cast<const uint4*>(flips + p * C::kSlot + 16 * c);
    const uint4 raw = *reinterpret_cast<const uint4*>(row + p * C::kSlot + 16 * c);
    float f[N];
    widen<T>(raw, fl, f);
    const int e = 64 * p + N * c;
    if (TURN == kPairs || (TURN == kPart && pairs)) {
      if (TURN == kPairs || e < rot) {
        // the pair's elements have signs of their own: turn them bare
        float z[N];
        widen<T>(raw, make_uint4(0, 0, 0, 0), z);
        constexpr uint32_t kBit = sizeof(T) == 4 ? 0x80000000u : 0x8000u;
        const uint32_t fw[4] = {fl.x, fl.y, fl.z, fl.w};
#pragma unroll
        for (int k = 0; k < N; k += 2) {
          const float co = __ldg(cs + (e + k) / 2), si = __ldg(sn + (e + k) / 2);
          const float a = fmaf(z[k], co, -(z[k + 1] * si)), b = fmaf(z[k + 1], co, z[k] * si);
          const bool na = sizeof(T) == 4 ? fw[k & 3] & kBit : fw[k / 2] & kBit;
          const bool nb = sizeof(T) == 4 ? fw[(k + 1) & 3] & kBit : fw[k / 2] & (kBit << 16);
          f[k] = na ? -a : a;
          f[k + 1] = nb ? -b : b;
        }
      }
    } else if (TURN == kWhole || TURN == kPart) {
      if (TURN == kWhole || e < rot) {
        const int half = TURN == kWhole ? D / 2 : rot >> 1;
        const bool second = TURN == kWhole ? p >= S / 2 : e >= half;
        const int o = second ? e - half : e + half, i = second ? o : e;
        float z[N];
        widen<T>(*reinterpret_cast<const uint4*>(row + (o >> 6) * C::kSlot +
                                                 (o & 63) * (int)sizeof(T)),
                 *reinterpret_cast<const uint4*>(flips + (8 + p) * C::kSlot + 16 * c), z);
#pragma unroll
        for (int k = 0; k < N; k += 4) {
          const float4 co = __ldg(reinterpret_cast<const float4*>(cs + i + k));
          const float4 si = __ldg(reinterpret_cast<const float4*>(sn + i + k));
          const float cc[4] = {co.x, co.y, co.z, co.w}, ss[4] = {si.x, si.y, si.z, si.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) f[k + q] = fmaf(f[k + q], cc[q], z[k + q] * ss[q]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) x[c * N + k] = f[k];
  }
}

template <typename T, int D, int TURN>
__global__ void __launch_bounds__(32 * kTileWarps, kTileCtas)
    paged_append_tiles_kernel(const __grid_constant__ TileParams P) {
  using C = TileCfg<T>;
  constexpr int J = D / 32;
  constexpr int S = D / 64;        // slots of a row
  constexpr int kRows = 32 / S;    // rows of a tile
  const PagedAppendRequest& r = P.a.r;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* buf = smem + C::kFlips + warp * 2 * C::kStage;
  // sign bits in the slots' layout: d of keys, d of values, and d of keys
  // times the sign of the pair's other element in the rotation
  for (int k = threadIdx.x; k < 3 * D; k += 32 * kTileWarps) {
    const int e = k % D, which = k / D;
    const uint32_t* neg = which == 1 ? r.dv_neg : r.dk_neg;
    const uint32_t bit = ((neg[e >> 5] >> (e & 31)) & 1) ^ (which == 2 && e < (r.rot_dim >> 1));
    uint8_t* at = smem + (which * 4 + e / 64) * C::kSlot + (e & 63) * sizeof(T);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(at) = bit << 31;
    else *reinterpret_cast<uint16_t*>(at) = (uint16_t)(bit << 15);
  }
  __syncthreads();
  const uint32_t rows = (uint32_t)(r.n_tokens * r.n_kv_heads);
  const uint32_t tiles = (rows + kRows - 1) / kRows;
  const uint32_t step = gridDim.x * kTileWarps;
  grid_dependency_wait();
  // first element of row i
  auto source = [&](uint32_t i, bool is_v) {
    const uint32_t t = P.by_heads(i), h = i - t * r.n_kv_heads;
    return is_v ? static_cast<const T*>(r.v) + t * r.v_stride_t + h * r.v_stride_h
                : static_cast<const T*>(r.k) + t * r.k_stride_t + h * r.k_stride_h;
  };
  auto issue = [&](uint32_t tile, int is_v) {
    const int stage = is_v;
    if (tile < tiles) {
      const uint32_t r0 = tile * kRows;
      const uint32_t left = rows - r0;  // rows of the tile, or more
      const uint32_t dst = smem_u32(buf + stage * C::kStage) + (lane / C::kPieces) * C::kSlot +
                           (lane % C::kPieces) * 16;
      const T* base = static_cast<const T*>(is_v ? r.v : r.k) + (int64_t)r0 * D + lane * C::N;
#pragma unroll
      for (int m = 0; m < C::kPieces; ++m) {
        const uint32_t k = lane + 32 * m, slot = k / C::kPieces;
        if (slot / S < left) {
          const T* src = P.contiguous ? base + 32 * m * C::N
                                      : source(r0 + slot / S, is_v) + (slot % S) * 64 +
                                            (k % C::kPieces) * C::N;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                           dst + m * (32 / C::kPieces) * C::kSlot),
                       "l"(src)
                       : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const uint32_t first = blockIdx.x * kTileWarps + warp;
  const int p = lane % S, rl = lane / S;
  issue(first, 0);
  issue(first, 1);
  // a tile's keys, then its values: both go to the same slots, and no warp is
  // left with keys alone, which cost more
  int64_t row = -1, angle = 0;
#pragma unroll 1
  for (uint32_t tile = first, is_v = 0; tile < tiles; tile += is_v ? step : 0, is_v ^= 1) {
    const uint32_t i = tile * kRows + rl;
    if (!is_v) {
      // a lane without a row goes along on stale values
      row = -1;
      angle = 0;
      if (i < rows) {
        const uint32_t t = P.by_heads(i), h = i - t * r.n_kv_heads;
        const int64_t slot = r.slots[t];
        bool ok = slot >= 0 && slot < r.n_pages * r.page_size;
        bool bad = !ok && slot != -1;
        if (TURN != kNone && slot != -1) {
          const int64_t pos = r.positions[t];
          const bool in = pos >= 0 && pos < r.n_positions;
          bad |= !in;
          ok = ok && in;
          angle = in ? pos * (r.rot_dim >> 1) : 0;
        }
        if (bad) flag_error(P.a.err, kErrBadIndex);
        if (ok) {
          const uint32_t page = P.by_page((uint32_t)slot);
          row = ((int64_t)page * r.n_kv_heads + h) * r.page_size +
                ((uint32_t)slot - page * r.page_size);
        }
      }
    }
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const uint8_t* src = buf + is_v * C::kStage + rl * S * C::kSlot;
    float x[64];
    if (TURN == kNone || is_v)
      load_slot<T, D, kNone>(src, smem + (is_v ? 4 * C::kSlot : 0), p, 0, false, nullptr, nullptr, x);
    else
      load_slot<T, D, TURN>(src, smem, p, r.rot_dim, r.interleaved, r.cos + angle, r.sin + angle, x);
    __syncwarp();
    issue(tile + step, is_v);  // the slots are in registers: the buffer takes the next tile's
    float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < 64; e += 2) {
      const float2 v = make_float2(x[e], x[e + 1]);
      s2 = __ffma2_rn(v, v, s2);
    }
    float ss = s2.x + s2.y;
#pragma unroll
    for (int o = 1; o < S; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float norm = sqrtf(ss);
    const float inv = 1.f / norm;
    fwht_regs<64>(x);
#pragma unroll
    for (int o = 1; o < S; o <<= 1) {
      const float sg = p & o ? -1.f : 1.f;
#pragma unroll
      for (int e = 0; e < 64; ++e) x[e] = fmaf(x[e], sg, __shfl_xor_sync(0xffffffffu, x[e], o));
    }
    // code bit = [u > 0] (an exact 0 lies inside the band); residual bit =
    // code bit xor [|y| < c1]
    uint32_t cw[2] = {0, 0}, tw[2] = {0, 0};
    float mu = INFINITY, mt = INFINITY;
    float2 v2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 30; k >= 0; k -= 2)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const float u0 = x[32 * w + k], u1 = x[32 * w + k + 1];
        const float t0 = fmaf(fabsf(u0), inv, -P.a.c1), t1 = fmaf(fabsf(u1), inv, -P.a.c1);
        cw[w] = push_sign(push_sign(cw[w], u1), u0);
        tw[w] = push_sign(push_sign(tw[w], t1), t0);
        mu = fminf(fminf(mu, fabsf(u0)), fabsf(u1));
        mt = fminf(fminf(mt, fabsf(t0)), fabsf(t1));
        const float2 tt = make_float2(t0, t1);
        v2 = __ffma2_rn(tt, tt, v2);
      }
    float vv = v2.x + v2.y;
#pragma unroll
    for (int o = 1; o < S; o <<= 1) vv += __shfl_xor_sync(0xffffffffu, vv, o);
    bool near = !(ss > kMinSquares && ss < kMaxSquares) || mu * inv < P.a.band || mt < P.a.band;
    near = near && row >= 0;
    uint32_t todo = __ballot_sync(0xffffffffu, near);
    // a row is near a border when one of its lanes is
#pragma unroll
    for (int o = 1; o < S; o <<= 1) {
      constexpr uint32_t kLow[3] = {0, 0x55555555u, 0x33333333u};
      todo |= ((todo & kLow[o]) << o) | ((todo >> o) & kLow[o]);
    }
    const PagedPool& pool = is_v ? r.vp : r.kp;
    if (row >= 0 && !(todo >> lane & 1)) {
      const uint2 c = make_uint2(~cw[0], ~cw[1]);
      *reinterpret_cast<uint2*>(pool.code + row * J + 2 * p) = c;
      *reinterpret_cast<uint2*>(pool.res + row * J + 2 * p) = make_uint2(c.x ^ tw[0], c.y ^ tw[1]);
      if (p == 0) {
        const float rn = norm * sqrtf(vv * (1.f / D));
        pool.norms[row] = norm;
        pool.rnorms[row] = rn == 0.f ? 1e-8f : rn;
      }
    }
#pragma unroll 1
    while (todo) {
      const int l = __ffs(todo) - 1;
      todo &= ~(((1u << S) - 1) << l);
      const int64_t ro = __shfl_sync(0xffffffffu, row, l);
      const int64_t an = __shfl_sync(0xffffffffu, angle, l);
      const Coded o = encode_row_64<T, J>(P.a, source(tile * kRows + l / S, is_v), is_v,
                                          is_v ? 0 : r.rot_dim, r.cos + an, r.sin + an, lane);
      if (lane < J) {
        pool.code[ro * J + lane] = o.code;
        pool.res[ro * J + lane] = o.res;
      }
      if (lane == 0) {
        pool.norms[ro] = o.norm;
        pool.rnorms[ro] = o.rnorm == 0.f ? 1e-8f : o.rnorm;
      }
    }
  }
  grid_dependents_launch();
}

template <typename T, int D>
kh_status launch_rows(const AppendParams& P, cudaStream_t stream) {
  const int64_t items = P.r.n_tokens * P.r.n_kv_heads * 2;
  const int64_t blocks = (items + 3) / 4;
  if (blocks > 0x7fffffffll) return KH_EINVAL;
  if (launch_programmatic(paged_append_kernel<T, D>, dim3((unsigned)blocks), dim3(128), 0, stream,
                          P) != cudaSuccess)
    return KH_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? KH_OK : KH_ELAUNCH;
}

template <typename T, int D, int TURN>
kh_status launch_tiles(const AppendParams& A, cudaStream_t stream) {
  using C = TileCfg<T>;
  auto kern = paged_append_tiles_kernel<T, D, TURN>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KH_ECUDA;
  static std::once_flag once[64];
  std::call_once(once[dev & 63], [&] {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  const PagedAppendRequest& r = A.r;
  TileParams P;
  P.a = A;
  P.by_heads = fast_div(r.n_kv_heads);
  P.by_page = fast_div(r.page_size);
  P.contiguous = r.k_stride_h == D && r.v_stride_h == D && r.k_stride_t == D * (int64_t)r.n_kv_heads &&
                 r.v_stride_t == r.k_stride_t;
  const int64_t rows = 32 * 64 / D;
  const int64_t tiles = (r.n_tokens * r.n_kv_heads + rows - 1) / rows;
  const int64_t blocks = std::min<int64_t>((tiles + kTileWarps - 1) / kTileWarps,
                                           (sizeof(T) == 4 ? 3 : kTileCtas) * sm_count());
  if (launch_programmatic(kern, dim3((unsigned)blocks), dim3(32 * kTileWarps), C::kSmem, stream,
                          P) != cudaSuccess)
    return KH_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? KH_OK : KH_ELAUNCH;
}

// The tiled kernel needs 16-byte pieces of rows and angles, rotation pairs
// that fall on whole pieces, levels -c, c, and 31-bit row and slot numbers.
template <typename T, int D>
bool tiles_fit(const PagedAppendRequest& r) {
  const auto on16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const int64_t n = 16 / sizeof(T);
  if (r.c0 != -r.c1 || !on16(r.k) || !on16(r.v)) return false;
  if (r.k_stride_t % n || r.k_stride_h % n || r.v_stride_t % n || r.v_stride_h % n) return false;
  if (r.n_tokens * r.n_kv_heads >= (int64_t(1) << 30) ||
      r.n_pages * r.page_size >= (int64_t(1) << 31))
    return false;
  if (r.rot_dim && !r.interleaved)
    return r.rot_dim % (2 * n) == 0 && r.rot_dim % 8 == 0 && on16(r.cos) && on16(r.sin);
  return r.rot_dim % n == 0;
}

template <typename T, int D>
kh_status launch_typed(const AppendParams& P, cudaStream_t stream) {
  const PagedAppendRequest& r = P.r;
  if (r.n_tokens * r.n_kv_heads < kTileRows || !tiles_fit<T, D>(r))
    return launch_rows<T, D>(P, stream);
  if (!r.rot_dim) return launch_tiles<T, D, kNone>(P, stream);
  if (r.rot_dim < D) return launch_tiles<T, D, kPart>(P, stream);
  return r.interleaved ? launch_tiles<T, D, kPairs>(P, stream)
                       : launch_tiles<T, D, kWhole>(P, stream);
}

template <typename T>
kh_status launch_dim(const AppendParams& P, cudaStream_t stream) {
  return P.r.D == 128 ? launch_typed<T, 128>(P, stream) : launch_typed<T, 256>(P, stream);
}

}  // namespace

kh_status launch_paged_append(const PagedAppendRequest& r, cudaStream_t stream) {
  AppendParams P;
  P.r = r;
  const double sd = std::sqrt((double)r.D);
  P.c0d = r.c0 * sd;
  P.c1d = r.c1 * sd;
  P.midd = 0.5 * ((double)r.c0 + (double)r.c1) * sd;
  P.c0 = (float)P.c0d;
  P.c1 = (float)P.c1d;
  P.mid = (float)P.midd;
  const double stages = r.D == 128 ? 7 : 8;
  P.band = (float)(std::ldexp((stages + 3) * sd + 16, -24));
  P.err = device_error_ptr();
  switch (r.dtype) {
    case KH_F32: return launch_dim<float>(P, stream);
    case KH_F16: return launch_dim<__half>(P, stream);
    case KH_BF16: return launch_dim<__nv_bfloat16>(P, stream);
  }
  return KH_EINVAL;
}

}  // namespace kh
