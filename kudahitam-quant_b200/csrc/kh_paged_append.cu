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
__device__ __forceinline__ Place place_of(const AppendParams& P, int64_t t, int h, bool is_v,
                                          bool report) {
  const PagedAppendRequest& r = P.r;
  Place p{-1, nullptr, nullptr};
  const int64_t slot = r.slots[t];
  if (slot == -1) return p;  // a padding token
  const int64_t pos = !is_v && r.positions ? r.positions[t] : 0;
  if (slot < 0 || slot >= r.n_pages * r.page_size ||
      (!is_v && r.positions && (pos < 0 || pos >= r.n_positions))) {
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
  const Place at = place_of(P, t, h, is_v, lane == 0);
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
// Many rows: a lane owns a row (D = 128) or half of one (D = 256, the first
// butterfly stage done while loading), so the transform stays in registers
// on packed adds and no value is exchanged.  A warp's tile is 4096 elements:
// 32 or 16 rows in (token, head) order, so that a token's angles serve its
// heads from L1.  Rows come by cp.async, 16 bytes a lane, into a private
// double buffer whose rows are 16 bytes longer than they need to be: the
// lanes' 16-byte reads, one row each, then hit different banks.
// 16-bit rows of D = 128 cost about 50 instructions a row against 296 bytes:
// bound by issue, not by HBM.
constexpr int kTileWarps = 4;
constexpr int64_t kTileRows = 8192;

template <typename T, int D>
struct TileCfg {
  static constexpr int kRows = 4096 / D;                // rows of a tile
  static constexpr int kBytes = D * (int)sizeof(T);     // of a row
  static constexpr int kPitch = kBytes + 16;
  static constexpr int kStage = kRows * kPitch;
  static constexpr int kSmem = kTileWarps * 2 * kStage;
};

template <typename T>
__device__ __forceinline__ void widen(const uint4& v, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
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

// 16-byte piece c of a staged row, rotated: ROT 0 not at all, 1 in pairs
// (i, i + rot / 2) (rot / 2 a multiple of a piece), 2 in pairs (2 i, 2 i + 1).
template <typename T, int ROT>
__device__ __forceinline__ void piece(const uint8_t* row, int c, int rot, const float* cs,
                                      const float* sn, float (&f)[16 / sizeof(T)]) {
  constexpr int N = 16 / sizeof(T);
  widen<T>(*reinterpret_cast<const uint4*>(row + 16 * c), f);
  if constexpr (ROT == 1) {
    if (c * N < rot) {
      const int half = rot / (2 * N);  // pieces
      const bool second = c >= half;
      const int i = (second ? c - half : c) * N;
      float z[N];
      widen<T>(*reinterpret_cast<const uint4*>(row + 16 * (second ? c - half : c + half)), z);
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const float4 co = __ldg(reinterpret_cast<const float4*>(cs + i + k));
        const float4 si = __ldg(reinterpret_cast<const float4*>(sn + i + k));
        const float cc[4] = {co.x, co.y, co.z, co.w}, ss[4] = {si.x, si.y, si.z, si.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = z[k + e] * ss[e];
          f[k + e] = fmaf(f[k + e], cc[e], second ? p : -p);
        }
      }
    }
  } else if constexpr (ROT == 2) {
    if (c * N < rot) {
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        const float co = __ldg(cs + (c * N + k) / 2), si = __ldg(sn + (c * N + k) / 2);
        const float a = f[k], b = f[k + 1];
        f[k] = fmaf(a, co, -(b * si));
        f[k + 1] = fmaf(b, co, a * si);
      }
    }
  }
}

// x[e] = this lane's 128 values of d . row: all of it at D = 128; at D = 256
// lo + hi (lanes 0 .. 15) or lo - hi, the first stage of the transform.
template <typename T, int D, int ROT>
__device__ __forceinline__ void load_row(const uint8_t* row, int rot, const float* cs,
                                         const float* sn, const uint32_t* flip, float sign,
                                         float (&x)[128]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int c = 0; c < 128 / N; ++c) {
    float f[N];
    piece<T, ROT>(row, c, rot, cs, sn, f);
    if constexpr (D == 128) {
#pragma unroll
      for (int k = 0; k < N; ++k)
        x[c * N + k] = __uint_as_float(__float_as_uint(f[k]) ^ flip[c * N + k]);
    } else {
      float z[N];
      piece<T, ROT>(row, c + 128 / N, rot, cs, sn, z);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float a = __uint_as_float(__float_as_uint(f[k]) ^ flip[c * N + k]);
        const float b = __uint_as_float(__float_as_uint(z[k]) ^ flip[128 + c * N + k]);
        x[c * N + k] = fmaf(b, sign, a);
      }
    }
  }
}

struct TileParams {
  AppendParams a;
  uint32_t dk_flip[256], dv_flip[256];  // sign bit where d is -1
};

template <typename T, int D>
__global__ void __launch_bounds__(32 * kTileWarps, 3)
    paged_append_tiles_kernel(const __grid_constant__ TileParams P) {
  using C = TileCfg<T, D>;
  constexpr int J = D / 32;
  const PagedAppendRequest& r = P.a.r;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* buf = smem + warp * 2 * C::kStage;
  const int64_t rows = r.n_tokens * r.n_kv_heads;
  const int64_t tiles = (rows + C::kRows - 1) / C::kRows * 2;  // keys and values in turn
  const int64_t step = (int64_t)gridDim.x * kTileWarps;
  grid_dependency_wait();
  // row i of the call as the source of its first element
  auto source = [&](int64_t i, bool is_v) {
    const int64_t t = i / r.n_kv_heads;
    const int h = (int)(i - t * r.n_kv_heads);
    return is_v ? static_cast<const T*>(r.v) + t * r.v_stride_t + h * r.v_stride_h
                : static_cast<const T*>(r.k) + t * r.k_stride_t + h * r.k_stride_h;
  };
  auto issue = [&](int64_t tile, int stage) {
    if (tile < tiles) {
      constexpr int kPieces = C::kBytes / 16;  // of a row: a power of two
      const int64_t r0 = (tile >> 1) * C::kRows;
      uint8_t* st = buf + stage * C::kStage;
#pragma unroll 4
      for (int k = lane; k < C::kRows * kPieces; k += 32) {
        const int64_t i = r0 + k / kPieces;
        if (i < rows) {
          const uint8_t* src = reinterpret_cast<const uint8_t*>(source(i, tile & 1));
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                           smem_u32(st + (k / kPieces) * C::kPitch + (k % kPieces) * 16)),
                       "l"(src + (k % kPieces) * 16)
                       : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int64_t first = (int64_t)blockIdx.x * kTileWarps + warp;
  issue(first, 0);
  int stage = 0;
#pragma unroll 1
  for (int64_t tile = first; tile < tiles; tile += step, stage ^= 1) {
    issue(tile + step, stage ^ 1);
    const bool is_v = tile & 1;
    const int rl = D == 128 ? lane : lane & 15;
    const int64_t i = (tile >> 1) * C::kRows + rl;
    Place at{-1, nullptr, nullptr};
    if (i < rows) {
      const int64_t t = i / r.n_kv_heads;
      at = place_of(P.a, t, (int)(i - t * r.n_kv_heads), is_v, true);
    }
    const bool on = at.row >= 0;
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const uint8_t* row = buf + stage * C::kStage + (on ? rl : 0) * C::kPitch;
    const float sign = lane < 16 ? 1.f : -1.f;
    float x[128];
    // a lane without a row goes along on another's (or on stale) values
    const int rot = is_v || !on ? 0 : r.rot_dim;
    if (is_v || !r.rot_dim) load_row<T, D, 0>(row, 0, nullptr, nullptr, is_v ? P.dv_flip : P.dk_flip, sign, x);
    else if (r.interleaved) load_row<T, D, 2>(row, rot, at.cs, at.sn, P.dk_flip, sign, x);
    else load_row<T, D, 1>(row, rot, at.cs, at.sn, P.dk_flip, sign, x);
    float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < 128; e += 2) {
      const float2 p = make_float2(x[e], x[e + 1]);
      s2 = __ffma2_rn(p, p, s2);
    }
    float ss = s2.x + s2.y;
    if (D == 256) ss = 0.5f * (ss + __shfl_xor_sync(0xffffffffu, ss, 16));
    const float norm = sqrtf(ss);
    const float inv = 1.f / norm;
    fwht_regs<128>(x);
    // code bit = [u > 0] (an exact 0 lies inside the band); residual bit =
    // code bit xor [|y| < c1]
    uint32_t cw[4] = {0, 0, 0, 0}, tw[4] = {0, 0, 0, 0};
    float mu = INFINITY, mt = INFINITY;
    float2 v2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 30; k >= 0; k -= 2)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
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
    bool near = !(ss > kMinSquares && ss < kMaxSquares) || mu * inv < P.a.band || mt < P.a.band;
    if (D == 256) {
      vv += __shfl_xor_sync(0xffffffffu, vv, 16);
      near |= __shfl_xor_sync(0xffffffffu, (int)near, 16) != 0;
    }
    near = near && on;
    const PagedPool& pool = is_v ? r.vp : r.kp;
    if (on && !near) {
      const int64_t o = D == 128 ? at.row * 4 : at.row * 8 + (lane >> 4) * 4;
      const uint4 c = make_uint4(~cw[0], ~cw[1], ~cw[2], ~cw[3]);
      *reinterpret_cast<uint4*>(pool.code + o) = c;
      *reinterpret_cast<uint4*>(pool.res + o) =
          make_uint4(c.x ^ tw[0], c.y ^ tw[1], c.z ^ tw[2], c.w ^ tw[3]);
      if (D == 128 || lane < 16) {
        const float rn = norm * sqrtf(vv * (1.f / D));
        pool.norms[at.row] = norm;
        pool.rnorms[at.row] = rn == 0.f ? 1e-8f : rn;
      }
    }
    uint32_t todo = __ballot_sync(0xffffffffu, near);
    if (D == 256) todo &= 0xffffu;
#pragma unroll 1
    while (todo) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1;
      const int64_t ti = (tile >> 1) * C::kRows + l;
      const int64_t ro = __shfl_sync(0xffffffffu, at.row, l);
      const float* cs = reinterpret_cast<const float*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(at.cs), l));
      const float* sn = reinterpret_cast<const float*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(at.sn), l));
      const Coded o = encode_row_64<T, J>(P.a, source(ti, is_v), is_v, is_v ? 0 : r.rot_dim, cs,
                                          sn, lane);
      if (lane < J) {
        pool.code[ro * J + lane] = o.code;
        pool.res[ro * J + lane] = o.res;
      }
      if (lane == 0) {
        pool.norms[ro] = o.norm;
        pool.rnorms[ro] = o.rnorm == 0.f ? 1e-8f : o.rnorm;
      }
    }
    __syncwarp();
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

template <typename T, int D>
kh_status launch_tiles(const AppendParams& A, cudaStream_t stream) {
  using C = TileCfg<T, D>;
  auto kern = paged_append_tiles_kernel<T, D>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return KH_ECUDA;
  static std::once_flag once[64];
  std::call_once(once[dev & 63], [&] {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  TileParams P;
  P.a = A;
  for (int e = 0; e < 256; ++e) {
    P.dk_flip[e] = (A.r.dk_neg[e >> 5] >> (e & 31) & 1) << 31;
    P.dv_flip[e] = (A.r.dv_neg[e >> 5] >> (e & 31) & 1) << 31;
  }
  const int64_t tiles = (A.r.n_tokens * A.r.n_kv_heads + C::kRows - 1) / C::kRows * 2;
  const int64_t blocks = std::min<int64_t>((tiles + kTileWarps - 1) / kTileWarps, 3 * sm_count());
  if (launch_programmatic(kern, dim3((unsigned)blocks), dim3(32 * kTileWarps), C::kSmem, stream,
                          P) != cudaSuccess)
    return KH_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? KH_OK : KH_ELAUNCH;
}

// The tiled kernel needs 16-byte pieces of rows and angles, rotation pairs
// that fall on whole pieces, and levels -c, c.
template <typename T, int D>
bool tiles_fit(const PagedAppendRequest& r) {
  const auto on16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const int64_t n = 16 / sizeof(T);
  if (r.c0 != -r.c1 || !on16(r.k) || !on16(r.v)) return false;
  if (r.k_stride_t % n || r.k_stride_h % n || r.v_stride_t % n || r.v_stride_h % n) return false;
  if (r.rot_dim && !r.interleaved)
    return r.rot_dim % (2 * n) == 0 && r.rot_dim % 8 == 0 && on16(r.cos) && on16(r.sin);
  return r.rot_dim == 0 || r.rot_dim % n == 0;
}

template <typename T, int D>
kh_status launch_typed(const AppendParams& P, cudaStream_t stream) {
  const int64_t rows = P.r.n_tokens * P.r.n_kv_heads * 2;
  return rows >= kTileRows && tiles_fit<T, D>(P.r) ? launch_tiles<T, D>(P, stream)
                                                   : launch_rows<T, D>(P, stream);
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
