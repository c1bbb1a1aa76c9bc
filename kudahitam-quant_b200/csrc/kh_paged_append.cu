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
#include <cmath>

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

template <typename T, int D>
__global__ void __launch_bounds__(128) paged_append_kernel(const __grid_constant__ AppendParams P) {
  constexpr int J = D / 32;
  const PagedAppendRequest& r = P.r;
  const int lane = threadIdx.x & 31;
  const int64_t n_items = r.n_tokens * r.n_kv_heads * 2;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  grid_dependency_wait();
  if (item >= n_items) return;
  // heads of one token side by side: the slot and the angles are read once
  const int64_t t = item / (2 * r.n_kv_heads);
  const int hv = (int)(item - t * 2 * r.n_kv_heads);
  const bool is_v = hv >= r.n_kv_heads;
  const int h = is_v ? hv - r.n_kv_heads : hv;
  const int64_t slot = r.slots[t];
  if (slot == -1) return;  // a padding token
  if (slot < 0 || slot >= r.n_pages * r.page_size) {
    if (lane == 0) flag_error(P.err, kErrBadIndex);
    return;
  }
  const T* src = is_v ? static_cast<const T*>(r.v) + t * r.v_stride_t + h * r.v_stride_h
                      : static_cast<const T*>(r.k) + t * r.k_stride_t + h * r.k_stride_h;
  int rot = 0;
  const float *cs = nullptr, *sn = nullptr;
  if (!is_v && r.positions) {
    const int64_t pos = r.positions[t];
    if (pos < 0 || pos >= r.n_positions) {
      if (lane == 0) flag_error(P.err, kErrBadIndex);
      return;
    }
    rot = r.rot_dim;
    cs = r.cos + pos * (rot >> 1);
    sn = r.sin + pos * (rot >> 1);
  }
  float x[J], ss = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint32_t neg = is_v ? r.dv_neg[j] : r.dk_neg[j];
    x[j] = element<float>(src, 32 * j + lane, rot, r.interleaved, cs, sn, (neg >> lane) & 1);
    ss = fmaf(x[j], x[j], ss);
  }
  ss = warp_sum(ss);
  float norm = sqrtf(ss);
  const float inv = 1.f / norm;
  fwht_warp<J>(x, lane);
  // squares that leave the 32-bit range (rows of zeros among them) go the
  // 64-bit way as well
  bool bit[J], res[J], near = !(ss > 1e-30f && ss < 1e37f);
  float vv = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const float y = x[j] * inv;
    bit[j] = y > P.mid;
    const float v = y - (bit[j] ? P.c1 : P.c0);
    res[j] = v >= 0.f;
    near |= fabsf(y - P.mid) < P.band || fabsf(v) < P.band;
    vv = fmaf(v, v, vv);
  }
  float rnorm = norm * sqrtf(warp_sum(vv) * (1.f / D));
  if (__any_sync(0xffffffffu, near)) {
    double xd[J], sd = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t neg = is_v ? r.dv_neg[j] : r.dk_neg[j];
      xd[j] = element<double>(src, 32 * j + lane, rot, r.interleaved, cs, sn, (neg >> lane) & 1);
      sd = fma(xd[j], xd[j], sd);
    }
    sd = warp_sum(sd);
    const double normd = sd == 0.0 ? 1e-8 : sqrt(sd);
    fwht_warp<J>(xd, lane);
    double vd = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      bit[j] = xd[j] > P.midd * normd;
      const double v = xd[j] - (bit[j] ? P.c1d : P.c0d) * normd;
      res[j] = v >= 0.0;
      vd = fma(v, v, vd);
    }
    vd = warp_sum(vd);
    norm = (float)normd;
    rnorm = (float)sqrt(vd * (1.0 / D));
  }
  const int64_t page = slot / r.page_size;
  const int64_t row = (page * r.n_kv_heads + h) * r.page_size + (slot - page * r.page_size);
  const PagedPool& pool = is_v ? r.vp : r.kp;
  uint32_t cw = 0, rw = 0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const uint32_t c = __ballot_sync(0xffffffffu, bit[j]);
    const uint32_t s = __ballot_sync(0xffffffffu, res[j]);
    if (lane == j) cw = c;
    if (lane == j) rw = s;
  }
  if (lane < J) {
    pool.code[row * J + lane] = cw;
    pool.res[row * J + lane] = rw;
  }
  if (lane == 0) {
    pool.norms[row] = norm;
    pool.rnorms[row] = rnorm == 0.f ? 1e-8f : rnorm;
  }
}

template <typename T, int D>
kh_status launch_typed(const AppendParams& P, cudaStream_t stream) {
  const int64_t items = P.r.n_tokens * P.r.n_kv_heads * 2;
  const int64_t blocks = (items + 3) / 4;
  if (blocks > 0x7fffffffll) return KH_EINVAL;
  if (launch_programmatic(paged_append_kernel<T, D>, dim3((unsigned)blocks), dim3(128), 0, stream,
                          P) != cudaSuccess)
    return KH_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? KH_OK : KH_ELAUNCH;
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
