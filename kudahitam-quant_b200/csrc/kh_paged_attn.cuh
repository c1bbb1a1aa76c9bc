// kh_paged_attn.cuh -- what the paged attention kernels share: the request as
// the device sees it, the rows a sequence attends, the score's cap.
#pragma once

#include "kh_common.cuh"
#include "kh_paged.h"

namespace kh {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// How the rows kernel's tiles are cut (kh_paged_attn.cu), and whose prefix is read.
struct Units {
  int64_t size;
  uint64_t mul;  // floor(2^64 / size) + 1: x / size while x size < 2^64
  // The prefix is read through the table of the first sequence that has all of
  // it, or else of the longest: places of a batch may be empty or short.
  int64_t source;
  int64_t pre_end;  // rows of it that `source` has
  __device__ __forceinline__ int64_t of(int64_t x) const {
    return (int64_t)__umul64hi((uint64_t)x, mul);
  }
};

struct AttnParams {
  PagedAttnRequest r;
  PagedPlan plan;
  float log_scale, inv_sd;  // sm_scale log2(e) / sqrt(D); 1 / sqrt(D)
  // j / page_size for j < 2^31: (j * mul) >> shift, mul = ceil(2^shift / page_size),
  // shift = 31 + ceil(log2 page_size) (the error j (mul page_size - 2^shift) / 2^shift stays under 1)
  uint64_t div_mul;
  int div_shift;
  uint32_t step_blocks, step_off;  // 32 rows on: whole pages and the rest
  // of the rows kernel (kh_paged_attn.cu)
  int64_t n_warps;
  float* records;
  int64_t* starts;
  int2* own;  // a sequence's own rows: first, end
  Units* units;
  void* frags;
  int pre_tensor;  // the prefix has its own launches (launch_paged_prefix)
  uint16_t* queries;  // workspace of those: q~ in fp16, tile by tile
  uint32_t* err;

  __device__ __forceinline__ uint32_t page_div(uint32_t j) const {
    return (uint32_t)((j * div_mul) >> div_shift);
  }
};

__device__ __forceinline__ float ld_any(const void* p, int dtype, int64_t i) {
  if (dtype == KH_F32) return static_cast<const float*>(p)[i];
  if (dtype == KH_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void st_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == KH_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == KH_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Attention of every sequence's queries over the shared prefix, a record per
// query row and chunk (kh_paged_prefix.cu).
kh_status launch_paged_prefix(const AttnParams& P, cudaStream_t stream);

// Its operand in the workspace: a KV head's query rows in groups of MT tiles of
// 128, then the group's scales, a float a row.
template <int D>
struct QueryTiles {
  static constexpr int MT = D == 128 ? 2 : 1;
  static constexpr int kTile = 128 * D * 2;  // bytes
  static constexpr int kGroup = MT * (kTile + 512);
};

// Length of sequence b, within what the table and max_len hold.
__device__ __forceinline__ int64_t length_of(const AttnParams& P, int64_t b) {
  int64_t n = P.r.lengths[b];
  if (n < 0 || n > P.r.max_len) {
    flag_error(P.err, kErrBadIndex);
    n = n < 0 ? 0 : P.r.max_len;
  }
  return n;
}
// First attended row of sequence b.
__device__ __forceinline__ int64_t first_of(const AttnParams& P, int64_t b, int64_t len) {
  int64_t lo = P.r.starts ? max((int64_t)P.r.starts[b], (int64_t)0) : 0;
  if (P.r.window > 0) lo = max(lo, len - P.r.window);
  return lo;
}
// Where a sequence's own rows begin.
__device__ __forceinline__ int64_t own_first(const AttnParams& P, int64_t b, int64_t len) {
  return max(first_of(P, b, len), P.r.prefix_len);
}
// cap tanh(t / cap): 1 - 2 / (e^2x + 1) loses what is left of small x, so
// below 0.3 the odd series (its next term is under 2^-33 of x there).  A NaN
// stays one: it compares false twice.
__device__ __forceinline__ float soft_cap(float t, float cap, float inv_cap) {
  const float x = t * inv_cap, a = fabsf(x);
  const float big = copysignf(1.f - 2.f / (__expf(2.f * (a > 20.f ? 20.f : a)) + 1.f), x);
  const float z = x * x;
  float s = fmaf(z, 0.0035921280f, -0.0088632355f);
  s = fmaf(z, s, 0.021869488f);
  s = fmaf(z, s, -0.053968254f);
  s = fmaf(z, s, 0.13333333f);
  s = fmaf(z, s, -0.33333333f);
  const float small = fmaf(x * z, s, x);
  return cap * (a < 0.3f ? small : big);
}

// The same for 16-bit queries: off by 2^-18 of it at most (2^-22 of the cap in
// the exponential and the reciprocal, from x = 1/16 up; the series' next term is
// 2^-28 there), a sixteenth of what the queries' own steps cost.  The division
// above takes so much code that the tensor-core kernel, which holds it 32 times,
// ran 165 us instead of 100 on 73 x 24 capped bf16 queries over 5188 rows.
__device__ __forceinline__ float soft_cap_16(float t, float cap, float inv_cap) {
  const float x = t * inv_cap, a = fabsf(x);
  float e, f;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(2.f * kLog2e * a));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(e + 1.f));
  const float z = x * x;
  const float small = fmaf(x * z, fmaf(z, 0.13333333f, -0.33333333f), x);
  return cap * (a < 0.0625f ? small : copysignf(fmaf(-2.f, f, 1.f), x));
}

// Walsh-Hadamard sums of a warp's row: element 32 j + lane in x[j].
template <int J>
__device__ __forceinline__ void fwht_lanes(float (&x)[J], int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const float y = __shfl_xor_sync(0xffffffffu, x[j], o);
      x[j] = up ? y - x[j] : x[j] + y;
    }
  }
#pragma unroll
  for (int h = 1; h < J; h <<= 1)
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (!(j & h)) {
        const float a = x[j], b = x[j + h];
        x[j] = a + b;
        x[j + h] = a - b;
      }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
constexpr float kNoRef = -1e30f;  // reference exponent before the first row
// Values count in full down to this norm (weights times norms have the references;
// at 2^-40 values of 1e-20 came out as noise); the weights alone then stay
// under 2^100, and sums of them in range.
constexpr float kLeastNorm = 0x1p-90f;

}  // namespace kh
