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

#include "kh_common.cuh"
#include "kh_paged.h"

namespace kh {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnParams {
  PagedAttnRequest r;
  PagedPlan plan;
  uint32_t* err;
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
// Flat plane row of position j of sequence b, or -1 (recorded) when the
// table holds no page of the pool there.
__device__ __forceinline__ int64_t row_of(const AttnParams& P, int64_t b, int h, int64_t j) {
  const int64_t blk = j / P.r.page_size;
  const int32_t page = P.r.table[b * P.r.table_stride + blk];
  if (page < 0 || page >= P.r.n_pages) {
    flag_error(P.err, kErrBadIndex);
    return -1;
  }
  return ((int64_t)page * P.r.n_kv_heads + h) * P.r.page_size + (j - blk * P.r.page_size);
}

// cap tanh(t / cap): 1 - 2 / (e^2x + 1) loses what is left of small x, so
// below 0.3 the odd series (next term x^13, under 2^-24 of x there).
__device__ __forceinline__ float soft_cap(float t, float cap, float inv_cap) {
  const float x = t * inv_cap, a = fabsf(x);
  const float big = copysignf(1.f - 2.f / (__expf(2.f * fminf(a, 20.f)) + 1.f), x);
  const float z = x * x;
  float s = fmaf(z, 0.0035921280f, -0.0088632355f);
  s = fmaf(z, s, 0.021869488f);
  s = fmaf(z, s, -0.053968254f);
  s = fmaf(z, s, 0.13333333f);
  s = fmaf(z, s, -0.33333333f);
  const float small = fmaf(x * z, s, x);
  return cap * (a < 0.3f ? small : big);
}

constexpr int kTile = 128;  // rows per step: one per thread
constexpr int kNq = 8;      // query rows per CTA

template <int D>
__global__ void __launch_bounds__(kTile) paged_attn_kernel(const __grid_constant__ AttnParams P) {
  constexpr int W = D / 32;
  const PagedAttnRequest& r = P.r;
  __shared__ float qt[kNq][D];
  __shared__ float w1[kNq][kTile], w2[kNq][kTile];
  __shared__ uint32_t vc[kTile][W + 1], vr[kTile][W + 1];
  __shared__ float red[kTile / 32];
  const int tid = threadIdx.x;
  const int h = blockIdx.y % r.n_kv_heads;
  const int64_t seq = blockIdx.y / r.n_kv_heads;  // 0: the prefix when there is one
  const bool pre = P.plan.pre_chunks > 0 && seq == 0;
  const int64_t b = pre ? 0 : seq - (P.plan.pre_chunks > 0 ? 1 : 0);
  const int chunk = blockIdx.x;
  if (chunk >= (pre ? P.plan.pre_chunks : P.plan.own_chunks)) return;
  const int64_t n_rows = pre ? r.n_seqs * r.n_q : r.n_q;
  const int64_t y0 = (int64_t)blockIdx.z * kNq;
  if (y0 >= n_rows) return;
  const int nq = (int)min((int64_t)kNq, n_rows - y0);
  grid_dependency_wait();
  int64_t lo, hi;
  if (pre) {
    lo = chunk * P.plan.pre_rows;
    hi = min(lo + P.plan.pre_rows, r.prefix_len);
  } else {
    const int64_t len = length_of(P, b);
    const int64_t base = own_first(P, b, len);
    lo = base + chunk * P.plan.own_rows;
    hi = min(lo + P.plan.own_rows, len);
    if (lo >= hi) return;
  }
  const int hq_all = r.n_kv_heads * r.n_q;
  auto seq_of = [&](int y) { return pre ? (y0 + y) / r.n_q : b; };
  auto head_of = [&](int y) { return h * r.n_q + (int)(pre ? (y0 + y) % r.n_q : y0 + y); };
  const float inv_sd = rsqrtf((float)D);
  for (int y = 0; y < nq; ++y) {
    const int64_t base = (seq_of(y) * hq_all + head_of(y)) * D;
    for (int e = tid; e < D; e += kTile) {
      const float v = ld_any(r.q, r.dtype, base + e);
      qt[y][e] = (r.dk_neg[e >> 5] >> (e & 31)) & 1 ? -v : v;
    }
  }
  __syncthreads();
  for (int s = 1; s < D; s <<= 1) {
    for (int i = tid; i < nq * (D / 2); i += kTile) {
      const int y = i / (D / 2), k = i % (D / 2);
      const int e = (k / s) * 2 * s + (k % s);
      const float a = qt[y][e], c = qt[y][e + s];
      qt[y][e] = a + c;
      qt[y][e + s] = a - c;
    }
    __syncthreads();
  }
  for (int i = tid; i < nq * D; i += kTile) qt[i / D][i % D] *= inv_sd;
  __syncthreads();

  float m[kNq], l[kNq], acc[kNq][D / kTile];
#pragma unroll
  for (int y = 0; y < kNq; ++y) {
    m[y] = -INFINITY;
    l[y] = 0.f;
#pragma unroll
    for (int i = 0; i < D / kTile; ++i) acc[y][i] = 0.f;
  }
  const float inv_cap = r.softcap > 0.f ? 1.f / r.softcap : 0.f;
  for (int64_t j0 = lo; j0 < hi; j0 += kTile) {
    const int64_t j = j0 + tid;
    const int64_t row = j < hi ? row_of(P, b, h, j) : -1;
    uint32_t kc[W], kr[W];
    float kn = 0.f, krn = 0.f, vn = 0.f, vrn = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      kc[w] = row >= 0 ? r.kp.code[row * W + w] : 0u;
      kr[w] = row >= 0 ? r.kp.res[row * W + w] : 0u;
      vc[tid][w] = row >= 0 ? r.vp.code[row * W + w] : 0u;
      vr[tid][w] = row >= 0 ? r.vp.res[row * W + w] : 0u;
    }
    if (row >= 0) {
      kn = r.kp.norms[row];
      krn = r.kp.rnorms[row] * inv_sd;
      vn = r.vp.norms[row] * inv_sd;
      vrn = r.vp.rnorms[row] * (0.7978845608028654f / D);
    }
#pragma unroll
    for (int y = 0; y < kNq; ++y) {
      if (y >= nq) break;
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
          const float q = qt[y][32 * w + i];
          s1 += q * ((kc[w] >> i) & 1 ? r.c1 : r.c0);
          s2 += (kr[w] >> i) & 1 ? q : -q;
        }
      float t = (kn * s1 + krn * s2) * r.sm_scale;
      if (r.softcap > 0.f) t = soft_cap(t, r.softcap, inv_cap);
      const int64_t len = length_of(P, seq_of(y));
      if (r.slopes) t -= r.slopes[head_of(y)] * (float)(len - 1 - j);
      const bool on = row >= 0 && j < len && j >= first_of(P, seq_of(y), len);
      t = on ? t * kLog2e : -INFINITY;
      float mx = t;
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      __syncthreads();
      if ((tid & 31) == 0) red[tid >> 5] = mx;
      __syncthreads();
      mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      const float mn = fmaxf(m[y], mx);
      const float f = mn == -INFINITY ? 1.f : exp2f(m[y] - mn);
      const float p = on ? exp2f(t - mn) : 0.f;
      w1[y][tid] = on ? p * vn : 0.f;
      w2[y][tid] = on ? p * vrn : 0.f;
      float ps = p;
      for (int o = 16; o; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
      __syncthreads();
      if ((tid & 31) == 0) red[tid >> 5] = ps;
      __syncthreads();
      l[y] = l[y] * f + ((red[0] + red[1]) + (red[2] + red[3]));
      m[y] = mn;
#pragma unroll
      for (int i = 0; i < D / kTile; ++i) acc[y][i] *= f;
    }
    __syncthreads();
    const int n = (int)min((int64_t)kTile, hi - j0);
    for (int k = 0; k < n; ++k)
#pragma unroll
      for (int i = 0; i < D / kTile; ++i) {
        const int e = tid + i * kTile;
        const float c = (vc[k][e >> 5] >> (e & 31)) & 1 ? r.c1 : r.c0;
        const bool s = (vr[k][e >> 5] >> (e & 31)) & 1;
#pragma unroll
        for (int y = 0; y < kNq; ++y)
          if (y < nq) acc[y][i] += w1[y][k] * c + (s ? w2[y][k] : -w2[y][k]);
      }
    __syncthreads();
  }
  const int part = pre ? chunk : P.plan.pre_chunks + chunk;
#pragma unroll
  for (int y = 0; y < kNq; ++y) {
    if (y >= nq) break;
    float* rec = r.workspace +
                 ((seq_of(y) * hq_all + head_of(y)) * P.plan.parts() + part) * (int64_t)(D + 2);
    if (tid == 0) {
      rec[0] = m[y];
      rec[1] = l[y];
    }
#pragma unroll
    for (int i = 0; i < D / kTile; ++i) rec[2 + tid + i * kTile] = acc[y][i];
  }
}

// One warp per query row: its records merged, element 32 j + lane in a[j].
template <int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const __grid_constant__ AttnParams P) {
  constexpr int J = D / 32;
  const PagedAttnRequest& r = P.r;
  const int lane = threadIdx.x & 31;
  const int hq_all = r.n_kv_heads * r.n_q;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  grid_dependency_wait();
  if (row >= r.n_seqs * hq_all) return;
  const int64_t b = row / hq_all;
  const int64_t len = length_of(P, b);
  const int64_t own = max((int64_t)0, len - own_first(P, b, len));
  const int n_own = P.plan.own_rows
                        ? (int)min((own + P.plan.own_rows - 1) / P.plan.own_rows,
                                   (int64_t)P.plan.own_chunks)
                        : 0;
  const int n = P.plan.pre_chunks + n_own;
  const float* rec = r.workspace + row * P.plan.parts() * (int64_t)(D + 2);
  float mx = -INFINITY;
  for (int p = lane; p < n; p += 32)
    if (rec[p * (D + 2) + 1] > 0.f) mx = fmaxf(mx, rec[p * (D + 2)]);
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float l = 0.f, a[J];
#pragma unroll
  for (int j = 0; j < J; ++j) a[j] = 0.f;
  for (int p = 0; p < n; ++p) {
    const float* q = rec + p * (D + 2);
    const float lp = q[1];
    if (!(lp > 0.f)) continue;  // nothing attended there
    const float f = exp2f(q[0] - mx);
    l = fmaf(lp, f, l);
#pragma unroll
    for (int j = 0; j < J; ++j) a[j] = fmaf(q[2 + 32 * j + lane], f, a[j]);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const float y = __shfl_xor_sync(0xffffffffu, a[j], o);
      a[j] = up ? y - a[j] : a[j] + y;
    }
  }
#pragma unroll
  for (int h = 1; h < J; h <<= 1)
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (!(j & h)) {
        const float x = a[j], y = a[j + h];
        a[j] = x + y;
        a[j + h] = x - y;
      }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const float v = l > 0.f ? a[j] * inv : 0.f;
    st_any(r.out, r.dtype, row * D + 32 * j + lane, (r.dv_neg[j] >> lane) & 1 ? -v : v);
  }
  if (r.lse && lane == 0) r.lse[row] = l > 0.f ? (mx + log2f(l)) * kLn2 : -INFINITY;
}

template <int D>
kh_status launch_dim(const AttnParams& P, cudaStream_t stream) {
  const PagedAttnRequest& r = P.r;
  const int64_t rows = r.n_seqs * r.n_kv_heads * r.n_q;
  if (P.plan.parts() > 0) {
    const int64_t gy = (r.n_seqs + (P.plan.pre_chunks > 0 ? 1 : 0)) * r.n_kv_heads;
    const int64_t nq = P.plan.pre_chunks > 0 ? r.n_seqs * r.n_q : r.n_q;
    const int64_t gz = (nq + kNq - 1) / kNq;
    if (gy > 65535 || gz > 65535) return KH_EINVAL;
    const dim3 grid((unsigned)std::max(P.plan.pre_chunks, P.plan.own_chunks), (unsigned)gy,
                    (unsigned)gz);
    if (launch_programmatic(paged_attn_kernel<D>, grid, dim3(kTile), 0, stream, P) != cudaSuccess)
      return KH_ELAUNCH;
  }
  if (launch_programmatic(paged_combine_kernel<D>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0,
                          stream, P) != cudaSuccess)
    return KH_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? KH_OK : KH_ELAUNCH;
}

}  // namespace

PagedPlan paged_plan(int64_t n_seqs, int n_q, int n_kv_heads, int D, int64_t max_len,
                     int64_t prefix_len, int64_t window, int n_sms) {
  PagedPlan p;
  (void)n_sms;
  (void)D;
  const int64_t chunk = 1024;
  const int64_t pre = std::min(prefix_len, max_len);
  int64_t own = max_len - pre;
  if (window > 0) own = std::min(own, window);
  if (pre > 0) {
    p.pre_rows = chunk;
    p.pre_chunks = (int)((pre + chunk - 1) / chunk);
  }
  if (own > 0) {
    p.own_rows = chunk;
    p.own_chunks = (int)((own + chunk - 1) / chunk);
  }
  return p;
}

kh_status launch_paged_attn(const PagedAttnRequest& r, cudaStream_t stream) {
  AttnParams P;
  P.r = r;
  P.plan = paged_plan(r.n_seqs, r.n_q, r.n_kv_heads, r.D, r.max_len, r.prefix_len, r.window,
                      sm_count());
  P.err = device_error_ptr();
  return r.D == 128 ? launch_dim<128>(P, stream) : launch_dim<256>(P, stream);
}

}  // namespace kh
