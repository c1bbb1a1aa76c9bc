// kh_paged.h -- host-side requests of the paged cache operators, shared by the
// C-ABI checks (kh_api.cu) and the kernels.
#pragma once

#include "kh_internal.h"

namespace kh {

// One tensor's page pool: row (page, kv head, offset) is row
// (page * n_kv_heads + head) * page_size + offset of the flat planes.
struct PagedPool {
  uint32_t* code;
  uint32_t* res;
  float* norms;
  float* rnorms;
};

struct PagedAppendRequest {
  const void *k, *v;
  int dtype;
  int64_t n_tokens;
  int n_kv_heads, D;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;  // elements
  const int64_t* slots;
  const int64_t* positions;  // nullptr: keys are not rotated
  const float *cos, *sin;    // [n_positions][rot_dim / 2]
  int64_t n_positions;
  int rot_dim;
  int interleaved;
  uint32_t dk_neg[8], dv_neg[8];  // bit i: d of element i is -1
  float c0, c1;
  PagedPool kp, vp;
  int64_t n_pages;
  int page_size;
};
kh_status launch_paged_append(const PagedAppendRequest& r, cudaStream_t stream);

struct PagedAttnRequest {
  const void* q;  // [n_seqs][n_kv_heads * n_q][D]
  int dtype;
  int64_t n_seqs;
  int n_q, n_kv_heads, D;
  PagedPool kp, vp;
  int64_t n_pages;
  int page_size;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* starts;  // may be null
  int64_t max_len, prefix_len;
  int64_t window;  // 0: none
  float softcap;   // 0: none
  const float* slopes;  // [n_kv_heads * n_q] or null
  float sm_scale;
  uint32_t dk_neg[8], dv_neg[8];
  float c0, c1;
  float* workspace;
  void* out;
  float* lse;  // may be null
};

// How a call's rows are cut, from what the host knows of it.
struct PagedPlan {
  // the rows kernel: query rows of a group, groups of a KV head (the prefix's,
  // and a sequence's own), their rows, tiles of 32 and units at most
  int block = 1, pre_blocks = 0, own_blocks = 0;
  int64_t pre_rows = 0, own_rows = 0, groups = 0, tiles = 0, max_units = 0;
  // the prefix on the tensor cores: chunks of chunk_rows rows
  int pre_chunks = 0;
  int64_t chunk_rows = 0;
};
PagedPlan paged_plan(int64_t n_seqs, int n_q, int n_kv_heads, int D, int64_t max_len,
                     int64_t prefix_len, int64_t window, int dtype, int n_sms);
int64_t paged_workspace_bytes(const PagedPlan& p, int64_t n_seqs, int n_q, int n_kv_heads, int D);
kh_status launch_paged_attn(const PagedAttnRequest& r, cudaStream_t stream);

}  // namespace kh
