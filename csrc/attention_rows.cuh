// Parameters of the attention calls with a 4-bit cache or a window (attention_rows.cu, kv4.cu).
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace braid {

struct RowsParams {
  const __nv_bfloat16* q;   // rows of [Hq, D], q_stride elements apart
  int64_t q_stride;
  const uint8_t* kv;        // bf16 pool [P, 2, Hkv, PS, D] or the 4-bit codes
  const uint32_t* scales;   // 4-bit (s, z) pairs
  __nv_bfloat16* out;       // [T, Hq, D]
  const int* qo_indptr;
  const int* positions;
  const int* seg_indptr;
  const int* seg_page_indptr;
  const int* seg_offset;
  const int* seg_len;
  const int* seg_pos0;
  const int* seg_delta;
  const int* page_ids;
  const float* cos;
  const float* sin;
  float scale_log2, q_sign;  // |scale| log2(e) (at least 1e-20), the sign of scale
  int use_rope, rope_len;
  int Hq, Hkv, G, PS, num_pages;
  int window, sinks;        // window 0: every earlier key
  int splits;               // CTAs per cluster
  int whole;                // 4-bit: a tile lies in one page (the page size is a multiple of it)
  unsigned long long* span;
};

}  // namespace braid
