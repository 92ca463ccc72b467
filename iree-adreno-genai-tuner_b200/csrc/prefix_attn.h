// Internal interface of the shared-prefix attention kernels.
#pragma once

#include "common.cuh"

namespace q4b {

struct PrefixArgs {
  const void* q;  // [rows, H, hd] of the cache's type
  long long q_stride, q_head_stride;
  int rows, H, Hkv, g;  // g = H / Hkv
  float scale2;         // scale * log2(e)
  q4b_batch b;
  q4b_paged_kv kv;
  const int32_t* prefix_pages;
  void* out;  // [rows, H * hd]
  int prefix_units;  // key tiles of the prefix's items
  int* cum;          // [batch + 1] key tiles of the own keys' items in front of sequence b
  float2* row_ml;    // [2][rows * H] (max, sum) of whole items, prefix then own keys
  float* row_o;      // [2][rows * H][hd] their weighted V
  float2* cut_ml;    // [CTAs][2][row tile] the same of cut items
  float* cut_o;
};

}  // namespace q4b
