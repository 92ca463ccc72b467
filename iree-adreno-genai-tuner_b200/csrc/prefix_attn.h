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
  // the prefix's whole 128-key tiles on the tensor cores (tc_splits 0: not used); the rest of the prefix, from key
  // prefix_skip, stays with the other kernel
  int tc_splits, tc_pairs, tc_tiles, prefix_skip;
  float2* tc_ml;  // [tc_splits][rows * H]
  float* tc_o;    // [tc_splits][rows * H][hd]
};

struct PrefixTcPlan {
  int splits, pairs, tiles;  // splits 0: the tensor-core kernel does not take this call
};
constexpr int kTcMaxSplits = 32;
constexpr int kTcMinRows = 33;
PrefixTcPlan prefix_tc_plan(int rows, int H, int prefix_len, const q4b_paged_kv& kv);
int prefix_tc_run(const PrefixArgs& a, cudaStream_t st);
unsigned prefix_status(bool reset);

}  // namespace q4b
