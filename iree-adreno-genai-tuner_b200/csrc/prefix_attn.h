// Internal interface of the shared-prefix attention kernels.
#pragma once

#include "common.cuh"

namespace q4b {

// The work of one kernel: items (KV head, row tile) of the prefix and of the sequences whose rows times heads per KV head
// lie in (own_lo, own_hi], all their key tiles ("units") in one line, of which each CTA takes an equal run.
struct AttnLine {
  int prefix_units;
  int own_lo, own_hi;
};

struct PrefixArgs {
  const void* q;  // [rows, H, hd] of the cache's type
  long long q_stride, q_head_stride;
  int rows, H, Hkv, g;  // g = H / Hkv
  float scale2;         // scale * log2(e)
  q4b_batch b;
  int table_keys;  // keys that a row of the page table holds
  q4b_paged_kv kv;
  const int32_t* prefix_pages;
  void* out;  // [rows, H * hd]
  int tc_ctas;       // CTAs of the tensor-core kernel, 0: not launched
  int mm_ctas;       // CTAs of the mma.sync kernel
  int mm_rows;       // its rows per row tile: 8 or 16 (narrow), 64 (wide)
  AttnLine tc, mm;
  int4* rec;         // [rows]: where the join finds a row's own item (join_records)
  int* totals;       // units of the mm line, own units of the tc line
  float2* row_ml;    // [2][rows * H] (max, sum) of items that one CTA did whole, prefix then own keys
  float* row_o;      // [2][rows * H][hd] their weighted V
  float2* mm_ml;     // [CTAs][2][mm_rows] the same of items cut between CTAs
  float* mm_o;
  float2* tc_ml;     // [prefix, own][CTAs][2][kTcRows]
  float* tc_o;
  unsigned long long wait_ns;  // limit of the kernels' waits
};

constexpr int kTcRows = 256, kTcKeys = 128, kTcCtas = 148;
constexpr int kTcWholeTiles = 8;  // own items of up to so many tiles are not cut between CTAs
constexpr int kMmKeys = 64;
constexpr int kTcMaxBatch = 2048;  // the sequences' table shares the tensor-core kernel's shared memory
// Prefix tiles of 16 rows x 64 keys from which the tensor-core kernel takes them. 32 single tokens of 3 heads a KV head, 60 own
// keys each: behind 768 keys (576 tiles) 17.3 us with it and 19.8 without, behind 2048 (1536) 20.0 and 31.3. The line was drawn
// for the kernels one behind the other; side by side it pays from fewer tiles on (512 keys, 384 tiles: 16.5 and 18.7).
constexpr int kTcMinUnits = 500;
constexpr int kTcMinRows = 64;     // rows x heads of a sequence from which it takes the own keys

// Rows of a TMA box: the largest power of two that divides both the page (a multiple of 8) and the tile, so that no box
// crosses a page or a tile.
__host__ __device__ inline int page_box(int page_size, int tile) {
  const int low = page_size & -page_size;
  return low < tile ? low : tile;
}

// whether the kernels that load by TMA can read this cache
bool prefix_tc_takes(const q4b_paged_kv& kv);
// whether the tensor-core kernel is as its register split needs it (asks the runtime); a build where it is not leaves all
// items to the other kernels
bool prefix_tc_built(const q4b_paged_kv& kv);
int prefix_tc_run(const PrefixArgs& a, cudaStream_t st);
unsigned prefix_tc_status(bool reset);
unsigned narrow_status(bool reset);

}  // namespace q4b
