// What the batched serving kernels share: the ragged batch, the paged cache, and 16-bit types.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace q4b {

// fp32 <-> the 16-bit cache types, pairwise (one packed 32-bit register)
template <typename T>
struct Half16;
template <>
struct Half16<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Half16<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Rows of sequence b, bounded: begin in [0, rows], end in [begin, rows].
__device__ __forceinline__ int2 batch_rows(const int32_t* q_start, int b, int rows) {
  const int lo = min(max(__ldg(q_start + b), 0), rows);
  return make_int2(lo, min(max(__ldg(q_start + b + 1), lo), rows));
}

// The sequence that holds row t, or -1: the last b with q_start[b] <= t, if its rows reach t. By a whole warp, 32
// probes a round: the loads of a round run side by side (one round up to 32 sequences, two up to 1055).
__device__ __forceinline__ int batch_find(const int32_t* q_start, int batch, int t, int lane) {
  int lo = 0, n = batch;  // the first b with q_start[b] > t is in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) / 32, at = lane * step;
    const int c = __popc(__ballot_sync(0xffffffffu, at < n && __ldg(q_start + lo + min(at, n - 1)) <= t));
    if (c == 0) break;
    const int skip = (c - 1) * step + 1;
    lo += skip;
    n = min(step - 1, n - skip);
  }
  if (lo == 0) return -1;
  return t < __ldg(q_start + lo) ? lo - 1 : -1;
}

// Host checks shared by the entry points; Q4B_OK or an error whose message names `what`.
int check_batch(const char* what, const q4b_batch* b, int rows);
int check_paged_kv(const char* what, const q4b_paged_kv* kv);

}  // namespace q4b
