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

// The sequence that holds row t, or -1: the last b with q_start[b] <= t, if its rows reach t.
__device__ __forceinline__ int batch_find(const int32_t* q_start, int batch, int t) {
  int lo = 0, hi = batch;  // first b in [0, batch] with q_start[b] > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(q_start + mid) <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  if (lo == 0) return -1;
  return t < __ldg(q_start + lo) ? lo - 1 : -1;
}

// Host checks shared by the entry points; Q4B_OK or an error whose message names `what`.
int check_batch(const char* what, const q4b_batch* b, int rows);
int check_paged_kv(const char* what, const q4b_paged_kv* kv);

}  // namespace q4b
