// A ragged batch's keys and values appended to a paged cache, with the rotary embedding applied to q and k
// on the way (the KV write and RoPE of scripts/llm/llama_q4.py:206-223, for a batch).
//
//   (a, b) -> (a cos - b sin, b cos + a sin) over the pairs (i, i + rot/2) or (2i, 2i + 1) of a head's first
//   rot elements; the other elements and v are copied.
//
// Bound by memory: every element is read once and written once (plus 4 rot bytes of table per token, read
// through L1 by the token's heads). A task is 16 elements of one head: both sides of eight pairs, so that
// every access is 16 or 32 bytes. A CTA takes `tok` tokens: first each token's place (sequence, page, slot,
// position) is found by one warp, then all threads walk the tasks. Few tokens get one CTA each (latency),
// many share CTAs so that the searches are paid once per 8 tokens. Measured: 13,375 rows of 32 + 2 * 8 heads of 128 in
// bf16 (336 MB) 59 us, 5.7 TB/s, 0.87 of the copy rate; one token 3.6 us, which is the launch. Stepping through the
// tasks without divisions, 16-byte table loads and four tokens a CTA changed nothing or cost time (58-67 us).
#include <algorithm>

#include "paged.cuh"

namespace q4b {

int check_batch(const char* what, const q4b_batch* b, int rows) {
  if (!b) return set_error(Q4B_EINVAL, "%s: null batch", what);
  if (rows < 0 || b->batch < 0 || b->table_width < 0 || b->prefix_len < 0 || b->max_new < 0 || b->own_keys < 0)
    return set_error(Q4B_EINVAL, "%s: negative size", what);
  if (b->prefix_len > 0x7fffff00) return set_error(Q4B_EINVAL, "%s: prefix_len %d is too large", what, b->prefix_len);
  if (!b->q_start || (b->batch > 0 && !b->seq_lens) || (b->batch > 0 && b->table_width > 0 && !b->page_table))
    return set_error(Q4B_EINVAL, "%s: null batch array", what);
  if (b->batch > 1 && b->table_stride < b->table_width)
    return set_error(Q4B_EINVAL, "%s: page table rows overlap (stride %lld < width %d)", what, b->table_stride,
                     b->table_width);
  return Q4B_OK;
}

int check_paged_kv(const char* what, const q4b_paged_kv* kv) {
  if (!kv || !kv->k || !kv->v) return set_error(Q4B_EINVAL, "%s: null cache", what);
  if (kv->dtype != Q4B_F16 && kv->dtype != Q4B_BF16)
    return set_error(Q4B_EINVAL, "%s: the cache is fp16 or bf16", what);
  if (kv->n_pages < 1 || kv->page_size < 1 || kv->n_kv_heads < 1 || kv->head_dim < 1)
    return set_error(Q4B_EINVAL, "%s: empty cache", what);
  if (kv->page_stride % 8 || kv->slot_stride % 8 || kv->head_stride % 8 || kv->page_stride < 0 ||
      kv->slot_stride < 0 || kv->head_stride < 0)
    return set_error(Q4B_EINVAL, "%s: cache strides must be multiples of 8 elements", what);
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return set_error(Q4B_EINVAL, "%s: cache bases must be 16-byte aligned", what);
  return Q4B_OK;
}

namespace {

constexpr int kAppendThreads = 256;
constexpr int kMaxTok = kAppendThreads / 32;

struct AppendArgs {
  const void *q, *k, *v;
  long long q_stride, k_stride, v_stride;
  int rows, H, Hkv, hd, rot;
  const float *cos, *sin;
  long long rope_stride;
  int table_rows;
  q4b_batch b;
  q4b_paged_kv kv;
  void* q_out;
  int tok;
};

// 8 elements -> fp32, and fp32 -> 8 elements of the cache type
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Half16<T>::unpack(w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 a;
  a.x = Half16<T>::pack(x[0], x[1]);
  a.y = Half16<T>::pack(x[2], x[3]);
  a.z = Half16<T>::pack(x[4], x[5]);
  a.w = Half16<T>::pack(x[6], x[7]);
  *reinterpret_cast<uint4*>(p) = a;
}

enum : int { kSkip = 0, kLive = 1, kZero = 2 };

template <typename TX, typename TC, bool INTER>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(AppendArgs a) {
  __shared__ int s_state[kMaxTok];
  __shared__ long long s_off[kMaxTok];  // element offset of the token's slot, or -1
  __shared__ long long s_pos[kMaxTok];
  const int t0 = blockIdx.x * a.tok, nt = min(a.tok, a.rows - t0);
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < nt) {
    const int t = t0 + warp;
    const int b = batch_find(a.b.q_start, a.b.batch, t, lane);
    int state = kSkip;
    long long off = -1, pos = 0;
    if (b >= 0) {
      const int2 r = batch_rows(a.b.q_start, b, a.rows);
      const long long cap = (long long)a.b.table_width * a.kv.page_size;
      // by the length as it is: behind the table's keys there is no slot, and no other token's slot is written instead
      const long long s = (long long)__ldg(a.b.seq_lens + b) - (r.y - r.x) + (t - r.x);
      pos = a.b.prefix_len + s;
      state = a.rot == 0 || (pos >= 0 && pos < a.table_rows) ? kLive : kZero;
      if (state == kLive && s >= 0 && s < cap) {
        const int pi = (int)(s / a.kv.page_size);
        const int page = __ldg(a.b.page_table + b * a.b.table_stride + pi);
        if (page >= 0 && page < a.kv.n_pages)
          off = page * a.kv.page_stride + (s - (long long)pi * a.kv.page_size) * a.kv.slot_stride;
      }
    }
    if (lane == 0) {
      s_state[warp] = state;
      s_off[warp] = off;
      s_pos[warp] = pos;
    }
  }
  __syncthreads();

  const int per_head = a.hd >> 4, heads = a.H + 2 * a.Hkv, per_tok = heads * per_head;
  const int rot_tasks = a.rot >> 4;
  for (int i = threadIdx.x; i < nt * per_tok; i += kAppendThreads) {
    const int ti = i / per_tok, w = i - ti * per_tok;
    const int head = w / per_head, c = w - head * per_head;
    const int state = s_state[ti];
    if (state == kSkip) continue;
    const int t = t0 + ti;
    const bool is_q = head < a.H, is_k = !is_q && head < a.H + a.Hkv;
    const long long off = s_off[ti];
    if (!is_q && (off < 0 || state == kZero)) continue;
    const TX* src;
    TC* dst;
    if (is_q) {
      src = static_cast<const TX*>(a.q) + t * a.q_stride + head * a.hd;
      dst = static_cast<TC*>(a.q_out) + ((long long)t * a.H + head) * a.hd;
    } else {
      const int kh = head - a.H - (is_k ? 0 : a.Hkv);
      src = is_k ? static_cast<const TX*>(a.k) + t * a.k_stride + kh * a.hd
                 : static_cast<const TX*>(a.v) + t * a.v_stride + kh * a.hd;
      dst = static_cast<TC*>(is_k ? a.kv.k : a.kv.v) + off + kh * a.kv.head_stride;
    }
    const bool turn = c < rot_tasks && (is_q || is_k);
    const int e0 = (!INTER && turn) ? 8 * c : 16 * c;
    const int e1 = (!INTER && turn) ? 8 * c + (a.rot >> 1) : 16 * c + 8;
    // v of a half-rotated head walks the head in order, so it takes elements 16 c .. 16 c + 15 like the rest
    float x[8], y[8];
    if (state == kZero) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.0f;
    } else {
      load8(src + e0, x);
      load8(src + e1, y);
      if (turn) {
        const float* cp = a.cos + s_pos[ti] * a.rope_stride + 8 * c;
        const float* sp = a.sin + s_pos[ti] * a.rope_stride + 8 * c;
        float cs[8], sn[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) cs[j] = __ldg(cp + j), sn[j] = __ldg(sp + j);
        if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float a0 = x[2 * j], b0 = x[2 * j + 1], a1 = y[2 * j], b1 = y[2 * j + 1];
            x[2 * j] = a0 * cs[j] - b0 * sn[j];
            x[2 * j + 1] = b0 * cs[j] + a0 * sn[j];
            y[2 * j] = a1 * cs[4 + j] - b1 * sn[4 + j];
            y[2 * j + 1] = b1 * cs[4 + j] + a1 * sn[4 + j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float a0 = x[j], b0 = y[j];
            x[j] = a0 * cs[j] - b0 * sn[j];
            y[j] = b0 * cs[j] + a0 * sn[j];
          }
        }
      }
    }
    store8(dst + e0, x);
    store8(dst + e1, y);
  }
}

template <typename TX, typename TC>
int launch(const AppendArgs& a, bool inter, cudaStream_t st) {
  const int grid = (a.rows + a.tok - 1) / a.tok;
  const cudaError_t e = inter ? launch_pdl(paged_append_kernel<TX, TC, true>, grid, kAppendThreads, 0, st, a)
                              : launch_pdl(paged_append_kernel<TX, TC, false>, grid, kAppendThreads, 0, st, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(Q4B_ELAUNCH, "paged_rope_append: launch failed: %s", cudaGetErrorString(e));
  }
  return Q4B_OK;
}

}  // namespace
}  // namespace q4b

using namespace q4b;

extern "C" int q4b_paged_rope_append(const void* q, const void* k, const void* v, int x_dtype, long long q_stride,
                                     long long k_stride, long long v_stride, int rows, int n_heads,
                                     const float* rope_cos, const float* rope_sin, long long rope_stride,
                                     int table_rows, int rot_dim, int interleaved, const q4b_batch* batch,
                                     const q4b_paged_kv* kv, void* q_out, q4b_stream_t stream) {
  const char* what = "paged_rope_append";
  if (int rc = check_batch(what, batch, rows)) return rc;
  if (int rc = check_paged_kv(what, kv)) return rc;
  if (!q || !k || !v || !q_out) return set_error(Q4B_EINVAL, "%s: null pointer", what);
  if ((kv->n_pages > 1 && kv->page_stride == 0) || (kv->page_size > 1 && kv->slot_stride == 0) ||
      (kv->n_kv_heads > 1 && kv->head_stride == 0))
    return set_error(Q4B_EINVAL, "%s: the cache's slots overlap (a stride of zero)", what);
  if (x_dtype != Q4B_F32 && x_dtype != kv->dtype)
    return set_error(Q4B_EINVAL, "%s: q, k and v are fp32 or of the cache's type", what);
  if (n_heads < 1) return set_error(Q4B_EINVAL, "%s: n_heads < 1", what);
  if (kv->head_dim % 16 || rot_dim < 0 || rot_dim % 16 || rot_dim > kv->head_dim)
    return set_error(Q4B_EINVAL, "%s: head_dim and rot_dim must be multiples of 16, rot_dim <= head_dim", what);
  if (rot_dim && (!rope_cos || !rope_sin || table_rows < 0 || (table_rows > 1 && rope_stride < rot_dim / 2)))
    return set_error(Q4B_EINVAL, "%s: bad rotation tables", what);
  if (q_stride % 8 || k_stride % 8 || v_stride % 8 || !aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) ||
      !aligned(q_out, 16))
    return set_error(Q4B_EINVAL, "%s: q, k, v, q_out must be 16-byte aligned with row strides that are multiples of 8", what);
  if ((long long)(n_heads + 2ll * kv->n_kv_heads) * kv->head_dim > (1 << 24))
    return set_error(Q4B_EUNSUPPORTED, "%s: more than 2^24 elements a row", what);
  if (rows == 0 || batch->batch == 0) return Q4B_OK;
  // A task reads its 16 elements before it writes them, so q_out may be q, element for element; any other overlap is read by
  // tasks that run after it was written.
  const size_t size = x_dtype == Q4B_F32 ? 4 : 2, q_row = (size_t)n_heads * kv->head_dim, kv_row = (size_t)kv->n_kv_heads * kv->head_dim;
  auto over = [&](const void* x, long long stride, size_t row) {
    return overlap(x, ((size_t)(rows - 1) * (size_t)stride + row) * size, q_out, (size_t)rows * q_row * 2);
  };
  const bool in_place = q_out == q && size == 2 && (rows == 1 || q_stride == (long long)q_row);
  if ((!in_place && over(q, q_stride, q_row)) || over(k, k_stride, kv_row) || over(v, v_stride, kv_row))
    return set_error(Q4B_EINVAL, "%s: q_out overlaps q, k or v (it may be q itself, of the cache's type and contiguous)", what);
  AppendArgs a;
  a.q = q, a.k = k, a.v = v;
  a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
  a.rows = rows, a.H = n_heads, a.Hkv = kv->n_kv_heads, a.hd = kv->head_dim, a.rot = rot_dim;
  a.cos = rope_cos, a.sin = rope_sin, a.rope_stride = rope_stride, a.table_rows = table_rows;
  a.b = *batch, a.kv = *kv, a.q_out = q_out;
  a.tok = rows <= 148 * 8 ? 1 : rows <= 148 * 16 ? 2 : rows <= 148 * 32 ? 4 : kMaxTok;
  const cudaStream_t st = as_stream(stream);
  if (kv->dtype == Q4B_F16)
    return x_dtype == Q4B_F32 ? launch<float, __half>(a, interleaved != 0, st) : launch<__half, __half>(a, interleaved != 0, st);
  return x_dtype == Q4B_F32 ? launch<float, __nv_bfloat16>(a, interleaved != 0, st)
                            : launch<__nv_bfloat16, __nv_bfloat16>(a, interleaved != 0, st);
}
