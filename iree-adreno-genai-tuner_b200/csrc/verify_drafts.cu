// Verification of drafted tokens against the target's probabilities, from given random numbers (the greedy
// head of scripts/llm/llama_q4.py:237-239, for sampling with a draft model).
//
//   draft x at row r is kept while u_r d_r(x) < p_r(x); behind the kept ones a token is drawn by inversion from
//   w = max(p - d, 0) of that row (p of the last row if all were kept): the first j with W_j > u W_{V-1}, W the
//   running sum of w.
//
// The sums have 43 bits and more (64-bit words where it matters, pairs of fp32 words over the values of a
// lane): a running sum of 10^5 probabilities in fp32 is off by more than a typical w, and the
// drawn index would depend on the order of the sum. The products u d of the tests are exact in 64 bits.
//
// Bound by memory: one row of p, and of d where a draft was rejected, per sequence; the acceptance tests read
// two numbers per draft. A cluster of CTAs takes one sequence, so that a row's read is spread over several
// SMs in one launch: each CTA sums its slice in tiles of 1024 values (a warp per tile, the tile sums stay
// in shared memory), the slices' sums meet through distributed shared memory, and the CTA whose slice holds
// the drawn index reads that one tile again (from L2) to find it.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace q4b {
namespace {

constexpr int kVfThreads = 256, kVfWarps = kVfThreads / 32;
constexpr int kTile = 1024;                  // values per tile
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxCluster = 8;

struct VerifyArgs {
  const void *target, *draft;
  long long target_stride, draft_stride;
  int vocab, rows, batch;
  const int32_t *tokens, *q_start;
  const float* uniforms;
  int32_t *out_tokens, *accepted;
};

template <typename T>
__device__ __forceinline__ float as_float(T v) {
  return static_cast<float>(v);
}
// a probability: negative, infinite and NaN count as zero
__device__ __forceinline__ float prob(float v) { return v > 0.0f && v < INFINITY ? v : 0.0f; }

// The weight of index i: how the residual and the plain row are drawn from with one code.
//   d != null: max(p - d, 0);  skip >= 0: p without index skip;  else p
template <typename T>
struct Weights {
  const T* p;
  const T* d;
  int skip;
  __device__ __forceinline__ double of(float pv, float dv) const {
    const double w = (double)prob(pv) - (double)prob(dv);
    return w > 0.0 ? w : 0.0;
  }
  __device__ __forceinline__ double at(int i) const {
    if (i == skip) return 0.0;
    return of(as_float(p[i]), d ? as_float(d[i]) : 0.0f);
  }
};

template <typename T, int N>
__device__ __forceinline__ void unpack16(const uint4& v, float (&x)[N]) {
  static_assert(N == 16 / sizeof(T), "one 16-byte vector");
  if constexpr (sizeof(T) == 4) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  } else {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Half16<T>::unpack(u[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}

// A sum in two fp32 words. The error of each fp32 addition and subtraction is itself an fp32 number, found
// by Knuth's two-sum; the errors are added up in `lo`. Over the 32 values of a lane hi + lo is off by
// less than 2^-43 of the sum, far below the share of one token, at fp32 speed: conversions to 64
// bits and 64-bit additions for every value took three times as long as the row's read.
struct Sum2 {
  float hi = 0.0f, lo = 0.0f;
  float top = 0.0f;  // largest value met: an infinite one sends the tile to the careful sum
  __device__ __forceinline__ void add(float x, float e) {
    const float s = __fadd_rn(hi, x), b = __fsub_rn(s, hi);
    lo = __fadd_rn(lo, __fadd_rn(__fadd_rn(__fsub_rn(hi, __fsub_rn(s, b)), __fsub_rn(x, b)), e));
    hi = s;
  }
  __device__ __forceinline__ void add_target(float p) {
    p = fmaxf(p, 0.0f);  // NaN and negative: zero
    top = fmaxf(top, p);
    add(p, 0.0f);
  }
  __device__ __forceinline__ void add_rest(float p, float d) {
    p = fmaxf(p, 0.0f), d = fmaxf(d, 0.0f);
    top = fmaxf(top, fmaxf(p, d));
    const float s = __fsub_rn(p, d), b = __fsub_rn(s, p);
    const float e = __fsub_rn(__fsub_rn(p, __fsub_rn(s, b)), __fadd_rn(d, b));
    if (s > 0.0f) add(s, e);  // the rounded difference has the exact one's sign
  }
};

// This lane's share of the weights of tile [lo, lo + kTile), whose bounds are 16-byte aligned in p and d: every
// 32nd vector (coalesced), or, with `runs`, the 32 values from lo + 32 lane.
template <typename T>
__device__ __forceinline__ double lane_sum_vec(const Weights<T>& w, int lo, int lane, bool runs) {
  constexpr int N = 16 / sizeof(T), U = kTile / (32 * N), HALF = U / 2;
  Sum2 sum;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint4 pv[HALF], dv[HALF];
    auto first = [&](int u) { return lo + N * (runs ? lane * U + h * HALF + u : (h * HALF + u) * 32 + lane); };
#pragma unroll
    for (int u = 0; u < HALF; ++u) {
      pv[u] = ld_stream_u4(w.p + first(u));
      if (w.d) dv[u] = ld_stream_u4(w.d + first(u));
    }
#pragma unroll
    for (int u = 0; u < HALF; ++u) {
      float a[N];
      unpack16<T>(pv[u], a);
      if (w.d) {
        float b[N];
        unpack16<T>(dv[u], b);
#pragma unroll
        for (int i = 0; i < N; ++i) sum.add_rest(a[i], b[i]);
      } else {
        const unsigned at = (unsigned)(w.skip - first(u));
#pragma unroll
        for (int i = 0; i < N; ++i) sum.add_target(at == (unsigned)i ? 0.0f : a[i]);
      }
    }
  }
  const bool odd = !(sum.top < INFINITY && sum.hi < INFINITY);
  if (__any_sync(0xffffffffu, odd)) {  // an infinite value counts as zero
    double s = 0.0;
    for (int i = 0; i < kTile / 32; ++i) s += w.at(lo + (runs ? lane * (kTile / 32) + i : i * 32 + lane));
    return s;
  }
  return (double)sum.hi + (double)sum.lo;
}

template <typename T>
__device__ __forceinline__ double tile_sum_any(const Weights<T>& w, int lo, int hi, int lane) {
  double s = 0.0;
#pragma unroll 8
  for (int i = lo + lane; i < hi; i += 32) s += w.at(i);
  return s;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// inclusive running sum over the lanes
__device__ __forceinline__ double warp_scan(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kVfThreads, 4) verify_kernel(VerifyArgs a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int nc = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / nc;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ double s_tile[kMaxVocab / kTile + 2];  // this CTA's tile sums
  __shared__ double s_cta[2][kMaxCluster];          // every CTA's sum (twice: the residual, then the target)
  __shared__ double s_part[kVfWarps];
  __shared__ int s_kept;
  cluster.barrier_arrive();  // waited for before the first write to another CTA: by then all have started
  griddep_launch_dependents();
  griddep_wait();
  const int2 r = batch_rows(a.q_start, b, a.rows);
  const int n = r.y - r.x;
  if (n == 0) {
    cluster.barrier_wait();
    if (rank == 0 && threadIdx.x == 0) a.accepted[b] = 0;
    return;
  }
  // acceptance: every CTA of the cluster makes the same test on two numbers per draft
  if (warp == 0) {
    int kept = n - 1;
    for (int i0 = 0; i0 < n - 1; i0 += 32) {
      bool ok = true;
      if (i0 + lane < n - 1) {
        const int row = r.x + i0 + lane;
        const int x = __ldg(a.tokens + row + 1);
        ok = false;
        if (x >= 0 && x < a.vocab) {
          const float p = prob(as_float(static_cast<const T*>(a.target)[row * a.target_stride + x]));
          const float d = a.draft ? prob(as_float(static_cast<const T*>(a.draft)[row * a.draft_stride + x])) : 1.0f;
          ok = (double)__ldg(a.uniforms + row) * (double)d < (double)p;
        }
      }
      const unsigned bad = __ballot_sync(0xffffffffu, !ok);
      if (bad) {
        kept = i0 + __ffs(bad) - 1;
        break;
      }
    }
    if (lane == 0) s_kept = kept;
  }
  __syncthreads();
  const int kept = s_kept;
  const long long row = r.x + kept;
  const bool cut = kept < n - 1;
  Weights<T> w;
  w.p = static_cast<const T*>(a.target) + row * a.target_stride;
  w.d = cut && a.draft ? static_cast<const T*>(a.draft) + row * a.draft_stride : nullptr;
  w.skip = cut && !a.draft ? __ldg(a.tokens + row + 1) : -1;

  // Tiles: `head` values up to p's first 16-byte boundary, then tiles of 1024, the last one short. Where d
  // is aligned otherwise than p, no tile takes the vector path.
  constexpr int N = 16 / sizeof(T);
  const int mis = (int)((reinterpret_cast<uintptr_t>(w.p) % 16) / sizeof(T));
  const int head = min(mis ? N - mis : 0, a.vocab);
  const int tiles = 1 + (a.vocab - head + kTile - 1) / kTile;
  const int t_lo = (int)((long long)tiles * rank / nc), t_hi = (int)((long long)tiles * (rank + 1) / nc);
  auto lo_of = [&](int t) { return t == 0 ? 0 : head + (t - 1) * kTile; };
  auto hi_of = [&](int t) { return t == 0 ? head : min(head + t * kTile, a.vocab); };

  double base = 0.0, total = 0.0;
  int round = 0;
  for (;; ++round) {
    const bool vec = !w.d || reinterpret_cast<uintptr_t>(w.d) % 16 == reinterpret_cast<uintptr_t>(w.p) % 16;
    double mine = 0.0;
    for (int t = t_lo + warp; t < t_hi; t += kVfWarps) {
      const int lo = lo_of(t), hi = hi_of(t);
      const double s = warp_sum(vec && hi - lo == kTile ? lane_sum_vec(w, lo, lane, false) : tile_sum_any(w, lo, hi, lane));
      if (lane == 0) s_tile[t - t_lo] = s;
      mine += s;
    }
    if (lane == 0) s_part[warp] = mine;
    __syncthreads();
    if (round == 0) cluster.barrier_wait();
    if (threadIdx.x < nc) {
      double s = 0.0;
      for (int i = 0; i < kVfWarps; ++i) s += s_part[i];
      *cluster.map_shared_rank(&s_cta[round][rank], threadIdx.x) = s;
    }
    cluster.sync();
    base = total = 0.0;
    for (int c = 0; c < nc; ++c) {
      if (c == rank) base = total;
      total += s_cta[round][c];
    }
    // an empty residual: draw from the target (the same decision in every CTA: they hold the same sums)
    if (total > 0.0 || (!w.d && w.skip < 0)) break;
    w.d = nullptr;
    w.skip = -1;
  }

  if (rank == 0) {
    for (int i = threadIdx.x; i < n; i += kVfThreads) {
      if (i < kept) a.out_tokens[r.x + i] = __ldg(a.tokens + r.x + i + 1);
      if (i > kept) a.out_tokens[r.x + i] = -1;
    }
    if (threadIdx.x == 0) {
      a.accepted[b] = kept;
      if (!(total > 0.0)) a.out_tokens[row] = -1;
    }
  }
  if (!(total > 0.0)) return;

  // The CTA whose slice holds the index: the first whose end lies above the mark; where rounding leaves the
  // mark at the very end, the last slice with any weight (every CTA decides the same).
  const double mark = (double)__ldg(a.uniforms + r.y - 1) * total;
  int owner = -1, some = 0;
  double run = 0.0;
  for (int c = 0; c < nc; ++c) {
    run += s_cta[round][c];
    if (owner < 0 && run > mark) owner = c;
    if (s_cta[round][c] > 0.0) some = c;
  }
  if (owner < 0) owner = some;
  if (owner != rank || warp != 0) return;

  // its tile, by the same rule
  int tile = -1, tile_some = t_lo;
  double cum = base, tile_base = base;
  for (int t0 = t_lo; t0 < t_hi && tile < 0; t0 += 32) {
    const double s = t0 + lane < t_hi ? s_tile[t0 + lane - t_lo] : 0.0;
    const double end = cum + warp_scan(s, lane);
    const unsigned above = __ballot_sync(0xffffffffu, s > 0.0 && end > mark), any = __ballot_sync(0xffffffffu, s > 0.0);
    const int f = above ? __ffs(above) - 1 : any ? 31 - __clz(any) : -1;
    if (f >= 0) {
      tile_some = t0 + f;
      tile_base = __shfl_sync(0xffffffffu, end - s, f);
      if (above) tile = t0 + f;
    }
    cum = __shfl_sync(0xffffffffu, end, 31);
  }
  if (tile < 0) tile = tile_some;

  // its run of values: lane l sums run l of the tile
  const int lo = lo_of(tile), hi = hi_of(tile), per = (hi - lo + 31) / 32;
  const int from = min(lo + lane * per, hi), to = min(from + per, hi);
  double s = 0.0;
  if (hi - lo == kTile && (!w.d || reinterpret_cast<uintptr_t>(w.d) % 16 == reinterpret_cast<uintptr_t>(w.p) % 16)) {
    s = lane_sum_vec(w, lo, lane, true);
  } else {
#pragma unroll 8
    for (int i = from; i < to; ++i) s += w.at(i);
  }
  double end = tile_base + warp_scan(s, lane);
  unsigned above = __ballot_sync(0xffffffffu, s > 0.0 && end > mark), any = __ballot_sync(0xffffffffu, s > 0.0);
  const int f = above ? __ffs(above) - 1 : 31 - __clz(any);
  // its value: lane l takes value l of the run
  const int i = __shfl_sync(0xffffffffu, from, f) + lane;
  const double run_base = __shfl_sync(0xffffffffu, end - s, f);
  s = i < __shfl_sync(0xffffffffu, to, f) ? w.at(i) : 0.0;
  end = run_base + warp_scan(s, lane);
  above = __ballot_sync(0xffffffffu, s > 0.0 && end > mark), any = __ballot_sync(0xffffffffu, s > 0.0);
  if (lane == (above ? __ffs(above) - 1 : 31 - __clz(any))) a.out_tokens[row] = i;
}

template <typename T>
int launch(const VerifyArgs& a, cudaStream_t st) {
  // Few sequences: 8 CTAs each, for the latency of one row's read. Many: 2 each, which fill the SMs by
  // themselves and exchange less.
  const int nc = a.batch <= 148 ? kMaxCluster : 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.batch * nc);
  cfg.blockDim = dim3(kVfThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = nc;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<T>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(Q4B_ELAUNCH, "verify_drafts: launch failed: %s", cudaGetErrorString(e));
  }
  return Q4B_OK;
}

}  // namespace
}  // namespace q4b

using namespace q4b;

extern "C" int q4b_verify_drafts(const void* target, const void* draft, int dtype, long long target_stride,
                                 long long draft_stride, int vocab, const int32_t* tokens, const float* uniforms,
                                 int rows, const int32_t* q_start, int batch, int32_t* out_tokens, int32_t* accepted,
                                 q4b_stream_t stream) {
  const char* what = "verify_drafts";
  if (rows < 0 || batch < 0) return set_error(Q4B_EINVAL, "%s: negative size", what);
  if (vocab < 1 || vocab > kMaxVocab) return set_error(Q4B_EINVAL, "%s: vocab %d outside 1..%d", what, vocab, kMaxVocab);
  if (dtype != Q4B_F32 && dtype != Q4B_F16 && dtype != Q4B_BF16)
    return set_error(Q4B_EINVAL, "%s: probabilities are fp32, fp16 or bf16", what);
  if (batch > (1 << 24)) return set_error(Q4B_EINVAL, "%s: batch %d over 2^24", what, batch);
  if (batch == 0) return Q4B_OK;
  if (!q_start || !accepted || (rows > 0 && (!target || !tokens || !uniforms || !out_tokens)))
    return set_error(Q4B_EINVAL, "%s: null pointer", what);
  if (rows > 1 && (target_stride < vocab || (draft && draft_stride < vocab)))
    return set_error(Q4B_EINVAL, "%s: rows overlap (stride below vocab)", what);
  const size_t size = dtype == Q4B_F32 ? 4 : 2;
  if (!aligned(target, size) || !aligned(draft, size)) return set_error(Q4B_EINVAL, "%s: misaligned probabilities", what);
  VerifyArgs a;
  a.target = target, a.draft = draft;
  a.target_stride = target_stride, a.draft_stride = draft_stride;
  a.vocab = vocab, a.rows = rows, a.batch = batch;
  a.tokens = tokens, a.q_start = q_start, a.uniforms = uniforms;
  a.out_tokens = out_tokens, a.accepted = accepted;
  const cudaStream_t st = as_stream(stream);
  if (dtype == Q4B_F32) return launch<float>(a, st);
  return dtype == Q4B_F16 ? launch<__half>(a, st) : launch<__nv_bfloat16>(a, st);
}
