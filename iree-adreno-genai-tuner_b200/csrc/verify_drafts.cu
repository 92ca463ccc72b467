// Verification of drafted tokens against the target's probabilities, from given random numbers (the greedy
// head of scripts/llm/llama_q4.py:237-239, for sampling with a draft model).
//
//   draft x at row r is kept while u_r d_r(x) < p_r(x); behind the kept ones a token is drawn by inversion from
//   w = max(p - d, 0) of that row (p of the last row if all were kept): the first j with W_j > u W_{V-1}, W the
//   running sum of w.
//
// The sums have 40 bits and more (64-bit words, and pairs of fp32 words over 16 values at a time): a running sum of 10^5
// probabilities in fp32 is off by more than a typical w, and the drawn index would depend on the order of the sum. The products u d of the tests are exact in 64 bits.
//
// Bound by memory: one row of p, and of d where a draft was rejected, per sequence; the acceptance tests read
// two numbers per draft. A cluster of CTAs takes one sequence, so that a row's read is spread over several
// SMs in one launch: each warp sums an equal piece of the row, the pieces' sums go to every CTA through
// distributed shared memory, and the CTA whose warp holds the drawn index reads that piece again (from L2),
// a few values a thread, to find it. What is left is latency: offsets, tokens, the tested numbers, the row, the
// exchange and the piece are dependent reads. Measured: one sequence over 32064 fp32 values 6.0 us; 64 sequences of up to
// 6 rows over 128256 values 17.6 us, of which the rows' 53 MB take 10; 155 over 49999 fp16 values 14.0 us.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace q4b {
namespace {

constexpr int kVfThreads = 256, kVfWarps = kVfThreads / 32;
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxCluster = 8, kMaxPieces = kMaxCluster * kVfWarps;

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

// A sum in two fp32 words, emptied into 64 bits after every kFlush values. The error of an fp32 addition or subtraction is
// itself an fp32 number, found by Dekker's fast two-sum (of numbers a >= b >= 0, s = a + b: b - (s - a), and s = a - b:
// (a - s) - b); the errors are added up in `lo`, which rounds too. With u = 2^-24 and S the sum of n values, an error is
// at most u S, those of the differences together u S, so |lo| <= (k + 1) u S after k values, and the roundings of lo and of
// its addends together u^2 S (n^2 / 2 + 5 n / 2 + 1): 169 u^2 S < 2^-40 S for n = 16. (Not emptied, over the 2048 values a
// lane that 2^20 values on 16 warps make, equal values far below one large one put the drawn index several tokens off.)
// Conversions to 64 bits and 64-bit additions for every value took three times as long as the row's read.
constexpr int kFlush = 16;
struct Sum2 {
  double sum = 0.0;
  float hi = 0.0f, lo = 0.0f;
  float top = 0.0f;  // largest value met: an infinite one sends the piece to the careful sum
  __device__ __forceinline__ void add(float x, float e) {  // x >= 0
    const float a = fmaxf(hi, x), b = fminf(hi, x);
    hi = __fadd_rn(a, b);
    lo = __fadd_rn(lo, __fadd_rn(__fsub_rn(b, __fsub_rn(hi, a)), e));
  }
  __device__ __forceinline__ void flush() {
    top = fmaxf(top, hi);
    sum += (double)hi + (double)lo;
    hi = lo = 0.0f;
  }
  __device__ __forceinline__ void add_target(float p) {
    p = fmaxf(p, 0.0f);  // NaN and negative: zero
    top = fmaxf(top, p);
    add(p, 0.0f);
  }
  __device__ __forceinline__ void add_rest(float p, float d) {
    p = fmaxf(p, 0.0f), d = fmaxf(d, 0.0f);
    top = fmaxf(top, fmaxf(p, d));
    const float s = __fsub_rn(p, d);  // has the exact difference's sign
    if (s > 0.0f) add(s, __fsub_rn(__fsub_rn(p, s), d));
  }
};

// A row cut into equal pieces, at 16-byte vectors where p and d are aligned alike (the first piece then takes the values
// in front of the first vector too, the last one those behind the last), else at single values (vectors 0).
template <typename T>
struct Row {
  static constexpr int N = 16 / sizeof(T);
  int vocab, pieces, head, vectors;
  __device__ __forceinline__ Row(const Weights<T>& w, int vocab, int pieces) : vocab(vocab), pieces(pieces) {
    const int mis = (int)(reinterpret_cast<uintptr_t>(w.p) % 16 / sizeof(T));
    head = min(mis ? N - mis : 0, vocab);
    vectors = (vocab - head) / N;
    if (w.d && reinterpret_cast<uintptr_t>(w.d) % 16 != reinterpret_cast<uintptr_t>(w.p) % 16) vectors = 0;
  }
  __device__ __forceinline__ int vector(int k) const { return (int)((long long)vectors * k / pieces); }
  __device__ __forceinline__ int value(int k) const {
    if (k == 0) return 0;
    if (k == pieces) return vocab;
    return vectors ? head + vector(k) * N : (int)((long long)vocab * k / pieces);
  }
};

// A lane's share of the weights of vectors [lo, hi), every 32nd; four 16-byte loads (p's, and d's) in flight.
template <typename T, bool REST>
__device__ __forceinline__ double lane_sum(const Weights<T>& w, int head, int lo, int hi, int lane) {
  constexpr int N = 16 / sizeof(T), U = 4;
  static_assert(U * N % kFlush == 0, "nothing is left in the fp32 words at the end");
  const T* p = w.p + head;
  const T* d = REST ? w.d + head : nullptr;
  Sum2 sum;
  for (int v0 = lo + lane; v0 < hi; v0 += 32 * U) {
    uint4 pv[U], dv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + 32 * u;
      pv[u] = dv[u] = make_uint4(0, 0, 0, 0);
      if (v < hi) pv[u] = ld_stream_u4(p + (long long)v * N);
      if (REST && v < hi) dv[u] = ld_stream_u4(d + (long long)v * N);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float a[N];
      unpack16<T>(pv[u], a);
      if constexpr (REST) {
        float b[N];
        unpack16<T>(dv[u], b);
#pragma unroll
        for (int i = 0; i < N; ++i) sum.add_rest(a[i], b[i]);
      } else {
        const unsigned at = (unsigned)(w.skip - head - (v0 + 32 * u) * N);
#pragma unroll
        for (int i = 0; i < N; ++i) sum.add_target(at == (unsigned)i ? 0.0f : a[i]);
      }
      if ((u + 1) * N % kFlush == 0) sum.flush();
    }
  }
  if (!(sum.top < INFINITY)) {  // an infinite value counts as zero
    double s = 0.0;
    for (int v = lo + lane; v < hi; v += 32)
      for (int i = 0; i < N; ++i) s += w.at(head + v * N + i);
    return s;
  }
  return sum.sum;
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

// CTAs that an SM holds: registers for p's and d's loads in flight, or p's alone.
template <bool DRAFT>
constexpr int kResident = DRAFT ? 4 : 5;

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(kVfThreads, kResident<DRAFT>) verify_kernel(VerifyArgs a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int nc = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / nc;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ double s_piece[2][kMaxPieces];  // every warp's sum (twice: the residual, then the target)
  __shared__ double s_part[kVfWarps];
  __shared__ int s_kept, s_first, s_some;
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
          const float d = DRAFT ? prob(as_float(static_cast<const T*>(a.draft)[row * a.draft_stride + x])) : 1.0f;
          ok = (double)__ldg(a.uniforms + row) * (double)d < (double)p;
        }
      }
      const unsigned bad = __ballot_sync(0xffffffffu, !ok);
      if (bad) {
        kept = i0 + __ffs(bad) - 1;
        break;
      }
    }
    if (lane == 0) {
      s_kept = kept;
      s_first = kVfThreads;
      s_some = 0;
    }
  }
  __syncthreads();
  const int kept = s_kept;
  const long long row = r.x + kept;
  const bool cut = kept < n - 1;
  Weights<T> w;
  w.p = static_cast<const T*>(a.target) + row * a.target_stride;
  w.d = DRAFT && cut ? static_cast<const T*>(a.draft) + row * a.draft_stride : nullptr;
  w.skip = !DRAFT && cut ? __ldg(a.tokens + row + 1) : -1;

  const int pieces = nc * kVfWarps, piece = rank * kVfWarps + warp;
  double total = 0.0, before = 0.0;  // before: of the pieces in front of this lane's two
  double mine0 = 0.0, mine1 = 0.0;   // pieces 2 lane and 2 lane + 1
  int round = 0;
  for (;; ++round) {
    const Row<T> row_of(w, a.vocab, pieces);
    double s = 0.0;
    int lo = row_of.value(piece), hi = row_of.value(piece + 1);
    if (row_of.vectors) {
      const int v0 = row_of.vector(piece), v1 = row_of.vector(piece + 1), h = row_of.head;
      s = DRAFT && w.d ? lane_sum<T, true>(w, h, v0, v1, lane) : lane_sum<T, false>(w, h, v0, v1, lane);
      // the values outside vectors: at most N - 1 in front and behind
      if (lo + lane < h + v0 * Row<T>::N) s += w.at(lo + lane);
      if (h + v1 * Row<T>::N + lane < hi) s += w.at(h + v1 * Row<T>::N + lane);
    } else {
#pragma unroll 8
      for (int i = lo + lane; i < hi; i += 32) s += w.at(i);
    }
    s = warp_sum(s);
    if (round == 0) cluster.barrier_wait();
    if (lane < nc) *cluster.map_shared_rank(&s_piece[round][piece], lane) = s;
    cluster.sync();
    mine0 = 2 * lane < pieces ? s_piece[round][2 * lane] : 0.0;
    mine1 = 2 * lane + 1 < pieces ? s_piece[round][2 * lane + 1] : 0.0;
    const double end = warp_scan(mine0 + mine1, lane);
    total = __shfl_sync(0xffffffffu, end, 31);
    before = end - (mine0 + mine1);
    // an empty residual: draw from the target (the same decision in every warp: they hold the same sums)
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

  // The piece that holds the index: the first whose end lies above the mark; where rounding leaves the mark at the
  // very end, the last one with any weight. Every warp decides the same.
  const double mark = (double)__ldg(a.uniforms + r.y - 1) * total;
  auto choose = [&](bool above, bool any, int& lane_of) {  // first lane above, else the last with weight
    const unsigned m = __ballot_sync(0xffffffffu, above), o = __ballot_sync(0xffffffffu, any);
    lane_of = m ? __ffs(m) - 1 : 31 - __clz(o);
    return m != 0;
  };
  int f;
  const double mid = before + mine0, end = mid + mine1;
  const bool above0 = mine0 > 0.0 && mid > mark, above1 = mine1 > 0.0 && end > mark;
  const bool found = choose(above0 || above1, mine0 > 0.0 || mine1 > 0.0, f);
  const bool second = found ? !above0 : mine1 > 0.0;
  const int at = __shfl_sync(0xffffffffu, 2 * lane + second, f);
  const double base = __shfl_sync(0xffffffffu, second ? mid : before, f);
  if (at / kVfWarps != rank) return;

  // Its values again, a run for each thread of the CTA, and the index by the same rule.
  const Row<T> row_of(w, a.vocab, pieces);
  const int lo = row_of.value(at), hi = row_of.value(at + 1), share = (hi - lo + kVfThreads - 1) / kVfThreads;
  const int from = min(lo + (int)threadIdx.x * share, hi), to = min(from + share, hi);
  double sum = 0.0;
#pragma unroll 8
  for (int i = from; i < to; ++i) sum += w.at(i);
  double run = warp_scan(sum, lane);
  if (lane == 31) s_part[warp] = run;
  __syncthreads();
  run += base;
  for (int k = 0; k < warp; ++k) run += s_part[k];
  if (sum > 0.0) {
    atomicMax(&s_some, (int)threadIdx.x);
    if (run > mark) atomicMin(&s_first, (int)threadIdx.x);
  }
  __syncthreads();
  if ((int)threadIdx.x != (s_first < kVfThreads ? s_first : s_some)) return;
  double cum = run - sum;
  int pick = -1;
  for (int i = from; i < to; ++i) {
    const double v = w.at(i);
    if (v > 0.0) {
      pick = i;
      cum += v;
      if (cum > mark) break;
    }
  }
  a.out_tokens[row] = pick;
}

template <typename T, bool DRAFT>
int launch(const VerifyArgs& a, cudaStream_t st) {
  // As many CTAs for each sequence as the SMs hold at once (a second wave for a few of them took half of the time again), 2 at
  // least.
  const int slots = 148 * kResident<DRAFT>;
  const int nc = a.batch * 8ll <= slots ? 8 : a.batch * 4ll <= slots ? 4 : 2;
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<T, DRAFT>, a);
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
  // other CTAs and warps read a sequence's tokens, numbers and offsets while its results are written
  const size_t n = 4 * (size_t)rows, nb = 4 * (size_t)batch;
  for (const void* in : {(const void*)tokens, (const void*)uniforms})
    if (overlap(in, n, out_tokens, n) || overlap(in, n, accepted, nb))
      return set_error(Q4B_EINVAL, "%s: the results overlap tokens or uniforms", what);
  if (overlap(q_start, nb + 4, out_tokens, n) || overlap(q_start, nb + 4, accepted, nb) || overlap(out_tokens, n, accepted, nb))
    return set_error(Q4B_EINVAL, "%s: the results overlap q_start or each other", what);
  VerifyArgs a;
  a.target = target, a.draft = draft;
  a.target_stride = target_stride, a.draft_stride = draft_stride;
  a.vocab = vocab, a.rows = rows, a.batch = batch;
  a.tokens = tokens, a.q_start = q_start, a.uniforms = uniforms;
  a.out_tokens = out_tokens, a.accepted = accepted;
  const cudaStream_t st = as_stream(stream);
  if (dtype == Q4B_F32) return draft ? launch<float, true>(a, st) : launch<float, false>(a, st);
  if (dtype == Q4B_F16) return draft ? launch<__half, true>(a, st) : launch<__half, false>(a, st);
  return draft ? launch<__nv_bfloat16, true>(a, st) : launch<__nv_bfloat16, false>(a, st);
}
