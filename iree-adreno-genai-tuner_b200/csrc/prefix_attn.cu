// Attention of a ragged batch over a paged cache whose sequences share a prefix (the GQA attention of
// scripts/llm/llama_q4.py:208-232, for a batch).
//
//   row (b, j), head h:  out = sum_s softmax_s(q . k_s * scale) v_s  over the prefix's keys and b's own keys
//   0 .. len_b - n_b + j;  zero if there are none.
//
// The prefix is read once for the whole batch: its queries are all rows of the step and all heads of a KV
// head's group. A sequence's own keys are read once for its rows and heads. Both are items (KV head, row tile)
// of key tiles, and all items' key tiles stand in one line, of which each CTA takes an equal run (whole
// items, and at most one cut item at either end): whatever the lengths, every SM streams the same number of
// bytes. Each run of an item leaves (max, sum, weighted V) in fp32; a last kernel joins a row's parts.
//
// Three kernels take items. The tensor-core kernel (prefix_attn_tc.cu) takes those with many rows. Here, with m16n8k16
// MMAs on the 16-bit values as stored, fp32 sums and an online softmax in base 2:
//
// Narrow (row tiles of 8 or 16: single tokens, a few drafts): bound by memory, or by the latency of a tile where a
// CTA has only a few. A producer warp looks the pages up and brings tiles of 64 keys by TMA (a box per page, 128-byte
// swizzle, a ring of STAGES tiles); four warps share a tile's keys, 16 each, and run free of one another but for
// the merge at an item's end. They hold S^T = K Q^T and O^T = V^T P^T: the keys fill the MMA's 16 rows and its 8
// columns are the query rows, where S = Q K^T would pad 3 or 4 query rows to 16. P^T moves from S^T's accumulator
// layout to a B operand by transposing 8 x 8 blocks in registers. Measured: 192 single tokens with 182,510 own keys
// (750 MB) 126 us, 5.9 TB/s, 0.91 of the copy rate, start and end included; with 16-byte copies by all threads
// instead of TMA 138 us (of the 1.5 us that a tile then took of a CTA's time 0.6 went into the copies' addresses).
// Wide (row tiles of 64): whatever the others cannot read (pages of other sizes, head_dim 32). 16-byte asynchronous
// copies, each warp 16 rows against all keys; items of up to 16 rows split the keys instead.
//
// P is rounded to the cache's type for the PV product: its error, half a step per weight, averages out over
// the keys and stays below the output's own rounding (fp16 ends early: kLift).
#include <algorithm>
#include <type_traits>

#include "attn_line.cuh"
#include "tc.cuh"

namespace q4b {
namespace {

constexpr int kThreads = 128;
constexpr int kRing = 8;  // page lookups in flight (tiles), >= STAGES + 2
constexpr int kSms = 148;
constexpr int kMaxBatch = 4096;

__device__ unsigned g_narrow_status = 0;

std::atomic<unsigned long long> g_wait_ns{kWaitLimitNs};

template <int HD>
struct Cfg {
  static constexpr int STAGES = HD == 128 ? 3 : 4;
  static constexpr int CTAS = HD == 128 ? 2 : 3;  // per SM
  static constexpr int HALF = kMmKeys * HD * 2;   // K (or V) of one tile
  static constexpr int STAGE = 2 * HALF;
  static constexpr int CHUNKS = HD / 8;           // 16-byte chunks of a row
};

// 16-byte chunk c of tile row r, swizzled so that 8 consecutive rows' equal chunks lie in 8 bank groups
template <int HD>
__device__ __forceinline__ uint32_t sw(int r, int c) {
  if constexpr (HD == 32) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  return r * (HD * 2) + ((c ^ (r & 7)) << 4);
}

// the same in the TMA's layout: 64-element (128-byte) halves of the tile one behind the other
__device__ __forceinline__ uint32_t sw_tma(int r, int c) { return (c >> 3) * (kMmKeys * 128) + r * 128 + (((c ^ r) & 7) << 4); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Zeros over shared memory that ldsm4 reads: a volatile asm like those, so that the compiler keeps their order.
__device__ __forceinline__ void st_zero16(uint32_t dst) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
// transposes an 8 x 8 block of 16-bit values held one row per four lanes
__device__ __forceinline__ uint32_t movm(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ const T* q_row(const PrefixArgs& a, const Cursor& c, int tr, int r) {
  const int rr = c.rt * tr + r, j = rr / a.g, head = c.h * a.g + rr - j * a.g;
  return static_cast<const T*>(a.q) + (long long)(c.q0 + j) * a.q_stride + (long long)head * a.q_head_stride;
}

// ---- wide form ---------------------------------------------------------------------------------------

template <typename T, int HD>
struct Wide {
  uint32_t q[HD / 16][4];
  float o[HD / 8][4];
  float m[2], l[2];
  int lim[2];  // keys that this lane's two rows see

  __device__ __forceinline__ void start(const PrefixArgs& a, const BatchTable& s, const Cursor& c, int r0, int lane) {
    const T* qp[2];
    bool on[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = r0 + (lane >> 2) + 8 * i;
      on[i] = r < c.nrows;
      qp[i] = q_row<T>(a, c, 64, r) + 2 * (lane & 3);
      lim[i] = row_limit(a, s, c, r, 64);
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < HD / 16; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        q[k][i] = on[i] ? __ldg(reinterpret_cast<const uint32_t*>(qp[i] + 16 * k)) : 0u;
        q[k][2 + i] = on[i] ? __ldg(reinterpret_cast<const uint32_t*>(qp[i] + 16 * k + 8)) : 0u;
      }
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
  }

  // NT n-tiles of 8 keys from key `k0` of the tile. `mask`: the tile's keys that exist; `whole`: all do,
  // for every row. `odd`: some V that not every row may see is infinite or NaN, so that 0 * v is not 0.
  template <int NT>
  __device__ __forceinline__ void tile(uint32_t ks, uint32_t vs, int k0, int key0, uint64_t mask, bool whole, bool odd,
                                       float scale2, int lane) {
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
    const int mat = lane >> 3, mr = lane & 7;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k)
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t f[4];
        ldsm4(f, ks + sw<HD>(k0 + n * 8 + (mat >> 1) * 8 + mr, 2 * k + (mat & 1)));
        mma<T>(s[n], q[k], f[0], f[1]);
        mma<T>(s[n + 1], q[k], f[2], f[3]);
      }
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = s[n][e] * scale2;
        if (!whole) {
          const int c = k0 + n * 8 + 2 * (lane & 3) + (e & 1);
          v = ((mask >> c) & 1) && key0 + c < lim[e >> 1] ? v : -INFINITY;
        }
        s[n][e] = v;
        mx[e >> 1] = fmaxf(mx[e >> 1], v);
      }
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      const float ref = mx[i] == -INFINITY ? 0.0f : mx[i];  // nothing seen yet: every weight below is exp2(-inf)
      f[i] = ex2(m[i] - ref);
      m[i] = mx[i];
      mx[i] = lifted<T, 0>(ref);
      l[i] *= f[i];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ex2(s[n][e] - mx[e >> 1]);
        l[e >> 1] += s[n][e];
      }
    if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= f[e >> 1];
    }
    if (!odd) {
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        const uint32_t p[4] = {Half16<T>::pack(s[n][0], s[n][1]), Half16<T>::pack(s[n][2], s[n][3]),
                               Half16<T>::pack(s[n + 1][0], s[n + 1][1]), Half16<T>::pack(s[n + 1][2], s[n + 1][3])};
#pragma unroll
        for (int d = 0; d < HD / 8; d += 2) {
          uint32_t v[4];
          ldsm4t(v, vs + sw<HD>(k0 + n * 8 + (mat & 1) * 8 + mr, d + (mat >> 1)));
          mma<T>(o[d], p, v[0], v[1]);
          mma<T>(o[d + 1], p, v[2], v[3]);
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll 1
        for (int c8 = 0; c8 < 8; ++c8) {
          const int src = (lane & ~3) | (c8 >> 1), c = k0 + n * 8 + c8;
          const float p0 = __shfl_sync(0xffffffffu, c8 & 1 ? s[n][1] : s[n][0], src);
          const float p1 = __shfl_sync(0xffffffffu, c8 & 1 ? s[n][3] : s[n][2], src);
          const bool there = (mask >> c) & 1;
          const bool see0 = there && key0 + c < lim[0], see1 = there && key0 + c < lim[1];
#pragma unroll
          for (int d = 0; d < HD / 8; ++d) {
            uint32_t w;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(vs + sw<HD>(c, d) + 4 * (lane & 3)));
            const float2 v = Half16<T>::unpack(w);
            if (see0) o[d][0] = fmaf(p0, v.x, o[d][0]), o[d][1] = fmaf(p0, v.y, o[d][1]);
            if (see1) o[d][2] = fmaf(p1, v.x, o[d][2]), o[d][3] = fmaf(p1, v.y, o[d][3]);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void end() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
  }
};

// column of element hd of row r in the merge buffers: spreads a warp's stores over the banks
__device__ __forceinline__ int merge_col(int r, int hd) { return hd ^ (((r >> 1) & 3) << 3); }

// For the join: where each row's own item lies. Sequences go round the CTAs. By all threads of the kernel that stands last in
// front of the join; waits for the kernel in front of it. Uses up the table's running sums.
template <int TR, int THREADS>
__device__ __forceinline__ void join_records(const PrefixArgs& a, const BatchTable& table, bool bad, int units, int* scan) {
  auto records = [&](const AttnLine& l, int first, int tr, bool tc) {
    for (int b = blockIdx.x; b < a.b.batch; b += gridDim.x) {
      const int n = table.q0[b + 1] - table.q0[b], mine = table.cum[b + 1] - table.cum[b];
      if (bad || n * a.g <= l.own_lo || n * a.g > l.own_hi) continue;
      const int row_tiles = (n * a.g + tr - 1) / tr, tiles = mine / (row_tiles * a.Hkv);
      for (int j = threadIdx.x; j < n; j += THREADS)
        a.rec[table.q0[b] + j] = make_int4(first + table.cum[b], tc ? -tiles : tiles, row_tiles, j);
    }
  };
  if (blockIdx.x == 0 && threadIdx.x == 0) a.totals[0] = units;
  records(a.mm, a.mm.prefix_units, TR, false);
  for (int t = blockIdx.x * THREADS + threadIdx.x; t < a.rows; t += gridDim.x * THREADS)
    if (bad || t < table.q0[0] || t >= table.q0[a.b.batch]) a.rec[t] = make_int4(0, 0, 1, -1);
  if (a.tc_ctas) {
    __syncthreads();
    const int own_units = line_table<THREADS, kTcRows, kTcKeys>(a, a.tc, table, bad, scan);
    records(a.tc, 0, kTcRows, true);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.totals[1] = own_units;
    griddep_wait();
  }
}


template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::CTAS) prefix_wide_kernel(PrefixArgs a) {
  using C = Cfg<HD>;
  constexpr int TR = 64, MERGE = 16;  // MERGE: rows of an item whose warps share the keys
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_koff[kRing][kMmKeys];  // byte offset of a tile's keys in the pools, -1: not there
  __shared__ unsigned s_mask[kRing][2];
  __shared__ int s_scan[kThreads / 32];
  __shared__ float s_m[4][MERGE], s_l[4][MERGE];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  BatchTable table;
  table.cum = reinterpret_cast<int*>(smem + C::STAGES * C::STAGE);
  table.q0 = table.cum + a.b.batch + 1;
  table.len = table.q0 + a.b.batch + 1;
  // Behind the tensor-core kernel the inputs are there already (it lets this kernel start only behind its own wait), and
  // its results matter to the join alone, which must find both kernels complete: so the wait comes last.
  griddep_launch_dependents();
  if (!a.tc_ctas) griddep_wait();
  const bool bad = batch_table<kThreads>(a, table);
  const int units = a.mm.prefix_units + line_table<kThreads, TR, kMmKeys>(a, a.mm, table, bad, s_scan);
  const Line<TR, kMmKeys> line{a, a.mm, table};
  const int ctas = min((int)gridDim.x, units);  // fewer units than CTAs: one each, so that no run is empty
  int u0 = 0, count = 0;
  if ((int)blockIdx.x < ctas) {
    u0 = cta_first(blockIdx.x, units, ctas);
    count = cta_first(blockIdx.x + 1, units, ctas) - u0;
  }

  const uint32_t s0 = smem_u32(smem);
  Cursor look = {};
  if (count) look = line.at(u0);
  Cursor cur = look;

  // Page lookup of a unit (the `look` cursor stands there): threads 0..63 take a key each. The load is left in flight.
  struct Lookup {
    int page, slot, h;
  };
  auto lookup = [&]() {
    Lookup l = {-1, 0, look.h};
    int key = look.tile * kMmKeys + tid;
    if (tid < kMmKeys && key < look.limit) {
      const int pi = key / a.kv.page_size;
      l.slot = key - pi * a.kv.page_size;
      l.page = __ldg(look.b < 0 ? a.prefix_pages + pi : a.b.page_table + look.b * a.b.table_stride + pi);
    }
    return l;
  };
  auto publish = [&](int x, const Lookup& l) {
    if (tid < kMmKeys) {
      const bool on = l.page >= 0 && l.page < a.kv.n_pages;
      s_koff[x % kRing][tid] = on ? 2 * (l.page * a.kv.page_stride + l.slot * a.kv.slot_stride + l.h * a.kv.head_stride) : -1;
      const unsigned bits = __ballot_sync(0xffffffffu, on);
      if (lane == 0) s_mask[x % kRing][warp] = bits;
    }
  };
  constexpr int PASS = kThreads / C::CHUNKS;  // tile rows per pass of the CTA's copies, a multiple of 8
  const int r0 = tid / C::CHUNKS;
  const uint32_t dst0 = s0 + sw<HD>(r0, tid % C::CHUNKS);
  const char* k0 = static_cast<const char*>(a.kv.k) + 16 * (tid % C::CHUNKS);
  const long long kv_gap = static_cast<const char*>(a.kv.v) - static_cast<const char*>(a.kv.k);
  auto issue = [&](int x) {
    const uint32_t dst = dst0 + (x % C::STAGES) * C::STAGE;
#pragma unroll
    for (int i = 0; i < kMmKeys / PASS; ++i) {
      const long long off = s_koff[x % kRing][r0 + i * PASS];
      const bool on = off >= 0;
      const char* src = k0 + (on ? off : 0);
      cp16(dst + i * PASS * HD * 2, src, on);
      cp16(dst + i * PASS * HD * 2 + C::HALF, src + kv_gap, on);
    }
  };

  Lookup pend = {-1, 0, 0};
  {
    Lookup l[C::STAGES];
#pragma unroll
    for (int x = 0; x < C::STAGES; ++x) {
      if (x < count) l[x] = lookup();
      if (x + 1 < count) line.next(look);
    }
#pragma unroll
    for (int x = 0; x < C::STAGES; ++x)
      if (x < count) publish(x, l[x]);
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < C::STAGES - 1; ++x) {
    if (x < count) issue(x);
    cp_commit();
  }

  Wide<T, HD> w;
  bool split_keys = false;  // the warps share the tile's keys, not the rows
  auto start = [&]() {
    split_keys = cur.nrows <= 16;
    w.start(a, table, cur, split_keys ? 0 : warp * 16, lane);
  };
  if (count) start();
  bool began = cur.tile == 0;  // the item's first unit is this CTA's
  for (int i = 0; i < count; ++i) {
    cp_wait<C::STAGES - 2>();
    __syncthreads();
    if (i + C::STAGES - 1 < count) issue(i + C::STAGES - 1);
    cp_commit();
    const bool more = i + C::STAGES < count;
    if (more) pend = lookup();
    const bool ends = cur.tile == cur.tiles - 1, run_ends = ends || i + 1 == count;

    const uint32_t ks = s0 + (i % C::STAGES) * C::STAGE, vs = ks + C::HALF;
    const uint64_t mask = (uint64_t)s_mask[i % kRing][1] << 32 | s_mask[i % kRing][0];
    const int key0 = cur.tile * kMmKeys;
    if (mask) {
      const bool whole = mask == ~0ull && key0 + kMmKeys <= cur.first;
      bool odd = false;
      if (cur.first < cur.limit && key0 + kMmKeys > cur.first) {
        // keys that the first row may not see and the last one does: is any of their V infinite or NaN?
        constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
        const int lo = max(cur.first - key0, 0);
        bool found = false;
        for (int x = tid + lo * C::CHUNKS; x < kMmKeys * C::CHUNKS; x += kThreads) {
          const uint4 v = *reinterpret_cast<const uint4*>(smem + (vs - s0) + sw<HD>(x / C::CHUNKS, x % C::CHUNKS));
          const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) found |= (vv[e] & E) == E || (vv[e] >> 16 & E) == E;
        }
        odd = __syncthreads_or(found);
      }
      if (split_keys)
        w.template tile<2>(ks, vs, warp * 16, key0, mask, whole, odd, a.scale2, lane);
      else if (warp * 16 < cur.nrows)
        w.template tile<8>(ks, vs, 0, key0, mask, whole, odd, a.scale2, lane);
    }
    if (more) {
      publish(i + C::STAGES, pend);
      if (i + C::STAGES + 1 < count) line.next(look);
    }

    if (!run_ends) {
      ++cur.tile;
      continue;
    }
    // the run of this item ends here: its part
    w.end();
    const Dest d = dest<TR>(a, cur, began, ends, 0, a.mm_o, a.mm_ml, HD);
    if (!split_keys) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = warp * 16 + (lane >> 2) + 8 * e;
        if (r < cur.nrows) {
          const long long row = d.row(r);
          float* op = d.o + row * HD + 2 * (lane & 3);
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(op + 8 * n) = make_float2(w.o[n][2 * e], w.o[n][2 * e + 1]);
          if ((lane & 3) == 0) d.ml[row] = make_float2(lifted<T, 0>(w.m[e]), w.l[e]);
        }
      }
    } else {
      // merge the warps' keys in the tile buffer just read ([4][MERGE][HD] fp32 is its size)
      float* so = reinterpret_cast<float*>(smem + (ks - s0)) + warp * MERGE * HD;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = (lane >> 2) + 8 * e;
        if (r < cur.nrows) {
#pragma unroll
          for (int n = 0; n < HD / 8; ++n)
            *reinterpret_cast<float2*>(so + r * HD + merge_col(r, 8 * n + 2 * (lane & 3))) = make_float2(w.o[n][2 * e], w.o[n][2 * e + 1]);
          if ((lane & 3) == 0) s_m[warp][r] = w.m[e], s_l[warp][r] = w.l[e];
        }
      }
      __syncthreads();
      so = reinterpret_cast<float*>(smem + (ks - s0));
      for (int x = tid; x < cur.nrows * HD; x += kThreads) {
        const int r = x / HD, e = x - r * HD;
        const float mm = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float o = 0.0f, l = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float f = ex2(s_m[k][r] - ref);
          o = fmaf(f, so[(k * MERGE + r) * HD + merge_col(r, e)], o);
          l = fmaf(f, s_l[k][r], l);
        }
        const long long row = d.row(r);
        d.o[row * HD + e] = o;
        if (e == 0) d.ml[row] = make_float2(lifted<T, 0>(mm), l);
      }
    }
    if (i + 1 < count) {
      line.next_item(cur);
      began = true;
      start();
    }
  }

  join_records<TR, kThreads>(a, table, bad, units, s_scan);
}

// ---- narrow form -------------------------------------------------------------------------------------

template <typename T, int HD, int TR>
struct Narrow {
  static constexpr int NR = TR / 8;  // n-tiles of 8 query rows
  uint32_t q[HD / 16][NR][2];
  float o[HD / 16][NR][4];
  float m[NR][2], l[NR][2];  // rows 8 n + 2 (lane % 4) + e
  int lim[NR][2];

  // Asks for the rows of the item to come while the last tile of this one runs: a lane a line of 128 bytes. (Held in registers
  // instead, they would cost more occupancy than the rest of the loads' latency does.)
  static __device__ __forceinline__ void ask(const PrefixArgs& a, const Cursor& c, int lane) {
    constexpr int LINES = HD / 64;
    const int r = lane / LINES;
    if (r < min(TR, c.nrows))
      asm volatile("prefetch.global.L1 [%0];" ::"l"(q_row<T>(a, c, TR, r) + lane % LINES * 64));
  }
  __device__ __forceinline__ void start(const PrefixArgs& a, const BatchTable& s, const Cursor& c, int lane) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = 8 * n + (lane >> 2);
      const bool on = r < c.nrows;
      const T* qp = q_row<T>(a, c, TR, r) + 2 * (lane & 3);
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        q[k][n][0] = on ? __ldg(reinterpret_cast<const uint32_t*>(qp + 16 * k)) : 0u;
        q[k][n][1] = on ? __ldg(reinterpret_cast<const uint32_t*>(qp + 16 * k + 8)) : 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][n][e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        lim[n][e] = row_limit(a, s, c, 8 * n + 2 * (lane & 3) + e, TR);
        m[n][e] = -INFINITY;
        l[n][e] = 0.0f;
      }
    }
  }

  // The 16 keys from key `k0` of the tile. `mask`: the tile's keys that exist; `whole`: all do, for every row.
  // `odd`: some V that not every row may see is infinite or NaN, so that 0 * v is not 0.
  __device__ __forceinline__ void tile(uint32_t ks, uint32_t vs, int k0, int key0, uint64_t mask, bool whole, bool odd,
                                       float scale2, int lane) {
    float s[NR][4], s2[NR][4];  // key k0 + lane / 4 + 8 (e / 2), row 8 n + 2 (lane % 4) + e % 2; two chains of sums
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.0f;
    const int mat = lane >> 3, mr = lane & 7;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
      uint32_t f[4];
      ldsm4(f, ks + sw_tma(k0 + (mat & 1) * 8 + mr, 2 * k + (mat >> 1)));
#pragma unroll
      for (int n = 0; n < NR; ++n) mma<T>(k & 1 ? s2[n] : s[n], f, q[k][n][0], q[k][n][1]);
    }
    bool moved = false;
    float f[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = (s[n][e] + s2[n][e]) * scale2;
        if (!whole) {
          const int c = k0 + (lane >> 2) + 8 * (e >> 1);
          if (!((mask >> c) & 1) || key0 + c >= lim[n][e & 1]) s[n][e] = -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(m[n][e], fmaxf(s[n][e], s[n][2 + e]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float ref = mx == -INFINITY ? 0.0f : mx;  // nothing seen yet: every weight below is exp2(-inf)
        f[n][e] = ex2(m[n][e] - ref);
        moved |= f[n][e] != 1.0f;
        m[n][e] = mx;
        const float against = lifted<T, 0>(ref);
        s[n][e] = ex2(s[n][e] - against);
        s[n][2 + e] = ex2(s[n][2 + e] - against);
        l[n][e] = fmaf(l[n][e], f[n][e], s[n][e] + s[n][2 + e]);
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[k][n][e] *= f[n][e & 1];
    }
    if (!odd) {
      uint32_t p[NR][2];
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        p[n][0] = movm(Half16<T>::pack(s[n][0], s[n][1]));
        p[n][1] = movm(Half16<T>::pack(s[n][2], s[n][3]));
      }
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        uint32_t v[4];
        ldsm4t(v, vs + sw_tma(k0 + (mat >> 1) * 8 + mr, 2 * k + (mat & 1)));
#pragma unroll
        for (int n = 0; n < NR; ++n) mma<T>(o[k][n], v, p[n][0], p[n][1]);
      }
    } else {
#pragma unroll 1
      for (int c16 = 0; c16 < 16; ++c16) {
        const int src = (c16 & 7) * 4 + (lane & 3), c = k0 + c16;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float p0 = __shfl_sync(0xffffffffu, c16 & 8 ? s[n][2] : s[n][0], src);
          const float p1 = __shfl_sync(0xffffffffu, c16 & 8 ? s[n][3] : s[n][1], src);
          const bool there = (mask >> c) & 1;
          const bool see0 = there && key0 + c < lim[n][0], see1 = there && key0 + c < lim[n][1];
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              unsigned short w;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(vs + sw_tma(c, 2 * k + h) + 2 * (lane >> 2)));
              const float v = Half16<T>::unpack(w).x;
              if (see0) o[k][n][2 * h] = fmaf(p0, v, o[k][n][2 * h]);
              if (see1) o[k][n][2 * h + 1] = fmaf(p1, v, o[k][n][2 * h + 1]);
            }
        }
      }
    }
  }

  __device__ __forceinline__ void end() {
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
  }
};


constexpr int kNarrowThreads = 160;  // four warps for the keys and the producer

template <typename T, int HD, int TR>
__global__ void __launch_bounds__(kNarrowThreads, Cfg<HD>::CTAS)
    prefix_narrow_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, PrefixArgs a) {
  using C = Cfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t s0 = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (s0 - smem_u32(smem_raw));
  __shared__ uint64_t full[C::STAGES], empty[C::STAGES];
  __shared__ unsigned long long s_mask[C::STAGES];
  __shared__ int s_scan[kNarrowThreads / 32], s_fail, s_issued;
  __shared__ float s_m[4][TR], s_l[4][TR];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    s_fail = s_issued = 0;
    fence_mbar_init();
    tma_prefetch_map(&tk);
    tma_prefetch_map(&tv);
  }
  BatchTable table;
  table.cum = reinterpret_cast<int*>(smem + C::STAGES * C::STAGE);
  table.q0 = table.cum + a.b.batch + 1;
  table.len = table.q0 + a.b.batch + 1;
  // Behind the tensor-core kernel the inputs are there already (it lets this kernel start only behind its own wait), and
  // its results matter to the join alone, which must find both kernels complete: so the wait comes last.
  griddep_launch_dependents();
  if (!a.tc_ctas) griddep_wait();
  const bool bad = batch_table<kNarrowThreads>(a, table);
  const int units = a.mm.prefix_units + line_table<kNarrowThreads, TR, kMmKeys>(a, a.mm, table, bad, s_scan);
  const Line<TR, kMmKeys> line{a, a.mm, table};
  const int ctas = min((int)gridDim.x, units);  // fewer units than CTAs: one each, so that no run is empty
  int u0 = 0, count = 0;
  if ((int)blockIdx.x < ctas) {
    u0 = cta_first(blockIdx.x, units, ctas);
    count = cta_first(blockIdx.x + 1, units, ctas) - u0;
  }
  volatile int* fail = &s_fail;

  if (warp == 4 && count) {
    // producer: lane l brings box l of each tile; its page is looked up one tile ahead
    const int box = page_box(a.kv.page_size, kMmKeys), boxes = kMmKeys / box;
    Cursor c = line.at(u0);
    auto page_of = [&]() {
      int page = -1;
      const int key = c.tile * kMmKeys + lane * box;
      if (lane < boxes && key < c.limit)
        page = __ldg((c.b < 0 ? a.prefix_pages : a.b.page_table + c.b * a.b.table_stride) + key / a.kv.page_size);
      return page;
    };
    int page = page_of();
    for (int i = 0; i < count; ++i) {
      const int s = i % C::STAGES, key = c.tile * kMmKeys + lane * box, left = c.limit - key, h = c.h;
      const bool there = page >= 0 && page < a.kv.n_pages;  // lanes without a box or with no key left: not
      unsigned long long mask = 0;
      if (there) mask = (left >= 64 ? ~0ull : (1ull << left) - 1) & (box == 64 ? ~0ull : (1ull << box) - 1);
      mask <<= (lane * box) & 63;
      unsigned lo = __reduce_or_sync(0xffffffffu, (unsigned)mask), hi = __reduce_or_sync(0xffffffffu, (unsigned)(mask >> 32));
      bool ok = true;
      if (lane == 0) {
        ok = i < C::STAGES || wait_for(a, &empty[s], (i / C::STAGES - 1) & 1);
        // A warp that gave up no longer waits for full, so its arrivals do not mean that the slot's copies have landed: nothing
        // more is brought then (a second arrival on a phase whose copies are in flight would be undefined).
        if (ok && !*fail) {
          s_mask[s] = (unsigned long long)hi << 32 | lo;
          mbar_arrive_expect_tx(&full[s], C::STAGE);
          s_issued = i + 1;
        } else {
          ok = false;
          *fail = 1;
        }
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      if (lane < boxes) {  // a page out of the pool reads as zeros
        const uint32_t dst = s0 + s * C::STAGE + lane * box * 128;
        const int slot = key % a.kv.page_size, from = there ? page : a.kv.n_pages;
#pragma unroll
        for (int x = 0; x < HD / 64; ++x) {
          tma_load_4d(dst + x * kMmKeys * 128, &tk, 64 * x, slot, h, from, &full[s]);
          tma_load_4d(dst + C::HALF + x * kMmKeys * 128, &tv, 64 * x, slot, h, from, &full[s]);
        }
      }
      if (i + 1 < count) {
        line.next(c);
        page = page_of();
      }
    }
  } else if (warp < 4 && count) {
    Cursor cur = line.at(u0);
    Narrow<T, HD, TR> w;
    w.start(a, table, cur, lane);
    bool began = cur.tile == 0;  // the item's first unit is this CTA's
    for (int i = 0; i < count; ++i) {
      const bool ends = cur.tile == cur.tiles - 1, run_ends = ends || i + 1 == count;
      Cursor next = cur;
      if (ends && i + 1 < count) {
        line.next_item(next);
        w.ask(a, next, lane);
      }
      const int s = i % C::STAGES, key0 = cur.tile * kMmKeys;
      // After a wait that gave up, the run goes on without waiting (the warps meet at barriers), to no use.
      if (!*fail && !wait_for(a, &full[s], (i / C::STAGES) & 1)) *fail = 1;
      __syncwarp();
      const uint32_t ks = s0 + s * C::STAGE, vs = ks + C::HALF;
      const unsigned long long mask = s_mask[s];
      const int k0 = warp * 16;
      bool wrote = false;
      if ((mask >> k0) & 0xffff) {
        bool odd = false;
        if (key0 + k0 + 16 > cur.first) {
          // Keys that the first row does not see: V of those that no row sees becomes zero (a page's rest holds anything);
          // is any of the others' infinite or NaN?
          constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
          bool found = false;
          for (int x = lane; x < 16 * C::CHUNKS; x += 32) {
            const int key = k0 + x / C::CHUNKS;
            uint4* v = reinterpret_cast<uint4*>(smem + (vs - s0) + sw_tma(key, x % C::CHUNKS));
            if (key0 + key >= cur.limit) {
              st_zero16(smem_u32(v));
            } else if (key0 + key >= cur.first) {
              const uint4 old = *v;
              const uint32_t vv[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) found |= (vv[e] & E) == E || (vv[e] >> 16 & E) == E;
            }
          }
          odd = __any_sync(0xffffffffu, found);
          wrote = true;
          __syncwarp();  // the zeros of other lanes: a vote does not order memory
        }
        const bool whole = mask == ~0ull && key0 + kMmKeys <= cur.first;
        w.tile(ks, vs, k0, key0, mask, whole, odd, a.scale2, lane);
      }
      if (!run_ends) {
        if (wrote) fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        ++cur.tile;
        continue;
      }
      // The run of this item ends here: merge the warps' keys in the tile buffer just read ([4][TR][HD] fp32 is at most
      // its size), and write the part.
      w.end();
      const Dest d = dest<TR>(a, cur, began, ends, 0, a.mm_o, a.mm_ml, HD);
      float* so = reinterpret_cast<float*>(smem + (ks - s0));
      named_bar_sync(1, 128);
#pragma unroll
      for (int n = 0; n < TR / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * n + 2 * (lane & 3) + e;
          if (r < cur.nrows) {
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
              for (int x = 0; x < 2; ++x) so[(warp * TR + r) * HD + merge_col(r, 16 * k + 8 * x + (lane >> 2))] = w.o[k][n][2 * x + e];
            if (lane < 4) s_m[warp][r] = w.m[n][e], s_l[warp][r] = w.l[n][e];
          }
        }
      named_bar_sync(1, 128);
      // HD / 4 lanes a row, four elements each
      constexpr int LANES = HD / 4;
#pragma unroll 2
      for (int r = threadIdx.x / LANES; r < cur.nrows; r += 128 / LANES) {
        const int e = threadIdx.x % LANES * 4;
        const float mm = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float f = ex2(s_m[k][r] - ref);
          const float4 v = *reinterpret_cast<const float4*>(so + (k * TR + r) * HD + merge_col(r, e));
          o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
          l = fmaf(f, s_l[k][r], l);
        }
        const long long row = d.row(r);
        *reinterpret_cast<float4*>(d.o + row * HD + e) = o;
        // a row whose work gave up is NaN
        if (e == 0) d.ml[row] = make_float2(lifted<T, 0>(mm), *fail ? __int_as_float(0x7fffffff) : l);
      }
      if (i + 1 < count) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        cur = next;
        began = true;
        w.start(a, table, cur, lane);
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && *fail) {
    atomicOr(&g_narrow_status, kStatusTimeout);
    for (int i = max(s_issued - C::STAGES, 0); i < s_issued; ++i)  // leave no copy in flight
      mbar_wait_bounded(&full[i % C::STAGES], (i / C::STAGES) & 1, kWaitLimitNs);
  }
  join_records<TR, kNarrowThreads>(a, table, bad, units, s_scan);
}

// Joins a row's parts, half a warp per (row, head): every part is (max, sum, weighted V); the prefix's and the own
// keys' come from whichever CTAs' runs the row's items lie in, 16 parts a round with all their loads side by
// side. Bound by latency (record, (max, sum), V: three dependent loads) until the parts outgrow L2: 6144 rows 10.8 us,
// 33,888 rows of three parts on average 17 us (3 TB/s).
constexpr int kJoinThreads = 128;

template <typename T, int HD>
__global__ void __launch_bounds__(kJoinThreads) prefix_join_kernel(PrefixArgs a) {
  constexpr int E = HD / 16;
  const int lane = threadIdx.x & 15;
  const unsigned half = 0xffffu << (threadIdx.x & 16);
  const int row = (blockIdx.x * kJoinThreads + threadIdx.x) / 16, n_rows = a.rows * a.H;  // at most 10^8
  griddep_launch_dependents();
  griddep_wait();
  if (row >= n_rows) return;
  const int t = row / a.H, head = row - t * a.H, h = head / a.g;
  const int4 rec = __ldcg(a.rec + t);
  const int mm_units = __ldcg(a.totals), tc_own_units = a.tc_ctas ? __ldcg(a.totals + 1) : 0;
  if (rec.w < 0) return;  // a row of no sequence

  // an item's parts: the first one's CTA, their number, the first place of cut items, this row's place in the row tile
  struct Item {
    int c0, n, cut0, r, tr;
    const float2* ml;
    const float* o;
  };
  auto find = [&](bool tc, bool pre, int first, int row_tiles, int tiles, int j) {
    Item it;
    it.cut0 = tc && !pre ? a.tc_ctas : 0;
    const int shift = tc ? 8 : a.mm_rows == 8 ? 3 : a.mm_rows == 16 ? 4 : 6;
    static_assert(kTcRows == 1 << 8, "the shift above");
    it.tr = 1 << shift;
    it.ml = tc ? a.tc_ml : a.mm_ml;
    it.o = tc ? a.tc_o : a.mm_o;
    const int units = !tc ? mm_units : pre ? a.tc.prefix_units : tc_own_units, ctas = min(tc ? a.tc_ctas : a.mm_ctas, units);
    const int rr = j * a.g + head - h * a.g, rt = rr >> shift;
    it.r = rr - (rt << shift);
    it.c0 = 0;
    it.n = tiles > 0;
    if (tiles > (tc && !pre ? kTcWholeTiles : 0)) {
      const int u = first + (h * row_tiles + rt) * tiles;
      it.c0 = cta_of(u, units, ctas);
      it.n = cta_of(u + tiles - 1, units, ctas) - it.c0 + 1;
    }
    return it;
  };
  const bool p_tc = a.tc.prefix_units > 0;
  const int tr = p_tc ? kTcRows : a.mm_rows, tk = p_tc ? kTcKeys : kMmKeys;
  const Item pre = find(p_tc, true, 0, (a.rows * a.g + tr - 1) / tr, (a.b.prefix_len + tk - 1) / tk, t);
  const Item own = find(rec.y < 0, false, rec.x, rec.z, abs(rec.y), rec.w);

  const int parts = pre.n + own.n;
  float acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  for (int k0 = 0; k0 < parts; k0 += 16) {
    float2 x = make_float2(-INFINITY, 0.0f);
    const float* o = a.row_o;
    if (k0 + lane < parts) {
      const bool first = k0 + lane < pre.n;
      const Item& it = first ? pre : own;
      const int k = k0 + lane - (first ? 0 : pre.n);
      const long long at = it.n == 1 ? row + (first ? 0ll : (long long)n_rows)
                                     : (2ll * (it.cut0 + it.c0 + k) + (k == 0)) * it.tr + it.r;
      x = __ldcg((it.n == 1 ? a.row_ml : it.ml) + at);
      o = (it.n == 1 ? a.row_o : it.o) + at * HD;
    }
    float mm = fmaxf(m, x.x);
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) mm = fmaxf(mm, __shfl_xor_sync(half, mm, s));
    const float ref = mm == -INFINITY ? 0.0f : mm;
    const float f = ex2(m - ref), weight = ex2(x.x - ref);  // a part without keys: 0
    float sum = x.y * weight;
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor_sync(half, sum, s);
    l = l * f + sum;
    m = mm;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= f;
    const int n = min(16, parts - k0);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(half, weight, i, 16);
      const float* src = reinterpret_cast<const float*>(
          __shfl_sync(half, (unsigned long long)reinterpret_cast<uintptr_t>(o), i, 16));
      if constexpr (E >= 4) {
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src) + lane + 16 * q);
          acc[4 * q] = fmaf(v.x, w, acc[4 * q]);
          acc[4 * q + 1] = fmaf(v.y, w, acc[4 * q + 1]);
          acc[4 * q + 2] = fmaf(v.z, w, acc[4 * q + 2]);
          acc[4 * q + 3] = fmaf(v.w, w, acc[4 * q + 3]);
        }
      } else {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(src) + lane);
        acc[0] = fmaf(v.x, w, acc[0]);
        acc[1] = fmaf(v.y, w, acc[1]);
      }
    }
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // no keys: zero
  T* out = static_cast<T*>(a.out) + (long long)row * HD;
  if constexpr (E >= 4) {
#pragma unroll
    for (int q = 0; q < E / 4; ++q)
      *reinterpret_cast<uint2*>(out + 4 * (lane + 16 * q)) =
          make_uint2(Half16<T>::pack(acc[4 * q] * inv, acc[4 * q + 1] * inv), Half16<T>::pack(acc[4 * q + 2] * inv, acc[4 * q + 3] * inv));
  } else {
    *reinterpret_cast<uint32_t*>(out + 2 * lane) = Half16<T>::pack(acc[0] * inv, acc[1] * inv);
  }
}

// ---- host --------------------------------------------------------------------------------------------

int mm_ctas_per_sm(int hd) { return hd == 128 ? Cfg<128>::CTAS : hd == 64 ? Cfg<64>::CTAS : Cfg<32>::CTAS; }

// Which kernel takes what; decided by what the host knows, so that a captured graph keeps its launches.
struct Plan {
  AttnLine tc, mm;
  int tc_ctas, mm_ctas, mm_rows;
};

int prefix_units(int rows, int g, int Hkv, int prefix_len, int tr, int tk) {
  return Hkv * ((rows * g + tr - 1) / tr) * ((prefix_len + tk - 1) / tk);
}

Plan plan(int rows, int H, const q4b_batch& b, const q4b_paged_kv& kv, bool tensor_cores) {
  constexpr int kAll = 0x7fffffff;
  const int Hkv = kv.n_kv_heads, g = H / Hkv, R = rows * g;
  Plan p = {};
  const bool tc = prefix_tc_takes(kv) && tensor_cores;
  const bool tc_prefix = tc && prefix_units(rows, g, Hkv, b.prefix_len, 16, kMmKeys) > kTcMinUnits;
  // several rows a sequence, as told or on average: those with many are worth the tensor cores
  const bool several = b.max_new ? b.max_new > 1 : rows > b.batch;
  const int most_rows = several ? (b.max_new ? std::min(b.max_new, rows) : rows) * g : g;  // of a sequence, times heads
  const bool tc_own = tc && several && most_rows > kTcMinRows && b.batch <= kTcMaxBatch;
  if (tc_prefix || tc_own) p.tc_ctas = kTcCtas;
  if (tc_prefix) p.tc.prefix_units = prefix_units(rows, g, Hkv, b.prefix_len, kTcRows, kTcKeys);
  p.tc.own_lo = tc_own ? kTcMinRows : kAll;
  p.tc.own_hi = kAll;
  p.mm.own_hi = tc_own ? kTcMinRows : kAll;
  // Row tiles: 8 for single tokens, 16 for a few rows; more rows are more tiles, whose keys come from L2 again.
  const bool prefix_here = !tc_prefix && b.prefix_len > 0;
  const int most = std::max(most_rows, prefix_here ? R : 0);
  p.mm_rows = !prefix_tc_takes(kv) ? 64 : most <= 8 ? 8 : 16;
  if (prefix_here) p.mm.prefix_units = prefix_units(rows, g, Hkv, b.prefix_len, p.mm_rows, kMmKeys);
  int mm_sms = kSms;
  // Small steps, where either kernel's start and end (some 10 us of launch, first reads and last parts) weigh as much as
  // its tiles: both at once, on disjoint SMs, instead of one behind the other. 61 sequences of 5 drafts behind 4099 keys: 45
  // us against 52; 192 single tokens behind 16384 keys, where a wrong guess at the own keys costs more than the start: 207 at
  // best against 210. Where the caller does not tell them, own keys are anything from none to full tables, and what counts is the
  // mean over four lengths between.
  const int per_sequence = (R + std::max(b.batch, 1) - 1) / std::max(b.batch, 1);
  const int items = Hkv * ((R + kTcRows - 1) / kTcRows);
  if (tc_prefix && per_sequence <= kTcMinRows && p.mm_rows < 64) {
    const int tiles = (b.prefix_len + kTcKeys - 1) / kTcKeys;
    const double tile_us = kv.head_dim == 128 ? 2.0 : 1.6;
    // row tiles of a sequence (ragged: a little above the mean), an item's start and end as 1.3 tiles
    const double row_tiles = !several ? (per_sequence + p.mm_rows - 1) / p.mm_rows
                                             : std::max(1.0, (double)R / std::max(b.batch, 1) / p.mm_rows + 0.2);
    const double full = (double)b.table_width * kv.page_size, known = std::min<double>(b.own_keys, full);
    auto mm_time = [&](double own) {
      return b.batch * (double)Hkv * row_tiles * (own / kMmKeys + 1.3) * 1.3 / (mm_ctas_per_sm(kv.head_dim) * kSms);
    };
    const double mm_us = mm_time(b.own_keys ? known : 0.5 * full);
    const double tc_us = (double)items * tiles * tile_us / kSms;
    if (tc_us + mm_us < 40) {
      // SMs for the prefix: a multiple of its items, so that no CTA has parts of two (that costs some 3 us), or the share of
      // the tiles' time. More CTAs an item are more parts for the join, 0.5 us each. Measured against the share alone: 24
      // sequences of 6 behind 3000 keys 35 us and 49, 32 single tokens behind 2048 25 and 28.5, 64 behind 1500 42.5 and 40.
      auto cost = [&](int ctas, double each, double parts) {
        double us = 0.0;
        for (double f : {0.125, 0.375, 0.625, 0.875})
          us += 0.25 * std::max(2.0 + each * tile_us, mm_time(b.own_keys ? known : f * full) * kSms / (kSms - ctas));
        return us + 0.5 * parts;
      };
      int best = 0;
      double least = 1e30;
      auto take = [&](int ctas, double us) {
        if (us < least) least = us, best = ctas;
      };
      for (int c = kSms / 6; c <= kSms * 3 / 4; c += 4) take(c, cost(c, items * (double)tiles / c + 3.0 / tile_us, 1.0 + c / (double)items));
      for (int m = 1; m <= tiles && m * items <= kSms * 3 / 4; ++m) take(m * items, cost(m * items, (tiles + m - 1) / m, m));
      p.tc_ctas = best;
      mm_sms = kSms - best;
    }
  }
  // A larger step of the prefix alone: the same multiple of the items, where it leaves no more than a 20th of the SMs idle.
  // 192 single tokens (24 items) behind 16384 keys, 144 CTAs against 148: 202.5 us against 205.5, short own keys 93 and 98.
  if (tc_prefix && !tc_own && p.tc_ctas == kSms && items <= kSms && kSms % items * 20 <= kSms) p.tc_ctas = kSms - kSms % items;
  p.mm_ctas = mm_ctas_per_sm(kv.head_dim) * mm_sms;
  return p;
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

struct Layout {
  size_t rec, totals, row_ml, row_o, mm_ml, mm_o, tc_ml, tc_o, total;
};
Layout layout(const Plan& p, int rows, int H, int hd) {
  Layout w;
  const size_t n = 2 * (size_t)rows * H, mm = 2 * (size_t)p.mm_ctas * p.mm_rows, tc = 4 * (size_t)p.tc_ctas * kTcRows;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += up256(bytes);
    return here;
  };
  w.rec = take(rows * sizeof(int4));
  w.totals = take(2 * sizeof(int));
  w.row_ml = take(n * sizeof(float2));
  w.row_o = take(n * hd * sizeof(float));
  w.mm_ml = take(mm * sizeof(float2));
  w.mm_o = take(mm * hd * sizeof(float));
  w.tc_ml = take(tc * sizeof(float2));
  w.tc_o = take(tc * hd * sizeof(float));
  w.total = at;
  return w;
}

size_t table_bytes(int batch) { return 12 * ((size_t)batch + 1); }

template <typename T, int HD>
cudaError_t launch_wide(const PrefixArgs& a, cudaStream_t st) {
  using C = Cfg<HD>;
  auto kern = prefix_wide_kernel<T, HD>;
  static std::atomic<unsigned long long> done;
  const cudaError_t e = set_max_dynamic_smem(kern, C::STAGES * C::STAGE + (int)table_bytes(kMaxBatch), done);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(a.mm_ctas), dim3(kThreads), C::STAGES * C::STAGE + table_bytes(a.b.batch), st, a);
}

template <typename T, int HD, int TR>
cudaError_t launch_narrow(const PrefixArgs& a, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  using C = Cfg<HD>;
  auto kern = prefix_narrow_kernel<T, HD, TR>;
  static std::atomic<unsigned long long> done;
  const cudaError_t e = set_max_dynamic_smem(kern, C::STAGES * C::STAGE + 1024 + (int)table_bytes(kMaxBatch), done);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(a.mm_ctas), dim3(kNarrowThreads), C::STAGES * C::STAGE + 1024 + table_bytes(a.b.batch), st, tk, tv, a);
}

template <typename T, int HD>
int launch(const PrefixArgs& a, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (a.mm_rows == 64) {
    e = launch_wide<T, HD>(a, st);
  } else if constexpr (HD >= 64) {
    CUtensorMap tk, tv;
    const int box = page_box(a.kv.page_size, kMmKeys);
    if (int rc = make_tmap_pages(&tk, a.kv, a.kv.k, box)) return rc;
    if (int rc = make_tmap_pages(&tv, a.kv, a.kv.v, box)) return rc;
    e = a.mm_rows == 8 ? launch_narrow<T, HD, 8>(a, tk, tv, st) : launch_narrow<T, HD, 16>(a, tk, tv, st);
  }
  if (e == cudaSuccess)
    e = launch_pdl(prefix_join_kernel<T, HD>, dim3((unsigned)(((long long)a.rows * a.H * 16 + kJoinThreads - 1) / kJoinThreads)),
                   dim3(kJoinThreads), 0, st, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(Q4B_ELAUNCH, "prefix_attention: launch failed: %s", cudaGetErrorString(e));
  }
  return Q4B_OK;
}

int check(const char* what, int rows, int n_heads, const q4b_batch* b, const q4b_paged_kv* kv) {
  if (int rc = check_batch(what, b, rows)) return rc;
  if (int rc = check_paged_kv(what, kv)) return rc;
  if (kv->head_dim != 32 && kv->head_dim != 64 && kv->head_dim != 128)
    return set_error(Q4B_EUNSUPPORTED, "%s: head_dim %d is not 32, 64 or 128", what, kv->head_dim);
  if (n_heads < 1 || n_heads % kv->n_kv_heads)
    return set_error(Q4B_EINVAL, "%s: need n_heads %% n_kv_heads == 0", what);
  if (b->batch > kMaxBatch) return set_error(Q4B_EUNSUPPORTED, "%s: more than %d sequences", what, kMaxBatch);
  // key tiles of all items, at most (row tiles of 8): they are counted in 32 bits
  const double g = n_heads / kv->n_kv_heads, tiles = (double)b->table_width * kv->page_size / kMmKeys + 1;
  if (((rows * g / 8 + b->batch) * tiles + (rows * g / 8 + 1) * (b->prefix_len / kMmKeys + 1.0)) * kv->n_kv_heads > 2e9 ||
      rows * (double)n_heads > 1e8)
    return set_error(Q4B_EUNSUPPORTED, "%s: the step is too large; split its rows", what);
  return Q4B_OK;
}

}  // namespace

unsigned narrow_status(bool reset) {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, g_narrow_status, sizeof(v));
  if (reset && v) {
    const unsigned zero = 0;
    cudaMemcpyToSymbol(g_narrow_status, &zero, sizeof(zero));
  }
  return v;
}

}  // namespace q4b

using namespace q4b;

extern "C" size_t q4b_prefix_attention_workspace(int rows, int n_heads, const q4b_batch* batch, const q4b_paged_kv* kv) {
  if (check("prefix_attention", rows, n_heads, batch, kv)) return 0;
  // whether the tensor-core kernel turns out to be used or not: that depends on q's alignment, and on the build
  return std::max(layout(plan(rows, n_heads, *batch, *kv, true), rows, n_heads, kv->head_dim).total,
                  layout(plan(rows, n_heads, *batch, *kv, false), rows, n_heads, kv->head_dim).total);
}

extern "C" int q4b_prefix_attention(const void* q, long long q_stride, long long q_head_stride, int rows, int n_heads,
                                    float scale, const int32_t* prefix_pages, const q4b_batch* batch,
                                    const q4b_paged_kv* kv, void* out, void* workspace, size_t workspace_bytes,
                                    q4b_stream_t stream) {
  const char* what = "prefix_attention";
  if (int rc = check(what, rows, n_heads, batch, kv)) return rc;
  if (rows == 0 || batch->batch == 0) return Q4B_OK;
  if (!q || !out || (batch->prefix_len > 0 && !prefix_pages)) return set_error(Q4B_EINVAL, "%s: null pointer", what);
  if (q_stride % 2 || q_head_stride % 2 || !aligned(q, 4) || !aligned(out, 16))
    return set_error(Q4B_EINVAL, "%s: q must be 4-byte aligned with even strides, out 16-byte aligned", what);
  if (!(scale > 0.0f) || !(scale < INFINITY)) return set_error(Q4B_EINVAL, "%s: scale must be positive", what);
  // the tensor-core kernel reads q in 16-byte pieces
  const bool wide_q = aligned(q, 16) && q_stride % 8 == 0 && q_head_stride % 8 == 0;
  const Plan p = plan(rows, n_heads, *batch, *kv, wide_q && prefix_tc_takes(*kv) && prefix_tc_built(*kv));
  const Layout w = layout(p, rows, n_heads, kv->head_dim);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < w.total)
    return set_error(Q4B_EINVAL, "%s: needs a 256-byte aligned workspace of %zu bytes", what, w.total);
  PrefixArgs a;
  a.q = q, a.q_stride = q_stride, a.q_head_stride = q_head_stride;
  a.rows = rows, a.H = n_heads, a.Hkv = kv->n_kv_heads, a.g = n_heads / kv->n_kv_heads;
  a.scale2 = scale * 1.44269504088896340736f;
  a.b = *batch, a.kv = *kv, a.prefix_pages = prefix_pages, a.out = out;
  a.table_keys = (int)std::min((long long)batch->table_width * kv->page_size, 0x7fffffffll - kTcKeys);
  a.tc_ctas = p.tc_ctas, a.mm_ctas = p.mm_ctas, a.mm_rows = p.mm_rows, a.tc = p.tc, a.mm = p.mm;
  char* base = static_cast<char*>(workspace);
  a.rec = reinterpret_cast<int4*>(base + w.rec);
  a.totals = reinterpret_cast<int*>(base + w.totals);
  a.row_ml = reinterpret_cast<float2*>(base + w.row_ml);
  a.row_o = reinterpret_cast<float*>(base + w.row_o);
  a.mm_ml = reinterpret_cast<float2*>(base + w.mm_ml);
  a.mm_o = reinterpret_cast<float*>(base + w.mm_o);
  a.tc_ml = reinterpret_cast<float2*>(base + w.tc_ml);
  a.tc_o = reinterpret_cast<float*>(base + w.tc_o);
  a.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
  const cudaStream_t st = as_stream(stream);
  if (a.tc_ctas)
    if (int rc = prefix_tc_run(a, st)) return rc;
  const bool h16 = kv->dtype == Q4B_F16;
  switch (kv->head_dim) {
    case 128: return h16 ? launch<__half, 128>(a, st) : launch<__nv_bfloat16, 128>(a, st);
    case 64: return h16 ? launch<__half, 64>(a, st) : launch<__nv_bfloat16, 64>(a, st);
    default: return h16 ? launch<__half, 32>(a, st) : launch<__nv_bfloat16, 32>(a, st);
  }
}

extern "C" void q4b_prefix_attention_wait_limit(unsigned long long ns) {
  g_wait_ns.store(std::min(ns, 10 * (unsigned long long)kWaitLimitNs), std::memory_order_relaxed);
}
