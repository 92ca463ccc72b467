// Attention of a ragged batch over a paged cache whose sequences share a prefix (the GQA attention of
// scripts/llm/llama_q4.py:208-232, for a batch).
//
//   row (b, j), head h:  out = sum_s softmax_s(q . k_s * scale) v_s  over the prefix's keys and b's own keys
//   0 .. len_b - n_b + j;  zero if there are none.
//
// The prefix is read once for the whole batch: its queries are all rows of the step and all heads of a KV
// head's group, tiled by 64; a sequence's own keys are read once for its rows and heads. Both are items
// (KV head, row tile) of key tiles of 64 keys, and all items' key tiles stand in one line, of which each CTA takes an
// equal run (whole items, and at most one cut item at either end): whatever the lengths, every SM
// streams the same number of bytes. Each run of an item leaves (max, sum, weighted V) in fp32; a second kernel
// joins a row's parts. Bound by memory for few rows per KV head (a step of single tokens: 2 hd bytes read per
// 2 g hd flops).
//
// In a CTA (4 warps): the tiles come by 16-byte asynchronous copies into a ring of swizzled buffers, STAGES - 1 ahead,
// with the page lookups one tile ahead of the copies. QK and PV are m16n8k16 MMAs on the 16-bit values
// as stored, fp32 sums, an online softmax in base 2. Items of up to 16 rows (single tokens) split a tile's 64
// keys over the warps and merge at the end; larger ones give each warp 16 rows. P is rounded to the
// cache's type for the PV product: its error, half a step per weight, averages out over the keys and stays
// below the output's own rounding.
#include <algorithm>

#include "paged.cuh"
#include "prefix_attn.h"

namespace q4b {
namespace {

constexpr int kThreads = 128;
constexpr int kTileKeys = 64, kTileRows = 64;
constexpr int kRing = 8;  // page lookups in flight (tiles), >= STAGES + 2
constexpr int kSms = 148;
constexpr int kMaxBatch = 4096;

template <int HD>
struct Cfg {
  static constexpr int STAGES = HD == 128 ? 3 : 4;
  static constexpr int CTAS = HD == 128 ? 2 : 3;  // per SM
  static constexpr int HALF = kTileKeys * HD * 2; // K (or V) of one tile
  static constexpr int STAGE = 2 * HALF;
  static constexpr int CHUNKS = HD / 8;           // 16-byte chunks of a row
};

// 16-byte chunk c of tile row r, swizzled so that 8 consecutive rows' equal chunks lie in 8 bank groups
template <int HD>
__device__ __forceinline__ uint32_t sw(int r, int c) {
  if constexpr (HD == 32) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  return r * (HD * 2) + ((c ^ (r & 7)) << 4);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
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

// first unit of CTA c, and the CTA that holds unit u, for `units` units over `ctas` CTAs
__host__ __device__ __forceinline__ int cta_first(int c, int units, int ctas) { return (int)((long long)c * units / ctas); }
__host__ __device__ __forceinline__ int cta_of(int u, int units, int ctas) {
  return (int)((((long long)u + 1) * ctas - 1) / units);
}

// One item's place and the tile of it that a unit stands for.
struct Cursor {
  int b;      // sequence, -1: the prefix
  int h, rt;  // KV head, row tile
  int tile, tiles, row_tiles;
  int q0, n, len;  // rows and own keys of the sequence (prefix: 0, all rows, prefix_len)
  int nrows;       // rows of this row tile
  int limit;       // keys that its last row sees
  int first;       // keys that its first row sees
};

struct Shared {
  int* cum;   // [batch + 1] units in front of sequence b (behind the prefix's)
  int* q0;    // [batch + 1] clamped
  int* len;   // [batch] clamped
};

__device__ __forceinline__ void cursor_item(Cursor& c, int g) {
  c.nrows = min(kTileRows, c.n * g - c.rt * kTileRows);
  if (c.b < 0) {
    c.limit = c.first = c.len;
  } else {
    const int j0 = c.rt * kTileRows / g, j1 = (c.rt * kTileRows + c.nrows - 1) / g;
    c.first = min(max(c.len - c.n + j0 + 1, 0), c.len);
    c.limit = min(max(c.len - c.n + j1 + 1, 0), c.len);
  }
}
__device__ __forceinline__ void cursor_seq(Cursor& c, const PrefixArgs& a, const Shared& s) {
  c.q0 = s.q0[c.b];
  c.n = s.q0[c.b + 1] - c.q0;
  c.len = s.len[c.b];
  c.row_tiles = (c.n * a.g + kTileRows - 1) / kTileRows;
  c.tiles = (c.len + kTileKeys - 1) / kTileKeys;
}
__device__ Cursor cursor_at(int u, const PrefixArgs& a, const Shared& s) {
  Cursor c;
  if (u < a.prefix_units) {
    c.b = -1;
    c.q0 = 0;
    c.n = a.rows;
    c.len = a.b.prefix_len - a.prefix_skip;
    c.row_tiles = (a.rows * a.g + kTileRows - 1) / kTileRows;
    c.tiles = (c.len + kTileKeys - 1) / kTileKeys;
  } else {
    u -= a.prefix_units;
    int lo = 0, hi = a.b.batch - 1;  // the last b with cum[b] <= u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s.cum[mid] <= u)
        lo = mid;
      else
        hi = mid - 1;
    }
    c.b = lo;
    u -= s.cum[lo];
    cursor_seq(c, a, s);
  }
  c.tile = u % c.tiles;
  u /= c.tiles;
  c.rt = u % c.row_tiles;
  c.h = u / c.row_tiles;
  cursor_item(c, a.g);
  return c;
}
// the next unit; the caller knows that there is one
__device__ __forceinline__ void cursor_next(Cursor& c, const PrefixArgs& a, const Shared& s) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.rt == c.row_tiles) {
    c.rt = 0;
    if (++c.h == a.Hkv) {
      c.h = 0;
      do ++c.b;
      while (s.cum[c.b + 1] == s.cum[c.b]);
      cursor_seq(c, a, s);
    }
  }
  cursor_item(c, a.g);
}

template <typename T, int HD>
struct Warp {
  uint32_t q[HD / 16][4];
  float o[HD / 8][4];
  float m[2], l[2];
  int lim[2];  // keys that this lane's two rows see

  __device__ __forceinline__ void start(const PrefixArgs& a, const Cursor& c, int r0, int lane) {
    const int q4 = lane & 3;
    const T* qp[2];
    bool on[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = r0 + (lane >> 2) + 8 * i, rr = c.rt * kTileRows + r;
      on[i] = r < c.nrows;
      const int j = rr / a.g, hh = c.h * a.g + rr - j * a.g;
      qp[i] = static_cast<const T*>(a.q) + (long long)(c.q0 + j) * a.q_stride + (long long)hh * a.q_head_stride + 2 * q4;
      lim[i] = c.b < 0 ? c.len : min(c.len - c.n + j + 1, c.len);
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
      f[i] = exp2f(m[i] - ref);
      m[i] = mx[i];
      mx[i] = ref;
      l[i] *= f[i];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = exp2f(s[n][e] - mx[e >> 1]);
        l[e >> 1] += s[n][e];
      }
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] *= f[e >> 1];
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

  __device__ __forceinline__ void sum_quads() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
  }
};

// Where a run of an item puts its (max, sum) and weighted V for row r of its row tile: by the output row if the
// run is the whole item, else in one of the CTA's two places for cut items.
struct Dest {
  float* o;
  float2* ml;
  bool whole;
  const PrefixArgs* a;
  int q0, base, h;
  __device__ __forceinline__ long long row(int r) const {
    if (!whole) return r;
    const int rr = base + r, j = rr / a->g;
    return (long long)(q0 + j) * a->H + h * a->g + rr - j * a->g;
  }
};

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::CTAS) prefix_attn_kernel(PrefixArgs a) {
  using C = Cfg<HD>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_koff[kRing][kTileKeys];  // element offset of a tile's keys, -1: not there
  __shared__ unsigned s_mask[kRing][2];
  __shared__ int s_scan[4];
  __shared__ float s_m[4][16], s_l[4][16];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Shared sh;
  sh.cum = reinterpret_cast<int*>(smem + C::STAGES * C::STAGE);
  sh.q0 = sh.cum + a.b.batch + 1;
  sh.len = sh.q0 + a.b.batch + 1;
  // Behind the tensor-core kernel the inputs are there already (it lets this kernel start only behind its own wait), and
  // its results matter to the join alone, which must find both kernels complete: so the wait comes last.
  griddep_launch_dependents();
  if (!a.tc_splits) griddep_wait();

  // the batch: rows, own keys and units of each sequence; thread t scans a run of sequences
  {
    const int B = a.b.batch, per = (B + kThreads - 1) / kThreads, b0 = min(tid * per, B), b1 = min(b0 + per, B);
    const long long cap = min((long long)a.b.table_width * a.kv.page_size, 0x7fffffffll - kTileKeys);
    int mine = 0;
    bool bad = false;  // offsets that decrease: no sequence gets own keys, and the units stay countable
    for (int b = b0; b < b1; ++b) {
      bad |= __ldg(a.b.q_start + b + 1) < __ldg(a.b.q_start + b);
      const int2 r = batch_rows(a.b.q_start, b, a.rows);
      const int len = (int)min((long long)max(__ldg(a.b.seq_lens + b), 0), cap);
      sh.q0[b] = r.x;
      sh.len[b] = len;
      const int n = r.y - r.x;
      const int units = a.Hkv * ((n * a.g + kTileRows - 1) / kTileRows) * ((len + kTileKeys - 1) / kTileKeys);
      sh.cum[b] = mine;
      mine += units;
      if (b == B - 1) sh.q0[B] = r.y;
    }
    bad = __syncthreads_or(bad);
    if (bad) mine = 0;
    int run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += v;
    }
    if (lane == 31) s_scan[warp] = run;
    __syncthreads();
    int before = run - mine;
    for (int w = 0; w < warp; ++w) before += s_scan[w];
    for (int b = b0; b < b1; ++b) sh.cum[b] = bad ? 0 : sh.cum[b] + before;
    if (tid == kThreads - 1) sh.cum[B] = before + mine;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int b = tid; b <= B; b += kThreads) a.cum[b] = sh.cum[b];
  }
  const int units = a.prefix_units + sh.cum[a.b.batch];
  const int ctas = min((int)gridDim.x, units);  // fewer units than CTAs: one each, so that no run is empty
  if ((int)blockIdx.x >= ctas) {
    if (a.tc_splits) griddep_wait();
    return;
  }
  const int u0 = cta_first(blockIdx.x, units, ctas), u1 = cta_first(blockIdx.x + 1, units, ctas);
  const int count = u1 - u0;

  const uint32_t s0 = smem_u32(smem);
  Cursor look = cursor_at(u0, a, sh), cur = look;

  // page lookup of unit x (the `look` cursor stands there): threads 0..63 take a key each
  long long pend = -1;
  auto lookup = [&]() {
    if (tid < kTileKeys) {
      int key = look.tile * kTileKeys + tid;
      pend = -1;
      if (key < look.limit) {
        if (look.b < 0) key += a.prefix_skip;
        const int pi = key / a.kv.page_size;
        const int page = __ldg(look.b < 0 ? a.prefix_pages + pi : a.b.page_table + look.b * a.b.table_stride + pi);
        if (page >= 0 && page < a.kv.n_pages)
          pend = page * a.kv.page_stride + (key - pi * a.kv.page_size) * a.kv.slot_stride + look.h * a.kv.head_stride;
      }
    }
  };
  auto publish = [&](int x) {
    if (tid < kTileKeys) {
      s_koff[x % kRing][tid] = pend;
      const unsigned bits = __ballot_sync(0xffffffffu, pend >= 0);
      if (lane == 0) s_mask[x % kRing][warp] = bits;
    }
  };
  auto issue = [&](int x) {
    const uint32_t dst = s0 + (x % C::STAGES) * C::STAGE;
    constexpr int PER = kThreads / C::CHUNKS;  // rows per pass
    const int c = tid % C::CHUNKS;
#pragma unroll
    for (int r = tid / C::CHUNKS; r < kTileKeys; r += PER) {
      const long long off = s_koff[x % kRing][r];
      const long long at = off < 0 ? 0 : off + 8 * c;
      cp16(dst + sw<HD>(r, c), static_cast<const T*>(a.kv.k) + at, off >= 0);
      cp16(dst + C::HALF + sw<HD>(r, c), static_cast<const T*>(a.kv.v) + at, off >= 0);
    }
  };

  for (int x = 0; x < C::STAGES && x < count; ++x) {
    lookup();
    publish(x);
    if (x + 1 < count) cursor_next(look, a, sh);
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < C::STAGES - 1; ++x) {
    if (x < count) issue(x);
    cp_commit();
  }

  Warp<T, HD> w;
  bool split_keys = cur.nrows <= 16;  // the warps share the tile's keys, not the rows
  w.start(a, cur, split_keys ? 0 : warp * 16, lane);
  int first_u = u0 - cur.tile;  // the item's first unit
  for (int i = 0; i < count; ++i) {
    cp_wait<C::STAGES - 2>();
    __syncthreads();
    if (i + C::STAGES - 1 < count) issue(i + C::STAGES - 1);
    cp_commit();
    const bool more = i + C::STAGES < count;
    if (more) lookup();

    const uint32_t ks = s0 + (i % C::STAGES) * C::STAGE, vs = ks + C::HALF;
    const uint64_t mask = (uint64_t)s_mask[i % kRing][1] << 32 | s_mask[i % kRing][0];
    const int key0 = cur.tile * kTileKeys;
    if (mask) {
      const bool whole = mask == ~0ull && key0 + kTileKeys <= cur.first;
      bool odd = false;
      if (cur.first < cur.limit && key0 + kTileKeys > cur.first) {
        // keys that the first row may not see and the last one does: is any of their V infinite or NaN?
        constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
        const int lo = max(cur.first - key0, 0);
        bool bad = false;
        for (int x = tid + lo * C::CHUNKS; x < kTileKeys * C::CHUNKS; x += kThreads) {
          const uint4 v = *reinterpret_cast<const uint4*>(smem + (vs - s0) + sw<HD>(x / C::CHUNKS, x % C::CHUNKS));
          const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) bad |= (vv[e] & E) == E || (vv[e] >> 16 & E) == E;
        }
        odd = __syncthreads_or(bad);
      }
      if (split_keys)
        w.template tile<2>(ks, vs, warp * 16, key0, mask, whole, odd, a.scale2, lane);
      else if (warp * 16 < cur.nrows)
        w.template tile<8>(ks, vs, 0, key0, mask, whole, odd, a.scale2, lane);
    }
    if (more) {
      publish(i + C::STAGES);
      if (i + C::STAGES + 1 < count) cursor_next(look, a, sh);
    }

    const bool item_end = cur.tile == cur.tiles - 1;
    if (!item_end && i + 1 < count) {
      ++cur.tile;
      continue;
    }
    // the run of this item ends here: its part
    w.sum_quads();
    Dest d;
    d.whole = item_end && first_u >= u0;
    d.a = &a;
    d.q0 = cur.q0;
    d.base = cur.rt * kTileRows;
    d.h = cur.h;
    if (d.whole) {
      const long long at = cur.b < 0 ? 0 : (long long)a.rows * a.H;
      d.o = a.row_o + at * HD;
      d.ml = a.row_ml + at;
    } else {
      const int at = (2 * blockIdx.x + (first_u >= u0)) * kTileRows;
      d.o = a.cut_o + (long long)at * HD;
      d.ml = a.cut_ml + at;
    }
    if (!split_keys) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = warp * 16 + (lane >> 2) + 8 * e;
        if (r < cur.nrows) {
          const long long row = d.row(r);
          float* op = d.o + row * HD + 2 * (lane & 3);
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(op + 8 * n) = make_float2(w.o[n][2 * e], w.o[n][2 * e + 1]);
          if ((lane & 3) == 0) d.ml[row] = make_float2(w.m[e], w.l[e]);
        }
      }
    } else {
      // merge the warps' keys in the tile buffer just read ([4][16][HD] fp32 is its size)
      float* so = reinterpret_cast<float*>(smem + (ks - s0));
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = (lane >> 2) + 8 * e;
        if (r < cur.nrows) {
          float* op = so + (warp * 16 + r) * HD + 2 * (lane & 3);
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(op + 8 * n) = make_float2(w.o[n][2 * e], w.o[n][2 * e + 1]);
          if ((lane & 3) == 0) s_m[warp][r] = w.m[e], s_l[warp][r] = w.l[e];
        }
      }
      __syncthreads();
      for (int x = tid; x < cur.nrows * HD; x += kThreads) {
        const int r = x / HD, e = x - r * HD;
        const float mm = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float o = 0.0f, l = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float f = exp2f(s_m[k][r] - ref);
          o = fmaf(f, so[(k * 16 + r) * HD + e], o);
          l = fmaf(f, s_l[k][r], l);
        }
        const long long row = d.row(r);
        d.o[row * HD + e] = o;
        if (e == 0) d.ml[row] = make_float2(mm, l);
      }
    }
    if (i + 1 < count) {
      cursor_next(cur, a, sh);
      first_u = u0 + i + 1;
      split_keys = cur.nrows <= 16;
      w.start(a, cur, split_keys ? 0 : warp * 16, lane);
    }
  }
  if (a.tc_splits) griddep_wait();
}

// Joins a row's parts, a warp per (row, head): every part is (max, sum, weighted V); the prefix's and the own keys'
// come from whichever CTAs' runs the row's items lie in, 32 parts a round with all their loads side by side.
// Bound by latency (batch search, (max, sum), V: three dependent loads) until the parts outgrow L2; `per`
// rows a warp keep the grid to one wave.
constexpr int kJoinWarps = 4, kJoinResident = kSms * 48;  // warps that run at once

template <typename T, int HD>
__global__ void __launch_bounds__(32 * kJoinWarps) prefix_join_kernel(PrefixArgs a, int grid, int per) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const long long n_rows = (long long)a.rows * a.H;
  const long long row0 = ((long long)blockIdx.x * kJoinWarps + (threadIdx.x >> 5)) * per;
  griddep_launch_dependents();
  griddep_wait();
  const int units = a.prefix_units + __ldcg(a.cum + a.b.batch), ctas = min(grid, units);
  const int p_row_tiles = (a.rows * a.g + kTileRows - 1) / kTileRows;
  const int p_tiles = (a.b.prefix_len - a.prefix_skip + kTileKeys - 1) / kTileKeys;
  int t = -1, b = -1, q0 = 0, own_first = 0, own_row_tiles = 1, own_tiles = 0;
  for (long long row = row0; row < min(row0 + per, n_rows); ++row) {
    const int head = (int)(row % a.H), h = head / a.g;
    if ((int)(row / a.H) != t) {
      t = (int)(row / a.H);
      b = batch_find(a.b.q_start, a.b.batch, t, lane);
      if (b >= 0) {
        const int2 r = batch_rows(a.b.q_start, b, a.rows);
        const int c0 = __ldcg(a.cum + b), c1 = __ldcg(a.cum + b + 1);
        q0 = r.x;
        own_first = a.prefix_units + c0;
        own_row_tiles = ((r.y - r.x) * a.g + kTileRows - 1) / kTileRows;
        own_tiles = (c1 - c0) / (max(own_row_tiles, 1) * a.Hkv);
      }
    }
    if (b < 0) continue;
    // the prefix's item and the own keys' item of this row: its row in the row tile, first CTA, number of parts
    const int pr = t * a.g + head - h * a.g, orow = (t - q0) * a.g + head - h * a.g;
    int p_c0 = 0, p_n = 0, o_c0 = 0, o_n = 0;
    if (p_tiles > 0) {
      const int u = (h * p_row_tiles + pr / kTileRows) * p_tiles;
      p_c0 = cta_of(u, units, ctas);
      p_n = cta_of(u + p_tiles - 1, units, ctas) - p_c0 + 1;
    }
    if (own_tiles > 0) {
      const int u = own_first + (h * own_row_tiles + orow / kTileRows) * own_tiles;
      o_c0 = cta_of(u, units, ctas);
      o_n = cta_of(u + own_tiles - 1, units, ctas) - o_c0 + 1;
    }
    const int parts = a.tc_splits + p_n + o_n;
    float acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int k0 = 0; k0 < parts; k0 += 32) {
      int k = k0 + lane;
      float2 x = make_float2(-INFINITY, 0.0f);
      const float* o = a.row_o;
      if (k < a.tc_splits) {
        x = __ldcg(a.tc_ml + k * n_rows + row);
        o = a.tc_o + (k * n_rows + row) * HD;
      } else if (k < parts) {
        k -= a.tc_splits;
        const bool pre = k < p_n;
        if (!pre) k -= p_n;
        if ((pre ? p_n : o_n) == 1) {
          const long long at = row + (pre ? 0 : n_rows);
          x = __ldcg(a.row_ml + at);
          o = a.row_o + at * HD;
        } else {
          const int at = (2 * ((pre ? p_c0 : o_c0) + k) + (k == 0)) * kTileRows + (pre ? pr : orow) % kTileRows;
          x = __ldcg(a.cut_ml + at);
          o = a.cut_o + (long long)at * HD;
        }
      }
      const float mm = fmaxf(m, warp_max(x.x)), ref = mm == -INFINITY ? 0.0f : mm;
      const float f = exp2f(m - ref), weight = exp2f(x.x - ref);  // a part without keys: 0
      l = l * f + warp_sum(x.y * weight);
      m = mm;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= f;
      const int n = min(32, parts - k0);
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float w = __shfl_sync(0xffffffffu, weight, i);
        const float* src = reinterpret_cast<const float*>(
            __shfl_sync(0xffffffffu, (unsigned long long)reinterpret_cast<uintptr_t>(o), i)) + lane * E;
        float v[E];
        if constexpr (E == 4)
          *reinterpret_cast<float4*>(v) = __ldcg(reinterpret_cast<const float4*>(src));
        else if constexpr (E == 2)
          *reinterpret_cast<float2*>(v) = __ldcg(reinterpret_cast<const float2*>(src));
        else
          v[0] = __ldcg(src);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(v[e], w, acc[e]);
      }
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // no keys: zero
    T* out = static_cast<T*>(a.out) + row * HD + lane * E;
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(out) = make_uint2(Half16<T>::pack(acc[0] * inv, acc[1] * inv), Half16<T>::pack(acc[2] * inv, acc[3] * inv));
    else if constexpr (E == 2)
      *reinterpret_cast<uint32_t*>(out) = Half16<T>::pack(acc[0] * inv, acc[1] * inv);
    else
      *out = T(acc[0] * inv);
  }
}

template <int HD>
constexpr int ctas() {
  return Cfg<HD>::CTAS * kSms;
}
int grid_of(int hd) { return hd == 128 ? ctas<128>() : hd == 64 ? ctas<64>() : ctas<32>(); }

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// workspace: cum | (max, sum) and weighted V by output row, prefix then own keys | the same of cut items
// | the same of the tensor-core kernel's splits
struct Plan {
  size_t cum, row_ml, row_o, cut_ml, cut_o, tc_ml, tc_o, total;
  PrefixTcPlan tc;
};
Plan plan(int rows, int H, const q4b_batch& b, const q4b_paged_kv& kv) {
  Plan p;
  const int hd = kv.head_dim, batch = b.batch;
  p.tc = prefix_tc_plan(rows, H, b.prefix_len, kv);
  const size_t tc = (size_t)p.tc.splits * rows * H;
  const size_t n = 2 * (size_t)rows * H, cut = 2 * (size_t)grid_of(hd) * kTileRows;
  p.cum = 0;
  p.row_ml = up256((batch + 1) * sizeof(int));
  p.row_o = p.row_ml + up256(n * sizeof(float2));
  p.cut_ml = p.row_o + up256(n * hd * sizeof(float));
  p.cut_o = p.cut_ml + up256(cut * sizeof(float2));
  p.tc_ml = p.cut_o + up256(cut * hd * sizeof(float));
  p.tc_o = p.tc_ml + up256(tc * sizeof(float2));
  p.total = p.tc_o + up256(tc * hd * sizeof(float));
  return p;
}

template <typename T, int HD>
int launch(const PrefixArgs& a, cudaStream_t st) {
  using C = Cfg<HD>;
  auto kern = prefix_attn_kernel<T, HD>;
  static std::atomic<unsigned long long> done;
  cudaError_t e = set_max_dynamic_smem(kern, C::STAGES * C::STAGE + 12 * (kMaxBatch + 1), done);
  if (e == cudaSuccess)
    e = launch_pdl(kern, dim3(ctas<HD>()), dim3(kThreads), C::STAGES * C::STAGE + 12 * (a.b.batch + 1), st, a);
  const long long n = (long long)a.rows * a.H;
  const int per = (int)((n + kJoinResident - 1) / kJoinResident);
  if (e == cudaSuccess)
    e = launch_pdl(prefix_join_kernel<T, HD>, dim3((unsigned)((n + kJoinWarps * per - 1) / (kJoinWarps * per))),
                   dim3(32 * kJoinWarps), 0, st, a, ctas<HD>(), per);
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
  // key tiles of all items, at most: they are counted in 32 bits
  const double g = n_heads / kv->n_kv_heads, tiles = (double)b->table_width * kv->page_size / kTileKeys + 1;
  if (((rows * g / kTileRows + b->batch) * tiles + (rows * g / kTileRows + 1) * (b->prefix_len / kTileKeys + 1.0)) *
              kv->n_kv_heads > 2e9 || rows * (double)n_heads > 2e9)
    return set_error(Q4B_EUNSUPPORTED, "%s: the step is too large; split its rows", what);
  return Q4B_OK;
}

}  // namespace
}  // namespace q4b

using namespace q4b;

extern "C" size_t q4b_prefix_attention_workspace(int rows, int n_heads, const q4b_batch* batch, const q4b_paged_kv* kv) {
  if (check("prefix_attention", rows, n_heads, batch, kv)) return 0;
  return plan(rows, n_heads, *batch, *kv).total;
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
  const Plan p = plan(rows, n_heads, *batch, *kv);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < p.total)
    return set_error(Q4B_EINVAL, "%s: needs a 256-byte aligned workspace of %zu bytes", what, p.total);
  PrefixArgs a;
  a.q = q, a.q_stride = q_stride, a.q_head_stride = q_head_stride;
  a.rows = rows, a.H = n_heads, a.Hkv = kv->n_kv_heads, a.g = n_heads / kv->n_kv_heads;
  a.scale2 = scale * 1.44269504088896340736f;
  a.b = *batch, a.kv = *kv, a.prefix_pages = prefix_pages, a.out = out;
  // the tensor-core kernel reads q in 16-byte pieces
  const bool tc = p.tc.splits && aligned(q, 16) && q_stride % 8 == 0 && q_head_stride % 8 == 0;
  a.tc_splits = tc ? p.tc.splits : 0, a.tc_pairs = p.tc.pairs, a.tc_tiles = p.tc.tiles;
  a.prefix_skip = tc ? p.tc.tiles * 128 : 0;
  a.prefix_units = a.Hkv * ((rows * a.g + kTileRows - 1) / kTileRows) *
                   ((batch->prefix_len - a.prefix_skip + kTileKeys - 1) / kTileKeys);
  char* w = static_cast<char*>(workspace);
  a.cum = reinterpret_cast<int*>(w + p.cum);
  a.row_ml = reinterpret_cast<float2*>(w + p.row_ml);
  a.row_o = reinterpret_cast<float*>(w + p.row_o);
  a.cut_ml = reinterpret_cast<float2*>(w + p.cut_ml);
  a.cut_o = reinterpret_cast<float*>(w + p.cut_o);
  a.tc_ml = reinterpret_cast<float2*>(w + p.tc_ml);
  a.tc_o = reinterpret_cast<float*>(w + p.tc_o);
  const cudaStream_t st = as_stream(stream);
  if (tc)
    if (int rc = prefix_tc_run(a, st)) return rc;
  const bool h16 = kv->dtype == Q4B_F16;
  switch (kv->head_dim) {
    case 128: return h16 ? launch<__half, 128>(a, st) : launch<__nv_bfloat16, 128>(a, st);
    case 64: return h16 ? launch<__half, 64>(a, st) : launch<__nv_bfloat16, 64>(a, st);
    default: return h16 ? launch<__half, 32>(a, st) : launch<__nv_bfloat16, 32>(a, st);
  }
}
