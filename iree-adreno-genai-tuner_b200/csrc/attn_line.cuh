// The line of key tiles that the batched attention kernels share their work by (AttnLine): units, runs and
// cursors. TR rows (tokens x heads of a KV head's group) per row tile, TK keys per unit.
#pragma once

#include <type_traits>

#include "paged.cuh"
#include "prefix_attn.h"

namespace q4b {

// A wait within the call's limit; a limit of zero gives up without a look.
__device__ __forceinline__ bool wait_for(const PrefixArgs& a, uint64_t* bar, uint32_t parity) {
  return a.wait_ns && mbar_wait_bounded(bar, parity, a.wait_ns);
}

// First unit of CTA c, and the CTA that holds unit u, for `units` units over `ctas` CTAs.
__device__ __forceinline__ int cta_first(int c, int units, int ctas) { return (int)((long long)c * units / ctas); }
// The largest c with cta_first(c) <= u, i.e. with c * units <= (u + 1) * ctas - 1: by a guess in fp32 (off by one at most:
// c is a few hundred), set right exactly. A 64-bit division would be most of the join's instructions.
__device__ __forceinline__ int cta_of(int u, int units, int ctas) {
  const long long n = ((long long)u + 1) * ctas - 1;
  int c = min((int)__fdividef((float)n, (float)units), ctas - 1);
  while ((long long)c * units > n) --c;
  while ((long long)(c + 1) * units <= n) ++c;
  return c;
}

// Weights are rounded to the cache's type for the PV product. fp16 ends at 2^-24: beside one large weight the small ones of a
// long context would be lost, all of them (40,000 keys of weight 2^-26 make 6e-4 of the result). So a kernel whose weights are
// at most 2^SLACK multiplies them by the power of two that brings them up to 2^15, and leaves its maxima that much smaller.
// What is then lost to fp16's end is less than 2^(SLACK - 40) of the largest weight a key.
template <typename T, int SLACK>
constexpr float kLift = std::is_same<T, __half>::value ? 15.0f - SLACK : 0.0f;
// The reference that weights are taken against, and the maximum that is left for the join. Rounded up: where a maximum is so large
// that the difference is not exact (2^24 and more), the lift becomes smaller, and no weight leaves fp16.
template <typename T, int SLACK>
__device__ __forceinline__ float lifted(float m) {
  if constexpr (kLift<T, SLACK> == 0.0f) return m;
  return __fsub_ru(m, kLift<T, SLACK>);
}

// Per sequence, in shared memory; every value bounded.
struct BatchTable {
  int* cum;  // [batch + 1] units of this line in front of sequence b, behind the prefix's
  int* q0;   // [batch + 1] first row
  int* len;  // [batch] own keys, those behind the page table among them
};

// Own keys of a sequence that its page table holds
__device__ __forceinline__ int held(const PrefixArgs& a, int len) { return min(len, a.table_keys); }

__device__ __forceinline__ int line_units(const PrefixArgs& a, const AttnLine& line, int n, int len, int tr, int tk) {
  const int r = n * a.g;
  return r > line.own_lo && r <= line.own_hi ? a.Hkv * ((r + tr - 1) / tr) * ((held(a, len) + tk - 1) / tk) : 0;
}

// Exclusive running sum of `mine` over the block's threads, and the total; `s` holds a word per warp and one more.
template <int THREADS>
__device__ __forceinline__ int block_scan(int mine, int* s, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  __syncthreads();
  if (lane == 31) s[warp] = run;
  __syncthreads();
  int before = run - mine;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s[w];
    total += s[w];
  }
  return before;
}

// Fills the table, thread t a run of sequences; returns whether the offsets decrease somewhere, in which case
// no sequence has rows (the units stay countable). Ends with a barrier still to come.
template <int THREADS>
__device__ __forceinline__ bool batch_table(const PrefixArgs& a, const BatchTable& s) {
  const int B = a.b.batch;
  bool bad = false;
  for (int b = threadIdx.x; b <= B; b += THREADS) {
    const int q = __ldg(a.b.q_start + b);
    s.q0[b] = min(max(q, 0), a.rows);
    if (b < B) {
      bad |= __ldg(a.b.q_start + b + 1) < q;
      s.len[b] = min(max(__ldg(a.b.seq_lens + b), 0), 0x7fffffff - kTcRows);  // row_limit counts on from here
    }
  }
  return __syncthreads_or(bad);
}

// The line's running sums into s.cum (behind batch_table); returns the own units.
template <int THREADS, int TR, int TK>
__device__ __forceinline__ int line_table(const PrefixArgs& a, const AttnLine& line, const BatchTable& s, bool bad, int* scan) {
  const int B = a.b.batch, per = (B + THREADS - 1) / THREADS;
  const int b0 = min((int)threadIdx.x * per, B), b1 = min(b0 + per, B);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += bad ? 0 : line_units(a, line, s.q0[b + 1] - s.q0[b], s.len[b], TR, TK);
  int total;
  int at = block_scan<THREADS>(mine, scan, total);
  for (int b = b0; b < b1; ++b) {
    s.cum[b] = at;
    at += bad ? 0 : line_units(a, line, s.q0[b + 1] - s.q0[b], s.len[b], TR, TK);
  }
  if (threadIdx.x == 0) s.cum[B] = total;
  __syncthreads();
  return total;
}

// An item, and the tile of it that a unit stands for.
struct Cursor {
  int b;      // sequence, -1: the prefix
  int h, rt;  // KV head, row tile
  int tile, tiles, row_tiles;
  int q0, n, len;  // first row, rows and keys (that are held) of the sequence (prefix: 0, all rows, prefix_len)
  int nrows;       // rows of this row tile
  int limit;       // keys that its last row sees
  int first;       // keys that its first row sees
};

template <int TR, int TK>
struct Line {
  const PrefixArgs& a;
  const AttnLine& line;
  const BatchTable& s;

  __device__ __forceinline__ void item(Cursor& c) const {
    c.nrows = min(TR, c.n * a.g - c.rt * TR);
    if (c.b < 0) {
      c.limit = c.first = c.len;
    } else {
      const int j0 = c.rt * TR / a.g, j1 = (c.rt * TR + c.nrows - 1) / a.g;
      const int seen = s.len[c.b] - c.n;  // own keys in front of the first row; negative: fewer keys than rows
      c.first = min(max(seen + j0 + 1, 0), c.len);
      c.limit = min(max(seen + j1 + 1, 0), c.len);
    }
  }
  __device__ __forceinline__ void sequence(Cursor& c) const {
    if (c.b < 0) {
      c.q0 = 0;
      c.n = a.rows;
      c.len = a.b.prefix_len;
    } else {
      c.q0 = s.q0[c.b];
      c.n = s.q0[c.b + 1] - c.q0;
      c.len = held(a, s.len[c.b]);
    }
    c.row_tiles = (c.n * a.g + TR - 1) / TR;
    c.tiles = (c.len + TK - 1) / TK;
  }
  __device__ Cursor at(int u) const {
    Cursor c;
    c.b = -1;
    if (u >= line.prefix_units) {
      u -= line.prefix_units;
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
    }
    sequence(c);
    c.tile = u % c.tiles;
    u /= c.tiles;
    c.rt = u % c.row_tiles;
    c.h = u / c.row_tiles;
    item(c);
    return c;
  }
  // the next item, at its first tile; the caller knows that there is one
  __device__ __forceinline__ void next_item(Cursor& c) const {
    c.tile = 0;
    if (++c.rt == c.row_tiles) {
      c.rt = 0;
      if (++c.h == a.Hkv) {
        c.h = 0;
        do ++c.b;
        while (s.cum[c.b + 1] == s.cum[c.b]);
        sequence(c);
      }
    }
    item(c);
  }
  __device__ __forceinline__ void next(Cursor& c) const {
    if (++c.tile == c.tiles) next_item(c);
  }
};

// keys that row r of the cursor's row tile sees
__device__ __forceinline__ int row_limit(const PrefixArgs& a, const BatchTable& s, const Cursor& c, int r, int tr) {
  return c.b < 0 ? c.len : min(s.len[c.b] - c.n + (c.rt * tr + r) / a.g + 1, c.len);
}

// Where a run of an item puts (max, sum) and weighted V of row r of its row tile: by the output row if the run is the
// whole item, else in one of the CTA's two places for cut items (0: it began in an earlier CTA); the
// places start with those of "CTA" cut0.
struct Dest {
  float* o;
  float2* ml;
  bool whole;
  int q0, base, h, g, H;
  __device__ __forceinline__ long long row(int r) const {
    if (!whole) return r;
    const int rr = base + r, j = rr / g;
    return (long long)(q0 + j) * H + h * g + rr - j * g;
  }
};
template <int TR>
__device__ __forceinline__ Dest dest(const PrefixArgs& a, const Cursor& c, bool began, bool ends, int cut0, float* cut_o, float2* cut_ml, int hd) {
  Dest d;
  d.whole = began && ends;
  d.q0 = c.q0, d.base = c.rt * TR, d.h = c.h, d.g = a.g, d.H = a.H;
  long long at;
  if (d.whole) {
    at = c.b < 0 ? 0 : (long long)a.rows * a.H;
    d.o = a.row_o, d.ml = a.row_ml;
  } else {
    at = (2ll * (cut0 + blockIdx.x) + began) * TR;
    d.o = cut_o, d.ml = cut_ml;
  }
  d.o += at * hd, d.ml += at;
  return d;
}

}  // namespace q4b
