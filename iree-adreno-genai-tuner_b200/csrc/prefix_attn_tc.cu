// Batched attention on the tcgen05 tensor cores, for the items with many rows: the shared prefix, where all
// rows of the step and all heads of a KV head's group attend to the same keys, and the sequences with many
// new rows. QK and PV are then matrix products with M = rows * heads per KV head.
//
//   S = Q K^T * scale;  P = exp2(S log2e - m);  O += P V;  l += sum P       (m: a running reference per row)
//
// One CTA per SM takes an equal run of the prefix's items and one of the own keys' (attn_line.cuh; row tiles of 256,
// key tiles of 128).
// Warps 0-3 and 4-7 are the softmax of one half of the row tile each, a thread a row; warp 8 brings K and V tiles by TMA
// (a box per page, 128-byte swizzle, a ring of tiles that runs on across items); one thread of warp 9 issues the
// MMAs (two more warps only fill up the warpgroup that gives up registers). S and O live in TMEM (2 x 128 + 2 x head_dim columns), and P goes back into S's columns as the A
// operand of the PV product, so nothing but K, V and Q passes through shared memory. The two halves alternate: while
// one's softmax runs, the tensor core works for the other, and both use every K and V tile that comes in. The
// next item's Q and first product overlap the end of the item before.
//
// m moves only when a row's maximum outgrows it by 2^8, which keeps P below 256 (times kLift) and spares most tiles the pass over
// O; exactness is not affected (l and O carry the same factor). P is rounded to the cache's type, as in
// the other kernel. Masks (the end of the keys, causal rows, pages that do not exist) cost only where a tile has
// any: scores by selection, and V by zeros written over the tile where some row may not see a key, since
// 0 * V is not 0 for infinite or NaN V; what such a V gives to the rows that do see it is added at the end.
//
// Bound by the chain of one half's tile, with the other half's beside it: S to P 2000 clocks (TMEM reads 300, maximum
// 280, exponentials 1350 at 16 a clock per SM), P to the next S 1300 (PV 500, QK 560, the barriers' latency the rest).
// The tensor pipe is active 0.51 of the time. Measured: 192 rows x 32 heads behind 65,536 keys (206 GFLOP) 194 us, 1.06
// PFLOP/s, and 1.2 PFLOP/s without start and end, 0.7 of the measured bf16 rate; start and end are some 25 us (first
// reads of offsets, pages, Q, K, the parts). Tried and slower: two threads a row (253 us), S in two buffers of 64 keys with
// the next products begun two ahead (243: an MMA of 64 columns takes as long as one of 128), the product of the first 64
// keys begun before the last exponentials (196), each TMEM read beside the maximum of the columns before (206), a
// quarter of the exponentials as polynomials (213), S read twice in rolled loops for fewer registers (241), weights against
// the old maximum and once more if it was outgrown (203), a ring of 5 single tiles (200), with head_dim 64 columns of their
// own for P and the next S begun when the last has been read (180 against 162). Neither pipe is full (tensor 0.50,
// exponentials 0.56, issue 0.33): a warp alone on its scheduler waits 2.3 clocks an instruction for its last results, and
// more warps have no registers.
#include <type_traits>

#include "attn_line.cuh"
#include "tc.cuh"

namespace q4b {
namespace {

constexpr int kTcThreads = 384;
// Registers: the softmax groups (256 threads) take from the four other warps; together no more than the 168
// a thread that the block is launched with (256 * 208 + 128 * 80 <= 384 * 168).
constexpr int kRegsLaunch = 168, kRegsSoftmax = 208, kRegsOther = 80;
static_assert(256 * kRegsSoftmax + 128 * kRegsOther <= kTcThreads * kRegsLaunch, "setmaxnreg draws on the block's own registers");
constexpr int kHalf = kTcRows / 2;  // rows of one softmax group and MMA
constexpr int kSlack = 8;  // base-2 growth of a row's maximum that its reference tolerates

__device__ unsigned g_prefix_status = 0;

template <int HD>
struct TcCfg {
  static constexpr int HALVES = HD / 64;                   // 64-column (128-byte) halves of a row
  static constexpr int ATOM = kTcKeys * 128;               // one half of a 128-row tile, bytes
  static constexpr int TILE = HALVES * ATOM;               // Q half, K or V tile
  static constexpr int SLOTS = HD == 128 ? 2 : 4;          // pairs of a V and the next K tile in flight
  static constexpr int SMEM = (2 + 2 * SLOTS) * TILE + 1024;  // + alignment to the swizzle's 1024 bytes
};

// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void tc_mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 columns of this warp's lanes, without the wait
__device__ __forceinline__ void tmem_ld_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// the wait; the registers pass through it, so that no use of them moves in front of it
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_st_32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 32 bytes, one whole sector, of one row
__device__ __forceinline__ void st_8(float* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The run of one item that a CTA takes: tiles [t0, t1) of the cursor's item, of which those from `e1` on hold no key
// that a row of it sees.
struct Seg {
  Cursor c;
  int t0, t1, e1;
  __device__ __forceinline__ int n() const { return max(e1 - t0, 0); }
  __device__ __forceinline__ int active() const { return c.nrows > kHalf ? 2 : 1; }
};

// The segments of a CTA's runs, in order: one run of the own keys' units and one of the prefix's. Each is an equal share,
// so that the two kinds, whose units cost differently, spread evenly.
struct Segs {
  const Line<kTcRows, kTcKeys>& line;
  int u, u1, then0, then1;
  Seg s;
  __device__ __forceinline__ Segs(const Line<kTcRows, kTcKeys>& line, int2 own, int2 prefix)
      : line(line), u(own.x), u1(own.y), then0(prefix.x), then1(prefix.y) {
    start();
  }
  __device__ __forceinline__ void start() {
    if (u >= u1) {
      u = then0, u1 = then1;
      then0 = then1 = 0;
    }
    if (u < u1) {
      s.c = line.at(u);
      set();
    }
  }
  __device__ __forceinline__ void set() {
    s.t0 = s.c.tile;
    s.t1 = min(s.c.tiles, s.t0 + u1 - u);
    s.e1 = min(s.t1, (s.c.limit + kTcKeys - 1) / kTcKeys);
  }
  __device__ __forceinline__ bool valid() const { return u < u1; }
  __device__ __forceinline__ void next() {
    u += s.t1 - s.t0;
    if (u < u1) {
      line.next_item(s.c);
      set();
    } else {
      start();
    }
  }
};

__device__ __forceinline__ const int32_t* page_row(const PrefixArgs& a, const Cursor& c) {
  return c.b < 0 ? a.prefix_pages : a.b.page_table + c.b * a.b.table_stride;
}

// The top bit of each half of the result: whether that half of v is an infinity or NaN (exponent all ones).
template <typename T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t v) {
  constexpr bool H16 = std::is_same<T, __half>::value;
  return (v & (H16 ? 0x7C007C00u : 0x7F807F80u)) + (H16 ? 0x04000400u : 0x00800080u);
}

// pairs of fp32 in one instruction
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, PrefixArgs a) {
  using C = TcCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  __shared__ uint64_t full[C::SLOTS], empty[C::SLOTS], q_full[2], s_full[2], p_full[2], o_full[2], drained;
  __shared__ uint32_t s_tmem;
  __shared__ int s_fail, s_issued, s_odd, s_scan[kTcThreads / 32];
  constexpr uint32_t kS = 0, kO = 256;  // TMEM columns: S (and P) of half i at 128 i, O at 256 + HD i

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], kHalf);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kHalf);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(&drained, 1);
    s_fail = s_issued = s_odd = 0;
    fence_mbar_init();
    tma_prefetch_map(&tk);
    tma_prefetch_map(&tv);
  }
  if (warp == 9) tmem_alloc(&s_tmem, 512);
  tc_fence_before();
  griddep_wait();
  griddep_launch_dependents();  // behind the wait: what runs next may read the inputs at once
  BatchTable table;
  table.cum = reinterpret_cast<int*>(smem + (2 + 2 * C::SLOTS) * C::TILE);
  table.q0 = table.cum + a.b.batch + 1;
  table.len = table.q0 + a.b.batch + 1;
  int own_units = 0;
  if (a.tc.own_lo < a.tc.own_hi) {
    const bool bad = batch_table<kTcThreads>(a, table);
    own_units = line_table<kTcThreads, kTcRows, kTcKeys>(a, a.tc, table, bad, s_scan);
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  volatile int* fail = &s_fail;
  const Line<kTcRows, kTcKeys> line{a, a.tc, table};
  const int cta = blockIdx.x;
  auto share = [&](int units) {
    const int ctas = min((int)gridDim.x, units);  // fewer units than CTAs: one each, no run is empty
    return cta < ctas ? make_int2(cta_first(cta, units, ctas), cta_first(cta + 1, units, ctas)) : make_int2(0, 0);
  };
  // A run of own keys begins and ends between items where the item is short: an item's start and end cost about as much as
  // two or three tiles, and another part for the join.
  auto whole = [&](int u) {
    if (u == 0 || u == own_units) return u;
    const Cursor c = line.at(a.tc.prefix_units + u);
    return c.tiles > kTcWholeTiles ? u : u - c.tile + (2 * c.tile < c.tiles ? 0 : c.tiles);
  };
  int2 run_own = share(own_units);
  run_own = make_int2(a.tc.prefix_units + whole(run_own.x), a.tc.prefix_units + whole(run_own.y));
  const int2 run_prefix = share(a.tc.prefix_units);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 8) {
      // producer: an item's run of n tiles is n + 1 entries of the ring, entry p its V tile p - 1 and K tile p: what one round of
      // the MMA thread needs, under one barrier
      const int box = page_box(a.kv.page_size, kTcKeys), boxes = kTcKeys / box;
      int x = 0;
      bool ok = true;
      for (Segs g(line, run_own, run_prefix); ok && g.valid(); g.next()) {
        const Seg& s = g.s;
        const int n = s.n();
        if (n == 0) continue;
        const int32_t* pages = page_row(a, s.c);
        auto page_of = [&](int j) {
          int page = a.kv.n_pages;  // out of the map: zeros
          const int key = j * kTcKeys + lane * box;
          if (lane < boxes && key < s.c.limit) {
            page = __ldg(pages + key / a.kv.page_size);
            if (page < 0 || page >= a.kv.n_pages) page = a.kv.n_pages;
          }
          return page;
        };
        int page = page_of(s.t0), before = 0;  // of K tile p, of V tile p - 1
        for (int p = 0; p <= n; ++p, ++x) {
          const int slot = x % C::SLOTS, r = x / C::SLOTS, j = s.t0 + p;
          if (lane == 0) {
            ok = r == 0 || wait_for(a, &empty[slot], (r - 1) & 1);
            if (ok) {
              mbar_arrive_expect_tx(&full[slot], p == 0 || p == n ? C::TILE : 2 * C::TILE);
              s_issued = x + 1;
            } else {
              *fail = 1;
            }
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          const int next = p + 1 < n ? page_of(j + 1) : 0;
          if (lane < boxes) {
            const uint32_t dst = base + (2 + 2 * slot) * C::TILE + lane * box * 128;
            const int key = j * kTcKeys + lane * box;
#pragma unroll
            for (int c = 0; c < C::HALVES; ++c) {
              if (p < n) tma_load_4d(dst + c * C::ATOM, &tk, 64 * c, key % a.kv.page_size, s.c.h, page, &full[slot]);
              if (p > 0) tma_load_4d(dst + C::TILE + c * C::ATOM, &tv, 64 * c, (key - kTcKeys) % a.kv.page_size, s.c.h, before, &full[slot]);
            }
          }
          before = page;
          page = next;
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      if (lane == 0) {
        constexpr uint32_t bf = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t idesc_s = idesc_f16_f32(kHalf, kTcKeys, false, false) | bf;
        constexpr uint32_t idesc_o = idesc_f16_f32(kHalf, HD, false, true) | bf;
        // Descriptors are made once and moved by adding to their address field (16-byte units): made anew for each MMA they
        // were most of this thread's time, and this thread was what the kernel waited for.
        const uint64_t q_desc = sw128_desc(base, 16, 1024), k_desc = sw128_desc(base + 2 * C::TILE, 16, 1024),
                       v_desc = sw128_desc(base + 3 * C::TILE, C::ATOM, 1024);
        auto wait_full = [&](int x) { return wait_for(a, &full[x % C::SLOTS], (x / C::SLOTS) & 1); };
        auto qk = [&](int i, int x) {
          const uint64_t q = q_desc + i * (C::TILE >> 4), k = k_desc + x % C::SLOTS * (2 * C::TILE >> 4);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const int off = ((kk / 4) * C::ATOM + (kk % 4) * 32) >> 4;
            tc_mma_f16(tmem + kS + 128 * i, q + off, k + off, idesc_s, kk != 0);
          }
          tc_commit(&s_full[i]);
        };
        auto pv = [&](int i, int x, bool first) {
          const uint64_t v = v_desc + x % C::SLOTS * (2 * C::TILE >> 4);
#pragma unroll
          for (int kk = 0; kk < kTcKeys / 16; ++kk)
            tc_mma_f16_ta(tmem + kO + HD * i, tmem + kS + 128 * i + 8 * kk, v + (kk * 2048 >> 4), idesc_o, !(first && kk == 0));
        };
        int x = 0, items = 0, items1 = 0, tiles = 0, tiles1 = 0;  // so far; ...1: those with a second half
        bool ok = true;
        for (Segs g(line, run_own, run_prefix); ok && g.valid(); g.next()) {
          const int n = g.s.n(), active = g.s.active();
          if (n == 0) continue;
          ok = wait_full(x);
          for (int i = 0; ok && i < active; ++i) {
            ok = wait_for(a, &q_full[i], (i ? items1 : items) & 1);
            if (!ok) break;
            tc_fence_after();
            qk(i, x);
          }
          if (ok) tc_commit(&empty[x % C::SLOTS]);
          for (int j = 0; ok && j < n; ++j) {
            ++x;
            ok = wait_full(x);
            for (int i = 0; ok && i < active; ++i) {
              ok = wait_for(a, &p_full[i], ((i ? tiles1 : tiles) + j) & 1);
              if (!ok) break;
              tc_fence_after();
              pv(i, x, j == 0);
              if (j + 1 < n)
                qk(i, x);
              else
                tc_commit(&o_full[i]);
            }
            if (ok) tc_commit(&empty[x % C::SLOTS]);
          }
          ++x;
          tiles += n, ++items;
          if (active == 2) tiles1 += n, ++items1;
        }
        if (!ok) *fail = 1;
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int i = warp / 4, row = (warp & 3) * 32 + lane;
    const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + kS + 128 * i;
    const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + kO + HD * i;
    auto load_q = [&](const Seg& s) {
      if (i >= s.active() || s.n() == 0) return;
      // Lane l finds row l of its warp; then HD / 8 lanes take a row, so that a load covers whole rows, all loads in flight
      // at once (they queue behind the first K and V tiles of all CTAs).
      constexpr int LANES = HD / 8, ROWS = 32 / LANES;
      const int rr = s.c.rt * kTcRows + i * kHalf + row, j = rr / a.g, c = lane % LANES;
      const long long mine = i * kHalf + row < s.c.nrows
                                 ? (s.c.q0 + j) * a.q_stride + (s.c.h * a.g + rr - j * a.g) * a.q_head_stride
                                 : -1;
      uint4 v[32 / ROWS];
#pragma unroll
      for (int y = 0; y < 32 / ROWS; ++y) {
        const long long off = __shfl_sync(0xffffffffu, mine, y * ROWS + lane / LANES);
        v[y] = off >= 0 ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + off) + c) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int y = 0; y < 32 / ROWS; ++y) {
        const int rw = (warp & 3) * 32 + y * ROWS + lane / LANES;
        *reinterpret_cast<uint4*>(smem + i * C::TILE + rw * 128 + (c / 8) * C::ATOM + (((c % 8) ^ (rw & 7)) << 4)) = v[y];
      }
      fence_async_smem();
      mbar_arrive(&q_full[i]);
    };
    int x = 0, tiles = 0, items = 0;  // ring entries so far; tiles and items of this half
    bool ok = true;
    Segs g(line, run_own, run_prefix);
    if (g.valid()) load_q(g.s);
    while (g.valid()) {
      const Seg s = g.s;
      const int n = s.n();
      g.next();
      if (i >= s.active()) {
        if (n > 0) x += n + 1;
        if (g.valid()) load_q(g.s);
        continue;
      }
      const int lim = row_limit(a, table, s.c, i * kHalf + row, kTcRows);
      const int32_t* pages = page_row(a, s.c);
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; ok && j < n; ++j) {
        const int key0 = (s.t0 + j) * kTcKeys;
        // a lane looks at the page of four keys (pages hold a multiple of 8)
        int page = 0;
        if (key0 + 4 * lane < s.c.limit) page = __ldg(pages + (key0 + 4 * lane) / a.kv.page_size);
        const unsigned there = __ballot_sync(0xffffffffu, page >= 0 && page < a.kv.n_pages);
        const bool edge = key0 + kTcKeys > s.c.first;  // some row does not see all of the tile's keys
        ok = wait_for(a, &s_full[i], (tiles + j) & 1);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (edge) {
          // Behind the wait for S: a half that sat out items may be ahead of the ring by more than the one phase that a
          // barrier's parity tells apart, but this tile's K is there, so its V is the barrier's current phase.
          const int xv = x + j + 1;
          ok = wait_for(a, &full[xv % C::SLOTS], (xv / C::SLOTS) & 1);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          // V of the keys that not every row sees: zeros behind the last one, and over what is not finite
          constexpr int ROW = 8 * C::HALVES;  // 16-byte chunks of a row
          const int from = max(s.c.first - key0, 0), to = min(s.c.limit - key0, kTcKeys);
          uint8_t* v = smem + (3 + 2 * (xv % C::SLOTS)) * C::TILE;
          auto chunk = [&](int y) { return reinterpret_cast<uint4*>(v + (y % ROW / 8) * C::ATOM + y / ROW * 128 + (y % 8) * 16); };
          uint32_t odd = 0;
#pragma unroll 4
          for (int y = from * ROW + row; y < to * ROW; y += kHalf) {
            const uint4 w = *chunk(y);
            odd |= odd_bits<T>(w.x) | odd_bits<T>(w.y) | odd_bits<T>(w.z) | odd_bits<T>(w.w);
          }
          for (int y = to * ROW + row; y < kTcKeys * ROW; y += kHalf) *chunk(y) = make_uint4(0, 0, 0, 0);
          if (odd & 0x80008000u) {
            *reinterpret_cast<volatile int*>(&s_odd) = 1;
            for (int y = from * ROW + row; y < to * ROW; y += kHalf) {
              const uint4 old = *chunk(y);
              uint32_t w[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t bits = odd_bits<T>(w[e]);
                if (bits & 0x8000u) w[e] &= 0xFFFF0000u;
                if (bits & 0x80000000u) w[e] &= 0x0000FFFFu;
              }
              *chunk(y) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          fence_async_smem();
          __syncwarp();  // the loops above end lane by lane, the TMEM loads below want the warp together
        }
        tc_fence_after();
        uint32_t sc[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_async(ts + 32 * c, sc[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_wait(sc[c]);
        if (edge) {
          const int vis = lim - key0;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * c + e >= vis) sc[c][e] = 0xff800000u;
        }
        if (there != 0xffffffffu) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((there >> (8 * c + e / 4)) & 1)) sc[c][e] = 0xff800000u;
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = __uint_as_float(sc[c][0]);
#pragma unroll
          for (int e = 1; e < 31; e += 2) mx[c] = max3(mx[c], __uint_as_float(sc[c][e]), __uint_as_float(sc[c][e + 1]));
          mx[c] = fmaxf(mx[c], __uint_as_float(sc[c][31]));
        }
        const float best = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const float top = best * a.scale2;
        // a row's reference moves for its own maximum only: its roundings do not depend on the rows beside it
        const bool grows = top > m + kSlack || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, grows)) {
          const float f = !grows ? 1.0f : m == -INFINITY ? 0.0f : ex2(m - top);
          if (grows) m = top;
          l *= f;
          if (j > 0) {  // PV of the tile before has ended: its S followed it
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              tmem_ld_async(to + 32 * c, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st_32(to + 32 * c, o);
            }
          }
        }
        const float ref = lifted<T, kSlack>(m == -INFINITY ? 0.0f : m);
        const uint64_t scale = pair(a.scale2, a.scale2), off = pair(-ref, -ref);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // P's 16 columns lie over columns of S that have been read
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 y = unpair(fma2(pair(__uint_as_float(sc[c][2 * e]), __uint_as_float(sc[c][2 * e + 1])), scale, off));
            y.x = ex2(y.x);
            y.y = ex2(y.y);
            sum[e & 1] = add2(sum[e & 1], pair(y.x, y.y));
            p[e] = Half16<T>::pack(y.x, y.y);
          }
          tmem_st_16(ts + 16 * c, p);
        }
        const float2 s01 = unpair(add2(sum[0], sum[1]));
        l += s01.x + s01.y;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[i]);
      }
      if (ok && g.valid()) load_q(g.s);  // the item's products with Q have ended
      if (ok && n > 0) {
        ok = wait_for(a, &o_full[i], items & 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (!ok) {
        *fail = 1;
        l = __int_as_float(0x7fffffff);  // a row whose work gave up is NaN, not stale
      }
      const Dest d = dest<kTcRows>(a, s.c, s.t0 == 0, s.t1 == s.c.tiles, s.c.b < 0 ? 0 : gridDim.x, a.tc_o, a.tc_ml, HD);
      const bool on = i * kHalf + row < s.c.nrows;
      const long long at = on ? d.row(i * kHalf + row) : 0;
      const bool odd = *reinterpret_cast<volatile int*>(&s_odd) != 0;
      if (ok) {
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          __syncwarp();  // behind the loop over `odd` keys, whose length differs by lane
          if (n > 0) {
            tmem_ld_async(to + 32 * c, o);
            tmem_ld_wait(o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
          }
          if (odd) {  // what the zeros written over V took from the rows that see it
            for (int key = max(s.c.first, s.t0 * kTcKeys); key < min(lim, s.e1 * kTcKeys); ++key) {
              const int page = __ldg(pages + key / a.kv.page_size);
              if (page < 0 || page >= a.kv.n_pages) continue;
              const uint32_t* v = reinterpret_cast<const uint32_t*>(
                  static_cast<const T*>(a.kv.v) + page * a.kv.page_stride + (key % a.kv.page_size) * a.kv.slot_stride +
                  s.c.h * a.kv.head_stride + 32 * c);
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const uint32_t w = __ldg(v + e);
                const float2 f = Half16<T>::unpack(w);
                if (odd_bits<T>(w) & 0x8000u) o[2 * e] = __float_as_uint(__uint_as_float(o[2 * e]) + f.x);
                if (odd_bits<T>(w) & 0x80000000u) o[2 * e + 1] = __float_as_uint(__uint_as_float(o[2 * e + 1]) + f.y);
              }
            }
          }
          if (on) {
#pragma unroll
            for (int e = 0; e < 4; ++e) st_8(d.o + at * HD + 32 * c + 8 * e, o + 8 * e);
          }
        }
      }
      if (on) d.ml[at] = make_float2(lifted<T, kSlack>(m), l);
      tc_fence_before();  // O has been read: the next item's first PV waits for this half's P
      tiles += n;
      if (n > 0) x += n + 1, ++items;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    if (*fail) {  // whoever gave up: let the products that were issued end before the TMEM goes back
      if (lane == 0) {
        tc_commit(&drained);
        mbar_wait_bounded(&drained, 0, kWaitLimitNs);
      }
      __syncwarp();
    }
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && *fail) {
    atomicOr(&g_prefix_status, kStatusTimeout);
    for (int x = max(s_issued - C::SLOTS, 0); x < s_issued; ++x)  // leave no copy in flight
      mbar_wait_bounded(&full[x % C::SLOTS], (x / C::SLOTS) & 1, kWaitLimitNs);
  }
}

// Whether the kernel was compiled to the launch registers that its split (setmaxnreg) was laid out for. Asked once.
template <typename T, int HD>
bool built() {
  static std::atomic<int> regs{0};
  if (!regs.load(std::memory_order_relaxed)) {
    cudaFuncAttributes f = {};
    if (cudaFuncGetAttributes(&f, prefix_tc_kernel<T, HD>) == cudaSuccess)
      regs.store(f.numRegs, std::memory_order_relaxed);
    else
      cudaGetLastError();
  }
  return regs.load(std::memory_order_relaxed) == kRegsLaunch;
}

template <typename T, int HD>
int launch(const PrefixArgs& a, cudaStream_t st) {
  CUtensorMap tk, tv;
  const int box = page_box(a.kv.page_size, kTcKeys);
  if (int rc = make_tmap_pages(&tk, a.kv, a.kv.k, box)) return rc;
  if (int rc = make_tmap_pages(&tv, a.kv, a.kv.v, box)) return rc;
  auto kern = prefix_tc_kernel<T, HD>;
  static std::atomic<unsigned long long> done;
  const int table = a.tc.own_lo < a.tc.own_hi ? 12 * (a.b.batch + 1) : 0;
  cudaError_t e = set_max_dynamic_smem(kern, TcCfg<HD>::SMEM + 12 * (kTcMaxBatch + 1), done);
  if (e == cudaSuccess) e = launch_pdl(kern, dim3(a.tc_ctas), dim3(kTcThreads), TcCfg<HD>::SMEM + table, st, tk, tv, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(Q4B_ELAUNCH, "prefix_attention: launch failed: %s", cudaGetErrorString(e));
  }
  return Q4B_OK;
}

}  // namespace

// Pages of whole swizzle groups (8 rows), and strides that a tensor map can describe.
bool prefix_tc_takes(const q4b_paged_kv& kv) {
  const bool strides = kv.slot_stride > 0 && (kv.n_kv_heads == 1 || kv.head_stride > 0) && (kv.n_pages == 1 || kv.page_stride > 0);
  return kv.head_dim >= 64 && kv.page_size % 8 == 0 && strides;
}

bool prefix_tc_built(const q4b_paged_kv& kv) {
  const bool h16 = kv.dtype == Q4B_F16;
  if (kv.head_dim == 128) return h16 ? built<__half, 128>() : built<__nv_bfloat16, 128>();
  return h16 ? built<__half, 64>() : built<__nv_bfloat16, 64>();
}

int prefix_tc_run(const PrefixArgs& a, cudaStream_t st) {
  const bool h16 = a.kv.dtype == Q4B_F16;
  if (a.kv.head_dim == 128) return h16 ? launch<__half, 128>(a, st) : launch<__nv_bfloat16, 128>(a, st);
  return h16 ? launch<__half, 64>(a, st) : launch<__nv_bfloat16, 64>(a, st);
}

unsigned prefix_tc_status(bool reset) {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, g_prefix_status, sizeof(v));
  if (reset && v) {
    const unsigned zero = 0;
    cudaMemcpyToSymbol(g_prefix_status, &zero, sizeof(zero));
  }
  return v;
}

}  // namespace q4b
