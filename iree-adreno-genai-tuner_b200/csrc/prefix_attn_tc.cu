// The shared prefix's part of the batched attention on the tcgen05 tensor cores, for steps whose rows fill
// them: all rows of the step and all heads of a KV head's group attend to the same keys, so QK and PV are
// matrix products with M = rows * H / n_kv_heads.
//
//   S = Q K^T * scale;  P = exp2(S log2e - m);  O += P V;  l += sum P       (m: a running reference per row)
//
// One CTA per SM takes 256 query rows (two tiles of 128) of one KV head and a run of 128-key tiles; a row
// tile's keys are split over several CTAs so that the CTAs fill the SMs, and each leaves (m, l) and O in
// fp32 for the join kernel. Warps 0-3 and 4-7 are the softmax of one query tile each, a thread a row; warp 8
// brings K and V tiles by TMA (a box per page, 128-byte swizzle, a ring of tiles); one thread of warp 9 issues
// the MMAs. S and O live in TMEM (2 x 128 + 2 x head_dim columns), and P goes back into S's
// columns as the A operand of the PV product, so nothing but K, V and Q passes through shared memory. The
// two query tiles alternate: while one's softmax runs, the tensor core works for the other, and both use every
// K and V tile that comes in.
//
// m moves only when a row's maximum outgrows it by 2^8, which keeps P below 256 and spares most tiles the pass over
// O; exactness is not affected (l and O carry the same factor). P is rounded to the cache's type, as in
// the other kernel. Bound by the tensor pipe and the exponentials (16 a clock per SM: 256 x 128 of them take as
// long as the tile's two MMAs at their nominal rate).
#include <type_traits>

#include "paged.cuh"
#include "prefix_attn.h"
#include "tc.cuh"

namespace q4b {
namespace {

constexpr int kTcThreads = 320;
constexpr int kTcRows = 128, kTcKeys = 128;
constexpr float kSlack = 8.0f;  // base-2 growth of a row's maximum that its reference tolerates

__device__ unsigned g_prefix_status = 0;

template <int HD>
struct TcCfg {
  static constexpr int HALVES = HD / 64;                   // 64-column (128-byte) halves of a row
  static constexpr int ATOM = kTcKeys * 128;               // one half of a 128-row tile, bytes
  static constexpr int TILE = HALVES * ATOM;               // Q, K or V tile
  static constexpr int SLOTS = HD == 128 ? 5 : 8;          // K and V tiles in flight
  static constexpr int SMEM = (2 + SLOTS) * TILE + 1024;   // + alignment to the swizzle's 1024 bytes
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

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
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, PrefixArgs a) {
  using C = TcCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  __shared__ uint64_t full[C::SLOTS], empty[C::SLOTS], q_full, s_full[2], p_full[2], o_full[2], drained;
  __shared__ uint32_t s_tmem;
  __shared__ int s_fail, s_issued;
  constexpr uint32_t kS = 0, kO = 256;  // TMEM columns: S (and P) of tile i at 128 i, O at 256 + HD i

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // item: KV head, pair of row tiles, run of key tiles
  const int sp = blockIdx.x % a.tc_splits, pair = blockIdx.x / a.tc_splits % a.tc_pairs,
            h = blockIdx.x / a.tc_splits / a.tc_pairs;
  const int j0 = (int)((long long)sp * a.tc_tiles / a.tc_splits), j1 = (int)((long long)(sp + 1) * a.tc_tiles / a.tc_splits);
  const int n = j1 - j0;  // >= 1: there are no more splits than tiles
  const int R = a.rows * a.g, r0 = pair * 2 * kTcRows;
  const int active = R - r0 > kTcRows ? 2 : 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&q_full, active * kTcRows);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kTcRows);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(&drained, 1);
    s_fail = s_issued = 0;
    fence_mbar_init();
    tma_prefetch_map(&tk);
    tma_prefetch_map(&tv);
  }
  if (warp == 9) tmem_alloc(&s_tmem, 512);
  tc_fence_before();
  griddep_wait();
  griddep_launch_dependents();  // behind the wait: what runs next may read the inputs at once
  // pages that do not exist: their keys are masked, which costs lookups, so only where there are any
  const int p0 = j0 * kTcKeys / a.kv.page_size, p1 = (j1 * kTcKeys - 1) / a.kv.page_size + 1;
  bool bad = false;
  for (int p = p0 + (int)threadIdx.x; p < p1; p += kTcThreads) {
    const int page = __ldg(a.prefix_pages + p);
    bad |= page < 0 || page >= a.kv.n_pages;
  }
  bad = __syncthreads_or(bad);
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  volatile int* fail = &s_fail;

  if (warp == 8) {
    // producer: tile n of the ring is K (even) or V (odd) of key tile j0 + n / 2
    const int box = min(a.kv.page_size, kTcKeys), boxes = kTcKeys / box;
    auto page_of = [&](int j) {
      int page = 0;
      if (lane < boxes && j < j1) {
        page = __ldg(a.prefix_pages + (j * kTcKeys + lane * box) / a.kv.page_size);
        if (page < 0 || page >= a.kv.n_pages) page = a.kv.n_pages;  // out of the map: zeros
      }
      return page;
    };
    int page = page_of(j0);
    for (int x = 0; x < 2 * n; ++x) {
      const int s = x % C::SLOTS, r = x / C::SLOTS, j = j0 + (x >> 1);
      bool ok = true;
      if (lane == 0) {
        ok = r == 0 || mbar_wait_bounded(&empty[s], (r - 1) & 1, kWaitLimitNs);
        if (ok) mbar_arrive_expect_tx(&full[s], C::TILE);
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) {
        if (lane == 0) *fail = 1;
        break;
      }
      const int next = x & 1 ? page_of(j + 1) : page;
      if (lane < boxes) {
        const int slot = (j * kTcKeys + lane * box) % a.kv.page_size;
        const uint32_t dst = base + (2 + s) * C::TILE + lane * box * 128;
#pragma unroll
        for (int c = 0; c < C::HALVES; ++c)
          tma_load_4d(dst + c * C::ATOM, x & 1 ? &tv : &tk, 64 * c, slot, h, page, &full[s]);
      }
      page = next;
      if (lane == 0) s_issued = x + 1;
    }
    __syncwarp();
  } else if (warp == 9) {
    if (lane == 0) {
      constexpr uint32_t bf = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
      constexpr uint32_t idesc_s = idesc_f16_f32(kTcRows, kTcKeys, false, false) | bf;
      constexpr uint32_t idesc_o = idesc_f16_f32(kTcRows, HD, false, true) | bf;
      auto slot = [&](int x) { return base + (2 + x % C::SLOTS) * C::TILE; };
      auto wait_full = [&](int x) { return mbar_wait_bounded(&full[x % C::SLOTS], (x / C::SLOTS) & 1, kWaitLimitNs); };
      auto qk = [&](int i, int x) {
        const uint32_t q = base + i * C::TILE, k = slot(x);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = (kk / 4) * C::ATOM + (kk % 4) * 32;
          tc_mma_f16(tmem + kS + 128 * i, sw128_desc(q + off, 16, 1024), sw128_desc(k + off, 16, 1024), idesc_s, kk != 0);
        }
        tc_commit(&s_full[i]);
      };
      auto pv = [&](int i, int x, bool first) {
        const uint32_t v = slot(x);
#pragma unroll
        for (int kk = 0; kk < kTcKeys / 16; ++kk)
          tc_mma_f16_ta(tmem + kO + HD * i, tmem + kS + 128 * i + 8 * kk, sw128_desc(v + kk * 2048, C::ATOM, 1024),
                        idesc_o, !(first && kk == 0));
      };
      bool ok = mbar_wait_bounded(&q_full, 0, kWaitLimitNs) && wait_full(0);
      if (ok) {
        tc_fence_after();
        for (int i = 0; i < active; ++i) qk(i, 0);
        tc_commit(&empty[0]);
      }
      for (int j = 0; ok && j < n; ++j) {
        const int xv = 2 * j + 1, xk = 2 * j + 2;
        ok = wait_full(xv);
        for (int i = 0; ok && i < active; ++i) {
          ok = mbar_wait_bounded(&p_full[i], j & 1, kWaitLimitNs);
          if (ok && i == 0 && j + 1 < n) ok = wait_full(xk);
          if (!ok) break;
          tc_fence_after();
          pv(i, xv, j == 0);
          if (j + 1 < n)
            qk(i, xk);
          else
            tc_commit(&o_full[i]);
        }
        if (ok) {
          tc_commit(&empty[xv % C::SLOTS]);
          if (j + 1 < n) tc_commit(&empty[xk % C::SLOTS]);
        }
      }
      if (!ok) {  // let what was issued end before the TMEM goes back
        *fail = 1;
        tc_commit(&drained);
        mbar_wait_bounded(&drained, 0, kWaitLimitNs);
      }
    }
    __syncwarp();
  } else if (warp / 4 < active) {
    const int i = warp / 4, row = (warp & 3) * 32 + lane, r = r0 + i * kTcRows + row;
    const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + kS + 128 * i;
    const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + kO + HD * i;
    const int t = r / a.g, head = h * a.g + r - t * a.g;
    {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (long long)t * a.q_stride +
                                                        (long long)head * a.q_head_stride);
      uint8_t* dst = smem + i * C::TILE + row * 128;
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) {
        const uint4 v = r < R ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + (c / 8) * C::ATOM + (((c % 8) ^ (row & 7)) << 4)) = v;
      }
      fence_async_smem();
      mbar_arrive(&q_full);
    }
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = mbar_wait_bounded(&s_full[i], j & 1, kWaitLimitNs);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_async(ts + 32 * c, s[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_wait(s[c]);
      if (bad) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int page = __ldg(a.prefix_pages + ((j0 + j) * kTcKeys + 32 * c + lane) / a.kv.page_size);
          const unsigned there = __ballot_sync(0xffffffffu, page >= 0 && page < a.kv.n_pages);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((there >> e) & 1)) s[c][e] = 0xff800000u;
        }
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
        for (int e = 1; e < 32; ++e) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][e]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2;
      if (__any_sync(0xffffffffu, top > m + kSlack || (m == -INFINITY && top > m))) {
        const float nm = fmaxf(m, top), f = m == -INFINITY ? 0.0f : ex2(m - nm);
        m = nm;
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
      const float ref = m == -INFINITY ? 0.0f : m;
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        uint32_t p[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = ex2(fmaf(__uint_as_float(s[c + e / 16][2 * e % 32]), a.scale2, -ref));
          const float y = ex2(fmaf(__uint_as_float(s[c + e / 16][2 * e % 32 + 1]), a.scale2, -ref));
          sum[e & 3] += x + y;
          p[e] = Half16<T>::pack(x, y);
        }
        tmem_st_32(ts + 16 * c, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[i]);
    }
    if (ok) ok = mbar_wait_bounded(&o_full[i], 0, kWaitLimitNs);
    ok = __all_sync(0xffffffffu, ok);
    const long long at = (long long)sp * a.rows * a.H + (long long)t * a.H + head;
    if (ok) {
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tmem_ld_async(to + 32 * c, o);
        tmem_ld_wait(o);
        if (r < R) {
          float4* dst = reinterpret_cast<float4*>(a.tc_o + at * HD + 32 * c);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                                 __uint_as_float(o[4 * e + 3]));
        }
      }
    } else {
      *fail = 1;
      l = __int_as_float(0x7fffffff);  // a row whose work gave up is NaN, not stale
    }
    if (r < R) a.tc_ml[at] = make_float2(m, l);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && *fail) {
    atomicOr(&g_prefix_status, kStatusTimeout);
    for (int x = max(s_issued - C::SLOTS, 0); x < s_issued; ++x)  // leave no copy in flight
      mbar_wait_bounded(&full[x % C::SLOTS], (x / C::SLOTS) & 1, kWaitLimitNs);
  }
}

template <typename T, int HD>
int launch(const PrefixArgs& a, cudaStream_t st) {
  CUtensorMap tk, tv;
  const int box = a.kv.page_size < kTcKeys ? a.kv.page_size : kTcKeys;
  if (int rc = make_tmap_pages(&tk, a.kv, a.kv.k, box)) return rc;
  if (int rc = make_tmap_pages(&tv, a.kv, a.kv.v, box)) return rc;
  auto kern = prefix_tc_kernel<T, HD>;
  static std::atomic<unsigned long long> done;
  cudaError_t e = set_max_dynamic_smem(kern, TcCfg<HD>::SMEM, done);
  if (e == cudaSuccess)
    e = launch_pdl(kern, dim3(a.Hkv * a.tc_pairs * a.tc_splits), dim3(kTcThreads), TcCfg<HD>::SMEM, st, tk, tv, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(Q4B_ELAUNCH, "prefix_attention: launch failed: %s", cudaGetErrorString(e));
  }
  return Q4B_OK;
}

}  // namespace

PrefixTcPlan prefix_tc_plan(int rows, int H, int prefix_len, const q4b_paged_kv& kv) {
  PrefixTcPlan p = {0, 0, 0};
  const int R = rows * (H / kv.n_kv_heads), ps = kv.page_size;
  const int tiles = prefix_len / kTcKeys;
  // Pages that a 128-key tile holds whole, or that hold whole tiles, in boxes of full swizzle groups (8 rows);
  // strides that a tensor map can describe.
  const bool boxes = ps % 8 == 0 && (ps % kTcKeys == 0 || kTcKeys % ps == 0);
  const bool strides = kv.slot_stride > 0 && (kv.n_kv_heads == 1 || kv.head_stride > 0) && (kv.n_pages == 1 || kv.page_stride > 0);
  if (kv.head_dim < 64 || !boxes || !strides || tiles == 0 || R < kTcMinRows) return p;
  p.tiles = tiles;
  p.pairs = (R + 2 * kTcRows - 1) / (2 * kTcRows);
  // Splits: the fewest rounds of (tiles + 3 tiles' worth of start and end) over the SMs.
  const int items = kv.n_kv_heads * p.pairs;
  double best = 0;
  for (int s = 1; s <= tiles && s <= kTcMaxSplits; ++s) {
    const double cost = (double)((items * (long long)s + 147) / 148) * ((tiles + s - 1) / s + 3);
    if (s == 1 || cost < best) best = cost, p.splits = s;
  }
  return p;
}

int prefix_tc_run(const PrefixArgs& a, cudaStream_t st) {
  const bool h16 = a.kv.dtype == Q4B_F16;
  if (a.kv.head_dim == 128) return h16 ? launch<__half, 128>(a, st) : launch<__nv_bfloat16, 128>(a, st);
  return h16 ? launch<__half, 64>(a, st) : launch<__nv_bfloat16, 64>(a, st);
}

unsigned prefix_status(bool reset) {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, g_prefix_status, sizeof(v));
  if (reset && v) {
    const unsigned zero = 0;
    cudaMemcpyToSymbol(g_prefix_status, &zero, sizeof(zero));
  }
  return v;
}

}  // namespace q4b
