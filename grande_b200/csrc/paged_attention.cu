// Attention over a paged K/V cache for groups of sequences that share a
// prefix (see paged.cuh): out = softmax(scale q K^T) V over the prefix keys
// and the sequence's own keys up to the query's position, inside the window.
//
// Three launches. The plan kernel (one CTA) cuts the query tokens into row
// tiles and lays their key tiles on one line (paged.cuh). The attention
// kernel gives every CTA an equal range of the line, whatever it crosses; a
// row tile inside one CTA's range is finished there, one that several CTAs
// cross leaves per CTA an unnormalised O and each row's (max, sum), which the
// merge kernel joins.
//
// Why all rows of a group in one tile: a prefix key is read from HBM once for
// all of them, and an M = 128 tensor-core tile costs 16 clocks per key at
// head_dim 256 however few rows it holds, against the 44 clocks that HBM
// takes to deliver the key's 1 KB to an SM. So a sequence's own keys, which
// only its few rows see, run through the same tile with the other rows'
// accumulator lanes switched off in the MMA: those rows are untouched, also
// by infinities or NaN among another sequence's values.
//
// Roles (192 threads): warp 0 loads Q and the K / V ring through TMA, a box
// per page; warp 1 issues S = Q K^T one tile ahead and O += P V; warps 2-5
// own one query row per thread: mask, online softmax, P, the rescale of O.
//
// Numerics: scores, max, exponentials and sums f32, O accumulated in f32; P
// enters the second product in the cache's 16-bit type (its rounding is of
// the size of the output's own and averages over keys). A row keeps a
// reference max and moves it only when exceeded by 2^11.5 (kTau), so P stays
// in range and O is rarely rescaled.
#include <algorithm>
#include <climits>
#include <cstdio>

#include "gemm.cuh"
#include "launch.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace omg {

namespace {

constexpr int kKeys = kPagedTileKeys;
constexpr int kRows = kPagedTileRows;
constexpr int kQChunk = kRows * 128;   // [128 rows][64 dims]
constexpr int kKvChunk = kKeys * 128;  // [64 keys][64 dims]
constexpr int kPBytes = kRows * kKeys * 2;
constexpr float kTau = 8.0f;           // slack of the reference max, in log2 units x ln 2
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPlanThreads = 1024;

template <int HD>
struct Shape {
  static constexpr int kV = HD < 256 ? HD : 256;    // dims of V and O per CTA
  static constexpr int kHalves = HD / kV;           // CTAs that share a row tile's softmax
  static constexpr int kChunks = kV / 64;           // 64-dim chunks of a ring stage
  static constexpr int kStage = kChunks * kKvChunk; // 64 keys x kV dims
  static constexpr int kQ = HD / 64 * kQChunk;
  static constexpr int kPSlots = 2;
  static constexpr int kCtasPerSm = HD <= 64 ? 2 : 1;
  static constexpr int kStages = HD == 512 ? 2 : HD == 256 ? 4 : HD == 128 ? 8 : 6;
  static constexpr int kTmemO = 128;                // S buffers at columns 0 and 64
  static constexpr uint32_t kTmemCols = HD >= 256 ? 512 : 256;
  static constexpr int kSmem = 1024 + kQ + kStages * kStage + kPSlots * kPBytes + 512;
};

// ---- plan -------------------------------------------------------------------

struct PlanSmem {
  int *gs, *gtok, *gtile;                // [groups + 1]: first sequence, token, row tile
  int *imin, *imax, *own, *seg0, *seg1;  // [max_tiles]
  int* cnt;                              // [max_segs] line tiles of each segment
};

__host__ __device__ inline size_t plan_smem_ints(int groups, int max_tiles, int max_segs) {
  return 3 * (static_cast<size_t>(groups) + 1) + 5 * static_cast<size_t>(max_tiles) + max_segs;
}

// Exclusive scan of v over the block, plus `carry`; returns the block's total.
__device__ __forceinline__ int block_scan(int v, int* excl) {
  __shared__ int ws[32];
  __shared__ int total;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) ws[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = ws[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    if (lane == 31) total = w;
    ws[lane] = w;
  }
  __syncthreads();
  *excl = x - v + (warp ? ws[warp - 1] : 0);
  const int t = total;
  __syncthreads();
  return t;
}

// Largest i with a[i] <= v in the ascending a[0..n), -1: none (shared memory).
__device__ __forceinline__ int last_le(const int* a, int n, int v) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo - 1;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedAttnArgs a) {
  extern __shared__ int sm[];
  const int groups = max(a.b.n_groups, 1), S = a.b.n_seqs, T = a.b.tokens;
  PlanSmem m;
  m.gs = sm;
  m.gtok = m.gs + groups + 1;
  m.gtile = m.gtok + groups + 1;
  m.imin = m.gtile + groups + 1;
  m.imax = m.imin + a.max_tiles;
  m.own = m.imax + a.max_tiles;
  m.seg0 = m.own + a.max_tiles;
  m.seg1 = m.seg0 + a.max_tiles;
  m.cnt = m.seg1 + a.max_tiles;
  const int tid = threadIdx.x;
  griddep_wait();
  griddep_launch();

  // Groups: first sequence and token, clipped to what exists.
  for (int g = tid; g <= groups; g += kPlanThreads) {
    int s = a.b.n_groups > 0 ? a.b.group_start[g] : g * S;
    s = min(max(s, 0), S);
    m.gs[g] = s;
    m.gtok[g] = min(max(a.b.q_start[s], 0), T);
  }
  for (int i = tid; i < a.max_segs; i += kPlanThreads) {
    m.cnt[i] = 0;
    a.segs[i].rows = 0;
  }
  for (int i = tid; i < a.max_tiles; i += kPlanThreads) {
    m.imin[i] = INT_MAX;
    m.imax[i] = INT_MIN;
    m.own[i] = 0;
    m.seg0[i] = INT_MAX;
    m.seg1[i] = -1;
  }
  __syncthreads();
  int n_tiles = 0;
  for (int g0 = 0; g0 < groups; g0 += kPlanThreads) {
    const int g = g0 + tid;
    const int n = g < groups ? (max(m.gtok[g + 1] - m.gtok[g], 0) + a.tpt - 1) / a.tpt : 0;
    int at;
    const int total = block_scan(n, &at);
    if (g < groups) m.gtile[g] = n_tiles + at;
    n_tiles += total;
  }
  n_tiles = min(n_tiles, a.max_tiles);  // only tables out of order make more
  if (tid == 0) m.gtile[groups] = n_tiles;
  __syncthreads();

  // (sequence, row tile) pairs.
  const int own_cap = a.b.max_pages << a.c.page_log2;
  for (int s = tid; s < S; s += kPlanThreads) {
    const int g = last_le(m.gs, groups + 1, s);
    if (g < 0 || g >= groups) continue;
    const int q0 = max(a.b.q_start[s], m.gtok[g]);
    const int q1 = min(a.b.q_start[s + 1], m.gtok[g + 1]);
    if (q0 >= q1) continue;
    const int len = a.b.lens[s];
    const int first = len - (a.b.q_start[s + 1] - q0);  // own index of token q0
    for (int k = (q0 - m.gtok[g]) / a.tpt; k <= (q1 - 1 - m.gtok[g]) / a.tpt; ++k) {
      const int rt = m.gtile[g] + k;
      const int t0 = m.gtok[g] + k * a.tpt;
      if (rt >= n_tiles) break;
      const int ta = max(q0, t0), tb = min(q1, t0 + a.tpt);
      const int i0 = first + (ta - q0), i1 = i0 + (tb - ta) - 1;
      PagedSeg sg;
      sg.s = s;
      sg.rt = rt;
      sg.rows = ((ta - t0) * a.hpg) | (((tb - t0) * a.hpg) << 16);
      sg.i0 = i0;
      sg.kend = min(i1 + 1, own_cap);
      const int lo = a.window > 0 ? max(0, i0 - a.window + 1) : 0;
      sg.own0 = lo / kKeys;
      sg.n_own = max(0, (sg.kend + kKeys - 1) / kKeys - sg.own0);
      if (sg.kend <= lo) sg.n_own = 0;
      sg.pad = 0;
      const int at = s + rt;
      a.segs[at] = sg;
      m.cnt[at] = sg.n_own;
      atomicMin(&m.imin[rt], i0);
      atomicMax(&m.imax[rt], i1);
      atomicAdd(&m.own[rt], sg.n_own);
      atomicMin(&m.seg0[rt], at);
      atomicMax(&m.seg1[rt], at);
    }
  }
  __syncthreads();

  // Row tiles: the prefix's key tiles come before the first segment's own.
  const int pre_cap = a.b.n_groups > 0 ? a.b.max_prefix_pages << a.c.page_log2 : 0;
  for (int rt = tid; rt < n_tiles; rt += kPlanThreads) {
    const int g = last_le(m.gtile, groups, rt);
    PagedTile t;
    t.tok0 = m.gtok[g] + (rt - m.gtile[g]) * a.tpt;
    t.ntok = min(a.tpt, m.gtok[g + 1] - t.tok0);
    t.group = g;
    t.prefix_len = a.b.n_groups > 0 ? max(a.b.prefix_lens[g], 0) : 0;
    t.seg0 = m.seg0[rt];
    t.nseg = m.seg1[rt] - m.seg0[rt] + 1;
    t.imin = m.imin[rt];
    t.imax = m.imax[rt];
    t.pre0 = t.npre = t.cum = t.ntiles = 0;
    if (m.seg1[rt] >= 0) {
      const int end = min(t.prefix_len, pre_cap);
      const int lo = a.window > 0 ? max(0, t.prefix_len + t.imin - a.window + 1) : 0;
      if (lo < end) {
        t.pre0 = lo / kKeys;
        t.npre = (end + kKeys - 1) / kKeys - t.pre0;
      }
      // Rows that see nothing at all still get their zeros: one key tile,
      // all of it masked.
      if (t.npre + m.own[rt] == 0) t.npre = 1;
      t.ntiles = t.npre + m.own[rt];
      m.cnt[t.seg0] += t.npre;
    }
    a.tiles[rt] = t;
  }
  __syncthreads();

  const int n_segs = S + n_tiles;
  int line = 0;
  for (int i0 = 0; i0 < n_segs; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int at;
    const int total = block_scan(i < n_segs ? m.cnt[i] : 0, &at);
    if (i < n_segs) {
      a.seg_cum[i] = line + at;
      const int rt = a.segs[i].rows ? a.segs[i].rt : -1;
      if (rt >= 0 && m.seg0[rt] == i) a.tiles[rt].cum = line + at;
    }
    line += total;
  }
  if (tid == 0) {
    a.seg_cum[n_segs] = line;
    *a.plan = PagedPlan{n_tiles, n_segs, line, 0};
  }
}

// ---- attention ----------------------------------------------------------------

// A position on the line, walked tile by tile by each role.
struct Walk {
  PagedTile t;   // row tile
  PagedSeg sg;   // segment whose own keys come next or are being read
  int kv, rt;    // KV head, row tile
  int pos, end;  // tile of the row tile, and where this CTA's range leaves it
  int seg, sub;  // segment index; own tile within it

  __device__ __forceinline__ void load_seg(const PagedAttnArgs& a) {
    while (a.segs[seg].rows == 0 || a.segs[seg].n_own == 0) {
      if (seg + 1 >= t.seg0 + t.nseg) break;
      ++seg;
    }
    sg = a.segs[seg];
  }
  // Enter the line at tile w of [w, w1); a full warp calls it.
  __device__ __forceinline__ void enter(const PagedAttnArgs& a, const PagedPlan& p, int w, int w1,
                                        int lane) {
    kv = w / p.line;
    const int wl = w - kv * p.line;
    seg = warp_count_le(a.seg_cum, p.n_segs, wl, lane) - 1;
    rt = a.segs[seg].rt;
    t = a.tiles[rt];
    pos = wl - t.cum;
    end = min(t.ntiles, pos + (w1 - w));
    if (pos < t.npre) {
      seg = t.seg0;
      sub = 0;
    } else {
      sub = wl - a.seg_cum[seg] - (seg == t.seg0 ? t.npre : 0);
    }
    load_seg(a);
  }
  __device__ __forceinline__ bool prefix() const { return pos < t.npre; }
  // Key tile number in its list of pages.
  __device__ __forceinline__ int key_tile() const {
    return prefix() ? t.pre0 + pos : sg.own0 + sub;
  }
  __device__ __forceinline__ void next(const PagedAttnArgs& a) {
    if (!prefix()) {
      if (++sub == sg.n_own && pos + 1 < t.ntiles) {
        ++seg;
        sub = 0;
        load_seg(a);
      }
    }
    ++pos;
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bits [a, b) of a 64-bit set, clipped to it.
__device__ __forceinline__ uint64_t bits_between(int a, int b) {
  a = min(max(a, 0), 64);
  b = min(max(b, 0), 64);
  if (a >= b) return 0;
  const uint64_t hi = b >= 64 ? ~0ull : (1ull << b) - 1;
  return hi & ~((1ull << a) - 1);
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          int lane) {
  int ok = 0;
  if (lane == 0) ok = mbar_wait(bar, parity, abort_flag, nullptr) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <class T>
__device__ __forceinline__ float to_float(uint16_t bits) {
  if constexpr (std::is_same<T, __half>::value)
    return __half2float(__ushort_as_half(bits));
  else
    return __bfloat162float(__ushort_as_bfloat16(bits));
}
// Does a pair of 16-bit values hold an infinity or a NaN?
template <class T>
__device__ __forceinline__ bool nonfinite2(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w >> 16 & e) == e;
}

// B_CLEAN: the softmax warps have looked through a partly seen V tile.
enum { B_Q = 0, B_QFREE, B_S0, B_S1, B_P0, B_P1, B_O0, B_O1, B_CLEAN, B_DRAIN, B_RING };
constexpr long long kDrainClocks = 1ll << 28;

template <int HD, class T>
__global__ void __launch_bounds__(192, Shape<HD>::kCtasPerSm)
    paged_attention_kernel(const __grid_constant__ CUtensorMap tq,
                           const __grid_constant__ CUtensorMap tkv, PagedAttnArgs a) {
  using Sh = Shape<HD>;
  constexpr int VD = Sh::kV, NST = Sh::kStages, CH = Sh::kChunks;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* qs = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ring = qs + Sh::kQ;
  uint8_t* ps = ring + NST * Sh::kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ps + Sh::kPSlots * kPBytes);
  // K stages and V tiles land on barriers of their own, in the order of their
  // own counts: a softmax warp waits for V tiles only, and a count that it
  // could fall two phases behind would read as done.
  uint64_t* kfull = bars + B_RING;
  uint64_t* vfull = kfull + NST;
  uint64_t* empty = vfull + NST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(empty + NST);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // [tile & 3][2]: a tile's keys with infinities or NaN in V. Four sets: a
  // warp can be two tiles ahead of the one that clears a set.
  uint32_t* bad_keys = tmem_slot + 2;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int vhalf = blockIdx.y;  // this CTA's dims of V (head_dim 512)

  if (threadIdx.x == 0) {
    for (int i = 0; i < B_RING; ++i) mbar_init(&bars[i], (i == B_P0 || i == B_P1 || i == B_CLEAN) ? 4 : 1);
    for (int i = 0; i < 3 * NST; ++i) mbar_init(&kfull[i], 1);
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) bad_keys[i] = 0;
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tkv);
  }
  if (warp == 1) tmem_alloc(tmem_slot, Sh::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch();

  const PagedPlan plan = *a.plan;
  const int total = plan.line * a.c.kv_heads;
  const int per = max((total + a.ctas - 1) / a.ctas, a.min_tiles);
  const int w0 = min(static_cast<int>(blockIdx.x) * per, total);
  const int w1 = min(w0 + per, total);
  const int pre_cap = a.b.n_groups > 0 ? a.b.max_prefix_pages << a.c.page_log2 : 0;
  constexpr int KST = Sh::kHalves;  // ring stages of a K tile (V: one)

  if (warp == 0) {
    // ---- loads: Q of each row tile; per tile K then, one tile behind, V.
    const int box = min(1 << a.c.page_log2, kKeys);  // rows per TMA box
    const int nbox = kKeys / box;
    const int lb = lane % nbox, lc = lane / nbox;
    int it = 0, nk = 0, nv = 0, nq = 0;
    bool ok = true;
    // First cache row of this lane's box of the walk's tile (-1: past the
    // keys that exist, nothing to load; a page outside the pool lies past
    // the map's end, where TMA fills zeros).
    auto box_row = [&](const Walk& w) -> int {
      const int key = w.key_tile() * kKeys + lb * box;
      const bool pre = w.prefix();
      const int kend = pre ? min(w.t.prefix_len, pre_cap) : w.sg.kend;
      if (key >= kend) return -1;
      const int pi = key >> a.c.page_log2;
      const int* table =
          pre ? a.b.prefix_pages + static_cast<int64_t>(w.t.group) * a.b.max_prefix_pages
              : a.b.pages + static_cast<int64_t>(w.sg.s) * a.b.max_pages;
      int page = table[pi];
      if (page < 0 || page >= a.c.n_pages) page = static_cast<int>(a.c.n_pages);
      return (page << a.c.page_log2) + (key & ((1 << a.c.page_log2) - 1));
    };
    // One ring stage: dims [x, x + kV) of the tile's keys.
    auto load_stage = [&](int row, int x, bool is_v) {
      const int s = it % NST, n = it / NST;
      if (n > 0 && !warp_wait(&empty[s], (n - 1) & 1, abort_flag, lane)) {
        ok = false;
        return;
      }
      ++it;
      uint64_t* full = is_v ? &vfull[nv++ % NST] : &kfull[nk++ % NST];
      const uint32_t live = __popc(__ballot_sync(0xffffffffu, row >= 0 && lc < CH));
      if (lane == 0) mbar_arrive_expect_tx(full, live * box * 128);
      __syncwarp();
      if (row >= 0 && lc < CH)
        tma_load_2d(ring + s * Sh::kStage + lc * kKvChunk + lb * box * 128, &tkv, full,
                    x + lc * 64, row);
    };
    for (int w = w0; w < w1 && ok;) {
      Walk wk;
      wk.enter(a, plan, w, w1, lane);
      if (nq > 0 && !warp_wait(&bars[B_QFREE], (nq - 1) & 1, abort_flag, lane)) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars[B_Q], HD * 2u * static_cast<uint32_t>(a.hpg * a.tpt));
#pragma unroll 1
        for (int c = 0; c < HD / 64; ++c)
          tma_load_4d(qs + c * kQChunk, &tq, &bars[B_Q], c * 64, 0, wk.kv, wk.t.tok0);
      }
      __syncwarp();
      ++nq;
      const int n = wk.end - wk.pos;
      const int kx = wk.kv * HD, vx = (a.c.kv_heads + wk.kv) * HD + vhalf * VD;
      int row = box_row(wk);
      for (int u = 0; u < KST && ok; ++u) load_stage(row, kx + u * VD, false);
      for (int j = 0; j < n && ok; ++j) {
        int ahead = -1;
        if (j + 1 < n) {
          wk.next(a);
          ahead = box_row(wk);
          for (int u = 0; u < KST && ok; ++u) load_stage(ahead, kx + u * VD, false);
        }
        if (ok) load_stage(row, vx, true);
        row = ahead;
      }
      w += n;
    }
    if (*abort_flag && lane == 0) {
      // Gave up: wait (bounded) for the copies in flight into this CTA.
      for (int i = max(0, nk - NST); i < nk; ++i)
        mbar_drain(&kfull[i % NST], (i / NST) & 1, kDrainClocks);
      for (int i = max(0, nv - NST); i < nv; ++i)
        mbar_drain(&vfull[i % NST], (i / NST) & 1, kDrainClocks);
      if (nq > 0) mbar_drain(&bars[B_Q], (nq - 1) & 1, kDrainClocks);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMA issue.
    constexpr uint32_t fs = idesc_f16_f32(kRows, kKeys), fo = idesc_f16_f32_bmn(kRows, VD);
    constexpr bool f16 = std::is_same<T, __half>::value;
    constexpr uint32_t idesc_s = f16 ? fs : idesc_bf16(fs);
    constexpr uint32_t idesc_o = f16 ? fo : idesc_bf16(fo);
    int it = 0, nk = 0, jt = 0, nq = 0;
    bool ok = true;
    for (int w = w0; w < w1 && ok;) {
      Walk wk;
      wk.enter(a, plan, w, w1, lane);
      const int n = wk.end - wk.pos;
      if (lane == 0) {
        auto issue_s = [&](int j) -> bool {
          const int b = (jt + j) & 1;
#pragma unroll 1
          for (int u = 0; u < KST; ++u, ++it, ++nk) {
            const int s = it % NST;
            if (!mbar_wait(&kfull[nk % NST], (nk / NST) & 1, abort_flag, nullptr)) return false;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < CH; ++c) {
              const uint64_t da = sw128_desc(qs + (u * CH + c) * kQChunk);
              const uint64_t db = sw128_desc(ring + s * Sh::kStage + c * kKvChunk);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16(tmem + b * kKeys, da + 2 * k, db + 2 * k, idesc_s, (u | c | k) ? 1u : 0u);
            }
            umma_commit(&empty[s]);
          }
          umma_commit(&bars[B_S0 + b]);
          if (j + 1 == n) umma_commit(&bars[B_QFREE]);
          return true;
        };
        ok = mbar_wait(&bars[B_Q], nq & 1, abort_flag, nullptr) && issue_s(0);
        for (int j = 0; ok && j < n; ++j) {
          // S one tile ahead; its buffer's last reader finished before the P
          // of two tiles back, waited for below.
          if (j + 1 < n && !issue_s(j + 1)) {
            ok = false;
            break;
          }
          const int g = jt + j, b = g & 1;
          const int s = it % NST;
          if (!mbar_wait(&bars[B_P0 + b], (g >> 1) & 1, abort_flag, nullptr) ||
              !mbar_wait(&vfull[g % NST], (g / NST) & 1, abort_flag, nullptr)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t off[4] = {0, 0, 0, 0};
          if (!wk.prefix()) {
            const int r0 = wk.sg.rows & 0xffff, r1 = wk.sg.rows >> 16;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              off[i] = ~static_cast<uint32_t>(bits_between(r0 - 32 * i, min(r1 - 32 * i, 32)));
          }
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk) {
            const uint64_t pa = sw128_desc(ps + b * kPBytes) + 2 * kk;
            const uint64_t vb = sw128_mn_desc(ring + s * Sh::kStage + kk * 2048, kKvChunk);
            umma_f16_lanes(tmem + Sh::kTmemO, pa, vb, idesc_o, 1u, off);
          }
          umma_commit(&bars[B_O0 + b]);
          umma_commit(&empty[s]);
          ++it;
          if (j + 1 < n) wk.next(a);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      ++nq;
      jt += n;
      w += n;
    }
    if (!ok && lane == 0) {
      // Gave up: let the MMAs in flight finish (bounded).
      umma_commit(&bars[B_DRAIN]);
      mbar_drain(&bars[B_DRAIN], 0, kDrainClocks);
    }
    __syncwarp();
  } else {
    // ---- softmax: one query row per thread, its TMEM lane.
    const int q4 = warp & 3;
    const int r = 32 * q4 + lane;
    const int tid = threadIdx.x - 64;
    const uint32_t trow = tmem + (static_cast<uint32_t>(32 * q4) << 16);
    uint8_t* my_stage[2] = {ps + 32 * q4 * 128, ps + kPBytes + 32 * q4 * 128};
    int it = 0, jt = 0, cleans = 0;
    bool ok = true;
    // All four softmax warps meet (a bounded wait, unlike a named barrier).
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[B_CLEAN]);
      return warp_wait(&bars[B_CLEAN], cleans++ & 1, abort_flag, lane);
    };
    for (int w = w0; w < w1;) {
      Walk wk;
      wk.enter(a, plan, w, w1, lane);
      const int n = wk.end - wk.pos;
      const int nrows = wk.t.ntok * a.hpg;
      const bool whole = n == wk.t.ntiles;
      // The row's own index, from its sequence's segment.
      int own = INT_MIN / 2;
      const bool valid = r < nrows;
      for (int i = wk.t.seg0; i < wk.t.seg0 + wk.t.nseg; ++i) {
        const int rows = a.segs[i].rows, i0 = a.segs[i].i0;
        const int r0 = rows & 0xffff;
        if (valid && r >= r0 && r < (rows >> 16)) own = i0 + (r - r0) / a.hpg;
      }
      const int nstart = it;
      float m_ref = -INFINITY, l = 0.f;
      if (ok && 32 * q4 < nrows) {
        // O starts from zero: an own tile only ever touches its rows' lanes.
        uint32_t z[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) z[e] = 0;
#pragma unroll 1
        for (int c = 0; c < VD / 32; ++c) tmem_st32(trow + Sh::kTmemO + c * 32, z);
        tmem_st_wait();
      }
      for (int j = 0; ok && j < n; ++j) {
        const int g = jt + j, b = g & 1;
        const bool pre = wk.prefix();
        const int k0 = wk.key_tile() * kKeys;
        const int r0 = pre ? 0 : wk.sg.rows & 0xffff, r1 = pre ? nrows : wk.sg.rows >> 16;
        const bool mine = r >= r0 && r < r1;
        // The row's keys of this tile; those of the tile's first and last
        // row bound what any and what all of its rows see.
        const int plen = wk.t.prefix_len;
        const int cap = pre ? min(plen, pre_cap) : wk.sg.kend;
        const int shift = pre ? plen : 0;
        const int ifirst = pre ? wk.t.imin : wk.sg.i0;
        const int ilast = pre ? wk.t.imax : wk.sg.i0 + (r1 - r0) / a.hpg - 1;
        auto sees = [&](int i) -> uint64_t {
          const int p = shift + i;
          return bits_between((a.window > 0 ? p - a.window + 1 : 0) - k0, min(p + 1, cap) - k0);
        };
        const uint64_t vis = mine ? sees(own) : 0;
        const uint64_t any =
            bits_between((a.window > 0 ? shift + ifirst - a.window + 1 : 0) - k0,
                         min(shift + ilast + 1, cap) - k0);
        const uint64_t all =
            bits_between((a.window > 0 ? shift + ilast - a.window + 1 : 0) - k0,
                         min(shift + ifirst + 1, cap) - k0);
        // FIFO place of this tile's V: K of tile j + 1 was loaded before it.
        const int vi = nstart + (j + 1 < n ? 2 * KST + j * (KST + 1) : n * (KST + 1) - 1);
        if (!warp_wait(&bars[B_S0 + b], (g >> 1) & 1, abort_flag, lane)) {
          ok = false;
          break;
        }
        uint64_t bad = 0;
        if (any != ~0ull || all != ~0ull) {
          // Keys that no row sees may hold anything: their V rows become
          // zeros. Of those that only some rows see, V rows with infinities
          // or NaN are taken out of the product and added by hand to the rows
          // that see them, so that a masked key never reaches a row.
          uint8_t* v = ring + (vi % NST) * Sh::kStage;
          if (!warp_wait(&vfull[g % NST], (g / NST) & 1, abort_flag, lane)) {
            ok = false;
            break;
          }
          const uint64_t part = any & ~all;
          for (int i = tid; i < kKeys * CH * 8; i += 128) {
            const int key = (i >> 3) & (kKeys - 1), chunk = i >> 9;
            uint4* p = reinterpret_cast<uint4*>(v + chunk * kKvChunk + key * 128 + (i & 7) * 16);
            if (!((any >> key) & 1)) {
              *p = make_uint4(0, 0, 0, 0);
            } else if ((part >> key) & 1) {
              const uint4 x = *p;
              if (nonfinite2<T>(x.x) || nonfinite2<T>(x.y) || nonfinite2<T>(x.z) ||
                  nonfinite2<T>(x.w))
                atomicOr(&bad_keys[2 * (g & 3) + (key >> 5)], 1u << (key & 31));
            }
          }
          if (part) {
            if (!meet()) {
              ok = false;
              break;
            }
            const volatile uint32_t* bk = bad_keys + 2 * (g & 3);
            bad = static_cast<uint64_t>(bk[0]) | (static_cast<uint64_t>(bk[1]) << 32);
          }
          if (bad) {
            for (int i = tid; i < kKeys * CH * 8; i += 128) {
              const int key = (i >> 3) & (kKeys - 1), chunk = i >> 9;
              if ((bad >> key) & 1)
                *reinterpret_cast<uint4*>(v + chunk * kKvChunk + key * 128 + (i & 7) * 16) =
                    make_uint4(0, 0, 0, 0);
            }
            if (!meet()) {
              ok = false;
              break;
            }
            if (tid < 2) bad_keys[2 * (g & 3) + tid] = 0;
          }
        }
        const bool active = __any_sync(0xffffffffu, vis != 0);
        uint8_t* pj = ps + b * kPBytes;
        if (active || (32 * q4 < r1 && 32 * q4 + 32 > r0)) {
          tc_fence_after();
          float s[kKeys];
          {
            uint32_t raw0[32], raw1[32];
            tmem_ld32_nowait(trow + b * kKeys, raw0);
            tmem_ld32_nowait(trow + b * kKeys + 32, raw1);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              s[c] = __uint_as_float(raw0[c]);
              s[32 + c] = __uint_as_float(raw1[c]);
            }
          }
          if (__any_sync(0xffffffffu, vis != ~0ull)) {
            const uint32_t vlo = static_cast<uint32_t>(vis), vhi = static_cast<uint32_t>(vis >> 32);
#pragma unroll
            for (int c = 0; c < kKeys; ++c) {
              const uint32_t m = c < 32 ? vlo : vhi;
              s[c] = ((m >> (c & 31)) & 1u) ? s[c] : -INFINITY;
            }
          }
          float mx[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) mx[e] = s[e];
#pragma unroll
          for (int c = 8; c < kKeys; ++c) mx[c & 7] = fmaxf(mx[c & 7], s[c]);
          const float mt = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                                 fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) *
                           a.scale_log2;
          float alpha = 1.f;
          bool rescale = false;
          if (mt > m_ref + kTau * kLog2e) {
            rescale = m_ref != -INFINITY;
            alpha = rescale ? exp2_fast(m_ref - mt) : 0.f;
            m_ref = mt;
          }
          float sum = 0.f;
          if (m_ref == -INFINITY) {
            // Nothing seen so far. A NaN score (fmaxf drops it) still counts.
#pragma unroll
            for (int c = 0; c < kKeys; ++c) {
              s[c] = s[c] != s[c] ? s[c] : 0.f;
              sum += s[c];
            }
          } else {
            float psum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < kKeys; ++c) {
              s[c] = exp2_fast(fmaf(s[c], a.scale_log2, -m_ref));
              psum[c & 7] += s[c];
            }
            sum = ((psum[0] + psum[1]) + (psum[2] + psum[3])) +
                  ((psum[4] + psum[5]) + (psum[6] + psum[7]));
          }
          l = l * alpha + sum;
          const bool any_rescale = __any_sync(0xffffffffu, rescale);
          // Rescaling O needs the P V before this one done; slot b was read by
          // the one before that.
          if (j > 0 && any_rescale) {
            if (!warp_wait(&bars[B_O0 + ((g - 1) & 1)], ((g - 1) >> 1) & 1, abort_flag, lane)) {
              ok = false;
              break;
            }
          }
          if (j > 1) {
            if (!warp_wait(&bars[B_O0 + b], ((g - 2) >> 1) & 1, abort_flag, lane)) {
              ok = false;
              break;
            }
          }
          if (any_rescale) {
            tc_fence_after();
            const float f = rescale ? alpha : 1.0f;
#pragma unroll 1
            for (int c = 0; c < VD / 32; ++c) {
              uint32_t o[32];
              tmem_ld32_nowait(trow + Sh::kTmemO + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(trow + Sh::kTmemO + c * 32, o);
            }
            tmem_st_wait();
          }
#pragma unroll
          for (int pw = 0; pw < kKeys / 8; ++pw) {
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = pack2<T>(s[pw * 8 + 2 * e], s[pw * 8 + 2 * e + 1]);
            *reinterpret_cast<uint4*>(pj + r * 128 + ((pw ^ (r & 7)) << 4)) =
                make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
        fence_proxy_async();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[B_P0 + b]);
        if (bad) {
          // The taken-out keys, for the rows that see them.
          if (!warp_wait(&bars[B_O0 + b], (g >> 1) & 1, abort_flag, lane)) {
            ok = false;
            break;
          }
          if (__any_sync(0xffffffffu, (vis & bad) != 0)) {
            tc_fence_after();
            for (uint64_t todo = bad; todo; todo &= todo - 1) {
              const int key = __ffsll(static_cast<long long>(todo)) - 1;
              const int pi = (k0 + key) >> a.c.page_log2;
              const int page =
                  pre ? a.b.prefix_pages[static_cast<int64_t>(wk.t.group) * a.b.max_prefix_pages + pi]
                      : a.b.pages[static_cast<int64_t>(wk.sg.s) * a.b.max_pages + pi];
              const int64_t row = (static_cast<int64_t>(page) << a.c.page_log2) +
                                  ((k0 + key) & ((1 << a.c.page_log2) - 1));
              const uint16_t* vrow = static_cast<const uint16_t*>(a.c.rows) +
                                     (row * 2 * a.c.kv_heads + a.c.kv_heads + wk.kv) * HD +
                                     vhalf * VD;
              const bool add = (vis >> key) & 1;
              const float p = to_float<T>(*reinterpret_cast<const uint16_t*>(
                  pj + r * 128 + (((key >> 3) ^ (r & 7)) << 4) + (key & 7) * 2));
#pragma unroll 1
              for (int c = 0; c < VD / 32; ++c) {
                uint32_t o[32];
                tmem_ld32_nowait(trow + Sh::kTmemO + c * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (add)
                    o[e] = __float_as_uint(
                        fmaf(p, to_float<T>(vrow[c * 32 + e]), __uint_as_float(o[e])));
                tmem_st32(trow + Sh::kTmemO + c * 32, o);
              }
              tmem_st_wait();
            }
            tc_fence_before();
          }
        }
        if (j + 1 < n) wk.next(a);
      }
      it += n * (KST + 1);
      jt += n;
      // O of the row tile, or this range's share of it.
      if (ok && !warp_wait(&bars[B_O0 + ((jt - 1) & 1)], ((jt - 1) >> 1) & 1, abort_flag, lane))
        ok = false;
      tc_fence_after();
      const bool first = w == w0;
      const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (first ? 0 : 1);
      float keep = 0.f;
      if (whole) {
        keep = l > 0.f ? 1.0f / l : 0.f;
        if (l != l) keep = l;
        if (!ok) keep = NAN;  // a wait ran out: no row passes for a result
      } else {
        keep = 1.f;
        if (vhalf == 0 && valid)
          a.part_ml[slot * kRows + r] = ok ? make_float2(m_ref, l) : make_float2(NAN, NAN);
      }
      const bool used = valid && (whole || l != 0.f || !ok);
      if (__any_sync(0xffffffffu, used)) {
        const int rows_here = min(32, nrows - 32 * q4);
        // Through the warp's rows of the P slots, whose products are done:
        // 128 bytes of each row at a time, then whole rows of it to memory.
        if (whole) {
          constexpr int kPass = 64;  // 16-bit values of 128 bytes
#pragma unroll 1
          for (int c = 0; c < VD / kPass; ++c) {
            uint8_t* st = my_stage[c & 1];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              float o[32];
              tmem_ld32(trow + Sh::kTmemO + c * kPass + hh * 32, o);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t h[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const float x = o[8 * e + 2 * q], y = o[8 * e + 2 * q + 1];
                  h[q] = pack2<T>(l == 0.f && ok ? 0.f : x * keep, l == 0.f && ok ? 0.f : y * keep);
                }
                *reinterpret_cast<uint4*>(st + lane * 128 + (((4 * hh + e) ^ (lane & 7)) << 4)) =
                    make_uint4(h[0], h[1], h[2], h[3]);
              }
            }
            __syncwarp();
#pragma unroll 1
            for (int i = lane >> 3; i < rows_here; i += 4) {
              const uint4 v =
                  *reinterpret_cast<const uint4*>(st + i * 128 + (((lane & 7) ^ (i & 7)) << 4));
              const int row = 32 * q4 + i, tok = row / a.hpg;
              T* o = static_cast<T*>(a.out) + (wk.t.tok0 + tok) * a.out_stride +
                     (wk.kv * a.hpg + row - tok * a.hpg) * HD + vhalf * VD + c * kPass;
              reinterpret_cast<uint4*>(o)[lane & 7] = v;
            }
            __syncwarp();
          }
        } else {
          const uint32_t live = __ballot_sync(0xffffffffu, used);
          float* po = a.part_o + slot * kRows * HD + vhalf * VD;
#pragma unroll 1
          for (int c = 0; c < VD / 32; ++c) {
            uint8_t* st = my_stage[c & 1];
            float o[32];
            tmem_ld32(trow + Sh::kTmemO + c * 32, o);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(st + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                  make_uint4(__float_as_uint(o[4 * e]), __float_as_uint(o[4 * e + 1]),
                             __float_as_uint(o[4 * e + 2]), __float_as_uint(o[4 * e + 3]));
            __syncwarp();
#pragma unroll 1
            for (int i = lane >> 3; i < rows_here; i += 4) {
              if (!((live >> i) & 1)) continue;
              const uint4 v =
                  *reinterpret_cast<const uint4*>(st + i * 128 + (((lane & 7) ^ (i & 7)) << 4));
              reinterpret_cast<uint4*>(po + static_cast<size_t>(32 * q4 + i) * HD + c * 32)[lane & 7] =
                  v;
            }
            __syncwarp();
          }
        }
      }
      tc_fence_before();
      w += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kTmemCols);
  }
}

// ---- merge ----------------------------------------------------------------------

// A block takes the row tile that the boundary between CTA i - 1 and i cuts
// first (later boundaries of the same tile leave), and of it the rows of its
// row group. A warp per row and 128 dims (64 at head_dim 64).
constexpr int kMergeWarps = 8;

template <int HD, class T>
__global__ void __launch_bounds__(32 * kMergeWarps) paged_merge_kernel(PagedAttnArgs a) {
  constexpr int kPer = HD < 128 ? HD : 128;       // dims per warp
  constexpr int kRowWarps = HD / kPer;            // warps per row
  constexpr int kRowsHere = kMergeWarps / kRowWarps;
  constexpr int kLane = kPer / 32;                // dims per lane
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedPlan plan = *a.plan;
  const int total = plan.line * a.c.kv_heads;
  const int per = max((total + a.ctas - 1) / a.ctas, a.min_tiles);
  const int i = blockIdx.x + 1;
  const int w = i * per;
  if (w >= total) return;
  const int kv = w / plan.line, wl = w - kv * plan.line;
  const int seg = warp_count_le(a.seg_cum, plan.n_segs, wl, lane) - 1;
  const PagedTile t = a.tiles[a.segs[seg].rt];
  const int e0 = kv * plan.line + t.cum;
  if (e0 == w || (i - 1) * per > e0) return;
  const int c0 = i - 1, c1 = (e0 + t.ntiles - 1) / per;
  const int r = blockIdx.y * kRowsHere + warp / kRowWarps;
  if (r >= t.ntok * a.hpg) return;
  const int d0 = (warp % kRowWarps) * kPer + lane * kLane;
  auto slot_row = [&](int c) {
    return (2 * static_cast<size_t>(c) + (c * per >= e0 ? 0 : 1)) * kRows + r;
  };
  float mmax = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) mmax = fmaxf(mmax, a.part_ml[slot_row(c)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mmax = fmaxf(mmax, __shfl_xor_sync(0xffffffffu, mmax, o));
  float acc[kLane], lsum = 0.f;
#pragma unroll
  for (int e = 0; e < kLane; ++e) acc[e] = 0.f;
  for (int cb = c0; cb <= c1; cb += 32) {
    const int c = cb + lane;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (c <= c1) ml = a.part_ml[slot_row(c)];
    // A range the row saw nothing of wrote no O. One whose scores were all
    // NaN has no max but a sum.
    const bool live = ml.y != 0.f;
    const float wt = ml.x == mmax || ml.x == -INFINITY ? 1.0f : exp2_fast(ml.x - mmax);
    uint32_t todo = __ballot_sync(0xffffffffu, live);
    while (todo) {
      // Four ranges' loads in flight.
      float v[4][kLane], wv[4], lv[4];
      int n = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int src = todo ? __ffs(todo) - 1 : 0;
        const bool on = todo != 0;
        if (on) ++n;
        todo &= todo - 1;
        wv[k] = __shfl_sync(0xffffffffu, wt, src);
        lv[k] = __shfl_sync(0xffffffffu, ml.y, src);
        const float* p = a.part_o + slot_row(cb + src) * HD + d0;
        if (on) {
          if constexpr (kLane == 4) {
            const float4 f = *reinterpret_cast<const float4*>(p);
            v[k][0] = f.x; v[k][1] = f.y; v[k][2] = f.z; v[k][3] = f.w;
          } else {
            const float2 f = *reinterpret_cast<const float2*>(p);
            v[k][0] = f.x; v[k][1] = f.y;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k < n) {
#pragma unroll
          for (int e = 0; e < kLane; ++e) acc[e] = fmaf(wv[k], v[k][e], acc[e]);
          lsum = fmaf(wv[k], lv[k], lsum);
        }
      }
    }
  }
  const float inv = lsum > 0.f ? 1.0f / lsum : lsum != lsum ? lsum : 0.f;
  const int tok = r / a.hpg;
  T* o = static_cast<T*>(a.out) + (t.tok0 + tok) * a.out_stride +
         (kv * a.hpg + r - tok * a.hpg) * HD + d0;
  uint32_t h[kLane / 2];
#pragma unroll
  for (int e = 0; e < kLane / 2; ++e) h[e] = pack2<T>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  if constexpr (kLane == 4)
    *reinterpret_cast<uint2*>(o) = make_uint2(h[0], h[1]);
  else
    *reinterpret_cast<uint32_t*>(o) = h[0];
}

template <int HD, class T>
void launch(const PagedAttnArgs& a, const CUtensorMap& tq, const CUtensorMap& tkv,
            cudaStream_t s) {
  const int groups = std::max(a.b.n_groups, 1);
  launch_pdl(paged_plan_kernel, dim3(1), dim3(kPlanThreads),
             plan_smem_ints(groups, a.max_tiles, a.max_segs) * 4, s, a);
  launch_pdl(paged_attention_kernel<HD, T>, dim3(a.ctas, Shape<HD>::kHalves), dim3(192),
             Shape<HD>::kSmem, s, tq, tkv, a);
  if (a.ctas > 1) {
    const int rows = std::min<int64_t>(kRows, static_cast<int64_t>(a.b.tokens) * a.hpg);
    constexpr int kRowsHere = kMergeWarps / (HD < 128 ? 1 : HD / 128);
    launch_pdl(paged_merge_kernel<HD, T>, dim3(a.ctas - 1, (rows + kRowsHere - 1) / kRowsHere),
               dim3(32 * kMergeWarps), 0, s, a);
  }
}

template <int HD>
void set_smem() {
  cudaFuncSetAttribute(paged_attention_kernel<HD, __half>,
                       cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<HD>::kSmem);
  cudaFuncSetAttribute(paged_attention_kernel<HD, __nv_bfloat16>,
                       cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<HD>::kSmem);
  static_assert(Shape<HD>::kSmem * Shape<HD>::kCtasPerSm <= 227 * 1024, "shared memory");
}

constexpr size_t kPlanSmemMax = 200 * 1024;

size_t align_up(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

void paged_attention_setup_device() {
  set_smem<64>();
  set_smem<128>();
  set_smem<256>();
  set_smem<512>();
  cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       static_cast<int>(kPlanSmemMax));
}

size_t paged_attention_layout(PagedAttnArgs* a, int num_sms) {
  const int groups = std::max(a->b.n_groups, 1);
  a->hpg = a->heads / a->c.kv_heads;
  a->tpt = kRows / a->hpg;
  const int64_t tiles = (static_cast<int64_t>(a->b.tokens) + a->tpt - 1) / a->tpt +
                        std::min<int64_t>(groups, a->b.tokens);
  const int64_t segs = tiles + a->b.n_seqs;
  if (plan_smem_ints(groups, 0, 0) * 4 > kPlanSmemMax || (5 * tiles + segs) * 4 > kPlanSmemMax ||
      plan_smem_ints(groups, static_cast<int>(tiles), static_cast<int>(segs)) * 4 > kPlanSmemMax)
    return 0;
  a->max_tiles = static_cast<int>(tiles);
  a->max_segs = static_cast<int>(segs);
  const int per_sm = a->c.hd == 64 ? Shape<64>::kCtasPerSm : 1;
  a->ctas = std::max(num_sms * per_sm / (a->c.hd == 512 ? 2 : 1), 1);
  a->min_tiles = 2;
  const size_t slots = 2 * static_cast<size_t>(a->ctas) * kRows;
  return align_up(sizeof(PagedPlan)) + align_up((segs + 1) * 4) + align_up(segs * sizeof(PagedSeg)) +
         align_up(tiles * sizeof(PagedTile)) + align_up(slots * 8) + slots * a->c.hd * 4;
}

void paged_attention_workspace(PagedAttnArgs* a, void* ws) {
  uint8_t* p = static_cast<uint8_t*>(ws);
  auto take = [&](size_t n) {
    void* q = p;
    p += align_up(n);
    return q;
  };
  const size_t slots = 2 * static_cast<size_t>(a->ctas) * kRows;
  a->plan = static_cast<PagedPlan*>(take(sizeof(PagedPlan)));
  a->seg_cum = static_cast<int*>(take((static_cast<size_t>(a->max_segs) + 1) * 4));
  a->segs = static_cast<PagedSeg*>(take(static_cast<size_t>(a->max_segs) * sizeof(PagedSeg)));
  a->tiles = static_cast<PagedTile*>(take(static_cast<size_t>(a->max_tiles) * sizeof(PagedTile)));
  a->part_ml = static_cast<float2*>(take(slots * 8));
  a->part_o = static_cast<float*>(take(slots * a->c.hd * 4));
}

bool paged_attention_maps(const PagedAttnArgs& a, const void* q, int64_t q_stride,
                          CUtensorMap* tq, CUtensorMap* tkv, char* err, size_t errlen) {
  const uint64_t hd = a.c.hd, kvh = a.c.kv_heads;
  const uint64_t qd[4] = {hd, static_cast<uint64_t>(a.hpg), kvh, static_cast<uint64_t>(a.b.tokens)};
  const uint64_t qst[3] = {hd * 2, a.hpg * hd * 2, static_cast<uint64_t>(q_stride) * 2};
  const uint32_t qb[4] = {64, static_cast<uint32_t>(a.hpg), 1, static_cast<uint32_t>(a.tpt)};
  if (!make_tmap_f16(tq, q, 4, qd, qst, qb, err, errlen)) return false;
  const uint64_t d[2] = {2 * kvh * hd, static_cast<uint64_t>(a.c.n_pages) << a.c.page_log2};
  const uint64_t st[1] = {2 * kvh * hd * 2};
  const uint32_t b[2] = {64, static_cast<uint32_t>(std::min(1 << a.c.page_log2, kKeys))};
  return make_tmap_f16(tkv, a.c.rows, 2, d, st, b, err, errlen);
}

void launch_paged_attention(const PagedAttnArgs& a, const CUtensorMap& tq, const CUtensorMap& tkv,
                            cudaStream_t s) {
  const bool f16 = a.c.dtype == kOpF16;
  switch (a.c.hd) {
    case 64: return f16 ? launch<64, __half>(a, tq, tkv, s) : launch<64, __nv_bfloat16>(a, tq, tkv, s);
    case 128:
      return f16 ? launch<128, __half>(a, tq, tkv, s) : launch<128, __nv_bfloat16>(a, tq, tkv, s);
    case 256:
      return f16 ? launch<256, __half>(a, tq, tkv, s) : launch<256, __nv_bfloat16>(a, tq, tkv, s);
    default:
      return f16 ? launch<512, __half>(a, tq, tkv, s) : launch<512, __nv_bfloat16>(a, tq, tkv, s);
  }
}

}  // namespace omg
