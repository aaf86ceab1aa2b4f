// Attention over a paged K/V cache for groups of sequences that share a
// prefix (see paged.cuh): out = softmax(scale q K^T) V over the prefix keys
// and the sequence's own keys up to the query's position, inside the window.
//
// Three launches, two for a single row tile, which the attention kernel plans
// itself. The plan kernel (one CTA) cuts the query tokens into row tiles and
// lays their key tiles on one line (paged.cuh). The attention kernel gives
// every CTA an equal range of the line, whatever it crosses; a row tile inside
// one CTA's range is finished there, one that several CTAs cross leaves per
// CTA an unnormalised O and each row's (reference, sum), which the merge kernel
// joins.
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
// per 16-key slot and 64 dims (boxes of whole pages took the same time within
// 2%, and a slot never straddles a page); warp 1 issues S = Q K^T one tile ahead and O += P V; warps 2-5
// own one query row per thread: mask, online softmax, P, the rescale of O.
//
// What bounds it. Prefixes of few rows: HBM; a 64-key tile of head_dim 256
// (64 KB) takes an SM 3,100 clocks, 90% of the copy rate, but slots hold more
// keys than a short branch has, and two partial O per CTA go out and back: 64
// states of up to 2,000 + 20 branches x 31 keys take 90 us, 2.8 TB/s. Long
// sequences of a few rows each: 122 us for 64 of up to 8,192 keys, 5.0 TB/s.
// Prompts: a tile's chain of scores, softmax and product, of which the two CTAs
// of an SM overlap two (head_dim 128: 1,570 clocks a tile, 512 of them the
// tensor pipe's): 770 TFLOP/s over 8,000 keys and more, 610 for a prompt of
// 8,192 tokens alone. One state's next token: latency; 13 to 19 us are two
// launches, the tables' chain of loads, a key tile per CTA and the merge.
//
// Numerics: scores, max, exponentials and sums f32, O accumulated in f32; P
// enters the second product in the cache's 16-bit type (its rounding is of
// the size of the output's own and averages over keys). A row's
// reference moves only when a score passes it by far (kReach), so that P stays
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
constexpr int kSlot = kPagedSlotKeys;
constexpr int kSlots = kKeys / kSlot;
constexpr int kRows = kPagedTileRows;
constexpr int kQChunk = kRows * 128;   // [128 rows][64 dims]
constexpr int kKvChunk = kKeys * 128;  // [64 keys][64 dims]
constexpr int kPBytes = kRows * kKeys * 2;
// A row's probabilities are 2^(score - m_ref) before their common division. At
// a new maximum m_ref is set kLift below it, and again once a score passes
// m_ref + kReach, so P stays below 2^kReach (f16 holds 2^16). f16's least is
// 2^-24: without the lift a key below 2^-25 of the largest had no part in O,
// but in the sum, and 40,000 of them beside a dominant key lost it 1e-3 of
// their V. With it that is below 2^-33; bf16 has f32's range.
template <class T> constexpr float kLift = std::is_same<T, __half>::value ? 8.0f : 0.0f;
template <class T> constexpr float kReach = std::is_same<T, __half>::value ? 15.0f : 11.5f;
constexpr int kPlanThreads = 1024;  // 32 warps (block_scan)
constexpr int kThreads = 192;
// What a row tile costs on the line beside its key tiles, in key tiles: its Q,
// the first tile's latency, the epilogue. Without it the CTA that the first,
// short row tiles of a prompt fall to holds up the rest. (us with 0, 2, 3, 4, 8:
// a prompt of 4,096 tokens, 8 heads of 128: 121, 98, 89, 86, 90; of 512: 378,
// 333, 333, 339, 351; 64 states' next tokens: 89.4, 88.7, 89.5, 90.5, 94.9.)
constexpr int kToll = 3;
// Runs (the prefix's included) that a CTA plans for itself in shared memory.
constexpr int one_tile_runs(int hd) { return hd == 128 ? 21 : 33; }

template <int HD>
struct Shape {
  static constexpr int kV = HD < 256 ? HD : 256;    // dims of V and O per CTA
  static constexpr int kHalves = HD / kV;           // CTAs that share a row tile's softmax
  static constexpr int kChunks = kV / 64;           // 64-dim chunks of a ring stage
  static constexpr int kStage = kChunks * kKvChunk; // 64 keys x kV dims
  static constexpr int kQ = HD / 64 * kQChunk;
  // Two CTAs of an SM hide each other's waits where both fit; at head_dim 128
  // one P slot each leaves room for rings of two whole tiles. (64 sequences of
  // up to 8,192 keys, head_dim 128: one CTA with 8 stages and 2 P slots 148 us,
  // two with 3 stages and 2 P slots 146, two with 4 stages and 1 P slot 118. At
  // head_dim 512 five stages of half the size and one P slot: 51 -> 57 us for
  // 288 tokens over 2,000 keys.)
  static constexpr int kPSlots = HD == 128 ? 1 : 2;
  static constexpr int kCtasPerSm = HD <= 128 ? 2 : 1;
  static constexpr int kStages = HD == 512 ? 2 : HD == 64 ? 6 : 4;
  static constexpr int kTmemO = 128;                // S buffers at columns 0 and 64
  static constexpr uint32_t kTmemCols = HD >= 256 ? 512 : 256;
  static constexpr int kSmem = kQ + kStages * kStage + kPSlots * kPBytes + 320 +
                               (1 + one_tile_runs(HD)) * 32;
};

// ---- plan -------------------------------------------------------------------

// Exclusive scan of v over the plan's block; returns its total. `ws`: 32 ints
// of shared memory.
__device__ __forceinline__ int block_scan(int v, int* excl, int* ws) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) ws[warp] = x;
  __syncthreads();
  // Every warp scans the warps' sums for itself.
  int w = ws[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  const int before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  *excl = x - v + (warp ? before : 0);
  const int total = __shfl_sync(0xffffffffu, w, 31);
  __syncthreads();
  return total;
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

// Row tile `rt`, tokens [t0, t1) of group g: its record and its runs; returns
// its key tiles. A full warp calls it, a lane per sequence; `first` is the
// first sequence that may have tokens there, `s_end` the group's end.
__device__ int plan_tile(const PagedAttnArgs& a, const int* q, const int* lens, int rt, int g,
                         int plen, int t0, int t1, int first, int s_end, PagedRun* runs,
                         PagedTile* out) {
  const int lane = threadIdx.x & 31;
  const int own_cap = a.b.max_pages << a.c.page_log2;
  const int pre_cap = a.b.n_groups > 0 ? a.b.max_prefix_pages << a.c.page_log2 : 0;
  // Sequence `s`'s tokens [ta, tb) of the tile; i0: own index of the first.
  auto part = [&](int s, int* ta, int* tb, int* i0) -> bool {
    *ta = *tb = 0;
    *i0 = 0;
    if (s >= s_end) return false;
    const int q0 = q[s], q1 = q[s + 1], len = lens[s];
    *ta = max(q0, t0);
    *tb = min(q1, t1);
    *i0 = len - (q1 - *ta);
    return q0 >= t1;  // the sequences from here on are past the tile
  };
  int imin = INT_MAX, imax = INT_MIN;
  int ta, tb, i0;
  int chunks = 0;
  for (int s = first; s < s_end; s += 32) {
    const bool past = part(s + lane, &ta, &tb, &i0);
    if (ta < tb) {
      imin = min(imin, i0);
      imax = max(imax, i0 + (tb - ta) - 1);
    }
    ++chunks;
    if (__any_sync(0xffffffffu, past)) break;
  }
  imin = __reduce_min_sync(0xffffffffu, imin);
  imax = __reduce_max_sync(0xffffffffu, imax);
  // The prefix's slots, then the own runs.
  const int end = min(plen, pre_cap);
  const int lo = a.window > 0 && imin != INT_MAX ? max(0, plen + imin - a.window + 1) : 0;
  int key0 = lo / kSlot * kSlot, kend = end;
  int pre = lo < end ? (end - key0 + kSlot - 1) / kSlot : 0;
  const int held = pre;
  int slots = 0, n_runs = 0;
  for (int c = 0; c < chunks; ++c) {
    const int me = first + 32 * c + lane;
    if (chunks > 1) part(me, &ta, &tb, &i0);  // one chunk: still at hand
    int n = 0, k0 = 0, ke = 0;
    if (ta < tb) {
      ke = min(i0 + (tb - ta), own_cap);
      const int l = a.window > 0 ? max(0, i0 - a.window + 1) : 0;
      k0 = l / kSlot * kSlot;
      n = ke > l ? (ke - k0 + kSlot - 1) / kSlot : 0;
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    // A sequence without a slot (a length below its query rows, a table of no
    // pages, a window past it) keeps its run: its rows' own indices are there.
    const bool here = ta < tb;
    const unsigned have = __ballot_sync(0xffffffffu, here);
    const int at = n_runs + __popc(have & ((1u << lane) - 1));
    // (No more runs than tokens in a tile, but for tables out of order.)
    if (here && at < a.tpt)
      runs[1 + at] = PagedRun{rt, held + slots + upto - n,
                              n,  k0,
                              ke, ((ta - t0) * a.hpg) | (((tb - t0) * a.hpg) << 16),
                              i0, me};
    n_runs = min(n_runs + __popc(have), a.tpt);
    slots += __shfl_sync(0xffffffffu, upto, 31);
  }
  // Rows that see nothing at all still get their zeros: one slot, all of it
  // masked. (A prefix run of no slots stays, before the own runs.)
  if (pre + slots == 0) {
    pre = 1;
    key0 = kend = 0;
  }
  const int ntiles = (pre + slots + kSlots - 1) / kSlots;
  if (lane == 0) {
    runs[0] = PagedRun{rt, 0, pre, key0, kend, ((t1 - t0) * a.hpg) << 16, 0, ~g};
    PagedTile t{};
    t.tok0 = t0;
    t.ntok = t1 - t0;
    t.prefix_len = plen;
    t.ntiles = ntiles;
    t.nruns = 1 + n_runs;
    t.imin = imin;
    t.imax = imax;
    *out = t;
  }
  __syncwarp();
  return ntiles;
}

// The place on the line that unit `w` of one KV head's `line` units is, in row
// tile `rt` that begins at unit `at` of it: the toll comes before the tiles.
__device__ __forceinline__ PagedStart place(int kv, int rt, int at, int w) {
  const int pos = w - at - kToll;
  return PagedStart{rt, max(pos, 0), kv, max(-pos, 0)};
}

__device__ __forceinline__ int tiles_per_cta(const PagedAttnArgs& a, int line) {
  // (At least 1, 2, 3, 4: one state with 12 branches 18.8, 20.4, 21.9, 24.1 us.)
  return max((line * a.c.kv_heads + a.ctas - 1) / a.ctas, 1);
}

__host__ __device__ inline size_t plan_smem_ints(int64_t seqs, int64_t groups, int64_t max_tiles) {
  return 32 + 2 * (seqs + 1) + 4 * (groups + 1) + max_tiles + 1;
}

// One block: groups to row tiles, a warp per row tile, and the CTAs' places on
// the line.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedAttnArgs a) {
  extern __shared__ __align__(16) int sm[];
  const int groups = max(a.b.n_groups, 1), S = a.b.n_seqs, T = a.b.tokens;
  int* q = sm + 32;            // [S + 1]
  int* len = q + S + 1;        // [S + 1]
  int* gs = len + S + 1;       // [groups + 1] first sequence, token, row tile; prefix length
  int* gtok = gs + groups + 1;
  int* gtile = gtok + groups + 1;
  int* plen = gtile + groups + 1;
  int* cum = plen + groups + 1;  // [max_tiles + 1] key tiles, then their running sum
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_wait();
  griddep_launch();
  for (int s = tid; s <= S; s += kPlanThreads) {
    q[s] = min(max(a.b.q_start[s], 0), T);
    len[s] = s < S ? a.b.lens[s] : 0;
  }
  for (int g = tid; g <= groups; g += kPlanThreads) {
    const int s = a.b.n_groups > 0 ? a.b.group_start[g] : g * S;
    gs[g] = min(max(s, 0), S);
    plen[g] = a.b.n_groups > 0 && g < groups ? max(a.b.prefix_lens[g], 0) : 0;
  }
  __syncthreads();
  int n_tiles = 0;
  for (int g0 = 0; g0 < groups; g0 += kPlanThreads) {
    const int g = g0 + tid;
    int n = 0;
    if (g < groups) {
      const int t0 = q[gs[g]], t1 = q[gs[g + 1]];
      gtok[g] = t0;
      n = (max(t1 - t0, 0) + a.tpt - 1) / a.tpt;
    }
    int at;
    const int total = block_scan(n, &at, sm);
    if (g < groups) gtile[g] = n_tiles + at;
    n_tiles += total;
  }
  n_tiles = min(n_tiles, a.max_tiles);  // only tables out of order make more
  __syncthreads();
  for (int rt = warp; rt < n_tiles; rt += kPlanThreads / 32) {
    const int g = last_le(gtile, groups, rt);
    const int t0 = gtok[g] + (rt - gtile[g]) * a.tpt;
    const int t1 = min(t0 + a.tpt, q[gs[g + 1]]);
    // The last sequence that starts at or before the first token.
    const int s = max(gs[g], warp_count_le(q + gs[g], gs[g + 1] - gs[g], t0, lane) - 1 + gs[g]);
    const int n = plan_tile(a, q, len, rt, g, plen[g], t0, t1, s, gs[g + 1],
                            a.runs + static_cast<int64_t>(rt) * (a.tpt + 1), a.tiles + rt);
    if (lane == 0) cum[rt] = n + kToll;
  }
  __syncthreads();
  int line = 0;
  for (int rt0 = 0; rt0 < n_tiles; rt0 += kPlanThreads) {
    const int rt = rt0 + tid;
    int at;
    const int total = block_scan(rt < n_tiles ? cum[rt] : 0, &at, sm);
    if (rt < n_tiles) cum[rt] = line + at;
    line += total;
  }
  __syncthreads();
  const int per = tiles_per_cta(a, line);
  for (int i = tid; i < a.ctas; i += kPlanThreads) {
    const int w = i * per;
    PagedStart st{0, 0, 0, 0};
    if (w < line * a.c.kv_heads) {
      const int kv = w / line, wl = w - kv * line, rt = last_le(cum, n_tiles, wl);
      st = place(kv, rt, cum[rt], wl);
    }
    a.starts[i] = st;
  }
  if (tid == 0) *a.plan = PagedPlan{n_tiles, line, per, 0};
}

// ---- attention ----------------------------------------------------------------

// A ring position and the parity of its current use.
template <int N>
struct Ring {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      ph ^= 1;
    }
  }
};

template <int N>
__device__ __forceinline__ int ring_add(int s, int n) {
  s += n;
  return s >= N ? s - N : s;
}

// One row tile's share of a CTA's range of the line, walked tile by tile by
// each role. Lane i keeps the run that slot i % 4 of the tile lies in.
struct Share {
  const PagedRun* runs;
  PagedTile tile;
  PagedRun run;   // rows 0: no such slot
  int kv, rt;
  int pos, end;   // key tiles [pos, end) of the row tile
  int slot, ri;   // this lane's slot of the row tile, and its run's index

  // Up to `left` tiles from tile `pos` of row tile `rt` on; a full warp calls
  // it. The row tile and its first runs, a lane each, come in one round trip.
  // `cap` runs are held for each row tile.
  __device__ __forceinline__ void load(const PagedTile* tiles, const PagedRun* all_runs, int cap,
                                       int left, int lane) {
    runs = all_runs + static_cast<int64_t>(rt) * cap;
    run = runs[min(lane, cap - 1)];
    tile = tiles[rt];
    end = min(tile.ntiles, pos + left);
    if (tile.nruns <= 32) {
      ri = __popc(__ballot_sync(0xffffffffu, lane < tile.nruns && run.slot0 <= pos * kSlots)) - 1;
      run.slot0 = __shfl_sync(0xffffffffu, run.slot0, ri);
      run.n = __shfl_sync(0xffffffffu, run.n, ri);
      run.key0 = __shfl_sync(0xffffffffu, run.key0, ri);
      run.kend = __shfl_sync(0xffffffffu, run.kend, ri);
      run.rows = __shfl_sync(0xffffffffu, run.rows, ri);
      run.i0 = __shfl_sync(0xffffffffu, run.i0, ri);
      run.owner = __shfl_sync(0xffffffffu, run.owner, ri);
    } else {
      ri = warp_count_le(&runs[0].slot0, tile.nruns, pos * kSlots, lane,
                         sizeof(PagedRun) / sizeof(int)) - 1;
      run = runs[ri];
    }
    slot = pos * kSlots + (lane & (kSlots - 1));
    settle();
  }
  // On to the next row tile, or the first of the next KV head.
  __device__ __forceinline__ void leave(int n_tiles) {
    pos = 0;
    if (++rt == n_tiles) {
      rt = 0;
      ++kv;
    }
  }
  __device__ __forceinline__ void settle() {
    while (slot >= run.slot0 + run.n) {
      if (++ri >= tile.nruns) {
        run.rows = 0;
        run.n = INT_MAX / 2;  // stays
        run.slot0 = 0;
        break;
      }
      run = runs[ri];
    }
  }
  __device__ __forceinline__ void next() {
    ++pos;
    slot += kSlots;
    settle();
  }
  __device__ __forceinline__ int key() const { return run.key0 + (slot - run.slot0) * kSlot; }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Every lane waits: a warp that is not split needs no broadcast.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity,
                                          volatile int* abort_flag) {
  const bool ok = mbar_wait(bar, parity, abort_flag, nullptr);
  return __all_sync(0xffffffffu, ok);
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
__global__ void __launch_bounds__(kThreads, Shape<HD>::kCtasPerSm)
    paged_attention_kernel(const __grid_constant__ PagedMaps maps, PagedAttnArgs a) {
  using Sh = Shape<HD>;
  constexpr int VD = Sh::kV, NST = Sh::kStages, CH = Sh::kChunks;
  extern __shared__ __align__(1024) uint8_t qs[];  // (the swizzle's atoms)
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
  // one_tile: the plan.
  PagedTile* my_tile = reinterpret_cast<PagedTile*>(reinterpret_cast<uint8_t*>(bars) + 320);
  PagedRun* my_runs = reinterpret_cast<PagedRun*>(my_tile + 1);
  static_assert((B_RING + 3 * NST) * 8 + 4 * (2 + 8) <= 320, "barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int vhalf = blockIdx.y;  // this CTA's dims of V (head_dim 512)

  if (threadIdx.x == 0) {
    for (int i = 0; i < B_RING; ++i) mbar_init(&bars[i], (i == B_P0 || i == B_P1 || i == B_CLEAN) ? 4 : 1);
    for (int i = 0; i < 3 * NST; ++i) mbar_init(&kfull[i], 1);
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) bad_keys[i] = 0;
    fence_barrier_init();
    prefetch_tmap(&maps.q);
    prefetch_tmap(&maps.kv);
  }
  if (warp == 1) tmem_alloc(tmem_slot, Sh::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch();
  PagedPlan plan;
  PagedStart start;
  const PagedRun* runs = a.runs;
  const PagedTile* tiles = a.tiles;
  const int run_cap = a.one_tile ? one_tile_runs(HD) : a.tpt + 1;
  if (a.one_tile) {
    // A single row tile: warp 2 of every CTA plans it here, in about the time
    // of three loads; the first CTA leaves it to the merge.
    if (warp == 2) {
      const int s0 = a.b.n_groups > 0 ? min(max(a.b.group_start[0], 0), a.b.n_seqs) : 0;
      const int s1 = a.b.n_groups > 0 ? min(max(a.b.group_start[1], s0), a.b.n_seqs) : a.b.n_seqs;
      const int plen = a.b.n_groups > 0 ? max(a.b.prefix_lens[0], 0) : 0;
      const int t0 = min(max(a.b.q_start[s0], 0), a.b.tokens);
      const int t1 = min(max(a.b.q_start[s1], t0), a.b.tokens);
      if (t1 > t0) plan_tile(a, a.b.q_start, a.b.lens, 0, 0, plen, t0, t1, s0, s1, my_runs, my_tile);
      if (t1 == t0 && lane == 0) my_tile->ntiles = -kToll;  // an empty line
      if (blockIdx.x == 0 && blockIdx.y == 0 && lane == 0) {
        const int line = my_tile->ntiles + kToll;
        *a.plan = PagedPlan{1, line, tiles_per_cta(a, line), 0};
        *a.tiles = *my_tile;
      }
    }
    __syncthreads();
    runs = my_runs;
    tiles = my_tile;
    const int line = my_tile->ntiles + kToll;
    plan = PagedPlan{1, line, tiles_per_cta(a, line), 0};
    const int w = blockIdx.x * plan.per, kv = line ? w / line : 0;
    start = place(kv, 0, 0, w - kv * line);
  } else {
    plan = *a.plan;
    start = a.starts[blockIdx.x];
  }
  const int total = plan.line * a.c.kv_heads;
  const int w0 = min(static_cast<int>(blockIdx.x) * plan.per, total);
  const int w1 = min(w0 + plan.per, total);
  constexpr int KST = Sh::kHalves;  // ring stages of a K tile (V: one)

  if (w0 >= w1) {
    // Nothing of the line: on to the end.
  } else if (warp == 0) {
    // ---- loads: Q of each row tile; K and V of each tile. At head_dim 512 V
    // comes after the next tile's K: the two stages that hold a K tile are all
    // the ring has, and S is issued a tile ahead.
    Ring<NST> slot, kr, vr;
    uint32_t qphase = 0;
    int issued_k = 0, issued_v = 0;  // for the drain
    bool ok = true, first_q = true;
    const int lg = a.c.page_log2;
    // A lane per box: slot lane % 4, 64-dim chunk lane / 4.
    const int lb = lane & (kSlots - 1), lc = lane / kSlots;
    // One ring stage: dims [x, x + kV) of the slots, whose first cache rows
    // are `row` (-1: no such keys).
    auto load_stage = [&](int row, int x, bool is_v) {
      if (!warp_wait(&empty[slot.s], slot.ph ^ 1, abort_flag)) {
        ok = false;
        return;
      }
      uint64_t* full = is_v ? &vfull[vr.s] : &kfull[kr.s];
      const bool on = row >= 0 && lc < CH;
      const uint32_t live = __popc(__ballot_sync(0xffffffffu, on));
      if (lane == 0) mbar_arrive_expect_tx(full, live * kSlot * 128);
      __syncwarp();
      if (on)
        tma_load_2d(ring + slot.s * Sh::kStage + lc * kKvChunk + lb * kSlot * 128, &maps.kv, full,
                    x + lc * 64, row);
      slot.next();
      if (is_v) {
        vr.next();
        ++issued_v;
      } else {
        kr.next();
        ++issued_k;
      }
    };
    // The page of this lane's slot and the slot's first key (-1: no such
    // keys), asked for a tile ahead; and the cache row they make. A page
    // outside the pool lies past the map's end, where TMA fills zeros.
    auto slot_page = [&](const Share& u, int* key) -> int {
      *key = u.key();
      if (u.run.rows == 0 || *key >= u.run.kend) {
        *key = -1;
        return 0;
      }
      const int* table =
          u.run.owner < 0
              ? a.b.prefix_pages + static_cast<int64_t>(~u.run.owner) * a.b.max_prefix_pages
              : a.b.pages + static_cast<int64_t>(u.run.owner) * a.b.max_pages;
      return table[*key >> lg];
    };
    auto row_of = [&](int page, int key) -> int {
      if (key < 0) return -1;
      if (page < 0 || page >= a.c.n_pages) page = static_cast<int>(a.c.n_pages);
      return (page << lg) + (key & ((1 << lg) - 1));
    };
    Share u;
    u.rt = start.rt;
    u.pos = start.pos;
    u.kv = start.kv;
    for (int w = w0 + start.toll; w < w1 && ok; u.leave(plan.n_tiles), w += kToll) {
      u.load(tiles, runs, run_cap, w1 - w, lane);
      const int n = u.end - u.pos;
      const int kx = u.kv * HD, vx = (a.c.kv_heads + u.kv) * HD + vhalf * VD;
      if (!first_q) {
        if (!warp_wait(&bars[B_QFREE], qphase, abort_flag)) break;
        qphase ^= 1;
      }
      first_q = false;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars[B_Q], HD * 2u * static_cast<uint32_t>(a.hpg * a.tpt));
#pragma unroll 1
        for (int c = 0; c < HD / 64; ++c)
          tma_load_4d(qs + c * kQChunk, &maps.q, &bars[B_Q], c * 64, 0, u.kv, u.tile.tok0);
      }
      __syncwarp();
      int key, page = slot_page(u, &key), before = -1;
      for (int t = 0; t < n && ok; ++t) {
        const int row = row_of(page, key);
        if (t + 1 < n) {
          u.next();
          page = slot_page(u, &key);
        }
        __syncwarp();
#pragma unroll
        for (int h = 0; h < KST; ++h)
          if (ok) load_stage(row, kx + h * VD, false);
        if constexpr (KST == 1) {
          if (ok) load_stage(row, vx, true);
        } else {
          if (t > 0 && ok) load_stage(before, vx, true);
          before = row;
        }
      }
      if (KST == 2 && ok) load_stage(before, vx, true);
      w += n;
    }
    if (*abort_flag && lane == 0) {
      // Gave up: wait (bounded) for the copies in flight into this CTA.
      for (int i = max(0, issued_k - NST); i < issued_k; ++i)
        mbar_drain(&kfull[i % NST], (i / NST) & 1, kDrainClocks);
      for (int i = max(0, issued_v - NST); i < issued_v; ++i)
        mbar_drain(&vfull[i % NST], (i / NST) & 1, kDrainClocks);
      mbar_drain(&bars[B_Q], 0, kDrainClocks);
      mbar_drain(&bars[B_Q], 1, kDrainClocks);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMA issue: S of a tile, then P V of the one before. The whole warp
    // runs the loop, one lane issues.
    constexpr uint32_t fs = idesc_f16_f32(kRows, kKeys), fo = idesc_f16_f32_bmn(kRows, VD);
    constexpr bool f16 = std::is_same<T, __half>::value;
    constexpr uint32_t idesc_s = f16 ? fs : idesc_bf16(fs);
    constexpr uint32_t idesc_o = f16 ? fo : idesc_bf16(fo);
    const uint64_t dq = sw128_desc(qs), dk = sw128_desc(ring), dp = sw128_desc(ps),
                   dv = sw128_mn_desc(ring, kKvChunk);
    // Ring places: at head_dim 512 in the order of use, otherwise K and V of a
    // tile side by side.
    Ring<NST> slot;
    int kslot = 0, vslot = 1;
    Ring<NST> kr, vr;
    uint32_t qphase = 0;
    int g = 0;  // tiles so far
    bool ok = true;
    // O += P V of tile `at`: a step per slot, for the lanes of its rows (rows
    // 0: no such slot).
    auto issue_pv = [&](int at, const int (&rows)[kSlots]) -> bool {
      const int b = at & 1;
      uint32_t off[kSlots][4];
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        if (i > 0 && rows[i] == rows[i - 1]) {
#pragma unroll
          for (int e = 0; e < 4; ++e) off[i][e] = off[i > 0 ? i - 1 : 0][e];
        } else {
          const int r0 = rows[i] & 0xffff, r1 = rows[i] >> 16;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // Lanes [lo, hi) stay on.
            const int lo = min(max(r0 - 32 * e, 0), 32), hi = min(max(r1 - 32 * e, 0), 32);
            off[i][e] = ~((hi == 32 ? ~0u : (1u << hi) - 1) & ~(lo == 32 ? ~0u : (1u << lo) - 1));
          }
        }
      }
      if (!warp_wait(&bars[B_P0 + b], (at >> 1) & 1, abort_flag) ||
          !warp_wait(&vfull[vr.s], vr.ph, abort_flag))
        return false;
      tc_fence_after();
      const int vs = KST == 1 ? vslot : slot.s;
      if (lane == 0) {
        const uint64_t pa = dp + (b & (Sh::kPSlots - 1)) * (kPBytes >> 4),
                       vb = dv + vs * (Sh::kStage >> 4);
#pragma unroll
        for (int i = 0; i < kSlots; ++i)
          if (rows[i] != 0)
            umma_f16_lanes(tmem + Sh::kTmemO, pa + 2 * i, vb + i * (2048 >> 4), idesc_o, 1u, off[i]);
        umma_commit(&bars[B_O0 + b]);
        umma_commit(&empty[vs]);
      }
      __syncwarp();
      slot.next();
      vslot = ring_add<NST>(vslot, 2);
      vr.next();
      return true;
    };
    Share u;
    u.rt = start.rt;
    u.pos = start.pos;
    u.kv = start.kv;
    for (int w = w0 + start.toll; w < w1 && ok; u.leave(plan.n_tiles), w += kToll) {
      u.load(tiles, runs, run_cap, w1 - w, lane);
      const int n = u.end - u.pos;
      if (!warp_wait(&bars[B_Q], qphase, abort_flag)) {
        ok = false;
        break;
      }
      qphase ^= 1;
      int before[kSlots] = {0, 0, 0, 0};
      for (int t = 0; t < n; ++t) {
        int rows[kSlots];
#pragma unroll
        for (int i = 0; i < kSlots; ++i) rows[i] = __shfl_sync(0xffffffffu, u.run.rows, i);
        if (t + 1 < n) u.next();
        __syncwarp();
        const int b = g & 1;
        // The score buffer's last reader finished before the P of two tiles
        // back, waited for with that tile's P V.
#pragma unroll
        for (int h = 0; h < KST; ++h) {
          if (!warp_wait(&kfull[kr.s], kr.ph, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int ks = KST == 1 ? kslot : slot.s;
          if (lane == 0) {
            const uint64_t kd = dk + ks * (Sh::kStage >> 4);
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16(tmem + b * kKeys, dq + (h * CH + c) * (kQChunk >> 4) + 2 * k,
                         kd + c * (kKvChunk >> 4) + 2 * k, idesc_s, (h | c | k) ? 1u : 0u);
            umma_commit(&empty[ks]);
            if (h == KST - 1) umma_commit(&bars[B_S0 + b]);
          }
          __syncwarp();
          slot.next();
          kslot = ring_add<NST>(kslot, 2);
          kr.next();
        }
        if (ok && t + 1 == n) {
          if (lane == 0) umma_commit(&bars[B_QFREE]);
          __syncwarp();
        }
        if (ok && t > 0) ok = issue_pv(g - 1, before);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) before[i] = rows[i];
        ++g;
      }
      if (ok) ok = issue_pv(g - 1, before);
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
    uint8_t* my_stage[2] = {ps + 32 * q4 * 128,
                            ps + (Sh::kPSlots - 1) * kPBytes + 32 * q4 * 128};
    int it = 0;     // ring stages before the row tile's (head_dim 512)
    int vslot = 1;  // ring place of the next V (otherwise)
    int g = 0;   // tiles so far
    Ring<NST> vr;
    uint32_t clean_phase = 0;
    bool ok = true;
    // All four softmax warps meet (a bounded wait, unlike a named barrier).
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[B_CLEAN]);
      const bool met = warp_wait(&bars[B_CLEAN], clean_phase, abort_flag);
      clean_phase ^= 1;
      return met;
    };
    Share u;
    u.rt = start.rt;
    u.pos = start.pos;
    u.kv = start.kv;
    bool first = true;
    for (int w = w0 + start.toll; w < w1; u.leave(plan.n_tiles), w += kToll) {
      u.load(tiles, runs, run_cap, w1 - w, lane);
      const PagedTile tile = u.tile;
      const int kv = u.kv, n = u.end - u.pos;
      const bool whole = n == tile.ntiles;
      const int nrows = tile.ntok * a.hpg;
      const bool valid = r < nrows;
      // The row's own index, from its sequence's run: a lane per run, and a
      // search over the lanes for the last run that starts at or before the
      // row (own runs ascend by row; a prefix run comes first).
      int own = INT_MIN / 2;
      for (int c = 0; c < tile.nruns; c += 32) {
        int start = kRows + 1, stop = 0, i0 = 0;
        if (c + lane < tile.nruns) {
          const PagedRun w = u.runs[c + lane];
          start = w.owner < 0 ? -1 : w.rows & 0xffff;
          stop = w.owner < 0 ? 0 : w.rows >> 16;
          i0 = w.i0;
        }
        int at = 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          if (__shfl_sync(0xffffffffu, start, at + o) <= r) at += o;
        const int s0 = __shfl_sync(0xffffffffu, start, at), s1 = __shfl_sync(0xffffffffu, stop, at),
                  si = __shfl_sync(0xffffffffu, i0, at);
        if (valid && r >= s0 && r < s1) own = si + ((r - s0) * a.hpg_recip >> 16);
      }
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
      const int wlo = a.window > 0 ? a.window - 1 : INT_MAX / 2;
      for (int done = 0; ok && done < n; ++done) {
        const int b = g & 1;
        // This lane's slot: the keys that any of its run's rows sees, and
        // those that all of them see (bounded by its first and last row).
        const int rows = u.run.rows, key0 = u.key(), owner = u.run.owner;
        const int r0 = rows & 0xffff, r1 = rows >> 16;
        const int shift = owner < 0 ? tile.prefix_len : 0, cap = u.run.kend;
        const int ifirst = shift + (owner < 0 ? tile.imin : u.run.i0);
        const int ilast = shift + (owner < 0 ? tile.imax
                                             : u.run.i0 + ((r1 - r0) * a.hpg_recip >> 16) - 1);
        const int all_lo = max(ilast - wlo, 0), all_hi = min(ifirst + 1, cap);
        const int rows0 = __shfl_sync(0xffffffffu, rows, 0);
        // A tile of one run all of whose rows see all of its keys: no mask.
        const bool edge = !__all_sync(0xffffffffu, rows == rows0 && rows != 0 && key0 >= all_lo &&
                                                       key0 + kSlot <= all_hi);
        // Ring place of this tile's V.
        const int vs =
            KST == 1 ? vslot : (it + done * (KST + 1) + (done + 1 == n ? KST : 2 * KST)) % NST;
        bool mine = r >= (rows0 & 0xffff) && r < (rows0 >> 16);
        uint64_t vis = ~0ull, any = ~0ull, all = ~0ull, exist = ~0ull;
        if (edge) {
          const int any_lo = max(ifirst - wlo, 0), any_hi = min(ilast + 1, cap);
          auto piece = [&](int lo, int hi) -> uint32_t {
            lo = min(max(lo - key0, 0), kSlot);
            hi = min(max(hi - key0, lo), kSlot);
            return rows ? (1u << hi) - (1u << lo) : 0u;
          };
          // Lanes 0 .. 3 hold the tile's four slots.
          auto whole64 = [&](uint32_t p) -> uint64_t {
            p <<= kSlot * (lane & 1);
            const uint32_t lo = __reduce_or_sync(0xffffffffu, lane < 2 ? p : 0u);
            const uint32_t hi = __reduce_or_sync(0xffffffffu, lane == 2 || lane == 3 ? p : 0u);
            return static_cast<uint64_t>(hi) << 32 | lo;
          };
          any = whole64(piece(any_lo, any_hi));
          all = whole64(piece(all_lo, all_hi));
          exist = whole64(rows ? 0xffffu : 0u);
          mine = false;
          vis = 0;
#pragma unroll
          for (int i = 0; i < kSlots; ++i) {
            const int ri = __shfl_sync(0xffffffffu, rows, i), ki = __shfl_sync(0xffffffffu, key0, i),
                      ci = __shfl_sync(0xffffffffu, cap, i), si = __shfl_sync(0xffffffffu, shift, i);
            if (r >= (ri & 0xffff) && r < (ri >> 16) && own > INT_MIN / 2) {
              mine = true;
              const int p = si + own;
              const int lo = min(max(p - wlo - ki, 0), kSlot), hi = min(max(min(p + 1, ci) - ki, lo), kSlot);
              vis |= static_cast<uint64_t>((1u << hi) - (1u << lo)) << (kSlot * i);
            }
          }
        }
        // (A row without a run, by tables out of order, sees nothing.)
        mine = mine && own > INT_MIN / 2;
        if (!warp_wait(&bars[B_S0 + b], (g >> 1) & 1, abort_flag)) {
          ok = false;
          break;
        }
        uint64_t bad = 0;
        if (edge) {
          // Keys that no row sees may hold anything: their V rows become
          // zeros. Of those that only some rows see, V rows with infinities or
          // NaN are taken out of the product and added by hand to the rows
          // that see them, so that a masked key never reaches a row. (Other
          // sequences' keys of the tile cannot: their steps of the product
          // leave the row's lane alone.)
          uint8_t* v = ring + vs * Sh::kStage;
          if (!warp_wait(&vfull[vr.s], vr.ph, abort_flag)) {
            ok = false;
            break;
          }
          // f(16-byte piece, key) over the V rows of `keys`, a key per warp.
          auto each_piece = [&](uint64_t keys, auto f) {
            for (keys &= 0x1111111111111111ull << q4; keys; keys &= keys - 1) {
              const int key = __ffsll(static_cast<long long>(keys)) - 1;
              if (lane < CH * 8)
                f(reinterpret_cast<uint4*>(v + (lane >> 3) * kKvChunk + key * 128 + (lane & 7) * 16),
                  key);
            }
          };
          auto zero = [](uint4* p, int) { *p = make_uint4(0, 0, 0, 0); };
          each_piece(exist & ~any, zero);
          const uint64_t part = any & ~all;
          if (part) {
            each_piece(part, [&](uint4* p, int key) {
              const uint4 x = *p;
              if (nonfinite2<T>(x.x) || nonfinite2<T>(x.y) || nonfinite2<T>(x.z) ||
                  nonfinite2<T>(x.w))
                atomicOr(&bad_keys[2 * (g & 3) + (key >> 5)], 1u << (key & 31));
            });
            if (!meet()) {
              ok = false;
              break;
            }
            const volatile uint32_t* bk = bad_keys + 2 * (g & 3);
            bad = static_cast<uint64_t>(bk[0]) | (static_cast<uint64_t>(bk[1]) << 32);
            if (bad) {
              each_piece(bad, zero);
              if (!meet()) {
                ok = false;
                break;
              }
              if (tid < 2) bad_keys[2 * (g & 3) + tid] = 0;
            }
          }
        }
        const bool my_warp = __any_sync(0xffffffffu, mine);
        uint8_t* pj = ps + (b & (Sh::kPSlots - 1)) * kPBytes;
        if (my_warp) {
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
          // Rows without a slot here see nothing: their lanes are off in the
          // product, so only their (max, sum) must not move and their
          // scores need no mask.
          if (__any_sync(0xffffffffu, vis != ~0ull && mine)) {
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
          if (mine && mt > m_ref + kReach<T>) {
            rescale = m_ref != -INFINITY;
            const float to = mt - kLift<T>;
            alpha = rescale ? exp2_fast(m_ref - to) : 0.f;
            m_ref = to;
          }
          // A row that has seen nothing yet has no reference: its scores are
          // all -infinity, or NaN, which counts (fmaxf drops it).
          const float ref = m_ref == -INFINITY ? 0.f : m_ref;
          float psum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < kKeys; ++c) {
            s[c] = exp2_fast(fmaf(s[c], a.scale_log2, -ref));
            psum[c & 7] += s[c];
          }
          const float sum = ((psum[0] + psum[1]) + (psum[2] + psum[3])) +
                            ((psum[4] + psum[5]) + (psum[6] + psum[7]));
          if (mine) l = l * alpha + sum;
          const bool any_rescale = __any_sync(0xffffffffu, rescale);
          // Rescaling O needs the P V before this one done; slot b was read
          // by the one before that.
          if (done > 0 && (any_rescale || Sh::kPSlots == 1)) {
            if (!warp_wait(&bars[B_O0 + ((g - 1) & 1)], ((g - 1) >> 1) & 1, abort_flag)) {
              ok = false;
              break;
            }
          }
          if (Sh::kPSlots == 2 && done > 1) {
            if (!warp_wait(&bars[B_O0 + b], ((g - 2) >> 1) & 1, abort_flag)) {
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
        if (my_warp || edge) fence_proxy_async();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[B_P0 + b]);
        if (bad) {
          // The taken-out keys, for the rows that see them.
          if (!warp_wait(&bars[B_O0 + b], (g >> 1) & 1, abort_flag)) {
            ok = false;
            break;
          }
          if (__any_sync(0xffffffffu, (vis & bad) != 0)) {
            tc_fence_after();
            for (uint64_t todo = bad; todo; todo &= todo - 1) {
              const int key = __ffsll(static_cast<long long>(todo)) - 1;
              // (All lanes take part: `todo` is the same in all of them.)
              const int from = __shfl_sync(0xffffffffu, owner, key / kSlot);
              const int at = __shfl_sync(0xffffffffu, key0, key / kSlot) + key % kSlot;
              const int pi = at >> a.c.page_log2;
              int page = from < 0 ? a.b.prefix_pages[static_cast<int64_t>(~from) *
                                                         a.b.max_prefix_pages + pi]
                                  : a.b.pages[static_cast<int64_t>(from) * a.b.max_pages + pi];
              const int64_t row = (static_cast<int64_t>(page) << a.c.page_log2) +
                                  (at & ((1 << a.c.page_log2) - 1));
              const uint16_t* vrow = static_cast<const uint16_t*>(a.c.rows) +
                                     (row * 2 * a.c.kv_heads + a.c.kv_heads + kv) * HD +
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
        ++g;
        vslot = ring_add<NST>(vslot, 2);
        vr.next();
        if (done + 1 < n) u.next();
        __syncwarp();
      }
      it += n * (KST + 1);
      // O of the row tile, or this range's share of it.
      if (ok && !warp_wait(&bars[B_O0 + ((g - 1) & 1)], ((g - 1) >> 1) & 1, abort_flag)) ok = false;
      tc_fence_after();
      const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (first ? 0 : 1);
      float keep = 0.f;
      const bool zero = l == 0.f && ok;  // O may hold anything
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
          uint32_t o[2][32];
          tmem_ld32_nowait(trow + Sh::kTmemO, o[0]);
          tmem_ld32_nowait(trow + Sh::kTmemO + 32, o[1]);
#pragma unroll 1
          for (int c = 0; c < VD / kPass; ++c) {
            uint8_t* st = my_stage[c & 1];
            tmem_ld_wait();
            if (Sh::kPSlots == 1) __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              uint32_t h[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float x = __uint_as_float(o[e >> 2][8 * (e & 3) + 2 * q]),
                            y = __uint_as_float(o[e >> 2][8 * (e & 3) + 2 * q + 1]);
                h[q] = zero ? 0u : pack2<T>(x * keep, y * keep);
              }
              *reinterpret_cast<uint4*>(st + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                  make_uint4(h[0], h[1], h[2], h[3]);
            }
            if (c + 1 < VD / kPass) {
              tmem_ld32_nowait(trow + Sh::kTmemO + (c + 1) * kPass, o[0]);
              tmem_ld32_nowait(trow + Sh::kTmemO + (c + 1) * kPass + 32, o[1]);
            }
            __syncwarp();
            uint4 v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int i = (lane >> 3) + 4 * e;
              v[e] = *reinterpret_cast<const uint4*>(st + i * 128 + (((lane & 7) ^ (i & 7)) << 4));
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int i = (lane >> 3) + 4 * e, row = 32 * q4 + i;
              const int tok = row * a.hpg_recip >> 16;
              T* o = static_cast<T*>(a.out) + (tile.tok0 + tok) * a.out_stride +
                     (kv * a.hpg + row - tok * a.hpg) * HD + vhalf * VD + c * kPass;
              if (i < rows_here) reinterpret_cast<uint4*>(o)[lane & 7] = v[e];
            }
          }
        } else {
          const uint32_t live = __ballot_sync(0xffffffffu, used);
          float* po = a.part_o + slot * kRows * HD + vhalf * VD;
          uint32_t o[32];
          tmem_ld32_nowait(trow + Sh::kTmemO, o);
#pragma unroll 1
          for (int c = 0; c < VD / 32; ++c) {
            uint8_t* st = my_stage[c & 1];
            tmem_ld_wait();
            if (Sh::kPSlots == 1) __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(st + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                  make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            if (c + 1 < VD / 32) tmem_ld32_nowait(trow + Sh::kTmemO + (c + 1) * 32, o);
            __syncwarp();
            uint4 v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int i = (lane >> 3) + 4 * e;
              v[e] = *reinterpret_cast<const uint4*>(st + i * 128 + (((lane & 7) ^ (i & 7)) << 4));
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int i = (lane >> 3) + 4 * e;
              if ((live >> i) & 1)
                reinterpret_cast<uint4*>(po + static_cast<size_t>(32 * q4 + i) * HD +
                                         c * 32)[lane & 7] = v[e];
            }
          }
          // Two CTAs share a row at head_dim 512 and one of them writes its sum:
          // each that gave up marks its own dims.
          if (Sh::kHalves > 1 && !ok) {
            __syncwarp();
            for (int d = 0; d < VD && valid; ++d) po[static_cast<size_t>(r) * HD + d] = NAN;
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      first = false;
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
// first (later boundaries of the same tile leave), and of it every
// gridDim.y-th row. A warp per row and 128 dims (64 at head_dim 64).
constexpr int kMergeWarps = 8;

// Blocks that share a cut row tile's rows. Few row tiles are cut by many CTAs
// each: many blocks, each with long sums. Many row tiles are cut once or
// twice: every boundary has work, and more blocks than fit at once wait.
// (One state, 12 branches: 8 blocks 22.4 us a call, 16 blocks 20.4; 64
// states: 8 blocks 90 us, 16 blocks 95.6.)
constexpr int merge_split(int64_t entries) { return entries < 64 ? 16 : 8; }

template <int HD, class T>
__global__ void __launch_bounds__(32 * kMergeWarps) paged_merge_kernel(PagedAttnArgs a) {
  constexpr int kPer = HD < 128 ? HD : 128;       // dims per warp
  constexpr int kRowWarps = HD / kPer;            // warps per row
  constexpr int kRowsHere = kMergeWarps / kRowWarps;
  constexpr int kLane = kPer / 32;                // dims per lane
  constexpr int kMany = 4;                        // ranges summed at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x + 1;
  griddep_wait();
  griddep_launch();
  const PagedPlan plan = *a.plan;
  PagedStart st;
  if (a.one_tile) {
    const int w = i * plan.per, kv = plan.line ? w / plan.line : 0;
    st = place(kv, 0, 0, w - kv * plan.line);
  } else {
    st = a.starts[i];
  }
  const PagedTile t = a.tiles[st.rt];
  const int per = plan.per, w = i * per;
  if (w >= plan.line * a.c.kv_heads) return;
  const int kv = st.kv, e0 = w - st.pos;  // the row tile's first key tile
  if (st.pos == 0 || (i - 1) * per > e0) return;
  const int c0 = i - 1, c1 = (e0 + t.ntiles - 1) / per;
  const int d0 = (warp % kRowWarps) * kPer + lane * kLane;
  const int nrows = t.ntok * a.hpg;
  for (int r = blockIdx.y + gridDim.y * (warp / kRowWarps); r < nrows;
       r += gridDim.y * kRowsHere) {
    auto slot_row = [&](int c) {
      return (2 * static_cast<size_t>(c) + (c * per >= e0 - kToll ? 0 : 1)) * kRows + r;
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
        // Several ranges' loads in flight.
        float v[kMany][kLane], wv[kMany], lv[kMany];
        int n = 0;
  #pragma unroll
        for (int k = 0; k < kMany; ++k) {
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
        for (int k = 0; k < kMany; ++k) {
          if (k < n) {
  #pragma unroll
            for (int e = 0; e < kLane; ++e) acc[e] = fmaf(wv[k], v[k][e], acc[e]);
            lsum = fmaf(wv[k], lv[k], lsum);
          }
        }
      }
    }
    const float inv = lsum > 0.f ? 1.0f / lsum : lsum != lsum ? lsum : 0.f;
    const int tok = r * a.hpg_recip >> 16;
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
}

template <int HD, class T>
void launch(const PagedAttnArgs& a, const PagedMaps& m, cudaStream_t s) {
  if (!a.one_tile)
    launch_pdl(paged_plan_kernel, dim3(1), dim3(kPlanThreads),
               plan_smem_ints(a.b.n_seqs, std::max(a.b.n_groups, 1), a.max_tiles) * 4, s, a);
  launch_pdl(paged_attention_kernel<HD, T>, dim3(a.ctas, Shape<HD>::kHalves), dim3(kThreads),
             Shape<HD>::kSmem, s, m, a);
  if (a.ctas > 1)
    launch_pdl(paged_merge_kernel<HD, T>,
               dim3(a.ctas - 1, merge_split(static_cast<int64_t>(a.max_tiles) * a.c.kv_heads)),
               dim3(32 * kMergeWarps), 0, s, a);
}

template <int HD>
void set_smem() {
  cudaFuncSetAttribute(paged_attention_kernel<HD, __half>,
                       cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<HD>::kSmem);
  cudaFuncSetAttribute(paged_attention_kernel<HD, __nv_bfloat16>,
                       cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<HD>::kSmem);
  static_assert((Shape<HD>::kSmem + 1024) * Shape<HD>::kCtasPerSm <= 228 * 1024, "shared memory");
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

bool paged_attention_shape(PagedAttnArgs* a) {
  const int groups = std::max(a->b.n_groups, 1);
  a->hpg = a->heads / a->c.kv_heads;
  a->tpt = kRows / a->hpg;
  a->hpg_recip = (65536 + a->hpg - 1) / a->hpg;
  const int64_t tiles = (static_cast<int64_t>(a->b.tokens) + a->tpt - 1) / a->tpt +
                        std::min<int64_t>(groups, a->b.tokens);
  if (plan_smem_ints(a->b.n_seqs, groups, tiles) * 4 > kPlanSmemMax) return false;
  a->max_tiles = static_cast<int>(tiles);
  // Units of the line are 32-bit numbers, so are the slots of a row tile: a
  // bound on them from the tables' widths. A run is a pair of a sequence and a
  // row tile that holds some of it.
  auto key_tiles = [&](int64_t pages) { return (pages << a->c.page_log2) / kKeys + 2; };
  const int64_t runs = a->b.n_seqs + tiles;
  const int64_t line = runs * key_tiles(a->b.max_pages) +
                       tiles * (kToll + (a->b.n_groups > 0 ? key_tiles(a->b.max_prefix_pages) : 0));
  if (line > (int64_t(1) << 29) / a->c.kv_heads) return false;
  // One row tile of few runs (a batch of branches of one state, a token each):
  // planned by every CTA for itself, which spares a launch. (One state with 12
  // branches: 26.8 us with the plan kernel, 22.4 without. More than 32 runs
  // take a second round of loads in every CTA: with up to 160, 7,400 clocks.)
  a->one_tile = a->b.n_groups <= 1 && a->b.tokens <= a->tpt &&
                std::min(a->b.n_seqs, a->tpt) < one_tile_runs(a->c.hd);
  return true;
}

size_t paged_attention_layout(PagedAttnArgs* a, int num_sms) {
  const int per_sm = a->c.hd <= 128 ? 2 : 1;
  a->ctas = std::max(num_sms * per_sm / (a->c.hd == 512 ? 2 : 1), 1);
  const size_t slots = 2 * static_cast<size_t>(a->ctas) * kRows;
  const size_t tiles = a->max_tiles;
  return align_up(sizeof(PagedPlan)) + align_up(a->ctas * sizeof(PagedStart)) +
         align_up(tiles * (a->tpt + 1) * sizeof(PagedRun)) + align_up(tiles * sizeof(PagedTile)) + align_up(slots * 8) + slots * a->c.hd * 4;
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
  a->starts = static_cast<PagedStart*>(take(a->ctas * sizeof(PagedStart)));
  a->runs = static_cast<PagedRun*>(
      take(static_cast<size_t>(a->max_tiles) * (a->tpt + 1) * sizeof(PagedRun)));
  a->tiles = static_cast<PagedTile*>(take(static_cast<size_t>(a->max_tiles) * sizeof(PagedTile)));
  a->part_ml = static_cast<float2*>(take(slots * 8));
  a->part_o = static_cast<float*>(take(slots * a->c.hd * 4));
}

bool paged_attention_maps(const PagedAttnArgs& a, const void* q, int64_t q_stride, PagedMaps* m,
                          char* err, size_t errlen) {
  const uint64_t hd = a.c.hd, kvh = a.c.kv_heads;
  const uint64_t qd[4] = {hd, static_cast<uint64_t>(a.hpg), kvh, static_cast<uint64_t>(a.b.tokens)};
  const uint64_t qst[3] = {hd * 2, a.hpg * hd * 2, static_cast<uint64_t>(q_stride) * 2};
  const uint32_t qb[4] = {64, static_cast<uint32_t>(a.hpg), 1, static_cast<uint32_t>(a.tpt)};
  if (!make_tmap_f16(&m->q, q, 4, qd, qst, qb, err, errlen)) return false;
  const uint64_t d[2] = {2 * kvh * hd, static_cast<uint64_t>(a.c.n_pages) << a.c.page_log2};
  const uint64_t st[1] = {2 * kvh * hd * 2};
  const uint32_t b[2] = {64, kSlot};
  return make_tmap_f16(&m->kv, a.c.rows, 2, d, st, b, err, errlen);
}

template <int HD>
static void launch_type(const PagedAttnArgs& a, const PagedMaps& m, cudaStream_t s) {
  if (a.c.dtype == kOpF16)
    launch<HD, __half>(a, m, s);
  else
    launch<HD, __nv_bfloat16>(a, m, s);
}

void launch_paged_attention(const PagedAttnArgs& a, const PagedMaps& m, cudaStream_t s) {
  switch (a.c.hd) {
    case 64: return launch_type<64>(a, m, s);
    case 128: return launch_type<128>(a, m, s);
    case 256: return launch_type<256>(a, m, s);
    default: return launch_type<512>(a, m, s);
  }
}

}  // namespace omg
