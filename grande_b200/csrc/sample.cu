// Sampling from logits rows (see sample.cuh). With x_i the row's logits, m
// its largest and T the temperature, w_i = exp((x_i - m) / T); in the order of
// descending x, equal ones by ascending index,
//   top-k keeps the first k,
//   top-p of those the shortest run whose w sums to at least p of their sum,
//   min-p of those the ones with w_i >= min_p;
// the token is the first in index order whose running sum of kept w exceeds
// u times their sum.
//
// A cluster of CTAs per row: each reads its slice of the row once from HBM
// into shared memory, and every later step runs from there. Nothing is
// sorted but short lists: a threshold (the k-th element, the p-th of the
// mass) is found by a histogram over log2 w in steps of 1/64, whose crossing
// bin is then refined by the exact (value, index) order until at most kList
// elements are left, which the first CTA sorts.
//
// The outcome is discrete, so sums have to be good to well under a border's
// width: a border of the running sum lies within 2^-24 of u times the total
// for about one row in 2^24 / vocab, far too often for f32. Weights are
// 64-bit integers in units of 2^-44 of the largest, from a 64-bit exp2 (table
// of 64 and a polynomial), so all sums are exact and the same in any order,
// atomics included.
//
// Bound: one read of the logits at HBM rate; above it stands the 64-bit
// exponential of every element where no top-k cuts the row first.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "ptx.cuh"
#include "sample.cuh"

namespace omg {

namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2944;      // log2 w from 0 to -46 in steps of 1/64
constexpr int kList = 2048;      // elements the first CTA sorts
constexpr int kScale = 44;       // weights in units of 2^-44
constexpr int kMaxCluster = 8;
constexpr int kSliceBytes = 160 * 1024;
constexpr int kSubBits = 11;     // refinement: up to 2^11 bins of the (value, index) order

struct Found {
  int ok, bin;
  unsigned above_cnt, bin_cnt;
  u64 above_mass, bin_mass;
};

struct Shared {
  union {
    struct {
      unsigned cnt[kBins], lo[kBins], hi[kBins];
    } h;
    struct {
      u64 comp[kList];
      u64 w[kList];
    } l;
  };
  double table[64];
  u64 red[kWarps];
  unsigned redc[kWarps];
  // Read by the other CTAs of the cluster.
  u64 best, part_mass, lo, hi;
  unsigned part_cnt, list_n;
  Found found;
  u64 threshold;
};

template <class T>
__device__ __forceinline__ float as_float(T v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (std::is_same<T, __half>::value)
    return __half2float(v);
  else
    return __bfloat162float(v);
}

// (value, index) order: descending value, then ascending index. NaN counts as
// -infinity, the two zeros are equal.
__device__ __forceinline__ u64 order_of(float x, unsigned idx) {
  x = x != x ? -INFINITY : x + 0.0f;
  const unsigned b = __float_as_uint(x);
  const unsigned key = b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
  return (static_cast<u64>(~key) << 32) | idx;
}
__device__ __forceinline__ float value_of(u64 comp) {
  const unsigned key = ~static_cast<unsigned>(comp >> 32);
  return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

// log2 w of a value, and w as an integer.
struct Weigher {
  double c, mc;  // log2(e) / T, the same times the row's largest
  float best;
  const double* table;

  // -64 log2 w rounded, or -1 when w is zero; *y: log2 w.
  __device__ __forceinline__ int bin(float x, double* y) const {
    const double v = x == best ? 0.0 : fma(static_cast<double>(x), c, -mc);
    if (!(v > -45.5)) return -1;
    *y = v;
    const double magic = 6755399441055744.0 / 64;  // 1.5 * 2^52 / 64: units of 1/64
    const int t = __double2loint(v + magic);
    return t > 0 ? 0 : -t;
  }
  __device__ __forceinline__ u64 weight(double y) const {
    const double magic = 6755399441055744.0 / 64;
    const double s = y + magic;
    const int t = __double2loint(s);
    const double r = y - (s - magic);  // |r| <= 1/128
    // 2^r - 1 = r (ln 2 + r (ln 2)^2 / 2 + ...), to 2^-44 of it.
    double p = fma(r, 9.618129107628477e-3, 5.550410866482158e-2);
    p = fma(p, r, 2.402265069591007e-1);
    p = fma(p, r, 6.931471805599453e-1);
    const double b = table[t & 63];
    const double m = fma(b * r, p, b);
    const long long bits = __double_as_longlong(m);
    const int e = static_cast<int>(bits >> 52) - 1023 + (t >> 6);
    const int shift = 52 - kScale - e;
    const u64 mant = (bits & 0xfffffffffffffll) | 0x10000000000000ll;
    return shift > 60 ? 0 : (mant + (1ull << (shift - 1))) >> shift;
  }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_min64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w < v ? w : v;
  }
  return v;
}

// Exclusive scans over the block; the totals come back through the pointers.
__device__ __forceinline__ void block_scan(Shared& sh, unsigned& c, u64& m, unsigned* ctot,
                                           u64* mtot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned ci = c;
  u64 mi = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned a = __shfl_up_sync(0xffffffffu, ci, o);
    const u64 b = __shfl_up_sync(0xffffffffu, mi, o);
    if (lane >= o) {
      ci += a;
      mi += b;
    }
  }
  if (lane == 31) {
    sh.redc[warp] = ci;
    sh.red[warp] = mi;
  }
  __syncthreads();
  if (warp == 0) {
    unsigned a = sh.redc[lane];
    u64 b = sh.red[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned a2 = __shfl_up_sync(0xffffffffu, a, o);
      const u64 b2 = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) {
        a += a2;
        b += b2;
      }
    }
    sh.redc[lane] = a;
    sh.red[lane] = b;
  }
  __syncthreads();
  c = ci - c + (warp ? sh.redc[warp - 1] : 0);
  m = mi - m + (warp ? sh.red[warp - 1] : 0);
  *ctot = sh.redc[kWarps - 1];
  *mtot = sh.red[kWarps - 1];
  __syncthreads();
}

// Smallest integer that is at least p times m, and the integer part of u
// times m (p, u in [0, 1)).
__device__ __forceinline__ u64 ceil_part(float p, u64 m) {
  const u64 f = __double2ull_rz(static_cast<double>(p) * 18446744073709551616.0);
  return __umul64hi(f, m) + (f * m != 0 ? 1 : 0);
}
__device__ __forceinline__ u64 floor_part(float u, u64 m) {
  return __umul64hi(__double2ull_rz(static_cast<double>(u) * 18446744073709551616.0), m);
}

// Sort sh.l.comp[0 .. n) ascending (n a power of two).
__device__ void sort_list(Shared& sh, int n) {
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 x = sh.l.comp[a], y = sh.l.comp[b];
        if ((x > y) == ((a & k) == 0)) {
          sh.l.comp[a] = y;
          sh.l.comp[b] = x;
        }
      }
      __syncthreads();
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto peer = [&](int r) -> Shared& { return *cluster.map_shared_rank(&sh, r); };

  // This CTA's slice [i0, i0 + n) of the row, kept at x[0 .. n).
  const int per = (a.vocab + C - 1) / C;
  const int i0 = min(rank * per, a.vocab), n = min(per, a.vocab - i0);
  const T* src = static_cast<const T*>(a.logits) + row * a.stride + i0;
  constexpr int kVec = 16 / sizeof(T);
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
  T* x = reinterpret_cast<T*>(smem + (sizeof(Shared) + 15) / 16 * 16) + lead;
  if (tid < 64) sh.table[tid] = exp2(tid / 64.0);
  if (tid == 0) {
    sh.list_n = 0;
    sh.threshold = ~0ull;
  }
  u64 best = ~0ull;
  {
    const int head = min(n, lead ? kVec - lead : 0);
    const int body = (n - head) / kVec;
    for (int i = tid; i < head; i += kThreads) {
      x[i] = src[i];
      best = min(best, order_of(as_float(x[i]), i0 + i));
    }
    const uint4* vs = reinterpret_cast<const uint4*>(src + head);
    uint4* vd = reinterpret_cast<uint4*>(x + head);
    for (int j0 = 0; j0 < body; j0 += 4 * kThreads) {
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + k * kThreads + tid;
        if (j < body) v[k] = __ldcs(vs + j);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + k * kThreads + tid;
        if (j >= body) break;
        vd[j] = v[k];
        const T* e = reinterpret_cast<const T*>(&v[k]);
        float m = -INFINITY;
        int at = 0;
#pragma unroll
        for (int q = 0; q < kVec; ++q) {
          const float f = as_float(e[q]);
          if (f > m) {
            m = f;
            at = q;
          }
        }
        best = min(best, order_of(m, i0 + head + j * kVec + at));
      }
    }
    for (int i = head + body * kVec + tid; i < n; i += kThreads) {
      x[i] = src[i];
      best = min(best, order_of(as_float(x[i]), i0 + i));
    }
  }
  best = warp_min64(best);
  if (lane == 0) sh.red[warp] = best;
  __syncthreads();
  if (warp == 0) {
    best = warp_min64(sh.red[lane]);
    if (lane == 0) sh.best = best;
  }
  cluster.sync();
  best = ~0ull;
  for (int r = 0; r < C; ++r) best = min(best, peer(r).best);

  const float temp = a.temperature ? a.temperature[row] : a.temperature1;
  int k = a.top_k ? a.top_k[row] : a.top_k1;
  float top_p = a.top_p ? a.top_p[row] : a.top_p1;
  float min_p = a.min_p ? a.min_p[row] : a.min_p1;
  min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
  const float u = fminf(fmaxf(a.u[row], 0.0f), 0.99999994f);
  if (k <= 0 || k >= a.vocab) k = INT_MAX;
  if (!(top_p < 1.0f)) top_p = 1.0f;
  Weigher wt;
  wt.best = value_of(best);
  const bool dead = wt.best == -INFINITY;
  if (dead || !(temp > 0.0f) || k == 1 || top_p <= 0.0f) {
    // The largest alone. (Every CTA of the cluster takes the same branches.)
    if (rank == 0 && tid == 0) {
      a.tokens[row] = dead ? -1 : static_cast<int>(best & 0xffffffffu);
      if (a.probs) a.probs[row] = dead ? 0.0f : 1.0f;
    }
    cluster.sync();  // no CTA leaves while another may read its memory
    return;
  }
  wt.c = 1.4426950408889634 / static_cast<double>(temp);
  wt.mc = static_cast<double>(wt.best) * wt.c;
  wt.table = sh.table;
  const double min_w = static_cast<double>(min_p) * static_cast<double>(1ull << kScale);

  // Element i of the slice: its order, and its bin (-1: no weight).
  auto comp_at = [&](int i) { return order_of(as_float(x[i]), i0 + i); };
  auto bin_at = [&](int i, double* y) {
    float v = as_float(x[i]);
    return wt.bin(v, y);
  };

  // Histograms of one sweep: elements of order at most `limit` that `key`
  // gives a bin >= 0.
  auto clear_hist = [&]() {
    for (int i = tid; i < kBins; i += kThreads) sh.h.cnt[i] = sh.h.lo[i] = sh.h.hi[i] = 0;
    if (tid == 0) sh.found.ok = 0;
    __syncthreads();
  };
  auto add = [&](int bin, u64 w, bool mass) {
    atomicAdd(&sh.h.cnt[bin], 1u);
    if (mass) {
      const unsigned lo = static_cast<unsigned>(w);
      const unsigned old = atomicAdd(&sh.h.lo[bin], lo);
      const unsigned hi = static_cast<unsigned>(w >> 32) + (old + lo < old ? 1u : 0u);
      if (hi) atomicAdd(&sh.h.hi[bin], hi);
    }
  };
  // The first bin at which the running count reaches `count`, or (mass) the
  // running mass reaches `target` (0: top_p of the total).
  auto find = [&](bool mass, unsigned count, u64 target) -> Found {
    cluster.sync();
    const int share = kBins / C;  // C divides it
    const int each = (share + kThreads - 1) / kThreads;
    unsigned c[3];
    u64 m[3];
    unsigned ct = 0;
    u64 mt = 0;
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      c[e] = 0;
      m[e] = 0;
      const int b = tid * each + e;
      if (e < each && b < share) {
        const int g = rank * share + b;
        for (int r = 0; r < C; ++r) {
          Shared& p = peer(r);
          c[e] += p.h.cnt[g];
          if (mass) m[e] += (static_cast<u64>(p.h.hi[g]) << 32) + p.h.lo[g];
        }
      }
      ct += c[e];
      mt += m[e];
    }
    unsigned cx = ct, ctot;
    u64 mx = mt, mtot;
    block_scan(sh, cx, mx, &ctot, &mtot);
    if (tid == 0) {
      sh.part_cnt = ctot;
      sh.part_mass = mtot;
    }
    cluster.sync();
    u64 all = 0;
    for (int r = 0; r < C; ++r) {
      const u64 pm = peer(r).part_mass;
      const unsigned pc = peer(r).part_cnt;
      all += pm;
      if (r < rank) {
        cx += pc;
        mx += pm;
      }
    }
    if (mass && target == 0) target = ceil_part(top_p, all);
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      const bool here = mass ? mx < target && mx + m[e] >= target
                             : cx < count && cx + c[e] >= count;
      if (here) {
        Found f;
        f.ok = 1;
        f.bin = rank * share + tid * each + e;
        f.above_cnt = cx;
        f.bin_cnt = c[e];
        f.above_mass = mx;
        f.bin_mass = target;  // handed on: the target of the mass
        for (int r = 0; r < C; ++r) peer(r).found = f;
      }
      cx += c[e];
      mx += m[e];
    }
    cluster.sync();
    const Found f = sh.found;
    __syncthreads();  // read by all before the next sweep clears it
    return f;
  };
  // Elements of `pred` (the same total in every CTA's eyes, at most kList)
  // into the first CTA's list; returns their number, padded list sorted there.
  auto gather = [&](auto pred) -> int {
    Shared& first = peer(0);
    const int rounds = (n + kThreads - 1) / kThreads;
    for (int q = 0; q < rounds; ++q) {
      const int i = q * kThreads + tid;
      const bool in = i < n && pred(i);
      const unsigned vote = __ballot_sync(0xffffffffu, in);
      if (!vote) continue;
      unsigned at = 0;
      if (lane == 0) at = atomicAdd(&first.list_n, static_cast<unsigned>(__popc(vote)));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(vote & ((1u << lane) - 1));
      if (in && at < kList) first.l.comp[at] = comp_at(i);
    }
    cluster.sync();
    int count = 0;
    if (rank == 0) {
      count = min(static_cast<int>(sh.list_n), kList);
      int pad = 2;
      while (pad < count) pad <<= 1;
      for (int i = count + tid; i < pad; i += kThreads) sh.l.comp[i] = ~0ull;
      __syncthreads();
      if (tid == 0) sh.list_n = 0;
      sort_list(sh, pad);
    }
    return count;
  };
  // Weight of list entry i.
  auto list_weight = [&](u64 comp) -> u64 {
    double y;
    return wt.bin(value_of(comp), &y) < 0 ? 0 : wt.weight(y);
  };

  // The order of the last element kept by top-k (mass false) or top-p, among
  // elements of order <= limit; ~0: all that have weight. With `whole` (a
  // count of at most kList) the elements down to the crossing go to the first
  // CTA's list instead, sorted, and their number is *listed there.
  auto search = [&](bool mass, unsigned count, u64 limit, bool whole, int* listed) -> u64 {
    clear_hist();
    for (int i = tid; i < n; i += kThreads) {
      if (limit != ~0ull && comp_at(i) > limit) continue;
      double y;
      const int b = bin_at(i, &y);
      if (b >= 0) add(b, mass ? wt.weight(y) : 0, mass);
    }
    Found f = find(mass, count, 0);
    if (!f.ok) {
      if (!whole) return limit;
      // Fewer than `count` elements have weight: all of them.
      *listed = gather([&](int i) {
        double y;
        return bin_at(i, &y) >= 0;
      });
      return limit;
    }
    const u64 target = f.bin_mass;
    const int bin = f.bin;
    unsigned above = f.above_cnt;
    u64 above_mass = f.above_mass;
    u64 lo = 0, hi = ~0ull;  // orders still in question, within the bin
    auto open = [&](int i) {
      double y;
      if (bin_at(i, &y) != bin) return false;
      const u64 o = comp_at(i);
      return o >= lo && o <= hi && o <= limit;
    };
    bool first = true;
    while ((whole ? above : 0) + f.bin_cnt > kList) {
      if (first) {
        // The bin's least and greatest order.
        u64 mn = ~0ull, mx = ~0ull;  // mx: the complement's least
        for (int i = tid; i < n; i += kThreads)
          if (open(i)) {
            const u64 o = comp_at(i);
            mn = min(mn, o);
            mx = min(mx, ~o);
          }
        mn = warp_min64(mn);
        mx = warp_min64(mx);
        __syncthreads();
        if (tid == 0) sh.lo = sh.hi = ~0ull;
        __syncthreads();
        if (lane == 0) {
          atomicMin(&sh.lo, mn);
          atomicMin(&sh.hi, mx);
        }
        cluster.sync();
        mn = mx = ~0ull;
        for (int r = 0; r < C; ++r) {
          mn = min(mn, peer(r).lo);
          mx = min(mx, peer(r).hi);
        }
        lo = mn;
        hi = ~mx;
        first = false;
      }
      const u64 span = hi - lo;
      const int bits = 64 - __clzll(static_cast<long long>(span));
      const int shift = max(0, bits - kSubBits);
      clear_hist();
      for (int i = tid; i < n; i += kThreads) {
        if (!open(i)) continue;
        double y;
        bin_at(i, &y);
        add(static_cast<int>((comp_at(i) - lo) >> shift), mass ? wt.weight(y) : 0, mass);
      }
      f = find(mass, count - above, mass ? target - above_mass : 0);
      above += f.above_cnt;
      above_mass += f.above_mass;
      lo += static_cast<u64>(f.bin) << shift;
      hi = min(hi, lo + (1ull << shift) - 1);
    }
    if (whole) {
      *listed = gather([&](int i) {
        double y;
        const int b = bin_at(i, &y);
        if (b < 0 || b > bin) return false;
        const u64 o = comp_at(i);
        return b < bin || (o <= hi && o <= limit);
      });
      return ~0ull;
    }
    const int got = gather(open);
    if (rank == 0) {
      u64 found = 0;
      if (mass) {
        // Two entries per thread.
        u64 w[2];
        unsigned none = 0, nt;
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * tid + e;
          w[e] = i < got ? list_weight(sh.l.comp[i]) : 0;
        }
        u64 at = w[0] + w[1], tot;
        block_scan(sh, none, at, &nt, &tot);
        at += above_mass;
        if (tid == 0) sh.threshold = sh.l.comp[max(got - 1, 0)];
        __syncthreads();
        for (int e = 0; e < 2; ++e) {
          if (at < target && at + w[e] >= target) {
            found = sh.l.comp[2 * tid + e];
            sh.threshold = found;
          }
          at += w[e];
        }
      } else if (tid == 0) {
        sh.threshold = sh.l.comp[min(static_cast<int>(count - above) - 1, got - 1)];
      }
    }
    cluster.sync();
    const u64 th = peer(0).threshold;
    cluster.sync();
    return min(th, limit);
  };

  auto finish = [&](int token, u64 w, u64 total) {
    a.tokens[row] = token;
    if (a.probs)
      a.probs[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(total));
  };

  if (k <= kList) {
    // The kept elements are few: the first CTA does the rest from its list.
    int listed = 0;
    search(false, k, ~0ull, true, &listed);
    if (rank == 0) {
      const int kept = min(listed, k);
      u64 w[2];
      unsigned none = 0, ntot;
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        w[e] = i < kept ? list_weight(sh.l.comp[i]) : 0;
      }
      u64 at = w[0] + w[1], total;
      block_scan(sh, none, at, &ntot, &total);
      const u64 target = top_p < 1.0f ? ceil_part(top_p, total) : ~0ull;
      // Those that stay, back in index order.
      int pad = 2;
      while (pad < kept) pad <<= 1;
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        if (i < pad) {
          const bool stays = i < kept && at < target && static_cast<double>(w[e]) >= min_w;
          const u64 idx = sh.l.comp[i] & 0xffffffffu;
          sh.l.comp[i] = stays ? (idx << 32) | i : ~0ull;
          sh.l.w[i] = w[e];
        }
        at += w[e];
      }
      __syncthreads();
      sort_list(sh, pad);
      u64 c[2];
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        c[e] = i < pad ? sh.l.comp[i] : ~0ull;
        w[e] = c[e] != ~0ull ? sh.l.w[c[e] & 0xffffffffu] : 0;
      }
      at = w[0] + w[1];
      none = 0;
      block_scan(sh, none, at, &ntot, &total);
      const u64 draw = floor_part(u, total);
      for (int e = 0; e < 2; ++e) {
        if (at <= draw && at + w[e] > draw) finish(static_cast<int>(c[e] >> 32), w[e], total);
        at += w[e];
      }
    }
    cluster.sync();
    return;
  }
  u64 limit = ~0ull;
  int listed;
  if (k != INT_MAX) limit = search(false, k, limit, false, &listed);
  if (top_p < 1.0f) limit = search(true, 0, limit, false, &listed);

  // The draw: every warp sums a run of consecutive elements, the one whose
  // run holds the drawn mass goes through it again.
  auto weight_at = [&](int i) -> u64 {
    if (limit != ~0ull && comp_at(i) > limit) return 0;
    double y;
    if (bin_at(i, &y) < 0) return 0;
    const u64 w = wt.weight(y);
    return static_cast<double>(w) >= min_w ? w : 0;
  };
  const int run = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int r0 = min(warp * run, n), r1 = min(r0 + run, n);
  u64 mine = 0;
  for (int i = r0 + lane; i < r1; i += 32) mine += weight_at(i);
  mine = warp_sum64(mine);
  __syncthreads();
  if (lane == 0) sh.red[warp] = mine;
  __syncthreads();
  u64 before = 0, total = 0;
  for (int wq = 0; wq < kWarps; ++wq) {
    if (wq < warp) before += sh.red[wq];
    total += sh.red[wq];
  }
  if (tid == 0) sh.part_mass = total;
  cluster.sync();
  total = 0;
  for (int r = 0; r < C; ++r) {
    const u64 p = peer(r).part_mass;
    if (r < rank) before += p;
    total += p;
  }
  const u64 draw = floor_part(u, total);
  if (before <= draw && draw < before + mine) {
    for (int i = r0; i < r1; i += 32) {
      const u64 w = i + lane < r1 ? weight_at(i + lane) : 0;
      u64 sum = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const bool hit = before + sum - w <= draw && draw < before + sum;
      if (hit) finish(i0 + i + lane, w, total);
      if (__any_sync(0xffffffffu, hit)) break;
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  cluster.sync();
}

constexpr int kShared = (sizeof(Shared) + 15) / 16 * 16;

template <class T>
void launch(const SampleArgs& a, int num_sms, cudaStream_t s) {
  // CTAs per row: enough that a slice fits shared memory, then more while
  // there are SMs without a row.
  int c = 1;
  while (c < kMaxCluster &&
         ((static_cast<int64_t>(a.vocab) + c - 1) / c * sizeof(T) > kSliceBytes ||
          static_cast<int64_t>(a.rows) * c * 2 <= num_sms))
    c *= 2;
  const int slice = (a.vocab + c - 1) / c * static_cast<int>(sizeof(T)) + 16;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kShared + (slice + 15) / 16 * 16;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
}

template <class T>
void set_smem() {
  cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       kShared + kSliceBytes + 32);
}

}  // namespace

int sample_max_vocab(int dtype) {
  // Slices in shared memory; and sums of 2^19 weights of 2^44 fit 64 bits.
  return std::min(kMaxCluster * kSliceBytes / (dtype == kOpF32 ? 4 : 2), 1 << 19);
}

void sample_setup_device() {
  set_smem<float>();
  set_smem<__half>();
  set_smem<__nv_bfloat16>();
}

void launch_sample(const SampleArgs& a, int num_sms, cudaStream_t s) {
  if (a.rows <= 0) return;
  if (a.dtype == kOpF32)
    launch<float>(a, num_sms, s);
  else if (a.dtype == kOpF16)
    launch<__half>(a, num_sms, s);
  else
    launch<__nv_bfloat16>(a, num_sms, s);
}

}  // namespace omg
