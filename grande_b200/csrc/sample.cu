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
// 64-bit integers in units of 2^-43 of the largest, from a 64-bit exp2, so all
// sums are exact and the same in any order, atomics included.
//
// Bound: one read of the logits at HBM rate is the floor; above it stand a
// sweep per step and, where no top-k cuts the row first, the 64-bit
// exponential of every element: 30 to 40 issue slots each, f64, integer and
// compare instructions at half rate. 128 rows of 262,144 f32, top-p: 124 us,
// 1.1 TB/s (a first read 14 us, counts 24, exponentials and sums 58, the rest
// the searches between); 64 rows of 56,000 bf16, settings of all kinds: 39 us;
// 5 rows of 25,000 with a top-k: 14 us, the steps' barriers. Slices up to
// kSliceBytes stay in shared memory, longer ones are read again: 128 rows of
// 56,000 bf16 41.0 us against 42.5, 5 rows of 262,144 34.9 against 36.9.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "ptx.cuh"
#include "sample.cuh"

namespace omg {

namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;
// The kernel is one body of lambdas; left to itself the compiler calls some
// of them, with their captures in local memory.
#define INLINE __attribute__((always_inline))

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2944;      // log2 w from 0 to -46 in steps of 1/64
constexpr int kList = 2048;      // elements the first CTA sorts
constexpr int kScale = 43;       // weights in units of 2^-43
constexpr int kMaxCluster = 16;
constexpr int kSliceBytes = 160 * 1024;     // of a row in a CTA's shared memory
constexpr int kEach = kList / kThreads;     // list entries per thread
constexpr int kRankSort = 256;              // lists up to this are sorted by counting
constexpr u64 kDropped = 1ull << 63;        // list entries that a filter took out
constexpr int kSubBits = 11;  // refinement: up to 2^11 bins of the (value, index) order

enum { kCount, kMass, kGuess };  // what a histogram's search sums

// The crossing bin of a search: what lies before it, what it holds, and the
// target (counts or masses).
struct Found {
  int ok, bin;
  u64 above, here, target;
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
    float queue[kWarps][8][32];  // the draw: each lane's kept values to weigh
  };
  double table[kBins];
  u64 red[kWarps];
  unsigned redc[kWarps];
  float redf[kWarps];
  u64 runs[kWarps], above[kWarps];
  int window_lo, window_hi;
  // Read by the other CTAs of the cluster.
  u64 part_mass, part_above, lo, hi;
  float top, part_sq;
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

// Bin and weight of a value. The bin is -64 log2 w rounded, in f32: monotone
// in the value, which is all that the search needs of it. The weight is
// 2^43 w rounded, from 64 bits: 2^(43 - bin / 64) from a table and
// 2^(r / 64), r what the bin's rounding left (|r| < 0.51), a polynomial of
// degree 4 in (ln 2 / 64)^k / k! r^k, good to 2^-44 of the weight.
__device__ __forceinline__ u64 whole_number(double x) { return __double2ull_rz(x); }

struct Weigher {
  float half, c128;     // half of the row's largest; 2 * 64 log2(e) / T
  double bestd, c64d;
  const double* table;

  static constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: units of 1
  // The bin as kMagic - bin; a weight below 2^-45.5 lies below kLast.
  static constexpr int kLastBin = 2912;
  static constexpr float kLast = kMagic - kLastBin;
  static constexpr float kFloor = kMagic - (kBins - 1);
  // Differences of halves: those of f32's largest values are finite, too.
  __device__ __forceinline__ float mark(float x) const {
    return fmaf(fmaf(x, 0.5f, -half), c128, kMagic);
  }
  static __device__ __forceinline__ int bin_of_mark(float m) {
    return 0x4B400000 - __float_as_int(m);
  }
  __device__ __forceinline__ int bin(float x) const {
    const float m = mark(x);
    return m >= kLast ? bin_of_mark(m) : -1;
  }
  __device__ __forceinline__ u64 weight(float x, unsigned bin) const {
    return weight(x, bin, table[bin]);
  }
  // The weight as a double, of a finite x and its mark, at least kFloor; the
  // table is 0 past kLastBin. (Integer instructions run at half the rate of
  // f32 ones, as f64 ones do: a sum of doubles below 2^53 costs half of a
  // 64-bit integer's, a maximum less than the selects it spares.)
  __device__ __forceinline__ double mass(float x, float m) const {
    const int bits = __float_as_int(m);
    const double db = 4503599627370496.0 + 0x4B400000 - __hiloint2double(0x43300000, bits);
    return power(x, db, table[0x4B400000 - bits]) - 4503599627370496.0;
  }
  // `b`: 2^(43 - bin / 64), the table's entry.
  __device__ __forceinline__ u64 weight(float x, unsigned bin, double b) const {
    // The bin as a double, through the low bits of 2^52.
    const double db = __hiloint2double(0x43300000, bin) - 4503599627370496.0;
    const double w = power(x, db, b);
    return (static_cast<u64>(__double2hiint(w) - 0x43300000) << 32) |
           static_cast<unsigned>(__double2loint(w));
  }
  // The weight + 2^52: rounded, its bits in the low word.
  __device__ __forceinline__ double power(float x, double db, double b) const {
    const double r = fma(static_cast<double>(x) - bestd, c64d, db);
    constexpr double l = 1.0830424696249145e-2;  // ln 2 / 64
    double p = fma(r, l * l * l * l / 24, l * l * l / 6);
    p = fma(p, r, l * l / 2);
    p = fma(p, r, l);
    return fma(b * r, p, b) + 4503599627370496.0;
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
    unsigned a = lane < kWarps ? sh.redc[lane] : 0;
    u64 b = lane < kWarps ? sh.red[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned a2 = __shfl_up_sync(0xffffffffu, a, o);
      const u64 b2 = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) {
        a += a2;
        b += b2;
      }
    }
    if (lane < kWarps) {
      sh.redc[lane] = a;
      sh.red[lane] = b;
    }
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

// Sort sh.l.comp[0 .. n) ascending, all distinct; n <= kList. Short lists by
// counting the smaller entries (n^2 / 128 times 5 instructions: 256 entries
// 2,600 clocks, the bitonic sort of as many 36 barriers), longer ones
// bitonically, padded to a power of two.
__device__ void sort_list(Shared& sh, int n) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (n <= kRankSort) {
    static_assert(kRankSort <= kThreads, "an entry per thread");
    // Threads side by side share an entry's count: as many as there are.
    int share = 32;
    while (share * n > kThreads) share >>= 1;
    const int entry = tid / share, part = tid & (share - 1);
    const u64 mine = entry < n ? sh.l.comp[entry] : ~0ull;
    int at = 0;
    if (entry < n) {
#pragma unroll 4
      for (int i = part; i < n; i += share) at += sh.l.comp[i] < mine;
    }
    for (int o = share >> 1; o > 0; o >>= 1) at += __shfl_xor_sync(0xffffffffu, at, o);
    __syncthreads();
    if (entry < n && part == 0) sh.l.comp[at] = mine;
    __syncthreads();
    return;
  }
  int pad = 2;
  while (pad < n) pad <<= 1;
  for (int i = n + tid; i < pad; i += kThreads) sh.l.comp[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= pad; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = tid; i < pad / 2; i += kThreads) {
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

template <class T, bool STAGED>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto peer = [&](int r) INLINE -> Shared& { return *cluster.map_shared_rank(&sh, r); };

  // This CTA's slice [i0, i0 + n) of the row, in blocks of 16 aligned bytes:
  // block j holds elements j kVec - lead and on; those outside the slice read
  // as -infinity, which nothing keeps.
  const int per = (a.vocab + C - 1) / C;
  const int i0 = min(rank * per, a.vocab), n = min(per, a.vocab - i0);
  const T* src = static_cast<const T*>(a.logits) + (a.row_of ? a.row_of[row] : row) * a.stride + i0;
  constexpr int kVec = 16 / sizeof(T);
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
  const int blocks = (lead + n + kVec - 1) / kVec;
  uint4* staged = reinterpret_cast<uint4*>(smem + (sizeof(Shared) + 15) / 16 * 16);
  auto fetch_global = [&](int j) INLINE -> uint4 {
    const int at = j * kVec - lead;
    if (at >= 0 && at + kVec <= n) return *reinterpret_cast<const uint4*>(src + at);
    union {
      T e[kVec];
      uint4 v;
    } u;
#pragma unroll
    for (int q = 0; q < kVec; ++q)
      u.e[q] = at + q >= 0 && at + q < n ? src[at + q] : static_cast<T>(-INFINITY);
    return u.v;
  };
  // The row's settings come while the row does.
  const float temp = a.temperature ? a.temperature[row] : a.temperature1;
  int k = a.top_k ? a.top_k[row] : a.top_k1;
  float top_p = a.top_p ? a.top_p[row] : a.top_p1;
  float min_p = a.min_p ? a.min_p[row] : a.min_p1;
  const float u = fminf(fmaxf(a.u[row], 0.0f), 0.99999994f);
  // A row of one CTA needs no barrier but the block's.
  auto sync = [&]() INLINE {
    if (C == 1)
      __syncthreads();
    else
      cluster.sync();
  };
  if (tid == 0) {
    sh.list_n = 0;
    sh.threshold = ~0ull;
  }
  // Whole blocks [b0, b1); only the first and the last can be cut.
  const int b0 = lead ? 1 : 0, b1 = max(b0, (lead + n) / kVec);
  const uint4* whole = reinterpret_cast<const uint4*>(src - lead);
  float top = -INFINITY;  // fmaxf passes over NaN
  auto top_of = [&](const uint4& v) INLINE {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int q = 0; q < kVec; ++q) top = fmaxf(top, as_float(e[q]));
  };
  {
    int j = b0 + tid;
    for (; j + 3 * kThreads < b1; j += 4 * kThreads) {
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = whole[j + k * kThreads];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (STAGED) staged[j + k * kThreads] = v[k];
        top_of(v[k]);
      }
    }
    for (; j < b1; j += kThreads) {
      const uint4 v = whole[j];
      if (STAGED) staged[j] = v;
      top_of(v);
    }
    // The cut blocks.
    const int edge = tid == 0 && b0 ? 0 : tid == 1 && b1 < blocks ? b1 : -1;
    if (edge >= 0) {
      const uint4 v = fetch_global(edge);
      if (STAGED) staged[edge] = v;
      top_of(v);
    }
  }
  top = warp_max(top);
  if (lane == 0) sh.redf[warp] = top;
  __syncthreads();
  if (warp == 0) {
    top = warp_max(sh.redf[lane]);
    if (lane == 0) sh.top = top;
  }
  sync();
  top = warp_max(lane < C ? peer(lane).top : -INFINITY);

  min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
  if (k <= 0 || k >= a.vocab) k = INT_MAX;
  if (!(top_p < 1.0f)) top_p = 1.0f;
  const bool dead = top == -INFINITY;
  const bool infinite = top == INFINITY;  // the infinite elements share the row
  if (infinite) top = 0.0f;
  // One sweep: f(index of the first, kVec values) for every block of
  // [first, last), `step` threads side by side. Rounds of whole blocks go
  // without checks, U at a time with their loads ahead; the rest is checked.
  // Whole warps stay together: blocks that are not there are -infinity.
  auto unpack = [&](const uint4& b, float (&v)[kVec]) INLINE {
    const T* e = reinterpret_cast<const T*>(&b);
#pragma unroll
    for (int q = 0; q < kVec; ++q) v[q] = as_float(e[q]);
    if (infinite) {
#pragma unroll
      for (int q = 0; q < kVec; ++q) v[q] = v[q] == INFINITY ? 0.0f : -INFINITY;
    }
  };
  auto sweep_run = [&](int first, int last, int step, auto unroll, auto f) INLINE {
    constexpr int U = decltype(unroll)::value;
    const int me = step == 32 ? lane : tid;
    const int lo = max(first, min(b0, last)), hi = max(lo, min(last, b1));
    const int rounds = (hi - lo) / step / U;
    const uint4* p = (STAGED ? staged : whole) + lo + me;
    int i = i0 + (lo + me) * kVec - lead;
#pragma unroll 1
    for (int r = 0; r < rounds; ++r) {
      uint4 b[U];
#pragma unroll
      for (int k = 0; k < U; ++k) b[k] = p[k * step];
      p += U * step;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        float v[kVec];
        unpack(b[k], v);
        f(i, v);
        i += step * kVec;
      }
    }
    // What is cut or left over: blocks [first, lo) and [at, last).
    const int at = lo + rounds * U * step, count = (lo - first) + (last - at);
#pragma unroll 1
    for (int q0 = 0; q0 < count; q0 += step) {
      const int q = q0 + me;
      const int j = q < lo - first ? first + q : at + q - (lo - first);
      float v[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = -INFINITY;
      if (q < count) unpack(STAGED ? staged[j] : fetch_global(j), v);
      f(i0 + j * kVec - lead, v);
    }
  };
  auto sweep = [&](auto unroll, auto f) INLINE { sweep_run(0, blocks, kThreads, unroll, f); };
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 4> light{};
  constexpr std::integral_constant<int, kVec == 4 ? 2 : 1> heavy{};

  if (dead || !(temp > 0.0f) || k == 1 || top_p <= 0.0f) {
    // The largest alone. (Every CTA of the cluster takes the same branches.)
    unsigned at = UINT_MAX;
    if (!dead)
      sweep(light, [&](int i, const float(&v)[kVec]) INLINE {
#pragma unroll
        for (int q = 0; q < kVec; ++q)
          if (v[q] == top) at = min(at, static_cast<unsigned>(i + q));
      });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) sh.redc[warp] = at;
    __syncthreads();
    if (warp == 0) {
      at = __reduce_min_sync(0xffffffffu, sh.redc[lane]);
      if (lane == 0) sh.part_cnt = at;
    }
    sync();
    if (rank == 0 && warp == 0) {
      at = __reduce_min_sync(0xffffffffu, lane < C ? peer(lane).part_cnt : UINT_MAX);
      if (lane == 0) {
        a.tokens[row] = dead ? -1 : static_cast<int>(at);
        if (a.probs) a.probs[row] = dead ? 0.0f : 1.0f;
      }
    }
    sync();  // no CTA leaves while another may read its memory
    return;
  }
  Weigher wt;
  wt.half = 0.5f * top;
  wt.bestd = top;
  // Finite for the least temperatures, too: the largest itself is in bin 0.
  wt.c64d = fmin(64 * 1.4426950408889634 / static_cast<double>(temp), 1e38);
  wt.c128 = static_cast<float>(2 * wt.c64d);
  wt.table = sh.table;
  const double min_w = static_cast<double>(min_p) * static_cast<double>(1ull << kScale);
  auto bin_of = [&](float v) INLINE { return wt.bin(v); };
  auto weight_of = [&](float v, int b) INLINE { return wt.weight(v, b); };

  // Histograms of one sweep over the slice, counts or masses.
  auto clear_hist = [&](bool mass) INLINE {
    for (int i = tid; i < kBins; i += kThreads) {
      if (mass)
        sh.h.lo[i] = sh.h.hi[i] = 0;
      else
        sh.h.cnt[i] = 0;
    }
    if (tid == 0) sh.found.ok = 0;
    __syncthreads();
  };
  auto add = [&](int bin, u64 w, bool mass) INLINE {
    if (mass) {
      // 64 bits from two 32-bit atomics: whoever wraps the low word carries.
      const unsigned lo = static_cast<unsigned>(w);
      const unsigned old = atomicAdd(&sh.h.lo[bin], lo);
      const unsigned hi = static_cast<unsigned>(w >> 32) + (old + lo < old ? 1u : 0u);
      if (hi) atomicAdd(&sh.h.hi[bin], hi);
    } else {
      atomicAdd(&sh.h.cnt[bin], 1u);
    }
  };
  // The first bin at which the running sum (of counts or masses) reaches
  // `target`; 0: top_p of the mass. kGuess: masses as counts times the bin's
  // weight; *tol is about three deviations of what that misses.
  auto find = [&](int of, u64 target, u64* tol) INLINE -> Found {
    const bool mass = of == kMass;
    sync();
    const int share = kBins / C;  // C divides it
    const int each = (share + kThreads - 1) / kThreads;
    constexpr int kMost = (kBins + kThreads - 1) / kThreads;
    // This thread's bins, from every CTA: all loads in flight together (a
    // load from a peer takes several hundred clocks).
    u64 m[kMost];
    u64 mt = 0;
    if (C == 1) {
#pragma unroll
      for (int e = 0; e < kMost; ++e) {
        const int b = tid * each + e;
        m[e] = e < each && b < share
                   ? (mass ? (static_cast<u64>(sh.h.hi[b]) << 32) + sh.h.lo[b] : sh.h.cnt[b])
                   : 0;
        mt += m[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < kMost; ++e) {
        m[e] = 0;
        const int b = tid * each + e;
        if (e < each && b < share) {
          const int g = rank * share + b;
#pragma unroll 1
          for (int r0 = 0; r0 < C; r0 += 8) {
            unsigned lo[8], hi[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              lo[r] = hi[r] = 0;
              if (r0 + r < C) {
                const Shared& p = peer(r0 + r);
                lo[r] = mass ? p.h.lo[g] : p.h.cnt[g];
                if (mass) hi[r] = p.h.hi[g];
              }
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) m[e] += (static_cast<u64>(hi[r]) << 32) + lo[r];
          }
        }
        mt += m[e];
      }
    }
    if (of == kGuess) {
      float sq = 0.0f;
      mt = 0;
#pragma unroll
      for (int e = 0; e < kMost; ++e) {
        const int b = tid * each + e;
        if (e < each && b < share)
          m[e] = static_cast<u64>(static_cast<double>(m[e]) * sh.table[rank * share + b]);
        const float x = static_cast<float>(m[e]);
        sq = fmaf(x, x, sq);
        mt += m[e];
      }
      sq = warp_sum(sq);
      if (lane == 0) sh.redf[warp] = sq;
    }
    unsigned none = 0, ntot;
    u64 mx = mt, mtot;
    block_scan(sh, none, mx, &ntot, &mtot);
    if (of == kGuess && warp == 0) {
      const float sq = warp_sum(sh.redf[lane]);
      if (lane == 0) sh.part_sq = sq;
    }
    if (tid == 0) sh.part_mass = mtot;
    sync();
    const u64 part = lane < C ? peer(lane).part_mass : 0;
    const u64 all = warp_sum64(part);
    if (of == kGuess) {
      const float sq = warp_sum(lane < C ? peer(lane).part_sq : 0.0f);
      *tol = static_cast<u64>(0.0094f * sqrtf(sq) + 5e-5f * static_cast<float>(all));
    }
    mx += warp_sum64(lane < rank ? part : 0);
    if (target == 0) target = ceil_part(top_p, all);
#pragma unroll
    for (int e = 0; e < kMost; ++e) {
      if (mx < target && mx + m[e] >= target) {
        Found f;
        f.ok = 1;
        f.bin = rank * share + tid * each + e;
        f.above = mx;
        f.here = m[e];
        f.target = target;
        for (int r = 0; r < C; ++r) peer(r).found = f;
      }
      mx += m[e];
    }
    sync();
    const Found f = sh.found;
    __syncthreads();  // read by all before the next sweep clears it
    return f;
  };
  // Elements of `pred(value, index)` (at most kList in the cluster) into the
  // first CTA's list, sorted there; returns their number there, 0 elsewhere.
  // `maybe(mark)` is a cheap test that they all pass; most warps go on from it.
  auto gather = [&](auto maybe, auto pred) INLINE -> int {
    Shared& first = peer(0);
    sweep(light, [&](int i, const float(&v)[kVec]) INLINE {
      bool any = false;
#pragma unroll
      for (int q = 0; q < kVec; ++q) any |= maybe(wt.mark(v[q]));
      if (!__any_sync(0xffffffffu, any)) return;
      unsigned in = 0;
#pragma unroll
      for (int q = 0; q < kVec; ++q)
        if (pred(v[q], i + q)) in |= 1u << q;
      unsigned upto = __popc(in);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      unsigned at = 0;
      if (lane == 31) at = atomicAdd(&first.list_n, upto);
      at = __shfl_sync(0xffffffffu, at, 31) + upto - __popc(in);
#pragma unroll
      for (int q = 0; q < kVec; ++q)
        if ((in >> q) & 1) {
          if (at < kList) first.l.comp[at] = order_of(v[q], i + q);
          ++at;
        }
    });
    sync();
    int count = 0;
    if (rank == 0) {
      count = min(static_cast<int>(sh.list_n), kList);
      sort_list(sh, count);
      if (tid == 0) sh.list_n = 0;
    }
    return count;
  };
  auto list_weight = [&](u64 comp) INLINE -> u64 {
    const float v = value_of(comp);
    const int b = bin_of(v);
    return b < 0 ? 0 : wt.weight(v, b, exp2(kScale - b / 64.0));
  };

  // Finds the last element that top-k (mass false, `count`) or top-p keeps
  // among those of order at most `limit`. If all the elements down to it fit
  // the list, they are in the first CTA's list, sorted, and *listed their
  // number there (top-k up to kList: always); otherwise *listed is -1 and its
  // order comes back (~0: every element with weight).
  auto search = [&](bool mass, unsigned count, u64 limit, int* listed, u64* goal) INLINE -> u64 {
    *listed = -1;
    clear_hist(mass);
    auto tally = [&](int i, const float(&v)[kVec], bool limited) INLINE {
#pragma unroll
      for (int q0 = 0; q0 < kVec; q0 += 4) {
        // Four weights first: their 64-bit chains overlap.
        unsigned b[4];
        bool on[4];
        u64 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float m = wt.mark(v[q0 + q]);
          on[q] = m >= Weigher::kLast;
          b[q] = on[q] ? Weigher::bin_of_mark(m) : 0;
          if (limited) on[q] = on[q] && order_of(v[q0 + q], i + q0 + q) <= limit;
          w[q] = mass ? weight_of(v[q0 + q], b[q]) : 0;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (on[q]) add(b[q], w[q], mass);
      }
    };
    if (limit == ~0ull)
      sweep(heavy, [&](int i, const float(&v)[kVec]) INLINE { tally(i, v, false); });
    else
      sweep(one, [&](int i, const float(&v)[kVec]) INLINE { tally(i, v, true); });
    Found f = find(mass ? kMass : kCount, mass ? 0 : count, nullptr);
    const u64 target = f.target;
    *goal = target;
    const int bin = f.bin;
    const float bin_mark = Weigher::kMagic - static_cast<float>(bin);
    if (!f.ok) {
      // Fewer than `count` elements have weight.
      if (count <= kList) *listed = gather([&](float m) INLINE { return m >= Weigher::kLast; },
                                        [&](float v, int) INLINE { return bin_of(v) >= 0; });
      return limit;
    }
    u64 above = f.above;
    // Bounds on numbers of elements: of a mass, it over its least weight.
    const u64 least = mass ? max(1ull, static_cast<u64>(exp2(kScale - (bin + 1.0) / 64))) : 1;
    if ((above + f.here) / least <= kList) {
      *listed = gather([&](float m) INLINE { return m >= bin_mark; }, [&](float v, int i) INLINE {
        const int b = bin_of(v);
        return b >= 0 && b <= bin && (limit == ~0ull || order_of(v, i) <= limit);
      });
      return limit;
    }
    u64 lo = 0, hi = ~0ull;  // orders still in question, within the bin
    auto open = [&](float v, int i) INLINE {
      if (wt.mark(v) != bin_mark) return false;
      const u64 o = order_of(v, i);
      return o >= lo && o <= hi && o <= limit;
    };
    const bool few = !mass && count <= kList;  // the list is to hold all of them
    bool first = true;
    while ((few ? above + f.here : f.here) / least > kList) {
      if (first) {
        // The bin's least and greatest order.
        u64 mn = ~0ull, mx = ~0ull;  // mx: the complement's least
        sweep(one, [&](int i, const float(&v)[kVec]) INLINE {
#pragma unroll
          for (int q = 0; q < kVec; ++q)
            if (open(v[q], i + q)) {
              const u64 o = order_of(v[q], i + q);
              mn = min(mn, o);
              mx = min(mx, ~o);
            }
        });
        mn = warp_min64(mn);
        mx = warp_min64(mx);
        __syncthreads();
        if (tid == 0) sh.lo = sh.hi = ~0ull;
        __syncthreads();
        if (lane == 0) {
          atomicMin(&sh.lo, mn);
          atomicMin(&sh.hi, mx);
        }
        sync();
        lo = warp_min64(lane < C ? peer(lane).lo : ~0ull);
        hi = ~warp_min64(lane < C ? peer(lane).hi : ~0ull);
        first = false;
      }
      if (lo == hi) break;  // one element is left, however heavy
      const u64 span = hi - lo;
      const int bits = 64 - __clzll(static_cast<long long>(span));
      const int shift = max(0, bits - kSubBits);
      clear_hist(mass);
      sweep(one, [&](int i, const float(&v)[kVec]) INLINE {
#pragma unroll
        for (int q = 0; q < kVec; ++q)
          if (open(v[q], i + q))
            add(static_cast<int>((order_of(v[q], i + q) - lo) >> shift),
                mass ? weight_of(v[q], bin) : 0, mass);
      });
      f = find(mass ? kMass : kCount, target - above, nullptr);
      above += f.above;
      lo += static_cast<u64>(f.bin) << shift;
      hi = min(hi, lo + (1ull << shift) - 1);
    }
    if (few) {
      *listed = gather([&](float m) INLINE { return m >= bin_mark; }, [&](float v, int i) INLINE {
        const int b = bin_of(v);
        return b >= 0 && (b < bin || (b == bin && order_of(v, i) <= hi));
      });
      return limit;
    }
    const int got = gather([&](float m) INLINE { return m == bin_mark; }, open);
    if (rank == 0) {
      u64 w[kEach];
      u64 at = 0, tot;
      unsigned none = 0, nt;
      for (int e = 0; e < kEach; ++e) {
        const int i = kEach * tid + e;
        w[e] = i < got ? (mass ? list_weight(sh.l.comp[i]) : 1) : 0;
        at += w[e];
      }
      block_scan(sh, none, at, &nt, &tot);
      at += above;
      for (int e = 0; e < kEach; ++e) {
        if (at < target && at + w[e] >= target) sh.threshold = sh.l.comp[kEach * tid + e];
        at += w[e];
      }
    }
    sync();
    const u64 th = peer(0).threshold;
    sync();
    return th;
  };
  auto finish = [&](int token, u64 w, u64 total) INLINE {
    a.tokens[row] = token;
    if (a.probs)
      a.probs[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(total));
  };

  // From a sorted list in the first CTA of which the first `kept` that lie
  // before `target` of the running mass stay (0: top_p of the list's).
  auto finish_list = [&](int kept, u64 target) INLINE {
    u64 w[kEach];
    u64 at = 0, total;
    unsigned none = 0, ntot;
    for (int e = 0; e < kEach; ++e) {
      const int i = kEach * tid + e;
      w[e] = i < kept ? list_weight(sh.l.comp[i]) : 0;
      at += w[e];
    }
    block_scan(sh, none, at, &ntot, &total);
    if (target == 0) target = top_p < 1.0f ? ceil_part(top_p, total) : ~0ull;
    // Those that stay, back in index order.
    for (int e = 0; e < kEach; ++e) {
      const int i = kEach * tid + e;
      if (i < kept) {
        const bool stays = at < target && static_cast<double>(w[e]) >= min_w;
        const u64 idx = sh.l.comp[i] & 0xffffffffu;
        sh.l.comp[i] = (stays ? idx << 32 : kDropped) | i;
        sh.l.w[i] = w[e];
      }
      at += w[e];
    }
    __syncthreads();
    sort_list(sh, kept);
    u64 c[kEach];
    at = 0;
    for (int e = 0; e < kEach; ++e) {
      const int i = kEach * tid + e;
      c[e] = i < kept ? sh.l.comp[i] : ~0ull;
      w[e] = c[e] < kDropped ? sh.l.w[c[e] & 0xffffffffu] : 0;
      at += w[e];
    }
    none = 0;
    block_scan(sh, none, at, &ntot, &total);
    const u64 draw = floor_part(u, total);
    for (int e = 0; e < kEach; ++e) {
      if (at <= draw && at + w[e] > draw) finish(static_cast<int>(c[e] >> 32), w[e], total);
      at += w[e];
    }
  };

  // (Lists compute the few entries they need.)
  if (k > kList)
    for (int i = tid; i < kBins; i += kThreads)
      sh.table[i] = i <= Weigher::kLastBin ? exp2(kScale - i / 64.0) : 0.0;
  u64 limit = ~0ull, goal = 0;
  int listed = -1;
  bool summed = false;  // sh.runs holds the warps' kept mass
  const int run = (blocks + kWarps - 1) / kWarps;
  const int r0 = min(warp * run, blocks), r1 = min(r0 + run, blocks);

  // top-p of a whole row. Counts times the bins' weights say within about a
  // bin where the mass is reached; one sweep then sums all that is above that
  // window, per warp as the draw wants it, and lists what is in it. One
  // exponential per element instead of two, and no 64-bit atomics: 128 rows of
  // 262,144 124 us, the histogram of masses below 157. False: the guess was
  // wrong, or more elements are in the window than the list holds (many equal
  // logits).
  auto window_search = [&]() INLINE -> bool {
    clear_hist(false);
    sweep(light, [&](int, const float(&v)[kVec]) INLINE {
#pragma unroll
      for (int q = 0; q < kVec; ++q) {
        const float m = wt.mark(v[q]);
        if (m >= Weigher::kLast) atomicAdd(&sh.h.cnt[Weigher::bin_of_mark(m)], 1u);
      }
    });
    u64 tol = 0;
    const Found f = find(kGuess, 0, &tol);
    if (!f.ok) return false;
    if (warp == 0) {
      // Bins on both sides, a lane each, until they hold `tol` beyond the
      // target.
      auto count_of = [&](int b) INLINE -> unsigned {
        unsigned c = 0;
        if (b >= 0 && b < kBins)
          for (int r = 0; r < C; ++r) c += peer(r).h.cnt[b];
        return c;
      };
      auto reach = [&](int dir, u64 held, unsigned* count) INLINE -> int {
        const int b = f.bin + dir * (1 + lane);
        unsigned c = count_of(b);
        u64 m = c ? static_cast<u64>(c * sh.table[b]) : 0;
        u64 before = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += y;
        }
        const bool in = held + before - m < tol;
        *count += __reduce_add_sync(0xffffffffu, in ? c : 0u);
        return __popc(__ballot_sync(0xffffffffu, in));
      };
      unsigned count = count_of(f.bin);
      const int up = reach(-1, f.target - f.above, &count);
      const int down = reach(1, f.above + f.here - f.target, &count);
      if (lane == 0) {
        sh.window_lo = f.bin - up;
        sh.window_hi = count <= kList ? f.bin + down : -1;
      }
    }
    sync();  // the list takes the histograms' place
    if (sh.window_hi < 0) return false;
    const float top_mark = Weigher::kMagic - static_cast<float>(sh.window_lo);
    const float low_mark = fmaxf(Weigher::kMagic - static_cast<float>(sh.window_hi), Weigher::kLast);
    Shared& head = peer(0);
    double dall = 0, dabove = 0, dkept = 0;  // of at most 2^10 weights: below 2^53
    sweep_run(r0, r1, 32, heavy, [&](int i, const float(&v)[kVec]) INLINE {
#pragma unroll
      for (int q0 = 0; q0 < kVec; q0 += 2) {
        float m[2];
        double w[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          // The mark of the logit as it is: -infinity and NaN get the floor's,
          // and with it no weight, at every temperature. (The mark of a finite
          // stand-in does not at great ones.) x only keeps the product finite.
          const float x = fmaxf(v[q0 + q], -FLT_MAX);
          m[q] = fmaxf(wt.mark(v[q0 + q]), Weigher::kFloor);
          w[q] = wt.mass(x, m[q]);
        }
        bool any = false;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          dall += w[q];
          if (m[q] > top_mark) dabove += w[q];
          any |= m[q] <= top_mark && m[q] >= low_mark;
        }
        if (min_p > 0.0f) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (m[q] > top_mark && w[q] >= min_w) dkept += w[q];
        }
        if (any) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (m[q] <= top_mark && m[q] >= low_mark) {
              const unsigned at = atomicAdd(&head.list_n, 1u);
              if (at < kList) head.l.comp[at] = order_of(v[q0 + q], i + q0 + q);
            }
        }
      }
    });
    u64 all = warp_sum64(whole_number(dall)), above = warp_sum64(whole_number(dabove));
    const u64 kept = min_p > 0.0f ? warp_sum64(whole_number(dkept)) : above;
    if (lane == 0) {
      sh.red[warp] = all;
      sh.above[warp] = above;
      sh.runs[warp] = kept;
    }
    __syncthreads();
    all = warp_sum64(sh.red[lane]);
    above = warp_sum64(sh.above[lane]);
    if (tid == 0) {
      sh.part_mass = all;
      sh.part_above = above;
    }
    sync();
    if (rank == 0) {
      const u64 target = ceil_part(top_p, warp_sum64(lane < C ? peer(lane).part_mass : 0));
      u64 above_all = warp_sum64(lane < C ? peer(lane).part_above : 0);
      const int got = min(static_cast<int>(sh.list_n), kList);
      // Their masses by order, in kList steps of the orders' range, and the
      // few of the crossing step sorted.
      u64 c[kEach], w[kEach];
      u64 mn = ~0ull, mx = ~0ull;  // mx: the complement's least
      __syncthreads();
      for (int e = 0; e < kEach; ++e) {
        const int i = tid + e * kThreads;
        c[e] = i < got ? sh.l.comp[i] : ~0ull;
        w[e] = 0;
        sh.l.w[i] = 0;
        if (i < got) {
          const float v = value_of(c[e]);
          w[e] = weight_of(v, bin_of(v));
          mn = min(mn, c[e]);
          mx = min(mx, ~c[e]);
        }
      }
      mn = warp_min64(mn);
      mx = warp_min64(mx);
      if (lane == 0) {
        sh.red[warp] = mn;
        sh.above[warp] = mx;
      }
      if (tid == 0) sh.list_n = 0;
      __syncthreads();
      mn = warp_min64(sh.red[lane]);
      mx = ~warp_min64(sh.above[lane]);
      const int shift = max(0, 64 - __clzll(static_cast<long long>(mx - mn)) - kSubBits);
      static_assert(1 << kSubBits == kList, "a step per list entry");
      for (int e = 0; e < kEach; ++e)
        if (w[e]) atomicAdd(&sh.l.w[(c[e] - mn) >> shift], w[e]);
      __syncthreads();
      u64 m[kEach];
      u64 at = 0, tot;
      unsigned none = 0, nt;
      for (int e = 0; e < kEach; ++e) {
        m[e] = sh.l.w[kEach * tid + e];
        at += m[e];
      }
      if (tid == 0) sh.found.ok = 0;
      block_scan(sh, none, at, &nt, &tot);
      at += above_all;
      for (int e = 0; e < kEach; ++e) {
        if (at < target && at + m[e] >= target) {
          sh.found.ok = 1;
          sh.found.bin = kEach * tid + e;
          sh.found.above = at;
        }
        at += m[e];
      }
      __syncthreads();
      if (sh.found.ok) {  // (else the guess was wrong)
        for (int e = 0; e < kEach; ++e)
          if (w[e] && static_cast<int>((c[e] - mn) >> shift) == sh.found.bin)
            sh.l.comp[atomicAdd(&sh.list_n, 1u)] = c[e];
        __syncthreads();
        const int few = sh.list_n;
        sort_list(sh, few);
        at = 0;
        for (int e = 0; e < kEach; ++e) {
          const int i = kEach * tid + e;
          m[e] = i < few ? list_weight(sh.l.comp[i]) : 0;
          at += m[e];
        }
        none = 0;
        block_scan(sh, none, at, &nt, &tot);
        at += sh.found.above;
        for (int e = 0; e < kEach; ++e) {
          if (at < target && at + m[e] >= target) sh.threshold = sh.l.comp[kEach * tid + e];
          at += m[e];
        }
        if (tid == 0) sh.list_n = 0;
        __syncthreads();
      }
      // Those of the window that stay, to the runs that they lie in.
      for (int e = 0; e < kEach; ++e) {
        if (w[e] && c[e] <= sh.threshold && static_cast<double>(w[e]) >= min_w) {
          const int idx = static_cast<int>(c[e] & 0xffffffffu);
          const int r = idx / per, first = r * per;
          const int cut = static_cast<int>(
              (reinterpret_cast<uintptr_t>(src + first) & 15) / sizeof(T));
          const int all_blocks = (cut + min(per, a.vocab - first) + kVec - 1) / kVec;
          const int of_warp = (idx - first + cut) / kVec / ((all_blocks + kWarps - 1) / kWarps);
          atomicAdd(&peer(r).runs[of_warp], w[e]);
        }
      }
    }
    sync();
    limit = peer(0).threshold;
    sync();
    return limit != ~0ull;
  };
  if (k != INT_MAX) {
    limit = search(false, k, limit, &listed, &goal);
    if (listed >= 0) {
      if (rank == 0) finish_list(min(listed, k), 0);
      sync();
      return;
    }
  }
  if (top_p < 1.0f && k == INT_MAX) summed = window_search();
  if (top_p < 1.0f && !summed) {
    limit = search(true, UINT_MAX, limit, &listed, &goal);
    if (listed >= 0) {
      if (rank == 0) finish_list(listed, goal);
      sync();
      return;
    }
  }

  // The draw: every warp sums a run of consecutive blocks; the run that holds
  // the drawn mass is then shared out over all warps of its CTA and gone
  // through again. Lanes queue the values they keep and weigh them together
  // once one of them has more than 4; nothing is queued when all are kept.
  const float edge = limit == ~0ull ? -INFINITY : value_of(limit);
  const int edge_idx = static_cast<int>(limit & 0x7fffffffu);
  auto kept = [&](float v, int i) INLINE {
    // What lies before the last kept element has weight, as that one has.
    if (limit == ~0ull) return bin_of(v) >= 0;
    return v > edge || (v == edge && i <= edge_idx);
  };
  auto weigh = [&](float v) INLINE -> u64 {
    const u64 w = weight_of(v, bin_of(v));
    return static_cast<double>(w) >= min_w ? w : 0;
  };
  float* queue = sh.queue[warp][0];
  u64 mine = 0;
  int waiting = 0;
  auto flush = [&]() INLINE {
#pragma unroll 1
    for (int e = 0; __any_sync(0xffffffffu, e < waiting); ++e)
      if (e < waiting) mine += weigh(queue[e * 32 + lane]);
    waiting = 0;
  };
  __syncthreads();  // the queues take the histograms' place
  if (summed)
    ;
  else if (limit == ~0ull)
    sweep_run(r0, r1, 32, heavy, [&](int i, const float(&v)[kVec]) INLINE {
#pragma unroll
      for (int q = 0; q < kVec; ++q) mine += bin_of(v[q]) >= 0 ? weigh(v[q]) : 0;
    });
  else
    sweep_run(r0, r1, 32, heavy, [&](int i, const float(&v)[kVec]) INLINE {
#pragma unroll
      for (int q = 0; q < kVec; ++q) {
        if (kept(v[q], i + q)) queue[waiting++ * 32 + lane] = v[q];
        if (q % 4 == 3 && __any_sync(0xffffffffu, waiting > 4)) flush();
      }
    });
  flush();
  mine = summed ? sh.runs[warp] : warp_sum64(mine);
  if (lane == 0) sh.red[warp] = mine;
  __syncthreads();
  const u64 of_warp = sh.red[lane];
  u64 total = warp_sum64(of_warp);
  if (tid == 0) sh.part_mass = total;
  sync();
  const u64 part = lane < C ? peer(lane).part_mass : 0;
  u64 before = warp_sum64(lane < rank ? part : 0);
  const u64 here = total;
  total = warp_sum64(part);
  const u64 draw = floor_part(u, total);
  if (before <= draw && draw < before + here) {
    u64 scan = of_warp;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    const int whose = __ffs(__ballot_sync(0xffffffffu, draw < before + scan)) - 1;
    before += __shfl_sync(0xffffffffu, scan - of_warp, whose);
    const int s0 = min(whose * run, blocks), s1 = min(s0 + run, blocks);
    const int piece = (s1 - s0 + kWarps - 1) / kWarps;
    const int p0 = min(s0 + warp * piece, s1), p1 = min(p0 + piece, s1);
    u64 sum = 0;
    sweep_run(p0, p1, 32, one, [&](int i, const float(&v)[kVec]) INLINE {
#pragma unroll
      for (int q = 0; q < kVec; ++q) sum += kept(v[q], i + q) ? weigh(v[q]) : 0;
    });
    sum = warp_sum64(sum);
    __syncthreads();
    if (lane == 0) sh.red[warp] = sum;
    __syncthreads();
    before += warp_sum64(lane < warp ? sh.red[lane] : 0);
    if (before <= draw && draw < before + sum) {
      sweep_run(p0, p1, 32, one, [&](int i, const float(&v)[kVec]) INLINE {
        u64 w[kVec], all = 0;
#pragma unroll
        for (int q = 0; q < kVec; ++q) {
          w[q] = kept(v[q], i + q) ? weigh(v[q]) : 0;
          all += w[q];
        }
        u64 upto = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += y;
        }
        u64 at = before + upto - all;
#pragma unroll
        for (int q = 0; q < kVec; ++q) {
          if (at <= draw && draw < at + w[q]) finish(i + q, w[q], total);
          at += w[q];
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      });
    }
  }
  sync();
}

constexpr int kShared = (sizeof(Shared) + 15) / 16 * 16;

template <class T>
void launch(const SampleArgs& a, int num_sms, cudaStream_t s) {
  // CTAs per row: more while there are SMs without a row and 8 elements per
  // thread; below that the cluster's barriers cost more than the sweeps gain.
  // (5 rows of 25,000: 20.1, 18.5, 16.4, 16.4, 20.5 us with 1, 2, 4, 8, 16.)
  int c = 1;
  while (c < kMaxCluster && static_cast<int64_t>(a.rows) * c * 2 <= num_sms &&
         a.vocab > c * 8 * kThreads)
    c *= 2;
  const int slice = (a.vocab + c - 1) / c * static_cast<int>(sizeof(T)) + 16;
  const bool staged = slice <= kSliceBytes;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kShared + (staged ? (slice + 15) / 16 * 16 : 0);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (staged)
    cudaLaunchKernelEx(&cfg, sample_kernel<T, true>, a);
  else
    cudaLaunchKernelEx(&cfg, sample_kernel<T, false>, a);
}

static_assert(kShared + kSliceBytes + 16 <= 227 * 1024, "shared memory");

template <class T, bool STAGED>
void set_attributes() {
  cudaFuncSetAttribute(sample_kernel<T, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       kShared + (STAGED ? kSliceBytes + 16 : 0));
  cudaFuncSetAttribute(sample_kernel<T, STAGED>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}

}  // namespace

int sample_max_vocab() { return 1 << 19; }  // (sums by thread stay below 2^53)

void sample_setup_device() {
  set_attributes<float, true>();
  set_attributes<float, false>();
  set_attributes<__half, true>();
  set_attributes<__half, false>();
  set_attributes<__nv_bfloat16, true>();
  set_attributes<__nv_bfloat16, false>();
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
