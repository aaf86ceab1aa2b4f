// Append to a paged K/V cache (see paged.cuh): per token of the fused
// projection row [q heads | k heads | v heads]
//   q, k:  x * rsqrt(mean x^2 + eps) * (offset + w), then the first n_freq
//          pairs (d, d + hd/2) rotated by position * inv_freq[d]
//   v:     as is, or normalised without a weight
// q times q_scale goes to q_out, k and v to the cache row of the token's page
// (qk_prep.wgsl does the same into a contiguous cache,
// crates/omg-wgpu/src/shaders/qk_prep.wgsl:1-80).
//
// Each value is read and written once and costs about ten operations, so HBM
// bounds it: 12,000 tokens of 8 + 2 x 2 heads of 512 from f32 take 70.6 us,
// 6.3 TB/s; 16,384 bf16 tokens of 16 + 2 x 4 heads of 128 take 45.1 us, 4.5
// TB/s. At a few tokens the chain of dependent loads does (sequence, length,
// page): 3.2 us for one. The heads' values are fetched before that chain, as
// they lie in memory so that four blocks fit an SM (values widened at the load
// hold twice the registers: 66 us for those 16,384 tokens, when it was 50).
//
// Numerics: everything in f32 and one rounding to the 16-bit outputs, except
// the angle. position * inv_freq passes 2^17 radians in long contexts, where
// f32 leaves 2^-7 of a radian: the turn count is a 64-bit product of which
// only the fraction goes on in f32.
#include <algorithm>

#include "launch.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace omg {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 4;  // tokens of a block, at most

// Eight values as they lie in memory, and as f32.
template <class T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <class T>
__device__ __forceinline__ void to_f32(const Raw8<T>& r, float (&v)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[2 * i] = __uint_as_float(w[2 * i]);
      v[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
    } else {
      float2 f;
      if constexpr (std::is_same<T, __half>::value)
        f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      else
        f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// A block takes `tb` tokens: a warp looks up each token's sequence, cache row
// and position, the block computes their rotations into shared memory, then
// sweeps their heads. A head takes HD / 16 threads, each 8 dims of its lower
// half and the 8 they are paired with.
template <int HD, class TI, class TO>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(PagedAppendArgs a, int tb) {
  constexpr int L = HD / 16;
  constexpr int kUnits = kThreads / L;
  constexpr int HALF = HD / 2;
  __shared__ float2 rot[kMaxTokens][HALF];  // dim 8 l + e at e L + l: no bank conflicts
  __shared__ long long s_row[kMaxTokens];  // cache row of the token, -1: none
  __shared__ int s_pos[kMaxTokens];        // its position
  __shared__ int s_live[kMaxTokens];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int l = tid % L, u_in = tid / L;
  const int kvh = a.c.kv_heads;
  const int nh = a.heads + (a.has_kv ? 2 * kvh : 0);
  const int t0 = blockIdx.x * tb, nt = min(tb, a.b.tokens - t0);
  const TI* qkv = static_cast<const TI*>(a.qkv) + t0 * a.qkv_stride;
  TO* q_out = static_cast<TO*>(a.q_out) + t0 * a.q_stride;
  TO* cache = static_cast<TO*>(a.c.rows);
  griddep_wait();
  griddep_launch();
  // The first heads' values are on their way while the tokens are looked up.
  Raw8<TI> x{}, y{};
  int u = u_in, tok = u / nh, h = u - tok * nh;
  auto fetch = [&]() {
    if (tok < nt) {
      const TI* row = qkv + tok * a.qkv_stride + h * HD + 8 * l;
      x = load8(row);
      y = load8(row + HALF);
    }
  };
  fetch();
  const double freq0 = tid < nt * a.n_freq ? a.inv_freq[tid % a.n_freq] : 0.0;
  if (warp < nt) {
    const int t = t0 + warp;
    const int s = warp_count_le(a.b.q_start, a.b.n_seqs + 1, t, lane) - 1;
    const bool live = s >= 0 && s < a.b.n_seqs;
    int pos = 0;
    long long crow = -1;
    if (live) {
      const int own = a.b.lens[s] - (a.b.q_start[s + 1] - t);
      // A token without a place (a length below its query rows, a page
      // outside the table or the pool) leaves the cache as it was.
      const int pi = own >> a.c.page_log2;
      int page = -1, prefix = 0;
      if (own >= 0 && pi < a.b.max_pages)
        page = a.b.pages[static_cast<int64_t>(s) * a.b.max_pages + pi];
      if (a.b.n_groups > 0) {
        const int g = warp_count_le(a.b.group_start, a.b.n_groups + 1, s, lane) - 1;
        if (g >= 0 && g < a.b.n_groups) prefix = a.b.prefix_lens[g];
      }
      pos = prefix + own;
      if (page >= 0 && page < a.c.n_pages)
        crow = (static_cast<long long>(page) << a.c.page_log2) +
               (own & ((1 << a.c.page_log2) - 1));
    }
    if (lane == 0) {
      s_row[warp] = crow;
      s_pos[warp] = pos;
      s_live[warp] = live;
    }
  }
  __syncthreads();
  for (int i = tid; i < nt * a.n_freq; i += kThreads) {
    const int k = i / a.n_freq, d = i - k * a.n_freq;
    const double turns = static_cast<double>(s_pos[k]) * ((i == tid ? freq0 : a.inv_freq[d]) * 0.15915494309189535);
    float sn, cs;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn, &cs);
    rot[k][(d & 7) * L + (d >> 3)] = make_float2(cs, sn);
  }
  __syncthreads();
  for (int u0 = 0; u0 < nt * nh; u0 += kUnits) {
    const int ht = h, tt = tok;
    const bool on = tt < nt && s_live[min(tt, kMaxTokens - 1)];
    const bool is_q = ht < a.heads, is_v = ht >= a.heads + kvh;
    const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    float v[8], z[8];
    float ss = 0.f;
    to_f32(x, v);
    to_f32(y, z);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += v[e] * v[e] + z[e] * z[e];
    // The next heads' values.
    u += kUnits;
    tok = u / nh;
    h = u - tok * nh;
    fetch();
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!on) continue;
    if (is_v ? a.v_norm : w != nullptr) {
      const float inv = rsqrtf(ss * (1.0f / HD) + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] *= inv;
        z[e] *= inv;
      }
    }
    if (!is_v) {
      if (w) {
        float wv[8], wz[8];
        to_f32(load8(w + 8 * l), wv);
        to_f32(load8(w + HALF + 8 * l), wz);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] *= a.norm_offset + wv[e];
          z[e] *= a.norm_offset + wz[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (8 * l + e < a.n_freq) {
          const float2 r = rot[tt][e * L + l];
          const float p = v[e] * r.x - z[e] * r.y;
          z[e] = z[e] * r.x + v[e] * r.y;
          v[e] = p;
        }
      }
    }
    if (is_q) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] *= a.q_scale;
        z[e] *= a.q_scale;
      }
      TO* o = q_out + tt * a.q_stride + ht * HD + 8 * l;
      store8(o, v);
      store8(o + HALF, z);
    } else if (s_row[tt] >= 0) {
      TO* o = cache + s_row[tt] * (2 * kvh * HD) + (ht - a.heads) * HD + 8 * l;
      store8(o, v);
      store8(o + HALF, z);
    }
  }
}

template <int HD, class TI, class TO>
void launch(const PagedAppendArgs& a, int num_sms, cudaStream_t s) {
  // Tokens per block: the lookups and barriers are paid once for all of them,
  // but few blocks leave SMs idle. us with 1, 2, 4, 8 tokens, 8 + 2 x 2 heads
  // of 512 from f32: 60 tokens 4.4, 5.1, 7.2, 11.7; 288 tokens 5.0, 5.3, 7.3,
  // 11.9; 720 tokens 10.0, 8.7, 9.1, 12.0; 3,000 tokens 25.8, 22.3, 24.1, 27.2;
  // 12,000 tokens 88.7, 74.0, 71.0, 73.2. 16 + 2 x 4 bf16 heads of 128: 512
  // tokens 4.6, 4.7, 4.9, 6.9; 1,024 tokens 7.1, 5.9, 5.7, 7.0; 6,503 tokens
  // 30.5, 24.1, 19.1, 19.0; 16,384 tokens 72.5, 57.6, 45.2, 42.5. (8 gains at
  // the last alone and needs twice the shared memory.)
  const int tb = a.b.tokens <= num_sms ? 1 : a.b.tokens <= 5 * num_sms ? 2 : kMaxTokens;
  launch_pdl(paged_append_kernel<HD, TI, TO>, dim3((a.b.tokens + tb - 1) / tb), dim3(kThreads), 0, s,
             a, tb);
}

template <int HD>
void launch_types(const PagedAppendArgs& a, int num_sms, cudaStream_t s) {
  if (a.c.dtype == kOpF16) {
    if (a.qkv_dtype == kOpF32)
      launch<HD, float, __half>(a, num_sms, s);
    else
      launch<HD, __half, __half>(a, num_sms, s);
  } else {
    if (a.qkv_dtype == kOpF32)
      launch<HD, float, __nv_bfloat16>(a, num_sms, s);
    else
      launch<HD, __nv_bfloat16, __nv_bfloat16>(a, num_sms, s);
  }
}

}  // namespace

void launch_paged_append(const PagedAppendArgs& a, int num_sms, cudaStream_t s) {
  if (a.b.tokens <= 0) return;
  switch (a.c.hd) {
    case 64: return launch_types<64>(a, num_sms, s);
    case 128: return launch_types<128>(a, num_sms, s);
    case 256: return launch_types<256>(a, num_sms, s);
    default: return launch_types<512>(a, num_sms, s);
  }
}

}  // namespace omg
