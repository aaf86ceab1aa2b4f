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
// bounds it; at a few tokens the chain of dependent loads does (sequence,
// length, page).
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

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0];
    const float4 b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
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

// A head takes HD / 16 threads, each 8 dims of its lower half and the 8 they
// are paired with; the block sweeps the heads of a token, all of them sharing
// the token's rotation in shared memory.
template <int HD, class TI, class TO>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(PagedAppendArgs a) {
  constexpr int L = HD / 16;
  constexpr int kUnits = kThreads / L;
  constexpr int HALF = HD / 2;
  __shared__ float2 rot[HALF];
  __shared__ long long s_row;  // cache row of the token, -1: none
  __shared__ int s_pos;        // its position
  __shared__ int s_live;
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x, lane = tid & 31;
  const int l = tid % L, u_in = tid / L;
  const int kvh = a.c.kv_heads;
  const int nh = a.heads + (a.has_kv ? 2 * kvh : 0);
  const TI* qkv = static_cast<const TI*>(a.qkv);
  TO* q_out = static_cast<TO*>(a.q_out);
  TO* cache = static_cast<TO*>(a.c.rows);
  for (int t = blockIdx.x; t < a.b.tokens; t += gridDim.x) {
    const TI* row = qkv + t * a.qkv_stride;
    if (tid < 32) {
      const int s = warp_count_le(a.b.q_start, a.b.n_seqs + 1, t, lane) - 1;
      const bool live = s >= 0 && s < a.b.n_seqs;
      int pos = 0;
      long long crow = -1;
      if (live) {
        const int own = a.b.lens[s] - (a.b.q_start[s + 1] - t);
        int prefix = 0;
        if (a.b.n_groups > 0) {
          const int g = warp_count_le(a.b.group_start, a.b.n_groups + 1, s, lane) - 1;
          if (g >= 0 && g < a.b.n_groups) prefix = a.b.prefix_lens[g];
        }
        pos = prefix + own;
        // A token without a place (a length below its query rows, a page
        // outside the table or the pool) leaves the cache as it was.
        const int pi = own >> a.c.page_log2;
        if (own >= 0 && pi < a.b.max_pages) {
          const int page = a.b.pages[static_cast<int64_t>(s) * a.b.max_pages + pi];
          if (page >= 0 && page < a.c.n_pages)
            crow = (static_cast<long long>(page) << a.c.page_log2) +
                   (own & ((1 << a.c.page_log2) - 1));
        }
      }
      if (lane == 0) {
        s_row = crow;
        s_pos = pos;
        s_live = live;
      }
    }
    __syncthreads();
    const bool live = s_live;
    const long long crow = s_row;
    if (live) {
      for (int d = tid; d < a.n_freq; d += kThreads) {
        const double turns = static_cast<double>(s_pos) * (a.inv_freq[d] * 0.15915494309189535);
        float sn, cs;
        sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn, &cs);
        rot[d] = make_float2(cs, sn);
      }
    }
    __syncthreads();
    for (int u0 = 0; live && u0 < nh; u0 += kUnits) {
      const int h = u0 + u_in;
      const bool on = h < nh;
      float x[8], y[8];
      if (on) {
        load8(row + h * HD + 8 * l, x);
        load8(row + h * HD + HALF + 8 * l, y);
      }
      const bool is_q = h < a.heads, is_v = h >= a.heads + kvh;
      const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (!on) continue;
      if (is_v ? a.v_norm : w != nullptr) {
        const float inv = rsqrtf(ss * (1.0f / HD) + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] *= inv;
          y[e] *= inv;
        }
      }
      if (!is_v) {
        if (w) {
          float wx[8], wy[8];
          load8(w + 8 * l, wx);
          load8(w + HALF + 8 * l, wy);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] *= a.norm_offset + wx[e];
            y[e] *= a.norm_offset + wy[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (8 * l + e < a.n_freq) {
            const float2 r = rot[8 * l + e];
            const float p = x[e] * r.x - y[e] * r.y;
            y[e] = y[e] * r.x + x[e] * r.y;
            x[e] = p;
          }
        }
      }
      if (is_q) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] *= a.q_scale;
          y[e] *= a.q_scale;
        }
        TO* o = q_out + t * a.q_stride + h * HD + 8 * l;
        store8(o, x);
        store8(o + HALF, y);
      } else if (crow >= 0) {
        TO* o = cache + crow * (2 * kvh * HD) + (h - a.heads) * HD + 8 * l;
        store8(o, x);
        store8(o + HALF, y);
      }
    }
    __syncthreads();
  }
}

template <int HD, class TI, class TO>
void launch(const PagedAppendArgs& a, int num_sms, cudaStream_t s) {
  const int grid = std::min(a.b.tokens, num_sms * 8);
  launch_pdl(paged_append_kernel<HD, TI, TO>, dim3(grid), dim3(kThreads), 0, s, a);
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
