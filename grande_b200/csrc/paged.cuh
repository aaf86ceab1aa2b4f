// Operators over a paged K/V cache: the append of projected rows (per-head
// norms, rotation, page lookup) and attention over shared prefixes.
//
// A cache is a pool of pages [n_pages][page rows][2 * kv_heads * hd], a row
// laid out as the engine's cache rows: kv_heads K heads, then kv_heads V
// heads. A sequence owns a list of pages holding its tokens in order; a group
// is a prefix with pages of its own and the consecutive sequences that
// continue from it, so own token i of a sequence sits at position
// prefix_len + i. All tables and lengths are device memory read by the
// kernels, so a captured graph follows them from step to step.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace omg {

enum OpType : int { kOpF16 = 0, kOpBf16 = 1, kOpF32 = 2 };

struct PagedBatch {
  const int* q_start;       // [n_seqs + 1] first query row of each sequence
  const int* lens;          // [n_seqs] own tokens, this call's included
  const int* pages;         // [n_seqs][max_pages]
  const int* group_start;   // [n_groups + 1] first sequence of each group
  const int* prefix_lens;   // [n_groups]
  const int* prefix_pages;  // [n_groups][max_prefix_pages]
  int n_seqs, n_groups;     // n_groups 0: no prefixes
  int max_pages, max_prefix_pages;
  int tokens;               // query rows; those from q_start[n_seqs] on are padding
};

struct PagedCache {
  void* rows;
  int64_t n_pages;
  int page_log2;  // rows per page = 1 << page_log2
  int kv_heads, hd;
  int dtype;      // kOpF16 or kOpBf16
};

struct PagedAppendArgs {
  PagedBatch b;
  PagedCache c;
  const void* qkv;       // [tokens] rows of (heads [+ 2 kv_heads]) * hd values
  int64_t qkv_stride;    // elements between rows
  int qkv_dtype;
  int heads;
  bool has_kv;           // false: q only (a layer that reads another layer's K/V)
  void* q_out;           // [tokens] rows of heads * hd
  int64_t q_stride;
  const float* q_norm;   // [hd] or null: no norm
  const float* k_norm;
  bool v_norm;
  float norm_offset, eps, q_scale;
  const double* inv_freq;  // [n_freq] radians per position, or null
  int n_freq;
};
void launch_paged_append(const PagedAppendArgs& a, int num_sms, cudaStream_t s);

// ---- attention ---------------------------------------------------------------
//
// A row tile is up to 128 / (query heads per KV head) consecutive query tokens
// of one group, all heads of one KV head: 128 query rows. It meets slots of 16
// keys: first its group's prefix, which all of its rows see, then the own keys
// of each of its sequences, which that sequence's rows see. Four slots in a
// row make a key tile, whosever they are; the key tiles of all (KV head, row
// tile) entries, in that order, form one line that the CTAs cut into equal
// ranges.

constexpr int kPagedTileRows = 128;
constexpr int kPagedTileKeys = 64;
constexpr int kPagedSlotKeys = 16;  // the K step of the P V product, the smallest page

// A run of slots of one row tile: its group's prefix, or one sequence's own
// keys.
struct alignas(16) PagedRun {
  int rt;          // row tile
  int slot0, n;    // slots [slot0, slot0 + n) of the row tile
  int key0;        // first key (a multiple of 16) of its list of pages
  int kend;        // keys of the list that exist (and, own: that any row sees)
  int rows;        // r0 | r1 << 16: the rows that see it
  int i0;          // own index of row r0's token
  int owner;       // the sequence; of a prefix ~group
};

struct alignas(16) PagedTile {
  int tok0, ntok;
  int prefix_len;
  int ntiles;        // key tiles
  int nruns, pad;
  int imin, imax;    // own indices of its rows
};

struct alignas(16) PagedPlan {
  int n_tiles;    // row tiles
  int line;       // units of one KV head
  int per;        // units per CTA
  int pad;
};

// Where a CTA's range of the line begins: tile `pos` of row tile `rt`, after
// `toll` more units of its toll.
struct alignas(16) PagedStart {
  int rt, pos, kv, toll;
};

struct PagedAttnArgs {
  PagedBatch b;
  PagedCache c;
  void* out;
  int64_t out_stride;
  int heads, hpg, tpt;  // query heads, per KV head, tokens per row tile
  int hpg_recip;        // ceil(2^16 / hpg): r / hpg = r hpg_recip >> 16 for r <= 128
  int window;           // 0: all keys
  float scale_log2;     // score scale x log2(e)
  // Workspace.
  PagedPlan* plan;
  PagedStart* starts;   // [ctas]
  PagedRun* runs;       // [max_tiles][tpt + 1]
  PagedTile* tiles;     // [max_tiles]
  float* part_o;        // [2 * ctas][128][hd]
  float2* part_ml;      // [2 * ctas][128]
  int max_tiles;
  int ctas;             // grid of the attention kernel
  bool one_tile;        // a single row tile, which every CTA plans for itself
};

// Row tiles of a call: fills hpg, tpt, max_tiles, one_tile of `a` from its batch
// and shape. False: more sequences and row tiles than the plan kernel holds, or
// a line of more than 2^29 key tiles.
bool paged_attention_shape(PagedAttnArgs* a);
// Then its grid, `ctas`; returns the workspace bytes.
size_t paged_attention_layout(PagedAttnArgs* a, int num_sms);
// Point the workspace members of `a` into `ws`.
void paged_attention_workspace(PagedAttnArgs* a, void* ws);
// Tensor maps: q, and the cache in boxes of a slot.
struct PagedMaps {
  CUtensorMap q, kv;
};
bool paged_attention_maps(const PagedAttnArgs& a, const void* q, int64_t q_stride, PagedMaps* m,
                          char* err, size_t errlen);
void launch_paged_attention(const PagedAttnArgs& a, const PagedMaps& m, cudaStream_t s);
// Shared-memory limits of its kernels (once per device).
void paged_attention_setup_device();

#ifdef __CUDACC__
// Entries of the ascending array a[0], a[stride] .. (n of them) that are <= t;
// a full warp calls it (each round every lane probes the last of its share).
__device__ __forceinline__ int warp_count_le(const int* __restrict__ a, int n, int t, int lane,
                                             int stride = 1) {
  int lo = 0;
  while (n > 0) {
    const int step = (n + 31) >> 5;
    const int e = (lane + 1) * step;
    const bool le = e <= n && a[static_cast<int64_t>(lo + e - 1) * stride] <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    lo += c * step;
    if (step == 1) break;
    n = min(step, n - c * step);
  }
  return lo;
}
#endif

}  // namespace omg
