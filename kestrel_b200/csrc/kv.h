// Paged key-value cache (kv.cu) and the attention over it (attn_decode.cu,
// attn_prompt.cu): the
// caller's buffers as the kernels see them, and the host-side launchers.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <map>

namespace kc {

enum : int { T_F16 = 1, T_BF16 = 30 };

// One registered cache. k and v are [n_layer][n_pages][nkv][page][hd]; table
// [n_seq][max_pages] (page ids, -1 past a sequence's last page); len [n_seq];
// refs [n_pages] (sequences that hold the page).
struct KvView {
  uint8_t *k, *v;
  int32_t *table, *len, *refs;
  int type, n_layer, n_pages, page, page_log2, nkv, hd, n_seq, max_pages;
  // Workspace of the page operations (one allocation, kv_workspace_ints):
  int *mark;               // [max(n_seq, n_pages)], all -1 between calls
  int *src, *dst, *rows;   // [max(n_seq, n_pages)] pages to copy and their rows
  int *last;               // [n_seq] extend: a sequence's partly full last page, or -1
  int *first;              // [n_seq] extend: its first entry of `fresh`
  int *fresh;              // [n_pages] extend: the pages it takes, ascending
  int *n_copy;             // entries of src / dst / rows
  int *both, *both_group, *lead, *plan;  // attention over shared prefixes (SharedArgs)
  int *status;
};

// CUtensorMaps (128 bytes each) of the k and v pools as [layer and page][head]
// [row][column], boxes of 64 columns x some rows of one page, 128B swizzle.
struct alignas(64) KvMap {
  unsigned char b[128];
};
struct KvMaps {
  KvMap k, v;
};
int make_kv_maps(const KvView& c, int box_rows, KvMaps& maps);

struct KvCache {
  KvView view;
  int* work;
  int64_t work_bytes;
  KvMaps rows16;  // boxes of 16 rows
  KvMaps tiles;   // boxes of attn_prompt_box_rows rows
};

// What a context holds of caches, and the attention kernels' workspace (made
// with the first cache).
struct KvState {
  std::map<int, KvCache> caches;
  float* part = nullptr;  // parts to be joined: the larger of the two kernels' needs
  int* count = nullptr;   // arrival counts, zero between launches
  int64_t count_bytes = 0;
  int64_t bytes = 0;      // of all
  bool share_always = false;  // KC_OPT_SHARE_ALWAYS
  float* shared = nullptr;  // between parts and counts: results of shared prefixes
};

int64_t kv_workspace_ints(const KvView& c);
// Points the view's workspace into `work` and clears the marks.
cudaError_t kv_workspace_init(KvView& c, int* work, cudaStream_t st);

void launch_kv_fork(const KvView& c, const int32_t* src, const int32_t* dst, int n, cudaStream_t st);
void launch_kv_free(const KvView& c, const int32_t* seqs, const int32_t* keep, int n, cudaStream_t st);
void launch_kv_extend(const KvView& c, const int32_t* seqs, const int32_t* n_new, int n, cudaStream_t st);
void launch_kv_compact(const KvView& c, int32_t* n_live, cudaStream_t st);
void launch_kv_copy_pages(const KvView& c, const int32_t* src, const int32_t* dst, int n, cudaStream_t st);
// Rows row_start[i] .. row_start[i+1]-1 of k / v (type t, row strides in
// elements) become the last positions of sequence seqs[i] (null: i) in `layer`;
// row_start null: one row each.
void launch_kv_write(const KvView& c, int layer, const int32_t* seqs, const int32_t* row_start, int n, int n_rows,
                     int t, const void* k, const void* v, int64_t k_stride, int64_t v_stride, cudaStream_t st);

struct AttnArgs {
  KvView c;
  int layer;
  const int32_t* seqs;       // null: 0 .. n-1
  const int32_t* row_start;  // [n + 1]; null: one row each
  int n, n_rows, nh, t_q;
  const void* q;             // [n_rows] rows of nh * hd, q_stride elements apart
  void* out;
  int64_t q_stride, out_stride;
  float scale;
  int window, sinks;         // window 0: none
};
// Decode attention of groups of entries whose sequences begin with the same pages:
// their prefix is computed once for a group (attn_prompt.cu's kernel, its rows the
// group's queries), the rest entry by entry (attn_decode.cu's), and both are joined
// by a kernel of their own (attn_shared.cu).
struct SharedArgs {
  const int32_t* group_start;  // [n_groups + 1]
  int n_groups;
  int32_t* of_entry;           // [n] positions that an entry's group has in common (a multiple of the page; 0: none)
  int32_t* of_group;           // [n_groups] the same of each group
  int32_t* lead;               // [n_groups] a sequence of it
  int32_t* plan;               // [SHARED_PLAN] what the device decides (below)
  int e0, e1;                  // entries of this launch
  int splits;                  // parts of a group's prefix, at most
  bool always;                 // (KC_OPT_SHARE_ALWAYS)
  // [split + 1][entry][head][64 * ceil(hd / 64) + 8]: result, maximum, sum; of the
  // parts of the prefix, then of the entries' own
  float* part;
};
// The plan: parts of a prefix (at most `splits`); blocks of the two kernels that
// work, the others leave their SMs at once.
enum { PLAN_SPLITS = 0, PLAN_PREFIX = 1, PLAN_OWN = 2, SHARED_PLAN = 4 };
__host__ __device__ inline int shared_tile(int hd) { return hd <= 128 ? 128 : 64; }
// Parts of a prefix of `both` positions: two tiles each at least, one a stream.
__host__ __device__ inline int shared_splits(int both, int hd, int most) {
  const int t = (both + shared_tile(hd) - 1) / shared_tile(hd) / 2;
  return t < 1 ? 1 : t < most ? t : most;
}
// (Whole 32-byte sectors.)
__host__ __device__ inline int shared_row_floats(int hd) { return (hd + 63) / 64 * 64 + 8; }

// The query rows of a call as [row][head][column], boxes of 128 (token, head)
// rows of one key-value head's group (which divides 128) x 128 bytes of columns.
int make_q_map(const AttnArgs& a, KvMap& map);

size_t attn_decode_part_bytes();
// One row per sequence (row_start null).
int launch_attn_decode(const AttnArgs& a, const KvMaps& rows16, float* part, int* count, cudaStream_t st);
// row_start non-null.
int attn_prompt_box_rows(int page, int hd);
size_t attn_prompt_part_bytes();
int attn_prompt_counts();
int launch_attn_prompt(const AttnArgs& a, const KvMaps& tiles, float* part, int* count, cudaStream_t st);

// (SharedArgs' e0, e1, splits and part are filled in here.)
int launch_attn_shared(const AttnArgs& a, SharedArgs sh, const KvMaps& rows16, const KvMaps& tiles, float* part,
                       int* count, float* shared_part, cudaStream_t st);
size_t attn_shared_part_bytes();
int attn_shared_counts();
int launch_attn_own(const AttnArgs& a, const SharedArgs& sh, const KvMaps& rows16, float* part, int* count,
                    cudaStream_t st);
int launch_attn_prefix(const AttnArgs& a, const SharedArgs& sh, const KvMaps& tiles, float* part, int* count,
                       cudaStream_t st);

}  // namespace kc
