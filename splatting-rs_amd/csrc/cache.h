// The paged cache's arguments, the checks of them and the rules that size its launches: host code without HIP,
// so that a plain C++ compiler builds it for the tests. Included by the kernels too, which use the same index
// checks on the device.
#pragma once

#include <cstddef>
#include <cstdint>

#include "errors.h"

#ifdef __HIPCC__
#define SPLAT_HD __host__ __device__
#else
#define SPLAT_HD
#endif

namespace splat {

// Pools of pages [pages][kv_heads][page_size][64], page_stride elements from page to page.
struct KvCache {
  int dt = 0, pages = 0, page_size = 0, kv_heads = 0;
  int shift = 0;  // log2(page_size), set by the checks
  long page_stride = 0;
  void* k = nullptr; void* v = nullptr;
};

enum TableStatus { TABLE_OK = 0, TABLE_BAD_LENGTH = 1, TABLE_POOL_EMPTY = 2, TABLE_SLOTS_FULL = 3 };
struct BlockTableArgs {
  int n = 0; const int* past = nullptr; const int* add = nullptr;
  int page_size = 0, shift = 0;
  const int* pool = nullptr; int pool_size = 0; const int* used = nullptr;
  int* table = nullptr; int width = 0;
  int* lens = nullptr; int* starts = nullptr; int* slots = nullptr; int* positions = nullptr; int cap = 0;
  int* used_out = nullptr; int* status = nullptr;
};

enum Norm { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };
enum Rope { ROPE_NONE = 0, ROPE_LINE = 1, ROPE_GRID = 2 };
struct QkArgs {
  int dt = 0; const void* qkv = nullptr; long ld = 0; int tokens = 0, heads = 0, kv_heads = 0;
  int norm = NORM_NONE; const float* qw = nullptr; const float* qb = nullptr; const float* kw = nullptr;
  const float* kb = nullptr; float eps = 0.f;
  int rope = ROPE_NONE; const int* positions = nullptr;
  void* q_out = nullptr; long ldq = 0; void* k_out = nullptr; long ldk = 0;
  bool has_cache = false; KvCache cache; const int* slots = nullptr;
  double freq[32];  // turns per position of the rotation's frequencies, set by the launcher
};

// bounds [pages][kv_heads][2][64] (lowest, highest key), for the pages that hold the last add[i]
// positions of each sequence (add NULL: all of its pages).
struct BoundsArgs {
  KvCache cache;
  int n = 0; const int* table = nullptr; int width = 0; const int* lens = nullptr; const int* add = nullptr;
  int max_add = 0; void* bounds = nullptr;
  int per_seq = 0;  // pages of a sequence taken at once, set by the check
};

struct PagedArgs {
  KvCache cache;
  const void* q = nullptr; long ldq = 0; int n = 0, heads = 0;
  const int* table = nullptr; int width = 0; const int* lens = nullptr; int max_len = 0;
  float scale = 1.f;
  void* out = nullptr; long ldo = 0;
};
struct SparseArgs {
  PagedArgs at;
  const void* bounds = nullptr; int topk = 0; int* selected = nullptr;
};

// Each throws Error(BAD_ARGUMENT, ...) for a call that is refused and sets what the launch derives. A call
// without rows (n or tokens 0) passes with its row pointers NULL.
void check_block_tables(BlockTableArgs& a);
void check_qk_norm_rope(QkArgs& a, double base);
void check_page_bounds(BoundsArgs& a);
void check_overlaps(const BoundsArgs& a);  // of outputs with index arrays and weights, after the checks above
void check_overlaps(const QkArgs& a);
void check_paged_attention(PagedArgs& a, const void* workspace, size_t bytes);
void check_sparse_attention(SparseArgs& a, const void* workspace, size_t bytes);

// How attention over the cache is launched: `cols` groups of up to 16 query heads of one key head, and for long
// sequences `workers` waves for each, which leave parts to join; 0: one block a sequence and group. topk 0: all
// pages.
constexpr int PART_HEAD = 68;  // floats of one head in one part
struct PagedPlan {
  int cols = 0, workers = 0;
  size_t before_bytes = 0, bytes = 0;  // of the workspace: the sequences' tile counts, and all of it
};
PagedPlan paged_plan(const KvCache& c, int n, int heads, int max_len, int topk);
size_t paged_attention_bytes(const KvCache& c, int n, int heads, int max_len);
size_t sparse_attention_bytes(const KvCache& c, int n, int heads, int max_len, int topk);

// base^(-i / h) / (2 pi), h = 32 (line) or 16 (grid): the turns per position of frequency i.
void rope_turns(int rope, double base, double (&freq)[32]);

// --- the kernels' own checks of what lies in device memory --------------------------------------

SPLAT_HD inline bool page_ok(int page, int pages) { return page >= 0 && page < pages; }
SPLAT_HD inline bool slot_ok(int slot, const KvCache& c) { return slot >= 0 && (slot >> c.shift) < c.pages; }
// Positions of a sequence that a call takes: no more than the table's row and `most` hold.
SPLAT_HD inline int length_of(int len, int width, int shift, int most) {
  const long row = long(width) << shift;
  long l = len < 0 ? 0 : len;
  if (l > row) l = row;
  return int(l > most ? most : l);
}
// Element offset of (page, head) in a pool.
SPLAT_HD inline long page_at(const KvCache& c, int page, int head) {
  return long(page) * c.page_stride + (long(head) << c.shift) * 64;
}
SPLAT_HD inline long slot_at(const KvCache& c, int slot, int head) {
  return page_at(c, slot >> c.shift, head) + long(slot & ((1 << c.shift) - 1)) * 64;
}

}  // namespace splat
