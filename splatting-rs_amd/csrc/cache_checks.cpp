// Checks and launch rules of the paged cache's operators (cache.h).
#include "cache.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <string>

namespace splat {

namespace {

// A launch has below 2^32 threads in x: up to 1024 for a query row, 64 for a token or for the page of a head.
constexpr long MOST_STRIDE = 1L << 31;  // elements from row to row: sizes in bytes stay within 64 bits
constexpr int FULL_BLOCKS = 1024;  // of attention in one launch, from which on they fill the chip several times
constexpr long MOST_ROWS = 1 << 21, MOST_TOKENS = 1 << 25, MOST_UNITS = 1 << 25;

long type_size(int dt) { return dt == 0 ? 4 : 2; }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(std::initializer_list<const void*> ps) {
  return std::all_of(ps.begin(), ps.end(), [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; });
}

void check_page_size(int page_size) {
  SPLAT_CHECK(page_size >= 8 && page_size <= 256 && (page_size & (page_size - 1)) == 0, BAD_ARGUMENT,
              "page_size must be a power of two from 8 to 256");
}

void check_width(int width, int page_size) {
  SPLAT_CHECK(width >= 1 && long(width) * page_size <= (1L << 30), BAD_ARGUMENT, "a table's row must hold 1 to 2^30 positions");
}

void check_sizes(const KvCache& c) {
  SPLAT_CHECK(c.dt >= 0 && c.dt <= 2, BAD_ARGUMENT, "cache: unknown dtype");
  check_page_size(c.page_size);
  SPLAT_CHECK(c.pages >= 1 && long(c.pages) * c.page_size <= 0x7fffffffL, BAD_ARGUMENT,
              "cache: pages times page_size must be 1 to 2^31 - 1");
  SPLAT_CHECK(c.kv_heads >= 1 && c.kv_heads <= 4096, BAD_ARGUMENT, "cache: kv_heads must be 1 to 4096");
}

void check_cache(KvCache& c) {
  check_sizes(c);
  SPLAT_CHECK(c.page_stride >= long(c.kv_heads) * c.page_size * 64 && c.page_stride % 8 == 0 && c.page_stride <= (1L << 31),
              BAD_ARGUMENT, "cache: page_stride must hold a page, be a multiple of 8 elements and at most 2^31");
  SPLAT_CHECK(c.k && c.v && aligned16(c.k) && aligned16(c.v), BAD_ARGUMENT, "cache: k and v must be 16-byte aligned");
  c.shift = __builtin_ctz(c.page_size);
}

// Whether rows of `wa` bytes every `sa` and rows of `wb` bytes every `sb` share memory. Rows of one stride may
// lie side by side, as the column blocks of one matrix do.
bool rows_meet(const void* a, long sa, long wa, const void* b, long sb, long wb, long rows) {
  if (!a || !b || rows <= 0) return false;
  const intptr_t pa = reinterpret_cast<intptr_t>(a), pb = reinterpret_cast<intptr_t>(b);
  if (pa + (rows - 1) * sa + wa <= pb || pb + (rows - 1) * sb + wb <= pa) return false;
  if (sa != sb || sa <= 0) return true;
  long d = (pb - pa) % sa;
  if (d < 0) d += sa;
  return d < wa || d + wb > sa;
}
bool meet(const void* a, long wa, const void* b, long wb) {
  return wa > 0 && wb > 0 && rows_meet(a, 0, wa, b, 0, wb, 1);
}

struct Range { const void* at; long bytes; };
bool meet(const Range& a, const Range& b) { return meet(a.at, a.bytes, b.at, b.bytes); }

long pool_bytes(const KvCache& c) {
  return ((c.pages - 1L) * c.page_stride + long(c.kv_heads) * c.page_size * 64) * type_size(c.dt);
}
long bounds_bytes(const KvCache& c) { return long(c.pages) * c.kv_heads * 128 * type_size(c.dt); }
bool meets_pools(const KvCache& c, const void* p, long bytes) {
  return meet(c.k, pool_bytes(c), p, bytes) || meet(c.v, pool_bytes(c), p, bytes);
}

// `count` rows of `width` bytes, `stride` apart.
struct Rows { const void* at; long stride, width, count; };
bool row_meets(const Rows& a, const Range& b) {
  if (!a.at || !b.at || a.count <= 0 || b.bytes <= 0) return false;
  const intptr_t pa = reinterpret_cast<intptr_t>(a.at), pb = reinterpret_cast<intptr_t>(b.at);
  const long row = std::max<long>(0, (pb - pa - a.width) / a.stride + (pb - pa >= a.width));  // the first that ends behind b's beginning
  return row < a.count && pa + row * a.stride < pb + b.bytes;
}

// A table's row holds up to 2^27 pages; the kernels count places past topk in 32 bits.
void check_topk(int topk) {
  SPLAT_CHECK(topk >= 1 && topk <= (1 << 27), BAD_ARGUMENT, "sparse attention: topk must be 1 to 2^27");
}

// What attention over the cache needs, whichever pages it takes.
void check_attention(PagedArgs& a) {
  check_cache(a.cache);
  SPLAT_CHECK(a.n >= 0 && a.heads >= 1 && a.heads <= 32768 && a.heads % a.cache.kv_heads == 0, BAD_ARGUMENT,
              "attention: heads must be a multiple of the cache's kv_heads");
  SPLAT_CHECK(long(a.n) * a.heads <= MOST_ROWS, BAD_ARGUMENT, "attention: more than 2^21 query rows");
  check_width(a.width, a.cache.page_size);
  SPLAT_CHECK(a.max_len >= 0, BAD_ARGUMENT, "attention: max_len is negative");
  // the kernels divide tile counts times waves (up to 2^13) as 64-bit floats
  SPLAT_CHECK(long(a.n) * std::min<long>(a.max_len, long(a.width) * a.cache.page_size) < (1L << 38), BAD_ARGUMENT,
              "attention: more than 2^38 positions");
  SPLAT_CHECK(std::isfinite(a.scale * 1.5f), BAD_ARGUMENT, "attention: scale is not finite, or too large");  // 1.5: a score of 1 stays finite in powers of two
  if (a.n == 0) return;
  SPLAT_CHECK(a.q && a.table && a.lens && a.out, BAD_ARGUMENT, "attention: a required pointer is NULL");
  const long es = type_size(a.cache.dt), w = a.heads * 64L;
  SPLAT_CHECK(aligned16(a.q) && aligned16(a.out) && a.ldq % 8 == 0 && a.ldo % 8 == 0 && a.ldq >= w && a.ldo >= w &&
                  a.ldq <= MOST_STRIDE && a.ldo <= MOST_STRIDE,
              BAD_ARGUMENT, "attention: rows of q and out must be 16-byte aligned, heads * 64 wide and a multiple of 8 elements (at most 2^31) apart");
  SPLAT_CHECK(!rows_meet(a.q, a.ldq * es, w * es, a.out, a.ldo * es, w * es, a.n), BAD_ARGUMENT, "attention: out overlaps q");
  SPLAT_CHECK(aligned4({a.table, a.lens}), BAD_ARGUMENT, "attention: table and lens must be 4-byte aligned");
  const Range out = {a.out, ((a.n - 1L) * a.ldo + w) * es};
  SPLAT_CHECK(!meets_pools(a.cache, out.at, out.bytes) && !meet(out, {a.table, 4L * a.n * a.width}) && !meet(out, {a.lens, 4L * a.n}),
              BAD_ARGUMENT, "attention: out overlaps the cache, the table or lens");
}

void check_workspace(const PagedArgs& a, const void* workspace, size_t bytes, size_t need) {
  if (need == 0) return;
  SPLAT_CHECK(workspace && aligned16(workspace) && bytes >= need, BAD_ARGUMENT,
              "the workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
  const long es = type_size(a.cache.dt), w = a.heads * 64L;
  const Range ws = {workspace, long(need)};
  SPLAT_CHECK(!meets_pools(a.cache, ws.at, ws.bytes) && !meet(ws, {a.q, ((a.n - 1L) * a.ldq + w) * es}) &&
                  !meet(ws, {a.out, ((a.n - 1L) * a.ldo + w) * es}) && !meet(ws, {a.table, 4L * a.n * a.width}) &&
                  !meet(ws, {a.lens, 4L * a.n}),
              BAD_ARGUMENT, "attention: the workspace overlaps another argument");
}

// The scores of every page that max_len allows.
size_t key_bytes(const KvCache& c, int n, int max_len) { return size_t(n) * c.kv_heads * ((long(max_len) + c.page_size - 1) / c.page_size) * 8; }

// A generous max_len sizes the workspace, which no shorter one needs more of, but not the launch.
void cut_to_row(PagedArgs& a) { a.max_len = int(std::min<long>(a.max_len, long(a.width) * a.cache.page_size)); }

}  // namespace

void check_block_tables(BlockTableArgs& a) {
  check_page_size(a.page_size);
  check_width(a.width, a.page_size);
  SPLAT_CHECK(a.n >= 0 && a.n <= 65536, BAD_ARGUMENT, "block tables: n must be 0 to 65536");
  SPLAT_CHECK(a.pool_size >= 0 && a.cap >= 0, BAD_ARGUMENT, "block tables: pool_size or cap is negative");
  SPLAT_CHECK(a.used && a.starts && a.used_out && a.status && (a.n == 0 || (a.past && a.add && a.table && a.lens)) &&
                  (a.pool_size == 0 || a.pool) && (a.cap == 0 || a.slots),
              BAD_ARGUMENT, "block tables: a required pointer is NULL");
  SPLAT_CHECK(aligned4({a.past, a.add, a.pool, a.used, a.table, a.lens, a.starts, a.slots, a.positions, a.used_out, a.status}),
              BAD_ARGUMENT, "block tables: every array must be 4-byte aligned");
  const Range in[] = {{a.past, a.n * 4L}, {a.add, a.n * 4L}, {a.pool, a.pool_size * 4L}, {a.used, 4}};
  const Range out[] = {{a.lens, a.n * 4L}, {a.used_out, 4}, {a.table, 4L * a.n * a.width}, {a.starts, 4L * (a.n + 1L)},
                       {a.slots, a.cap * 4L}, {a.positions, a.cap * 4L}, {a.status, 4}};
  for (int o = 0; o < 7; ++o) {
    for (int i = 0; i < 4; ++i) {
      if ((o == 0 && i == 0 && a.lens == a.past) || (o == 1 && i == 3 && a.used_out == a.used)) continue;
      SPLAT_CHECK(!meet(out[o], in[i]), BAD_ARGUMENT, "block tables: an output overlaps an input");
    }
    for (int i = 0; i < o; ++i)
      SPLAT_CHECK(!meet(out[o], out[i]), BAD_ARGUMENT, "block tables: two outputs overlap");
  }
  a.shift = __builtin_ctz(a.page_size);
}

void check_qk_norm_rope(QkArgs& a, double base) {
  SPLAT_CHECK(a.dt >= 0 && a.dt <= 2, BAD_ARGUMENT, "unknown dtype");
  SPLAT_CHECK(a.tokens >= 0 && a.tokens <= MOST_TOKENS && a.heads >= 1 && a.kv_heads >= 1 && a.heads <= 65536 && a.kv_heads <= 4096, BAD_ARGUMENT,
              "qk norm: tokens, heads or kv_heads");
  SPLAT_CHECK(a.norm >= NORM_NONE && a.norm <= NORM_RMS, BAD_ARGUMENT, "qk norm: unknown norm");
  SPLAT_CHECK(a.rope >= ROPE_NONE && a.rope <= ROPE_GRID, BAD_ARGUMENT, "qk norm: unknown rotation");
  SPLAT_CHECK(a.norm == NORM_NONE || (std::isfinite(a.eps) && a.eps >= 0.f), BAD_ARGUMENT, "qk norm: eps must be finite and not negative");
  SPLAT_CHECK(a.rope == ROPE_NONE || (std::isfinite(base) && base >= 1.0), BAD_ARGUMENT, "qk norm: rope_base must be at least 1");
  SPLAT_CHECK(a.has_cache == (a.slots != nullptr), BAD_ARGUMENT, "qk norm: a cache needs slots, and slots a cache");
  if (a.has_cache) {
    check_cache(a.cache);
    SPLAT_CHECK(a.cache.dt == a.dt && a.cache.kv_heads == a.kv_heads, BAD_ARGUMENT,
                "qk norm: the cache has another dtype or other kv_heads");
  }
  SPLAT_CHECK(aligned16(a.qw) && aligned16(a.qb) && aligned16(a.kw) && aligned16(a.kb), BAD_ARGUMENT,
              "qk norm: qw, qb, kw and kb must be 16-byte aligned");
  SPLAT_CHECK(aligned4({a.positions, a.slots}), BAD_ARGUMENT, "qk norm: positions and slots must be 4-byte aligned");
  if (a.tokens == 0) return;
  SPLAT_CHECK(a.qkv && a.q_out && (a.rope == ROPE_NONE || a.positions), BAD_ARGUMENT, "qk norm: a required pointer is NULL");
  const long es = type_size(a.dt), cols = (a.heads + 2L * a.kv_heads) * 64, wq = a.heads * 64L, wk = a.kv_heads * 64L;
  SPLAT_CHECK(aligned16(a.qkv) && aligned16(a.q_out) && aligned16(a.k_out) && a.ld % 8 == 0 && a.ldq % 8 == 0 && a.ld >= cols &&
                  a.ldq >= wq && a.ld <= MOST_STRIDE && a.ldq <= MOST_STRIDE &&
                  (!a.k_out || (a.ldk % 8 == 0 && a.ldk >= wk && a.ldk <= MOST_STRIDE)),
              BAD_ARGUMENT, "qk norm: rows must be 16-byte aligned, as wide as their heads and a multiple of 8 elements (at most 2^31) apart");
  const char* in = static_cast<const char*>(a.qkv);
  SPLAT_CHECK((a.q_out == in && a.ldq == a.ld) || !rows_meet(in, a.ld * es, cols * es, a.q_out, a.ldq * es, wq * es, a.tokens),
              BAD_ARGUMENT, "qk norm: q_out overlaps qkv and is not its query block");
  SPLAT_CHECK((a.k_out == in + wq * es && a.ldk == a.ld) || !rows_meet(in, a.ld * es, cols * es, a.k_out, a.ldk * es, wk * es, a.tokens),
              BAD_ARGUMENT, "qk norm: k_out overlaps qkv and is not its key block");
  SPLAT_CHECK(!rows_meet(a.q_out, a.ldq * es, wq * es, a.k_out, a.ldk * es, wk * es, a.tokens), BAD_ARGUMENT, "qk norm: q_out overlaps k_out");
  if (a.has_cache) {
    const long before = a.tokens - 1L;
    SPLAT_CHECK(!meets_pools(a.cache, in, (before * a.ld + cols) * es) && !meets_pools(a.cache, a.q_out, (before * a.ldq + wq) * es) &&
                    (!a.k_out || !meets_pools(a.cache, a.k_out, (before * a.ldk + wk) * es)),
                BAD_ARGUMENT, "qk norm: the cache overlaps the rows");
    const long stride = a.cache.page_stride * es, page = wk * a.cache.page_size * es;  // k and v may share pages
    SPLAT_CHECK(!rows_meet(a.cache.k, stride, page, a.cache.v, stride, page, a.cache.pages), BAD_ARGUMENT,
                "qk norm: the cache's keys and values overlap");
  }
}

void check_page_bounds(BoundsArgs& a) {
  check_cache(a.cache);
  SPLAT_CHECK(a.n >= 0 && a.max_add >= 0, BAD_ARGUMENT, "page bounds: n or max_add is negative");
  check_width(a.width, a.cache.page_size);
  if (a.n == 0) return;
  SPLAT_CHECK(a.table && a.lens && a.bounds && aligned16(a.bounds), BAD_ARGUMENT,
              "page bounds: a required pointer is NULL, or bounds not 16-byte aligned");
  SPLAT_CHECK(aligned4({a.table, a.lens, a.add}), BAD_ARGUMENT, "page bounds: table, lens and add must be 4-byte aligned");
  SPLAT_CHECK(!meets_pools(a.cache, a.bounds, bounds_bytes(a.cache)), BAD_ARGUMENT, "page bounds: bounds overlap the cache");
  // add positions that end anywhere lie in one page more than they fill
  a.per_seq = int(std::min<long>(a.width, a.add ? (long(a.max_add) + a.cache.page_size - 1) / a.cache.page_size + 1 : a.width));
  SPLAT_CHECK(long(a.n) * a.cache.kv_heads <= MOST_UNITS, BAD_ARGUMENT, "page bounds: more than 2^25 sequences and heads");
  a.per_seq = int(std::min<long>(a.per_seq, MOST_UNITS / (long(a.n) * a.cache.kv_heads)));  // a wave goes on to the next ones
}

void check_overlaps(const BoundsArgs& a) {
  if (a.n == 0) return;
  const Range out = {a.bounds, bounds_bytes(a.cache)};
  SPLAT_CHECK(!meet(out, {a.table, 4L * a.n * a.width}) && !meet(out, {a.lens, 4L * a.n}) && !meet(out, {a.add, 4L * a.n}), BAD_ARGUMENT,
              "page bounds: bounds overlap the table, lens or add");
}

void check_overlaps(const QkArgs& a) {
  if (a.tokens == 0) return;
  const long es = type_size(a.dt), page = a.kv_heads * 64L * a.cache.page_size * es, stride = a.cache.page_stride * es;
  const Rows out[] = {{a.q_out, a.ldq * es, a.heads * 64 * es, a.tokens}, {a.k_out, a.ldk * es, a.kv_heads * 64 * es, a.tokens},
                      {a.has_cache ? a.cache.k : nullptr, stride, page, a.cache.pages}, {a.has_cache ? a.cache.v : nullptr, stride, page, a.cache.pages}};
  const long position = a.rope == ROPE_GRID ? 8 : a.rope == ROPE_LINE ? 4 : 0, weight = a.norm == NORM_NONE ? 0 : 256;
  const Range in[] = {{a.positions, position * a.tokens}, {a.slots, 4L * a.tokens}, {a.qw, weight}, {a.qb, weight}, {a.kw, weight}, {a.kb, weight}};
  for (const Rows& o : out)
    for (const Range& i : in)
      SPLAT_CHECK(!row_meets(o, i), BAD_ARGUMENT, "qk norm: an output or the cache overlaps the positions, the slots or a weight");
}

void check_paged_attention(PagedArgs& a, const void* workspace, size_t bytes) {
  check_attention(a);
  if (a.n == 0) return;
  check_workspace(a, workspace, bytes, paged_plan(a.cache, a.n, a.heads, a.max_len, 0).bytes);
  cut_to_row(a);
}

void check_sparse_attention(SparseArgs& a, const void* workspace, size_t bytes) {
  check_attention(a.at);
  check_topk(a.topk);
  SPLAT_CHECK(a.at.scale > 0.f, BAD_ARGUMENT, "sparse attention: scale must be positive");
  if (a.at.n == 0) return;
  SPLAT_CHECK(a.bounds && aligned16(a.bounds) && a.selected, BAD_ARGUMENT,
              "sparse attention: a required pointer is NULL, or bounds not 16-byte aligned");
  const PagedArgs& p = a.at;
  const long es = type_size(p.cache.dt), w = p.heads * 64L;
  const Range sel = {a.selected, 4L * p.n * p.cache.kv_heads * a.topk}, low = {a.bounds, bounds_bytes(p.cache)};
  const Range out = {p.out, ((p.n - 1L) * p.ldo + w) * es};
  SPLAT_CHECK(aligned4({a.selected}), BAD_ARGUMENT, "sparse attention: selected must be 4-byte aligned");
  SPLAT_CHECK(!meets_pools(p.cache, sel.at, sel.bytes) && !meet(sel, {p.q, ((p.n - 1L) * p.ldq + w) * es}) && !meet(sel, out) &&
                  !meet(sel, {p.table, 4L * p.n * p.width}) && !meet(sel, {p.lens, 4L * p.n}) && !meet(sel, low) && !meet(out, low),
              BAD_ARGUMENT, "sparse attention: selected or out overlaps another argument");
  const size_t need = paged_plan(p.cache, p.n, p.heads, p.max_len, a.topk).bytes + key_bytes(p.cache, p.n, p.max_len);
  check_workspace(p, workspace, bytes, need);
  SPLAT_CHECK(!meet({workspace, long(need)}, sel) && !meet({workspace, long(need)}, low), BAD_ARGUMENT,
              "sparse attention: the workspace overlaps another argument");
  cut_to_row(a.at);
  // four threads a page in whole blocks of 64 pages
  SPLAT_CHECK(long(p.n) * p.cache.kv_heads * ((long(p.max_len) + p.cache.page_size - 1) / p.cache.page_size + 63) < (1L << 30),
              BAD_ARGUMENT, "sparse attention: more than 2^30 pages and heads");
}

namespace {
void check_workspace_sizes(const KvCache& c, int n, int heads, int max_len) {
  check_sizes(c);
  SPLAT_CHECK(n >= 0 && max_len >= 0 && heads >= 1 && heads <= 32768 && heads % c.kv_heads == 0 && long(n) * heads <= MOST_ROWS, BAD_ARGUMENT,
              "workspace: n, heads or max_len");
}
}  // namespace

PagedPlan paged_plan(const KvCache& c, int n, int heads, int max_len, int topk) {
  const int G = heads / c.kv_heads, keys = c.dt == 0 ? 16 : 32;  // positions of a tile
  PagedPlan plan;
  plan.cols = c.kv_heads * ((G + 15) / 16);
  const long most = topk ? std::min<long>(max_len, long(topk) * c.page_size) : max_len, longest = (most + keys - 1) / keys;
  // One block a sequence, without a join, for few tiles a sequence. Measured, one launch against two, a call among others: one
  // sequence of 12 heads (bf16) 10.2 : 11.4 us at 1024 positions, 11.7 : 11.3 at 1280, 12.4 : 11.3 at 1300; 32 heads on 4 11.4 : 11.5 at
  // 1280; in fp32 (tiles of 16) 10.9 : 12.3 at 448 and 11.9 : 11.9 at 512; and where the blocks fill the chip several times
  // (200 sequences of up to 2000, 12 heads) 39.0 : 47.5, up to 4000 70.5 : 69.
  if (longest <= (long(n) * plan.cols >= FULL_BLOCKS ? 128 : c.dt == 0 ? 28 : 40)) return plan;
  // eight waves on each of 256 CUs, but two tiles at least for each where all sequences are as long as may be
  const long tiles = n * longest;
  const long workers = std::min<long>(2048 / plan.cols, (tiles + 1) / 2);
  plan.workers = int(std::max<long>(4, workers / 4 * 4));
  plan.before_bytes = ((n + 1) * 8L + 15) / 16 * 16;
  plan.bytes = plan.before_bytes + size_t(plan.workers) * plan.cols * 2 * std::min(G, 16) * PART_HEAD * 4;
  // no more than give the longest part its tiles: 778 tiles of 12 heads 17.3 us by 168 waves of 4 or 5, 16.7 by 156 of 5. The
  // workspace stays that of all of them, so that it never shrinks as max_len grows.
  const long each = (tiles + plan.workers - 1) / plan.workers, enough = (tiles + each - 1) / each;
  plan.workers = int(std::min<long>(plan.workers, (enough + 3) / 4 * 4));
  return plan;
}

namespace {
// What the plan takes for n sequences or fewer: few sequences may leave parts where many leave none.
size_t plan_bytes(const KvCache& c, int n, int heads, int max_len, int topk) {
  const PagedPlan all = paged_plan(c, n, heads, max_len, topk);
  const int few = std::min(n, (FULL_BLOCKS - 1) / all.cols);
  return few ? std::max(all.bytes, paged_plan(c, few, heads, max_len, topk).bytes) : all.bytes;
}
}  // namespace

size_t paged_attention_bytes(const KvCache& c, int n, int heads, int max_len) {
  check_workspace_sizes(c, n, heads, max_len);
  return plan_bytes(c, n, heads, max_len, 0);
}

size_t sparse_attention_bytes(const KvCache& c, int n, int heads, int max_len, int topk) {
  check_workspace_sizes(c, n, heads, max_len);
  check_topk(topk);
  return plan_bytes(c, n, heads, max_len, topk) + key_bytes(c, n, max_len);
}

void rope_turns(int rope, double base, double (&freq)[32]) {
  // products of powers of two of the step: at most five roundings each
  const int h = rope == ROPE_LINE ? 32 : 16;
  double step[5];
  for (int b = 0; b < 5; ++b) step[b] = std::pow(base, -double(1 << b) / h);
  for (int i = 0; i < 32; ++i) {
    double f = 0.15915494309189535;  // 1 / (2 pi)
    for (int b = 0; b < 5; ++b)
      if (i >> b & 1) f *= step[b];
    freq[i] = f;
  }
}

}  // namespace splat
