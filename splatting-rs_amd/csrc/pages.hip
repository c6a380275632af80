// What happens to the pages of a cache: rows that become forks of others and share their pages, pages given back that no row
// holds any more, pages moved so that those in use come first, and the copies that forks and moves ask for.
//
// Which pages are in use follows from the tables alone: no counts of holders are kept that a call could miss. Maps of the
// pages are filled from the rows and read in the order of the pages, so that what is given back, and what moves where,
// does not hang on the order in which threads come. Entries outside [0, pages) are no pages.
#include "paged.h"

namespace splat {

namespace {

// The sums before thread tid and over all of the block's; `sums` has room for a value a wave.
template <int THREADS> __device__ inline uint64_t scan_block(uint64_t v, uint64_t* sums, uint64_t& total) {
  const auto plus = [](uint64_t a, uint64_t b) { return a + b; };
  const uint64_t s = scan_wave(v, uint64_t(0), plus);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();  // the sums of the call before are read
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  uint64_t before = s - v;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  return before;
}

__device__ inline int places_of(int len, int shift) { return int((long(len) + (1 << shift) - 1) >> shift); }

// --- forks --------------------------------------------------------------------------------------

// Every block looks the rows over and sums up the pages that begun pages need (a thread its k rows), so that the call takes
// effect whole or not at all without a launch before; then each wave takes its share of a row's full pages from the parent's, and
// block 0 writes what there is one of for a row. FILL and COMMIT as in block_tables_kernel: two launches where lens_out lies over
// lens or used_out over used and there are several blocks.
// Bound by its chain of loads (parents, lengths, entries, the pool): 28 of 64 rows 5.0 us, a call among others, a thousand (2.3 MB of entries
// read and written) 5.6, where an empty call takes 3.9.
constexpr int FORK_THREADS = 1024;  // a row each up to as many; blocks of 256 take as long for 64 rows and 12.7 us for 1024, these 5.6
constexpr int FORK_UNIT = 512;      // entries of a row that a wave takes at once
template <bool FILL, bool COMMIT>
__global__ void __launch_bounds__(FORK_THREADS) fork_pages_kernel(const ForkArgs a) {
  __shared__ uint64_t sums[FORK_THREADS / 64];
  const PagesArgs& p = a.at;
  const int tid = threadIdx.x, k = (p.n + FORK_THREADS - 1) / FORK_THREADS, ps = 1 << p.shift;
  const int i0 = int(min(long(tid) * k, long(p.n))), i1 = int(min(long(i0) + k, long(p.n)));
  const long most = long(p.width) << p.shift;
  const int used = *p.used;
  bool bad = used < 0 || used > p.pool_size, no_row = false;
  auto in_pool = [&](long k) { return !bad && used + k < p.pool_size; };
  const int next = in_pool(tid) ? p.pool[used + tid] : 0;  // asked for beside the rows
  int need = 0;
  // the entry of the page that the fork begins with a copy, -1: none
  auto begun = [&](int from, int len) { return len & (ps - 1) ? p.table[long(from) * p.width + (len >> p.shift)] : -1; };
  for (int i = i0; i < i1; ++i) {
    const int from = a.parents[i];
    if (from == -1) continue;
    if (from < 0 || from >= p.n || a.parents[from] != -1 || p.lens[i] != 0) {
      no_row = true;
      continue;
    }
    const int have = p.lens[from], len = a.keep ? a.keep[i] : have;
    if (have < 0 || have > most || len < 0 || len > have) bad = true;
    else need += page_ok(begun(from, len), p.pages);
  }
  // pages (up to n) in the low half of a sum, threads with a bad length and with a bad row above
  uint64_t sum;
  long rank = long(uint32_t(scan_block<FORK_THREADS>(uint64_t(no_row) << 48 | uint64_t(bad) << 32 | uint32_t(need), sums, sum)));
  const int total = int(uint32_t(sum));
  bool none = false;  // a page that is to be taken
  for (long k = tid; k < total && in_pool(k); k += FORK_THREADS) none |= !page_ok(k == tid ? next : p.pool[used + k], p.pages);
  const bool no_page = __syncthreads_or(none);
  const int status = sum >> 32 & 0xffff ? TABLE_BAD_LENGTH : sum >> 48 ? TABLE_BAD_ROW : total > long(p.pool_size) - used ? TABLE_POOL_EMPTY
                     : no_page ? TABLE_BAD_PAGE : TABLE_OK;
  if constexpr (FILL) {
    if (status == TABLE_OK) {
      const int lane = tid & 63, segs = (p.width + FORK_UNIT - 1) / FORK_UNIT;
      for (long u = long(blockIdx.x) * (FORK_THREADS / 64) + (tid >> 6); u < long(p.n) * segs; u += long(gridDim.x) * (FORK_THREADS / 64)) {
        const int i = int(quotient(u, segs)), j0 = int(u - long(i) * segs) * FORK_UNIT + lane;
        const int from = a.parents[i];
        if (from == -1) continue;
        const int full = (a.keep ? a.keep[i] : p.lens[from]) >> p.shift;
        const int* old = p.table + long(from) * p.width;
        int* row = p.table + long(i) * p.width;
        int page[FORK_UNIT / 64];
#pragma unroll
        for (int k = 0; k < FORK_UNIT / 64; ++k)
          if (j0 + 64 * k < full) page[k] = old[j0 + 64 * k];
#pragma unroll
        for (int k = 0; k < FORK_UNIT / 64; ++k)
          if (j0 + 64 * k < full) row[j0 + 64 * k] = page[k];
      }
    }
  }
  if constexpr (COMMIT) {
    if (blockIdx.x) return;
    for (int i = i0; i < i1; ++i) {
      const int from = status == TABLE_OK ? a.parents[i] : -1;
      int len = p.lens[i], src = -1, dst = -1, rows = 0;
      if (from != -1) {
        len = a.keep ? a.keep[i] : p.lens[from];
        const int page = begun(from, len);
        if (page_ok(page, p.pages)) {
          src = page;
          dst = p.pool[used + rank++];
          rows = len & (ps - 1);
        }
        if (len & (ps - 1)) p.table[long(i) * p.width + (len >> p.shift)] = rows ? dst : page;
      }
      a.lens_out[i] = len;
      a.src[i] = src;
      a.dst[i] = dst;
      a.rows[i] = rows;
    }
    if (tid == 0) {
      *a.used_out = status == TABLE_OK ? used + total : used;
      *p.status = status;
    }
  }
}

// --- maps of pages ------------------------------------------------------------------------------
//
// Over many pages a map has a byte a page and the XCDs' caches store into it as they like: all of them store 1. (Bits, set with atomic
// operations of the device, took 95 us for 320 thousand entries of a thousand rows that share their pages, where the bytes take 6.) Few
// pages are bits in one block's LDS (bytes there, without atomics, took as long).
//
// Measured, a call among others: 64 rows of 8 thousand positions give pages back in 8.4 us, by one block, which its CU's loads of the
// entries bound; a thousand rows of up to 25 thousand positions (320 thousand entries) in 15.1, by four launches (clear 2, marks 7, counts
// 2, pages 4) that stores of a byte from each lane and the launches bound. 16 rows compact in 6.7 us by one block; 512 rows and a hundred
// thousand pages in 24.4, by five launches (clear 2, marks 5, counts 2, moves 8, entries 8), each two to four dependent loads.

constexpr int MAP_THREADS = PAGE_CHUNK;
constexpr int UNIT = 256;  // places of a row that a wave takes at once
struct MapHead {  // in the workspace, one for the launches of a call
  int used, bad;  // bad: bit 0 a length, bit 1 a page
  int kept, status;  // of compact_pages: live pages that stay
};

struct ByteMap {
  uint8_t* at;
  __device__ inline void set(int page) const { at[page] = 1; }
};
struct BitMap {
  uint32_t* at;
  __device__ inline void set(int page) const { atomicOr(at + (page >> 5), 1u << (page & 31)); }
};

// Places of row i that its keep[i] first positions fill (keep NULL: all), and its lens[i]; false where a length is none.
__device__ inline bool places_of_row(const PagesArgs& p, const int* keep, int i, int& kept, int& all) {
  const int len = p.lens[i], stays = keep ? keep[i] : len;
  const bool ok = len >= 0 && len <= (long(p.width) << p.shift) && stays >= 0 && stays <= len;
  kept = ok ? places_of(stays, p.shift) : 0;
  all = ok ? places_of(len, p.shift) : 0;
  return ok;
}
// The pages at places j0 on of row i: kept ones in `held`, the others below `all` in `gone`.
template <typename Map> struct RowUnit {
  int page[UNIT / 64], j, kept, all;
  __device__ inline void load(const PagesArgs& p, int i, int j0, int kept_, int all_) {
    j = j0 + int(threadIdx.x & 63);
    kept = kept_;
    all = all_;
    const int* row = p.table + long(i) * p.width;
#pragma unroll
    for (int k = 0; k < UNIT / 64; ++k)
      if (j + 64 * k < all) page[k] = row[j + 64 * k];
  }
  __device__ inline void mark(const PagesArgs& p, const Map& held, const Map& gone) const {
#pragma unroll
    for (int k = 0; k < UNIT / 64; ++k)
      if (j + 64 * k < all && page_ok(page[k], p.pages)) (j + 64 * k < kept ? held : gone).set(page[k]);
  }
};

// The free pages from the first-th on; true where one is none.
template <typename Map> __device__ inline bool mark_pool(const PagesArgs& p, long first, const Map& map, long thread, long threads) {
  bool bad = false;
  for (long k = first + thread; k < p.pool_size; k += threads) {
    const int page = p.pool[k];
    if (page_ok(page, p.pages)) map.set(page);
    else bad = true;
  }
  return bad;
}

__global__ void __launch_bounds__(256) pages_clear_kernel(uint4* maps, long count, MapHead* head, const int* used) {
  const long t = long(blockIdx.x) * 256 + threadIdx.x;
  for (long w = t; w < count; w += long(gridDim.x) * 256) maps[w] = make_uint4(0, 0, 0, 0);
  if (t == 0) *head = {*used, 0, 0, 0};
}

// The first map from kept places (and free pages), the second from those given back; compact: live pages, then free ones.
template <bool COMPACT>
__global__ void __launch_bounds__(256) pages_mark_kernel(const PagesArgs p, const int* keep, uint8_t* first, uint8_t* second, MapHead* head) {
  const long t = long(blockIdx.x) * 256 + threadIdx.x, all_threads = long(gridDim.x) * 256;
  const int used = head->used, segs = (p.width + UNIT - 1) / UNIT;
  int bad = 0;
  if (used < 0 || used > p.pool_size) bad = 1;
  else if (mark_pool(p, used, ByteMap{COMPACT ? second : first}, t, all_threads) && COMPACT) bad = 2;
  for (long u = t >> 6; u < long(p.n) * segs; u += all_threads >> 6) {
    const int i = int(quotient(u, segs)), j0 = int(u - long(i) * segs) * UNIT;
    int kept, all;
    if (!places_of_row(p, keep, i, kept, all)) bad |= 1;
    if (j0 >= all) continue;
    RowUnit<ByteMap> unit;
    unit.load(p, i, j0, kept, all);
    unit.mark(p, {first}, {second});
  }
  if (bad) atomicOr(&head->bad, bad);
}

// The same by one block in LDS. Lengths come first, for all rows at once, then POOL_AHEAD thousand free pages and four units of each wave
// are under way. bad: a length; none: a free page.
constexpr int SMALL_ROWS = 2048;
__device__ inline void mark_small(const PagesArgs& p, const int* keep, int used, const BitMap& pool, const BitMap& held, const BitMap& gone, int2* places, bool& bad,
                                  bool& none) {
  constexpr int WAVES = MAP_THREADS / 64, AHEAD = 4, POOL_AHEAD = 4;
  const int tid = threadIdx.x, wave = tid >> 6, segs = (p.width + UNIT - 1) / UNIT, units = p.n * segs;
  for (int i = tid; i < p.n; i += MAP_THREADS) bad |= !places_of_row(p, keep, i, places[i].x, places[i].y);
  const bool inside = used >= 0 && used <= p.pool_size;
  int free_page[POOL_AHEAD];
  auto in_pool = [&](int k) { return inside && k * MAP_THREADS + tid < p.pool_size - used; };
#pragma unroll
  for (int k = 0; k < POOL_AHEAD; ++k)
    if (in_pool(k)) free_page[k] = p.pool[used + k * MAP_THREADS + tid];
  __syncthreads();  // the maps are empty, the places there
  bad |= !inside;
  none = false;
  for (int u0 = wave; u0 < units; u0 += AHEAD * WAVES) {
    RowUnit<BitMap> unit[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int u = min(u0 + k * WAVES, units - 1), i = u / segs;  // the last one again changes nothing
      unit[k].load(p, i, (u - i * segs) * UNIT, places[i].x, places[i].y);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) unit[k].mark(p, held, gone);
  }
#pragma unroll
  for (int k = 0; k < POOL_AHEAD; ++k) {
    if (!in_pool(k)) continue;
    if (page_ok(free_page[k], p.pages)) pool.set(free_page[k]);
    else none = true;
  }
  if (inside) none |= mark_pool(p, long(used) + POOL_AHEAD * MAP_THREADS, pool, tid, MAP_THREADS);
}

// Four bytes of a map as four bits.
__device__ inline uint32_t bits_of(uint32_t bytes) { return ((bytes & 0x01010101u) * 0x01020408u) >> 24 & 15u; }

// Pages of a word that are given back; live and free pages (low and high half). A page that is both is bad.
template <bool COMPACT> __device__ inline uint64_t count_word(uint32_t first, uint32_t second, bool& bad) {
  if (!COMPACT) return __popc(second & ~first);
  bad |= (first & second) != 0;
  return uint64_t(__popc(second)) << 32 | uint64_t(__popc(first));
}

// A thread four pages: the counts of each chunk of 4096.
template <bool COMPACT>
__global__ void __launch_bounds__(MAP_THREADS) pages_count_kernel(const uint32_t* first, const uint32_t* second, long words, uint64_t* counts, MapHead* head) {
  __shared__ uint64_t sums[MAP_THREADS / 64];
  const long w = long(blockIdx.x) * MAP_THREADS + threadIdx.x;
  bool bad = false;
  const uint64_t v = w < words ? count_word<COMPACT>(bits_of(first[w]), bits_of(second[w]), bad) : 0;
  uint64_t total;
  scan_block<MAP_THREADS>(v, sums, total);
  if (threadIdx.x == 0) counts[blockIdx.x] = total;
  if (bad) atomicOr(&head->bad, 2);
}

// The counts' (below 2^32) sums before chunk `chunk`, in the high half, and of all of them: this thread's share.
__device__ inline uint64_t share_of_counts(const uint64_t* counts, long chunks, long chunk) {
  uint64_t v = 0;
  for (long c = threadIdx.x; c < chunks; c += MAP_THREADS) v += counts[c] * (c < chunk ? 0x100000001u : 1u);
  return v;
}

// What becomes of `total` pages that are to be given back; the rows' lengths.
__device__ inline int write_lengths(const FreeArgs& a, uint64_t total, int used, int bad, long thread, long threads) {
  const PagesArgs& p = a.at;
  const int status = bad & 1 ? TABLE_BAD_LENGTH : long(total) > used ? TABLE_BAD_PAGE : TABLE_OK;
  for (long i = thread; i < p.n; i += threads) a.lens_out[i] = status == TABLE_OK ? a.keep[i] : p.lens[i];
  if (thread == 0) {
    *a.used_out = status == TABLE_OK ? used - int(total) : used;
    *p.status = status;
  }
  return status;
}

__global__ void __launch_bounds__(MAP_THREADS) pages_free_kernel(const FreeArgs a, const uint32_t* held, const uint32_t* gone, long words, const uint64_t* counts,
                                                                 const MapHead* head) {
  __shared__ uint64_t sums[MAP_THREADS / 64];
  const long w = long(blockIdx.x) * MAP_THREADS + threadIdx.x;
  const uint32_t bits = w < words ? bits_of(gone[w]) & ~bits_of(held[w]) : 0;
  const uint64_t share = gridDim.x > 1 ? share_of_counts(counts, gridDim.x, blockIdx.x) : 0;
  const int used = head->used, bad = head->bad;
  uint64_t total;
  uint64_t rank = scan_block<MAP_THREADS>(__popc(bits), sums, total);
  if (gridDim.x > 1) {
    uint64_t both;
    scan_block<MAP_THREADS>(share, sums, both);
    rank += both >> 32;
    total = both & 0xffffffffu;
  }
  if (write_lengths(a, total, used, bad, w, long(gridDim.x) * MAP_THREADS) != TABLE_OK) return;
  // in their order in front of the free ones
  int* to = a.at.pool + (used - long(total) + long(rank));
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (bits >> k & 1) *to++ = int(w * 4) + k;
}

// Few rows and pages: the maps in LDS and all of it in one launch.
__global__ void __launch_bounds__(MAP_THREADS) pages_free_small_kernel(const FreeArgs a) {
  __shared__ uint64_t sums[MAP_THREADS / 64];
  __shared__ uint32_t held[MAP_THREADS], gone[MAP_THREADS];
  __shared__ int before[MAP_THREADS];
  __shared__ int2 places[SMALL_ROWS];
  const int tid = threadIdx.x, used = *a.at.used;
  held[tid] = gone[tid] = 0;
  bool bad = false, none;
  mark_small(a.at, a.keep, used, {held}, {held}, {gone}, places, bad, none);
  bad = __syncthreads_or(bad);
  const uint32_t bits = gone[tid] & ~held[tid];
  uint64_t total;
  before[tid] = int(scan_block<MAP_THREADS>(__popc(bits), sums, total));
  gone[tid] = bits;  // only this thread has read it since the marks
  __syncthreads();
  if (write_lengths(a, total, used, bad, tid, MAP_THREADS) != TABLE_OK) return;
  int* to = a.at.pool + (used - long(total));
  for (int page = tid; page < a.at.pages; page += MAP_THREADS) {
    const uint32_t word = gone[page >> 5], bit = 1u << (page & 31);
    if (word & bit) to[before[page >> 5] + __popc(word & (bit - 1))] = page;
  }
}

// --- compaction ---------------------------------------------------------------------------------

// Of the pages in use (L) and the free ones, in their order, the first L are to be in use. The free ones among those are the holes,
// M of them, and the live ones behind them move there, both in their order: the first L - M live pages stay.

// Free pages among the first `need` (at least one, as many as there are at most) of a word's pages.
__device__ inline int holes_in(uint32_t live, uint32_t free, int need) {
  uint32_t last = 0;  // the bit of the need-th page
#pragma unroll
  for (uint32_t s = 16; s; s >>= 1)
    if (__popc((live | free) & ((1u << (last + s)) - 1)) < need) last += s;
  return __popc(free & ((2u << last) - 1));
}

// A page's part of the result. l, f: live and free pages before it.
__device__ inline void write_move(const CompactArgs& a, int page, bool is_live, long l, long f, int used, long in_use, long moved) {
  const long rank = l + f - in_use;  // among the pages that are to be free
  if (rank >= 0) a.pool_out[used + rank] = page;
  if (is_live && rank >= 0) a.src[l - (in_use - moved)] = page;
  if (!is_live && rank < 0) a.dst[f] = page;
}

// What there is besides the moves: places of src and dst behind them, and the pool as it was where nothing is done.
__device__ inline void write_rest(const CompactArgs& a, int status, int used, long moved, long thread, long threads) {
  for (long k = (status == TABLE_OK ? moved : 0) + thread; k < a.cap; k += threads) a.src[k] = a.dst[k] = -1;
  if (status != TABLE_OK && a.pool_out != a.at.pool && used >= 0)
    for (long k = used + thread; k < a.at.pool_size; k += threads) a.pool_out[k] = a.at.pool[k];
  if (thread == 0) {
    *a.count = status == TABLE_OK ? int(moved) : 0;
    *a.at.status = status;
  }
}

// The rows' entries where their pages are now. rank_of(page): how many live pages are before it; places(i): the pages of row i.
template <typename Rank, typename Places>
__device__ inline void rewrite_rows(const CompactArgs& a, int status, int kept, long wave, long waves, Rank&& rank_of, Places&& places) {
  const PagesArgs& p = a.at;
  const bool in_place = a.table_out == p.table;
  const int lane = threadIdx.x & 63, segs = (p.width + UNIT - 1) / UNIT;
  if (status != TABLE_OK && in_place) return;
  for (long u = wave; u < long(p.n) * segs; u += waves) {
    const int i = int(quotient(u, segs)), j0 = int(u - long(i) * segs) * UNIT;
    const int all = status == TABLE_OK ? places(i) : 0, end = in_place ? all : p.width;
    if (j0 >= end) continue;
    const int* row = p.table + long(i) * p.width;
    int* out = a.table_out + long(i) * p.width;
    int page[UNIT / 64], rank[UNIT / 64];
#pragma unroll
    for (int k = 0; k < UNIT / 64; ++k) {
      const int j = j0 + 64 * k + lane;
      page[k] = j < end ? row[j] : -1;
    }
#pragma unroll
    for (int k = 0; k < UNIT / 64; ++k) rank[k] = j0 + 64 * k + lane < all && page_ok(page[k], p.pages) ? rank_of(page[k]) : -1;
#pragma unroll
    for (int k = 0; k < UNIT / 64; ++k)
      if (rank[k] >= kept) page[k] = a.dst[rank[k] - kept];  // kept is not negative
#pragma unroll
    for (int k = 0; k < UNIT / 64; ++k) {
      const int j = j0 + 64 * k + lane;
      if (j < end) out[j] = page[k];
    }
  }
}

__global__ void __launch_bounds__(MAP_THREADS) pages_move_kernel(const CompactArgs a, const uint32_t* live, const uint32_t* free, long words, int* before,
                                                                 const uint64_t* counts, MapHead* head) {
  __shared__ uint64_t sums[MAP_THREADS / 64];
  __shared__ long at_chunk, at_count;
  __shared__ uint64_t at_before, at_mine;
  const int tid = threadIdx.x, used = head->used, head_bad = head->bad;
  const long w = long(blockIdx.x) * MAP_THREADS + tid, chunks = gridDim.x;
  const uint32_t l = w < words ? bits_of(live[w]) : 0, f = w < words ? bits_of(free[w]) : 0;
  // one chunk's counts are its block's, of which there is one
  auto count_of = [&](long c) { return chunks > 1 && c < chunks ? counts[c] : 0; };
  uint64_t v = count_of(tid), b = 0;
  if (tid == 0) at_chunk = at_count = at_before = at_mine = 0;
  bool both = false;
  uint64_t total, ahead = scan_block<MAP_THREADS>(count_word<true>(l, f, both), sums, total);
  const bool twice = __syncthreads_or(both);  // with several chunks the count has looked at all of them
  auto pages_in = [](uint64_t v) { return long(v & 0xffffffffu) + long(v >> 32); };
  // the sums before each of MAP_THREADS chunks from c0 on, one a thread
  auto sums_before = [&](long c0, uint64_t& base) {
    if (c0) v = count_of(c0 + tid);
    uint64_t sum;
    b = base + scan_block<MAP_THREADS>(v, sums, sum);
    base += sum;
  };
  if (chunks > 1) {
    total = 0;
    for (long c0 = 0; c0 < chunks; c0 += MAP_THREADS) {
      sums_before(c0, total);
      if (c0 + tid == long(blockIdx.x)) at_mine = b;
    }
  }
  const long in_use = long(total & 0xffffffffu);
  // the chunk that holds the last of the first `in_use` pages, then the word in it: the holes are the free pages before there
  if (chunks > 1) {
    uint64_t base = 0;
    for (long c0 = 0; c0 < chunks; c0 += MAP_THREADS) {
      if (chunks > MAP_THREADS) {
        v = count_of(c0 + tid);
        sums_before(c0, base);
      }
      if (pages_in(b) < in_use && in_use <= pages_in(b) + pages_in(v)) {
        at_chunk = c0 + tid;
        at_before = b;
      }
    }
    __syncthreads();
    ahead += at_mine;
  }
  const long w2 = at_chunk * MAP_THREADS + tid;
  const uint32_t l2 = w2 < words ? bits_of(live[w2]) : 0, f2 = w2 < words ? bits_of(free[w2]) : 0;
  uint64_t sum2;
  const uint64_t v2 = count_word<true>(l2, f2, both), b2 = at_before + scan_block<MAP_THREADS>(v2, sums, sum2);
  if (pages_in(b2) < in_use && in_use <= pages_in(b2) + pages_in(v2)) at_count = long(b2 >> 32) + holes_in(l2, f2, int(in_use - pages_in(b2)));
  __syncthreads();
  const long moved = at_count;
  // a free page that is there twice leaves fewer of them than the pool has
  const int bad = head_bad | (twice || (!(head_bad & 1) && long(total >> 32) != long(a.at.pool_size) - used) ? 2 : 0);
  const int status = bad & 1 ? TABLE_BAD_LENGTH : bad ? TABLE_BAD_PAGE : moved > a.cap ? TABLE_SLOTS_FULL : TABLE_OK;
  if (w < words) before[w] = int(ahead & 0xffffffffu);
  if (status == TABLE_OK && w < words) {
    long lives = long(ahead & 0xffffffffu), frees = long(ahead >> 32);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!((l | f) >> k & 1)) continue;
      write_move(a, int(w * 4) + k, l >> k & 1, lives, frees, used, in_use, moved);
      ++(l >> k & 1 ? lives : frees);
    }
  }
  write_rest(a, status, used, moved, w, chunks * MAP_THREADS);
  if (w == 0) {
    head->kept = int(in_use - moved);
    head->status = status;
  }
}

__global__ void __launch_bounds__(256) pages_rewrite_kernel(const CompactArgs a, const uint32_t* live, const int* before, const MapHead* head) {
  const long t = long(blockIdx.x) * 256 + threadIdx.x;
  rewrite_rows(a, head->status, head->kept, t >> 6, long(gridDim.x) * 4, [&](int page) {
    const int w = page >> 2;
    return before[w] + __popc(live[w] & 0x01010101u & ((1u << (8 * (page & 3))) - 1));
  }, [&](int i) { return places_of(a.at.lens[i], a.at.shift); });
}

// Few rows and pages: the maps in LDS and all of it in one launch.
__global__ void __launch_bounds__(MAP_THREADS) pages_compact_small_kernel(const CompactArgs a) {
  __shared__ uint64_t sums[MAP_THREADS / 64];
  __shared__ uint32_t live[MAP_THREADS], free[MAP_THREADS];
  __shared__ int before[MAP_THREADS], frees[MAP_THREADS];  // live and free pages before a word
  __shared__ int2 places[SMALL_ROWS];
  __shared__ long holes;
  const int tid = threadIdx.x, used = *a.at.used;
  live[tid] = free[tid] = 0;
  if (tid == 0) holes = 0;
  bool bad = false, none;
  mark_small(a.at, nullptr, used, {free}, {live}, {live}, places, bad, none);
  bad = __syncthreads_or(bad);
  const uint32_t l = live[tid], f = free[tid];
  uint64_t total;
  const uint64_t v = count_word<true>(l, f, none), ahead = scan_block<MAP_THREADS>(v, sums, total);
  none |= !bad && long(total >> 32) != long(a.at.pool_size) - used;  // a free page that is there twice
  none = __syncthreads_or(none);
  const long in_use = long(total & 0xffffffffu), first = long(ahead & 0xffffffffu) + long(ahead >> 32), here = long(v & 0xffffffffu) + long(v >> 32);
  if (first < in_use && in_use <= first + here) holes = long(ahead >> 32) + holes_in(l, f, int(in_use - first));
  before[tid] = int(ahead & 0xffffffffu);
  frees[tid] = int(ahead >> 32);
  __syncthreads();
  const long moved = holes;
  const int status = bad ? TABLE_BAD_LENGTH : none ? TABLE_BAD_PAGE : moved > a.cap ? TABLE_SLOTS_FULL : TABLE_OK;
  if (status == TABLE_OK) {
    for (int page = tid; page < a.at.pages; page += MAP_THREADS) {
      const int w = page >> 5;
      const uint32_t lives = live[w], open = free[w], bit = 1u << (page & 31);
      if ((lives | open) & bit) write_move(a, page, lives & bit, before[w] + __popc(lives & (bit - 1)), frees[w] + __popc(open & (bit - 1)), used, in_use, moved);
    }
  }
  write_rest(a, status, used, moved, tid, MAP_THREADS);
  __syncthreads();  // dst is there
  rewrite_rows(a, status, int(in_use - moved), tid >> 6, MAP_THREADS / 64,
               [&](int page) { return before[page >> 5] + __popc(live[page >> 5] & ((1u << (page & 31)) - 1)); }, [&](int i) { return places[i].y; });
}

// --- copies -------------------------------------------------------------------------------------

constexpr int COPY_THREADS = 256, COPY_AT_ONCE = 4;
constexpr int COPY_PIECE = COPY_THREADS * COPY_AT_ONCE;  // pieces of 16 bytes a block has under way

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes a thread, four of them under way. A block takes (pair, array, part of a page) units in turn; arrays are the layers' keys,
// values and bounds. Bound by HBM: 1000 pages of 64 KB of two layers, 268 MB read and as many written, 112.0 us (4.8 TB/s); 32 begun pages of four
// layers 5.7, where an empty call takes 3.9.
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(const CopyArgs a, int es, int parts, long units) {
  const KvCache& c = a.cache;
  const int arrays = a.layers * (a.has_bounds ? 3 : 2), row_shift = es == 4 ? 4 : 3;  // 16-byte pieces of a row
  const int page16 = c.kv_heads << (c.shift + row_shift), bounds16 = c.kv_heads << (row_shift + 1);
  if (a.count) units = min(units, long(min(max(*a.count, 0), a.n)) * arrays * parts);
  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    const int i = int(quotient(u, long(arrays) * parts)), r = int(u - long(i) * arrays * parts), array = r / parts, part = r - array * parts;
    const int src = a.src[i], dst = a.dst[i];
    if (!page_ok(src, c.pages) || !page_ok(dst, c.pages) || src == dst) continue;
    const int layer = array < a.layers ? array : array < 2 * a.layers ? array - a.layers : array - 2 * a.layers;
    const bool bounds = array >= 2 * a.layers;
    char* base = static_cast<char*>(bounds ? a.bounds[layer] : array < a.layers ? a.k[layer] : a.v[layer]);
    const long stride = bounds ? bounds16 * 16L : c.page_stride * es;
    const int end = bounds ? bounds16 : page16, rows = bounds || !a.rows ? 1 << c.shift : a.rows[i];
    const u32x4* from = reinterpret_cast<const u32x4*>(base + src * stride);
    u32x4* to = reinterpret_cast<u32x4*>(base + dst * stride);
    u32x4 v[COPY_AT_ONCE];
    auto there = [&](int q) { return q < end && (bounds || ((q >> row_shift) & ((1 << c.shift) - 1)) < rows); };
#pragma unroll
    for (int k = 0; k < COPY_AT_ONCE; ++k) {
      const int q = part * COPY_PIECE + k * COPY_THREADS + int(threadIdx.x);
      if (there(q)) v[k] = from[q];
    }
#pragma unroll
    for (int k = 0; k < COPY_AT_ONCE; ++k) {
      const int q = part * COPY_PIECE + k * COPY_THREADS + int(threadIdx.x);
      if (there(q)) to[q] = v[k];
    }
  }
}

constexpr long FORK_BLOCKS = 256;  // each of which looks all rows over

// Pages, rows and places of all rows up to which one block takes them in LDS, where a CU reads alone. Measured, one block / several
// launches, 520 places a row of 16 positions: 16 rows given back 5.4 / 10.6 us, 64 8.5 / 10.5, 128 13.3 / 10.5; 16 compacted 9.1 / 13.2, 64 20.5 /
// 13.5 (each entry is read again and its page's new place looked up).
constexpr int SMALL_PAGES = MAP_THREADS * 32;
constexpr long SMALL_FREE = 49152, SMALL_COMPACT = 16384;
bool small(const PagesArgs& p, long places) { return p.pages <= SMALL_PAGES && p.n <= SMALL_ROWS && long(p.n) * p.width <= places; }

// Waves that the rows' units fill, four a block, no more than the chip holds several times.
int mark_blocks(const PagesArgs& p) { return int(std::max<long>(1, std::min<long>(2048, (long(p.n) * cdiv(p.width, UNIT) + 3) / 4))); }

struct Maps {
  uint8_t* first; uint8_t* second; int* before; uint64_t* counts; MapHead* head;
  Maps(const PagesPlan& plan, void* workspace) {
    char* ws = static_cast<char*>(workspace);
    first = reinterpret_cast<uint8_t*>(ws);
    second = reinterpret_cast<uint8_t*>(ws + plan.second);
    before = reinterpret_cast<int*>(ws + plan.before);
    counts = reinterpret_cast<uint64_t*>(ws + plan.counts);
    head = reinterpret_cast<MapHead*>(ws + plan.head);
  }
  const uint32_t* first4() const { return reinterpret_cast<const uint32_t*>(first); }
  const uint32_t* second4() const { return reinterpret_cast<const uint32_t*>(second); }
};

// The maps of a call's pages, and the counts of their chunks where there are several.
template <bool COMPACT> void fill_maps(const Exec& ex, const PagesArgs& p, const int* keep, const PagesPlan& plan, const Maps& m) {
  const long count = long(plan.before / 16);  // both maps
  pages_clear_kernel<<<int(std::max<long>(1, std::min<long>((count + 255) / 256, 2048))), 256, 0, ex.stream>>>(reinterpret_cast<uint4*>(m.first), count, m.head, p.used);
  pages_mark_kernel<COMPACT><<<mark_blocks(p), 256, 0, ex.stream>>>(p, keep, m.first, m.second, m.head);
  if (plan.chunks > 1) pages_count_kernel<COMPACT><<<int(plan.chunks), MAP_THREADS, 0, ex.stream>>>(m.first4(), m.second4(), plan.words, m.counts, m.head);
}

}  // namespace

void fork_pages(const Exec& ex, const ForkArgs& args) {
  ForkArgs a = args;
  check_fork_pages(a);
  if (ex.dry) return;
  const PagesArgs& p = a.at;
  ProfScope prof(ex, "fork_pages", 0, 8.0 * p.n * p.width + 32.0 * p.n);
  const int grid = int(std::max<long>(1, std::min<long>(FORK_BLOCKS, (long(p.n) * cdiv(p.width, FORK_UNIT) + FORK_THREADS / 64 - 1) / (FORK_THREADS / 64))));
  if (grid == 1 || (a.lens_out != p.lens && a.used_out != p.used)) {
    fork_pages_kernel<true, true><<<grid, FORK_THREADS, 0, ex.stream>>>(a);
  } else {
    fork_pages_kernel<true, false><<<grid, FORK_THREADS, 0, ex.stream>>>(a);
    fork_pages_kernel<false, true><<<1, FORK_THREADS, 0, ex.stream>>>(a);
  }
  SPLAT_HIP(hipGetLastError());
}

void free_pages(const Exec& ex, const FreeArgs& args, void* workspace, size_t bytes) {
  FreeArgs a = args;
  check_free_pages(a, workspace, bytes);
  if (ex.dry) return;
  const PagesArgs& p = a.at;
  ProfScope prof(ex, "free_pages", 0, 4.0 * p.n * p.width + 12.0 * p.n);
  if (small(p, SMALL_FREE)) {
    pages_free_small_kernel<<<1, MAP_THREADS, 0, ex.stream>>>(a);
  } else {
    const PagesPlan plan = pages_plan(p.pages);
    const Maps m(plan, workspace);
    fill_maps<false>(ex, p, a.keep, plan, m);
    pages_free_kernel<<<int(plan.chunks), MAP_THREADS, 0, ex.stream>>>(a, m.first4(), m.second4(), plan.words, m.counts, m.head);
  }
  SPLAT_HIP(hipGetLastError());
}

void compact_pages(const Exec& ex, const CompactArgs& args, void* workspace, size_t bytes) {
  CompactArgs a = args;
  check_compact_pages(a, workspace, bytes);
  if (ex.dry) return;
  const PagesArgs& p = a.at;
  ProfScope prof(ex, "compact_pages", 0, 8.0 * p.n * p.width + 8.0 * p.pages);
  if (small(p, SMALL_COMPACT)) {
    pages_compact_small_kernel<<<1, MAP_THREADS, 0, ex.stream>>>(a);
  } else {
    const PagesPlan plan = pages_plan(p.pages);
    const Maps m(plan, workspace);
    fill_maps<true>(ex, p, nullptr, plan, m);
    pages_move_kernel<<<int(plan.chunks), MAP_THREADS, 0, ex.stream>>>(a, m.first4(), m.second4(), plan.words, m.before, m.counts, m.head);
    pages_rewrite_kernel<<<mark_blocks(p), 256, 0, ex.stream>>>(a, m.first4(), m.before, m.head);
  }
  SPLAT_HIP(hipGetLastError());
}

void copy_pages(const Exec& ex, const CopyArgs& args) {
  CopyArgs a = args;
  check_copy_pages(a);
  if (a.n == 0 || a.layers == 0 || ex.dry) return;
  const KvCache& c = a.cache;
  const int es = int(dtype_size(c.dt));
  const long page16 = long(c.kv_heads) * c.page_size * 4 * es;  // 16-byte pieces
  const int parts = cdiv(page16, COPY_PIECE), arrays = a.layers * (a.has_bounds ? 3 : 2);
  ProfScope prof(ex, "copy_pages", 0, 2.0 * a.n * a.layers * (2.0 * page16 + (a.has_bounds ? c.kv_heads * 8.0 * es : 0.0)) * 16);
  const long units = long(a.n) * arrays * parts;
  copy_pages_kernel<<<int(std::min<long>(units, 16384)), COPY_THREADS, 0, ex.stream>>>(a, es, parts, units);
  SPLAT_HIP(hipGetLastError());
}

}  // namespace splat
