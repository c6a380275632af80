// A paged cache of keys and values and the operators on it: block tables and slot maps, per-head norms
// with the position rotation (storing into the cache), key bounds per page, attention of one token per
// sequence over its pages, and the same over the pages that a score selects.
//
// Head dim 64, as everywhere in the library. Position p of a sequence lies in row p % page_size of the page
// its table names for p / page_size; (page, head) holds page_size rows of 64 channels back to back.
// Entries of a table outside [0, pages) hold no keys: every kernel checks them before it forms an address.
#include "paged.h"

namespace splat {

namespace {

// --- block tables and slot maps -----------------------------------------------------------------

// Request i holds past[i] positions in ceil(past / ps) pages; its add[i] new ones take the next pages of
// the pool, requests in order. Every block sums the requests up again (thread t its k of them, then one scan
// over the threads), so that a token finds its request and its page without a pass before: a binary search
// over the threads' sums for four tokens at a time, then a walk over at most k requests. A new page begins with
// a new token, whose thread writes the table's entry.
// The call takes effect whole or not at all: the status is known before anything is written.
// Bound by its chain of loads (requests; past and add again; the pool), not by its bytes: 32 requests of one token 4.6 us,
// 64 of up to 24 views (813008 tokens, 6.6 MB) 6.1 us, where an empty kernel takes 2.2. A thread that searched for each
// of its tokens took 14.7 us for the same tokens, and the commit as a second launch 3.8 more.
// FILL writes the table, slots and positions, COMMIT (block 0) lens, starts, used and status; where those lie over
// past and used and there are several blocks, it runs as a second launch.
template <int THREADS, bool FILL, bool COMMIT>
__global__ void __launch_bounds__(THREADS) block_tables_kernel(const BlockTableArgs p, bool vec) {
  constexpr int WAVES = THREADS / 64;
  __shared__ long tok[THREADS], pag[THREADS], wtok[WAVES], wpag[WAVES];
  const int tid = threadIdx.x, k = (p.n + THREADS - 1) / THREADS;
  const int i0 = int(min(long(tid) * k, long(p.n))), i1 = int(min(long(i0) + k, long(p.n)));
  const int ps = 1 << p.shift;
  const long most = long(p.width) << p.shift;
  const int used = *p.used;
  long nt = 0, np = 0;
  bool bad = used < 0 || used > p.pool_size;
  for (int i = i0; i < i1; ++i) {
    const long a = p.past[i], d = p.add[i];
    bad |= a < 0 || d < 0 || a + d > most;
    nt += d;
    np += ((a + d + ps - 1) >> p.shift) - ((a + ps - 1) >> p.shift);
  }
  const auto plus = [](uint64_t a, uint64_t b) { return a + b; };
  const long st = long(scan_wave(uint64_t(nt), uint64_t(0), plus)), sp = long(scan_wave(uint64_t(np), uint64_t(0), plus));
  const int lane = tid & 63, wave = tid >> 6;
  if (lane == 63) { wtok[wave] = st; wpag[wave] = sp; }
  const bool broken = __syncthreads_or(bad);
  long et = st - nt, ep = sp - np, total = 0, pages = 0;  // exclusive sums and all
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) { et += wtok[w]; ep += wpag[w]; }
    total += wtok[w];
    pages += wpag[w];
  }
  const int status = broken ? TABLE_BAD_LENGTH : pages > long(p.pool_size) - used ? TABLE_POOL_EMPTY
                     : total > p.cap ? TABLE_SLOTS_FULL : TABLE_OK;
  if constexpr (FILL) {
    tok[tid] = et;
    pag[tid] = ep;
    __syncthreads();
    const long count = status == TABLE_OK ? total : 0;
    for (long t = (long(blockIdx.x) * THREADS + tid) * 4; t < p.cap; t += long(gridDim.x) * THREADS * 4) {
      int slot[4] = {-1, -1, -1, -1}, pos[4] = {};
      if (t < count) {
        int lo = 0;  // the last thread whose sum is at most t
#pragma unroll
        for (int half = THREADS / 2; half; half >>= 1)
          if (tok[lo + half] <= t) lo += half;
        long r = t - tok[lo], pg = pag[lo];
        int i = lo * k, a = p.past[i], d = p.add[i], held = -1, page = -1;
#pragma unroll
        for (int u = 0; u < 4; ++u, ++r) {
          if (t + u >= count) break;
          while (r >= d) {  // ends: token t + u belongs to a request
            r -= d;
            pg += ((long(a) + d + ps - 1) >> p.shift) - ((long(a) + ps - 1) >> p.shift);
            ++i;
            a = p.past[i];
            d = p.add[i];
            held = -1;
          }
          pos[u] = a + int(r);
          const int j = pos[u] >> p.shift, have = int((long(a) + ps - 1) >> p.shift);
          if (j != held) {
            held = j;
            page = j < have ? p.table[long(i) * p.width + j] : p.pool[used + pg + (j - have)];
          }
          if (j >= have && (pos[u] & (ps - 1)) == 0) p.table[long(i) * p.width + j] = page;
          const long s = (long(page) << p.shift) + (pos[u] & (ps - 1));
          slot[u] = page < 0 || s > 0x7fffffffL ? -1 : int(s);
        }
      }
      if (vec && t + 4 <= p.cap) {
        *reinterpret_cast<int4*>(p.slots + t) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        if (p.positions) *reinterpret_cast<int4*>(p.positions + t) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        continue;
      }
      for (int u = 0; u < 4 && t + u < p.cap; ++u) {
        p.slots[t + u] = slot[u];
        if (p.positions) p.positions[t + u] = pos[u];
      }
    }
  }
  if constexpr (COMMIT) {
    if (blockIdx.x != 0) return;
    if (FILL) __syncthreads();  // the block's tokens have read past
    long t = et;
    for (int i = i0; i < i1; ++i) {
      const int a = p.past[i], d = p.add[i];
      p.starts[i] = status == TABLE_OK ? int(t) : 0;
      p.lens[i] = status == TABLE_OK ? a + d : a;
      t += d;
    }
    if (tid == 0) {
      p.starts[p.n] = status == TABLE_OK ? int(total) : 0;
      *p.used_out = status == TABLE_OK ? used + int(pages) : used;
      *p.status = status;
    }
  }
}

// --- norms of queries and keys with the rotation ------------------------------------------------

// 4 consecutive channels, as they lie in memory and as floats.
template <typename T> struct Quad {
  using Raw = uint2;
  __device__ static inline void get(const uint2& w, float* x) {
    x[0] = u16f<T>(w.x);
    x[1] = u16f<T>(w.x >> 16);
    x[2] = u16f<T>(w.y);
    x[3] = u16f<T>(w.y >> 16);
  }
  __device__ static inline uint2 put(const float* x) { return make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])); }
};
template <> struct Quad<float> {
  using Raw = float4;
  __device__ static inline void get(const float4& w, float* x) { x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w; }
  __device__ static inline float4 put(const float* x) { return make_float4(x[0], x[1], x[2], x[3]); }
};

// A wave takes one token and up to IT steps of 8 head rows, 8 lanes a row; a step's rows are all queries, keys
// or values. A lane holds the two quads of channels that turn together, (c, c + 32) on a line and (c, c + 16)
// in each half on a grid, so that no value crosses lanes but in the sums. Lane l < 32 takes frequency l's angle
// once for all heads, in 64 bits up to the fraction of a quarter turn; all loads are under way before it.
// Bound by HBM where there are many tokens: 24889 of 24 + 8 + 8 heads (f16) 54 us, 4.7 TB/s, a large copy's rate (one head
// row over 8 lanes of 8 channels, whose partners and sums crossed lanes through LDS, took 100). 32 tokens of 36 heads
// (bf16) 3.6 us, 973 of 18 (fp32) 4.4: the launch and two dependent loads (10.1 and 9.1 before the steps were dealt to waves).
template <typename T, int IT, int ROPE>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QkArgs p) {
  using Raw = typename Quad<T>::Raw;
  __shared__ __attribute__((aligned(16))) float turn[4][2][32];  // cosines, sines
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), j = lane & 7, in_step = lane >> 3;
  const int t = blockIdx.x * 4 + wave;
  if (t >= p.tokens) return;
  constexpr int SPAN = ROPE == ROPE_GRID ? 16 : 32;
  const int c0 = ROPE == ROPE_GRID ? (j >> 2) * 32 + (j & 3) * 4 : j * 4;
  const int nq = (p.heads + 7) >> 3, nk = (p.kv_heads + 7) >> 3, steps = nq + (p.slots ? 2 : 1) * nk, s0 = blockIdx.y * IT;
  // the step's kind (0 queries, 1 keys, 2 values) and this lane's head
  auto kind_of = [&](int s) { return s < nq ? 0 : s < nq + nk ? 1 : 2; };
  auto head_of = [&](int s, int kind) { return (kind == 0 ? s : kind == 1 ? s - nq : s - nq - nk) * 8 + in_step; };
  auto heads_of = [&](int kind) { return kind == 0 ? p.heads : p.kv_heads; };
  Raw raw[IT][2];
  const T* row = static_cast<const T*>(p.qkv) + t * p.ld + c0;
#pragma unroll
  for (int s = 0; s < IT; ++s) {
    if (s0 + s >= steps) break;
    const int kind = kind_of(s0 + s), h = head_of(s0 + s, kind);
    if (h >= heads_of(kind)) continue;
    const T* at = row + ((kind == 0 ? 0 : kind == 1 ? p.heads : p.heads + p.kv_heads) + h) * 64L;
    raw[s][0] = *reinterpret_cast<const Raw*>(at);
    raw[s][1] = *reinterpret_cast<const Raw*>(at + SPAN);
  }
  const int slot = p.slots ? uload(p.slots + t) : -1;
  const bool cached = p.slots && slot_ok(slot, p.cache);
  float cs[4], sn[4];
  if constexpr (ROPE != ROPE_NONE) {
    if (lane < 32) {
      const int pos = ROPE == ROPE_LINE ? p.positions[t] : p.positions[2L * t + (lane >> 4)];
      // less whole quarters of a turn (below 2^31), so that 32 bits hold what is left to 2^-27 of a half turn
      const double x = double(pos) * p.freq[ROPE == ROPE_LINE ? lane : lane & 15], quarters = rint(4.0 * x);
      const int quarter = int(quarters);
      float s, c;
      sincospif(float(2.0 * (x - 0.25 * quarters)), &s, &c);
      if (quarter & 1) {
        const float t = c;
        c = -s;
        s = t;
      }
      turn[wave][0][lane] = quarter & 2 ? -c : c;
      turn[wave][1][lane] = quarter & 2 ? -s : s;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's own rows: its LDS operations stay in order
    __builtin_amdgcn_wave_barrier();
    *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(&turn[wave][0][4 * j]);
    *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(&turn[wave][1][4 * j]);
  }
#pragma unroll
  for (int s = 0; s < IT; ++s) {
    if (s0 + s >= steps) break;
    const int kind = kind_of(s0 + s), h = head_of(s0 + s, kind);
    if (kind < 2) {
      float x[8];
      Quad<T>::get(raw[s][0], x);
      Quad<T>::get(raw[s][1], x + 4);
      if (p.norm != NORM_NONE) {
        if (p.norm == NORM_LAYER) {
          const float m = sum8(((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]))) * (1.f / 64.f);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] -= m;
        }
        float v = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) v += x[e] * x[e];
        const float r = 1.f / sqrtf(sum8(v) * (1.f / 64.f) + p.eps);
        const float* w = kind == 0 ? p.qw : p.kw;
        const float* b = kind == 0 ? p.qb : p.kb;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= r;
        if (w) {
          *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(w + c0);
          *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(w + c0 + SPAN);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= f[e];
        }
        if (b) {
          *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(b + c0);
          *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(b + c0 + SPAN);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] += f[e];
        }
      }
      if constexpr (ROPE != ROPE_NONE) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = x[e], b = x[e + 4];
          x[e] = a * cs[e] - b * sn[e];
          x[e + 4] = b * cs[e] + a * sn[e];
        }
      }
      raw[s][0] = Quad<T>::put(x);
      raw[s][1] = Quad<T>::put(x + 4);
    }
    if (h >= heads_of(kind)) continue;
    auto put = [&](T* at) {
      *reinterpret_cast<Raw*>(at) = raw[s][0];
      *reinterpret_cast<Raw*>(at + SPAN) = raw[s][1];
    };
    if (kind == 0) put(static_cast<T*>(p.q_out) + t * p.ldq + h * 64L + c0);
    if (kind == 1 && p.k_out) put(static_cast<T*>(p.k_out) + t * p.ldk + h * 64L + c0);
    if (kind && cached) put(static_cast<T*>(kind == 1 ? p.cache.k : p.cache.v) + slot_at(p.cache, slot, h) + c0);
  }
}

// --- key bounds per page ------------------------------------------------------------------------

// NaN in either operand gives NaN.
__device__ inline float low(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ inline float high(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// One wave a (sequence, page, head), 8 lanes a row, 8 rows a load, 8 loads under way. 1556 pages of 64 rows and 8 heads
// (f16, 28 MB) 8.2 us, 3.4 TB/s: short waves, whose comparisons and the joining of their 16 values over the lanes take
// half of that (10.4 with the joining through LDS; two heads a wave 12.4, four 18.2: fewer waves hide less). The pages of
// 32 new tokens (bf16, 12 heads) 3.5 us: the launch and three dependent loads.
template <typename T>
__global__ void __launch_bounds__(256) page_bounds_kernel(const BoundsArgs p) {
  const KvCache& c = p.cache;
  const long unit = long(blockIdx.x) * 4 + uniform(threadIdx.x >> 6);
  if (unit >= long(p.n) * p.per_seq * c.kv_heads) return;
  const int lane = threadIdx.x & 63, j = lane & 7, ps = 1 << c.shift;
  const long of_seq = long(p.per_seq) * c.kv_heads;
  const int i = int(quotient(unit, of_seq)), first = int(quotient(unit - i * of_seq, c.kv_heads)), h = int(unit - i * of_seq - long(first) * c.kv_heads);
  const int len = length_of(uload(p.lens + i), p.width, c.shift, 0x7fffffff);
  const int fresh = p.add ? min(max(uload(p.add + i), 0), len) : len;
  if (fresh == 0) return;
  const int last = int((long(len) + ps - 1) >> c.shift);
  for (int g = ((len - fresh) >> c.shift) + first; g < last; g += p.per_seq) {
    const int page = uload(p.table + long(i) * p.width + g);
    if (!page_ok(page, c.pages)) continue;
    const int rows = min(ps, len - (g << c.shift));
    const T* k = static_cast<const T*>(c.k) + page_at(c, page, h) + j * 8;
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] = INFINITY; hi[e] = -INFINITY; }
    for (int r0 = lane >> 3; r0 < rows; r0 += 64) {
      uint4 raw[8][sizeof(T) / 2];  // as they lie in memory: the conversions would double the registers
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (8 * u < rows)  // the last row again changes nothing
#pragma unroll
          for (int w = 0; w < int(sizeof(T) / 2); ++w) raw[u][w] = reinterpret_cast<const uint4*>(k + min(r0 + 8 * u, rows - 1) * 64)[w];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (8 * u < rows) {
          float x[8];
          load8(reinterpret_cast<const T*>(raw[u]), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) { lo[e] = low(lo[e], x[e]); hi[e] = high(hi[e], x[e]); }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = over_halves(lo[e], low);
      hi[e] = over_halves(hi[e], high);
    }
    T* out = static_cast<T*>(p.bounds) + (long(page) * c.kv_heads + h) * 128 + j * 8;
    if (lane < 8) store8(out, lo);
    else if (lane < 16) store8(out + 64, hi);
  }
}

// --- attention of one token over the cache ------------------------------------------------------
//
// S^T = K Q^T and O^T = V^T P^T on the 16x16 matrix instructions, the query heads that share a key head as the
// 16 columns (fewer: columns of zeros, which cost nothing, since the bytes of K and V bound the kernel).
// The scores come out with a lane holding one head (lane % 16) and keys 4 (lane / 16) + r, which is the
// operand layout of the second product as it stands; V is read transposed from LDS.
//
// Bound by the bytes of K and V: 48 sequences (f16, 8 key heads, 295 MB) in 59 us, 5.0 TB/s, where a kernel that only reads
// reaches 5.7 and a large copy 4.7. A kernel of the vector unit, one wave a query head, took 1.8 ms.
//
// A wave works alone: tiles of 32 keys (16 in fp32: 4 KB of K and 4 KB of V in every type) stream into its own
// ring in LDS, four loads of 1 KB for each, that many bytes ahead, and no barrier holds it up. A load covers 8
// rows (4 in fp32) of one page, and the rows that are not there (past the length, a missing page) lie outside
// its buffer, so that they arrive as zeros whatever memory holds.

constexpr int STAGES = 2;  // run() takes two

// Tiles of a sequence: of its positions, or of the pages that were selected.
template <int KEYS> __device__ inline int tiles_in(int len, const KvCache& c, int topk) {
  if (!topk) return int((long(len) + KEYS - 1) / KEYS);
  const int held = int((long(len) + c.page_size - 1) >> c.shift);
  return int(((long(min(held, topk)) << c.shift) + KEYS - 1) / KEYS);
}

// One wave: the running softmax of one group of heads over tiles of one sequence (SPARSE: of its selected pages).
template <typename T, bool SPARSE> struct PagedWave {
  using Ops = TileOps<T>;
  static constexpr int KEYS = Ops::KEYS, PIECE = Ops::PIECE;
  const PagedArgs& p;
  const int* sel;  // [n, kv_heads, topk] (SPARSE)
  const int topk, kh, lane;
  const bool in;  // the lane's column has a head
  const uint32_t lds;   // of the wave's ring
  const char* ring;
  Ops ops;
  f32x4 o[4];
  float m, l;
  int some;  // keys were there
  int len, held;
  const int *row, *chosen;

  __device__ inline void begin(int i) {
    row = p.table + long(i) * p.width;
    if (SPARSE) chosen = sel + (long(i) * p.cache.kv_heads + kh) * topk;
    len = length_of(uload(p.lens + i), p.width, p.cache.shift, p.max_len);
    held = int((long(len) + p.cache.page_size - 1) >> p.cache.shift);
  }

  // Loads tile t, which lies in E pages, into slot b of the ring; the rows of each piece that are there, 8 bits a piece.
  // The table's entries are read whatever the length is, so that both loads are under way together.
  template <int E> __device__ inline uint32_t load_tile(int t, int b) {
    constexpr int PIECES = 4 / E, ROWS = PIECES * PIECE;  // of one page
    const KvCache& c = p.cache;
    uint32_t k_off[4], v_off[4], there = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      k_off[k] = Ops::k_off(lane, k);
      v_off[k] = Ops::v_off(lane, k);
    }
    int place[E], entry[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int at = (t * KEYS + e * ROWS) >> c.shift;
      place[e] = SPARSE ? at < topk ? uload(chosen + min(at, topk - 1)) : -1 : at;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) entry[e] = uload(row + (SPARSE ? max(min(place[e], p.width - 1), 0) : min(place[e], p.width - 1)));
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int in_page = E > 1 ? 0 : (t * KEYS) & (c.page_size - 1);
      const bool ok = place[e] >= 0 && place[e] < held && page_ok(entry[e], c.pages);
      const int rows = ok ? max(0, min(ROWS, len - (place[e] << c.shift) - in_page)) : 0;
#pragma unroll
      for (int k = 0; k < PIECES; ++k) there |= uint32_t(max(0, min(PIECE, rows - k * PIECE))) << (8 * (e * PIECES + k));
      const long at = (ok ? page_at(c, entry[e], kh) : 0) + in_page * 64;
      const uint32_t bytes = uint32_t(rows) * 64 * sizeof(T), to = lds + b * TILE_BYTES + e * PIECES * 1024;
      load_lds<PIECES>(static_cast<const T*>(c.k) + at, bytes, k_off, e * PIECES, to);
      load_lds<PIECES>(static_cast<const T*>(c.v) + at, bytes, v_off, e * PIECES, to + TILE_BYTES / 2);
    }
    return uniform(int(there));
  }
  __device__ inline uint32_t issue(int t, int b) {
    if (p.cache.page_size >= KEYS) return load_tile<1>(t, b);
    if (KEYS == 16 || p.cache.page_size == 16) return load_tile<2>(t, b);
    return load_tile<4>(t, b);
  }

  __device__ inline void tile(int b, uint32_t there, float scale, bool rest) {
    constexpr uint32_t ALL = PIECE * 0x01010101u;
    const char* kt = ring + b * TILE_BYTES;
    f32x4 x[Ops::T16];
    ops.scores(kt, lane, x);
    const typename Ops::Values v = Ops::values(kt + TILE_BYTES / 2, lane);  // under way during the softmax
    const int g = lane >> 4;
#pragma unroll
    for (int t = 0; t < Ops::T16; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[t][r] *= scale;
    if (there != ALL) {
#pragma unroll
      for (int t = 0; t < Ops::T16; ++t) {
        const int key = 16 * t + 4 * g, rows = int((there >> (8 * (key / PIECE))) & 255u) - key % PIECE;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r >= rows) x[t][r] = -INFINITY;
      }
    }
    some |= there != 0;
    float mx = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
    if constexpr (Ops::T16 == 2) mx = fmaxf(mx, fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    const float mn = fmaxf(m, max_groups(mx));
    const float ref = mn == -INFINITY ? 0.f : mn;
    // the weights are 2^TOP e^(x - ref); what was summed against another reference moves along
    const float keep = m == -INFINITY ? 0.f : exp_of(m - mn);
    m = mn;
    l *= keep;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[d][r] *= keep;
#pragma unroll
    for (int t = 0; t < Ops::T16; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[t][r] = exp_of<Ops::TOP>(x[t][r] - ref);
        l += x[t][r];
      }
    Ops::weigh(v, x, o, rest);
  }

  // Tiles t, t + step, ... below end: tile k is asked for while tile k - 2 is used, in one copy of either's code (a
  // launch begins with a cold instruction cache). Where a sum is NaN they are taken again without the weights' second terms:
  // beside an infinite value these make inf - inf or 0 inf. Columns of zeros do not count, which an infinite key makes NaN.
  __device__ inline void run(int t, int step, int end, float scale) {
    const int count = t < end ? (end - t + step - 1) / step : 0;
    bool rest = sizeof(T) == 2;
    ops.pin_q();
#pragma unroll 1
    while (true) {
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
      m = -INFINITY;
      l = 0.f;
      some = 0;
      uint32_t there = 0, next = 0;  // of tiles k - 2 and k - 1
#pragma unroll 1
      for (int k = 0; k < count + 2; ++k) {
        if (k >= 2) {
          if (k - 1 < count) wait_loads<8>();
          else wait_loads<0>();
          tile(k & 1, there, scale, rest);
        }
        there = next;
        if (k < count) next = issue(t + k * step, k & 1);
      }
      if (sizeof(T) == 4 || !rest) return;
      bool nan = false;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) nan |= o[d][r] != o[d][r];
      if (!__any(nan && in)) return;
      rest = false;
    }
  }

  // The normalised result, or zeros where no key was there.
  __device__ inline void store(int i, int head, float sum) const {
    const float inv = 1.f / sum;
    T* out = static_cast<T*>(p.out) + i * p.ldo + long(head) * 64 + 4 * (lane >> 4);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = some ? o[d][r] * inv : 0.f;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out + 16 * d) = make_float4(v[0], v[1], v[2], v[3]);
      else *reinterpret_cast<uint2*>(out + 16 * d) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    }
  }
};

constexpr int PAGED_WAVES = 4;

// A part: `heads` (up to 16) times 64 sums, then (m, l) of each head; l is -1 where no key was there. PART_HEAD
// floats a head keep the parts 16-byte aligned.
struct Part {
  const int heads;
  __device__ inline explicit Part(int G) : heads(min(G, 16)) {}
  __device__ inline long size() const { return heads * long(PART_HEAD); }
  __device__ inline int ml(int g) const { return heads * 64 + g * 2; }
};

// What the waves of a block ended with. Waves r, r + 1, ... whose last part is of one sequence, the later ones' only
// part, join in LDS: wave d adds up channels 16 d + (0..15). The result is written normalised if the sequence lies in
// them as a whole, else as one part in the place of the first of them.
struct BlockEnds {
  int seq[PAGED_WAVES];  // -1: nothing left to write
  bool only[PAGED_WAVES], begins[PAGED_WAVES], ends[PAGED_WAVES];
};
template <typename T, typename Wave, typename Place>
__device__ inline void join_block(const PagedArgs& p, const Wave& w, char* smem, BlockEnds& at, int wave, int head, bool in,
                                  const Part& part, Place&& place) {
  const int lane = w.lane, col = lane & 15, g = lane >> 4;
  float* own = reinterpret_cast<float*>(smem + wave * STAGES * TILE_BYTES);  // its tiles are used up
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) own[(d * 4 + r) * 64 + lane] = w.o[d][r];
  if (lane < 16) {
    float* ml = own + 1024 + lane * 4;
    ml[0] = w.m;
    ml[1] = w.l;
    ml[2] = __int_as_float(w.some);
  }
  __syncthreads();
  for (int r = 0; r < PAGED_WAVES;) {
    const int seq = at.seq[r];
    int e = r + 1;
    while (seq >= 0 && e < PAGED_WAVES && at.seq[e] == seq && at.only[e]) ++e;
    if (seq >= 0) {
      float mn = -INFINITY, sum = 0.f, f[PAGED_WAVES], v[4] = {};
      int some = 0;
      auto state = [&](int k) { return reinterpret_cast<const float*>(smem + k * STAGES * TILE_BYTES); };
#pragma unroll
      for (int k = 0; k < PAGED_WAVES; ++k)
        if (k >= r && k < e) mn = fmaxf(mn, state(k)[1024 + col * 4]);
#pragma unroll
      for (int k = 0; k < PAGED_WAVES; ++k) {
        if (k < r || k >= e) continue;
        const float* ml = state(k) + 1024 + col * 4;
        const int had = __float_as_int(ml[2]);
        f[k] = !had || ml[0] == -INFINITY ? 0.f : exp_of(ml[0] - mn);
        if (!had) continue;  // no key: its sums are zeros, whatever the others hold
        some = 1;
        sum += ml[1] * f[k];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] += state(k)[(wave * 4 + c) * 64 + lane] * f[k];
      }
      if (in) {
        if (at.begins[r] && at.ends[e - 1]) {
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = some ? v[c] / sum : 0.f;
          T* out = static_cast<T*>(p.out) + seq * p.ldo + long(head) * 64 + 16 * wave + 4 * g;
          if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
          else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
        } else {
          float* to = place(r, at.only[r]);
          *reinterpret_cast<float4*>(to + col * 64 + 16 * wave + 4 * g) = make_float4(v[0], v[1], v[2], v[3]);
          if (wave == 0 && g == 0) *reinterpret_cast<float2*>(to + part.ml(col)) = make_float2(mn, some ? sum : -1.f);
        }
      }
    }
    r = e;
  }
}

// One block a (sequence, group of up to 16 heads of one key head): its waves take equal parts of the tiles
// and join their sums in LDS. For short sequences (paged_plan has the rule and both sides' times): three of up to 188
// positions (fp32, 6 heads) 7.8 us, of which the launch and the length take 2.6, the first tiles 2.0, the products of
// three tiles in fp32 (matrix instructions of 4 keys) 2.2 and the join 0.8.
template <typename T, bool SPARSE>
__global__ void __launch_bounds__(PAGED_WAVES * 64, 2) paged_whole_kernel(const PagedArgs p, const int* sel, int topk, float scale) {
  using Wave = PagedWave<T, SPARSE>;
  __shared__ __attribute__((aligned(1024))) char smem[PAGED_WAVES * STAGES * TILE_BYTES];
  __shared__ BlockEnds ends;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int G = p.heads / p.cache.kv_heads, groups = (G + 15) / 16;
  const int i = blockIdx.x, kh = int(blockIdx.y) / groups, g0 = int(blockIdx.y) % groups * 16;
  const int col = lane & 15, head = kh * G + g0 + col;
  char* ring = smem + wave * STAGES * TILE_BYTES;
  Wave w{p, sel, topk, kh, lane, g0 + col < G, uint32_t(reinterpret_cast<uintptr_t>((lds_cptr)ring)), ring};
  w.ops.load_q(static_cast<const T*>(p.q) + i * p.ldq + long(head) * 64, lane >> 4, g0 + col < G);
  w.begin(i);
  if (threadIdx.x < PAGED_WAVES) {
    ends.seq[threadIdx.x] = i;
    ends.only[threadIdx.x] = ends.begins[threadIdx.x] = ends.ends[threadIdx.x] = true;
  }
  // every fourth tile: the first ones do not hang on the length
  w.run(wave, PAGED_WAVES, tiles_in<Wave::KEYS>(w.len, p.cache, topk), scale);
  w.l = sum_groups(w.l);
  join_block<T>(p, w, smem, ends, wave, head, g0 + col < G, Part(G), [](int, bool) { return static_cast<float*>(nullptr); });
}

// Long or uneven sequences: the tiles of all sequences in a row, cut into one equal part a wave. A sequence that
// lies within one part or one block's is written at once; of the others the parts' sums, unnormalised, are left
// for paged_join_kernel: slot 0 for the sequence that a wave's part begins in, slot 1 for one that it ends in. With
// span = PAGED_WAVES the parts that a block's waves end with are joined where they are of one sequence, so that a
// long sequence leaves one part a block instead of one a wave (span = 1). That costs this kernel 1.5 us and spares the join its
// batches: one sequence, 12 heads (156 waves each) 22.9 -> 22.4 us, 2 groups of 16 heads (260 waves) 16.4 -> 13.3; with fewer waves a
// sequence it gives or costs a microsecond (8 sequences of 8000, 12 heads on 12 38.5 -> 39.6; 48 sequences, 32 heads on 8 57.6 ->
// 56.8), so it is done from 128 waves a sequence on.
constexpr int SCAN_MAX = 1024;


// before[i]: tiles of the sequences before i, for i in [0, n]. By one block of NT threads.
template <int KEYS, int NT> __device__ inline void scan_tiles(const PagedArgs& p, int topk, long* before) {
  __shared__ long wsum[NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  long base = 0;
  for (int i0 = 0; i0 <= p.n; i0 += NT) {
    const int i = i0 + tid;
    const long c = i < p.n ? tiles_in<KEYS>(length_of(p.lens[i], p.width, p.cache.shift, p.max_len), p.cache, topk) : 0;
    long inc = c;
    for (int m = 1; m < 64; m <<= 1) {
      const long o = __shfl_up(inc, m);
      if (lane >= m) inc += o;
    }
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    long at = base + inc - c;
    for (int k = 0; k < NT / 64; ++k) {
      if (k < wave) at += wsum[k];
      base += wsum[k];
    }
    if (i <= p.n) before[i] = at;
    __syncthreads();
  }
}

template <int KEYS> __global__ void __launch_bounds__(1024) paged_scan_kernel(const PagedArgs p, int topk, long* before) {
  scan_tiles<KEYS, 1024>(p, topk, before);
}

template <typename T, bool SPARSE, bool SCAN>
__global__ void __launch_bounds__(PAGED_WAVES * 64, 2) paged_parts_kernel(const PagedArgs p, const int* sel, int topk, float scale,
                                                                          int workers, int span, long* before, float* parts) {
  using Wave = PagedWave<T, SPARSE>;
  __shared__ __attribute__((aligned(1024))) char smem[PAGED_WAVES * STAGES * TILE_BYTES];
  __shared__ long own[SCAN ? SCAN_MAX + 1 : 1];
  __shared__ BlockEnds ends;
  const long* pre = before;
  if constexpr (SCAN) {  // few sequences: every block counts for itself, one leaves the counts for the join
    scan_tiles<Wave::KEYS, PAGED_WAVES * 64>(p, topk, own);
    if (blockIdx.x == 0 && blockIdx.y == 0)
      for (int i = threadIdx.x; i <= p.n; i += PAGED_WAVES * 64) before[i] = own[i];
    pre = own;
  }
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int G = p.heads / p.cache.kv_heads, groups = (G + 15) / 16, cols = p.cache.kv_heads * groups;
  const int kh = int(blockIdx.y) / groups, g0 = int(blockIdx.y) % groups * 16;
  const int col = lane & 15, head = kh * G + g0 + col;
  const long worker = long(blockIdx.x) * PAGED_WAVES + wave, total = pre[p.n];
  const long W = min(long(workers), total);  // each has a tile at least
  if (long(blockIdx.x) * PAGED_WAVES >= W) return;
  const Part part(G);
  auto place = [&](long worker, bool only) { return parts + ((worker * cols + blockIdx.y) * 2 + (only ? 0 : 1)) * part.size(); };
  char* ring = smem + wave * STAGES * TILE_BYTES;
  Wave w{p, sel, topk, kh, lane, g0 + col < G, uint32_t(reinterpret_cast<uintptr_t>((lds_cptr)ring)), ring};
  w.m = w.l = 0.f;
  w.some = 0;
#pragma unroll
  for (int d = 0; d < 4; ++d) w.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  int last = -1;
  bool only = false, begins = false, stops = false;
  if (worker < W) {
    long t = quotient(total * worker, W);
    const long first = t, end = quotient(total * (worker + 1), W);
    int lo = 0, hi = p.n;  // the sequence that tile t belongs to
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= t) lo = mid;
      else hi = mid;
    }
    for (int i = uniform(lo); t < end; i = uniform(i + 1)) {
      const long b0 = pre[i], b1 = pre[i + 1];
      const long stop = min(end, b1);
      if (stop <= t) continue;
      w.ops.load_q(static_cast<const T*>(p.q) + i * p.ldq + long(head) * 64, lane >> 4, g0 + col < G);
      w.begin(i);
      w.run(uniform(int(t - b0)), 1, uniform(int(stop - b0)), scale);
      w.l = sum_groups(w.l);
      if (t == b0 && stop == b1) {
        if (g0 + col < G) w.store(i, head, w.l);
      } else if (stop == end && span > 1) {  // for the join with the next waves
        last = i;
        only = t == first;
        begins = t == b0;
        stops = stop == b1;
      } else if (g0 + col < G) {
        float* at = place(worker, t == first);
#pragma unroll
        for (int d = 0; d < 4; ++d)
          *reinterpret_cast<float4*>(at + col * 64 + 16 * d + 4 * (lane >> 4)) = make_float4(w.o[d][0], w.o[d][1], w.o[d][2], w.o[d][3]);
        if (lane < 16) *reinterpret_cast<float2*>(at + part.ml(col)) = make_float2(w.m, w.some ? w.l : -1.f);
      }
      t = stop;
    }
  }
  if (span == 1) return;
  if (lane == 0) {
    ends.seq[wave] = last;
    ends.only[wave] = only;
    ends.begins[wave] = begins;
    ends.ends[wave] = stops;
  }
  const long worker0 = long(blockIdx.x) * PAGED_WAVES;
  join_block<T>(p, w, smem, ends, wave, head, g0 + col < G, part, [&](int r, bool only) { return place(worker0 + r, only); });
}

// One block a (sequence, `per` heads of a group): the parts of a sequence that several waves had. SPLIT waves share a
// head (all eight where the block has one), each with every SPLIT-th part, a channel a lane, JOIN_PARTS parts under way.
// Bound by its chain of loads (counts, then parts), not by their bytes: 39 parts of 12 heads 5.0 us, parts of 48 sequences of
// 32 heads 8.8. Blocks of 4 or 16 waves, 4 to 24 parts under way and other numbers of heads a block were no faster; 64-bit
// integer divisions for the parts' places made it 18.6.
constexpr int JOIN_WAVES = 8, JOIN_PARTS = 8;
template <typename T>
__global__ void __launch_bounds__(JOIN_WAVES * 64) paged_join_kernel(const PagedArgs p, int workers, int span, int per, const long* before, const float* parts) {
  __shared__ float accs[JOIN_WAVES][64], sums[JOIN_WAVES], refs[JOIN_WAVES];
  __shared__ int somes[JOIN_WAVES];
  const int i = blockIdx.x, G = p.heads / p.cache.kv_heads, groups = (G + 15) / 16, cols = p.cache.kv_heads * groups;
  const int blocks = (min(G, 16) + per - 1) / per, col = blockIdx.y / blocks, first_head = blockIdx.y % blocks * per;  // in the group
  const int group = col % groups * 16, heads = min(per, min(16, G - group) - first_head);
  if (heads <= 0) return;
  const int head0 = col / groups * G + group + first_head;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const long b0 = before[i], b1 = before[i + 1], total = before[p.n];
  T* out = static_cast<T*>(p.out) + i * p.ldo + long(head0) * 64;
  if (b0 == b1) {
    for (int e = threadIdx.x; e < heads * 64; e += JOIN_WAVES * 64) out[e] = from_f<T>(0.f);
    return;
  }
  // the last worker that begins at or before tile b: begin(w) = floor(total w / W)
  const long W = min(long(workers), total);
  const long w0 = quotient((b0 + 1) * W - 1, total), w1 = quotient(b1 * W - 1, total);
  if (w0 == w1) return;  // written whole
  // Each `span` workers (one, or a block's) leave one part in the place of the first; the last worker's is one of its
  // own where it went on to other sequences.
  const bool went_on = quotient(total * (w1 + 1), W) != b1;
  const long block0 = w0 / span, block1 = (went_on ? w1 - 1 : w1) / span;
  if (!went_on && block0 == block1) return;  // written whole
  const int joined = int(block1 - block0) + 1, count = joined + went_on;
  const Part layout(G);
  // floats from `parts`: below 2^31, as the plan's sizes are
  const int size = int(layout.size()) * 2, step = span * cols * size, base = int(block0) * step + col * size;
  const int first = int(w0) * cols * size + col * size + (quotient(total * w0, W) < b0 ? size / 2 : 0);  // w0's second part
  const int last = int(w1) * cols * size + col * size;
  auto part = [&](int k) { return parts + (k == 0 ? first : k < joined ? base + k * step : last); };
  const int split = heads >= 5 ? 1 : JOIN_WAVES / heads, at_once = JOIN_WAVES / split;
  for (int g0 = 0; g0 < heads; g0 += at_once) {
    const int g = g0 + wave / split;
    float acc = 0.f, sum = 0.f, m = -INFINITY;
    int some = 0;
    if (g < heads && wave < split * at_once)
      for (int k0 = wave % split; k0 < count; k0 += JOIN_PARTS * split) {
        float2 ml[JOIN_PARTS];
        float o[JOIN_PARTS], mx = m;
#pragma unroll
        for (int u = 0; u < JOIN_PARTS; ++u) {
          const int k = min(k0 + u * split, count - 1);
          const float* at = part(k);
          ml[u] = *reinterpret_cast<const float2*>(at + layout.ml(first_head + g));
          o[u] = at[(first_head + g) * 64 + lane];
        }
#pragma unroll
        for (int u = 0; u < JOIN_PARTS; ++u)
          if (k0 + u * split < count && !(ml[u].y < 0.f)) {  // NaN stays
            mx = fmaxf(mx, ml[u].x);
            some = 1;
          }
        const float keep = m == -INFINITY ? 0.f : exp_of(m - mx);
        acc *= keep;
        sum *= keep;
        m = mx;
#pragma unroll
        for (int u = 0; u < JOIN_PARTS; ++u)
          if (k0 + u * split < count && !(ml[u].y < 0.f)) {
            const float f = ml[u].x == -INFINITY ? 0.f : exp_of(ml[u].x - mx);
            acc += o[u] * f;
            sum += ml[u].y * f;
          }
      }
    if (split > 1) {
      accs[wave][lane] = acc;
      if (lane == 0) {
        sums[wave] = sum;
        refs[wave] = m;
        somes[wave] = some;
      }
      __syncthreads();
      if (wave % split == 0) {
        float mx = m;
        for (int k = 1; k < split; ++k) mx = fmaxf(mx, refs[wave + k]);
        acc = sum = 0.f;
        for (int k = 0; k < split; ++k) {
          if (!somes[wave + k]) continue;
          some = 1;
          const float f = refs[wave + k] == -INFINITY ? 0.f : exp_of(refs[wave + k] - mx);
          acc += accs[wave + k][lane] * f;
          sum += sums[wave + k] * f;
        }
      }
    }
    if (g < heads && wave % split == 0 && wave < split * at_once) out[g * 64 + lane] = from_f<T>(some ? acc / sum : 0.f);
  }
}

// --- selection of pages -------------------------------------------------------------------------

// Scores as whole numbers in the order of the scores, NaN above all; 0: no page there.
__device__ inline uint64_t order_of(double s) {
  if (s != s) return ~0ull;
  const uint64_t b = __double_as_longlong(s);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

// The most that each head's q k can be for a key between the page's bounds, summed over the group's heads (bounding a page's
// scores by its keys' lowest and highest channels: Tang et al., query-aware sparsity for long contexts, 2024), is
// sum_c hi_c A_c + lo_c B_c, with A and B the sums of the positive and the negative parts of the heads' queries:
// 128 products a page, however many heads share it. In 64 bits: which of two pages next to the border is
// taken can hang on less than 32 bits hold. 8 lanes a page, 16 products each. An infinite bound of the other side, whose
// factor is 0 because no head has that sign, takes no part: 0 inf would be NaN and place the page first. Such sums are taken again, so
// that finite ones cost a comparison.
template <typename T> struct PageScore {
  const PagedArgs& p;
  const T* bounds;
  const int kh, lane;
  const T* q;  // the sequence's
  double A[8], B[8];
  __device__ inline void load_q(int i) {
    q = static_cast<const T*>(p.q) + i * p.ldq;
    const int G = p.heads / p.cache.kv_heads, j = lane & 7;
#pragma unroll
    for (int e = 0; e < 8; ++e) A[e] = B[e] = 0.0;
    for (int g0 = 0; g0 < G; g0 += 4) {  // four heads under way
      float x[4][8] = {};
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (g0 + g < G) load8(q + (long(kh) * G + g0 + g) * 64 + j * 8, x[g]);
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          A[e] += x[g][e] > 0.f ? double(x[g][e]) : 0.0;
          B[e] += x[g][e] > 0.f ? 0.0 : double(x[g][e]);
        }
    }
  }
  // The lane's products as the definition has them, where the plain sum is NaN: a query of 0 beside an infinite bound gives NaN
  // (as q k does with such a key), one of the other sign leaves it out. All of it read again, one channel at a time: the
  // registers of the way without it are kept.
  __device__ inline double careful(int page) const {
    if (!page_ok(page, p.cache.pages)) return 0.0;  // no place's score
    const int G = p.heads / p.cache.kv_heads, j = lane & 7;
    double s = 0;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const T* at = bounds + (long(page) * p.cache.kv_heads + kh) * 128 + j * 8 + e;
      double l = to_f(at[0]), h = to_f(at[64]), a = 0, b = 0;
      bool zero = false;
#pragma unroll 1
      for (int g = 0; g < G; ++g) {
        const float x = to_f(q[(long(kh) * G + g) * 64 + j * 8 + e]);
        a += x > 0.f ? double(x) : 0.0;
        b += x > 0.f ? 0.0 : double(x);
        zero |= x == 0.f;
      }
      if (!zero && b == 0.0 && fabs(l) == double(INFINITY)) l = 0.0;
      if (!zero && a == 0.0 && fabs(h) == double(INFINITY)) h = 0.0;
      s += l * b + h * a;
      if (zero) s += 0.0 * l + 0.0 * h;
    }
    return s;
  }
  // 16 pages, two for each 8 lanes: page[k] is place + 8 k's (below 0: none); put(place, key) once for each place.
  template <typename Put> __device__ inline void score(const int (&page)[2], int place, Put&& put) const {
    const int j = lane & 7;
    float lo[2][8] = {}, hi[2][8] = {};
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (page_ok(page[k], p.cache.pages)) {
        const T* at = bounds + (long(page[k]) * p.cache.kv_heads + kh) * 128 + j * 8;
        load8(at, lo[k]);
        load8(at + 64, hi[k]);
      }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      double s = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) s += double(lo[k][e]) * B[e] + double(hi[k][e]) * A[e];
      if (s != s) s = careful(page[k]);
      s = sum8(s);
      if (j == 0) put(place + 8 * k, page_ok(page[k], p.cache.pages) ? order_of(s) : 0);
    }
  }
};

// A wave takes 16 pages of one (sequence, key head); bound by its two dependent loads (the table's entry with the
// length, the bounds) and, in 64 bits, its products: 3241 pages of 12 heads (bf16) 6.2 us, 1 us of it for the 64 bits; 16
// lanes a page took 6.4, 64 pages a wave 6.6.
constexpr int SCORE_PAGES = 64;  // a block
template <typename T>
__global__ void __launch_bounds__(256) page_score_kernel(const PagedArgs p, const T* bounds, int maxp, uint64_t* keys) {
  const KvCache& c = p.cache;
  const int chunks = (maxp + SCORE_PAGES - 1) / SCORE_PAGES, chunk = blockIdx.x % chunks, pair = blockIdx.x / chunks;
  const int i = pair / c.kv_heads, lane = threadIdx.x & 63;
  const int held = int((long(length_of(uload(p.lens + i), p.width, c.shift, p.max_len)) + c.page_size - 1) >> c.shift);
  const int p0 = chunk * SCORE_PAGES + (threadIdx.x >> 6) * 16 + (lane >> 3);
  int page[2];  // read together with the length, whatever it is
#pragma unroll
  for (int k = 0; k < 2; ++k) page[k] = p.table[long(i) * p.width + min(p0 + 8 * k, p.width - 1)];
  if (chunk * SCORE_PAGES >= held) return;
  PageScore<T> score{p, bounds, pair % c.kv_heads, lane};
  score.load_q(i);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (p0 + 8 * k >= held) page[k] = -1;
  score.score(page, p0, [&](int at, uint64_t key) {
    if (at < held) keys[long(pair) * maxp + at] = key;
  });
}

// One block a (sequence, key head): the topk largest keys' places, ascending, the lowest place first among equal
// keys, -1 behind them; the newest page is taken first. The keys that are still undecided lie in [lo, hi]; they
// are counted into up to 512 equal bins of that range, the bins above the border's are taken, and its bin is the
// next range: two rounds for most scores, seven at most. Counts do not hang on the order of the atomic adds, and
// every wave reads all bins for itself, so that a round has one barrier: of three sets of bins one is counted
// into, one cleared, and one may still be read. What bounds the kernel is the chain of these steps: 405 of 3241 pages, 12
// heads, 6.0 us on 512 threads (256: 8.9, 1024: 6.5; with block-wide sums between the steps 11.3).
// Thread t holds keys [t K, (t + 1) K) in registers (K > 0), or reads them every round (K = 0, `k` each). FUSED (K = 1, a
// wave for every 16 pages): the block scores the pages itself, a launch less for sequences of few pages (3 pages 4.9 us
// against 3.5 + 4.0, 125 pages 6.9 against 4.3 + 4.7; 256 pages 9.2 against 4.0 + 4.4).
constexpr int SELECT_BINS = 512;
template <int THREADS, int K, typename T = void>
__global__ void __launch_bounds__(THREADS) page_select_kernel(const PagedArgs p, const uint64_t* keys, const void* bounds, int maxp, int k, int topk, int* sel) {
  constexpr bool FUSED = !std::is_void<T>::value;
  constexpr int WAVES = THREADS / 64, EACH = SELECT_BINS / 64;
  __shared__ __attribute__((aligned(16))) int bins[3][SELECT_BINS];
  __shared__ int room[2][WAVES];
  __shared__ uint32_t ends[2][WAVES];
  const KvCache& c = p.cache;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = blockIdx.x / c.kv_heads;
  const uint64_t* in = keys + long(blockIdx.x) * maxp;
  int* out = sel + long(blockIdx.x) * topk;
  uint64_t mine[K > 0 ? K : 1];
  if constexpr (K > 0 && !FUSED) {  // with the length, whatever it is
    k = K;
#pragma unroll
    for (int e = 0; e < K; ++e) mine[e] = tid * K + e < maxp ? in[tid * K + e] : 0;
  }
  const int held = int((long(length_of(uload(p.lens + i), p.width, c.shift, p.max_len)) + c.page_size - 1) >> c.shift);
  const int newest = held - 1;
  const bool newest_there = held > 0 && page_ok(uload(p.table + long(i) * p.width + max(newest, 0)), c.pages);
  if constexpr (FUSED) {
    static_assert(K == 1, "a key a thread");
    __shared__ uint64_t scored[WAVES * 16];
    PageScore<T> score{p, static_cast<const T*>(bounds), int(blockIdx.x % c.kv_heads), lane};
    const int at = wave * 16 + (lane >> 3);
    int page[2];  // read together with the length, whatever it is
#pragma unroll
    for (int e = 0; e < 2; ++e) page[e] = p.table[long(i) * p.width + min(at + 8 * e, p.width - 1)];
    score.load_q(i);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (at + 8 * e >= held) page[e] = -1;
    score.score(page, at, [&](int place, uint64_t key) { scored[place] = key; });
    __syncthreads();
    mine[0] = tid < WAVES * 16 ? scored[tid] : 0;
  }
  // fn(place, key) for this thread's places before the newest; 0: no page there
  auto each = [&](auto&& fn) {
    if constexpr (K > 0) {
#pragma unroll
      for (int e = 0; e < K; ++e) fn(tid * K + e, mine[e]);
    } else {
      for (int e = 0; e < k; ++e) {
        const long at = long(tid) * k + e;
        if (at < newest) fn(int(at), in[at]);
      }
    }
  };
  if constexpr (K > 0) {
#pragma unroll
    for (int e = 0; e < K; ++e)
      if (tid * K + e >= newest) mine[e] = 0;
  }
  for (int b = tid; b < SELECT_BINS; b += THREADS) bins[0][b] = 0;
  // the range of the keys' upper halves
  uint32_t low32 = ~0u, high32 = 0;
  each([&](int, uint64_t key) {
    if (key) low32 = min(low32, uint32_t(key >> 32));
    high32 = max(high32, uint32_t(key >> 32));
  });
  low32 = scan_wave(int(low32), -1, [](int a, int b) { return int(min(uint32_t(a), uint32_t(b))); });
  high32 = scan_wave(int(high32), 0, [](int a, int b) { return int(max(uint32_t(a), uint32_t(b))); });
  if (lane == 63) {
    ends[0][wave] = low32;
    ends[1][wave] = high32;
  }
  __syncthreads();
  low32 = ends[0][0];
  high32 = ends[1][0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    low32 = min(low32, ends[0][w]);
    high32 = max(high32, ends[1][w]);
  }
  uint64_t lo = uint64_t(low32) << 32, hi = uint64_t(high32) << 32 | 0xffffffffu;
  if (lo == 0) lo = 1;  // 0 is no key
  int need = topk - int(newest_there), inside = -1;  // to take from [lo, hi], and how many lie in it: known from the first round on
  for (int round = 0; need > 0 && need != inside && lo < hi; ++round) {
    const int shift = max(0, 55 - __clzll(hi - lo));  // (hi - lo) >> shift < 512
    int* now = bins[round % 3];
    int* next = bins[(round + 1) % 3];
    for (int b = tid; b < SELECT_BINS; b += THREADS) next[b] = 0;
    each([&](int, uint64_t key) {
      if (key >= lo && key <= hi) atomicAdd(&now[int((key - lo) >> shift)], 1);
    });
    __syncthreads();
    // lane t has the t-th EACH bins from above
    int cnt[EACH], sum = 0;
#pragma unroll
    for (int b = 0; b < EACH; b += 4) *reinterpret_cast<int4*>(cnt + b) = *reinterpret_cast<const int4*>(now + SELECT_BINS - EACH * (lane + 1) + b);
#pragma unroll
    for (int b = 0; b < EACH; ++b) sum += cnt[b];
    const int upto = sum_wave(sum), all = __builtin_amdgcn_readlane(upto, 63);
    if (round == 0) need = min(need, all);
    if (need == 0 || need == all) {
      inside = all;
      break;
    }
    int above = upto - sum, bin = 0, got = 0, passed = 0;
#pragma unroll
    for (int b = EACH - 1; b >= 0; --b) {
      if (above < need && need <= above + cnt[b]) {
        bin = SELECT_BINS - EACH * (lane + 1) + b;
        got = cnt[b];
        passed = above;
      }
      above += cnt[b];
    }
    const int who = __builtin_ctzll(__ballot(got > 0));
    need -= __builtin_amdgcn_readlane(passed, who);
    inside = __builtin_amdgcn_readlane(got, who);
    const uint64_t at = lo + (uint64_t(__builtin_amdgcn_readlane(bin, who)) << shift), last = (1ull << shift) - 1;
    if (hi - at > last) hi = at + last;
    lo = at;
  }
  // taken: the newest, what lies above the range, and of the range all or (equal keys) the first `need`
  const bool some = need > 0 && need != inside;
  int eq = 0, before = 0, total = 0;
  if (some) {
    int equal = 0;
    each([&](int, uint64_t key) { equal += key >= lo && key <= hi; });
    const int upto = sum_wave(equal);
    if (lane == 63) room[1][wave] = upto;
    __syncthreads();
    eq = upto - equal;
    for (int w = 0; w < wave; ++w) eq += room[1][w];
  }
  const int first = need > 0 ? need - eq : 0;  // of this thread's equal keys
  int left = some ? first : need > 0 ? k : 0;
  auto takes = [&](uint64_t key, int& left) {
    if (key > hi) return true;
    return key >= lo && key != 0 && left-- > 0;
  };
  int count = 0, l = left;
  each([&](int, uint64_t key) { count += takes(key, l); });
  const int upto = sum_wave(count);
  if (lane == 63) room[0][wave] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += room[0][w];
    total += room[0][w];
  }
  before += upto - count;
  each([&](int at, uint64_t key) {
    if (takes(key, left)) out[before++] = at;
  });
  if (tid == 0 && newest_there) out[total] = newest;
  total += newest_there;
  for (int e = total + tid; e < topk; e += THREADS) out[e] = -1;
}

// Waves up to which a wave of qk_norm_rope_kernel takes one step (five beyond): 2800 tokens of 6 steps 8.7 us against 9.9,
// 5600 tokens 14.1 against 13.9.
constexpr long QK_WAVES = 24576;
constexpr long JOIN_BLOCKS = 256;  // of paged_join_kernel, beyond which a block takes several heads
constexpr int FUSE_MAX = 128;      // pages up to which page_select_kernel scores them itself

}  // namespace

void block_tables(const Exec& ex, const BlockTableArgs& args) {
  BlockTableArgs a = args;
  check_block_tables(a);
  if (ex.dry) return;
  ProfScope prof(ex, "block_tables", 4.0 * a.cap, 8.0 * a.cap + 16.0 * a.n);
  const bool vec = ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
  // 256 threads a block where each has at most four requests to sum up
  auto launch = [&](auto threads) {
    constexpr int N = decltype(threads)::value;
    const int blocks = int(std::min<long>((long(a.cap) + 4 * N - 1) / (4 * N), N == 256 ? 1024 : 256));
    if (blocks <= 1 || (a.lens != a.past && a.used_out != a.used)) {
      block_tables_kernel<N, true, true><<<std::max(blocks, 1), N, 0, ex.stream>>>(a, vec);
    } else {
      block_tables_kernel<N, true, false><<<blocks, N, 0, ex.stream>>>(a, vec);
      block_tables_kernel<N, false, true><<<1, N, 0, ex.stream>>>(a, vec);
    }
  };
  if (a.n <= 1024) launch(std::integral_constant<int, 256>());
  else launch(std::integral_constant<int, 1024>());
  SPLAT_HIP(hipGetLastError());
}

void qk_norm_rope(const Exec& ex, const QkArgs& args, double base) {
  QkArgs a = args;
  check_qk_norm_rope(a, base);
  check_overlaps(a);
  if (a.tokens == 0 || ex.dry) return;
  if (a.rope != ROPE_NONE) rope_turns(a.rope, base, a.freq);
  const double values = double(a.tokens) * (a.heads + (a.has_cache ? 2 : 1) * a.kv_heads) * 64;
  ProfScope prof(ex, "qk_norm_rope", 12 * values, 2 * values * dtype_size(a.dt));
  by_type(a.dt, [&](auto t) {
    using T = decltype(t);
    // a step of 8 head rows a wave while that leaves waves to spare, else five steps, whose angles are taken once
    const int steps = cdiv(a.heads, 8) + (a.has_cache ? 2 : 1) * cdiv(a.kv_heads, 8), tokens = cdiv(a.tokens, 4);
    auto launch = [&](auto rope) {
      constexpr int R = decltype(rope)::value;
      if (long(a.tokens) * steps <= QK_WAVES) qk_norm_rope_kernel<T, 1, R><<<dim3(tokens, steps), 256, 0, ex.stream>>>(a);
      else qk_norm_rope_kernel<T, 5, R><<<dim3(tokens, cdiv(steps, 5)), 256, 0, ex.stream>>>(a);
    };
    if (a.rope == ROPE_NONE) launch(std::integral_constant<int, ROPE_NONE>());
    else if (a.rope == ROPE_LINE) launch(std::integral_constant<int, ROPE_LINE>());
    else launch(std::integral_constant<int, ROPE_GRID>());
  });
  SPLAT_HIP(hipGetLastError());
}

void page_bounds(const Exec& ex, const BoundsArgs& args) {
  BoundsArgs a = args;
  check_page_bounds(a);
  check_overlaps(a);
  if (a.n == 0 || ex.dry) return;
  const long units = long(a.n) * a.per_seq * a.cache.kv_heads;
  ProfScope prof(ex, "page_bounds", 128.0 * units * a.cache.page_size,
                 units * (a.cache.page_size + 2) * 64.0 * dtype_size(a.cache.dt));
  by_type(a.cache.dt, [&](auto t) { page_bounds_kernel<decltype(t)><<<cdiv(units, 4), 256, 0, ex.stream>>>(a); });
  SPLAT_HIP(hipGetLastError());
}

// The launches of attention over the cache. topk: 0, or the pages that sel lists.
void attend(const Exec& ex, const PagedArgs& a, const int* sel, int topk, char* workspace) {
  const PagedPlan plan = paged_plan(a.cache, a.n, a.heads, a.max_len, topk);
  long* before = reinterpret_cast<long*>(workspace);
  float* parts = reinterpret_cast<float*>(workspace + plan.before_bytes);
  auto launch = [&](auto t, auto sparse) {
    using T = decltype(t);
    constexpr bool S = decltype(sparse)::value;
    if (!plan.workers) {
      paged_whole_kernel<T, S><<<dim3(a.n, plan.cols), PAGED_WAVES * 64, 0, ex.stream>>>(a, sel, topk, a.scale);
      return;
    }
    const dim3 grid(plan.workers / PAGED_WAVES, plan.cols);
    const int span = plan.workers >= 128L * a.n ? PAGED_WAVES : 1;
    if (a.n <= SCAN_MAX) {
      paged_parts_kernel<T, S, true><<<grid, PAGED_WAVES * 64, 0, ex.stream>>>(a, sel, topk, a.scale, plan.workers, span, before, parts);
    } else {
      paged_scan_kernel<TileOps<T>::KEYS><<<1, 1024, 0, ex.stream>>>(a, topk, before);
      paged_parts_kernel<T, S, false><<<grid, PAGED_WAVES * 64, 0, ex.stream>>>(a, sel, topk, a.scale, plan.workers, span, before, parts);
    }
    // a head a block, with eight waves on its parts, until there are blocks enough
    const int most = std::min(a.heads / a.cache.kv_heads, 16), per = int(std::min<long>(most, std::max<long>(1, long(a.n) * a.heads / JOIN_BLOCKS)));
    paged_join_kernel<T><<<dim3(a.n, plan.cols * cdiv(most, per)), JOIN_WAVES * 64, 0, ex.stream>>>(a, plan.workers, span, per, before, parts);
  };
  by_type(a.cache.dt, [&](auto t) {
    if (topk) launch(t, std::true_type());
    else launch(t, std::false_type());
  });
}

void paged_attention(const Exec& ex, const PagedArgs& args, void* workspace, size_t bytes) {
  PagedArgs a = args;
  check_paged_attention(a, workspace, bytes);
  if (a.n == 0 || ex.dry) return;
  const double keys = double(a.n) * a.max_len;
  ProfScope prof(ex, "paged_attention", 256 * keys * a.heads, 128 * keys * a.cache.kv_heads * dtype_size(a.cache.dt));
  attend(ex, a, nullptr, 0, static_cast<char*>(workspace));
  SPLAT_HIP(hipGetLastError());
}

void sparse_attention(const Exec& ex, const SparseArgs& args, void* workspace, size_t bytes) {
  SparseArgs s = args;
  check_sparse_attention(s, workspace, bytes);
  const PagedArgs& a = s.at;
  if (a.n == 0 || ex.dry) return;
  const int pairs = a.n * a.cache.kv_heads, maxp = cdiv(a.max_len, a.cache.page_size);
  const double rows = 2.0 * maxp + 2.0 * std::min(s.topk, maxp) * a.cache.page_size;
  ProfScope prof(ex, "sparse_attention", 256.0 * a.n * a.heads * std::min(s.topk, maxp) * a.cache.page_size,
                 pairs * rows * 64 * dtype_size(a.cache.dt));
  char* ws = static_cast<char*>(workspace);
  uint64_t* keys = reinterpret_cast<uint64_t*>(ws + paged_plan(a.cache, a.n, a.heads, a.max_len, s.topk).bytes);
  by_type(a.cache.dt, [&](auto t) {
    using T = decltype(t);
    auto select = [&](auto kernel, int threads) {
      kernel<<<pairs, threads, 0, ex.stream>>>(a, keys, s.bounds, maxp, cdiv(maxp, threads), s.topk, s.selected);
    };
    if (maxp <= FUSE_MAX) {
      // 16 pages a wave, all at once
      if (maxp <= 64) select(page_select_kernel<256, 1, T>, 256);
      else select(page_select_kernel<512, 1, T>, 512);
      return;
    }
    page_score_kernel<T><<<pairs * cdiv(maxp, SCORE_PAGES), 256, 0, ex.stream>>>(a, static_cast<const T*>(s.bounds), maxp, keys);
    if (maxp <= 1024) select(page_select_kernel<256, 4>, 256);
    else if (maxp <= 4096) select(page_select_kernel<512, 8>, 512);
    else if (maxp <= 16384) select(page_select_kernel<1024, 16>, 1024);
    else select(page_select_kernel<1024, 0>, 1024);
  });
  attend(ex, a, s.selected, s.topk, ws);
  SPLAT_HIP(hipGetLastError());
}

}  // namespace splat
