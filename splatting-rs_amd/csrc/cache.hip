// A paged cache of keys and values and the operators on it: block tables and slot maps, per-head norms
// with the position rotation (storing into the cache), key bounds per page, attention of one token per
// sequence over its pages, and the same over the pages that a score selects.
//
// Head dim 64, as everywhere in the library. Position p of a sequence lies in row p % page_size of the page
// its table names for p / page_size; (page, head) holds page_size rows of 64 channels back to back.
// Entries of a table outside [0, pages) hold no keys: every kernel checks them before it forms an address.
#include "kernels.h"

#include <algorithm>

namespace splat {

namespace {

// Sum over the 8 lanes of a head row; every lane gets it.
__device__ inline float sum8(float v) {
#pragma unroll
  for (int m = 1; m < 8; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// 8 consecutive channels.
template <typename T> __device__ inline void load8(const T* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = u16f<T>(u[i]);
    x[2 * i + 1] = u16f<T>(u[i] >> 16);
  }
}
template <> __device__ inline void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <typename T> __device__ inline void store8(T* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}
template <> __device__ inline void store8<float>(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// --- block tables and slot maps -----------------------------------------------------------------

constexpr int TABLE_THREADS = 1024;

// Request i holds past[i] positions in ceil(past / ps) pages; its add[i] new ones take the next pages of
// the pool, requests in order. Every block sums the requests up again (thread t its k of them, then one scan
// over the threads), so that a token finds its request and its page without a pass before: a binary search
// over the threads' sums, then a walk over at most k requests. A new page begins with a new token, whose
// thread writes the table's entry.
// The call takes effect whole or not at all: the status is known before anything is written.
// FILL writes the table, slots and positions, COMMIT lens, starts, used and status, which may lie over
// past and used: with several blocks it runs as a second launch.
template <bool FILL, bool COMMIT>
__global__ void __launch_bounds__(TABLE_THREADS) block_tables_kernel(const BlockTableArgs p) {
  __shared__ long tok[TABLE_THREADS + 1], pag[TABLE_THREADS + 1];
  __shared__ long wtok[16], wpag[16];
  __shared__ int bad_any;
  const int tid = threadIdx.x, k = (p.n + TABLE_THREADS - 1) / TABLE_THREADS;
  const int i0 = int(min(long(tid) * k, long(p.n))), i1 = int(min(long(i0) + k, long(p.n)));
  const int ps = 1 << p.shift;
  const long most = long(p.width) << p.shift;
  if (tid == 0) bad_any = 0;
  const int used = *p.used;
  long nt = 0, np = 0;
  bool bad = false;
  for (int i = i0; i < i1; ++i) {
    const long a = p.past[i], d = p.add[i];
    bad |= a < 0 || d < 0 || a + d > most;
    nt += d;
    np += ((a + d + ps - 1) >> p.shift) - ((a + ps - 1) >> p.shift);
  }
  __syncthreads();
  if (bad) bad_any = 1;
  long st = nt, sp = np;  // inclusive scan over the wave, then over the waves
  const int lane = tid & 63, wave = tid >> 6;
  for (int m = 1; m < 64; m <<= 1) {
    const long ot = __shfl_up(st, m), op = __shfl_up(sp, m);
    if (lane >= m) { st += ot; sp += op; }
  }
  if (lane == 63) { wtok[wave] = st; wpag[wave] = sp; }
  __syncthreads();
  long bt = 0, bp = 0, total = 0, pages = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) { bt += wtok[w]; bp += wpag[w]; }
    total += wtok[w];
    pages += wpag[w];
  }
  const long et = bt + st - nt, ep = bp + sp - np;  // exclusive
  tok[tid] = et;
  pag[tid] = ep;
  const bool broken = bad_any != 0 || used < 0 || used > p.pool_size;
  const int status = broken ? TABLE_BAD_LENGTH : pages > long(p.pool_size) - used ? TABLE_POOL_EMPTY
                     : total > p.cap ? TABLE_SLOTS_FULL : TABLE_OK;
  __syncthreads();
  if constexpr (FILL) {
    const long count = status == TABLE_OK ? total : 0;
    for (long t = long(blockIdx.x) * TABLE_THREADS + tid; t < p.cap; t += long(gridDim.x) * TABLE_THREADS) {
      int slot = -1, pos = 0;
      if (t < count) {
        int lo = 0, hi = TABLE_THREADS;  // the last thread whose sum is at most t
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (tok[mid] <= t) lo = mid;
          else hi = mid;
        }
        long r = t - tok[lo], pg = pag[lo];
        int i = int(min(long(lo) * k, long(p.n)));
        int a = p.past[i], d = p.add[i];
        while (r >= d) {  // ends: the thread's requests hold more than r tokens
          r -= d;
          pg += ((long(a) + d + ps - 1) >> p.shift) - ((long(a) + ps - 1) >> p.shift);
          ++i;
          a = p.past[i];
          d = p.add[i];
        }
        pos = a + int(r);
        const int j = pos >> p.shift, have = int((long(a) + ps - 1) >> p.shift);
        int page;
        if (j < have) {
          page = p.table[long(i) * p.width + j];
        } else {
          page = p.pool[used + pg + (j - have)];
          if ((pos & (ps - 1)) == 0) p.table[long(i) * p.width + j] = page;
        }
        const long s = (long(page) << p.shift) + (pos & (ps - 1));
        slot = page < 0 || s > 0x7fffffffL ? -1 : int(s);
      }
      p.slots[t] = slot;
      if (p.positions) p.positions[t] = pos;
    }
  }
  if constexpr (COMMIT) {
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

// One wave a token: 8 lanes hold a head row (8 channels each), 8 rows at a time. Lane l < 32 takes
// frequency l's angle once for all heads, in 64 bits up to the fraction of a turn.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QkArgs p) {
  __shared__ float2 turn[4][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long t = long(blockIdx.x) * 4 + wave;
  if (t >= p.tokens) return;
  const int j = lane & 7;
  if (p.rope != ROPE_NONE) {
    if (lane < 32) {
      const int pos = p.rope == ROPE_LINE ? p.positions[t] : p.positions[2 * t + (lane >> 4)];
      const double x = double(pos) * p.freq[p.rope == ROPE_LINE ? lane : lane & 15];
      float s, c;
      sincospif(float(2.0 * (x - rint(x))), &s, &c);
      turn[wave][lane] = make_float2(c, s);
    }
    __builtin_amdgcn_wave_barrier();
  }
  const int slot = p.slots ? p.slots[t] : -1;
  const bool cached = p.slots && slot_ok(slot, p.cache);
  const int R = p.heads + (p.slots ? 2 : 1) * p.kv_heads;
  for (int r0 = 0; r0 < R; r0 += 8) {
    const int r = r0 + (lane >> 3);
    const bool in = r < R;
    float x[8] = {};
    if (in) load8(static_cast<const T*>(p.qkv) + t * p.ld + r * 64 + j * 8, x);
    const bool isq = r < p.heads, isk = !isq && r < p.heads + p.kv_heads;
    if (isq || isk) {
      const float* w = isq ? p.qw : p.kw;
      const float* b = isq ? p.qb : p.kb;
      if (p.norm != NORM_NONE) {
        float m = 0.f, v = 0.f;
        if (p.norm == NORM_LAYER) {
#pragma unroll
          for (int e = 0; e < 8; ++e) m += x[e];
          m = sum8(m) * (1.f / 64.f);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[e] -= m; v += x[e] * x[e]; }
        const float s = 1.f / sqrtf(sum8(v) * (1.f / 64.f) + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] *= s;
          if (w) x[e] *= w[j * 8 + e];
          if (b) x[e] += b[j * 8 + e];
        }
      }
      if (p.rope != ROPE_NONE) {
        const int span = p.rope == ROPE_LINE ? 4 : 2;  // the partner's lane, and this lane's first frequency
        const int f0 = p.rope == ROPE_LINE ? (j & 3) * 8 : (j >> 2) * 16 + (j & 1) * 8;
        const float sign = (j & span) ? 1.f : -1.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 cs = turn[wave][f0 + e];
          const float o = __shfl_xor(x[e], span);
          x[e] = x[e] * cs.x + sign * o * cs.y;
        }
      }
    }
    if (!in) continue;
    if (isq) {
      store8(static_cast<T*>(p.q_out) + t * p.ldq + r * 64 + j * 8, x);
      continue;
    }
    const int h = isk ? r - p.heads : r - p.heads - p.kv_heads;
    if (isk && p.k_out) store8(static_cast<T*>(p.k_out) + t * p.ldk + h * 64 + j * 8, x);
    if (cached) {
      store8(static_cast<T*>(isk ? p.cache.k : p.cache.v) + slot_at(p.cache, slot, h) + j * 8, x);
    }
  }
}

// --- key bounds per page ------------------------------------------------------------------------

// NaN in either operand gives NaN.
__device__ inline float low(float a, float b) { return b < a || b != b ? b : a; }
__device__ inline float high(float a, float b) { return b > a || b != b ? b : a; }

// One wave a (sequence, page, head), 8 lanes a row, 8 rows at a time.
template <typename T>
__global__ void __launch_bounds__(256) page_bounds_kernel(const BoundsArgs p) {
  const KvCache& c = p.cache;
  const long unit = long(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (unit >= long(p.n) * p.per_seq * c.kv_heads) return;
  const int lane = threadIdx.x & 63, j = lane & 7, ps = 1 << c.shift;
  const int h = int(unit % c.kv_heads), first = int(unit / c.kv_heads % p.per_seq), i = int(unit / c.kv_heads / p.per_seq);
  const int len = length_of(p.lens[i], p.width, c.shift, 0x7fffffff);
  const int fresh = p.add ? min(max(p.add[i], 0), len) : len;
  if (fresh == 0) return;
  const int last = (len + ps - 1) >> c.shift;
  for (int g = ((len - fresh) >> c.shift) + first; g < last; g += p.per_seq) {
    const int page = p.table[long(i) * p.width + g];
    if (!page_ok(page, c.pages)) continue;
    const int rows = min(ps, len - (g << c.shift));
    const T* k = static_cast<const T*>(c.k) + page_at(c, page, h) + j * 8;
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] = INFINITY; hi[e] = -INFINITY; }
    for (int r = lane >> 3; r < rows; r += 8) {
      float x[8];
      load8(k + r * 64, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) { lo[e] = low(lo[e], x[e]); hi[e] = high(hi[e], x[e]); }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int m = 8; m < 64; m <<= 1) {
        lo[e] = low(lo[e], __shfl_xor(lo[e], m));
        hi[e] = high(hi[e], __shfl_xor(hi[e], m));
      }
    T* out = static_cast<T*>(p.bounds) + (long(page) * c.kv_heads + h) * 128 + j * 8;
    if (lane < 8) store8(out, lo);
    else if (lane < 16) store8(out + 64, hi);
  }
}

// --- attention of one token over the cache ------------------------------------------------------

// One wave a (sequence, query head): 8 lanes a key row, 8 keys at a time, a running maximum and sum for
// each of the 8 groups of lanes, joined at the end. `sel` != null: only the pages that it lists.
template <typename T>
__global__ void __launch_bounds__(64) paged_attention_kernel(const PagedArgs p, const int* sel, int topk) {
  const int lane = threadIdx.x, g = lane >> 3, j = lane & 7;
  const int h = blockIdx.x % p.heads, i = blockIdx.x / p.heads, kh = h / (p.heads / p.cache.kv_heads);
  const KvCache& c = p.cache;
  const int ps = 1 << c.shift;
  const int len = length_of(p.lens[i], p.width, c.shift, p.max_len);
  float q[8], o[8] = {};
  load8(static_cast<const T*>(p.q) + i * p.ldq + h * 64 + j * 8, q);
  const float scale = p.scale * 1.44269504088896341f;
  float m = -INFINITY, l = 0.f;
  bool some = false;
  const int count = sel ? topk : (len + ps - 1) >> c.shift;
  for (int a = 0; a < count; ++a) {
    const int pi = sel ? sel[(long(i) * c.kv_heads + kh) * topk + a] : a;
    if (pi < 0) break;
    const int page = p.table[long(i) * p.width + pi];
    if (!page_ok(page, c.pages)) continue;
    const int rows = min(ps, len - (pi << c.shift));
    const long at = page_at(c, page, kh) + j * 8;
    for (int r = g; r < rows; r += 8) {
      float x[8], s = 0.f;
      load8(static_cast<const T*>(c.k) + at + r * 64, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += q[e] * x[e];
      s = sum8(s) * scale;
      const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;
      const float keep = exp2f(m - ref), w = exp2f(s - ref);
      load8(static_cast<const T*>(c.v) + at + r * 64, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = o[e] * keep + w * x[e];
      l = l * keep + w;
      m = mn;
      some = true;
    }
  }
#pragma unroll
  for (int d = 8; d < 64; d <<= 1) {
    const float om = __shfl_xor(m, d), ol = __shfl_xor(l, d);
    const bool os = __shfl_xor(int(some), d);
    const float mn = fmaxf(m, om), ref = mn == -INFINITY ? 0.f : mn;
    // a side without keys has no part, whatever the other holds
    const float a = some ? exp2f(m - ref) : 0.f, b = os ? exp2f(om - ref) : 0.f;
    l = l * a + ol * b;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * a + __shfl_xor(o[e], d) * b;
    m = mn;
    some |= os;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = some ? o[e] / l : 0.f;
  if (lane < 8) store8(static_cast<T*>(p.out) + i * p.ldo + h * 64 + j * 8, o);
}

// --- selection of pages -------------------------------------------------------------------------

// Scores as whole numbers in the order of the scores, NaN above all; 0: not a page of the sequence.
__device__ inline uint64_t order_of(double s) {
  if (s != s) return ~0ull - 1;
  const uint64_t b = __double_as_longlong(s);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

// One block a (sequence, key head). The most that q k can be for a key between the page's bounds, summed
// over the group's heads, is sum_c hi_c A_c + lo_c B_c with A and B the sums of the positive and the negative
// parts of the heads' queries. In 64 bits: a page next to the border is chosen or not by less than 32 bits
// hold.
template <typename T>
__global__ void __launch_bounds__(256) page_score_kernel(const PagedArgs p, const T* bounds, int maxp, uint64_t* keys) {
  __shared__ double A[64], B[64];
  const KvCache& c = p.cache;
  const int i = blockIdx.x / c.kv_heads, kh = blockIdx.x % c.kv_heads, G = p.heads / c.kv_heads;
  if (threadIdx.x < 64) {
    double a = 0, b = 0;
    for (int g = 0; g < G; ++g) {
      const double x = to_f<T>(static_cast<const T*>(p.q)[i * p.ldq + (kh * G + g) * 64 + threadIdx.x]);
      if (x > 0) a += x;
      else b += x;
    }
    A[threadIdx.x] = a;
    B[threadIdx.x] = b;
  }
  __syncthreads();
  const int ps = 1 << c.shift;
  const int len = length_of(p.lens[i], p.width, c.shift, p.max_len);
  const int held = (len + ps - 1) >> c.shift;
  for (int j = threadIdx.x; j < maxp; j += 256) {
    uint64_t key = 0;
    const int page = j < held ? p.table[long(i) * p.width + j] : -1;
    if (page_ok(page, c.pages)) {
      const T* lo = bounds + (long(page) * c.kv_heads + kh) * 128;
      double s = 0;
      for (int d = 0; d < 64; ++d) s += double(to_f<T>(lo[d])) * B[d] + double(to_f<T>(lo[64 + d])) * A[d];
      key = j == held - 1 ? ~0ull : order_of(s);
    }
    keys[(long(i) * c.kv_heads + kh) * maxp + j] = key;
  }
}

// The topk largest keys' places in ascending order, the lowest place first among equal keys, -1 behind them.
__global__ void __launch_bounds__(256) page_select_kernel(const uint64_t* keys, int maxp, int topk, int* sel) {
  const uint64_t* k = keys + long(blockIdx.x) * maxp;
  int* out = sel + long(blockIdx.x) * topk;
  __shared__ int total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  for (int b = 0; b < maxp; b += 256) {
    const int j = b + threadIdx.x;
    bool take = false;
    if (j < maxp && k[j] != 0) {
      int ahead = 0;
      for (int o = 0; o < maxp; ++o) ahead += k[o] > k[j] || (k[o] == k[j] && o < j);
      take = ahead < topk;
    }
    __shared__ int flags[256];
    flags[threadIdx.x] = take;
    __syncthreads();
    int at = total, all = 0;
    for (int o = 0; o < 256; ++o) {
      if (o < int(threadIdx.x)) at += flags[o];
      all += flags[o];
    }
    if (take) out[at] = j;
    __syncthreads();
    if (threadIdx.x == 0) total += all;
    __syncthreads();
  }
  for (int a = total + threadIdx.x; a < topk; a += 256) out[a] = -1;
}

// Runs fn with the storage type dt as a value.
template <typename F> void by_type(int dt, F&& fn) {
  if (dt == F32) fn(float());
  else if (dt == BF16) fn(bf16());
  else fn(f16());
}

}  // namespace

void block_tables(const Exec& ex, const BlockTableArgs& args) {
  BlockTableArgs a = args;
  check_block_tables(a);
  if (ex.dry) return;
  ProfScope prof(ex, "block_tables", 4.0 * a.cap, 8.0 * a.cap + 16.0 * a.n);
  const int blocks = std::min(cdiv(a.cap, TABLE_THREADS), 512);
  if (blocks <= 1) {
    block_tables_kernel<true, true><<<1, TABLE_THREADS, 0, ex.stream>>>(a);
  } else {
    block_tables_kernel<true, false><<<blocks, TABLE_THREADS, 0, ex.stream>>>(a);
    block_tables_kernel<false, true><<<1, TABLE_THREADS, 0, ex.stream>>>(a);
  }
  SPLAT_HIP(hipGetLastError());
}

void qk_norm_rope(const Exec& ex, const QkArgs& args, double base) {
  QkArgs a = args;
  check_qk_norm_rope(a, base);
  if (a.tokens == 0 || ex.dry) return;
  if (a.rope != ROPE_NONE) rope_turns(a.rope, base, a.freq);
  const double values = double(a.tokens) * (a.heads + (a.has_cache ? 2 : 1) * a.kv_heads) * 64;
  ProfScope prof(ex, "qk_norm_rope", 12 * values, 2 * values * dtype_size(a.dt));
  by_type(a.dt, [&](auto t) {
    qk_norm_rope_kernel<decltype(t)><<<cdiv(a.tokens, 4), 256, 0, ex.stream>>>(a);
  });
  SPLAT_HIP(hipGetLastError());
}

void page_bounds(const Exec& ex, const BoundsArgs& args) {
  BoundsArgs a = args;
  check_page_bounds(a);
  if (a.n == 0 || ex.dry) return;
  const long units = long(a.n) * a.per_seq * a.cache.kv_heads;
  ProfScope prof(ex, "page_bounds", 128.0 * units * a.cache.page_size,
                 units * (a.cache.page_size + 2) * 64.0 * dtype_size(a.cache.dt));
  by_type(a.cache.dt, [&](auto t) { page_bounds_kernel<decltype(t)><<<cdiv(units, 4), 256, 0, ex.stream>>>(a); });
  SPLAT_HIP(hipGetLastError());
}

void paged_attention(const Exec& ex, const PagedArgs& args, void* workspace, size_t bytes) {
  PagedArgs a = args;
  check_paged_attention(a, workspace, bytes);
  if (a.n == 0 || ex.dry) return;
  const double keys = double(a.n) * a.max_len;
  ProfScope prof(ex, "paged_attention", 256 * keys * a.heads, 128 * keys * a.cache.kv_heads * dtype_size(a.cache.dt));
  by_type(a.cache.dt, [&](auto t) {
    paged_attention_kernel<decltype(t)><<<a.n * a.heads, 64, 0, ex.stream>>>(a, nullptr, 0);
  });
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
  uint64_t* keys = static_cast<uint64_t*>(workspace);
  by_type(a.cache.dt, [&](auto t) {
    using T = decltype(t);
    page_score_kernel<T><<<pairs, 256, 0, ex.stream>>>(a, static_cast<const T*>(s.bounds), maxp, keys);
    page_select_kernel<<<pairs, 256, 0, ex.stream>>>(keys, maxp, s.topk, s.selected);
    paged_attention_kernel<T><<<a.n * a.heads, 64, 0, ex.stream>>>(a, s.selected, s.topk);
  });
  SPLAT_HIP(hipGetLastError());
}

}  // namespace splat
