// A paged cache of keys and values and the operators on it: block tables and slot maps, per-head norms
// with the position rotation (storing into the cache), key bounds per page, attention of one token per
// sequence over its pages, and the same over the pages that a score selects.
//
// Head dim 64, as everywhere in the library. Position p of a sequence lies in row p % page_size of the page
// its table names for p / page_size; (page, head) holds page_size rows of 64 channels back to back.
// Entries of a table outside [0, pages) hold no keys: every kernel checks them before it forms an address.
#include "kernels.h"

#include <algorithm>
#include <type_traits>

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
//
// S^T = K Q^T and O^T = V^T P^T on the 16x16 matrix instructions, the query heads that share a key head as the
// 16 columns (fewer: columns of zeros, which cost nothing, since the bytes of K and V bound the kernel).
// The scores come out with a lane holding one head (lane % 16) and keys 4 (lane / 16) + r, which is the
// operand layout of the second product as it stands; V is read transposed from LDS.
//
// A wave works alone: tiles of 32 keys (16 in fp32: 4 KB of K and 4 KB of V in every type) stream into its own
// ring in LDS, four loads of 1 KB for each, that many bytes ahead, and no barrier holds it up. A load covers 8
// rows (4 in fp32) of one page, and the rows that are not there (past the length, a missing page) lie outside
// its buffer, so that they arrive as zeros whatever memory holds.

typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int int32x4_v __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(3))) char* lds_cptr;

// A wave-uniform load of memory that the launch only reads.
__device__ inline int uload(const int* p) { return *(const __attribute__((address_space(4))) int*)p; }
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// 16 bytes a lane from `base + off` into LDS at lds + 16 * lane; offsets from `bytes` on read as zeros.
__device__ inline void load_lds(const void* base, uint32_t bytes, uint32_t off, uint32_t lds) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const int32x4_v r = {uniform(int(uint32_t(a))), uniform(int(uint32_t(a >> 32))), uniform(int(bytes)), 0x00020000};
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(uniform(int(lds))), "v"(off), "s"(r)
               : "memory");
}
template <int N> __device__ inline void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// Maximum (sum) over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ inline float max_groups(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float sum_groups(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The two products on a tile in LDS. KEYS keys in T16 groups of 16; PIECE rows to a load.
template <typename T> struct TileOps {  // bf16, f16: rows of 128 bytes
  static constexpr int KEYS = 32, T16 = 2, PIECE = 8;
  // f16 weights below 2^-14 lose bits: the largest one is 2^12, so that they do so from 2^-26 of it on.
  static constexpr float TOP = std::is_same<T, f16>::value ? 12.f : 0.f;
  uint4 q[2];
  __device__ inline void load_q(const T* row, int g, bool in) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
      q[s] = in ? *reinterpret_cast<const uint4*>(row + 32 * s + 8 * g) : make_uint4(0, 0, 0, 0);
  }
  // Takes the loads as done here: inside the loop the compiler's wait for them would be one for every tile in flight.
  __device__ inline void pin_q() {
#pragma unroll
    for (int s = 0; s < 2; ++s) asm volatile("" : "+v"(q[s].x), "+v"(q[s].y), "+v"(q[s].z), "+v"(q[s].w));
  }
  // Offset of this lane's 16 bytes within piece `p` (1 KB, 8 rows): chunk c of row r lies in slot c ^ ((r / 2) & 7)
  // for keys, c ^ 2 ((r / 2) & 3) for values, so that the rows that a read takes lie in different banks.
  __device__ static inline uint32_t k_off(int lane, int p) { return (lane >> 3) * 128 + (((lane & 7) ^ (((lane >> 4) + 4 * p) & 7)) * 16); }
  __device__ static inline uint32_t v_off(int lane, int) { return (lane >> 3) * 128 + (((lane & 7) ^ (2 * ((lane >> 4) & 3))) * 16); }
  __device__ static inline f32x4 mma(const uint4& a, const uint4& b, const f32x4& c) {
    if constexpr (std::is_same<T, bf16>::value)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0, 0, 0);
  }
  __device__ inline void scores(const char* kt, int lane, f32x4 (&x)[T16]) const {
    const int row = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 2; ++s)
        a = mma(*reinterpret_cast<const uint4*>(kt + (16 * t + row) * 128 + (((4 * s + g) ^ ((row >> 1) & 7)) * 16)), q[s], a);
      x[t] = a;
    }
  }
  __device__ static inline void weigh(const char* vt, int lane, const f32x4 (&w)[T16], f32x4 (&o)[4]) {
    const int g = lane >> 4, j = (lane >> 2) & 3, cc = lane & 3;
    const uint4 p = make_uint4(pack2<T>(w[0][0], w[0][1]), pack2<T>(w[0][2], w[0][3]), pack2<T>(w[1][0], w[1][1]),
                               pack2<T>(w[1][2], w[1][3]));
    const int row = 4 * g + j;  // and 16 + row, whose chunks lie alike
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      typedef short v4s __attribute__((ext_vector_type(4)));
      const char* at = vt + row * 128 + (((2 * d + (cc >> 1)) ^ (2 * ((row >> 1) & 3))) * 16) + (cc & 1) * 8;
      uint32_t f[4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const v4s r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)((lds_cptr)(at + t * 2048)));
        const uint2 u = __builtin_bit_cast(uint2, r);
        f[2 * t] = u.x;
        f[2 * t + 1] = u.y;
      }
      o[d] = mma(make_uint4(f[0], f[1], f[2], f[3]), p, o[d]);
    }
  }
};
template <> struct TileOps<float> {  // rows of 256 bytes
  static constexpr int KEYS = 16, T16 = 1, PIECE = 4;
  static constexpr float TOP = 0.f;
  float4 q[4];
  __device__ inline void load_q(const float* row, int g, bool in) {
#pragma unroll
    for (int b = 0; b < 4; ++b)
      q[b] = in ? *reinterpret_cast<const float4*>(row + 16 * b + 4 * g) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ inline void pin_q() {
#pragma unroll
    for (int b = 0; b < 4; ++b) asm volatile("" : "+v"(q[b].x), "+v"(q[b].y), "+v"(q[b].z), "+v"(q[b].w));
  }
  // chunk c of row r in slot c ^ r for keys, c ^ 4 (r / 4) for values
  __device__ static inline uint32_t k_off(int lane, int p) { return (lane >> 4) * 256 + (((lane & 15) ^ (4 * p + (lane >> 4))) * 16); }
  __device__ static inline uint32_t v_off(int lane, int p) { return (lane >> 4) * 256 + (((lane & 15) ^ (4 * p)) * 16); }
  __device__ inline void scores(const char* kt, int lane, f32x4 (&x)[T16]) const {
    const int row = lane & 15, g = lane >> 4;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float4 k = *reinterpret_cast<const float4*>(kt + row * 256 + (((4 * b + g) ^ row) * 16));
      a = __builtin_amdgcn_mfma_f32_16x16x4f32(k.x, q[b].x, a, 0, 0, 0);
      a = __builtin_amdgcn_mfma_f32_16x16x4f32(k.y, q[b].y, a, 0, 0, 0);
      a = __builtin_amdgcn_mfma_f32_16x16x4f32(k.z, q[b].z, a, 0, 0, 0);
      a = __builtin_amdgcn_mfma_f32_16x16x4f32(k.w, q[b].w, a, 0, 0, 0);
    }
    x[0] = a;
  }
  __device__ static inline void weigh(const char* vt, int lane, const f32x4 (&w)[T16], f32x4 (&o)[4]) {
    const int g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = *reinterpret_cast<const float*>(vt + (4 * g + r) * 256 + (((4 * d + (c >> 2)) ^ (4 * g)) * 16) + (c & 3) * 4);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, w[0][r], o[d], 0, 0, 0);
      }
  }
};

constexpr int TILE_BYTES = 8192;  // K, then V
constexpr int STAGES = 2;

// Where a wave stands: sequence i holds tiles [base, next) of the launch's row of tiles.
struct Cursor {
  int i;
  long base, next;
};

// Tiles of sequence i: of its positions, or of the pages that were selected.
template <int KEYS> __device__ inline int tiles_of(const PagedArgs& p, int i, int topk) {
  const int len = length_of(p.lens[i], p.width, p.cache.shift, p.max_len);
  if (!topk) return int((long(len) + KEYS - 1) / KEYS);
  const int held = int((long(len) + p.cache.page_size - 1) >> p.cache.shift);
  return int(((long(min(held, topk)) << p.cache.shift) + KEYS - 1) / KEYS);
}

// One wave: the running softmax of one group of heads over tiles [t, end), which may cross sequences.
// finish(cursor, first tile, state) is called at the end of each sequence's part.
template <typename T> struct PagedWave {
  using Ops = TileOps<T>;
  static constexpr int KEYS = Ops::KEYS, PIECE = Ops::PIECE;
  const PagedArgs& p;
  const int* sel;  // [n, kv_heads, topk] or null
  const int topk, kh, lane;
  const uint32_t lds;   // of the wave's ring
  const char* ring;
  Ops ops;
  f32x4 o[4];
  float m, l;
  int some;  // keys were there

  __device__ inline void clear() {
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
    some = 0;
  }

  // Loads local tile t of sequence i into slot b of the ring; the rows of each piece that are there, 8 bits a piece.
  __device__ inline uint32_t issue(int i, int t, int b) {
    const KvCache& c = p.cache;
    const int len = uniform(length_of(uload(p.lens + i), p.width, c.shift, p.max_len)), ps = c.page_size;
    const int held = int((long(len) + ps - 1) >> c.shift), count = topk ? min(held, topk) : held;
    const int* row = p.table + long(i) * p.width;
    uint32_t there = 0;
    int entry[4], rows[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int pos = t * KEYS + k * PIECE, e = pos >> c.shift;
      int j = min(e, count - 1);
      if (topk) j = uload(sel + (long(i) * c.kv_heads + kh) * topk + j);
      entry[k] = uload(row + max(j, 0));
      const int left = len - int(long(j) << c.shift) - (pos & (ps - 1));
      rows[k] = e < count && j >= 0 ? max(0, min(PIECE, left)) : 0;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool ok = page_ok(entry[k], c.pages);
      const int r = ok ? rows[k] : 0;
      there |= uint32_t(r) << (8 * k);
      const long at = (ok ? page_at(c, entry[k], kh) : 0) + long((t * KEYS + k * PIECE) & (ps - 1)) * 64;
      const uint32_t bytes = uint32_t(r) * 64 * sizeof(T), to = lds + b * TILE_BYTES + k * 1024;
      load_lds(static_cast<const T*>(c.k) + at, bytes, Ops::k_off(lane, k), to);
      load_lds(static_cast<const T*>(c.v) + at, bytes, Ops::v_off(lane, k), to + TILE_BYTES / 2);
    }
    return uniform(int(there));
  }

  __device__ inline void tile(int b, uint32_t there, float scale) {
    constexpr uint32_t ALL = PIECE * 0x01010101u;
    const char* kt = ring + b * TILE_BYTES;
    f32x4 x[Ops::T16];
    ops.scores(kt, lane, x);
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
    const float ref = mn == -INFINITY ? 0.f : mn - Ops::TOP;
    // the weights are 2^(x - ref); what was summed against another reference moves along
    const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
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
        x[t][r] = __builtin_amdgcn_exp2f(x[t][r] - ref);
        l += x[t][r];
      }
    Ops::weigh(kt + TILE_BYTES / 2, lane, x, o);
  }

  // Local tiles [t, end) of one sequence with nothing in flight before or after.
  __device__ inline void run(int i, int t, int end, float scale) {
    uint32_t there[STAGES];
#pragma unroll
    for (int b = 0; b < STAGES; ++b) there[b] = t + b < end ? issue(i, t + b, b) : 0;
    ops.pin_q();
    while (t < end) {
#pragma unroll
      for (int b = 0; b < STAGES; ++b) {
        if (t + b >= end) break;
        if (t + b + 1 < end) wait_loads<8 * (STAGES - 1)>();
        else wait_loads<0>();
        tile(b, there[b], scale);
        if (t + b + STAGES < end) there[b] = issue(i, t + b + STAGES, b);
      }
      t += STAGES;
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

// One block a (sequence, group of up to 16 heads of one key head): its waves take a quarter of the tiles each
// and join their sums in LDS.
template <typename T>
__global__ void __launch_bounds__(PAGED_WAVES * 64, 2) paged_whole_kernel(const PagedArgs p, const int* sel, int topk, float scale) {
  using Wave = PagedWave<T>;
  __shared__ __attribute__((aligned(1024))) char smem[PAGED_WAVES * STAGES * TILE_BYTES];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int G = p.heads / p.cache.kv_heads, parts = (G + 15) / 16;
  const int i = blockIdx.x, kh = int(blockIdx.y) / parts, g0 = int(blockIdx.y) % parts * 16;
  const int col = lane & 15, head = kh * G + g0 + col;
  char* ring = smem + wave * STAGES * TILE_BYTES;
  Wave w{p, sel, topk, kh, lane, uint32_t(reinterpret_cast<uintptr_t>((lds_cptr)ring)), ring};
  w.ops.load_q(static_cast<const T*>(p.q) + i * p.ldq + long(head) * 64, lane >> 4, g0 + col < G);
  w.clear();
  const int nt = uniform(tiles_of<Wave::KEYS>(p, i, topk));
  w.run(i, int(long(nt) * wave / PAGED_WAVES), int(long(nt) * (wave + 1) / PAGED_WAVES), scale);
  w.l = sum_groups(w.l);
  // the join: every wave's m, l and whether it had keys, then the sums moved to the common reference
  float* ml = reinterpret_cast<float*>(smem);
  __syncthreads();
  if (lane < 16) {
    float* at = ml + (wave * 16 + lane) * 4;
    at[0] = w.m;
    at[1] = w.l;
    at[2] = __int_as_float(w.some);
  }
  __syncthreads();
  float mn = -INFINITY;
  for (int k = 0; k < PAGED_WAVES; ++k) mn = fmaxf(mn, ml[(k * 16 + col) * 4]);
  float sum = 0.f;
  int some = 0;
  for (int k = 0; k < PAGED_WAVES; ++k) {
    const float* at = ml + (k * 16 + col) * 4;
    if (!__float_as_int(at[2])) continue;
    some = 1;
    sum += at[1] * (at[0] == -INFINITY ? 0.f : exp2f(at[0] - mn));
  }
  const float keep = !w.some ? 0.f : w.m == -INFINITY ? 0.f : exp2f(w.m - mn);
  float* os = ml + 1024;  // [wave][d][r][lane]
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) os[((wave * 4 + d) * 4 + r) * 64 + lane] = w.some ? w.o[d][r] * keep : 0.f;
  __syncthreads();
  if (g0 + col >= G) return;
  // wave d writes channels 16 d + 4 (lane / 16) + (0..3)
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float a = 0.f;
    for (int k = 0; k < PAGED_WAVES; ++k) a += os[((k * 4 + wave) * 4 + r) * 64 + lane];
    v[r] = some ? a / sum : 0.f;
  }
  T* out = static_cast<T*>(p.out) + i * p.ldo + long(head) * 64 + 16 * wave + 4 * (lane >> 4);
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
  else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
}

// Long or uneven sequences: the tiles of all sequences in a row, cut into one equal part a wave. A sequence that
// lies within one part is written at once; of the others each wave leaves its part's sums, unnormalised, for
// paged_join_kernel: slot 0 for the sequence that the part begins in, slot 1 for one that it ends in.
constexpr int SCAN_MAX = 1024;


// before[i]: tiles of the sequences before i, for i in [0, n]. By one block of NT threads.
template <int KEYS, int NT> __device__ inline void scan_tiles(const PagedArgs& p, int topk, long* before) {
  __shared__ long wsum[NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  long base = 0;
  for (int i0 = 0; i0 <= p.n; i0 += NT) {
    const int i = i0 + tid;
    const long c = i < p.n ? tiles_of<KEYS>(p, i, topk) : 0;
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

// A part: `heads` (up to 16) times 64 sums, then (m, l) of each head; l is -1 where no key was there. PART_HEAD
// floats a head keep the parts 16-byte aligned.
struct Part {
  const int heads;
  __device__ inline explicit Part(int G) : heads(min(G, 16)) {}
  __device__ inline long size() const { return heads * long(PART_HEAD); }
  __device__ inline int ml(int g) const { return heads * 64 + g * 2; }
};

template <typename T, bool SCAN>
__global__ void __launch_bounds__(PAGED_WAVES * 64, 2) paged_parts_kernel(const PagedArgs p, const int* sel, int topk, float scale,
                                                                          int workers, long* before, float* parts) {
  using Wave = PagedWave<T>;
  __shared__ __attribute__((aligned(1024))) char smem[PAGED_WAVES * STAGES * TILE_BYTES];
  __shared__ long own[SCAN ? SCAN_MAX + 1 : 1];
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
  if (worker >= W) return;
  long t = total * worker / W;
  const long end = total * (worker + 1) / W;
  const Part part(G);
  char* ring = smem + wave * STAGES * TILE_BYTES;
  Wave w{p, sel, topk, kh, lane, uint32_t(reinterpret_cast<uintptr_t>((lds_cptr)ring)), ring};
  int lo = 0, hi = p.n;  // the sequence that tile t belongs to
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= t) lo = mid;
    else hi = mid;
  }
  const long first = t;
  for (int i = uniform(lo); t < end; i = uniform(i + 1)) {
    const long b0 = pre[i], b1 = pre[i + 1];
    const long stop = min(end, b1);
    if (stop <= t) continue;
    w.ops.load_q(static_cast<const T*>(p.q) + i * p.ldq + long(head) * 64, lane >> 4, g0 + col < G);
    w.clear();
    w.run(i, uniform(int(t - b0)), uniform(int(stop - b0)), scale);
    w.l = sum_groups(w.l);
    if (g0 + col < G) {
      if (t == b0 && stop == b1) {
        w.store(i, head, w.l);
      } else {
        float* at = parts + ((worker * cols + blockIdx.y) * 2 + (t == first ? 0 : 1)) * part.size();
#pragma unroll
        for (int d = 0; d < 4; ++d)
          *reinterpret_cast<float4*>(at + col * 64 + 16 * d + 4 * (lane >> 4)) = make_float4(w.o[d][0], w.o[d][1], w.o[d][2], w.o[d][3]);
        if (lane < 16) *reinterpret_cast<float2*>(at + part.ml(col)) = make_float2(w.m, w.some ? w.l : -1.f);
      }
    }
    t = stop;
  }
}

// One block a (sequence, head): the parts of a sequence that several waves had. Every wave finds the common
// reference from all parts' (m, l), then sums every JOIN_WAVES-th part, a channel a lane.
constexpr int JOIN_WAVES = 8;
template <typename T>
__global__ void __launch_bounds__(JOIN_WAVES * 64) paged_join_kernel(const PagedArgs p, int workers, const long* before, const float* parts) {
  const int i = blockIdx.x, head = blockIdx.y, G = p.heads / p.cache.kv_heads, groups = (G + 15) / 16, cols = p.cache.kv_heads * groups;
  const int col = head / G * groups + head % G / 16, g = head % G % 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long b0 = before[i], b1 = before[i + 1], total = before[p.n];
  T* out = static_cast<T*>(p.out) + i * p.ldo + long(head) * 64;
  if (b0 == b1) {
    if (threadIdx.x < 64) out[threadIdx.x] = from_f<T>(0.f);
    return;
  }
  // the last worker that begins at or before tile b: begin(w) = floor(total w / W)
  const long W = min(long(workers), total);
  auto holder = [&](long b) { return ((b + 1) * W - 1) / total; };
  const long w0 = holder(b0), w1 = holder(b1 - 1);
  if (w0 == w1) return;  // written whole
  const long count = w1 - w0 + 1;
  const Part layout(G);
  auto part = [&](long k) {
    const long w = w0 + k;
    return parts + ((w * cols + col) * 2 + (total * w / W >= b0 ? 0 : 1)) * layout.size();
  };
  float mx = -INFINITY;
  int some = 0;
  for (long k = lane; k < count; k += 64) {
    const float2 ml = *reinterpret_cast<const float2*>(part(k) + layout.ml(g));
    if (ml.y < 0.f) continue;  // NaN stays
    mx = fmaxf(mx, ml.x);
    some = 1;
  }
  for (int d = 1; d < 64; d <<= 1) {
    mx = fmaxf(mx, __shfl_xor(mx, d));
    some |= __shfl_xor(some, d);
  }
  float acc = 0.f, sum = 0.f;
#pragma unroll 8
  for (long k = wave; k < count; k += JOIN_WAVES) {
    const float* at = part(k);
    const float2 ml = *reinterpret_cast<const float2*>(at + layout.ml(g));
    const float o = at[g * 64 + lane];
    const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
    if (ml.y < 0.f) continue;
    acc += o * f;
    sum += ml.y * f;
  }
  __shared__ float accs[JOIN_WAVES][64], sums[JOIN_WAVES];
  accs[wave][lane] = acc;
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (wave) return;
  acc = sum = 0.f;
  for (int k = 0; k < JOIN_WAVES; ++k) {
    acc += accs[k][lane];
    sum += sums[k];
  }
  out[lane] = from_f<T>(some ? acc / sum : 0.f);
}

// --- selection of pages -------------------------------------------------------------------------

// Scores as whole numbers in the order of the scores, NaN above all; 0: no page there.
__device__ inline uint64_t order_of(double s) {
  if (s != s) return ~0ull;
  const uint64_t b = __double_as_longlong(s);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

// The most that q k can be for a key between the page's bounds, summed over the group's heads, is
// sum_c hi_c A_c + lo_c B_c, with A and B the sums of the positive and the negative parts of the heads' queries:
// 128 products a page, however many heads share it. In 64 bits: which of two pages next to the border is
// taken can hang on less than 32 bits hold. 16 lanes a page, 8 products each, 16 pages a wave whose loads fly
// together; bound by its two dependent loads (the table's entry, the bounds).
constexpr int SCORE_PAGES = 64;  // a block
template <typename T>
__global__ void __launch_bounds__(256) page_score_kernel(const PagedArgs p, const T* bounds, int maxp, uint64_t* keys) {
  const KvCache& c = p.cache;
  const int chunks = (maxp + SCORE_PAGES - 1) / SCORE_PAGES, chunk = blockIdx.x % chunks, pair = blockIdx.x / chunks;
  const int i = pair / c.kv_heads, kh = pair % c.kv_heads, G = p.heads / c.kv_heads;
  const int lane = threadIdx.x & 63, sub = lane & 15, hi = sub >> 3, j = sub & 7;
  const int held = int((long(length_of(p.lens[i], p.width, c.shift, p.max_len)) + c.page_size - 1) >> c.shift);
  const int p0 = chunk * SCORE_PAGES + (threadIdx.x >> 6) * 16 + (lane >> 4);
  if (chunk * SCORE_PAGES >= held) return;
  int page[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) page[k] = p0 + 4 * k < held ? p.table[long(i) * p.width + p0 + 4 * k] : -1;
  double cf[8] = {};
  for (int g = 0; g < G; ++g) {
    float x[8];
    load8(static_cast<const T*>(p.q) + i * p.ldq + (long(kh) * G + g) * 64 + j * 8, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) cf[e] += (x[e] > 0.f) == (hi != 0) ? double(x[e]) : 0.0;
  }
  float v[4][8] = {};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (page_ok(page[k], c.pages)) load8(bounds + (long(page[k]) * c.kv_heads + kh) * 128 + sub * 8, v[k]);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    double s = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) s += double(v[k][e]) * cf[e];
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) s += __shfl_xor(s, m);
    if (sub == 0 && p0 + 4 * k < held)
      keys[long(pair) * maxp + p0 + 4 * k] = page_ok(page[k], c.pages) ? order_of(s) : 0;
  }
}

// Exclusive sum over the block's threads; `total` gets all of it. `room`: one int a wave and one.
constexpr int SELECT_THREADS = 1024, SELECT_BINS = 2048;
__device__ inline int scan_block(int v, int* room, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int inc = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(inc, m);
    if (lane >= m) inc += o;
  }
  __syncthreads();  // the room's last readers
  if (lane == 63) room[wave] = inc;
  __syncthreads();
  int before = inc - v;
  total = 0;
#pragma unroll
  for (int k = 0; k < SELECT_THREADS / 64; ++k) {
    const int r = room[k];
    if (k < wave) before += r;
    total += r;
  }
  return before;
}

// One block a (sequence, key head): the topk largest keys' places, ascending, the lowest place first among equal
// keys, -1 behind them; the newest page is taken first. The keys that are still undecided lie in [lo, hi]; they
// are counted into up to 2048 equal bins of that range, the bins above the border's are taken, and its bin is the
// next range: two rounds for most scores, six at most. Counts do not hang on the order of the atomic adds.
// Thread t holds keys [t K, (t + 1) K) in registers (K > 0), or reads them every round (K = 0, `k` each).
template <int K>
__global__ void __launch_bounds__(SELECT_THREADS) page_select_kernel(const PagedArgs p, const uint64_t* keys, int maxp, int k,
                                                                     int topk, int* sel) {
  __shared__ int bins[SELECT_BINS], room[SELECT_THREADS / 64], found[3];
  __shared__ uint64_t ends[2][SELECT_THREADS / 64];
  const KvCache& c = p.cache;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = blockIdx.x / c.kv_heads;
  const int held = int((long(length_of(p.lens[i], p.width, c.shift, p.max_len)) + c.page_size - 1) >> c.shift);
  const uint64_t* in = keys + long(blockIdx.x) * maxp;
  int* out = sel + long(blockIdx.x) * topk;
  if (K > 0) k = K;
  uint64_t mine[K > 0 ? K : 1];
  if constexpr (K > 0) {
#pragma unroll
    for (int e = 0; e < K; ++e) mine[e] = tid * K + e < held ? in[tid * K + e] : 0;
  }
  auto each = [&](auto&& fn) {
    if constexpr (K > 0) {
#pragma unroll
      for (int e = 0; e < K; ++e) fn(tid * K + e, mine[e]);
    } else {
      for (int e = 0; e < k; ++e) {
        const long at = long(tid) * k + e;
        if (at < held) fn(int(at), in[at]);
      }
    }
  };
  // the newest page aside: how many there are, and their range
  const int newest = held - 1;
  uint64_t lo = ~0ull, hi = 0;
  int mycount = 0, there, first = 0;
  each([&](int at, uint64_t key) {
    if (key == 0) return;
    if (at == newest) {
      first = 1;
      return;
    }
    ++mycount;
    lo = min(lo, key);
    hi = max(hi, key);
  });
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    lo = min(lo, uint64_t(__shfl_xor((unsigned long long)lo, m)));
    hi = max(hi, uint64_t(__shfl_xor((unsigned long long)hi, m)));
  }
  if (lane == 0) {
    ends[0][wave] = lo;
    ends[1][wave] = hi;
  }
  scan_block(mycount, room, there);
#pragma unroll
  for (int w = 0; w < SELECT_THREADS / 64; ++w) {
    lo = min(lo, ends[0][w]);
    hi = max(hi, ends[1][w]);
  }
  const bool newest_there = __syncthreads_or(first);
  int need = min(topk - int(newest_there), there), inside = there;  // to take from [lo, hi], and how many lie in it
  while (need < inside && need > 0 && lo < hi) {
    const int shift = max(0, 53 - __clzll(hi - lo));  // (hi - lo) >> shift < 2048
    for (int b = tid; b < SELECT_BINS; b += SELECT_THREADS) bins[b] = 0;
    __syncthreads();
    each([&](int at, uint64_t key) {
      if (key >= lo && key <= hi && at != newest) atomicAdd(&bins[int((key - lo) >> shift)], 1);
    });
    __syncthreads();
    // thread t has the t-th pair of bins from above
    const int b1 = bins[SELECT_BINS - 1 - 2 * tid], b0 = bins[SELECT_BINS - 2 - 2 * tid];
    int all;
    const int above = scan_block(b1 + b0, room, all);
    if (above < need && need <= above + b1 + b0) {
      const bool up = need <= above + b1;
      found[0] = SELECT_BINS - 1 - 2 * tid - (up ? 0 : 1);
      found[1] = up ? above : above + b1;
      found[2] = up ? b1 : b0;
    }
    __syncthreads();
    need -= found[1];
    inside = found[2];
    const uint64_t at = lo + (uint64_t(found[0]) << shift);
    const uint64_t last = (1ull << shift) - 1;
    if (hi - at > last) hi = at + last;
    lo = at;
    __syncthreads();  // found and bins are written again
  }
  // taken: the newest, what lies above the range, and of the range all or (equal keys) the first `need`
  const bool all = need == inside;
  int equal = 0, eq_total;
  if (!all && need > 0) each([&](int at, uint64_t key) { equal += key >= lo && key <= hi && at != newest; });
  int eq_before = scan_block(equal, room, eq_total);
  auto takes = [&](int at, uint64_t key, int& eq) {
    if (key == 0) return false;
    if (at == newest || key > hi) return true;
    if (key < lo || need == 0) return false;
    return all || eq++ < need;
  };
  int count = 0, total, eq = eq_before;
  each([&](int at, uint64_t key) { count += takes(at, key, eq); });
  int to = scan_block(count, room, total);
  eq = eq_before;
  each([&](int at, uint64_t key) {
    if (takes(at, key, eq)) out[to++] = at;
  });
  for (int e = total + tid; e < topk; e += SELECT_THREADS) out[e] = -1;
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

// The launches of attention over the cache. topk: 0, or the pages that sel lists.
void attend(const Exec& ex, const PagedArgs& a, const int* sel, int topk, char* workspace) {
  const PagedPlan plan = paged_plan(a.cache, a.n, a.heads, a.max_len, topk);
  const float scale = a.scale * 1.44269504088896341f;  // scores as exponents of 2
  long* before = reinterpret_cast<long*>(workspace);
  float* parts = reinterpret_cast<float*>(workspace + plan.before_bytes);
  by_type(a.cache.dt, [&](auto t) {
    using T = decltype(t);
    if (!plan.workers) {
      paged_whole_kernel<T><<<dim3(a.n, plan.cols), PAGED_WAVES * 64, 0, ex.stream>>>(a, sel, topk, scale);
      return;
    }
    const dim3 grid(plan.workers / PAGED_WAVES, plan.cols);
    if (a.n <= SCAN_MAX) {
      paged_parts_kernel<T, true><<<grid, PAGED_WAVES * 64, 0, ex.stream>>>(a, sel, topk, scale, plan.workers, before, parts);
    } else {
      paged_scan_kernel<TileOps<T>::KEYS><<<1, 1024, 0, ex.stream>>>(a, topk, before);
      paged_parts_kernel<T, false><<<grid, PAGED_WAVES * 64, 0, ex.stream>>>(a, sel, topk, scale, plan.workers, before, parts);
    }
    paged_join_kernel<T><<<dim3(a.n, a.heads), JOIN_WAVES * 64, 0, ex.stream>>>(a, plan.workers, before, parts);
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
    if (maxp > 0)
      page_score_kernel<T><<<pairs * cdiv(maxp, SCORE_PAGES), 256, 0, ex.stream>>>(a, static_cast<const T*>(s.bounds), maxp, keys);
  });
  const int each = cdiv(maxp, SELECT_THREADS);
  auto select = [&](auto kernel) { kernel<<<pairs, SELECT_THREADS, 0, ex.stream>>>(a, keys, maxp, each, s.topk, s.selected); };
  if (each <= 1) select(page_select_kernel<1>);
  else if (each <= 4) select(page_select_kernel<4>);
  else if (each <= 16) select(page_select_kernel<16>);
  else select(page_select_kernel<0>);
  attend(ex, a, s.selected, s.topk, ws);
  SPLAT_HIP(hipGetLastError());
}

}  // namespace splat
