// What the paged cache's kernels share on the device: lanes of a wave, loads into LDS, and the two products of attention on a
// tile of a page. Each file of kernels has its own copy.
#pragma once

#include "kernels.h"

#include <algorithm>
#include <type_traits>

namespace splat {

namespace {

// The value of the lane that CTRL names (a DPP control), `old` in the rows that ROWS leaves out and for lanes without one.
template <int CTRL, int ROWS> __device__ inline int from_lane(int old, int v) {
  return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> __device__ inline uint64_t from_lane(uint64_t old, uint64_t v) {
  const uint32_t l = from_lane<CTRL, ROWS>(int(uint32_t(old)), int(uint32_t(v))), h = from_lane<CTRL, ROWS>(int(old >> 32), int(v >> 32));
  return uint64_t(h) << 32 | l;
}
template <int CTRL, int ROWS> __device__ inline float from_lane(float old, float v) {
  return __int_as_float(from_lane<CTRL, ROWS>(__float_as_int(old), __float_as_int(v)));
}
template <int CTRL, int ROWS> __device__ inline double from_lane(double old, double v) {
  return __longlong_as_double(from_lane<CTRL, ROWS>(uint64_t(__double_as_longlong(old)), uint64_t(__double_as_longlong(v))));
}
// Combines every lane with those before it: 1, 2, 4 and 8 to the left in its row of 16, then the rows'
// last lanes (0x142 and 0x143 hand lane 15 of a row and lane 31 on). Lane 63 ends with all 64.
template <typename V, typename F> __device__ inline V scan_wave(V v, V none, F&& fn) {
  v = fn(v, from_lane<0x111, 0xf>(none, v));
  v = fn(v, from_lane<0x112, 0xf>(none, v));
  v = fn(v, from_lane<0x114, 0xf>(none, v));
  v = fn(v, from_lane<0x118, 0xf>(none, v));
  v = fn(v, from_lane<0x142, 0xa>(none, v));
  return fn(v, from_lane<0x143, 0xc>(none, v));
}
__device__ inline int sum_wave(int v) {
  return scan_wave(v, 0, [](int a, int b) { return a + b; });
}

// Sum over the 8 lanes of a head row; every lane gets it (lanes l ^ 1, l ^ 2, then the other quad's mirror).
template <typename V> __device__ inline V sum8(V v) {
  v += from_lane<0xB1, 0xf>(v, v);
  v += from_lane<0x4E, 0xf>(v, v);
  return v + from_lane<0x141, 0xf>(v, v);
}

// A wave-uniform load of memory that the launch only reads.
__device__ inline int uload(const int* p) { return *(const __attribute__((address_space(4))) int*)p; }
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// floor(a / b) for 0 <= a < 2^52 and 0 < b < 2^52: a quotient below a whole number is so by more than the
// rounding of the 64-bit float division. The integer division is a hundred instructions.
__device__ inline long quotient(long a, long b) { return long(floor(double(a) / double(b))); }

// fn over lanes l, l ^ 16, l ^ 32, l ^ 48 (over_rows) and l, l ^ 8, ... (over_halves, then over_rows).
template <typename F> __device__ inline float over_rows(float v, F&& fn) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fn(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fn(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
template <typename F> __device__ inline float over_halves(float v, F&& fn) {
  return over_rows(fn(v, from_lane<0x128, 0xf>(v, v)), fn);
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

// --- tiles of keys and values -------------------------------------------------------------------

typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int int32x4_v __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(3))) char* lds_cptr;

// N loads of 16 bytes a lane, 1 KB each, from base + off[k] + 1024 k into LDS at lds + 1024 k + 16 * lane; offsets
// from `bytes` on read as zeros. The instruction's offset goes into both addresses.
// A load wants one wait state after the write of m0, and five after a vector instruction wrote its descriptor, which the compiler
// does not insert before inline assembly: the write and s_nop 3 are five.
template <int N> __device__ inline void load_lds(const void* base, uint32_t bytes, const uint32_t (&off)[4], int p, uint32_t lds) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const int32x4_v r = {uniform(int(uint32_t(a))), uniform(int(uint32_t(a >> 32))), uniform(int(bytes)), 0x00020000};
  const int m0 = uniform(int(lds));
  if constexpr (N == 4)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\t"
        "buffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
        "buffer_load_dwordx4 %2, %5, 0 offen offset:%6 lds\n\t"
        "buffer_load_dwordx4 %3, %5, 0 offen offset:%7 lds\n\t"
        "buffer_load_dwordx4 %4, %5, 0 offen offset:%8 lds" ::"s"(m0),
        "v"(off[p]), "v"(off[p + 1]), "v"(off[p + 2]), "v"(off[p + 3]), "s"(r), "n"(1024), "n"(2 * 1024), "n"(3 * 1024)
        : "memory");
  else if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\t"
        "buffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
        "buffer_load_dwordx4 %2, %3, 0 offen offset:1024 lds" ::"s"(m0),
        "v"(off[p]), "v"(off[p + 1]), "s"(r)
        : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(m0), "v"(off[p]), "s"(r) : "memory");
}
template <int N> __device__ inline void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// 2^TOP e^d. Scores are subtracted from the largest one before the turn to powers of two: log2(e) times a large score would round
// off what the difference holds.
template <int TOP = 0> __device__ inline float exp_of(float d) { return __builtin_amdgcn_exp2f(fmaf(d, 1.44269504088896341f, float(TOP))); }

__device__ inline float max_groups(float v) { return over_rows(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ inline float sum_groups(float v) { return over_rows(v, [](float a, float b) { return a + b; }); }
// The two products on a tile in LDS. KEYS keys in T16 groups of 16; PIECE rows to a load.
template <typename T> struct TileOps {  // bf16, f16: rows of 128 bytes
  static constexpr int KEYS = 32, T16 = 2, PIECE = 8;
  // f16 weights below 2^-14 lose bits: the largest one is 2^12, so that they do so from 2^-26 of it on.
  static constexpr int TOP = std::is_same<T, f16>::value ? 12 : 0;
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
  // V^T of the tile as the second product's operand: 16 channels each, keys 4 g + (0..3) and 16 + 4 g + (0..3).
  struct Values { uint4 f[4]; };
  __device__ static inline Values values(const char* vt, int lane) {
    const int g = lane >> 4, j = (lane >> 2) & 3, cc = lane & 3, row = 4 * g + j;  // and 16 + row, whose chunks lie alike
    Values v;
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
      v.f[d] = make_uint4(f[0], f[1], f[2], f[3]);
    }
    return v;
  }
  // A weight is two terms of the type, itself rounded and (rest) what that left: the sums keep 16 bits of it in bf16, 22 in f16,
  // for four more matrix instructions a tile (one scene of 24889 positions 16.6 -> 17.1 us, 48 sequences 58 -> 59). The weight
  // rounded alone was most of the result's error before its own rounding.
  __device__ static inline void weigh(const Values& v, const f32x4 (&w)[T16], f32x4 (&o)[4], bool rest) {
    uint32_t p[4], r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = pack2<T>(w[k >> 1][2 * (k & 1)], w[k >> 1][2 * (k & 1) + 1]);
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = mma(v.f[d], make_uint4(p[0], p[1], p[2], p[3]), o[d]);
    if (!rest) return;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      r[k] = pack2<T>(w[k >> 1][2 * (k & 1)] - u16f<T>(p[k]), w[k >> 1][2 * (k & 1) + 1] - u16f<T>(p[k] >> 16));
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = mma(v.f[d], make_uint4(r[0], r[1], r[2], r[3]), o[d]);
  }
};
template <> struct TileOps<float> {  // rows of 256 bytes
  static constexpr int KEYS = 16, T16 = 1, PIECE = 4;
  static constexpr int TOP = 0;
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
    // Four chains of 4 and not one of 16, whose every step rounds the whole sum: results off by 7e-8 instead of 1.1e-7, in the same time.
    f32x4 a[4] = {};
    float4 ks[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) ks[b] = *reinterpret_cast<const float4*>(kt + row * 256 + (((4 * b + g) ^ row) * 16));
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float4& k = ks[b];
      a[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.x, q[b].x, a[b], 0, 0, 0);
      a[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.y, q[b].y, a[b], 0, 0, 0);
      a[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.z, q[b].z, a[b], 0, 0, 0);
      a[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.w, q[b].w, a[b], 0, 0, 0);
    }
    x[0] = (a[0] + a[1]) + (a[2] + a[3]);
  }
  struct Values { float f[4][4]; };  // [key 4 g + r][channel 16 d + lane % 16]
  __device__ static inline Values values(const char* vt, int lane) {
    const int g = lane >> 4, c = lane & 15;
    Values v;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int d = 0; d < 4; ++d)
        v.f[r][d] = *reinterpret_cast<const float*>(vt + (4 * g + r) * 256 + (((4 * d + (c >> 2)) ^ (4 * g)) * 16) + (c & 3) * 4);
    return v;
  }
  __device__ static inline void weigh(const Values& v, const f32x4 (&w)[T16], f32x4 (&o)[4], bool) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v.f[r][d], w[0][r], o[d], 0, 0, 0);
  }
};

constexpr int TILE_BYTES = 8192;  // K, then V

// Runs fn with the storage type dt as a value.
template <typename F> void by_type(int dt, F&& fn) {
  if (dt == F32) fn(float());
  else if (dt == BF16) fn(bf16());
  else fn(f16());
}

}  // namespace

}  // namespace splat
