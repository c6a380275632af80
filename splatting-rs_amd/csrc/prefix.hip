// Attention of many tokens over a prefix that they share, read once for all of them, joined with each token's own positions.
//
// The tokens of a group times the query heads of a key head are the columns of S^T = K Q^T and O^T = V^T P^T (paged.h has
// the products). An item is up to R columns of one group and key head. With the running maximum m and the sum l of a
// softmax, parts over any sets of positions join: O = sum e^(m_i - m) O_i, l = sum e^(m_i - m) l_i.
//
// The first blocks of a launch take the prefixes' items. All items' tiles are cut into about equal parts, so that few items
// fill the chip too: every block sums the groups up and finds its own part, without a launch before. The other blocks take
// the tokens' own positions. Parts are left in the workspace for a joining launch where there are several of a column.
#include "paged.h"

namespace splat {

namespace {

constexpr int WAVES = 4;
constexpr int RING = 2;  // tiles of a wave's ring: run() takes two

// What block 0 leaves for the join: of each group the first block of its items, and the parts that its tiles are cut into.
struct GroupPlan { int block0, parts, items, row0; };  // items: of one key head
struct PlanHead { int valid, pad[3]; };

__device__ inline int shared_of(const PrefixArgs& a, int g) { return length_of(a.shared[g], a.prefix_width, a.cache.shift, a.max_shared); }
// The first token of group g and of the next one, within [0, n].
__device__ inline int start_of(const PrefixArgs& a, int g) { return min(max(a.starts[g], 0), a.n); }

// The group of token i, by a wave, -1: none. The group is the last one that begins at or before i.
__device__ inline int group_of(const PrefixArgs& a, int i) {
  const int lane = threadIdx.x & 63;
  int lo = 0, count = a.groups;  // among groups lo .. lo + count - 1
  while (count > 1) {
    const int step = (count + 63) / 64, g = lo + lane * step;
    const uint64_t begun = __ballot(lane * step < count && start_of(a, g) <= i);
    const int at = begun ? 63 - __builtin_clzll(begun) : 0;
    lo += at * step;
    count = min(step, count - at * step);
  }
  return uniform(start_of(a, lo) <= i && i < start_of(a, lo + 1) ? lo : -1);
}

// --- one wave -----------------------------------------------------------------------------------

// The values as floats, element by element.
template <typename T, typename F> __device__ inline typename TileOps<T>::Values map_values(const typename TileOps<T>::Values& v, F&& fn) {
  typename TileOps<T>::Values out;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int d = 0; d < 4; ++d) out.f[r][d] = fn(v.f[r][d], r);
  } else {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const uint32_t u[4] = {v.f[d].x, v.f[d].y, v.f[d].z, v.f[d].w};
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = pack2<T>(fn(u16f<T>(u[k]), 2 * k), fn(u16f<T>(u[k] >> 16), 2 * k + 1));
      out.f[d] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  return out;
}

// The running softmax of NT times 16 columns over tiles of one row of pages. Column t, lane % 16 sees positions [lo, hi[t]).
template <typename T, int NT> struct PrefixWave {
  using Ops = TileOps<T>;
  static constexpr int KEYS = Ops::KEYS, PIECE = Ops::PIECE;
  const KvCache& c;
  const int kh, lane;
  const uint32_t lds;  // of the wave's ring
  const char* ring;
  const int* row;      // of pages, `width` entries
  int width;
  int lo, end, least;  // positions at or past `end` are seen by no column, those in [lo, least) by all
  int hi[NT];
  Ops ops[NT];
  f32x4 o[NT][4];
  float m[NT], l[NT];
  int some[NT];        // keys were there

  // Loads tile t, which lies in E pages, into slot b of the ring; the rows of each piece that are there, 8 bits a piece.
  template <int E> __device__ inline uint32_t load_tile(int t, int b) {
    constexpr int PIECES = 4 / E, ROWS = PIECES * PIECE;  // of one page
    uint32_t k_off[4], v_off[4], there = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      k_off[k] = Ops::k_off(lane, k);
      v_off[k] = Ops::v_off(lane, k);
    }
    int entry[E];
#pragma unroll
    for (int e = 0; e < E; ++e) entry[e] = uload(row + min((t * KEYS + e * ROWS) >> c.shift, width - 1));
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int first = t * KEYS + e * ROWS, in_page = E > 1 ? 0 : first & (c.page_size - 1);
      const int rows = page_ok(entry[e], c.pages) ? max(0, min(ROWS, end - first)) : 0;
#pragma unroll
      for (int k = 0; k < PIECES; ++k) there |= uint32_t(max(0, min(PIECE, rows - k * PIECE))) << (8 * (e * PIECES + k));
      const long at = (rows ? page_at(c, entry[e], kh) : 0) + in_page * 64;
      const uint32_t bytes = uint32_t(rows) * 64 * sizeof(T), to = lds + b * TILE_BYTES + e * PIECES * 1024;
      load_lds<PIECES>(static_cast<const T*>(c.k) + at, bytes, k_off, e * PIECES, to);
      load_lds<PIECES>(static_cast<const T*>(c.v) + at, bytes, v_off, e * PIECES, to + TILE_BYTES / 2);
    }
    return uniform(int(there));
  }
  __device__ inline uint32_t issue(int t, int b) {
    if (c.page_size >= KEYS) return load_tile<1>(t, b);
    if (KEYS == 16 || c.page_size == 16) return load_tile<2>(t, b);
    return load_tile<4>(t, b);
  }

  // CAREFUL: infinities and NaN among the values count where they are seen and nowhere else.
  template <bool CAREFUL> __device__ inline void tile(int b, int t, uint32_t there, float scale) {
    constexpr uint32_t ALL = PIECE * 0x01010101u;
    const char* kt = ring + b * TILE_BYTES;
    const int g = lane >> 4, first = t * KEYS;
    typename Ops::Values v = Ops::values(kt + TILE_BYTES / 2, lane);
    const bool edge = there != ALL || first < lo || first + KEYS > least;
    if (edge && first < lo) {  // positions that belong to another part may hold anything
      v = map_values<T>(v, [&](float x, int e) {
        const int key = sizeof(T) == 4 ? 4 * g + e : 16 * (e >> 2) + 4 * g + (e & 3);
        return first + key < lo ? 0.f : x;
      });
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 x[Ops::T16], seen[Ops::T16];
      ops[n].scores(kt, lane, x);
#pragma unroll
      for (int s = 0; s < Ops::T16; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[s][r] *= scale;
          if (CAREFUL) seen[s][r] = 1.f;
        }
      int any = 1;
      if (edge) {
        any = 0;
#pragma unroll
        for (int s = 0; s < Ops::T16; ++s) {
          const int key = 16 * s + 4 * g, rows = int((there >> (8 * (key / PIECE))) & 255u) - key % PIECE;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int p = first + key + r;
            if (r < rows && p >= lo && p < hi[n]) any = 1;
            else {
              x[s][r] = -INFINITY;
              if (CAREFUL) seen[s][r] = 0.f;
            }
          }
        }
      }
      some[n] |= any;
      float mx = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
      if constexpr (Ops::T16 == 2) mx = fmaxf(mx, fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
      const float mn = fmaxf(m[n], max_groups(mx));
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float keep = m[n] == -INFINITY ? 0.f : exp_of(m[n] - mn);
      m[n] = mn;
      l[n] *= keep;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[n][d][r] *= keep;
#pragma unroll
      for (int s = 0; s < Ops::T16; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[s][r] = exp_of<Ops::TOP>(x[s][r] - ref);
          l[n] += x[s][r];
        }
      if constexpr (!CAREFUL) {
        Ops::weigh(v, x, o[n], sizeof(T) == 2);
      } else {
        // the finite ones as always, then how many of each other kind the column sees
        auto kind = [&](auto&& is) { return map_values<T>(v, [&](float y, int) { return is(y) ? 1.f : 0.f; }); };
        Ops::weigh(map_values<T>(v, [](float y, int) { return fabsf(y) < INFINITY ? y : 0.f; }), x, o[n], sizeof(T) == 2);
        auto add = [&](const typename Ops::Values& w, float what) {
          f32x4 count[4] = {};
          Ops::weigh(w, seen, count, false);
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[n][d][r] += count[d][r] > 0.f ? what : 0.f;
        };
        add(kind([](float y) { return y != y; }), NAN);
        add(kind([](float y) { return y == INFINITY; }), INFINITY);
        add(kind([](float y) { return y == -INFINITY; }), -INFINITY);
      }
    }
  }

  // Tiles t, t + step, ...: tile k is asked for while tile k - 2 is used. Where a sum is NaN they are to be taken again with care: a
  // weight of 0 times an infinity, or an infinity beside the second term of a weight, is no answer.
  template <bool CAREFUL> __device__ inline bool pass(int t, int step, int count, float scale) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int d = 0; d < 4; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[n] = -INFINITY;
      l[n] = 0.f;
      some[n] = 0;
    }
    uint32_t there = 0, next = 0;  // of tiles k - 2 and k - 1
#pragma unroll 1
    for (int k = 0; k < count + 2; ++k) {
      if (k >= 2) {
        if (k - 1 < count) wait_loads<8>();
        else wait_loads<0>();
        tile<CAREFUL>(k & 1, t + (k - 2) * step, there, scale);
      }
      there = next;
      if (k < count) next = issue(t + k * step, k & 1);
    }
    bool nan = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) nan |= o[n][d][r] != o[n][d][r];
    return __any(nan);
  }
  // True where a sum is NaN: then again, with care.
  template <bool CAREFUL> __device__ inline bool run(int t, int step, int stop, float scale) {
#pragma unroll
    for (int n = 0; n < NT; ++n) ops[n].pin_q();
    const bool nan = pass<CAREFUL>(t, step, t < stop ? (stop - t + step - 1) / step : 0, scale);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      l[n] = sum_groups(l[n]);
      some[n] = over_rows(float(some[n]), [](float a, float b) { return fmaxf(a, b); }) > 0.f;
    }
    return nan;
  }
};

// --- a block ------------------------------------------------------------------------------------

// A part: `columns` times 64 sums, then (m, l) of each, the sums being of weights e^(x - m), m the largest score as it is: a logarithm of the
// forms' factors 2^TOP taken off it would round it, at scores of 8192 by up to 2^-11. l is -1 where no key was there.
__device__ inline float* part_at(char* workspace, size_t offset, long index, int columns) {
  return reinterpret_cast<float*>(workspace + offset) + index * columns * long(PART_HEAD);
}

// The waves' sums join in LDS: wave d adds up channels 16 d + (0..15) of columns first, first + 1, ... place(n) gives the output's row
// for the lane's column of NT (normalised, where `whole`) or nullptr if there is none; else they go to `part`.
template <typename T, int NT, typename Place>
__device__ inline void join_waves(const PrefixWave<T, NT>& w, char* smem, float (*stats)[4], int wave, bool whole, float* part, int first, int columns, Place&& place) {
  const int lane = w.lane, col = lane & 15, g = lane >> 4;
  float* mine = reinterpret_cast<float*>(smem + wave * RING * TILE_BYTES);  // its tiles are used up
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) mine[((n * 4 + d) * 4 + r) * 64 + lane] = w.o[n][d][r];
    if (g == 0) {
      float* s = stats[(wave * NT + n) * 16 + col];
      s[0] = w.m[n];
      s[1] = w.l[n];
      s[2] = float(w.some[n]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int column = first + n * 16 + col;
    float mn = -INFINITY, sum = 0.f, v[4] = {};
    bool some = false;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) mn = fmaxf(mn, stats[(k * NT + n) * 16 + col][0]);
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const float* s = stats[(k * NT + n) * 16 + col];
      if (s[2] == 0.f) continue;  // no key: its sums are zeros, whatever the others hold
      some = true;
      const float f = s[0] == -INFINITY ? 0.f : exp_of(s[0] - mn);
      sum += s[1] * f;
      const float* theirs = reinterpret_cast<const float*>(smem + k * RING * TILE_BYTES);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += theirs[((n * 4 + wave) * 4 + r) * 64 + lane] * f;
    }
    if (column >= columns) continue;
    if (whole) {
      T* out = place(n);
      if (!out) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = some ? v[r] / sum : 0.f;
      out += 16 * wave + 4 * g;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
      else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
      constexpr float f = 1.f / (1 << TileOps<T>::TOP);
      *reinterpret_cast<float4*>(part + column * 64 + 16 * wave + 4 * g) = make_float4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
      if (wave == 0 && g == 0) *reinterpret_cast<float2*>(part + columns * 64 + column * 2) = make_float2(mn, some ? sum * f : -1.f);
    }
  }
}

// A block's part of the groups' items.
struct Mine {
  int id;  // of the block among those with work, -1: nothing to do
  int group, item, kh, part, parts;
  int start, tokens, shared;
};

// Every wave for itself, 64 groups at a time, a group a lane: two loads one after the other and no barrier where there are no more of
// them. Block 0 leaves the plan for the join. The tiles of a part: as few as leave no more parts than blocks. All tiles / blocks is
// tried first, which fits where the groups are alike; an item of T tiles has at most T / each + 1 parts, so that all tiles /
// (blocks - items) always fits.
template <int KEYS, int R> __device__ inline Mine find_item(const PrefixArgs& a, int blocks, char* workspace, bool join) {
  const int lane = threadIdx.x & 63, G = a.heads / a.cache.kv_heads, kv = a.cache.kv_heads, rounds = (a.groups + 63) / 64;
  struct Group { int start, tokens, shared, items, tiles; bool descends; };  // items of a key head
  auto group_at = [&](int k) {
    const int g = 64 * k + lane, at = min(g, a.groups - 1);
    Group x;
    x.start = start_of(a, at);
    const int count = g < a.groups ? start_of(a, at + 1) - x.start : 0;
    x.tokens = max(0, count);
    x.descends = count < 0;
    x.shared = shared_of(a, at);
    x.items = (x.tokens * G + R - 1) / R;  // tokens times G are below 2^21
    x.tiles = (x.shared + KEYS - 1) / KEYS;
    return x;
  };
  const Group first = group_at(0);
  auto group_of_round = [&](int k) { return k == 0 ? first : group_at(k); };
  const auto plus = [](uint64_t x, uint64_t y) { return x + y; };
  auto last = [&](uint64_t v) { return long(uint64_t(uint32_t(__builtin_amdgcn_readlane(int(v >> 32), 63))) << 32 | uint32_t(__builtin_amdgcn_readlane(int(v), 63))); };
  long items = 0, tiles = 0, total = 0, each = 1L << 40;
  bool valid = true;  // starts ascend: no token is in two groups
  for (int k = 0; k < rounds; ++k) {
    const Group x = group_of_round(k);
    valid &= !__ballot(x.descends);
    items += last(scan_wave(uint64_t(x.items) * kv, uint64_t(0), plus));
    tiles += last(scan_wave(uint64_t(x.items) * kv * x.tiles, uint64_t(0), plus));
  }
  auto parts_of = [&](const Group& x) { return int(max(1L, quotient(x.tiles + each - 1, each))); };
  for (int attempt = 0; attempt < 2; ++attempt) {
    const long share = attempt == 0 ? blocks : blocks - items;
    each = join && share > 0 ? max(1L, quotient(tiles + share - 1, share)) : 1L << 40;
    total = 0;
    for (int k = 0; k < rounds; ++k) {
      const Group x = group_of_round(k);
      total += last(scan_wave(uint64_t(x.items) * kv * parts_of(x), uint64_t(0), plus));
    }
    if (total <= blocks) break;
  }
  Mine mine;
  mine.id = valid && long(blockIdx.x) < total ? xcd_contiguous(int(blockIdx.x), int(total)) : -1;
  const bool leave = join && blockIdx.x == 0 && threadIdx.x < 64;
  if (leave && lane == 0) reinterpret_cast<PlanHead*>(workspace)->valid = valid;
  if (!valid || (mine.id < 0 && !leave)) return mine;
  // those that read the same keys run at the same time on the same XCD: items fastest, contiguous ids an XCD
  uint64_t before = 0;
  for (int k = 0; k < rounds; ++k) {
    const Group x = group_of_round(k);
    const int parts = parts_of(x), here = x.items * kv * parts;
    const uint64_t sum = scan_wave(uint64_t(here), uint64_t(0), plus);
    const int at = int(before + sum) - here;  // below `blocks`
    if (leave && 64 * k + lane < a.groups)
      reinterpret_cast<GroupPlan*>(workspace + sizeof(PlanHead))[64 * k + lane] = {at, parts, x.items, x.start};
    const uint64_t there = __ballot(mine.id >= at && mine.id < at + here);
    if (there) {
      const int l = __builtin_ctzll(there);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int its = of(x.items), r = mine.id - of(at), rest = r / its;
      mine.group = 64 * k + l;
      mine.item = r % its;
      mine.parts = of(parts);
      mine.kh = rest / mine.parts;
      mine.part = rest % mine.parts;
      mine.start = of(x.start);
      mine.tokens = of(x.tokens);
      mine.shared = of(x.shared);
      if (!leave) break;
    }
    before += last(sum);
  }
  return mine;
}

// A token's own positions: part `part` of `of` of those of token i and up to 16 heads (column group `group` of the key heads'), every
// step-th tile from the first-th on by this wave. Returns the wave, whose sums are there.
template <typename T>
__device__ inline PrefixWave<T, 1> own_tiles(const PrefixArgs& a, int i, int group, int part, int of, int first, int step, char* ring) {
  constexpr int KEYS = TileOps<T>::KEYS;
  const KvCache& c = a.cache;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int G = a.heads / c.kv_heads, groups = (G + 15) / 16, kh = group / groups, h0 = group % groups * 16;
  PrefixWave<T, 1> w{c, kh, lane, uint32_t(reinterpret_cast<uintptr_t>((lds_cptr)ring)), ring, a.table + long(i) * a.width, a.width};
  const bool in = h0 + col < G;
  w.ops[0].load_q(static_cast<const T*>(a.q) + long(i) * a.ldq + long(kh * G + h0 + (in ? col : 0)) * 64, g, in);
  // for up to 64 groups what is asked of them comes in one load, a group a lane
  const int near = min(lane, a.groups - 1), begin = start_of(a, near), end = start_of(a, near + 1);
  int shared = a.shared[near], len = a.lens[i], at = -1;  // whole: where the prefix is cut, own positions begin behind it all the same
  if (a.groups <= 64) {
    const uint64_t of_token = __ballot(lane < a.groups && begin <= i && i < end);
    if (of_token) {
      at = 63 - __builtin_clzll(of_token);
      shared = __builtin_amdgcn_readlane(shared, at);
    }
  } else if ((at = group_of(a, i)) >= 0) {
    shared = a.shared[at];
  }
  w.lo = at < 0 ? 0 : uniform(max(shared, 0));
  w.end = at < 0 ? 0 : uniform(int(min(long(length_of(len, a.width, c.shift, 0x7fffffff)), long(w.lo) + a.max_own)));
  w.least = w.hi[0] = w.end;
  const int from = w.lo / KEYS, tiles = w.end > w.lo ? (w.end + KEYS - 1) / KEYS - from : 0;
  const int t0 = from + int(long(tiles) * part / of) + first, t1 = from + int(long(tiles) * (part + 1) / of);
  if (w.template run<false>(t0, step, t1, a.scale)) w.template run<true>(t0, step, t1, a.scale);
  return w;
}

// Block `u` of those for the tokens' own positions, whose waves share one of `own` parts. (A wave with a token by itself, of which 64 forks
// of 12 heads have enough: 52 -> 62 us, by the longest of them.)
template <typename T>
__device__ inline void own_block(const PrefixArgs& a, int u, int own, size_t own_parts, char* workspace, char* smem, float (*stats)[4]) {
  const int wave = uniform(threadIdx.x >> 6), G = a.heads / a.cache.kv_heads, cols = a.cache.kv_heads * ((G + 15) / 16), columns = min(G, 16);
  const PrefixWave<T, 1> w = own_tiles<T>(a, u / own / cols, u / own % cols, u % own, own, wave, WAVES, smem + wave * RING * TILE_BYTES);
  join_waves<T, 1>(w, smem, stats, wave, false, part_at(workspace, own_parts, u, columns), 0, columns, [](int) { return static_cast<T*>(nullptr); });
}

// The tokens' own positions by themselves, beside the wide form, whose blocks leave no room for these.
template <typename T>
__global__ void __launch_bounds__(WAVES * 64, 2) prefix_own_kernel(const PrefixArgs a, int own, size_t own_parts, char* workspace) {
  __shared__ __attribute__((aligned(1024))) char smem[WAVES * RING * TILE_BYTES];
  __shared__ float stats[WAVES * 16][4];
  own_block<T>(a, int(blockIdx.x), own, own_parts, workspace, smem, stats);
}

// Few rows an item: each wave streams its own tiles through a ring of its own, and the block's waves join in LDS.
template <typename T, int NT>
__global__ void __launch_bounds__(WAVES * 64, 2) prefix_parts_kernel(const PrefixArgs a, int blocks, int own, bool join, size_t parts, size_t own_parts, char* workspace) {
  constexpr int KEYS = TileOps<T>::KEYS, R = NT * 16;
  __shared__ __attribute__((aligned(1024))) char smem[WAVES * RING * TILE_BYTES];
  __shared__ float stats[WAVES * R][4];
  if (int(blockIdx.x) >= blocks) {
    own_block<T>(a, int(blockIdx.x) - blocks, own, own_parts, workspace, smem, stats);
    return;
  }
  const Mine mine = find_item<KEYS, R>(a, blocks, workspace, join);
  if (uniform(mine.id) < 0) return;
  const KvCache& c = a.cache;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, G = a.heads / c.kv_heads;
  const int kh = uniform(mine.kh), shared = uniform(mine.shared), rows = uniform(mine.tokens) * G, item = uniform(mine.item), start = uniform(mine.start);
  char* ring = smem + wave * RING * TILE_BYTES;
  const uint32_t lds = uint32_t(reinterpret_cast<uintptr_t>((lds_cptr)ring));
  const int* row = a.prefix + long(uniform(mine.group)) * a.prefix_width;
  float* part = part_at(workspace, parts, uniform(mine.id), R);
  // The item's columns from `first` on: M times 16. True where a sum is NaN, and nothing is written then.
  auto columns = [&](auto count, auto careful, int first) {
    constexpr int M = decltype(count)::value;
    constexpr bool CAREFUL = decltype(careful)::value;
    PrefixWave<T, M> w{c, kh, lane, lds, ring, row, a.prefix_width};
    int most = 0, least = 0x7fffffff, token[M], head[M];
#pragma unroll
    for (int n = 0; n < M; ++n) {
      const int r = item * R + first + n * 16 + col;  // below 2^21
      const bool in = r < rows;
      token[n] = start + (in ? r / G : 0);
      head[n] = in ? kh * G + r % G : -1;
      w.hi[n] = in ? max(0, min(a.lens ? a.lens[token[n]] : shared, shared)) : 0;
      w.ops[n].load_q(static_cast<const T*>(a.q) + long(token[n]) * a.ldq + long(max(head[n], 0)) * 64, lane >> 4, in);
      most = max(most, w.hi[n]);
      if (in) least = min(least, w.hi[n]);
    }
    // over the lanes: 16 columns (the four groups of lanes hold the same)
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
      most = max(most, __shfl_xor(most, x));
      least = min(least, __shfl_xor(least, x));
    }
    w.lo = 0;
    w.end = uniform(most);
    w.least = uniform(least);
    const int tiles = (shared + KEYS - 1) / KEYS, seen = (w.end + KEYS - 1) / KEYS, k = uniform(mine.part), of = uniform(mine.parts);
    const int t0 = int(long(tiles) * k / of), t1 = min(seen, int(long(tiles) * (k + 1) / of));
    const bool nan = w.template run<CAREFUL>(t0 + wave, WAVES, t1, a.scale);
    if (!CAREFUL && __syncthreads_or(nan)) return true;
    join_waves<T, M>(w, smem, stats, wave, !join, part, first, R, [&](int n) {
      T* out = nullptr;
#pragma unroll
      for (int k = 0; k < M; ++k)
        if (k == n && head[k] >= 0) out = static_cast<T*>(a.out) + long(token[k]) * a.ldo + long(head[k]) * 64;
      return out;
    });
    return false;
  };
  if (!columns(std::integral_constant<int, NT>(), std::false_type(), 0)) return;
#pragma unroll 1
  for (int n = 0; n < NT; ++n) {  // a few columns at a time: what the careful form keeps leaves no registers for more
    __syncthreads();              // the ring and the statistics are read
    columns(std::integral_constant<int, 1>(), std::true_type(), n * 16);
  }
}

// --- many rows an item --------------------------------------------------------------------------
//
// Four waves of 32 columns each share tiles of 64 keys, on the 32x32 matrix instructions: S^T = K Q^T leaves a lane one
// column (lane % 32) and 16 keys of each 32, which is the second operand of O^T = V^T P^T as it stands.
//
// Bound by the matrix instructions and by the vector unit's work on the scores, about as much of either: so half a tile's products
// with K and the half before the last one's with V are under way while the half between becomes weights, all in one wave's stream,
// and three waves share a SIMD. 1037 tokens of 12 heads on 24889 positions (bf16, 79 GFLOP): 158 us, the join's 10 among them (0.50 PFLOP/s,
// and half as many operations again for the weights' second terms: 0.8 PFLOP/s while the parts are formed). Of the 3600 cycles that a tile
// of 64 columns takes a SIMD 1550 go to the matrix instructions and 2000 to the vector unit (by their counters). With weights of one term, when all of
// it took 115 us: two blocks a CU with a tile more under way 130, waves of 64 columns 125, two teams of waves that multiply and exponentiate in
// turn 140, the compiler's own order of the same instructions 6% more.
//
// The weights are 2^(c s + ref), c = |scale| log2(e), in one fused multiply-add: its one rounding is of the difference, and what ref =
// -c r was rounded by is the same for all weights of a column: parts are freed of it. r is the largest product of the first half tile with a key; sums that overflow
// with it (2^64, in f16 weights of 2^16) are taken again with care. A weight is two terms of the values' type, as in TileOps: 16 bits of it in
// bf16, 22 in f16. Rounded to one (115 us for 158) a bf16 view is off by 1.9e-3 where the output's own rounding is 1.65e-3, and the same
// token by as much between a call of few rows and one of many.

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T> __device__ inline f32x16 mma32(const uint4& a, const uint4& b, const f32x16& c) {
  if constexpr (std::is_same<T, bf16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0, 0, 0);
}
// What one value of a packed pair leaves of x, which it is x rounded to: exact, by a product with (-1, 0) or (0, -1). The factors stay in
// registers: a 16-bit constant of an instruction's own is not in the half that it is in here.
typedef __bf16 bf16x2_v __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_v __attribute__((ext_vector_type(2)));
template <typename T, int WHICH> __device__ inline float rest_of(uint32_t pair, float x) {
  uint32_t minus = (std::is_same<T, bf16>::value ? 0xbf80u : 0xbc00u) << (16 * WHICH);
  asm("" : "+s"(minus));
  if constexpr (std::is_same<T, bf16>::value)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_v, pair), __builtin_bit_cast(bf16x2_v, minus), x, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_v, pair), __builtin_bit_cast(f16x2_v, minus), x, false);
}
__device__ inline float most_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // NaN stays
// fn over lanes l and l ^ 32
template <typename F> __device__ inline float over_two(float v, F&& fn) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fn(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

constexpr int WIDE_KEYS = 64, WIDE_BYTES = WIDE_KEYS * 256;  // a tile: K, then V
constexpr int WIDE_RING = 3, WIDE_OCCUPANCY = 3;

template <typename T> struct WideWave {
  // f16 weights below 2^-14 lose bits and 2^16 is beyond them: the first tile's largest weight is 2^4
  static constexpr float TOP = std::is_same<T, f16>::value ? 4.f : 0.f;
  const KvCache& c;
  const int kh, lane, wave;
  char* ring;
  const int* row;  // of pages
  int width, end;  // positions from `end` on are seen by no column of the block
  // 64 entries of the row, one a lane: where the keys of the pages lie that tiles are loaded from now (ok: which are pages), and the
  // next entries
  int chunk, ahead;
  uint32_t at_lo, at_hi;
  uint64_t ok;
  uint32_t full;        // bits of a tile's pages
  int hi, most, least;  // what the lane's column sees; of the wave's columns
  uint4 q[4];
  f32x16 o[2];
  float r, l;
  int key0;  // the first position of the tiles with a page: a column that sees it has met a key

  __device__ inline int load_entries(int k) const { return row[min(long(k) * 64 + lane, long(width) - 1)]; }
  __device__ inline void take_entries(int k, int these) {
    chunk = k;
    asm volatile("" : "+v"(these));  // these are here: the wait for them is not to be one for the next
    const bool page = page_ok(these, c.pages);
    const uint64_t at = reinterpret_cast<uint64_t>(static_cast<const T*>(c.k) + (page ? page_at(c, these, kh) : 0));
    at_lo = uint32_t(at);
    at_hi = uint32_t(at >> 32);
    ok = __ballot(page);
    ahead = load_entries(k + 1);
  }
  // Before tile t is asked for: which of its pages are there, a bit each.
  __device__ inline uint32_t pages_of(int t) {
    const int place0 = (t * WIDE_KEYS) >> c.shift;
    if ((place0 >> 6) != chunk) take_entries(place0 >> 6, (place0 >> 6) == chunk + 1 ? ahead : load_entries(place0 >> 6));
    return uint32_t(ok >> (place0 & 63)) & full;
  }
  // Asks for this wave's 16 rows of tile t (16 w on), which lie in PIECES pages, into slot b of the ring. What is behind `end` reads as zeros.
  // Chunk x of row y lies in slot x ^ (y / 2) of keys and x ^ 2 (y % 4) of values, so that the rows that a read takes lie in different banks.
  template <int PIECES> __device__ inline void ask(int t, int b, uint32_t pages) const {
    const int lrow = lane >> 3;
    const uint32_t k_off[4] = {uint32_t(lrow * 128 + (((lane & 7) ^ (lrow >> 1)) * 16)), uint32_t(lrow * 128 + (((lane & 7) ^ (4 + (lrow >> 1))) * 16))};
    const uint32_t v_off[4] = {uint32_t(lrow * 128 + (((lane & 7) ^ ((lrow & 3) << 1)) * 16)), uint32_t(lrow * 128 + (((lane & 7) ^ ((lrow & 3) << 1)) * 16))};
    const uint32_t lds = uint32_t(reinterpret_cast<uintptr_t>((lds_cptr)ring)) + b * WIDE_BYTES + wave * 2048;
    const uint64_t apart = reinterpret_cast<uint64_t>(c.v) - reinterpret_cast<uint64_t>(c.k);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int first = t * WIDE_KEYS + 16 * wave + 8 * i, from = first >> c.shift;
      int rows = 16 / PIECES;
      if (pages != full || first + rows > end) {
        const int here = c.page_size < WIDE_KEYS ? (16 * wave + 8 * i) >> c.shift : 0;
        rows = pages >> here & 1 ? uniform(max(0, min(rows, end - first))) : 0;
      }
      uint64_t k = uint64_t(uint32_t(__builtin_amdgcn_readlane(int(at_hi), from & 63))) << 32 | uint32_t(__builtin_amdgcn_readlane(int(at_lo), from & 63));
      k += (first & (c.page_size - 1)) * 128;
      load_lds<2 / PIECES>(reinterpret_cast<const void*>(k), rows * 128, k_off, i, lds + i * 1024);
      load_lds<2 / PIECES>(reinterpret_cast<const void*>(k + apart), rows * 128, v_off, i, lds + WIDE_BYTES / 2 + i * 1024);
    }
  }
  __device__ inline uint32_t issue(int t) {
    const uint32_t pages = pages_of(t);
    if (c.page_size >= 16) ask<1>(t, t % WIDE_RING, pages);
    else ask<2>(t, t % WIDE_RING, pages);
    return pages;
  }

  // V^T of 16 keys from 32 half + 16 hh on and channels 32 dt on, in the order of the weights (as in TileOps, for 32 rows of output).
  __device__ inline uint4 values(int b, int half, int hh, int dt) const {
    typedef short v4s __attribute__((ext_vector_type(4)));
    const char* vt = ring + b * WIDE_BYTES + WIDE_BYTES / 2;
    const int G = lane >> 4, j = (lane >> 2) & 3, cc = lane & 3;
    const int at = (4 * (G >> 1) + j) * 128 + (((4 * dt + 2 * (G & 1) + (cc >> 1)) ^ (j << 1)) * 16) + (cc & 1) * 8;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)((lds_cptr)(vt + (half * 32 + 16 * hh + 8 * e) * 128 + at)));
      const uint2 u = __builtin_bit_cast(uint2, x);
      w[2 * e] = u.x;
      w[2 * e + 1] = u.y;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // K of 32 keys from 32 half on and 16 channels from 16 st on.
  __device__ inline uint4 keys(int b, int half, int st) const {
    const int g = lane >> 5, l32 = lane & 31, sw = (l32 >> 1) & 7;
    return *reinterpret_cast<const uint4*>(ring + b * WIDE_BYTES + (half * 32 + l32) * 128 + ((2 * st + g) ^ sw) * 16);
  }
  template <typename F> __device__ static inline uint4 map_pairs(const uint4& v, F&& fn) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = pack2<T>(fn(u16f<T>(u[k])), fn(u16f<T>(u[k] >> 16)));
    return make_uint4(w[0], w[1], w[2], w[3]);
  }

  // Half a tile: its operands, scores, weights, and what those add to the sums.
  struct Weights { uint32_t p[8], rest[8]; };
  __device__ inline void load_keys(uint4 (&kf)[4], int b, int half) const {
#pragma unroll
    for (int st = 0; st < 4; ++st) kf[st] = keys(b, half, st);
  }
  __device__ inline void load_values(uint4 (&vf)[4], int b, int half) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) vf[k] = values(b, half, k >> 1, k & 1);
  }
  __device__ inline void score(f32x16& s, const uint4 (&kf)[4]) const {
    const f32x16 zero = {};
#pragma unroll
    for (int st = 0; st < 4; ++st) s = mma32<T>(kf[st], q[st], st == 0 ? zero : s);
  }
  __device__ inline void weights(Weights& w, const f32x16& s, float scale, float ref) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * e], scale, ref)), y = __builtin_amdgcn_exp2f(fmaf(s[2 * e + 1], scale, ref));
      w.p[e] = pack2<T>(x, y);
      w.rest[e] = pack2<T>(rest_of<T, 0>(w.p[e], x), rest_of<T, 1>(w.p[e], y));
      sum += x + y;
    }
    l += sum;
  }
  __device__ inline void weigh_one(const Weights& w, int k, const uint4& v) {
    const int p = 4 * (k >> 1);
    o[k & 1] = mma32<T>(v, make_uint4(w.p[p], w.p[p + 1], w.p[p + 2], w.p[p + 3]), o[k & 1]);
    o[k & 1] = mma32<T>(v, make_uint4(w.rest[p], w.rest[p + 1], w.rest[p + 2], w.rest[p + 3]), o[k & 1]);
  }
  __device__ inline void weigh(const Weights& w, const uint4 (&vf)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t* p = w.p + 4 * (k >> 1);
      o[k & 1] = mma32<T>(vf[k], make_uint4(p[0], p[1], p[2], p[3]), o[k & 1]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t* p = w.rest + 4 * (k >> 1);
      o[k & 1] = mma32<T>(vf[k], make_uint4(p[0], p[1], p[2], p[3]), o[k & 1]);
    }
  }
  // The weights are 2^(scale s + ref) of products s.
  __device__ inline float ref_of(float scale) const { return r == -INFINITY ? TOP : fmaf(-r, scale, TOP); }
  // The largest product of the lane's column.
  __device__ static inline float largest(const f32x16& s) {
    float m = most_of(most_of(s[0], s[1]), s[2]);
#pragma unroll
    for (int e = 3; e < 15; e += 2) m = most_of(most_of(m, s[e]), s[e + 1]);
    return over_two(most_of(m, s[15]), most_of);
  }
  // Of half a tile from position `first` on (a multiple of 32), in the group of 8 keys in one page: how many from the lane's own first
  // one on its column sees.
  __device__ inline int limit(int first, uint32_t pages, int group) const {
    const int at = (first & (WIDE_KEYS - 1)) + group * 8, bit = c.page_size < WIDE_KEYS ? at >> c.shift : 0;
    return pages >> bit & 1 ? hi - first - 4 * (lane >> 5) - 8 * group : -WIDE_KEYS;
  }

  // Half a tile by itself: keys that not all columns see, and columns whose reference is not there yet. CAREFUL: the reference follows
  // the largest score, and infinities and NaN among the values count where they are seen and nowhere else.
  template <bool CAREFUL> __device__ inline void half_tile(int t, int half, uint32_t pages, float scale, float& ref) {
    const int b = t % WIDE_RING, first = t * WIDE_KEYS + half * 32;
    uint4 kf[4], vf[4];
    f32x16 s;
    Weights w;
    load_keys(kf, b, half);
    score(s, kf);
    load_values(vf, b, half);
#pragma unroll
    for (int x4 = 0; x4 < 4; ++x4) {
      const int below = limit(first, pages, x4);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * x4 + e] = e < below ? s[4 * x4 + e] : -INFINITY;
    }
    const float mx = largest(s), old = r, was = ref;
    r = r == -INFINITY || (CAREFUL && mx > r) ? mx : r;
    ref = ref_of(scale);
    if (CAREFUL) {  // where there was none, the sums are zeros
      const float keep = r == old ? 1.f : old == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - was);
      l *= keep;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        o[0][e] *= keep;
        o[1][e] *= keep;
      }
    }
    weights(w, s, scale, ref);
    if constexpr (CAREFUL) {
      const f32x16 zero = {};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 raw = vf[k];
        weigh_one(w, k, map_pairs(raw, [](float y) { return fabsf(y) < INFINITY ? y : 0.f; }));
        uint32_t one[4];  // how many of each other kind the column sees
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int below = limit(first, pages, 2 * (k >> 1) + e / 2) - 2 * (e & 1);
          one[e] = pack2<T>(below > 0 ? 1.f : 0.f, below > 1 ? 1.f : 0.f);
        }
        const uint4 sees = make_uint4(one[0], one[1], one[2], one[3]);
        auto add = [&](auto&& kind, float what) {
          const f32x16 count = mma32<T>(map_pairs(raw, [&](float y) { return kind(y) ? 1.f : 0.f; }), sees, zero);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[k & 1][e] += count[e] > 0.f ? what : 0.f;
        };
        add([](float y) { return y != y; }, NAN);
        add([](float y) { return y == INFINITY; }, INFINITY);
        add([](float y) { return y == -INFINITY; }, -INFINITY);
      }
    } else {
      weigh(w, vf);
    }
  }

  // Weights are taken here, not where they are used first: that is behind the next barrier.
  __device__ inline void pin(Weights& w) {
    asm volatile("" : "+v"(l));
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      asm volatile("" : "+v"(w.p[e]), "+v"(w.p[e + 1]), "+v"(w.p[e + 2]), "+v"(w.p[e + 3]));
      asm volatile("" : "+v"(w.rest[e]), "+v"(w.rest[e + 1]), "+v"(w.rest[e + 2]), "+v"(w.rest[e + 3]));
    }
  }
  // Beside the twelve matrix instructions of half a tile: the vector unit's work, six of its instructions between each two (4, 5, 7
  // and 9 take as long, 8 are 6% slower).
  __device__ static inline void interleave() {
#pragma unroll
    for (int k = 0; k < 12; ++k) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
    }
  }

  // Tiles t0 up to t1. True where the sums are not to be taken: a NaN, an infinity, or weights beyond 2^64.
  template <bool CAREFUL> __device__ inline bool pass(int t0, int t1, float scale) {
    float ref = TOP;
#pragma unroll
    for (int x = 0; x < 16; ++x) o[0][x] = o[1][x] = 0.f;
    r = -INFINITY;
    l = 0.f;
    key0 = 0x7fffffff;
    full = (1u << max(1, WIDE_KEYS >> c.shift)) - 1;
    uint32_t pages = 0, next = 0;  // of tiles t and t + 1
    if (t0 < t1) {
      const int k = ((t0 * WIDE_KEYS) >> c.shift) >> 6;
      take_entries(k, load_entries(k));
      next = issue(t0);
    }
    // Tile t is there, all waves' loads, and tile t - 2 used up: its slot is tile t + 1's.
    auto arrive = [&](int t) {
      wait_loads<0>();
      asm volatile("s_barrier" ::: "memory");
      pages = next;
      if (t + 1 < t1) next = issue(t + 1);
    };
    auto plain = [&](int t) {  // all columns see all of tile t, and have their reference
      return !CAREFUL && pages == full && (t + 1) * WIDE_KEYS <= least && !__builtin_amdgcn_ballot_w64(r == -INFINITY && hi > 0);
    };
    int t = t0;
    if (t < t1) arrive(t);
#pragma unroll 1
    while (t < t1) {
      if (!plain(t)) {
        if (t * WIDE_KEYS < most) {
          if (pages && key0 == 0x7fffffff) key0 = t * WIDE_KEYS + (__builtin_ctz(pages) << c.shift);
          half_tile<CAREFUL>(t, 0, pages, scale, ref);
          half_tile<CAREFUL>(t, 1, pages, scale, ref);
        }
        if (++t < t1) arrive(t);
        continue;
      }
      if constexpr (!CAREFUL) {
        // the first half's scores, and weights of 0 in the place of the half before it
        f32x16 sa, sb;
        Weights pa, pb = {};
        uint4 kf[4], vf[4];
        load_keys(kf, t % WIDE_RING, 0);
        load_values(vf, t % WIDE_RING, 0);
        score(sa, kf);
        bool more;
#pragma unroll 1
        do {
          const int b = t % WIDE_RING;
          load_keys(kf, b, 1);
          weigh(pb, vf);
          weights(pa, sa, scale, ref);
          load_values(vf, b, 0);
          score(sb, kf);
          interleave();
          pin(pa);
          more = ++t < t1;
          if (more) {
            arrive(t);
            more = plain(t);
          }
          load_keys(kf, (b + 1) % WIDE_RING, 0);  // where that is no plain tile, of any: its scores are not used
          weigh(pa, vf);
          weights(pb, sb, scale, ref);
          load_values(vf, b, 1);
          score(sa, kf);
          interleave();
          pin(pb);
        } while (more);
        weigh(pb, vf);
      }
    }
    bool bad = !(l <= 18446744073709551616.f);
#pragma unroll
    for (int x = 0; x < 16; ++x) bad |= !(fabsf(o[0][x]) < INFINITY) || !(fabsf(o[1][x]) < INFINITY);
    return __syncthreads_or(bad && most > 0);
  }
};

template <typename T>
__global__ void __launch_bounds__(WAVES * 64, WIDE_OCCUPANCY) prefix_wide_kernel(const PrefixArgs a, int blocks, bool join, size_t parts, char* workspace) {
  constexpr int R = WAVES * 32;
  __shared__ __attribute__((aligned(1024))) char smem[WIDE_RING * WIDE_BYTES];
  __shared__ int ends[WAVES];
  const Mine mine = find_item<WIDE_KEYS, R>(a, blocks, workspace, join);
  if (uniform(mine.id) < 0) return;
  const KvCache& c = a.cache;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 5, G = a.heads / c.kv_heads;
  const int kh = uniform(mine.kh), shared = uniform(mine.shared), rows = uniform(mine.tokens) * G, start = uniform(mine.start);
  WideWave<T> w{c, kh, lane, wave, smem, a.prefix + long(uniform(mine.group)) * a.prefix_width, a.prefix_width};
  // a scale's sign goes into the queries, exactly, and a scale of 0: the largest score is then the largest product
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, hold = a.scale == 0.f ? 0u : ~0u;
  const float scale = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.44269504088896341f;
  const int column = wave * 32 + (lane & 31), row = uniform(mine.item) * R + column;
  const bool in = row < rows;
  const int token = start + (in ? row / G : 0), head = kh * G + (in ? row % G : 0);
  w.hi = in ? max(0, min(a.lens ? a.lens[token] : shared, shared)) : 0;
#pragma unroll
  for (int st = 0; st < 4; ++st) {
    const uint4 x = in ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + long(token) * a.ldq + long(head) * 64 + st * 16 + g * 8) : make_uint4(0, 0, 0, 0);
    w.q[st] = make_uint4((x.x ^ flip) & hold, (x.y ^ flip) & hold, (x.z ^ flip) & hold, (x.w ^ flip) & hold);
  }
  int most = w.hi, least = in ? w.hi : 0x7fffffff;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    most = max(most, __shfl_xor(most, x));
    least = min(least, __shfl_xor(least, x));
  }
  w.most = uniform(most);
  w.least = uniform(least);
  if (lane == 0) ends[wave] = most;
  __syncthreads();
  w.end = 0;
#pragma unroll
  for (int k = 0; k < WAVES; ++k) w.end = max(w.end, uniform(ends[k]));
  const int tiles = (shared + WIDE_KEYS - 1) / WIDE_KEYS, seen = (w.end + WIDE_KEYS - 1) / WIDE_KEYS, k = uniform(mine.part), of = uniform(mine.parts);
  const int t0 = int(long(tiles) * k / of), t1 = min(seen, int(long(tiles) * (k + 1) / of));
  if (w.template pass<false>(t0, t1, scale)) w.template pass<true>(t0, t1, scale);
  const float sum = over_two(w.l, [](float x, float y) { return x + y; });
  const bool some = w.hi > w.key0;
  if (join) {
    float* part = part_at(workspace, parts, uniform(mine.id), R);
    // the largest score as it is: what its weight is other than 1 goes into the sums, 2^TOP and what rounding ref left of scale r
    const bool none = w.r == -INFINITY;
    const float f = none ? 1.f : __builtin_amdgcn_exp2f(-fmaf(w.r, scale, w.ref_of(scale))), m = none ? w.r : w.r * fabsf(a.scale);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<float4*>(part + column * 64 + dt * 32 + 8 * k + 4 * g) =
            make_float4(w.o[dt][4 * k] * f, w.o[dt][4 * k + 1] * f, w.o[dt][4 * k + 2] * f, w.o[dt][4 * k + 3] * f);
    if (g == 0) *reinterpret_cast<float2*>(part + R * 64 + column * 2) = make_float2(m, some ? sum * f : -1.f);
  } else if (in) {
    const float inv = 1.f / sum;
    T* out = static_cast<T*>(a.out) + long(token) * a.ldo + long(head) * 64 + 4 * g;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = some ? w.o[dt][4 * k + e] * inv : 0.f;
        *reinterpret_cast<uint2*>(out + dt * 32 + 8 * k) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
      }
  }
}

// --- the join -----------------------------------------------------------------------------------

// 16 lanes hold a part's column, four channels each. A wave takes one (token, head), four parts a load and 4 AT_ONCE under way, or four
// (token, head)s, a part of each a load, where there are MANY_COLUMNS, so that all of them are on the chip at once. Bound by its chain of
// loads (starts, the plan, the parts), and by the parts' bytes where there are many rows. Measured, one / four a wave: 768 of them 5.7 / 6.9 us,
// 1536 7.4 / 8.9, 12444 (seven parts, 26 MB) 14.2 / 9.8; of whole calls 4800 65.3 / 65.9, 7200 80.0 / 78.9, 9600 99.6 / 97.4.
constexpr int JOIN_WAVES = 4, AT_ONCE = 8;
constexpr long MANY_COLUMNS = 6144;  // (token, head)s
template <typename T, int COLUMNS>
__global__ void __launch_bounds__(JOIN_WAVES * 64) prefix_join_kernel(const PrefixArgs a, int R, int own, size_t parts, size_t own_parts, char* workspace) {
  constexpr int ACROSS = 4 / COLUMNS;  // parts of a load
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), quad = lane & 15, g = lane >> 4;
  const int u0 = (int(blockIdx.x) * JOIN_WAVES + wave) * COLUMNS, all_columns = a.n * a.heads;  // below 2^21
  if (u0 >= all_columns) return;
  const GroupPlan* plans = reinterpret_cast<const GroupPlan*>(workspace + sizeof(PlanHead));
  // for up to 64 groups what is asked of them comes in one load, a group a lane
  const int near = min(lane, a.groups - 1), valid = reinterpret_cast<const PlanHead*>(workspace)->valid, begin = start_of(a, near), end = start_of(a, near + 1);
  const GroupPlan near_plan = plans[near];
  if (!valid) return;
  const int u = u0 + (COLUMNS > 1 ? g : 0), i = u / a.heads, head = u - i * a.heads;
  GroupPlan plan = {};
  bool found = false;
#pragma unroll
  for (int x = 0; x < COLUMNS; ++x) {
    const int token = COLUMNS > 1 ? __builtin_amdgcn_readlane(i, 16 * x) : i;
    GroupPlan its;
    if (a.groups <= 64) {
      const uint64_t in = __ballot(lane < a.groups && begin <= token && token < end);
      if (!in) continue;
      const int l = 63 - __builtin_clzll(in);
      its = {__builtin_amdgcn_readlane(near_plan.block0, l), __builtin_amdgcn_readlane(near_plan.parts, l), __builtin_amdgcn_readlane(near_plan.items, l),
             __builtin_amdgcn_readlane(near_plan.row0, l)};
    } else {
      const int group = group_of(a, min(token, a.n - 1));
      if (group < 0) continue;
      its = plans[group];
    }
    if (COLUMNS == 1 || g == x) {
      plan = its;
      found = true;
    }
  }
  found &= u < all_columns;
  const KvCache& c = a.cache;
  const int G = a.heads / c.kv_heads, kh = head / G, e = head - kh * G;
  const int r = (i - plan.row0) * G + e, item = r / R, column = r - item * R, columns = min(G, 16), cols = c.kv_heads * ((G + 15) / 16);
  const long own0 = (long(i) * cols + kh * ((G + 15) / 16) + e / 16) * own;
  const int count = found ? plan.parts + own : 0;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f, m = -INFINITY;
  bool some = false;
  for (int k0 = 0; k0 < count; k0 += ACROSS * AT_ONCE) {
    float2 ml[AT_ONCE];
    float4 o[AT_ONCE];
    float mx = m;
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      const int k = k0 + ACROSS * x + (COLUMNS > 1 ? 0 : g);
      ml[x] = make_float2(0.f, -1.f);
      if (k0 + ACROSS * x >= count || k >= count) continue;
      const bool mine = k >= plan.parts;
      const int width = mine ? columns : R, at = mine ? e % 16 : column;
      const float* p = mine ? part_at(workspace, own_parts, own0 + k - plan.parts, columns)
                            : part_at(workspace, parts, plan.block0 + (long(kh) * plan.parts + k) * plan.items + item, R);
      ml[x] = *reinterpret_cast<const float2*>(p + width * 64 + at * 2);
      o[x] = *reinterpret_cast<const float4*>(p + at * 64 + quad * 4);
    }
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x)
      if (!(ml[x].y < 0.f)) {  // NaN stays
        mx = fmaxf(mx, ml[x].x);
        some = true;
      }
    const float keep = m == -INFINITY ? 0.f : exp_of(m - mx);
    acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
    sum *= keep;
    m = mx;
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x)
      if (!(ml[x].y < 0.f)) {
        const float f = ml[x].x == -INFINITY ? 0.f : exp_of(ml[x].x - mx);
        acc = make_float4(acc.x + o[x].x * f, acc.y + o[x].y * f, acc.z + o[x].z * f, acc.w + o[x].w * f);
        sum += ml[x].y * f;
      }
  }
  float v[4] = {acc.x, acc.y, acc.z, acc.w};
  if constexpr (COLUMNS == 1) {  // the four groups of lanes; one without a key has zeros, whatever the others hold
    const float top = max_groups(m), f = m == -INFINITY ? 0.f : exp_of(m - top);
    auto all = [&](float x) { return sum_groups(some ? x * f : 0.f); };
    sum = all(sum);
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = all(v[x]);
    some = max_groups(some ? 1.f : 0.f) > 0.f;
    if (g) return;
  }
  if (!found) return;
#pragma unroll
  for (int x = 0; x < 4; ++x) v[x] = some ? v[x] / sum : 0.f;
  T* out = static_cast<T*>(a.out) + long(i) * a.ldo + long(head) * 64 + quad * 4;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
  else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
}

}  // namespace

void prefix_attention(const Exec& ex, const PrefixArgs& args, void* workspace, size_t bytes) {
  PrefixArgs a = args;
  check_prefix_attention(a, workspace, bytes);
  if (a.n == 0 || a.groups == 0 || ex.dry) return;
  const KvCache& c = a.cache;
  const PrefixPlan plan = prefix_plan(a);
  const double seen = double(a.n) * (double(a.max_shared) + a.max_own);
  ProfScope prof(ex, "prefix_attention", 256 * seen * a.heads,
                 128.0 * c.kv_heads * dtype_size(c.dt) * (double(a.groups) * a.max_shared + double(a.n) * a.max_own));
  const int G = a.heads / c.kv_heads;
  const long own = long(a.n) * c.kv_heads * ((G + 15) / 16) * plan.own;
  char* ws = static_cast<char*>(workspace);
  by_type(c.dt, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto kernel) {
      kernel<<<int(plan.blocks + own), WAVES * 64, 0, ex.stream>>>(a, plan.blocks, plan.own, plan.join, plan.parts, plan.own_parts, ws);
    };
    if (plan.rows == 16) launch(prefix_parts_kernel<T, 1>);
    else if (plan.rows == 32) launch(prefix_parts_kernel<T, 2>);
    else if constexpr (sizeof(T) == 4) launch(prefix_parts_kernel<T, 4>);
    else {
      if (own) prefix_own_kernel<T><<<int(own), WAVES * 64, 0, ex.stream>>>(a, plan.own, plan.own_parts, ws);
      prefix_wide_kernel<T><<<plan.blocks, WAVES * 64, 0, ex.stream>>>(a, plan.blocks, plan.join, plan.parts, ws);
    }
    auto join = [&](auto columns) {
      constexpr int N = decltype(columns)::value;
      prefix_join_kernel<T, N><<<cdiv(long(a.n) * a.heads, JOIN_WAVES * N), JOIN_WAVES * 64, 0, ex.stream>>>(a, plan.rows, plan.own, plan.parts, plan.own_parts, ws);
    };
    if (!plan.join) return;
    if (long(a.n) * a.heads >= MANY_COLUMNS) join(std::integral_constant<int, 4>());
    else join(std::integral_constant<int, 1>());
  });
  SPLAT_HIP(hipGetLastError());
}

}  // namespace splat
