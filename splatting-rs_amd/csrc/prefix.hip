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

  // Tiles t, t + step, ... below stop: tile k is asked for while tile k - 2 is used. Where a sum is NaN they are taken again with
  // care: a weight of 0 times an infinity, or one beside the second term of a weight, is no answer.
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
  __device__ inline void run(int t, int step, int stop, float scale) {
    const int count = t < stop ? (stop - t + step - 1) / step : 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) ops[n].pin_q();
    if (pass<false>(t, step, count, scale)) pass<true>(t, step, count, scale);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      l[n] = sum_groups(l[n]);
      some[n] = over_rows(float(some[n]), [](float a, float b) { return fmaxf(a, b); }) > 0.f;
    }
  }
};

// --- a block ------------------------------------------------------------------------------------

// A part: `columns` times 64 sums, then (m, l) of each; l is -1 where no key was there.
__device__ inline float* part_at(char* workspace, size_t offset, long index, int columns) {
  return reinterpret_cast<float*>(workspace + offset) + index * columns * long(PART_HEAD);
}

// The waves' sums join in LDS: wave d adds up channels 16 d + (0..15) of every column. place(column) gives the output's row
// (normalised, where `whole`) or nullptr for columns without one; the others go to `part`.
template <typename T, int NT, typename Place>
__device__ inline void join_waves(const PrefixWave<T, NT>& w, char* smem, float (*stats)[NT * 16][4], int wave, bool whole, float* part, int columns, Place&& place) {
  const int lane = w.lane, col = lane & 15, g = lane >> 4;
  float* mine = reinterpret_cast<float*>(smem + wave * RING * TILE_BYTES);  // its tiles are used up
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) mine[((n * 4 + d) * 4 + r) * 64 + lane] = w.o[n][d][r];
    if (g == 0) {
      float* s = stats[wave][n * 16 + col];
      s[0] = w.m[n];
      s[1] = w.l[n];
      s[2] = float(w.some[n]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int column = n * 16 + col;
    float mn = -INFINITY, sum = 0.f, v[4] = {};
    bool some = false;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) mn = fmaxf(mn, stats[k][column][0]);
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const float* s = stats[k][column];
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
      T* out = place(column);
      if (!out) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = some ? v[r] / sum : 0.f;
      out += 16 * wave + 4 * g;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
      else *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
      *reinterpret_cast<float4*>(part + column * 64 + 16 * wave + 4 * g) = make_float4(v[0], v[1], v[2], v[3]);
      if (wave == 0 && g == 0) *reinterpret_cast<float2*>(part + columns * 64 + column * 2) = make_float2(mn, some ? sum : -1.f);
    }
  }
}

// A block's part of the groups' items.
struct Mine {
  int group, item, kh, part, parts;  // group -1: nothing
  int start, tokens, shared;
};

// Thread t sums up its k groups; block 0 leaves the plan for the join. The tiles of a part: as many as leave no more parts
// than blocks (an item of T tiles has at most T / each + 1).
template <int KEYS, int R> __device__ inline Mine find_item(const PrefixArgs& a, int blocks, char* workspace, bool join) {
  __shared__ long sums[WAVES];
  __shared__ Mine found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, G = a.heads / a.cache.kv_heads, kv = a.cache.kv_heads;
  const int k = (a.groups + WAVES * 64 - 1) / (WAVES * 64), g0 = min(tid * k, a.groups), g1 = min(g0 + k, a.groups);
  auto total_of = [&](long v, long& before) {
    const long s = long(scan_wave(uint64_t(v), uint64_t(0), [](uint64_t x, uint64_t y) { return x + y; }));
    __syncthreads();
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    before = s - v;
    long total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) before += sums[w];
      total += sums[w];
    }
    return total;
  };
  if (tid == 0) found.group = -1;
  long items = 0, tiles = 0, tokens = 0, before;
  for (int g = g0; g < g1; ++g) {
    const int m = max(0, start_of(a, g + 1) - start_of(a, g));
    const long its = (long(m) * G + R - 1) / R;
    items += its * kv;
    tiles += its * kv * ((shared_of(a, g) + KEYS - 1) / KEYS);
    tokens += m;
  }
  const bool valid = total_of(tokens, before) <= a.n;  // more only where starts descend: nothing is done
  const long all_items = total_of(items, before), all_tiles = total_of(tiles, before);
  const long spare = blocks - all_items, each = join && spare > 0 ? max(1L, quotient(all_tiles + spare - 1, spare)) : 1L << 40;
  long count = 0;
  auto parts_of = [&](int shared) { return int(max(1L, quotient((shared + KEYS - 1) / KEYS + each - 1, each))); };
  for (int g = g0; g < g1; ++g) {
    const int m = max(0, start_of(a, g + 1) - start_of(a, g));
    count += (long(m) * G + R - 1) / R * kv * parts_of(shared_of(a, g));
  }
  total_of(valid ? count : 0, before);
  if (valid) {
    long at = before;
    for (int g = g0; g < g1; ++g) {
      const int start = start_of(a, g), m = max(0, start_of(a, g + 1) - start), shared = shared_of(a, g), parts = parts_of(shared);
      const int its = int((long(m) * G + R - 1) / R);
      const long here = long(its) * kv * parts;
      if (join && blockIdx.x == 0) reinterpret_cast<GroupPlan*>(workspace + sizeof(PlanHead))[g] = {int(at), parts, its, start};
      if (long(blockIdx.x) >= at && long(blockIdx.x) < at + here) {
        // items fastest: those that read the same keys run at the same time
        const int r = int(blockIdx.x - at), item = r % its, rest = r / its;
        found = {g, item, rest / parts, rest % parts, parts, start, m, shared};
      }
      at += here;
    }
  }
  if (join && blockIdx.x == 0 && tid == 0) reinterpret_cast<PlanHead*>(workspace)->valid = valid;
  __syncthreads();
  return found;
}

template <typename T, int NT>
__global__ void __launch_bounds__(WAVES * 64, 2) prefix_parts_kernel(const PrefixArgs a, int blocks, int own, bool join, size_t parts, size_t own_parts, char* workspace) {
  using Ops = TileOps<T>;
  constexpr int KEYS = Ops::KEYS, R = NT * 16;
  __shared__ __attribute__((aligned(1024))) char smem[WAVES * RING * TILE_BYTES];
  __shared__ float stats[WAVES][R][4];
  const KvCache& c = a.cache;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int G = a.heads / c.kv_heads;
  char* ring = smem + wave * RING * TILE_BYTES;
  const uint32_t lds = uint32_t(reinterpret_cast<uintptr_t>((lds_cptr)ring));
  if (int(blockIdx.x) < blocks) {
    const Mine mine = find_item<KEYS, R>(a, blocks, workspace, join);
    if (uniform(mine.group) < 0) return;
    const int kh = uniform(mine.kh), shared = uniform(mine.shared);
    PrefixWave<T, NT> w{c, kh, lane, lds, ring, a.prefix + long(uniform(mine.group)) * a.prefix_width, a.prefix_width};
    const int rows = uniform(mine.tokens) * G;
    int most = 0, least = 0x7fffffff;
    int token[NT], head[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = uniform(mine.item) * R + n * 16 + col;  // below 2^21
      const bool in = r < rows;
      token[n] = uniform(mine.start) + (in ? r / G : 0);
      head[n] = in ? kh * G + r % G : -1;
      w.hi[n] = in ? max(0, min(a.lens ? a.lens[token[n]] : shared, shared)) : 0;
      w.ops[n].load_q(static_cast<const T*>(a.q) + long(token[n]) * a.ldq + long(max(head[n], 0)) * 64, g, in);
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
    const int tiles = (shared + KEYS - 1) / KEYS, seen = (w.end + KEYS - 1) / KEYS, part = uniform(mine.part), of = uniform(mine.parts);
    const int t0 = int(long(tiles) * part / of), t1 = min(seen, int(long(tiles) * (part + 1) / of));
    w.run(t0 + wave, WAVES, t1, a.scale);
    join_waves<T, NT>(w, smem, stats, wave, !join, part_at(workspace, parts, blockIdx.x, R), R, [&](int column) {
      const int n = column >> 4;
      T* out = nullptr;
#pragma unroll
      for (int k = 0; k < NT; ++k)
        if (k == n && head[k] >= 0) out = static_cast<T*>(a.out) + long(token[k]) * a.ldo + long(head[k]) * 64;
      return out;
    });
    return;
  }
  // a token's own positions
  const int cols = c.kv_heads * ((G + 15) / 16), columns = min(G, 16);
  const int u = int(blockIdx.x) - blocks, part = u % own, i = u / own / cols, group = u / own % cols, kh = group / ((G + 15) / 16), h0 = group % ((G + 15) / 16) * 16;
  const int grp = group_of(a, i);
  PrefixWave<T, 1> w{c, kh, lane, lds, ring, a.table + long(i) * a.width, a.width};
  const bool in = h0 + col < G;
  w.ops[0].load_q(static_cast<const T*>(a.q) + long(i) * a.ldq + long(kh * G + h0 + (in ? col : 0)) * 64, g, in);
  w.lo = grp < 0 ? 0 : uniform(shared_of(a, grp));
  w.end = grp < 0 ? 0 : uniform(int(min(long(length_of(a.lens[i], a.width, c.shift, 0x7fffffff)), long(w.lo) + a.max_own)));
  w.least = w.hi[0] = w.end;
  const int first = w.lo / KEYS, tiles = w.end > w.lo ? (w.end + KEYS - 1) / KEYS - first : 0;
  w.run(first + int(long(tiles) * part / own) + wave, WAVES, first + int(long(tiles) * (part + 1) / own), a.scale);
  float* to = part_at(workspace, own_parts, u, columns);
  __shared__ float own_stats[WAVES][16][4];
  join_waves<T, 1>(w, smem, own_stats, wave, false, to, columns, [](int) { return static_cast<T*>(nullptr); });
}

// --- the join -----------------------------------------------------------------------------------

// One wave a (token, head): a channel a lane, AT_ONCE parts under way.
constexpr int JOIN_WAVES = 4, AT_ONCE = 8;
template <typename T, int R>
__global__ void __launch_bounds__(JOIN_WAVES * 64) prefix_join_kernel(const PrefixArgs a, int own, size_t parts, size_t own_parts, char* workspace) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int u = int(blockIdx.x) * JOIN_WAVES + wave;  // below 2^21
  if (u >= a.n * a.heads || !reinterpret_cast<const PlanHead*>(workspace)->valid) return;
  const int i = u / a.heads, head = u % a.heads, g = group_of(a, i);
  if (g < 0) return;
  const KvCache& c = a.cache;
  const int G = a.heads / c.kv_heads, kh = head / G, e = head % G;
  const GroupPlan plan = reinterpret_cast<const GroupPlan*>(workspace + sizeof(PlanHead))[g];
  const int r = (i - plan.row0) * G + e, item = r / R, column = r % R, columns = min(G, 16), cols = c.kv_heads * ((G + 15) / 16);
  const long own0 = (long(i) * cols + kh * ((G + 15) / 16) + e / 16) * own;
  const int count = plan.parts + own;
  float acc = 0.f, sum = 0.f, m = -INFINITY;
  bool some = false;
  for (int k0 = 0; k0 < count; k0 += AT_ONCE) {
    float2 ml[AT_ONCE];
    float o[AT_ONCE], mx = m;
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      const int k = min(k0 + x, count - 1);
      const bool mine = k >= plan.parts;
      const int width = mine ? columns : R, at = mine ? e % 16 : column;
      const float* p = mine ? part_at(workspace, own_parts, own0 + k - plan.parts, columns)
                            : part_at(workspace, parts, plan.block0 + (long(kh) * plan.parts + k) * plan.items + item, R);
      ml[x] = *reinterpret_cast<const float2*>(p + width * 64 + at * 2);
      o[x] = p[at * 64 + lane];
    }
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x)
      if (k0 + x < count && !(ml[x].y < 0.f)) {  // NaN stays
        mx = fmaxf(mx, ml[x].x);
        some = true;
      }
    const float keep = m == -INFINITY ? 0.f : exp_of(m - mx);
    acc *= keep;
    sum *= keep;
    m = mx;
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x)
      if (k0 + x < count && !(ml[x].y < 0.f)) {
        const float f = ml[x].x == -INFINITY ? 0.f : exp_of(ml[x].x - mx);
        acc += o[x] * f;
        sum += ml[x].y * f;
      }
  }
  static_cast<T*>(a.out)[long(i) * a.ldo + long(head) * 64 + lane] = from_f<T>(some ? acc / sum : 0.f);
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
    prefix_parts_kernel<T, 1><<<int(plan.blocks + own), WAVES * 64, 0, ex.stream>>>(a, plan.blocks, plan.own, plan.join, plan.parts, plan.own_parts, ws);
    if (plan.join)
      prefix_join_kernel<T, 16><<<cdiv(long(a.n) * a.heads, JOIN_WAVES), JOIN_WAVES * 64, 0, ex.stream>>>(a, plan.own, plan.parts, plan.own_parts, ws);
  });
  SPLAT_HIP(hipGetLastError());
}

}  // namespace splat
