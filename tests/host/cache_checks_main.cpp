// The argument checks of the paged cache's operators, without a GPU: each named call starts from one that is
// accepted and changes one thing. Prints "name OK" or "name ERR code message". The pointers are never followed.
#include <cmath>
#include <cstdio>
#include <functional>
#include <limits>
#include <string>

#include "../../splatting-rs_amd/csrc/cache.h"

using namespace splat;

namespace {

char* at(long offset) { return reinterpret_cast<char*>((1L << 40) + offset); }
int* ints(long offset) { return reinterpret_cast<int*>(at(offset)); }
constexpr long MB = 1L << 20;

KvCache cache() {  // bf16, 100 pages of 16 rows, 4 heads: pools of 819200 bytes
  KvCache c;
  c.dt = 1;
  c.pages = 100;
  c.page_size = 16;
  c.kv_heads = 4;
  c.page_stride = 4 * 16 * 64;
  c.k = at(0);
  c.v = at(MB);
  return c;
}

BlockTableArgs tables() {
  BlockTableArgs a;
  a.n = 10;
  a.page_size = 16;
  a.past = ints(0);
  a.add = ints(64);
  a.pool = ints(128);
  a.pool_size = 100;
  a.used = ints(1024);
  a.table = ints(2048);
  a.width = 8;
  a.lens = ints(4096);
  a.starts = ints(4160);
  a.slots = ints(8192);
  a.positions = ints(16384);
  a.cap = 1000;
  a.used_out = ints(32768);
  a.status = ints(32772);
  return a;
}

QkArgs qk() {
  QkArgs a;
  a.dt = 1;
  a.tokens = 10;
  a.heads = 8;
  a.kv_heads = 4;
  a.qkv = at(8 * MB);
  a.ld = 16 * 64;
  a.norm = NORM_LAYER;
  a.eps = 1e-5f;
  a.rope = ROPE_GRID;
  a.positions = ints(16 * MB);
  a.q_out = at(12 * MB);
  a.ldq = 8 * 64;
  a.k_out = at(13 * MB);
  a.ldk = 4 * 64;
  a.has_cache = true;
  a.cache = cache();
  a.slots = ints(17 * MB);
  return a;
}

BoundsArgs bounds() {
  BoundsArgs a;
  a.cache = cache();
  a.n = 3;
  a.table = ints(8 * MB);
  a.width = 20;
  a.lens = ints(9 * MB);
  a.add = ints(9 * MB + 64);
  a.max_add = 40;
  a.bounds = at(10 * MB);
  return a;
}

PagedArgs paged() {
  PagedArgs a;
  a.cache = cache();
  a.n = 3;
  a.heads = 8;
  a.q = at(8 * MB);
  a.ldq = 8 * 64;
  a.table = ints(9 * MB);
  a.width = 20;
  a.lens = ints(10 * MB);
  a.max_len = 300;
  a.scale = 0.125f;
  a.out = at(11 * MB);
  a.ldo = 8 * 64;
  return a;
}

SparseArgs sparse() {
  SparseArgs a;
  a.at = paged();
  a.bounds = at(12 * MB);
  a.topk = 5;
  a.selected = ints(13 * MB);
  return a;
}

void say(const char* name, const std::function<void()>& f) {
  try {
    f();
    std::printf("%s OK\n", name);
  } catch (const Error& e) {
    std::printf("%s ERR %d %s\n", name, e.code, e.what());
  }
}

template <typename A> void on(const char* name, A a, void (*check)(A&), const std::function<void(A&)>& change) {
  say(name, [&] {
    change(a);
    check(a);
  });
}

void check_qk(QkArgs& a) { check_qk_norm_rope(a, 100.0); }
void check_paged(PagedArgs& a) { check_paged_attention(a, at(4096 * MB), size_t(1) << 40); }
void check_sparse(SparseArgs& a) { check_sparse_attention(a, at(4096 * MB), size_t(1) << 40); }

}  // namespace

int main() {
  const float inf = std::numeric_limits<float>::infinity(), nan = std::nanf("");
  auto T = [&](const char* n, const std::function<void(BlockTableArgs&)>& f) { on<BlockTableArgs>(n, tables(), check_block_tables, f); };
  T("tables ok", [](auto&) {});
  T("tables ok lens over past", [](auto& a) { a.lens = const_cast<int*>(a.past); });
  T("tables ok used over used", [](auto& a) { a.used_out = const_cast<int*>(a.used); });
  T("tables ok no positions", [](auto& a) { a.positions = nullptr; });
  T("tables ok no requests", [](auto& a) { a.n = 0; a.past = a.add = nullptr; a.table = a.lens = nullptr; });
  T("tables ok no slots", [](auto& a) { a.cap = 0; a.slots = nullptr; a.positions = nullptr; });
  T("tables ok no pool", [](auto& a) { a.pool_size = 0; a.pool = nullptr; });
  T("tables n -1", [](auto& a) { a.n = -1; });
  T("tables n 65537", [](auto& a) { a.n = 65537; });
  T("tables page 4", [](auto& a) { a.page_size = 4; });
  T("tables page 24", [](auto& a) { a.page_size = 24; });
  T("tables page 512", [](auto& a) { a.page_size = 512; });
  T("tables page 0", [](auto& a) { a.page_size = 0; });
  T("tables page -16", [](auto& a) { a.page_size = -16; });
  T("tables width 0", [](auto& a) { a.width = 0; });
  T("tables width 2^27", [](auto& a) { a.width = 1 << 27; });
  T("tables pool -1", [](auto& a) { a.pool_size = -1; });
  T("tables cap -1", [](auto& a) { a.cap = -1; });
  T("tables past NULL", [](auto& a) { a.past = nullptr; });
  T("tables pool NULL", [](auto& a) { a.pool = nullptr; });
  T("tables slots NULL", [](auto& a) { a.slots = nullptr; });
  T("tables status NULL", [](auto& a) { a.status = nullptr; });
  T("tables lens into past", [](auto& a) { a.lens = const_cast<int*>(a.past) + 1; });
  T("tables slots over table", [](auto& a) { a.slots = a.table + 79; });
  T("tables used_out over pool", [](auto& a) { a.used_out = const_cast<int*>(a.pool) + 99; });
  T("tables odd lens", [](auto& a) { a.lens = reinterpret_cast<int*>(at(4 * 4096 + 2)); });
  T("tables status over used_out", [](auto& a) { a.status = a.used_out; });

  auto Q = [&](const char* n, const std::function<void(QkArgs&)>& f) { on<QkArgs>(n, qk(), check_qk, f); };
  Q("qk ok", [](auto&) {});
  Q("qk ok in place", [](auto& a) { a.q_out = const_cast<void*>(a.qkv); a.ldq = a.ld; a.k_out = at(8 * MB + 1024); a.ldk = a.ld; });
  Q("qk ok no cache", [](auto& a) { a.has_cache = false; a.slots = nullptr; });
  Q("qk ok side by side", [](auto& a) { a.ldq = a.ldk = 12 * 64; a.k_out = at(12 * MB + 1024); });
  Q("qk ok nothing", [](auto& a) { a.tokens = 0; a.qkv = a.q_out = a.k_out = nullptr; a.positions = nullptr; });
  Q("qk ok keys and values share pages", [](auto& a) { a.cache.page_stride *= 2; a.cache.v = at(4 * 16 * 64 * 2); });
  Q("qk keys over values", [](auto& a) { a.cache.v = at(16); });
  Q("qk dtype 3", [](auto& a) { a.dt = 3; });
  Q("qk heads 0", [](auto& a) { a.heads = 0; });
  Q("qk kv_heads 0", [](auto& a) { a.kv_heads = 0; });
  Q("qk tokens 2^25 + 1", [](auto& a) { a.tokens = (1 << 25) + 1; a.qkv = at(1L << 42); a.q_out = at(1L << 43); a.k_out = at(1L << 44); });
  Q("qk tokens -1", [](auto& a) { a.tokens = -1; });
  Q("qk norm 3", [](auto& a) { a.norm = 3; });
  Q("qk rope -1", [](auto& a) { a.rope = -1; });
  Q("qk eps nan", [&](auto& a) { a.eps = nan; });
  Q("qk eps -1", [](auto& a) { a.eps = -1.f; });
  Q("qk slots without cache", [](auto& a) { a.has_cache = false; });
  Q("qk cache without slots", [](auto& a) { a.slots = nullptr; });
  Q("qk cache dtype", [](auto& a) { a.cache.dt = 2; });
  Q("qk cache heads", [](auto& a) { a.cache.kv_heads = 2; });
  Q("qk qkv NULL", [](auto& a) { a.qkv = nullptr; });
  Q("qk positions NULL", [](auto& a) { a.positions = nullptr; });
  Q("qk odd qkv", [](auto& a) { a.qkv = at(8 * MB + 2); });
  Q("qk odd slots", [](auto& a) { a.slots = reinterpret_cast<int*>(at(17 * 4 * MB + 1)); });
  Q("qk odd qw", [](auto& a) { a.qw = reinterpret_cast<float*>(at(20 * MB + 4)); });
  Q("qk odd kb", [](auto& a) { a.kb = reinterpret_cast<float*>(at(20 * MB + 8)); });
  Q("qk ld 1028", [](auto& a) { a.ld = 1028; });
  Q("qk ld short", [](auto& a) { a.ld = 15 * 64; });
  Q("qk ldq short", [](auto& a) { a.ldq = 7 * 64; });
  Q("qk ld 2^61", [](auto& a) { a.ld = 1L << 61; });
  Q("qk ldq 2^62", [](auto& a) { a.ldq = 1L << 62; });
  Q("qk ldk 2^62", [](auto& a) { a.ldk = 1L << 62; });
  Q("qk ldk short", [](auto& a) { a.ldk = 3 * 64; });
  Q("qk q_out over keys", [](auto& a) { a.q_out = at(8 * MB + 1024); a.ldq = a.ld; });
  Q("qk q_out another stride", [](auto& a) { a.q_out = const_cast<void*>(a.qkv); });
  Q("qk k_out over q_out", [](auto& a) { a.k_out = at(12 * MB + 512); });
  Q("qk rows over cache", [](auto& a) { a.q_out = a.cache.k; });
  say("qk base nan", [&] { QkArgs a = qk(); check_qk_norm_rope(a, nan); });
  say("qk base 0.5", [] { QkArgs a = qk(); check_qk_norm_rope(a, 0.5); });
  say("qk ok base 0.5 without rotation", [] { QkArgs a = qk(); a.rope = ROPE_NONE; check_qk_norm_rope(a, 0.5); });

  auto B = [&](const char* n, const std::function<void(BoundsArgs&)>& f) { on<BoundsArgs>(n, bounds(), check_page_bounds, f); };
  B("bounds ok", [](auto&) {});
  B("bounds ok all", [](auto& a) { a.add = nullptr; });
  B("bounds ok none", [](auto& a) { a.n = 0; a.table = a.lens = nullptr; a.bounds = nullptr; });
  B("bounds n -1", [](auto& a) { a.n = -1; });
  B("bounds max_add -1", [](auto& a) { a.max_add = -1; });
  B("bounds lens NULL", [](auto& a) { a.lens = nullptr; });
  B("bounds odd lens", [](auto& a) { a.lens = reinterpret_cast<int*>(at(36 * MB + 2)); });
  B("bounds odd", [](auto& a) { a.bounds = at(10 * MB + 4); });
  B("bounds over cache", [](auto& a) { a.bounds = a.cache.v; });
  say("bounds ok launch", [] {  // the pages of a sequence are dealt out in turns where all at once are too many
    BoundsArgs a = bounds();
    a.n = 1 << 20;
    a.width = 1 << 20;
    a.add = nullptr;
    check_page_bounds(a);
    if (a.per_seq != 8) throw Error(BAD_ARGUMENT, "per_seq " + std::to_string(a.per_seq));
  });
  B("bounds too many", [](auto& a) { a.n = 0x7fffffff; a.add = nullptr; });
  B("cache dtype -1", [](auto& a) { a.cache.dt = -1; });
  B("cache pages 0", [](auto& a) { a.cache.pages = 0; });
  B("cache pages 2^27", [](auto& a) { a.cache.pages = 1 << 27; });
  B("cache page 7", [](auto& a) { a.cache.page_size = 7; });
  B("cache kv_heads 0", [](auto& a) { a.cache.kv_heads = 0; });
  B("cache kv_heads 5000", [](auto& a) { a.cache.kv_heads = 5000; a.cache.page_stride = 5000 * 16 * 64; });
  B("cache stride short", [](auto& a) { a.cache.page_stride -= 8; });
  B("cache stride odd", [](auto& a) { a.cache.page_stride += 4; });
  B("cache stride negative", [](auto& a) { a.cache.page_stride = -a.cache.page_stride; });
  B("cache k NULL", [](auto& a) { a.cache.k = nullptr; });
  B("cache v odd", [](auto& a) { a.cache.v = at(MB + 8); });

  auto P = [&](const char* n, const std::function<void(PagedArgs&)>& f) { on<PagedArgs>(n, paged(), check_paged, f); };
  P("paged ok", [](auto&) {});
  P("paged ok none", [](auto& a) { a.n = 0; a.q = nullptr; a.out = nullptr; a.table = a.lens = nullptr; });
  P("paged ok max_len 0", [](auto& a) { a.max_len = 0; });
  P("paged ok strides", [](auto& a) { a.ldq = 520; a.ldo = 1024; });
  P("paged heads 6", [](auto& a) { a.heads = 6; });
  P("paged heads 0", [](auto& a) { a.heads = 0; });
  P("paged n -1", [](auto& a) { a.n = -1; });
  P("paged n 2^22", [](auto& a) { a.n = 1 << 22; });
  P("paged ok n 2^18", [](auto& a) { a.n = 1 << 18; a.q = at(1L << 36); a.out = at(1L << 37); a.table = ints(1L << 38); a.lens = ints(1L << 39); });
  P("paged n 2^18 + 1", [](auto& a) { a.n = (1 << 18) + 1; a.q = at(1L << 36); a.out = at(1L << 37); a.table = ints(1L << 38); a.lens = ints(1L << 39); });
  P("paged width 0", [](auto& a) { a.width = 0; });
  P("paged max_len -1", [](auto& a) { a.max_len = -1; });
  P("paged scale inf", [&](auto& a) { a.scale = inf; });
  P("paged q NULL", [](auto& a) { a.q = nullptr; });
  P("paged ldo 500", [](auto& a) { a.ldo = 500; });
  P("paged ldq 2^61", [](auto& a) { a.ldq = 1L << 61; });
  P("paged ldo 2^62", [](auto& a) { a.ldo = 1L << 62; });
  P("paged ldq 516", [](auto& a) { a.ldq = 516; });
  P("paged scale 3e38", [](auto& a) { a.scale = 3e38f; });
  P("paged width 2^27", [](auto& a) { a.width = 1 << 27; });
  P("paged odd table", [](auto& a) { a.table = reinterpret_cast<int*>(at(36 * MB + 2)); });
  P("paged out over table", [](auto& a) { a.out = const_cast<int*>(a.table); });
  P("paged out over q", [](auto& a) { a.out = const_cast<void*>(a.q); });
  P("paged out over cache", [](auto& a) { a.out = a.cache.k; });

  say("paged workspace odd", [] {
    PagedArgs a = paged();
    a.max_len = 1 << 20;
    a.width = 1 << 16;
    check_paged_attention(a, at(4), size_t(1) << 40);
  });
  say("paged workspace over q", [] {
    PagedArgs a = paged();
    a.max_len = 1 << 20;
    a.width = 1 << 16;
    check_paged_attention(a, a.q, size_t(1) << 40);
  });
  say("paged workspace small", [] {
    PagedArgs a = paged();
    a.max_len = 1 << 20;
    a.width = 1 << 16;
    check_paged_attention(a, at(4096 * MB), paged_attention_bytes(a.cache, a.n, a.heads, a.max_len) - 1);
  });

  auto S = [&](const char* n, const std::function<void(SparseArgs&)>& f) { on<SparseArgs>(n, sparse(), check_sparse, f); };
  S("sparse ok", [](auto&) {});
  S("sparse ok topk 2^20", [](auto& a) { a.topk = 1 << 20; });
  S("sparse ok topk 2^27", [](auto& a) { a.topk = 1 << 27; a.selected = ints(1L << 36); });
  S("sparse topk past 2^27", [](auto& a) { a.topk = (1 << 27) + 1; a.selected = ints(1L << 36); });
  S("sparse topk 2^31 - 1", [](auto& a) { a.topk = 0x7fffffff; a.selected = ints(1L << 36); });
  S("sparse ok max_len 2^31 - 1", [](auto& a) { a.at.max_len = 0x7fffffff; });
  S("sparse 2^30 pages", [](auto& a) { a.at.max_len = 0x7fffffff; a.at.width = 1 << 26; a.at.n = 4; a.at.table = ints(1L << 38); });
  S("sparse topk 0", [](auto& a) { a.topk = 0; });
  S("sparse scale 0", [](auto& a) { a.at.scale = 0.f; });
  S("sparse scale nan", [&](auto& a) { a.at.scale = nan; });
  S("sparse bounds NULL", [](auto& a) { a.bounds = nullptr; });
  S("sparse selected NULL", [](auto& a) { a.selected = nullptr; });
  S("sparse selected over cache", [](auto& a) { a.selected = static_cast<int*>(a.at.cache.k); });
  S("sparse selected over lens", [](auto& a) { a.selected = const_cast<int*>(a.at.lens); });
  S("sparse selected over bounds", [](auto& a) { a.selected = const_cast<int*>(static_cast<const int*>(a.bounds)); });
  S("sparse out over bounds", [](auto& a) { a.bounds = a.at.out; });
  S("sparse odd selected", [](auto& a) { a.selected = reinterpret_cast<int*>(at(13 * 4 * MB + 2)); });
  S("sparse heads 3", [](auto& a) { a.at.heads = 3; });
  say("sparse workspace small", [] {
    SparseArgs a = sparse();
    check_sparse_attention(a, at(4096 * MB), sparse_attention_bytes(a.at.cache, 3, 8, 300, 5) - 1);
  });
  say("sparse workspace over selected", [] {
    SparseArgs a = sparse();
    check_sparse_attention(a, a.selected, size_t(1) << 40);
  });
  say("paged ok max_len sizes no launch past the row", [] {
    for (int dt = 0; dt < 3; ++dt)
      for (int topk : {0, 1, 40, 5000}) {
        KvCache c = cache();
        c.dt = dt;
        for (int n : {1, 7, 300}) {
          size_t most = 0;
          for (int len = 1; len > 0 && len < 0x7fffffff / 3; len = len * 3 / 2 + 1) {  // workspaces grow with max_len
            const size_t bytes = paged_plan(c, n, 8, len, topk).bytes;
            if (bytes < most) throw Error(BAD_ARGUMENT, "a longer max_len takes a smaller workspace");
            most = bytes;
          }
        }
      }
    PagedArgs a = paged();
    a.max_len = 0x7fffffff;
    check_paged(a);
    if (a.max_len != 320) throw Error(BAD_ARGUMENT, "max_len " + std::to_string(a.max_len));
  });
  say("workspace ok", [] {
    paged_attention_bytes(cache(), 0, 8, 0);
    sparse_attention_bytes(cache(), 0, 8, 0, 1);
  });
  say("workspace heads 5", [] { paged_attention_bytes(cache(), 1, 5, 10); });
  say("workspace topk 2^31 - 1", [] { sparse_attention_bytes(cache(), 1, 8, 10, 0x7fffffff); });
  say("workspace topk 0", [] { sparse_attention_bytes(cache(), 1, 8, 10, 0); });
  say("workspace page 0", [] {
    KvCache c = cache();
    c.page_size = 0;
    sparse_attention_bytes(c, 1, 8, 10, 1);
  });

  // What the kernels check on the device.
  KvCache c = cache();
  c.shift = 4;
  std::printf("pages %d %d %d %d\n", page_ok(-1, 100), page_ok(0, 100), page_ok(99, 100), page_ok(100, 100));
  std::printf("slots %d %d %d %d %d\n", slot_ok(-1, c), slot_ok(0, c), slot_ok(1599, c), slot_ok(1600, c), slot_ok(0x7fffffff, c));
  std::printf("lengths %d %d %d %d %d\n", length_of(-5, 20, 4, 300), length_of(0, 20, 4, 300), length_of(299, 20, 4, 300),
              length_of(310, 20, 4, 1000), length_of(0x7fffffff, 1 << 22, 8, 0x7fffffff));
  c.page_stride = 1L << 31;
  std::printf("offsets %ld %ld\n", page_at(c, 99, 3), slot_at(c, 1599, 3));
  double f[32];
  rope_turns(ROPE_LINE, 10000.0, f);
  double worst = 0;
  for (int i = 0; i < 32; ++i)
    worst = std::fmax(worst, std::fabs(f[i] * 6.283185307179586 / std::pow(10000.0, -i / 32.0) - 1));
  std::printf("turns %d\n", worst < 1e-15 * 2);
  return 0;
}
