// The argument checks of the calls on a cache's pages and of attention over a shared prefix, without a GPU: each named call
// starts from one that is accepted and changes one thing. Prints "name OK" or "name ERR code message". The pointers are never followed.
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
constexpr size_t LOTS = size_t(1) << 40;

PagesArgs pages() {
  PagesArgs a;
  a.n = 10;
  a.page_size = 16;
  a.pages = 100;
  a.pool = ints(0);
  a.pool_size = 100;
  a.used = ints(1024);
  a.table = ints(2048);
  a.width = 8;
  a.lens = ints(4096);
  a.status = ints(8192);
  return a;
}
ForkArgs forks() {
  ForkArgs a;
  a.at = pages();
  a.parents = ints(16384);
  a.keep = ints(16448);
  a.lens_out = ints(16512);
  a.src = ints(16576);
  a.dst = ints(16640);
  a.rows = ints(16704);
  a.used_out = ints(16768);
  return a;
}
FreeArgs frees() {
  FreeArgs a;
  a.at = pages();
  a.keep = ints(16384);
  a.lens_out = ints(16448);
  a.used_out = ints(16512);
  return a;
}
CompactArgs compacts() {
  CompactArgs a;
  a.at = pages();
  a.table_out = ints(16384);
  a.pool_out = ints(32768);
  a.src = ints(65536);
  a.dst = ints(81920);
  a.cap = 50;
  a.count = ints(98304);
  return a;
}
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
CopyArgs copies() {
  CopyArgs a;
  a.cache = cache();
  a.layers = 3;
  a.has_bounds = true;
  for (int i = 0; i < 3; ++i) {
    a.k[i] = at(i * 4 * MB);
    a.v[i] = at(i * 4 * MB + MB);
    a.bounds[i] = at(i * 4 * MB + 2 * MB);
  }
  a.n = 20;
  a.src = ints(16 * MB);
  a.dst = ints(16 * MB + 80);
  a.rows = ints(16 * MB + 160);
  a.count = ints(16 * MB + 240);
  return a;
}
PrefixArgs prefix() {
  PrefixArgs a;
  a.cache = cache();
  a.n = 30;
  a.heads = 8;
  a.q = at(8 * MB);
  a.ldq = a.ldo = 8 * 64;
  a.starts = ints(9 * MB);
  a.groups = 3;
  a.prefix = ints(10 * MB);
  a.prefix_width = 20;
  a.shared = ints(11 * MB);
  a.max_shared = 300;
  a.table = ints(12 * MB);
  a.width = 30;
  a.lens = ints(13 * MB);
  a.max_own = 100;
  a.scale = 0.125f;
  a.out = at(14 * MB);
  return a;
}

void say(const std::string& name, const std::function<void()>& f) {
  try {
    f();
    std::printf("%s OK\n", name.c_str());
  } catch (const Error& e) {
    std::printf("%s ERR %d %s\n", name.c_str(), e.code, e.what());
  }
}
template <typename A> void on(const char* name, A a, const std::function<void(A&)>& check, const std::function<void(A&)>& change) {
  say(name, [&] {
    change(a);
    check(a);
  });
}
void expect(bool ok, const std::string& what) {
  if (!ok) throw Error(1, what);
}

// A workspace serves every smaller call, and holds what the launch takes.
void workspaces() {
  say("workspace ok pages", [] {
    size_t most = 0;
    for (long p = 1; p <= 1 << 28; p += 1 + p / 7) {
      const size_t b = pages_bytes(int(p));
      const PagesPlan plan = pages_plan(int(p));
      expect(b >= most && b == plan.bytes, "less for more pages");
      expect(plan.second >= size_t(p) && plan.before >= plan.second + p && plan.counts >= plan.before + size_t(plan.words) * 4 &&
                 plan.head >= plan.counts + size_t(plan.chunks) * 8 && b >= plan.head + 16 && plan.words * 4 >= p && plan.chunks * PAGE_CHUNK >= plan.words,
             "a map that does not fit");
      expect(plan.second % 16 == 0 && plan.before % 16 == 0 && plan.counts % 16 == 0 && plan.head % 16 == 0, "alignment");
      most = b;
    }
  });
  say("workspace no pages", [] { pages_bytes(0); });
  say("workspace too many pages", [] { pages_bytes((1 << 28) + 1); });
  for (int dt : {0, 1, 2})
    for (int kv : {1, 4, 12})
      for (int G : {1, 3, 20})
        say("workspace ok prefix " + std::to_string(dt) + " " + std::to_string(kv) + " " + std::to_string(G), [&] {
          KvCache c = cache();
          c.dt = dt;
          c.kv_heads = kv;
          c.page_stride = kv * 16 * 64;
          for (int n = 1; n < 3000; n += 1 + n / 4)
            for (int groups : {1, 2, 7, 50, 1000})
              for (int shared : {0, 1, 33, 500, 5000, 30000})
                for (int own : {0, 1, 100, 40000}) {
                  PrefixArgs a = prefix();
                  a.cache = c;
                  a.n = n;
                  a.heads = kv * G;
                  a.groups = groups;
                  a.max_shared = shared;
                  a.max_own = own;
                  const size_t b = prefix_attention_bytes(c, n, kv * G, groups, shared, own);
                  const PrefixPlan plan = prefix_plan(a);
                  expect(plan.bytes <= b, "a plan of " + std::to_string(plan.bytes) + " bytes in " + std::to_string(b));
                  const long items = (long(n) * G / plan.rows + std::min(groups, n)) * kv;
                  expect(plan.blocks >= items, "an item without a block");
                  expect(plan.join || plan.blocks == items, "parts without a join");
                  expect(prefix_attention_bytes(c, n + 1, kv * G, groups, shared, own) >= b && prefix_attention_bytes(c, n, kv * G, groups + 1, shared, own) >= b &&
                             prefix_attention_bytes(c, n, kv * G, groups, shared + 1, own) >= b && prefix_attention_bytes(c, n, kv * G, groups, shared, own + 1) >= b,
                         "less for a larger call");
                }
        });
  say("workspace heads 3 on 4", [] { prefix_attention_bytes(cache(), 1, 3, 1, 10, 0); });
  say("workspace rows 2^21 + 8", [] { prefix_attention_bytes(cache(), (1 << 18) + 1, 8, 1, 10, 0); });
  say("workspace groups 65537", [] { prefix_attention_bytes(cache(), 10, 8, 65537, 10, 0); });
  say("workspace shared -1", [] { prefix_attention_bytes(cache(), 10, 8, 1, -1, 0); });
  say("workspace own -1", [] { prefix_attention_bytes(cache(), 10, 8, 1, 1, -1); });
}

template <typename A> void table_cases(const std::string& what, const std::function<A()>& make, const std::function<void(A&)>& check) {
  auto T = [&](const char* n, const std::function<void(PagesArgs&)>& f) { on<A>((what + " " + n).c_str(), make(), check, [&](A& a) { f(a.at); }); };
  T("ok", [](auto&) {});
  T("ok no pool", [](auto& a) { a.pool_size = 0; a.pool = nullptr; });
  T("n -1", [](auto& a) { a.n = -1; });
  T("n 65537", [](auto& a) { a.n = 65537; });
  T("page 4", [](auto& a) { a.page_size = 4; });
  T("page 24", [](auto& a) { a.page_size = 24; });
  T("page 0", [](auto& a) { a.page_size = 0; });
  T("pages 0", [](auto& a) { a.pages = 0; });
  T("pages past 2^31 positions", [](auto& a) { a.pages = 1 << 27; });
  T("width 0", [](auto& a) { a.width = 0; });
  T("width 2^27", [](auto& a) { a.width = 1 << 27; });
  T("pool -1", [](auto& a) { a.pool_size = -1; });
  T("pool NULL", [](auto& a) { a.pool = nullptr; });
  T("used NULL", [](auto& a) { a.used = nullptr; });
  T("table NULL", [](auto& a) { a.table = nullptr; });
  T("lens NULL", [](auto& a) { a.lens = nullptr; });
  T("status NULL", [](auto& a) { a.status = nullptr; });
  T("lens odd", [](auto& a) { a.lens = reinterpret_cast<int*>(at(4097)); });
  T("status over lens", [](auto& a) { a.status = const_cast<int*>(a.lens) + 3; });
  T("status over table", [](auto& a) { a.status = a.table + 79; });
  T("status over used", [](auto& a) { a.status = const_cast<int*>(a.used); });
}

}  // namespace

int main() {
  const float inf = std::numeric_limits<float>::infinity();
  table_cases<ForkArgs>("fork", forks, check_fork_pages);
  auto F = [&](const char* n, const std::function<void(ForkArgs&)>& f) { on<ForkArgs>(n, forks(), check_fork_pages, f); };
  F("fork ok no keep", [](auto& a) { a.keep = nullptr; });
  F("fork ok lens over lens", [](auto& a) { a.lens_out = const_cast<int*>(a.at.lens); a.used_out = const_cast<int*>(a.at.used); });
  F("fork ok no rows", [](auto& a) { a.at.n = 0; a.parents = a.keep = nullptr; a.lens_out = a.src = a.dst = a.rows = a.at.table = nullptr; a.at.lens = nullptr; });
  F("fork parents NULL", [](auto& a) { a.parents = nullptr; });
  F("fork lens_out NULL", [](auto& a) { a.lens_out = nullptr; });
  F("fork src NULL", [](auto& a) { a.src = nullptr; });
  F("fork dst NULL", [](auto& a) { a.dst = nullptr; });
  F("fork rows NULL", [](auto& a) { a.rows = nullptr; });
  F("fork used_out NULL", [](auto& a) { a.used_out = nullptr; });
  F("fork lens_out into lens", [](auto& a) { a.lens_out = const_cast<int*>(a.at.lens) + 1; });
  F("fork lens_out over keep", [](auto& a) { a.lens_out = const_cast<int*>(a.keep); });
  F("fork table over the pool", [](auto& a) { a.at.table = a.at.pool; });
  F("fork src over parents", [](auto& a) { a.src = const_cast<int*>(a.parents); });
  F("fork src over dst", [](auto& a) { a.src = a.dst + 9; });
  F("fork rows over lens", [](auto& a) { a.rows = const_cast<int*>(a.at.lens); });
  F("fork used_out into lens_out", [](auto& a) { a.used_out = a.lens_out + 2; });
  F("fork keep odd", [](auto& a) { a.keep = reinterpret_cast<int*>(at(16449)); });

  const auto free_ = [](FreeArgs& a) { check_free_pages(a, at(MB), pages_bytes(a.at.pages > 0 ? a.at.pages : 1)); };
  table_cases<FreeArgs>("free", frees, free_);
  auto G = [&](const char* n, const std::function<void(FreeArgs&)>& f) { on<FreeArgs>(n, frees(), free_, f); };
  G("free ok in place", [](auto& a) { a.lens_out = const_cast<int*>(a.at.lens); a.used_out = const_cast<int*>(a.at.used); });
  G("free ok over keep", [](auto& a) { a.lens_out = const_cast<int*>(a.keep); });
  G("free ok no rows", [](auto& a) { a.at.n = 0; a.keep = nullptr; a.lens_out = a.at.table = nullptr; a.at.lens = nullptr; });
  G("free keep NULL", [](auto& a) { a.keep = nullptr; });
  G("free lens_out NULL", [](auto& a) { a.lens_out = nullptr; });
  G("free used_out NULL", [](auto& a) { a.used_out = nullptr; });
  G("free pool over table", [](auto& a) { a.at.pool = a.at.table; });
  G("free pool over lens", [](auto& a) { a.at.pool = const_cast<int*>(a.at.lens); });
  G("free lens_out over table", [](auto& a) { a.lens_out = a.at.table; });
  G("free lens_out into keep", [](auto& a) { a.lens_out = const_cast<int*>(a.keep) + 1; });
  G("free used_out over the pool", [](auto& a) { a.used_out = a.at.pool + 99; });
  on<FreeArgs>("free no workspace", frees(), [](auto& a) { check_free_pages(a, nullptr, LOTS); }, [](auto&) {});
  on<FreeArgs>("free workspace small", frees(), [](auto& a) { check_free_pages(a, at(MB), pages_bytes(100) - 1); }, [](auto&) {});
  on<FreeArgs>("free workspace odd", frees(), [](auto& a) { check_free_pages(a, at(MB + 8), LOTS); }, [](auto&) {});
  on<FreeArgs>("free workspace over the table", frees(), [](auto& a) { check_free_pages(a, at(2048), LOTS); }, [](auto&) {});
  on<FreeArgs>("free workspace over the pool", frees(), [](auto& a) { check_free_pages(a, at(16), LOTS); }, [](auto&) {});

  const auto compact = [](CompactArgs& a) { check_compact_pages(a, at(MB), pages_bytes(a.at.pages > 0 ? a.at.pages : 1)); };
  table_cases<CompactArgs>("compact", compacts, compact);
  auto C = [&](const char* n, const std::function<void(CompactArgs&)>& f) { on<CompactArgs>(n, compacts(), compact, f); };
  C("compact ok in place", [](auto& a) { a.table_out = a.at.table; a.pool_out = a.at.pool; });
  C("compact ok no moves", [](auto& a) { a.cap = 0; a.src = a.dst = nullptr; });
  C("compact ok no rows", [](auto& a) { a.at.n = 0; a.table_out = a.at.table = nullptr; a.at.lens = nullptr; });
  C("compact cap -1", [](auto& a) { a.cap = -1; });
  C("compact table_out NULL", [](auto& a) { a.table_out = nullptr; });
  C("compact pool_out NULL", [](auto& a) { a.pool_out = nullptr; });
  C("compact src NULL", [](auto& a) { a.src = nullptr; });
  C("compact dst NULL", [](auto& a) { a.dst = nullptr; });
  C("compact count NULL", [](auto& a) { a.count = nullptr; });
  C("compact table_out into table", [](auto& a) { a.table_out = a.at.table + 8; });
  C("compact pool_out into pool", [](auto& a) { a.pool_out = a.at.pool + 1; });
  C("compact table_out over the pool", [](auto& a) { a.table_out = a.at.pool; });
  C("compact src over dst", [](auto& a) { a.src = a.dst + 49; });
  C("compact src over lens", [](auto& a) { a.src = const_cast<int*>(a.at.lens); });
  C("compact count over src", [](auto& a) { a.count = a.src; });
  on<CompactArgs>("compact workspace over dst", compacts(), [](auto& a) { check_compact_pages(a, a.dst, LOTS); }, [](auto&) {});
  on<CompactArgs>("compact no workspace", compacts(), [](auto& a) { check_compact_pages(a, nullptr, 0); }, [](auto&) {});

  auto P = [&](const char* n, const std::function<void(CopyArgs&)>& f) { on<CopyArgs>(n, copies(), check_copy_pages, f); };
  P("copy ok", [](auto&) {});
  P("copy ok no bounds", [](auto& a) { a.has_bounds = false; a.bounds[0] = nullptr; });
  P("copy ok all rows, no count", [](auto& a) { a.rows = a.count = nullptr; });
  P("copy ok no pairs", [](auto& a) { a.n = 0; a.src = a.dst = a.rows = a.count = nullptr; });
  P("copy ok no layers", [](auto& a) { a.layers = 0; });
  P("copy ok keys and values in turn", [](auto& a) { a.cache.page_stride = 2 * 4096; a.layers = 1; a.v[0] = at(8192); });
  P("copy layers 65", [](auto& a) { a.layers = 65; });
  P("copy layers -1", [](auto& a) { a.layers = -1; });
  P("copy n -1", [](auto& a) { a.n = -1; });
  P("copy src NULL", [](auto& a) { a.src = nullptr; });
  P("copy dst NULL", [](auto& a) { a.dst = nullptr; });
  P("copy rows odd", [](auto& a) { a.rows = reinterpret_cast<int*>(at(16 * MB + 161)); });
  P("copy k NULL", [](auto& a) { a.k[2] = nullptr; });
  P("copy v odd", [](auto& a) { a.v[1] = at(8); });
  P("copy bounds NULL", [](auto& a) { a.bounds[1] = nullptr; });
  P("copy bounds odd", [](auto& a) { a.bounds[1] = at(6 * MB + 8); });
  P("copy stride short", [](auto& a) { a.cache.page_stride = 4096 - 8; });
  P("copy dtype", [](auto& a) { a.cache.dt = 3; });
  P("copy k over v", [](auto& a) { a.v[0] = a.k[0]; });
  P("copy k into v", [](auto& a) { a.v[0] = at(819200 - 16); });
  P("copy k of two layers", [](auto& a) { a.k[2] = a.k[0]; });
  P("copy bounds over keys", [](auto& a) { a.bounds[2] = a.k[0]; });
  P("copy bounds of two layers", [](auto& a) { a.bounds[2] = a.bounds[1]; });
  P("copy pool over src", [](auto& a) { a.src = reinterpret_cast<const int*>(at(4)); });
  P("copy bounds over dst", [](auto& a) { a.dst = reinterpret_cast<const int*>(at(2 * MB + 64)); });
  P("copy too much", [](auto& a) {
    a.n = 0x7fffffff;
    a.src = ints(1L << 55);
    a.dst = ints(1L << 56);
    a.rows = a.count = nullptr;
    a.cache.dt = 0;
    a.cache.kv_heads = 4096;
    a.cache.page_size = 256;
    a.cache.page_stride = 4096L * 256 * 64;
    a.layers = 64;
    for (int i = 0; i < 64; ++i) a.k[i] = at((1L + 3 * i) << 44), a.v[i] = at((2L + 3 * i) << 44), a.bounds[i] = at((3L + 3 * i) << 44);
  });

  const auto attend = [](PrefixArgs& a) { check_prefix_attention(a, at(4096 * MB), LOTS); };
  auto A = [&](const char* n, const std::function<void(PrefixArgs&)>& f) { on<PrefixArgs>(n, prefix(), attend, f); };
  A("prefix ok", [](auto&) {});
  A("prefix ok no table", [](auto& a) { a.table = nullptr; a.width = 0; });
  A("prefix ok no table and lens", [](auto& a) { a.table = a.lens = nullptr; a.width = 0; });
  A("prefix ok no tokens", [](auto& a) { a.n = 0; a.q = nullptr; a.out = nullptr; a.starts = a.prefix = a.shared = a.table = a.lens = nullptr; });
  A("prefix ok no groups", [](auto& a) { a.groups = 0; a.starts = a.prefix = a.shared = nullptr; });
  A("prefix ok table is prefix", [](auto& a) { a.table = a.prefix + 100; });
  A("prefix ok rows apart", [](auto& a) { a.ldq = 520; a.ldo = 1024; });
  A("prefix heads 6 on 4", [](auto& a) { a.heads = 6; });
  A("prefix heads 0", [](auto& a) { a.heads = 0; });
  A("prefix n -1", [](auto& a) { a.n = -1; });
  A("prefix too many rows", [](auto& a) { a.n = 1 << 19; });
  A("prefix groups -1", [](auto& a) { a.groups = -1; });
  A("prefix groups 65537", [](auto& a) { a.groups = 65537; });
  A("prefix width 0", [](auto& a) { a.prefix_width = 0; });
  A("prefix table width 0", [](auto& a) { a.width = 0; });
  A("prefix table width 2^27", [](auto& a) { a.width = 1 << 27; });
  A("prefix table without lens", [](auto& a) { a.lens = nullptr; });
  A("prefix max_shared -1", [](auto& a) { a.max_shared = -1; });
  A("prefix max_own -1", [](auto& a) { a.max_own = -1; });
  A("prefix scale inf", [&](auto& a) { a.scale = inf; });
  A("prefix scale nan", [](auto& a) { a.scale = std::nanf(""); });
  A("prefix scale huge", [](auto& a) { a.scale = 3e38f; });
  A("prefix q NULL", [](auto& a) { a.q = nullptr; });
  A("prefix out NULL", [](auto& a) { a.out = nullptr; });
  A("prefix starts NULL", [](auto& a) { a.starts = nullptr; });
  A("prefix row NULL", [](auto& a) { a.prefix = nullptr; });
  A("prefix shared NULL", [](auto& a) { a.shared = nullptr; });
  A("prefix q odd", [](auto& a) { a.q = at(8 * MB + 8); });
  A("prefix ldq 508", [](auto& a) { a.ldq = 508; });
  A("prefix ldq 504", [](auto& a) { a.ldq = 504; });
  A("prefix ldo 2^32", [](auto& a) { a.ldo = 1L << 32; });
  A("prefix out over q", [](auto& a) { a.out = const_cast<void*>(a.q); });
  A("prefix out over the cache", [](auto& a) { a.out = at(16); });
  A("prefix out over starts", [](auto& a) { a.out = at(9 * MB); });
  A("prefix out over the prefix", [](auto& a) { a.out = at(10 * MB + 16); });
  A("prefix out over the table", [](auto& a) { a.out = at(12 * MB); });
  A("prefix out over lens", [](auto& a) { a.out = at(13 * MB); });
  A("prefix starts odd", [](auto& a) { a.starts = reinterpret_cast<int*>(at(9 * MB + 2)); });
  A("prefix cache k NULL", [](auto& a) { a.cache.k = nullptr; });
  const size_t need = prefix_attention_bytes(cache(), 30, 8, 3, 300, 100);
  on<PrefixArgs>("prefix ok workspace exact", prefix(), [&](auto& a) { check_prefix_attention(a, at(4096 * MB), need); }, [](auto&) {});
  on<PrefixArgs>("prefix workspace short", prefix(), [&](auto& a) { check_prefix_attention(a, at(4096 * MB), need - 1); }, [](auto&) {});
  on<PrefixArgs>("prefix workspace NULL", prefix(), [&](auto& a) { check_prefix_attention(a, nullptr, need); }, [](auto&) {});
  on<PrefixArgs>("prefix workspace odd", prefix(), [&](auto& a) { check_prefix_attention(a, at(4096 * MB + 8), LOTS); }, [](auto&) {});
  on<PrefixArgs>("prefix workspace over q", prefix(), [&](auto& a) { check_prefix_attention(a, at(8 * MB), LOTS); }, [](auto&) {});
  on<PrefixArgs>("prefix workspace over lens", prefix(), [&](auto& a) { check_prefix_attention(a, at(13 * MB + 64), LOTS); }, [](auto&) {});
  on<PrefixArgs>("prefix workspace over the cache", prefix(), [&](auto& a) { check_prefix_attention(a, at(64), LOTS); }, [](auto&) {});
  say("cut shared and own", [&] {
    PrefixArgs a = prefix();
    a.max_shared = a.max_own = 0x7fffffff;
    attend(a);
    std::printf("cuts %d %d\n", a.max_shared, a.max_own);
  });
  workspaces();
  return 0;
}
