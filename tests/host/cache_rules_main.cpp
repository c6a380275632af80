// Rules of the paged cache's calls that a table of single changes does not show, without a GPU. Prints "name OK" or
// "name ERR code message". The pointers are never followed.
#include <algorithm>
#include <cstdio>
#include <functional>
#include <string>

#include "../../splatting-rs_amd/csrc/cache.h"

using namespace splat;

namespace {

char* at(long offset) { return reinterpret_cast<char*>((1L << 40) + offset); }
int* ints(long offset) { return reinterpret_cast<int*>(at(offset)); }
float* floats(long offset) { return reinterpret_cast<float*>(at(offset)); }
constexpr long MB = 1L << 20;

KvCache cache(int dt = 1, int heads = 4) {  // 100 pages of 16 rows
  KvCache c;
  c.dt = dt;
  c.pages = 100;
  c.page_size = 16;
  c.kv_heads = heads;
  c.page_stride = heads * 16L * 64;
  c.k = at(0);
  c.v = at(64 * MB);
  return c;
}

void say(const std::string& name, const std::function<void()>& f) {
  try {
    f();
    std::printf("%s OK\n", name.c_str());
  } catch (const Error& e) {
    std::printf("%s ERR %d %s\n", name.c_str(), e.code, e.what());
  }
}

void expect(bool ok, const std::string& what) {
  if (!ok) throw Error(HIP_ERROR, what);
}

BoundsArgs bounds() {
  BoundsArgs a;
  a.cache = cache();
  a.n = 3;
  a.table = ints(200 * MB);
  a.width = 20;
  a.lens = ints(201 * MB);
  a.add = ints(202 * MB);
  a.max_add = 40;
  a.bounds = at(300 * MB);  // 100 * 4 * 128 values: 102400 bytes
  return a;
}

void bounds_overlaps() {
  const auto B = [](const std::string& n, const std::function<void(BoundsArgs&)>& f) {
    say("bounds " + n, [&] {
      BoundsArgs a = bounds();
      f(a);
      check_page_bounds(a);
      check_overlaps(a);
    });
  };
  B("ok", [](auto&) {});
  B("ok table behind", [](auto& a) { a.table = ints(300 * MB + 102400); });
  B("ok table before", [](auto& a) { a.table = ints(300 * MB - 240); });
  B("ok no add", [](auto& a) { a.add = nullptr; });
  B("over table", [](auto& a) { a.table = ints(300 * MB + 102396); });
  B("over table's end", [](auto& a) { a.table = ints(300 * MB - 236); });
  B("over lens", [](auto& a) { a.lens = ints(300 * MB + 64); });
  B("over add", [](auto& a) { a.add = ints(300 * MB - 8); });
}

// 10 rows of 8 + 4 heads of 64 bf16: q_out 10 rows of 1024 bytes, 1536 apart; pools of 100 pages of 8192 bytes.
QkArgs qk() {
  QkArgs a;
  a.dt = 1;
  a.tokens = 10;
  a.heads = 8;
  a.kv_heads = 4;
  a.qkv = at(200 * MB);
  a.ld = 16 * 64;
  a.norm = NORM_LAYER;
  a.eps = 1e-5f;
  a.rope = ROPE_GRID;
  a.positions = ints(300 * MB);
  a.q_out = at(400 * MB);
  a.ldq = 12 * 64;
  a.k_out = at(500 * MB);
  a.ldk = 4 * 64;
  a.has_cache = true;
  a.cache = cache();
  a.slots = ints(600 * MB);
  a.qw = floats(700 * MB);
  a.qb = floats(701 * MB);
  a.kw = floats(702 * MB);
  a.kb = floats(703 * MB);
  return a;
}

void qk_overlaps() {
  const auto Q = [](const std::string& n, const std::function<void(QkArgs&)>& f) {
    say("qk " + n, [&] {
      QkArgs a = qk();
      f(a);
      check_qk_norm_rope(a, 100.0);
      check_overlaps(a);
    });
  };
  Q("ok", [](auto&) {});
  Q("ok no weights", [](auto& a) { a.qw = a.qb = a.kw = a.kb = nullptr; });
  Q("ok one weight for both", [](auto& a) { a.kw = a.qw; a.kb = a.qb; });
  Q("ok nothing", [](auto& a) { a.tokens = 0; a.positions = static_cast<const int*>(a.q_out); });
  Q("ok weights between rows", [](auto& a) { a.qw = floats(400 * MB + 1024); a.kw = floats(400 * MB + 1536 + 1280); });
  Q("ok slots behind the last row", [](auto& a) { a.slots = ints(400 * MB + 9 * 1536 + 1024); });
  Q("ok slots before k_out", [](auto& a) { a.slots = ints(500 * MB - 40); });
  Q("ok weights in a page's gap", [](auto& a) { a.cache.page_stride += 128; a.kb = floats(7 * (8192 + 256) + 8192); });
  Q("ok positions unread", [](auto& a) { a.rope = ROPE_NONE; a.positions = static_cast<const int*>(a.q_out); });
  Q("ok weights unread", [](auto& a) { a.norm = NORM_NONE; a.qw = static_cast<const float*>(a.q_out); });
  Q("q_out over positions", [](auto& a) { a.positions = ints(400 * MB - 76); });
  Q("q_out over the grid's second positions", [](auto& a) { a.positions = ints(400 * MB - 44); });
  Q("q_out over slots", [](auto& a) { a.slots = ints(400 * MB + 9 * 1536 + 1020); });
  Q("q_out over qw", [](auto& a) { a.qw = floats(400 * MB + 1024 - 16); });
  Q("q_out over qb", [](auto& a) { a.qb = floats(400 * MB + 3 * 1536 - 128); });
  Q("q_out over kw", [](auto& a) { a.kw = floats(400 * MB + 9 * 1536); });
  Q("q_out over kb", [](auto& a) { a.kb = floats(400 * MB - 240); });
  Q("k_out over positions", [](auto& a) { a.positions = ints(500 * MB + 100); });
  Q("k_out over slots", [](auto& a) { a.slots = ints(500 * MB + 5116); });
  Q("k_out over kw", [](auto& a) { a.kw = floats(500 * MB + 512); });
  Q("keys over positions", [](auto& a) { a.positions = ints(50 * 8192); });
  Q("keys over slots", [](auto& a) { a.slots = ints(100 * 8192 - 4); });
  Q("values over slots", [](auto& a) { a.slots = ints(64 * MB - 36); });
  Q("values over kb", [](auto& a) { a.kb = floats(64 * MB + 99 * 8192); });
}

// A workspace that is sized for the largest batch, length and selection serves every smaller call.
void workspaces() {
  for (int dt = 0; dt < 3; ++dt)
    for (int kv : {1, 2, 12, 300})
      for (int group : {1, 8, 20})
        for (int topk : {0, 1, 60, 100, 3000})
          say("workspace ok " + std::to_string(dt) + " " + std::to_string(kv) + " " + std::to_string(group) + " " + std::to_string(topk), [&] {
            const KvCache c = cache(dt, kv);
            const auto bytes = [&](int n, int len, int k) {
              return topk ? sparse_attention_bytes(c, n, kv * group, len, k) : paged_attention_bytes(c, n, kv * group, len);
            };
            for (int len : {1, 440, 500, 900, 1500, 2000, 4000, 4200, 30000}) {
              size_t most = 0;
              for (int n = 1; n <= 1500 && long(n) * kv * group < 1 << 21; n += 1 + n / 60) {
                const size_t b = bytes(n, len, topk);
                expect(b >= most, "less for " + std::to_string(n) + " sequences of " + std::to_string(len));
                expect(bytes(n, len + 1, topk) >= b, "less for a longer max_len");
                expect(!topk || bytes(n, len, topk + 1) >= b, "less for more pages");
                most = b;
              }
            }
          });
  for (int topk : {0, 100})
    for (int n : {1, 3, 85, 86, 87, 200})
      say("workspace ok of a larger batch " + std::to_string(topk) + " " + std::to_string(n), [&] {
        SparseArgs s;
        PagedArgs& a = s.at;
        a.cache = cache(1, 12);
        a.n = n;
        a.heads = 12;
        a.q = at(200 * MB);
        a.ldq = a.ldo = 12 * 64;
        a.table = ints(300 * MB);
        a.width = 300;
        a.lens = ints(400 * MB);
        a.max_len = topk ? 4000 : 2000;
        a.scale = 0.125f;
        a.out = at(500 * MB);
        s.bounds = at(600 * MB);
        s.topk = topk;
        s.selected = ints(700 * MB);
        if (topk) check_sparse_attention(s, at(800 * MB), sparse_attention_bytes(a.cache, 200, 12, a.max_len, topk));
        else check_paged_attention(a, at(800 * MB), paged_attention_bytes(a.cache, 200, 12, a.max_len));
      });
  say("workspace ok none where no parts are left", [] {
    PagedArgs a;
    a.cache = cache(1, 12);
    a.n = 200;
    a.heads = 12;
    a.q = at(200 * MB);
    a.ldq = a.ldo = 12 * 64;
    a.table = ints(300 * MB);
    a.width = 300;
    a.lens = ints(400 * MB);
    a.max_len = 2000;
    a.out = at(500 * MB);
    check_paged_attention(a, nullptr, 0);
  });
}

}  // namespace

int main() {
  workspaces();
  bounds_overlaps();
  qk_overlaps();
  return 0;
}
