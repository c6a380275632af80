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

}  // namespace

int main() {
  bounds_overlaps();
  return 0;
}
