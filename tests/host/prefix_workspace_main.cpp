// What attention over a shared prefix writes into its workspace, by the kernels' own indexes, in the bytes that a caller is asked for: the
// parts of the items (block `id` of plan.blocks leaves plan.rows columns), then those of the tokens' own positions (block u of n *
// kv_heads * ceil(G / 16) * plan.own leaves min(G, 16) columns, those of heads that the last group has not among them).
// Prints "name OK" or "name ERR code message".
#include <algorithm>
#include <cstdio>
#include <string>

#include "../../splatting-rs_amd/csrc/cache.h"

using namespace splat;

namespace {

KvCache cache(int dt, int kv) {
  KvCache c;
  c.dt = dt;
  c.pages = 100;
  c.page_size = 16;
  c.shift = 4;
  c.kv_heads = kv;
  c.page_stride = kv * 16 * 64;
  return c;
}
PrefixArgs call(const KvCache& c, int n, int G, int groups, int shared, int own) {
  PrefixArgs a;
  a.cache = c;
  a.n = n;
  a.heads = c.kv_heads * G;
  a.groups = groups;
  a.max_shared = shared;
  a.max_own = own;
  return a;
}
void fits(const PrefixArgs& a, size_t bytes) {
  const PrefixPlan plan = prefix_plan(a);
  if (!plan.join) return;
  const int G = a.heads / a.cache.kv_heads;
  const size_t items = plan.parts + size_t(plan.blocks) * plan.rows * PART_HEAD * 4;
  const size_t blocks = size_t(a.n) * a.cache.kv_heads * ((G + 15) / 16) * plan.own, end = plan.own_parts + blocks * std::min(G, 16) * PART_HEAD * 4;
  const std::string what = "n " + std::to_string(a.n) + " groups " + std::to_string(a.groups) + " shared " + std::to_string(a.max_shared) + " own " +
                           std::to_string(a.max_own) + ": ";
  SPLAT_CHECK(plan.parts >= 16 + size_t(a.groups) * 16 && plan.parts % 16 == 0 && plan.own_parts % 16 == 0, BAD_ARGUMENT, what + "the groups' plan");
  SPLAT_CHECK(items <= plan.own_parts, BAD_ARGUMENT, what + "items' parts up to " + std::to_string(items) + " behind " + std::to_string(plan.own_parts));
  SPLAT_CHECK(end <= plan.bytes, BAD_ARGUMENT, what + std::to_string(end) + " bytes written, " + std::to_string(plan.bytes) + " in the plan");
  SPLAT_CHECK(end <= bytes, BAD_ARGUMENT, what + std::to_string(end) + " bytes written, " + std::to_string(bytes) + " asked for");
}

}  // namespace

int main() {
  for (int dt : {0, 1, 2})
    for (int kv : {1, 3})
      for (int G = 1; G <= 40; ++G) {
        const std::string name = "extent ok " + std::to_string(dt) + " " + std::to_string(kv) + " " + std::to_string(G);
        try {
          const KvCache c = cache(dt, kv);
          for (int n = 1; n < 3000; n += 1 + n / 3)
            for (int groups : {1, 3, 60, 1000}) {
              size_t before = 0;
              for (int shared : {0, 1, 33, 64, 100, 128, 500, 30000}) {
                size_t less = 0;
                for (int own : {0, 1, 64, 600, 8192, 16384, 24889, 1000000}) {
                  const size_t bytes = prefix_attention_bytes(c, n, kv * G, groups, shared, own);
                  SPLAT_CHECK(bytes >= less && bytes >= before, BAD_ARGUMENT, "less for a larger call");
                  less = bytes;
                  fits(call(c, n, G, groups, shared, own), bytes);
                  // every smaller call in the same workspace
                  for (int few : {1, 2, n / 2, n - 1})
                    if (few >= 1 && few <= n) fits(call(c, few, G, std::max(1, groups / 2), shared / 2, own / 2), bytes);
                }
                before = prefix_attention_bytes(c, n, kv * G, groups, shared, 0);
              }
            }
          std::printf("%s OK\n", name.c_str());
        } catch (const Error& e) {
          std::printf("%s ERR %d %s\n", name.c_str(), e.code, e.what());
        }
      }
  return 0;
}
