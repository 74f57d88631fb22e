// Host-only harness run under AddressSanitizer and UndefinedBehaviorSanitizer by
// tests/test_generation_oracle.py: the index arithmetic of the cache's kernels
// (femtochat_amd/csrc/cache_index.hpp), which lengths, counts, page tables and parents
// of any value reach on the device.
#include "../../femtochat_amd/csrc/cache_index.hpp"

#include <climits>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

static int failures = 0;
#define CHECK(cond)                                                                 \
  do {                                                                              \
    if (!(cond)) {                                                                  \
      std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond);        \
      if (++failures > 20) std::exit(1);                                            \
    }                                                                               \
  } while (0)

static std::mt19937 rng(7);
static int any(const std::vector<int>& v) { return v[rng() % v.size()]; }

// Every row that comes back lies in the pool, and rows of good tokens are distinct.
static void rows() {
  for (int round = 0; round < 300; ++round) {
    fc_cache_desc d;
    std::memset(&d, 0, sizeof d);
    d.D = 16, d.Hkv = 1 + rng() % 3, d.B = 1 + rng() % 4, d.layers = 1 + rng() % 2, d.type = 1 + rng() % 3;
    const bool table = rng() % 2;
    d.page_size = table ? 16 << rng() % 3 : 16 * (1 + rng() % 5);
    d.max_pages = table ? 1 + rng() % 4 : 0;
    d.pages = table ? 1 + rng() % 12 : d.B;
    fc::CacheGeom g;
    char msg[200];
    CHECK(fc::make_cache(&d, &g, msg, sizeof msg) == FC_OK);
    std::vector<int32_t> t(table ? d.B * d.max_pages : 0);
    for (auto& p : t) p = rng() % 3 ? (int)(rng() % d.pages) : any({-1, INT_MIN, INT_MAX, d.pages});
    const int64_t all = (int64_t)d.layers * d.pages * d.Hkv * d.page_size;
    for (int n = 0; n < 400; ++n) {
      const int length = any({0, 1, g.capacity - 1, g.capacity, g.capacity + 1, -1, INT_MIN, INT_MAX, (int)(rng() % g.capacity)});
      const int k = any({0, 1, 63, -1, INT_MAX, (int)(rng() % 100)});
      const int pos = fc::behind(g, length, k);
      CHECK(pos >= -1 && pos < g.capacity);
      if (length >= 0 && length <= g.capacity && k >= 0 && k < g.capacity - length) CHECK(pos == length + k);
      const int b = rng() % d.B, h = rng() % d.Hkv, layer = rng() % d.layers;
      const int64_t row = fc::cache_row(g, table ? t.data() : nullptr, layer, b, h, rng() % 4 ? pos : any({INT_MIN, INT_MAX, -5}));
      CHECK(row >= -1 && row < all);
      // a kernel's block of 16 keys lies within one page
      if (pos >= 0) {
        const int first = pos / 16 * 16;
        CHECK(first + 15 < g.capacity && fc::cache_place(g, table ? t.data() : nullptr, first) + 15 < g.page_size);
      }
    }
  }
}

// Slots: all tiles of all sequences are in exactly one, and there are at most share + B.
static void slots() {
  for (int round = 0; round < 2000; ++round) {
    const int B = 1 + rng() % 80, shares = 1 + rng() % 300, least = any({fc::kBegin + 1, 12, 16, 1 << 30}), N = 1 + rng() % 64;
    const int capacity = 16 * (1 + rng() % any({3, 100, 5000})), left = any({0, 1, 31, 512, INT_MAX / 2});
    int64_t total = 0;
    std::vector<fc::Span> spans;
    for (int b = 0; b < B; ++b) {
      const int length = rng() % 6 ? (int)(rng() % (capacity + 1)) : any({-3, INT_MIN, INT_MAX, capacity, capacity + 1});
      const int count = rng() % 6 ? (int)(rng() % (N + 1)) : any({-1, INT_MIN, INT_MAX});
      spans.push_back(fc::span_of(length, count, N, left, capacity));
      const fc::Span& s = spans.back();
      const int end = s.length + s.count < capacity ? s.length + s.count : capacity;
      CHECK(s.length >= 0 && s.length <= capacity && s.count >= 0 && s.count <= N && s.tiles >= 1 && s.first >= 0);
      if (s.count > 0) {
        CHECK((s.first + s.tiles) * fc::kTileKeys >= end);
        CHECK((s.first + s.tiles - 1) * fc::kTileKeys <= end);  // the last tile begins within the sequence, or at its capacity
        CHECK(s.first * (int64_t)fc::kTileKeys <= s.length);
        if (s.length > left) CHECK(s.first * fc::kTileKeys <= s.length - left);
      }
      total += fc::line_length(s.tiles);
    }
    // The line: every tile of every sequence is in one share, a share has at most two parts of
    // sequences that it does not hold whole, and no two parts share a slot.
    const int64_t each = fc::share_of(total, shares, least);
    CHECK(each >= least && each * shares >= total);
    std::vector<int> slots(2 * (size_t)shares, 0);
    int64_t start = 0;
    for (const auto& s : spans) {
      int upto = 0;
      for (int64_t x = start / each; x * each < start + fc::line_length(s.tiles); ++x) {
        CHECK(x < shares);
        const fc::Stretch st = fc::stretch_of(start, s.tiles, x, each);
        CHECK(st.first <= st.last && (st.first == upto || st.last == 0));
        CHECK(fc::line_quotient(start, each) == start / each);
        if (st.first >= st.last) {  // the room in front alone, in the first share that has any of it, or what fills the last four
          CHECK((x == start / each && upto == 0) || (upto == s.tiles && x * each >= start + s.tiles + fc::kBegin));
          continue;
        }
        upto = st.last;
        if (st.first == 0 && st.last == s.tiles) continue;
        const int64_t slot = fc::part_slot(start, x, each);
        CHECK(slot >= 0 && slot < 2 * shares && ++slots[slot] == 1);
        if (st.first > 0) CHECK(slot == 2 * x);  // (behind the first part, every second slot)
      }
      CHECK(upto == s.tiles);
      // The shares beside it hold nothing of it.
      const fc::Stretch before = fc::stretch_of(start, s.tiles, start / each - 1, each);
      const fc::Stretch behind = fc::stretch_of(start, s.tiles, (start + s.tiles + fc::kBegin - 1) / each + 1, each);
      CHECK(before.last == 0 && behind.first == s.tiles);
      start += fc::line_length(s.tiles);
    }
  }
  CHECK(fc::share_of((int64_t)1 << 50, 1, 12) == (int64_t)1 << 50);
}

// The mask of 32 keys against key by key.
static void masks() {
  for (int round = 0; round < 200000; ++round) {
    const int length = rng() % 5 ? (int)(rng() % 200) : (1 << 28) - (int)(rng() % 70), key0 = 4 * (int)(rng() % 80) + (length > 1000 ? length / 4 * 4 - 160 : 0);
    const int low = any({0, length, INT_MAX, (int)(rng() % (length + 1)), key0, key0 + 31, key0 + 32});
    const uint64_t sees = rng() % 4 == 0 ? ~0ull : ((uint64_t)rng() << 32 | rng());
    const uint32_t got = fc::seen_keys(key0, low, sees, length);
    for (int i = 0; i < 32; ++i) {
      const int key = key0 + i, node = key - length;
      const bool want = node < 0 ? key >= low : node < 64 && ((sees >> node) & 1) != 0;
      CHECK((((got >> i) & 1) != 0) == want);
    }
  }
}

int main() {
  rows();
  slots();
  masks();
  if (failures == 0) std::puts("ok");
  return failures != 0;
}
