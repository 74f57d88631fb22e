// Where a cache's tokens lie, and the checks of its descriptor: host and device
// code, also built alone by the host harness (tests/sanitize/cache_harness.cpp).
#pragma once

#include <stddef.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/femtochat_cache.h"
#include "attn_index.hpp"

namespace fc {

// A cache's sizes as the kernels take them.
struct CacheGeom {
  int D, Hkv, B, layers, pages, page_size, max_pages, type;
  int shift;     // log2(page_size) with a table
  int capacity;  // tokens of a sequence
};

FC_HD inline int cache_value_bytes(int type) { return type == FC_CACHE_BF16 ? 2 : 1; }

// The row (token of one head: D values, one scale) of a token at `position` of
// sequence b: layer's, page's and head's rows one after another.  -1 where the
// position is beyond the capacity (or below 0) or the page is not in the pool.
FC_HD inline int64_t cache_page(const CacheGeom& g, const int32_t* table, int b, int position) {
  if (position < 0 || position >= g.capacity) return -1;
  if (table == nullptr) return b;
  const int p = table[(int64_t)b * g.max_pages + (position >> g.shift)];
  return p >= 0 && p < g.pages ? p : -1;
}
FC_HD inline int cache_place(const CacheGeom& g, const int32_t* table, int position) {
  return table == nullptr ? position : position & (g.page_size - 1);
}
FC_HD inline int64_t cache_row(const CacheGeom& g, const int32_t* table, int layer, int b, int h, int position) {
  const int64_t p = cache_page(g, table, b, position);
  if (p < 0) return -1;
  return (((int64_t)layer * g.pages + p) * g.Hkv + h) * g.page_size + cache_place(g, table, position);
}

// The position of a sequence's token t behind `length`, -1 where it has none: a sum that stays in 32 bits.
FC_HD inline int behind(const CacheGeom& g, int length, int t) {
  const int n = imin(imax(length, 0), g.capacity);
  return t < 0 || t >= g.capacity - n ? -1 : n + t;
}

// ---- attention over the cache: which keys a workgroup takes, and what a node sees ----

constexpr int kTileKeys = 32;
constexpr int kMaxNodes = 64;

// Sequence b's tiles: from that of the first key any of its nodes sees to that of its last node.
struct Span {
  int length, count, first, tiles;
};
FC_HD inline Span span_of(int length, int count, int N, int left, int capacity) {
  Span s;
  s.length = imin(imax(length, 0), capacity);
  s.count = imin(imax(count, 0), N);
  const int end = imin(s.length + s.count, capacity);  // at most 2^28 + 64
  s.first = s.count == 0 ? 0 : imax(s.length - left, 0) / kTileKeys;
  s.tiles = s.count == 0 ? 1 : imax(1, (end + kTileKeys - 1) / kTileKeys - s.first);
  return s;
}
// A batch's work is shared out as one line, each sequence's tiles behind the ones before,
// in fours, as a workgroup's four waves take them, and with room in front for what beginning a
// sequence costs (in tiles): workgroup x takes the x-th stretch of the line.  One share, and with
// it one workgroup, may end a sequence, hold others whole and begin another.
constexpr int kBegin = 8;

FC_HD inline int line_length(int tiles) { return kBegin + (tiles + 3) / 4 * 4; }
// (a 64-bit quotient is some 150 instructions)
FC_HD inline int64_t line_quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
FC_HD inline int64_t share_of(int64_t total, int shares, int least) {
  const int64_t s = line_quotient(total + shares - 1, shares);
  return s > least ? s : least;
}
// The tiles (first, last: counted from the sequence's first) of a sequence at `start` of the
// line that share x holds: none where it has only the room in front, or nothing, of it.
struct Stretch {
  int first, last;
};
FC_HD inline Stretch stretch_of(int64_t start, int tiles, int64_t x, int64_t share) {
  const int64_t from = x * share - start, upto = from + share;
  Stretch s;
  s.first = from <= kBegin ? 0 : (int)(from - kBegin < tiles ? from - kBegin : tiles);
  s.last = upto <= kBegin ? 0 : (int)(upto - kBegin < tiles ? upto - kBegin : tiles);
  return s;
}
// Where share x leaves its part of a sequence: it has at most two parts that are not whole.
FC_HD inline int64_t part_slot(int64_t start, int64_t x, int64_t share) { return 2 * x + (start >= x * share ? 1 : 0); }

// Which of the 32 keys from key0 on are seen: those of the sequence (below length)
// from `low` on, and the nodes' behind it.
FC_HD inline uint32_t seen_keys(int key0, int low, uint64_t sees, int length) {
  const int node0 = key0 - length, from = low - key0;  // bits: the sequence's are below -node0
  const uint32_t upto = node0 >= 0 ? 0u : node0 <= -32 ? ~0u : (1u << -node0) - 1;
  const uint32_t behind_low = from <= 0 ? ~0u : from >= 32 ? 0u : ~0u << from;
  const uint32_t of_nodes = node0 >= 64 || node0 <= -32 ? 0u : (uint32_t)(node0 >= 0 ? sees >> node0 : sees << -node0);
  return (upto & behind_low) | of_nodes;
}

// Checks a descriptor; on failure a message and its status.
inline fc_status make_cache(const fc_cache_desc* d, CacheGeom* g, char* msg, size_t n) {
  const auto no = [&](const char* what, fc_status code = FC_ERR_INVALID_ARGUMENT) {
    snprintf(msg, n, "%s", what);
    return code;
  };
  if (d == nullptr) return no("descriptor is null");
  if (d->D <= 0 || d->D % 16 != 0 || d->D > 128) return no("head_dim must be a multiple of 16 up to 128");
  if (d->Hkv <= 0 || d->B <= 0 || d->layers <= 0 || d->pages <= 0 || d->page_size <= 0)
    return no("Hkv, B, layers, pages and page_size must be positive");
  if (d->type < FC_CACHE_BF16 || d->type > FC_CACHE_F8) return no("unknown cache type");
  if (d->page_size % 16 != 0) return no("page_size must be a multiple of 16");
  if (d->max_pages < 0) return no("max_pages must not be negative");
  if (d->max_pages > 0 && (d->page_size & (d->page_size - 1)) != 0) return no("pages of a table hold a power of two of tokens");
  if (d->max_pages == 0 && d->pages != d->B) return no("without a table every sequence has one page");
  // 64 sequences' tiles of 32 tokens sum up in 32 bits; a launch's grid has 65535 along y and z.
  const int64_t capacity = d->max_pages > 0 ? (int64_t)d->max_pages * d->page_size : d->page_size;
  if (capacity > (int64_t)1 << 28) return no("a sequence holds at most 2^28 tokens", FC_ERR_UNSUPPORTED);
  if (d->B > 65535 || d->layers > 65535) return no("at most 65535 sequences and layers", FC_ERR_UNSUPPORTED);
  if (d->Hkv > 1024) return no("at most 1024 KV heads", FC_ERR_UNSUPPORTED);
  g->D = d->D, g->Hkv = d->Hkv, g->B = d->B, g->layers = d->layers, g->pages = d->pages;
  g->page_size = d->page_size, g->max_pages = d->max_pages, g->type = d->type;
  g->shift = 0;
  while ((1 << g->shift) < d->page_size) ++g->shift;
  g->capacity = (int)capacity;
  return FC_OK;
}

}  // namespace fc
