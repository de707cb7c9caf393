// Whether two strided sets of rows share memory (host code).  A call must not
// write rows that other threads of it still read, or write twice; the slices of
// a projection that these operators take are strided, so the ranges of their
// addresses say too little.
#pragma once

#include <algorithm>
#include <cstdint>
#include <vector>

namespace fkv {

// `tokens` x `heads` pieces of `bytes` bytes; strides in bytes, not negative, 0 along an axis of one entry.
struct RowSet {
  uintptr_t base;
  int64_t tokens, heads, token, head, bytes;
  bool same_place(const RowSet &o) const { return base == o.base && token == o.token && head == o.head; }
};

// Of two sets of the same shape.
inline bool rows_share_memory(RowSet a, RowSet b) {
  if (a.tokens <= 0 || a.heads <= 0 || a.bytes <= 0) return false;
  auto end = [](const RowSet &r) { return r.base + (r.tokens - 1) * r.token + (r.heads - 1) * r.head + r.bytes; };
  if (end(a) <= b.base || end(b) <= a.base) return false;
  if (a.token == b.token && a.head == b.head) {
    // Pieces differ by apart + u * token + w * head for all |u| < tokens, |w| < heads: for each w (of the shorter
    // axis) the u that brings it next to 0, from either side.
    if (a.heads > a.tokens) std::swap(a.tokens, a.heads), std::swap(a.token, a.head);
    const int64_t apart = (int64_t)(b.base - a.base), most = a.tokens - 1;
    for (int64_t w = 1 - a.heads; w < a.heads; ++w) {
      const int64_t x = apart + w * a.head, u = a.token ? -x / a.token : 0;
      for (int64_t k = u - 1; k <= u + 1; ++k) {
        const int64_t d = x + std::clamp(k, -most, most) * a.token;
        if (d > -a.bytes && d < a.bytes) return true;
      }
    }
    return false;
  }
  // Unlike strides in one range of addresses: piece by piece; beyond 2^24 of them taken as shared.
  if (a.tokens > ((int64_t)1 << 24) / a.heads) return true;
  std::vector<uintptr_t> at(a.tokens * a.heads);
  for (int64_t i = 0; i < a.tokens; ++i)
    for (int64_t h = 0; h < a.heads; ++h) at[i * a.heads + h] = a.base + i * a.token + h * a.head;
  std::sort(at.begin(), at.end());
  for (int64_t i = 0; i < b.tokens; ++i)
    for (int64_t h = 0; h < b.heads; ++h) {
      const uintptr_t x = b.base + i * b.token + h * b.head;
      const auto next = std::upper_bound(at.begin(), at.end(), x - a.bytes);  // the first piece that ends behind x
      if (next != at.end() && *next < x + b.bytes) return true;
    }
  return false;
}

}  // namespace fkv
