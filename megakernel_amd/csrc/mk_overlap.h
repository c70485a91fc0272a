// Whether two tensors lie on each other.  Plain C++ (no HIP), so that the CPU
// tests run the same code.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace mk {

// Rows [tokens][heads] of `width` bytes each, bytes from one token / head to the
// next (neither negative).
struct Span {
  uintptr_t p;
  long long tokens, heads, ts, hs, width;
};

// Some byte of a is one of b.  Tensors of other strides than each other's whose
// ranges meet (two shapes of one buffer) are not compared: false.
inline bool overlap(Span a, Span b) {
  if (a.tokens < 1 || b.tokens < 1 || a.heads < 1 || b.heads < 1 || a.width < 1 || b.width < 1) return false;
  for (Span* s : {&a, &b}) {
    if (s->heads > 1 && s->hs == s->width) s->width *= s->heads, s->heads = 1;  // heads side by side are one row
    if (s->heads == 1 && s->tokens > 1 && s->ts == s->width) s->width *= s->tokens, s->tokens = 1;  // and so are tokens
    if (s->heads == 1) s->hs = 0;
    if (s->tokens == 1) s->ts = 0;
  }
  const auto last = [](const Span& s) { return s.p + (uintptr_t)((s.tokens - 1) * s.ts + (s.heads - 1) * s.hs + s.width - 1); };
  if (last(a) < b.p || last(b) < a.p) return false;
  if ((a.tokens > 1 && b.tokens > 1 && a.ts != b.ts) || (a.heads > 1 && b.heads > 1 && a.hs != b.hs)) return false;
  const long long t = std::max(a.ts, b.ts), h = std::max(a.hs, b.hs), delta = (long long)(b.p - a.p);
  // row (x, y) of a and row (x', y') of b, j = y - y', i = x - x': they meet where
  // lo < i t < hi.  i from 1 - b.tokens to a.tokens - 1: the first that is above lo.
  for (long long j = 1 - b.heads; j < a.heads; ++j) {
    const long long lo = delta - j * h - a.width, hi = delta - j * h + b.width;
    long long i = 0;
    if (t) {
      i = lo / t - (lo % t < 0) + 1;
      i = std::max(i, 1 - b.tokens);
      if (i > a.tokens - 1) continue;
    }
    if (lo < i * t && i * t < hi) return true;
  }
  return false;
}

}  // namespace mk
