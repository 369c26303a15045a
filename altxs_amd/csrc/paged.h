// Index arithmetic of the paged KV cache (include/altxs.h), shared by the
// kernels and, compiled for the host, by the tests: which segment a token or a
// tile of query rows belongs to, which keys a row sees, and where a key lies.
// Every function is total: whatever the device arrays hold, the results stay
// inside the bounds that the callers index with.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define ALTXS_HD __host__ __device__ __forceinline__
#else
#define ALTXS_HD inline
#endif

namespace altxs_paged {

// Exact n / d for 0 <= n < 2^31 by a multiplication (d >= 1): m = ceil(2^(32+s) / d)
// with 2^s >= d has an error below 2^s / 2^(32+s) per unit of n.
struct FastDiv {
  uint32_t m, s, d;
};
inline FastDiv fast_div(uint32_t d) {
  FastDiv f;
  f.d = d;
  f.s = 0;
  while ((1u << f.s) < d) ++f.s;
  f.m = (uint32_t)((((uint64_t)1 << (32 + f.s)) + d - 1) / d - ((uint64_t)1 << 32));
  return f;
}
ALTXS_HD uint32_t div_by(uint32_t n, const FastDiv f) {
  const uint64_t h = ((uint64_t)n * f.m >> 32) + n;  // n * (2^32 + m) >> 32, below 2^33
  return (uint32_t)(h >> f.s);
}

// First slot of segment b among the row tiles of `br` rows, when its tokens start at
// row `start` and every token makes `g` rows.  Slots f(b) .. f(b+1)-1 are enough for
// its tiles (floor((a + n) / br) - floor(a / br) + 1 >= ceil(n / br)), need no sum
// over the segments, and ascend with b as cu does.
ALTXS_HD int64_t first_slot(int64_t start, int g, int br, int64_t b) { return start * g / br + b; }
ALTXS_HD int64_t slot_count(int64_t T, int g, int br, int64_t B) { return T * g / br + B; }

// A segment's share of the call, made safe: rows [t0, t0 + n) of the token
// arrays, first position pos.  ok = 0: the segment is left out (flagged).
struct Segment {
  int32_t t0, n, pos, ok;
};
ALTXS_HD Segment segment_of(int32_t c0, int32_t c1, int32_t pos, int64_t T, int32_t cap) {
  Segment s;
  s.ok = c0 >= 0 && c1 >= c0 && c1 <= T && pos >= 0 && (int64_t)pos + (c1 - c0) <= cap;
  s.t0 = c0 < 0 ? 0 : c0;
  if (s.t0 > T) s.t0 = (int32_t)T;
  s.n = c1 <= s.t0 ? 0 : (int32_t)((c1 < T ? c1 : T) - s.t0);
  s.pos = pos;
  return s;
}

// Keys [lo, hi) seen by the token at position p (hi <= len <= cap); empty when lo >= hi.
struct Range {
  int32_t lo, hi;
};
ALTXS_HD Range keys_seen(int32_t p, int32_t len, int32_t window, int32_t start, int32_t prefix) {
  Range r;
  const int32_t pre = prefix < len ? prefix : len;
  r.hi = p + 1 > pre ? p + 1 : pre;
  r.lo = start > 0 ? start : 0;
  if (window > 0 && p - window + 1 > r.lo) r.lo = p - window + 1;
  if (r.lo >= r.hi) r.lo = r.hi = 0;
  return r;
}

// Page of key row t, or -1: t outside the table or a page id outside [0, n_pages).
ALTXS_HD int32_t page_of(const int32_t* row, int32_t width, int32_t shift, int64_t n_pages, int32_t t) {
  const int32_t i = t >> shift;
  if (t < 0 || i >= width) return -1;
  const int32_t g = row[i];
  return g < 0 || g >= n_pages ? -1 : g;
}

// Segments lo .. lo + n - 1 in 64 parts: the last segment of part `lane` (its own, or that of
// the last part that has any), and the first part whose bit is set (else the last).
struct Block {
  int32_t lo, n;
};
ALTXS_HD int32_t part_end(const Block b, int lane) {
  const int64_t end = (int64_t)(lane + 1) * ((b.n - 1) / 64 + 1);
  return b.lo + (int32_t)(end < b.n ? end : b.n) - 1;
}
ALTXS_HD Block part_of(const Block b, uint64_t bits) {
  const int32_t step = (b.n - 1) / 64 + 1, k = bits ? __builtin_ctzll(bits) : (b.n - 1) / step, left = b.n - k * step;
  return Block{b.lo + k * step, left < step ? left : step};
}

#if defined(__HIPCC__)
// The first of a block of at most 64 segments that holds the first one of which `later` holds,
// asked by a whole wave: two steps serve 4096 segments.  `later` is false, then true, when cu
// ascends; with any other cu some block comes out.
// (Decoding 4096 ragged segments of 100 keys takes 211 us, equal ones, which need no
// search, 183; 64 segments after the other it took 532.)
template <class F> __device__ __forceinline__ int block_with_first(int B, int lane, F later) {
  Block b = {0, B};
  while (b.n > 64) b = part_of(b, __ballot(later(part_end(b, lane))));
  return b.lo;
}

// The segment of token t, asked by a whole wave, each lane with one's bounds and position (so
// nothing is read again once it is found); -1: the token belongs to nobody.  cu = NULL: every
// segment has W tokens.
__device__ __forceinline__ int token_segment(const int32_t* cu, const int32_t* pos, int B, int W, int64_t t, int64_t T, int cap,
                                             int lane, Segment& s) {
  if (!cu) {
    const int b = (int)(t / W);
    s = segment_of(b * W, b * W + W, pos[b], T, cap);
    return b;
  }
  const int i = block_with_first(B, lane, [&](int j) { return cu[j + 1] > t; });
  const int j = i + lane < B ? i + lane : B - 1;
  const int c0 = cu[j], c1 = cu[j + 1], p = pos[j];
  const uint64_t later = __ballot(i + lane < B && c1 > t);
  if (later) {
    const int l = __builtin_ctzll(later);
    s = segment_of(__builtin_amdgcn_readlane(c0, l), __builtin_amdgcn_readlane(c1, l), __builtin_amdgcn_readlane(p, l), T, cap);
    return i + l;
  }
  s = Segment{0, 0, 0, 0};
  return -1;
}
#endif

}  // namespace altxs_paged
