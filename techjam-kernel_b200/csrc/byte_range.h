// byte_range.h — address ranges of row-major operands, for the host-side
// overlap checks of the entry points (an output whose stores race the reads
// of an input is rejected before launch).
#pragma once

#include <cstdint>

namespace b200attn {

struct ByteRange {
  uintptr_t lo = 0, hi = 0;  // [lo, hi)
  bool overlaps(const ByteRange& o) const { return lo < o.hi && o.lo < hi; }
};

// Bytes spanned by a [rows, cols] matrix of `elem`-byte elements whose rows
// start `ld` elements apart (the last dimension contiguous).
inline ByteRange rows_range(const void* base, int64_t rows, int64_t cols, int64_t ld,
                            int64_t elem = 2) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(base);
  const int64_t span = (rows > 1 ? (rows - 1) * ld : 0) + cols;
  return ByteRange{lo, lo + static_cast<uintptr_t>(span * elem)};
}

// The bytes of a strided view: stretches of `run` bytes that start at whole multiples of
// `pitch` from the first one (0: there is one stretch).
struct Stretches {
  ByteRange all;
  int64_t run = 0, pitch = 0;
};

inline int64_t common_divisor(int64_t a, int64_t b) {
  while (b) {
    const int64_t r = a % b;
    a = b;
    b = r;
  }
  return a;
}

// Of `n` (up to 4) dimensions with strides of no less than 0 elements, and `cols` contiguous
// elements at each place.  Dimensions that continue the stretch become part of it.
inline Stretches stretches_of(const void* base, const int64_t* stride, const int64_t* extent,
                              int n, int64_t cols, int64_t elem) {
  Stretches s;
  s.run = cols * elem;
  bool part[4] = {};
  int64_t last = s.run;
  for (int d = 0; d < n; ++d) {
    part[d] = extent[d] <= 1;
    if (!part[d]) last += (extent[d] - 1) * stride[d] * elem;
  }
  for (bool grew = true; grew;) {
    grew = false;
    for (int d = 0; d < n; ++d)
      if (!part[d] && stride[d] * elem == s.run) {
        s.run *= extent[d];
        part[d] = grew = true;
      }
  }
  for (int d = 0; d < n; ++d)
    if (!part[d]) s.pitch = common_divisor(s.pitch, stride[d] * elem);
  s.all.lo = reinterpret_cast<uintptr_t>(base);
  s.all.hi = s.all.lo + static_cast<uintptr_t>(last);
  return s;
}

// Whether two views can have a byte in common.  Views that lie side by side in the rows of one
// tensor do not: their stretches keep to different places of the common pitch.
inline bool may_overlap(const Stretches& a, const Stretches& b) {
  if (!a.all.overlaps(b.all)) return false;
  const int64_t pitch = common_divisor(a.pitch, b.pitch);
  if (pitch == 0 || a.run + b.run > pitch) return true;
  const int64_t away = static_cast<int64_t>(b.all.lo - a.all.lo) % pitch;
  const int64_t at = away < 0 ? away + pitch : away;  // of b's stretches, seen from a's
  return at < a.run || at + b.run > pitch;
}

}  // namespace b200attn
