// What the entry points over a paged key-value cache share.
//
// A cache is [pages, Hkv, page, head_dim]: one (page, head) block is contiguous, so
// the keys that a decode wave streams for its head come in runs of page rows.
// Position p of a sequence lies in page table[row][p / page], slot p % page.
#pragma once

#include <stdint.h>

namespace llmy {

constexpr int32_t kCacheBf16 = 0, kCacheE4m3 = 1;
constexpr int32_t kMaxHeads = 1024;

// log2 of a page's tokens, or -1 where the kernels do not take that size: 16 rows, the
// keys of one MFMA tile, never cross a page, and a slot is a mask and a shift.
inline int page_shift(int32_t page) {
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

// Scores: a scale of at least 0 that is finite in log2 units too; a cap of 0 (none) or up to
// 1024, since the fp32 form of the cap is off by 2^-23 of it, and not so small beside the
// scale that their ratio overflows.
inline bool scale_ok(float scale, float softcap) {
  const float inf = __builtin_inff();
  return scale >= 0.f && scale * 1.4426950408889634f < inf && softcap >= 0.f && softcap <= 1024.f &&
         (softcap == 0.f || 4.f * scale / softcap < inf);
}

// A distance bias a position, in log2 units.  Cut off at kMaxSlope, where a neighbour's
// weight is e^-1024: a larger one times a distance could pass fp32, and 0 times it is NaN.
constexpr float kMaxSlope = 1024.f;

__device__ __forceinline__ float slope_log2(float slope, float most) {
  return (fabsf(slope) > most ? copysignf(most, slope) : slope) * 1.4426950408889634f;
}

// Elements from the first to the last of strided rows [n, H, hd].
inline int64_t rows_extent(int64_t row, int64_t head, int32_t n, int32_t H, int32_t hd) {
  return (n - 1) * row + (H - 1) * head + hd;
}

// Strided rows of 16-bit words [n, H, hd], whose memory may interleave with other rows' (the
// q and k of a fused projection), so that only an exact look tells whether they meet.
struct Rows {
  const void* p;
  int64_t row, head;  // strides, in elements
  int32_t n, H, hd;

  // Elements to the end of the last; a double, since strides are any 63-bit number.
  double extent() const {
    return static_cast<double>(n - 1) * row + static_cast<double>(H - 1) * head + hd;
  }
  bool same(const Rows& o) const {
    return p == o.p && (n == 1 || row == o.row) && (H == 1 || head == o.head);
  }
};

// Whether the blocks of hd elements at d + i r, -n < i < n, miss the one at 0 (i = 0 left
// out where `others`).
inline bool misses(int64_t d, int64_t r, int32_t n, int32_t hd, bool others = false) {
  const auto miss = [&](int64_t i) {
    const int64_t at = d + i * r;
    return i <= -n || i >= n || (others && i == 0) || at >= hd || at <= -hd;
  };
  // the blocks next to 0, among them the nearest
  const int64_t most = n - 1, i = r == 0 ? 0 : -d / r < -most ? -most : -d / r > most ? most : -d / r;
  return miss(i - 1) && miss(i) && miss(i + 1);
}

constexpr double kMaxExtent = 0x1p52;  // past any memory; the sums below stay exact

// Whether no block of one is touched by a block of the other, of as many rows.
inline bool rows_apart(const Rows& a, const Rows& b) {
  if (a.extent() > kMaxExtent || b.extent() > kMaxExtent) return false;
  const int64_t ea = static_cast<int64_t>(a.extent()), eb = static_cast<int64_t>(b.extent());
  const int64_t d = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.p) -
                                         reinterpret_cast<uintptr_t>(a.p)) / 2;
  if (d >= ea || d <= -eb) return true;
  const int64_t r = a.n == 1 ? 0 : a.row;
  if (a.n > 1 && a.row != b.row) return false;  // entwined at two pitches: not looked into
  const int64_t sa = (a.H - 1) * a.head + a.hd, sb = (b.H - 1) * b.head + b.hd;
  if (r > 0 && sa <= r && sb <= r) {  // beside each other in one wider row
    const int64_t at = (d % r + r) % r;
    if (at >= sa && at + sb <= r) return true;
  }
  if (a.H == 1 || b.H == 1 || a.head == b.head) {
    const int64_t s = a.H == 1 ? b.head : a.head;
    for (int64_t h = 1 - a.H; h < b.H; ++h)
      if (!misses(d + h * s, r, a.n, a.hd)) return false;
    return true;
  }
  for (int64_t i = 0; i < a.H; ++i)
    for (int64_t j = 0; j < b.H; ++j)
      if (!misses(d + j * b.head - i * a.head, r, a.n, a.hd)) return false;
  return true;
}

// Whether no two blocks of rows that are written share an element.
inline bool rows_apart(const Rows& a) {
  if (a.extent() > kMaxExtent) return false;
  const int64_t r = a.n == 1 ? 0 : a.row;
  if (a.n > 1 && !misses(0, r, a.n, a.hd, true)) return false;
  if ((a.H - 1) * a.head + a.hd <= r || (a.H > 1 && (a.n - 1) * r + a.hd <= a.head)) return true;
  for (int64_t h = 1; h < a.H; ++h)
    if (!misses(h * a.head, r, a.n, a.hd)) return false;
  return true;
}

// Whether two ranges of bytes lie apart; an empty one always does.
inline bool bytes_apart(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na == 0 || nb == 0 || x + na <= y || y + nb <= x;
}

// Whether strided rows lie apart from a range of bytes.
inline bool rows_apart(const Rows& a, const void* p, int64_t bytes) {
  const double x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(p);
  return bytes == 0 || y + bytes <= x || y >= x + 2. * a.extent();
}

// Rows written in place of others are exactly those, or apart from them.
inline bool in_place_or_apart(const Rows& out, const Rows& in) {
  return out.same(in) || rows_apart(out, in);
}

// Whether two ranges of 16-bit words lie apart.
inline bool apart(const uint16_t* a, int64_t na, const uint16_t* b, int64_t nb) {
  return a + na <= b || b + nb <= a;
}

// An 8-bit cache holds x / scale, a bf16 one x itself.  From 2^-100 to 2^100 a scale's
// reciprocal, its quotients' remainders and its share of a sum are ordinary fp32 numbers;
// the reciprocal of one below 2^-128 is infinite, and 0 times that is NaN.
inline bool scales_ok(int32_t cache_type, float k_scale, float v_scale) {
  const auto ok = [](float s) { return s >= 0x1p-100f && s <= 0x1p100f; };
  return cache_type == kCacheBf16 ? k_scale == 1.f && v_scale == 1.f : ok(k_scale) && ok(v_scale);
}

}  // namespace llmy
