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
