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

// An 8-bit cache holds x / scale; a bf16 one x itself.
inline bool scales_ok(int32_t cache_type, float k_scale, float v_scale) {
  const float inf = __builtin_inff();
  return cache_type == kCacheBf16 ? k_scale == 1.f && v_scale == 1.f
                                  : k_scale > 0.f && v_scale > 0.f && k_scale < inf && v_scale < inf;
}

}  // namespace llmy
