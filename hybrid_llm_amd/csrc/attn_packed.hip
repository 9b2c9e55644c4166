// Attention over packed prompts: row i of document [a, e) (from the running sums of the
// documents' lengths) with window W and a two-way prefix of p rows sees the keys
//   lo_i <= j < hi_i,  lo_i = max(a, i - W + 1),  hi_i = max(i + 1, min(a + p, e)),
// an interval for every mask this entry has; scores z = scale q . k, capped
// c tanh(z / c), less slope_h |i - j|; o = sum_j softmax(z)_j v_j.  Query head h reads
// key-value head h / (Hq / Hkv).
//
// Matrix work in the transposed form of attn_prefill.hip (S^T = K Q^T, O^T = V^T P^T on
// v_mfma_f32_32x32x16_bf16, P never leaves its registers, K and V by DMA into two
// swizzled LDS stages): a workgroup owns 128 consecutive rows of one head, whatever
// documents they belong to, and walks the 64-key tiles that any of its rows sees; a
// wave skips 32-key sub-tiles that none of its 32 rows sees and masks only those that
// some of its rows see and some do not.
// What a masked place holds, NaN and infinities included, must reach no row, and 0 * inf
// is NaN in the product: such values are zeroed in the fragments of a sub-tile that
// some row does not see in full, and the rows that do see them get them at the end.
// Blocks run from the last rows to the first, the longest ones of a document first,
// heads fastest: with 8 or 16 heads a head's blocks share an XCD's L2.
#include "common.hpp"
#include "abi_util.hpp"
#include "attn_tile.hpp"
#include "paged.hpp"

namespace llmy {

typedef float f32x16v __attribute__((ext_vector_type(16)));

constexpr int kPN = 64;   // keys per staged tile

struct PackedArgs {
  const uint16_t *q, *k, *v;
  long long qr, qh, kr, kh, vr, vh;  // strides by row and head (elements)
  uint16_t* o;
  const int32_t *cu, *prefix;
  const float* slopes;
  float scale_log2, cap_log2, cap_x2;
  int N, docs, hq, G, window;
};

__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v = min(v, __shfl_xor(v, d, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}

__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v = max(v, __shfl_xor(v, d, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}

// Fragment reads at a fixed distance from an address register (the immediate saves an
// add), and the wait for them.  AG: into accumulation registers, which the matrix
// instructions read as well: with 64 rows a wave of 128-wide heads, the fragments and
// the output tiles together are more than the 256 that vector instructions reach.
template <bool AG, int OFF>
__device__ __forceinline__ u32x4 lds_b128_at(uint32_t addr) {
  u32x4 v;
  if constexpr (AG)
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=a"(v) : "v"(addr), "n"(OFF) : "memory");
  else
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF) : "memory");
  return v;
}

template <bool AG, int OFF>
__device__ __forceinline__ u32x2 lds_tr16_at(uint32_t addr) {
  u32x2 v;
  if constexpr (AG)
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=a"(v) : "v"(addr), "n"(OFF) : "memory");
  else
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF) : "memory");
  return v;
}

template <bool AG>
__device__ __forceinline__ void settle4(u32x4* f) {
  if constexpr (AG)
    asm volatile("s_waitcnt lgkmcnt(0)" : "+a"(f[0]), "+a"(f[1]), "+a"(f[2]), "+a"(f[3])::"memory");
  else
    lds_settle4(f);
}

template <bool AG>
__device__ __forceinline__ void settle8(u32x2* f) {
  if constexpr (AG)
    asm volatile("s_waitcnt lgkmcnt(0)"
                 : "+a"(f[0]), "+a"(f[1]), "+a"(f[2]), "+a"(f[3]), "+a"(f[4]), "+a"(f[5]),
                   "+a"(f[6]), "+a"(f[7])::"memory");
  else
    lds_settle_v(f);
}

// Per 16-bit half, 0xffff where its exponent is all ones (infinities and NaN).
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return (((w & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u) * 0xffffu;
}

typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

template <int V>
struct Int {
  static constexpr int value = V;
};

// SCORE: scores are capped or biased (otherwise the scale goes into the exponent).
// QT: 32-row tiles of a wave.
template <int HD, bool SCORE, int QT>
__global__ __launch_bounds__(256, HD == 64 || QT == 1 ? 2 : 1) void packed_attn_kernel(
    const PackedArgs a) {
  constexpr int ND = HD / 32;         // 32-dim output tiles
  constexpr int NS = HD / 16;         // 16-dim slices of the score product
  constexpr int RB = 2 * HD;          // bytes of a staged row
  constexpr int TB = kPN * RB;        // bytes of a staged K or V tile
  constexpr int PM = 128 * QT;        // rows per workgroup
  constexpr int ST = 3;               // stages
  constexpr bool AG = HD == 128;      // where the fragments lie
  __shared__ __align__(1024) uint8_t smem[ST * 2 * TB];
  __shared__ int range[2][4];

  const int nblk = (a.N + PM - 1) / PM;
  const int h = blockIdx.x % a.hq;
  const int q0 = (nblk - 1 - static_cast<int>(blockIdx.x / a.hq)) * PM;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5;
  const int col = lane & 31;
  const int qw = q0 + 32 * QT * wave;  // this wave's first row; tile x: 32 x more

  // this lane's rows: their documents by bisection, their keys [lo, lo + n); none for a
  // row of no document.  A tile's sub-tile is whole (needs no mask) in [ilo, ihi).
  int lo[QT], ilo[QT], ihi[QT];
  unsigned n[QT];
  bool mine[QT];
  const int big = 0x7fffffff;
  int wlo = big, whi = 0;
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const int qi = qw + 32 * x + col;
    int hi = 0;
    lo[x] = 0;
    mine[x] = false;
    if (qi < a.N) {
      int b = 0, e = a.docs + 1;  // the first entry past qi
      while (b < e) {
        const int mid = (b + e) >> 1;
        if (a.cu[mid] <= qi) b = mid + 1;
        else e = mid;
      }
      if (b > 0 && b <= a.docs) {
        const int first = max(a.cu[b - 1], 0), end = min(a.cu[b], a.N);
        const int two_way = a.prefix ? min(max(a.prefix[b - 1], 0), end - first) : 0;
        mine[x] = true;
        lo[x] = a.window > 0 ? max(first, qi - min(a.window - 1, qi)) : first;
        hi = max(qi + 1, first + two_way);
      }
    }
    n[x] = hi - lo[x];
    wlo = min(wlo, wave_min_i(mine[x] ? lo[x] : big));
    whi = max(whi, wave_max_i(mine[x] ? hi : 0));
    ilo[x] = wave_max_i(mine[x] ? lo[x] : 0);
    ihi[x] = wave_min_i(mine[x] ? hi : big);
  }
  if (lane == 0) {
    range[0][wave] = wlo;
    range[1][wave] = whi;
  }
  __syncthreads();
  const int glo = min(min(range[0][0], range[0][1]), min(range[0][2], range[0][3]));
  const int ghi = max(max(range[1][0], range[1][1]), max(range[1][2], range[1][3]));
  if (ghi <= 0) return;  // no row of any document
  const int t_lo = __builtin_amdgcn_readfirstlane(glo / kPN);
  const int t_hi = __builtin_amdgcn_readfirstlane((ghi - 1) / kPN);
  // the wave's sub-tiles, from an even one on
  const int j0 = whi > 0 ? wlo / kPN * 2 : big, j1 = whi > 0 ? (whi + 31) / 32 : 0;

  uint4 qf[QT][NS];
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const uint16_t* qp = a.q + min(qw + 32 * x + col, a.N - 1) * a.qr + h * a.qh + 8 * half;
#pragma unroll
    for (int t = 0; t < NS; ++t) qf[x][t] = *reinterpret_cast<const uint4*>(qp + 16 * t);
  }
  float slope = 0.f;
  if (SCORE && a.slopes) slope = a.slopes[h] * 1.4426950408889634f;
  const float sc = SCORE ? 1.f : a.scale_log2;

  f32x16v acc[QT][ND], s[QT];
  float m[QT], l[QT];  // the exponent's offset (scaled, log2) and the sum of weights
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    m[x] = -1e38f;
    l[x] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][d][r] = 0.f;
  }

  // DMA: 1 KiB blocks j = wave + 4 i of RPB rows; lane p fills row RPB j + p / CH, chunk
  // slot p % CH.  Rows past the last re-read it (no row sees them).
  constexpr int CH = HD / 8;
  constexpr int RPB = 64 / CH;
  constexpr int BPW = kPN / RPB / 4;
  const uint16_t* kb = a.k + (h / a.G) * a.kh;
  const uint16_t* vb = a.v + (h / a.G) * a.vh;
  const int kr = static_cast<int>(a.kr), vr = static_cast<int>(a.vr);
  uint32_t kdo[BPW], vdo[BPW];
#pragma unroll
  for (int i = 0; i < BPW; ++i) {
    const int r = RPB * (wave + 4 * i) + lane / CH, sl = lane % CH;
    kdo[i] = r * kr + 8 * (sl ^ (r & 7));
    vdo[i] = r * vr + 8 * (sl ^ (2 * (r & 3)));
  }
  auto issue = [&](int tile, int st) __attribute__((always_inline)) {
    const int kt = tile * kPN;
    uint8_t* sk = smem + st * 2 * TB + wave * 1024;
    const uint16_t* kp = kb + kt * a.kr;
    const uint16_t* vp = vb + kt * a.vr;
    if (kt + kPN <= a.N) {
#pragma unroll
      for (int i = 0; i < BPW; ++i) {
        dma16(kp + kdo[i], sk + 4096 * i);
        dma16(vp + vdo[i], sk + TB + 4096 * i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < BPW; ++i) {
        const int r = RPB * (wave + 4 * i) + lane / CH;
        const int back = max(0, r - (a.N - 1 - kt));
        dma16(kp + (static_cast<int>(kdo[i]) - back * kr), sk + 4096 * i);
        dma16(vp + (static_cast<int>(vdo[i]) - back * vr), sk + TB + 4096 * i);
      }
    }
  };

  // fragment addresses in stage 0: K slice t at ka[t % 4] (+ 128 bytes for t >= 4), V
  // tile d at va[d % 2] (+ 128 for d >= 2); the swizzle spares the higher bits
  uint32_t ka[4], va[2];
  {
    const uint32_t sbase = lds_addr(smem);
#pragma unroll
    for (int t = 0; t < 4; ++t) ka[t] = sbase + col * RB + 16 * ((2 * t + half) ^ (col & 7));
    const int y = lane & 15, g = lane >> 4, i = y >> 2;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int dim0 = 32 * d + 16 * (g & 1) + 4 * (y & 3);
      va[d] = sbase + TB + (4 * half + i) * RB + 16 * ((dim0 >> 3) ^ (2 * i)) + 2 * (dim0 & 7);
    }
  }
  u32x4 kf[2][NS];           // K fragments by the sub-tile's parity
  u32x2 vf[2][2 * ND * 2];   // V fragments: [slice][tile][lo, hi 8 keys]
  auto read_k = [&](auto par, uint32_t off) __attribute__((always_inline)) {
    constexpr int P = decltype(par)::value;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      kf[P][t] = lds_b128_at<AG, P * 32 * RB>(ka[t] + off);
      if constexpr (NS == 8) kf[P][t + 4] = lds_b128_at<AG, P * 32 * RB + 128>(ka[t] + off);
    }
  };
  auto read_v = [&](auto par, uint32_t off) __attribute__((always_inline)) {
    constexpr int P = decltype(par)::value;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const uint32_t at = va[d] + off;
      vf[P][2 * d] = lds_tr16_at<AG, P * 32 * RB>(at);
      vf[P][2 * d + 1] = lds_tr16_at<AG, P * 32 * RB + 8 * RB>(at);
      vf[P][2 * ND + 2 * d] = lds_tr16_at<AG, P * 32 * RB + 16 * RB>(at);
      vf[P][2 * ND + 2 * d + 1] = lds_tr16_at<AG, P * 32 * RB + 24 * RB>(at);
      if constexpr (ND == 4) {
        vf[P][2 * d + 4] = lds_tr16_at<AG, P * 32 * RB + 128>(at);
        vf[P][2 * d + 5] = lds_tr16_at<AG, P * 32 * RB + 8 * RB + 128>(at);
        vf[P][2 * ND + 2 * d + 4] = lds_tr16_at<AG, P * 32 * RB + 16 * RB + 128>(at);
        vf[P][2 * ND + 2 * d + 5] = lds_tr16_at<AG, P * 32 * RB + 24 * RB + 128>(at);
      }
    }
  };
  auto settle_k = [&](auto par) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NS; t += 4) settle4<AG>(kf[decltype(par)::value] + t);
  };
  auto settle_v = [&](auto par) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 4 * ND; t += 8) settle8<AG>(vf[decltype(par)::value] + t);
  };

  // scores of tile y and the sub-tile whose K fragments have parity KP
  auto scores = [&](auto yc, auto kp) __attribute__((always_inline)) {
    constexpr int Y = decltype(yc)::value, KP = decltype(kp)::value;
    f32x16v z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
#pragma unroll
    for (int t = 0; t < NS; ++t)
      z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kf[KP][t]),
                                                  as_bf16x8(qf[Y][t]), z, 0, 0, 0);
    s[Y] = z;
  };
  // cap, bias and (EDGE) mask of tile y's scores of sub-tile j; register r holds key
  // 32 j + (r & 3) + 8 (r >> 2) + 4 half
  auto finish_scores = [&](auto yc, auto edge, int j) __attribute__((always_inline)) {
    constexpr int Y = decltype(yc)::value;
    const int k0 = 32 * j + 4 * half;
    if (SCORE) {
      const float dq = static_cast<float>(qw + 32 * Y + col - k0);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float c = (r & 3) + 8 * (r >> 2);
        float z = a.cap_x2 > 0.f ? softcap_log2(s[Y][r] * a.cap_x2, a.cap_log2)
                                 : s[Y][r] * a.scale_log2;
        if (a.slopes) z = fmaf(-slope, fabsf(dq - c), z);
        s[Y][r] = z;
      }
    }
    if constexpr (decltype(edge)::value != 0) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int cr = (r & 3) + 8 * (r >> 2);
        s[Y][r] = static_cast<unsigned>(k0 + cr - lo[Y]) < n[Y] ? s[Y][r] : -INFINITY;
      }
    }
  };
  // the largest score of each row; moves the offset when some row's passes it by 8
  // (log2), decided by the wave, so most sub-tiles rescale nothing
  auto row_max = [&](auto yc) __attribute__((always_inline)) -> float {
    constexpr int Y = decltype(yc)::value;
    float x = s[Y][0];
#pragma unroll
    for (int r = 1; r < 16; ++r) x = fmaxf(x, s[Y][r]);
    // the other lane half's (lanes l and l ^ 32 hold one row)
    const auto sw =
        __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
  };
  auto rescale = [&](auto yc, float x) __attribute__((always_inline)) {
    constexpr int Y = decltype(yc)::value;
    if (__ballot(fmaf(x, sc, -8.f) > m[Y])) {
      const float m_new = fmaxf(m[Y], x * sc);
      const float alpha = exp2_fast(m[Y] - m_new);
      m[Y] = m_new;
      l[Y] *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[Y][d][r] *= alpha;
    }
  };
  // weights of tile x: rounded, and the sum of the rounded ones
  auto weights = [&](auto xc, uint4* pb) __attribute__((always_inline)) {
    constexpr int X = decltype(xc)::value;
    float p[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = exp2_fast(fmaf(s[X][r], sc, -m[X]));
    pb[0] = pack8_bf16(p);
    pb[1] = pack8_bf16(p + 8);
    const bf16x2v one = __builtin_bit_cast(bf16x2v, 0x3f803f80u);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[X] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, pb[i].x), one, l[X], false);
      l[X] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, pb[i].y), one, l[X], false);
      l[X] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, pb[i].z), one, l[X], false);
      l[X] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, pb[i].w), one, l[X], false);
    }
  };
  auto add_values = [&](auto xc, auto vp, const uint4* pb) __attribute__((always_inline)) {
    constexpr int X = decltype(xc)::value, VP = decltype(vp)::value;
#pragma unroll
    for (int sl = 0; sl < 2; ++sl)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const u32x2 f0 = vf[VP][2 * ND * sl + 2 * d], f1 = vf[VP][2 * ND * sl + 2 * d + 1];
        acc[X][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            as_bf16x8(uint4{f0.x, f0.y, f1.x, f1.y}), as_bf16x8(pb[sl]), acc[X][d], 0, 0, 0);
      }
  };
  // Values that are not finite, in a sub-tile that some row does not see: zeroed in the V
  // fragments; the rows that see them get them after the last tile.
  bool dirty = false;
  auto clean_values = [&](auto vp) __attribute__((always_inline)) {
    constexpr int VP = decltype(vp)::value;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4 * ND; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) top |= (vf[VP][i][e] & 0x7f807f80u) + 0x00800080u;
    if (!__ballot((top & 0x80008000u) != 0)) return;
    dirty = true;
#pragma unroll
    for (int i = 0; i < 4 * ND; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) vf[VP][i][e] &= ~not_finite(vf[VP][i][e]);
  };
  auto whole = [&](int x, int j) { return 32 * j >= ilo[x] && 32 * j + 32 <= ihi[x]; };

  // One unit, tile x of sub-tile jx (its scores and offset ready): the scores of the next
  // unit (tile y of sub-tile jy) run on the matrix cores under this one's exponentials,
  // its own product under the next one's maximum.  Units with a masked row go one thing
  // after the other.
  auto unit = [&](auto xc, auto yc, auto vp, auto kp, int jx, int jy)
                  __attribute__((always_inline)) {
    constexpr int X = decltype(xc)::value, Y = decltype(yc)::value;
    uint4 pb[2];
    float x;
    if (whole(X, jx) && whole(Y, jy)) {
      f32x16v keep;
      if constexpr (X == Y) {  // one tile a wave: its next scores beside its present ones
        keep = s[X];
        scores(yc, kp);
        const f32x16v nextv = s[X];
        s[X] = keep;
        weights(xc, pb);
        s[X] = nextv;
      } else {
        scores(yc, kp);
        weights(xc, pb);
      }
      add_values(xc, vp, pb);
      finish_scores(yc, Int<0>{}, jy);
      x = row_max(yc);
    } else {
      weights(xc, pb);
      if (!whole(X, jx)) clean_values(vp);
      add_values(xc, vp, pb);
      scores(yc, kp);
      finish_scores(yc, Int<1>{}, jy);
      x = row_max(yc);
    }
    rescale(yc, x);
  };

  const Int<0> A{};
  const Int<QT - 1> Z{};
  const Int<0> P0{};
  const Int<1> P1{};
  issue(t_lo, 0);
  if (t_lo < t_hi) issue(t_lo + 1, 1);
  int st = 0;
  for (int tile = t_lo; tile <= t_hi; ++tile) {
    // this tile's and the next one's DMAs have landed and, after the barrier, every
    // wave's have, and every wave is done with the stage before, which the tile after the
    // next then fills
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const int st1 = st == ST - 1 ? 0 : st + 1, st2 = st1 == ST - 1 ? 0 : st1 + 1;
    if (tile + 2 <= t_hi) issue(tile + 2, st2);
    const int j = 2 * tile;
    const uint32_t here = st * 2 * TB, next = st1 * 2 * TB;
    if (j >= j0 && j < j1) {
      if (j == j0) {
        read_k(P0, here);
        read_v(P0, here);
        if constexpr (QT == 1) read_k(P1, here);
        settle_k(P0);
        scores(A, P0);
        finish_scores(A, Int<1>{}, j);
        rescale(A, row_max(A));
      }
      if constexpr (QT == 2) {
        settle_v(P0);
        read_k(P1, here);
        unit(A, Z, P0, P0, j, j);
        settle_k(P1);
        read_v(P1, here);
        unit(Z, A, P0, P1, j, j + 1);
        settle_v(P1);
        if (j + 1 < j1) {
          read_k(P0, next);
          unit(A, Z, P1, P1, j + 1, j + 1);
          settle_k(P0);
          read_v(P0, next);
          unit(Z, A, P1, P0, j + 1, j + 2);
        }
      } else {
        settle_v(P0);
        settle_k(P1);
        read_v(P1, here);
        read_k(P0, next);
        unit(A, A, P0, P1, j, j + 1);
        settle_v(P1);
        settle_k(P0);
        if (j + 1 < j1) {
          read_v(P0, next);
          read_k(P1, next);
          unit(A, A, P1, P0, j + 1, j + 2);
        }
      }
    }
    st = st1;
  }
  // reads of a sub-tile that does not exist may still be under way
  settle_k(P0);
  settle_k(P1);
  settle_v(P0);

  if (dirty) {
    // the values left out, straight from memory: lane's dims 32 d + 8 g + 4 half .. + 3 of
    // every key that its rows see (one that was added before adds nothing new: inf + inf)
    for (int key = wlo; key < whi; ++key) {
      const uint16_t* row = vb + key * a.vr + 4 * half;
#pragma unroll
      for (int e = 0; e < 4 * ND; ++e) {
        const uint2 w = *reinterpret_cast<const uint2*>(row + 8 * e);
        const uint32_t f[2] = {w.x & not_finite(w.x), w.y & not_finite(w.y)};
#pragma unroll
        for (int x = 0; x < QT; ++x) {
          const uint32_t sees = static_cast<unsigned>(key - lo[x]) < n[x] ? 0xffffffffu : 0u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t b = f[i >> 1] & sees;
            acc[x][e >> 2][4 * (e & 3) + i] += __uint_as_float(i & 1 ? b & 0xffff0000u : b << 16);
          }
        }
      }
    }
  }

#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const float l_tot = l[x] + __shfl_xor(l[x], 32, kWave);
    if (!mine[x]) continue;
    const float inv = 1.0f / l_tot;
    uint16_t* orow = a.o + (static_cast<long long>(qw + 32 * x + col) * a.hq + h) * HD;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const int dim = 32 * d + 8 * g4 + 4 * half;
        *reinterpret_cast<uint2*>(orow + dim) =
            make_uint2(pack_bf2(acc[x][d][4 * g4] * inv, acc[x][d][4 * g4 + 1] * inv),
                       pack_bf2(acc[x][d][4 * g4 + 2] * inv, acc[x][d][4 * g4 + 3] * inv));
      }
  }
}

template <int HD, bool SCORE>
void launch_packed(const PackedArgs& a, int qt, unsigned blocks, hipStream_t s) {
  if (qt == 2)
    hipLaunchKernelGGL((packed_attn_kernel<HD, SCORE, 2>), dim3(blocks), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((packed_attn_kernel<HD, SCORE, 1>), dim3(blocks), dim3(256), 0, s, a);
}

}  // namespace llmy

using namespace llmy;

extern "C" int32_t llmy_packed_attn_prefill_bf16(
    const llmy_bf16* q, int64_t q_row, int64_t q_head, const llmy_bf16* k, int64_t k_row,
    int64_t k_head, const llmy_bf16* v, int64_t v_row, int64_t v_head, const int32_t* cu_seqlens,
    const int32_t* prefix, const float* slopes, llmy_bf16* out, int32_t N, int32_t docs,
    int32_t Hq, int32_t Hkv, int32_t head_dim, int32_t window, float scale, float softcap,
    void* stream) {
  LLMY_REQUIRE(N >= 0 && docs >= 0 && docs < (1 << 30) && Hq > 0 && Hkv > 0 && Hq <= kMaxHeads &&
               Hq % Hkv == 0);
  LLMY_REQUIRE((head_dim == 64 || head_dim == 128) && window >= 0 && scale >= 0.f &&
               softcap >= 0.f);
  LLMY_REQUIRE(N < (1 << 30));  // positions and tile ends are 32-bit
  if (N == 0 || docs == 0) return 0;
  LLMY_REQUIRE(q && k && v && out && cu_seqlens);
  LLMY_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16));
  for (const int64_t x : {q_row, q_head, k_row, k_head, v_row, v_head})
    LLMY_REQUIRE(x >= 0 && x % 8 == 0);
  LLMY_REQUIRE(k_row < (1 << 22) && v_row < (1 << 22));  // 64-row offsets are 32-bit
  // 256 rows a workgroup where that fills the chip twice over, else 128
  const int qt = static_cast<long long>((N + 255) / 256) * Hq >= 2ll * compute_units() ? 2 : 1;
  const long long blocks = static_cast<long long>((N + 128 * qt - 1) / (128 * qt)) * Hq;
  LLMY_REQUIRE(blocks < (1ll << 31));
  // out is written while other workgroups still read k and v
  const int64_t hd = head_dim;
  const auto apart = [&](const llmy_bf16* p, int64_t row, int64_t head) {
    const llmy_bf16* end = p + (N - 1) * row + (Hkv - 1) * head + hd;
    return end <= out || out + static_cast<int64_t>(N) * Hq * hd <= p;
  };
  LLMY_REQUIRE(apart(k, k_row, k_head) && apart(v, v_row, v_head));
  PackedArgs a{};
  a.q = q; a.qr = q_row; a.qh = q_head;
  a.k = k; a.kr = k_row; a.kh = k_head;
  a.v = v; a.vr = v_row; a.vh = v_head;
  a.o = out; a.cu = cu_seqlens; a.prefix = prefix; a.slopes = slopes;
  const float log2e = 1.4426950408889634f;
  a.scale_log2 = scale * log2e;
  a.cap_log2 = softcap * log2e;
  a.cap_x2 = softcap > 0.f ? 2.f * log2e * scale / softcap : 0.f;
  a.N = N; a.docs = docs; a.hq = Hq; a.G = Hq / Hkv; a.window = window;
  const hipStream_t st = as_stream(stream);
  const unsigned grid = static_cast<unsigned>(blocks);
  // a scale of 0 would turn the masked scores' -inf into NaN in the exponent
  const bool score = softcap > 0.f || slopes || scale == 0.f;
  if (head_dim == 64)
    score ? launch_packed<64, true>(a, qt, grid, st) : launch_packed<64, false>(a, qt, grid, st);
  else
    score ? launch_packed<128, true>(a, qt, grid, st) : launch_packed<128, false>(a, qt, grid, st);
  return launch_status();
}
