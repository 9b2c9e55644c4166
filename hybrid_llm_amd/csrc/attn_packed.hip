// Attention over packed prompts: row i of document [a, e) (from the running sums of the
// documents' lengths) with window W and a two-way prefix of p rows sees the keys
//   lo_i <= j < hi_i,  lo_i = max(a, i - W + 1),  hi_i = max(i + 1, min(a + p, e)),
// an interval for every mask this entry has; scores z = scale q . k, capped
// c tanh(z / c), less slope_h |i - j|; o = sum_j softmax(z)_j v_j.  Query head h reads
// key-value head h / (Hq / Hkv).
//
// Matrix work in the transposed form of attn_prefill.hip (S^T = K Q^T, O^T = V^T P^T on
// v_mfma_f32_32x32x16_bf16, P never leaves its registers, K and V copied into two
// swizzled LDS stages): a wave owns 32 consecutive rows of one head, whatever documents
// they belong to, and takes 32 keys at a time; it skips those that none of its rows
// sees and masks only those that some of its rows see and some do not.
//   * Many rows: the four waves of a workgroup own 128 rows and share 64-key tiles.  A
//     sub-tile is 82 vector instructions beside its 16 (128-wide heads) or 8 matrix
//     ones, and two or four waves a SIMD run the one kind under the other's.
//   * Few rows: two or four waves own the same 32 rows and take a half of each 64-key or
//     a quarter of each 128-key tile; their sums are joined in LDS.  The longest chain
//     of sub-tiles, 1100 cycles each where a SIMD has little else, is a half or a quarter
//     as long and there are more workgroups, against two or four times the copies.
//     One prompt, 16 heads over 4, us with 1 / 2 / 4 waves along the keys (a workgroup a
//     128 rows and head): 1024 rows (128 workgroups) x 64 21 / 15 / 12, x 128 31 / 22 / 22;
//     2048 (256) 40 / 30 / 28, 57 / 41 / 60; 4096 (512) 78 / 61 / 82, 112 / 98 / 197;
//     8192 (1024) 175 / 178 / 285, 307 / 350 / 744.  So four up to half a workgroup a
//     CU, two up to two.  (Whole prompts: a window and short documents, which shorten
//     the chain that more waves cut, are not part of the rule.)
// Blocks run from the last rows to the first, the longest ones of a document first; the
// query heads of a key-value head run side by side on one XCD and share its L2.
//
// What a masked place holds, NaN and infinities included, must reach no row, what a visible
// one holds every row that sees it, however small its weight, and 0 * inf is NaN in the
// product.  The values are not looked at as they pass (96 instructions a sub-tile): a
// workgroup that ends with an output that is not finite runs once more, with such values
// zeroed and given to the rows that see them at the end.
//
// An exponent s scale - m is one multiply-add, its product not rounded, while m is the
// rounded product of the largest score: the weights are off by one factor 2^d, |d| half a
// step of m.  It leaves with the division by their sum, as long as it stays inside the
// exponent's range: d is 8 at most where |m| < 2^28.  A workgroup with an m past that
// runs the second time too, which rounds the products first (a multiply a score, 2% of a
// long prompt's time if all took it).
#include "common.hpp"
#include "abi_util.hpp"
#include "attn_tile.hpp"
#include "paged.hpp"

namespace llmy {

typedef float f32x16v __attribute__((ext_vector_type(16)));

constexpr int kDocsInLds = 511;

// A row's offset before its first score: every finite score reaches it.
constexpr float kNoScore = -3.402823466e38f;
// From here on (log2 units) a workgroup runs its second time: see below.
constexpr float kFar = 0x1p28f;

struct PackedArgs {
  const uint16_t *q, *k, *v;
  long long qr, qh, kr, kh, vr, vh;  // strides by row and head (elements)
  uint16_t* o;
  const int32_t *cu, *prefix;
  const float* slopes;
  float scale_log2, cap_log2, cap_x2;
  int N, docs, hq, hkv, G, window;
};

// Per 16-bit half, 0xffff where its exponent is all ones (infinities and NaN).
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return (((w & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u) * 0xffffu;
}

typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

template <int V>
struct Int {
  static constexpr int value = V;
};

// kBiased: a distance bias alone; kAny: with a cap or a two-way prefix
// too, or a scale near 0
enum { kPlain = 0, kCapped = 1, kBiased = 2, kAny = 3 };

// KW: waves along the keys (1, 2 or 4); 4 / KW waves along the rows.
template <int HD, int MODE, int KW>
__global__ __launch_bounds__(256, (HD == 128 ? 2 : MODE == kAny ? 3 : 4) / (KW == 4 ? 2 : 1))
void packed_attn_kernel(const PackedArgs a) {
  constexpr int ND = HD / 32;             // 32-dim output tiles
  constexpr int NS = HD / 16;             // 16-dim slices of the score product
  constexpr int RB = 2 * HD;              // bytes of a staged row
  constexpr int PM = 128 / KW;            // rows per workgroup
  constexpr int PN = KW == 4 ? 128 : 64;  // keys per staged tile
  constexpr int TB = PN * RB;             // bytes of a staged K or V tile
  // the two stages; with two waves along the keys the join takes 4 KiB more
  __shared__ __align__(1024) uint8_t smem[2 * 2 * TB + (KW == 2 ? 4096 : 0)];
  __shared__ int range[2][4];
  __shared__ int cu_s[kDocsInLds + 1];

  // workgroup i runs on XCD i % 8: a unit, PM rows of one key-value head, goes to one of
  // them with all its query heads
  const int nblk = (a.N + PM - 1) / PM;
  const int unit = static_cast<int>(blockIdx.x / (8u * a.G)) * 8 + static_cast<int>(blockIdx.x % 8u);
  const int qb = unit / a.hkv;
  if (qb >= nblk) return;
  const int kvh = unit - qb * a.hkv;
  const int h = kvh * a.G + static_cast<int>(blockIdx.x / 8u) % a.G;
  const int q0 = (nblk - 1 - qb) * PM;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5;
  const int col = lane & 31;
  const int rg = wave / KW, part = wave % KW;  // 32 rows, 1 / KW of the sub-tiles
  const int qi = q0 + 32 * rg + col;           // this lane's row

  u32x4 qf[NS];
  {
    const uint16_t* qp = a.q + min(qi, a.N - 1) * a.qr + h * a.qh + 8 * half;
#pragma unroll
    for (int t = 0; t < NS; ++t) qf[t] = *reinterpret_cast<const u32x4*>(qp + 16 * t);
  }

  // its document by bisection (few documents: in LDS, one load's latency instead of a
  // chain), its keys [lo, hi); none for a row of no document
  const bool few = a.docs <= kDocsInLds;
  if (few)
    for (int i = threadIdx.x; i <= a.docs; i += 256) cu_s[i] = a.cu[i];
  __syncthreads();
  auto cu = [&](int i) { return few ? cu_s[i] : a.cu[i]; };
  int lo = 0, hi = 0;
  bool mine = false;
  if (qi < a.N) {
    int b = 0, e = a.docs + 1;  // the first entry past qi
    while (b < e) {
      const int mid = (b + e) >> 1;
      if (cu(mid) <= qi) b = mid + 1;
      else e = mid;
    }
    if (b > 0 && b <= a.docs) {
      const int first = max(cu(b - 1), 0), end = min(cu(b), a.N);
      const int two_way = a.prefix ? min(max(a.prefix[b - 1], 0), end - first) : 0;
      mine = true;
      lo = a.window > 0 ? max(first, qi - min(a.window - 1, qi)) : first;
      hi = max(qi + 1, first + two_way);
    }
  }
  // the wave's rows see keys in [wlo, whi), all of them those in [ilo, ihi): both bounds
  // ascend with the row, so the first and the last row of a document say it
  const uint32_t rows = static_cast<uint32_t>(__ballot(mine));
  const int r0 = rows ? __ffs(rows) - 1 : 0, r1 = rows ? 31 - __clz(rows) : 0;
  const int wlo = rows ? __builtin_amdgcn_readlane(lo, r0) : 0x7fffffff;
  const int whi = rows ? __builtin_amdgcn_readlane(hi, r1) : 0;
  const int ilo = __builtin_amdgcn_readlane(lo, r1), ihi = __builtin_amdgcn_readlane(hi, r0);
  if (lane == 0) {
    range[0][wave] = wlo;
    range[1][wave] = whi;
  }
  __syncthreads();
  const int glo = min(min(range[0][0], range[0][1]), min(range[0][2], range[0][3]));
  const int ghi = max(max(range[1][0], range[1][1]), max(range[1][2], range[1][3]));
  if (glo >= ghi) return;  // no row of any document (or bounds that do not ascend)
  const int t_lo = __builtin_amdgcn_readfirstlane(glo / PN);
  const int t_hi = __builtin_amdgcn_readfirstlane((ghi - 1) / PN);

  // kBiased rounds the bias and the largest score apart: 2^-24 of the farthest row's
  // bias, 2^31 at the most, stays inside the exponent's range
  const float slope = MODE >= kBiased && a.slopes
      ? slope_log2(a.slopes[h], fminf(kMaxSlope, 0x1p31f / a.N)) : 0.f;
  const float ratio = MODE == kBiased ? slope / a.scale_log2 : 0.f;

  f32x16v acc[ND];
  float m, l;  // the exponent's offset (scaled, log2) and the sum of weights

  // DMA: 1 KiB blocks j = wave + 4 i of RPB rows; lane p fills row RPB j + p / CH, chunk
  // slot p % CH.  Rows past the last re-read it (no row sees them).
  constexpr int CH = HD / 8;
  constexpr int RPB = 64 / CH;
  constexpr int BPW = PN / RPB / 4;
  const uint16_t* kb = a.k + kvh * a.kh;
  const uint16_t* vb = a.v + kvh * a.vh;
  const int kr = static_cast<int>(a.kr), vr = static_cast<int>(a.vr);
  uint32_t kdo[BPW], vdo[BPW];
#pragma unroll
  for (int i = 0; i < BPW; ++i) {
    const int r = RPB * (wave + 4 * i) + lane / CH, sl = lane % CH;
    kdo[i] = 2 * r * kr + 16 * (sl ^ (r & 7));
    vdo[i] = 2 * r * vr + 16 * (sl ^ (2 * (r & 3)));
  }
  const uint32_t sbase = lds_addr(smem);
  auto issue = [&](int tile, int st) __attribute__((always_inline)) {
    const int kt = tile * PN;
    const uint32_t dst = sbase + st * 2 * TB + wave * 1024;
    const uint16_t* kp = kb + kt * a.kr;
    const uint16_t* vp = vb + kt * a.vr;
    if (kt + PN <= a.N) {
#pragma unroll
      for (int i = 0; i < BPW; ++i) {
        lds_fill16(kp, kdo[i], dst + 4096 * i);
        lds_fill16(vp, vdo[i], dst + TB + 4096 * i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < BPW; ++i) {
        const int r = RPB * (wave + 4 * i) + lane / CH;
        const int back = 2 * max(0, r - (a.N - 1 - kt));
        lds_fill16(kp, kdo[i] - back * kr, dst + 4096 * i);
        lds_fill16(vp, vdo[i] - back * vr, dst + TB + 4096 * i);
      }
    }
  };

  // fragment addresses in stage 0: K slice t at ka[t % 4] (+ 128 bytes for t >= 4), V
  // tile d at va[d % 2] (+ 128 for d >= 2); the swizzle spares the higher bits
  uint32_t ka[4], va[2];
  {
#pragma unroll
    for (int t = 0; t < 4; ++t) ka[t] = sbase + col * RB + 16 * ((2 * t + half) ^ (col & 7));
    const int y = lane & 15, g = lane >> 4, i = y >> 2;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int dim0 = 32 * d + 16 * (g & 1) + 4 * (y & 3);
      va[d] = sbase + TB + (4 * half + i) * RB + 16 * ((dim0 >> 3) ^ (2 * i)) + 2 * (dim0 & 7);
    }
  }
  bool careful = false;  // the second run: see the top
  float factor = a.scale_log2;  // of the scores that meet the offset; 1 in the second run
  auto sub_tile = [&](auto subc, int ks, uint32_t off) __attribute__((always_inline)) {
    constexpr int S = decltype(subc)::value * 32 * RB;
    if (ks >= whi || ks + 32 <= wlo) return;  // no row of this wave sees it
    f32x16v s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      const u32x4 kf = lds_get16(ka[t & 3] + off + (S + 128 * (t >> 2)));
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kf),
                                                  __builtin_bit_cast(bf16x8, qf[t]), s, 0, 0, 0);
    }
    // V fragments, asked for ahead of the softmax: [16-key slice][tile][lo, hi 8 keys]
    u32x2 vf[2][ND][2];
#pragma unroll
    for (int sl = 0; sl < 2; ++sl)
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          vf[sl][d][e] =
              lds_get_tr16(va[d & 1] + off + (S + (16 * sl + 8 * e) * RB + 128 * (d >> 1)));
    // register r holds key ks + 4 half + c(r), c(r) = (r & 3) + 8 (r >> 2)
    const bool whole = ks >= ilo && ks + 32 <= ihi;
    // No key after its row: the bias -slope (row - key) is slope c(r), the same for every
    // lane, plus a lane's own part, which joins the offset; in units of the raw scores the
    // first is one multiply-add by a constant
    const float dq = static_cast<float>(qi - ks - 4 * half);
    float lane_bias = MODE == kBiased ? -slope * dq : 0.f;
    if (MODE == kBiased) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fmaf(ratio, (r & 3) + 8 * (r >> 2), s[r]);
    }
    if (MODE == kAny) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float c = (r & 3) + 8 * (r >> 2);
        const float z = a.cap_x2 > 0.f ? softcap_log2(s[r] * a.cap_x2, a.cap_log2)
                                       : s[r] * a.scale_log2;
        s[r] = fmaf(-slope, fabsf(dq - c), z);
      }
    }
    uint32_t seen = 0xffffffffu;  // bit c(r): this lane's row sees the key
    if (!whole) {
      const uint64_t one = 1;
      seen = static_cast<uint32_t>((one << min(max(hi - ks, 0), 32)) -
                                   (one << min(max(lo - ks, 0), 32))) >> (4 * half);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t v = __builtin_amdgcn_sbfe(seen, (r & 3) + 8 * (r >> 2), 1);
        s[r] = __uint_as_float((v & __float_as_uint(s[r])) | (~v & 0xff800000u));  // else -inf
      }
    }
    if (careful) {
#pragma unroll
      for (int i = 0; i < 4 * ND; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          (&vf[0][0][0])[i][e] &= ~not_finite((&vf[0][0][0])[i][e]);
    }
    if ((MODE == kPlain || MODE == kBiased) && careful) {  // the products, rounded
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], a.scale_log2, lane_bias);
      lane_bias = 0.f;
    }
    float x = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) x = fmaxf(x, s[r]);
    if (MODE == kBiased) x = fmaf(x, factor, lane_bias);
    // the cap ascends, so the largest score is the largest capped one.  A visible -inf is
    // capped to -cap, so whether there is a score says the mask (bits c(r)), not the value
    if (MODE == kCapped)
      x = seen & 0x0f0f0f0fu ? softcap_log2(x * a.cap_x2, a.cap_log2) : -INFINITY;
    {  // the other lane half's (lanes l and l ^ 32 hold one row)
      const auto sw =
          __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      x = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    }
    if (MODE == kPlain) x *= factor;
    // the offset moves when some row's largest score passes it by 8 (log2), decided by
    // the wave, so most sub-tiles rescale nothing
    if (__ballot(x - 8.f > m)) {
      const float m_new = fmaxf(m, x);
      const float alpha = exp2_fast(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
    }
    // weights rounded to bf16 (a second product for what that leaves would add half to the
    // matrix work, which bounds long prompts) and the sum of the rounded ones, so that they
    // still average: 2^-8 of a weight at the most; the error against 64 bits of 16384 rows,
    // mostly the store's, is 2.0e-3 of the output where fp32 weights give 1.5e-3
    float p[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (MODE == kPlain) p[r] = exp2_fast(fmaf(s[r], factor, -m));
      if (MODE == kCapped) p[r] = exp2_fast(softcap_log2(s[r] * a.cap_x2, a.cap_log2) - m);
      if (MODE == kBiased) p[r] = exp2_fast(fmaf(s[r], factor, lane_bias - m));
      if (MODE == kAny) p[r] = exp2_fast(s[r] - m);
    }
    if (MODE == kCapped && !whole) {  // -inf is capped to -cap: out of the sum here
#pragma unroll
      for (int r = 0; r < 16; ++r)
        p[r] = __uint_as_float(__float_as_uint(p[r]) &
                               __builtin_amdgcn_sbfe(seen, (r & 3) + 8 * (r >> 2), 1));
    }
    const uint4 pb[2] = {pack8_bf16(p), pack8_bf16(p + 8)};
    const bf16x2v one = __builtin_bit_cast(bf16x2v, 0x3f803f80u);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      for (const uint32_t w : {pb[i].x, pb[i].y, pb[i].z, pb[i].w})
        l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, w), one, l, false);
#pragma unroll
    for (int sl = 0; sl < 2; ++sl)
#pragma unroll
      for (int d = 0; d < ND; ++d)
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            as_bf16x8(uint4{vf[sl][d][0].x, vf[sl][d][0].y, vf[sl][d][1].x, vf[sl][d][1].y}),
            as_bf16x8(pb[sl]), acc[d], 0, 0, 0);
  };

  for (;;) {
    m = kNoScore;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    issue(t_lo, 0);
    for (int tile = t_lo; tile <= t_hi; ++tile) {
      const int st = (tile - t_lo) & 1;
      // this wave's copies of the tile have landed; after the barrier every wave's have,
      // and every wave is done with the other stage, which the next tile then fills
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tile < t_hi) issue(tile + 1, st ^ 1);
      const int ks = tile * PN;
      const uint32_t off = st * 2 * TB;
      if (KW == 1) {
        sub_tile(Int<0>{}, ks, off);
        sub_tile(Int<1>{}, ks + 32, off);
      } else {
        sub_tile(Int<0>{}, ks + 32 * part, off + 32 * RB * part);
      }
    }
    if (careful) break;
    float bad = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) bad = fmaf(acc[d][r], 0.f, bad);
    // NaN: some value is not finite, or a weight overflowed
    const bool far = (MODE == kPlain || MODE == kBiased) && m != kNoScore && !(fabsf(m) < kFar);
    if (!__syncthreads_or(mine && (bad != 0.f || far))) break;
    careful = true;
    factor = 1.f;
  }
  if (careful) {
    // the values left out, straight from memory: this lane's dims 8 e + 4 half .. + 3 of
    // every key that its row sees
    for (int key = wlo; key < whi; key += 4) {
#pragma unroll
      for (int e = 0; e < 4 * ND; ++e) {
        uint2 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = *reinterpret_cast<const uint2*>(vb + min(key + i, whi - 1) * a.vr + 4 * half + 8 * e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t sees = key + i >= lo && key + i < hi ? 0xffffffffu : 0u;
          const uint32_t f[2] = {w[i].x & not_finite(w[i].x) & sees,
                                 w[i].y & not_finite(w[i].y) & sees};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[e >> 2][4 * (e & 3) + j] +=
                __uint_as_float(j & 1 ? f[j >> 1] & 0xffff0000u : f[j >> 1] << 16);
        }
      }
    }
  }

  float l_tot = l + __shfl_xor(l, 32, kWave);
  if constexpr (KW > 1) {
    // the (m, l, acc) of the KW waves of each 32 rows joined, HD / LPR dims a thread
    constexpr int PMR = 128 / KW, LPR = 256 / PMR, NO = HD / LPR, LD = HD + 4;
    float* const so = reinterpret_cast<float*>(smem);
    float* const sm = so + 128 * LD;
    float* const sl = sm + 128;
    static_assert((128 * LD + 256) * 4 <= 2 * 2 * TB + (KW == 2 ? 4096 : 0), "the join fits");
    // the barrier of the check above is behind every read of a stage, but for a second run
    if (careful) __syncthreads();
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<float4*>(so + (32 * wave + col) * LD + 32 * d + 8 * g4 + 4 * half) =
            make_float4(acc[d][4 * g4], acc[d][4 * g4 + 1], acc[d][4 * g4 + 2],
                        acc[d][4 * g4 + 3]);
    if (half == 0) {
      sm[32 * wave + col] = mine ? m : NAN;  // a row of no document: not stored
      sl[32 * wave + col] = l_tot;
    }
    __syncthreads();
    const int row = threadIdx.x / LPR, c0 = (threadIdx.x % LPR) * NO;
    const int at = (row >> 5) * KW * 32 + (row & 31);  // of its first wave
    float mx = sm[at];
    if (mx != mx) return;
#pragma unroll
    for (int w = 1; w < KW; ++w) mx = fmaxf(mx, sm[at + 32 * w]);
    float o[NO], den = 0.f;
#pragma unroll
    for (int i = 0; i < NO; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const float e = exp2_fast(sm[at + 32 * w] - mx);
      // the sum of a part without weight is finite or, of a visible NaN score alone (no
      // maximum sees one), NaN, and then the row's is; its infinities, which the others
      // have too, would add NaN
      den = fmaf(sl[at + 32 * w], e, den);
      if (e == 0.f) continue;
#pragma unroll
      for (int i = 0; i < NO; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(so + (at + 32 * w) * LD + c0 + i);
        o[i] = fmaf(v.x, e, o[i]);
        o[i + 1] = fmaf(v.y, e, o[i + 1]);
        o[i + 2] = fmaf(v.z, e, o[i + 2]);
        o[i + 3] = fmaf(v.w, e, o[i + 3]);
      }
    }
    const float inv = 1.0f / den;
#pragma unroll
    for (int i = 0; i < NO; ++i) o[i] *= inv;
    uint16_t* dst = a.o + (static_cast<long long>(q0 + row) * a.hq + h) * HD + c0;
#pragma unroll
    for (int i = 0; i < NO; i += 8) *reinterpret_cast<uint4*>(dst + i) = pack8_bf16(o + i);
    return;
  }
  // rows put together in LDS, so that whole ones are stored: a lane holds 4 dims of every 8
  // (8192 rows x 16 heads x 64: 5 us of 34 less).  The barrier of the check above is
  // behind every read of a stage, but for a second run
  if (careful) __syncthreads();
  constexpr int LB = RB + 16;  // bytes a row
  uint8_t* const so = smem + 32 * LB * wave;
  static_assert(128 * LB <= 2 * 2 * TB, "the rows fit the stages");
  const float inv = 1.0f / l_tot;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      *reinterpret_cast<uint2*>(so + col * LB + 2 * (32 * d + 8 * g4 + 4 * half)) =
          make_uint2(pack_bf2(acc[d][4 * g4] * inv, acc[d][4 * g4 + 1] * inv),
                     pack_bf2(acc[d][4 * g4 + 2] * inv, acc[d][4 * g4 + 3] * inv));
  wave_lds_order();
#pragma unroll
  for (int i = 0; i < CH / 2; ++i) {
    const int row = (64 / CH) * i + lane / CH, c = lane % CH;
    if ((rows >> row) & 1u)
      *reinterpret_cast<uint4*>(
          a.o + (static_cast<long long>(q0 + 32 * rg + row) * a.hq + h) * HD + 8 * c) =
          *reinterpret_cast<const uint4*>(so + row * LB + 16 * c);
  }
}

template <int HD, int MODE>
int32_t launch_packed(const PackedArgs& a, hipStream_t s) {
  const long long wide = static_cast<long long>((a.N + 127) / 128) * a.hq;
  const int cus = compute_units();
  const int kw = wide <= cus / 2 ? 4 : wide <= 2 * cus ? 2 : 1;
  const long long units = static_cast<long long>((a.N + 128 / kw - 1) / (128 / kw)) * a.hkv;
  const long long blocks = (units + 7) / 8 * 8 * a.G;
  LLMY_REQUIRE(blocks < (1ll << 31));
  const dim3 grid(static_cast<unsigned>(blocks));
  if (kw == 4)
    hipLaunchKernelGGL((packed_attn_kernel<HD, MODE, 4>), grid, dim3(256), 0, s, a);
  else if (kw == 2)
    hipLaunchKernelGGL((packed_attn_kernel<HD, MODE, 2>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((packed_attn_kernel<HD, MODE, 1>), grid, dim3(256), 0, s, a);
  return launch_status();
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
  LLMY_REQUIRE((head_dim == 64 || head_dim == 128) && window >= 0 && scale_ok(scale, softcap));
  LLMY_REQUIRE(N < (1 << 30));  // positions and tile ends are 32-bit
  if (N == 0 || docs == 0) return 0;
  LLMY_REQUIRE(q && k && v && out && cu_seqlens);
  LLMY_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16));
  for (const int64_t x : {q_row, q_head, k_row, k_head, v_row, v_head})
    LLMY_REQUIRE(x >= 0 && x % 8 == 0);
  LLMY_REQUIRE(k_row < (1 << 22) && v_row < (1 << 22));  // a tile's offsets are 32-bit
  // out is written while other workgroups still read
  const int64_t out_n = static_cast<int64_t>(N) * Hq * head_dim;
  LLMY_REQUIRE(apart(q, rows_extent(q_row, q_head, N, Hq, head_dim), out, out_n) &&
               apart(k, rows_extent(k_row, k_head, N, Hkv, head_dim), out, out_n) &&
               apart(v, rows_extent(v_row, v_head, N, Hkv, head_dim), out, out_n));
  PackedArgs a{};
  a.q = q; a.qr = q_row; a.qh = q_head;
  a.k = k; a.kr = k_row; a.kh = k_head;
  a.v = v; a.vr = v_row; a.vh = v_head;
  a.o = out; a.cu = cu_seqlens; a.prefix = prefix; a.slopes = slopes;
  const float log2e = 1.4426950408889634f;
  a.scale_log2 = scale * log2e;
  a.cap_log2 = softcap * log2e;
  a.cap_x2 = softcap > 0.f ? 2.f * log2e * scale / softcap : 0.f;
  a.N = N; a.docs = docs; a.hq = Hq; a.hkv = Hkv; a.G = Hq / Hkv; a.window = window;
  const hipStream_t st = as_stream(stream);
  // a scale of 0 would turn the masked scores' -inf into NaN in the exponent of kPlain
  const bool cap = softcap > 0.f;
  const int mode = scale == 0.f || (slopes && (cap || prefix || scale < 1e-6f)) ? kAny
                   : slopes ? kBiased : cap ? kCapped : kPlain;
  const auto launch = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    return mode == kPlain    ? launch_packed<HD, kPlain>(a, st)
           : mode == kCapped ? launch_packed<HD, kCapped>(a, st)
           : mode == kBiased ? launch_packed<HD, kBiased>(a, st)
                             : launch_packed<HD, kAny>(a, st);
  };
  return head_dim == 64 ? launch(Int<64>{}) : launch(Int<128>{});
}
