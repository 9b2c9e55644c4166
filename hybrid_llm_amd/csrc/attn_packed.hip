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

constexpr int kPM = 128;  // rows per workgroup
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
template <int HD, bool SCORE>
__global__ __launch_bounds__(256, HD == 64 ? 4 : 2) void packed_attn_kernel(const PackedArgs a) {
  constexpr int ND = HD / 32;   // 32-dim output tiles
  constexpr int NS = HD / 16;   // 16-dim slices of the score product
  constexpr int RB = 2 * HD;    // bytes of a staged row
  constexpr int TB = kPN * RB;  // bytes of a staged K or V tile
  __shared__ __align__(1024) uint8_t smem[2 * 2 * TB];
  __shared__ int range[2][4];

  const int nblk = (a.N + kPM - 1) / kPM;
  const int h = blockIdx.x % a.hq;
  const int q0 = (nblk - 1 - static_cast<int>(blockIdx.x / a.hq)) * kPM;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5;
  const int col = lane & 31;
  const int qi = q0 + 32 * wave + col;  // this lane's row

  // its document by bisection, its keys [lo, lo + n); none for a row of no document
  int lo = 0, hi = 0;
  bool mine = false;
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
      mine = true;
      lo = a.window > 0 ? max(first, qi - min(a.window - 1, qi)) : first;
      hi = max(qi + 1, first + two_way);
    }
  }
  const unsigned n = hi - lo;
  // the wave's rows see keys in [wlo, whi), all of them those in [ilo, ihi)
  const int big = 0x7fffffff;
  const int wlo = wave_min_i(mine ? lo : big), whi = wave_max_i(mine ? hi : 0);
  const int ilo = wave_max_i(mine ? lo : 0), ihi = wave_min_i(mine ? hi : big);
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

  u32x4 qf[NS];
  {
    const uint16_t* qp = a.q + min(qi, a.N - 1) * a.qr + h * a.qh + 8 * half;
#pragma unroll
    for (int t = 0; t < NS; ++t) qf[t] = *reinterpret_cast<const u32x4*>(qp + 16 * t);
  }
  float slope = 0.f;
  if (SCORE && a.slopes) slope = a.slopes[h] * 1.4426950408889634f;
  const float sc = SCORE ? 1.f : a.scale_log2;

  f32x16v acc[ND];
  float m = -1e38f, l = 0.f;  // the exponent's offset (scaled, log2) and the sum of weights
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;

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
    kdo[i] = 2 * r * kr + 16 * (sl ^ (r & 7));
    vdo[i] = 2 * r * vr + 16 * (sl ^ (2 * (r & 3)));
  }
  const uint32_t sbase = lds_addr(smem);
  auto issue = [&](int tile, int st) __attribute__((always_inline)) {
    const int kt = tile * kPN;
    const uint32_t dst = sbase + st * 2 * TB + wave * 1024;
    const uint16_t* kp = kb + kt * a.kr;
    const uint16_t* vp = vb + kt * a.vr;
    if (kt + kPN <= a.N) {
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
  bool dirty = false;
  auto sub_tile = [&](auto subc, int tile, uint32_t off) __attribute__((always_inline)) {
    constexpr int S = decltype(subc)::value * 32 * RB;
    const int ks = tile * kPN + 32 * decltype(subc)::value;
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
    // register r holds key ks + (r & 3) + 8 (r >> 2) + 4 half
    const int k0 = ks + 4 * half;
    if (SCORE) {
      const float dq = static_cast<float>(qi - k0);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float c = (r & 3) + 8 * (r >> 2);
        float z = a.cap_x2 > 0.f ? softcap_log2(s[r] * a.cap_x2, a.cap_log2)
                                 : s[r] * a.scale_log2;
        if (a.slopes) z = fmaf(-slope, fabsf(dq - c), z);
        s[r] = z;
      }
    }
    const bool whole = ks >= ilo && ks + 32 <= ihi;
    if (!whole) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int cr = (r & 3) + 8 * (r >> 2);
        s[r] = static_cast<unsigned>(k0 + cr - lo) < n ? s[r] : -INFINITY;
      }
      // values that are not finite are left out here; the rows that see them get them
      // after the last tile
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4 * ND; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) top |= ((&vf[0][0][0])[i][e] & 0x7f807f80u) + 0x00800080u;
      if (__ballot((top & 0x80008000u) != 0)) {
        dirty = true;
#pragma unroll
        for (int i = 0; i < 4 * ND; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            (&vf[0][0][0])[i][e] &= ~not_finite((&vf[0][0][0])[i][e]);
      }
    }
    float x = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) x = fmaxf(x, s[r]);
    {  // the other lane half's (lanes l and l ^ 32 hold one row)
      const auto sw =
          __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      x = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    }
    // the offset moves when some row's largest score passes it by 8 (log2), decided by
    // the wave, so most sub-tiles rescale nothing
    if (__ballot(fmaf(x, sc, -8.f) > m)) {
      const float m_new = fmaxf(m, x * sc);
      const float alpha = exp2_fast(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
    }
    // weights, rounded, and the sum of the rounded ones
    float p[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = exp2_fast(fmaf(s[r], sc, -m));
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

  issue(t_lo, 0);
  for (int tile = t_lo; tile <= t_hi; ++tile) {
    const int st = (tile - t_lo) & 1;
    // this wave's copies of the tile have landed; after the barrier every wave's have,
    // and every wave is done with the other stage, which the next tile then fills
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tile < t_hi) issue(tile + 1, st ^ 1);
    sub_tile(Int<0>{}, tile, st * 2 * TB);
    sub_tile(Int<1>{}, tile, st * 2 * TB);
  }

  if (dirty) {
    // the values left out, straight from memory: this lane's dims 8 e + 4 half .. + 3 of
    // every key that its row sees (one that was added before adds nothing new: inf + inf)
    for (int key = wlo; key < whi; ++key) {
      const uint16_t* row = vb + key * a.vr + 4 * half;
      const uint32_t sees = static_cast<unsigned>(key - lo) < n ? 0xffffffffu : 0u;
#pragma unroll
      for (int e = 0; e < 4 * ND; ++e) {
        const uint2 w = *reinterpret_cast<const uint2*>(row + 8 * e);
        const uint32_t f[2] = {w.x & not_finite(w.x) & sees, w.y & not_finite(w.y) & sees};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[e >> 2][4 * (e & 3) + i] +=
              __uint_as_float(i & 1 ? f[i >> 1] & 0xffff0000u : f[i >> 1] << 16);
      }
    }
  }

  const float l_tot = l + __shfl_xor(l, 32, kWave);
  if (!mine) return;
  const float inv = 1.0f / l_tot;
  uint16_t* orow = a.o + (static_cast<long long>(qi) * a.hq + h) * HD;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const int dim = 32 * d + 8 * g4 + 4 * half;
      *reinterpret_cast<uint2*>(orow + dim) =
          make_uint2(pack_bf2(acc[d][4 * g4] * inv, acc[d][4 * g4 + 1] * inv),
                     pack_bf2(acc[d][4 * g4 + 2] * inv, acc[d][4 * g4 + 3] * inv));
    }
}

template <int HD, bool SCORE>
void launch_packed(const PackedArgs& a, unsigned blocks, hipStream_t s) {
  hipLaunchKernelGGL((packed_attn_kernel<HD, SCORE>), dim3(blocks), dim3(256), 0, s, a);
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
  const long long blocks = static_cast<long long>((N + kPM - 1) / kPM) * Hq;
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
    score ? launch_packed<64, true>(a, grid, st) : launch_packed<64, false>(a, grid, st);
  else
    score ? launch_packed<128, true>(a, grid, st) : launch_packed<128, false>(a, grid, st);
  return launch_status();
}
