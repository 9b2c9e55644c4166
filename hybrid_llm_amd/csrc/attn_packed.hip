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
// A sub-tile that is masked for some row may hold anything there, NaN and infinities
// included, and 0 * inf is NaN in the product: a masked sub-tile whose V has such a
// value takes its finite part through the product, then adds the infinities of the
// rows that see them (a product of the visibility with the places of +inf, -inf, NaN).
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

// SCORE: scores are capped or biased (otherwise the scale goes into the exponent).
template <int HD, bool SCORE>
__global__ __launch_bounds__(256) void packed_attn_kernel(const PackedArgs a) {
  constexpr int ND = HD / 32;     // 32-dim output tiles
  constexpr int NS = HD / 16;     // 16-dim slices of the score product
  constexpr int TILE = kPN * HD;  // elements of a staged K or V tile
  constexpr int RB = 2 * HD;      // bytes of a staged row
  __shared__ __align__(1024) uint16_t smem[2 * 2 * TILE];
  __shared__ int range[2][4];

  const int nblk = (a.N + kPM - 1) / kPM;
  const int h = blockIdx.x % a.hq;
  const int q0 = (nblk - 1 - static_cast<int>(blockIdx.x / a.hq)) * kPM;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int half = lane >> 5;
  const int col = lane & 31;
  const int qi = q0 + 32 * wave + col;

  // this lane's row: its document by bisection, its keys [lo, hi); none for a row of no
  // document
  int lo = 0, hi = 0;
  bool mine = false;
  if (qi < a.N) {
    int x = 0, y = a.docs + 1;  // the first entry past qi
    while (x < y) {
      const int mid = (x + y) >> 1;
      if (a.cu[mid] <= qi) x = mid + 1;
      else y = mid;
    }
    if (x > 0 && x <= a.docs) {
      const int first = max(a.cu[x - 1], 0), end = min(a.cu[x], a.N);
      const int two_way = a.prefix ? min(max(a.prefix[x - 1], 0), end - first) : 0;
      mine = true;
      lo = a.window > 0 ? max(first, qi - min(a.window - 1, qi)) : first;
      hi = max(qi + 1, first + two_way);
    }
  }
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
  const int t_lo = glo / kPN, t_hi = (ghi - 1) / kPN;

  uint4 qf[NS];
  {
    const uint16_t* qp = a.q + min(qi, a.N - 1) * a.qr + h * a.qh + 8 * half;
#pragma unroll
    for (int t = 0; t < NS; ++t) qf[t] = *reinterpret_cast<const uint4*>(qp + 16 * t);
  }
  float slope = 0.f;
  if (SCORE && a.slopes) slope = a.slopes[h] * 1.4426950408889634f;

  f32x16v acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  const float sc = SCORE ? 1.f : a.scale_log2;

  // DMA lanes, as in attn_prefill.hip; rows past the last re-read it (no row sees them)
  constexpr int CH = HD / 8;
  constexpr int RPB = 64 / CH;
  constexpr int BPW = kPN / RPB / 4;
  const uint16_t* kb = a.k + (h / a.G) * a.kh;
  const uint16_t* vb = a.v + (h / a.G) * a.vh;
  const int kr = static_cast<int>(a.kr), vr = static_cast<int>(a.vr);
  auto issue = [&](int tile, int st) {
    const int kt = tile * kPN;
    uint16_t* sk = smem + st * 2 * TILE;
    const uint16_t* kp = kb + kt * a.kr;
    const uint16_t* vp = vb + kt * a.vr;
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      const int r = RPB * (wave + 4 * i) + lane / CH, sl = lane % CH;
      const int row = min(r, a.N - 1 - kt);
      dma16(kp + row * kr + 8 * (sl ^ (r & 7)), sk + (wave + 4 * i) * 512);
      dma16(vp + row * vr + 8 * (sl ^ (2 * (r & 3))), sk + TILE + (wave + 4 * i) * 512);
    }
  };
  const uint32_t sbase = lds_addr(smem);
  uint32_t koff[NS], voff[ND];
#pragma unroll
  for (int t = 0; t < NS; ++t) koff[t] = col * RB + 16 * ((2 * t + half) ^ (col & 7));
  {
    const int y = lane & 15, g = lane >> 4, i = y >> 2;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int dim0 = 32 * d + 16 * (g & 1) + 4 * (y & 3);
      voff[d] = (4 * half + i) * RB + 16 * ((dim0 >> 3) ^ (2 * i)) + 2 * (dim0 & 7);
    }
  }
  issue(t_lo, 0);
  for (int tile = t_lo; tile <= t_hi; ++tile) {
    const int st = (tile - t_lo) & 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tile < t_hi) issue(tile + 1, st ^ 1);
    const uint32_t kst = sbase + st * 4 * TILE, vst = kst + 2 * TILE;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const int ks = tile * kPN + 32 * sub;
      if (ks >= whi || ks + 32 <= wlo) continue;  // no row of this wave sees it
      f32x16v s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
      u32x4 kf[NS];
#pragma unroll
      for (int t = 0; t < NS; ++t) kf[t] = lds_b128(kst + 32 * sub * RB + koff[t]);
#pragma unroll
      for (int t = 0; t < NS; t += 4) lds_settle4(kf + t);
#pragma unroll
      for (int t = 0; t < NS; ++t)
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kf[t]),
                                                    as_bf16x8(qf[t]), s, 0, 0, 0);
      u32x2 vf[2][ND][2];
#pragma unroll
      for (int sl = 0; sl < 2; ++sl)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const uint32_t va = vst + (32 * sub + 16 * sl) * RB + voff[d];
          vf[sl][d][0] = lds_tr16(va);
          vf[sl][d][1] = lds_tr16(va + 8 * RB);
        }
      if (SCORE) {
        const float dq = static_cast<float>(qi - ks - 4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float c = (r & 3) + 8 * (r >> 2);
          float z = a.cap_x2 > 0.f ? softcap_log2(s[r] * a.cap_x2, a.cap_log2)
                                   : s[r] * a.scale_log2;
          if (a.slopes) z = fmaf(-slope, fabsf(dq - c), z);
          s[r] = z;
        }
      }
      // register r holds key ks + (r & 3) + 8 (r >> 2) + 4 half
      const bool whole = ks >= ilo && ks + 32 <= ihi;
      if (!whole) {
        const int k0 = ks + 4 * half;
        const unsigned n = hi - lo;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int cr = (r & 3) + 8 * (r >> 2);
          s[r] = static_cast<unsigned>(k0 + cr - lo) < n ? s[r] : -INFINITY;
        }
      }
      float mloc = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) mloc = fmaxf(mloc, s[r]);
      {  // the other lane half's maximum (lanes l and l ^ 32 hold one row)
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mloc),
                                                         __float_as_uint(mloc), false, false);
        mloc = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      }
      // lazy rescale: the offset moves when some row's maximum passes it by 8 (log2)
      if (__ballot(!(mloc * sc <= m_run * sc + 8.f))) {
        const float m_new = fmaxf(m_run, mloc);
        const float alpha = m_new == -INFINITY ? 1.f : exp2_fast((m_run - m_new) * sc);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
      }
      const float m_sc = m_run == -INFINITY ? 0.f : m_run * sc;
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = exp2_fast(fmaf(s[r], sc, -m_sc));
      const uint4 pb[2] = {pack8_bf16(p), pack8_bf16(p + 8)};
#pragma unroll
      for (int sl = 0; sl < 2; ++sl) {  // the sum of the rounded weights
        unpack8(pb[sl], p);
#pragma unroll
        for (int j = 0; j < 8; ++j) l_run += p[j];
      }
#pragma unroll
      for (int i = 0; i < ND / 2; ++i) lds_settle_v(&vf[0][0][0] + 8 * i);
      if (!whole) {  // values that are not finite, where some row does not see their key
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4 * ND; ++i) {
          const u32x2 w = (&vf[0][0][0])[i];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            top |= static_cast<uint32_t>((w[e] & 0x7f80u) == 0x7f80u) |
                   static_cast<uint32_t>((w[e] & 0x7f800000u) == 0x7f800000u);
        }
        if (__ballot(top)) {
          const int k0 = ks + 4 * half;
          const unsigned n = hi - lo;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            f32x16v up, dn;
#pragma unroll
            for (int r = 0; r < 16; ++r) up[r] = dn[r] = 0.f;
#pragma unroll
            for (int sl = 0; sl < 2; ++sl) {
              uint32_t pu[4], pd[4], see[4];
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                uint32_t& x = reinterpret_cast<uint32_t*>(&vf[sl][d][0])[w];
                uint32_t keep = 0xffffffffu, u = 0, m = 0, vis = 0;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t b = (x >> (16 * e)) & 0xffffu;
                  if ((b & 0x7f80u) == 0x7f80u) {
                    keep &= ~(0xffffu << (16 * e));
                    if (b != 0xff80u) u |= 0x3f80u << (16 * e);  // 1 where +inf or NaN
                    if (b != 0x7f80u) m |= 0x3f80u << (16 * e);  // 1 where -inf or NaN
                  }
                  const int j = 2 * w + e, r = 8 * sl + j, cr = (r & 3) + 8 * (r >> 2);
                  if (static_cast<unsigned>(k0 + cr - lo) < n) vis |= 0x3f80u << (16 * e);
                }
                x &= keep;
                pu[w] = u;
                pd[w] = m;
                see[w] = vis;
              }
              const bf16x8 sv = as_bf16x8(uint4{see[0], see[1], see[2], see[3]});
              up = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  as_bf16x8(uint4{pu[0], pu[1], pu[2], pu[3]}), sv, up, 0, 0, 0);
              dn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  as_bf16x8(uint4{pd[0], pd[1], pd[2], pd[3]}), sv, dn, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              acc[d][r] += up[r] > 0.f ? INFINITY : 0.f;
              acc[d][r] += dn[r] > 0.f ? -INFINITY : 0.f;
            }
          }
        }
      }
#pragma unroll
      for (int sl = 0; sl < 2; ++sl)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const uint4 va = uint4{vf[sl][d][0].x, vf[sl][d][0].y, vf[sl][d][1].x, vf[sl][d][1].y};
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(va), as_bf16x8(pb[sl]),
                                                           acc[d], 0, 0, 0);
        }
    }
  }

  const float l_tot = l_run + __shfl_xor(l_run, 32, kWave);
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
  for (const int64_t st : {q_row, q_head, k_row, k_head, v_row, v_head})
    LLMY_REQUIRE(st >= 0 && st % 8 == 0);
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
  const dim3 grid(static_cast<unsigned>(blocks));
  const hipStream_t s = as_stream(stream);
  // a scale of 0 would turn the masked scores' -inf into NaN in the exponent
  const bool score = softcap > 0.f || slopes || scale == 0.f;
  if (head_dim == 64) {
    if (score) hipLaunchKernelGGL((packed_attn_kernel<64, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((packed_attn_kernel<64, false>), grid, dim3(256), 0, s, a);
  } else {
    if (score) hipLaunchKernelGGL((packed_attn_kernel<128, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((packed_attn_kernel<128, false>), grid, dim3(256), 0, s, a);
  }
  return launch_status();
}
