// Attention of one or several new tokens per sequence over a paged cache held in 4 bits:
//   z_j = scale q . k_j, capped: c tanh(z / c), less slope_h (e_t - 1 - j);
//   o = sum_j softmax(z)_j v_j over the positions max(0, e_t - W) <= j < e_t,
// e_t = len - (T - 1 - t) for token t of T, query head h reading key-value head
// h / (Hq / Hkv).  Cache and page table as in paged.hpp.
//
// Bound by the read of K and V, 17 / 32 of a byte a value.  A key-value head's T G query
// rows (G = Hq / Hkv) are columns of 16 x 16 x 32 MFMAs, up to 16 NT of them a wave, so
// several drafted tokens cost the bytes of one.
//   * codes become bf16 by the chip's conversion under a block scale, two values an
//     instruction and without rounding.  (The scaled matrix products that take 4-bit operands
//     themselves align a block's products to its largest and lose what lies 2^-17 under it.)
//   * S^T = K Q^T: a lane's K operand is its key's 16 bytes (8 for 64 dims) as they lie in
//     the cache, loaded straight to registers, three steps ahead.  Lane l (g = l / 16)
//     gets keys 4 g + r of a 16-key tile for column l % 16; two such tiles are, register
//     by register, the B operand of a 32-key product O^T += V^T P^T under the key order
//     4 g + j, 16 + 4 g + j.
//   * V, loaded the same way, is put in bf16 into the wave's own 32 rows of LDS, whose
//     transposing reads give V^T in that order.  A block scale belongs to a key and 32 dims,
//     so scaling V costs nothing beyond its conversion, and scaling the weights would
//     take one set of them per block.
//   * a wave works alone and waits for no other; waves share a head tile where tables are
//     short, and otherwise each takes an equal run of the flat list of all (sequence, head
//     tile, step), found from the lengths on the device: partials of heads that are cut go to
//     the workspace, and a second kernel joins them.
// Masked keys (past the length, before the window, in a page that the table does not name)
// have their scores set to -inf and their V rows zeroed, so nothing that such a place holds
// reaches a sum.  A block of V that is NaN counts as zeros in the product, and as NaN
// afterwards for the rows that see its key.
//
// Weights enter the product as the sum of two bf16, 16 bits of each.
#include "common.hpp"
#include "abi_util.hpp"
#include "attn_tile.hpp"
#include "paged.hpp"

namespace llmy {

typedef const int32_t __attribute__((address_space(4)))* const_i32;

__device__ __forceinline__ int32_t uniform_at(const int32_t* p, long long i) {
  return reinterpret_cast<const_i32>(reinterpret_cast<uintptr_t>(p))[i];
}

constexpr int kMxStep = 32;      // keys a step
constexpr int kMxAhead = 3;      // steps in registers
constexpr float kMxLowest = -3.402823466e38f;
constexpr uint32_t kMxOne = 127u;   // the scale byte of 1
constexpr uint32_t kMxLost = 253u;  // from here on codes pass fp32, or the block is NaN

struct Mx4Args {
  const uint16_t* q;
  long long qb, qt, qh;        // strides of q by sequence, token and head (elements)
  const uint8_t *kc, *vc, *ks, *vs;
  const int32_t *table, *lengths;
  uint16_t* out;               // [B, T, Hq, HD]
  float *po, *pml;             // partials: O [2 runs, GT, HD] and (m, l) [2 runs, GT, 2]
  int32_t* starts;             // [B + 1]: steps of the sequences before each, and of all
  const float* slopes;
  float scale_log2, cap_log2, cap_x2;
  int B, T, hq, hkv, G, HT, GT;  // T G columns in HT tiles of GT <= 16 NT
  int width, shift, pages, window, cap_len;
  int runs;
};

struct MxSeq {
  int len, lo, s0, s1;         // positions [lo, len) seen by any token, steps [s0, s1)
};

__device__ __forceinline__ MxSeq mx_seq(int len, const Mx4Args& a) {
  MxSeq s;
  s.len = min(max(len, 0), a.cap_len);
  s.lo = a.window > 0 ? static_cast<int>(max(0ll, s.len - (a.T - 1ll) - a.window)) : 0;
  s.s0 = s.lo / kMxStep;
  s.s1 = static_cast<int>((static_cast<unsigned>(s.len) + kMxStep - 1) / kMxStep);
  return s;
}

// Steps of all sequences (the host sees to it that they fit 31 bits), as sums over 64
// blocks of `per` sequences, one per lane.
struct MxScan {
  int before, upto, total;  // this lane's block: exclusive and inclusive sums
  int per;
};

__device__ __forceinline__ MxScan mx_scan(const Mx4Args& a, int lane) {
  MxScan r;
  r.per = (a.B + kWave - 1) / kWave;
  int n = 0;
  const int b1 = min(a.B, (lane + 1) * r.per);
  for (int b = lane * r.per; b < b1; ++b) {
    const MxSeq s = mx_seq(a.lengths[b], a);
    n += s.s1 - s.s0;
  }
  r.upto = n;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(r.upto, d, kWave);
    if (lane >= d) r.upto += o;
  }
  r.before = r.upto - n;
  r.total = __builtin_amdgcn_readlane(r.upto, kWave - 1);
  return r;
}

__device__ __forceinline__ int mx_run(long long total, int runs) {
  const long long q = (total + runs - 1) / runs;
  return static_cast<int>(q > 1 ? q : 1);
}

// 1 over a row's sum of weights; without a visible key (m -inf) 0, with only scores of -inf
// NaN.
__device__ __forceinline__ float mx_share(float m, float l) {
  return l != 0.f ? 1.f / l : m == -INFINITY ? 0.f : NAN;
}

// A part's sum under its weight beside the others, which may have vanished: infinities and
// NaN stay all the same.
__device__ __forceinline__ float mx_weighted(float x, float f) {
  return f != 0.f ? x * f : fabsf(x) < INFINITY ? 0.f : x;
}

// V rows lie in LDS with their 16-byte chunks XOR-swizzled: 8 consecutive rows put one chunk
// into 8 different places, and the two chunks of 4 rows that a transposing read takes into 8.
__device__ __forceinline__ int mx_swz(int row) { return 2 * (row & 3) | ((row >> 2) & 1); }

// What one step loads: a 16-key tile's codes (a lane: its key's quarter of the dims) and the
// scale byte over them, twice; V's codes by 16 bytes with theirs.
template <int HD>
struct MxStage {
  static constexpr int NV = HD / 64;
  uint32_t k[2][HD / 32];
  uint32_t ks[2];
  u32x4 v[NV];
  uint32_t vs[NV];
};

// W waves: 1: a run of the flat list; more: a head tile, each wave every W-th of its steps.
template <int HD, int NT, int W>
__global__ __launch_bounds__(64 * W, W > 1 ? W / 4 : NT == 1 ? 2 : 1)
void mx4_attn_kernel(const Mx4Args a) {
  constexpr int RB = 2 * HD;                  // bytes of a V row in LDS
  constexpr int CB = HD / 2, SB = HD / 32;    // bytes of a stored row: codes, scales
  constexpr int NS = HD / 32;                 // 32-dim slices of the score product
  constexpr int ND = HD / 16;                 // 16-dim output tiles
  constexpr int NV = MxStage<HD>::NV;
  constexpr int CPR = HD / 32;                // 16-byte chunks of a stored row
  constexpr int LD = HD + 4;                  // of a column's part in the waves' join
  constexpr int TILE = kMxStep * RB, JOIN = W > 1 ? 16 * NT * (LD + 2) * 4 : 0;
  constexpr int LDS = TILE > JOIN ? TILE : JOIN;
  __shared__ __align__(1024) uint8_t smem[W * LDS];

  const int lane = threadIdx.x & 63;
  const int wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int g = lane >> 4, col = lane & 15;
  const int units = a.hkv * a.HT, TG = a.T * a.G;

  // this wave's run: `count` steps from step s of head tile u of sequence b on
  int b, u, s, count, run_q = 0;
  long long run_at = 0;
  MxSeq cur;
  if (W > 1) {
    b = blockIdx.x / units;
    u = blockIdx.x - b * units;
    cur = mx_seq(uniform_at(a.lengths, b), a);
    s = cur.s0 + wave;
    count = max(0, (cur.s1 - s + W - 1) / W);
  } else {
    const MxScan sc = mx_scan(a, lane);
    if (blockIdx.x == 0) {  // where each sequence's steps begin, for the join
      int at = sc.before;
      const int b1 = min(a.B, (lane + 1) * sc.per);
      for (int i = lane * sc.per; i < b1; ++i) {
        a.starts[i] = at;
        const MxSeq q = mx_seq(a.lengths[i], a);
        at += q.s1 - q.s0;
      }
      if (lane == 0) a.starts[a.B] = sc.total;
    }
    const long long total = static_cast<long long>(sc.total) * units;
    run_q = mx_run(total, a.runs);
    run_at = static_cast<long long>(blockIdx.x) * run_q;
    if (run_at >= total) return;
    count = static_cast<int>(min(static_cast<long long>(run_q), total - run_at));
    const uint64_t past = __ballot(static_cast<long long>(sc.upto) * units > run_at);
    const int blk = __ffsll(static_cast<unsigned long long>(past)) - 1;
    long long at = __builtin_amdgcn_readlane(sc.before, blk);
    b = blk * sc.per;
    for (;; ++b) {  // ends: the block's sum passes run_at
      cur = mx_seq(uniform_at(a.lengths, b), a);
      if ((at + cur.s1 - cur.s0) * units > run_at) break;
      at += cur.s1 - cur.s0;
    }
    const long long rem = run_at - at * units;
    u = static_cast<int>(rem / (cur.s1 - cur.s0));
    s = cur.s0 + static_cast<int>(rem - static_cast<long long>(u) * (cur.s1 - cur.s0));
  }

  // byte offsets of this lane's loads from its tile's first row
  const uint32_t k_at = col * CB + g * (CB / 4), ks_at = col * SB + g * SB / 4;
  const uint32_t v_at = (HD == 128 ? lane : lane & 31) * 16, vs_at = HD == 128 ? lane : lane & 31;
  uint8_t* const mem = smem + wave * LDS;
  const uint32_t base = lds_addr(mem);

  int ib = b, iu = u, is = s;
  MxSeq icur = cur;
  auto next = [&](int& nb, int& nu, int& ns, MxSeq& q) {  // the step after; the caller counts
    ns += W;
    if (W > 1 || ns < q.s1) return;
    if (++nu == units) {
      nu = 0;
      do {
        q = mx_seq(uniform_at(a.lengths, ++nb), a);
      } while (q.s0 == q.s1);
    }
    ns = q.s0;
  };
  unsigned holes[kMxAhead];  // of each stage: its 16-key tiles whose page the table does not name
  MxStage<HD> stage[kMxAhead];
  auto issue = [&](int d) __attribute__((always_inline)) {
    const int kvh = iu / a.HT;
    const long long row = static_cast<long long>(ib) * a.width;
    const int last = (icur.len - 1) >> a.shift;  // keys past the length stay in its page
    long long at[2];
    holes[d] = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = is * kMxStep + 16 * h;
      const int page = uniform_at(a.table, row + min(key >> a.shift, last));
      const bool ok = page >= 0 && page < a.pages;
      if (!ok) holes[d] |= 1u << h;
      at[h] = ((static_cast<long long>(ok ? page : 0) * a.hkv + kvh) << a.shift) +
              (key & ((1 << a.shift) - 1));
      const uint8_t* kp = a.kc + at[h] * CB + k_at;
      if constexpr (HD == 128) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(kp);
        stage[d].k[h][0] = w.x; stage[d].k[h][1] = w.y;
        stage[d].k[h][2] = w.z; stage[d].k[h][3] = w.w;
      } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(kp);
        stage[d].k[h][0] = w.x; stage[d].k[h][1] = w.y;
      }
      stage[d].ks[h] = a.ks[at[h] * SB + ks_at];
    }
    if constexpr (HD == 128) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        stage[d].v[j] = *reinterpret_cast<const u32x4*>(a.vc + at[j] * CB + v_at);
        stage[d].vs[j] = a.vs[at[j] * SB + vs_at];
      }
    } else {
      const long long mine = lane < 32 ? at[0] : at[1];
      stage[d].v[0] = *reinterpret_cast<const u32x4*>(a.vc + mine * CB + v_at);
      stage[d].vs[0] = a.vs[mine * SB + vs_at];
    }
  };

  // LDS offsets: this lane's V row(s) and its transposing reads
  const int v_row = lane / CPR, v_ch = 4 * (lane % CPR);
  uint32_t vput[4], voff[ND];
#pragma unroll
  for (int i = 0; i < 4; ++i) vput[i] = v_row * RB + 16 * ((v_ch + i) ^ mx_swz(v_row));
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int row = 4 * g + (col >> 2), dim = 16 * d + 4 * (col & 3);
    voff[d] = row * RB + 16 * ((dim >> 3) ^ mx_swz(row)) + 2 * (dim & 7);
  }

  int issued = 0;
#pragma unroll
  for (int d = 0; d < kMxAhead; ++d)
    if (d < count) {
      if (d) next(ib, iu, is, icur);
      issue(d);
      ++issued;
    }

  uint4 qf[NT][NS];
  f32x4 acc[NT][ND];
  float m_run[NT], l_run[NT], slope[NT];
  int lo[NT], end[NT];  // what each column sees
  bool fresh = true;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m_run[n] = -INFINITY;
    l_run[n] = slope[n] = 0.f;
    lo[n] = end[n] = 0;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto step = [&](int d, int i) __attribute__((always_inline)) {
    const int kvh = u / a.HT, ht = u - kvh * a.HT;
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int c = min(16 * (NT * ht + n) + col, TG - 1), t = c / a.G;
        const int h = kvh * a.G + c - t * a.G;
        end[n] = cur.len - (a.T - 1 - t);
        lo[n] = a.window > 0 ? max(0, end[n] - a.window) : 0;
        const uint16_t* qp = a.q + b * a.qb + t * a.qt + h * a.qh + g * (HD / 4);
#pragma unroll
        for (int x = 0; x < NS; ++x) qf[n][x] = *reinterpret_cast<const uint4*>(qp + 8 * x);
        if (a.slopes) slope[n] = slope_log2(a.slopes[h], kMaxSlope);
        m_run[n] = -INFINITY;
        l_run[n] = 0.f;
#pragma unroll
        for (int x = 0; x < ND; ++x) acc[n][x] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
    const int key0 = s * kMxStep;
    const unsigned hole = holes[d];
    // whether some column does not see some key of the step
    const bool edge = (a.window > 0 && key0 < cur.len - a.window) ||
                      key0 + kMxStep > cur.len - (a.T - 1) || hole;
    MxStage<HD>& st = stage[d];

    f32x4 sc[NT][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int n = 0; n < NT; ++n) sc[n][k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const bf16x8 kk = as_bf16x8(mx4_to_bf16(st.k[k][x], st.ks[k]));
#pragma unroll
        for (int n = 0; n < NT; ++n)
          sc[n][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, as_bf16x8(qf[n][x]), sc[n][k], 0, 0, 0);
      }
    }

    if (edge) {  // rows that no column sees become zeros
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int row = 16 * j + v_row, key = key0 + row;
        if (key < cur.lo || key >= cur.len || ((hole >> (row >> 4)) & 1u)) {
          st.v[j] = u32x4{0u, 0u, 0u, 0u};
          st.vs[j] = kMxOne;
        }
      }
    }
    bool lost = false;
#pragma unroll
    for (int j = 0; j < NV; ++j) lost |= st.vs[j] >= kMxLost;
    if (__ballot(lost)) {  // blocks that are NaN: zeros here, and NaN to the rows that see them
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        uint64_t todo = __ballot(st.vs[j] >= kMxLost);
        while (todo) {
          const int l = __ffsll(static_cast<unsigned long long>(todo)) - 1;
          todo &= todo - 1;
          const int key = key0 + 16 * j + l / CPR, blk = l % CPR;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < ND; ++x)
              if (key >= lo[n] && key < end[n] && (x >> 1) == blk) acc[n][x] += NAN;
        }
        if (st.vs[j] >= kMxLost) {
          st.v[j] = u32x4{0u, 0u, 0u, 0u};
          st.vs[j] = kMxOne;
        }
      }
    }
    wave_lds_order();  // behind the last step's reads
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t w[4] = {st.v[j].x, st.v[j].y, st.v[j].z, st.v[j].w};
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<uint4*>(mem + 16 * j * RB + vput[x]) = mx4_to_bf16(w[x], st.vs[j]);
    }
    if (issued < count) {
      next(ib, iu, is, icur);
      issue(d);
      ++issued;
    }
    wave_lds_order();
    u32x2 vf[2 * ND];
#pragma unroll
    for (int x = 0; x < ND; ++x) {
      vf[2 * x] = lds_get_tr16(base + voff[x]);
      vf[2 * x + 1] = lds_get_tr16(base + voff[x] + 16 * RB);
    }

#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float z[8];
      // a step with a visible key lifts the maximum to the lowest finite number, also if they
      // all score -inf: softmax over such alone is NaN, over no key it gives zeros
      const auto shows = [&](int h) {
        const int first = key0 + 16 * h;
        return !((hole >> h) & 1u) && max(first, lo[n]) < min(first + 16, end[n]);
      };
      float mloc = !edge || shows(0) || shows(1) ? kMxLowest : -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float x = sc[n][j >> 2][j & 3];
        x = a.cap_x2 > 0.f ? softcap_log2(x * a.cap_x2, a.cap_log2) : x * a.scale_log2;
        const int key = key0 + 16 * (j >> 2) + 4 * g + (j & 3);
        if (a.slopes) x -= slope[n] * static_cast<float>(end[n] - 1 - key);
        if (edge && (key < lo[n] || key >= end[n] || ((hole >> (j >> 2)) & 1u))) x = -INFINITY;
        z[j] = x;
        mloc = fmaxf(mloc, x);
      }
      // the offset moves only when some score passes it by more than 8 (weights stay
      // below 2^8), decided by the wave; all four lanes of a column take the same one
      if (__ballot(!(mloc <= m_run[n] + 8.f))) {
        mloc = fmaxf(mloc, __shfl_xor(mloc, 16, kWave));
        mloc = fmaxf(mloc, __shfl_xor(mloc, 32, kWave));
        const float m_new = fmaxf(m_run[n], mloc);
        const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m_run[n] - m_new);
        m_run[n] = m_new;
        l_run[n] *= alpha;
#pragma unroll
        for (int x = 0; x < ND; ++x) acc[n][x] *= alpha;
      }
      const float m_sub = m_run[n] == -INFINITY ? 0.f : m_run[n];
      // the weights as a sum of two bf16, the first cut off
      uint32_t h8[8];
      float lo8[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = exp2_fast(z[j] - m_sub);
        l_run[n] += p;
        h8[j] = __float_as_uint(p) & 0xffff0000u;
        lo8[j] = p - __uint_as_float(h8[j]);
      }
      const uint4 pb = uint4{h8[0] >> 16 | h8[1], h8[2] >> 16 | h8[3], h8[4] >> 16 | h8[5],
                             h8[6] >> 16 | h8[7]};
      const uint4 pl = pack8_bf16(lo8);
#pragma unroll
      for (int x = 0; x < ND; ++x) {
        const bf16x8 vv = as_bf16x8(uint4{vf[2 * x].x, vf[2 * x].y, vf[2 * x + 1].x, vf[2 * x + 1].y});
        acc[n][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, as_bf16x8(pb), acc[n][x], 0, 0, 0);
        acc[n][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, as_bf16x8(pl), acc[n][x], 0, 0, 0);
      }
    }

    const bool head_end = s + 1 == cur.s1;
    if (W == 1 && (head_end || i + 1 == count)) {
      // whole: the head's first step lies in this run too
      const bool whole = head_end && i >= s - cur.s0;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int c = 16 * (NT * ht + n) + col;
        float l = l_run[n] + __shfl_xor(l_run[n], 16, kWave);
        l += __shfl_xor(l, 32, kWave);
        if (c >= TG) continue;
        if (whole) {
          const float f = mx_share(m_run[n], l);
          const int t = c / a.G, h = kvh * a.G + c - t * a.G;
          uint16_t* o = a.out + ((static_cast<long long>(b) * a.T + t) * a.hq + h) * HD + 4 * g;
#pragma unroll
          for (int x = 0; x < ND; ++x)
            *reinterpret_cast<uint2*>(o + 16 * x) =
                make_uint2(pack_bf2(acc[n][x][0] * f, acc[n][x][1] * f),
                           pack_bf2(acc[n][x][2] * f, acc[n][x][3] * f));
        } else {
          // the run starts in this head (or at its first step): 0; else it ends in it: 1
          const int part = i > s - cur.s0 ? 1 : 0;
          const long long at = (2ll * blockIdx.x + part) * a.GT + c - 16 * NT * ht;
          float* o = a.po + at * HD + 4 * g;
#pragma unroll
          for (int x = 0; x < ND; ++x)
            *reinterpret_cast<float4*>(o + 16 * x) =
                make_float4(acc[n][x][0], acc[n][x][1], acc[n][x][2], acc[n][x][3]);
          if (g == 0) *reinterpret_cast<float2*>(a.pml + 2 * at) = make_float2(m_run[n], l);
        }
      }
      fresh = true;
    }
    if (i + 1 < count) next(b, u, s, cur);
  };
  for (int i = 0; i < count; i += kMxAhead) {
#pragma unroll
    for (int d = 0; d < kMxAhead; ++d)
      if (i + d < count) step(d, i + d);
  }

  if constexpr (W > 1) {
    // the waves' (m, l, O) joined through each one's LDS, which it has done with
    const int kvh = u / a.HT, ht = u - kvh * a.HT;
    wave_lds_order();
    float* const so = reinterpret_cast<float*>(mem);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float l = l_run[n] + __shfl_xor(l_run[n], 16, kWave);
      l += __shfl_xor(l, 32, kWave);
#pragma unroll
      for (int x = 0; x < ND; ++x)
        *reinterpret_cast<float4*>(so + (16 * n + col) * LD + 16 * x + 4 * g) =
            make_float4(acc[n][x][0], acc[n][x][1], acc[n][x][2], acc[n][x][3]);
      if (g == 0)
        *reinterpret_cast<float2*>(so + 16 * NT * LD + 2 * (16 * n + col)) =
            make_float2(m_run[n], l);
    }
    __syncthreads();
    const int cols = min(16 * NT, TG - 16 * NT * ht);
    for (int e = threadIdx.x; e < cols * (HD / 4); e += 64 * W) {
      const int c = e / (HD / 4), x = 4 * (e - c * (HD / 4));
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w)
        mx = fmaxf(mx, reinterpret_cast<const float*>(smem + w * LDS)[16 * NT * LD + 2 * c]);
      const float m_sub = mx == -INFINITY ? 0.f : mx;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float* part = reinterpret_cast<const float*>(smem + w * LDS);
        const float2 ml = *reinterpret_cast<const float2*>(part + 16 * NT * LD + 2 * c);
        const float4 y = *reinterpret_cast<const float4*>(part + c * LD + x);
        const float f = exp2_fast(ml.x - m_sub);
        den = fmaf(ml.y, f, den);  // NaN of a NaN score, whatever its part's weight
        sum.x += mx_weighted(y.x, f);
        sum.y += mx_weighted(y.y, f);
        sum.z += mx_weighted(y.z, f);
        sum.w += mx_weighted(y.w, f);
      }
      const float r = mx_share(mx, den);
      const int ci = 16 * NT * ht + c, t = ci / a.G, h = kvh * a.G + ci - t * a.G;
      *reinterpret_cast<uint2*>(a.out + ((static_cast<long long>(b) * a.T + t) * a.hq + h) * HD + x) =
          make_uint2(pack_bf2(sum.x * r, sum.y * r), pack_bf2(sum.z * r, sum.w * r));
    }
  }
}

// Joins the partials of one (sequence, token, query head): o = sum_i 2^(m_i - m) O_i /
// sum_i 2^(m_i - m) l_i, in the runs' order within each of T / (HD / 4) lane groups and
// then over the groups, so the result does not depend on timing.
template <int HD, int TH>
__global__ __launch_bounds__(TH) void mx4_join_kernel(const Mx4Args a, int cols) {
  constexpr int LPP = HD / 4;       // lanes a partial
  constexpr int NG = TH / LPP;
  __shared__ __align__(16) float so[NG][HD];
  __shared__ float sm[NG], sl[NG];
  const int grp = threadIdx.x / LPP, c = threadIdx.x % LPP;
  const int bt = blockIdx.x / a.hq, h = blockIdx.x - bt * a.hq;
  const int b = bt / a.T, t = bt - b * a.T;
  const int kvh = h / a.G, ci = t * a.G + h - kvh * a.G, ht = ci / cols, row = ci - ht * cols;
  const int units = a.hkv * a.HT, u = kvh * a.HT + ht;
  uint16_t* out = a.out + static_cast<long long>(blockIdx.x) * HD;

  const int start = uniform_at(a.starts, b), n = uniform_at(a.starts, b + 1) - start;
  if (n == 0) {  // nothing visible: zeros
    if (threadIdx.x < LPP) *reinterpret_cast<uint2*>(out + 4 * c) = make_uint2(0u, 0u);
    return;
  }
  const int q = mx_run(static_cast<long long>(uniform_at(a.starts, a.B)) * units, a.runs);
  const long long first = static_cast<long long>(start) * units + static_cast<long long>(u) * n;
  const int w0 = static_cast<int>(first / q), w1 = static_cast<int>((first + n - 1) / q);
  if (w0 == w1) return;  // stored by its run
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = w0 + grp; w <= w1; w += NG) {
    const int part = w == w0 && first != static_cast<long long>(w0) * q ? 1 : 0;
    const long long i = (2ll * w + part) * a.GT + row;
    const float2 ml = *reinterpret_cast<const float2*>(a.pml + 2 * i);
    const float4 x = *reinterpret_cast<const float4*>(a.po + i * HD + 4 * c);
    const float m_new = fmaxf(m, ml.x);
    const float m_sub = m_new == -INFINITY ? 0.f : m_new;
    const float f = exp2_fast(m - m_sub), e = exp2_fast(ml.x - m_sub);
    m = m_new;
    l = fmaf(ml.y, e, l * f);  // NaN of a NaN score, whatever its part's weight
    o.x = mx_weighted(x.x, e) + mx_weighted(o.x, f);
    o.y = mx_weighted(x.y, e) + mx_weighted(o.y, f);
    o.z = mx_weighted(x.z, e) + mx_weighted(o.z, f);
    o.w = mx_weighted(x.w, e) + mx_weighted(o.w, f);
  }
  *reinterpret_cast<float4*>(&so[grp][4 * c]) = o;
  if (c == 0) {
    sm[grp] = m;
    sl[grp] = l;
  }
  __syncthreads();
  float mx = sm[0];
#pragma unroll
  for (int i = 1; i < NG; ++i) mx = fmaxf(mx, sm[i]);
  const float m_sub = mx == -INFINITY ? 0.f : mx;
  for (int d = threadIdx.x; d < HD; d += TH) {
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const float e = exp2_fast(sm[i] - m_sub);
      den = fmaf(sl[i], e, den);
      num += mx_weighted(so[i][d], e);
    }
    out[d] = f2bf(num * mx_share(mx, den));
  }
}

struct Mx4Plan {
  int G, HT, GT, NT, runs;
  bool wide;  // a workgroup a head tile, its waves every 8th (4th) step; else runs and their join
  long long cap_len, groups, ws;
};

inline bool mx4_plan(int B, int T, int Hq, int Hkv, int hd, int width, int page, Mx4Plan* p) {
  if (B < 0 || T < 1 || T > 64 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq > kMaxHeads ||
      (hd != 64 && hd != 128) || width < 0 || page_shift(page) < 0)
    return false;
  p->G = Hq / Hkv;
  const int tg = T * p->G;
  p->NT = tg > 16 ? 2 : 1;
  const int cols = 16 * p->NT;
  p->HT = (tg + cols - 1) / cols;
  p->GT = tg < cols ? tg : cols;
  p->cap_len = static_cast<long long>(width) * page;
  if (p->cap_len >= (1ll << 31) - kMxStep) return false;  // positions are 32-bit
  const long long units = static_cast<long long>(B) * Hkv * p->HT;
  const int W = p->NT == 1 ? 8 : 4;
  const long long deep = (p->cap_len + kMxStep * W - 1) / (kMxStep * W);
  p->wide = deep <= 4 || (W == 8 && deep <= 8 && 2 * units >= compute_units());
  p->runs = p->wide ? 0 : compute_units() * (p->NT == 1 ? 8 : 4);
  p->groups = p->wide ? units : p->runs;
  p->ws = p->wide ? 0
                  : 2ll * p->runs * p->GT * (hd + 2) * 4 + (static_cast<long long>(B) + 1) * 4;
  // all steps, a run's steps and the grids are 32-bit
  const double steps = static_cast<double>(B) * (p->cap_len / kMxStep + 1);
  return steps < 2147483647. &&
         (p->wide || steps * Hkv * p->HT / p->runs < 2147483647.) && p->groups < (1ll << 31) &&
         static_cast<double>(B) * T * Hq < 2147483647.;
}

template <int HD, int NT>
int32_t launch_mx4(const Mx4Args& a, const Mx4Plan& p, hipStream_t s) {
  constexpr int W = NT == 1 ? 8 : 4;
  const dim3 grid(static_cast<unsigned>(p.groups));
  if (p.wide) {
    hipLaunchKernelGGL((mx4_attn_kernel<HD, NT, W>), grid, dim3(64 * W), 0, s, a);
    return launch_status();
  }
  const dim3 heads(static_cast<unsigned>(a.B) * a.T * a.hq);
  hipLaunchKernelGGL((mx4_attn_kernel<HD, NT, 1>), grid, dim3(64), 0, s, a);
  if (heads.x >= 1024)
    hipLaunchKernelGGL((mx4_join_kernel<HD, 64>), heads, dim3(64), 0, s, a, 16 * NT);
  else
    hipLaunchKernelGGL((mx4_join_kernel<HD, 512>), heads, dim3(512), 0, s, a, 16 * NT);
  return launch_status();
}

}  // namespace llmy

using namespace llmy;

extern "C" int64_t llmy_paged_attn_mx4_workspace_bytes(int32_t B, int32_t T, int32_t Hq,
                                                       int32_t Hkv, int32_t head_dim,
                                                       int32_t width, int32_t page) {
  Mx4Plan p;
  return mx4_plan(B, T, Hq, Hkv, head_dim, width, page, &p) ? p.ws : -1;
}

extern "C" int32_t llmy_paged_attn_mx4(
    const llmy_bf16* q, int64_t q_seq, int64_t q_row, int64_t q_head, const void* k_cache,
    const void* v_cache, const void* k_scales, const void* v_scales, const int32_t* page_table,
    const int32_t* lengths, const float* slopes, llmy_bf16* out, void* workspace,
    int64_t workspace_bytes, int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t head_dim,
    int32_t width, int32_t page, int32_t pages, int32_t window, float scale, float softcap,
    void* stream) {
  Mx4Plan p;
  LLMY_REQUIRE(mx4_plan(B, T, Hq, Hkv, head_dim, width, page, &p));
  LLMY_REQUIRE(pages >= 0 && window >= 0 && scale_ok(scale, softcap));
  if (B == 0) return 0;
  LLMY_REQUIRE(q && out && lengths && aligned(q, 16) && aligned(out, 16));
  LLMY_REQUIRE(q_seq % 8 == 0 && q_row % 8 == 0 && q_head % 8 == 0 && q_seq >= 0 && q_row >= 0 &&
               q_head >= 0);
  LLMY_REQUIRE(width == 0 || page_table);
  const Mx4Cache c{const_cast<void*>(k_cache), const_cast<void*>(v_cache),
                   const_cast<void*>(k_scales), const_cast<void*>(v_scales)};
  const int64_t slots = static_cast<int64_t>(pages) * Hkv * page;
  LLMY_REQUIRE(c.ok(slots, head_dim));  // with no page at all every length counts as 0
  LLMY_REQUIRE(p.ws == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= p.ws));
  // out and the workspace are written while other workgroups still read
  const int64_t out_bytes = 2ll * B * T * Hq * head_dim;
  const double q_extent = 2. * ((B - 1.) * q_seq + (T - 1.) * q_row + (Hq - 1.) * q_head + head_dim);
  LLMY_REQUIRE(q_extent < kMaxExtent);
  const int64_t q_bytes = static_cast<int64_t>(q_extent);
  LLMY_REQUIRE(bytes_apart(out, out_bytes, q, q_bytes) && bytes_apart(workspace, p.ws, q, q_bytes) &&
               bytes_apart(workspace, p.ws, out, out_bytes));
  for (int i = 0; i < 4; ++i)
    LLMY_REQUIRE(bytes_apart(out, out_bytes, c.part(i), c.bytes(i, slots, head_dim)) &&
                 bytes_apart(workspace, p.ws, c.part(i), c.bytes(i, slots, head_dim)));
  Mx4Args a{};
  a.q = q; a.qb = q_seq; a.qt = q_row; a.qh = q_head;
  a.kc = static_cast<const uint8_t*>(k_cache); a.vc = static_cast<const uint8_t*>(v_cache);
  a.ks = static_cast<const uint8_t*>(k_scales); a.vs = static_cast<const uint8_t*>(v_scales);
  a.table = page_table; a.lengths = lengths; a.out = out; a.slopes = slopes;
  a.po = static_cast<float*>(workspace);
  a.pml = a.po + 2ll * p.runs * p.GT * head_dim;
  a.starts = reinterpret_cast<int32_t*>(a.pml + 4ll * p.runs * p.GT);
  const float log2e = 1.4426950408889634f;
  a.scale_log2 = scale * log2e;
  a.cap_log2 = softcap * log2e;
  a.cap_x2 = softcap > 0.f ? 2.f * log2e * scale / softcap : 0.f;
  a.B = B; a.T = T; a.hq = Hq; a.hkv = Hkv; a.G = p.G; a.HT = p.HT; a.GT = p.GT;
  a.width = width; a.shift = page_shift(page); a.pages = pages; a.window = window;
  a.cap_len = pages ? static_cast<int>(p.cap_len) : 0;
  a.runs = p.runs;
  const hipStream_t s = as_stream(stream);
  if (head_dim == 64)
    return p.NT == 1 ? launch_mx4<64, 1>(a, p, s) : launch_mx4<64, 2>(a, p, s);
  return p.NT == 1 ? launch_mx4<128, 1>(a, p, s) : launch_mx4<128, 2>(a, p, s);
}
