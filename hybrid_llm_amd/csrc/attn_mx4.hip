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
//     the cache, loaded straight to registers, two rounds of the waves ahead.  Lane l (g = l /
//     16) gets keys 4 g + r of a 16-key tile for column l % 16; two such tiles are, register
//     by register, the B operand of a 32-key product O^T += V^T P^T under the key order
//     4 g + j, 16 + 4 g + j.
//   * V, loaded the same way, is put in bf16 into the wave's own 32 rows of LDS, whose
//     transposing reads give V^T in that order.  A block scale belongs to a key and 32 dims,
//     so scaling V costs nothing beyond its conversion, and scaling the weights would
//     take one set of them per block.
//   * the waves of a workgroup take the 32-key steps of a head tile in turn and join their
//     (m, l, O) in LDS.  Where tables are short a workgroup has a whole tile; otherwise an equal
//     run of the flat list of all (sequence, head tile, step), found from the lengths on the
//     device: partials of tiles that are cut go to the workspace, and a second kernel joins
//     them.  A run of four waves instead of one has a quarter of the parts to store and join.
// Measured, the call's kernels together (32 heads over 8 x 128): 4 sequences of 131072 tokens,
// 570 MB, 106 us, 5.4 TB/s; 64 ragged ones of up to 4096 with 4 tokens each and capped scores,
// 143 MB, 49 us, of which the join takes 6 and the first loads and the changes of tiles most of
// what is past 28; 16 x 64 over 4, one sequence of 1023, 10 us, a chain of latencies.
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
constexpr int kMxAhead = 2;      // steps of a wave in registers
constexpr int kMxPad = 8;        // steps that a head tile costs besides
constexpr int kMxLeast = 16;     // places of a run at the least
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
  int32_t* starts;             // [B + 1]: places of the sequences before each, and of all
  const float* slopes;
  float scale_log2, cap_log2, cap_x2;
  int B, T, hq, hkv, G, HT, GT;  // T G columns in HT tiles of GT <= 16 NT
  int width, shift, pages, window, cap_len;
  uint32_t page_bytes;         // of a page's codes
  int runs;
};

struct MxSeq {
  int len, lo, s0, s1;         // positions [lo, len) seen by any token, steps [s0, s1)

  // A head tile's places on the flat list: kMxPad for what it costs beside its steps (its
  // queries, the waves' join, the round that its last steps do not fill), then they.
  __device__ __forceinline__ int places() const { return s1 > s0 ? s1 - s0 + kMxPad : 0; }
};

__device__ __forceinline__ MxSeq mx_seq(int len, const Mx4Args& a) {
  MxSeq s;
  s.len = min(max(len, 0), a.cap_len);
  s.lo = a.window > 0 ? static_cast<int>(max(0ll, s.len - (a.T - 1ll) - a.window)) : 0;
  s.s0 = s.lo / kMxStep;
  s.s1 = static_cast<int>((static_cast<unsigned>(s.len) + kMxStep - 1) / kMxStep);
  return s;
}

// Places of all sequences (the host sees to it that they fit 31 bits), as sums over 64
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
    n += mx_seq(a.lengths[b], a).places();
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
  return static_cast<int>(q > kMxLeast ? q : kMxLeast);
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
template <class T>
__device__ __forceinline__ void mx_swap(T& a, T& b) {
  const T t = a;
  a = b;
  b = t;
}

template <int HD>
struct MxStage {
  static constexpr int NV = HD / 64;
  uint32_t k[2][HD / 32];
  uint32_t ks[2];
  u32x4 v[NV];
  uint32_t vs[NV];

  __device__ __forceinline__ void swap(MxStage& o) {  // (whole structures would go through memory)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) mx_swap(k[i][j], o.k[i][j]);
      mx_swap(ks[i], o.ks[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      mx_swap(v[i], o.v[i]);
      mx_swap(vs[i], o.vs[i]);
    }
  }
};

// Waves a SIMD: as many as the registers of each form take.
constexpr int mx4_waves(int hd, int nt) { return hd == 64 ? (nt == 1 ? 3 : 2) : nt == 1 ? 3 : 2; }

// Waves of the workgroups that take a head tile among few: what fits a CU without spilling, which
// costs most where it is least work (28 bytes of scratch a lane: the first round 6 to 16 us).
constexpr int mx4_most(int hd, int nt) { return hd == 64 && nt == 1 ? 12 : 8; }

// A place in a workgroup's run: steps [begin, end) of one head tile, `it` of its rounds (a
// step for each wave) done, and `left` steps of the run behind this tile's.
struct MxPlace {
  int b, kvh, ht, len, lo, begin, end, it, left;

  // its sequence's page ids, and the last that its keys reach: those past the length stay there
  const int32_t* table;
  int last;

  __device__ __forceinline__ void sequence(const Mx4Args& a, int n, int first) {
    len = n;
    lo = first;
    table = a.table + static_cast<long long>(b) * a.width;
    last = (n - 1) >> a.shift;
  }
};

// A global address from an SGPR pair and a lane's 32-bit offset: kept from being folded into
// one 64-bit address a lane, which costs an addition each time.
typedef const uint8_t __attribute__((address_space(1)))* global_u8;

__device__ __forceinline__ global_u8 mx_base(const uint8_t* p, uint64_t off) {
  uint64_t at = reinterpret_cast<uint64_t>(p) + off;
  asm("" : "+s"(at));
  return reinterpret_cast<global_u8>(at);
}

template <class T>
__device__ __forceinline__ T mx_load(global_u8 p) {
  return __builtin_nontemporal_load(reinterpret_cast<const T __attribute__((address_space(1)))*>(p));
}

// W waves: a run of the flat list (runs > 0), or a whole head tile.
template <int HD, int NT, int W>
__global__ __launch_bounds__(64 * W, W > 4 ? W / 4 : mx4_waves(HD, NT))
void mx4_attn_kernel(const Mx4Args a) {
  constexpr int RB = 2 * HD;                  // bytes of a V row in LDS
  constexpr int CB = HD / 2, SB = HD / 32;    // bytes of a stored row: codes, scales
  constexpr int NS = HD / 32;                 // 32-dim slices of the score product
  constexpr int ND = HD / 16;                 // 16-dim output tiles
  constexpr int NV = MxStage<HD>::NV;
  constexpr int CPR = HD / 32;                // 16-byte chunks of a stored row
  constexpr int LD = HD + 4;                  // of a column's part in the waves' join
  constexpr int TILE = kMxStep * RB, JOIN = 16 * NT * (LD + 2) * 4;
  constexpr int LDS = TILE > JOIN ? TILE : JOIN;
  static_assert(LDS % 128 == 0, "the waves' rows start on one bank");
  __shared__ __align__(1024) uint8_t smem[W * LDS];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int units = a.hkv * a.HT, TG = a.T * a.G;

  MxPlace at;  // where this workgroup's run starts
  {
    MxSeq cur;
    int u;
    at.it = 0;
    if (a.runs == 0) {
      at.b = blockIdx.x / units;
      u = blockIdx.x - at.b * units;
      cur = mx_seq(uniform_at(a.lengths, at.b), a);
      at.begin = cur.s0;
      at.end = cur.s1;
      at.left = 0;
    } else {
      const MxScan sc = mx_scan(a, lane);
      if (blockIdx.x == 0 && wave == 0) {  // where each sequence's places begin, for the join
        int x = sc.before;
        const int b1 = min(a.B, (lane + 1) * sc.per);
        for (int i = lane * sc.per; i < b1; ++i) {
          a.starts[i] = x;
          x += mx_seq(a.lengths[i], a).places();
        }
        if (lane == 0) a.starts[a.B] = sc.total;
      }
      const long long total = static_cast<long long>(sc.total) * units;
      const int run_q = mx_run(total, a.runs);
      const long long run_at = static_cast<long long>(blockIdx.x) * run_q;
      if (run_at >= total) return;
      const int count = static_cast<int>(min(static_cast<long long>(run_q), total - run_at));
      const uint64_t past = __ballot(static_cast<long long>(sc.upto) * units > run_at);
      const int blk = __ffsll(static_cast<unsigned long long>(past)) - 1;
      long long before = __builtin_amdgcn_readlane(sc.before, blk);
      at.b = blk * sc.per;
      for (;; ++at.b) {  // ends: the block's sum passes run_at
        cur = mx_seq(uniform_at(a.lengths, at.b), a);
        if ((before + cur.places()) * units > run_at) break;
        before += cur.places();
      }
      const long long rem = run_at - before * units;
      u = static_cast<int>(rem / cur.places());
      const int p0 = static_cast<int>(rem - static_cast<long long>(u) * cur.places());
      const int p1 = min(cur.places(), p0 + count);
      at.begin = cur.s0 + max(0, p0 - kMxPad);
      at.end = cur.s0 + max(0, p1 - kMxPad);
      at.left = count - (p1 - p0);
      // (at least a step: a run is longer than a tile's pad, and the last one ends with a tile)
      static_assert(kMxLeast > kMxPad, "a run of a pad alone");
    }
    at.sequence(a, cur.len, cur.lo);
    if (at.begin == at.end) {  // nothing to see (a whole tile): zeros
      const int kvh = u / a.HT, ht = u - kvh * a.HT;
      const int cols = min(16 * NT, TG - 16 * NT * ht);
      for (int e = threadIdx.x; e < cols * (HD / 4); e += 64 * W) {
        const int ci = 16 * NT * ht + e / (HD / 4), t = ci / a.G;
        *reinterpret_cast<uint2*>(a.out + ((static_cast<long long>(at.b) * a.T + t) * a.hq +
                                           kvh * a.G + ci - t * a.G) * HD + 4 * (e % (HD / 4))) =
            make_uint2(0u, 0u);
      }
      return;
    }
    at.kvh = u / a.HT;
    at.ht = u - at.kvh * a.HT;
  }

  // one round on; false behind the run's last
  const auto advance = [&](MxPlace& p) __attribute__((always_inline)) {
    ++p.it;
    if (p.begin + p.it * W < p.end) return true;
    if (p.left <= kMxPad) return false;  // no step of the next tile
    p.it = 0;
    if (++p.ht == a.HT) {
      p.ht = 0;
      if (++p.kvh == a.hkv) {
        p.kvh = 0;
        MxSeq q;
        do {
          q = mx_seq(uniform_at(a.lengths, ++p.b), a);
        } while (q.s0 == q.s1);
        p.sequence(a, q.len, q.lo);
      }
    }
    p.begin = p.lo / kMxStep;
    const int all = (p.len + kMxStep - 1) / kMxStep - p.begin;
    p.end = p.begin + min(all, p.left - kMxPad);
    p.left = max(0, p.left - kMxPad - all);
    return true;
  };

  // byte offsets of this lane's loads from its tile's first row
  const uint32_t k_at = col * CB + g * (CB / 4), ks_at = col * SB + g * SB / 4;
  const uint32_t v_at = (HD == 128 ? lane : lane & 31) * 16, vs_at = HD == 128 ? lane : lane & 31;
  uint8_t* const mem = smem + wave * LDS;
  const uint32_t base = lds_addr(mem);

  // The round that is loaded next, and its page ids.  Every wave loads something every round,
  // the cache's first rows where it has no step, so that the compiler can count the loads that
  // are in flight: past a branch around them it would wait for all.
  MxPlace to = at;
  bool more = true;
  int ipage[2], istep;
  const auto look = [&]() __attribute__((always_inline)) {
    istep = min(to.begin + to.it * W + wave, to.end - 1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      ipage[h] = uniform_at(to.table, min((istep * kMxStep + 16 * h) >> a.shift, to.last));
  };
  // of each stage: its 16-key tiles that are not there, no step's or in a page without a name
  unsigned holes[kMxAhead];
  MxStage<HD> stage[kMxAhead];
  const auto issue = [&](int d) __attribute__((always_inline)) {
    const bool none = !more || to.begin + to.it * W + wave >= to.end;
    holes[d] = 0u;
    global_u8 kp[2], vp[2], ksp[2], vsp[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = istep * kMxStep + 16 * h;
      const bool ok = !none && ipage[h] >= 0 && ipage[h] < a.pages;
      if (!ok) holes[d] |= 1u << h;
      const uint64_t off = ok ? static_cast<uint64_t>(ipage[h]) * a.page_bytes +
                                    static_cast<uint32_t>((to.kvh << a.shift) + (key & ((1 << a.shift) - 1))) * CB
                              : 0;
      static_assert(CB == 16 * SB, "scales lie as the codes do");
      kp[h] = mx_base(a.kc, off);
      vp[h] = mx_base(a.vc, off);
      ksp[h] = mx_base(a.ks, off / 16);
      vsp[h] = mx_base(a.vs, off / 16);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (HD == 128) {
        const u32x4 w = mx_load<u32x4>(kp[h] + k_at);
        stage[d].k[h][0] = w.x; stage[d].k[h][1] = w.y;
        stage[d].k[h][2] = w.z; stage[d].k[h][3] = w.w;
      } else {
        const u32x2 w = mx_load<u32x2>(kp[h] + k_at);
        stage[d].k[h][0] = w.x; stage[d].k[h][1] = w.y;
      }
      stage[d].ks[h] = ksp[h][ks_at];
    }
    if constexpr (HD == 128) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        stage[d].v[j] = mx_load<u32x4>(vp[j] + v_at);
        stage[d].vs[j] = vsp[j][vs_at];
      }
    } else {
      stage[d].v[0] = mx_load<u32x4>((lane < 32 ? vp[0] : vp[1]) + v_at);
      stage[d].vs[0] = (lane < 32 ? vsp[0] : vsp[1])[vs_at];
    }
    more = more && advance(to);
    look();
  };

  // LDS offsets: this lane's V row(s) and its transposing reads
  // (chunk c of a row lies at c ^ swz, which the bits of c over and under split)
  const int v_row = lane / CPR, v_ch = 4 * (lane % CPR), t_row = 4 * g + (col >> 2);
  const uint32_t vput = v_row * RB + 16 * (v_ch ^ mx_swz(v_row));
  const uint32_t vget = base + t_row * RB + 16 * (((col >> 1) & 1) ^ mx_swz(t_row)) + 8 * (col & 1);

  uint4 qf[NT][NS];
  f32x4 acc[NT][ND];
  float m_run[NT], l_run[NT], slope[NT];
  int lo[NT], end[NT];  // what each column sees
  bool rough[NT];       // some column's offset is as large as below
  const auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = min(16 * (NT * at.ht + n) + col, TG - 1), t = a.T == 1 ? 0 : c / a.G;
      const int h = at.kvh * a.G + c - t * a.G;
      end[n] = at.len - (a.T - 1 - t);
      lo[n] = a.window > 0 ? max(0, max(0, end[n]) - a.window) : 0;
      const uint16_t* qp = a.q + at.b * a.qb + t * a.qt + h * a.qh + g * (HD / 4);
#pragma unroll
      for (int x = 0; x < NS; ++x) qf[n][x] = *reinterpret_cast<const uint4*>(qp + 8 * x);
      slope[n] = a.slopes ? slope_log2(a.slopes[h], kMaxSlope) : 0.f;
      m_run[n] = -INFINITY;
      l_run[n] = 0.f;
      rough[n] = true;
#pragma unroll
      for (int x = 0; x < ND; ++x) acc[n][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  // waited for before a tile's rounds: left pending, each of them would wait as its first does
  const auto settle = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int x = 0; x < NS; ++x)
        asm volatile("" : "+v"(qf[n][x].x), "+v"(qf[n][x].y), "+v"(qf[n][x].z), "+v"(qf[n][x].w));
      asm volatile("" : "+v"(slope[n]));
    }
  };
  look();
  begin();
#pragma unroll
  for (int d = 0; d < kMxAhead; ++d) issue(d);
  settle();

  const bool special = a.cap_x2 > 0.f || a.slopes;
  const auto step = [&](int d, int s) __attribute__((always_inline)) {
    const int key0 = s * kMxStep;
    const unsigned hole = holes[d];
    // whether some column does not see some key of the step
    const bool edge = (a.window > 0 && key0 < at.len - a.window) ||
                      key0 + kMxStep > at.len - (a.T - 1) || hole;
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
        if (key < at.lo || key >= at.len || ((hole >> (row >> 4)) & 1u)) {
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
        *reinterpret_cast<uint4*>(mem + 16 * j * RB + (vput ^ (16 * x))) = mx4_to_bf16(w[x], st.vs[j]);
    }
    wave_lds_order();
    issue(d);

    uint4 pb[NT], pl[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // scores: products to scale by `mul`, or, where more is done to them, in log2 units
      float z[8], mul = a.scale_log2;
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = sc[n][j >> 2][j & 3];
      float least = kMxLowest;
      if (special || edge) {
        mul = 1.f;
        if (a.cap_x2 > 0.f) {
#pragma unroll
          for (int j = 0; j < 8; ++j) z[j] = softcap_log2(z[j] * a.cap_x2, a.cap_log2);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) z[j] *= a.scale_log2;
        }
        const int key = key0 + 4 * g;
        if (a.slopes) {
          const float far = static_cast<float>(end[n] - 1 - key);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            z[j] -= slope[n] * (far - static_cast<float>(16 * (j >> 2) + (j & 3)));
        }
        if (edge) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int at_key = key + 16 * (j >> 2) + (j & 3);
            const bool seen = at_key >= lo[n] && at_key < end[n] && !((hole >> (j >> 2)) & 1u);
            z[j] = seen ? z[j] : -INFINITY;
          }
          const auto shows = [&](int h) {
            const int from = key0 + 16 * h;
            return !((hole >> h) & 1u) && max(from, lo[n]) < min(from + 16, end[n]);
          };
          least = shows(0) || shows(1) ? kMxLowest : -INFINITY;
        }
      }
      // a step with a visible key lifts the maximum to the lowest finite number, also if they
      // all score -inf: softmax over such alone is NaN, over no key it gives zeros
      float mloc = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])),
                         fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7])));
      mloc = fmaxf(mloc * mul, least);
      // the offset moves only when some score passes it by more than 8 (weights stay
      // below 2^8), decided by the wave; all four lanes of a column take the same one
      if (__ballot(!(mloc <= m_run[n] + 8.f))) {
        mloc = fmaxf(mloc, __shfl_xor(mloc, 16, kWave));
        mloc = fmaxf(mloc, __shfl_xor(mloc, 32, kWave));
        const float m_new = fmaxf(m_run[n], mloc);
        const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m_run[n] - m_new);
        m_run[n] = m_new;
        rough[n] = __ballot(!(fabsf(m_new) < 0x1p20f)) != 0;
        l_run[n] *= alpha;
#pragma unroll
        for (int x = 0; x < ND; ++x) acc[n][x] *= alpha;
      }
      // One rounding for product and difference, which leaves all weights the same factor from
      // the offset's own; not so where that is 2^20 or more, and the factor any
      if (rough[n]) {
#pragma clang fp contract(off)
        const float m_sub = m_run[n] == -INFINITY ? 0.f : m_run[n];
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = z[j] * mul - m_sub;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = fmaf(z[j], mul, -m_run[n]);
      }
      // the weights as a sum of two bf16, the first cut off
      uint32_t h8[8];
      float lo8[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = exp2_fast(z[j]);
        l_run[n] += p;
        h8[j] = __float_as_uint(p) & 0xffff0000u;
        lo8[j] = p - __uint_as_float(h8[j]);
      }
      pb[n] = uint4{h8[0] >> 16 | h8[1], h8[2] >> 16 | h8[3], h8[4] >> 16 | h8[5],
                    h8[6] >> 16 | h8[7]};
      pl[n] = pack8_bf16(lo8);
    }
#pragma unroll
    for (int x = 0; x < ND; ++x) {
      const uint32_t from = (vget ^ (32 * (x & 3))) + 128 * (x >> 2);
      const u32x2 v0 = lds_get_tr16(from), v1 = lds_get_tr16(from + 16 * RB);
      const bf16x8 vv = as_bf16x8(uint4{v0.x, v0.y, v1.x, v1.y});
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[n][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, as_bf16x8(pb[n]), acc[n][x], 0, 0, 0);
        acc[n][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, as_bf16x8(pl[n]), acc[n][x], 0, 0, 0);
      }
    }
  };

  // The waves' (m, l, O) of a head tile joined through each one's LDS: to the output where the
  // run has all of its steps, else to the workspace, where the run's first tile takes place 0
  // and its last one place 1.
  const auto join = [&](bool first) __attribute__((always_inline)) {
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
    const bool whole = at.begin == at.lo / kMxStep && at.end == (at.len + kMxStep - 1) / kMxStep;
    const int cols = min(16 * NT, TG - 16 * NT * at.ht);
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
      if (whole) {
        const float r = mx_share(mx, den);
        const int ci = 16 * NT * at.ht + c, t = a.T == 1 ? 0 : ci / a.G;
        const int h = at.kvh * a.G + ci - t * a.G;
        *reinterpret_cast<uint2*>(a.out + ((static_cast<long long>(at.b) * a.T + t) * a.hq + h) * HD + x) =
            make_uint2(pack_bf2(sum.x * r, sum.y * r), pack_bf2(sum.z * r, sum.w * r));
      } else {
        const long long i = (2ll * blockIdx.x + (first ? 0 : 1)) * a.GT + c;
        *reinterpret_cast<float4*>(a.po + i * HD + x) = sum;
        if (x == 0) *reinterpret_cast<float2*>(a.pml + 2 * i) = make_float2(mx, den);
      }
    }
  };

  // A tile's rounds by twos, so that each stage keeps its registers, in a loop of one exit: past
  // a second one the compiler would again wait for all loads.  An odd round leaves the stages
  // in the other order.
  static_assert(kMxAhead == 2, "the loop below");
  for (bool first = true;; first = false) {
    const int rounds = (at.end - at.begin + W - 1) / W;
    int s = at.begin + wave;
    for (int r = rounds >> 1; r > 0; --r, s += 2 * W) {
      step(0, s);
      step(1, s + W);
    }
    if (rounds & 1) step(0, s);
    join(first);
    at.it = rounds - 1;
    if (!advance(at)) break;
    if (rounds & 1) {
      stage[0].swap(stage[1]);
      mx_swap(holes[0], holes[1]);
    }
    __syncthreads();  // before its parts are written over
    begin();
    settle();
  }
}

// Joins the partials of one (sequence, head tile): o = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i -
// m) l_i, for kMxJoinCols of its columns a workgroup, in the runs' order within each of a number
// of lane groups and then over the groups, so the result does not depend on timing.
constexpr int kMxJoin = 512, kMxJoinCols = 8;

template <int HD>
__global__ __launch_bounds__(kMxJoin) void mx4_join_kernel(const Mx4Args a, int cols, int parts) {
  constexpr int LPP = HD / 4;                       // lanes a column
  constexpr int ITEMS = kMxJoinCols * LPP, GROUPS = kMxJoin / ITEMS;
  __shared__ __align__(16) float so[kMxJoin][4];
  __shared__ float2 sml[kMxJoin];
  const int units = a.hkv * a.HT;
  const int tile = blockIdx.x / parts, row = (blockIdx.x - tile * parts) * kMxJoinCols +
                                             threadIdx.x % ITEMS / LPP;
  const int b = tile / units, u = tile - b * units;
  const int kvh = u / a.HT, ht = u - kvh * a.HT;
  const int start = uniform_at(a.starts, b), n = uniform_at(a.starts, b + 1) - start;
  const int q = mx_run(static_cast<long long>(uniform_at(a.starts, a.B)) * units, a.runs);
  const long long first = static_cast<long long>(start) * units + static_cast<long long>(u) * n;
  // the runs of its first and last step
  const int w0 = static_cast<int>((first + kMxPad) / q);
  const int w1 = n ? static_cast<int>((first + n - 1) / q) : -1;
  if (w0 == w1) return;  // stored by its run
  const int ci = cols * ht + row, c = threadIdx.x % LPP, grp = threadIdx.x / ITEMS;
  const bool here = row < cols && ci < a.T * a.G;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (here) {
#pragma unroll 4
    for (int w = w0 + grp; w <= w1; w += GROUPS) {
      const int part = w == w0 && first > static_cast<long long>(w0) * q ? 1 : 0;
      const long long i = (2ll * w + part) * a.GT + row;
      const float2 ml = *reinterpret_cast<const float2*>(a.pml + 2 * i);
      const float4 x = *reinterpret_cast<const float4*>(a.po + i * HD + 4 * c);
      const float m_new = fmaxf(m, ml.x);
      const float m_sub = m_new == -INFINITY ? 0.f : m_new;
      const float f = exp2_fast(m - m_sub), y = exp2_fast(ml.x - m_sub);
      m = m_new;
      l = fmaf(ml.y, y, l * f);  // NaN of a NaN score, whatever its part's weight
      o.x = mx_weighted(x.x, y) + mx_weighted(o.x, f);
      o.y = mx_weighted(x.y, y) + mx_weighted(o.y, f);
      o.z = mx_weighted(x.z, y) + mx_weighted(o.z, f);
      o.w = mx_weighted(x.w, y) + mx_weighted(o.w, f);
    }
  }
  *reinterpret_cast<float4*>(so[threadIdx.x]) = o;
  sml[threadIdx.x] = make_float2(m, l);
  __syncthreads();
  if (grp > 0 || !here) return;
  float mx = m;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) mx = fmaxf(mx, sml[threadIdx.x + i * ITEMS].x);
  const float m_sub = mx == -INFINITY ? 0.f : mx, f = exp2_fast(m - m_sub);
  l *= f;
  o = make_float4(mx_weighted(o.x, f), mx_weighted(o.y, f), mx_weighted(o.z, f),
                  mx_weighted(o.w, f));
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    const float2 ml = sml[threadIdx.x + i * ITEMS];
    const float4 x = *reinterpret_cast<const float4*>(so[threadIdx.x + i * ITEMS]);
    const float y = exp2_fast(ml.x - m_sub);
    l = fmaf(ml.y, y, l);
    o.x += mx_weighted(x.x, y);
    o.y += mx_weighted(x.y, y);
    o.z += mx_weighted(x.z, y);
    o.w += mx_weighted(x.w, y);
  }
  const float r = mx_share(mx, l);  // (without a part, a sequence of length 0: zeros)
  const int t = ci / a.G, h = kvh * a.G + ci - t * a.G;
  *reinterpret_cast<uint2*>(a.out + ((static_cast<long long>(b) * a.T + t) * a.hq + h) * HD + 4 * c) =
      make_uint2(pack_bf2(o.x * r, o.y * r), pack_bf2(o.z * r, o.w * r));
}

struct Mx4Plan {
  int G, HT, GT, NT, runs;
  int W;  // waves of a workgroup: of a whole head tile (runs 0), or of a run, whose parts are joined
  long long cap_len, groups, ws;
};

inline bool mx4_plan(int B, int T, int Hq, int Hkv, int hd, int width, int page, int window,
                     Mx4Plan* p) {
  if (B < 0 || T < 1 || T > 64 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq > kMaxHeads ||
      (hd != 64 && hd != 128) || width < 0 || page_shift(page) < 0 || window < 0)
    return false;
  p->G = Hq / Hkv;
  const int tg = T * p->G;
  p->NT = tg > 16 ? 2 : 1;
  const int cols = 16 * p->NT;
  p->HT = (tg + cols - 1) / cols;
  p->GT = tg < cols ? tg : cols;
  p->cap_len = static_cast<long long>(width) * page;
  if (p->cap_len >= (1ll << 31) - kMxStep) return false;  // positions are 32-bit
  const long long units = static_cast<long long>(B) * Hkv * p->HT, cus = compute_units();
  // Whole head tiles by workgroups need one launch and no parts, but take as long as the longest
  // of them; four waves share a CU with others, a CU's own serve few tiles.  By the rounds of
  // four waves that the table (or the window) can fill; us of four waves a tile / of a CU's / of
  // runs, lengths even: 16 heads over 4 x 64, one sequence of 1000 tokens 13 / 13 / 18, 2000 19
  // / 16 / 19, 4000 34 / 23 / 18, 64 of 2000 21 / 17 / 22, 4000 36 / 26 / 30 (ragged 35 / 25 /
  // 24); 32 heads over 8 x 128, 1 x 1000 16 / 13 / 16, 2000 25 / 19 / 16, 16 x 2000 26 / 19 / 22,
  // 64 x 1000 22 / 27 / 30, 2000 36 / 41 / 42 (ragged 32 / 37 / 32), 4000 63 / 67 / 65 (ragged
  // 55 / 60 / 44).  Two column tiles a wave (8 tokens): 4 x 64, 64 x 2000 29 / 22 / 33, 4000 51
  // / 37 / 46; 8 x 128, 16 x 2000 35 / 28 / 32, 64 x 2000 51 / 58 / 67.
  const long long span = static_cast<long long>(window) + T;
  const long long seen = window > 0 && span < p->cap_len ? span : p->cap_len;
  const long long rounds = (seen + 4 * kMxStep - 1) / (4 * kMxStep);
  bool whole;
  if (hd == 128 && units >= cus) {
    whole = rounds <= 16;
    p->W = 4;
  } else {
    whole = rounds <= 8 || (rounds <= 16 && (hd == 64 || 4 * units >= cus)) ||
            (rounds <= 32 && hd == 64 && units >= cus);
    p->W = whole ? mx4_most(hd, p->NT) : 4;
  }
  p->runs = whole ? 0 : static_cast<int>(cus) * mx4_waves(hd, p->NT);
  p->groups = whole ? units : p->runs;
  p->ws = whole ? 0
                : 2ll * p->runs * p->GT * (hd + 2) * 4 + (static_cast<long long>(B) + 1) * 4;
  // all steps, a run's steps and the grids are 32-bit
  const double steps = static_cast<double>(B) * (p->cap_len / kMxStep + 1 + kMxPad);
  return steps < 2147483647. &&
         (whole || steps * Hkv * p->HT / p->runs < 2147483647.) && p->groups < (1ll << 31) &&
         static_cast<double>(B) * T * Hq < 2147483647. && 4 * units < (1ll << 31);
}

template <int HD, int NT>
int32_t launch_mx4(const Mx4Args& a, const Mx4Plan& p, hipStream_t s) {
  constexpr int MOST = mx4_most(HD, NT);
  const dim3 grid(static_cast<unsigned>(p.groups));
  if (p.W == 4)
    hipLaunchKernelGGL((mx4_attn_kernel<HD, NT, 4>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((mx4_attn_kernel<HD, NT, MOST>), grid, dim3(64 * MOST), 0, s, a);
  if (p.runs == 0) return launch_status();
  const int parts = (p.GT + kMxJoinCols - 1) / kMxJoinCols;
  hipLaunchKernelGGL(mx4_join_kernel<HD>,
                     dim3(static_cast<unsigned>(a.B) * a.hkv * a.HT * parts), dim3(kMxJoin), 0, s,
                     a, 16 * NT, parts);
  return launch_status();
}

}  // namespace llmy

using namespace llmy;

extern "C" int64_t llmy_paged_attn_mx4_workspace_bytes(int32_t B, int32_t T, int32_t Hq,
                                                       int32_t Hkv, int32_t head_dim,
                                                       int32_t width, int32_t page,
                                                       int32_t window) {
  Mx4Plan p;
  return mx4_plan(B, T, Hq, Hkv, head_dim, width, page, window, &p) ? p.ws : -1;
}

extern "C" int32_t llmy_paged_attn_mx4(
    const llmy_bf16* q, int64_t q_seq, int64_t q_row, int64_t q_head, const void* k_cache,
    const void* v_cache, const void* k_scales, const void* v_scales, const int32_t* page_table,
    const int32_t* lengths, const float* slopes, llmy_bf16* out, void* workspace,
    int64_t workspace_bytes, int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t head_dim,
    int32_t width, int32_t page, int32_t pages, int32_t window, float scale, float softcap,
    void* stream) {
  Mx4Plan p;
  LLMY_REQUIRE(mx4_plan(B, T, Hq, Hkv, head_dim, width, page, window, &p));
  LLMY_REQUIRE(pages >= 0 && scale_ok(scale, softcap));
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
  a.page_bytes = static_cast<uint32_t>(Hkv) * page * (head_dim / 2);
  a.runs = p.runs;
  const hipStream_t s = as_stream(stream);
  if (head_dim == 64)
    return p.NT == 1 ? launch_mx4<64, 1>(a, p, s) : launch_mx4<64, 2>(a, p, s);
  return p.NT == 1 ? launch_mx4<128, 1>(a, p, s) : launch_mx4<128, 2>(a, p, s);
}
