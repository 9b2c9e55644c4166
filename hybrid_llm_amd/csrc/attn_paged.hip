// Attention of one new token per sequence over a paged key-value cache:
//   z_j = scale q . k_j, capped: c tanh(z / c), less slope_h (len - 1 - j);
//   o = sum_j softmax(z)_j v_j over the positions max(0, len - W) <= j < len,
// query head h reading key-value head h / (Hq / Hkv).  Cache and page table as in
// paged.hpp, bf16 or e4m3 times a scale.
//
// Bound by the read of K and V, whatever the grouping: a group's query heads (up to
// 16) are the columns of one 16 x 16 x 32 MFMA, so a key row is read once for all of
// them, and the matrix cores do with 16 columns what vector code would have to do once
// per head.
//   * S^T = K Q^T: lane l (g = l / 16) gets keys 4 g + r of a 16-key tile for head
//     l % 16.  Two such tiles are, register by register, the B operand of a 32-key
//     product O^T += V^T P^T under the key order 4 g + j, 16 + 4 g + j, so the
//     weights never leave their registers; V^T comes from transposing LDS reads of
//     row-major V rows in that order.
//   * a wave works alone: its 32-key steps arrive by DMA into 2 or 3 LDS stages of its
//     own and it waits for no other wave.  Four to twelve waves a CU keep 64 KiB and
//     more in flight per CU, several times what the read rate needs to cover a load's
//     latency.
//   * short tables: a workgroup takes a head, its waves every fourth or eighth step, and
//     joins their (m, l, O) in LDS.
//   * long ones: the work is the flat list of all (sequence, key-value head, step), cut into
//     equal runs: one run per wave, found from the lengths on the device.  A batch of
//     any mixture of lengths is balanced, and the host never learns the lengths.  A
//     run that starts or ends inside a head's steps leaves (m, l, O) partials in the
//     workspace, at most two, and a second kernel joins them; a head that lies in
//     one run is stored by that wave.  64 sequences of up to 4096 tokens, 32 heads
//     over 8 x 128: 95-100 us, 5.6 TB/s of the visible keys (all of 4096: 169 us, 6.1); four of
//     131072 in e4m3: 179 us, 5.9.
//   * the page ids come by scalar loads (a page holds whole 16-key tiles, so they are
//     the same for every lane of a DMA), which leaves the vector counter to the DMAs.
// Masked keys (past the length, before the window, in a page that the table does not
// name) have their scores set to -inf and their V rows zeroed in LDS, so nothing
// that such a place holds, NaN and infinities included, reaches a sum.
//
// Weights enter the product as the sum of two bf16, 16 bits of each, which the idle matrix
// cores do on the side (within 2% of the time): the store is the only rounding that
// shows.  e4m3 converts to bf16 without rounding; its scales go into the score scale and
// the final factor.
#include "common.hpp"
#include "abi_util.hpp"
#include "attn_tile.hpp"
#include "paged.hpp"

namespace llmy {

// Read-only words at wave-uniform addresses, by scalar loads.
typedef const int32_t __attribute__((address_space(4)))* const_i32;

__device__ __forceinline__ int32_t scalar_at(const int32_t* p, long long i) {
  return reinterpret_cast<const_i32>(reinterpret_cast<uintptr_t>(p))[i];
}

constexpr int kStep = 32;      // keys a step
constexpr float kLowest = -3.402823466e38f;

struct PagedArgs {
  const uint16_t* q;
  long long qb, qh;            // strides of q by sequence and head (elements)
  const uint8_t *kc, *vc;
  const int32_t *table, *lengths;
  uint16_t* out;               // [B, Hq, HD]
  float *po, *pml;             // partials: O [2 runs, GT, HD] and (m, l) [2 runs, GT, 2]
  int32_t* starts;             // [B + 1]: steps of the sequences before each, and of all
  const float* slopes;
  float scale_log2, cap_log2, cap_x2, v_scale;
  int B, hq, hkv, G, HT, GT;   // G = Hq / Hkv in HT tiles of GT <= 16 heads
  int width, shift, pages, window, cap_len;
  int runs;
};

struct Seq {
  int len, lo, s0, s1;         // visible positions [lo, len), steps [s0, s1)
};

__device__ __forceinline__ Seq seq_of(int len, int cap_len, int window) {
  Seq s;
  s.len = min(max(len, 0), cap_len);
  s.lo = window > 0 ? max(0, s.len - window) : 0;
  s.s0 = s.lo / kStep;
  s.s1 = static_cast<int>((static_cast<unsigned>(s.len) + kStep - 1) / kStep);
  return s;
}

// Steps of all sequences (the host sees to it that they fit 31 bits), as sums over 64
// blocks of `per` sequences, one per lane.
struct StepScan {
  int before, upto, total;  // this lane's block: exclusive and inclusive sums
  int per;
};

__device__ __forceinline__ StepScan scan_steps(const PagedArgs& a, int lane) {
  StepScan r;
  r.per = (a.B + kWave - 1) / kWave;
  int n = 0;
  const int b1 = min(a.B, (lane + 1) * r.per);
  for (int b = lane * r.per; b < b1; ++b) {
    const Seq s = seq_of(a.lengths[b], a.cap_len, a.window);
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

__device__ __forceinline__ int run_steps(long long total, int runs) {
  const long long q = (total + runs - 1) / runs;
  return static_cast<int>(q > 1 ? q : 1);
}

// What turns a row's sum of weighted values into its output: scale / sum of weights; without
// a visible key (m -inf) 0, with only scores of -inf NaN.
__device__ __forceinline__ float share(float m, float l, float scale) {
  return l != 0.f ? scale / l : m == -INFINITY ? 0.f : NAN;
}

// A part's sum under its weight beside the others, which may have vanished: infinities and
// NaN, those of visible values, stay all the same.
__device__ __forceinline__ float weighted(float x, float f) {
  return f != 0.f ? x * f : fabsf(x) < INFINITY ? 0.f : x;
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 8 e4m3 codes as bf16 (exact).
__device__ __forceinline__ bf16x8 e4m3_to_bf16(uint32_t lo, uint32_t hi) {
  uint4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
  return as_bf16x8(r);
}

// Staged rows keep their 16-byte chunks XOR-swizzled so that the fragment reads below
// spread over the banks: 8 lanes reading one chunk of 8 consecutive key rows, and a
// 16-lane group reading 4 (bf16) or 8 (e4m3) key rows of one transposed V tile.
template <int HD, bool F8, int W>
struct Tile {
  static constexpr int RB = HD * (F8 ? 1 : 2);       // bytes a row
  static constexpr int CH = RB / 16;                 // chunks a row
  static constexpr int RPB = 64 / CH;                // rows of one 1 KiB DMA
  static constexpr int NB = kStep / RPB;             // DMAs of a K or V tile
  static constexpr int BYTES = kStep * RB;           // of a K or V tile
  static constexpr int STAGES = F8 || HD == 128 || W > 1 ? 2 : 3;
  static constexpr int LDS = 2 * STAGES * BYTES;     // of a wave
  static __device__ __forceinline__ int kswz(int row) {
    return CH == 4 ? (row >> 1) & 3 : row & 7;
  }
  static __device__ __forceinline__ int vswz(int row) {
    if (!F8) return 2 * (row & 3);
    const int n = (row & 3) | ((row >> 2) & 4);  // its place among the group's 8 rows
    return CH == 4 ? n >> 1 : n;
  }
};

// W waves: 1: a run of the flat list; more: a head tile, each wave every W-th of its steps.
// (Waves a SIMD: as many as paged_runs counts on; 129 registers for e4m3 of 128 dims.)
template <int HD, bool F8, int W>
__global__ __launch_bounds__(64 * W, W > 1 ? W / 4 : F8 ? 3 : HD == 64 ? 2 : 1)
void paged_attn_kernel(const PagedArgs a) {
  using T = Tile<HD, F8, W>;
  constexpr int RB = T::RB, NB = T::NB, ST = T::STAGES;
  constexpr int NS = HD / 32;                 // 32-dim slices of the score product
  constexpr int ND = HD / 16;                 // 16-dim output tiles
  constexpr int NK = F8 ? HD / 64 : HD / 32;  // 16-byte K reads of a 16-key tile
  __shared__ __align__(1024) uint8_t smem[W * T::LDS];

  const int lane = threadIdx.x & 63;
  const int wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int g = lane >> 4, col = lane & 15;
  const int units = a.hkv * a.HT;

  // this wave's run: `count` steps from step s of head tile u of sequence b on
  int b, u, s, count, run_q = 0;
  long long run_at = 0;
  Seq cur;
  if (W > 1) {
    b = blockIdx.x / units;
    u = blockIdx.x - b * units;
    cur = seq_of(scalar_at(a.lengths, b), a.cap_len, a.window);
    s = cur.s0 + wave;
    count = max(0, (cur.s1 - s + W - 1) / W);
    if (cur.s0 == cur.s1) {  // nothing visible: zeros
      const int kvh = u / a.HT, ht = u - kvh * a.HT;
      const int heads = min(16, a.G - 16 * ht);
      uint16_t* o = a.out + (static_cast<long long>(b) * a.hq + kvh * a.G + 16 * ht) * HD;
      for (int e = 8 * threadIdx.x; e < heads * HD; e += 512 * W)
        *reinterpret_cast<uint4*>(o + e) = uint4{0u, 0u, 0u, 0u};
      return;
    }
  } else {
    const StepScan sc = scan_steps(a, lane);
    if (blockIdx.x == 0) {  // where each sequence's steps begin, for the join
      int at = sc.before;
      const int b1 = min(a.B, (lane + 1) * sc.per);
      for (int i = lane * sc.per; i < b1; ++i) {
        a.starts[i] = at;
        const Seq q = seq_of(a.lengths[i], a.cap_len, a.window);
        at += q.s1 - q.s0;
      }
      if (lane == 0) a.starts[a.B] = sc.total;
    }
    const long long total = static_cast<long long>(sc.total) * units;
    run_q = run_steps(total, a.runs);
    run_at = static_cast<long long>(blockIdx.x) * run_q;
    if (run_at >= total) return;
    count = static_cast<int>(min(static_cast<long long>(run_q), total - run_at));
    const uint64_t past = __ballot(static_cast<long long>(sc.upto) * units > run_at);
    const int blk = __ffsll(static_cast<unsigned long long>(past)) - 1;
    long long at = __builtin_amdgcn_readlane(sc.before, blk);
    b = blk * sc.per;
    for (;; ++b) {  // ends: the block's sum passes run_at
      cur = seq_of(scalar_at(a.lengths, b), a.cap_len, a.window);
      if ((at + cur.s1 - cur.s0) * units > run_at) break;
      at += cur.s1 - cur.s0;
    }
    const long long rem = run_at - at * units;
    u = static_cast<int>(rem / (cur.s1 - cur.s0));
    s = cur.s0 + static_cast<int>(rem - static_cast<long long>(u) * (cur.s1 - cur.s0));
  }

  // DMA lanes: lane p of block j fills row RPB j + p / CH, chunk slot p % CH
  uint32_t kdo[NB], vdo[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int r = T::RPB * j + lane / T::CH, sl = lane % T::CH;
    kdo[j] = (lane / T::CH) * RB + 16 * (sl ^ T::kswz(r));
    vdo[j] = (lane / T::CH) * RB + 16 * (sl ^ T::vswz(r));
  }
  uint8_t* const mem = smem + wave * T::LDS;  // this wave's stages
  const uint32_t sbase = lds_addr(mem);
  unsigned bad = 0;  // two bits a stage: its 16-key tiles whose page the table does not name
  int ib = b, iu = u, is = s;
  Seq icur = cur;
  auto next = [&](int& nb, int& nu, int& ns, Seq& q) {  // the step after; the caller counts
    ns += W;
    if (W > 1 || ns < q.s1) return;
    if (++nu == units) {
      nu = 0;
      do {
        q = seq_of(scalar_at(a.lengths, ++nb), a.cap_len, a.window);
      } while (q.s0 == q.s1);
    }
    ns = q.s0;
  };
  auto issue = [&](int st) {
    const int kvh = iu / a.HT;
    const long long row = static_cast<long long>(ib) * a.width;
    const int key0 = is * kStep;
    const int last = (icur.len - 1) >> a.shift;  // keys past the length stay in its page
    const uint32_t dst = sbase + st * 2 * T::BYTES;
    bad &= ~(3u << (2 * st));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = key0 + 16 * h;
      const int page = scalar_at(a.table, row + min(key >> a.shift, last));
      const bool ok = page >= 0 && page < a.pages;
      if (!ok) bad |= 1u << (2 * st + h);
      const long long at = (((static_cast<long long>(ok ? page : 0) * a.hkv + kvh) << a.shift) +
                            (key & ((1 << a.shift) - 1))) * RB;
      const uint8_t *kp = a.kc + at, *vp = a.vc + at;
#pragma unroll
      for (int j = 0; j < NB / 2; ++j) {
        const int blk = h * (NB / 2) + j;
        lds_fill16<true>(kp + j * 1024, kdo[blk], dst + blk * 1024);
        lds_fill16<true>(vp + j * 1024, vdo[blk], dst + T::BYTES + blk * 1024);
      }
    }
  };

  // fragment offsets (bytes from a stage's K or V tile)
  uint32_t koff[NK], voff[ND];
#pragma unroll
  for (int t = 0; t < NK; ++t) koff[t] = col * RB + 16 * ((4 * t + g) ^ T::kswz(col));
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    if (F8) {
      const int n = col >> 1, row = (n < 4 ? 0 : 16) + 4 * g + (n & 3);
      voff[d] = row * RB + 16 * (d ^ T::vswz(row)) + 8 * (col & 1);
    } else {
      const int row = 4 * g + (col >> 2), dim = 16 * d + 4 * (col & 3);
      voff[d] = row * RB + 16 * ((dim >> 3) ^ T::vswz(row)) + 2 * (dim & 7);
    }
  }

  int issued = 0;
  for (; issued < ST && issued < count; ++issued) {
    if (issued) next(ib, iu, is, icur);
    issue(issued);
  }

  uint4 qf[NS];
  f32x4 acc[ND];
  float m_run = -INFINITY, l_run = 0.f, slope = 0.f;
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  // After a part, the steps from `from` to `to` of a head: a visible value that is not finite
  // is what its dim becomes for every head, but left NaN there under a weight that had
  // vanished.  Seen by the sums, then looked up in memory, but for rows that are NaN as a
  // whole (l, their sum of weights).  (e4m3 has no infinities.)
  auto settle = [&](int from, int to, float l) __attribute__((always_inline)) {
    if (F8) return;
    float bad = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) bad = fmaf(acc[d][r], 0.f, bad);
    if (!__ballot(bad != 0.f && l == l)) return;  // bad: NaN of an infinity or a NaN
    const long long row = static_cast<long long>(b) * a.width;
    const int kvh = u / a.HT;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma nounroll
      for (int at = from; at <= to; at += W) {
        const int first = max(at * kStep, cur.lo), end = min((at + 1) * kStep, cur.len);
#pragma nounroll
        for (int key = first; key < end; ++key) {
          const int page = scalar_at(a.table, row + (key >> a.shift));
          if (page < 0 || page >= a.pages) continue;
          const long long slot = ((static_cast<long long>(page) * a.hkv + kvh) << a.shift) +
                                 (key & ((1 << a.shift) - 1));
          const uint2 w = *reinterpret_cast<const uint2*>(a.vc + slot * RB + 32 * d + 8 * g);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t half = r < 2 ? w.x : w.y;
            const float v = __uint_as_float(r & 1 ? half & 0xffff0000u : half << 16);
            if (!(fabsf(v) < INFINITY)) t[r] += v;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!(fabsf(t[r]) < INFINITY)) acc[d][r] = t[r];
    }
  };
  bool fresh = true;
  int st = 0;
  for (int i = 0; i < count; ++i) {
    const int kvh = u / a.HT, ht = u - kvh * a.HT;
    const int heads = min(16, a.G - 16 * ht);
    const int h0 = kvh * a.G + 16 * ht;
    if (fresh) {
      fresh = false;
      const uint16_t* qp = a.q + b * a.qb + (h0 + min(col, heads - 1)) * a.qh;
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        const int d0 = F8 ? 64 * (t / 2) + 16 * g + 8 * (t & 1) : 32 * t + 8 * g;
        qf[t] = *reinterpret_cast<const uint4*>(qp + d0);
      }
      if (a.slopes) slope = slope_log2(a.slopes[h0 + min(col, heads - 1)], kMaxSlope);
      m_run = -INFINITY;
      l_run = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // DMAs complete in order: this stage has landed once only later stages' are out
    if (issued - i == ST) wait_vm<(ST - 1) * 2 * NB>();
    else wait_vm<0>();
    const uint32_t kst = sbase + st * 2 * T::BYTES, vst = kst + T::BYTES;
    const int key0 = s * kStep;
    const unsigned hole = (bad >> (2 * st)) & 3u;
    const bool edge = key0 < cur.lo || key0 + kStep > cur.len || hole;

    u32x4 kf[2 * NK];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int t = 0; t < NK; ++t) kf[k * NK + t] = lds_get16(kst + 16 * k * RB + koff[t]);
    if (edge) {  // masked keys' V rows are zeroed
      for (int e = lane; e < kStep * T::CH; e += 64) {
        const int row = e / T::CH, key = key0 + row;
        if (key < cur.lo || key >= cur.len || ((hole >> (row >> 4)) & 1u))
          *reinterpret_cast<uint4*>(mem + st * 2 * T::BYTES + T::BYTES + 16 * e) =
              uint4{0u, 0u, 0u, 0u};
      }
      wave_lds_order();
    }
    constexpr int NV = F8 ? ND : 2 * ND;
    u32x2 vf[NV];
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      if (F8) {
        vf[d] = lds_get_tr8(vst + voff[d]);
      } else {
        vf[2 * d] = lds_get_tr16(vst + voff[d]);
        vf[2 * d + 1] = lds_get_tr16(vst + voff[d] + 16 * RB);
      }
    }
    f32x4 sc[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      sc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        bf16x8 kk;
        if (F8) {
          const u32x4 w = kf[k * NK + t / 2];
          kk = (t & 1) ? e4m3_to_bf16(w.z, w.w) : e4m3_to_bf16(w.x, w.y);
        } else {
          kk = __builtin_bit_cast(bf16x8, kf[k * NK + t]);
        }
        sc[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, as_bf16x8(qf[t]), sc[k], 0, 0, 0);
      }
    }
    float z[8];
    // a step with a visible key lifts the maximum to the lowest finite number, also if they
    // all score -inf: softmax over such alone is NaN, over no key it gives zeros
    const auto shows = [&](int h) {
      const int first = key0 + 16 * h;
      return !((hole >> h) & 1u) && max(first, cur.lo) < min(first + 16, cur.len);
    };
    float mloc = !edge || shows(0) || shows(1) ? kLowest : -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x = sc[j >> 2][j & 3];
      x = a.cap_x2 > 0.f ? softcap_log2(x * a.cap_x2, a.cap_log2) : x * a.scale_log2;
      const int key = key0 + 16 * (j >> 2) + 4 * g + (j & 3);
      if (a.slopes) x -= slope * static_cast<float>(cur.len - 1 - key);
      if (edge && (key < cur.lo || key >= cur.len || ((hole >> (j >> 2)) & 1u))) x = -INFINITY;
      z[j] = x;
      mloc = fmaxf(mloc, x);
    }
    // the offset moves only when some score passes it by more than 8 (weights stay
    // below 2^8), decided by the wave; all four lanes of a head take the same one
    if (__ballot(!(mloc <= m_run + 8.f))) {
      mloc = fmaxf(mloc, __shfl_xor(mloc, 16, kWave));
      mloc = fmaxf(mloc, __shfl_xor(mloc, 32, kWave));
      const float m_new = fmaxf(m_run, mloc);
      const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] *= alpha;
    }
    const float m_sub = m_run == -INFINITY ? 0.f : m_run;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = exp2_fast(z[j] - m_sub);
    // the weights as a sum of two bf16: the matrix cores have time to spare here.  The
    // first is cut off below the weight, so both are positive and an infinite value
    // stays that infinity
    uint32_t h8[8];
    float lo8[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      l_run += p[j];
      h8[j] = __float_as_uint(p[j] * (1.f - 0x1p-8f)) & 0xffff0000u;
      lo8[j] = p[j] - __uint_as_float(h8[j]);
    }
    const uint4 pb = uint4{h8[0] >> 16 | h8[1], h8[2] >> 16 | h8[3], h8[4] >> 16 | h8[5],
                           h8[6] >> 16 | h8[7]};
    const uint4 pl = pack8_bf16(lo8);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const bf16x8 vv = F8 ? e4m3_to_bf16(vf[d].x, vf[d].y)
                           : as_bf16x8(uint4{vf[F8 ? 0 : 2 * d].x, vf[F8 ? 0 : 2 * d].y,
                                             vf[F8 ? 0 : 2 * d + 1].x, vf[F8 ? 0 : 2 * d + 1].y});
      acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, as_bf16x8(pb), acc[d], 0, 0, 0);
      acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, as_bf16x8(pl), acc[d], 0, 0, 0);
    }
    // once every read of this stage has returned, the next step may land in it
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (issued < count) {
      next(ib, iu, is, icur);
      issue(st);
      ++issued;
    }
    st = st + 1 == ST ? 0 : st + 1;

    const bool head_end = s + 1 == cur.s1;
    if (W == 1 && (head_end || i + 1 == count)) {
      float l = l_run + __shfl_xor(l_run, 16, kWave);
      l += __shfl_xor(l, 32, kWave);
      // whole: the head's first step lies in this run too
      const bool whole = head_end && i >= s - cur.s0;
      settle(max(cur.s0, s - i), s, l);
      if (whole) {
        const float f = share(m_run, l, a.v_scale);
        uint16_t* o = a.out + (static_cast<long long>(b) * a.hq + h0 + col) * HD + 4 * g;
        if (col < heads)
#pragma unroll
          for (int d = 0; d < ND; ++d)
            *reinterpret_cast<uint2*>(o + 16 * d) =
                make_uint2(pack_bf2(acc[d][0] * f, acc[d][1] * f),
                           pack_bf2(acc[d][2] * f, acc[d][3] * f));
      } else if (col < heads) {
        // the run starts in this head (or at its first step): 0; else it ends in it: 1
        const int part = i > s - cur.s0 ? 1 : 0;
        const long long at = (2ll * blockIdx.x + part) * a.GT + col;
        float* o = a.po + at * HD + 4 * g;
#pragma unroll
        for (int d = 0; d < ND; ++d)
          *reinterpret_cast<float4*>(o + 16 * d) =
              make_float4(acc[d][0], acc[d][1], acc[d][2], acc[d][3]);
        if (g == 0) *reinterpret_cast<float2*>(a.pml + 2 * at) = make_float2(m_run, l);
      }
      fresh = true;
    }
    if (i + 1 < count) next(b, u, s, cur);
  }
  if constexpr (W > 1) {
    // the waves' (m, l, O) joined through each one's stages, which it has done with
    constexpr int LD = HD + 4;
    static_assert((16 * LD + 32) * 4 <= T::LDS, "a wave's part fits its stages");
    const int kvh = u / a.HT, ht = u - kvh * a.HT;
    const int heads = min(16, a.G - 16 * ht);
    float l = l_run + __shfl_xor(l_run, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
    settle(cur.s0 + wave, cur.s1 - 1, l);
    float* const so = reinterpret_cast<float*>(mem);
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *reinterpret_cast<float4*>(so + col * LD + 16 * d + 4 * g) =
          make_float4(acc[d][0], acc[d][1], acc[d][2], acc[d][3]);
    if (g == 0) *reinterpret_cast<float2*>(so + 16 * LD + 2 * col) = make_float2(m_run, l);
    __syncthreads();
    uint16_t* o = a.out + (static_cast<long long>(b) * a.hq + kvh * a.G + 16 * ht) * HD;
    for (int e = threadIdx.x; e < heads * (HD / 4); e += 64 * W) {
      const int h = e / (HD / 4), c = 4 * (e - h * (HD / 4));
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w)
        mx = fmaxf(mx, reinterpret_cast<const float*>(smem + w * T::LDS)[16 * LD + 2 * h]);
      const float m_sub = mx == -INFINITY ? 0.f : mx;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float* part = reinterpret_cast<const float*>(smem + w * T::LDS);
        const float2 ml = *reinterpret_cast<const float2*>(part + 16 * LD + 2 * h);
        const float4 x = *reinterpret_cast<const float4*>(part + h * LD + c);
        const float f = exp2_fast(ml.x - m_sub);
        den = fmaf(ml.y, f, den);  // NaN of a NaN score, whatever its part's weight
        sum.x += weighted(x.x, f);
        sum.y += weighted(x.y, f);
        sum.z += weighted(x.z, f);
        sum.w += weighted(x.w, f);
      }
      const float r = share(mx, den, a.v_scale);
      *reinterpret_cast<uint2*>(o + h * HD + c) =
          make_uint2(pack_bf2(sum.x * r, sum.y * r), pack_bf2(sum.z * r, sum.w * r));
    }
  }
}

// Joins the partials of one (sequence, query head): o = sum_i 2^(m_i - m) O_i /
// sum_i 2^(m_i - m) l_i, in the runs' order within each of T / (HD / 4) lane groups and
// then over the groups, so the result does not depend on timing.  A part without weight
// still adds its infinities, and its l, which is finite or, of a visible NaN score (no
// maximum sees one), NaN: then the row is NaN, however its head was cut.  T threads: 64
// where the heads alone fill the chip, 512 where few heads have many partials each.
template <int HD, int T>
__global__ __launch_bounds__(T) void paged_join_kernel(const PagedArgs a) {
  constexpr int LPP = HD / 4;       // lanes a partial
  constexpr int NG = T / LPP;
  __shared__ __align__(16) float so[NG][HD];
  __shared__ float sm[NG], sl[NG];
  const int grp = threadIdx.x / LPP, c = threadIdx.x % LPP;
  const int b = blockIdx.x / a.hq, h = blockIdx.x - b * a.hq;
  const int kvh = h / a.G, ht = (h - kvh * a.G) / 16, row = h - kvh * a.G - 16 * ht;
  const int units = a.hkv * a.HT, u = kvh * a.HT + ht;
  uint16_t* out = a.out + static_cast<long long>(blockIdx.x) * HD;

  const int start = scalar_at(a.starts, b), n = scalar_at(a.starts, b + 1) - start;
  if (n == 0) {  // nothing visible: zeros
    if (threadIdx.x < LPP) *reinterpret_cast<uint2*>(out + 4 * c) = make_uint2(0u, 0u);
    return;
  }
  const int q = run_steps(static_cast<long long>(scalar_at(a.starts, a.B)) * units, a.runs);
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
    o.x = weighted(x.x, e) + weighted(o.x, f);
    o.y = weighted(x.y, e) + weighted(o.y, f);
    o.z = weighted(x.z, e) + weighted(o.z, f);
    o.w = weighted(x.w, e) + weighted(o.w, f);
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
  for (int d = threadIdx.x; d < HD; d += T) {
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const float e = exp2_fast(sm[i] - m_sub);
      den = fmaf(sl[i], e, den);
      num += weighted(so[i][d], e);
    }
    out[d] = f2bf(num * share(mx, den, a.v_scale));
  }
}

// Waves that the chip holds at once: what a CU's 160 KiB of LDS take, 12 at most.
inline int paged_runs(int head_dim, bool f8) {
  const int lds = head_dim == 128 ? (f8 ? Tile<128, true, 1>::LDS : Tile<128, false, 1>::LDS)
                                  : (f8 ? Tile<64, true, 1>::LDS : Tile<64, false, 1>::LDS);
  const int per_cu = (163840 - 1) / lds;  // five of 32 KiB do not fit beside each other
  return compute_units() * (per_cu < 12 ? per_cu : 12);
}

struct PagedPlan {
  int G, HT, GT, waves, runs;
  bool wide;  // a workgroup of `waves` waves a head tile; else `runs` waves and their join
  long long cap_len, groups, ws;
};

inline bool paged_plan(int B, int Hq, int Hkv, int hd, int width, int page, int type,
                       PagedPlan* p) {
  if (B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq > kMaxHeads || (hd != 64 && hd != 128) ||
      width < 0 || page_shift(page) < 0 || (type != kCacheBf16 && type != kCacheE4m3))
    return false;
  p->G = Hq / Hkv;
  p->HT = (p->G + 15) / 16;
  p->GT = p->G < 16 ? p->G : 16;
  p->cap_len = static_cast<long long>(width) * page;
  if (p->cap_len >= (1ll << 31) - kStep) return false;  // positions are 32-bit
  const long long units = static_cast<long long>(B) * Hkv * p->HT;
  // Short tables: a head tile a workgroup, one launch.  us of it / of runs and their join,
  // lengths near the table's unless ragged: 1 x 16 heads over 4 x 64, 256 tokens 4.3 / 8.6,
  // 1024 8.0 / 9.4, 2048 13 / 10; 64 sequences of them, 1024 14 / 21, 2048 24 / 31 (ragged
  // 19 / 22), 4096 ragged 33 / 34; 32 heads over 8 x 128 in e4m3, 64 x 1024 29 / 34, 2048
  // 48 / 55 (ragged 37 / 37), in bf16, 1 x 256 6.2 / 8.8, 512 9.8 / 9.2, 64 x 512 30 / 32,
  // 1024 49 / 52 (ragged 41 / 36).  So up to four steps a wave, and up to eight where
  // there are many heads and eight waves.
  const int W = p->waves = hd == 128 && type == kCacheBf16 ? 4 : 8;
  const long long deep = (p->cap_len + kStep * W - 1) / (kStep * W);
  p->wide = deep <= 4 || (W == 8 && deep <= 8 && 2 * units >= compute_units());
  p->runs = p->wide ? 0 : paged_runs(hd, type == kCacheE4m3);
  p->groups = p->wide ? units : p->runs;
  p->ws = p->wide ? 0
                  : 2ll * p->runs * p->GT * (hd + 2) * 4 + (static_cast<long long>(B) + 1) * 4;
  // all steps, a run's steps and the grids are 32-bit
  const double steps = static_cast<double>(B) * (p->cap_len / kStep + 1);
  return steps < 2147483647. &&
         (p->wide || steps * Hkv * p->HT / p->runs < 2147483647.) && p->groups < (1ll << 31) &&
         static_cast<long long>(B) * Hq < (1ll << 31);
}

template <int HD, bool F8>
int32_t launch_paged(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  constexpr int W = HD == 128 && !F8 ? 4 : 8;  // 128 KiB of stages at the most (p.waves)
  const dim3 grid(static_cast<unsigned>(p.groups)), heads(static_cast<unsigned>(a.B) * a.hq);
  if (p.wide) {
    hipLaunchKernelGGL((paged_attn_kernel<HD, F8, W>), grid, dim3(64 * W), 0, s, a);
    return launch_status();
  }
  hipLaunchKernelGGL((paged_attn_kernel<HD, F8, 1>), grid, dim3(64), 0, s, a);
  if (heads.x >= 1024)
    hipLaunchKernelGGL((paged_join_kernel<HD, 64>), heads, dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL((paged_join_kernel<HD, 512>), heads, dim3(512), 0, s, a);
  return launch_status();
}

}  // namespace llmy

using namespace llmy;

extern "C" int64_t llmy_paged_attn_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv,
                                                   int32_t head_dim, int32_t width, int32_t page,
                                                   int32_t cache_type) {
  PagedPlan p;
  return paged_plan(B, Hq, Hkv, head_dim, width, page, cache_type, &p) ? p.ws : -1;
}

extern "C" int32_t llmy_paged_attn_decode(
    const llmy_bf16* q, int64_t q_row, int64_t q_head, const void* k_cache, const void* v_cache,
    int32_t cache_type, float k_scale, float v_scale, const int32_t* page_table,
    const int32_t* lengths, const float* slopes, llmy_bf16* out, void* workspace,
    int64_t workspace_bytes, int32_t B, int32_t Hq, int32_t Hkv, int32_t head_dim, int32_t width,
    int32_t page, int32_t pages, int32_t window, float scale, float softcap, void* stream) {
  PagedPlan p;
  LLMY_REQUIRE(paged_plan(B, Hq, Hkv, head_dim, width, page, cache_type, &p));
  LLMY_REQUIRE(pages >= 0 && window >= 0 && scales_ok(cache_type, k_scale, v_scale) &&
               scale_ok(scale * k_scale, softcap));
  if (B == 0) return 0;
  LLMY_REQUIRE(q && out && lengths && aligned(q, 16) && aligned(out, 16));
  LLMY_REQUIRE(q_row % 8 == 0 && q_head % 8 == 0 && q_row >= 0 && q_head >= 0);
  LLMY_REQUIRE(apart(q, rows_extent(q_row, q_head, B, Hq, head_dim), out,
                     static_cast<int64_t>(B) * Hq * head_dim));
  LLMY_REQUIRE(width == 0 || page_table);
  // with no page at all every length counts as 0
  LLMY_REQUIRE(pages == 0 || (k_cache && v_cache && aligned(k_cache, 16) && aligned(v_cache, 16)));
  LLMY_REQUIRE(p.ws == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= p.ws));
  // out and the workspace are written while other workgroups still read
  const int64_t out_bytes = 2ll * B * Hq * head_dim;
  const int64_t cache_bytes = static_cast<int64_t>(pages) * Hkv * page * head_dim *
                              (cache_type == kCacheE4m3 ? 1 : 2);
  LLMY_REQUIRE(bytes_apart(out, out_bytes, k_cache, cache_bytes) &&
               bytes_apart(out, out_bytes, v_cache, cache_bytes) &&
               bytes_apart(workspace, p.ws, k_cache, cache_bytes) &&
               bytes_apart(workspace, p.ws, v_cache, cache_bytes) &&
               bytes_apart(workspace, p.ws, out, out_bytes) &&
               rows_apart(Rows{q, q_row, q_head, B, Hq, head_dim}, workspace, p.ws));
  PagedArgs a{};
  a.q = q; a.qb = q_row; a.qh = q_head;
  a.kc = static_cast<const uint8_t*>(k_cache);
  a.vc = static_cast<const uint8_t*>(v_cache);
  a.table = page_table; a.lengths = lengths; a.out = out; a.slopes = slopes;
  a.po = static_cast<float*>(workspace);
  a.pml = a.po + 2ll * p.runs * p.GT * head_dim;
  a.starts = reinterpret_cast<int32_t*>(a.pml + 4ll * p.runs * p.GT);
  const float log2e = 1.4426950408889634f, qk = scale * k_scale;
  a.scale_log2 = qk * log2e;
  a.cap_log2 = softcap * log2e;
  a.cap_x2 = softcap > 0.f ? 2.f * log2e * qk / softcap : 0.f;
  a.v_scale = v_scale;
  a.B = B; a.hq = Hq; a.hkv = Hkv; a.G = p.G; a.HT = p.HT; a.GT = p.GT;
  a.width = width; a.shift = page_shift(page); a.pages = pages; a.window = window;
  a.cap_len = pages ? static_cast<int>(p.cap_len) : 0;
  a.runs = p.runs;
  const hipStream_t s = as_stream(stream);
  return cache_type == kCacheE4m3
             ? (head_dim == 64 ? launch_paged<64, true>(a, p, s) : launch_paged<128, true>(a, p, s))
             : (head_dim == 64 ? launch_paged<64, false>(a, p, s)
                               : launch_paged<128, false>(a, p, s));
}
