// Verification of drafted tokens against the target's probabilities, from given uniforms.
//
// Row t of a sequence is the target's after t of its drafts: p_t = softmax(logits_t / T).
// Draft x_t, drawn from q_t, is kept while u_t q_t(x_t) < p_t(x_t); the first that is not is
// replaced by a draw from max(p_t - q_t, 0), and behind the last draft comes one from p:
// the ids that come out are distributed as the target's own.  The draw is the first id, in
// their order, at which the running sum passes u times the whole.
//
// The draw looks for a border among up to V of them, and sums in 32 bits move a border by
// more than their distance at large V; so exponentials and sums are in 64 bits, which this
// chip adds and multiplies at the rate of single 32-bit ones.
//
// Bound by the read of the logits (then of one draft row a sequence) where there are many rows,
// by latency where there are few.  Rows are cut into chunks, so that one sequence's rows fill
// the chip too:
//   1. a workgroup's chunks of a row: their maximum and sum of exponentials under it;
//   2. per sequence: from those, which drafts are kept;
//   3. per sequence and chunk: its sum of the distribution to draw from;
//   4. per sequence: the chunk in which the sum passes the threshold, and the id in it.
// 2 to 4 are one launch for few sequences, where launches are what takes long.
// Greedy (T = 0): each row's first largest id, then the comparison: two launches.
// Measured, 64 sequences of 4 drafts, 128256 ids: 40 to 42 + 5 + 19 to 20 + 6.5 us, the first at 4 TB/s
// (its exponentials in 64 bits alone take 31 us, under the loads), the third at 3.0 to 3.2; greedy,
// 64 x 4 rows of 32000: 9.4 + 2 to 3 us, 3.5 TB/s; one sequence of 4 drafts, 32000 ids: 4.2 + 9.6.
#include "common.hpp"
#include "abi_util.hpp"
#include "paged.hpp"

namespace llmy {

constexpr int kVerThreads = 256, kVerPer = 16;
constexpr int kVerChunk = kVerThreads * kVerPer;
constexpr int kVerWaves = kVerThreads / kWave;
// Ids a thread of a draw, few, so that one sequence spreads over the chip and many hide their
// loads (1 x 32000 ids, 16 a thread against 4: 14 and 8 us; 64 x 128256: 28 and 25).
constexpr int kVerDraw = 4, kVerDrawChunk = kVerThreads * kVerDraw;
static_assert(kVerDraw == 4, "sums in the ids' order: a thread's are neighbours");
constexpr int kMaxDrafts = 63;  // rows of a sequence in LDS

struct VerifyArgs {
  const float* logits;          // [B, K + 1, V]
  const int32_t* drafts;        // [B, K]
  const float* probs;           // [B, K, V] or null: the drafts were certain
  const int32_t* counts;        // [B] or null: K
  const float* u;               // [B, K + 1]
  int32_t *tokens, *accepted;   // [B, K + 1], [B]
  uint64_t* best;               // [B (K + 1), parts]: largest (value, lowest id) of a part
  double* sum;                  // [B (K + 1), parts]: its sum under that maximum
  double *rest, *plain;         // [B, chunks]: of max(e - q Z, 0) and e of the drawn row
  struct Decision* decided;     // [B]
  uint32_t* done;               // [B] in their place: chunks whose sums are stored
  double c;                     // log2(e) / T
  int B, K, V;
  int row_chunks, per_part, parts;  // chunks of a row, of a first workgroup, and those of a row
  int chunks;                   // of a row that is drawn from
  bool vec4;
};

// 2^y for y up to about 0: 2^n 2^f, y = n + f, |f| <= 1/2, 2^f by the polynomial that meets it at
// ten Chebyshev points: off by 2^-45 of it.  0 below 2^-1075, also for -inf.  Adding 1.5 x 2^52
// rounds to a whole number and leaves it in the low word.
__device__ __forceinline__ double exp2_neg(double y) {
  y = fmax(y, -1100.0);
  const double t = y + 0x1.8p52, f = y - (t - 0x1.8p52);
  double s = 1.0212097549811005e-07;
  s = fma(s, f, 1.3259945262689143e-06);
  s = fma(s, f, 1.5252640059770786e-05);
  s = fma(s, f, 0.00015403432339553542);
  s = fma(s, f, 0.001333355825801874);
  s = fma(s, f, 0.009618129195951041);
  s = fma(s, f, 0.05550410866428854);
  s = fma(s, f, 0.24022650695631514);
  s = fma(s, f, 0.6931471805599526);
  s = fma(s, f, 1.000000000000014);
  return ldexp(s, static_cast<int>(static_cast<uint32_t>(__builtin_bit_cast(uint64_t, t))));
}

// e^((x - top) / T) for x at most top.  The difference first: where top c passes 2^53 (a
// temperature near 0), a product's rounding would pass whole powers of two.
__device__ __forceinline__ double weight(float x, double c, double top) {
  return exp2_neg((static_cast<double>(x) - top) * c);
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v += __shfl_xor(v, d, kWave);
  return v;
}

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t k = static_cast<uint32_t>(key >> 32);
  return k == 0xffffffffu ? __uint_as_float(0x7fc00000u)
                          : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// This thread's PER ids of a part of a row: the four from base + 1024 i + 4 t on, i < PER / 4;
// `none` past the row.  (All loads of a part that lies in the row go out together; a test
// around each would wait for the one before.)
template <int PER>
__device__ __forceinline__ void load_ids(const float* row, int V, int base, bool vec4, float none,
                                         float* v) {
  const float* own = row + base + 4 * static_cast<int>(threadIdx.x);
  if (vec4 && base + kVerThreads * PER <= V) {
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
      const float4 w = *reinterpret_cast<const float4*>(own + 1024 * i);
      v[4 * i] = w.x; v[4 * i + 1] = w.y; v[4 * i + 2] = w.z; v[4 * i + 3] = w.w;
    }
    return;
  }
  // else every address lies in the row, and what is past it is put right afterwards
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = base + 1024 * (i >> 2) + 4 * static_cast<int>(threadIdx.x) + (i & 3);
    v[i] = row[min(at, V - 1)];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = base + 1024 * (i >> 2) + 4 * static_cast<int>(threadIdx.x) + (i & 3);
    v[i] = at < V ? v[i] : none;
  }
}

// The lowest id of this thread's largest value `most` among its ids of a chunk (NaN above all); none:
// 2^31 - 1.  (A thread past the row's end has -inf, at ids behind it.)
__device__ __forceinline__ uint64_t first_key(const float* v, float most, int base, int V) {
  uint32_t at = 0x7fffffffu;
#pragma unroll
  for (int k = kVerPer - 1; k >= 0; --k) {
    const bool same = v[k] == most || (v[k] != v[k] && most != most);
    at = same ? base + 1024 * (k >> 2) + 4 * threadIdx.x + (k & 3) : at;
  }
  return at < static_cast<uint32_t>(V) ? value_index_key(most, at) : 0ull;
}

__device__ __forceinline__ float largest(const float* v) {
  float most = v[0];
#pragma unroll
  for (int k = 1; k < kVerPer; ++k) most = __builtin_elementwise_maximum(most, v[k]);
  return most;
}

// A part of a row: `per_part` chunks, the next one loaded under the present one's exponentials.
// Each thread keeps a maximum and a sum under it; the workgroup's are formed once, at the end.
template <bool GREEDY>
__global__ __launch_bounds__(kVerThreads) void verify_rows_kernel(const VerifyArgs a) {
  __shared__ uint64_t keys[kVerWaves];
  __shared__ double sums[kVerWaves];
  __shared__ float tops[kVerWaves];
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  const int c0 = part * a.per_part, c1 = min(a.row_chunks, c0 + a.per_part), wave = threadIdx.x >> 6;
  const float* x = a.logits + static_cast<long long>(row) * a.V;
  if (!GREEDY && part == 0 && threadIdx.x == 0 && row % (a.K + 1) == 0) a.done[row / (a.K + 1)] = 0u;
  float v[kVerPer], next[kVerPer];
  load_ids<kVerPer>(x, a.V, c0 * kVerChunk, a.vec4, -INFINITY, v);
  float top = -INFINITY;
  double s = 0;
  uint64_t key = 0;
  for (int c = c0; c < c1; ++c) {
    if (c + 1 < c1) load_ids<kVerPer>(x, a.V, (c + 1) * kVerChunk, a.vec4, -INFINITY, next);
    const float most = largest(v);
    if (GREEDY) {
      key = umax64(key, first_key(v, most, c * kVerChunk, a.V));
    } else {
      const float old = top;
      top = __builtin_elementwise_maximum(top, most);
      // (under a row's first -inf alone the offset is the lowest number: weights 0)
      const double under = fmaxf(top, -3.402823466e38f);
      s *= weight(old, a.c, under);
#pragma unroll
      for (int k = 0; k < kVerPer; ++k) s += weight(v[k], a.c, under);
    }
#pragma unroll
    for (int k = 0; k < kVerPer; ++k) v[k] = next[k];
  }
  if (!GREEDY) {
    float all = top;
    all = __builtin_elementwise_maximum(all, dpp_f<kDppXor1>(all));
    all = __builtin_elementwise_maximum(all, dpp_f<kDppXor2>(all));
    all = __builtin_elementwise_maximum(all, dpp_f<kDppHalfMirror>(all));
    all = __builtin_elementwise_maximum(all, dpp_f<kDppMirror>(all));
    all = __builtin_elementwise_maximum(
        __builtin_elementwise_maximum(readlane_f(all, 0), readlane_f(all, 16)),
        __builtin_elementwise_maximum(readlane_f(all, 32), readlane_f(all, 48)));
    if ((threadIdx.x & 63) == 0) tops[wave] = all;
    __syncthreads();
    all = __builtin_elementwise_maximum(__builtin_elementwise_maximum(tops[0], tops[1]),
                                        __builtin_elementwise_maximum(tops[2], tops[3]));
    if (fabsf(all) < INFINITY) {
      s = wave_sum_d(s * weight(top, a.c, all));
      if ((threadIdx.x & 63) == 0) sums[wave] = s;
      __syncthreads();
      if (threadIdx.x == 0) {
        a.best[blockIdx.x] = value_index_key(all, 0u);
        a.sum[blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
      }
      return;
    }
    // no finite largest: its id is looked for after all
    for (int c = c0; c < c1; ++c) {
      load_ids<kVerPer>(x, a.V, c * kVerChunk, a.vec4, -INFINITY, v);
      key = umax64(key, first_key(v, largest(v), c * kVerChunk, a.V));
    }
    if (threadIdx.x == 0) a.sum[blockIdx.x] = 0.;
  }
  key = wave_max_u64(key);
  if ((threadIdx.x & 63) == 0) keys[wave] = key;
  __syncthreads();
  if (threadIdx.x == 0)
    a.best[blockIdx.x] = umax64(umax64(keys[0], keys[1]), umax64(keys[2], keys[3]));
}

struct Row {
  uint64_t key;   // its largest value and that one's lowest id
  double z;       // sum of e^((x - largest) / T); rows without a finite largest: 1
  bool sure;      // no finite largest: the id of the key alone
};

struct Decision {
  Row row;        // the row that the new token comes from
  int kept;       // drafts kept before it
  bool rejected;  // a draft was put away there
};

// Which drafts of a sequence are kept: every row by 16 lanes, their verdicts through LDS.  By a
// workgroup, with the same result in each.
template <bool GREEDY>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, int b) {
  __shared__ Row rows[kMaxDrafts + 1];
  __shared__ int keep[kMaxDrafts + 1];
  const int sub = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int count = a.counts ? min(max(a.counts[b], 0), a.K) : a.K;
  for (int t0 = 0; t0 <= count; t0 += kVerThreads / 16) {
    const int t = min(t0 + sub, count);  // (the last row again by what lanes are left)
    const long long row = static_cast<long long>(b) * (a.K + 1) + t;
    const long long draft = static_cast<long long>(b) * a.K + min(t, a.K - 1);
    const int id = a.drafts[draft];
    const bool named = t < count && id >= 0 && id < a.V;
    float x = 0.f, q = 1.f, u = 0.f;
    if (!GREEDY && named) {
      x = a.logits[row * a.V + id];
      if (a.probs) q = a.probs[draft * a.V + id];
      u = a.u[row];
    }
    Row r;
    r.key = 0;
    for (int c = lane; c < a.parts; c += 16) r.key = umax64(r.key, a.best[row * a.parts + c]);
    r.key = umax64(r.key, dpp_u64<kDppXor1>(r.key));
    r.key = umax64(r.key, dpp_u64<kDppXor2>(r.key));
    r.key = umax64(r.key, dpp_u64<kDppHalfMirror>(r.key));
    r.key = umax64(r.key, dpp_u64<kDppMirror>(r.key));
    const float top = key_value(r.key);
    r.sure = GREEDY || !(fabsf(top) < INFINITY);
    r.z = 1.0;
    if (!GREEDY) {
      double z = 0;
      if (!r.sure)
        for (int c = lane; c < a.parts; c += 16)
          z += a.sum[row * a.parts + c] * weight(key_value(a.best[row * a.parts + c]), a.c, top);
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) z += __shfl_xor(z, d, kWave);
      if (!r.sure) r.z = z;
    }
    if (lane == 0) {
      rows[t] = r;
      const bool best = static_cast<uint32_t>(id) == key_index(r.key);
      const double e = r.sure ? (best ? 1.0 : 0.0) : weight(x, a.c, top);
      keep[t] = named && (GREEDY ? best : static_cast<double>(u) * q * r.z < e);
    }
  }
  __syncthreads();
  Decision d;
  d.kept = 0;
  while (d.kept < count && keep[d.kept]) ++d.kept;
  d.rejected = d.kept < count;
  d.row = rows[d.kept];
  return d;
}

// A sequence's outputs: the kept drafts, the new token, then -1.
__device__ __forceinline__ void put_tokens(const VerifyArgs& a, int b, const Decision& d, int id) {
  for (int t = threadIdx.x; t <= a.K; t += kVerThreads) {
    const int64_t at = static_cast<int64_t>(b) * (a.K + 1) + t;
    a.tokens[at] = t < d.kept ? a.drafts[static_cast<int64_t>(b) * a.K + t] : t == d.kept ? id : -1;
  }
  if (threadIdx.x == 0) a.accepted[b] = d.kept;
}

template <bool GREEDY>
__global__ __launch_bounds__(kVerThreads) void verify_decide_kernel(const VerifyArgs a) {
  const int b = blockIdx.x;
  const Decision d = decide<GREEDY>(a, b);
  if (GREEDY)
    put_tokens(a, b, d, static_cast<int>(key_index(d.row.key)));
  else if (threadIdx.x == 0)
    a.decided[b] = d;
}

// Weights of the drawn row at this thread's ids of a chunk, in order: put(k, e, max(e - q Z, 0)).
template <class Put>
__device__ __forceinline__ void draw_weights(const VerifyArgs& a, int b, const Decision& d, int base,
                                             Put put) {
  const long long row = static_cast<long long>(b) * (a.K + 1) + d.kept;
  float x[kVerDraw], q[kVerDraw];
  load_ids<kVerDraw>(a.logits + row * a.V, a.V, base, a.vec4, -INFINITY, x);
  const long long draft = static_cast<long long>(b) * a.K + d.kept;
#pragma unroll
  for (int k = 0; k < kVerDraw; ++k) q[k] = 0.f;
  if (d.rejected && a.probs) load_ids<kVerDraw>(a.probs + draft * a.V, a.V, base, a.vec4, 0.f, q);
  const int certain = d.rejected && !a.probs ? a.drafts[draft] : -1;
  const double top = key_value(d.row.key);
#pragma unroll
  for (int k = 0; k < kVerDraw; ++k) {
    const int id = base + kVerDraw * static_cast<int>(threadIdx.x) + k;
    const double e = d.row.sure ? (static_cast<uint32_t>(id) == key_index(d.row.key) ? 1.0 : 0.0)
                                : weight(x[k], a.c, top);
    const float qk = q[k] == q[k] ? q[k] : 0.f;  // (a NaN in q takes nothing off)
    const double less = id == certain ? d.row.z : static_cast<double>(qk) * d.row.z;
    put(k, e, e > less ? e - less : 0.0);
  }
}

// A chunk's sums of the distribution to draw from, stored by thread 0.
__device__ __forceinline__ void chunk_sums(const VerifyArgs& a, int b, const Decision& d) {
  __shared__ double sums[2][kVerWaves];
  const int chunk = blockIdx.x - b * a.chunks;
  double se = 0, sr = 0;
  draw_weights(a, b, d, chunk * kVerDrawChunk, [&](int, double e, double rest) {
    se += e;
    sr += rest;
  });
  se = wave_sum_d(se);
  sr = wave_sum_d(sr);
  if ((threadIdx.x & 63) == 0) {
    sums[0][threadIdx.x >> 6] = se;
    sums[1][threadIdx.x >> 6] = sr;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.plain[blockIdx.x] = (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]);
    a.rest[blockIdx.x] = (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3]);
  }
}

__global__ __launch_bounds__(kVerThreads) void verify_sums_kernel(const VerifyArgs a) {
  const int b = blockIdx.x / a.chunks;
  chunk_sums(a, b, a.decided[b]);
}

// The draw: a workgroup a sequence, or (JOINED) one a chunk, which decides and sums by itself and
// draws if it is its sequence's last to come so far.  None waits for another; which one comes
// last has no effect on what it reads or adds up.
template <bool JOINED>
__global__ __launch_bounds__(kVerThreads) void verify_draw_kernel(const VerifyArgs a) {
  __shared__ double part[kVerWaves];
  __shared__ int first, last, closes;
  const int b = JOINED ? blockIdx.x / a.chunks : blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Decision d = JOINED ? decide<false>(a, b) : a.decided[b];
  if (JOINED) {
    chunk_sums(a, b, d);
    if (threadIdx.x == 0) {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
      const uint32_t before = __hip_atomic_fetch_add(a.done + b, 1u, __ATOMIC_RELAXED,
                                                     __HIP_MEMORY_SCOPE_AGENT);
      closes = before + 1u == static_cast<uint32_t>(a.chunks);
    }
    __syncthreads();
    if (!closes) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  }
  // The chunk in which the running sum passes the threshold, by every wave alike: sums of 64
  // chunks at a time, each lane's in the chunks' order behind those before them.
  const double* sums = a.rest + static_cast<long long>(b) * a.chunks;
  const auto upto = [&](int c0, double& mine) {  // inclusive, of the chunks from c0 to this lane's
    mine = c0 + lane < a.chunks ? sums[c0 + lane] : 0.;
    double s = mine;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const double x = __shfl_up(s, o, kWave);
      if (lane >= o) s += x;
    }
    return s;
  };
  const auto whole = [&]() {
    double all = 0, mine;
    for (int c0 = 0; c0 < a.chunks; c0 += kWave) all += __shfl(upto(c0, mine), kWave - 1, kWave);
    return all;
  };
  double total = whole();
  const bool spare = total > 0;  // else nothing is left beside the draft: from p itself
  if (!spare) {
    sums = a.plain + static_cast<long long>(b) * a.chunks;
    total = whole();
  }
  const double goal = static_cast<double>(a.u[static_cast<long long>(b) * (a.K + 1) + a.K]) * total;
  int chunk = 0;
  double before = 0, run = 0;
  for (int c0 = 0; c0 < a.chunks; c0 += kWave) {
    double mine;
    const double s = upto(c0, mine);
    const uint64_t any = __ballot(mine > 0), past = __ballot(mine > 0 && run + s > goal);
    // the first chunk past the threshold; none (yet): the last that has any weight
    const int l = past ? __ffsll(static_cast<unsigned long long>(past)) - 1
                       : 63 - __clzll(static_cast<long long>(any));
    if (past | any) {
      chunk = c0 + l;
      before = run + __shfl(s, l, kWave) - __shfl(mine, l, kWave);
    }
    if (past) break;
    run += __shfl(s, kWave - 1, kWave);
  }
  if (threadIdx.x == 0) first = a.V, last = -1;
  double rest[kVerDraw];
  const int base = chunk * kVerDrawChunk;
  draw_weights(a, b, d, base, [&](int k, double e, double r) { rest[k] = spare ? r : e; });
  // running sums in the ids' order
  double sum = (rest[0] + rest[1]) + (rest[2] + rest[3]);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const double x = __shfl_up(sum, o, kWave);
    if (lane >= o) sum += x;
  }
  if (lane == kWave - 1) part[wave] = sum;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVerWaves; ++w)
    if (w < wave) before += part[w];
  const double prev = __shfl_up(sum, 1, kWave);
  if (lane) before += prev;
  int at_first = a.V, at_last = -1;
#pragma unroll
  for (int j = 0; j < kVerDraw; ++j) {
    before += rest[j];
    const int id = base + kVerDraw * static_cast<int>(threadIdx.x) + j;
    if (rest[j] > 0) {
      if (before > goal) at_first = min(at_first, id);
      at_last = max(at_last, id);
    }
  }
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    at_first = min(at_first, __shfl_xor(at_first, o, kWave));
    at_last = max(at_last, __shfl_xor(at_last, o, kWave));
  }
  if (lane == 0) {
    atomicMin(&first, at_first);
    atomicMax(&last, at_last);
  }
  __syncthreads();
  // u at 1, or sums that rounded below the threshold: the last id with any weight
  put_tokens(a, b, d, first < a.V ? first : last);
}

inline int verify_chunks(int V, int chunk) { return (V + chunk - 1) / chunk; }

// Whether decisions, sums and draw are one launch: each workgroup then hands its sums to the other
// dies' caches, which takes longer the more of them do.  us of a call joined / in three launches,
// 4 drafts: 1 x 32000 ids 13.2 / 17.8 (in a graph 13.0 / 14.5), 4 x 32000, 128 workgroups, 14.0 /
// 18.8 (14.1 / 14.9), 8 x 32000 18.4 / 18.8 (18.7 / 15.7), 31 x 32000 34 / 21, 1 x 128256 14.7 / 18.3.
inline bool verify_joined(int B, int chunks) {
  return 2ll * B * chunks <= compute_units();
}

// Chunks of a row that one workgroup of the first kernel takes: as many as leave five a CU, which
// are resident together (64 x 5 rows of 32 chunks: one each 46 us, eight each 39).
inline int verify_per_part(int64_t rows, int chunks) {
  const int64_t n = rows * chunks / (5ll * compute_units());
  return static_cast<int>(n < 1 ? 1 : n > chunks ? chunks : n);
}

}  // namespace llmy

using namespace llmy;

extern "C" int64_t llmy_verify_drafts_workspace_bytes(int32_t B, int32_t K, int32_t V) {
  if (B < 0 || K < 1 || K > kMaxDrafts || V < 1 || V > (1 << 30)) return -1;
  const int64_t rows = static_cast<int64_t>(B) * (K + 1);
  const int64_t parts = rows * verify_chunks(V, kVerChunk);
  const int64_t draws = static_cast<int64_t>(B) * verify_chunks(V, kVerDrawChunk);
  if (parts >= (1ll << 31) || draws >= (1ll << 31)) return -1;  // the grids
  return 16 * (parts + draws) + static_cast<int64_t>(sizeof(Decision)) * B;
}

extern "C" int32_t llmy_verify_drafts_f32(const float* logits, const int32_t* draft_tokens,
                                          const float* draft_probs, const int32_t* counts,
                                          const float* u, double temperature, int32_t* tokens,
                                          int32_t* accepted, void* workspace,
                                          int64_t workspace_bytes, int32_t B, int32_t K, int32_t V,
                                          void* stream) {
  const int64_t ws = llmy_verify_drafts_workspace_bytes(B, K, V);
  LLMY_REQUIRE(ws >= 0 && temperature == temperature && temperature < __builtin_inf());
  if (B == 0) return 0;
  const bool greedy = temperature <= 0.;
  LLMY_REQUIRE(logits && draft_tokens && tokens && accepted && (greedy || u));
  LLMY_REQUIRE(workspace && aligned(workspace, 8) && workspace_bytes >= ws);
  const int64_t rows = static_cast<int64_t>(B) * (K + 1), drafts = rows - B;
  const struct { const void* p; int64_t n; } all[] = {
      {tokens, 4 * rows}, {accepted, 4ll * B}, {workspace, ws}, {logits, 4 * rows * V},
      {draft_tokens, 4 * drafts}, {draft_probs, draft_probs ? 4 * drafts * V : 0},
      {counts, counts ? 4ll * B : 0}, {u, u ? 4 * rows : 0}};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 8; ++j)
      LLMY_REQUIRE(bytes_apart(all[i].p, all[i].n, all[j].p, all[j].n));
  VerifyArgs a{};
  a.logits = logits; a.drafts = draft_tokens; a.probs = draft_probs; a.counts = counts; a.u = u;
  a.tokens = tokens; a.accepted = accepted;
  a.B = B; a.K = K; a.V = V;
  a.row_chunks = verify_chunks(V, kVerChunk);
  a.chunks = verify_chunks(V, kVerDrawChunk);
  // (2^800 already takes the least difference of two logits, 2^-149, past every weight)
  a.c = greedy ? 0. : fmin(1.4426950408889634 / temperature, 0x1p800);
  a.vec4 = V % 4 == 0 && aligned(logits, 16) && (!draft_probs || aligned(draft_probs, 16));
  a.per_part = verify_per_part(rows, a.row_chunks);
  a.parts = (a.row_chunks + a.per_part - 1) / a.per_part;
  a.best = static_cast<uint64_t*>(workspace);
  a.sum = reinterpret_cast<double*>(a.best + rows * a.parts);
  a.rest = a.sum + rows * a.parts;
  a.plain = a.rest + static_cast<int64_t>(B) * a.chunks;
  a.decided = reinterpret_cast<Decision*>(a.plain + static_cast<int64_t>(B) * a.chunks);
  a.done = reinterpret_cast<uint32_t*>(a.decided);  // (of a joined draw, which stores no decisions)
  const hipStream_t s = as_stream(stream);
  const dim3 grid(static_cast<unsigned>(rows * a.parts)), draws(static_cast<unsigned>(B) * a.chunks);
  if (greedy) {
    hipLaunchKernelGGL(verify_rows_kernel<true>, grid, dim3(kVerThreads), 0, s, a);
    hipLaunchKernelGGL(verify_decide_kernel<true>, dim3(B), dim3(kVerThreads), 0, s, a);
    return launch_status();
  }
  hipLaunchKernelGGL(verify_rows_kernel<false>, grid, dim3(kVerThreads), 0, s, a);
  if (verify_joined(B, a.chunks)) {
    hipLaunchKernelGGL(verify_draw_kernel<true>, draws, dim3(kVerThreads), 0, s, a);
    return launch_status();
  }
  hipLaunchKernelGGL(verify_decide_kernel<false>, dim3(B), dim3(kVerThreads), 0, s, a);
  hipLaunchKernelGGL(verify_sums_kernel, draws, dim3(kVerThreads), 0, s, a);
  hipLaunchKernelGGL(verify_draw_kernel<false>, dim3(B), dim3(kVerThreads), 0, s, a);
  return launch_status();
}
