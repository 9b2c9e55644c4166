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
// chip adds and multiplies at the rate of single 32-bit ones: 2^x of a reduced argument by
// its Taylor sum.
//
// Bound by the read of the logits (then of one draft row a sequence).  Rows are cut into
// chunks of 4096 ids, a workgroup each, so that one sequence's rows fill the chip too:
//   1. each chunk's maximum and sum of exponentials under it;
//   2. per (sequence, chunk): from those, which drafts are kept (few numbers, repeated by
//      each chunk's workgroup), and the chunk's sum of the distribution to draw from;
//   3. per sequence: the chunk in which the sum passes the threshold, and the id in it.
// Greedy (T = 0): each row's first largest id, then the comparison: two launches.
#include "common.hpp"
#include "abi_util.hpp"
#include "paged.hpp"

namespace llmy {

constexpr int kVerThreads = 256, kVerPer = 16;
constexpr int kVerChunk = kVerThreads * kVerPer;
constexpr int kVerWaves = kVerThreads / kWave;
constexpr int kMaxDrafts = 63;  // a wave looks at all rows of a sequence at once

struct VerifyArgs {
  const float* logits;          // [B, K + 1, V]
  const int32_t* drafts;        // [B, K]
  const float* probs;           // [B, K, V] or null: the drafts were certain
  const int32_t* counts;        // [B] or null: K
  const float* u;               // [B, K + 1]
  int32_t *tokens, *accepted;   // [B, K + 1], [B]
  uint64_t* best;               // [B (K + 1), chunks]: largest (value, lowest id) of a chunk
  double* sum;                  // [B (K + 1), chunks]: its sum under that maximum
  double *rest, *plain;         // [B, chunks]: of max(e - q Z, 0) and e of the drawn row
  double inv_t;
  int B, K, V, chunks;
  bool vec4;
};

// e^x for x <= 0: 2^n sum_k r^k / k!, x = n ln 2 + r, |r| <= ln 2 / 2; the remainder
// after k = 12 is under 2^-52 of it.  0 below -745, also for -inf.
__device__ __forceinline__ double exp_neg(double x) {
  x = fmax(x, -746.0);
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, -0.6931471805599453, x);  // ln 2 rounded to 64 bits, and what that left
  r = fma(n, -2.3190468138462996e-17, r);
  double s = 1.0 / 479001600.0;
  s = fma(s, r, 1.0 / 39916800.0);
  s = fma(s, r, 1.0 / 3628800.0);
  s = fma(s, r, 1.0 / 362880.0);
  s = fma(s, r, 1.0 / 40320.0);
  s = fma(s, r, 1.0 / 5040.0);
  s = fma(s, r, 1.0 / 720.0);
  s = fma(s, r, 1.0 / 120.0);
  s = fma(s, r, 1.0 / 24.0);
  s = fma(s, r, 1.0 / 6.0);
  s = fma(s, r, 0.5);
  s = fma(s, r, 1.0);
  s = fma(s, r, 1.0);
  return ldexp(s, static_cast<int>(n));
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

// This thread's 16 ids of a chunk of a row: the four from base + 1024 i + 4 t on, i < 4;
// `none` past the row.
__device__ __forceinline__ void load_ids(const float* row, int V, int base, bool vec4, float none,
                                         float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = base + 1024 * i + 4 * static_cast<int>(threadIdx.x);
    if (vec4) {
      float4 w = make_float4(none, none, none, none);
      if (at < V) w = *reinterpret_cast<const float4*>(row + at);  // V % 4 == 0
      v[4 * i] = w.x; v[4 * i + 1] = w.y; v[4 * i + 2] = w.z; v[4 * i + 3] = w.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = at + j < V ? row[at + j] : none;
    }
  }
}

template <bool GREEDY>
__global__ __launch_bounds__(kVerThreads) void verify_rows_kernel(const VerifyArgs a) {
  __shared__ uint64_t keys[kVerWaves];
  __shared__ double sums[kVerWaves];
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const int base = chunk * kVerChunk;
  float v[kVerPer];
  load_ids(a.logits + static_cast<long long>(row) * a.V, a.V, base, a.vec4, -INFINITY, v);
  uint64_t key = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int id = base + 1024 * i + 4 * static_cast<int>(threadIdx.x) + j;
      if (id < a.V) key = umax64(key, value_index_key(v[4 * i + j], id));
    }
  key = wave_max_u64(key);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) keys[wave] = key;
  __syncthreads();
  key = umax64(umax64(keys[0], keys[1]), umax64(keys[2], keys[3]));
  const float top = key_value(key);
  double s = 0;
  if (!GREEDY && fabsf(top) < INFINITY) {
#pragma unroll
    for (int k = 0; k < kVerPer; ++k)
      s += exp_neg((static_cast<double>(v[k]) - static_cast<double>(top)) * a.inv_t);
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) sums[wave] = s;
    __syncthreads();
    s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
  if (threadIdx.x == 0) {
    a.best[blockIdx.x] = key;
    if (!GREEDY) a.sum[blockIdx.x] = s;
  }
}

struct Row {
  uint64_t key;   // its largest value and that one's lowest id
  double z;       // sum of e^((x - largest) / T); rows without a finite largest: 1
  bool sure;      // no finite largest: the id of the key alone
};

// A row from its chunks, by one wave.
__device__ __forceinline__ Row whole_row(const VerifyArgs& a, long long row, bool greedy) {
  const int lane = threadIdx.x & 63;
  Row r;
  r.key = 0;
  for (int c = lane; c < a.chunks; c += kWave) r.key = umax64(r.key, a.best[row * a.chunks + c]);
  r.key = wave_max_u64(r.key);
  const float top = key_value(r.key);
  r.sure = greedy || !(fabsf(top) < INFINITY);
  r.z = 1.0;
  if (!r.sure) {
    double z = 0;
    for (int c = lane; c < a.chunks; c += kWave) {
      const float m = key_value(a.best[row * a.chunks + c]);
      z += a.sum[row * a.chunks + c] *
           exp_neg((static_cast<double>(m) - static_cast<double>(top)) * a.inv_t);
    }
    r.z = wave_sum_d(z);
  }
  return r;
}

struct Decision {
  Row row;        // the row that the new token comes from
  int kept;       // drafts kept before it
  bool rejected;  // a draft was put away there
};

// Which drafts of sequence b are kept: every row by a wave, their verdicts through LDS.
template <bool GREEDY>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, int b, Row* rows, int* keep) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int count = a.counts ? min(max(a.counts[b], 0), a.K) : a.K;
  for (int t = wave; t <= count; t += kVerWaves) {
    const long long row = static_cast<long long>(b) * (a.K + 1) + t;
    const Row r = whole_row(a, row, GREEDY);
    if (lane == 0) {
      rows[t] = r;
      bool ok = false;
      if (t < count) {
        const int id = a.drafts[static_cast<long long>(b) * a.K + t];
        if (id >= 0 && id < a.V) {
          if (GREEDY) {
            ok = static_cast<uint32_t>(id) == key_index(r.key);
          } else {
            const float x = a.logits[row * a.V + id];
            const double e = r.sure ? (static_cast<uint32_t>(id) == key_index(r.key) ? 1.0 : 0.0)
                                    : exp_neg((static_cast<double>(x) -
                                               static_cast<double>(key_value(r.key))) * a.inv_t);
            const double q =
                a.probs ? a.probs[(static_cast<long long>(b) * a.K + t) * a.V + id] : 1.0;
            ok = static_cast<double>(a.u[row]) * q * r.z < e;
          }
        }
      }
      keep[t] = ok;
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

// Weights of the drawn row at this thread's 16 ids of a chunk: e and max(e - q Z, 0).
__device__ __forceinline__ void draw_weights(const VerifyArgs& a, int b, const Decision& d, int base,
                                             double* e, double* rest) {
  const long long row = static_cast<long long>(b) * (a.K + 1) + d.kept;
  float x[kVerPer], q[kVerPer];
  load_ids(a.logits + row * a.V, a.V, base, a.vec4, -INFINITY, x);
  const long long draft = static_cast<long long>(b) * a.K + d.kept;
#pragma unroll
  for (int k = 0; k < kVerPer; ++k) q[k] = 0.f;
  if (d.rejected && a.probs) load_ids(a.probs + draft * a.V, a.V, base, a.vec4, 0.f, q);
  const int certain = d.rejected && !a.probs ? a.drafts[draft] : -1;
  const double top = key_value(d.row.key);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = 4 * i + j, id = base + 1024 * i + 4 * static_cast<int>(threadIdx.x) + j;
      e[k] = d.row.sure ? (static_cast<uint32_t>(id) == key_index(d.row.key) ? 1.0 : 0.0)
                        : exp_neg((static_cast<double>(x[k]) - top) * a.inv_t);
      const double less = id == certain ? d.row.z : static_cast<double>(q[k]) * d.row.z;
      rest[k] = e[k] > less ? e[k] - less : 0.0;  // (a NaN in q: 0)
    }
}

__device__ __forceinline__ void put_tokens(const VerifyArgs& a, int b, int kept, int fresh) {
  for (int t = threadIdx.x; t <= a.K; t += kVerThreads) {
    const int id = t < kept ? a.drafts[static_cast<long long>(b) * a.K + t] : t == kept ? fresh : -1;
    a.tokens[static_cast<long long>(b) * (a.K + 1) + t] = id;
  }
  if (threadIdx.x == 0) a.accepted[b] = kept;
}

__global__ __launch_bounds__(kVerThreads) void verify_greedy_kernel(const VerifyArgs a) {
  __shared__ Row rows[kMaxDrafts + 1];
  __shared__ int keep[kMaxDrafts + 1];
  const Decision d = decide<true>(a, blockIdx.x, rows, keep);
  put_tokens(a, blockIdx.x, d.kept, static_cast<int>(key_index(d.row.key)));
}

__global__ __launch_bounds__(kVerThreads) void verify_sums_kernel(const VerifyArgs a) {
  __shared__ Row rows[kMaxDrafts + 1];
  __shared__ int keep[kMaxDrafts + 1];
  __shared__ double sums[2][kVerWaves];
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  const Decision d = decide<false>(a, b, rows, keep);
  double e[kVerPer], rest[kVerPer];
  draw_weights(a, b, d, chunk * kVerChunk, e, rest);
  double se = 0, sr = 0;
#pragma unroll
  for (int k = 0; k < kVerPer; ++k) {
    se += e[k];
    sr += rest[k];
  }
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

__global__ __launch_bounds__(kVerThreads) void verify_draw_kernel(const VerifyArgs a) {
  __shared__ Row rows[kMaxDrafts + 1];
  __shared__ int keep[kMaxDrafts + 1];
  __shared__ double part[4][kVerWaves];
  __shared__ int first, last;
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Decision d = decide<false>(a, b, rows, keep);
  // the whole, the chunk that passes the threshold, and the sum before it, by every wave alike
  const double* sums = a.rest + static_cast<long long>(b) * a.chunks;
  double all = 0;
  for (int c = lane; c < a.chunks; c += kWave) all += sums[c];
  all = wave_sum_d(all);
  const bool spare = all > 0;  // else nothing is left beside the draft: from p itself
  if (!spare) sums = a.plain + static_cast<long long>(b) * a.chunks;
  // sums in the chunks' order: the total is the last running sum, as a threshold needs
  double total = 0;
  for (int c = 0; c < a.chunks; ++c) total += sums[c];
  const double goal = static_cast<double>(a.u[static_cast<long long>(b) * (a.K + 1) + a.K]) * total;
  int chunk = 0;
  double before = 0, run = 0;
  bool passed = false;
  for (int c = 0; c < a.chunks; ++c) {
    const double s = sums[c];
    if (s > 0 && !passed) {
      chunk = c;
      before = run;
      passed = run + s > goal;
    }
    run += s;
  }
  if (threadIdx.x == 0) first = a.V, last = -1;
  double e[kVerPer], rest[kVerPer];
  const int base = chunk * kVerChunk;
  draw_weights(a, b, d, base, e, rest);
#pragma unroll
  for (int k = 0; k < kVerPer; ++k)
    if (!spare) rest[k] = e[k];
  // running sums in the ids' order: four blocks of 1024 ids, 4 a thread
  double upto[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    double s = (rest[4 * i] + rest[4 * i + 1]) + (rest[4 * i + 2] + rest[4 * i + 3]);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const double x = __shfl_up(s, o, kWave);
      if (lane >= o) s += x;
    }
    upto[i] = s;
    if (lane == kWave - 1) part[i][wave] = s;
  }
  __syncthreads();
  double start = before;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    double c = start;
#pragma unroll
    for (int w = 0; w < kVerWaves; ++w) {
      if (w < wave) c += part[i][w];
      start += part[i][w];
    }
    const double prev = __shfl_up(upto[i], 1, kWave);
    if (lane) c += prev;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double w = rest[4 * i + j];
      c += w;
      const int id = base + 1024 * i + 4 * static_cast<int>(threadIdx.x) + j;
      if (w > 0) {
        if (c > goal) atomicMin(&first, id);
        atomicMax(&last, id);
      }
    }
  }
  __syncthreads();
  // u at 1, or sums that rounded below the threshold: the last id with any weight
  put_tokens(a, b, d.kept, first < a.V ? first : last);
}

inline int verify_chunks(int V) { return (V + kVerChunk - 1) / kVerChunk; }

}  // namespace llmy

using namespace llmy;

extern "C" int64_t llmy_verify_drafts_workspace_bytes(int32_t B, int32_t K, int32_t V) {
  if (B < 0 || K < 1 || K > kMaxDrafts || V < 1 || V > (1 << 30)) return -1;
  const int64_t chunks = verify_chunks(V), rows = static_cast<int64_t>(B) * (K + 1);
  if (rows * chunks >= (1ll << 31)) return -1;  // the grid
  return 16 * chunks * (rows + B);
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
  a.B = B; a.K = K; a.V = V; a.chunks = verify_chunks(V);
  a.inv_t = greedy ? 0. : fmin(1. / temperature, 0x1p1023);
  a.vec4 = V % 4 == 0 && aligned(logits, 16) && (!draft_probs || aligned(draft_probs, 16));
  const int64_t parts = rows * a.chunks;
  a.best = static_cast<uint64_t*>(workspace);
  a.sum = reinterpret_cast<double*>(a.best + parts);
  a.rest = a.sum + parts;
  a.plain = a.rest + static_cast<int64_t>(B) * a.chunks;
  const hipStream_t s = as_stream(stream);
  const dim3 grid(static_cast<unsigned>(parts)), draws(static_cast<unsigned>(B) * a.chunks);
  if (greedy) {
    hipLaunchKernelGGL(verify_rows_kernel<true>, grid, dim3(kVerThreads), 0, s, a);
    hipLaunchKernelGGL(verify_greedy_kernel, dim3(B), dim3(kVerThreads), 0, s, a);
    return launch_status();
  }
  hipLaunchKernelGGL(verify_rows_kernel<false>, grid, dim3(kVerThreads), 0, s, a);
  hipLaunchKernelGGL(verify_sums_kernel, draws, dim3(kVerThreads), 0, s, a);
  hipLaunchKernelGGL(verify_draw_kernel, dim3(B), dim3(kVerThreads), 0, s, a);
  return launch_status();
}
