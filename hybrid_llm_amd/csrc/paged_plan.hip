// Pages and slots for a batch's new tokens, from its lengths, on the GPU: which pages go
// back to the free stack, which are handed out, and where each packed token lies.
//
// Sums over the sequences in their order decide everything (b a sequence, P a page's tokens):
//   back_b = held_b where reset_b, else 0        pushed on the stack in order of b
//   need_b = max(0, ceil((len_b + new_b) / P) - held_b) where new_b > 0 and the tokens fit
//   given_b: need_b = 0 or sum_{a <= b} need_a <= free pages, len_b + new_b <= width P and
//            sum_{a <= b} new_a <= capacity
// so every result is a whole number that does not depend on timing.  A sequence's i-th new
// page is entry top - 1 - (sum_{a < b} need_a + i) of the stack: those that are given pages
// come before those that are not, so the popped entries have no holes.
//
// Bound by latency, not by its bytes (12 a token and page): few launches.  A call of up to
// 4096 tokens is one workgroup and one launch; a larger one spreads its tokens over many
// workgroups that each repeat the scan of the sequences (up to 4 a thread, in registers)
// and stores what the second launch needs to hand the pages out, since a page may be pushed
// and popped in one call.  Measured: 64 sequences of a token each 4.3 us; 127 prompts of
// 262139 tokens 9.6 + 4.0.
#include "common.hpp"
#include "abi_util.hpp"
#include "paged.hpp"

namespace llmy {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / kWave;
constexpr int kPlanPer = 4;                           // sequences a thread
constexpr int kPlanMost = kPlanThreads * kPlanPer;
constexpr int kPlanTokens = 4 * kPlanThreads;         // of a workgroup

struct PlanArgs {
  const int32_t *lengths, *fresh, *reset;
  int32_t *table, *held, *stack, *n_free;
  int32_t *cu, *rows, *pos, *out_len;
  int32_t* ws;                    // [2 + 3 B]: top, popped; held after resets, pages got, first
  int B, width, page, shift, F, N;
  bool vec4;                      // rows and positions by 16 bytes
};

// Sums stop at 2^32 - 1, past every bound that they are held against (all below 2^31), which
// leaves the order of additions without effect.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  return __builtin_elementwise_add_sat(a, b);
}

// Inclusive sums over the wave: the previous 1, 2, 4 and 8 lanes of each row of 16, then the last
// lane of the row and of the half before.
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
#define LLMY_STEP(ctrl, rows) \
  v = add_sat(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl, rows, 0xf, false)))
  LLMY_STEP(0x111, 0xf);  // row_shr:1
  LLMY_STEP(0x112, 0xf);
  LLMY_STEP(0x114, 0xf);
  LLMY_STEP(0x118, 0xf);
  LLMY_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
  LLMY_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef LLMY_STEP
  return v;
}

// Sums over the block of the threads before this one, and of all; scratch: a word a wave.
__device__ __forceinline__ uint32_t plan_scan(uint32_t v, uint32_t* scratch, int waves, uint32_t* total) {
  const int wave = threadIdx.x / kWave;
  const uint32_t upto = wave_upto(v);
  // exclusive within the wave: the lane before's, 0 at the first (a saturated sum has no difference)
  uint32_t before = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(upto), 0x138, 0xf, 0xf, false));
  uint32_t all = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), kWave - 1));
  if (waves > 1) {
    if ((threadIdx.x & (kWave - 1)) == 0) scratch[wave] = all;
    __syncthreads();
    all = 0;
    for (int w = 0; w < waves; ++w) {
      const uint32_t x = scratch[w];
      if (w < wave) before = add_sat(before, x);
      all = add_sat(all, x);
    }
  }
  *total = all;
  return before;
}

// The last of n ascending entries that is at most x (the first is).
__device__ __forceinline__ int plan_find(const int32_t* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// One wave hands a sequence its pages: entries at, at - 1, ... of the stack into its row's
// entries from held on.
__device__ __forceinline__ void plan_pop(const PlanArgs& a, int b, int held, int got, int at,
                                         int lane) {
  for (int i = lane; i < got; i += kWave)
    a.table[static_cast<long long>(b) * a.width + held + i] = a.stack[at - i];
}

// One workgroup of many, or (ONE) the whole call; PER sequences a thread.
template <bool ONE, int PER>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const PlanArgs a) {
  extern __shared__ int32_t lds[];      // cu [B + 1], pushed before [B + 1], position - row [B]
  __shared__ uint32_t scratch[3][kPlanWaves];
  __shared__ int popped;
  int32_t *const s_cu = lds, *const s_back = lds + a.B + 1, *const s_base = s_back + a.B + 1;
  const int b0 = threadIdx.x * PER, b1 = min(a.B, b0 + PER);
  const int t = threadIdx.x, lane = t & (kWave - 1), threads = blockDim.x, waves = threads / kWave;
  const bool tells = ONE || blockIdx.x == 0;

  int len[PER], fresh[PER], held[PER], back[PER];
  uint32_t sum_new = 0, sum_back = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = b0 + k;
    len[k] = fresh[k] = held[k] = back[k] = 0;
    if (b < b1) {
      const int n = a.lengths[b], f = a.fresh[b], h = a.held[b];
      const bool over = a.reset && a.reset[b] != 0;
      len[k] = over ? 0 : max(n, 0);
      fresh[k] = max(f, 0);
      held[k] = min(max(h, 0), a.width);
      if (over) {
        back[k] = held[k];
        held[k] = 0;
      }
      sum_new = add_sat(sum_new, fresh[k]);
      sum_back = add_sat(sum_back, back[k]);
    }
  }
  const int n0 = min(max(*a.n_free, 0), a.F);
  if (t == 0) popped = 0;
  uint32_t all_new, all_back, all_need;
  uint32_t at_new = plan_scan(sum_new, scratch[0], waves, &all_new);
  uint32_t at_back = plan_scan(sum_back, scratch[1], waves, &all_back);
  const uint32_t top = min(static_cast<uint32_t>(a.F), add_sat(n0, all_back));
  const long long cap = static_cast<long long>(a.width) << a.shift;

  int need[PER];
  bool fits[PER];
  uint32_t sum_need = 0, end = at_new;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    need[k] = 0;
    fits[k] = false;
    if (b0 + k < b1) {
      end = add_sat(end, fresh[k]);
      const long long total = static_cast<long long>(len[k]) + fresh[k];
      fits[k] = total <= cap && end <= static_cast<uint32_t>(a.N);
      if (fits[k] && fresh[k] > 0)
        need[k] = max(0, static_cast<int>((total + a.page - 1) >> a.shift) - held[k]);
      sum_need = add_sat(sum_need, need[k]);
    }
  }
  uint32_t upto = plan_scan(sum_need, scratch[2], waves, &all_need);
  int got[PER], first[PER], most = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    got[k] = first[k] = 0;
    const int b = b0 + k;
    if (b < b1) {
      first[k] = static_cast<int>(top - 1 - min(upto, top));
      upto = add_sat(upto, need[k]);
      const bool given = fits[k] && (need[k] == 0 || upto <= top);
      got[k] = given ? need[k] : 0;
      if (got[k] > 0) most = static_cast<int>(upto);  // those that are given pages come first
      const int from = static_cast<int>(min(at_new, static_cast<uint32_t>(a.N)));
      s_cu[b] = from;
      s_back[b] = static_cast<int>(min(at_back, 0x7fffffffu));
      s_base[b] = given ? len[k] - from : INT32_MIN;  // (given: from is exact, at most N)
      at_new = add_sat(at_new, fresh[k]);
      at_back = add_sat(at_back, back[k]);
      if (tells) {
        a.cu[b] = from;
        a.out_len[b] = len[k] + (given ? fresh[k] : 0);
        if (!ONE) {
          a.ws[2 + b] = held[k];
          a.ws[2 + a.B + b] = got[k];
          a.ws[2 + 2 * a.B + b] = first[k];
        }
      }
    }
  }
  if (most > 0) atomicMax(&popped, most);  // (the barriers of the scans lie behind its 0)
  if (t == 0) {
    s_cu[a.B] = static_cast<int>(min(all_new, static_cast<uint32_t>(a.N)));
    s_back[a.B] = static_cast<int>(top) - n0;               // what the stack takes
    if (tells) a.cu[a.B] = s_cu[a.B];
  }
  __syncthreads();

  // finished sequences' pages onto the stack
  const int pushed = s_back[a.B], step = ONE ? threads : gridDim.x * threads;
  for (int i = (ONE ? 0 : blockIdx.x * threads) + t; i < pushed; i += step) {
    const int b = plan_find(s_back, a.B, i);
    a.stack[n0 + i] = a.table[static_cast<long long>(b) * a.width + i - s_back[b]];
  }
  // the tokens' rows and positions
  const int end_all = s_cu[a.B];
  const long long j0 = ONE ? 0 : blockIdx.x * static_cast<long long>(kPlanTokens);
  const int j1 = static_cast<int>(min(static_cast<long long>(a.N), j0 + kPlanTokens));
  // (a few: one a thread, whose searches overlap; many: four together, of one row mostly)
  constexpr int TPT = ONE ? 1 : 4;
  for (long long j = j0 + TPT * t; j < j1; j += TPT * threads) {
    int row[TPT], p[TPT], at = 0;
#pragma unroll
    for (int i = 0; i < TPT; ++i) {
      row[i] = p[i] = -1;
      const int x = static_cast<int>(j) + i;
      if (x < end_all) {
        if (i == 0 || s_cu[at + 1] <= x) at = plan_find(s_cu, a.B, x);
        row[i] = at;
        if (s_base[at] != INT32_MIN) p[i] = s_base[at] + x;
      }
    }
    if (!ONE && a.vec4) {  // (N % 4 == 0)
      *reinterpret_cast<int4*>(a.rows + j) = make_int4(row[0], row[1 % TPT], row[2 % TPT], row[3 % TPT]);
      *reinterpret_cast<int4*>(a.pos + j) = make_int4(p[0], p[1 % TPT], p[2 % TPT], p[3 % TPT]);
    } else {
#pragma unroll
      for (int i = 0; i < TPT; ++i)
        if (j + i < j1) {
          a.rows[j + i] = row[i];
          a.pos[j + i] = p[i];
        }
    }
  }
  if (!ONE) {
    if (blockIdx.x == 0 && t == 0) {
      a.ws[0] = static_cast<int>(top);
      a.ws[1] = popped;
    }
    return;
  }
  __syncthreads();  // behind this workgroup's pushes, and its reads of the table
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (b0 + k < b1) a.held[b0 + k] = held[k] + got[k];
    // a wave's sequences one after the other, each by all of its lanes
    uint64_t todo = __ballot(b0 + k < b1 && got[k] > 0);
    while (todo) {
      const int l = __ffsll(static_cast<unsigned long long>(todo)) - 1;
      todo &= todo - 1;
      plan_pop(a, __builtin_amdgcn_readlane(b0 + k, l), __builtin_amdgcn_readlane(held[k], l),
               __builtin_amdgcn_readlane(got[k], l), __builtin_amdgcn_readlane(first[k], l), lane);
    }
  }
  if (t == 0) *a.n_free = static_cast<int>(top) - popped;
}

// The second launch: a wave a sequence.
__global__ __launch_bounds__(256) void plan_pop_kernel(const PlanArgs a) {
  const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.n_free = a.ws[0] - a.ws[1];
  if (b >= a.B) return;
  const int held = a.ws[2 + b], got = a.ws[2 + a.B + b];
  plan_pop(a, b, held, got, a.ws[2 + 2 * a.B + b], threadIdx.x & (kWave - 1));
  if ((threadIdx.x & 63) == 0) a.held[b] = held + got;
}

}  // namespace llmy

using namespace llmy;

extern "C" int64_t llmy_paged_plan_workspace_bytes(int32_t B, int32_t capacity) {
  if (B < 0 || B > kPlanMost || capacity < 0) return -1;
  return capacity <= kPlanTokens ? 0 : 4ll * (2 + 3ll * B);
}

extern "C" int32_t llmy_paged_plan(const int32_t* lengths, const int32_t* new_tokens,
                                   const int32_t* reset, int32_t* page_table, int32_t* held,
                                   int32_t* free_pages, int32_t* n_free, int32_t* cu_seqlens,
                                   int32_t* rows, int32_t* positions, int32_t* lengths_out,
                                   void* workspace, int64_t workspace_bytes, int32_t B,
                                   int32_t width, int32_t page, int32_t free_capacity,
                                   int32_t capacity, void* stream) {
  const int64_t ws = llmy_paged_plan_workspace_bytes(B, capacity);
  LLMY_REQUIRE(ws >= 0 && width >= 0 && free_capacity >= 0 && page_shift(page) > 0);
  LLMY_REQUIRE((static_cast<int64_t>(width) << page_shift(page)) < (1ll << 31));
  LLMY_REQUIRE(n_free && cu_seqlens && (capacity == 0 || (rows && positions)) &&
               (free_capacity == 0 || free_pages));
  LLMY_REQUIRE(B == 0 || (lengths && new_tokens && held && lengths_out));
  LLMY_REQUIRE(B == 0 || width == 0 || page_table);
  LLMY_REQUIRE(ws == 0 || (workspace && aligned(workspace, 4) && workspace_bytes >= ws));
  // what the call writes lies apart from all else
  const struct { const void* p; int64_t n; } all[] = {
      {page_table, 4ll * B * width}, {held, 4ll * B}, {free_pages, 4ll * free_capacity},
      {n_free, 4}, {cu_seqlens, 4ll * (B + 1ll)}, {rows, 4ll * capacity},
      {positions, 4ll * capacity}, {lengths_out, 4ll * B}, {workspace, ws},
      {lengths, 4ll * B}, {new_tokens, 4ll * B}, {reset, reset ? 4ll * B : 0}};
  for (int i = 0; i < 9; ++i)
    for (int j = i + 1; j < 12; ++j)
      LLMY_REQUIRE(bytes_apart(all[i].p, all[i].n, all[j].p, all[j].n));
  PlanArgs a{};
  a.lengths = lengths; a.fresh = new_tokens; a.reset = reset;
  a.table = page_table; a.held = held; a.stack = free_pages; a.n_free = n_free;
  a.cu = cu_seqlens; a.rows = rows; a.pos = positions; a.out_len = lengths_out;
  a.ws = static_cast<int32_t*>(workspace);
  a.B = B; a.width = width; a.page = page; a.shift = page_shift(page);
  a.F = free_capacity; a.N = capacity;
  a.vec4 = capacity % 4 == 0 && aligned(rows, 16) && aligned(positions, 16);
  const hipStream_t s = as_stream(stream);
  const unsigned lds = 4u * (3u * B + 2u);
  // threads: a sequence each and a few tokens; waves that have neither only lengthen the barriers
  const int threads = ws ? kPlanThreads
                         : 64 * ((B > capacity / 4 ? B : capacity / 4) / 64 + 1 < kPlanWaves
                                     ? (B > capacity / 4 ? B : capacity / 4) / 64 + 1
                                     : kPlanWaves);
  if (ws == 0) {
    if (B <= threads)
      hipLaunchKernelGGL((plan_kernel<true, 1>), dim3(1), dim3(threads), lds, s, a);
    else
      hipLaunchKernelGGL((plan_kernel<true, kPlanPer>), dim3(1), dim3(kPlanThreads), lds, s, a);
    return launch_status();
  }
  const unsigned groups = static_cast<unsigned>((capacity + kPlanTokens - 1ll) / kPlanTokens);
  if (B <= kPlanThreads)
    hipLaunchKernelGGL((plan_kernel<false, 1>), dim3(groups), dim3(kPlanThreads), lds, s, a);
  else
    hipLaunchKernelGGL((plan_kernel<false, kPlanPer>), dim3(groups), dim3(kPlanThreads), lds, s, a);
  hipLaunchKernelGGL(plan_pop_kernel, dim3(static_cast<unsigned>(B / 4 + 1)), dim3(256), 0, s, a);
  return launch_status();
}
