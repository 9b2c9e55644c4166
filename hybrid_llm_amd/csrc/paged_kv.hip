// Per-head norms and position rotation of query and key rows, and the append of
// keys and values to a paged cache in the same pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w        over one head's HD values (optional)
//   (y_a, y_b) -> (y_a cos t - y_b sin t, y_b cos t + y_a sin t),  t = pos * inv_freq[i]
//
// for the pairs (a, b) = (i, i + half) or (2i, 2i + 1) of the first 2 half dims; the
// other dims pass.  In fp32 from the bf16 rows to one rounding at the store; keys of a 4-bit
// cache in fp64.
//
// The angle of a far position has more digits than fp32 holds (pos 2^20 at
// inv_freq 1 leaves 2^-3 of a radian), so pos * inv_freq / 2 pi is formed in fp64,
// its whole turns dropped there, and only the fraction goes on in fp32.  A table of
// cosines would cost max_pos * half * 8 bytes and bound the positions; one sincospi
// a lane and task costs less than the task's loads.
//
// Bound by memory: a wave takes one token and IT * 512 / HD of its rows (a row: one
// head of q, k or v), HD / 8 lanes a row, all rows' loads issued before the first is
// used.  A lane holds 4 dims of each half of its pairs, dims 4c.. and half + 4c..,
// so a pair never crosses lanes; lane l forms the cosine and sine of pair l once
// and hands them round through LDS.
//
// A 4-bit cache (kCacheMx4) stores blocks of 32 dims: the smallest power of two of which 7
// cover the block's largest magnitude, and each value over it as a 4-bit float, to nearest
// even.  7 and not 6, the largest code: what lies between is off by no more than half of
// the code's last step, like the values under 6, and the finer scale serves the other 31.
// A key next to a border between two codes is a whole step off if its rounding crosses it: of
// 262144 normed and rotated keys in fp32 one did in a few calls, so 4-bit keys are formed in
// 64 bits (3.6 -> 4.4 us for one token, 5.1 -> 6.4 for 256 of 8 x 128, 7.0 -> 11.6 for 8191 of
// 2 x 128) and come to fp32 by rounding to odd, after which a second rounding to fewer bits is
// as good as the only one.
#include "common.hpp"
#include "abi_util.hpp"
#include "paged.hpp"

namespace llmy {

struct RopeArgs {
  const uint16_t* x[3];          // q, k, v rows [N, H, HD]
  long long xr[3], xh[3];        // their strides (elements) by row and head
  uint16_t* o[2];                // q_out; k_out (null: k and v go to the cache)
  long long orow[2], ohead[2];
  const float* w[2];             // norm weights [HD] or null
  const int32_t* pos;
  const float* inv_freq;
  const int32_t* rows;           // page-table row of token n, or null: n
  const int32_t* table;
  void *kc, *vc;
  uint8_t *ks, *vs;              // a 4-bit cache's block scales
  float eps, scale[2], inv[2];   // of an 8-bit cache: k's and v's scale, 1 / it
  int half, interleaved;
  int N, hq, hkv, heads;         // heads: rows of one token (q, k and, with a cache, v)
  int chunks;                    // tasks of one token
  int B, width, shift, pages;    // page table [B, width], tokens a page = 1 << shift
};

__device__ __forceinline__ void unpack4(const uint2& v, float* out) {
  out[0] = __uint_as_float(v.x << 16);
  out[1] = __uint_as_float(v.x & 0xffff0000u);
  out[2] = __uint_as_float(v.y << 16);
  out[3] = __uint_as_float(v.y & 0xffff0000u);
}

// 4 values over their scale as e4m3: saturated at the largest finite one (NaN stays NaN), to
// nearest even.  A product with the reciprocal alone would move a quotient half way
// between two codes to the wrong one (under 7 / 64 or 0.3 some bf16 values are), so its
// remainder corrects it: the rounded quotient, for the scales that scales_ok lets
// through.  (8191 x 4 rows: 6.1 us, with the product
// alone 6.0, with a division 6.9.)
__device__ __forceinline__ uint32_t pack4_e4m3(const float* v, float scale, float inv) {
  float t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = __builtin_amdgcn_fmed3f(v[i] * inv, -448.f, 448.f);
    const float s = fmaf(-fmaf(q, scale, -v[i]), inv, q);  // (so a zero keeps its sign)
    t[i] = __builtin_elementwise_maximum(__builtin_elementwise_minimum(s, 448.f), -448.f);
  }
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], r, true));
}

// The mean square of a row, of which this lane has y.
template <int HD>
__device__ __forceinline__ float mean_square(const float* y) {
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
  ss += dpp_f<kDppXor1>(ss);
  ss += dpp_f<kDppXor2>(ss);
  ss += dpp_f<kDppHalfMirror>(ss);
  if (HD == 128) ss += dpp_f<kDppMirror>(ss);
  return ss * (1.f / HD);
}

// To fp32: what is not exact to the neighbour with an odd last bit.
__device__ __forceinline__ float to_odd(double d) {
  const float f = static_cast<float>(d);
  const double back = f;
  const uint32_t u = __float_as_uint(f);
  if (back == d || (u & 1u)) return f;
  return __uint_as_float(fabs(back) > fabs(d) ? u - 1u : u + 1u);  // (NaN stays one)
}

// Below this mean square the squares may have lost bits to fp32's end; such rows, all under
// 2^-41, are raised so that bf16's smallest squares to a normal number.  Rows whose
// squares overflowed reach past 2^60 and are lowered; what that takes below the
// smallest normal is under 2^-100 of the row.
constexpr float kLeastMean = 0x1p-90f, kRaise = 0x1p100f, kLower = 0x1p-70f;

// 8 values under a block scale 2^(byte - 127), byte 1 to 254, as 4-bit floats in order from
// the lowest bits; magnitudes past 6 steps become 6.
__device__ __forceinline__ uint32_t pack8_mx4(const float* v, uint32_t byte) {
  const float step = __uint_as_float(byte << 23);
  uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], step, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], step, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], step, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], step, 3);
}

// The scale byte of a block of 32 dims, 8 on each of four neighbouring lanes: 255 where one
// is not finite.  Magnitudes compare as integers, NaN past infinity; adding all but 1 of a
// quarter of the mantissa's range carries into the exponent past 1.75, 7 / 4.  Largest
// magnitudes over 1.5 x 2^127 count as that, or their code would stand for 2^128.
__device__ __forceinline__ uint32_t mx4_scale(const float* y) {
  uint32_t most = 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(y[j]) & 0x7fffffffu);
  most = max(most, dpp_u<kDppXor1>(most));
  most = max(most, dpp_u<kDppXor2>(most));
  if (most >= 0x7f800000u) return 255u;
  const uint32_t e = (min(most, 0x7f400000u) + 0x1fffffu) >> 23;
  return max(e, 3u) - 2u;
}

template <int HD, int IT, bool CACHE, int CT>
__global__ __launch_bounds__(256) void norm_rope_kernel(const RopeArgs a) {
  constexpr bool F8 = CT == kCacheE4m3, M4 = CT == kCacheMx4;
  constexpr int LPR = HD / 8;   // lanes a row
  constexpr int RPI = 64 / LPR; // rows an iteration
  __shared__ __align__(16) float trig[4][2][64];
  __shared__ __align__(16) float turn[M4 ? 4 : 1][M4 ? 512 : 4];
  __shared__ __align__(16) double trig64[M4 ? 4 : 1][2][M4 ? 64 : 2];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const uint32_t task = blockIdx.x * 4u + wave;
  const int n = static_cast<int>(task / static_cast<uint32_t>(a.chunks));
  if (n >= a.N) return;
  const int p = a.pos[n];
  if (p < 0) return;  // a padding row: left as it was
  const int first = static_cast<int>(task - static_cast<uint32_t>(n) * a.chunks) * (IT * RPI);
  const int g = lane / LPR, c = lane % LPR;
  const bool turned = c < a.half / 4;
  const bool split = turned && !a.interleaved;
  const int d0 = split ? 4 * c : 8 * c;
  const int d1 = split ? a.half + 4 * c : 8 * c + 4;

  // where this token's keys and values go; nowhere without a valid slot
  long long slot = -1;  // element of head 0's row in the cache
  if (CACHE) {
    const int row = a.rows ? a.rows[n] : n;
    const int pi = p >> a.shift;
    if (row >= 0 && row < a.B && pi < a.width) {
      const int page = a.table[static_cast<long long>(row) * a.width + pi];
      if (page >= 0 && page < a.pages)
        slot = ((static_cast<long long>(page) * a.hkv << a.shift) + (p & ((1 << a.shift) - 1))) * HD;
    }
  }

  uint2 x0[IT], x1[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int r = first + i * RPI + g;
    x0[i] = x1[i] = make_uint2(0u, 0u);
    if (r < a.heads) {
      const int kind = r < a.hq ? 0 : r < a.hq + a.hkv ? 1 : 2;
      const int h = r - (kind == 0 ? 0 : kind == 1 ? a.hq : a.hq + a.hkv);
      const uint16_t* src = kind == 0   ? a.x[0] + n * a.xr[0] + h * a.xh[0]
                            : kind == 1 ? a.x[1] + n * a.xr[1] + h * a.xh[1]
                                        : a.x[2] + n * a.xr[2] + h * a.xh[2];
      x0[i] = *reinterpret_cast<const uint2*>(src + d0);
      x1[i] = *reinterpret_cast<const uint2*>(src + d1);
    }
  }

  float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
  if (lane < a.half) {
    const double turns = static_cast<double>(p) * static_cast<double>(a.inv_freq[lane]) *
                         0.15915494309189535;  // 1 / (2 pi)
    float s, co;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &co);
    trig[wave][0][lane] = co;
    trig[wave][1][lane] = s;
    if (M4 && first < a.hq + a.hkv && first + IT * RPI > a.hq) {  // this wave has keys
      double s64, c64;
      sincospi(2. * (turns - rint(turns)), &s64, &c64);
      trig64[M4 ? wave : 0][0][M4 ? lane : 0] = c64;
      trig64[M4 ? wave : 0][1][M4 ? lane : 0] = s64;
    }
  }
  wave_lds_order();
  if (turned) {
    *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(&trig[wave][0][4 * c]);
    *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(&trig[wave][1][4 * c]);
  }

  const bool normed = a.w[0] || a.w[1];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int r = first + i * RPI + g;
    const int kind = r < a.hq ? 0 : r < a.hq + a.hkv ? 1 : 2;
    const int h = r - (kind == 0 ? 0 : kind == 1 ? a.hq : a.hq + a.hkv);
    float y[8];
    unpack4(x0[i], y);
    unpack4(x1[i], y + 4);
    const float* w = kind == 0 ? a.w[0] : kind == 1 ? a.w[1] : nullptr;
    float mean = mean_square<HD>(y) + a.eps;
    // rows whose squares overflow, or vanish with an eps that does too: times a power of
    // two, which the norm takes out (1 for the other rows of such a wave)
    const bool odd = w && r < a.heads && !(mean >= kLeastMean && mean < INFINITY);
    if (normed && __ballot(odd)) {
      const float by = !odd ? 1.f : mean < 1.f ? kRaise : kLower;
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= by;
      mean = mean_square<HD>(y) + a.eps * by * by;
    }
    if (!M4 && r >= a.heads) continue;  // (4 bits: all lanes meet again below)
    if (w) {
      const float rs = rsqrtf(mean);
      const float4 w0 = *reinterpret_cast<const float4*>(w + d0);
      const float4 w1 = *reinterpret_cast<const float4*>(w + d1);
      y[0] *= rs * w0.x; y[1] *= rs * w0.y; y[2] *= rs * w0.z; y[3] *= rs * w0.w;
      y[4] *= rs * w1.x; y[5] *= rs * w1.y; y[6] *= rs * w1.z; y[7] *= rs * w1.w;
    }
    if (turned && kind != 2) {
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = y[2 * j], v = y[2 * j + 1];
          y[2 * j] = u * cs[j] - v * sn[j];
          y[2 * j + 1] = v * cs[j] + u * sn[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = y[j], v = y[j + 4];
          y[j] = u * cs[j] - v * sn[j];
          y[j + 4] = v * cs[j] + u * sn[j];
        }
      }
    }
    if (M4 && (a.w[1] || a.half > 0) && __ballot(kind == 1)) {  // keys again, in 64 bits
      float x[8];
      unpack4(x0[i], x);
      unpack4(x1[i], x + 4);
      double z[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = x[j];
      if (a.w[1]) {
        double ss = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fma(z[j], z[j], ss);
        ss += __builtin_bit_cast(double, dpp_u64<kDppXor1>(__builtin_bit_cast(uint64_t, ss)));
        ss += __builtin_bit_cast(double, dpp_u64<kDppXor2>(__builtin_bit_cast(uint64_t, ss)));
        ss += __builtin_bit_cast(double, dpp_u64<kDppHalfMirror>(__builtin_bit_cast(uint64_t, ss)));
        if (HD == 128)
          ss += __builtin_bit_cast(double, dpp_u64<kDppMirror>(__builtin_bit_cast(uint64_t, ss)));
        const double rs = 1. / sqrt(ss * (1. / HD) + static_cast<double>(a.eps));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          z[j] *= rs * static_cast<double>(a.w[1][d0 + j]);
          z[j + 4] *= rs * static_cast<double>(a.w[1][d1 + j]);
        }
      }
      if (turned) {
        const double* c64 = trig64[M4 ? wave : 0][0] + (M4 ? 4 * c : 0);
        const double* s64 = trig64[M4 ? wave : 0][1] + (M4 ? 4 * c : 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double u = z[j], v = z[j + 4];
          if (!a.interleaved) {
            z[j] = u * c64[j] - v * s64[j];
            z[j + 4] = v * c64[j] + u * s64[j];
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double u = z[2 * j], v = z[2 * j + 1];
          if (a.interleaved) {
            z[2 * j] = u * c64[j] - v * s64[j];
            z[2 * j + 1] = v * c64[j] + u * s64[j];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = kind == 1 ? to_odd(z[j]) : y[j];
    }
    if (M4) {
      // blocks are of neighbouring dims: each row's values in order through LDS
      float z[8];
      float* const own = turn[M4 ? wave : 0] + g * HD;
      wave_lds_order();  // behind the last iteration's reads
      *reinterpret_cast<float4*>(own + d0) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(own + d1) = make_float4(y[4], y[5], y[6], y[7]);
      wave_lds_order();
      *reinterpret_cast<float4*>(z) = *reinterpret_cast<const float4*>(own + 8 * c);
      *reinterpret_cast<float4*>(z + 4) = *reinterpret_cast<const float4*>(own + 8 * c + 4);
      const uint32_t byte = mx4_scale(z);
      if (kind != 0 && r < a.heads && slot >= 0) {
        const long long row = slot / HD + (static_cast<long long>(h) << a.shift);
        const uint32_t codes = byte == 255u ? 0u : pack8_mx4(z, byte);
        uint8_t* const to = static_cast<uint8_t*>(kind == 1 ? a.kc : a.vc);
        *reinterpret_cast<uint32_t*>(to + row * (HD / 2) + 4 * c) = codes;
        if ((c & 3) == 0) (kind == 1 ? a.ks : a.vs)[row * (HD / 32) + (c >> 2)] = byte;
      }
      if (kind != 0 || r >= a.heads) continue;
    }
    if (CACHE && kind != 0) {
      if (slot < 0) continue;
      const long long at = slot + (static_cast<long long>(h) << a.shift) * HD;
      if (F8) {
        uint8_t* dst = static_cast<uint8_t*>(kind == 1 ? a.kc : a.vc) + at;
        const float scale = kind == 1 ? a.scale[0] : a.scale[1],
                    inv = kind == 1 ? a.inv[0] : a.inv[1];
        *reinterpret_cast<uint32_t*>(dst + d0) = pack4_e4m3(y, scale, inv);
        *reinterpret_cast<uint32_t*>(dst + d1) = pack4_e4m3(y + 4, scale, inv);
      } else {
        uint16_t* dst = static_cast<uint16_t*>(kind == 1 ? a.kc : a.vc) + at;
        *reinterpret_cast<uint2*>(dst + d0) = make_uint2(pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]));
        *reinterpret_cast<uint2*>(dst + d1) = make_uint2(pack_bf2(y[4], y[5]), pack_bf2(y[6], y[7]));
      }
    } else {
      uint16_t* dst = kind == 0 ? a.o[0] + n * a.orow[0] + h * a.ohead[0]
                                : a.o[1] + n * a.orow[1] + h * a.ohead[1];
      *reinterpret_cast<uint2*>(dst + d0) = make_uint2(pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]));
      *reinterpret_cast<uint2*>(dst + d1) = make_uint2(pack_bf2(y[4], y[5]), pack_bf2(y[6], y[7]));
    }
  }
}

// Stored rows back as bf16, which holds each of them exactly (a code has two significant
// bits); zeros for a token without a slot.  8 dims a lane: 4 bytes in, 16 out; bound by the
// writes.
struct ReadArgs {
  const uint8_t *kc, *vc, *ks, *vs;
  const int32_t *table, *rows, *pos;
  uint16_t *k, *v;               // [N, Hkv, HD]
  int N, hkv, B, width, shift, pages;
};

template <int HD>
__global__ __launch_bounds__(256) void mx4_read_kernel(const ReadArgs a) {
  constexpr int LPR = HD / 8;
  const long long at = blockIdx.x * 256ll + threadIdx.x;
  const int c = static_cast<int>(at % LPR);
  long long row = at / LPR;  // token, k or v, head
  const int h = static_cast<int>(row % a.hkv);
  row /= a.hkv;
  const bool is_v = row & 1;
  row >>= 1;
  if (row >= a.N) return;
  const int n = static_cast<int>(row), p = a.pos[n], r = a.rows ? a.rows[n] : n;
  uint4 out = uint4{0u, 0u, 0u, 0u};
  if (p >= 0 && r >= 0 && r < a.B && (p >> a.shift) < a.width) {
    const int page = a.table[static_cast<long long>(r) * a.width + (p >> a.shift)];
    if (page >= 0 && page < a.pages) {
      const long long s = ((static_cast<long long>(page) * a.hkv + h) << a.shift) +
                          (p & ((1 << a.shift) - 1));
      const uint32_t w = *reinterpret_cast<const uint32_t*>((is_v ? a.vc : a.kc) + s * (HD / 2) + 4 * c);
      out = mx4_to_bf16(w, (is_v ? a.vs : a.ks)[s * (HD / 32) + (c >> 2)]);
    }
  }
  *reinterpret_cast<uint4*>((is_v ? a.v : a.k) + (static_cast<long long>(n) * a.hkv + h) * HD + 8 * c) = out;
}

template <bool CACHE, int CT>
int32_t launch_norm_rope(RopeArgs a, int head_dim, hipStream_t s) {
  const int rpi = 512 / head_dim;
  // Four iterations a wave read at the rate of a copy (16384 tokens x 40 rows of 128: 65 us,
  // 5.2 TB/s; one iteration 91 us), one spreads a small call over more waves (1003 x 18: 4.8
  // us against 5.2) and leaves none of a token's last wave idle, since a wave stays with
  // its token (8191 x 4 into an e4m3 cache, 12 of 16 row slots empty: 6.3 against 6.9); but
  // 4096 x 20 rows of 64: 8.3 against 7.0.  The border lies somewhere between 33 and 82
  // thousand rows; nothing in between was measured, nor rows of both widths at one size.
  const int it = static_cast<long long>(a.N) * a.heads >= 65536 ? 4 : 1;
  a.chunks = (a.heads + it * rpi - 1) / (it * rpi);
  const long long wgs = (static_cast<long long>(a.N) * a.chunks + 3) / 4;
  LLMY_REQUIRE(wgs < (1ll << 29));  // task numbers are 32-bit
  const dim3 grid(static_cast<unsigned>(wgs));
  if (head_dim == 64) {
    if (it == 1)
      hipLaunchKernelGGL((norm_rope_kernel<64, 1, CACHE, CT>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((norm_rope_kernel<64, 4, CACHE, CT>), grid, dim3(256), 0, s, a);
  } else {
    if (it == 1)
      hipLaunchKernelGGL((norm_rope_kernel<128, 1, CACHE, CT>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((norm_rope_kernel<128, 4, CACHE, CT>), grid, dim3(256), 0, s, a);
  }
  return launch_status();
}

// Rows [N, H, HD] of 16-bit words that 8-byte accesses reach.
inline bool rows_ok(const void* p, int64_t row, int64_t head, int32_t H, int32_t hd) {
  return p && aligned(p, 8) && row % 4 == 0 && head % 4 == 0 && row >= 0 && head >= 0 &&
         (H <= 1 || head >= hd);
}

}  // namespace llmy

using namespace llmy;

extern "C" int32_t llmy_qk_norm_rope_bf16(
    const llmy_bf16* q, int64_t q_row, int64_t q_head, const llmy_bf16* k, int64_t k_row,
    int64_t k_head, const int32_t* positions, const float* inv_freq, int32_t half,
    const float* q_norm, const float* k_norm, float eps, int32_t interleaved, llmy_bf16* q_out,
    int64_t qo_row, int64_t qo_head, llmy_bf16* k_out, int64_t ko_row, int64_t ko_head, int32_t N,
    int32_t Hq, int32_t Hkv, int32_t head_dim, void* stream) {
  LLMY_REQUIRE(N >= 0 && Hq > 0 && Hkv > 0 && Hq <= kMaxHeads && Hkv <= kMaxHeads);
  LLMY_REQUIRE(head_dim == 64 || head_dim == 128);
  LLMY_REQUIRE(half >= 0 && half % 4 == 0 && 2 * half <= head_dim && (half == 0 || inv_freq));
  LLMY_REQUIRE(eps >= 0.f);
  if (N == 0) return 0;
  LLMY_REQUIRE(positions && rows_ok(q, q_row, q_head, Hq, head_dim) &&
               rows_ok(k, k_row, k_head, Hkv, head_dim) &&
               rows_ok(q_out, qo_row, qo_head, Hq, head_dim) &&
               rows_ok(k_out, ko_row, ko_head, Hkv, head_dim));
  LLMY_REQUIRE(aligned(q_norm, 16) && aligned(k_norm, 16));
  // rows are written while other waves still read theirs
  const Rows qi{q, q_row, q_head, N, Hq, head_dim}, ki{k, k_row, k_head, N, Hkv, head_dim},
      qo{q_out, qo_row, qo_head, N, Hq, head_dim}, ko{k_out, ko_row, ko_head, N, Hkv, head_dim};
  LLMY_REQUIRE(rows_apart(qo) && rows_apart(ko) && rows_apart(qo, ko) &&
               in_place_or_apart(qo, qi) && in_place_or_apart(ko, ki) && rows_apart(qo, ki) &&
               rows_apart(ko, qi));
  RopeArgs a{};
  a.x[0] = q; a.xr[0] = q_row; a.xh[0] = q_head;
  a.x[1] = k; a.xr[1] = k_row; a.xh[1] = k_head;
  a.o[0] = q_out; a.orow[0] = qo_row; a.ohead[0] = qo_head;
  a.o[1] = k_out; a.orow[1] = ko_row; a.ohead[1] = ko_head;
  a.w[0] = q_norm; a.w[1] = k_norm;
  a.pos = positions; a.inv_freq = inv_freq; a.eps = eps;
  a.half = half; a.interleaved = interleaved != 0;
  a.N = N; a.hq = Hq; a.hkv = Hkv; a.heads = Hq + Hkv;
  return launch_norm_rope<false, kCacheBf16>(a, head_dim, as_stream(stream));
}

extern "C" int32_t llmy_paged_kv_append(
    const llmy_bf16* k, int64_t k_row, int64_t k_head, const llmy_bf16* v, int64_t v_row,
    int64_t v_head, void* k_cache, void* v_cache, int32_t cache_type, float k_scale,
    float v_scale, const int32_t* page_table, const int32_t* rows, const int32_t* positions,
    const float* inv_freq, int32_t half, const float* k_norm, float eps, int32_t interleaved,
    const llmy_bf16* q, int64_t q_row, int64_t q_head, const float* q_norm, llmy_bf16* q_out,
    int64_t qo_row, int64_t qo_head, int32_t N, int32_t Hq, int32_t Hkv, int32_t head_dim,
    int32_t B, int32_t width, int32_t page, int32_t pages, void* stream) {
  LLMY_REQUIRE(N >= 0 && Hq >= 0 && Hkv > 0 && Hq <= kMaxHeads && Hkv <= kMaxHeads);
  LLMY_REQUIRE(head_dim == 64 || head_dim == 128);
  LLMY_REQUIRE(half >= 0 && half % 4 == 0 && 2 * half <= head_dim && (half == 0 || inv_freq));
  LLMY_REQUIRE(eps >= 0.f);
  LLMY_REQUIRE(B >= 0 && width >= 0 && pages >= 0 && page_shift(page) > 0);
  LLMY_REQUIRE(cache_type == kCacheBf16 || cache_type == kCacheE4m3);
  LLMY_REQUIRE(scales_ok(cache_type, k_scale, v_scale));
  if (N == 0) return 0;
  LLMY_REQUIRE(positions && rows_ok(k, k_row, k_head, Hkv, head_dim) &&
               rows_ok(v, v_row, v_head, Hkv, head_dim));
  LLMY_REQUIRE((B == 0 || width == 0 || page_table) &&
               (pages == 0 || (k_cache && v_cache && aligned(k_cache, 16) && aligned(v_cache, 16))));
  const int64_t cache_words = static_cast<int64_t>(pages) * Hkv * page * head_dim /
                              (cache_type == kCacheE4m3 ? 2 : 1);
  LLMY_REQUIRE(apart(static_cast<uint16_t*>(k_cache), cache_words,
                     static_cast<uint16_t*>(v_cache), cache_words));
  LLMY_REQUIRE(aligned(q_norm, 16) && aligned(k_norm, 16));
  if (Hq > 0) {
    LLMY_REQUIRE(rows_ok(q, q_row, q_head, Hq, head_dim) &&
                 rows_ok(q_out, qo_row, qo_head, Hq, head_dim));
    // rows are written while other waves still read theirs
    const Rows qo{q_out, qo_row, qo_head, N, Hq, head_dim};
    LLMY_REQUIRE(rows_apart(qo) &&
                 in_place_or_apart(qo, Rows{q, q_row, q_head, N, Hq, head_dim}) &&
                 rows_apart(qo, Rows{k, k_row, k_head, N, Hkv, head_dim}) &&
                 rows_apart(qo, Rows{v, v_row, v_head, N, Hkv, head_dim}) &&
                 rows_apart(qo, k_cache, 2 * cache_words) &&
                 rows_apart(qo, v_cache, 2 * cache_words));
  }
  RopeArgs a{};
  a.x[0] = q; a.xr[0] = q_row; a.xh[0] = q_head;
  a.x[1] = k; a.xr[1] = k_row; a.xh[1] = k_head;
  a.x[2] = v; a.xr[2] = v_row; a.xh[2] = v_head;
  a.o[0] = q_out; a.orow[0] = qo_row; a.ohead[0] = qo_head;
  a.w[0] = q_norm; a.w[1] = k_norm;
  a.pos = positions; a.inv_freq = inv_freq; a.eps = eps;
  a.half = half; a.interleaved = interleaved != 0;
  a.rows = rows; a.table = page_table; a.kc = k_cache; a.vc = v_cache;
  a.scale[0] = k_scale; a.scale[1] = v_scale;
  a.inv[0] = 1.f / k_scale; a.inv[1] = 1.f / v_scale;
  a.N = N; a.hq = Hq; a.hkv = Hkv; a.heads = Hq + 2 * Hkv;
  a.B = B; a.width = width; a.shift = page_shift(page); a.pages = pages;
  return cache_type == kCacheE4m3
             ? launch_norm_rope<true, kCacheE4m3>(a, head_dim, as_stream(stream))
             : launch_norm_rope<true, kCacheBf16>(a, head_dim, as_stream(stream));
}

extern "C" int32_t llmy_paged_kv_append_mx4(
    const llmy_bf16* k, int64_t k_row, int64_t k_head, const llmy_bf16* v, int64_t v_row,
    int64_t v_head, void* k_cache, void* v_cache, void* k_scales, void* v_scales,
    const int32_t* page_table, const int32_t* rows, const int32_t* positions,
    const float* inv_freq, int32_t half, const float* k_norm, float eps, int32_t interleaved,
    const llmy_bf16* q, int64_t q_row, int64_t q_head, const float* q_norm, llmy_bf16* q_out,
    int64_t qo_row, int64_t qo_head, int32_t N, int32_t Hq, int32_t Hkv, int32_t head_dim,
    int32_t B, int32_t width, int32_t page, int32_t pages, void* stream) {
  LLMY_REQUIRE(N >= 0 && Hq >= 0 && Hkv > 0 && Hq <= kMaxHeads && Hkv <= kMaxHeads);
  LLMY_REQUIRE(head_dim == 64 || head_dim == 128);
  LLMY_REQUIRE(half >= 0 && half % 4 == 0 && 2 * half <= head_dim && (half == 0 || inv_freq));
  LLMY_REQUIRE(eps >= 0.f);
  LLMY_REQUIRE(B >= 0 && width >= 0 && pages >= 0 && page_shift(page) > 0);
  if (N == 0) return 0;
  LLMY_REQUIRE(positions && rows_ok(k, k_row, k_head, Hkv, head_dim) &&
               rows_ok(v, v_row, v_head, Hkv, head_dim));
  const Mx4Cache c{k_cache, v_cache, k_scales, v_scales};
  const int64_t slots = static_cast<int64_t>(pages) * Hkv * page;
  LLMY_REQUIRE((B == 0 || width == 0 || page_table) && c.ok(slots, head_dim) &&
               c.apart(slots, head_dim));
  LLMY_REQUIRE(aligned(q_norm, 16) && aligned(k_norm, 16));
  // the caches are written while other waves still read rows and weights
  for (int i = 0; i < 4; ++i)
    LLMY_REQUIRE(rows_apart(Rows{k, k_row, k_head, N, Hkv, head_dim}, c.part(i),
                            c.bytes(i, slots, head_dim)) &&
                 rows_apart(Rows{v, v_row, v_head, N, Hkv, head_dim}, c.part(i),
                            c.bytes(i, slots, head_dim)));
  if (Hq > 0) {
    LLMY_REQUIRE(rows_ok(q, q_row, q_head, Hq, head_dim) &&
                 rows_ok(q_out, qo_row, qo_head, Hq, head_dim));
    const Rows qi{q, q_row, q_head, N, Hq, head_dim}, qo{q_out, qo_row, qo_head, N, Hq, head_dim};
    LLMY_REQUIRE(rows_apart(qo) && in_place_or_apart(qo, qi) &&
                 rows_apart(qo, Rows{k, k_row, k_head, N, Hkv, head_dim}) &&
                 rows_apart(qo, Rows{v, v_row, v_head, N, Hkv, head_dim}));
    for (int i = 0; i < 4; ++i)
      LLMY_REQUIRE(rows_apart(qo, c.part(i), c.bytes(i, slots, head_dim)) &&
                   rows_apart(qi, c.part(i), c.bytes(i, slots, head_dim)));
  }
  RopeArgs a{};
  a.x[0] = q; a.xr[0] = q_row; a.xh[0] = q_head;
  a.x[1] = k; a.xr[1] = k_row; a.xh[1] = k_head;
  a.x[2] = v; a.xr[2] = v_row; a.xh[2] = v_head;
  a.o[0] = q_out; a.orow[0] = qo_row; a.ohead[0] = qo_head;
  a.w[0] = q_norm; a.w[1] = k_norm;
  a.pos = positions; a.inv_freq = inv_freq; a.eps = eps;
  a.half = half; a.interleaved = interleaved != 0;
  a.rows = rows; a.table = page_table; a.kc = k_cache; a.vc = v_cache;
  a.ks = static_cast<uint8_t*>(k_scales); a.vs = static_cast<uint8_t*>(v_scales);
  a.N = N; a.hq = Hq; a.hkv = Hkv; a.heads = Hq + 2 * Hkv;
  a.B = B; a.width = width; a.shift = page_shift(page); a.pages = pages;
  return launch_norm_rope<true, kCacheMx4>(a, head_dim, as_stream(stream));
}

extern "C" int32_t llmy_paged_kv_read_mx4(const void* k_cache, const void* v_cache,
                                          const void* k_scales, const void* v_scales,
                                          const int32_t* page_table, const int32_t* rows,
                                          const int32_t* positions, llmy_bf16* k, llmy_bf16* v,
                                          int32_t N, int32_t Hkv, int32_t head_dim, int32_t B,
                                          int32_t width, int32_t page, int32_t pages,
                                          void* stream) {
  LLMY_REQUIRE(N >= 0 && Hkv > 0 && Hkv <= kMaxHeads && (head_dim == 64 || head_dim == 128));
  LLMY_REQUIRE(B >= 0 && width >= 0 && pages >= 0 && page_shift(page) > 0);
  if (N == 0) return 0;
  const Mx4Cache c{const_cast<void*>(k_cache), const_cast<void*>(v_cache),
                   const_cast<void*>(k_scales), const_cast<void*>(v_scales)};
  const int64_t slots = static_cast<int64_t>(pages) * Hkv * page;
  LLMY_REQUIRE(positions && k && v && aligned(k, 16) && aligned(v, 16) &&
               (B == 0 || width == 0 || page_table) && c.ok(slots, head_dim));
  const int64_t bytes = 2ll * N * Hkv * head_dim;
  LLMY_REQUIRE(bytes_apart(k, bytes, v, bytes));
  for (int i = 0; i < 4; ++i)
    LLMY_REQUIRE(bytes_apart(k, bytes, c.part(i), c.bytes(i, slots, head_dim)) &&
                 bytes_apart(v, bytes, c.part(i), c.bytes(i, slots, head_dim)));
  ReadArgs a{};
  a.kc = static_cast<const uint8_t*>(k_cache); a.vc = static_cast<const uint8_t*>(v_cache);
  a.ks = static_cast<const uint8_t*>(k_scales); a.vs = static_cast<const uint8_t*>(v_scales);
  a.table = page_table; a.rows = rows; a.pos = positions; a.k = k; a.v = v;
  a.N = N; a.hkv = Hkv; a.B = B; a.width = width; a.shift = page_shift(page); a.pages = pages;
  const long long lanes = static_cast<long long>(N) * Hkv * 2 * (head_dim / 8);
  LLMY_REQUIRE(lanes < (1ll << 38));  // workgroups are 31-bit
  const dim3 grid(static_cast<unsigned>((lanes + 255) / 256));
  const hipStream_t s = as_stream(stream);
  if (head_dim == 64)
    hipLaunchKernelGGL(mx4_read_kernel<64>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(mx4_read_kernel<128>, grid, dim3(256), 0, s, a);
  return launch_status();
}
