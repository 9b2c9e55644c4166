// Staging and fragment reads shared by the attention kernels whose K and V tiles
// arrive by DMA into swizzled LDS stages.
#pragma once

#include "common.hpp"

namespace llmy {

typedef __attribute__((address_space(3))) void lds_void;
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// 16 bytes a lane from global memory straight into LDS: lane l's land at dst + 16 l.
__device__ __forceinline__ void dma16(const void* src, void* lds_dst) {
  __builtin_amdgcn_global_load_lds(src, (lds_void*)lds_dst, 16, 0, 0);
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_void*)p));
}

// LDS reads as inline asm: with a DMA into another stage in flight, the
// compiler would make every LDS read wait for it.  Their results are valid
// after lds_settle.
__device__ __forceinline__ u32x4 lds_b128(uint32_t addr) {
  u32x4 v;
  asm volatile("ds_read_b128 %0, %1" : "=v"(v) : "v"(addr) : "memory");
  return v;
}

__device__ __forceinline__ u32x2 lds_tr16(uint32_t addr) {
  u32x2 v;
  asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(v) : "v"(addr) : "memory");
  return v;
}

// Wait for every LDS read of this wave and tie the registers they filled to
// the wait, so no use is scheduled above it.
__device__ __forceinline__ void lds_settle4(u32x4* f) {
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3])::"memory");
}

__device__ __forceinline__ void lds_settle_v(u32x2* f) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]), "+v"(f[4]), "+v"(f[5]),
                 "+v"(f[6]), "+v"(f[7])::"memory");
}

// The same copy as a statement the compiler knows nothing of but its memory clobber, so
// that LDS reads need not wait for copies into other stages; the kernel waits for its
// copies (vmcnt) itself.  base is the same for every lane, off a lane's bytes from it,
// dst the wave's LDS byte address.  s_nop 3 after the move of m0 makes the five wait
// states that the load needs after a VALU write of an SGPR that it reads.  m0 is
// reserved (hence a warning), but the compiler keeps values there for its own use:
// the clobber says that they are gone.  STREAM: data read once, not kept in the caches.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <bool STREAM = false>
__device__ __forceinline__ void lds_fill16(const void* base, uint32_t off, uint32_t dst) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 ::"s"(dst), "v"(off), "s"(base) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2"
                 ::"s"(dst), "v"(off), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

// LDS reads at a byte address, for kernels that fill LDS by lds_fill16: the compiler
// waits for each result where it is used.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ u32x4 lds_get16(uint32_t addr) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(addr);
}

// In each 16-lane group lane y addresses 8 bytes, 4 columns 4 (y & 3) .. of row y / 4, and
// receives column y of the 4 rows.
__device__ __forceinline__ u32x2 lds_get_tr16(uint32_t addr) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      reinterpret_cast<__attribute__((address_space(3))) s16x4*>(addr)));
}

// Lane y of a group addresses 8 bytes, half y & 1 of row y / 2 of 8 rows of 16 bytes, and
// receives column y of the 8 rows.
__device__ __forceinline__ u32x2 lds_get_tr8(uint32_t addr) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
      reinterpret_cast<__attribute__((address_space(3))) i32x2*>(addr)));
}

__device__ __forceinline__ uint4 pack8_bf16(const float* v) {
  return uint4{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]),
               pack_bf2(v[6], v[7])};
}

// cap * tanh(x / cap) * log2(e) of a score x, x2 = x * 2 log2(e) / cap: from one
// exponential and one reciprocal, 1 - 2 / (2^x2 + 1), which saturates at both ends
// (2^x2 = inf or 0).  Its error is a few 2^-24 of the cap.
__device__ __forceinline__ float softcap_log2(float x2, float cap_log2) {
  return fmaf(-2.f * cap_log2, __builtin_amdgcn_rcpf(exp2_fast(x2) + 1.f), cap_log2);
}

}  // namespace llmy
