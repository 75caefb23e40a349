// What the attention kernels over the paged cache share on the device: exchange between
// lanes, loads to LDS, the matrix instructions' operand types, and the sharing out of
// work among workgroups.
#ifndef RPG_AMD_ATTENTION_DEV_H_
#define RPG_AMD_ATTENTION_DEV_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "dev_util.h"

namespace rpg {
namespace attn {

using Half2 = _Float16 __attribute__((ext_vector_type(2)));
using Half8 = _Float16 __attribute__((ext_vector_type(8)));
using F32x4 = float __attribute__((ext_vector_type(4)));
using I32x4 = int __attribute__((ext_vector_type(4)));
using I32x2 = int __attribute__((ext_vector_type(2)));
using S16x4 = short __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- lane exchange

// x of the lane kBy before it in its row of 16, which goes round.
template <int kBy>
__device__ __forceinline__ float Ror(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x120 + kBy, 0xF, 0xF, false));
}

// f over the four lanes l, l ^ 16, l ^ 32, l ^ 48; every one of them has the result.
template <class F>
__device__ __forceinline__ float AcrossRows(float x, F f) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = f(__int_as_float(a[0]), __int_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return f(__int_as_float(b[0]), __int_as_float(b[1]));
}
__device__ __forceinline__ float MaxAcrossRows(float x) {
  return AcrossRows(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float SumAcrossRows(float x) {
  return AcrossRows(x, [](float a, float b) { return a + b; });
}

// ---------------------------------------------------------------- operands

__device__ __forceinline__ uint32_t Bits(Half2 h) { return __builtin_bit_cast(uint32_t, h); }

__device__ __forceinline__ Half8 AsHalf8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const dev::U32x4 w = {a, b, c, d};
  return __builtin_bit_cast(Half8, w);
}

// ---------------------------------------------------------------- LDS

using Lds = __attribute__((address_space(3))) char;

// Loads straight to LDS are written out, and so are the waits for them: the compiler
// lets an LDS read wait for every such load before it, where the loop below needs it
// to wait for the older half of them. The waits count on the kernel's main loop to
// make no other vector memory access in between; any that the compiler does make
// (a piece's queries and outputs) only makes a wait longer.
using Resource = dev::U32x4;
__device__ __forceinline__ Resource RowsResource(const void* base, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  return Resource{static_cast<uint32_t>(at), static_cast<uint32_t>(at >> 32) & 0xFFFFu, bytes, 0x00020000u};
}
__device__ __forceinline__ uint32_t LdsAddress(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const Lds*)(static_cast<const char*>(p))));
}
// kN times 16 bytes a lane from rs: time i from byte off[i % kOff] + 1024 i, lane j's to LDS address `to` + 1024 i +
// 16 j (an instruction's offset counts on both sides). What is read once is loaded with the streaming hint: without it
// 32 x 4096 positions take 55.4 us and not 50.0, 128 x 8192 in 8 bits 214 and not 190. M0 holds the
// LDS address: an operand, so that the compiler writes it and knows what is there. It is read one wait state after it is
// written; five are waited, which M0 and a resource need where a vector instruction wrote them.
template <int kN, int kOff>
__device__ __forceinline__ void LoadToLds(Resource rs, const uint32_t (&off)[kOff], uint32_t to) {
  static_assert(kN == 1 || kN == 2 || kN == 4, "");
  if constexpr (kN == 1) {
    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
                 :
                 : "{m0}"(to), "v"(off[0]), "s"(rs)
                 : "memory");
  } else if constexpr (kN == 2) {
    asm volatile(
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %1, %3, 0 offen nt lds\n\t"
        "buffer_load_dwordx4 %2, %3, 0 offen offset:1024 nt lds"
        :
        : "{m0}"(to), "v"(off[0]), "v"(off[1 % kOff]), "s"(rs)
        : "memory");
  } else {
    asm volatile(
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %1, %5, 0 offen nt lds\n\t"
        "buffer_load_dwordx4 %2, %5, 0 offen offset:1024 nt lds\n\t"
        "buffer_load_dwordx4 %3, %5, 0 offen offset:2048 nt lds\n\t"
        "buffer_load_dwordx4 %4, %5, 0 offen offset:0xc00 nt lds"
        :
        : "{m0}"(to), "v"(off[0]), "v"(off[1 % kOff]), "v"(off[2 % kOff]), "v"(off[3 % kOff]), "s"(rs)
        : "memory");
  }
}
// 4 bytes a lane, from an address of its own.
__device__ __forceinline__ void LoadWordToLds(const float* from, uint32_t to) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %1, off" : : "{m0}"(to), "v"(from) : "memory");
}
// Waits until at most kLeft vector memory accesses are under way.
template <int kLeft>
__device__ __forceinline__ void WaitLoads() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLeft) : "memory");
}
// Waits for the LDS reads under way, before what they read is loaded over.
__device__ __forceinline__ void WaitLdsReads() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// A scalar load: p is the same in every lane, and what it points to does not change while the kernel runs.
template <class T>
__device__ __forceinline__ T ScalarLoad(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(p);
}

// Four halves, one of each of four rows: in each 16-lane group, lane j receives
// element j % 4 of the 8 bytes addressed by lanes j / 4, 4 + j / 4, ...
__device__ __forceinline__ uint2 ReadHalvesAcross(const char* at) {
  const S16x4 v =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S16x4*)(Lds*)(const_cast<char*>(at)));
  return __builtin_bit_cast(uint2, v);
}
// Eight bytes, one of each of eight rows: in each 16-lane group, lane j receives
// byte j % 8 of the 8 bytes addressed by lanes j / 8, 2 + j / 8, ...
__device__ __forceinline__ I32x2 ReadBytesAcross(const char* at) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) I32x2*)(Lds*)(const_cast<char*>(at)));
}

// ---------------------------------------------------------------- sharing out

__device__ __forceinline__ uint32_t Scalar(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// Everything here is the same in every lane of a wave, and kept in scalar registers.
struct Share {
  uint32_t per;  // a workgroup's items: per, and one more in the first `rem` of them
  uint32_t rem;

  __device__ __forceinline__ Share(uint32_t items, uint32_t groups) {
    per = Scalar(items / groups);
    rem = items - per * groups;
  }
  __device__ __forceinline__ uint32_t Begin(uint32_t w) const { return w * per + min(w, rem); }
  // The workgroup whose share holds item x.
  __device__ __forceinline__ uint32_t Holder(uint32_t x) const {
    return Scalar(HolderOfLane(x));
  }
  __device__ __forceinline__ uint32_t HolderOfLane(uint32_t x) const {
    const uint32_t big = rem * (per + 1);
    return x < big ? x / (per + 1) : rem + (x - big) / per;
  }
};

// Sum of x over the lanes up to and with this one.
__device__ __forceinline__ uint32_t ScanAdd(uint32_t x) {
  int v = static_cast<int>(x);
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8: within rows of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // lane 15's into row 1, lane 47's into row 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31's into rows 2 and 3
  return static_cast<uint32_t>(v);
}

// Counts in at a counter; whether that was the last of `all`, which leaves the counter ready for the next call.
__device__ __forceinline__ int Count(char* workspace, uint32_t counter, uint32_t all) {
  uint32_t* at = reinterpret_cast<uint32_t*>(workspace) + counter;
  const bool last = __hip_atomic_fetch_add(at, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
  if (last) __hip_atomic_store(at, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return last ? 1 : 0;
}

}  // namespace attn
}  // namespace rpg

#endif  // RPG_AMD_ATTENTION_DEV_H_
