// Pieces shared by the matrix-core attention and product kernels: operand vector
// types, a compile-time loop, LDS reads that the compiler does not order after
// direct-to-LDS loads, and such loads that it does not know of.
#pragma once

#include <type_traits>
#include <utility>

#include "common.h"

namespace evo2 {

typedef __attribute__((ext_vector_type(8))) __bf16 abf16x8_t;
typedef __attribute__((ext_vector_type(4))) float af32x4_t;
typedef __attribute__((ext_vector_type(4))) unsigned int au32x4_t;
typedef __attribute__((address_space(3))) void alds_void;

// f(integral_constant<int, 0>) .. f(integral_constant<int, N - 1>): the
// index is a constant expression inside f.
template <typename F, int... I>
__device__ __forceinline__ void static_for_seq(F &f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F &&f) {
  static_for_seq(f, std::make_integer_sequence<int, N>{});
}

// Eight 16-byte LDS reads at byte address a + STRIDE j, then a wait for them.
// Inline assembly: the compiler would otherwise wait for every direct-to-LDS
// load in flight before any LDS read; the caller waits for the ones it reads.
template <int STRIDE>
__device__ __forceinline__ void lds_read8(au32x4_t (&r)[8], uint32_t a) {
  static_assert(STRIDE > 0 && 7 * STRIDE < 65536, "ds_read offsets are 16 bits");
  asm volatile(
      "ds_read_b128 %0, %8\n"
      "ds_read_b128 %1, %8 offset:%9\n"
      "ds_read_b128 %2, %8 offset:%10\n"
      "ds_read_b128 %3, %8 offset:%11\n"
      "ds_read_b128 %4, %8 offset:%12\n"
      "ds_read_b128 %5, %8 offset:%13\n"
      "ds_read_b128 %6, %8 offset:%14\n"
      "ds_read_b128 %7, %8 offset:%15\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]),
        "=&v"(r[7])
      : "v"(a), "i"(STRIDE), "i"(2 * STRIDE), "i"(3 * STRIDE), "i"(4 * STRIDE), "i"(5 * STRIDE),
        "i"(6 * STRIDE), "i"(7 * STRIDE)
      : "memory");
}

// Four 16-byte LDS reads at byte address a + STRIDE j, then a wait for them.
template <int STRIDE>
__device__ __forceinline__ void lds_read4(au32x4_t (&r)[4], uint32_t a) {
  static_assert(STRIDE > 0 && 3 * STRIDE < 65536, "ds_read offsets are 16 bits");
  asm volatile(
      "ds_read_b128 %0, %4\n"
      "ds_read_b128 %1, %4 offset:%5\n"
      "ds_read_b128 %2, %4 offset:%6\n"
      "ds_read_b128 %3, %4 offset:%7\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
      : "v"(a), "i"(STRIDE), "i"(2 * STRIDE), "i"(3 * STRIDE)
      : "memory");
}

// LDS byte address of a pointer into a __shared__ array.
__device__ __forceinline__ uint32_t lds_addr(const void *p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p));
}

// A raw buffer descriptor over `bytes` bytes from p.
__device__ __forceinline__ au32x4_t lds_rsrc(const void *p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  // (uniform values; stated, for an operand that has to be in SGPRs)
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
  return au32x4_t{lo, hi & 0xffffu, static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(bytes)), 0x00020000u};
}

// (m0, a reserved register, is named as clobbered below)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"

// One direct-to-LDS load: 64 lanes x 16 bytes at byte offset v (zeros past the
// descriptor) to lds .. lds + 1 KB.  In asm so that the compiler does not know of it:
// before each transposing LDS read it would wait for all such loads in flight.  The
// kernel waits for them itself (lds_sync), and no register is written.  The wait states
// that the compiler would put before the load stand in the asm: one after the write of m0,
// and five after a vector instruction that wrote part of the descriptor (lds_rsrc's
// readfirstlane, or the reload of a spilled register, wherever those land), which the
// hardware does not interlock: the load would go by the old word.  (Two loads to an asm
// block, with the wait states once, were no faster: gated step of 8192 rows 3904 and 3915 us,
// loss of 131072 columns 13.9 ms both.)
__device__ __forceinline__ void lds_load(au32x4_t rsrc, uint32_t v, const bf16_t *lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds_addr(lds)), "v"(v), "s"(rsrc)
               : "m0");
}

// The same, 64 lanes x 4 bytes.
__device__ __forceinline__ void lds_load4(au32x4_t rsrc, uint32_t v, const void *lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds_addr(lds)), "v"(v), "s"(rsrc)
               : "m0");
}

#pragma clang diagnostic pop

// All but N of the wave's loads and stores and all its LDS reads are done; then the
// workgroup meets, and LDS holds what every wave's loads brought.
template <int N>
__device__ __forceinline__ void lds_sync() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

}  // namespace evo2
