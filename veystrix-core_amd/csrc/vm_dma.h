// Tiles staged in LDS by DMA (global_load_lds_dwordx4: no registers held) as rows of 128 bytes, eight 16-byte units
// each, and read back as MFMA operands.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace vm {

constexpr uint32_t kChunk = 128;          // bytes of a row per step

// Unit u of row r lies at unit u ^ swz(r) of its 128 bytes: an operand read (lane: row lane % 16, unit lane / 16 or
// 4 + lane / 16) then spreads over all 64 banks in every lane grouping of the read.
__device__ __forceinline__ uint32_t tile_swz(uint32_t r) { return ((r >> 1) & 2u) | ((r << 1) & 4u); }

// One kilobyte from the lanes' addresses to LDS, lane j's 16 bytes at dst + 16 j; dst is the same in all lanes.  ONCE:
// non-temporal, for data that is read once.
template <bool ONCE = false>
__device__ __forceinline__ void load_to_lds(const void* src, uint8_t* dst) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 16, 0, ONCE ? 2 : 0);
}

// s_waitcnt for a vector memory count of N, or the LDS count at zero, the others left alone
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt is six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4)); }

template <int J, int N, class F>
__device__ __forceinline__ void unroll(F&& f) {
  if constexpr (J < N) {
    f(std::integral_constant<int, J>{});
    unroll<J + 1, N>(f);
  }
}

// A block barrier that no memory access is moved across and that waits for none by itself.
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace vm
