// lds_copy.hpp — copies from global memory straight into LDS (decode3.hpp,
// prefill_stage.hpp), the waits that go with them, and pairs of bf16.
#pragma once

#include "tq_common.hpp"

namespace tq {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    v2bf v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}

typedef __attribute__((address_space(3))) unsigned char lds_u8;

// 16 bytes from each lane's global address into LDS at dst + 16*lane
// (global_load_lds_dwordx4; M0 holds the LDS byte address and is restored; a
// scalar write of M0 needs one wait state before the copy, the s_nop).
// Issued as inline assembly so that the compiler does not follow every such
// copy with a full vmcnt(0) wait before LDS accesses: the kernel waits for
// exactly the copies it needs (wait_vm), counting them in issue order.
// No memory clobber: LDS reads of a slot are ordered before a refill by
// wait_lds() (a compiler barrier plus lgkmcnt(0)) and after its copies by
// wait_vm(); leaving memory unclobbered keeps the uniform loads that
// precede the copies scalar.
__device__ __forceinline__ void dma16(const void *src, unsigned char *dst) {
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_u8 *)dst;
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(src), "s"(lds));
}
// The same copy from a scalar base address plus each lane's 32-bit offset
// (the saddr form): a uniform base costs no vector address arithmetic.
__device__ __forceinline__ void dma16s(const unsigned char *base, uint32_t off, unsigned char *dst) {
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_u8 *)dst;
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(off), "s"(base), "s"(lds));
}
// 4 bytes per lane, the same way (into LDS at dst + 4*lane).
__device__ __forceinline__ void dma4s(const unsigned char *base, uint32_t off, unsigned char *dst) {
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_u8 *)dst;
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"
        "global_load_lds_dword %1, %2\n\ts_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(off), "s"(base), "s"(lds));
}
// Wait until at most N vector memory operations of this wave are outstanding (the copies
// above are counted in issue order).
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt immediate");
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// Every LDS access issued so far has completed (before a copy may land on
// memory those accesses touch).
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

}  // namespace tq
