// What the products on token rows have in common: requests that fill LDS past the registers, the waits for them, and the activation as
// a constant of an epilogue.
#pragma once
#include "elements.hpp"

namespace tsx {

#ifdef __HIPCC__

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// 64 lanes x 16 bytes, from an address for each lane to consecutive bytes of LDS.  Complete when vmcnt says so.
__device__ __forceinline__ void to_lds(const int8_t *at, int8_t *lds) {
    __builtin_amdgcn_global_load_lds((global_void *)at, (lds_void *)lds, 16, 0, 0);
}

// f(the activation as a constant): one branch around all of a wavefront's values
template <class F>
__device__ __forceinline__ void by_act(int act, F &&f) {
    switch (act) {
        case TSX_ACT_RELU: f(std::integral_constant<int, TSX_ACT_RELU>{}); break;
        case TSX_ACT_LEAKY_RELU: f(std::integral_constant<int, TSX_ACT_LEAKY_RELU>{}); break;
        case TSX_ACT_MISH_FAST: f(std::integral_constant<int, TSX_ACT_MISH_FAST>{}); break;
        case TSX_ACT_SILU: f(std::integral_constant<int, TSX_ACT_SILU>{}); break;
        default: f(std::integral_constant<int, TSX_ACT_NONE>{}); break;
    }
}

// LDS is this workgroup's own: what was read from it is read, and what the wavefronts wrote is there, behind the barrier.  Requests to
// memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
template <int N>
__device__ __forceinline__ void wait_for_all_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

#endif  // __HIPCC__

}  // namespace tsx
