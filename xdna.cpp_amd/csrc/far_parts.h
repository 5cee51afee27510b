// Results that travel between the workgroups of one launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.h"

namespace mi355x {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_a __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_a __attribute__((ext_vector_type(4)));

// Parts of a row's sums that travel between workgroups of one launch, whose dies'
// L2s do not see each other: stored and read past them, so that no L2 has to be
// written back or emptied (fences that do so made 64 ragged requests 454 us
// instead of 196).  A workgroup that has waited for its stores and met a barrier
// may then count itself in.
constexpr int kPastL2 = 16;  // the sc1 bit of a buffer operation
struct FarParts {
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ explicit FarParts(float *base)
        : rsrc(__builtin_amdgcn_make_buffer_rsrc(base, 0, 0xFFFFFFFFu, kBufferWord3)) {}
    __device__ __forceinline__ void store(int at, float v) const {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), rsrc, 4 * at, 0, kPastL2);
    }
    __device__ __forceinline__ void store4(int at, f32x4 v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_a, v), rsrc, 4 * at, 0, kPastL2);
    }
    __device__ __forceinline__ void store2(int at, u32x2_a v) const {
        __builtin_amdgcn_raw_buffer_store_b64(v, rsrc, 4 * at, 0, kPastL2);
    }
    __device__ __forceinline__ u32x2_a load2(int at) const {
        return __builtin_bit_cast(u32x2_a, __builtin_amdgcn_raw_buffer_load_b64(rsrc, 4 * at, 0, kPastL2));
    }
    __device__ __forceinline__ float load(int at) const {
        return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, 4 * at, 0, kPastL2));
    }
    __device__ __forceinline__ f32x4 load4(int at) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, 4 * at, 0, kPastL2));
    }
};
// Counts this workgroup in at *counter, which `n` of them do; true for the last
// one, which finds the others' parts complete and leaves the counter at 0.
// Called by all threads; `flag` is LDS.
__device__ __forceinline__ bool last_of(int *counter, int n, int *flag) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wavefront's stores
    __syncthreads();
    if (threadIdx.x == 0) {
        const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (before == n - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = before == n - 1;
    }
    __syncthreads();
    return *flag != 0;
}

}  // namespace mi355x
