// Rows of f32, f16 or bf16 values, read and written eight at a time at any
// alignment of their type, and reductions of 64-bit values over a workgroup.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "device_common.h"
#include "mi355x-attention.h"

namespace mi355x {

template <int TYPE>
struct RowElem;
template <>
struct RowElem<MI355X_TYPE_F32> {
    typedef float T;
    typedef float Raw8 __attribute__((ext_vector_type(8), aligned(4)));
};
template <>
struct RowElem<MI355X_TYPE_F16> {
    typedef _Float16 T;
    typedef _Float16 Raw8 __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct RowElem<MI355X_TYPE_BF16> {
    typedef __bf16 T;
    typedef __bf16 Raw8 __attribute__((ext_vector_type(8), aligned(2)));
};

// Values i .. i + 7 of a row of n, zeros behind its end.
template <int TYPE>
__device__ __forceinline__ typename RowElem<TYPE>::Raw8 row_load8(const void *row, int i, int n) {
    typedef typename RowElem<TYPE>::T T;
    typedef typename RowElem<TYPE>::Raw8 R;
    const T *p = static_cast<const T *>(row) + i;
    R r = {};
    if (i + 8 <= n) {
        r = *reinterpret_cast<const R *>(p);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j < n) r[j] = p[j];
    }
    return r;
}

// Values 1 .. 7 of eight, and a zero.
template <class R>
__device__ __forceinline__ R shifted(R r) {
    return __builtin_shufflevector(r, R{}, 1, 2, 3, 4, 5, 6, 7, 8);
}

// The same without a branch, of a row of 8 or more: a run that the row ends in is taken from
// the row's last eight, as row_end then has to put right.
template <int TYPE>
__device__ __forceinline__ typename RowElem<TYPE>::Raw8 row_load8_near(const void *row, int i, int n) {
    typedef typename RowElem<TYPE>::T T;
    return *reinterpret_cast<const typename RowElem<TYPE>::Raw8 *>(static_cast<const T *>(row) + min(i, n - 8));
}
template <int TYPE>
__device__ __forceinline__ void row_end(typename RowElem<TYPE>::Raw8 &r, int i, int n) {
#pragma unroll 1
    for (int k = min(i + 8 - n, 8); k > 0; --k) r = shifted(r);
}

// (The tail's loops are not unrolled: their conditions would take a kernel's scalar registers.)
template <int TYPE>
__device__ __forceinline__ void row_store8(void *row, int i, int n, typename RowElem<TYPE>::Raw8 r) {
    typedef typename RowElem<TYPE>::T T;
    typedef typename RowElem<TYPE>::Raw8 R;
    T *p = static_cast<T *>(row) + i;
    if (i + 8 <= n) {
        *reinterpret_cast<R *>(p) = r;
    } else {
#pragma unroll 1
        for (int j = 0; i + j < n; ++j, r = shifted(r)) p[j] = r[0];
    }
}

// Eight codes, a byte each, to codes i .. i + 7 of a row of n.
__device__ __forceinline__ void row_store_codes(int8_t *row, int i, int n, uint64_t codes) {
    typedef uint64_t U8 __attribute__((aligned(1)));
    int8_t *p = row + i;
    if (i + 8 <= n) {
        *reinterpret_cast<U8 *>(p) = codes;
    } else {
#pragma unroll 1
        for (int j = 0; i + j < n; ++j, codes >>= 8) p[j] = static_cast<int8_t>(codes);
    }
}

// The other lane's 64-bit value of a DPP move (0 where no lane is read).
template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ double dpp_mov64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROW_MASK, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROW_MASK, 0xF, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ __forceinline__ double last_lane64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), 63);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), 63);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Sum, and largest of values that are not negative, over a wavefront whose lanes
// are all active; the same in every lane.
__device__ __forceinline__ double wave_sum64(double v) {
    v += dpp_mov64<0xB1>(v);        // quad_perm [1,0,3,2]
    v += dpp_mov64<0x4E>(v);        // quad_perm [2,3,0,1]
    v += dpp_mov64<0x141>(v);       // row_half_mirror
    v += dpp_mov64<0x140>(v);       // row_mirror
    v += dpp_mov64<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
    v += dpp_mov64<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
    return last_lane64(v);
}
__device__ __forceinline__ double wave_max64(double v) {
    v = fmax(v, dpp_mov64<0xB1>(v));
    v = fmax(v, dpp_mov64<0x4E>(v));
    v = fmax(v, dpp_mov64<0x141>(v));
    v = fmax(v, dpp_mov64<0x140>(v));
    v = fmax(v, dpp_mov64<0x142, 0xA>(v));
    v = fmax(v, dpp_mov64<0x143, 0xC>(v));
    return last_lane64(v);
}

// Largest over a wavefront whose lanes are all active (NaN does not count); the same in
// every lane.
__device__ __forceinline__ float wave_max(float v) {
    // lanes that no move writes read -inf: the identity
    const int none = __builtin_bit_cast(int, -INFINITY);
    auto mov = [&](auto ctrl, auto mask) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(none, __builtin_bit_cast(int, v), decltype(ctrl)::value,
                                                                     decltype(mask)::value, 0xF, false));
    };
    typedef std::integral_constant<int, 0xF> All;
    v = fmaxf(v, mov(std::integral_constant<int, 0xB1>{}, All{}));
    v = fmaxf(v, mov(std::integral_constant<int, 0x4E>{}, All{}));
    v = fmaxf(v, mov(std::integral_constant<int, 0x141>{}, All{}));
    v = fmaxf(v, mov(std::integral_constant<int, 0x140>{}, All{}));
    v = fmaxf(v, mov(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{}));
    v = fmaxf(v, mov(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{}));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

}  // namespace mi355x
