// Eight neighbouring elements of a row in float registers: the unit of the row kernels of
// rowwise.hpp.  float and bfloat16 rows of any alignment and width: a chunk that lies inside the row is
// moved by 16-byte accesses (global memory takes them at any element's address), the one that
// the row's end cuts element by element.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bf {

using bf16 = __bf16;

typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

// (round to nearest even, NaN stays NaN: v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    const floatx2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return (float)v; }

// (vectors at an element's alignment)
typedef float quad_at_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t quad_at_2 __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ void load8_whole(const float *p, float (&v)[8])
{
    const quad_at_4 a = *reinterpret_cast<const quad_at_4 *>(p), b = *reinterpret_cast<const quad_at_4 *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ void store8_whole(float *p, const float (&v)[8])
{
    const quad_at_4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
    *reinterpret_cast<quad_at_4 *>(p) = a;
    *reinterpret_cast<quad_at_4 *>(p + 4) = b;
}
__device__ __forceinline__ void load8_whole(const bf16 *p, float (&v)[8])
{
    const quad_at_2 a = *reinterpret_cast<const quad_at_2 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __builtin_bit_cast(float, a[i] << 16);
        v[2 * i + 1] = __builtin_bit_cast(float, a[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store8_whole(bf16 *p, const float (&v)[8])
{
    const quad_at_2 a = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    *reinterpret_cast<quad_at_2 *>(p) = a;
}

// Elements col .. col + 7 of a row of `cols`; those past its end are `fill`.
template <typename T>
__device__ __forceinline__ void load8(const T *row, int col, int cols, float fill, float (&v)[8])
{
    if (col + 8 <= cols) {
        load8_whole(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? to_float(row[col + i]) : fill;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *row, int col, int cols, const float (&v)[8])
{
    if (col + 8 <= cols) {
        store8_whole(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < cols) row[col + i] = (T)v[i];
    }
}

// Sum over L neighbouring lanes (L a power of two, at most 64), the same in each of them.
template <int L>
__device__ __forceinline__ float lanes_sum(float v)
{
#pragma unroll
    for (int d = 1; d < L; d *= 2) v += __shfl_xor(v, d, 64);
    return v;
}

}  // namespace bf
