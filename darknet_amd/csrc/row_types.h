/*
 * row_types.h - what the row operators (norm.hip, q4.hip, sample.hip) share: element types, their
 * loads and stores as float, reductions over a wavefront, and how a call is refused.
 */
#ifndef DN_ROW_TYPES_H
#define DN_ROW_TYPES_H

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "hip.h"

static inline hipStream_t dn_stream() { return (hipStream_t)hip_get_stream(); }

/* A call that the kernels cannot honour: a message, and -1 to the caller; nothing has been launched. */
static inline int dn_refuse(const char *call, const char *why)
{
    fprintf(stderr, "%s: %s\n", call, why);
    return -1;
}

/* Storage of an element type and its conversions; stores round to nearest even. */
template <int T> struct dn_elt;
template <> struct dn_elt<DN_F32> { typedef float store; };
template <> struct dn_elt<DN_F16> { typedef _Float16 store; };
template <> struct dn_elt<DN_BF16> { typedef __bf16 store; };
template <> struct dn_elt<DN_I8> { typedef signed char store; };

static inline int dn_type_bytes(int type) { return type == DN_F32 ? 4 : type == DN_I8 ? 1 : 2; }
static inline bool dn_is_float_type(int type) { return type == DN_F32 || type == DN_F16 || type == DN_BF16; }
static inline bool dn_aligned(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

__device__ __forceinline__ double dn_wave_sum(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ double dn_wave_max(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
    return v;
}

__device__ __forceinline__ float dn_wave_max(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

__device__ __forceinline__ unsigned long long dn_wave_sum(unsigned long long v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

#endif
