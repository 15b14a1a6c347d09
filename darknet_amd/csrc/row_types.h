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

/* Reductions and running sums over the 64 lanes by data-parallel-primitive moves between registers (rows of 16
 * lanes, then row 0 to 1 and 2 to 3, then the lower half to the upper), which wait for no LDS as shuffles do.  All 64 lanes must be active.  Lanes without a source take `none`. */
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dn_move(unsigned none, unsigned v)
{
    return (unsigned)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long dn_move(unsigned long long none, unsigned long long v)
{
    const unsigned lo = dn_move<CTRL, ROWS>((unsigned)none, (unsigned)v);
    const unsigned hi = dn_move<CTRL, ROWS>((unsigned)(none >> 32), (unsigned)(v >> 32));
    return (unsigned long long)hi << 32 | lo;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dn_move(double none, double v)
{
    return __longlong_as_double((long long)dn_move<CTRL, ROWS>((unsigned long long)__double_as_longlong(none),
                                                              (unsigned long long)__double_as_longlong(v)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dn_move(float none, float v)
{
    return __uint_as_float(dn_move<CTRL, ROWS>(__float_as_uint(none), __float_as_uint(v)));
}

/* The running result of op in lane order, from lane 0 to each lane. */
template <class T, class Op>
__device__ __forceinline__ T dn_wave_scan(T v, T none, Op op)
{
    v = op(v, dn_move<0x111, 0xf>(none, v));
    v = op(v, dn_move<0x112, 0xf>(none, v));
    v = op(v, dn_move<0x114, 0xf>(none, v));
    v = op(v, dn_move<0x118, 0xf>(none, v));
    v = op(v, dn_move<0x142, 0xa>(none, v));
    v = op(v, dn_move<0x143, 0xc>(none, v));
    return v;
}

__device__ __forceinline__ unsigned dn_lane(unsigned v, int lane) { return (unsigned)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ unsigned long long dn_lane(unsigned long long v, int lane)
{
    return (unsigned long long)dn_lane((unsigned)(v >> 32), lane) << 32 | dn_lane((unsigned)v, lane);
}
__device__ __forceinline__ double dn_lane(double v, int lane)
{
    return __longlong_as_double((long long)dn_lane((unsigned long long)__double_as_longlong(v), lane));
}
__device__ __forceinline__ float dn_lane(float v, int lane) { return __uint_as_float(dn_lane(__float_as_uint(v), lane)); }

template <class T>
__device__ __forceinline__ T dn_wave_sum(T v)
{
    return dn_lane(dn_wave_scan(v, (T)0, [](T a, T b) { return a + b; }), 63);
}
__device__ __forceinline__ double dn_wave_max(double v)
{
    return dn_lane(dn_wave_scan(v, v, [](double a, double b) { return fmax(a, b); }), 63);
}
__device__ __forceinline__ float dn_wave_max(float v)
{
    return dn_lane(dn_wave_scan(v, v, [](float a, float b) { return fmaxf(a, b); }), 63);
}
__device__ __forceinline__ unsigned dn_wave_max(unsigned v)
{
    return dn_lane(dn_wave_scan(v, v, [](unsigned a, unsigned b) { return a > b ? a : b; }), 63);
}
__device__ __forceinline__ unsigned long long dn_wave_max(unsigned long long v)
{
    typedef unsigned long long u64;
    return dn_lane(dn_wave_scan(v, v, [](u64 a, u64 b) { return a > b ? a : b; }), 63);
}

#endif
