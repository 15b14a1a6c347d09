/*
 * q4.hip - products with 4-bit weights: a connected layer whose weights are held as
 *
 *   w[o][k] = (code[o][k] - zero[o][k / G]) * scale[o][k / G],   code and zero 0 .. 15, G = 32, 64 or 128
 *   output[b][o] = activation(bias[o] + sum_k x[b][k] * w[o][k])
 *
 * Packed weights, written once when they are loaded: tiles of 16 outputs x 128 inputs, a kilobyte each, in
 * the order [outputs / 16][inputs / 128][lane 0..63][4 dwords], so that a wave reads a tile with one 16-byte load
 * a lane.  Dword s of lane r + 16*j holds output r, inputs 32*s + 8*j + i (i = 0..7), which is what that lane
 * gives to the matrix instruction of 16 x 16 x 32; input i stands in the four bits from
 * 4 * (i / 2) + 16 * (i % 2) on, so that a mask leaves two neighbours in the two halves of a register.
 * Behind the codes the scales, [outputs / 16][inputs / 128][16][groups in 128] floats, and the zeros, the same in
 * bytes.  What fills the last tiles up has code, scale and zero 0.
 */
#include <math.h>

#include "device_math.h"
#include "row_types.h"

struct q4_shape {
    int inputs, outputs, group;
    int kblocks, tiles, groups; /* groups of the filled-up length */
    long scales_at, zeros_at;   /* byte offsets of the two tables */
};

static q4_shape q4_shape_of(int inputs, int outputs, int group)
{
    q4_shape s;
    s.inputs = inputs;
    s.outputs = outputs;
    s.group = group;
    s.kblocks = (int)(((long)inputs + 127) / 128);
    s.tiles = (int)(((long)outputs + 15) / 16);
    s.groups = s.kblocks * (128 / group);
    s.scales_at = (long)s.tiles * s.kblocks * 1024;
    s.zeros_at = s.scales_at + (long)s.tiles * s.groups * 64;
    return s;
}

static bool q4_shape_ok(int inputs, int outputs, int group)
{
    /* what is below 2^31 by more than a launch's stride: loops and filled-up tiles stay within an int */
    return inputs >= 1 && outputs >= 1 && inputs <= 0x7fff0000 && outputs <= 0x7fff0000 && (group == 32 || group == 64 || group == 128);
}

extern "C" size_t q4_packed_bytes(int inputs, int outputs, int group)
{
    if (!q4_shape_ok(inputs, outputs, group)) return 0;
    const q4_shape s = q4_shape_of(inputs, outputs, group);
    return (size_t)s.zeros_at + (size_t)s.tiles * s.groups * 16;
}

__device__ __forceinline__ long q4_dword_at(const q4_shape &s, int o, int k)
{
    return (((long)(o >> 4) * s.kblocks + (k >> 7)) * 64 + (o & 15) + ((k >> 3) & 3) * 16) * 4 + ((k >> 5) & 3);
}
__device__ __forceinline__ int q4_bit_of(int k) { return ((k & 6) << 1) + ((k & 1) << 4); }
__device__ __forceinline__ long q4_group_at(const q4_shape &s, int o, int g)
{
    const int per = 128 / s.group;
    return (((long)(o >> 4) * s.kblocks + g / per) * 16 + (o & 15)) * per + g % per;
}

/* One thread for each (output, 32 inputs) of the filled-up matrix: its four dwords are written by it alone. */
__global__ void q4_pack_codes_kernel(const unsigned char *codes, const float *scales, const unsigned char *zeros,
                                     unsigned char *packed, q4_shape s)
{
    const long chunks = (long)s.kblocks * 4, total = (long)s.tiles * 16 * chunks;
    const int groups = (s.inputs + s.group - 1) / s.group;
    const long row_bytes = ((long)s.inputs + 1) / 2;
    for (long t = blockIdx.x * (long)blockDim.x + threadIdx.x; t < total; t += (long)gridDim.x * blockDim.x) {
        const int o = (int)(t / chunks), k0 = (int)(t % chunks) * 32;
        for (int j = 0; j < 4; ++j) {
            unsigned v = 0;
            for (int i = 0; i < 8; ++i) {
                const int k = k0 + j * 8 + i;
                if (o < s.outputs && k < s.inputs)
                    v |= (unsigned)((codes[o * row_bytes + (k >> 1)] >> ((k & 1) * 4)) & 15) << q4_bit_of(k);
            }
            ((unsigned *)packed)[q4_dword_at(s, o, k0 + j * 8)] = v;
        }
        if (k0 % s.group == 0) {
            const int g = k0 / s.group;
            const bool in = o < s.outputs && g < groups;
            ((float *)(packed + s.scales_at))[q4_group_at(s, o, g)] = in ? scales[(long)o * groups + g] : 0.f;
            packed[s.zeros_at + q4_group_at(s, o, g)] = in ? (zeros ? zeros[(long)o * groups + g] & 15 : 8) : 0;
        }
    }
}

/* Quantises as it packs, one thread for each (output, group): the range of the group, widened to hold
 * zero, in 15 steps. */
__global__ void q4_pack_weights_kernel(const float *weights, unsigned char *packed, q4_shape s)
{
    const long total = (long)s.tiles * 16 * s.groups;
    for (long t = blockIdx.x * (long)blockDim.x + threadIdx.x; t < total; t += (long)gridDim.x * blockDim.x) {
        const int o = (int)(t / s.groups), g = (int)(t % s.groups), lo_k = g * s.group;
        const int n = o < s.outputs ? min(s.group, s.inputs - lo_k) : 0;
        const float *w = weights + (long)o * s.inputs + lo_k;
        float lo = 0, hi = 0;
        for (int i = 0; i < n; ++i) {
            lo = fminf(lo, w[i]);
            hi = fmaxf(hi, w[i]);
        }
        const float scale = (float)(((double)hi - (double)lo) / 15);
        const double zero = scale > 0 ? fmin(rint(-(double)lo / scale), 15.) : 0;
        for (int j = 0; j < s.group / 8; ++j) {
            unsigned v = 0;
            for (int i = 0; i < 8; ++i) {
                const int at = j * 8 + i;
                if (at < n && scale > 0)
                    v |= (unsigned)fmin(fmax(rint((double)w[at] / scale) + zero, 0.), 15.) << q4_bit_of(at);
            }
            ((unsigned *)packed)[q4_dword_at(s, o, lo_k + j * 8)] = v;
        }
        ((float *)(packed + s.scales_at))[q4_group_at(s, o, g)] = scale;
        packed[s.zeros_at + q4_group_at(s, o, g)] = (unsigned char)zero;
    }
}

__global__ void q4_unpack_kernel(const unsigned char *packed, float *weights, q4_shape s)
{
    const long total = (long)s.outputs * s.inputs;
    for (long t = blockIdx.x * (long)blockDim.x + threadIdx.x; t < total; t += (long)gridDim.x * blockDim.x) {
        const int o = (int)(t / s.inputs), k = (int)(t % s.inputs);
        const long at = q4_group_at(s, o, k / s.group);
        const int code = (((const unsigned *)packed)[q4_dword_at(s, o, k)] >> q4_bit_of(k)) & 15;
        weights[t] = (float)(code - (int)packed[s.zeros_at + at]) * ((const float *)(packed + s.scales_at))[at];
    }
}

static dim3 q4_grid(long threads)
{
    const long b = (threads + 255) / 256;
    return dim3((unsigned)(b < 8192 ? b : 8192));
}

extern "C" int q4_pack_codes_gpu(const unsigned char *codes, const float *scales, const unsigned char *zeros,
                                 void *packed, int inputs, int outputs, int group)
{
    const char *me = "q4_pack_codes_gpu";
    if (!q4_shape_ok(inputs, outputs, group)) return dn_refuse(me, "bad geometry (group must be 32, 64 or 128)");
    if (!codes || !scales || !packed) return dn_refuse(me, "a buffer is missing");
    if (!dn_aligned(packed, 16) || !dn_aligned(scales, 4)) return dn_refuse(me, "packed must be aligned to 16 bytes, scales to 4");
    hip_require_device(me);
    const q4_shape s = q4_shape_of(inputs, outputs, group);
    hipLaunchKernelGGL(q4_pack_codes_kernel, q4_grid((long)s.tiles * 16 * s.kblocks * 4), dim3(256), 0, dn_stream(),
                       codes, scales, zeros, (unsigned char *)packed, s);
    dn_check_launch(me);
    return 0;
}

extern "C" int q4_pack_weights_gpu(const float *weights, void *packed, int inputs, int outputs, int group)
{
    const char *me = "q4_pack_weights_gpu";
    if (!q4_shape_ok(inputs, outputs, group)) return dn_refuse(me, "bad geometry (group must be 32, 64 or 128)");
    if (!weights || !packed) return dn_refuse(me, "a buffer is missing");
    if (!dn_aligned(packed, 16) || !dn_aligned(weights, 4)) return dn_refuse(me, "packed must be aligned to 16 bytes, weights to 4");
    hip_require_device(me);
    const q4_shape s = q4_shape_of(inputs, outputs, group);
    hipLaunchKernelGGL(q4_pack_weights_kernel, q4_grid((long)s.tiles * 16 * s.groups), dim3(256), 0, dn_stream(),
                       weights, (unsigned char *)packed, s);
    dn_check_launch(me);
    return 0;
}

extern "C" int q4_unpack_weights_gpu(const void *packed, float *weights, int inputs, int outputs, int group)
{
    const char *me = "q4_unpack_weights_gpu";
    if (!q4_shape_ok(inputs, outputs, group)) return dn_refuse(me, "bad geometry (group must be 32, 64 or 128)");
    if (!weights || !packed) return dn_refuse(me, "a buffer is missing");
    if (!dn_aligned(packed, 16) || !dn_aligned(weights, 4)) return dn_refuse(me, "packed must be aligned to 16 bytes, weights to 4");
    hip_require_device(me);
    const q4_shape s = q4_shape_of(inputs, outputs, group);
    hipLaunchKernelGGL(q4_unpack_kernel, q4_grid((long)outputs * inputs), dim3(256), 0, dn_stream(),
                       (const unsigned char *)packed, weights, s);
    dn_check_launch(me);
    return 0;
}

/* ---- the product --------------------------------------------------------------------------------------
 * On the fp16 matrix instruction: code - zero is a whole number of at most 15, exact in fp16.  8-bit and fp16 input is
 * exact there.  fp32 and bf16 input is scaled by a power of two that brings the largest value (of the row, or of 128
 * inputs) to 2^14 .. 2^15, and held as one fp16 value (bf16: exact from 2^-31 of the largest up) or as two, of which the
 * second is the 2^12-fold of what the first leaves (fp32: to 2^-23 of each value from 2^-28 of the largest up; the weights
 * that the second meets are 2^-12 times the others).  Where values lie further apart some are left out there (the scale of a
 * row is then the one under which most are held); each eight inputs that have such values are marked, and their products
 * are added to the output at the end, one by one: an ordinary row has hardly any, but an output whose weights avoid the
 * large inputs would miss the small ones.  Products are exact in the fp32 accumulators, which
 * a group starts from zero; its sum is then multiplied with the scale and added to the output's, the factors of the input
 * last: a factor times a scale may be below the normal range where the output is not.  Where a value is not finite the
 * factor that undoes the scaling is NaN.
 *
 * The input is the instruction's first operand and the weights the second, so that a lane's results are those
 * of one output, whose scale and zero it has read beside the codes.
 *
 * What bounds it: the weights are read once, half a byte each, and up to some 64 rows nothing else takes as long.  The
 * products take a quarter of that at 16 rows; unpacking (9 vector instructions for 8 codes of a lane) is shared
 * by all rows of a workgroup.  So each form below is built around loads that stay in flight. */
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef unsigned uint4_t __attribute__((ext_vector_type(4)));

#define Q4_THREADS 512 /* 8 waves */
#define Q4_WAVES 8

struct q4_args {
    const void *input;
    const float *input_scales;
    const unsigned char *packed;
    const float *biases;
    void *output;
    unsigned char *workspace;
    int output_type;
    bool ranged;        /* input whose values may be too far apart for the pieces */
    int batch, x_group; /* x_group: 0, or the inputs that share one of input_scales */
    int activation;
    int ksplit; /* direct form: waves of a workgroup that share a row tile, each taking a part of the inputs */
    int run;    /* stream form: blocks of the inputs that a workgroup has */
    q4_shape s;
};

/* Input types whose values may be too far apart for the pieces, and what these take: absolute values (as bits) from `least`
 * on and below `most`.  What is below would be subnormal in the first piece (fp32; the matrix instruction aligns its
 * addends by their exponents, and takes that of a subnormal factor as 2^-14), or lose bits (bf16). */
template <int TI>
struct q4_range {
    static constexpr bool wide = TI == DN_F32 || TI == DN_BF16;
    static constexpr int exponents = TI == DN_F32 ? 29 : 32;
    unsigned least, most;
    __device__ q4_range(float factor) : least(__float_as_uint((TI == DN_F32 ? 0x1p-14f : 0x1p-17f) * factor)), most(__float_as_uint(0x1p15f * factor)) {}
    __device__ bool holds(float x) const /* 0 is not said to be held: it makes no difference */
    {
        const unsigned v = __float_as_uint(x) & 0x7fffffffu;
        return v >= least && v < most;
    }
};

/* The power of two that values are scaled by, from the largest of their absolute values' bits, and the factor that undoes
 * it: a power of two, NaN if a value is not finite.  fp16 input is not scaled down: it fits, and would lose its last bit. */
template <int TI>
__device__ __forceinline__ float q4_scaling(unsigned largest, float &factor)
{
    int e = 15;
    if (largest - 1u < 0x7f7fffffu) (void)frexpf(__uint_as_float(largest), &e); /* largest < 2^e */
    int shift = min(15 - e, 126);                                              /* 2^-126: the factor is not rounded */
    if (TI == DN_F16) shift = max(shift, 0);
    factor = largest < 0x7f800000u ? ldexpf(1.f, -shift) : __uint_as_float(0x7fc00000u);
    return ldexpf(1.f, shift);
}

/* A scale of 8-bit input: NaN if it is not finite, as an infinite one times a code may be either. */
__device__ __forceinline__ float q4_input_scale(const float *p)
{
    return fabsf(*p) <= 3.402823466e38f ? *p : __uint_as_float(0x7fc00000u);
}

/* Eight inputs from k on, zeros behind the row's end, in one access (two of fp32) whatever their alignment: the run that
 * the end cuts is read from eight before the end, and moved. */
template <int TI>
__device__ __forceinline__ void q4_load8(const void *row, int k, int inputs, float x[8])
{
    typedef typename dn_elt<TI>::store E;
    typedef E E8 __attribute__((ext_vector_type(8)));
    typedef E8 E8U __attribute__((aligned(sizeof(E))));
    const E *p = (const E *)row;
    if (inputs < 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = k + i < inputs ? (float)p[k + i] : 0.f;
        return;
    }
    const int from = min(k, inputs - 8), cut = k - from;
    const E8 v = *(const E8U *)(p + from);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
    if (cut > 0) {
#pragma unroll
        for (int d = 1; d <= 4; d *= 2)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = cut & d ? (i + d < 8 ? x[i + d] : 0.f) : x[i];
        if (cut >= 8)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0;
    }
}

__device__ __forceinline__ unsigned q4_largest8(unsigned m, const float x[8])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
}

/* The least of eight absolute values that are not 0, as the maximum of 0 - its bits. */
__device__ __forceinline__ unsigned q4_least8(unsigned m, const float x[8])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, 0u - (__float_as_uint(x[i]) & 0x7fffffffu));
    return m;
}

/* Whether a value that is not 0 lies below what the pieces hold (never where the factor is NaN). */
template <int TI>
__device__ __forceinline__ bool q4_below(unsigned least, float factor)
{
    return q4_range<TI>::wide && factor > 0 && least > 0u - q4_range<TI>(factor).least;
}

/* The operand form of eight inputs, scaled by a power of two: hi, and 2^12 times what it leaves of the value in lo.
 * Returns the least of the scaled values (below what the pieces hold if one of them is, or is 0). */
#define Q4_LO 0x1p-12f
__device__ __forceinline__ float q4_split8(const float x[8], float scale, half8_t &hi, half8_t &lo)
{
    float least = 1, v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = x[i] * scale;
        least = fminf(least, fabsf(v[i]));
        hi[i] = (_Float16)v[i];
    }
    /* Behind the empty statements the compiler does not know where a half came from: it converts in pairs then, where it
     * would else round each value again in a slower mixed instruction (12544 values 0.25 us). */
    uint4_t w = __builtin_bit_cast(uint4_t, hi);
    asm("" : "+v"(w));
    hi = __builtin_bit_cast(half8_t, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float t = fmaf((float)hi[i], -1 / Q4_LO, v[i] * (1 / Q4_LO)); /* exact before it is rounded */
        asm("" : "+v"(t));
        lo[i] = (_Float16)t;
    }
    return least;
}

/* Of eight inputs those that the pieces take.  Returns whether there are others. */
template <int TI>
__device__ __forceinline__ bool q4_keep_held(float x[8], float factor)
{
    const q4_range<TI> range(factor);
    bool others = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool holds = range.holds(x[i]);
        others = others || (!holds && x[i] != 0);
        x[i] = holds ? x[i] : 0.f;
    }
    return others;
}

/* What the pieces leave of row b's sums with N outputs from o on: the values of marked eights that they do not hold.  Of
 * blocks of 128 inputs: some(kb), whether one of eight from kb on has marks; marks(kb), 16 bits (eights that hold all may be
 * marked too); factor(kb).  One thread's work, for the few rows that need it. */
template <int TI, int N, class Some, class Marks, class Factor>
__device__ __forceinline__ void q4_left_out(const q4_args &a, int b, int o, float (&sum)[N], Some some, Marks marks, Factor factor)
{
    typedef typename dn_elt<TI>::store E;
    const E *row = (const E *)a.input + (long)b * a.s.inputs;
#pragma unroll
    for (int n = 0; n < N; ++n) sum[n] = 0;
#pragma unroll 1
    for (int kb0 = 0; kb0 < a.s.kblocks; kb0 += 8) {
        if (!some(kb0)) continue;
#pragma unroll 1
        for (int kb = kb0; kb < min(kb0 + 8, a.s.kblocks); ++kb) {
#pragma unroll 1
            for (unsigned m = marks(kb); m; m &= m - 1) {
                const int k = kb * 128 + (__ffs((int)m) - 1) * 8;
                const q4_range<TI> range(factor(kb));
                float x[8];
                q4_load8<TI>(row, k, a.s.inputs, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = range.holds(x[i]) ? 0.f : x[i];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int on = min(o + n, a.s.outputs - 1);
                    const unsigned codes = ((const unsigned *)a.packed)[q4_dword_at(a.s, on, k)];
                    const long g = q4_group_at(a.s, on, k / a.s.group);
                    const int zero = a.packed[a.s.zeros_at + g];
                    const float scale = ((const float *)(a.packed + a.s.scales_at))[g];
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[n] = fmaf(x[i], (float)((int)(codes >> q4_bit_of(i) & 15) - zero) * scale, sum[n]);
                }
            }
        }
    }
}

/* One tile of 16 outputs x 128 inputs as a lane holds it; PER groups in 128 inputs. */
template <int PER>
struct q4_tile {
    uint4_t code;
    float scale[PER];
    unsigned zero; /* a byte for each group, from byte zero_at(lane) on */
    static __device__ unsigned zero_at(int lane) { return (unsigned)(lane * PER) & 3; }
};

template <int PER>
__device__ __forceinline__ q4_tile<PER> q4_load_tile(const q4_args &a, int tile, int kb, int lane) /* lane: whose part */
{
    typedef float scales_t __attribute__((ext_vector_type(PER)));
    q4_tile<PER> t;
    const long at = (long)tile * a.s.kblocks + kb, own = (at * 16 + (lane & 15)) * PER;
    t.code = ((const uint4_t *)a.packed)[at * 64 + lane];
    const float *scale = (const float *)(a.packed + a.s.scales_at) + own;
    /* a whole word: after a load of one or two bytes the compiler masks them at once, and so waits for a tile that
     * is not wanted before the next round */
    t.zero = *(const unsigned *)(a.packed + a.s.zeros_at + (own & ~3l));
    if constexpr (PER == 1) {
        t.scale[0] = *scale;
    } else {
        const scales_t v = *(const scales_t *)scale;
#pragma unroll
        for (int g = 0; g < PER; ++g) t.scale[g] = v[g];
    }
    return t;
}

__device__ __forceinline__ half2_t q4_as_half2(unsigned v) { return __builtin_bit_cast(half2_t, v); }

/* The constants of the unpacking, held in registers that the compiler does not see through: it then masks and merges
 * in one instruction, which takes no two literals. */
struct q4_masks {
    unsigned low, high, magic;
    __device__ q4_masks() : low(0x000f000fu), high(0x00f000f0u), magic(0x64006400u)
    {
        asm("" : "+s"(low), "+s"(high), "+v"(magic));
    }
};

/* Eight codes less their zero as fp16: 0x6400 | c is 1024 + c, and with the code four bits up 1024 + 16 c. */
__device__ __forceinline__ half8_t q4_unpack8(unsigned v, half2_t z1024, half2_t z64, const q4_masks &k)
{
    const half2_t sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const unsigned w = v >> 8;
    const half2_t a = q4_as_half2((v & k.low) | k.magic) + z1024;
    const half2_t b = __builtin_elementwise_fma(q4_as_half2((v & k.high) | k.magic), sixteenth, z64);
    const half2_t c = q4_as_half2((w & k.low) | k.magic) + z1024;
    const half2_t d = __builtin_elementwise_fma(q4_as_half2((w & k.high) | k.magic), sixteenth, z64);
    return (half8_t){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

/* The zero of group g of a tile in both halves, as -(1024 + z) and -(64 + z). */
template <int PER>
__device__ __forceinline__ void q4_zeros(const q4_tile<PER> &w, int g, half2_t &z1024, half2_t &z64)
{
    const unsigned select = 0x0c000c00u + 0x00010001u * (q4_tile<PER>::zero_at(threadIdx.x & 63) + g);
    const unsigned z2 = __builtin_amdgcn_perm(0, w.zero, select);
    z1024 = q4_as_half2(0xe400e400u | z2);
    z64 = q4_as_half2(0xd400d400u | z2 << 4);
}

/* Adds the products of R tiles of outputs with T tiles of 16 input rows.  operand(t, piece, step): the lane's eight
 * inputs of a row; x_scale(t, g): the factors of its four rows of results, where they change along the row (XS). */
template <int T, int R, int PIECES, int PER, bool XS, class Operand, class Scale>
__device__ __forceinline__ void q4_multiply(const q4_masks &masks, const q4_tile<PER> (&w)[R], float4_t (&sum)[R][T],
                                            Operand operand, Scale x_scale)
{
#pragma unroll
    for (int g = 0; g < PER; ++g) {
        /* the second piece has sums of its own (4 instructions for a group and tile of 16 rows, not 4 for each 8 weights of a
         * lane: 64 x 4096 -> 32768 fp32 53.1 us, 55.4 with the weights multiplied; in groups of 32 60.7 and 58.0) */
        constexpr int SUMS = PIECES == 2 && PER < 4 && R * T <= 4 ? 2 : 1;
        float4_t part[SUMS][R][T], acc[R][T];
        half2_t z1024[R], z64[R];
#pragma unroll
        for (int r = 0; r < R; ++r) q4_zeros(w[r], g, z1024[r], z64[r]);
#pragma unroll
        for (int i = 0; i < 4 / PER; ++i) {
            const int step = g * (4 / PER) + i;
            half8_t wv[R], wl[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                wv[r] = q4_unpack8(w[r].code[step], z1024[r], z64[r], masks);
                if (PIECES == 2 && SUMS == 1) wl[r] = wv[r] * (_Float16)Q4_LO; /* exact: 15 * 2^-12 at most, 2^-12 at least */
            }
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    const half8_t x = operand(t, p, step);
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        part[p % SUMS][r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            x, p && SUMS == 1 ? wl[r] : wv[r], i || p >= SUMS ? part[p % SUMS][r][t] : (float4_t){0, 0, 0, 0}, 0, 0, 0);
                }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < T; ++t)
                acc[r][t] = SUMS == 2 ? __builtin_elementwise_fma(part[SUMS - 1][r][t], (float4_t){Q4_LO, Q4_LO, Q4_LO, Q4_LO}, part[0][r][t]) : part[0][r][t];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float4_t f = {1, 1, 1, 1};
            if (XS) f = x_scale(t, g);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float4_t scale = {w[r].scale[g], w[r].scale[g], w[r].scale[g], w[r].scale[g]};
                sum[r][t] = XS ? __builtin_elementwise_fma(acc[r][t] * scale, f, sum[r][t]) : __builtin_elementwise_fma(acc[r][t], scale, sum[r][t]);
            }
        }
    }
}

/* An output: bias, activation, rounding, store. */
__device__ __forceinline__ void q4_store(const q4_args &a, int b, int o, float y, float bias)
{
    y += bias;
    y = a.activation == DN_LINEAR ? y : dn_activate(y, a.activation);
    const long at = (long)b * a.s.outputs + o;
    if (a.output_type == DN_F32) ((float *)a.output)[at] = y;
    else if (a.output_type == DN_F16) ((_Float16 *)a.output)[at] = (_Float16)y;
    else ((__bf16 *)a.output)[at] = (__bf16)y;
}

__device__ __forceinline__ float q4_bias(const q4_args &a, int o) { return a.biases && o < a.s.outputs ? a.biases[o] : 0.f; }

/* ---- small input: at most 4 rows that fit into LDS whole.  Each workgroup scales and splits the input itself, block
 * by block of 128 values, and then streams the weights, AHEAD loads of a wave in flight.
 *
 * The matrix instruction has 16 rows, and the input at most 4: where there are fewer tiles of outputs than CUs, its rows
 * are 4 rows of H neighbouring blocks, and its columns the weights of 16 / H outputs in these blocks.  A column's
 * result with its own block is what counts.  So a workgroup has fewer outputs, and each operand that is read from LDS
 * serves H blocks; but a wave then reads pieces of 256 / H bytes, which costs more than it gives with many tiles.
 *
 * Measured, fp32 input: 4096 -> 4096 in groups of 128 5.4 us (1.7 TB/s; a launch that does nothing 3; 6.7 with weights
 * that come from memory), 12544 -> 1715 in groups of 32 8.9 us (1.6 TB/s), 25088 -> 4096 17.8 us (3.1 TB/s); bf16, weights
 * from memory: 8192 -> 28672 28 us, 4096 -> 131072 60 us (4.8 TB/s).  Of the second 4 us are the launch, the first loads
 * and the join, 2 the scaling of the input, the rest the weights: few CUs, each at what it can have in flight.  A block
 * of 128 values far below an outlier costs some 10 us more. */
template <int TI, int PER, bool XG, int H>
__global__ __launch_bounds__(Q4_THREADS, 4) void q4_direct_kernel(q4_args a)
{
    constexpr int THREADS = Q4_THREADS, WAVES = Q4_WAVES;
    constexpr int PIECES = TI == DN_F32 ? 2 : 1, WIDTH = 16 / H;
    constexpr int BLOCK = H > 1 ? 272 : 256; /* bytes of a block: 16 more put the blocks of an operand in other banks */
    constexpr int AHEAD = 4, MOVES = 2;
    extern __shared__ char lds[];
    __shared__ float s_red[WAVES][4][WIDTH];
    __shared__ unsigned s_below[WAVES]; /* whether a wave has met values below what the pieces hold */
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kblocks = a.s.kblocks, steps = (kblocks + H - 1) / H, kpad = steps * H * 128;
    const int plane = kpad / 128 * BLOCK, pitch = plane * PIECES + 16; /* bytes of a row's halves, and of a row */
    const int part = wave % a.ksplit, own_unit = wave / a.ksplit, units_per = WAVES / a.ksplit;
    const int mine = (steps - part + a.ksplit - 1) / a.ksplit; /* this wave's steps of H blocks: part, part + ksplit, ... */
    const int stride = gridDim.x * units_per, units = a.s.tiles * H; /* a unit: WIDTH outputs */
    const int own_block = (lane & 15) / WIDTH, own_row = lane >> 4;
    int unit0 = blockIdx.x * units_per;

    auto fetch = [&](int u, int n) {
        const int unit = min(u, units - 1), kb = (part + a.ksplit * n) * H + own_block;
        /* behind the last block: its weights again, for input that is 0 */
        return q4_load_tile<PER>(a, unit / H, min(kb, kblocks - 1), (lane & 48) + unit % H * WIDTH + lane % WIDTH);
    };
    const q4_masks masks;
    q4_tile<PER> w[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (u < mine) w[u] = fetch(unit0 + own_unit, u);

    /* the input: [row][pitch] halves, and [block (8-bit input with groups: group)][4 rows] factors behind them, negative
     * (fp32 and bf16 input) where values lie below what the pieces hold */
    const size_t row_bytes = (size_t)a.s.inputs * (TI == DN_F32 ? 4 : TI == DN_I8 ? 1 : 2);
    float *factors = (float *)(lds + a.batch * pitch);
    if (q4_range<TI>::wide && lane == 0) s_below[wave] = 0;
    const int eights = kpad / 8;
    for (int b = 0, q = tid; b < a.batch;) {
        float x[MOVES][8];
        int of[MOVES], at[MOVES]; /* row and eight of the next items of this lane, whose loads go together */
#pragma unroll
        for (int m = 0; m < MOVES; ++m) {
            const bool in = q < eights; /* (a row shorter than the workgroup leaves some lanes out) */
            of[m] = in ? b : a.batch;
            at[m] = q;
            q4_load8<TI>((const char *)a.input + min(b, a.batch - 1) * row_bytes, min(q, eights - 1) * 8, a.s.inputs, x[m]);
            q += THREADS;
            if (q >= eights) {
                q = tid;
                ++b;
            }
        }
#pragma unroll
        for (int m = 0; m < MOVES; ++m) { /* 16 lanes have a block */
            if (of[m] >= a.batch) continue;
            float factor = 1, scale = 1;
            half8_t hi, lo;
            if (TI != DN_I8) {
                unsigned m8 = q4_largest8(0, x[m]);
                m8 = max(m8, dn_move<0xb1, 0xf>(m8, m8));
                m8 = max(m8, dn_move<0x4e, 0xf>(m8, m8));
                m8 = max(m8, dn_move<0x141, 0xf>(m8, m8));
                m8 = max(m8, dn_move<0x140, 0xf>(m8, m8));
                scale = q4_scaling<TI>(m8, factor);
                if ((tid & 15) == 0) factors[(at[m] >> 4) * 4 + of[m]] = factor;
            }
            const float least = q4_split8(x[m], scale, hi, lo);
            if (q4_range<TI>::wide && least < 0x1p-14f && q4_below<TI>(q4_least8(0, x[m]), factor)) {
                (void)q4_keep_held<TI>(x[m], factor);
                (void)q4_split8(x[m], scale, hi, lo);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* behind the write above, which is the same wave's */
                factors[(at[m] >> 4) * 4 + of[m]] = -factor;
                s_below[wave] = 1;
            }
            char *to = lds + of[m] * pitch + (at[m] >> 4) * BLOCK + (at[m] & 15) * 16;
            *(half8_t *)to = hi;
            if (PIECES == 2) *(half8_t *)(to + plane) = lo;
        }
    }
    if (XG) {
        const int x_groups = (a.s.inputs + a.x_group - 1) / a.x_group, groups = kpad / 128 * PER;
        for (int i = tid; i < a.batch * groups; i += THREADS) {
            const int b = i / groups, g = i - b * groups;
            factors[g * 4 + b] = g < x_groups ? q4_input_scale(a.input_scales + (long)b * x_groups + g) : 0.f;
        }
    }
    __syncthreads();

    const char *base = lds + min((lane & 15) >> 2, a.batch - 1) * pitch + (lane & 3) % H * BLOCK + (lane >> 4) * 16;
    const float *own_factors = factors + own_block * (XG ? PER : 1) * 4 + own_row;
    for (; unit0 < units; unit0 += stride) {
        const int unit = unit0 + own_unit;
        float sum = 0;
        for (int n = 0; n < mine; n += AHEAD) {
            const bool last = n + AHEAD >= mine; /* what comes next is of the next unit */
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (n + u < mine) {
                    const int kb = (part + a.ksplit * (n + u)) * H;
#pragma unroll
                    for (int g = 0; g < PER; ++g) {
                        half2_t z1024, z64;
                        q4_zeros(w[u], g, z1024, z64);
                        /* the second piece has a sum of its own (one or two instructions more for a group, not four for each 8
                         * weights), or goes first where that would take more registers than there are (a group is one step there) */
                        constexpr int SUMS = PIECES == 2 && (PER < 4 || H < 4) ? 2 : 1;
                        float4_t acc[SUMS];
#pragma unroll
                        for (int p = 0; p < SUMS; ++p) acc[p] = (float4_t){0, 0, 0, 0};
#pragma unroll
                        for (int step = g * (4 / PER); step < (g + 1) * (4 / PER); ++step) {
                            half8_t x[PIECES];
#pragma unroll
                            for (int p = 0; p < PIECES; ++p) x[p] = *(const half8_t *)(base + p * plane + kb * BLOCK + step * 64);
                            const half8_t wv = q4_unpack8(w[u].code[step], z1024, z64, masks);
#pragma unroll
                            for (int p = PIECES - 1; p >= 0; --p) {
                                acc[p % SUMS] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[p], wv, acc[p % SUMS], 0, 0, 0);
                                if (SUMS == 1 && p == 1) acc[0] *= (float4_t){Q4_LO, Q4_LO, Q4_LO, Q4_LO};
                            }
                        }
                        auto own = [&](float4_t v) { return own_block == 0 ? v[0] : own_block == 1 ? v[1] : own_block == 2 ? v[2] : v[3]; };
                        const float v = SUMS == 2 ? fmaf(own(acc[SUMS - 1]), Q4_LO, own(acc[0])) : own(acc[0]);
                        const float f = TI != DN_I8 || XG ? own_factors[(XG ? kb * PER + g : kb) * 4] : 1.f;
                        sum = fmaf(v * w[u].scale[g], q4_range<TI>::wide ? fabsf(f) : f, sum);
                    }
                }
                if (last ? u < mine && unit0 + stride < units : n + AHEAD + u < mine)
                    w[u] = fetch(last ? unit + stride : unit, last ? u : n + AHEAD + u);
            }
        }
        /* what the blocks and the waves of a unit have, added in their order; a thread for each output of each row */
        if (H >= 2) sum += dn_move<0x128, 0xf>(sum, sum); /* the lane 8, then 4 on among 16 */
        if (H == 4) sum += dn_move<0x124, 0xf>(sum, sum);
        __syncthreads();
        if (own_block == 0) s_red[wave][own_row][lane % WIDTH] = sum;
        __syncthreads();
        for (int i = tid; i < units_per * a.batch * WIDTH; i += THREADS) {
            const int r = i / (a.batch * WIDTH), b = i / WIDTH % a.batch, o = (unit0 + r) * WIDTH + i % WIDTH;
            if (o >= a.s.outputs) continue;
            const float bias = q4_bias(a, o);
            float y = 0;
#pragma unroll
            for (int q = 0; q < WAVES; ++q)
                if (q < a.ksplit) y += s_red[r * a.ksplit + q][b][i % WIDTH];
            if (TI == DN_I8 && !XG) y *= q4_input_scale(a.input_scales + b);
            if constexpr (q4_range<TI>::wide) {
                unsigned any = 0;
#pragma unroll
                for (int q = 0; q < WAVES; ++q) any |= s_below[q];
                if (__builtin_expect(any != 0, 0)) {
                    auto factor = [&](int kb) { return -factors[kb * 4 + b]; };
                    float left[1];
                    q4_left_out<TI>(a, b, o, left, [](int) { return true; }, [&](int kb) { return factor(kb) > 0 ? 0xffffu : 0u; }, factor);
                    y += left[0];
                }
            }
            q4_store(a, b, o, y, bias);
        }
    }
}

/* ---- larger input, first pass: one workgroup for each row scales it and writes it in the order in which the second
 * pass feeds it to the matrix instruction: [row / 16][inputs / 128] blocks of [piece][step][lane][8 halves] and, for
 * 8-bit input with groups, [group in 128][16] factors.  Behind the blocks a factor for each row, negative (fp32 and bf16
 * input) where the pieces do not hold all values; then [row][inputs / 128, in eights] the 16 bits of the eights that have
 * such values, written for these rows only.  A pass over a few kilobytes, 3 to 5 us with its launch; it saves every
 * workgroup of the second pass a scaling of its own (16 rows of 8192 values read as they are by that pass, without this
 * one: the same time in groups of 128, 27 us against 20 in groups of 32).  1024 threads for long rows: 8 rows of 20787
 * in all 17.8 us, 21 with 256. */
__host__ __device__ static inline int q4_block_bytes(const q4_shape &s, int pieces, bool groups)
{
    return pieces * 4096 + (groups ? 128 / s.group * 64 : 0);
}

__host__ __device__ static inline size_t q4_rows_at(const q4_shape &s, int pieces, int batch, bool groups)
{
    return ((size_t)batch + 15) / 16 * s.kblocks * q4_block_bytes(s, pieces, groups);
}

__host__ __device__ static inline size_t q4_marks_at(const q4_shape &s, int pieces, int batch, bool groups)
{
    return (q4_rows_at(s, pieces, batch, groups) + (size_t)batch * 4 + 15) / 16 * 16;
}
__host__ __device__ static inline size_t q4_marks_pitch(const q4_shape &s) { return ((size_t)s.kblocks + 7) / 8 * 8; }

/* The factor under which the pieces hold most of a row's values: of the runs of as many exponents as they hold the one
 * with most values.  The whole workgroup. */
template <int TI, int THREADS>
__device__ __forceinline__ float q4_factor_for_most(const char *row, int inputs, float &scale)
{
    typedef unsigned long long u64;
    __shared__ unsigned s_exponents[256];
    __shared__ u64 s_best[THREADS / 64];
    const int tid = threadIdx.x;
    static_assert(THREADS >= 256, "a thread for each exponent");
    if (tid < 256) s_exponents[tid] = 0;
    __syncthreads();
    for (int k = tid * 8; k < inputs; k += THREADS * 8) {
        float x[8];
        q4_load8<TI>(row, k, inputs, x);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (x[i] != 0) atomicAdd(&s_exponents[(__float_as_uint(x[i]) & 0x7fffffffu) >> 23], 1u);
    }
    __syncthreads();
    u64 best = 0; /* the number of values, and the last exponent of the run */
    if (tid < 255) {
        for (int e = max(tid - q4_range<TI>::exponents + 1, 0); e <= tid; ++e) best += s_exponents[e];
        best = best << 8 | (unsigned)tid;
    }
    best = dn_wave_max(best);
    if ((tid & 63) == 0) s_best[tid >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) best = best > s_best[w] ? best : s_best[w];
    const int shift = min(141 - (int)(best & 255), 126); /* the values are below 2^(exponent - 126) */
    scale = ldexpf(1.f, shift);
    return ldexpf(1.f, -shift);
}

template <int TI, bool XG, int THREADS>
__global__ __launch_bounds__(THREADS) void q4_prepare_kernel(q4_args a)
{
    constexpr int PIECES = TI == DN_F32 ? 2 : 1;
    __shared__ unsigned s_largest[THREADS / 64], s_least[THREADS / 64];
    const int tid = threadIdx.x, b = blockIdx.x, block = q4_block_bytes(a.s, PIECES, XG);
    const size_t row_bytes = (size_t)a.s.inputs * (TI == DN_F32 ? 4 : TI == DN_I8 ? 1 : 2);
    const char *row = (const char *)a.input + b * row_bytes;
    float factor = 1, scale = 1;
    bool below = false;
    if (TI != DN_I8) {
        unsigned m = 0, least = 0;
#pragma unroll 4
        for (int k = tid * 8; k < a.s.inputs; k += THREADS * 8) {
            float x[8];
            q4_load8<TI>(row, k, a.s.inputs, x);
            m = q4_largest8(m, x);
            if (q4_range<TI>::wide) least = q4_least8(least, x);
        }
        m = dn_wave_max(m);
        if (q4_range<TI>::wide) least = dn_wave_max(least);
        if ((tid & 63) == 0) {
            s_largest[tid >> 6] = m;
            s_least[tid >> 6] = least;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) {
            m = max(m, s_largest[w]);
            if (q4_range<TI>::wide) least = max(least, s_least[w]);
        }
        scale = q4_scaling<TI>(m, factor);
        below = q4_below<TI>(least, factor);
        if constexpr (q4_range<TI>::wide)
            if (below) factor = q4_factor_for_most<TI, THREADS>(row, a.s.inputs, scale);
    }
    if (tid == 0)
        ((float *)(a.workspace + q4_rows_at(a.s, PIECES, a.batch, XG)))[b] = TI == DN_I8 ? (XG ? 1.f : q4_input_scale(a.input_scales + b)) : below ? -factor : factor;
    unsigned char *out = a.workspace + (size_t)(b >> 4) * a.s.kblocks * block + (b & 15) * 16;
    unsigned short *marks = (unsigned short *)(a.workspace + q4_marks_at(a.s, PIECES, a.batch, XG)) + b * q4_marks_pitch(a.s);
    if (q4_range<TI>::wide && below && tid < 8 && a.s.kblocks + tid < q4_marks_pitch(a.s)) marks[a.s.kblocks + tid] = 0;
    for (int k = tid * 8; k < a.s.kblocks * 128; k += THREADS * 8) {
        float x[8];
        half8_t hi, lo;
        q4_load8<TI>(row, k, a.s.inputs, x);
        if (q4_range<TI>::wide && below) { /* 16 lanes have a block */
            const unsigned mark = (unsigned)(__ballot(q4_keep_held<TI>(x, factor)) >> (tid & 48)) & 0xffffu;
            if ((tid & 15) == 0) marks[k >> 7] = (unsigned short)mark;
        }
        q4_split8(x, scale, hi, lo);
        unsigned char *to = out + (size_t)(k >> 7) * block + ((k >> 5) & 3) * 1024 + ((k >> 3) & 3) * 256;
        *(half8_t *)to = hi;
        if (PIECES == 2) *(half8_t *)(to + 4096) = lo;
    }
    if (XG) {
        const int x_groups = (a.s.inputs + a.x_group - 1) / a.x_group, per = 128 / a.s.group;
        unsigned char *to = a.workspace + (size_t)(b >> 4) * a.s.kblocks * block + PIECES * 4096 + (b & 15) * 4;
        for (int g = tid; g < a.s.groups; g += THREADS)
            *(float *)(to + (size_t)(g / per) * block + g % per * 64) = g < x_groups ? q4_input_scale(a.input_scales + (long)b * x_groups + g) : 0.f;
    }
}

/* Whether a row has values that the pieces do not hold, and what they leave of its sums with N outputs. */
template <bool XG>
__device__ __forceinline__ bool q4_is_below(const q4_args &a, float row_factor) { return !XG && a.ranged && row_factor < 0; }

template <int PIECES, int N>
__device__ __forceinline__ void q4_left_out_of(const q4_args &a, float row_factor, int b, int o, float (&left)[N])
{
    const unsigned short *marks = (const unsigned short *)(a.workspace + q4_marks_at(a.s, PIECES, a.batch, false)) + b * q4_marks_pitch(a.s);
    q4_left_out<PIECES == 2 ? DN_F32 : DN_BF16>(
        a, b, o, left,
        [&](int kb) {
            const uint4_t m = *(const uint4_t *)(marks + kb);
            return (m[0] | m[1] | m[2] | m[3]) != 0;
        },
        [&](int kb) { return (unsigned)marks[kb]; }, [&](int) { return -row_factor; });
}

/* A sum with its row's factor. */
template <int PIECES, bool XG>
__device__ __forceinline__ float q4_scaled(const q4_args &a, float row_factor, int b, int o, float y)
{
    if (!q4_is_below<XG>(a, row_factor)) return y * row_factor;
    float left[1];
    q4_left_out_of<PIECES>(a, row_factor, b, o, left);
    return fmaf(y, -row_factor, left[0]);
}

/* A lane's results of one tile of outputs and 16 rows, with the rows' own factors. */
template <int PIECES, bool XG>
__device__ __forceinline__ void q4_store_tile(const q4_args &a, const float *row_factors, int tile, int b0, float4_t v)
{
    const int lane = threadIdx.x & 63, o = tile * 16 + (lane & 15);
    if (o >= a.s.outputs) return;
    const float bias = q4_bias(a, o);
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        const int b = b0 + (lane >> 4) * 4 + i;
        const float y = i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3];
        if (b < a.batch) q4_store(a, b, o, q4_scaled<PIECES, XG>(a, row_factors[b], b, o, y), bias);
    }
}

/* The same as one of several parts of the sums, which the next pass joins. */
__host__ __device__ static inline size_t q4_parts_at(const q4_shape &s, int pieces, int batch, bool groups)
{
    return q4_marks_at(s, pieces, batch, groups) + batch * q4_marks_pitch(s) * 2;
}

__device__ __forceinline__ void q4_store_part(const q4_args &a, size_t parts_at, int tile, int b0, float4_t v)
{
    const int lane = threadIdx.x & 63, o = tile * 16 + (lane & 15);
    if (o >= a.s.outputs) return;
    float *parts = (float *)(a.workspace + parts_at) + (size_t)blockIdx.z * a.batch * a.s.outputs;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int b = b0 + (lane >> 4) * 4 + i;
        if (b < a.batch) parts[(size_t)b * a.s.outputs + o] = v[i];
    }
}

/* Third pass, where the inputs were cut: the parts' sums of an output, in their order. */
template <int PIECES, bool XG>
__global__ __launch_bounds__(256) void q4_join_kernel(q4_args a, size_t rows_at, size_t parts_at, int parts)
{
    const int o = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (o >= a.s.outputs) return;
    const float *part = (const float *)(a.workspace + parts_at) + (size_t)b * a.s.outputs + o;
    const float bias = q4_bias(a, o), factor = ((const float *)(a.workspace + rows_at))[b];
    float y = 0;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) y += part[(size_t)p * a.batch * a.s.outputs];
    q4_store(a, b, o, q4_scaled<PIECES, XG>(a, factor, b, o, y), bias);
}

/* ---- second pass, few outputs: a workgroup takes R row tiles and a tile of input rows, its eight waves an eighth of
 * the inputs each.  No two waves read the same input, so that it comes straight into registers like the weights, both
 * a block ahead, and nothing waits for another wave before the end.
 *
 * Measured: 16 rows of 8-bit input, 8192 -> 8192 in groups of 128, 14.1 us for both passes, 11 for this one (3.3 TB/s);
 * 16 x 4096 -> 32768 bf16 21.5 us (3.4 TB/s).  Two tiles of input rows in a workgroup took longer (64 x 4096 -> 8192:
 * 23.7 against 20.4 us: fewer waves have the registers). */
template <int R, int PIECES, int PER, bool XG>
__global__ __launch_bounds__(Q4_THREADS) void q4_stream_kernel(q4_args a)
{
    __shared__ float4_t s_red[Q4_WAVES][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int block = q4_block_bytes(a.s, PIECES, XG), x_tile = blockIdx.y, tile0 = blockIdx.x * R;
    const int kb0 = blockIdx.z * a.run, mine = (min(a.run, a.s.kblocks - kb0) - wave + Q4_WAVES - 1) / Q4_WAVES;
    struct block_data {
        q4_tile<PER> w[R];
        half8_t x[PIECES][4];
        float4_t f[PER];
    };
    auto fetch = [&](int n, block_data &d) {
        const int kb = kb0 + wave + n * Q4_WAVES;
#pragma unroll
        for (int r = 0; r < R; ++r) d.w[r] = q4_load_tile<PER>(a, min(tile0 + r, a.s.tiles - 1), kb, lane);
        const unsigned char *p = a.workspace + ((size_t)x_tile * a.s.kblocks + kb) * block;
#pragma unroll
        for (int i = 0; i < 4 * PIECES; ++i) d.x[i / 4][i % 4] = *(const half8_t *)(p + i * 1024 + lane * 16);
        if (XG)
#pragma unroll
            for (int g = 0; g < PER; ++g) d.f[g] = *(const float4_t *)(p + PIECES * 4096 + g * 64 + (lane >> 4) * 16);
    };
    float4_t sum[R][1];
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r][0] = (float4_t){0, 0, 0, 0};
    const q4_masks masks;
    auto multiply = [&](const block_data &d) {
        q4_multiply<1, R, PIECES, PER, XG>(
            masks, d.w, sum, [&](int, int piece, int step) { return d.x[piece][step]; }, [&](int, int g) { return d.f[g]; });
    };
    block_data one, two;
    if (mine > 0) fetch(0, one);
    for (int n = 0; n < mine; n += 2) {
        if (n + 1 < mine) fetch(n + 1, two);
        multiply(one);
        if (n + 2 < mine) fetch(n + 2, one);
        if (n + 1 < mine) multiply(two);
    }
    /* the waves' sums, in their order; each wave joins what falls to it */
    const float *row_factors = (const float *)(a.workspace + q4_rows_at(a.s, PIECES, a.batch, XG));
#pragma unroll 1
    for (int k = 0; k < R; ++k) {
        __syncthreads();
        s_red[wave][lane] = R > 1 && k == 1 ? sum[R - 1][0] : sum[0][0];
        __syncthreads();
        if (wave == k && tile0 + k < a.s.tiles) {
            float4_t v = s_red[0][lane];
#pragma unroll
            for (int q = 1; q < Q4_WAVES; ++q) v += s_red[q][lane];
            if (gridDim.z > 1) q4_store_part(a, q4_parts_at(a.s, PIECES, a.batch, XG), tile0 + k, x_tile * 16, v);
            else q4_store_tile<PIECES, XG>(a, row_factors, tile0 + k, x_tile * 16, v);
        }
    }
}

/* Four neighbouring outputs of a row, in one access where they exist, whatever their alignment. */
template <class E>
__device__ __forceinline__ void q4_put4(E *p, int n, float4_t y)
{
    typedef E E4 __attribute__((ext_vector_type(4)));
    typedef E4 E4U __attribute__((aligned(sizeof(E))));
    if (n >= 4) {
        *(E4U *)p = __builtin_convertvector(y, E4);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) p[i] = (E)y[i];
    }
}

__device__ __forceinline__ void q4_store4(const q4_args &a, int b, int o, float4_t y)
{
    if (a.activation != DN_LINEAR)
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            const float x = dn_activate(i == 0 ? y[0] : i == 1 ? y[1] : i == 2 ? y[2] : y[3], a.activation);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = i == e ? x : y[e];
        }
    const long at = (long)b * a.s.outputs + o;
    const int n = a.s.outputs - o;
    if (a.output_type == DN_F32) q4_put4((float *)a.output + at, n, y);
    else if (a.output_type == DN_F16) q4_put4((_Float16 *)a.output + at, n, y);
    else q4_put4((__bf16 *)a.output + at, n, y);
}

/* ---- second pass, many outputs: a workgroup takes 4 * R row tiles, R for each wave, and T tiles of input rows.  The
 * input goes through LDS in chunks that all waves read; each wave's weights come straight from memory, as nobody else
 * needs them.
 *
 * Measured: 64 x 4096 -> 131072 bf16, groups of 128, fp32 output: 100 us, 3.2 TB/s and 690 TFLOP/s; its bytes alone
 * take 54 us at the rate of a large addition and its products 52 at that of a large product.  A SIMD has two waves, and an
 * instruction count of 40 us of vector and 27 us of matrix instructions, which overlap in part.  One chunk on its way
 * instead of two 117 us; four row tiles a wave or three workgroups a CU gave nothing. */
#define Q4_STAGED_WAVES 4
template <int T, int R, int PIECES, int PER, bool XG>
__global__ __launch_bounds__(Q4_STAGED_WAVES * 64, 2) void q4_staged_kernel(q4_args a)
{
    constexpr int THREADS = Q4_STAGED_WAVES * 64;
    constexpr int UNITS = T * PIECES >= 2 ? 1 : 2; /* blocks of a chunk */
    constexpr int BLOCK = PIECES * 4096 + (XG ? PER * 64 : 0), SPAN = UNITS * BLOCK, CHUNK = T * SPAN;
    constexpr int MOVES = (CHUNK + THREADS * 16 - 1) / (THREADS * 16);
    __shared__ uint4_t s_input[2][CHUNK / 16];
    __shared__ float s_factors[T * 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int x_tiles = (a.batch + 15) / 16, x0 = blockIdx.y * T, tile0 = (blockIdx.x * Q4_STAGED_WAVES + wave) * R;
    const int kblocks = a.s.kblocks, chunks = (kblocks + UNITS - 1) / UNITS;
    float4_t sum[R][T];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) sum[r][t] = (float4_t){0, 0, 0, 0};

    if (tid < T * 16) s_factors[tid] = ((const float *)(a.workspace + q4_rows_at(a.s, PIECES, a.batch, XG)))[min(x0 * 16 + tid, a.batch - 1)];
    const q4_masks masks;
    uint4_t moved[2][MOVES];
    auto input_of = [&](int c, uint4_t (&to)[MOVES]) {
#pragma unroll
        for (int m = 0; m < MOVES; ++m) { /* what lies behind the last block or tile is read at its place, and not multiplied */
            const int at = (m * THREADS + tid) * 16, i = (m + 1) * THREADS * 16 <= CHUNK ? at : min(at, CHUNK - 16), t = i / SPAN, in = i % SPAN;
            const int kb = min(c * UNITS + in / BLOCK, kblocks - 1);
            to[m] = *(const uint4_t *)(a.workspace + ((size_t)min(x0 + t, x_tiles - 1) * kblocks + kb) * BLOCK + in % BLOCK);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto keep_input = [&](int buffer, const uint4_t (&from)[MOVES]) {
#pragma unroll
        for (int m = 0; m < MOVES; ++m)
            if ((m + 1) * THREADS * 16 <= CHUNK || (m * THREADS + tid) * 16 < CHUNK) s_input[buffer][m * THREADS + tid] = from[m];
    };
    q4_tile<PER> w[2][UNITS][R];
    auto fetch = [&](int c, int u, q4_tile<PER> (&to)[R]) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < R; ++r)
            to[r] = q4_load_tile<PER>(a, min(tile0 + r, a.s.tiles - 1), min(c * UNITS + u, kblocks - 1), lane);
        __builtin_amdgcn_sched_barrier(0);
    };
    /* Two chunks on their way, input and weights in turn: loads return in their order, so that a wait for input that was
     * asked for behind weights would be a wait for those as well.  No load is conditional (behind the last chunk they
     * repeat the last block): the compiler waits for every load that may have been left out. */
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        input_of(h, moved[h]);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) fetch(h, u, w[h][u]);
    }
    keep_input(0, moved[0]);
    __syncthreads();
    for (int c0 = 0; c0 < chunks; c0 += 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = c0 + h;
            input_of(c + 2, moved[h]);
            const char *base = (const char *)s_input[h];
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                if (c * UNITS + u < kblocks)
                    q4_multiply<T, R, PIECES, PER, XG>(
                        masks, w[h][u], sum,
                        [&](int t, int piece, int step) {
                            return *(const half8_t *)(base + t * SPAN + u * BLOCK + piece * 4096 + step * 1024 + lane * 16);
                        },
                        [&](int t, int g) { return *(const float4_t *)(base + t * SPAN + u * BLOCK + PIECES * 4096 + g * 64 + (lane >> 4) * 16); });
                fetch(c + 2, u, w[h][u]);
            }
            keep_input(h ^ 1, moved[h ^ 1]); /* the buffer that all waves have left at the last barrier */
            __syncthreads();
        }
    }
    /* The sums go through LDS, a tile of input rows at a time, so that neighbouring lanes store neighbouring outputs
     * (16 of a row alone are half a line), four each, and there is one copy of the activation's code. */
    constexpr int WIDTH = Q4_STAGED_WAVES * R * 16, PITCH = WIDTH + 4;
    static_assert(sizeof s_input >= 16 * PITCH * 4, "room for a tile's sums");
    float *s_sum = (float *)s_input;
    const int column = tid % (WIDTH / 4) * 4, o = blockIdx.x * WIDTH + column;
    const float4_t bias = {q4_bias(a, o), q4_bias(a, o + 1), q4_bias(a, o + 2), q4_bias(a, o + 3)};
#pragma unroll 1
    for (int x = 0; x < T; ++x) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float4_t v = sum[r][0];
#pragma unroll
            for (int m = 1; m < T; ++m) v = x == m ? sum[r][m] : v;
#pragma unroll
            for (int i = 0; i < 4; ++i) s_sum[((lane >> 4) * 4 + i) * PITCH + (wave * R + r) * 16 + (lane & 15)] = v[i];
        }
        __syncthreads();
#pragma unroll 1
        for (int row = tid / (WIDTH / 4); row < 16; row += THREADS / (WIDTH / 4)) {
            const int b = (x0 + x) * 16 + row;
            const float f = s_factors[x * 16 + row];
            if (b >= a.batch || o >= a.s.outputs) continue;
            float4_t y = *(const float4_t *)(s_sum + row * PITCH + column);
            if (q4_is_below<XG>(a, f)) {
                float left[4];
                q4_left_out_of<PIECES>(a, f, b, o, left);
                y = __builtin_elementwise_fma(y, (float4_t){-f, -f, -f, -f}, (float4_t){left[0], left[1], left[2], left[3]}) + bias;
            } else {
                y = __builtin_elementwise_fma(y, (float4_t){f, f, f, f}, bias);
            }
            q4_store4(a, b, o, y);
        }
        __syncthreads();
    }
}

/* Which form a product takes (times of both sides, groups of 128):
 *   direct  at most 4 rows (the matrix instruction's rows and columns are laid out for that) which fit into LDS: one row
 *           25088 -> 4096 fp32 18.3 us, by the second pass below 29.4; four rows 4096 -> 4096 bf16 6.4 us against 8.8.
 *           The border is rough: four rows of 18000 bf16 21.3 against 16.9.
 *   staged  so many tiles that workgroups of 4 or 8 of them fill the chip: its time hardly depends on their number
 *           up to there, while stream's grows with it.  64 x 4096 -> 11200 (2800 tiles) bf16 25.2 against 31.3 us, fp32
 *           36.1 and 46.9; 9216 (2304) 24.9 and 26.2, 36.0 and 40.1; 8192 (2048) 24.8 and 22.4, 35.9 and 34.4.  (Fewer
 *           rows would have it lower: 32 x 4096 -> 16384, 2048 tiles, bf16 18.7 and 22.5.)
 *   stream  the others
 * Blocks (H): 12544 -> 1715 (108 tiles) 7.3 us by two, 9.5 by one; 160 tiles 10.1 by two, 9.6 by one; 63 tiles of
 * 8192 5.3 by four, 5.7 by two, 7.2 by one.
 * Row tiles (R): staged 64 x 4096 -> 131072 100 us by two, 113 by one, no difference at 49152; stream 16 x 8192 -> 8192
 * 15.0 and 15.4. */
struct q4_plan {
    enum { DIRECT, STREAM, STAGED } form;
    int ksplit, h, t, r, run;
    unsigned gx, gy, gz;
    size_t lds;
};

static q4_plan q4_plan_of(const q4_shape &s, int type, int batch)
{
    q4_plan p;
    const int pieces = type == DN_F32 ? 2 : 1, x_tiles = (int)(((long)batch + 15) / 16);
    p.ksplit = p.h = p.t = p.r = 1;
    p.gy = p.gz = 1;
    p.run = s.kblocks;
    while (p.h < 4 && (long)s.tiles * p.h <= 128 && s.kblocks > p.h) p.h *= 2;
    const int steps = (s.kblocks + p.h - 1) / p.h;
    p.lds = batch * ((size_t)steps * p.h * (p.h > 1 ? 272 : 256) * pieces + 16) + (size_t)steps * p.h * (type == DN_I8 ? 128 / s.group : 1) * 16;
    if (batch <= 4 && p.lds <= 150 << 10) {
        p.form = q4_plan::DIRECT;
        /* waves share outputs as long as each has blocks and two workgroups a CU are not reached */
        while (p.ksplit < Q4_WAVES && (long)s.tiles * p.h * p.ksplit <= 256 * Q4_WAVES && p.ksplit * 2 <= steps) p.ksplit *= 2;
        const long groups = ((long)s.tiles * p.h * p.ksplit + Q4_WAVES - 1) / Q4_WAVES;
        p.gx = (unsigned)(groups < 512 ? groups : 512);
        return p;
    }
    p.lds = 0;
    const int passes = (x_tiles + 3) / 4;
    if ((long)s.tiles * x_tiles >= 2300) {
        p.form = q4_plan::STAGED;
        p.t = (x_tiles + passes - 1) / passes;
        p.r = s.group > 32 && (long)s.tiles * passes >= Q4_STAGED_WAVES * 2 * 384 ? 2 : 1;
        p.gx = (unsigned)((s.tiles + Q4_STAGED_WAVES * p.r - 1) / (Q4_STAGED_WAVES * p.r));
    } else {
        p.form = q4_plan::STREAM;
        p.r = s.group > 32 && s.tiles >= 2 * 192 ? 2 : 1;
        p.gx = (unsigned)((s.tiles + p.r - 1) / p.r);
    }
    p.gy = (unsigned)((x_tiles + p.t - 1) / p.t);
    /* Far fewer workgroups than CUs, and long rows: the inputs are cut over workgroups.  The third launch costs some 3 us:
     * 8 x 20787 -> 512 bf16 17.8 us uncut, 12.8 cut; 5 x 22144 -> 1778 19.2 and 16.4; 16 x 8192 -> 1000 10.4 and 10.0;
     * below that nothing. */
    if (p.form == q4_plan::STREAM && s.kblocks >= 64) {
        while ((long)p.gx * p.gy * p.gz * 2 <= 256 && p.run >= 32) {
            p.run = (p.run + 1) / 2;
            p.gz = (unsigned)((s.kblocks + p.run - 1) / p.run);
        }
    }
    return p;
}

extern "C" size_t connected_q4_workspace_bytes(int input_type, int batch, int inputs, int outputs, int group)
{
    if (!q4_shape_ok(inputs, outputs, group) || batch < 1) return 0;
    const q4_shape s = q4_shape_of(inputs, outputs, group);
    const q4_plan p = q4_plan_of(s, input_type, batch);
    if (p.form == q4_plan::DIRECT) return 0;
    const int pieces = input_type == DN_F32 ? 2 : 1;
    return q4_parts_at(s, pieces, batch, input_type == DN_I8) + (p.gz > 1 ? (size_t)p.gz * batch * outputs * 4 : 0);
}

template <int T, int R, int PIECES, int PER, bool XG>
static void q4_launch_second(const q4_args &a, const q4_plan &p)
{
    const dim3 grid(p.gx, p.gy, p.gz);
    if (p.form == q4_plan::STAGED)
        hipLaunchKernelGGL((q4_staged_kernel<T, R, PIECES, PER, XG>), grid, dim3(Q4_STAGED_WAVES * 64), 0, dn_stream(), a);
    else if constexpr (T == 1) {
        hipLaunchKernelGGL((q4_stream_kernel<R, PIECES, PER, XG>), grid, dim3(Q4_THREADS), 0, dn_stream(), a);
        if (p.gz > 1)
            hipLaunchKernelGGL((q4_join_kernel<PIECES, XG>), dim3((unsigned)((a.s.outputs + 255) / 256), (unsigned)a.batch), dim3(256), 0, dn_stream(), a,
                               q4_rows_at(a.s, PIECES, a.batch, XG), q4_parts_at(a.s, PIECES, a.batch, XG), (int)p.gz);
    }
}

template <int TI, int PER, bool XG>
static void q4_launch(const q4_args &a, const q4_plan &p)
{
    constexpr int PIECES = TI == DN_F32 ? 2 : 1;
    if (p.form == q4_plan::DIRECT) {
        const dim3 grid(p.gx), block(Q4_THREADS);
        if (p.h == 1) hipLaunchKernelGGL((q4_direct_kernel<TI, PER, XG, 1>), grid, block, p.lds, dn_stream(), a);
        else if (p.h == 2) hipLaunchKernelGGL((q4_direct_kernel<TI, PER, XG, 2>), grid, block, p.lds, dn_stream(), a);
        else hipLaunchKernelGGL((q4_direct_kernel<TI, PER, XG, 4>), grid, block, p.lds, dn_stream(), a);
        return;
    }
    if (a.s.inputs > 4096) hipLaunchKernelGGL((q4_prepare_kernel<TI, XG, 1024>), dim3((unsigned)a.batch), dim3(1024), 0, dn_stream(), a);
    else hipLaunchKernelGGL((q4_prepare_kernel<TI, XG, 256>), dim3((unsigned)a.batch), dim3(256), 0, dn_stream(), a);
    if constexpr (PER < 4) /* four groups in a block fill the registers with R = 1 */
        if (p.r == 2) {
            if (p.t == 1) q4_launch_second<1, 2, PIECES, PER, XG>(a, p);
            else if (p.t == 2) q4_launch_second<2, 2, PIECES, PER, XG>(a, p);
            else if (p.t == 3) q4_launch_second<3, 2, PIECES, PER, XG>(a, p);
            else q4_launch_second<4, 2, PIECES, PER, XG>(a, p);
            return;
        }
    if (p.t == 1) q4_launch_second<1, 1, PIECES, PER, XG>(a, p);
    else if (p.t == 2) q4_launch_second<2, 1, PIECES, PER, XG>(a, p);
    else if (p.t == 3) q4_launch_second<3, 1, PIECES, PER, XG>(a, p);
    else q4_launch_second<4, 1, PIECES, PER, XG>(a, p);
}

template <int TI, bool XG>
static void q4_launch_group(const q4_args &a, const q4_plan &p)
{
    if (a.s.group == 32) q4_launch<TI, 4, XG>(a, p);
    else if (a.s.group == 64) q4_launch<TI, 2, XG>(a, p);
    else q4_launch<TI, 1, XG>(a, p);
}

extern "C" int forward_connected_q4_gpu(const void *input, int input_type, const float *input_scales, int input_group,
                                        const void *packed, const float *biases, void *output, int output_type,
                                        int batch, int inputs, int outputs, int group, int activation, void *workspace)
{
    const char *me = "forward_connected_q4_gpu";
    if (!dn_is_float_type(input_type) && input_type != DN_I8) return dn_refuse(me, "unknown input type");
    if (!dn_is_float_type(output_type)) return dn_refuse(me, "unknown output type");
    if (batch < 0 || !q4_shape_ok(inputs, outputs, group)) return dn_refuse(me, "bad geometry (group must be 32, 64 or 128)");
    if (activation < 0 || activation > DN_SELU) return dn_refuse(me, "unknown activation");
    if (batch == 0) return 0;
    if (!input || !packed || !output) return dn_refuse(me, "a buffer is missing");
    if (input_type == DN_I8 && !input_scales) return dn_refuse(me, "8-bit input needs its scales");
    if (input_type == DN_I8 && input_group != 0 && input_group != group)
        return dn_refuse(me, "input_group must be 0 (the row) or the weights' group");
    if (!dn_aligned(input, dn_type_bytes(input_type)) || !dn_aligned(output, dn_type_bytes(output_type)) ||
        (input_type == DN_I8 && !dn_aligned(input_scales, 4)) || !dn_aligned(biases, 4) || !dn_aligned(packed, 16) || !dn_aligned(workspace, 16))
        return dn_refuse(me, "a buffer is not aligned to its element type, or packed or workspace not to 16 bytes");
    const q4_shape s = q4_shape_of(inputs, outputs, group);
    const bool xg = input_type == DN_I8 && input_group != 0;
    const q4_plan p = q4_plan_of(s, input_type, batch);
    if (p.form != q4_plan::DIRECT && !workspace) return dn_refuse(me, "the workspace is missing");
    if (p.gx > 0x7fffffu || p.gy > 65535u) return dn_refuse(me, "too many outputs or rows for one call");
    hip_require_device(me);
    const q4_args a = {input, input_scales, (const unsigned char *)packed, biases, output, (unsigned char *)workspace,
                       output_type, input_type == DN_F32 || input_type == DN_BF16, batch, xg ? input_group : 0, activation, p.ksplit, p.run, s};
    if (input_type == DN_F32) q4_launch_group<DN_F32, false>(a, p);
    else if (input_type == DN_F16) q4_launch_group<DN_F16, false>(a, p);
    else if (input_type == DN_BF16) q4_launch_group<DN_BF16, false>(a, p);
    else if (xg) q4_launch_group<DN_I8, true>(a, p);
    else q4_launch_group<DN_I8, false>(a, p);
    dn_check_launch(me);
    return 0;
}
