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
 * Behind the codes the scales, [outputs / 16][groups][16] floats, and the zeros, [outputs / 16][inputs / 128]
 * [16][groups in 128] bytes.  What fills the last tiles up has code, scale and zero 0.
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
    return inputs >= 1 && outputs >= 1 && inputs <= 0x7fffff80 && (group == 32 || group == 64 || group == 128);
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
    return ((long)(o >> 4) * s.groups + g) * 16 + (o & 15);
}
__device__ __forceinline__ long q4_zero_at(const q4_shape &s, int o, int g)
{
    const int per = 128 / s.group;
    return s.zeros_at + (((long)(o >> 4) * s.kblocks + g / per) * 16 + (o & 15)) * per + g % per;
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
            packed[q4_zero_at(s, o, g)] = in ? (zeros ? zeros[(long)o * groups + g] & 15 : 8) : 0;
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
        packed[q4_zero_at(s, o, g)] = (unsigned char)zero;
    }
}

__global__ void q4_unpack_kernel(const unsigned char *packed, float *weights, q4_shape s)
{
    const long total = (long)s.outputs * s.inputs;
    for (long t = blockIdx.x * (long)blockDim.x + threadIdx.x; t < total; t += (long)gridDim.x * blockDim.x) {
        const int o = (int)(t / s.inputs), k = (int)(t % s.inputs);
        const long at = q4_group_at(s, o, k / s.group);
        const int code = (((const unsigned *)packed)[q4_dword_at(s, o, k)] >> q4_bit_of(k)) & 15;
        weights[t] = (float)(code - (int)packed[q4_zero_at(s, o, k / s.group)]) * ((const float *)(packed + s.scales_at))[at];
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
 * On the fp16 matrix instruction: code - zero is a whole number of at most 15, exact in fp16.  A row of the
 * input is scaled by a power of two that brings its largest value to 2^14 .. 2^15 and held as one fp16 value (8-bit,
 * fp16 and bf16 input: exact, short of values 2^-29 below the row's largest) or as the sum of two (fp32 input:
 * to 2^-23 of each value).  Products are exact in the fp32 accumulators, which a group starts
 * from zero; its sum is then multiplied with the scale and added to the output's.  A row with a value that is
 * not finite gets NaN for the factor that undoes its scaling. */
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));

#define Q4_THREADS 512 /* 8 waves */
#define Q4_WAVES 8

struct q4_args {
    const void *input;
    const float *input_scales;
    const unsigned char *packed;
    const float *biases;
    void *output;
    unsigned char *workspace;
    int input_type, output_type;
    int batch, x_group; /* x_group: 0, or the inputs that share one of input_scales */
    int activation;
    int ksplit;         /* waves of a workgroup that share a row tile, each taking a part of the inputs */
    int chunk;          /* staged form: 128-input blocks in LDS at a time */
    q4_shape s;
};

/* The exponent a row is scaled by, from the largest of its absolute values' bits; 0x7fffffff: not finite. */
__device__ __forceinline__ int q4_row_shift(unsigned largest)
{
    if (largest >= 0x7f800000u) return 0x7fffffff;
    if (largest == 0) return 0;
    int e;
    (void)frexpf(__uint_as_float(largest), &e); /* largest < 2^e */
    return 15 - e;
}

__device__ __forceinline__ float q4_row_factor(int shift)
{
    return shift == 0x7fffffff ? __uint_as_float(0x7fc00000u) : 1.f;
}

/* Four inputs from k on (zeros behind the row's end). */
template <int TI>
__device__ __forceinline__ void q4_load4(const void *row, int k, int inputs, bool vectors, float x[4])
{
    typedef typename dn_elt<TI>::store E;
    typedef E E4 __attribute__((ext_vector_type(4)));
    const E *p = (const E *)row + k;
    if (vectors && k + 4 <= inputs) {
        const E4 v = *(const E4 *)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = k + i < inputs ? (float)p[i] : 0.f;
    }
}

__device__ __forceinline__ unsigned q4_largest4(unsigned m, const float x[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
}

/* The operand form of four inputs: hi, and what it leaves of the value in lo. */
__device__ __forceinline__ void q4_split4(const float x[4], int shift, half4_t &hi, half4_t &lo)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = ldexpf(x[i], shift);
        hi[i] = (_Float16)v;
        lo[i] = (_Float16)(v - (float)hi[i]);
    }
}

/* One tile of 16 outputs x 128 inputs as a lane holds it; PER groups in 128 inputs. */
template <int PER>
struct q4_tile {
    uint4 code;
    float4_t scale[PER]; /* of the lane's four outputs of the result */
    unsigned zero;       /* of the lane's output of the operand, a byte for each group */
};

template <int PER>
__device__ __forceinline__ q4_tile<PER> q4_load_tile(const q4_args &a, int tile, int kb, int lane)
{
    q4_tile<PER> t;
    const long at = (long)tile * a.s.kblocks + kb;
    t.code = ((const uint4 *)a.packed)[at * 64 + lane];
#pragma unroll
    for (int g = 0; g < PER; ++g)
        t.scale[g] = ((const float4_t *)(a.packed + a.s.scales_at))[(at * PER + g) * 4 + (lane >> 4)];
    const unsigned char *z = a.packed + a.s.zeros_at + (at * 16 + (lane & 15)) * PER;
    t.zero = PER == 4 ? *(const unsigned *)z : PER == 2 ? *(const unsigned short *)z : *z;
    return t;
}

__device__ __forceinline__ half2_t q4_as_half2(unsigned v) { return __builtin_bit_cast(half2_t, v); }

/* Eight codes less their zero as fp16: 0x6400 | c is 1024 + c, and with the code four bits up 1024 + 16 c. */
__device__ __forceinline__ half8_t q4_unpack8(unsigned v, unsigned zero)
{
    const unsigned z2 = zero | zero << 16;
    const half2_t z1024 = q4_as_half2(0xe400e400u | z2), z64 = q4_as_half2(0xd400d400u | z2 << 4); /* -(1024 + z), -(64 + z) */
    const half2_t sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const unsigned w = v >> 8;
    const half2_t a = q4_as_half2((v & 0x000f000fu) | 0x64006400u) + z1024;
    const half2_t b = __builtin_elementwise_fma(q4_as_half2((v & 0x00f000f0u) | 0x64006400u), sixteenth, z64);
    const half2_t c = q4_as_half2((w & 0x000f000fu) | 0x64006400u) + z1024;
    const half2_t d = __builtin_elementwise_fma(q4_as_half2((w & 0x00f000f0u) | 0x64006400u), sixteenth, z64);
    return (half8_t){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float4_t q4_mfma(half8_t a, half8_t b, float4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

/* Adds the products of one tile with T tiles of 16 input rows.  operand(t, piece, step): the lane's eight
 * inputs; x_scale(t, g): the input's own scale of the group, where it has one (XG). */
template <int T, int PIECES, int PER, bool XG, class Operand, class Scale>
__device__ __forceinline__ void q4_multiply(const q4_tile<PER> &w, float4_t (&sum)[T], Operand operand, Scale x_scale)
{
    const unsigned code[4] = {w.code.x, w.code.y, w.code.z, w.code.w};
#pragma unroll
    for (int g = 0; g < PER; ++g) {
        float4_t acc[T];
        const unsigned zero = (w.zero >> (8 * g)) & 0xff;
#pragma unroll
        for (int i = 0; i < 4 / PER; ++i) {
            const int step = g * (4 / PER) + i;
            const half8_t av = q4_unpack8(code[step], zero);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                acc[t] = q4_mfma(av, operand(t, 0, step), i ? acc[t] : (float4_t){0, 0, 0, 0});
                if (PIECES == 2) acc[t] = q4_mfma(av, operand(t, 1, step), acc[t]);
            }
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float4_t f = XG ? w.scale[g] * x_scale(t, g) : w.scale[g];
            sum[t] = __builtin_elementwise_fma(acc[t], f, sum[t]);
        }
    }
}

/* Four neighbouring outputs of one input row: undoes the row's scaling, bias, activation, rounding, store. */
__device__ __forceinline__ void q4_store4(const q4_args &a, int b, int o, float4_t v, int shift, float factor)
{
    if (b >= a.batch) return;
    const long at = (long)b * a.s.outputs + o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float y = ldexpf(v[i], -shift) * factor;
        if (o + i >= a.s.outputs) continue;
        if (a.biases) y += a.biases[o + i];
        y = a.activation == DN_LINEAR ? y : dn_activate(y, a.activation);
        if (a.output_type == DN_F32) ((float *)a.output)[at + i] = y;
        else if (a.output_type == DN_F16) ((_Float16 *)a.output)[at + i] = (_Float16)y;
        else ((__bf16 *)a.output)[at + i] = (__bf16)y;
    }
}

/* Adds what the waves of a row tile have, in the order of the waves, and stores it.  `red`: 8 KB. */
__device__ __forceinline__ void q4_join(const q4_args &a, float4_t (*red)[64], float4_t own, int tile, int b0, int shift, float factor)
{
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (a.ksplit > 1) {
        __syncthreads();
        red[wave][lane] = own;
        __syncthreads();
        if (wave % a.ksplit) return;
        for (int q = 1; q < a.ksplit; ++q) own += red[wave + q][lane];
    }
    if (tile < a.s.tiles) q4_store4(a, b0 + (lane & 15), tile * 16 + (lane >> 4) * 4, own, shift, factor);
}

/* Small input (the whole of it in LDS, at most 16 rows): each workgroup scales and splits the input itself and
 * then streams row tiles of the weights, the next tiles' loads in flight over the current ones' products. */
template <int TI, int PER, bool XG>
__global__ __launch_bounds__(Q4_THREADS) void q4_direct_kernel(q4_args a)
{
    constexpr int PIECES = TI == DN_F32 ? 2 : 1;
    constexpr int AHEAD = 4; /* blocks in flight */
    extern __shared__ char lds[];
    __shared__ unsigned s_largest[16][Q4_WAVES];
    __shared__ float4_t s_red[Q4_WAVES][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kpad = a.s.kblocks * 128, pitch = kpad * 2 * PIECES + 16; /* bytes of a row: 16 more, for the banks */
    const int part = wave % a.ksplit, rows_per = Q4_WAVES / a.ksplit;
    const int mine = (a.s.kblocks - part + a.ksplit - 1) / a.ksplit; /* this wave's blocks: part, part + ksplit, ... */
    const int stride = gridDim.x * rows_per;
    int tile = blockIdx.x * rows_per + wave / a.ksplit;

    /* block n of this wave in a row tile; one behind the last counts nothing */
    auto fetch = [&](int t, int n) {
        q4_tile<PER> w = q4_load_tile<PER>(a, min(t, a.s.tiles - 1), part + a.ksplit * min(n, mine - 1), lane);
        if (n >= mine)
#pragma unroll
            for (int g = 0; g < PER; ++g) w.scale[g] = (float4_t){0, 0, 0, 0};
        return w;
    };
    q4_tile<PER> w[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) w[u] = fetch(tile, u);

    const size_t row_bytes = (size_t)a.s.inputs * (TI == DN_F32 ? 4 : TI == DN_I8 ? 1 : 2);
    const bool vectors = ((uintptr_t)a.input & 15) == 0 && (row_bytes & 15) == 0;
    if (TI != DN_I8) {
        for (int b = 0; b < a.batch; ++b) {
            unsigned m = 0;
            for (int k = tid * 4; k < a.s.inputs; k += Q4_THREADS * 4) {
                float x[4];
                q4_load4<TI>((const char *)a.input + b * row_bytes, k, a.s.inputs, vectors, x);
                m = q4_largest4(m, x);
            }
            m = dn_wave_max(m);
            if (lane == 0) s_largest[b][wave] = m;
        }
        __syncthreads();
    }
    auto shift_of = [&](int b) {
        if (TI == DN_I8) return 0;
        unsigned m = s_largest[b][0];
#pragma unroll
        for (int w = 1; w < Q4_WAVES; ++w) m = max(m, s_largest[b][w]);
        return q4_row_shift(m);
    };
    for (int b = 0; b < a.batch; ++b) {
        const int sh = shift_of(b);
        for (int k = tid * 4; k < kpad; k += Q4_THREADS * 4) {
            float x[4];
            half4_t hi, lo;
            q4_load4<TI>((const char *)a.input + b * row_bytes, k, a.s.inputs, vectors, x);
            q4_split4(x, sh == 0x7fffffff ? 0 : sh, hi, lo);
            *(half4_t *)(lds + b * pitch + k * 2) = hi;
            if (PIECES == 2) *(half4_t *)(lds + b * pitch + kpad * 2 + k * 2) = lo;
        }
    }
    const int x_groups = XG ? (a.s.inputs + a.x_group - 1) / a.x_group : 1;
    float *x_scales = (float *)(lds + a.batch * pitch); /* [row][group], only XG */
    if (XG)
        for (int i = tid; i < a.batch * a.s.groups; i += Q4_THREADS) {
            const int b = i / a.s.groups, g = i % a.s.groups;
            x_scales[i] = g < x_groups ? a.input_scales[(long)b * x_groups + g] : 0.f;
        }
    const int col = min(lane & 15, a.batch - 1);
    int shift = shift_of(col);
    float factor = TI == DN_I8 ? (XG ? 1.f : a.input_scales[col]) : q4_row_factor(shift);
    if (shift == 0x7fffffff) shift = 0;
    __syncthreads();

    const char *base = lds + col * pitch + (lane >> 4) * 16;
    for (; tile - wave / a.ksplit < a.s.tiles; tile += stride) {
        float4_t sum[1] = {{0, 0, 0, 0}};
        for (int n = 0; n < mine; n += AHEAD) {
            const bool last = n + AHEAD >= mine; /* what comes next is of the next row tile */
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int kb = part + a.ksplit * min(n + u, mine - 1);
                q4_multiply<1, PIECES, PER, XG>(
                    w[u], sum,
                    [&](int, int piece, int step) { return *(const half8_t *)(base + piece * kpad * 2 + kb * 256 + step * 64); },
                    [&](int, int g) { return x_scales[col * a.s.groups + kb * PER + g]; });
                w[u] = fetch(last ? tile + stride : tile, last ? u : n + AHEAD + u);
            }
        }
        q4_join(a, s_red, sum[0], tile, 0, shift, factor);
    }
}

/* Larger input, first pass: one workgroup for each row scales it and writes it in the order in which the second
 * pass feeds it to the matrix instruction: [row / 16][inputs / 128][piece][step][lane][8 halves].  Behind that
 * [row] factors and shifts and, for 8-bit input with groups, [row / 16][groups][16] scales. */
struct q4_space {
    size_t rows_at, scales_at, bytes;
};

__host__ __device__ static inline q4_space q4_space_of(const q4_shape &s, int pieces, int batch, bool groups)
{
    q4_space w;
    const size_t tiles = ((size_t)batch + 15) / 16;
    w.rows_at = tiles * s.kblocks * pieces * 4096;
    w.scales_at = w.rows_at + tiles * 16 * 8;
    w.bytes = w.scales_at + (groups ? tiles * s.groups * 64 : 0);
    return w;
}

template <int TI>
__global__ __launch_bounds__(256) void q4_prepare_kernel(q4_args a)
{
    constexpr int PIECES = TI == DN_F32 ? 2 : 1;
    __shared__ unsigned s_largest[4];
    const int tid = threadIdx.x, b = blockIdx.x;
    const bool xg = TI == DN_I8 && a.x_group;
    const q4_space ws = q4_space_of(a.s, PIECES, a.batch, xg);
    const size_t row_bytes = (size_t)a.s.inputs * (TI == DN_F32 ? 4 : TI == DN_I8 ? 1 : 2);
    const bool vectors = ((uintptr_t)a.input & 15) == 0 && (row_bytes & 15) == 0;
    const char *row = (const char *)a.input + b * row_bytes;
    int shift = 0;
    if (TI != DN_I8) {
        unsigned m = 0;
        for (int k = tid * 4; k < a.s.inputs; k += 1024) {
            float x[4];
            q4_load4<TI>(row, k, a.s.inputs, vectors, x);
            m = q4_largest4(m, x);
        }
        m = dn_wave_max(m);
        if ((tid & 63) == 0) s_largest[tid >> 6] = m;
        __syncthreads();
        shift = q4_row_shift(max(max(s_largest[0], s_largest[1]), max(s_largest[2], s_largest[3])));
    }
    if (tid == 0) {
        ((float *)(a.workspace + ws.rows_at))[2 * b] = TI == DN_I8 ? (xg ? 1.f : a.input_scales[b]) : q4_row_factor(shift);
        ((int *)(a.workspace + ws.rows_at))[2 * b + 1] = shift == 0x7fffffff ? 0 : shift;
    }
    if (shift == 0x7fffffff) shift = 0;
    unsigned char *out = a.workspace + (size_t)(b >> 4) * a.s.kblocks * PIECES * 4096 + (b & 15) * 16;
    for (int k = tid * 8; k < a.s.kblocks * 128; k += 2048) {
        float x[8];
        half4_t hi[2], lo[2];
        q4_load4<TI>(row, k, a.s.inputs, vectors, x);
        q4_load4<TI>(row, k + 4, a.s.inputs, vectors, x + 4);
        q4_split4(x, shift, hi[0], lo[0]);
        q4_split4(x + 4, shift, hi[1], lo[1]);
        unsigned char *to = out + (size_t)(k >> 7) * PIECES * 4096 + ((k >> 5) & 3) * 1024 + ((k >> 3) & 3) * 256;
        ((half4_t *)to)[0] = hi[0];
        ((half4_t *)to)[1] = hi[1];
        if (PIECES == 2) {
            ((half4_t *)(to + 4096))[0] = lo[0];
            ((half4_t *)(to + 4096))[1] = lo[1];
        }
    }
    if (xg) {
        const int x_groups = (a.s.inputs + a.x_group - 1) / a.x_group;
        float *to = (float *)(a.workspace + ws.scales_at) + ((size_t)(b >> 4) * a.s.groups) * 16 + (b & 15);
        for (int g = tid; g < a.s.groups; g += 256) to[g * 16] = g < x_groups ? a.input_scales[(long)b * x_groups + g] : 0.f;
    }
}

/* Second pass: a workgroup takes 8 / ksplit * R row tiles and T tiles of 16 input rows.  The input goes through
 * LDS in chunks that all its waves read; each wave's own weights come straight from memory, a chunk ahead. */
__host__ __device__ constexpr int q4_units(int r, int per) /* blocks of a wave in a chunk, at most */
{
    return per == 4 ? 2 / r : 4 / r;
}

template <int T, int R, int PIECES, int PER, bool XG>
__global__ __launch_bounds__(Q4_THREADS) void q4_staged_kernel(q4_args a)
{
    constexpr int UNITS = q4_units(R, PER);
    extern __shared__ char lds[];
    __shared__ float4_t s_red[Q4_WAVES][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const q4_space ws = q4_space_of(a.s, PIECES, a.batch, XG);
    const int part = wave % a.ksplit, x_tiles = (a.batch + 15) / 16, x0 = blockIdx.y * T;
    const int tile0 = (blockIdx.x * (Q4_WAVES / a.ksplit) + wave / a.ksplit) * R;
    const int units = a.chunk / a.ksplit, chunks = (a.s.kblocks + a.chunk - 1) / a.chunk;
    const float *x_scales = (const float *)(a.workspace + ws.scales_at);
    float4_t sum[R][T];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) sum[r][t] = (float4_t){0, 0, 0, 0};

    auto fetch = [&](int c, int u, int r) {
        const int kb = c * a.chunk + part + u * a.ksplit;
        q4_tile<PER> w = q4_load_tile<PER>(a, min(tile0 + r, a.s.tiles - 1), min(kb, a.s.kblocks - 1), lane);
        if (kb >= a.s.kblocks)
#pragma unroll
            for (int g = 0; g < PER; ++g) w.scale[g] = (float4_t){0, 0, 0, 0};
        return w;
    };
    q4_tile<PER> w[UNITS][R];
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (u < units) w[u][r] = fetch(0, u, r);
    const int block = PIECES * 4096, span = a.chunk * block; /* bytes of one input tile's block, and of its chunk */
    for (int c = 0; c < chunks; ++c) {
        /* stage chunk c: blocks behind the last are not read by a product with a scale, but must be finite */
        __syncthreads();
        for (int i = tid * 16; i < T * span; i += Q4_THREADS * 16) {
            const int t = i / span, in = i % span, kb = c * a.chunk + in / block;
            uint4 v = {0, 0, 0, 0};
            if (x0 + t < x_tiles && kb < a.s.kblocks)
                v = *(const uint4 *)(a.workspace + ((size_t)(x0 + t) * a.s.kblocks + c * a.chunk) * block + in);
            *(uint4 *)(lds + i) = v;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            if (u >= units) break;
            const int at = part + u * a.ksplit, kb = min(c * a.chunk + at, a.s.kblocks - 1);
            const char *base = lds + at * block + lane * 16;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                q4_multiply<T, PIECES, PER, XG>(
                    w[u][r], sum[r],
                    [&](int t, int piece, int step) { return *(const half8_t *)(base + t * span + piece * 4096 + step * 1024); },
                    [&](int t, int g) {
                        return x_scales[((size_t)min(x0 + t, x_tiles - 1) * a.s.groups + kb * PER + g) * 16 + (lane & 15)];
                    });
                w[u][r] = fetch(c + 1, u, r);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const int b0 = (x0 + t) * 16, b = min(b0 + (lane & 15), a.batch - 1);
        const float factor = ((const float *)(a.workspace + ws.rows_at))[2 * b];
        const int shift = ((const int *)(a.workspace + ws.rows_at))[2 * b + 1];
#pragma unroll
        for (int r = 0; r < R; ++r) q4_join(a, s_red, sum[r][t], tile0 + r, b0, shift, factor);
    }
}

/* Which form a product takes.  Direct: up to 16 rows and 16384 inputs in all (what a workgroup can scale while its
 * first weights arrive). */
struct q4_plan {
    bool direct;
    int pieces, ksplit, t, r, chunk;
    unsigned gx, gy;
    size_t lds;
};

static q4_plan q4_plan_of(const q4_shape &s, int type, int batch, bool xg)
{
    q4_plan p;
    p.pieces = type == DN_F32 ? 2 : 1;
    p.t = p.r = p.chunk = 1;
    p.gy = 1;
    const size_t pitch = (size_t)s.kblocks * 256 * p.pieces + 16, need = batch * (pitch + (xg ? (size_t)s.groups * 4 : 0));
    p.direct = batch <= 16 && (long)batch * s.inputs <= 16384 && need <= 128 << 10;
    if (p.direct) {
        p.lds = need;
        /* waves share a row tile as long as that leaves each of them a block and the chip is not full */
        p.ksplit = 1;
        while (p.ksplit < 8 && (long)s.tiles * p.ksplit < 256 * Q4_WAVES && p.ksplit * 2 <= s.kblocks) p.ksplit *= 2;
        const int groups = (s.tiles * p.ksplit + Q4_WAVES - 1) / Q4_WAVES;
        p.gx = groups < 512 ? groups : 512;
        return p;
    }
    const int x_tiles = (batch + 15) / 16, passes = (x_tiles + 3) / 4;
    auto grid = [&]() {
        const int per = Q4_WAVES / p.ksplit * p.r;
        p.gx = (unsigned)((s.tiles + per - 1) / per);
        p.gy = (unsigned)((x_tiles + p.t - 1) / p.t);
        return (long)p.gx * p.gy;
    };
    p.t = (x_tiles + passes - 1) / passes;
    p.ksplit = 1;
    p.r = 2;
    if (grid() < 256) p.r = 1;
    while (grid() < 256 && p.ksplit < 8) {
        if (p.t * p.pieces * p.ksplit * 2 <= 16) p.ksplit *= 2;
        else if (p.t > 1) p.t = (p.t + 1) / 2;
        else break;
    }
    grid();
    const int most = 16 / (p.t * p.pieces) > 0 ? 16 / (p.t * p.pieces) : 1; /* blocks in 64 KB */
    p.chunk = most / p.ksplit * p.ksplit;
    if (p.chunk < p.ksplit) p.chunk = p.ksplit;
    const int units = q4_units(p.r, 128 / s.group);
    if (p.chunk > units * p.ksplit) p.chunk = units * p.ksplit;
    p.lds = (size_t)p.t * p.chunk * p.pieces * 4096;
    return p;
}

extern "C" size_t connected_q4_workspace_bytes(int input_type, int batch, int inputs, int outputs, int group)
{
    if (!q4_shape_ok(inputs, outputs, group) || batch < 1) return 0;
    const q4_shape s = q4_shape_of(inputs, outputs, group);
    if (q4_plan_of(s, input_type, batch, input_type == DN_I8).direct) return 0;
    return q4_space_of(s, input_type == DN_F32 ? 2 : 1, batch, input_type == DN_I8).bytes;
}

template <int TI, int PER, bool XG>
static void q4_launch_direct(const q4_args &a, const q4_plan &p)
{
    hipLaunchKernelGGL((q4_direct_kernel<TI, PER, XG>), dim3(p.gx), dim3(Q4_THREADS), p.lds, dn_stream(), a);
}

template <int T, int PIECES, int PER, bool XG>
static void q4_launch_staged(const q4_args &a, const q4_plan &p)
{
    const dim3 grid(p.gx, p.gy), block(Q4_THREADS);
    if (p.r == 2) hipLaunchKernelGGL((q4_staged_kernel<T, 2, PIECES, PER, XG>), grid, block, p.lds, dn_stream(), a);
    else hipLaunchKernelGGL((q4_staged_kernel<T, 1, PIECES, PER, XG>), grid, block, p.lds, dn_stream(), a);
}

template <int TI, int PER, bool XG>
static void q4_launch(const q4_args &a, const q4_plan &p)
{
    constexpr int PIECES = TI == DN_F32 ? 2 : 1;
    if (p.direct) {
        q4_launch_direct<TI, PER, XG>(a, p);
        return;
    }
    hipLaunchKernelGGL((q4_prepare_kernel<TI>), dim3((unsigned)a.batch), dim3(256), 0, dn_stream(), a);
    if (p.t == 1) q4_launch_staged<1, PIECES, PER, XG>(a, p);
    else if (p.t == 2) q4_launch_staged<2, PIECES, PER, XG>(a, p);
    else if (p.t == 3) q4_launch_staged<3, PIECES, PER, XG>(a, p);
    else q4_launch_staged<4, PIECES, PER, XG>(a, p);
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
    if (!input || !packed || !output) return dn_refuse(me, "a buffer is missing");
    if (input_type == DN_I8 && !input_scales) return dn_refuse(me, "8-bit input needs its scales");
    if (input_type == DN_I8 && input_group != 0 && input_group != group)
        return dn_refuse(me, "input_group must be 0 (the row) or the weights' group");
    if (!dn_aligned(input, dn_type_bytes(input_type)) || !dn_aligned(output, dn_type_bytes(output_type)) ||
        !dn_aligned(input_scales, 4) || !dn_aligned(biases, 4) || !dn_aligned(packed, 16) || !dn_aligned(workspace, 16))
        return dn_refuse(me, "a buffer is not aligned to its element type, or packed or workspace not to 16 bytes");
    if (batch == 0) return 0;
    const q4_shape s = q4_shape_of(inputs, outputs, group);
    const bool xg = input_type == DN_I8 && input_group != 0;
    const q4_plan p = q4_plan_of(s, input_type, batch, input_type == DN_I8);
    if (!p.direct && !workspace) return dn_refuse(me, "the workspace is missing");
    if (p.gx > 0x7fffffu || p.gy > 65535u) return dn_refuse(me, "too many outputs or rows for one call");
    hip_require_device(me);
    const q4_args a = {input, input_scales, (const unsigned char *)packed, biases, output, (unsigned char *)workspace,
                       input_type, output_type, batch, xg ? input_group : 0, activation, p.ksplit, p.chunk, s};
    if (input_type == DN_F32) q4_launch_group<DN_F32, false>(a, p);
    else if (input_type == DN_F16) q4_launch_group<DN_F16, false>(a, p);
    else if (input_type == DN_BF16) q4_launch_group<DN_BF16, false>(a, p);
    else if (xg) q4_launch_group<DN_I8, true>(a, p);
    else q4_launch_group<DN_I8, false>(a, p);
    dn_check_launch(me);
    return 0;
}
