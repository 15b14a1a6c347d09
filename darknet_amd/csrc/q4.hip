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
 * On the fp16 matrix instruction: code - zero is a whole number of at most 15, exact in fp16.  The input is
 * scaled by a power of two that brings its largest value to 2^14 .. 2^15 and held as one fp16 value (8-bit, fp16
 * and bf16 input: exact, short of values 2^-29 below the largest) or as the sum of two (fp32 input: to
 * 2^-23 of each value).  Products are exact in the fp32 accumulators, which a group starts from zero; its sum
 * is then multiplied with the scale and added to the output's.  Where a value is not finite the factor that
 * undoes the scaling is NaN.
 *
 * The input is the instruction's first operand and the weights the second, so that a lane's results are those
 * of one output, whose scale and zero it has read beside the codes. */
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
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
    int batch, x_group; /* x_group: 0, or the inputs that share one of input_scales */
    int activation;
    int ksplit; /* direct form: waves of a workgroup that share a row tile, each taking a part of the inputs */
    q4_shape s;
};

/* The exponent that values are scaled by, from the largest of their absolute values' bits, and the factor that undoes
 * it: a power of two, NaN if a value is not finite. */
__device__ __forceinline__ int q4_shift(unsigned largest, float &factor)
{
    int e = 15;
    if (largest - 1u < 0x7f7fffffu) (void)frexpf(__uint_as_float(largest), &e); /* largest < 2^e */
    const int shift = min(15 - e, 126);                                        /* 2^-126: the factor is not rounded */
    factor = largest < 0x7f800000u ? ldexpf(1.f, -shift) : __uint_as_float(0x7fc00000u);
    return shift;
}

/* Four inputs from k on (zeros behind the row's end), in one access where they exist, whatever their alignment. */
template <int TI>
__device__ __forceinline__ void q4_load4(const void *row, int k, int inputs, float x[4])
{
    typedef typename dn_elt<TI>::store E;
    typedef E E4 __attribute__((ext_vector_type(4)));
    typedef E4 E4U __attribute__((aligned(sizeof(E))));
    const E *p = (const E *)row + k;
    if (k + 4 <= inputs) {
        const E4 v = *(const E4U *)p;
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
    uint4_t code;
    float scale[PER];
    unsigned zero; /* a byte for each group */
};

template <int PER>
__device__ __forceinline__ q4_tile<PER> q4_load_tile(const q4_args &a, int tile, int kb, int lane)
{
    typedef float scales_t __attribute__((ext_vector_type(PER)));
    q4_tile<PER> t;
    const long at = (long)tile * a.s.kblocks + kb, own = (at * 16 + (lane & 15)) * PER;
    t.code = ((const uint4_t *)a.packed)[at * 64 + lane];
    const float *scale = (const float *)(a.packed + a.s.scales_at) + own;
    const unsigned char *z = a.packed + a.s.zeros_at + own;
    if constexpr (PER == 1) {
        t.scale[0] = *scale;
        t.zero = *z;
    } else {
        const scales_t v = *(const scales_t *)scale;
#pragma unroll
        for (int g = 0; g < PER; ++g) t.scale[g] = v[g];
        t.zero = PER == 4 ? *(const unsigned *)z : *(const unsigned short *)z;
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

/* Adds the products of R tiles of outputs with T tiles of 16 input rows.  operand(t, piece, step): the lane's eight
 * inputs of a row; x_scale(t, g): the factors of its four rows of results, where they change along the row (XS).  ONE:
 * there is one input row, and only the first result of a lane counts. */
template <int T, int R, int PIECES, int PER, bool XS, bool ONE = false, class Operand, class Scale>
__device__ __forceinline__ void q4_multiply(const q4_masks &masks, const q4_tile<PER> (&w)[R], float4_t (&sum)[R][T],
                                            Operand operand, Scale x_scale)
{
#pragma unroll
    for (int g = 0; g < PER; ++g) {
        float4_t acc[R][T];
        half2_t z1024[R], z64[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const unsigned z2 = __builtin_amdgcn_perm(0, w[r].zero, 0x0c000c00u + 0x00010001u * g); /* the byte in both halves */
            z1024[r] = q4_as_half2(0xe400e400u | z2); /* -(1024 + z), -(64 + z) */
            z64[r] = q4_as_half2(0xd400d400u | z2 << 4);
        }
#pragma unroll
        for (int i = 0; i < 4 / PER; ++i) {
            const int step = g * (4 / PER) + i;
            half8_t wv[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const unsigned code = step == 0 ? w[r].code.x : step == 1 ? w[r].code.y : step == 2 ? w[r].code.z : w[r].code.w;
                wv[r] = q4_unpack8(code, z1024[r], z64[r], masks);
            }
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    const half8_t x = operand(t, p, step);
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            x, wv[r], i || p ? acc[r][t] : (float4_t){0, 0, 0, 0}, 0, 0, 0);
                }
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float4_t f = {1, 1, 1, 1};
            if (XS) f = x_scale(t, g);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (ONE) {
                    sum[r][t][0] = fmaf(acc[r][t][0], XS ? f[0] * w[r].scale[g] : w[r].scale[g], sum[r][t][0]);
                    continue;
                }
                const float4_t scale = {w[r].scale[g], w[r].scale[g], w[r].scale[g], w[r].scale[g]};
                sum[r][t] = __builtin_elementwise_fma(acc[r][t], XS ? f * scale : scale, sum[r][t]);
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

/* ---- small input: at most 16 rows that fit into LDS whole.  Each workgroup scales and splits the input itself, block
 * by block of 128 values, and then streams row tiles of the weights, AHEAD blocks of a wave in flight. */
template <int TI, int PER, bool XG, bool ONE>
__global__ __launch_bounds__(Q4_THREADS) void q4_direct_kernel(q4_args a)
{
    constexpr int THREADS = Q4_THREADS, WAVES = Q4_WAVES;
    constexpr int PIECES = TI == DN_F32 ? 2 : 1;
    constexpr int AHEAD = PER == 4 ? 6 : 8, MOVES = 4;
    extern __shared__ char lds[];
    __shared__ float s_red[WAVES][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kpad = a.s.kblocks * 128, pitch = kpad * 2 * PIECES + 16; /* bytes of a row: 16 more, for the banks */
    const int part = wave % a.ksplit, own_tile = wave / a.ksplit, rows_per = WAVES / a.ksplit;
    const int mine = (a.s.kblocks - part + a.ksplit - 1) / a.ksplit; /* this wave's blocks: part, part + ksplit, ... */
    const int stride = gridDim.x * rows_per;
    int tile0 = blockIdx.x * rows_per;

    auto fetch = [&](int t, int n) { return q4_load_tile<PER>(a, min(t, a.s.tiles - 1), part + a.ksplit * n, lane); };
    const q4_masks masks;
    q4_tile<PER> w[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (u < mine) w[u] = fetch(tile0 + own_tile, u);

    /* the input: [row][pitch] halves, and [block (8-bit input with groups: group)][16 rows] factors behind them */
    const size_t row_bytes = (size_t)a.s.inputs * (TI == DN_F32 ? 4 : TI == DN_I8 ? 1 : 2);
    float *factors = (float *)(lds + a.batch * pitch);
    const int quads = kpad / 4;
    for (int b = 0, q = tid; b < a.batch;) {
        float x[MOVES][4];
        int of[MOVES], at[MOVES]; /* row and four of the next items of this lane, whose loads go together */
#pragma unroll
        for (int m = 0; m < MOVES; ++m) {
            const bool in = q < quads; /* (a row shorter than the workgroup leaves some lanes out) */
            of[m] = in ? b : a.batch;
            at[m] = q;
            q4_load4<TI>((const char *)a.input + min(b, a.batch - 1) * row_bytes, min(q, quads - 1) * 4, a.s.inputs, x[m]);
            q += THREADS;
            if (q >= quads) {
                q = tid;
                ++b;
            }
        }
#pragma unroll
        for (int m = 0; m < MOVES; ++m) { /* 32 lanes have a block */
            if (of[m] >= a.batch) continue;
            float factor = 1;
            half4_t hi, lo;
            int shift = 0;
            if (TI != DN_I8) {
                unsigned m4 = q4_largest4(0, x[m]);
                m4 = max(m4, dn_move<0xb1, 0xf>(m4, m4));
                m4 = max(m4, dn_move<0x4e, 0xf>(m4, m4));
                m4 = max(m4, dn_move<0x141, 0xf>(m4, m4));
                m4 = max(m4, dn_move<0x140, 0xf>(m4, m4));
                m4 = max(m4, (unsigned)__shfl_xor((int)m4, 16, 64));
                shift = q4_shift(m4, factor);
                if ((tid & 31) == 0) factors[(at[m] >> 5) * 16 + of[m]] = factor;
            }
            q4_split4(x[m], shift, hi, lo);
            char *to = lds + of[m] * pitch + at[m] * 8;
            *(half4_t *)to = hi;
            if (PIECES == 2) *(half4_t *)(to + kpad * 2) = lo;
        }
    }
    if (XG) {
        const int x_groups = (a.s.inputs + a.x_group - 1) / a.x_group;
        for (int i = tid; i < a.batch * a.s.groups; i += THREADS) {
            const int b = i / a.s.groups, g = i - b * a.s.groups;
            factors[g * 16 + b] = g < x_groups ? a.input_scales[(long)b * x_groups + g] : 0.f;
        }
    }
    __syncthreads();

    constexpr bool XS = TI != DN_I8 || XG;
    const char *base = lds + min(lane & 15, a.batch - 1) * pitch + (lane >> 4) * 16;
    const float *row_factors = factors + (ONE ? 0 : (lane >> 4) * 4);
    for (; tile0 < a.s.tiles; tile0 += stride) {
        const int tile = tile0 + own_tile;
        float4_t sum[1][1] = {{{0, 0, 0, 0}}};
        for (int n = 0; n < mine; n += AHEAD) {
            const bool last = n + AHEAD >= mine; /* what comes next is of the next row tile */
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (n + u < mine) {
                    const int kb = part + a.ksplit * (n + u);
                    const q4_tile<PER> one[1] = {w[u]};
                    q4_multiply<1, 1, PIECES, PER, XS, ONE>(
                        masks, one, sum,
                        [&](int, int piece, int step) { return *(const half8_t *)(base + piece * kpad * 2 + kb * 256 + step * 64); },
                        [&](int, int g) {
                            const float *f = row_factors + (XG ? kb * PER + g : kb) * 16;
                            return ONE ? (float4_t){*f, 0, 0, 0} : *(const float4_t *)f;
                        });
                }
                if (last ? u < mine && tile0 + stride < a.s.tiles : n + AHEAD + u < mine)
                    w[u] = fetch(last ? tile + stride : tile, last ? u : n + AHEAD + u);
            }
        }
        /* what the waves of a row tile have, added in their order; a thread for each output of each row */
        __syncthreads();
#pragma unroll
        for (int i = 0; i < (ONE ? 1 : 4); ++i) s_red[wave][(lane >> 4) * 4 + i][lane & 15] = sum[0][0][i];
        __syncthreads();
        for (int i = tid; i < rows_per * a.batch * 16; i += THREADS) {
            const int r = i / (a.batch * 16), b = (i >> 4) % a.batch, o = (tile0 + r) * 16 + (i & 15);
            if (o >= a.s.outputs) continue;
            const float bias = q4_bias(a, o);
            float y = 0;
#pragma unroll
            for (int q = 0; q < WAVES; ++q)
                if (q < a.ksplit) y += s_red[r * a.ksplit + q][b][i & 15];
            if (TI == DN_I8 && !XG) y *= a.input_scales[b];
            q4_store(a, b, o, y, bias);
        }
    }
}

/* ---- larger input, first pass: one workgroup for each row scales it and writes it in the order in which the second
 * pass feeds it to the matrix instruction: [row / 16][inputs / 128] blocks of [piece][step][lane][8 halves] and, for
 * 8-bit input with groups, [group in 128][16] factors.  Behind the blocks a factor for each row. */
__host__ __device__ static inline int q4_block_bytes(const q4_shape &s, int pieces, bool groups)
{
    return pieces * 4096 + (groups ? 128 / s.group * 64 : 0);
}

__host__ __device__ static inline size_t q4_rows_at(const q4_shape &s, int pieces, int batch, bool groups)
{
    return ((size_t)batch + 15) / 16 * s.kblocks * q4_block_bytes(s, pieces, groups);
}

template <int TI, bool XG>
__global__ __launch_bounds__(256) void q4_prepare_kernel(q4_args a)
{
    constexpr int PIECES = TI == DN_F32 ? 2 : 1;
    __shared__ unsigned s_largest[4];
    const int tid = threadIdx.x, b = blockIdx.x, block = q4_block_bytes(a.s, PIECES, XG);
    const size_t row_bytes = (size_t)a.s.inputs * (TI == DN_F32 ? 4 : TI == DN_I8 ? 1 : 2);
    const char *row = (const char *)a.input + b * row_bytes;
    int shift = 0;
    float factor = 1;
    if (TI != DN_I8) {
        unsigned m = 0;
#pragma unroll 4
        for (int k = tid * 4; k < a.s.inputs; k += 1024) {
            float x[4];
            q4_load4<TI>(row, k, a.s.inputs, x);
            m = q4_largest4(m, x);
        }
        m = dn_wave_max(m);
        if ((tid & 63) == 0) s_largest[tid >> 6] = m;
        __syncthreads();
        shift = q4_shift(max(max(s_largest[0], s_largest[1]), max(s_largest[2], s_largest[3])), factor);
    }
    if (tid == 0)
        ((float *)(a.workspace + q4_rows_at(a.s, PIECES, a.batch, XG)))[b] = TI == DN_I8 ? (XG ? 1.f : a.input_scales[b]) : factor;
    unsigned char *out = a.workspace + (size_t)(b >> 4) * a.s.kblocks * block + (b & 15) * 16;
    for (int k = tid * 8; k < a.s.kblocks * 128; k += 2048) {
        float x[8];
        half4_t hi[2], lo[2];
        q4_load4<TI>(row, k, a.s.inputs, x);
        q4_load4<TI>(row, k + 4, a.s.inputs, x + 4);
        q4_split4(x, shift, hi[0], lo[0]);
        q4_split4(x + 4, shift, hi[1], lo[1]);
        unsigned char *to = out + (size_t)(k >> 7) * block + ((k >> 5) & 3) * 1024 + ((k >> 3) & 3) * 256;
        ((half4_t *)to)[0] = hi[0];
        ((half4_t *)to)[1] = hi[1];
        if (PIECES == 2) {
            ((half4_t *)(to + 4096))[0] = lo[0];
            ((half4_t *)(to + 4096))[1] = lo[1];
        }
    }
    if (XG) {
        const int x_groups = (a.s.inputs + a.x_group - 1) / a.x_group, per = 128 / a.s.group;
        unsigned char *to = a.workspace + (size_t)(b >> 4) * a.s.kblocks * block + PIECES * 4096 + (b & 15) * 4;
        for (int g = tid; g < a.s.groups; g += 256)
            *(float *)(to + (size_t)(g / per) * block + g % per * 64) = g < x_groups ? a.input_scales[(long)b * x_groups + g] : 0.f;
    }
}

/* A lane's results of one tile of outputs and 16 rows, with the rows' own factors. */
__device__ __forceinline__ void q4_store_tile(const q4_args &a, const float *row_factors, int tile, int b0, float4_t v)
{
    const int lane = threadIdx.x & 63, o = tile * 16 + (lane & 15);
    if (o >= a.s.outputs) return;
    const float bias = q4_bias(a, o);
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        const int b = b0 + (lane >> 4) * 4 + i;
        const float y = i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3];
        if (b < a.batch) q4_store(a, b, o, y * row_factors[b], bias);
    }
}

/* ---- second pass, few outputs: a workgroup takes R row tiles and T tiles of input rows, its eight waves an eighth of
 * the inputs each.  No two waves read the same input, so that it comes straight into registers like the weights, both
 * a block ahead, and nothing waits for another wave before the end. */
template <int T, int R, int PIECES, int PER, bool XG>
__global__ __launch_bounds__(Q4_THREADS) void q4_stream_kernel(q4_args a)
{
    __shared__ float4_t s_red[Q4_WAVES][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int block = q4_block_bytes(a.s, PIECES, XG), x_tiles = (a.batch + 15) / 16, x0 = blockIdx.y * T, tile0 = blockIdx.x * R;
    const int mine = (a.s.kblocks - wave + Q4_WAVES - 1) / Q4_WAVES;
    struct block_data {
        q4_tile<PER> w[R];
        half8_t x[T][PIECES][4];
        float4_t f[T][PER];
    };
    auto fetch = [&](int n, block_data &d) {
        const int kb = wave + n * Q4_WAVES;
#pragma unroll
        for (int r = 0; r < R; ++r) d.w[r] = q4_load_tile<PER>(a, min(tile0 + r, a.s.tiles - 1), kb, lane);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const unsigned char *p = a.workspace + ((size_t)min(x0 + t, x_tiles - 1) * a.s.kblocks + kb) * block;
#pragma unroll
            for (int i = 0; i < 4 * PIECES; ++i) d.x[t][i / 4][i % 4] = *(const half8_t *)(p + i * 1024 + lane * 16);
            if (XG)
#pragma unroll
                for (int g = 0; g < PER; ++g) d.f[t][g] = *(const float4_t *)(p + PIECES * 4096 + g * 64 + (lane >> 4) * 16);
        }
    };
    float4_t sum[R][T];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) sum[r][t] = (float4_t){0, 0, 0, 0};
    const q4_masks masks;
    auto multiply = [&](const block_data &d) {
        q4_multiply<T, R, PIECES, PER, XG>(
            masks, d.w, sum, [&](int t, int piece, int step) { return d.x[t][piece][step]; }, [&](int t, int g) { return d.f[t][g]; });
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
    for (int k = 0; k < R * T; ++k) {
        float4_t v = sum[0][0];
#pragma unroll
        for (int m = 1; m < R * T; ++m) v = k == m ? sum[m / T][m % T] : v;
        __syncthreads();
        s_red[wave][lane] = v;
        __syncthreads();
        if (wave == k && tile0 + k / T < a.s.tiles && x0 + k % T < x_tiles) { /* R * T <= 8 */
            v = s_red[0][lane];
#pragma unroll
            for (int q = 1; q < Q4_WAVES; ++q) v += s_red[q][lane];
            q4_store_tile(a, row_factors, tile0 + k / T, (x0 + k % T) * 16, v);
        }
    }
}

/* Stores 16 rows of WIDTH outputs from LDS. */
template <int THREADS, int WIDTH, int PITCH>
__device__ __forceinline__ void q4_store_rows(const q4_args &a, const float *s_sum, const float *row_factors, int b0, int o0)
{
    const int rows = min(16, a.batch - b0);
#pragma unroll 2
    for (int i = threadIdx.x; i < rows * WIDTH; i += THREADS) {
        const int row = i / WIDTH, o = o0 + i % WIDTH;
        if (o < a.s.outputs) q4_store(a, b0 + row, o, s_sum[row * PITCH + i % WIDTH] * row_factors[b0 + row], q4_bias(a, o));
    }
}

/* ---- second pass, many outputs: a workgroup takes 4 * R row tiles, R for each wave, and T tiles of input rows.  The
 * input goes through LDS in chunks that all waves read, the next chunk on its way (through registers) during the
 * products of the present one; each wave's weights come straight from memory, a chunk ahead as well. */
#define Q4_STAGED_WAVES 4
template <int T, int R, int PIECES, int PER, bool XG>
__global__ __launch_bounds__(Q4_STAGED_WAVES * 64, 2) void q4_staged_kernel(q4_args a)
{
    constexpr int THREADS = Q4_STAGED_WAVES * 64;
    constexpr int UNITS = 4 / (T * PIECES > 4 ? 4 : T * PIECES); /* blocks of a chunk */
    constexpr int BLOCK = PIECES * 4096 + (XG ? PER * 64 : 0), SPAN = UNITS * BLOCK, CHUNK = T * SPAN;
    constexpr int MOVES = (CHUNK + THREADS * 16 - 1) / (THREADS * 16);
    __shared__ uint4_t s_input[2][CHUNK / 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int x_tiles = (a.batch + 15) / 16, x0 = blockIdx.y * T, tile0 = (blockIdx.x * Q4_STAGED_WAVES + wave) * R;
    const int kblocks = a.s.kblocks, chunks = (kblocks + UNITS - 1) / UNITS;
    float4_t sum[R][T];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) sum[r][t] = (float4_t){0, 0, 0, 0};

    const q4_masks masks;
    uint4_t moved[MOVES];
    auto input_of = [&](int c) {
#pragma unroll
        for (int m = 0; m < MOVES; ++m) { /* what lies behind the last block or tile is read at its place, and not multiplied */
            const int i = min((m * THREADS + tid) * 16, CHUNK - 16), t = i / SPAN, in = i % SPAN;
            const int kb = min(c * UNITS + in / BLOCK, kblocks - 1);
            moved[m] = *(const uint4_t *)(a.workspace + ((size_t)min(x0 + t, x_tiles - 1) * kblocks + kb) * BLOCK + in % BLOCK);
        }
    };
    auto keep_input = [&](int buffer) {
#pragma unroll
        for (int m = 0; m < MOVES; ++m)
            if ((m * THREADS + tid) * 16 < CHUNK) s_input[buffer][m * THREADS + tid] = moved[m];
    };
    q4_tile<PER> w[UNITS][R];
    auto fetch = [&](int c, int u) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            w[u][r] = q4_load_tile<PER>(a, min(tile0 + r, a.s.tiles - 1), min(c * UNITS + u, kblocks - 1), lane);
    };
    input_of(0);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) fetch(0, u);
    keep_input(0);
    __syncthreads();
    for (int c = 0; c < chunks; ++c) {
        if (c + 1 < chunks) input_of(c + 1);
        const char *base = (const char *)s_input[c & 1];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            if (c * UNITS + u < kblocks)
                q4_multiply<T, R, PIECES, PER, XG>(
                    masks, w[u], sum,
                    [&](int t, int piece, int step) {
                        return *(const half8_t *)(base + t * SPAN + u * BLOCK + piece * 4096 + step * 1024 + lane * 16);
                    },
                    [&](int t, int g) { return *(const float4_t *)(base + t * SPAN + u * BLOCK + PIECES * 4096 + g * 64 + (lane >> 4) * 16); });
            if (c + 1 < chunks) fetch(c + 1, u);
        }
        if (c + 1 < chunks) keep_input((c + 1) & 1); /* the buffer that all waves have left at the last barrier */
        __syncthreads();
    }
    /* The sums go through LDS, a tile of input rows at a time, so that neighbouring lanes store neighbouring outputs
     * (16 of a row alone are half a line) and there is one copy of the activation's code. */
    const float *row_factors = (const float *)(a.workspace + q4_rows_at(a.s, PIECES, a.batch, XG));
    constexpr int WIDTH = Q4_STAGED_WAVES * R * 16, PITCH = WIDTH + 4;
    static_assert(sizeof s_input >= 16 * PITCH * 4, "room for a tile's sums");
    float *s_sum = (float *)s_input;
    const int o0 = blockIdx.x * WIDTH;
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
        q4_store_rows<THREADS, WIDTH, PITCH>(a, s_sum, row_factors, (x0 + x) * 16, o0);
        __syncthreads();
    }
}

/* Which form a product takes.
 *   direct  at most 16 rows that are short enough for every workgroup to scale them while its first weights arrive: a
 *           second launch and the way of the input through memory cost more.  Longer ones (25088 values in two rows)
 *           are better scaled once.
 *   staged  so many outputs that workgroups of 64 (R = 1) or 128 (R = 2) of them fill the chip
 *   stream  the others */
struct q4_plan {
    enum { DIRECT, STREAM, STAGED } form;
    int ksplit, t, r;
    unsigned gx, gy;
    size_t lds;
};

static q4_plan q4_plan_of(const q4_shape &s, int type, int batch)
{
    q4_plan p;
    const int pieces = type == DN_F32 ? 2 : 1, x_tiles = (int)(((long)batch + 15) / 16);
    p.ksplit = p.t = p.r = 1;
    p.gy = 1;
    p.lds = batch * ((size_t)s.kblocks * 256 * pieces + 16) + (size_t)(type == DN_I8 ? s.groups : s.kblocks) * 64;
    if (batch <= 4 && (long)batch * s.inputs <= 28672 && p.lds <= 120 << 10) {
        p.form = q4_plan::DIRECT;
        /* waves share a row tile as long as each has a block and the chip is not full */
        while (p.ksplit < Q4_WAVES && (long)s.tiles * p.ksplit < 256 * Q4_WAVES && p.ksplit * 2 <= s.kblocks) p.ksplit *= 2;
        const long groups = ((long)s.tiles * p.ksplit + Q4_WAVES - 1) / Q4_WAVES;
        p.gx = (unsigned)(groups < 512 ? groups : 512);
        return p;
    }
    p.lds = 0;
    const int passes = (x_tiles + 3) / 4;
    if ((long)s.tiles * x_tiles >= 2800) {
        p.form = q4_plan::STAGED;
        p.t = (x_tiles + passes - 1) / passes;
        p.r = s.group > 32 && (long)s.tiles * passes >= Q4_STAGED_WAVES * 2 * 384 ? 2 : 1;
        p.gx = (unsigned)((s.tiles + Q4_STAGED_WAVES * p.r - 1) / (Q4_STAGED_WAVES * p.r));
    } else {
        p.form = q4_plan::STREAM;
        p.t = pieces == 1 && x_tiles > 1 ? 2 : 1;
        p.r = s.group > 32 && s.tiles >= 2 * 192 ? 2 : 1;
        p.gx = (unsigned)((s.tiles + p.r - 1) / p.r);
    }
    p.gy = (unsigned)((x_tiles + p.t - 1) / p.t);
    return p;
}

extern "C" size_t connected_q4_workspace_bytes(int input_type, int batch, int inputs, int outputs, int group)
{
    if (!q4_shape_ok(inputs, outputs, group) || batch < 1) return 0;
    const q4_shape s = q4_shape_of(inputs, outputs, group);
    if (q4_plan_of(s, input_type, batch).form == q4_plan::DIRECT) return 0;
    return q4_rows_at(s, input_type == DN_F32 ? 2 : 1, batch, input_type == DN_I8) + (size_t)batch * 4;
}

template <int T, int R, int PIECES, int PER, bool XG>
static void q4_launch_second(const q4_args &a, const q4_plan &p)
{
    const dim3 grid(p.gx, p.gy);
    if (p.form == q4_plan::STAGED)
        hipLaunchKernelGGL((q4_staged_kernel<T, R, PIECES, PER, XG>), grid, dim3(Q4_STAGED_WAVES * 64), 0, dn_stream(), a);
    else if constexpr (T * PIECES <= 2)
        hipLaunchKernelGGL((q4_stream_kernel<T, R, PIECES, PER, XG>), grid, dim3(Q4_THREADS), 0, dn_stream(), a);
}

template <int TI, int PER, bool XG>
static void q4_launch(const q4_args &a, const q4_plan &p)
{
    constexpr int PIECES = TI == DN_F32 ? 2 : 1;
    if (p.form == q4_plan::DIRECT) {
        if (a.batch == 1) hipLaunchKernelGGL((q4_direct_kernel<TI, PER, XG, true>), dim3(p.gx), dim3(Q4_THREADS), p.lds, dn_stream(), a);
        else hipLaunchKernelGGL((q4_direct_kernel<TI, PER, XG, false>), dim3(p.gx), dim3(Q4_THREADS), p.lds, dn_stream(), a);
        return;
    }
    hipLaunchKernelGGL((q4_prepare_kernel<TI, XG>), dim3((unsigned)a.batch), dim3(256), 0, dn_stream(), a);
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
                       output_type, batch, xg ? input_group : 0, activation, p.ksplit, s};
    if (input_type == DN_F32) q4_launch_group<DN_F32, false>(a, p);
    else if (input_type == DN_F16) q4_launch_group<DN_F16, false>(a, p);
    else if (input_type == DN_BF16) q4_launch_group<DN_BF16, false>(a, p);
    else if (xg) q4_launch_group<DN_I8, true>(a, p);
    else q4_launch_group<DN_I8, false>(a, p);
    dn_check_launch(me);
    return 0;
}
