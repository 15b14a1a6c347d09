/*
 * q4.hip - products with 4-bit weights: a connected layer whose weights are held as
 *
 *   w[o][k] = (code[o][k] - zero[o][k / G]) * scale[o][k / G],   code and zero 0 .. 15, G = 32, 64 or 128
 *   output[b][o] = activation(bias[o] + sum_k x[b][k] * w[o][k])
 *
 * Packed weights, written once when they are loaded: tiles of 16 outputs x 128 inputs, a kilobyte each, in
 * the order [outputs / 16][inputs / 128][lane 0..63][4 dwords].  Dword s of lane r + 16*j holds output r,
 * inputs 32*s + 8*j + i: i = 0..3 in the low halves of its bytes 0..3, i = 4..7 in the high halves.
 * Masking a dword with 0x0f0f0f0f, and so after a shift by 4, gives a lane its bytes of a matrix operand.
 * Behind the codes the scales, [outputs / 16][groups][16] floats, and the zeros, the same in bytes.  What
 * fills the last tiles up has code, scale and zero 0.
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
__device__ __forceinline__ int q4_bit_of(int k) { return ((k & 3) << 3) + (k & 4); }
__device__ __forceinline__ long q4_group_at(const q4_shape &s, int o, int g)
{
    return ((long)(o >> 4) * s.groups + g) * 16 + (o & 15);
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

struct q4_args {
    const void *input;
    const float *input_scales;
    const unsigned char *packed;
    const float *biases;
    void *output;
    int batch, input_group, activation;
    q4_shape s;
};

/* One wave for each output and batch row: a lane takes 8 inputs of every 512, products and sums in fp32. */
template <int TI, int TO>
__global__ __launch_bounds__(256) void q4_rows_kernel(q4_args a)
{
    const q4_shape s = a.s;
    const int lane = threadIdx.x & 63;
    const long item = blockIdx.x * 4L + (threadIdx.x >> 6);
    if (item >= (long)a.batch * s.outputs) return;
    const int b = (int)(item / s.outputs), o = (int)(item % s.outputs);
    const typename dn_elt<TI>::store *x = (const typename dn_elt<TI>::store *)a.input + (long)b * s.inputs;
    const int x_groups = a.input_group ? (s.inputs + a.input_group - 1) / a.input_group : 1;
    float sum = 0, poison = 0;
    for (int k0 = lane * 8; k0 < s.inputs; k0 += 512) {
        const unsigned v = ((const unsigned *)a.packed)[q4_dword_at(s, o, k0)];
        const long at = q4_group_at(s, o, k0 / s.group);
        const int zero = a.packed[s.zeros_at + at];
        float part = 0;
        for (int i = 0; i < 8 && k0 + i < s.inputs; ++i) {
            poison = fmaf((float)x[k0 + i], 0.f, poison); /* NaN from a value that is not finite */
            part = fmaf((float)((int)((v >> q4_bit_of(i)) & 15) - zero), (float)x[k0 + i], part);
        }
        float scale = ((const float *)(a.packed + s.scales_at))[at];
        if (TI == DN_I8) scale *= a.input_scales[(long)b * x_groups + (a.input_group ? k0 / a.input_group : 0)];
        sum = fmaf(scale, part, sum);
    }
    sum += poison;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) {
        if (a.biases) sum += a.biases[o];
        ((typename dn_elt<TO>::store *)a.output)[item] = (typename dn_elt<TO>::store)dn_activate(sum, a.activation);
    }
}

extern "C" size_t connected_q4_workspace_bytes(int input_type, int batch, int inputs, int outputs, int group)
{
    (void)input_type;
    (void)batch;
    (void)inputs;
    (void)outputs;
    (void)group;
    return 0;
}

template <int TI>
static void q4_launch(const q4_args &a, int output_type)
{
    const dim3 grid((unsigned)(((long)a.batch * a.s.outputs + 3) / 4)), block(256);
    if (output_type == DN_F32) hipLaunchKernelGGL((q4_rows_kernel<TI, DN_F32>), grid, block, 0, dn_stream(), a);
    else if (output_type == DN_F16) hipLaunchKernelGGL((q4_rows_kernel<TI, DN_F16>), grid, block, 0, dn_stream(), a);
    else hipLaunchKernelGGL((q4_rows_kernel<TI, DN_BF16>), grid, block, 0, dn_stream(), a);
}

extern "C" int forward_connected_q4_gpu(const void *input, int input_type, const float *input_scales, int input_group,
                                        const void *packed, const float *biases, void *output, int output_type,
                                        int batch, int inputs, int outputs, int group, int activation, void *workspace)
{
    const char *me = "forward_connected_q4_gpu";
    if (!dn_is_float_type(input_type) && input_type != DN_I8) return dn_refuse(me, "unknown input type");
    if (!dn_is_float_type(output_type)) return dn_refuse(me, "unknown output type");
    if (batch < 0 || !q4_shape_ok(inputs, outputs, group)) return dn_refuse(me, "bad geometry (group must be 32, 64 or 128)");
    if ((long)batch * outputs > 0x1ffffffffL) return dn_refuse(me, "too many outputs for one call");
    if (activation < 0 || activation > DN_SELU) return dn_refuse(me, "unknown activation");
    if (!input || !packed || !output) return dn_refuse(me, "a buffer is missing");
    if (input_type == DN_I8 && !input_scales) return dn_refuse(me, "8-bit input needs its scales");
    if (input_type == DN_I8 && input_group != 0 && input_group != group)
        return dn_refuse(me, "input_group must be 0 (the row) or the weights' group");
    if (!dn_aligned(input, dn_type_bytes(input_type)) || !dn_aligned(output, dn_type_bytes(output_type)) ||
        !dn_aligned(input_scales, 4) || !dn_aligned(biases, 4) || !dn_aligned(packed, 16))
        return dn_refuse(me, "a buffer is not aligned to its element type, or packed not to 16 bytes");
    (void)workspace;
    if (batch == 0) return 0;
    hip_require_device(me);
    const q4_args a = {input, input_scales, (const unsigned char *)packed, biases, output, batch, input_group,
                       activation, q4_shape_of(inputs, outputs, group)};
    if (input_type == DN_F32) q4_launch<DN_F32>(a, output_type);
    else if (input_type == DN_F16) q4_launch<DN_F16>(a, output_type);
    else if (input_type == DN_BF16) q4_launch<DN_BF16>(a, output_type);
    else q4_launch<DN_I8>(a, output_type);
    dn_check_launch(me);
    return 0;
}
