/*
 * norm.hip - root-mean-square norm of the rows of a matrix, with the addition of a residual in front of it
 * and an 8-bit form of the result behind it.
 *
 *   s[i] = round_T(input[i] + add[i])      r = 1 / sqrt(sum(s^2) / n + eps)      y[i] = s[i] * r * scales[i]
 *   8 bit, for each row or group:          c = (float)(max|y| / 127)             q[i] = rint(y[i] / c)
 *
 * The sum of squares is held in 64 bits: a product of two 24-bit values is exact there and the fp64
 * rate of a vector ALU on this part equals its fp32 rate.  The 8-bit form evaluates y in 64 bits as well, so
 * that a value next to the border between two steps goes to the step that the formula gives.
 */
#include <math.h>

#include "row_types.h"

#define NM_THREADS 256

struct norm_args {
    const void *input, *add;
    const float *scales;
    void *sum, *output;
    signed char *q8;
    float *q8_scales;
    int rows, n, group; /* group: values that share a scale, 0 = the row */
    float eps;
};

/* Sum (or maximum) over the workgroup, the same bits on every lane and in every run. */
template <bool MAX>
__device__ __forceinline__ double block_all(double v, double *lds)
{
    v = MAX ? dn_wave_max(v) : dn_wave_sum(v);
    __syncthreads(); /* the last use of lds is over */
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = lds[0];
    for (int w = 1; w < (int)blockDim.x / 64; ++w) t = MAX ? fmax(t, lds[w]) : t + lds[w];
    return t;
}

/* |y| for the maximum: a value that is not finite counts as infinity and so marks its group. */
__device__ __forceinline__ double finite_abs(double y)
{
    const double a = fabs(y);
    return a <= 1.7976931348623157e308 ? a : __longlong_as_double(0x7ff0000000000000LL);
}

__device__ __forceinline__ float q8_step(double largest)
{
    const float c = (float)(largest / 127);
    return c <= 3.402823466e38f ? c : __int_as_float(0x7fc00000);
}

__device__ __forceinline__ signed char q8_code(double y, float c)
{
    if (!(c > 0)) return 0; /* nothing but zeros, or a group with a value that is not finite */
    return (signed char)fmin(fmax(rint(y / (double)c), -127.), 127.);
}

template <int T>
__global__ __launch_bounds__(NM_THREADS) void rmsnorm_kernel(norm_args a)
{
    typedef typename dn_elt<T>::store E;
    __shared__ double lds[NM_THREADS / 64];
    const int tid = threadIdx.x, n = a.n;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const E *in = (const E *)a.input + row * n;
        const E *add = a.add ? (const E *)a.add + row * n : 0;
        E *sum = a.sum ? (E *)a.sum + row * n : 0;
        double acc = 0;
        for (int i = tid; i < n; i += NM_THREADS) {
            float s = (float)in[i];
            if (add) s = (float)(E)(s + (float)add[i]);
            if (sum) sum[i] = (E)s;
            acc += (double)s * s;
        }
        acc = block_all<false>(acc, lds);
        const double r = 1. / sqrt(acc / n + (double)a.eps);
        /* the sum where it was stored (it may have taken the input's place), else added again */
        auto value = [&](int i) {
            if (sum) return (float)sum[i];
            const float s = (float)in[i];
            return add ? (float)(E)(s + (float)add[i]) : s;
        };
        auto norm = [&](int i) { return (double)value(i) * r * (a.scales ? (double)a.scales[i] : 1.); };
        if (a.q8) {
            signed char *q = a.q8 + row * n;
            if (a.group == 0) {
                double largest = 0;
                for (int i = tid; i < n; i += NM_THREADS) largest = fmax(largest, finite_abs(norm(i)));
                const float c = q8_step(block_all<true>(largest, lds));
                if (tid == 0) a.q8_scales[row] = c;
                for (int i = tid; i < n; i += NM_THREADS) q[i] = q8_code(norm(i), c);
            } else {
                const int groups = (n + a.group - 1) / a.group;
                __syncthreads(); /* a group's values may have been stored by another wave */
                for (int g = tid >> 6; g < groups; g += NM_THREADS / 64) {
                    const int lo = g * a.group, hi = min(n, lo + a.group);
                    double largest = 0;
                    for (int i = lo + (tid & 63); i < hi; i += 64) largest = fmax(largest, finite_abs(norm(i)));
                    const float c = q8_step(dn_wave_max(largest));
                    if ((tid & 63) == 0) a.q8_scales[row * groups + g] = c;
                    for (int i = lo + (tid & 63); i < hi; i += 64) q[i] = q8_code(norm(i), c);
                }
            }
        }
        if (a.output) {
            E *out = (E *)a.output + row * n;
            if (a.q8) __syncthreads(); /* it may take the input's place, which the groups above read */
            for (int i = tid; i < n; i += NM_THREADS) out[i] = (E)(float)norm(i);
        }
    }
}

extern "C" int forward_rmsnorm_gpu(const void *input, const void *add, const float *scales, void *sum_output,
                                   void *output, signed char *q8_output, float *q8_scales, int type, int rows,
                                   int n, int q8_group, float eps)
{
    const char *me = "forward_rmsnorm_gpu";
    if (!dn_is_float_type(type)) return dn_refuse(me, "unknown element type");
    if (rows < 0 || n < 1) return dn_refuse(me, "bad geometry");
    if (!(eps >= 0) || !(eps <= 3.402823466e38f)) return dn_refuse(me, "eps must be a finite number that is not negative");
    if (!input) return dn_refuse(me, "input is missing");
    if (!output && !q8_output) return dn_refuse(me, "neither output nor q8_output is given");
    if (!q8_output != !q8_scales) return dn_refuse(me, "q8_output and q8_scales come together");
    if (q8_group != 0 && q8_group != 32 && q8_group != 64 && q8_group != 128)
        return dn_refuse(me, "q8_group must be 0 (the row), 32, 64 or 128");
    if (sum_output && !add) return dn_refuse(me, "sum_output needs add");
    if (sum_output && sum_output == output) return dn_refuse(me, "sum_output and output must be two buffers");
    const size_t e = dn_type_bytes(type);
    if (!dn_aligned(input, e) || !dn_aligned(add, e) || !dn_aligned(sum_output, e) || !dn_aligned(output, e) ||
        !dn_aligned(scales, 4) || !dn_aligned(q8_scales, 4))
        return dn_refuse(me, "a buffer is not aligned to its element type");
    if (rows == 0) return 0;
    hip_require_device(me);
    const norm_args a = {input, add, scales, sum_output, output, q8_output, q8_scales, rows, n, q8_group, eps};
    const dim3 grid(rows < 65536 ? rows : 65536), block(NM_THREADS);
    if (type == DN_F32) hipLaunchKernelGGL((rmsnorm_kernel<DN_F32>), grid, block, 0, dn_stream(), a);
    else if (type == DN_F16) hipLaunchKernelGGL((rmsnorm_kernel<DN_F16>), grid, block, 0, dn_stream(), a);
    else hipLaunchKernelGGL((rmsnorm_kernel<DN_BF16>), grid, block, 0, dn_stream(), a);
    dn_check_launch(me);
    return 0;
}
