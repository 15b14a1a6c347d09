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
template <int THREADS, bool MAX>
__device__ __forceinline__ double block_all(double v, double *lds)
{
    v = MAX ? dn_wave_max(v) : dn_wave_sum(v);
    if (THREADS == 64) return v;
    __syncthreads(); /* the last use of lds is over */
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = lds[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) t = MAX ? fmax(t, lds[w]) : t + lds[w];
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

/* The code of y for a step of c, inv = 1 / (double)c: the product differs from the quotient by its last bit, which
 * matters to a rounding as little as the last bit of y. */
__device__ __forceinline__ int q8_code(double y, float c, double inv)
{
    if (!(c > 0)) return 0; /* nothing but zeros, or a group with a value that is not finite */
    return (int)fmin(fmax(rint(y * inv), -127.), 127.);
}

/* V neighbouring elements as floats; VECTORS: they all exist, on a boundary of V elements. */
template <int T, int V, bool VECTORS>
__device__ __forceinline__ void load_run(const typename dn_elt<T>::store *p, int i, int n, float *v)
{
    typedef typename dn_elt<T>::store E;
    typedef E EV __attribute__((ext_vector_type(V)));
    if (VECTORS) {
        const EV x = *(const EV *)(p + i);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)x[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = i + e < n ? (float)p[i + e] : 0.f;
    }
}

template <int T, int V, bool VECTORS>
__device__ __forceinline__ void store_run(typename dn_elt<T>::store *p, int i, int n, const float *v)
{
    typedef typename dn_elt<T>::store E;
    typedef E EV __attribute__((ext_vector_type(V)));
    if (VECTORS) {
        EV x;
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = (E)v[e];
        *(EV *)(p + i) = x;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (i + e < n) p[i + e] = (E)v[e];
    }
}

/* One workgroup for each row, which it holds in registers: RUNS runs of V neighbouring values a lane, the runs of
 * the lanes next to each other (lane t, run j: values (j * THREADS + t) * V on).  Every buffer is read and written once.
 * A group of 8-bit values is a power of two of neighbouring lanes' runs, so that its maximum takes lane moves only. */
template <int T, int THREADS, int RUNS, int V, bool VECTORS, bool Q8>
__global__ __launch_bounds__(THREADS) void rmsnorm_kernel(norm_args a)
{
    typedef typename dn_elt<T>::store E;
    __shared__ double lds[THREADS / 64];
    const int tid = threadIdx.x, n = a.n;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float s[RUNS][V];
        double acc = 0;
        {
            float add[RUNS][V];
#pragma unroll
            for (int j = 0; j < RUNS; ++j) {
                const int i = (j * THREADS + tid) * V;
                if (i < n) load_run<T, V, VECTORS>((const E *)a.input + row * n, i, n, s[j]);
                else
#pragma unroll
                    for (int e = 0; e < V; ++e) s[j][e] = 0;
            }
            if (a.add) {
#pragma unroll
                for (int j = 0; j < RUNS; ++j) {
                    const int i = (j * THREADS + tid) * V;
                    if (i < n) load_run<T, V, VECTORS>((const E *)a.add + row * n, i, n, add[j]);
                }
#pragma unroll
                for (int j = 0; j < RUNS; ++j) {
                    const int i = (j * THREADS + tid) * V;
                    if (i >= n) continue;
#pragma unroll
                    for (int e = 0; e < V; ++e) s[j][e] = (float)(E)(s[j][e] + add[j][e]);
                    if (a.sum) store_run<T, V, VECTORS>((E *)a.sum + row * n, i, n, s[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < RUNS; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) acc = fma((double)s[j][e], (double)s[j][e], acc);
        acc = block_all<THREADS, false>(acc, lds);
        const double r = 1. / sqrt(acc / n + (double)a.eps);
        auto scales = [&](int i, float g[V]) {
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] = 1;
            if (a.scales && i < n) load_run<DN_F32, V, VECTORS>(a.scales, i, n, g);
        };
        if (a.output) {
            const float rf = (float)r;
#pragma unroll
            for (int j = 0; j < RUNS; ++j) {
                const int i = (j * THREADS + tid) * V;
                float y[V], g[V];
                scales(i, g);
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = s[j][e] * rf * g[e];
                if (i < n) store_run<T, V, VECTORS>((E *)a.output + row * n, i, n, y);
            }
        }
        if (!Q8) continue;
        const int lanes = a.group / V, groups = a.group ? (n + a.group - 1) / a.group : 1;
        double row_largest = 0;
        if (a.group == 0) {
#pragma unroll
            for (int j = 0; j < RUNS; ++j) {
                float g[V];
                scales((j * THREADS + tid) * V, g);
#pragma unroll
                for (int e = 0; e < V; ++e) row_largest = fmax(row_largest, finite_abs((double)s[j][e] * r * (double)g[e]));
            }
            row_largest = block_all<THREADS, true>(row_largest, lds);
            if (tid == 0) a.q8_scales[row] = q8_step(row_largest);
        }
#pragma unroll
        for (int j = 0; j < RUNS; ++j) {
            const int i = (j * THREADS + tid) * V;
            float g[V];
            double y[V], largest = 0;
            scales(i, g);
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = (double)s[j][e] * r * (double)g[e];
            if (a.group) {
#pragma unroll
                for (int e = 0; e < V; ++e) largest = fmax(largest, finite_abs(y[e]));
                for (int o = 1; o < lanes; o <<= 1) largest = fmax(largest, __shfl_xor(largest, o, 64));
            } else {
                largest = row_largest;
            }
            const float c = q8_step(largest);
            const double inv = 1. / (double)c;
            if (a.group && i < n && (tid & (lanes - 1)) == 0) a.q8_scales[row * groups + i / a.group] = c;
            if (i >= n) continue;
            signed char *q = a.q8 + row * n;
            if (VECTORS) {
                typedef signed char QV __attribute__((ext_vector_type(V)));
                QV x;
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = (signed char)q8_code(y[e], c, inv);
                *(QV *)(q + i) = x;
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (i + e < n) q[i + e] = (signed char)q8_code(y[e], c, inv);
            }
        }
    }
}

/* Rows that no workgroup holds in registers: read again for each step. */
template <int T>
__global__ __launch_bounds__(1024) void rmsnorm_long_kernel(norm_args a)
{
    typedef typename dn_elt<T>::store E;
    constexpr int THREADS = 1024;
    __shared__ double lds[THREADS / 64];
    const int tid = threadIdx.x, n = a.n;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const E *in = (const E *)a.input + row * n;
        const E *add = a.add ? (const E *)a.add + row * n : 0;
        E *sum = a.sum ? (E *)a.sum + row * n : 0;
        double acc = 0;
        for (int i = tid; i < n; i += THREADS) {
            float s = (float)in[i];
            if (add) s = (float)(E)(s + (float)add[i]);
            if (sum) sum[i] = (E)s;
            acc += (double)s * s;
        }
        acc = block_all<THREADS, false>(acc, lds);
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
                for (int i = tid; i < n; i += THREADS) largest = fmax(largest, finite_abs(norm(i)));
                const float c = q8_step(block_all<THREADS, true>(largest, lds));
                const double inv = 1. / (double)c;
                if (tid == 0) a.q8_scales[row] = c;
                for (int i = tid; i < n; i += THREADS) q[i] = (signed char)q8_code(norm(i), c, inv);
            } else {
                const int groups = (n + a.group - 1) / a.group;
                __syncthreads(); /* a group's values may have been stored by another wave */
                for (int g = tid >> 6; g < groups; g += THREADS / 64) {
                    const int lo = g * a.group, hi = min(n, lo + a.group);
                    double largest = 0;
                    for (int i = lo + (tid & 63); i < hi; i += 64) largest = fmax(largest, finite_abs(norm(i)));
                    const float c = q8_step(dn_wave_max(largest));
                    const double inv = 1. / (double)c;
                    if ((tid & 63) == 0) a.q8_scales[row * groups + g] = c;
                    for (int i = lo + (tid & 63); i < hi; i += 64) q[i] = (signed char)q8_code(norm(i), c, inv);
                }
            }
        }
        if (a.output) {
            E *out = (E *)a.output + row * n;
            if (a.q8) __syncthreads(); /* it may take the input's place, which the groups above read */
            for (int i = tid; i < n; i += THREADS) out[i] = (E)(float)norm(i);
        }
    }
}

/* Which form a row takes: one run a lane up to 256 lanes, then two, so that several rows share a CU and their loads
 * and stores overlap; a row of more than 16384 values is read again for each step. */
template <int T, bool VECTORS, bool Q8>
static void norm_launch(const norm_args &a)
{
    constexpr int V = T == DN_F32 ? 4 : 8;
    const dim3 grid(a.rows < 65536 ? a.rows : 65536);
    const int runs = (int)(((long)a.n + V - 1) / V);
#define NM_LAUNCH(THREADS, RUNS) \
    hipLaunchKernelGGL((rmsnorm_kernel<T, THREADS, RUNS, V, VECTORS, Q8>), grid, dim3(THREADS), 0, dn_stream(), a)
    if (runs <= 64) NM_LAUNCH(64, 1);
    else if (runs <= 128) NM_LAUNCH(128, 1);
    else if (runs <= 256) NM_LAUNCH(256, 1);
    else if (runs <= 512) NM_LAUNCH(256, 2);
    else if (runs <= 1024) NM_LAUNCH(512, 2);
    else if (runs <= 2048) NM_LAUNCH(1024, 2);
    else if (V == 4 && runs <= 4096) NM_LAUNCH(1024, 16 / V);
    else hipLaunchKernelGGL((rmsnorm_long_kernel<T>), grid, dim3(1024), 0, dn_stream(), a);
#undef NM_LAUNCH
}

/* Sixteen-byte runs want rows of whole runs from 16-byte boundaries on (8-bit codes: from V-byte boundaries). */
template <int T>
static void norm_launch_type(const norm_args &a)
{
    const int v = T == DN_F32 ? 4 : 8;
    const bool vectors = a.n % v == 0 && dn_aligned(a.input, 16) && dn_aligned(a.add, 16) && dn_aligned(a.sum, 16) &&
                         dn_aligned(a.output, 16) && dn_aligned(a.scales, 16) && dn_aligned(a.q8, v);
    if (a.q8) {
        if (vectors) norm_launch<T, true, true>(a);
        else norm_launch<T, false, true>(a);
    } else {
        if (vectors) norm_launch<T, true, false>(a);
        else norm_launch<T, false, false>(a);
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
    if (type == DN_F32) norm_launch_type<DN_F32>(a);
    else if (type == DN_F16) norm_launch_type<DN_F16>(a);
    else norm_launch_type<DN_BF16>(a);
    dn_check_launch(me);
    return 0;
}
