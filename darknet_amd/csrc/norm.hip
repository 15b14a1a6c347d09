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
    double inv_n;
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

/* A value y can lie half-way between two steps only if the row's root mean square has few bits: y = p / rms, where p = s *
 * scales has 48 at most, is then a product of the step, a float, and a number of 8 bits.  In such rows (all values alike, say,
 * without eps) what reciprocals give is looked at once more. */
__device__ __forceinline__ bool q8_may_tie(double rms) { return ((unsigned long long)__double_as_longlong(rms) & 0xffffff) == 0; }

/* The scale of a group whose largest |p| is given; NaN where that is not finite. */
__device__ __forceinline__ float q8_step(double largest, double rms, double r, bool ties)
{
    const float c = ties ? (float)(largest / rms / 127) : (float)(largest * r * (1. / 127));
    return c <= 3.402823466e38f ? c : __int_as_float(0x7fc00000);
}

/* r / c for a step c > 0: the hardware's reciprocal after two steps of Newton's iteration, in 64 bits. */
__device__ __forceinline__ double q8_factor(double r, float c)
{
    const double d = (double)c;
    double x = __builtin_amdgcn_rcp(d);
    x = fma(fma(-d, x, 1.), x, x);
    x = fma(fma(-d, x, 1.), x, x);
    return r * x;
}

/* The maximum over 4, 8, 16 or 32 neighbouring lanes, on each of them: the lane's pair, the other
 * pair of its quad, the other quad of its 8, the other 8 of its 16, and the other 16. */
__device__ __forceinline__ double group_largest(double v, int lanes)
{
    v = fmax(v, dn_move<0xb1, 0xf>(v, v));
    v = fmax(v, dn_move<0x4e, 0xf>(v, v));
    if (lanes >= 8) v = fmax(v, dn_move<0x141, 0xf>(v, v));
    if (lanes >= 16) v = fmax(v, dn_move<0x140, 0xf>(v, v));
    if (lanes >= 32) v = fmax(v, __shfl_xor(v, 16, 64));
    return v;
}

/* rint(p * factor) within -127 .. 127: added to 1.5 * 2^52 the whole number stands in the low word of the sum. */
__device__ __forceinline__ int q8_code(double p, double factor)
{
    const int q = (int)__double_as_longlong(fma(p, factor, 0x1.8p52));
    return max(-127, min(127, q));
}

/* rint(p / step) next to q, ties to even: the sign of a remainder that is rounded once is exact. */
__device__ __forceinline__ int q8_nearest(int q, double p, double step)
{
    const double above = fma(-(q + .5), step, p), below = fma(-(q - .5), step, p);
    if (above > 0 || (above == 0 && q & 1)) ++q;
    else if (below < 0 || (below == 0 && q & 1)) --q;
    return max(-127, min(127, q));
}

/* V neighbouring elements as floats, 0 behind the row's end.  Runs that lie within the row go in one access whatever
 * their alignment. */
template <int T, int V>
__device__ __forceinline__ void load_run(const typename dn_elt<T>::store *p, int i, int n, float *v)
{
    typedef typename dn_elt<T>::store E;
    typedef E EV __attribute__((ext_vector_type(V)));
    typedef EV EU __attribute__((aligned(sizeof(E))));
    if (i + V <= n) {
        const EV x = *(const EU *)(p + i);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)x[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = i + e < n ? (float)p[i + e] : 0.f;
    }
}

template <class E, int V>
__device__ __forceinline__ void store_run(E *p, int i, int n, const float *v)
{
    typedef E EV __attribute__((ext_vector_type(V)));
    typedef EV EU __attribute__((aligned(sizeof(E))));
    if (i + V <= n) {
        EV x;
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = (E)v[e];
        *(EU *)(p + i) = x;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (i + e < n) p[i + e] = (E)v[e];
    }
}

/* One workgroup for each row, which it holds in registers: RUNS runs of V neighbouring values a lane, the runs of
 * the lanes next to each other (lane t, run j: values (j * THREADS + t) * V on).  Every buffer is read and written once.
 * RUNS = 0: as many runs as the row has, read again for each step (from the stored sum, if there is one).
 * A group of 8-bit values is a power of two of neighbouring lanes' runs, so that its maximum takes lane moves only.
 *
 * The 8-bit form works on p = s * scales, exact in 64 bits: max|y| = max|p| * r, and code = rint(p * (r / c)).
 *
 * Bound by memory: 16384 x 4096 fp32 with residual, sum and output (1.07 GB) 187 us, 5.7 TB/s, where a large copy reaches
 * 5.1 and an addition 6.0; 4096 x 8192 bf16 likewise 50 us, 5.3 TB/s.  With 8-bit output in groups of 128 (236 MB) 50
 * us, 4.7 TB/s, beside 540 vector instructions for 16 values a lane.  One row of 4096: 3 us, a launch. */
template <int T, int THREADS, int RUNS, int V, bool Q8>
__global__ __launch_bounds__(THREADS) void rmsnorm_kernel(norm_args a)
{
    typedef typename dn_elt<T>::store E;
    __shared__ double lds[THREADS / 64];
    const int tid = threadIdx.x, n = a.n, runs = RUNS ? RUNS : (n + THREADS * V - 1) / (THREADS * V);
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const E *in = (const E *)a.input + row * n, *add = a.add ? (const E *)a.add + row * n : 0;
        E *sum = a.sum ? (E *)a.sum + row * n : 0;
        /* Behind the empty statement the compiler knows nothing of where a run lies, and does not prepare the loads and
         * stores of all runs beforehand: 58 registers instead of 95 with 8-bit output, and a third more waves. */
        int first = tid * V;
        asm("" : "+v"(first));
        auto at = [&](int j) { return j * THREADS * V + first; };
        auto added = [&](float s[V], const float t[V]) {
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] = (float)(E)(s[e] + t[e]);
        };
        float s[RUNS ? RUNS : 1][V];
        double acc = 0;
        auto square = [&](const float v[V]) {
#pragma unroll
            for (int e = 0; e < V; ++e) acc = fma((double)v[e], (double)v[e], acc);
        };
        if (RUNS) {
            float t[RUNS ? RUNS : 1][V];
#pragma unroll
            for (int j = 0; j < RUNS; ++j) load_run<T, V>(in, at(j), n, s[j]);
            if (add) {
#pragma unroll
                for (int j = 0; j < RUNS; ++j) load_run<T, V>(add, at(j), n, t[j]);
#pragma unroll
                for (int j = 0; j < RUNS; ++j) {
                    added(s[j], t[j]);
                    if (sum) store_run<E, V>(sum, at(j), n, s[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < RUNS; ++j) square(s[j]);
        } else {
            for (int j = 0; j < runs; ++j) {
                float v[V], t[V];
                load_run<T, V>(in, at(j), n, v);
                if (add) {
                    load_run<T, V>(add, at(j), n, t);
                    added(v, t);
                    if (sum) store_run<E, V>(sum, at(j), n, v);
                }
                square(v);
            }
        }
        acc = block_all<THREADS, false>(acc, lds);
        double mean = acc * a.inv_n;
        if (Q8 && acc <= 1.7976931348623157e308) mean = fma(fma(-mean, (double)n, acc), a.inv_n, mean); /* acc / n as it rounds */
        const double rms = sqrt(mean + (double)a.eps), r = 1. / rms;
        auto values = [&](int j, float v[V]) {
            if (RUNS) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = s[j][e];
                return;
            }
            load_run<T, V>(sum ? sum : in, at(j), n, v);
            if (add && !sum) {
                float t[V];
                load_run<T, V>(add, at(j), n, t);
                added(v, t);
            }
        };
        auto scales = [&](int j, float g[V]) {
            if (a.scales) load_run<DN_F32, V>(a.scales, at(j), n, g);
            else
#pragma unroll
                for (int e = 0; e < V; ++e) g[e] = 1;
        };
        if (Q8) { /* before the output, which may take the place of what is read here */
            /* convert s again below rather than hold its 64-bit forms: with fewer registers more rows fit on a CU */
#pragma unroll
            for (int j = 0; j < RUNS; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) asm volatile("" : "+v"(s[j][e]));
            const int lanes = a.group / V, groups = a.group ? (n + a.group - 1) / a.group : 1;
            const bool finite = acc <= 1.7976931348623157e308; /* and so every s */
            const bool ties = __builtin_amdgcn_readfirstlane(q8_may_tie(rms));
            const double inf = __longlong_as_double(0x7ff0000000000000LL);
            /* p of a run, and max|p|: infinity where a factor is not finite (x * 0 is NaN then) */
            auto products = [&](int j, double p[V]) {
                float v[V], g[V], poison = 0;
                double largest = 0;
                values(j, v);
                scales(j, g);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    p[e] = (double)v[e] * (double)g[e];
                    poison = fmaf(g[e], 0.f, poison);
                    largest = fmax(largest, fabs(p[e]));
                }
                if (!finite)
#pragma unroll
                    for (int e = 0; e < V; ++e) poison = fmaf(v[e], 0.f, poison);
                return poison == 0 && r == r ? largest : inf;
            };
            double row_largest = 0;
            if (a.group == 0) {
#pragma unroll
                for (int j = 0; j < runs; ++j) {
                    double p[V];
                    row_largest = fmax(row_largest, products(j, p));
                }
                row_largest = block_all<THREADS, true>(row_largest, lds);
            }
#pragma unroll
            for (int j = 0; j < runs; ++j) {
                const int i = at(j);
                double p[V];
                const double largest = a.group ? group_largest(products(j, p), lanes) : (products(j, p), row_largest);
                /* an infinite maximum stays one: r may be 0 then */
                const float c = largest < inf ? q8_step(largest, rms, r, ties) : __int_as_float(0x7fc00000);
                const double factor = c > 0 ? q8_factor(r, c) : 0; /* codes are 0 where c is 0 or NaN */
                if (a.group ? i < n && (tid & (lanes - 1)) == 0 : i == 0) a.q8_scales[row * groups + (a.group ? i / a.group : 0)] = c;
                unsigned q[V];
                if (ties) {
                    const double step = rms * (double)c; /* 29 and 24 bits: exact */
#pragma unroll
                    for (int e = 0; e < V; ++e) q[e] = (unsigned)(c > 0 ? q8_nearest(q8_code(p[e], factor), p[e], step) : 0);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) q[e] = (unsigned)(c > 0 ? q8_code(p[e], factor) : 0);
                }
                signed char *to = a.q8 + row * n;
                if (i + V <= n) {
                    typedef unsigned __attribute__((ext_vector_type(V / 4))) words;
                    typedef words __attribute__((aligned(1))) words_anywhere;
                    words w;
#pragma unroll
                    for (int e = 0; e < V; e += 4)
                        w[e / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[e + 3], q[e + 2], 0x0c0c0400),
                                                         __builtin_amdgcn_perm(q[e + 1], q[e], 0x0c0c0400), 0x05040100);
                    *(words_anywhere *)(to + i) = w;
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (i + e < n) to[i + e] = (signed char)q[e];
                }
            }
        }
        if (a.output) {
            /* in 64 bits: either product of two factors may leave the range of 32 where the result does not */
#pragma unroll
            for (int j = 0; j < runs; ++j) {
                float v[V], g[V];
                values(j, v);
                scales(j, g);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = (float)((double)v[e] * r * (double)g[e]);
                store_run<E, V>((E *)a.output + row * n, at(j), n, v);
            }
        }
    }
}

/* Which form a row takes: one run a lane up to 256 lanes, then two, so that several rows share a CU and their loads
 * and stores overlap (8192 bf16, 4096 rows: 50 us by 512 lanes with two, 58 by 1024 with one, 56 by 256 with four), but
 * for 16-bit rows of 257 to 512 runs of eight, whose two runs take the registers of a row more (4096 bf16, 16384 rows with
 * residual: 92 us by 512, 94 by 256; without one 55 and 51, and to 8 bits 123 and 103: there 256 would be ahead).  768
 * lanes for what leaves a third of 1024 idle (3795 x 6000 fp32 69 us, 77 by 1024; bf16 43 and 54; 384 below 512 gave
 * nothing).  A row of more than 16384 values is read again for each step. */
template <int T, bool Q8>
static void norm_launch(const norm_args &a)
{
    constexpr int V = T == DN_F32 ? 4 : 8;
    const dim3 grid(a.rows < 65536 ? a.rows : 65536);
    const int runs = (int)(((long)a.n + V - 1) / V);
#define NM_LAUNCH(THREADS, RUNS) \
    hipLaunchKernelGGL((rmsnorm_kernel<T, THREADS, RUNS, V, Q8>), grid, dim3(THREADS), 0, dn_stream(), a)
    if (runs <= 64) NM_LAUNCH(64, 1);
    else if (runs <= 128) NM_LAUNCH(128, 1);
    else if (runs <= 256) NM_LAUNCH(256, 1);
    else if (V == 8 && runs <= 512) NM_LAUNCH(512, 1);
    else if (runs <= 512) NM_LAUNCH(256, 2);
    else if (runs <= 1024) NM_LAUNCH(512, 2);
    else if (runs <= 1536) NM_LAUNCH(768, 2);
    else if (runs <= 2048) NM_LAUNCH(1024, 2);
    else if (V == 4 && runs <= 4096) NM_LAUNCH(1024, 16 / V);
    else NM_LAUNCH(1024, 0);
#undef NM_LAUNCH
}

extern "C" int forward_rmsnorm_gpu(const void *input, const void *add, const float *scales, void *sum_output,
                                   void *output, signed char *q8_output, float *q8_scales, int type, int rows,
                                   int n, int q8_group, float eps)
{
    const char *me = "forward_rmsnorm_gpu";
    if (!dn_is_float_type(type)) return dn_refuse(me, "unknown element type");
    if (rows < 0 || n < 1 || n > 0x7fff0000) return dn_refuse(me, "bad geometry"); /* indexes of a row stay within an int */
    if (!(eps >= 0) || !(eps <= 3.402823466e38f)) return dn_refuse(me, "eps must be a finite number that is not negative");
    if (rows == 0) return 0;
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
    hip_require_device(me);
    const norm_args a = {input, add, scales, sum_output, output, q8_output, q8_scales, rows, n, q8_group, eps, 1. / n};
    if (type == DN_F32) q8_output ? norm_launch<DN_F32, true>(a) : norm_launch<DN_F32, false>(a);
    else if (type == DN_F16) q8_output ? norm_launch<DN_F16, true>(a) : norm_launch<DN_F16, false>(a);
    else q8_output ? norm_launch<DN_BF16, true>(a) : norm_launch<DN_BF16, false>(a);
    dn_check_launch(me);
    return 0;
}
