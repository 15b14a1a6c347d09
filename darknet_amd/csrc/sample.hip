/*
 * sample.hip - one token for each row of logits from a random number: temperature, top-k, top-p, min-p.
 *
 * The tokens of a row are ordered by (logit descending, index ascending).  w = exp((logit - largest) / T).
 *   top-k   the first k
 *   top-p   the shortest run of first tokens whose mass is at least p times the mass of what top-k left
 *   min-p   of these the tokens with w >= min_p (the largest has w = 1)
 * The answer is the first token in index order at which the running mass reaches u times the mass kept.
 *
 * Masses are whole numbers, rint(w * 2^shift) with w in 64 bits: their sums do not depend on the
 * order in which lanes and atomics add them, so the same row gives the same token in every run, and a
 * border between two tokens lies where the formula puts it to within 2^-shift of the largest mass.
 */
#include <math.h>

#include "row_types.h"

#define SM_THREADS 1024

struct sample_args {
    const void *logits;
    const float *temperature, *top_p, *min_p, *uniform;
    const int *top_k;
    int *tokens;
    float *probs;
    long stride;
    int rows, n, shift;
};

/* A token's place in the order as one number: larger is earlier.  0 for a token that cannot be drawn (NaN, -inf). */
__device__ __forceinline__ unsigned long long place_of(float l, int i)
{
    if (!(l > -INFINITY)) return 0;
    const unsigned b = __float_as_uint(l + 0.f); /* -0 ranks as 0 */
    const unsigned key = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((unsigned long long)key << 32) | (0xffffffffu - (unsigned)i);
}

__device__ __forceinline__ double weight_of(float l, float largest, double temperature)
{
    if (l == largest) return 1;
    return exp(((double)l - (double)largest) / temperature);
}

__device__ __forceinline__ unsigned long long mass_of(double w, int shift)
{
    return (unsigned long long)rint(ldexp(w, shift));
}

template <int T>
__global__ __launch_bounds__(SM_THREADS) void sample_kernel(sample_args a)
{
    typedef unsigned long long u64;
    typedef typename dn_elt<T>::store E;
    __shared__ u64 hist[256], part[SM_THREADS];
    __shared__ u64 s_prefix, s_above;
    __shared__ int s_token;
    const int tid = threadIdx.x, n = a.n;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const E *x = (const E *)a.logits + row * a.stride;
        float t = a.temperature ? a.temperature[row] : 1.f;
        int k = a.top_k ? a.top_k[row] : 0;
        if (!(t > 0)) { /* the largest */
            t = 1;
            k = 1;
        }
        const float p = a.top_p ? a.top_p[row] : 1.f;
        const float floor_w = a.min_p ? fminf(a.min_p[row], 1.f) : 0.f;

        float largest = -INFINITY;
        for (int i = tid; i < n; i += SM_THREADS)
            if ((float)x[i] > largest) largest = (float)x[i];
        largest = dn_wave_max(largest);
        __syncthreads();
        if ((tid & 63) == 0) part[tid >> 6] = __float_as_uint(largest);
        __syncthreads();
        for (int w = 0; w < SM_THREADS / 64; ++w) largest = fmaxf(largest, __uint_as_float((unsigned)part[w]));
        if (!(largest > -INFINITY)) {
            if (tid == 0) {
                a.tokens[row] = -1;
                if (a.probs) a.probs[row] = 0;
            }
            continue;
        }
        /* The place at which the running count (or mass) of the order reaches `target`, among the
         * places from `least` on; 0 if it never does. */
        auto find = [&](bool mass, double target, u64 least) {
            u64 prefix = 0, above = 0;
            for (int bit = 56; bit >= 0; bit -= 8) {
                __syncthreads();
                if (tid < 256) hist[tid] = 0;
                __syncthreads();
                for (int i = tid; i < n; i += SM_THREADS) {
                    const float l = (float)x[i];
                    const u64 c = place_of(l, i);
                    if (c < least || !c || (bit < 56 && c >> (bit + 8) != prefix)) continue;
                    atomicAdd(&hist[(c >> bit) & 255], mass ? mass_of(weight_of(l, largest, t), a.shift) : 1ull);
                }
                __syncthreads();
                if (tid == 0) {
                    int d = 255;
                    u64 sum = above;
                    while (d > 0 && (double)(sum + hist[d]) < target) sum += hist[d--];
                    if ((double)(sum + hist[d]) < target) d = -1;
                    s_above = sum;
                    s_prefix = d < 0 ? ~0ull : prefix << 8 | (u64)d;
                }
                __syncthreads();
                prefix = s_prefix;
                above = s_above;
                if (prefix == ~0ull) return (u64)0;
            }
            return prefix;
        };
        auto block_sum = [&](u64 v) {
            __syncthreads();
            v = dn_wave_sum(v);
            if ((tid & 63) == 0) part[tid >> 6] = v;
            __syncthreads();
            u64 s = 0;
            for (int w = 0; w < SM_THREADS / 64; ++w) s += part[w];
            return s;
        };
        auto kept_mass = [&](int i, u64 least, double floor_of) {
            const float l = (float)x[i];
            const u64 c = place_of(l, i);
            if (!c || c < least) return (u64)0;
            const double w = weight_of(l, largest, t);
            return w >= floor_of ? mass_of(w, a.shift) : (u64)0;
        };
        u64 least = 0;
        if (k > 0 && k < n) least = find(false, (double)k, 0);
        if (p < 1) {
            u64 m = 0;
            for (int i = tid; i < n; i += SM_THREADS) m += kept_mass(i, least, 0.);
            m = block_sum(m);
            const u64 at = find(true, fmax((double)p * (double)m, 1.), least); /* one token at least */
            if (at > least) least = at;
        }
        /* the running mass in index order: each lane a piece of the row */
        const int piece = (n + SM_THREADS - 1) / SM_THREADS, lo = (int)min((long)n, (long)tid * piece), hi = min(n, lo + piece);
        const double floor_of = floor_w > 0 ? (double)floor_w : 0.;
        u64 own = 0;
        for (int i = lo; i < hi; ++i) own += kept_mass(i, least, floor_of);
        const u64 total = block_sum(own);
        __syncthreads();
        part[tid] = own;
        if (tid == 0) s_token = n;
        __syncthreads();
        u64 run = 0;
        for (int j = 0; j < tid; ++j) run += part[j];
        const double u = a.uniform[row], target = (u > 0 ? fmin(u, 1.) : 0.) * (double)total;
        if (own && (double)(run + own) >= target) {
            int i = lo;
            u64 m;
            for (; i < hi; ++i) {
                m = kept_mass(i, least, floor_of);
                run += m;
                if (m && (double)run >= target) break;
            }
            atomicMin(&s_token, i);
        }
        __syncthreads();
        if (tid == 0) {
            const int token = s_token;
            a.tokens[row] = token;
            if (a.probs) a.probs[row] = (float)((double)kept_mass(token, least, floor_of) / (double)total);
        }
        __syncthreads();
    }
}

extern "C" size_t sample_workspace_bytes(int rows, int n)
{
    (void)rows;
    (void)n;
    return 0;
}

extern "C" int sample_rows_gpu(const void *logits, int type, int rows, int n, long stride, const float *temperature,
                               const int *top_k, const float *top_p, const float *min_p, const float *uniform,
                               int *tokens, float *probs, void *workspace)
{
    const char *me = "sample_rows_gpu";
    if (!dn_is_float_type(type)) return dn_refuse(me, "unknown element type");
    if (rows < 0 || n < 1 || n > (1 << 24)) return dn_refuse(me, "bad geometry (1 to 2^24 tokens)");
    if (stride < n) return dn_refuse(me, "the stride is shorter than a row");
    if (!logits || !uniform || !tokens) return dn_refuse(me, "a buffer is missing");
    if (!dn_aligned(logits, dn_type_bytes(type)) || !dn_aligned(temperature, 4) || !dn_aligned(top_k, 4) ||
        !dn_aligned(top_p, 4) || !dn_aligned(min_p, 4) || !dn_aligned(uniform, 4) || !dn_aligned(tokens, 4) ||
        !dn_aligned(probs, 4))
        return dn_refuse(me, "a buffer is not aligned to its element type");
    (void)workspace;
    if (rows == 0) return 0;
    hip_require_device(me);
    int shift = 62; /* n * 2^shift <= 2^62, and a weight keeps the 52 bits it has */
    while ((long)n > 1L << (62 - shift)) --shift;
    if (shift > 52) shift = 52;
    const sample_args a = {logits, temperature, top_p, min_p, uniform, top_k, tokens, probs, stride, rows, n, shift};
    const dim3 grid(rows < 65536 ? rows : 65536), block(SM_THREADS);
    if (type == DN_F32) hipLaunchKernelGGL((sample_kernel<DN_F32>), grid, block, 0, dn_stream(), a);
    else if (type == DN_F16) hipLaunchKernelGGL((sample_kernel<DN_F16>), grid, block, 0, dn_stream(), a);
    else hipLaunchKernelGGL((sample_kernel<DN_BF16>), grid, block, 0, dn_stream(), a);
    dn_check_launch(me);
    return 0;
}
