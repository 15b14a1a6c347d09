/*
 * sample.hip - one token for each row of logits from a random number: temperature, top-k, top-p, min-p.
 *
 * The tokens of a row are ordered by (logit descending, index ascending).  w = exp((logit - largest) / T).
 *   top-k   the first k
 *   top-p   the shortest run of first tokens whose mass is at least p times the mass of what top-k left
 *   min-p   of these the tokens with w >= min_p (the largest has w = 1)
 * The answer is the first token in index order at which the running mass reaches u times the mass kept.
 *
 * Masses are whole numbers, rint(w * 2^38) with w in 64 bits: their sums do not depend on the order in which
 * lanes and atomics add them, so the same row gives the same token in every run, and a border between two
 * tokens lies where the formula puts it to within 2^-38 of the largest mass.
 *
 * No row is sorted.  The logits are counted and weighed in 512 bins, an eighth of T wide, below the largest; the
 * bin in which the order's prefix ends is known from the running sums, everything in the bins before it is
 * kept, and only that bin's tokens (the candidates) are looked at more closely: digit by digit of their places.
 */
#include <math.h>

#include "row_types.h"

typedef unsigned long long u64;

#define SM_BINS 512
#define SM_PER_T 8
#define SM_SHIFT 38
#define SM_CANDIDATES 4096 /* that fit into LDS */
#define SM_SEGMENTS 32

struct sample_args {
    const void *logits;
    const float *temperature, *top_p, *min_p, *uniform;
    const int *top_k;
    int *tokens;
    float *probs;
    unsigned char *workspace;
    long stride;
    int rows, n, segments, length, block; /* length: tokens of a segment, block: of what its mass is summed over */
};

/* A row's settings, those that are off in one form. */
struct sample_row {
    double log2_per_logit; /* log2(e) / T */
    double floor;          /* min-p */
    double uniform;        /* in 0 .. 1 */
    float bins_per_logit;
    float p;               /* 2: off */
    int k;                 /* 0: off */
};

/* Every array is read, a missing one at another's place, so that the loads are in flight together. */
__device__ __forceinline__ sample_row settings_of(const sample_args &a, long row)
{
    sample_row s;
    const float t_of = (a.temperature ? a.temperature : a.uniform)[row], p_of = (a.top_p ? a.top_p : a.uniform)[row];
    const float m_of = (a.min_p ? a.min_p : a.uniform)[row];
    const int k_of = (a.top_k ? a.top_k : (const int *)a.uniform)[row];
    const float u = a.uniform[row];
    float t = a.temperature ? t_of : 1.f;
    int k = a.top_k ? k_of : 0;
    if (!(t > 0)) { /* the first of the order */
        t = 1;
        k = 1;
    }
    s.k = k > 0 && k < a.n ? k : 0;
    s.p = a.top_p && p_of < 1 ? p_of : 2.f;
    s.floor = a.min_p && m_of > 0 ? (double)fminf(m_of, 1.f) : 0.;
    s.uniform = u > 0 ? (double)fminf(u, 1.f) : 0.;
    s.log2_per_logit = 1.4426950408889634 / (double)t;
    s.bins_per_logit = fminf(SM_PER_T / t, 3.402823466e38f);
    return s;
}

/* A token's place in the order as one number: larger is earlier.  0 for a token that cannot be drawn (NaN, -inf). */
__device__ __forceinline__ u64 place_of(float l, int i)
{
    if (!(l > -INFINITY)) return 0;
    const unsigned b = __float_as_uint(l + 0.f); /* -0 ranks as 0 */
    const unsigned key = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((u64)key << 32) | (0xffffffffu - (unsigned)i);
}

__device__ __forceinline__ float logit_of(u64 place)
{
    const unsigned key = (unsigned)(place >> 32);
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

/* 2^x for x <= 0 as the first ten terms of its series around the nearest whole exponent: to 7e-12. */
__device__ __forceinline__ double weight_of(float l, float largest, const sample_row &s)
{
    if (l == largest) return 1; /* also where both are infinite */
    const double x = ((double)l - (double)largest) * s.log2_per_logit;
    if (!(x > -64)) return 0;
    const double whole = rint(x), f = x - whole;
    double p = 1.0178086009239696e-07;
    p = fma(p, f, 1.3215486790144305e-06);
    p = fma(p, f, 1.5252733804059838e-05);
    p = fma(p, f, 0.00015403530393381606);
    p = fma(p, f, 0.0013333558146428441);
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.055504108664821576);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.);
    return ldexp(p, (int)whole);
}

/* rint(w * 2^38): added to 2^52 the number stands in the low bits of the sum. */
__device__ __forceinline__ u64 mass_of(double w)
{
    return (u64)__double_as_longlong(w * 0x1p38 + 0x1p52) & 0xfffffffffffffull;
}

__device__ __forceinline__ int bin_of(float l, float largest, const sample_row &s)
{
    const float below = (largest - l) * s.bins_per_logit;
    return l == largest ? 0 : below < SM_BINS - 1 ? (int)below : SM_BINS - 1;
}

/* Where the ordered prefix of a row ends, as far as the bins tell. */
struct sample_border {
    int first;         /* tokens in the bins before this one are in the prefix */
    int lo, hi, k_bin; /* candidates: the tokens in bins lo .. hi and k_bin */
    int k_need;        /* top-k: how many of k_bin's tokens are among the first k */
    u64 mass_lo, mass_k; /* mass in the bins before lo, before k_bin */
};

struct sample_lds {
    u64 mass[SM_BINS + 64];
    unsigned count[SM_BINS + 64];
    u64 digit[256 + 64], part[16];
    unsigned digit_count[256];
    u64 prefix, base, found;
    unsigned single;
    sample_border border;
};

template <class V>
__device__ __forceinline__ V wave_scan(V v)
{
    return dn_wave_scan(v, (V)0, [](V a, V b) { return a + b; });
}

/* Where bin b stands in LDS: a gap after every E bins spreads the runs of E that the lanes read over the banks. */
template <int E>
__device__ __forceinline__ int slot_of(int b)
{
    return b + b / E;
}
#define SM_SLOTS (SM_BINS + 64)
__device__ __forceinline__ int bin_slot(int b) { return slot_of<SM_BINS / 64>(b); }
__device__ __forceinline__ int digit_slot(int d) { return slot_of<4>(d); }

/* One wave: the first of N bins (in order, or from the last one down) at which base + running sum reaches the
 * target, and the sum before it; N if none does.  The target is at least 1. */
template <int N, bool DOWN, class V>
__device__ __forceinline__ int find_bin(const V *bins, u64 base, double target, u64 &before, int lane)
{
    constexpr int E = N / 64;
    u64 own = 0, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int b = lane * E + e;
        v[e] = bins[slot_of<E>(DOWN ? N - 1 - b : b)];
        own += v[e];
    }
    u64 run = base + wave_scan(own) - own;
    int at = N;
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (at == N && v[e] && (double)(run + v[e]) >= target) {
            at = lane * E + e;
            sum = run;
        }
        run += v[e];
    }
    const u64 any = __ballot(at < N);
    if (!any) {
        before = 0;
        return N;
    }
    const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)any) - 1);
    before = dn_lane(sum, src);
    at = (int)dn_lane((unsigned)at, src);
    return DOWN ? N - 1 - at : at;
}

/* One wave: the borders from the bins in LDS. */
__device__ __forceinline__ sample_border border_of(const sample_lds &s, const sample_row &r, int lane)
{
    sample_border b = {SM_BINS, SM_BINS, SM_BINS - 1, -1, 0, 0, 0};
    u64 mass_least = 0, mass_most = 0, count = 0;
    if (r.p < 1 || r.k) {
        u64 own_mass = 0;
        if (r.k) {
            b.k_bin = find_bin<SM_BINS, false>(s.count, 0, (double)r.k, count, lane);
            if (b.k_bin == SM_BINS) b.k_bin = -1; /* fewer than k tokens can be drawn at all */
            else b.k_need = r.k - (int)count;
        }
#pragma unroll
        for (int e = 0; e < SM_BINS / 64; ++e) {
            const int at = lane * (SM_BINS / 64) + e;
            if (b.k_bin < 0 || at < b.k_bin) own_mass += s.mass[bin_slot(at)];
        }
        mass_least = dn_wave_sum(own_mass);
        mass_most = b.k_bin < 0 ? mass_least : mass_least + s.mass[bin_slot(b.k_bin)];
        b.mass_k = mass_least;
    }
    if (r.p < 1) {
        u64 ignore;
        b.lo = find_bin<SM_BINS, false>(s.mass, 0, fmax((double)r.p * (double)mass_least, 1.), b.mass_lo, lane);
        b.hi = find_bin<SM_BINS, false>(s.mass, 0, fmax((double)r.p * (double)mass_most, 1.), ignore, lane);
        b.first = b.lo;
    } else if (b.k_bin >= 0) {
        b.first = b.k_bin;
    }
    return b;
}

__device__ __forceinline__ bool is_candidate(const sample_border &b, int bin)
{
    return (bin >= b.lo && bin <= b.hi) || bin == b.k_bin;
}

template <class T>
__device__ __forceinline__ T block_sum(T v, sample_lds &s)
{
    v = dn_wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = v;
    __syncthreads();
    T t = 0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) t += s.part[w];
    return t;
}

__device__ __forceinline__ float block_largest(float v, sample_lds &s)
{
    v = dn_wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = __float_as_uint(v);
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x / 64; ++w) v = fmaxf(v, __uint_as_float((unsigned)s.part[w]));
    return v;
}

__device__ __forceinline__ u64 shift_right(u64 v, int bits) { return bits > 63 ? 0 : v >> bits; }

/* The place at which base + the running sum of value(place) over the places handed out by each(), from the largest
 * down, reaches the target.  By eight bits a round, from the first bit in which two of the places differ. */
template <class Each, class Value>
__device__ __forceinline__ u64 find_place(Each each, Value value, u64 base, double target, sample_lds &s)
{
    const int tid = threadIdx.x, lane = tid & 63;
    u64 most = 0, least = ~0ull;
    each([&](u64 c) {
        most = c > most ? c : most;
        least = c < least ? c : least;
    });
    most = dn_wave_max(most);
    least = ~dn_wave_max(~least);
    __syncthreads();
    if (tid == 0) {
        s.prefix = 0;
        s.found = ~0ull;
    }
    __syncthreads();
    if (lane == 0) {
        atomicMax(&s.prefix, most);
        atomicMin(&s.found, least);
    }
    __syncthreads();
    most = s.prefix;
    least = s.found;
    if (most <= least) return most;
    int bit = 64 - __clzll((long long)(most ^ least));
    u64 prefix = shift_right(most, bit);
    while (bit > 0) {
        const int next = bit > 8 ? bit - 8 : 0;
        __syncthreads();
        if (tid < 256) {
            s.digit[digit_slot(tid)] = 0;
            s.digit_count[tid] = 0;
        }
        __syncthreads();
        each([&](u64 c) {
            if (shift_right(c, bit) != prefix) return;
            const int d = (int)(c >> next) & ((1 << (bit - next)) - 1);
            atomicAdd(&s.digit[digit_slot(d)], value(c));
            atomicAdd(&s.digit_count[d], 1u);
        });
        __syncthreads();
        if (tid < 64) {
            u64 before;
            const int d = find_bin<256, true>(s.digit, base, target, before, lane);
            if (lane == 0) {
                s.prefix = prefix << (bit - next) | (u64)(d & 255);
                s.base = before;
                s.single = s.digit_count[d & 255] == 1;
            }
        }
        __syncthreads();
        prefix = s.prefix;
        base = s.base;
        bit = next;
        if (bit > 0 && s.single) {
            each([&](u64 c) {
                if (shift_right(c, bit) == prefix) s.found = c;
            });
            __syncthreads();
            return s.found;
        }
    }
    return prefix;
}

/* The last place of the kept prefix, from the candidates: top-k first, then top-p of what it left. */
template <class Each>
__device__ __forceinline__ u64 last_place(Each each, const sample_border &b, const sample_row &r, float largest, sample_lds &s)
{
    auto mass = [&](u64 c) { return mass_of(weight_of(logit_of(c), largest, r)); };
    u64 k_place = 0, p_place = 0, mass_k = b.mass_k;
    if (b.k_bin >= 0) {
        auto in_k_bin = [&](auto f) {
            each([&](u64 c) {
                if (bin_of(logit_of(c), largest, r) == b.k_bin) f(c);
            });
        };
        k_place = find_place(in_k_bin, [](u64) { return (u64)1; }, 0, (double)b.k_need, s);
        if (r.p < 1) {
            u64 m = 0;
            in_k_bin([&](u64 c) { m += c >= k_place ? mass(c) : 0; });
            mass_k += block_sum(m, s);
        }
    }
    if (r.p < 1)
        p_place = find_place([&](auto f) { each([&](u64 c) { if (c >= k_place) f(c); }); }, mass, b.mass_lo,
                             fmax((double)r.p * (double)mass_k, 1.), s);
    return k_place > p_place ? k_place : p_place;
}

/* Each lane has `own`, the mass of its piece of consecutive tokens; pieces follow each other in lane order.  Finds the
 * piece in which base + running mass reaches the target: true for its lane, with the sum before it. */
__device__ __forceinline__ bool reaches(u64 own, u64 base, double target, u64 &before, sample_lds &s)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 incl = wave_scan(own);
    __syncthreads();
    if (lane == 63) s.part[wave] = incl;
    __syncthreads();
    u64 run = base + incl - own;
    for (int w = 0; w < wave; ++w) run += s.part[w];
    before = run;
    return own && (double)run < target && (double)(run + own) >= target;
}

__device__ __forceinline__ double draw_target(const sample_row &r, u64 total) { return fmax(r.uniform * (double)total, 1.); }

__device__ __forceinline__ void answer(const sample_args &a, long row, int token, u64 mass, u64 total)
{
    a.tokens[row] = token;
    if (a.probs) a.probs[row] = total ? (float)((double)mass / (double)total) : 0.f;
}

/* Eight neighbouring tokens from i on; -inf behind `end`. */
template <int T>
__device__ __forceinline__ void load8(const typename dn_elt<T>::store *x, int i, int end, bool vectors, float l[8])
{
    typedef typename dn_elt<T>::store S;
    typedef S S4 __attribute__((ext_vector_type(4)));
    if (vectors && i + 8 <= end) {
        const S4 u = *(const S4 *)(x + i), v = *(const S4 *)(x + i + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            l[e] = (float)u[e];
            l[e + 4] = (float)v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) l[e] = i + e < end ? (float)x[i + e] : -INFINITY;
    }
}

template <int T>
__device__ __forceinline__ bool rows_aligned(const sample_args &a)
{
    const int size = sizeof(typename dn_elt<T>::store);
    return ((uintptr_t)a.logits & 15) == 0 && ((a.stride * size) & 15) == 0;
}

/* ---- a row of up to 8192 tokens: one workgroup, the row in registers ---------------------------------- */
template <int T, int E, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_row_kernel(sample_args a)
{
    typedef typename dn_elt<T>::store S;
    __shared__ sample_lds s;
    __shared__ u64 candidates[SM_CANDIDATES];
    __shared__ unsigned s_count;
    const int tid = threadIdx.x;
    const bool vectors = rows_aligned<T>(a);
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const S *x = (const S *)a.logits + row * a.stride;
        const sample_row r = settings_of(a, row);
        float l[E];
#pragma unroll
        for (int e = 0; e < E; e += 8) load8<T>(x, tid * E + e, a.n, vectors, l + e);
        float largest = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) largest = l[e] > largest ? l[e] : largest;
        largest = block_largest(largest, s);
        if (!(largest > -INFINITY)) {
            if (tid == 0) answer(a, row, -1, 0, 0);
            continue;
        }
        u64 last = 0;
        if (r.k || r.p < 1) {
            for (int i = tid; i < SM_SLOTS; i += THREADS) {
                s.count[i] = 0;
                s.mass[i] = 0;
            }
            if (tid == 0) s_count = 0;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (l[e] > -INFINITY) {
                    const int b = bin_slot(bin_of(l[e], largest, r));
                    if (r.k) atomicAdd(&s.count[b], 1u);
                    if (r.p < 1) atomicAdd(&s.mass[b], mass_of(weight_of(l[e], largest, r)));
                }
            __syncthreads();
            if (tid < 64) {
                const sample_border b = border_of(s, r, tid);
                if (tid == 0) s.border = b;
            }
            __syncthreads();
            const sample_border b = s.border;
            if (b.k_bin >= 0 || r.p < 1) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (l[e] > -INFINITY && is_candidate(b, bin_of(l[e], largest, r))) {
                        const unsigned at = atomicAdd(&s_count, 1u);
                        if (at < SM_CANDIDATES) candidates[at] = place_of(l[e], tid * E + e);
                    }
                __syncthreads();
                const int count = (int)s_count;
                last = last_place([&](auto f) {
                    if (count <= SM_CANDIDATES) {
                        for (int i = tid; i < count; i += THREADS) f(candidates[i]);
                        return;
                    }
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (l[e] > -INFINITY && is_candidate(b, bin_of(l[e], largest, r))) f(place_of(l[e], tid * E + e));
                }, b, r, largest, s);
            }
        }
        auto kept_mass = [&](int e) {
            const u64 c = place_of(l[e], tid * E + e);
            if (!c || c < last) return (u64)0;
            const double w = weight_of(l[e], largest, r);
            return w >= r.floor ? mass_of(w) : (u64)0;
        };
        u64 own = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) own += kept_mass(e);
        const u64 total = block_sum(own, s);
        const double target = draw_target(r, total);
        u64 run;
        if (reaches(own, 0, target, run, s)) {
            bool done = false;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const u64 m = done ? 0 : kept_mass(e);
                run += m;
                if (m && (double)run >= target) {
                    answer(a, row, tid * E + e, m, total);
                    done = true;
                }
            }
        }
        __syncthreads();
    }
}

/* ---- longer rows: cut into segments, four passes ---------------------------------------------------------
 * 1 largest of each segment (and the row's bins cleared)
 * 2 bins of the row, rows with top-k or top-p only: each segment's in LDS, then added to the row's
 * 3 borders from the bins; the kept mass of each block of tokens and each segment's candidates
 * 4 one workgroup a row: the prefix' end among the candidates, the block that the draw falls into, the token */
#define SM_SPLIT_THREADS 256
#define SM_STRIP (SM_SPLIT_THREADS * 8) /* tokens that a workgroup takes at a time */
#define SM_BLOCKS 512                   /* of a row, at most: they are summed in LDS */
#define SM_LISTED 512                   /* candidates that a segment keeps a list of */

struct sample_space {
    size_t kept, bins_mass, border, list, bins_count, largest, found, bytes;
};

__host__ __device__ static inline sample_space space_of(int rows, int segments)
{
    sample_space w;
    const size_t all = (size_t)rows * segments;
    w.kept = 0;
    w.bins_mass = w.kept + (size_t)rows * SM_BLOCKS * 8;
    w.border = w.bins_mass + (size_t)rows * SM_BINS * 8;
    w.list = w.border + (size_t)rows * sizeof(sample_border);
    w.bins_count = w.list + all * SM_LISTED * 8;
    w.largest = w.bins_count + (size_t)rows * SM_BINS * 4;
    w.found = w.largest + all * 4;
    w.bytes = w.found + all * 4;
    return w;
}

template <int T>
__global__ __launch_bounds__(SM_SPLIT_THREADS) void sample_largest_kernel(sample_args a)
{
    typedef typename dn_elt<T>::store S;
    __shared__ float part[SM_SPLIT_THREADS / 64];
    const sample_space ws = space_of(a.rows, a.segments);
    const bool vectors = rows_aligned<T>(a);
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const S *x = (const S *)a.logits + row * a.stride;
        const int lo = blockIdx.x * a.length, hi = min(a.n, lo + a.length);
        float m = -INFINITY;
        for (int i = lo + threadIdx.x * 8; i < hi; i += SM_STRIP) {
            float l[8];
            load8<T>(x, i, hi, vectors, l);
#pragma unroll
            for (int e = 0; e < 8; ++e) m = l[e] > m ? l[e] : m;
        }
        m = dn_wave_max(m);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
        __syncthreads();
        if (threadIdx.x == 0)
            ((float *)(a.workspace + ws.largest))[row * a.segments + blockIdx.x] = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i < SM_BINS; i += SM_SPLIT_THREADS) {
                ((u64 *)(a.workspace + ws.bins_mass))[row * SM_BINS + i] = 0;
                ((unsigned *)(a.workspace + ws.bins_count))[row * SM_BINS + i] = 0;
            }
    }
}

__device__ __forceinline__ float row_largest(const sample_args &a, const sample_space &ws, long row)
{
    const int lane = threadIdx.x & 63;
    const float *m = (const float *)(a.workspace + ws.largest) + row * a.segments;
    return dn_wave_max(lane < a.segments ? m[lane] : -INFINITY);
}

template <int T>
__global__ __launch_bounds__(SM_SPLIT_THREADS) void sample_bins_kernel(sample_args a)
{
    typedef typename dn_elt<T>::store S;
    __shared__ u64 mass[SM_BINS];
    __shared__ unsigned count[SM_BINS];
    const sample_space ws = space_of(a.rows, a.segments);
    const bool vectors = rows_aligned<T>(a);
    const int tid = threadIdx.x;
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const sample_row r = settings_of(a, row);
        if (!r.k && !(r.p < 1)) continue;
        const float largest = row_largest(a, ws, row);
        const S *x = (const S *)a.logits + row * a.stride;
        const int lo = blockIdx.x * a.length, hi = min(a.n, lo + a.length);
        __syncthreads();
        for (int i = tid; i < SM_BINS; i += SM_SPLIT_THREADS) {
            mass[i] = 0;
            count[i] = 0;
        }
        __syncthreads();
        for (int i = lo + tid * 8; i < hi; i += SM_STRIP) {
            float l[8];
            load8<T>(x, i, hi, vectors, l);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (!(l[e] > -INFINITY)) continue;
                const int b = bin_of(l[e], largest, r);
                if (r.k) atomicAdd(&count[b], 1u);
                if (r.p < 1) atomicAdd(&mass[b], mass_of(weight_of(l[e], largest, r)));
            }
        }
        __syncthreads();
        for (int i = tid; i < SM_BINS; i += SM_SPLIT_THREADS) {
            if (mass[i]) atomicAdd((u64 *)(a.workspace + ws.bins_mass) + row * SM_BINS + i, mass[i]);
            if (count[i]) atomicAdd((unsigned *)(a.workspace + ws.bins_count) + row * SM_BINS + i, count[i]);
        }
    }
}

template <int T>
__global__ __launch_bounds__(SM_SPLIT_THREADS) void sample_kept_kernel(sample_args a)
{
    typedef typename dn_elt<T>::store S;
    __shared__ sample_lds s;
    __shared__ unsigned s_count;
    const sample_space ws = space_of(a.rows, a.segments);
    const bool vectors = rows_aligned<T>(a);
    const int tid = threadIdx.x;
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const sample_row r = settings_of(a, row);
        const float largest = row_largest(a, ws, row);
        __syncthreads();
        if (r.k || r.p < 1)
            for (int i = tid; i < SM_BINS; i += SM_SPLIT_THREADS) {
                s.mass[bin_slot(i)] = ((const u64 *)(a.workspace + ws.bins_mass))[row * SM_BINS + i];
                s.count[bin_slot(i)] = ((const unsigned *)(a.workspace + ws.bins_count))[row * SM_BINS + i];
            }
        if (tid == 0) s_count = 0;
        __syncthreads();
        if (tid < 64) {
            const sample_border b = border_of(s, r, tid);
            if (tid == 0) {
                s.border = b;
                if (blockIdx.x == 0) ((sample_border *)(a.workspace + ws.border))[row] = b;
            }
        }
        __syncthreads();
        const sample_border b = s.border;
        const S *x = (const S *)a.logits + row * a.stride;
        const int lo = blockIdx.x * a.length, hi = min(a.n, lo + a.length);
        u64 *list = (u64 *)(a.workspace + ws.list) + ((size_t)row * a.segments + blockIdx.x) * SM_LISTED;
        for (int from = lo; from < hi; from += a.block) {
            u64 own = 0;
            const int to = min(hi, from + a.block);
            for (int i = from + tid * 8; i < to; i += SM_STRIP) {
                float l[8];
                load8<T>(x, i, to, vectors, l);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (!(l[e] > -INFINITY)) continue;
                    const int bin = bin_of(l[e], largest, r);
                    if (bin < b.first) {
                        const double w = weight_of(l[e], largest, r);
                        if (w >= r.floor) own += mass_of(w);
                    } else if (is_candidate(b, bin)) {
                        const unsigned at = atomicAdd(&s_count, 1u);
                        if (at < SM_LISTED) list[at] = place_of(l[e], i + e);
                    }
                }
            }
            const u64 kept = block_sum(own, s);
            if (tid == 0) ((u64 *)(a.workspace + ws.kept))[row * SM_BLOCKS + from / a.block] = kept;
        }
        __syncthreads();
        if (tid == 0) ((int *)(a.workspace + ws.found))[row * a.segments + blockIdx.x] = (int)s_count;
    }
}

template <int T>
__global__ __launch_bounds__(SM_SPLIT_THREADS) void sample_draw_kernel(sample_args a)
{
    typedef typename dn_elt<T>::store S;
    __shared__ sample_lds s;
    __shared__ u64 candidates[SM_CANDIDATES];
    __shared__ u64 s_kept[SM_BLOCKS];
    __shared__ int s_from[SM_SEGMENTS + 1], s_listed;
    __shared__ u64 s_before;
    __shared__ int s_block;
    const sample_space ws = space_of(a.rows, a.segments);
    const bool vectors = rows_aligned<T>(a);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, blocks = (a.n + a.block - 1) / a.block;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const sample_row r = settings_of(a, row);
        const float largest = row_largest(a, ws, row);
        if (!(largest > -INFINITY)) {
            if (tid == 0) answer(a, row, -1, 0, 0);
            continue;
        }
        const S *x = (const S *)a.logits + row * a.stride;
        const sample_border b = ((const sample_border *)(a.workspace + ws.border))[row];
        __syncthreads();
        for (int i = tid; i < SM_BLOCKS; i += SM_SPLIT_THREADS)
            s_kept[i] = i < blocks ? ((const u64 *)(a.workspace + ws.kept))[row * SM_BLOCKS + i] : 0;
        if (wave == 0) {
            const int c = lane < a.segments ? ((const int *)(a.workspace + ws.found))[row * a.segments + lane] : 0;
            const int upto = (int)wave_scan((unsigned)c);
            if (lane < a.segments) s_from[lane + 1] = upto;
            if (lane == 0) s_from[0] = 0;
            const bool whole = __all(c <= SM_LISTED);
            if (lane == 63) s_listed = whole && upto <= SM_CANDIDATES;
        }
        __syncthreads();
        const int count = s_from[a.segments];
        u64 last = 0;
        if (count) {
            const bool fits = s_listed;
            if (fits) {
                for (int g = wave; g < a.segments; g += SM_SPLIT_THREADS / 64) {
                    const u64 *list = (const u64 *)(a.workspace + ws.list) + ((size_t)row * a.segments + g) * SM_LISTED;
                    for (int j = lane; j < s_from[g + 1] - s_from[g]; j += 64) candidates[s_from[g] + j] = list[j];
                }
                __syncthreads();
            }
            auto each = [&](auto f) {
                if (fits) {
                    for (int i = tid; i < count; i += SM_SPLIT_THREADS) f(candidates[i]);
                    return;
                }
                for (int i = tid * 8; i < a.n; i += SM_STRIP) { /* too many for the lists: from the row again */
                    float l[8];
                    load8<T>(x, i, a.n, vectors, l);
                    for (int e = 0; e < 8; ++e)
                        if (l[e] > -INFINITY && is_candidate(b, bin_of(l[e], largest, r))) f(place_of(l[e], i + e));
                }
            };
            last = last_place(each, b, r, largest, s);
            each([&](u64 c) {
                if (c < last) return;
                const double w = weight_of(logit_of(c), largest, r);
                if (w >= r.floor) atomicAdd(&s_kept[(int)(0xffffffffu - (unsigned)c) / a.block], mass_of(w));
            });
        }
        __syncthreads();
        u64 own = 0, run;
        constexpr int E = SM_BLOCKS / SM_SPLIT_THREADS;
#pragma unroll
        for (int e = 0; e < E; ++e) own += s_kept[tid * E + e];
        const u64 total = block_sum(own, s);
        const double target = draw_target(r, total);
        if (reaches(own, 0, target, run, s)) {
            int at = tid * E;
            while ((double)(run + s_kept[at]) < target) run += s_kept[at++];
            s_block = at;
            s_before = run;
        }
        __syncthreads();
        /* the block, a strip at a time, eight tokens a lane */
        run = s_before;
        const int lo = s_block * a.block, hi = min(a.n, lo + a.block);
        for (int from = lo; from < hi; from += SM_STRIP) {
            const int i = from + tid * 8;
            float l[8];
            u64 m[8], before;
            load8<T>(x, i, hi, vectors, l);
            own = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const u64 c = place_of(l[e], i + e);
                m[e] = 0;
                if (c && c >= last) {
                    const double w = weight_of(l[e], largest, r);
                    if (w >= r.floor) m[e] = mass_of(w);
                }
                own += m[e];
            }
            if (reaches(own, run, target, before, s)) {
                bool done = false;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    before += m[e];
                    if (!done && m[e] && (double)before >= target) {
                        answer(a, row, i + e, m[e], total);
                        done = true;
                    }
                }
            }
            if (from + SM_STRIP < hi) {
                run += block_sum(own, s);
                if ((double)run >= target) break;
            }
        }
    }
}

/* Rows of up to 8192 tokens take one workgroup each.  Longer ones are cut so that about 1024 workgroups have a
 * share of one block of tokens at least. */
static bool sample_in_one(int n) { return n <= 8192; }

static void sample_cut(sample_args &a)
{
    a.block = (int)(((long)a.n + (long)SM_STRIP * SM_BLOCKS - 1) / ((long)SM_STRIP * SM_BLOCKS)) * SM_STRIP;
    const int blocks = (a.n + a.block - 1) / a.block;
    int segments = 1;
    while (segments < SM_SEGMENTS && (long)a.rows * segments < 1024 && segments * 2 <= blocks) segments *= 2;
    a.segments = segments;
    a.length = (blocks + segments - 1) / segments * a.block;
}

extern "C" size_t sample_workspace_bytes(int rows, int n)
{
    if (rows < 1 || n < 1 || n > (1 << 24) || sample_in_one(n)) return 0;
    sample_args a = {};
    a.rows = rows;
    a.n = n;
    sample_cut(a);
    return space_of(rows, a.segments).bytes;
}

template <int T>
static void sample_launch(const sample_args &a)
{
    if (sample_in_one(a.n)) {
        const dim3 grid(a.rows < 65536 ? a.rows : 65536);
        if (a.n <= 2048) hipLaunchKernelGGL((sample_row_kernel<T, 8, 256>), grid, dim3(256), 0, dn_stream(), a);
        else hipLaunchKernelGGL((sample_row_kernel<T, 16, 512>), grid, dim3(512), 0, dn_stream(), a);
        return;
    }
    const dim3 grid(a.segments, a.rows < 65535 ? a.rows : 65535), block(SM_SPLIT_THREADS);
    hipLaunchKernelGGL((sample_largest_kernel<T>), grid, block, 0, dn_stream(), a);
    if (a.top_k || a.top_p || a.temperature) hipLaunchKernelGGL((sample_bins_kernel<T>), grid, block, 0, dn_stream(), a);
    hipLaunchKernelGGL((sample_kept_kernel<T>), grid, block, 0, dn_stream(), a);
    hipLaunchKernelGGL((sample_draw_kernel<T>), dim3(a.rows < 65535 ? a.rows : 65535), block, 0, dn_stream(), a);
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
        !dn_aligned(probs, 4) || !dn_aligned(workspace, 16))
        return dn_refuse(me, "a buffer is not aligned to its element type, or the workspace not to 16 bytes");
    if (rows == 0) return 0;
    if (!workspace && !sample_in_one(n)) return dn_refuse(me, "the workspace is missing");
    hip_require_device(me);
    sample_args a = {logits, temperature, top_p, min_p, uniform, top_k, tokens, probs, (unsigned char *)workspace,
                     stride, rows, n, 1, n, n};
    if (!sample_in_one(n)) sample_cut(a);
    if (type == DN_F32) sample_launch<DN_F32>(a);
    else if (type == DN_F16) sample_launch<DN_F16>(a);
    else sample_launch<DN_BF16>(a);
    dn_check_launch(me);
    return 0;
}
