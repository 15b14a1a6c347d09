/*
 * sample.hip - one token for each row of logits from a random number: temperature, top-k, top-p, min-p.
 *
 * The tokens of a row are ordered by (logit descending, index ascending).  w = exp((logit - largest) / T).
 *   top-k   the first k
 *   top-p   the shortest run of first tokens whose mass is at least p times the mass of what top-k left
 *   min-p   of these the tokens with w >= min_p (the largest has w = 1)
 * The answer is the first token in index order at which the running mass reaches u times the mass kept.
 *
 * Masses are whole numbers, rint(w * 2^b) with w in 64 bits: their sums do not depend on the order in which
 * lanes and atomics add them, so the same row gives the same token in every run.  b is as large as the sum of a row
 * whose tokens are all alike allows, 63 less the bits of an index: 46 for 131072 tokens, 39 for 2^24; and 48 at most, as
 * the last bin has to weigh nothing.  Each mass is off by 2^-(b + 1) of the largest token's at most, in the same direction
 * where logits are the same: a border between two tokens lies where the formula puts it to within n * 2^-(b + 1) of the
 * largest mass, 2^-30 for 131072 tokens, and 2^-16 for 2^24.
 *
 * No row is sorted.  The logits are counted and weighed in 512 bins below the largest, a fifteenth of T wide (what is
 * further below weighs nothing) or, where the row's logits lie closer together, as much narrower.  The bin in which the
 * order's prefix ends is known from the running sums, everything in the bins before it is kept, and only that
 * bin's tokens (the candidates) are looked at more closely: digit by digit of their places.
 */
#include <math.h>

#include "row_types.h"

typedef unsigned long long u64;

typedef float float2_t __attribute__((ext_vector_type(2)));

#define SM_BINS 512
#define SM_PER_T 15
#define SM_SHIFT 48 /* of a mass, at most: what lies 511 / SM_PER_T times T below the largest has a weight below 2^-49 */
#define SM_CANDIDATES 2048 /* that are kept in LDS */
#define SM_LISTED 8192     /* of a long row that are kept in memory */
#define SM_FOUND 512       /* of a segment that are handed on */
#define SM_SEGMENTS 32

struct sample_args {
    const void *logits;
    const float *temperature, *top_p, *min_p, *uniform;
    const int *top_k;
    int *tokens;
    float *probs;
    unsigned char *workspace;
    long stride;
    int rows, n;
    int index_bits; /* that hold n - 1 */
    double unit;    /* the mass of the largest token */
    int segments, length, block; /* length: tokens of a segment, block: of what its mass is summed over */
};

/* A row's settings, those that are off in one form. */
struct sample_row {
    double log2_per_logit; /* log2(e) / T */
    double floor;          /* min-p */
    double uniform;        /* in 0 .. 1 */
    double unit;           /* the mass of the largest token */
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
    s.unit = a.unit;
    s.bins_per_logit = fminf(SM_PER_T / t, 3.402823466e38f);
    return s;
}

/* A token's place in the order as one number, larger is earlier: the logit's bits in their order, without those that
 * are the same in every value of the type (the fewer bits, the fewer rounds find one), and the index from the end.
 * 0 for a token that cannot be drawn (NaN, -inf). */
template <int T>
struct sample_places {
    static constexpr int SAME = T == DN_F32 ? 0 : T == DN_BF16 ? 16 : 13;
    int bits; /* of an index */
    __device__ u64 of(float l, int i) const
    {
        if (!(l > -INFINITY)) return 0;
        const unsigned b = __float_as_uint(l + 0.f); /* -0 ranks as 0 */
        const unsigned key = b & 0x80000000u ? ~b : b | 0x80000000u;
        return ((u64)(key >> SAME) << bits) + ((1u << bits) - 1 - (unsigned)i);
    }
    __device__ float logit(u64 place) const
    {
        const unsigned key = ((unsigned)(place >> bits) << SAME) | ((1u << SAME) - 1);
        return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu & ~((1u << SAME) - 1) : ~key);
    }
    __device__ int index(u64 place) const { return (int)((1u << bits) - 1 - ((unsigned)place & ((1u << bits) - 1))); }
};

/* 2^x for x <= 0 around the nearest whole exponent: 1 + f * q(f), q the polynomial that meets (2^f - 1) / f in the ten
 * Chebyshev points of -1/2 .. 1/2; to 2^-50. */
__device__ __forceinline__ double weight_of(float l, float largest, const sample_row &s)
{
    if (l == largest) return 1; /* also where both are infinite */
    const double x = ((double)l - (double)largest) * s.log2_per_logit;
    if (!(x > -64)) return 0;
    const double whole = rint(x), f = x - whole;
    double p = 7.070977866508138e-09;
    p = fma(p, f, 1.0205905413765595e-07);
    p = fma(p, f, 1.3215451633221434e-06);
    p = fma(p, f, 1.5252672924850737e-05);
    p = fma(p, f, 0.00015403530424776529);
    p = fma(p, f, 0.0013333558200794592);
    p = fma(p, f, 0.009618129107618665);
    p = fma(p, f, 0.05550410866465167);
    p = fma(p, f, 0.24022650695910075);
    p = fma(p, f, 0.6931471805599462);
    p = fma(p, f, 1.);
    return ldexp(p, (int)whole);
}

/* rint(w * 2^b): added to 2^52 the number stands in the low bits of the sum. */
__device__ __forceinline__ u64 mass_of(double w, const sample_row &s)
{
    return (u64)__double_as_longlong(fma(w, s.unit, 0x1p52)) & 0xfffffffffffffull;
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

#define SM_DIGIT_SLOTS (256 + 64)
struct sample_lds {
    u64 mass[SM_BINS + 64];
    unsigned count[SM_BINS + 64];
    u64 digit[2][SM_DIGIT_SLOTS], part[16];
    unsigned digit_count[2][256];
    u64 digit_place[256], prefix, base, found;
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

/* A share of a mass as the whole number that a running sum has to reach: at least 1, at most the mass. */
__device__ __forceinline__ u64 share_of(double share, u64 mass)
{
    const u64 t = (u64)ceil(fmax(share * (double)mass, 1.));
    return t < mass || !mass ? t : mass;
}

/* N bins (in order, or from the last one down) over the lanes of a wave, and where running sums over them reach a
 * target. */
template <int N, bool DOWN, class V>
struct sample_sums {
    static constexpr int E = N / 64;
    V v[E];
    u64 own, upto; /* a lane's sum, and the running sum through it */
    int lane;

    __device__ void read(const V *bins, int lane_)
    {
        lane = lane_;
        own = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int b = lane * E + e;
            v[e] = bins[slot_of<E>(DOWN ? N - 1 - b : b)];
            own += v[e];
        }
        upto = wave_scan(own);
    }
    __device__ u64 total() const { return dn_lane(upto, 63); }
    /* the first bin at which base + running sum reaches the target (at least 1), and the sum before it; N: none */
    __device__ int find(u64 base, u64 target, u64 &before) const
    {
        const u64 any = __ballot(base + upto >= target);
        before = 0;
        if (!any) return N;
        const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)any) - 1);
        u64 run = base + upto - own;
        int at = lane * E;
        bool done = false;
#pragma unroll
        for (int e = 0; e < E; ++e) { /* of use in lane src only */
            done = done || run + v[e] >= target;
            run += done ? 0 : v[e];
            at += done ? 0 : 1;
        }
        before = dn_lane(run, src);
        at = (int)dn_lane((unsigned)at, src);
        return DOWN ? N - 1 - at : at;
    }
    /* the sum before bin b, and with it */
    __device__ u64 sum_to(int b, u64 &with) const
    {
        u64 run = upto - own, next = run;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            run += e < b % E ? v[e] : 0;
            next += e <= b % E ? v[e] : 0;
        }
        with = dn_lane(next, b / E);
        return dn_lane(run, b / E);
    }
};

/* The workgroup: the borders from the bins in LDS, into LDS.  The first wave counts, the second weighs. */
__device__ __forceinline__ void find_border(sample_lds &s, const sample_row &r)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    sample_sums<SM_BINS, false, u64> sums;
    __syncthreads();
    if (wave == 0) {
        int bin = -1, need = 0;
        if (r.k) {
            sample_sums<SM_BINS, false, unsigned> counts;
            counts.read(s.count, lane);
            u64 before;
            bin = counts.find(0, (u64)r.k, before);
            need = r.k - (int)before;
            /* all that weighs anything is among the first k: what is in the last bin lies 34 T or more below the largest
             * (but for a T next to which the difference of two logits is infinite) */
            if (bin == SM_BINS || (bin == SM_BINS - 1 && r.bins_per_logit > 1e-30f)) bin = -1;
        }
        if (lane == 0) {
            s.border.k_bin = bin;
            s.border.k_need = need;
        }
    } else if (wave == 1) {
        sums.read(s.mass, lane);
    }
    __syncthreads();
    if (wave == 1) {
        const int k_bin = __builtin_amdgcn_readfirstlane(s.border.k_bin);
        u64 least, most, mass_lo = 0, ignore;
        if (k_bin < 0) least = most = sums.total();
        else least = sums.sum_to(k_bin, most);
        int lo = SM_BINS, hi = SM_BINS - 1;
        if (r.p < 1) {
            lo = hi = sums.find(0, share_of(r.p, least), mass_lo);
            if (most > least) hi = sums.find(0, share_of(r.p, most), ignore);
        }
        if (lane == 0) {
            s.border.first = r.p < 1 ? lo : k_bin >= 0 ? k_bin : SM_BINS;
            s.border.lo = lo;
            s.border.hi = hi;
            s.border.mass_lo = mass_lo;
            s.border.mass_k = least;
        }
    }
    __syncthreads();
}

__device__ __forceinline__ bool is_candidate(const sample_border &b, int bin)
{
    return (bin >= b.lo && bin <= b.hi) || bin == b.k_bin;
}

template <int THREADS>
__device__ __forceinline__ u64 block_sum(u64 v, sample_lds &s)
{
    v = dn_wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) t += s.part[w];
    return t;
}

template <int THREADS>
__device__ __forceinline__ float2_t block_ends(float2_t v, sample_lds &s)
{
    v = (float2_t){dn_wave_max(v.x), -dn_wave_max(-v.y)};
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = __builtin_bit_cast(u64, v);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        const float2_t o = __builtin_bit_cast(float2_t, s.part[w]);
        v = (float2_t){fmaxf(v.x, o.x), fminf(v.y, o.y)};
    }
    return v;
}

/* A row's largest and least logit (of those above -inf), of four more. */
__device__ __forceinline__ void widen(float2_t &ends, const float l[4])
{
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        ends.x = l[e] > ends.x ? l[e] : ends.x;
        ends.y = l[e] < ends.y && l[e] > -INFINITY ? l[e] : ends.y;
    }
}

/* Where all logits lie closer to the largest than the bins reach, the bins are made as much narrower: the fewer
 * tokens share the one that has to be looked at. */
__device__ __forceinline__ void narrow_bins(sample_row &r, float2_t ends)
{
    r.bins_per_logit = fminf(fmaxf(r.bins_per_logit, (SM_BINS - 2) / (ends.x - ends.y)), 3.402823466e38f);
}

/* mass_of the weight, and in the top bit whether min-p keeps it. */
#define SM_KEPT (1ull << 63)
__device__ __forceinline__ u64 weigh(float l, float largest, const sample_row &r)
{
    const double w = weight_of(l, largest, r);
    return mass_of(w, r) | (w >= r.floor ? SM_KEPT : 0);
}

/* The candidates of a row: places and what weigh() says of them in LDS; where they are too many, a list of places
 * in memory; where they are too many for that (values that most tokens share), the row itself, a strip of 8 tokens a
 * lane at a time.  Loops over them are kept rolled, here and below: these kernels run their code about once, so
 * that its size is time. */
struct sample_candidates {
    u64 place[SM_CANDIDATES], weight[SM_CANDIDATES];
};

template <int T, int THREADS, class Strip, class F>
__device__ __forceinline__ void each_candidate(const sample_candidates &c, const u64 *list, int count, int n, Strip strip,
                                               const sample_places<T> &places, const sample_border &b,
                                               const sample_row &r, float largest, F f)
{
    const bool in_lds = count <= SM_CANDIDATES, in_row = !in_lds && !list;
    const int end = in_row ? n : count, step = in_row ? 8 : 1;
#pragma unroll 1
    for (int i = threadIdx.x * step; i < end; i += THREADS * step) {
        const float *l = in_row ? strip(i) : 0;
#pragma unroll 1
        for (int e = 0; e < step; ++e) {
            u64 place;
            if (in_row) {
                if (!(l[e] > -INFINITY) || !is_candidate(b, bin_of(l[e], largest, r))) continue;
                place = places.of(l[e], i + e);
            } else {
                place = in_lds ? c.place[i] : list[i];
            }
            f(place, in_lds ? c.weight[i] : weigh(places.logit(place), largest, r));
        }
    }
}

/* The last place of the kept prefix, from the candidates: top-k among those of its bin, then top-p among those that it
 * left.  Each is found by eight bits a round, from the first bit in which two logits of these bins can differ. */
template <int T, int THREADS, class Each>
__device__ __forceinline__ u64 last_place(Each each, const sample_places<T> &places, const sample_border &b,
                                          const sample_row &r, float largest, sample_lds &s)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    u64 last = 0, mass_k = b.mass_k;
#pragma unroll 1
    for (int stage = 0; stage < 2; ++stage) {
        const bool by_mass = stage == 1;
        if (by_mass ? !(r.p < 1) : b.k_bin < 0) continue;
        const int from = by_mass ? b.lo : b.k_bin, to = by_mass ? b.hi : b.k_bin;
        auto bin = [&](u64 c) { return bin_of(places.logit(c), largest, r); };
        __syncthreads(); /* the last use of s is over */
        for (int i = tid; i < SM_DIGIT_SLOTS; i += THREADS) s.digit[0][i] = 0;
        for (int i = tid; i < 256; i += THREADS) s.digit_count[0][i] = 0;
        if (by_mass && b.k_bin >= 0) {
            u64 in_k = 0;
            each([&](u64 c, u64 w) { in_k += c >= last && bin(c) == b.k_bin ? w & ~SM_KEPT : 0; });
            mass_k += block_sum<THREADS>(in_k, s);
        }
        __syncthreads();
        const u64 target = by_mass ? share_of(r.p, mass_k) : (u64)b.k_need;
        u64 base = by_mass ? b.mass_lo : 0;
        /* logits of bins from .. to, a hundredth of a bin more on either side than the rounding of bin_of needs */
        const float up = largest - (from - 0.01f) / r.bins_per_logit;
        const float upper = up >= -3.402823466e38f && up < largest ? up : largest; /* (bins may be infinitely wide) */
        const float lower = to < SM_BINS - 1 ? largest - (to + 1.01f) / r.bins_per_logit : -INFINITY;
        const u64 most = places.of(upper, 0), least = places.of(lower, (1 << places.bits) - 1);
        int bit = most > least ? 64 - __clzll((long long)(most ^ least)) : 0, turn = 0;
        u64 prefix = most >> bit; /* places have 56 bits at most */
        while (bit > 0) {
            const int next = bit > 8 ? bit - 8 : 0;
            each([&](u64 c, u64 w) {
                const int in = bin(c);
                if (in < from || in > to || c < last || c >> bit != prefix) return;
                const int d = (int)(c >> next) & ((1 << (bit - next)) - 1);
                atomicAdd(&s.digit[turn][digit_slot(d)], by_mass ? w & ~SM_KEPT : 1ull);
                if (atomicAdd(&s.digit_count[turn][d], 1u) == 0) s.digit_place[d] = c;
            });
            __syncthreads();
            if (wave == 0) {
                u64 before;
                sample_sums<256, true, u64> sums;
                sums.read(s.digit[turn], lane);
                const int d = sums.find(base, target, before) & 255;
                if (lane == 0) {
                    s.prefix = prefix << (bit - next) | (u64)d;
                    s.base = before;
                    s.found = s.digit_count[turn][d] == 1 ? s.digit_place[d] : 0;
                }
            } else { /* what the next round counts in */
                for (int i = tid - 64; i < SM_DIGIT_SLOTS; i += THREADS - 64) s.digit[turn ^ 1][i] = 0;
                for (int i = tid - 64; i < 256; i += THREADS - 64) s.digit_count[turn ^ 1][i] = 0;
            }
            __syncthreads();
            prefix = s.prefix;
            base = s.base;
            bit = next;
            turn ^= 1;
            if (s.found) { /* the only one with this digit */
                prefix = s.found;
                break;
            }
        }
        last = prefix > last ? prefix : last;
    }
    return last;
}

/* Each lane has `own`, the mass of its piece of consecutive tokens; pieces follow each other in lane order.  Finds the
 * piece in which base + running mass reaches the target: true for its lane, with the sum before it. */
template <int THREADS>
__device__ __forceinline__ bool reaches(u64 own, u64 base, u64 target, u64 &before, sample_lds &s)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 incl = wave_scan(own);
    __syncthreads();
    if (lane == 63) s.part[wave] = incl;
    __syncthreads();
    u64 run = base + incl - own;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) run += w < wave ? s.part[w] : 0;
    before = run;
    return run < target && run + own >= target;
}

__device__ __forceinline__ void answer(const sample_args &a, long row, int token, u64 mass, u64 total)
{
    a.tokens[row] = token;
    if (a.probs) a.probs[row] = total ? (float)((double)mass / (double)total) : 0.f;
}

/* Four (eight) neighbouring tokens from i on, in one access whatever their alignment; -inf behind `end`. */
template <int T>
__device__ __forceinline__ void load4(const typename dn_elt<T>::store *x, int i, int end, float *l)
{
    typedef typename dn_elt<T>::store S;
    typedef S S4 __attribute__((ext_vector_type(4)));
    typedef S4 S4U __attribute__((aligned(sizeof(S))));
    if (i + 4 <= end) {
        const S4 u = *(const S4U *)(x + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) l[e] = (float)u[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) l[e] = i + e < end ? (float)x[i + e] : -INFINITY;
    }
}

template <int T>
__device__ __forceinline__ void load8(const typename dn_elt<T>::store *x, int i, int end, float l[8])
{
    typedef typename dn_elt<T>::store S;
    typedef S S8 __attribute__((ext_vector_type(8)));
    typedef S8 S8U __attribute__((aligned(sizeof(S))));
    if (i + 8 <= end) {
        const S8 u = *(const S8U *)(x + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) l[e] = (float)u[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) l[e] = i + e < end ? (float)x[i + e] : -INFINITY;
    }
}

/* ---- a row of up to 8192 tokens: one workgroup, the row in LDS, one launch --------------------------------
 * Bound by the latency of its steps (largest, bins, border, candidates, kept mass, token), each behind a barrier: 1000
 * tokens 10 us, 8000 16 us, 256 rows of 8000 19 us. */
template <int T, int E, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_row_kernel(sample_args a)
{
    typedef typename dn_elt<T>::store S;
    __shared__ sample_lds s;
    __shared__ sample_candidates c;
    __shared__ float row_lds[THREADS * (E + 1)]; /* E neighbours a lane; the gap spreads them over the banks */
    __shared__ unsigned s_count;
    const int tid = threadIdx.x;
    const sample_places<T> places = {a.index_bits};
    float *own_l = row_lds + tid * (E + 1);
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const S *x = (const S *)a.logits + row * a.stride;
        sample_row r = settings_of(a, row);
        float2_t ends = {-INFINITY, INFINITY};
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            float l[4];
            load4<T>(x, tid * E + e, a.n, l);
            widen(ends, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) own_l[e + i] = l[i];
        }
        if (r.k || r.p < 1)
            for (int i = tid; i < SM_SLOTS; i += THREADS) {
                s.count[i] = 0;
                s.mass[i] = 0;
            }
        if (tid == 0) s_count = 0;
        ends = block_ends<THREADS>(ends, s);
        narrow_bins(r, ends);
        const float largest = ends.x;
        if (!(largest > -INFINITY)) {
            if (tid == 0) answer(a, row, -1, 0, 0);
            continue;
        }
        u64 last = 0;
        if (r.k || r.p < 1) {
#pragma unroll 4
            for (int e = 0; e < E; ++e) {
                const float l = own_l[e];
                if (!(l > -INFINITY)) continue;
                const int b = bin_slot(bin_of(l, largest, r));
                if (r.k) atomicAdd(&s.count[b], 1u);
                if (r.p < 1) atomicAdd(&s.mass[b], mass_of(weight_of(l, largest, r), r));
            }
            find_border(s, r);
            const sample_border b = s.border;
            if (b.k_bin >= 0 || r.p < 1) {
#pragma unroll 1
                for (int e = 0; e < E; ++e) {
                    const float l = own_l[e];
                    if (!(l > -INFINITY) || !is_candidate(b, bin_of(l, largest, r))) continue;
                    const unsigned at = atomicAdd(&s_count, 1u);
                    if (at >= SM_CANDIDATES) continue;
                    c.place[at] = places.of(l, tid * E + e);
                    c.weight[at] = weigh(l, largest, r);
                }
                __syncthreads();
                const int count = (int)s_count;
                auto strip = [&](int i) { return row_lds + i + i / E; }; /* (E = 4: a row has no more tokens than the list holds) */
                last = last_place<T, THREADS>([&](auto f) { each_candidate<T, THREADS>(c, 0, count, a.n, strip, places, b, r, largest, f); },
                                     places, b, r, largest, s);
            }
        }
        auto kept_mass = [&](int e) {
            const u64 place = places.of(own_l[e], tid * E + e);
            if (!place || place < last) return (u64)0;
            const u64 w = weigh(own_l[e], largest, r);
            return w & SM_KEPT ? w & ~SM_KEPT : 0;
        };
        u64 own = 0, run;
#pragma unroll 1
        for (int e = 0; e < E; ++e) own += kept_mass(e);
        const u64 total = block_sum<THREADS>(own, s), target = share_of(r.uniform, total);
        if (reaches<THREADS>(own, 0, target, run, s)) {
#pragma unroll 1
            for (int e = 0; e < E; ++e) {
                const u64 m = kept_mass(e);
                run += m;
                if (run >= target) {
                    answer(a, row, tid * E + e, m, total);
                    break;
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
 * 4 one workgroup a row: the prefix' end among the candidates, the block that the draw falls into, the token
 *
 * Measured: one row of 32768 fp32, top-k and top-p, 22 us (2, 4, 6 and 8 in the four); 64 rows of 131072 with settings of
 * all kinds 51 us (7, 15, 17, 10).  A pass over the logits is 6 us at the memory's
 * rate; the second and third are bound by their instructions: a weight is 23 of 64 bits, the additions to 64-bit bins
 * wait for each other, and a token of a bin that is kept is weighed twice rather than 8 bytes stored for each.  The
 * fourth is a chain of latencies. */
#define SM_SPLIT_THREADS 256
#define SM_STRIP (SM_SPLIT_THREADS * 8) /* tokens that a workgroup takes at a time */
#define SM_DRAW_THREADS 512
#define SM_BLOCKS 512                   /* of a row, at most: they are summed in LDS */

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
    w.bins_count = w.list + (size_t)rows * SM_LISTED * 8;
    w.largest = w.bins_count + (size_t)rows * SM_BINS * 4;
    w.found = w.largest + all * 8;
    w.bytes = w.found + (size_t)rows * 8;
    return w;
}

template <int T>
__global__ __launch_bounds__(SM_SPLIT_THREADS) void sample_largest_kernel(sample_args a)
{
    typedef typename dn_elt<T>::store S;
    __shared__ float2_t part[SM_SPLIT_THREADS / 64];
    const sample_space ws = space_of(a.rows, a.segments);
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const S *x = (const S *)a.logits + row * a.stride;
        const int lo = blockIdx.x * a.length, hi = min(a.n, lo + a.length);
        float2_t ends = {-INFINITY, INFINITY};
        for (int i = lo + threadIdx.x * 8; i < hi; i += SM_STRIP) {
            float l[8];
            load8<T>(x, i, hi, l);
            widen(ends, l);
            widen(ends, l + 4);
        }
        ends = (float2_t){dn_wave_max(ends.x), -dn_wave_max(-ends.y)};
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ends;
        __syncthreads();
        if (threadIdx.x == 0) {
            float2_t t = part[0];
            for (int w = 1; w < SM_SPLIT_THREADS / 64; ++w) t = (float2_t){fmaxf(t.x, part[w].x), fminf(t.y, part[w].y)};
            ((float2_t *)(a.workspace + ws.largest))[row * a.segments + blockIdx.x] = t;
        }
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i < SM_BINS; i += SM_SPLIT_THREADS) {
                ((u64 *)(a.workspace + ws.bins_mass))[row * SM_BINS + i] = 0;
                ((unsigned *)(a.workspace + ws.bins_count))[row * SM_BINS + i] = 0;
                if (i < 2) ((unsigned *)(a.workspace + ws.found))[row * 2 + i] = 0;
            }
    }
}

/* The row's largest logit, and the bins' width. */
__device__ __forceinline__ float row_largest(const sample_args &a, const sample_space &ws, long row, sample_row &r)
{
    const int lane = threadIdx.x & 63;
    const float2_t *m = (const float2_t *)(a.workspace + ws.largest) + row * a.segments;
    const float2_t own = lane < a.segments ? m[lane] : (float2_t){-INFINITY, INFINITY};
    const float2_t ends = {dn_wave_max(own.x), -dn_wave_max(-own.y)};
    narrow_bins(r, ends);
    return ends.x;
}

template <int T>
__global__ __launch_bounds__(SM_SPLIT_THREADS) void sample_bins_kernel(sample_args a)
{
    typedef typename dn_elt<T>::store S;
    __shared__ u64 mass[SM_BINS];
    __shared__ unsigned count[SM_BINS];
    const sample_space ws = space_of(a.rows, a.segments);
    const int tid = threadIdx.x;
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        sample_row r = settings_of(a, row);
        if (!r.k && !(r.p < 1)) continue;
        const float largest = row_largest(a, ws, row, r);
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
            load8<T>(x, i, hi, l);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (!(l[e] > -INFINITY)) continue;
                const int b = bin_of(l[e], largest, r);
                if (r.k) atomicAdd(&count[b], 1u);
                if (r.p < 1) atomicAdd(&mass[b], mass_of(weight_of(l[e], largest, r), r));
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
    __shared__ u64 s_list[SM_FOUND];
    __shared__ unsigned s_count, s_from;
    const sample_space ws = space_of(a.rows, a.segments);
    const sample_places<T> places = {a.index_bits};
    const int tid = threadIdx.x;
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        sample_row r = settings_of(a, row);
        const float largest = row_largest(a, ws, row, r);
        __syncthreads();
        if (r.k || r.p < 1)
            for (int i = tid; i < SM_BINS; i += SM_SPLIT_THREADS) {
                s.mass[bin_slot(i)] = ((const u64 *)(a.workspace + ws.bins_mass))[row * SM_BINS + i];
                s.count[bin_slot(i)] = ((const unsigned *)(a.workspace + ws.bins_count))[row * SM_BINS + i];
            }
        if (tid == 0) s_count = 0;
        find_border(s, r);
        if (tid == 0 && blockIdx.x == 0) ((sample_border *)(a.workspace + ws.border))[row] = s.border;
        const sample_border b = s.border;
        const S *x = (const S *)a.logits + row * a.stride;
        const int lo = blockIdx.x * a.length, hi = min(a.n, lo + a.length);
        for (int from = lo; from < hi; from += a.block) {
            u64 own = 0;
            const int to = min(hi, from + a.block);
            for (int i = from + tid * 8; i < to; i += SM_STRIP) {
                float l[8];
                load8<T>(x, i, to, l);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (!(l[e] > -INFINITY)) continue;
                    const int bin = bin_of(l[e], largest, r);
                    if (bin < b.first) {
                        const double w = weight_of(l[e], largest, r);
                        if (w >= r.floor) own += mass_of(w, r);
                    } else if (is_candidate(b, bin)) {
                        const unsigned at = atomicAdd(&s_count, 1u);
                        if (at < SM_FOUND) s_list[at] = places.of(l[e], i + e);
                    }
                }
            }
            const u64 kept = block_sum<SM_SPLIT_THREADS>(own, s);
            if (tid == 0) ((u64 *)(a.workspace + ws.kept))[row * SM_BLOCKS + from / a.block] = kept;
        }
        /* the segment's candidates behind those of the segments that came first; their order does not matter.  More than
         * can be handed on: the second number */
        __syncthreads();
        const unsigned count = s_count;
        unsigned *found = (unsigned *)(a.workspace + ws.found) + row * 2;
        if (tid == 0 && count) {
            if (count > SM_FOUND) atomicAdd(found + 1, 1u);
            s_from = atomicAdd(found, count);
        }
        __syncthreads();
        u64 *list = (u64 *)(a.workspace + ws.list) + (size_t)row * SM_LISTED;
        for (unsigned i = tid; i < count && i < SM_FOUND; i += SM_SPLIT_THREADS)
            if (s_from + i < SM_LISTED) list[s_from + i] = s_list[i];
    }
}

template <int T>
__global__ __launch_bounds__(SM_DRAW_THREADS) void sample_draw_kernel(sample_args a)
{
    typedef typename dn_elt<T>::store S;
    __shared__ sample_lds s;
    __shared__ sample_candidates c;
    __shared__ u64 s_kept[SM_BLOCKS];
    constexpr int P = 9; /* a lane's tokens and a gap */
    __shared__ float strip[SM_DRAW_THREADS * P];
    __shared__ u64 s_before;
    __shared__ int s_block;
    const sample_space ws = space_of(a.rows, a.segments);
    const sample_places<T> places = {a.index_bits};
    const int tid = threadIdx.x, blocks = (a.n + a.block - 1) / a.block;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        /* all that the first steps read is asked for at once */
        sample_row r = settings_of(a, row);
        const sample_border b = ((const sample_border *)(a.workspace + ws.border))[row];
        const u64 *kept = (const u64 *)(a.workspace + ws.kept) + row * SM_BLOCKS;
        const u64 own_kept = tid < blocks ? kept[tid] : 0;
        const int count = ((const int *)(a.workspace + ws.found))[row * 2], lost = ((const int *)(a.workspace + ws.found))[row * 2 + 1];
        const u64 *in_memory = (const u64 *)(a.workspace + ws.list) + (size_t)row * SM_LISTED;
        const float largest = row_largest(a, ws, row, r);
        const S *x = (const S *)a.logits + row * a.stride;
        if (!(largest > -INFINITY)) {
            if (tid == 0) answer(a, row, -1, 0, 0);
            continue;
        }
        __syncthreads();
        s_kept[tid] = own_kept;
        u64 last = 0;
        if (count) {
            const bool whole = !lost && count <= SM_LISTED;
            const u64 *list = whole ? in_memory : 0;
            const int held = whole ? count : 0x7fffffff;
            if (held <= SM_CANDIDATES)
#pragma unroll 1
                for (int i = tid; i < held; i += SM_DRAW_THREADS) {
                    c.place[i] = list[i];
                    c.weight[i] = weigh(places.logit(list[i]), largest, r);
                }
            __syncthreads();
            auto strip_at = [&](int i) {
                float l[8], *to = strip + tid * P;
                load8<T>(x, i, a.n, l);
#pragma unroll
                for (int e = 0; e < 8; ++e) to[e] = l[e];
                return to;
            };
            auto each = [&](auto f) { each_candidate<T, SM_DRAW_THREADS>(c, list, held, a.n, strip_at, places, b, r, largest, f); };
            last = last_place<T, SM_DRAW_THREADS>(each, places, b, r, largest, s);
            each([&](u64 place, u64 w) {
                if (place >= last && w & SM_KEPT) atomicAdd(&s_kept[places.index(place) / a.block], w & ~SM_KEPT);
            });
        }
        __syncthreads();
        static_assert(SM_BLOCKS == SM_DRAW_THREADS, "a block a lane");
        u64 own = s_kept[tid], run;
        const u64 total = block_sum<SM_DRAW_THREADS>(own, s), target = share_of(r.uniform, total);
        if (reaches<SM_DRAW_THREADS>(own, 0, target, run, s)) {
            s_block = tid;
            s_before = run;
        }
        __syncthreads();
        /* the block, a strip at a time, four tokens a lane */
        run = s_before;
        const int lo = s_block * a.block, hi = min(a.n, lo + a.block);
#pragma unroll 1
        for (int from = lo; from < hi; from += SM_STRIP) {
            const int i = from + tid * 4;
            float l[4];
            load4<T>(x, i, hi, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) strip[tid * P + e] = l[e];
            auto kept_mass = [&](int e) {
                const u64 place = places.of(strip[tid * P + e], i + e);
                if (!place || place < last) return (u64)0;
                const u64 w = weigh(strip[tid * P + e], largest, r);
                return w & SM_KEPT ? w & ~SM_KEPT : 0;
            };
            own = 0;
#pragma unroll 1
            for (int e = 0; e < 4; ++e) own += kept_mass(e);
            u64 before;
            if (reaches<SM_DRAW_THREADS>(own, run, target, before, s)) {
#pragma unroll 1
                for (int e = 0; e < 4; ++e) {
                    const u64 m = kept_mass(e);
                    before += m;
                    if (before >= target) {
                        answer(a, row, i + e, m, total);
                        break;
                    }
                }
            }
            if (from + SM_STRIP < hi) {
                run += block_sum<SM_DRAW_THREADS>(own, s);
                if (run >= target) break;
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
        if (a.n <= 1024) hipLaunchKernelGGL((sample_row_kernel<T, 4, 256>), grid, dim3(256), 0, dn_stream(), a);
        else if (a.n <= 4096) hipLaunchKernelGGL((sample_row_kernel<T, 8, 512>), grid, dim3(512), 0, dn_stream(), a);
        else hipLaunchKernelGGL((sample_row_kernel<T, 8, 1024>), grid, dim3(1024), 0, dn_stream(), a);
        return;
    }
    const dim3 grid(a.segments, a.rows < 65535 ? a.rows : 65535), block(SM_SPLIT_THREADS);
    hipLaunchKernelGGL((sample_largest_kernel<T>), grid, block, 0, dn_stream(), a);
    if (a.top_k || a.top_p || a.temperature) hipLaunchKernelGGL((sample_bins_kernel<T>), grid, block, 0, dn_stream(), a);
    hipLaunchKernelGGL((sample_kept_kernel<T>), grid, block, 0, dn_stream(), a);
    hipLaunchKernelGGL((sample_draw_kernel<T>), dim3(a.rows < 65535 ? a.rows : 65535), dim3(SM_DRAW_THREADS), 0, dn_stream(), a);
}

extern "C" int sample_rows_gpu(const void *logits, int type, int rows, int n, long stride, const float *temperature,
                               const int *top_k, const float *top_p, const float *min_p, const float *uniform,
                               int *tokens, float *probs, void *workspace)
{
    const char *me = "sample_rows_gpu";
    if (!dn_is_float_type(type)) return dn_refuse(me, "unknown element type");
    if (rows < 0 || n < 1 || n > (1 << 24)) return dn_refuse(me, "bad geometry (1 to 2^24 tokens)");
    if (stride < n) return dn_refuse(me, "the stride is shorter than a row");
    if (rows == 0) return 0;
    if (!logits || !uniform || !tokens) return dn_refuse(me, "a buffer is missing");
    if (!dn_aligned(logits, dn_type_bytes(type)) || !dn_aligned(temperature, 4) || !dn_aligned(top_k, 4) ||
        !dn_aligned(top_p, 4) || !dn_aligned(min_p, 4) || !dn_aligned(uniform, 4) || !dn_aligned(tokens, 4) ||
        !dn_aligned(probs, 4) || !dn_aligned(workspace, 16))
        return dn_refuse(me, "a buffer is not aligned to its element type, or the workspace not to 16 bytes");
    if (!workspace && !sample_in_one(n)) return dn_refuse(me, "the workspace is missing");
    hip_require_device(me);
    sample_args a = {logits, temperature, top_p, min_p, uniform, top_k, tokens, probs, (unsigned char *)workspace,
                     stride, rows, n, 1, 0, 1, n, n};
    while (1 << a.index_bits < n) ++a.index_bits;
    a.unit = ldexp(1., 63 - a.index_bits < SM_SHIFT ? 63 - a.index_bits : SM_SHIFT);
    if (!sample_in_one(n)) sample_cut(a);
    if (type == DN_F32) sample_launch<DN_F32>(a);
    else if (type == DN_F16) sample_launch<DN_F16>(a);
    else sample_launch<DN_BF16>(a);
    dn_check_launch(me);
    return 0;
}
