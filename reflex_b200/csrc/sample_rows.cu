// One token a row from 32-bit logits [B, V], every row with its own temperature, top-k, top-p and min-p.
//
// With e_i = exp((l_i - max) / T), the tokens in descending order of l (ties: the lower index first) are kept
// while their place is below k, the sum of the e before them is below p * (the sum of all), and e_i is at
// least min_p; each of the three keeps a prefix of the same order, so the shortest decides.  The token is the
// first in index order at which the running sum of the kept e reaches u * (their sum).  T <= 0 or NaN: the
// largest logit, ties to the highest index.  Infinite logits share everything between them, -inf and NaN are
// never picked, and a row with nothing else gives 0.
//
// A thread-block cluster takes a row: its CTAs hold a piece of it each in shared memory, so the logits are
// read once, and exchange maxima, sums and histograms through distributed shared memory; one launch does
// everything.  The cut is found by narrowing an interval of the logits' ordered bit patterns: 2,048 bins, the
// first of them at which the count or the mass is reached, then that bin's interval, until it is one value.
// Counts are integers and a bin's mass is 64-bit fixed point (rounded), so no result depends on the order in
// which threads add; the sums that the draw walks are 64-bit, in index order.
//
// e itself is taken in 64 bits: a draw that falls near one of 150,000 borders between tokens lands on the
// same side as in exact arithmetic only if the borders are good to about 1e-12 of the sum (with 32-bit
// exponentials one row in ten thousand of a flat distribution differs).
#include <cooperative_groups.h>
#include <float.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

using namespace rfx;

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 2048, PER = BINS / THREADS, MAX_CLUSTER = 8;
constexpr int TABLE = 64;
constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.69314718055994530942;
typedef unsigned long long u64;

// bit patterns in the order of the values; -0 and 0 are one
__device__ __forceinline__ unsigned key_of(float l) {
    const unsigned u = __float_as_uint(l + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// 2^y for y <= 0: y = (64 m + j) / 64 + f, 2^m 2^(j/64) e^(f ln 2), the last by its series to the fourth
// power, |f ln 2| <= ln 2 / 128 (off by 4e-14).  Zero below 2^-1000.
__device__ __forceinline__ double pow2(double y, const double* table) {
    if (!(y > -1000.0)) return 0.0;
    const double t = y * TABLE, r = rint(t), f = (t - r) * (LN2 / TABLE);
    const int n = (int)r;
    const double s = fma(fma(fma(fma(f, 1.0 / 24, 1.0 / 6), f, 0.5), f, 1.0), f, 1.0);
    return s * table[n & (TABLE - 1)] * __hiloint2double(((n >> 6) + 1023) << 20, 0);
}

struct Params {
    const float* logits;
    long long ld;
    int V, chunk;
    const float *temperature, *uniform, *top_p, *min_p;
    const int* top_k;
    int* out;
};

// What the leader decides after a round of narrowing.
struct Cut {
    unsigned lo, hi;     // the interval of patterns that holds the cut
    int above, in;       // entries above the interval, and in it
    u64 mass_above;
    int found, last;     // a rule stops the row here; the interval is one value
};

struct Shared {
    double table[TABLE];
    double warp_d[WARPS + 1];
    double total[MAX_CLUSTER], kept[MAX_CLUSTER];
    float top[MAX_CLUSTER];
    int ties[MAX_CLUSTER], best[MAX_CLUSTER];
    u64 warp_m[WARPS];
    int warp_i[WARPS + 1];
    float warp_f[WARPS];
    Cut cut;
    int stop, who, last;
};

template <typename T>
__device__ __forceinline__ void tell_all(cg::cluster_group& cluster, T* slots, T v) {
    const int C = cluster.num_blocks();
    if ((int)threadIdx.x < C) cluster.map_shared_rank(slots, threadIdx.x)[cluster.block_rank()] = v;
    cluster.sync();
}

// Sum over the block in a fixed order; every thread gets it.
__device__ __forceinline__ double block_total(double v, double* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < WARPS; ++w) t += scratch[w];
    return t;
}

// STAGED: the CTA's piece of the row lies in shared memory; otherwise it is read again by every pass (from L2).
template <bool STAGED>
__global__ void __launch_bounds__(THREADS) sample_rows_kernel(const Params p) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), c = cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int* hist_n = reinterpret_cast<int*>(dynamic);
    unsigned* hist_lo = reinterpret_cast<unsigned*>(hist_n + BINS);
    unsigned* hist_hi = hist_lo + BINS;
    float* piece = reinterpret_cast<float*>(hist_hi + BINS);
    if (tid < TABLE) sh.table[tid] = exp2((double)tid / TABLE);
    pdl_prologue();
    const size_t b = blockIdx.x;
    const int lo = min(p.V, c * p.chunk), n = min(p.V, lo + p.chunk) - lo;
    const float* row = p.logits + b * p.ld + lo;
    auto at = [&](int i) { return STAGED ? piece[i] : row[i]; };

    // ---- the piece, and the row's maximum
    float mx = -INFINITY;
    if (STAGED && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
        const int n4 = n / 4;
#pragma unroll 4
        for (int i = tid; i < n4; i += THREADS) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(row) + i);
            reinterpret_cast<float4*>(piece)[i] = v;
            mx = fmaxf(fmaxf(mx, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
        }
        for (int i = n4 * 4 + tid; i < n; i += THREADS) {
            const float v = row[i];
            piece[i] = v;
            mx = fmaxf(mx, v);
        }
    } else {
#pragma unroll 4
        for (int i = tid; i < n; i += THREADS) {
            const float v = row[i];
            if (STAGED) piece[i] = v;
            mx = fmaxf(mx, v);
        }
    }
    mx = warp_max(mx);
    if (lane == 0) sh.warp_f[warp] = mx;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, sh.warp_f[w]);
    tell_all(cluster, sh.top, mx);
    for (int i = 0; i < C; ++i) mx = fmaxf(mx, sh.top[i]);
    if (mx == -INFINITY) {  // nothing left
        if (c == 0 && tid == 0) p.out[b] = 0;
        return;
    }
    const float T = p.temperature[b];
    if (!(T > 0.0f)) {
        int best = -1;
        for (int i = tid; i < n; i += THREADS)
            if (at(i) == mx) best = lo + i;
        best = __reduce_max_sync(0xffffffffu, best);
        if (lane == 0) sh.warp_i[warp] = best;
        __syncthreads();
        for (int w = 0; w < WARPS; ++w) best = max(best, sh.warp_i[w]);
        tell_all(cluster, sh.best, best);
        if (c == 0 && tid == 0) {
            for (int i = 0; i < C; ++i) best = max(best, sh.best[i]);
            p.out[b] = best;
        }
        return;
    }

    // ---- the rules
    const double per_t = LOG2E / (double)T;
    auto mass = [&](float l) { return l == mx ? 1.0 : pow2(((double)l - (double)mx) * per_t, sh.table); };
    const int k = p.top_k ? p.top_k[b] : 0;
    const bool k_on = k > 0 && k < p.V;
    const float tp = p.top_p ? fmaxf(p.top_p[b], 0.0f) : 1.0f;
    const bool p_on = p.top_p && p.top_p[b] < 1.0f;
    const float mp = p.min_p && p.min_p[b] > 0.0f ? fminf(p.min_p[b], 1.0f) : 0.0f;
    double reach = INFINITY;  // how far below the maximum a kept logit may lie
    if (mp > 0.0f) reach = -(double)T * log((double)mp);
    double total = 0.0;
    if (p_on) {
        for (int i = tid; i < n; i += THREADS) {
            const float l = at(i);
            if (l > -INFINITY) total += mass(l);
        }
        total = block_total(total, sh.warp_d);
        tell_all(cluster, sh.total, total);
        total = 0.0;
        for (int i = 0; i < C; ++i) total += sh.total[i];
        // entries below (1 - p) total / V have less than (1 - p) total between them: what lies above them
        // reaches p total (half of that bound, for the roundings)
        reach = fmin(reach, -(double)T * log((1.0 - (double)tp) * total / p.V * 0.5));
    }
    float least = -FLT_MAX;  // the smallest logit within reach
    if (reach < INFINITY) {
        least = (float)((double)mx - reach);
        if (mx == INFINITY) least = mx;
        for (int i = 0; i < 4 && (double)mx - (double)least > reach; ++i) least = nextafterf(least, INFINITY);
        const float below = nextafterf(least, -INFINITY);
        if (mx < INFINITY && (double)mx - (double)below <= reach) least = below;
        least = fmaxf(fminf(least, mx), -FLT_MAX);
    }

    // ---- the cut
    float cut = least;
    int ties_kept = 0x7fffffff, ties = 0;
    if (k_on || p_on) {
        int bits = 1;
        while (bits < 31 && (1 << bits) < p.V) ++bits;
        const double one = __hiloint2double((62 - bits + 1023) << 20, 0);  // 2^(62 - bits): V masses of 1 fit
        const u64 want = (u64)((double)tp * total * one);
        Cut st = {key_of(least), key_of(mx), 0, 0, 0ull, 1, 0};
        for (int round = 0; round < 4 && st.found && !st.last; ++round) {
            const unsigned range = st.hi - st.lo;
            const int shift = range < BINS ? 0 : 21 - __clz(range);
            for (int i = tid; i < BINS; i += THREADS) hist_n[i] = 0, hist_lo[i] = 0, hist_hi[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += THREADS) {
                const float l = at(i);
                if (l >= least) {
                    const unsigned key = key_of(l);
                    if (key >= st.lo && key <= st.hi) {
                        const unsigned bin = (st.hi - key) >> shift;
                        atomicAdd(&hist_n[bin], 1);
                        if (p_on) {
                            // two 32-bit halves: the addition that wraps the low one carries into the high one
                            const u64 m = (u64)(mass(l) * one + 0.5);
                            const unsigned m_lo = (unsigned)m, m_hi = (unsigned)(m >> 32);
                            const unsigned old = atomicAdd(&hist_lo[bin], m_lo);
                            const unsigned up = m_hi + (old + m_lo < old ? 1u : 0u);
                            if (up) atomicAdd(&hist_hi[bin], up);
                        }
                    }
                }
            }
            cluster.sync();
            if (c == 0) {  // the leader: every CTA's bins together, and the first at which a rule stops the row
                int cn[PER] = {}, tn = 0;
                u64 cm[PER] = {}, tm = 0;
                for (int i = 0; i < C; ++i) {
                    const int4 h = reinterpret_cast<const int4*>(cluster.map_shared_rank(hist_n, i))[tid];
                    cn[0] += h.x, cn[1] += h.y, cn[2] += h.z, cn[3] += h.w;
                    if (p_on) {
                        const uint4 l = reinterpret_cast<const uint4*>(cluster.map_shared_rank(hist_lo, i))[tid];
                        const uint4 u = reinterpret_cast<const uint4*>(cluster.map_shared_rank(hist_hi, i))[tid];
                        cm[0] += ((u64)u.x << 32) + l.x, cm[1] += ((u64)u.y << 32) + l.y;
                        cm[2] += ((u64)u.z << 32) + l.z, cm[3] += ((u64)u.w << 32) + l.w;
                    }
                }
                for (int q = 0; q < PER; ++q) tn += cn[q], tm += cm[q];
                int in = tn;
                u64 im = tm;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int a = __shfl_up_sync(0xffffffffu, in, o);
                    const u64 m = __shfl_up_sync(0xffffffffu, im, o);
                    if (lane >= o) in += a, im += m;
                }
                if (lane == 31) sh.warp_i[warp] = in, sh.warp_m[warp] = im;
                if (tid == 0) sh.stop = BINS;
                __syncthreads();
                int above = st.above + in - tn;
                u64 mass_above = st.mass_above + im - tm;
                for (int w = 0; w < warp; ++w) above += sh.warp_i[w], mass_above += sh.warp_m[w];
                int stop = BINS, q = 0;
                for (; q < PER; ++q) {
                    if (cn[q] && ((k_on && above + cn[q] >= k) || (p_on && mass_above + cm[q] >= want))) {
                        stop = tid * PER + q;
                        break;
                    }
                    above += cn[q];
                    mass_above += cm[q];
                }
                if (stop < BINS) atomicMin(&sh.stop, stop);
                __syncthreads();
                if (sh.stop == stop && stop < BINS) {
                    Cut next;
                    next.hi = st.hi - ((unsigned)stop << shift);
                    next.lo = max(st.lo, next.hi - min(next.hi, (1u << shift) - 1u));
                    next.above = above;
                    next.in = cn[q];
                    next.mass_above = mass_above;
                    next.found = 1;
                    next.last = shift == 0;
                    for (int i = 0; i < C; ++i) *cluster.map_shared_rank(&sh.cut, i) = next;
                }
                if (sh.stop == BINS && tid < C) cluster.map_shared_rank(&sh.cut, tid)->found = 0;  // all within reach
            }
            cluster.sync();
            if (!sh.cut.found) st.found = 0;
            else st = sh.cut;
        }
        if (st.found) {
            cut = value_of(st.hi);
            ties = ties_kept = st.in;
            if (k_on) ties_kept = min(ties_kept, max(1, k - st.above));
            if (p_on) {
                const u64 each = (u64)(mass(cut) * one + 0.5);
                u64 need = 1;
                if (each > 0 && want > st.mass_above) need = (want - st.mass_above + each - 1) / each;
                if (need < (u64)ties_kept) ties_kept = max((int)need, 1);
            }
        }
    }

    // ---- the draw: a thread's entries lie side by side (an odd number: no bank twice)
    const int per = ((p.chunk + THREADS - 1) / THREADS) | 1;
    const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
    int seen = 0;  // entries equal to the cut before this thread's
    const bool some_ties = ties_kept < ties;
    if (some_ties) {
        int mine = 0;
        for (int i = i0; i < i1; ++i) mine += at(i) == cut;
        int in = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, in, o);
            if (lane >= o) in += a;
        }
        __syncthreads();
        if (lane == 31) sh.warp_i[warp] = in;
        __syncthreads();
        seen = in - mine;
        int all = 0;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) seen += sh.warp_i[w];
            all += sh.warp_i[w];
        }
        tell_all(cluster, sh.ties, all);
        for (int i = 0; i < c; ++i) seen += sh.ties[i];
    }
    auto kept = [&](float l, int& s) { return l > cut || (l == cut && (!some_ties || s++ < ties_kept)); };
    double mine = 0.0;
    {
        int s = seen;
        for (int i = i0; i < i1; ++i) {
            const float l = at(i);
            if (kept(l, s)) mine += mass(l);
        }
    }
    double in = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double a = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += a;
    }
    __syncthreads();
    if (lane == 31) sh.warp_d[warp] = in;
    if (tid == 0) sh.who = THREADS, sh.last = -1;
    __syncthreads();
    double before = in - mine, all = 0.0;
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += sh.warp_d[w];
        all += sh.warp_d[w];
    }
    tell_all(cluster, sh.kept, all);
    double sum = 0.0;
    for (int i = 0; i < C; ++i) sum += sh.kept[i];
    const double draw = (double)p.uniform[b] * sum;
    int owner = -1, last = -1;
    double start = 0.0;
    {
        double acc = 0.0, last_start = 0.0;
        for (int i = 0; i < C; ++i) {
            if (sh.kept[i] > 0.0) {
                last = i, last_start = acc;
                if (owner < 0 && draw <= acc + sh.kept[i]) owner = i, start = acc;
            }
            acc += sh.kept[i];
        }
        if (owner < 0) owner = last, start = last_start;  // (u beyond 1: the last that is kept)
    }
    if (owner != c) return;
    before += start;
    if (mine > 0.0) {
        atomicMax(&sh.last, tid);
        if (draw <= before + mine) atomicMin(&sh.who, tid);
    }
    __syncthreads();
    if (tid == (sh.who < THREADS ? sh.who : sh.last)) {
        int s = seen, token = 0;
        double acc = before;
        for (int i = i0; i < i1; ++i) {
            const float l = at(i);
            if (!kept(l, s)) continue;
            const double e = mass(l);
            if (e > 0.0) token = lo + i;  // (what rounds to nothing is never the pick)
            acc += e;
            if (e > 0.0 && draw <= acc) break;
        }
        p.out[b] = token;
    }
}

}  // namespace

// temperature [B] (<= 0 or NaN: greedy), uniform [B] in [0, 1); top_k (<= 0 or >= V: off), top_p (>= 1: off)
// and min_p (<= 0: off, above 1 as 1) [B] or null.
extern "C" int rfx_sample_rows(const float* logits, long long ld, int B, int V, const float* temperature,
                               const float* uniform, const int* top_k, const float* top_p, const float* min_p, int* out,
                               void* stream) {
    if (B <= 0) return 0;
    if (V <= 0 || ld < V) return RFX_ERR_BAD_ARG;
    int C = 1;
    while (C < MAX_CLUSTER && (long long)C * 4096 < V) C *= 2;
    const int chunk = ((V + C - 1) / C + 3) / 4 * 4;
    const size_t hist = (size_t)BINS * 12, piece = (size_t)chunk * 4;
    const bool staged = hist + piece <= 200 * 1024;
    Params p{logits, ld, V, chunk, temperature, uniform, top_p, min_p, top_k, out};
    auto kernel = staged ? sample_rows_kernel<true> : sample_rows_kernel<false>;
    const size_t smem = hist + (staged ? piece : 0);
    static SmemLimit limits[2];
    cudaError_t e = limits[staged].raise(kernel, smem);
    if (e == cudaSuccess)
        e = launch(kernel, dim3(B, 1, C), THREADS, smem, (cudaStream_t)stream, C, p);
    return (int)e;
}
