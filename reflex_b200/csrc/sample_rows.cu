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
// everything.  For top-k and top-p the cut is found in a histogram of 2,048 bins of 1/32 octave of e; the entries
// of the chosen bin, up to 512 or 1,024, go to every CTA, and the cut is found among them.  Where they are more, 2,048
// bins inside the bin follow, and, if several share one of those too (equal logits, a temperature that makes all
// alike), their bit patterns are narrowed 2,048 bins at a time until one value is left.
//
// A mass is good to 2e-9 of itself (about 24 instructions: see `Scale`) and sums are 64-bit fixed point: they do not
// depend on the order in which threads add, and a draw near one of 150,000 borders between tokens lands on the
// side that exact arithmetic gives (with plain 32-bit exponentials one row in ten thousand of a flat distribution
// does not; 64-bit ones throughout are as good and cost as much as all the rest).
//
// The row is read once (64 rows of 151,936: 39 MB, 6 us at the memory's rate), but every logit costs a mass, a
// histogram's atomics with a cut, and a place in a running sum: instructions bound it, and with few rows the
// cluster's barriers.  Rows of 151,936: one with top-p 15 to 22 us, eight without a cut 11, 64 with all kinds of cuts 64;
// 256 rows of 32,003 with all three 60.
#include <cooperative_groups.h>
#include <float.h>

#include <type_traits>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

using namespace rfx;

constexpr int BINS = 2048, COARSE = 64, MAX_WARPS = 32;
constexpr int PER_OCTAVE = 32;               // bins an octave: e below 2^-64 of the maximum is nothing
constexpr float FINE = PER_OCTAVE * (BINS / 2.0f);  // fine bins an octave: a bin and its roundings hold 2,048
typedef unsigned long long u64;

// bit patterns in the order of the values; -0 and 0 are one
__device__ __forceinline__ unsigned key_of(float l) {
    const unsigned u = __float_as_uint(l + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

struct Params {
    const float* logits;
    long long ld;
    int V, chunk, unit;  // a mass of 1 is 2^unit
    const float *temperature, *uniform, *top_p, *min_p;
    const int* top_k;
    int* out;
};

// Where an entry lies: y = (l - max) log2(e) / T = f - bin / 32, |f| <= 1/32.
struct Point {
    int bin;  // 0 .. 2048, at 2048 (and beyond) its mass is nothing
    float f;
};

// A row's scale.  c = log2(e) / T is kept in two floats, c max as m / 32 + g.  l c = n / 32 + r + s with n the nearest
// integer to 32 fl(l c_hi), r the exact rest of that product and s what the product left out; so the
// difference from the maximum loses no bits to its size, and f is good to 2^-30.  Rows whose c max is beyond
// 2^16 (logits or 1 / T in the tens of thousands) take 64-bit products instead.
struct Scale {
    float mx, hi, lo, floor, g;
    int m, unit;
    bool wide;
    double c;
    __device__ __forceinline__ static float rest(float l, float hi, float lo, float product) {
        return fmaf(l, lo, fmaf(l, hi, -product));
    }
    __device__ void set(float maximum, float T, int unit_) {
        mx = maximum, unit = unit_;
        c = 1.4426950408889634074 / (double)T;
        wide = !(fabs((double)mx * c) < 65536.0 && c < 1e30);
        hi = (float)c, lo = (float)(c - (double)hi);
        floor = (float)((double)mx - 70.0 / c);  // below 2^-64, and harmless
        if (!wide) {
            const float product = mx * hi, magic = fmaf(product, (float)PER_OCTAVE, 12582912.0f);
            m = __float_as_int(magic);
            g = fmaf(magic - 12582912.0f, -1.0f / PER_OCTAVE, product) + rest(mx, hi, lo, product);
        }
    }
    template <bool WIDE>
    __device__ __forceinline__ Point at(float l) const {
        if (WIDE) {
            const double y = l == mx ? 0.0 : fmax(((double)l - (double)mx) * c, -70.0), n = rint(y * PER_OCTAVE);
            return Point{min((int)-n, BINS), (float)(y - n * (1.0 / PER_OCTAVE))};
        }
        const float z = fmaxf(l, floor), product = z * hi;
        const float magic = fmaf(product, (float)PER_OCTAVE, 12582912.0f);  // its low bits are n
        const float r = fmaf(magic - 12582912.0f, -1.0f / PER_OCTAVE, product);
        return Point{min(m - __float_as_int(magic), BINS), r + (rest(z, hi, lo, product) - g)};
    }
    // 2^y in fixed point, 2^unit a one: 2^(-bin / 32) from a table and the exponent, 2^f - 1 by a polynomial (off by 4e-11); adding
    // 2^(52 - unit) leaves the integer in the sum's low bits
    __device__ __forceinline__ u64 mass(const Point& p, const double* table) const {
        const float q = p.f * fmaf(p.f, fmaf(p.f, fmaf(p.f, 0.009618129f, 0.05550411f), 0.24022651f), 0.69314718f);
        const double u = table[p.bin % PER_OCTAVE], one = __hiloint2double((52 - unit + 1023) << 20, 0);
        const double t = __hiloint2double(__double2hiint(u) - ((p.bin / PER_OCTAVE) << 20), __double2loint(u));
        const double sum = fma((double)q, t, t) + one;
        return ((u64)(unsigned)(__double2hiint(sum) - __double2hiint(one)) << 32) | (unsigned)__double2loint(sum);
    }
    // the distance below the maximum in fine bins; never decreasing as l falls (as `bin` is)
    __device__ __forceinline__ int fine(float l) const {
        if (l == mx) return 0;
        return (int)fminf((mx - l) * fminf(hi, FLT_MAX) * FINE, (float)(1 << 23));
    }
};

// CLUSTER: the most CTAs a row may have; LIST: the most entries of a bin among which the cut is looked for one by one.
template <int CLUSTER, int LIST_>
struct Shared {
    static constexpr int LIST = LIST_;
    u64 list_m[LIST];
    double table[PER_OCTAVE];  // 2^(-i / 32)
    u64 coarse_m[COARSE], all_m[CLUSTER][COARSE];  // this CTA's, and every CTA's
    u64 kept[CLUSTER], far[CLUSTER];
    u64 warp_m[MAX_WARPS];
    u64 mass_above, total;
    int coarse_n[COARSE], all_n[CLUSTER][COARSE];
    float list[LIST];
    float top[CLUSTER];
    int ties[CLUSTER], best[CLUSTER];
    int warp_i[MAX_WARPS];
    float warp_f[MAX_WARPS];
    int bin, above, in, who, listed;
    float cut;
};

template <typename T>
__device__ __forceinline__ void tell_all(cg::cluster_group& cluster, T* slots, T v) {
    const int C = cluster.num_blocks();
    if ((int)threadIdx.x < C) cluster.map_shared_rank(slots, threadIdx.x)[cluster.block_rank()] = v;
    cluster.sync();
}

template <typename T>
__device__ __forceinline__ T warp_inclusive(T v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

struct Hist {
    int* n;
    unsigned *lo, *hi;  // a bin's mass in two 32-bit halves
    __device__ __forceinline__ Hist(int* bins) : n(bins), lo((unsigned*)bins + BINS), hi((unsigned*)bins + 2 * BINS) {}
    __device__ __forceinline__ void clear() const {
        for (int i = threadIdx.x; i < BINS * 3 / 4; i += blockDim.x) reinterpret_cast<int4*>(n)[i] = make_int4(0, 0, 0, 0);
        __syncthreads();
    }
    __device__ __forceinline__ void add(int bin) const { atomicAdd(n + bin, 1); }
    // the addition that wraps the low half carries into the high one
    __device__ __forceinline__ void add(int bin, u64 m) const {
        atomicAdd(n + bin, 1);
        const unsigned m_lo = (unsigned)m, m_hi = (unsigned)(m >> 32);
        const unsigned old = atomicAdd(lo + bin, m_lo);
        const unsigned up = m_hi + (old + m_lo < old ? 1u : 0u);
        if (up) atomicAdd(hi + bin, up);
    }
};

// The rules of a row that cut by place in the descending order, and what lies above the bins now looked at.
struct Rules {
    int k;          // 0: no top-k
    bool p_on;
    float p;
    u64 want;       // top_p times the whole mass, one unit at least: the first token is kept whatever top_p is
    int above;
    u64 mass_above;
    int in;         // entries in the bin last chosen
};

// Whether the rules stop a row that has kept so much.
__device__ __forceinline__ bool stops(const Rules& r, int count, u64 mass) {
    return (r.k && count >= r.k) || (r.p_on && mass >= r.want);
}

// The first bin, over the cluster's histograms, at which a rule stops the row; -1: none does.  Every CTA finds it
// for itself, from 64 sums of 32 bins and then those 32.  `totals`: the bins hold the whole row but for the
// mass that every CTA told apart (`far`), and the sum gives `want`.  The cluster meets once more before the histogram is used again.
template <typename Sh>
__device__ int choose(cg::cluster_group& cluster, Sh& sh, const Hist& hist, Rules& rules, bool totals) {
    const int C = cluster.num_blocks(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    for (int q = warp; q < COARSE; q += blockDim.x / 32) {
        const int bin = q * 32 + lane, n = __reduce_add_sync(0xffffffffu, hist.n[bin]);
        if (lane == 0) sh.coarse_n[q] = n;
        if (rules.p_on) {
            // in three sums of 32-bit numbers: 32 times 22 bits fit
            const u64 m = ((u64)hist.hi[bin] << 32) + hist.lo[bin];
            const unsigned a = __reduce_add_sync(0xffffffffu, (unsigned)(m & 0x3fffffu));
            const unsigned b = __reduce_add_sync(0xffffffffu, (unsigned)((m >> 22) & 0x3fffffu));
            const unsigned d = __reduce_add_sync(0xffffffffu, (unsigned)(m >> 44));
            if (lane == 0) sh.coarse_m[q] = a + ((u64)b << 22) + ((u64)d << 44);
        }
    }
    __syncthreads();
    const int2 coarse_n = reinterpret_cast<const int2*>(sh.coarse_n)[lane];
    const ulonglong2 coarse_m = reinterpret_cast<const ulonglong2*>(sh.coarse_m)[lane];
    for (int r = warp; r < C; r += blockDim.x / 32) {
        reinterpret_cast<int2*>(cluster.map_shared_rank(sh.all_n[cluster.block_rank()], r))[lane] = coarse_n;
        if (rules.p_on)
            reinterpret_cast<ulonglong2*>(cluster.map_shared_rank(sh.all_m[cluster.block_rank()], r))[lane] = coarse_m;
    }
    cluster.sync();
    if (warp == 0) {
        int n[2] = {};
        u64 m[2] = {};
        for (int r = 0; r < C; ++r) {
            const int2 cn = reinterpret_cast<const int2*>(sh.all_n[r])[lane];
            n[0] += cn.x, n[1] += cn.y;
            if (rules.p_on) {
                const ulonglong2 cm = reinterpret_cast<const ulonglong2*>(sh.all_m[r])[lane];
                m[0] += cm.x, m[1] += cm.y;
            }
        }
        const int in = warp_inclusive(n[0] + n[1]);
        const u64 im = rules.p_on ? warp_inclusive(m[0] + m[1]) : 0ull;
        if (totals && rules.p_on) {
            u64 all = __shfl_sync(0xffffffffu, im, 31);
            for (int r = 0; r < C; ++r) all += sh.far[r];
            rules.want = max((u64)ceil((double)rules.p * (double)all), 1ull);
            if (lane == 0) sh.total = all;
        }
        // two coarse bins a lane
        const int n_before = rules.above + in - n[0] - n[1];
        const u64 m_before = rules.mass_above + im - m[0] - m[1];
        const bool first = n[0] && stops(rules, n_before + n[0], m_before + m[0]);
        const bool second = n[1] && stops(rules, n_before + n[0] + n[1], m_before + m[0] + m[1]);
        const unsigned any = __ballot_sync(0xffffffffu, first || second);
        if (lane == 0) sh.bin = -1;
        __syncwarp();
        if (any && lane == __ffs(any) - 1) {
            sh.bin = first ? 2 * lane : 2 * lane + 1;
            sh.above = first ? n_before : n_before + n[0];
            sh.mass_above = first ? m_before : m_before + m[0];
        }
    }
    __syncthreads();
    if (totals && rules.p_on) rules.want = max((u64)ceil((double)rules.p * (double)sh.total), 1ull);
    const int q = sh.bin;
    if (q < 0) return q;
    // the 32 bins of the chosen one, a warp a CTA
    for (int r = warp; r < C; r += blockDim.x / 32) {
        sh.all_n[r][lane] = cluster.map_shared_rank(hist.n, r)[q * 32 + lane];
        if (rules.p_on) {
            const unsigned hi = cluster.map_shared_rank(hist.hi, r)[q * 32 + lane];
            sh.all_m[r][lane] = ((u64)hi << 32) + cluster.map_shared_rank(hist.lo, r)[q * 32 + lane];
        }
    }
    __syncthreads();
    if (warp == 0) {
        int n = 0;
        u64 m = 0;
        for (int r = 0; r < C; ++r) {
            n += sh.all_n[r][lane];
            if (rules.p_on) m += sh.all_m[r][lane];
        }
        const int above = sh.above + warp_inclusive(n);
        const u64 mass_above = sh.mass_above + (rules.p_on ? warp_inclusive(m) : 0ull);
        const unsigned any = __ballot_sync(0xffffffffu, n && stops(rules, above, mass_above));
        // (the coarse bin stops the row, so one of its bins does)
        if (lane == __ffs(any) - 1) sh.bin = q * 32 + lane, sh.above = above - n, sh.mass_above = mass_above - m, sh.in = n;
    }
    __syncthreads();
    const int found = sh.bin;
    rules.above = sh.above, rules.mass_above = sh.mass_above, rules.in = sh.in;
    __syncthreads();  // (sh.bin may be written again)
    return found;
}

// STAGED: the CTA's piece of the row lies in shared memory; otherwise it is read again by every pass (from L2).
template <bool STAGED, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) sample_rows_kernel(const Params p) {
    constexpr int WARPS = THREADS / 32;
    extern __shared__ __align__(16) uint8_t dynamic[];
    // (rows with few CTAs beside them on an SM may have clusters of 16: two CTAs an SM have no room for that)
    using Sh = std::conditional_t<THREADS == 1024, Shared<16, 1024>, Shared<8, 512>>;
    __shared__ __align__(16) Sh sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), c = cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Hist hist(reinterpret_cast<int*>(dynamic));
    float* piece = reinterpret_cast<float*>(dynamic) + 3 * BINS;
    if (tid < PER_OCTAVE) sh.table[tid] = exp2((double)-tid / PER_OCTAVE);
    if (tid == 0) sh.listed = 0;
    cluster.barrier_arrive();  // met below: every CTA has begun before another writes into its memory
    pdl_prologue();
    const size_t b = blockIdx.x;
    const int lo = min(p.V, c * p.chunk), n = min(p.V, lo + p.chunk) - lo;
    const float* row = p.logits + b * p.ld + lo;
    auto at = [&](int i) { return STAGED ? piece[i] : __ldg(row + i); };

    // ---- the piece, and the row's maximum
    float mx = -INFINITY;
    if (STAGED && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
        const int n4 = n / 4;
#pragma unroll 5
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
    cluster.barrier_wait();
    tell_all(cluster, sh.top, mx);
    for (int i = 0; i < C; ++i) mx = fmaxf(mx, sh.top[i]);
    if (mx == -INFINITY) {  // nothing left
        if (c == 0 && tid == 0) p.out[b] = 0;
        return;
    }
    const float T = p.temperature[b];
    if (!(T > 0.0f)) {
        int best = -1;
#pragma unroll 4
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
    Scale scale;
    scale.set(mx, T, p.unit);
    const int k = p.top_k ? p.top_k[b] : 0;
    const float tp = p.top_p ? p.top_p[b] : 1.0f;
    Rules rules{k > 0 && k < p.V ? k : 0, tp < 1.0f, fmaxf(tp, 0.0f), 0ull, 0, 0ull, 0};
    float least = -FLT_MAX;  // the smallest logit that min-p keeps
    const float mp = p.min_p && p.min_p[b] > 0.0f ? fminf(p.min_p[b], 1.0f) : 0.0f;
    if (mp > 0.0f) {
        const double reach = -(double)T * log((double)mp);  // how far below the maximum it may lie
        least = mx;
        if (mx < INFINITY) {
            least = (float)((double)mx - reach);
            for (int i = 0; i < 4 && (double)mx - (double)least > reach; ++i) least = nextafterf(least, INFINITY);
            const float below = nextafterf(least, -INFINITY);
            if ((double)mx - (double)below <= reach) least = below;
        }
        least = fmaxf(fminf(least, mx), -FLT_MAX);
    }

    auto go = [&](auto is_wide) {
        constexpr bool WIDE = decltype(is_wide)::value;
        // ---- the cut: kept are the entries of bins above `bin_cut`, and in that bin those of fine bins above
        // `fine_cut`, and of those at it the ones above the value `cut` and `ties_kept` of those equal to it
        int bin_cut = BINS + 1, fine_cut = 0x7fffffff, ties_kept = 0x7fffffff, ties = 0;
        float cut = -INFINITY, bin_from = -FLT_MAX, bin_to = INFINITY;
        if (rules.k || rules.p_on) {
            hist.clear();
            // The mass that top-p goes by is the whole row's, so entries below min-p's reach count too.  Entries below
            // (1 - p) / 2V of the maximum have less than (1 - p) / 2 of the mass between them: they are beyond every
            // top-p cut, and their mass goes by a thread's sum.
            const float from = rules.p_on ? -FLT_MAX : least;
            const int far_bin = rules.p_on
                                    ? (int)fminf(PER_OCTAVE * (1.0f - log2f((1.0f - rules.p) / (2.0f * p.V))), (float)BINS)
                                    : BINS;
            u64 far = 0;
#pragma unroll 4
            for (int i = tid; i < n; i += THREADS) {
                const float l = at(i);
                const Point q = scale.template at<WIDE>(l);
                if (l >= from) {
                    if (rules.p_on) {
                        const u64 m = scale.mass(q, sh.table);
                        if (q.bin > far_bin) far += m;
                        else hist.add(min(q.bin, BINS - 1), m);
                    } else hist.add(min(q.bin, BINS - 1));
                }
            }
            if (rules.p_on) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) far += __shfl_xor_sync(0xffffffffu, far, o);
                if (lane == 0) sh.warp_m[warp] = far;
                __syncthreads();
                if (warp == 0) {
                    u64 f = lane < WARPS ? sh.warp_m[lane] : 0ull;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) f += __shfl_xor_sync(0xffffffffu, f, o);
                    if (lane < C) cluster.map_shared_rank(sh.far, lane)[c] = f;
                }
            }
            const int bin = choose(cluster, sh, hist, rules, true);
            if (bin >= 0) bin_cut = bin;
            // the logits that may lie in the bin: a bin to either side (both products are rounded to bins), and what
            // the product with c may be off
            if (bin >= 0) {
                const double off = 1.01 + 4e-6 * (fabs((double)mx * scale.c) + 70.0);
                if (bin < BINS - 1) bin_from = (float)((double)mx - (bin + off) / (PER_OCTAVE * scale.c));
                bin_to = (float)((double)mx - (bin - off) / (PER_OCTAVE * scale.c));
                if (WIDE) bin_from = -FLT_MAX, bin_to = mx;
            }
            auto in_bin = [&](float l) {
                return l >= from && !(l < bin_from || l > bin_to) && min(scale.template at<WIDE>(l).bin, BINS - 1) == bin;
            };
            if (bin >= 0 && rules.in > 1 && rules.in <= Sh::LIST) {
                // the bin's entries to every CTA, in any order, and the cut among them: the largest value at which a
                // rule stops the row, eight lanes an entry
#pragma unroll 4
                for (int i = tid; i < n; i += THREADS) {
                    const float l = at(i);
                    if (in_bin(l)) {
                        const int slot = atomicAdd(cluster.map_shared_rank(&sh.listed, 0), 1);
                        for (int r = 0; r < C; ++r) cluster.map_shared_rank(sh.list, r)[slot] = l;
                    }
                }
                cluster.sync();
                for (int i = tid; i < rules.in; i += THREADS)
                    sh.list_m[i] = rules.p_on ? scale.mass(scale.template at<WIDE>(sh.list[i]), sh.table) : 0ull;
                __syncthreads();
                // (more than 64 comparisons a thread: each CTA takes its share and tells the others, one more meeting of
                // 1.7 us; 64 rows of 151,936 with all kinds of cuts took 67 us on average where it now takes 57, logits in L2)
                const bool shared = C > 1 && rules.in * rules.in > 64 * THREADS;
                const int step = shared ? C : 1, mine = shared ? c : 0;
                for (int e0 = 0; e0 < rules.in; e0 += step * (THREADS / 8)) {
                    const int e = e0 + mine + step * (tid >> 3);
                    const float l = e < rules.in ? sh.list[e] : 0.f;
                    int above = 0, equal = 0;
                    u64 mass_above = 0;
#pragma unroll 4
                    for (int i = tid & 7; i < rules.in; i += 8) {
                        const float o = sh.list[i];
                        const u64 m = sh.list_m[i];
                        above += o > l;
                        mass_above += o > l ? m : 0ull;
                        equal += o == l;
                    }
#pragma unroll
                    for (int o = 4; o > 0; o >>= 1) {
                        above += __shfl_xor_sync(0xffffffffu, above, o);
                        equal += __shfl_xor_sync(0xffffffffu, equal, o);
                        mass_above += __shfl_xor_sync(0xffffffffu, mass_above, o);
                    }
                    above += rules.above, mass_above += rules.mass_above;
                    if (e < rules.in && (tid & 7) == 0) {
                        const u64 each = sh.list_m[e];
                        if (!stops(rules, above, mass_above) && stops(rules, above + equal, mass_above + equal * each))
                            for (int r = shared ? 0 : c; r < (shared ? C : c + 1); ++r) {  // (equal ones write the same)
                                Sh& to = *cluster.map_shared_rank(&sh, r);
                                to.above = above, to.mass_above = mass_above, to.in = equal, to.cut = l;
                            }
                    }
                }
                if (shared) cluster.sync();
                else __syncthreads();
                rules.above = sh.above, rules.mass_above = sh.mass_above, rules.in = sh.in;
                cut = sh.cut;
            } else if (bin >= 0 && rules.in > 1) {
                const int first = (bin - 1) * (BINS / 2);  // the bin's fine bins, half as many more on either side
                auto fine_of = [&](float l) { return min(max(scale.fine(l) - first, 0), BINS - 1); };
                cluster.sync();
                hist.clear();
#pragma unroll 4
                for (int i = tid; i < n; i += THREADS) {
                    const float l = at(i);
                    if (in_bin(l)) {
                        if (rules.p_on) hist.add(fine_of(l), scale.mass(scale.template at<WIDE>(l), sh.table));
                        else hist.add(fine_of(l));
                    }
                }
                const int fine = choose(cluster, sh, hist, rules, false);
                // the bit patterns there, until one value is left
                unsigned k_lo = key_of(-FLT_MAX), k_hi = key_of(mx);
                for (int round = 0; round < 4 && rules.in > 1; ++round) {
                    const unsigned range = k_hi - k_lo;
                    const int shift = range < BINS ? 0 : 21 - __clz(range);
                    cluster.sync();
                    hist.clear();
#pragma unroll 4
                    for (int i = tid; i < n; i += THREADS) {
                        const float l = at(i);
                        if (in_bin(l) && fine_of(l) == fine) {
                            const unsigned key = key_of(l);
                            if (key >= k_lo && key <= k_hi) {
                                if (rules.p_on) hist.add((k_hi - key) >> shift, scale.mass(scale.template at<WIDE>(l), sh.table));
                                else hist.add((k_hi - key) >> shift);
                            }
                        }
                    }
                    const unsigned q = choose(cluster, sh, hist, rules, false);
                    k_hi -= q << shift;
                    k_lo = max(k_lo, k_hi - min(k_hi, (1u << shift) - 1u));
                    cut = value_of(k_lo);
                    if (shift == 0) break;
                }
                fine_cut = fine + first;
                // (one entry left in a wider interval: it lies at or above the interval's end)
            }
            if (bin >= 0 && rules.in > 1) {  // all of one value
                ties = ties_kept = rules.in;
                if (rules.k) ties_kept = min(ties_kept, max(1, rules.k - rules.above));
                if (rules.p_on) {
                    const u64 each = scale.mass(scale.template at<WIDE>(cut), sh.table);
                    u64 need = 1;
                    if (each > 0 && rules.want > rules.mass_above) need = (rules.want - rules.mass_above + each - 1) / each;
                    if (need < (u64)ties_kept) ties_kept = max((int)need, 1);
                }
            }
        }

        // ---- the draw: a thread's entries lie side by side (an odd number: no bank twice)
        const int per = ((p.chunk + THREADS - 1) / THREADS) | 1;
        const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
        const bool some_ties = ties_kept < ties;
        const int fine_first = (bin_cut - 1) * (BINS / 2);
        int seen = 0;  // entries equal to the cut before this thread's
        if (some_ties) {
            int mine = 0;
            for (int i = i0; i < i1; ++i) mine += at(i) == cut;
            const int in = warp_inclusive(mine);
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
        const float lowest = fmaxf(least, bin_cut < BINS ? bin_from : -FLT_MAX);  // nothing below it is kept
        auto kept = [&](float l, const Point& q) {  // but for ties that are not all kept
            const int bin = min(q.bin, BINS - 1);
            if (!(l >= least) || bin > bin_cut) return false;
            if (bin < bin_cut) return true;
            if (fine_cut != 0x7fffffff) {
                const int fine = min(max(scale.fine(l) - fine_first, 0), BINS - 1) + fine_first;
                if (fine != fine_cut) return fine < fine_cut;
            }
            return l >= cut;
        };
        u64 mine = 0;
        if (bin_cut > BINS) {  // no cut but min-p's
#pragma unroll 4
            for (int i = i0; i < i1; ++i) {
                const float l = at(i);
                const u64 m = scale.mass(scale.template at<WIDE>(l), sh.table);
                mine += l >= least ? m : 0ull;
            }
        } else {
            int s = seen;
#pragma unroll 2
            for (int i = i0; i < i1; ++i) {
                const float l = at(i);
                if (!(l >= lowest)) continue;
                const Point q = scale.template at<WIDE>(l);
                if (kept(l, q) && !(some_ties && l == cut && s++ >= ties_kept)) mine += scale.mass(q, sh.table);
            }
        }
        const u64 in = warp_inclusive(mine);
        __syncthreads();
        if (lane == 31) sh.warp_m[warp] = in;
        __syncthreads();
        u64 before = in - mine, all = 0;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += sh.warp_m[w];
            all += sh.warp_m[w];
        }
        tell_all(cluster, sh.kept, all);
        u64 sum = 0, start = 0;
        for (int i = 0; i < C; ++i) {
            if (i < c) start += sh.kept[i];
            sum += sh.kept[i];
        }
        // the first at which the sum reaches u times the whole; a mass of one unit at least, the whole at most
        u64 draw = (u64)ceil((double)p.uniform[b] * (double)sum);
        draw = min(max(draw, (u64)1), sum);
        if (draw <= start || draw > start + all) return;  // another CTA's
        before += start;
        if (draw > before && draw <= before + mine) sh.who = tid;  // one thread's
        __syncthreads();
        if (warp != sh.who / 32) return;
        // its warp goes over its entries together
        const int who = sh.who % 32, w0 = __shfl_sync(0xffffffffu, i0, who), w1 = __shfl_sync(0xffffffffu, i1, who);
        u64 sums = __shfl_sync(0xffffffffu, before, who);
        int tied = __shfl_sync(0xffffffffu, seen, who);
        for (int i = w0; i < w1; i += 32) {
            const float l = i + lane < w1 ? at(i + lane) : -INFINITY;
            const unsigned equal = __ballot_sync(0xffffffffu, some_ties && l == cut);
            const Point q = scale.template at<WIDE>(l);
            bool take = kept(l, q);
            if (some_ties && l == cut) take = take && tied + __popc(equal & ((1u << lane) - 1)) < ties_kept;
            tied += __popc(equal);
            const u64 m = warp_inclusive(take ? scale.mass(q, sh.table) : 0ull);
            const unsigned hit = __ballot_sync(0xffffffffu, sums + m >= draw);
            if (hit) {
                if (lane == __ffs(hit) - 1) p.out[b] = lo + i + lane;
                return;
            }
            sums += __shfl_sync(0xffffffffu, m, 31);
        }
    };
    if (scale.wide) go(std::true_type{});
    else go(std::false_type{});
}

}  // namespace

// CTAs a row.  A cluster of 16 halves what its CTAs have to go over (a row of 151,936 with top-p: 23 -> 20 us), but a
// group of SMs holds one: eight rows took 16 us where clusters of eight take 11.  Only CTAs that each have an SM to
// themselves have room for what sixteen exchange.
extern "C" int rfx_sample_rows_ctas(int B, int V, int sms) {
    const int most = B <= 4 && 16 * B <= sms ? 16 : 8;
    int C = 1;
    while (C < most && (long long)C * 4096 < V && ((long long)B * C < 2 * sms || (long long)C * 19200 < V)) C *= 2;
    return C;
}

// temperature [B] (<= 0 or NaN: greedy), uniform [B] in [0, 1); top_k (<= 0 or >= V: off), top_p (>= 1: off)
// and min_p (<= 0: off, above 1 as 1) [B] or null.
extern "C" int rfx_sample_rows(const float* logits, long long ld, int B, int V, const float* temperature,
                               const float* uniform, const int* top_k, const float* top_p, const float* min_p, int* out,
                               void* stream) {
    if (B <= 0) return 0;
    if (V <= 0 || ld < V) return RFX_ERR_BAD_ARG;
    const int C = rfx_sample_rows_ctas(B, V, sm_count());
    const int chunk = ((V + C - 1) / C + 3) / 4 * 4;
    const size_t hist = (size_t)BINS * 12, piece = (size_t)chunk * 4;
    const bool staged = hist + piece <= 200 * 1024;
    int bits = 1;
    while (bits < 31 && (1LL << bits) < V) ++bits;
    // V masses of one fit 63 bits; more than 2^-44 is not asked of a mass
    const int unit = 62 - bits < 44 ? 62 - bits : 44;
    Params p{logits, ld, V, chunk, unit, temperature, uniform, top_p, min_p, top_k, out};
    // One CTA an SM: twice the threads hide the arithmetic's latency
    const bool few = (long long)B * C <= sm_count();
    const size_t smem = hist + (staged ? piece : 0);
    static SmemLimit limits[4];
    auto go = [&](auto kernel, int threads, SmemLimit& limit) {
        cudaError_t e = limit.raise(kernel, smem, C > 8);
        if (e == cudaSuccess) e = launch(kernel, dim3(B, 1, C), threads, smem, (cudaStream_t)stream, C, p);
        return (int)e;
    };
    if (staged)
        return few ? go(sample_rows_kernel<true, 1024>, 1024, limits[0]) : go(sample_rows_kernel<true, 512>, 512, limits[1]);
    return few ? go(sample_rows_kernel<false, 1024>, 1024, limits[2]) : go(sample_rows_kernel<false, 512>, 512, limits[3]);
}
