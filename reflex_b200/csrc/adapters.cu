// Adapters of a step's requests: the rows grouped by adapter, and the low-rank products in 32-bit
// multiply-adds.
//
//  * rows: a stable counting sort of the rows by their adapter's number, rows without one last, and the
//    groups cut into tiles of at most T rows.  One block: every warp counts a piece of the rows; a prefix over
//    (number, warp) gives each warp the place at which its rows of a number go, and lanes with the same number
//    find their order by a match, so nothing depends on the order of atomics.  Latency bounds it: 64 rows
//    4.0 us, 16,384 rows of 48 prompts over 500 adapters 11 us.
//  * add: out[r, c] = base[r, c] + s_a sum_i B_a[c, i] (sum_k A_a[part(c), i, k] x[r, k]), a the row's
//    adapter, in two launches: the low-rank rows v = A x (k in LOW_SPLITS pieces that depend on K alone, an
//    element's products added in k's order, the pieces' sums in order, so that a row's bits do not depend on
//    what else is in the step), then out.  Any sizes, strides and alignment, 32-bit and bfloat16.  The multiply-adds
//    and the shared memory that feeds them bound it: 701 rows by 1,024, rank 16, 2,048 columns 20 us.
#include "adapters.cuh"

namespace {

using namespace rfx;
using namespace adapters;

constexpr int GROUP_THREADS = 1024;
constexpr int MAX_ADAPTERS = 1024;

__device__ __forceinline__ int warp_inclusive(int v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Exclusive prefix over the block of a value a thread; `total` is the sum.  `scratch` holds 33 ints.
__device__ __forceinline__ int block_exclusive(int v, int* scratch, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int in = warp_inclusive(v);
    __syncthreads();
    if (lane == 31) scratch[warp] = in;
    __syncthreads();
    if (warp == 0) {
        const int w = scratch[lane];
        const int s = warp_inclusive(w);
        scratch[lane] = s - w;
        if (lane == 31) scratch[32] = s;
    }
    __syncthreads();
    *total = scratch[32];
    return scratch[warp] + in - v;
}

// cnt[w][key]: rows of a key in warp w's piece, then the place of the first of them; two more rows: the
// first place of every key, and the first tile of every key.
__global__ void __launch_bounds__(GROUP_THREADS)
adapter_rows_kernel(const int* __restrict__ ids, int R, int n, int T, int* __restrict__ order, int* __restrict__ first,
                    int* __restrict__ tiles, int max_tiles, int* __restrict__ err) {
    extern __shared__ int sh[];
    __shared__ int scratch[33];
    pdl_prologue();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = GROUP_THREADS / 32;
    const int keys = n + 1;
    int* cnt = sh;
    int* s_first = sh + warps * keys;
    int* s_tile = s_first + keys + 1;
    const int piece = ((R + warps - 1) / warps + 31) / 32 * 32;
    const int lo = min(R, warp * piece), hi = min(R, lo + piece);
    for (int i = threadIdx.x; i < warps * keys; i += GROUP_THREADS) cnt[i] = 0;
    __syncthreads();
    int* mine = cnt + warp * keys;
    bool bad = false;
    constexpr int AHEAD = 8;  // rows a lane has loaded before it looks at the first
    int key[AHEAD];
    auto load_keys = [&](int r0) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) key[i] = r0 + i * 32 + lane < hi ? ids[r0 + i * 32 + lane] : -2;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const bool in = r0 + i * 32 + lane < hi;
            bad |= in && (key[i] < -1 || key[i] >= n);
            key[i] = !in ? -1 : (key[i] < 0 || key[i] >= n ? n : key[i]);
        }
    };
    for (int r0 = lo; r0 < hi; r0 += 32 * AHEAD) {
        load_keys(r0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (r0 + i * 32 >= hi) break;
            if (key[i] >= 0) atomicAdd(mine + key[i], 1);  // (a warp's own counters, and whole numbers)
        }
    }
    if (bad) atomicExch(err, 2);
    __syncthreads();
    // a key's count over the warps, the keys' first places and first tiles, a block's threads at a time
    int placed = 0, tiled = 0;
    for (int k0 = 0; k0 < keys; k0 += GROUP_THREADS) {
        const int k = k0 + threadIdx.x;
        int total = 0;
        if (k < keys)
#pragma unroll 8
            for (int w = 0; w < warps; ++w) {
                const int c = cnt[w * keys + k];
                cnt[w * keys + k] = total;
                total += c;
            }
        int all, all_tiles;
        const int at = placed + block_exclusive(total, scratch, &all);
        const int tile = tiled + block_exclusive((total + T - 1) / T, scratch, &all_tiles);
        if (k < keys) {
            s_first[k] = at;
            s_tile[k] = tile;
            first[k] = at;
        }
        placed += all;
        tiled += all_tiles;
    }
    if (threadIdx.x == 0) {
        s_first[keys] = placed;
        s_tile[keys] = tiled;
        first[keys] = placed;
    }
    __syncthreads();
    for (int r0 = lo; r0 < hi; r0 += 32 * AHEAD) {
        load_keys(r0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (r0 + i * 32 >= hi) break;
            // rows of one prompt are one number: the match, which takes as long as all the rest, is for others
            const int k = key[i];
            unsigned same = 0xffffffffu;
            if (!__all_sync(0xffffffffu, k == __shfl_sync(0xffffffffu, k, 0))) same = __match_any_sync(0xffffffffu, k);
            if (k >= 0) order[s_first[k] + mine[k] + __popc(same & ((1u << lane) - 1))] = r0 + i * 32 + lane;
            __syncwarp();
            if (k >= 0 && lane == __ffs(same) - 1) mine[k] += __popc(same);
            __syncwarp();
        }
    }
    for (int t = threadIdx.x; t < max_tiles; t += GROUP_THREADS) {
        int a = -1, place = 0, count = 0;
        if (t < tiled) {
            int l = 0, h = keys - 1;  // the last key whose first tile is at or before t and that has rows
            while (l < h) {
                const int m = (l + h + 1) / 2;
                if (s_tile[m] <= t) l = m;
                else h = m - 1;
            }
            a = l;
            place = s_first[l] + (t - s_tile[l]) * T;
            count = min(T, s_first[l + 1] - place);
        }
        tiles[3 * t] = a;
        tiles[3 * t + 1] = place;
        tiles[3 * t + 2] = count;
    }
}

// ---- the products in 32-bit multiply-adds ------------------------------------------------------------
constexpr int LOW_SPLITS = 8, ROWS = 32, COLS = 32, BK = 32, OUT_COLS = 64, FIRST = 4, MAX_TURNS = 8;

__host__ __device__ inline int k_piece(int K) { return ((K + LOW_SPLITS - 1) / LOW_SPLITS + BK - 1) / BK * BK; }
__host__ __device__ inline int k_pieces(int K) { return (K + k_piece(K) - 1) / k_piece(K); }

// Four neighbours of a row's first `left`, zeros beyond; `whole`: the row's fours lie on their own size.
template <typename T>
__device__ __forceinline__ float4 four(const T* p, int left, bool whole) {
    if (whole && left >= 4) return load4(p);
    return make_float4(left > 0 ? ld(p, 0) : 0.f, left > 1 ? ld(p, 1) : 0.f, left > 2 ? ld(p, 2) : 0.f,
                       left > 3 ? ld(p, 3) : 0.f);
}
__device__ __forceinline__ void fma4(float& s, const float4& a, const float4& b) {
    s = fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, s))));
}

// low[piece][place][part * rank + i]: 32 rows x 32 rank rows a block, four sums a thread; the next 32 of K are on
// their way while these are multiplied.
template <typename T>
__global__ void __launch_bounds__(256) adapter_low_kernel(const Args p, int x_whole, int a_whole) {
    constexpr int LD = BK + 4;
    __shared__ __align__(16) float xs[2][ROWS][LD], as[2][COLS][LD];
    pdl_prologue();
    const int subs = (p.tile + ROWS - 1) / ROWS;
    const Tile t = load_tile(p.tiles, blockIdx.x / subs);
    const int sub = blockIdx.x % subs * ROWS, W = p.parts.n * p.rank;
    if (t.adapter < 0 || t.adapter >= p.n || sub >= t.count) return;
    const int here = min(ROWS, t.count - sub), w0 = blockIdx.y * COLS, rank = p.rank_of(t.adapter);
    const int k0 = blockIdx.z * k_piece(p.K), k1 = min(p.K, k0 + k_piece(p.K));
    // what this thread brings: four of K of a row of x and of a rank row
    const int row = threadIdx.x >> 3, k4 = (threadIdx.x & 7) * 4, w = w0 + row;
    const T* x = (const T*)p.x + (size_t)p.order[t.place + sub + min(row, here - 1)] * p.ld_x;
    const T* a = (const T*)p.a + ((size_t)t.adapter * W + min(w, W - 1)) * p.lda;
    const bool a_on = w < W && w % p.rank < rank;
    auto load_x = [&](int k) { return four(x + k + k4, k1 - k - k4, x_whole); };
    auto load_a = [&](int k) { return four(a + k + k4, a_on ? k1 - k - k4 : 0, a_whole); };
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    float4 nx = load_x(k0), na = load_a(k0);
    for (int k = k0, s = 0; k < k1; k += BK, s ^= 1) {
        store4(&xs[s][row][k4], nx);
        store4(&as[s][row][k4], na);
        __syncthreads();
        if (k + BK < k1) nx = load_x(k + BK), na = load_a(k + BK);
#pragma unroll
        for (int kk = 0; kk < BK; kk += 4) {
            const float4 av = load4(&as[s][tx][kk]);
#pragma unroll
            for (int j = 0; j < 4; ++j) fma4(acc[j], load4(&xs[s][ty * 4 + j][kk]), av);
        }
    }
    if (w0 + tx < W)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (ty * 4 + j < here)
                p.low[((size_t)blockIdx.z * p.R + t.place + sub + ty * 4 + j) * W + w0 + tx] = acc[j];
}

// 32 rows by `turns` times 64 columns a block, eight rows of a column a thread.  What hangs on the tile alone (the rows'
// places, B's first numbers, the pieces' sums) is asked for at once; rows behind the tile's last are its last again and
// not stored.
template <typename T, typename TO>
__global__ void __launch_bounds__(256) adapter_up_kernel(const Args p, int turns, int b_whole) {
    extern __shared__ __align__(16) float vs[];  // [ROWS][parts][rank in fours]
    pdl_prologue();
    const int subs = (p.tile + ROWS - 1) / ROWS;
    const Tile t = load_tile(p.tiles, blockIdx.x / subs);
    const int sub = blockIdx.x % subs * ROWS, W = p.parts.n * p.rank, wide = (p.rank + 3) / 4 * 4, LD = p.parts.n * wide;
    if (t.adapter < 0 || sub >= t.count) return;
    const bool none = t.adapter >= p.n;
    if (none && p.out == p.base) return;
    const int here = min(ROWS, t.count - sub), r0 = (threadIdx.x >> 6) * 8;
    const int rank = none ? 0 : p.rank_of(t.adapter);
    const float scale = none ? 0.f : p.scale[t.adapter];
    const TO* base = (const TO*)p.base;
    TO* out = (TO*)p.out;
    int rows[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) rows[j] = p.order[t.place + sub + min(r0 + j, here - 1)];
    int c = blockIdx.y * turns * OUT_COLS + (threadIdx.x & 63);
    for (int turn = 0; turn < turns; ++turn, c += OUT_COLS) {
        const T* b = (const T*)p.b + ((size_t)t.adapter * p.N + c) * p.rank;
        float4 ahead[FIRST];
        float y[8], acc[8] = {};
        if (c < p.N) {
#pragma unroll
            for (int i = 0; i < FIRST; ++i)
                if (4 * i < rank) ahead[i] = four(b + 4 * i, rank - 4 * i, b_whole);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = ld(base, (size_t)rows[j] * p.ld_base + c);
        }
        if (turn == 0 && !none) {
            const int pieces = k_pieces(p.K);
            const float* low = p.low + ((size_t)t.place + sub) * W;
            const size_t apart = (size_t)p.R * W;
            if (wide == p.rank) {  // (the rows lie in memory as in vs)
                for (int i = threadIdx.x * 4; i < here * W; i += 1024) {
                    float4 v = load4(low + i);
                    for (int s = 1; s < pieces; ++s) {
                        const float4 d = load4(low + s * apart + i);
                        v.x += d.x, v.y += d.y, v.z += d.z, v.w += d.w;
                    }
                    store4(vs + i, v);
                }
            } else {
                for (int i = threadIdx.x; i < here * LD; i += 256) {
                    const int r = i / LD, q = (i - r * LD) / wide, k = i - r * LD - q * wide;
                    float v = 0.f;
                    if (k < p.rank)
                        for (int s = 0; s < pieces; ++s) v += low[s * apart + r * W + q * p.rank + k];
                    vs[i] = v;
                }
            }
            __syncthreads();
        }
        if (c >= p.N) continue;
        if (!none) {
            const float* v = vs + p.parts.part_of(c) * wide + r0 * LD;
            auto add = [&](int i, const float4& bi) {
#pragma unroll
                for (int j = 0; j < 8; ++j) fma4(acc[j], load4(v + j * LD + i), bi);
            };
#pragma unroll
            for (int i = 0; i < FIRST; ++i)
                if (4 * i < rank) add(4 * i, ahead[i]);
#pragma unroll 2
            for (int i = 4 * FIRST; i < rank; i += 4) add(i, four(b + i, p.rank - i, b_whole));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (r0 + j < here) st(out, (size_t)rows[j] * p.ld_out + c, none ? y[j] : fmaf(scale, acc[j], y[j]));
    }
}

template <typename T, typename TO>
int fma_form(const Args& p, cudaStream_t s) {
    const int W = p.parts.n * p.rank, subs = (p.tile + ROWS - 1) / ROWS;
    const long long blocks = (long long)p.max_tiles * subs;
    if (blocks > 0x7fffffffLL || (p.N + OUT_COLS - 1) / OUT_COLS > 65535 || (W + COLS - 1) / COLS > 65535)
        return RFX_ERR_UNSUPPORTED;
    const size_t smem = (size_t)ROWS * p.parts.n * ((p.rank + 3) / 4 * 4) * sizeof(float);
    // rows that can be read by fours
    const size_t mask = 4 * sizeof(T) - 1;
    const int x_whole = (((size_t)p.x | (size_t)(p.ld_x * sizeof(T))) & mask) == 0;
    const int a_whole = (((size_t)p.a | (size_t)(p.lda * sizeof(T))) & mask) == 0;
    const int b_whole = (((size_t)p.b | (size_t)(p.rank * sizeof(T))) & mask) == 0;
    // As many turns as leave every SM its two blocks, which add the pieces up once (701 rows by 2,048 columns: 22.2 us
    // with one turn, 19.9 with two)
    const int groups = (p.N + OUT_COLS - 1) / OUT_COLS;
    const long long all = (long long)((p.R + ROWS - 1) / ROWS) * groups, fill = 2LL * sm_count();
    const int turns = (int)min((long long)MAX_TURNS, max(1LL, (all + fill - 1) / fill));
    static SmemLimit limit;
    cudaError_t e = limit.raise(adapter_up_kernel<T, TO>, smem);
    if (e != cudaSuccess) return (int)e;
    RFX_LAUNCH(adapter_low_kernel<T>, dim3((unsigned)blocks, (W + COLS - 1) / COLS, k_pieces(p.K)), 256, 0, s, p, x_whole, a_whole);
    RFX_LAUNCH((adapter_up_kernel<T, TO>), dim3((unsigned)blocks, (groups + turns - 1) / turns), 256, smem, s, p, turns, b_whole);
    return 0;
}

}  // namespace

// order [R], first [n + 2], tiles [max_tiles][3]; an id below -1 or from n on counts as none and sets *err.
extern "C" int rfx_adapter_rows(const int* ids, int R, int n, int tile, int* order, int* first, int* tiles,
                                int max_tiles, int* err, void* stream) {
    if (R <= 0 || n <= 0 || tile <= 0 || max_tiles < min(R, n + 1) + R / tile) return RFX_ERR_BAD_ARG;
    if (n > MAX_ADAPTERS) return RFX_ERR_UNSUPPORTED;
    const size_t smem = ((size_t)(GROUP_THREADS / 32) * (n + 1) + 2 * (n + 2)) * sizeof(int);
    static SmemLimit limit;
    cudaError_t e = limit.raise(adapter_rows_kernel, smem);
    if (e != cudaSuccess) return (int)e;
    RFX_LAUNCH(adapter_rows_kernel, 1, GROUP_THREADS, smem, (cudaStream_t)stream, ids, R, n, tile, order, first, tiles,
               max_tiles, err);
    return 0;
}

// A projection's adapters (the fields of ops.AdapterBank's `_Bank`).
struct AdapterBank {
    const void *a, *b;
    const float* scale;
    const int* ranks;
    int n, K, lda, N, rank, parts, woven, dt;
    int ends[MAX_PARTS];  // a part's last column and one
};

// The form that takes tiles of so many rows where x's lie on 16 bytes (0 takes them all): what rfx_adapter_add is
// given as `form`.
extern "C" int rfx_adapter_form(const AdapterBank* k, int tile, int dt_out) {
    if (!k || k->dt != RFX_DT_BF16 || k->K <= 0 || k->rank <= 0 || k->parts <= 0 || k->parts > MAX_PARTS) return 0;
    Args p{nullptr, nullptr, nullptr, k->a, k->b, k->scale, k->ranks, nullptr, nullptr, nullptr, 0, 0, 0, k->n, 1, k->K,
           k->lda, k->N, k->rank, 1, tile, {}};
    p.parts.n = k->parts;
    p.parts.woven = k->woven;
    return step_takes(p) ? 1 : prompt_takes(p, dt_out) ? 2 : 0;
}

// Floats of scratch that rfx_adapter_add needs in a form: 0 the products in 32-bit multiply-adds, 1 tiles of
// 16 rows and 2 tiles of 128 rows on the tensor cores.
extern "C" long long rfx_adapter_low_floats(const AdapterBank* k, int R, int form) {
    if (R <= 0 || !k || k->K <= 0 || form == 1) return 0;
    if (form == 2) return prompt_low_floats(R, k->parts * k->rank);
    return (long long)k_pieces(k->K) * R * k->parts * k->rank;
}

// dt_out: of base and out (32-bit, or bfloat16 beside bfloat16).
extern "C" int rfx_adapter_add(const AdapterBank* k, const int* order, const int* tiles, int max_tiles, int tile,
                               const void* base, long long ld_base, void* out, long long ld_out, int dt_out, const void* x,
                               long long ld_x, float* low, int R, int form, int* err, void* stream) {
    if (!k) return RFX_ERR_BAD_ARG;
    if (R <= 0 || k->N <= 0) return 0;
    if (k->K <= 0 || k->rank <= 0 || k->n <= 0 || tile <= 0 || max_tiles <= 0 || k->parts <= 0 || k->lda < k->K ||
        ld_x < k->K || ld_base < k->N || ld_out < k->N || (k->woven && (k->parts != 2 || k->N % 2)))
        return RFX_ERR_BAD_ARG;
    if (k->parts > MAX_PARTS || k->parts * k->rank > 1024 || (k->dt != RFX_DT_F32 && k->dt != RFX_DT_BF16) ||
        (k->dt == RFX_DT_F32 && dt_out != RFX_DT_F32) || (dt_out != RFX_DT_F32 && dt_out != RFX_DT_BF16))
        return RFX_ERR_UNSUPPORTED;
    Args p{base, out, x, k->a, k->b, k->scale, k->ranks, order, tiles, low, ld_base, ld_out, ld_x, k->n, R, k->K, k->lda,
           k->N, k->rank, max_tiles, tile, {}};
    p.parts.n = k->parts;
    p.parts.woven = k->woven;
    for (int i = 0; i < k->parts; ++i) p.parts.end[i] = k->ends[i];
    cudaStream_t s = (cudaStream_t)stream;
    if (form == 1) return k->dt == RFX_DT_BF16 && step_takes(p) ? step_form(p, dt_out, s) : RFX_ERR_UNSUPPORTED;
    if (form == 2 && low)
        return k->dt == RFX_DT_BF16 && prompt_takes(p, dt_out) ? prompt_form(p, dt_out, err, s) : RFX_ERR_UNSUPPORTED;
    if (form != 0 || !low) return RFX_ERR_BAD_ARG;
    if (k->dt == RFX_DT_F32) return fma_form<float, float>(p, s);
    if (dt_out == RFX_DT_F32) return fma_form<__nv_bfloat16, float>(p, s);
    return fma_form<__nv_bfloat16, __nv_bfloat16>(p, s);
}
