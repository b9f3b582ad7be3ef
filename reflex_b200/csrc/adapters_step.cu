// The adapters of a step's requests, a row or a few each: tiles of at most 16 rows, bfloat16, one launch.
//
// A thread-block cluster takes a tile and both products.  Each of its eight CTAs multiplies the tile's rows
// with A over an eighth of K on the tensor cores (m16n8k16: 16 rows, 8 rank rows), a warp every eighth 8 rank rows;
// the partial sums of a few rows go straight to all eight CTAs' shared memory (of many, each CTA fetches them there,
// and the cluster meets once more: 0.5 us), and each adds them up in the same order; then it multiplies the low-rank
// rows with its share of B's columns and adds the base.  Nothing but the result goes back to memory, and there is one
// launch where two would have to follow one another.
//
// It is latency that counts, the chain tile -> row -> x and A -> cluster -> B, and then the adapters' bytes: one row
// with an adapter of rank 16 beside 4,096 x 6,144 (0.6 MB) takes 5.8 us, 64 rows over 32 adapters of ranks to 64
// (33 MB with base and out) 19 us, eight through 4,096 x 24,576 11 us.  So a warp's batches of A and then of B follow
// one another through a ring of shared memory, 4 KB on their way, B's first while the cluster meets; every lane
// reads what it brought itself (no barrier), k permuted alike on both sides so that its numbers lie side by side.
// A deeper ring is slower (four batches: 20 us): at 64 rows the memory is busy as it is, and the adapters of small
// rank then take more of it from those of large rank, which end last.
//
// The low-rank rows are kept in 32 bits and go into the second product as three bfloat16 parts (24 bits).  What the tensor
// cores cut off is kept small: sums over K in chains of a batch, added in 32 bits, and the smallest part first (one
// row with a 32-bit result is off by 1.3e-7; 4.4e-7 in chains of a whole slice).
// How K is cut depends on K alone, and a row's sums on nothing else in the tile, so a row has the same bits
// whatever shares its step.
#include <cooperative_groups.h>

#include "adapters.cuh"
#include "attn_mma.cuh"

namespace cg = cooperative_groups;

namespace {

using namespace rfx;
using namespace adapters;

constexpr int CLUSTER = 8, THREADS = 256, WARPS = THREADS / 32, TILE = 16;
constexpr int RING = 3;    // a warp's batches of A and B on their way or in use
constexpr int BATCH = 4;   // of A: 8 rank rows by 4 times 32 of K; of B: a group of columns by 32 of the rank
constexpr int GROUP = 32;  // columns a warp makes at a time

// (in whole batches of 128)
__host__ __device__ inline int k_slice(int K) { return ((K + CLUSTER - 1) / CLUSTER + 127) / 128 * 128; }
// elements from row to row: 64 bytes from where a row's banks begin, so that 16-byte reads by four lanes of two rows meet
// different ones
__host__ __device__ inline int ld_x_of(int K) { return k_slice(K) + 32; }
__host__ __device__ inline int ld_v_of(int W) { return (W + 63) / 64 * 64 + 32; }
// bytes of shared memory: the warps' rings; the rows of x and, when they have been read, v's three parts; partial rows
__host__ __device__ inline int rows_bytes(int W, int K) { return max(TILE * ld_x_of(K) * 2, 3 * TILE * ld_v_of(W) * 2); }
__host__ __device__ inline int sums_bytes(int W) { return max(TILE * W * 4, min(2 * TILE * W * 4, 24 * 1024)); }
inline int step_smem(int W, int K) { return WARPS * RING * BATCH * 512 + rows_bytes(W, K) + sums_bytes(W); }

__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}

template <typename TO>
__device__ __forceinline__ void load8(const TO* p, float (&v)[8]) {
    const float4 a = load4(p), b = load4(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

template <typename TO>
__global__ void __launch_bounds__(THREADS, 2) adapter_step_kernel(const Args p, int groups, int vec) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    cg::cluster_group cluster = cg::this_cluster();
    const int W = p.parts.n * p.rank, LDV = ld_v_of(W), slice = k_slice(p.K), LDX = ld_x_of(p.K);
    uint8_t* ring = dynamic;                                                                  // [WARPS][RING][BATCH][lane]
    __nv_bfloat16* xs = reinterpret_cast<__nv_bfloat16*>(ring + WARPS * RING * BATCH * 512);  // [TILE][LDX]
    __nv_bfloat16* vs = xs;                                                                   // [3][TILE][LDV]
    float* sums = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(xs) + rows_bytes(W, p.K));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_prologue();
    const Tile tile = load_tile(p.tiles, blockIdx.y);
    if (tile.adapter < 0) return;  // (the same for the whole cluster)
    const bool none = tile.adapter >= p.n;
    if (none && p.out == p.base) return;
    const int count = min(tile.count, TILE), c = cluster.block_rank();
    const int row_lo = p.order[tile.place + min(g, count - 1)], row_hi = p.order[tile.place + min(g + 8, count - 1)];
    const int rank = none ? 0 : p.rank_of(tile.adapter);
    const float scale = none ? 0.f : p.scale[tile.adapter];
    const int per = (rank + 7) / 8, tiles = per * p.parts.n, b_batches = (per + 3) / 4;
    if (!none) cluster_arrive();  // (the cluster's CTAs have begun: waited for before the first store to another)
    // ---- x's rows over this CTA's slice of K
    const int k0 = c * slice, k1 = min(p.K, k0 + slice), blocks = k0 < k1 ? (k1 - k0 + 31) / 32 : 0;
    if (!none) {
        const __nv_bfloat16* x = (const __nv_bfloat16*)p.x;
        const int padded = (blocks + BATCH - 1) / BATCH * BATCH * 32;
        const int rows[2] = {__shfl_sync(0xffffffffu, row_lo, warp * 4), __shfl_sync(0xffffffffu, row_hi, warp * 4)};
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (warp + 8 * h < count)
                for (int k = lane * 8; k < padded; k += 256)
                    attn::cp_async_16(xs + (warp + 8 * h) * LDX + k, k0 + k < k1 ? x + (size_t)rows[h] * p.ld_x + k0 + k : x,
                                      k0 + k < k1);
    }
    attn::cp_async_commit();

    // a warp's columns: groups of 32 from the start of a part (woven: of the whole), lane (g, t) has columns
    // 8 t .. 8 t + 7 of rows g and g + 8
    const __nv_bfloat16* b = (const __nv_bfloat16*)p.b + (size_t)tile.adapter * p.N * p.rank;
    int group = (blockIdx.x * CLUSTER + c) * WARPS + warp;
    const int stride = gridDim.x * CLUSTER * WARPS;
    auto locate = [&](int q, int& col, int& end, int& part) {
        int first = 0;
        part = 0;
        if (!p.parts.woven)
            while (true) {
                const int n = (p.parts.end[part] - first + GROUP - 1) / GROUP;
                if (q < n || part + 1 == p.parts.n) break;
                q -= n;
                first = p.parts.end[part++];
            }
        col = first + q * GROUP;
        end = p.parts.woven ? p.N : p.parts.end[part];
    };
    // ---- a warp's batches of A, then of B: tiles of 8 rank rows n = warp, warp + 8, ..., 128 of K at a time, then its
    // groups of columns, 32 of the rank at a time; a lane brings, and reads, its own 16 bytes of each 32 numbers
    const __nv_bfloat16* a = (const __nv_bfloat16*)p.a + (size_t)tile.adapter * W * p.lda;
    const uint32_t my_ring = attn::smem_u32(ring) + warp * RING * BATCH * 512 + lane * 16;
    int next_n = blocks ? warp : tiles, next_b = 0, next_slot = 0, next_group = b_batches ? group : groups;
    int next_part = 0, next_in = warp;  // tile next_n is number next_in of its part
    auto settle = [&]() {
        while (per && next_in >= per) next_in -= per, ++next_part;
    };
    settle();
    auto copy = [&](int j, const __nv_bfloat16* src, bool there) {  // (zeros if not)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(my_ring + (next_slot * BATCH + j) * 512),
                     "l"(there ? src : a), "r"(there ? 16 : 0)
                     : "memory");
    };
    auto bring = [&]() {
        if (next_n < tiles) {
            const int row = next_part * p.rank + next_in * 8 + g;
            const __nv_bfloat16* src = a + (size_t)row * p.lda + k0 + next_b * 32 + t * 8;
#pragma unroll
            for (int j = 0; j < BATCH; ++j) copy(j, src + j * 32, k0 + (next_b + j) * 32 + t * 8 < k1);
            if ((next_b += BATCH) >= blocks) {
                next_b = 0, next_n += WARPS, next_in += WARPS;
                settle();
            }
            if (++next_slot == RING) next_slot = 0;
        } else if (next_group < groups) {
            int col, end, part;
            locate(next_group, col, end, part);
            const int k = next_b * 32 + t * 8;
#pragma unroll
            for (int j = 0; j < BATCH; ++j)  // tile j: columns col + 4 n + j
                copy(j, b + (size_t)min(col + 4 * g + j, end - 1) * p.rank + k, k < per * 8);
            if (++next_b == b_batches) next_b = 0, next_group += stride;
            if (++next_slot == RING) next_slot = 0;
        }
        attn::cp_async_commit();
    };
    for (int i = 0; i < RING - 1; ++i) bring();
    const TO* base = (const TO*)p.base;
    TO* out = (TO*)p.out;
    auto load_base = [&](int col, int end, int r, int row, float (&v)[8]) {
        const int at = col + 8 * t;
        if (r < count) {
            const TO* src = base + (size_t)row * p.ld_base + at;
            if (vec && at + 8 <= end && (at & 7) == 0) load8(src, v);
            else
                for (int i = 0; i < 8; ++i) v[i] = at + i < end ? ld(src, i) : 0.f;
        }
    };
    float base_lo[8], base_hi[8];
    int col = 0, end = 0, part = 0;
    if (group < groups) {
        locate(group, col, end, part);
        load_base(col, end, g, row_lo, base_lo);
        load_base(col, end, g + 8, row_hi, base_hi);
    }

    int slot = 0;
    if (!none) {
        // ---- the low-rank rows over this CTA's slice of K
        attn::cp_async_wait<RING - 1>();
        __syncthreads();  // x is there
        // (few rows: straight to where each CTA adds them up; else each CTA fetches them)
        const int wide = tiles * 8;
        const bool push = CLUSTER * count * wide * 4 <= sums_bytes(W);
        cluster_wait();
        const uint32_t x_at = attn::smem_u32(xs) + (g * LDX + t * 8) * 2;
        for (int n = warp; n < tiles; n += WARPS) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            for (int i = 0; i < blocks; i += BATCH) {
                float some[4] = {0.f, 0.f, 0.f, 0.f};  // a batch's: the tensor cores cut sums off, and chains are kept short
                bring();
                attn::cp_async_wait<RING - 1>();
                uint4 w[BATCH], xa[BATCH], xb[BATCH];
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    w[j] = lds16(my_ring + (slot * BATCH + j) * 512);
                    xa[j] = lds16(x_at + (i + j) * 64);
                    xb[j] = lds16(x_at + 8 * LDX * 2 + (i + j) * 64);
                }
                if (++slot == RING) slot = 0;
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const uint32_t f0[4] = {xa[j].x, xb[j].x, xa[j].y, xb[j].y}, f1[4] = {xa[j].z, xb[j].z, xa[j].w, xb[j].w};
                    attn::mma_bf16(some, f0, w[j].x, w[j].y);
                    attn::mma_bf16(some, f1, w[j].z, w[j].w);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] += some[j];
            }
            if (push) {
#pragma unroll
                for (int q = 0; q < CLUSTER; ++q) {
                    float* to = cluster.map_shared_rank(sums, q) + c * count * wide + n * 8 + t * 2;
                    if (g < count) store2(to + g * wide, acc[0], acc[1]);
                    if (g + 8 < count) store2(to + (g + 8) * wide, acc[2], acc[3]);
                }
            } else {
                store2(sums + g * wide + n * 8 + t * 2, acc[0], acc[1]);
                store2(sums + (g + 8) * wide + n * 8 + t * 2, acc[2], acc[3]);
            }
        }
        cluster_arrive();
        cluster_wait();
        // ---- the cluster's sums, in three parts of bfloat16
        for (int i = tid; i < count * wide; i += THREADS) {
            const int r = i / wide, n = i - r * wide;
            float d[CLUSTER], v = 0.f;
#pragma unroll
            for (int q = 0; q < CLUSTER; ++q) d[q] = push ? sums[q * count * wide + i] : cluster.map_shared_rank(sums, q)[i];
#pragma unroll
            for (int q = 0; q < CLUSTER; ++q) v += d[q];
            const int at = r * LDV + n;
            const __nv_bfloat16 hi = __float2bfloat16_rn(v);
            const float rest = v - __bfloat162float(hi);
            const __nv_bfloat16 mid = __float2bfloat16_rn(rest);
            vs[at] = hi;
            vs[TILE * LDV + at] = mid;
            vs[2 * TILE * LDV + at] = __float2bfloat16_rn(rest - __bfloat162float(mid));
        }
        if (push) __syncthreads();
        else {  // no CTA leaves while another reads its sums
            cluster_arrive();
            cluster_wait();
        }
    }

    // ---- the columns
    const uint32_t v_at = attn::smem_u32(vs) + (g * LDV + t * 8) * 2;
    for (; group < groups; group += stride) {
        // the next group's base is on its way meanwhile
        int next_col = 0, next_end = 0, next_part = 0;
        float next_lo[8], next_hi[8];
        if (group + stride < groups) {
            locate(group + stride, next_col, next_end, next_part);
            load_base(next_col, next_end, g, row_lo, next_lo);
            load_base(next_col, next_end, g + 8, row_hi, next_hi);
        }
        float acc[4][4] = {};
        for (int i = 0; i < b_batches; ++i) {
            bring();
            attn::cp_async_wait<RING - 1>();
            uint4 w[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) w[j] = lds16(my_ring + (slot * BATCH + j) * 512);
            if (++slot == RING) slot = 0;
            const bool there = i * 32 + t * 8 < per * 8;  // (what lies beyond is no number of this part)
#pragma unroll
            for (int q = 2; q >= 0; --q) {  // the smallest part first
                auto frag = [&](int sp, uint4& lo, uint4& hi) {
                    const uint32_t at = v_at + (q * TILE * LDV + sp * per * 8 + i * 32) * 2;
                    lo = hi = make_uint4(0, 0, 0, 0);
                    if (there && g < count) lo = lds16(at);
                    if (there && g + 8 < count) hi = lds16(at + 8 * LDV * 2);
                };
                auto multiply = [&](int j, const uint4& lo, const uint4& hi) {
                    const uint32_t f0[4] = {lo.x, hi.x, lo.y, hi.y}, f1[4] = {lo.z, hi.z, lo.w, hi.w};
                    attn::mma_bf16(acc[j], f0, w[j].x, w[j].y);
                    attn::mma_bf16(acc[j], f1, w[j].z, w[j].w);
                };
                uint4 lo, hi;
                frag(part, lo, hi);
                multiply(0, lo, hi);
                multiply(2, lo, hi);
                if (p.parts.woven) frag(1, lo, hi);
                multiply(1, lo, hi);
                multiply(3, lo, hi);
            }
        }
        auto store = [&](int r, int row, const float (&y)[8], int h) {
            const int at = col + 8 * t;
            if (r >= count) return;
            TO* dst = out + (size_t)row * p.ld_out + at;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = none ? y[i] : fmaf(scale, acc[i & 3][h + (i >> 2)], y[i]);
            if (vec && at + 8 <= end && (at & 7) == 0) {
                store4(dst, make_float4(v[0], v[1], v[2], v[3]));
                store4(dst + 4, make_float4(v[4], v[5], v[6], v[7]));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at + i < end) st(dst, i, v[i]);
            }
        };
        store(g, row_lo, base_lo, 0);
        store(g + 8, row_hi, base_hi, 2);
        col = next_col, end = next_end, part = next_part;
#pragma unroll
        for (int i = 0; i < 8; ++i) base_lo[i] = next_lo[i], base_hi[i] = next_hi[i];
    }
}

template <typename TO>
int go(const Args& p, cudaStream_t s) {
    const int W = p.parts.n * p.rank;
    int groups = 0;
    for (int i = 0, first = 0; i < p.parts.n; first = p.parts.end[i++])
        groups += (p.parts.end[i] - first + GROUP - 1) / GROUP;
    if (p.parts.woven) groups = (p.N + GROUP - 1) / GROUP;
    // Several clusters share a tile's columns (each makes the low-rank rows for itself, A comes from L2) until
    // the grid holds two CTAs for every SM, or every warp has one group of columns.
    int share = 2 * sm_count() / (CLUSTER * p.max_tiles);
    if (share < 1) share = 1;
    const int most = (groups + CLUSTER * WARPS - 1) / (CLUSTER * WARPS);
    if (share > most) share = most;
    // rows of base and out by 16 bytes
    const size_t align = (size_t)p.base | (size_t)p.out | (size_t)(p.ld_base * sizeof(TO)) | (size_t)(p.ld_out * sizeof(TO));
    const int vec = (align & 15) == 0;
    const size_t smem = step_smem(W, p.K);
    static SmemLimit limit;
    cudaError_t e = limit.raise(adapter_step_kernel<TO>, smem);
    if (e == cudaSuccess)
        e = launch(adapter_step_kernel<TO>, dim3(share, p.max_tiles, CLUSTER), THREADS, smem, s, CLUSTER, p, groups, vec);
    return (int)e;
}

}  // namespace

namespace adapters {

// Whether the cluster form takes these: x, a and b by 16 bytes, ranks in sixteens.
bool step_takes(const Args& p) {
    const size_t align = (size_t)p.x | (size_t)p.a | (size_t)p.b | (size_t)(p.ld_x * 2) | (size_t)(p.lda * 2);
    return p.tile == TILE && (align & 15) == 0 && p.K % 8 == 0 && p.rank % 16 == 0 && p.max_tiles <= 65535 &&
           step_smem(p.parts.n * p.rank, p.K) <= 220 * 1024;
}

int step_form(const Args& p, int dt_out, cudaStream_t s) {
    return dt_out == RFX_DT_F32 ? go<float>(p, s) : go<__nv_bfloat16>(p, s);
}

}  // namespace adapters
