// The adapters of a step's requests, a row or a few each: tiles of at most 16 rows, bfloat16, one launch.
//
// A thread-block cluster takes a tile and both products.  Each of its eight CTAs multiplies the tile's rows
// with A over an eighth of K on the tensor cores (m16n8k16: 16 rows, 8 rank rows), a warp every eighth 8 rank rows;
// the partial sums meet in distributed shared memory, in rank order; then each CTA multiplies the low-rank rows
// with its share of B's columns and adds the base.  Nothing but the result goes back to memory, and there is
// one launch where two would have to follow one another.
//
// It is latency that counts, the chain tile -> row -> x and A -> cluster -> B, and then the adapters' bytes (an
// adapter of rank 16 beside 4,096 x 6,144: 0.6 MB, which one row takes 6.5 us for; 64 rows over 32 adapters of
// rank 64, 33 MB with base and out: 27 us).  So a warp
// has 6 KB of A on their way, in a ring of shared memory of which every lane reads what it brought itself (no
// barrier), k permuted alike on both sides so that a lane's elements lie side by side; B's columns are asked
// for ahead, and a warp's first ones and their base are loaded before the cluster meets.
//
// The low-rank rows are kept in 32 bits and go into the second product as three bfloat16 parts (24 bits).
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
constexpr int RING = 3, BATCH = 4;          // a warp's batches of A under way, of 8 rank rows by 4 times 32 of K
constexpr int GROUP = 32;                   // columns a warp makes at a time
constexpr int AHEAD = 2;                    // steps of 16 along the rank whose B is loaded before the cluster meets

// (in whole batches of 128)
__host__ __device__ inline int k_slice(int K) { return ((K + CLUSTER - 1) / CLUSTER + 127) / 128 * 128; }
// the warps' pieces of A, the rows of x, the partial rows, and the three parts' bfloat16s
inline size_t step_smem(int W, int K) {
    return (size_t)WARPS * RING * BATCH * 512 + (size_t)TILE * (k_slice(K) + 8) * 2 + (size_t)TILE * W * 4 +
           (size_t)3 * TILE * (W + 8) * 2;
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

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

template <typename TO>
__global__ void __launch_bounds__(THREADS, 2) adapter_step_kernel(const Args p, int groups, int vec) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ int rows[TILE];
    cg::cluster_group cluster = cg::this_cluster();
    const int W = p.parts.n * p.rank, LDV = W + 8, slice = k_slice(p.K), LDX = slice + 8;
    uint8_t* ring = dynamic;                                                              // [WARPS][RING][BATCH][lane]
    __nv_bfloat16* xs = reinterpret_cast<__nv_bfloat16*>(ring + WARPS * RING * BATCH * 512);  // [TILE][LDX]
    float* part_v = reinterpret_cast<float*>(xs + TILE * LDX);                            // [TILE][W]
    __nv_bfloat16* vs = reinterpret_cast<__nv_bfloat16*>(part_v + TILE * W);              // [3][TILE][LDV]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_prologue();
    const Tile tile = load_tile(p.tiles, blockIdx.y);
    if (tile.adapter < 0) return;  // (the same for the whole cluster)
    const bool none = tile.adapter >= p.n;
    if (none && p.out == p.base) return;
    const int count = min(tile.count, TILE), c = cluster.block_rank();
    const int rank = none ? 0 : p.rank_of(tile.adapter);
    const int per = (rank + 7) / 8, steps = (rank + 15) / 16, tiles = per * p.parts.n;
    // ---- a warp's first pieces of A: tiles of 8 rank rows n = warp, warp + 8, ..., 128 of K at a time; a lane brings,
    // and reads, its own 16 bytes of each 32
    const int k0 = c * slice, k1 = min(p.K, k0 + slice), blocks = k0 < k1 ? (k1 - k0 + 31) / 32 : 0;
    const __nv_bfloat16* a = (const __nv_bfloat16*)p.a + (size_t)tile.adapter * W * p.lda;
    const uint32_t my_ring = attn::smem_u32(ring) + warp * RING * BATCH * 512 + lane * 16;
    int next_n = blocks ? warp : tiles, next_b = 0, next_slot = 0;
    auto bring = [&]() {
        if (next_n < tiles) {
            const int s = next_n / per, row = s * p.rank + (next_n - s * per) * 8 + g;
            const __nv_bfloat16* src = a + (size_t)row * p.lda + k0 + next_b * 32 + t * 8;
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int bytes = k0 + (next_b + j) * 32 + t * 8 < k1 ? 16 : 0;  // (zeros beyond)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(my_ring + (next_slot * BATCH + j) * 512),
                             "l"(bytes ? src + j * 32 : a), "r"(bytes)
                             : "memory");
            }
            if ((next_b += BATCH) >= blocks) next_b = 0, next_n += WARPS;
            if (++next_slot == RING) next_slot = 0;
        }
        attn::cp_async_commit();
    };
    for (int i = 0; i < RING - 1; ++i) bring();
    if (tid < TILE) rows[tid] = p.order[tile.place + min(tid, count - 1)];
    __syncthreads();
    // ---- x's rows over this CTA's slice of K
    if (!none) {
        const __nv_bfloat16* x = (const __nv_bfloat16*)p.x;
        const int padded = (blocks + BATCH - 1) / BATCH * BATCH * 32;
        for (int r = warp; r < count; r += WARPS)
            for (int k = lane * 8; k < padded; k += 256)
                attn::cp_async_16(xs + r * LDX + k, k0 + k < k1 ? x + (size_t)rows[r] * p.ld_x + k0 + k : x, k0 + k < k1);
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
    auto load_b = [&](int col, int end, int s, int j) {  // step s of tile j: columns col + 4 n + j
        const int at = min(col + 4 * g + j, end - 1);
        return __ldg(reinterpret_cast<const uint2*>(b + (size_t)at * p.rank + s * 16 + t * 4));
    };
    const TO* base = (const TO*)p.base;
    TO* out = (TO*)p.out;
    auto load_base = [&](int col, int end, int r, float (&v)[8]) {
        const int at = col + 8 * t;
        if (r < count) {
            const TO* src = base + (size_t)rows[r] * p.ld_base + at;
            if (vec && at + 8 <= end && (at & 7) == 0) load8(src, v);
            else
                for (int i = 0; i < 8; ++i) v[i] = at + i < end ? ld(src, i) : 0.f;
        }
    };
    uint2 ahead[AHEAD][4];
    float base_lo[8], base_hi[8];
    int col = 0, end = 0, part = 0;
    const bool any = group < groups;
    if (any) {
        locate(group, col, end, part);
#pragma unroll
        for (int s = 0; s < AHEAD; ++s)
            if (s < steps)
#pragma unroll
                for (int j = 0; j < 4; ++j) ahead[s][j] = load_b(col, end, s, j);
        load_base(col, end, g, base_lo);
        load_base(col, end, g + 8, base_hi);
        // this warp's columns of B and of base are asked for, and come from L2 when their turn has come
        if (!none)
            for (int q = group; q < groups; q += stride) {
                int col_q, end_q, part_q;
                locate(q, col_q, end_q, part_q);
                const int n = min(GROUP, end_q - col_q) * p.rank;  // (one stretch of memory)
                for (int i = lane * 64; i < n; i += 32 * 64) prefetch_l2(b + (size_t)col_q * p.rank + i);
                if (q != group && lane < count) prefetch_l2(base + (size_t)rows[lane] * p.ld_base + col_q);
            }
    }

    if (!none) {
        // ---- the low-rank rows over this CTA's slice of K
        for (int i = tid; i < 3 * TILE * LDV / 2; i += THREADS) reinterpret_cast<uint32_t*>(vs)[i] = 0u;
        attn::cp_async_wait<0>();
        __syncthreads();  // x is there
        const uint32_t x_at = attn::smem_u32(xs) + (g * LDX + t * 8) * 2;
        int slot = 0;
        for (int n = warp; n < tiles; n += WARPS) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            for (int i = 0; i < blocks; i += BATCH) {
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
                    attn::mma_bf16(acc, f0, w[j].x, w[j].y);
                    attn::mma_bf16(acc, f1, w[j].z, w[j].w);
                }
            }
            store2(part_v + g * W + n * 8 + t * 2, acc[0], acc[1]);
            store2(part_v + (g + 8) * W + n * 8 + t * 2, acc[2], acc[3]);
        }
        attn::cp_async_wait<0>();
        cluster.sync();
        // ---- the cluster's sums, in three parts of bfloat16
        for (int i = tid; i < count * tiles * 8; i += THREADS) {
            const int r = i / (tiles * 8), n = i - r * tiles * 8;
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < CLUSTER; ++q) v += cluster.map_shared_rank(part_v, q)[r * W + n];
            const int s = n / (per * 8), at = r * LDV + s * p.rank + n - s * per * 8;
            const __nv_bfloat16 hi = __float2bfloat16_rn(v);
            const float rest = v - __bfloat162float(hi);
            const __nv_bfloat16 mid = __float2bfloat16_rn(rest);
            vs[at] = hi;
            vs[TILE * LDV + at] = mid;
            vs[2 * TILE * LDV + at] = __float2bfloat16_rn(rest - __bfloat162float(mid));
        }
        cluster.sync();  // no CTA leaves while another reads its sums
    }

    // ---- the columns
    const float scale = none ? 0.f : p.scale[tile.adapter];
    for (bool first = true; group < groups; group += stride, first = false) {
        if (!first) {
            locate(group, col, end, part);
            load_base(col, end, g, base_lo);
            load_base(col, end, g + 8, base_hi);
        }
        float acc[4][4] = {};
        for (int s0 = 0; s0 < steps; s0 += AHEAD) {
            if (!first || s0)
#pragma unroll
                for (int s = 0; s < AHEAD; ++s)
                    if (s0 + s < steps)
#pragma unroll
                        for (int j = 0; j < 4; ++j) ahead[s][j] = load_b(col, end, s0 + s, j);
#pragma unroll
            for (int s = 0; s < AHEAD; ++s)
                if (s0 + s < steps)
#pragma unroll
                    for (int q = 0; q < 3; ++q) {
                        const __nv_bfloat16* v = vs + q * TILE * LDV + (s0 + s) * 16 + t * 4;
                        auto frag = [&](int sp, uint32_t (&f)[4]) {
                            const uint2 lo = *reinterpret_cast<const uint2*>(v + g * LDV + sp * p.rank);
                            const uint2 hi = *reinterpret_cast<const uint2*>(v + (g + 8) * LDV + sp * p.rank);
                            f[0] = lo.x, f[1] = hi.x, f[2] = lo.y, f[3] = hi.y;
                        };
                        uint32_t f[4], odd[4];
                        frag(part, f);
                        if (p.parts.woven) frag(1, odd);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if ((j & 1) && p.parts.woven) attn::mma_bf16(acc[j], odd, ahead[s][j].x, ahead[s][j].y);
                            else attn::mma_bf16(acc[j], f, ahead[s][j].x, ahead[s][j].y);
                        }
                    }
        }
        auto store = [&](int r, const float (&y)[8], int h) {
            const int at = col + 8 * t;
            if (r >= count) return;
            TO* dst = out + (size_t)rows[r] * p.ld_out + at;
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
        store(g, base_lo, 0);
        store(g + 8, base_hi, 2);
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
    const size_t smem = step_smem(W, p.K);
    // rows of base and out by 16 bytes
    const size_t align = (size_t)p.base | (size_t)p.out | (size_t)(p.ld_base * sizeof(TO)) | (size_t)(p.ld_out * sizeof(TO));
    const int vec = (align & 15) == 0;
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
