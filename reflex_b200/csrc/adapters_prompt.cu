// The adapters of prompts: tiles of up to 128 rows of one adapter, bfloat16, two launches.
//
//  * low: v = A x, 128 rows by all rank rows of all parts, on tcgen05 with 32-bit sums in tensor memory.  A's rows
//    come by TMA, and so do the tile's where they follow one another (a prompt's); other tiles (where two prompts
//    of one adapter meet, decoding rows by the hundred) are brought by four warps with 16-byte asynchronous copies
//    straight into the operand's swizzled layout.  K goes in up to eight pieces while that fills the GPU, a tile's
//    pieces are a cluster, and their sums meet in distributed shared memory, in order.  v goes to memory in
//    three bfloat16 parts (24 bits; large ranks of a bfloat16 result: two, see splits_of).  x is read once, A once a tile
//    from the L2 cache.  8,192 rows by 4,096, three parts of rank 64: 30 us where x alone would take 10; 2,047 rows by
//    12,288, rank 32: 17 us where prompts fill their tiles, 25 where they do not (x alone: 8).  What a block does once
//    bounds it, the barriers, the pieces' meeting and the parts' stores, beside A's way out of the cache.
//  * up: out = base + scale B v, 128 rows by up to 4,096 of one part's columns.  v comes by TMA as the operand that it
//    is, B's columns follow by asynchronous copies, the products go to one of two accumulators in tensor
//    memory, and sixteen warps add them to base's rows, of which several groups of columns are always on their way.
//    Base and out move in whole sectors, once: memory bounds it (8,192 rows by 6,144 columns: 53 us in bfloat16, 201 MB,
//    105 us in 32 bits, 403 MB: 3.8 TB/s, the first and the last columns of a block included, when it only reads or only
//    writes).
#include <cooperative_groups.h>

#include "adapters.cuh"
#include "attn_mma.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace cg = cooperative_groups;

namespace {

using namespace rfx;
using namespace adapters;
using namespace sm100;

constexpr int TILE = 128, BK = 64, LOW_THREADS = 384, MAX_STAGES = 8, MAX_W = 512, CHUNK = 256, MAX_PIECES = 8;
constexpr int MAX_SUMS = 4;  // accumulators that take turns
constexpr int X_BYTES = TILE * BK * 2;

// Stages, of `subs` blocks of 64 along K, that each of `pieces` takes.
__host__ __device__ inline int piece_stages(int K, int subs, int pieces) {
    const int all = (K + subs * BK - 1) / (subs * BK);
    return (all + pieces - 1) / pieces;
}

// Shared memory by its own addresses: through generic ones a load takes several times as long, and the compiler orders
// it with the stores to memory around it.
__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}

// Four numbers in two or three bfloat16 parts, which follow one another by `apart` elements.
__device__ __forceinline__ void store_parts(__nv_bfloat16* dst, size_t apart, int splits, float4 v) {
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        if (s == splits) break;
        const uint2 h = {attn::pack_bf16(v.x, v.y), attn::pack_bf16(v.z, v.w)};
        *reinterpret_cast<uint2*>(dst + s * apart) = h;
        v.x -= __uint_as_float(h.x << 16), v.y -= __uint_as_float(h.x & 0xffff0000u);
        v.z -= __uint_as_float(h.y << 16), v.w -= __uint_as_float(h.y & 0xffff0000u);
    }
}

__global__ void __launch_bounds__(LOW_THREADS)
adapter_low_tc_kernel(const Args p, const __grid_constant__ CUtensorMap map_a,
                      const __grid_constant__ CUtensorMap map_x, int box, int subs, int stages, int splits,
                      uint32_t tmem_cols, int turns, int* __restrict__ err) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], done_bar;
    __shared__ uint32_t tmem_base;
    __shared__ int rows[TILE];
    uint8_t* stage0 = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int W = p.parts.n * p.rank, stage_bytes = subs * (X_BYTES + W * BK * 2);
    pdl_wait();
    const Tile t = load_tile(p.tiles, blockIdx.x);
    if (t.adapter < 0 || t.adapter >= p.n) return;
    if (p.rank_of(t.adapter) == 0) return;  // (nothing reads its rows)
    // (a tile's pieces are a cluster; what returns here, returns as one)
    cg::cluster_group cluster = cg::this_cluster();
    const int pieces = cluster.num_blocks(), piece = cluster.block_rank();
    const int step = subs * BK, per = piece_stages(p.K, subs, pieces), kb0 = piece * per;
    const int nkb = min((p.K + step - 1) / step, kb0 + per) - kb0;  // (one at least)
    if (tid < TILE) rows[tid] = p.order[t.place + min(tid, t.count - 1)];
    const int row0 = p.order[t.place];
    const bool run = p.order[t.place + t.count - 1] - row0 == t.count - 1;  // (in order within a tile)
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full_bar[s], run ? 1 : TILE + 1);  // the bytes that TMA brings, and the threads that bring x
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&done_bar, 1);
        fence_barrier_init();
        prefetch_tensormap(&map_a);
        prefetch_tensormap(&map_x);
    }
    if (warp == 4) {
        tmem_alloc(&tmem_base, tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_launch_dependents();  // (not before tensor memory is this block's: the next kernel's blocks would take it)
    const uint32_t tmem = tmem_base, apart = tmem_cols / turns;  // `turns` accumulators, a stage each in turn
    if (warp < 4) {
        auto bring = [&](int s, int k) {  // A's rows of all parts, and the tile's where they follow one another
            uint8_t *dst = stage0 + (size_t)s * stage_bytes, *a = dst + subs * X_BYTES;
            mbar_expect_tx(&full_bar[s], (uint32_t)(subs * (W * BK * 2 + (run ? X_BYTES : 0))));
            for (int b = 0; b < subs; ++b, k += BK, dst += X_BYTES) {
                if (run) {
                    tma_load_2d(dst, &map_x, &full_bar[s], k, row0);
                    tma_load_2d(dst + X_BYTES / 2, &map_x, &full_bar[s], k, row0 + TILE / 2);
                }
                for (int w = 0; w < W; w += box, a += box * 128) tma_load_2d(a, &map_a, &full_bar[s], k, t.adapter * W + w);
            }
        };
        int s = 0, ph = 1;
        if (run) {
            if (warp == 0 && elect_one()) {
                for (int i = 0; i < nkb; ++i) {
                    if (i >= stages && !mbar_wait(&empty_bar[s], ph)) {
                        atomicExch(err, 61);
                        break;
                    }
                    bring(s, (kb0 + i) * step);
                    if (++s == stages) s = 0, ph ^= 1;
                }
            }
        } else {
            // thread: 16-byte unit u of the rows r0, r0 + 16, ...; a row's 128 bytes swizzled by its place among eight
            const int u = tid & 7, r0 = tid >> 3;
            const __nv_bfloat16* x = (const __nv_bfloat16*)p.x;
            for (int i = 0; i < nkb; ++i) {
                if (i >= stages && !mbar_wait(&empty_bar[s], ph)) {
                    atomicExch(err, 61);
                    break;
                }
                uint8_t* dst = stage0 + (size_t)s * stage_bytes;
                for (int b = 0; b < subs; ++b, dst += X_BYTES) {
                    const int k = (kb0 + i) * step + b * BK + u * 8;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int r = r0 + 16 * j;
                        const __nv_bfloat16* src = x + (size_t)rows[r] * p.ld_x + k;
                        attn::cp_async_16(dst + r * 128 + ((u ^ (r & 7)) << 4), k < p.K ? src : x, k < p.K);
                    }
                }
                // this thread's arrival follows its copies
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full_bar[s])) : "memory");
                if (tid == 0) bring(s, (kb0 + i) * step);
                if (++s == stages) s = 0, ph ^= 1;
            }
            attn::cp_async_wait<0>();
        }
        if (!mbar_wait(&done_bar, 0)) {
            atomicExch(err, 62);
            mbar_wait(&done_bar, 0);  // as long again for what is still being multiplied
        }
        tc_fence_after_sync();
        __syncwarp();
    } else if (warp == 4) {
        if (elect_one()) {
            // (one thread's instructions follow one another: what can be made ahead of the loop is)
            const uint64_t desc0 = umma_desc_k_sw128(smem_u32(stage0));
            const uint32_t stage_step = (uint32_t)stage_bytes >> 4;
            const uint32_t idesc = umma_idesc_bf16(TILE, min(256, W)), idesc2 = umma_idesc_bf16(TILE, max(16, W - 256));
            uint64_t dx = desc0;
            int s = 0, ph = 0, turn = 0;
            for (int i = 0; i < nkb; ++i) {
                if (!mbar_wait(&full_bar[s], ph)) {
                    atomicExch(err, 63);
                    // nothing more is begun; the stages that may still be on their way get as long again each
                    for (int j = i; j < min(nkb, i + stages); ++j) mbar_wait(&full_bar[j % stages], j / stages & 1);
                    break;
                }
                // rows brought by threads were written by the generic proxy; the tensor cores read by the asynchronous one
                if (!run) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_after_sync();
                const uint32_t d = tmem + turn * apart;
                uint32_t more = i >= turns;
                if (++turn == turns) turn = 0;
                for (int b = 0; b < subs; ++b) {
                    const uint64_t db = dx + b * (X_BYTES / 16), da = dx + subs * (X_BYTES / 16) + b * (W * 8);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k) {
                        umma_bf16(d, db + 2 * k, da + 2 * k, idesc, more);
                        if (W > 256) umma_bf16(d + 256, db + 2 * k, da + 256 * 8 + 2 * k, idesc2, more);
                        more = 1;
                    }
                }
                umma_commit(&empty_bar[s]);
                dx += stage_step;
                if (++s == stages) s = 0, ph ^= 1, dx = desc0;
            }
            umma_commit(&done_bar);  // (after a wait that ran out too: for the products before it)
        }
        __syncwarp();
    }
    // ---- the sums: each CTA of the cluster gets a share of the rows from all pieces (its stages are free by then), adds
    // them in order and stores them in their bfloat16 parts
    float* sums = reinterpret_cast<float*>(stage0);  // [piece][share][LD]
    __nv_bfloat16* low = reinterpret_cast<__nv_bfloat16*>(p.low);
    const int share = (TILE + pieces - 1) / pieces, r0 = piece * share, r1 = min(t.count, r0 + share);
    for (int c0 = 0; c0 < W; c0 += CHUNK) {
        const int wide = min(CHUNK, W - c0), LD = wide + 4;
        if (pieces > 1) cluster.sync();
        else __syncthreads();
        const int row = warp * 32 + lane, owner = row / share;
        if (warp < 4) {
            float* dst = pieces > 1 ? cluster.map_shared_rank(sums, owner) : sums;
            dst += (piece * share + row - owner * share) * LD;
            for (int c = 0; c < wide; c += 16) {
                float v[16];
                tmem_ld_16(tmem + ((uint32_t)(warp * 32) << 16) + c0 + c, v);
                for (int q = 1; q < min(turns, nkb); ++q) {
                    float u[16];
                    tmem_ld_16(tmem + ((uint32_t)(warp * 32) << 16) + q * apart + c0 + c, u);
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] += u[j];
                }
                if (row < t.count)
#pragma unroll
                    for (int j = 0; j < 16; j += 4) store4(dst + c + j, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
            }
        }
        if (pieces > 1) cluster.sync();
        else __syncthreads();
        // (twelve warps and a short loop: code that runs once a block costs more than what it does)
        const uint32_t sums_at = smem_u32(sums), next = share * LD * 4;
        for (int c = lane * 4; c < wide; c += 128)
#pragma unroll 1
            for (int r = warp; r < r1 - r0; r += LOW_THREADS / 32) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int q = 0; q < pieces; ++q) {
                    const uint4 a = lds16(sums_at + q * next + (r * LD + c) * 4);
                    v.x += __uint_as_float(a.x), v.y += __uint_as_float(a.y);
                    v.z += __uint_as_float(a.z), v.w += __uint_as_float(a.w);
                }
                store_parts(low + ((size_t)t.place + r0 + r) * W + c0 + c, (size_t)p.R * W, splits, v);
            }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, tmem_cols);
    }
}

// ---- out = base + scale B v ------------------------------------------------------------------------------
constexpr int UP_WARPS = 16, UP_THREADS = (UP_WARPS + 3) * 32, UP_STAGES = 2, GROUP = 32, STRIDE = 4 * GROUP;  // columns that a warp makes at a time

// Eight neighbouring elements of base as they lie.
template <typename TO> struct Eight;
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = load4(p), b = load4(p + 4); }
    __device__ __forceinline__ void load_shared(uint32_t at) {
        const uint4 u = lds16(at), v = lds16(at + 16);
        a = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
        b = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    }
    __device__ __forceinline__ void store(float* p) const { store4(p, a), store4(p + 4, b); }
    __device__ __forceinline__ float get(int i) const {
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        return v[i];
    }
};
template <> struct Eight<__nv_bfloat16> {
    uint4 a;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void load_shared(uint32_t at) { a = lds16(at); }
    __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = a; }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t v[4] = {a.x, a.y, a.z, a.w};
        return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
    }
};
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    store4(p, make_float4(v[0], v[1], v[2], v[3]));
    store4(p + 4, make_float4(v[4], v[5], v[6], v[7]));
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 u = {attn::pack_bf16(v[0], v[1]), attn::pack_bf16(v[2], v[3]), attn::pack_bf16(v[4], v[5]),
               attn::pack_bf16(v[6], v[7])};
    *reinterpret_cast<uint4*>(p) = u;
}

// SPLITS bfloat16 parts of v; a block: 128 rows by `span` turns of `cols` (128 or 64) columns of one part (woven: of
// both).  Warps 0 to 15 make the sums, 32 rows by every fourth 32 columns each; warp 16 issues the products, 17 and 18
// bring B.  AHEAD groups of base a warp are on their way or in use, 128 KB where there is room: an SM that reads
// and writes at its share of the memory's rate waits 3 to 4 us for a load, and with 64 KB on their way (two blocks
// of four such warps) the kernel took 58 us where one of sixteen took 51 us for 8,192 rows by 6,144 columns (v in two
// parts).  B's columns lie in the operand, and so in tensor memory, in an order that leaves a lane of the accumulator layout
// with eight neighbours of a row: of a group of 32, column 4 n + j is number 8 j + n (woven: even j in the first
// half of the turn's columns, odd j in the second, each half a product with its own part of v).
template <typename TO, int SPLITS, bool WOVEN, int AHEAD>
__global__ void __launch_bounds__(UP_THREADS, 1)
adapter_up_tc_kernel(const Args p, const __grid_constant__ CUtensorMap map_v, int span, int cols, int vec,
                     int* __restrict__ err) {
    constexpr int PARTS = WOVEN ? 2 : 1, stages = UP_STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t b_full[UP_STAGES], b_empty[UP_STAGES], acc_full[2], acc_empty[2], v_full;
    __shared__ uint32_t tmem_base;
    __shared__ int rows[TILE];
    const int kb = (p.rank + BK - 1) / BK;  // blocks of 64 along the rank
    uint8_t* vs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* bs = vs + SPLITS * PARTS * kb * X_BYTES;  // v: [SPLITS][PARTS][kb] blocks of 128 rows; B: [stages][kb]
    uint8_t* ys = bs + (size_t)stages * kb * cols * 128;  // base, a lane's own pieces: [warp][ahead][4 rows][lane]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_wait();
    const Tile tile = load_tile(p.tiles, blockIdx.x);
    if (tile.adapter < 0) return;
    const bool none = tile.adapter >= p.n;
    if (none && p.out == p.base) return;
    if (tid < TILE) rows[tid] = p.order[tile.place + min(tid, tile.count - 1)];
    const int rank = none ? 0 : p.rank_of(tile.adapter), steps = (rank + 15) / 16;
    // this block's part and columns
    int part = 0, first = 0, block = blockIdx.y;
    if (!WOVEN)
        while (part + 1 < p.parts.n) {
            const int n = ((p.parts.end[part] - first + cols - 1) / cols + span - 1) / span;
            if (block < n) break;
            block -= n;
            first = p.parts.end[part++];
        }
    const int end = WOVEN ? p.N : p.parts.end[part];
    first += block * span * cols;
    const int turns = min(span, (end - first + cols - 1) / cols);
    if (steps && tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&b_full[s], 64);
            mbar_init(&b_empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&acc_full[s], 1);
            mbar_init(&acc_empty[s], 4 * (cols / GROUP));
        }
        mbar_init(&v_full, 1);
        fence_barrier_init();
        // v lies by place: a tile's rows follow one another, and what is beyond them is multiplied and dropped
        const int blocks = (steps + 3) / 4;
        mbar_expect_tx(&v_full, SPLITS * PARTS * blocks * X_BYTES);
        for (int s = 0; s < SPLITS; ++s)
            for (int q = 0; q < PARTS; ++q)
                for (int k = 0; k < blocks; ++k)
                    tma_load_2d(vs + ((s * PARTS + q) * kb + k) * X_BYTES, &map_v, &v_full,
                                (WOVEN ? q : part) * p.rank + k * BK, s * p.R + tile.place);
    }
    if (steps && warp == UP_WARPS) {
        tmem_alloc(&tmem_base, 256);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_launch_dependents();  // (not before tensor memory is this block's)
    if (warp < UP_WARPS) {
        const int m0 = (warp & 3) * 32, quarter = warp >> 2;
        // this lane's pieces: columns 8 t .. of rows m0 + g, + 8, + 16, + 24, from its warp's first group on
        const int col0 = first + quarter * GROUP + 8 * t;
        const TO* base[4];
        TO* out[4];
        int rows_on = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = m0 + g + 8 * i;
            if (r < tile.count) rows_on |= 1 << i;
            base[i] = (const TO*)p.base + (size_t)rows[r] * p.ld_base + col0;
            out[i] = (TO*)p.out + (size_t)rows[r] * p.ld_out + col0;
        }
        // its groups, and whether a piece of one can be moved whole
        const int groups = (min(turns * cols, end - first) - quarter * GROUP + STRIDE - 1) / STRIDE;
        const int wholes = vec && (first & 7) == 0 ? (end - col0 - 8 + STRIDE) / STRIDE : 0;
        if (steps == 0) {  // rows without an adapter (or with one of rank 0) go over as they are
            for (int q = 0; q < groups; ++q) {
                Eight<TO> v[4];
                if (q < wholes)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (rows_on >> j & 1) v[j].load(base[j] + q * STRIDE);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!(rows_on >> j & 1)) continue;
                    if (q < wholes) v[j].store(out[j] + q * STRIDE);
                    else
                        for (int i = q * STRIDE; i < q * STRIDE + 8 && col0 + i < end; ++i) out[j][i] = base[j][i];
                }
            }
            return;
        }
        constexpr int PIECE = 8 * sizeof(TO), SLOT = 4 * 32 * PIECE;  // bytes of eight neighbours, of a warp's group
        const uint32_t mine = smem_u32(ys) + warp * AHEAD * SLOT + lane * PIECE;
        auto bring_base = [&](int q) {
            if (q < wholes && q < groups) {
                const uint32_t dst = mine + (q & (AHEAD - 1)) * SLOT;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (rows_on >> j & 1)
#pragma unroll
                        for (int c = 0; c < PIECE; c += 16)
                            asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst + j * 32 * PIECE + c),
                                         "l"(reinterpret_cast<const uint8_t*>(base[j] + q * STRIDE) + c)
                                         : "memory");
            }
            attn::cp_async_commit();
        };
        const uint32_t tmem = tmem_base + ((uint32_t)m0 << 16);
        const float scale = p.scale[tile.adapter];
        const int per = cols == 128 ? 2 : 1;  // (the logarithm of) the groups of a turn
        bool ok = true;
        for (int q = 0; q < AHEAD - 1; ++q) bring_base(q);
        for (int q = 0; q < groups; ++q) {
            bring_base(q + AHEAD - 1);
            const int i = (q * 4 + quarter) >> per, h = quarter & (cols / GROUP - 1);  // the turn, and the group in it
            ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[i & 1], i >> 1 & 1));
            tc_fence_after_sync();
            __syncwarp();
            uint32_t acc[2][16];  // 16 rows each: [tile of 8 columns][row g: two columns, row g + 8: two]
            const uint32_t at_t = tmem + (i & 1) * cols + h * (WOVEN ? 16 : 32);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if (WOVEN) {
                    tmem_ld_frag2_nowait(at_t + ((uint32_t)m << 20), acc[m]);
                    tmem_ld_frag2_nowait(at_t + cols / 2 + ((uint32_t)m << 20), acc[m] + 8);
                } else {
                    tmem_ld_frag4_nowait(at_t + ((uint32_t)m << 20), acc[m]);
                }
            }
            attn::cp_async_wait<AHEAD - 1>();  // a lane reads what it brought itself
            Eight<TO> y[4];                    // (what no copy brought is not used)
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j].load_shared(mine + (q & (AHEAD - 1)) * SLOT + j * 32 * PIECE);
            tmem_ld_wait_16(acc[0]);
            tmem_loaded_16(acc[1]);
            tc_fence_before_sync();  // the group's sums are read
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[i & 1]);
            if (!ok) break;
            const bool fast = q < wholes;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!(rows_on >> j & 1)) continue;
                float d[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    // column 4 n + jj of the group, n = 2 t or 2 t + 1: tile jj (woven: 0, 2, 1, 3 lie in order)
                    const int jj = c & 3, at_acc = WOVEN ? (jj & 1) * 2 + (jj >> 1) : jj;
                    d[c] = __uint_as_float(acc[j >> 1][at_acc * 4 + (j & 1) * 2 + (c >> 2)]);
                }
                const int at = q * STRIDE;
                if (fast) {
                    float o[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) o[c] = fmaf(scale, d[c], y[j].get(c));
                    store8(out[j] + at, o);
                } else {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (col0 + at + c < end) st(out[j], at + c, fmaf(scale, d[c], ld(base[j], at + c)));
                }
            }
        }
        if (!ok) atomicExch(err, 64);
        attn::cp_async_wait<0>();
        tc_fence_before_sync();
    } else if (warp == UP_WARPS) {
        if (steps && elect_one()) {
            const uint32_t idesc = umma_idesc_bf16(TILE, cols / PARTS), b_step = (uint32_t)(kb * cols * 8);
            const uint64_t desc_v = umma_desc_k_sw128(smem_u32(vs)), desc_b = umma_desc_k_sw128(smem_u32(bs));
            int s = 0, ph = 0;
            const bool ok = mbar_wait(&v_full, 0);
            if (!ok) {
                atomicExch(err, 67);
                mbar_wait(&v_full, 0);  // as long again for the copies on their way
            }
            for (int i = 0; i < turns && ok; ++i) {
                if ((i >= 2 && !mbar_wait(&acc_empty[i & 1], (i >> 1 & 1) ^ 1)) || !mbar_wait(&b_full[s], ph)) {
                    atomicExch(err, 65);
                    // nothing more is begun; the products on their way get as long again
                    for (int j = max(i - 2, 0); j < i; ++j) mbar_wait(&acc_full[j & 1], j >> 1 & 1);
                    break;
                }
                // B's columns were written by the generic proxy; the tensor cores read by the asynchronous one
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_after_sync();
                const uint64_t db0 = desc_b + s * b_step;
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    const uint32_t d = tmem_base + (i & 1) * cols + q * (cols / 2);
                    uint32_t more = 0;
#pragma unroll
                    for (int sp = SPLITS - 1; sp >= 0; --sp) {  // the smallest first: what is cut off is small as well
                        uint64_t dv = desc_v + (uint32_t)((sp * PARTS + q) * kb) * (X_BYTES / 16), db = db0 + q * (cols / 2) * 8;
                        for (int k = 0; k < steps; ++k) {
                            umma_bf16(d, dv, db, idesc, more);
                            more = 1;
                            // 16 further along the rank; the fourth time into the next block of 64
                            const bool over = (k & 3) == 3;
                            dv += over ? X_BYTES / 16 - 6 : 2;
                            db += over ? cols * 8 - 6 : 2;
                        }
                    }
                }
                umma_commit(&b_empty[s]);
                umma_commit(&acc_full[i & 1]);
                if (++s == stages) s = 0, ph ^= 1;
            }
        }
        __syncwarp();
        tc_fence_before_sync();
    } else if (steps) {
        // four threads a column, each every fourth 16 bytes of it
        const __nv_bfloat16* b = (const __nv_bfloat16*)p.b + (size_t)tile.adapter * p.N * p.rank + (lane & 3) * 8;
        const int c0 = (tid - (UP_WARPS + 1) * 32) >> 2;
        int s = 0, ph = 1;
        for (int i = 0; i < turns; ++i) {
            if (i >= stages && !mbar_wait(&b_empty[s], ph)) {
                atomicExch(err, 66);
                break;
            }
            uint8_t* dst = bs + s * kb * cols * 128;
#pragma unroll 2
            for (int c = c0; c < cols; c += 16) {
                const int n = (c & (GROUP - 1)) >> 2, j = c & 3;
                const int d = WOVEN ? (j & 1) * (cols / 2) + (c >> 5) * 16 + (j >> 1) * 8 + n : (c & ~(GROUP - 1)) + j * 8 + n;
                const __nv_bfloat16* src = b + (size_t)min(first + i * cols + c, end - 1) * p.rank;
                for (int u = lane & 3; u < steps * 2; u += 4)
                    attn::cp_async_16(dst + ((u >> 3) * cols + d) * 128 + (((u ^ d) & 7) << 4), src + (u & ~3) * 8, true);
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&b_full[s])) : "memory");
            if (++s == stages) s = 0, ph ^= 1;
        }
        attn::cp_async_wait<0>();
    }
    if (steps == 0) return;
    __syncthreads();
    if (warp == UP_WARPS) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 256);
    }
}

// Blocks of 64 along K a stage: two where at least two such stages have room, for a stage costs the thread that
// issues its products about as much as their issue (2,047 rows by 12,288, rank 32: 28.5 us with one, 25 with two).
int subs_of(int W) { return 2 * 2 * (X_BYTES + W * BK * 2) <= 200 * 1024 ? 2 : 1; }

// Pieces of K: the waves of clusters times the stages that each block takes and what its beginning and end cost, at
// their least; as few as give each a stage.
int pieces_of(int K, int subs, int max_tiles) {
    const int all = (K + subs * BK - 1) / (subs * BK), sms = sm_count();
    int best = 1;
    long long least = 0;
    for (int n = 1; n <= MAX_PIECES && n <= (all + 1) / 2; ++n) {
        const int at_once = n <= 2 ? sms / n : 8 * (18 / n);  // clusters: eight groups of 18 SMs or a few more
        const long long cost = (long long)(max_tiles + at_once - 1) / at_once * ((all + n - 1) / n * subs + 10);
        if (n == 1 || cost < least) best = n, least = cost;
    }
    const int per = piece_stages(K, subs, best);
    return (all + per - 1) / per;
}

// Blocks of 64 along the rank that v takes in shared memory (16 KB each), all its bfloat16 parts together: beside
// them B and base's groups find room for eight of a bfloat16 result, six of a 32-bit one.
constexpr size_t MOST_SMEM = 226 * 1024;
int v_blocks(const Args& p, int splits) { return splits * (p.parts.woven ? 2 : 1) * ((p.rank + BK - 1) / BK); }
// The parts in which v goes from one product to the other: three (24 bits) wherever they find room, ranks to 128 (woven:
// to 64); a bfloat16 result of larger ranks has two (16 bits: v is off by 2^-17 of itself at most, 2^-9 of the result's
// own rounding).
int splits_of(const Args& p, int dt_out) { return dt_out == RFX_DT_F32 || v_blocks(p, 3) <= 6 ? 3 : 2; }

template <typename TO, int SPLITS, bool WOVEN>
int up(const Args& p, int* err, cudaStream_t s) {
    CUtensorMap map_v;
    const int W = p.parts.n * p.rank;
    if (!rfx::tma::make_map_rows64(&map_v, p.low, (long long)SPLITS * p.R, W, TILE)) return RFX_ERR_UNSUPPORTED;
    const int kb = (p.rank + BK - 1) / BK, cols = kb > 2 ? 64 : 128, parts = WOVEN ? 1 : p.parts.n;
    int turns[MAX_PARTS];
    for (int i = 0, first = 0; i < parts; first = p.parts.end[i++])
        turns[i] = ((WOVEN ? p.N : p.parts.end[i]) - first + cols - 1) / cols;
    // Turns a block: the waves of blocks, one an SM and part by part as the grid has them, each wave at its longest
    // block's turns and about three for a block's beginning, at their least.
    int span = 1;
    long long least = -1;
    for (int n : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        long long cost = 0, ctas = 0, wave = -1;
        int longest = 0;
        for (int i = 0; i < parts; ++i)
            for (int left = turns[i]; left > 0; left -= n, ctas += p.max_tiles) {
                const int here = left < n ? left : n;
                const long long from = ctas / sm_count(), to = (ctas + p.max_tiles - 1) / sm_count();
                if (from == wave) {  // the wave that the block before began
                    if (here > longest) cost += here - longest, longest = here;
                }
                if (to > wave) cost += (to - (from > wave ? from - 1 : wave)) * (here + 3), longest = here, wave = to;
            }
        if (least < 0 || cost < least) span = n, least = cost;
    }
    int blocks = 0;
    for (int i = 0; i < parts; ++i) blocks += (turns[i] + span - 1) / span;
    const size_t v = (size_t)v_blocks(p, SPLITS) * X_BYTES, b = (size_t)kb * cols * 128;
    const size_t group = (size_t)UP_WARPS * 4 * 32 * 8 * sizeof(TO), rest = v + UP_STAGES * b + 1024;
    int ahead = 1;  // groups of base a warp: 128 KB at most
    while (ahead * group < 128 * 1024 && rest + 2 * ahead * group <= MOST_SMEM) ahead *= 2;
    const size_t smem = rest + ahead * group;
    const size_t align = (size_t)p.base | (size_t)p.out | (size_t)(p.ld_base * sizeof(TO)) | (size_t)(p.ld_out * sizeof(TO));
    static SmemLimit limits[3];
    auto go = [&](auto kernel, SmemLimit& limit) {
        cudaError_t e = limit.raise(kernel, smem);
        if (e == cudaSuccess)
            e = launch(kernel, dim3(p.max_tiles, blocks), UP_THREADS, smem, s, 1, p, map_v, span, cols,
                       (align & 15) == 0 ? 1 : 0, err);
        return (int)e;
    };
    if (ahead == 1) return go(adapter_up_tc_kernel<TO, SPLITS, WOVEN, 1>, limits[0]);
    if (ahead == 2) return go(adapter_up_tc_kernel<TO, SPLITS, WOVEN, 2>, limits[1]);
    return go(adapter_up_tc_kernel<TO, SPLITS, WOVEN, 4>, limits[2]);
}

}  // namespace

namespace adapters {

// Whether the tcgen05 form takes these: x, a and b by 16 bytes, ranks in sixteens, the rank rows in tensor memory and
// the low-rank rows in shared memory.
bool prompt_takes(const Args& p, int dt_out) {
    const size_t align = (size_t)p.x | (size_t)p.a | (size_t)p.b | (size_t)(p.ld_x * 2) | (size_t)(p.lda * 2);
    const int splits = splits_of(p, dt_out);
    return p.tile == TILE && (align & 15) == 0 && p.K % 8 == 0 && p.K >= BK && p.lda == p.K && p.rank % 16 == 0 &&
           p.parts.n * p.rank <= MAX_W && v_blocks(p, splits) <= (splits == 3 ? 6 : 8) && p.N <= 65535 * 64;
}

long long prompt_low_floats(int R, int W) { return ((long long)3 * R * W + 1) / 2; }  // three bfloat16 parts at most

int prompt_form(const Args& p, int dt_out, int* err, cudaStream_t s) {
    const int W = p.parts.n * p.rank, subs = subs_of(W), pieces = pieces_of(p.K, subs, p.max_tiles);
    CUtensorMap map_a, map_x;
    const int box = W <= 256 ? W : 16;  // rows of A a copy brings (they come 53 cycles apart)
    if (!rfx::tma::make_map_rows64(&map_a, p.a, (long long)p.n * W, p.K, box) ||
        !rfx::tma::make_map_rows64(&map_x, p.x, p.R, p.K, TILE / 2, p.ld_x))
        return RFX_ERR_UNSUPPORTED;
    const int stage = subs * (X_BYTES + W * BK * 2);
    int stages = 200 * 1024 / stage;  // one block an SM: what is on its way hides the memory's latency
    if (stages < 2) stages = 2;
    if (stages > 6) stages = 6;
    uint32_t cols = 32;
    while ((int)cols < W) cols *= 2;
    // A tensor core cuts sums off, always towards zero: accumulators that take turns keep the chains short
    const int turns = (int)min((uint32_t)MAX_SUMS, 512 / cols);
    const size_t smem = (size_t)stages * stage + 1024;
    static SmemLimit limit;
    cudaError_t e = limit.raise(adapter_low_tc_kernel, smem);
    if (e != cudaSuccess) return (int)e;
    const int splits = splits_of(p, dt_out);
    e = launch(adapter_low_tc_kernel, dim3(p.max_tiles, 1, pieces), LOW_THREADS, smem, s, pieces, p, map_a, map_x, box, subs, stages,
               splits, cols * turns, turns, err);
    if (e != cudaSuccess) return (int)e;
    if (dt_out == RFX_DT_F32) return p.parts.woven ? up<float, 3, true>(p, err, s) : up<float, 3, false>(p, err, s);
    if (splits == 3) return p.parts.woven ? up<__nv_bfloat16, 3, true>(p, err, s) : up<__nv_bfloat16, 3, false>(p, err, s);
    return p.parts.woven ? up<__nv_bfloat16, 2, true>(p, err, s) : up<__nv_bfloat16, 2, false>(p, err, s);
}

}  // namespace adapters
