// The adapters of prompts: tiles of up to 128 rows of one adapter, bfloat16, two launches.
//
//  * low: v = A x, 128 rows by all rank rows of all parts, on tcgen05 with 32-bit sums in tensor memory.  A's
//    rows come by TMA, and so do the tile's where they follow one another (a prompt's); other tiles (where two prompts of one adapter meet, decoding rows by the hundred) are brought by
//    four warps with 16-byte asynchronous copies straight into the operand's swizzled layout.  K goes in several
//    pieces side by side while that fills the GPU.  It reads x once, and memory bounds it.
//  * up: out = base + scale B v, 128 rows by up to 4,096 of one part's columns.  v is summed over the pieces, in
//    order, into two bfloat16 parts (16 bits: its error is 2^-9 of the result's rounding to bfloat16; three parts
//    for a 32-bit result) in shared memory; B's columns follow by asynchronous copies, the products go to one of two
//    accumulators in tensor memory, and four warps add them to base's rows, which are a group of columns ahead
//    in registers.  Base and out move in whole sectors, once: memory bounds it.
#include "adapters.cuh"
#include "attn_mma.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace {

using namespace rfx;
using namespace adapters;
using namespace sm100;

constexpr int TILE = 128, BK = 64, LOW_THREADS = 160, MAX_STAGES = 8, MAX_W = 512;
constexpr int X_BYTES = TILE * BK * 2;

// K blocks of 64 a piece takes
__host__ __device__ inline int piece_blocks(int K, int pieces) {
    const int blocks = (K + BK - 1) / BK;
    return (blocks + pieces - 1) / pieces;
}

__global__ void __launch_bounds__(LOW_THREADS)
adapter_low_tc_kernel(const Args p, const __grid_constant__ CUtensorMap map_a,
                      const __grid_constant__ CUtensorMap map_x, int box, int stages, int pieces, uint32_t tmem_cols,
                      int* __restrict__ err) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], done_bar;
    __shared__ uint32_t tmem_base;
    __shared__ int rows[TILE];
    uint8_t* stage0 = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int W = p.parts.n * p.rank, stage_bytes = X_BYTES + W * BK * 2;
    pdl_wait();
    const Tile t = load_tile(p.tiles, blockIdx.x);
    if (t.adapter < 0 || t.adapter >= p.n) return;
    const int per = piece_blocks(p.K, pieces), kb0 = blockIdx.y * per;
    const int nkb = min((p.K + BK - 1) / BK, kb0 + per) - kb0;
    if (nkb <= 0 || p.rank_of(t.adapter) == 0) return;  // (what nothing is left of is not read either)
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
    const uint32_t tmem = tmem_base;
    bool ok = true;
    if (warp < 4) {
        auto bring = [&](int s, int k) {  // A's rows of all parts, and the tile's where they follow one another
            uint8_t* dst = stage0 + (size_t)s * stage_bytes;
            mbar_expect_tx(&full_bar[s], (uint32_t)(W * BK * 2 + (run ? X_BYTES : 0)));
            if (run) {
                tma_load_2d(dst, &map_x, &full_bar[s], k, row0);
                tma_load_2d(dst + X_BYTES / 2, &map_x, &full_bar[s], k, row0 + TILE / 2);
            }
            for (int w = 0; w < W; w += box)
                tma_load_2d(dst + X_BYTES + w * 128, &map_a, &full_bar[s], k, t.adapter * W + w);
        };
        int s = 0, ph = 1;
        if (run) {
            if (warp == 0 && elect_one()) {
                for (int i = 0; i < nkb; ++i) {
                    if (i >= stages && !mbar_wait(&empty_bar[s], ph)) {
                        atomicExch(err, 61);
                        ok = false;
                        break;
                    }
                    bring(s, (kb0 + i) * BK);
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
                    ok = false;
                    break;
                }
                uint8_t* dst = stage0 + (size_t)s * stage_bytes;
                const int k = (kb0 + i) * BK;
                const bool in = k + u * 8 < p.K;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int r = r0 + 16 * j;
                    const __nv_bfloat16* src = x + (size_t)rows[r] * p.ld_x + k + u * 8;
                    attn::cp_async_16(dst + r * 128 + ((u ^ (r & 7)) << 4), in ? src : x, in);
                }
                // this thread's arrival follows its copies
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full_bar[s])) : "memory");
                if (tid == 0) bring(s, k);
                if (++s == stages) s = 0, ph ^= 1;
            }
            attn::cp_async_wait<0>();
        }
        // ---- the sums: a thread has a row; rows go out through shared memory (the stages are free), whole
        const bool have = mbar_wait(&done_bar, 0);
        if (!have) atomicExch(err, 62);
        ok = __all_sync(0xffffffffu, have && ok);
        tc_fence_after_sync();
        const uint32_t at = tmem + ((uint32_t)(warp * 32) << 16);
        constexpr int LD = 68;  // 64 columns at a time
        float* out = reinterpret_cast<float*>(stage0) + warp * 32 * LD;
        const int here = min(32, t.count - warp * 32);
        float* dst = p.low + ((size_t)blockIdx.y * p.R + t.place + warp * 32) * W;
        for (int c0 = 0; c0 < W && ok; c0 += 64) {
            const int wide = min(64, W - c0);
            for (int c = 0; c < wide; c += 16) {
                float v[16];
                tmem_ld_16(at + c0 + c, v);
#pragma unroll
                for (int j = 0; j < 16; j += 4)
                    store4(out + lane * LD + c + j, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
            }
            __syncwarp();
            const int c = (lane & 15) * 4;  // sixteen lanes a row
            if (c < wide)
#pragma unroll 4
                for (int r = lane >> 4; r < here; r += 2) store4(dst + (size_t)r * W + c0 + c, load4(out + r * LD + c));
            __syncwarp();
        }
        tc_fence_before_sync();
    } else {
        if (elect_one()) {
            int s = 0, ph = 0;
            for (int i = 0; i < nkb; ++i) {
                if (!mbar_wait(&full_bar[s], ph)) {
                    atomicExch(err, 63);
                    ok = false;
                    break;
                }
                // rows brought by threads were written by the generic proxy; the tensor cores read by the asynchronous one
                if (!run) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_after_sync();
                const uint32_t a = smem_u32(stage0 + (size_t)s * stage_bytes);
                const uint64_t dx = umma_desc_k_sw128(a);
                for (int n0 = 0; n0 < W; n0 += 256) {
                    const uint32_t idesc = umma_idesc_bf16(TILE, min(256, W - n0));
                    const uint64_t da = umma_desc_k_sw128(a + X_BYTES + n0 * 128);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k)
                        umma_bf16(tmem + n0, dx + 2 * k, da + 2 * k, idesc, (i > 0 || k > 0) ? 1u : 0u);
                }
                umma_commit(&empty_bar[s]);
                if (++s == stages) s = 0, ph ^= 1;
            }
            if (ok) umma_commit(&done_bar);
        }
        __syncwarp();
        tc_fence_before_sync();
    }
    __syncthreads();
    if (warp == 4) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, tmem_cols);
    }
}

// ---- out = base + scale B v ------------------------------------------------------------------------------
constexpr int UP_THREADS = 224, UP_STAGES = 3, GROUP = 32;  // columns that a warp makes at a time

// Eight neighbouring elements of base as they lie.
template <typename TO> struct Eight;
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = load4(p), b = load4(p + 4); }
    __device__ __forceinline__ void store(float* p) const { store4(p, a), store4(p + 4, b); }
    __device__ __forceinline__ float get(int i) const {
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        return v[i];
    }
};
template <> struct Eight<__nv_bfloat16> {
    uint4 a;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
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
// both).  Warps 0 to 3 have 32 rows each and make the sums, warp 4 issues the products, 5 and 6 bring B.  B's
// columns lie in the operand, and so in tensor memory, in an order that leaves a lane of the accumulator layout
// with eight neighbours of a row: of a group of 32, column 4 n + j is number 8 j + n (woven: even j in the first
// half of the turn's columns, odd j in the second, each half a product with its own part of v).
template <typename TO, int SPLITS, bool WOVEN>
__global__ void __launch_bounds__(UP_THREADS, 2)
adapter_up_tc_kernel(const Args p, int pieces, int span, int cols, int stages, int vec, int* __restrict__ err) {
    constexpr int PARTS = WOVEN ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t b_full[UP_STAGES], b_empty[UP_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_base;
    __shared__ int rows[TILE];
    const int kb = (p.rank + BK - 1) / BK;  // blocks of 64 along the rank
    uint8_t* vs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* bs = vs + SPLITS * PARTS * kb * X_BYTES;  // v: [SPLITS][PARTS][kb] blocks of 128 rows; B: [stages][kb]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_wait();
    const Tile tile = load_tile(p.tiles, blockIdx.y);
    if (tile.adapter < 0) return;
    const bool none = tile.adapter >= p.n;
    if (none && p.out == p.base) return;
    if (tid < TILE) rows[tid] = p.order[tile.place + min(tid, tile.count - 1)];
    const int rank = none ? 0 : p.rank_of(tile.adapter), steps = (rank + 15) / 16, W = p.parts.n * p.rank;
    // this block's part and columns
    int part = 0, first = 0, block = blockIdx.x;
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
            mbar_init(&acc_empty[s], 4);
        }
        fence_barrier_init();
    }
    if (steps && warp == 4) {
        tmem_alloc(&tmem_base, 256);
        tmem_relinquish();
    }
    if (steps) {
        // v: four lanes a row, a row's numbers four at a time
        const int per = piece_blocks(p.K, pieces);
        const int full = ((p.K + BK - 1) / BK + per - 1) / per;  // pieces that have blocks
        for (int r = warp * 8 + (lane >> 2); r < TILE; r += UP_THREADS / 4) {
            const float* low = p.low + ((size_t)tile.place + min(r, tile.count - 1)) * W + (WOVEN ? 0 : part * p.rank);
            for (int q = 0; q < PARTS; ++q)
#pragma unroll 4
                for (int k = t * 4; k < steps * 16; k += 16) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int s = 0; s < full; ++s) {
                        const float4 a = load4(low + (size_t)s * p.R * W + q * p.rank + k);
                        v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
                    }
                    uint8_t* dst = vs + (q * kb + (k >> 6)) * X_BYTES + r * 128 + ((((k >> 3) ^ r) & 7) << 4) + (k & 4) * 2;
#pragma unroll
                    for (int s = 0; s < SPLITS; ++s) {
                        const uint2 h = {attn::pack_bf16(v.x, v.y), attn::pack_bf16(v.z, v.w)};
                        *reinterpret_cast<uint2*>(dst + s * PARTS * kb * X_BYTES) = h;
                        v.x -= __uint_as_float(h.x << 16), v.y -= __uint_as_float(h.x & 0xffff0000u);
                        v.z -= __uint_as_float(h.y << 16), v.w -= __uint_as_float(h.y & 0xffff0000u);
                    }
                }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_launch_dependents();  // (not before tensor memory is this block's)
    if (warp < 4) {
        const int m0 = warp * 32;
        const TO* base[4];
        TO* out[4];
        bool row_on[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = m0 + g + 8 * i;
            row_on[i] = r < tile.count;
            base[i] = (const TO*)p.base + (size_t)rows[r] * p.ld_base;
            out[i] = (TO*)p.out + (size_t)rows[r] * p.ld_out;
        }
        const int per_turn = cols / GROUP, groups = min(turns * per_turn, (end - first + GROUP - 1) / GROUP);
        auto whole = [&](int at) { return vec && at + 8 <= end && (at & 7) == 0; };
        auto load_base = [&](int q, Eight<TO> (&v)[4]) {
            const int at = first + q * GROUP + 8 * t;
            if (q < groups && whole(at))
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (row_on[j]) v[j].load(base[j] + at);
        };
        if (steps == 0) {  // rows without an adapter (or with one of rank 0) go over as they are
            for (int q = 0; q < groups; ++q) {
                const int at = first + q * GROUP + 8 * t;
                Eight<TO> v[4];
                load_base(q, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!row_on[j]) continue;
                    if (whole(at)) v[j].store(out[j] + at);
                    else
                        for (int i = 0; i < 8; ++i)
                            if (at + i < end) out[j][at + i] = base[j][at + i];
                }
            }
            return;
        }
        const uint32_t tmem = tmem_base + ((uint32_t)m0 << 16);
        const float scale = p.scale[tile.adapter];
        bool ok = true;
        auto make = [&](int q, const Eight<TO> (&y)[4]) {
            const int i = q / per_turn, h = q - i * per_turn;
            if (h == 0) {
                ok = ok && mbar_wait(&acc_full[i & 1], i >> 1 & 1);
                if (!ok) atomicExch(err, 64);
                tc_fence_after_sync();
            }
            __syncwarp();
            uint32_t acc[2][16];  // 16 rows each: [tile of 8 columns][row g: two columns, row g + 8: two]
            const uint32_t at_t = tmem + (i & 1) * cols + (WOVEN ? h * 16 : h * 32);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if (WOVEN) {
                    tmem_ld_frag2_nowait(at_t + ((uint32_t)m << 20), acc[m]);
                    tmem_ld_frag2_nowait(at_t + cols / 2 + ((uint32_t)m << 20), acc[m] + 8);
                } else {
                    tmem_ld_frag4_nowait(at_t + ((uint32_t)m << 20), acc[m]);
                }
            }
            tmem_ld_wait_16(acc[0]);
            tmem_loaded_16(acc[1]);
            if (h == per_turn - 1 || q == groups - 1) {  // the turn's sums are read
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[i & 1]);
            }
            const int at = first + q * GROUP + 8 * t;
            const bool fast = whole(at);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!row_on[j]) continue;
                float d[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    // column 4 n + jj of the group, n = 2 t or 2 t + 1: tile jj (woven: 0, 2, 1, 3 lie in order)
                    const int jj = c & 3, at_acc = WOVEN ? (jj & 1) * 2 + (jj >> 1) : jj;
                    d[c] = __uint_as_float(acc[j >> 1][at_acc * 4 + (j & 1) * 2 + (c >> 2)]);
                }
                if (fast) {
                    float o[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) o[c] = fmaf(scale, d[c], y[j].get(c));
                    if (ok) store8(out[j] + at, o);
                } else {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (at + c < end && ok) st(out[j], at + c, fmaf(scale, d[c], ld(base[j], at + c)));
                }
            }
        };
        // base's rows are on their way while the group before is made
        Eight<TO> y0[4], y1[4];
        load_base(0, y0);
        for (int q = 0; q < groups; q += 2) {
            load_base(q + 1, y1);
            make(q, y0);
            load_base(q + 2, y0);
            if (q + 1 < groups) make(q + 1, y1);
        }
        tc_fence_before_sync();
    } else if (warp == 4) {
        if (steps && elect_one()) {
            const uint32_t idesc = umma_idesc_bf16(TILE, cols / PARTS);
            int s = 0, ph = 0;
            for (int i = 0; i < turns; ++i) {
                if ((i >= 2 && !mbar_wait(&acc_empty[i & 1], (i >> 1 & 1) ^ 1)) || !mbar_wait(&b_full[s], ph)) {
                    atomicExch(err, 65);
                    break;
                }
                // B's columns were written by the generic proxy; the tensor cores read by the asynchronous one
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_after_sync();
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    const uint32_t d = tmem_base + (i & 1) * cols + q * (cols / 2);
                    uint32_t more = 0;
                    for (int sp = 0; sp < SPLITS; ++sp)
                        for (int k = 0; k < steps; ++k) {
                            const uint64_t dv = umma_desc_k_sw128(smem_u32(vs + ((sp * PARTS + q) * kb + (k >> 2)) * X_BYTES));
                            const uint64_t db = umma_desc_k_sw128(
                                smem_u32(bs + ((s * kb + (k >> 2)) * cols + q * (cols / 2)) * 128));
                            umma_bf16(d, dv + 2 * (k & 3), db + 2 * (k & 3), idesc, more);
                            more = 1;
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
        const int c0 = (tid - 160) >> 2;
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
    if (warp == 4) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 256);
    }
}

// Pieces of K: the waves of blocks, an SM holding one, times the blocks of 64 that each takes and about eight for
// its beginning and end, at their least.
int pieces_of(int K, int max_tiles) {
    const int blocks = (K + BK - 1) / BK, sms = sm_count();
    int best = 1;
    long long least = 0;
    for (int n = 1; n <= 16 && n <= (blocks + 3) / 4; ++n) {
        const long long cost = ((long long)max_tiles * n + sms - 1) / sms * ((blocks + n - 1) / n + 8);
        if (n == 1 || cost < least) best = n, least = cost;
    }
    return best;
}

// Blocks of 64 along the rank that v takes in shared memory (16 KB each), all its bfloat16 parts together: the
// kernel takes nine.
int v_blocks(const Args& p, int splits) { return splits * (p.parts.woven ? 2 : 1) * ((p.rank + BK - 1) / BK); }

template <typename TO, int SPLITS, bool WOVEN>
int up(const Args& p, int pieces, int* err, cudaStream_t s) {
    const int kb = (p.rank + BK - 1) / BK, cols = kb > 2 ? 64 : 128, parts = WOVEN ? 1 : p.parts.n;
    int turns[MAX_PARTS];
    for (int i = 0, first = 0; i < parts; first = p.parts.end[i++])
        turns[i] = ((WOVEN ? p.N : p.parts.end[i]) - first + cols - 1) / cols;
    // turns a block: the waves of blocks, two an SM, times the turns of each and about two for its beginning (v), at
    // their least
    int span = 1;
    long long least = 0;
    for (int n = 1; n <= 32; ++n) {
        long long blocks = 0;
        for (int i = 0; i < parts; ++i) blocks += (turns[i] + n - 1) / n;
        const long long cost = (blocks * p.max_tiles + 2 * sm_count() - 1) / (2 * sm_count()) * (n + 2);
        if (n == 1 || cost < least) span = n, least = cost;
    }
    int blocks = 0;
    for (int i = 0; i < parts; ++i) blocks += (turns[i] + span - 1) / span;
    const size_t v = (size_t)v_blocks(p, SPLITS) * X_BYTES, b = (size_t)kb * cols * 128;
    // two blocks an SM where three or two stages of B leave room for that
    int stages = v + 3 * b <= 110 * 1024 ? 3 : 2;
    const size_t smem = v + stages * b + 1024;
    const size_t align = (size_t)p.base | (size_t)p.out | (size_t)(p.ld_base * sizeof(TO)) | (size_t)(p.ld_out * sizeof(TO));
    static SmemLimit limit;
    cudaError_t e = limit.raise(adapter_up_tc_kernel<TO, SPLITS, WOVEN>, smem);
    if (e != cudaSuccess) return (int)e;
    RFX_LAUNCH((adapter_up_tc_kernel<TO, SPLITS, WOVEN>), dim3(blocks, p.max_tiles), UP_THREADS, smem, s, p, pieces, span,
               cols, stages, (align & 15) == 0 ? 1 : 0, err);
    return 0;
}

}  // namespace

namespace adapters {

// Whether the tcgen05 form takes these: x, a and b by 16 bytes, ranks in sixteens, the rank rows in tensor memory and
// the low-rank rows in shared memory.
bool prompt_takes(const Args& p, int dt_out) {
    const size_t align = (size_t)p.x | (size_t)p.a | (size_t)p.b | (size_t)(p.ld_x * 2) | (size_t)(p.lda * 2);
    return p.tile == TILE && (align & 15) == 0 && p.K % 8 == 0 && p.K >= BK && p.lda == p.K && p.rank % 16 == 0 &&
           p.parts.n * p.rank <= MAX_W && v_blocks(p, dt_out == RFX_DT_F32 ? 3 : 2) <= 9 && p.max_tiles <= 65535;
}

long long prompt_low_floats(int R, int K, int W, int max_tiles) { return (long long)pieces_of(K, max_tiles) * R * W; }

int prompt_form(const Args& p, int dt_out, int* err, cudaStream_t s) {
    const int W = p.parts.n * p.rank, pieces = pieces_of(p.K, p.max_tiles);
    CUtensorMap map_a, map_x;
    const int box = W <= 256 ? W : 16;  // rows of A a copy brings (they come 53 cycles apart)
    if (!rfx::tma::make_map_rows64(&map_a, p.a, (long long)p.n * W, p.K, box) ||
        !rfx::tma::make_map_rows64(&map_x, p.x, p.R, p.K, TILE / 2, p.ld_x))
        return RFX_ERR_UNSUPPORTED;
    const int stage = X_BYTES + W * BK * 2;
    int stages = 200 * 1024 / stage;  // one block an SM: what is on its way hides the memory's latency
    if (stages < 2) stages = 2;
    if (stages > 6) stages = 6;
    uint32_t cols = 32;
    while ((int)cols < W) cols *= 2;
    const size_t smem = (size_t)stages * stage + 1024;
    static SmemLimit limit;
    cudaError_t e = limit.raise(adapter_low_tc_kernel, smem);
    if (e != cudaSuccess) return (int)e;
    RFX_LAUNCH(adapter_low_tc_kernel, dim3(p.max_tiles, pieces), LOW_THREADS, smem, s, p, map_a, map_x, box, stages, pieces,
               cols, err);
    if (dt_out == RFX_DT_F32)
        return p.parts.woven ? up<float, 3, true>(p, pieces, err, s) : up<float, 3, false>(p, pieces, err, s);
    return p.parts.woven ? up<__nv_bfloat16, 2, true>(p, pieces, err, s) : up<__nv_bfloat16, 2, false>(p, pieces, err, s);
}

}  // namespace adapters
