// The adapters of prompts: tiles of up to 128 rows of one adapter, bfloat16, two launches.
//
//  * low: v = A x, 128 rows by all rank rows of all parts, on tcgen05 with 32-bit sums in tensor memory.  A
//    tile's rows may lie anywhere (the packed rows of several prompts), so four warps bring them by 16-byte
//    asynchronous copies straight into the swizzled layout of the tensor cores' operand; A's rows, as many
//    as the adapter has, come by TMA.  K goes in several pieces side by side while that fills the GPU.  It reads
//    x once, and memory bounds it.
//  * up: out = base + scale B v, 128 rows by a span of one part's columns.  v is summed over the pieces, in
//    order, into two bfloat16 parts (16 bits: its error is 2^-9 of the result's rounding to bfloat16; three parts
//    for a 32-bit result) in shared memory; B's fragments come straight from memory (from L1 for all but one warp)
//    with k permuted so that a lane's elements lie side by side, and columns dealt so that a lane ends with
//    eight neighbours: base and out move in whole sectors.  The product is short (the rank), so the legacy
//    tensor instructions keep ahead of the memory that bounds this kernel.
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
adapter_low_tc_kernel(const Args p, const __grid_constant__ CUtensorMap map_a, int stages, int pieces, uint32_t tmem_cols,
                      int* __restrict__ err) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], done_bar;
    __shared__ uint32_t tmem_base;
    __shared__ int rows[TILE];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int W = p.parts.n * p.rank, stage_bytes = X_BYTES + W * BK * 2;
    pdl_prologue();
    const Tile t = load_tile(p.tiles, blockIdx.x);
    if (t.adapter < 0 || t.adapter >= p.n) return;
    const int rank = p.rank_of(t.adapter), steps = (rank + 15) / 16, N = p.parts.n * steps * 16;
    const int per = piece_blocks(p.K, pieces), kb0 = blockIdx.y * per;
    const int nkb = min((p.K + BK - 1) / BK, kb0 + per) - kb0;
    if (steps == 0 || nkb <= 0) return;  // (pieces without blocks are not read either)
    if (tid < TILE) rows[tid] = p.order[t.place + min(tid, t.count - 1)];
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full_bar[s], TILE + 1);  // the threads that bring x, and the bytes of A
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&done_bar, 1);
        fence_barrier_init();
        prefetch_tensormap(&map_a);
    }
    if (warp == 4) {
        tmem_alloc(&tmem_base, tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_base;
    if (warp < 4) {
        // thread: 16-byte unit u of the rows r0, r0 + 16, ...; a row's 128 bytes swizzled by its place among eight
        const int u = tid & 7, r0 = tid >> 3;
        const __nv_bfloat16* x = (const __nv_bfloat16*)p.x;
        const __nv_bfloat16* src[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) src[i] = x + (size_t)rows[r0 + 16 * i] * p.ld_x + u * 8;
        bool ok = true;
        auto arrive = [&](int i) {  // block i has landed: visible to the tensor cores
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&full_bar[i % stages]);
        };
        const int behind = stages - 1;
        for (int i = 0; i < nkb; ++i) {
            const int s = i % stages;
            if (i >= stages && !mbar_wait(&empty_bar[s], (i / stages - 1) & 1)) {
                atomicExch(err, 61);
                ok = false;
                break;
            }
            uint8_t* dst = tiles + (size_t)s * stage_bytes;
            const int k = (kb0 + i) * BK;
            const bool in = k + u * 8 < p.K;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = r0 + 16 * j;
                attn::cp_async_16(dst + r * 128 + ((u ^ (r & 7)) << 4), in ? src[j] + k : x, in);
            }
            attn::cp_async_commit();
            if (tid == 0) {
                mbar_expect_tx(&full_bar[s], (uint32_t)(N * BK * 2));
                for (int q = 0; q < p.parts.n; ++q)
                    for (int w = 0; w < steps; ++w)
                        tma_load_2d(dst + X_BYTES + (q * steps + w) * 16 * 128, &map_a, &full_bar[s], k,
                                    (t.adapter * p.parts.n + q) * p.rank + w * 16);
            }
            // all but the last `behind` blocks have landed once no more than that many groups are open
            if (i >= behind) {
                switch (behind) {
                    case 1: attn::cp_async_wait<1>(); break;
                    case 2: attn::cp_async_wait<2>(); break;
                    case 3: attn::cp_async_wait<3>(); break;
                    case 4: attn::cp_async_wait<4>(); break;
                    case 5: attn::cp_async_wait<5>(); break;
                    case 6: attn::cp_async_wait<6>(); break;
                    default: attn::cp_async_wait<7>(); break;
                }
                arrive(i - behind);
            }
        }
        attn::cp_async_wait<0>();
        if (ok)
            for (int i = max(0, nkb - behind); i < nkb; ++i) arrive(i);
        // ---- the sums: a thread has a row
        const bool have = ok && mbar_wait(&done_bar, 0);
        if (!have) atomicExch(err, 62);
        tc_fence_after_sync();
        const bool any = __any_sync(0xffffffffu, have);  // (the loads below are the whole warp's)
        const int m = warp * 32 + lane;
        const uint32_t at = tmem + ((uint32_t)(warp * 32) << 16);
        float* dst = p.low + ((size_t)blockIdx.y * p.R + t.place + m) * W;
        if (any) {
            for (int c = 0; c < N / 16; ++c) {
                float v[16];
                tmem_ld_16(at + c * 16, v);
                const int q = c / steps;
                if (m < t.count && have)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        store4(dst + q * p.rank + (c - q * steps) * 16 + j * 4,
                               make_float4(v[j * 4], v[j * 4 + 1], v[j * 4 + 2], v[j * 4 + 3]));
            }
        }
        tc_fence_before_sync();
    } else {
        if (elect_one()) {
            bool ok = true;
            for (int i = 0; i < nkb; ++i) {
                const int s = i % stages;
                if (!mbar_wait(&full_bar[s], (i / stages) & 1)) {
                    atomicExch(err, 63);
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const uint32_t a = smem_u32(tiles + (size_t)s * stage_bytes);
                const uint64_t dx = umma_desc_k_sw128(a);
                for (int n0 = 0; n0 < N; n0 += 256) {
                    const uint32_t idesc = umma_idesc_bf16(TILE, min(256, N - n0));
                    const uint64_t da = umma_desc_k_sw128(a + X_BYTES + n0 * 128);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k)
                        umma_bf16(tmem + n0, dx + 2 * k, da + 2 * k, idesc, (i > 0 || k > 0) ? 1u : 0u);
                }
                umma_commit(&empty_bar[s]);
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
constexpr int UP_THREADS = 256, GROUP = 32;

// SPLITS bfloat16 parts of v; a block: 128 rows by `span` groups of 32 columns, warps 4 (32 rows) x 2 (groups)
template <typename TO, int SPLITS, bool WOVEN>
__global__ void __launch_bounds__(UP_THREADS, 2) adapter_up_tc_kernel(const Args p, int pieces, int span, int vec) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ int rows[TILE];
    __nv_bfloat16* vs = reinterpret_cast<__nv_bfloat16*>(dynamic);  // [SPLITS][TILE][parts here * rank + 8]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_prologue();
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
            const int n = ((p.parts.end[part] - first + GROUP - 1) / GROUP + span - 1) / span;
            if (block < n) break;
            block -= n;
            first = p.parts.end[part++];
        }
    const int end = WOVEN ? p.N : p.parts.end[part];
    const int g0 = block * span, g1 = min(g0 + span, (end - first + GROUP - 1) / GROUP);
    const int here = WOVEN ? 2 * p.rank : p.rank, LDV = here + 8;
    if (steps) {
        const int units = (WOVEN ? 2 : 1) * steps * 4;  // of four numbers
        const int used = min((p.K + BK - 1) / BK, pieces * piece_blocks(p.K, pieces));
        const int full = (used + piece_blocks(p.K, pieces) - 1) / piece_blocks(p.K, pieces);  // pieces that have blocks
        for (int i = tid; i < TILE * units; i += UP_THREADS) {
            const int r = i / units, u = i - r * units, q = u / (steps * 4), at = q * p.rank + (u - q * steps * 4) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < tile.count) {
                const float* src = p.low + ((size_t)tile.place + r) * W + (WOVEN ? 0 : part * p.rank) + at;
                for (int s = 0; s < full; ++s) {
                    const float4 a = load4(src + (size_t)s * p.R * W);
                    v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
                }
            }
#pragma unroll
            for (int s = 0; s < SPLITS; ++s) {
                __nv_bfloat16* dst = vs + ((size_t)s * TILE + r) * LDV + at;
                store4(dst, v);
                const float4 f = load4(dst);
                v.x -= f.x, v.y -= f.y, v.z -= f.z, v.w -= f.w;
            }
        }
    }
    __syncthreads();
    const float scale = none ? 0.f : p.scale[tile.adapter];
    const __nv_bfloat16* b = (const __nv_bfloat16*)p.b + (none ? 0 : (size_t)tile.adapter * p.N * p.rank);
    const TO* base = (const TO*)p.base;
    TO* out = (TO*)p.out;
    const int m0 = (warp >> 1) * 32;
    if (m0 >= tile.count) return;
    for (int q = g0 + (warp & 1); q < g1; q += 2) {
        const int col = first + q * GROUP, at = col + 8 * t;
        const bool whole = vec && at + 8 <= end && (at & 7) == 0;
        float y[4][8];  // rows m0 + g, + 8, + 16, + 24
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = m0 + g + 8 * i;
            if (r < tile.count) {
                const TO* src = base + (size_t)rows[r] * p.ld_base + at;
                if (whole) {
                    const float4 lo = load4(src), hi = load4(src + 4);
                    y[i][0] = lo.x, y[i][1] = lo.y, y[i][2] = lo.z, y[i][3] = lo.w;
                    y[i][4] = hi.x, y[i][5] = hi.y, y[i][6] = hi.z, y[i][7] = hi.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[i][j] = at + j < end ? ld(src, j) : 0.f;
                }
            }
        }
        float acc[2][4][4] = {};
        const __nv_bfloat16* b_col[4];  // tile j has columns col + 4 n + j: a lane ends with eight neighbours
#pragma unroll
        for (int j = 0; j < 4; ++j) b_col[j] = b + (size_t)min(col + 4 * g + j, end - 1) * p.rank + t * 4;
#pragma unroll 2
        for (int s = 0; s < steps; ++s) {
            uint2 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __ldg(reinterpret_cast<const uint2*>(b_col[j] + s * 16));
#pragma unroll
            for (int sp = 0; sp < SPLITS; ++sp)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const __nv_bfloat16* v = vs + ((size_t)sp * TILE + m0 + m * 16 + g) * LDV + s * 16 + t * 4;
                    auto frag = [&](const __nv_bfloat16* f, uint32_t (&o)[4]) {
                        const uint2 lo = *reinterpret_cast<const uint2*>(f);
                        const uint2 hi = *reinterpret_cast<const uint2*>(f + 8 * LDV);
                        o[0] = lo.x, o[1] = hi.x, o[2] = lo.y, o[3] = hi.y;
                    };
                    uint32_t f[4], odd[4];
                    frag(v, f);
                    if (WOVEN) frag(v + p.rank, odd);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (WOVEN && (j & 1)) attn::mma_bf16(acc[m][j], odd, w[j].x, w[j].y);
                        else attn::mma_bf16(acc[m][j], f, w[j].x, w[j].y);
                    }
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = m0 + g + 8 * i;
            if (r >= tile.count) continue;
            TO* dst = out + (size_t)rows[r] * p.ld_out + at;
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                o[j] = none ? y[i][j] : fmaf(scale, acc[i >> 1][j & 3][(i & 1) * 2 + (j >> 2)], y[i][j]);
            if (whole) {
                store4(dst, make_float4(o[0], o[1], o[2], o[3]));
                store4(dst + 4, make_float4(o[4], o[5], o[6], o[7]));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at + j < end) st(dst, j, o[j]);
            }
        }
    }
}

// Pieces of K: as many as fill the GPU twice, at least four blocks of 64 each.
int pieces_of(int K, int max_tiles) {
    int n = (2 * sm_count() + max_tiles - 1) / max_tiles;
    const int most = ((K + BK - 1) / BK + 3) / 4;
    if (n > most) n = most;
    return n > 16 ? 16 : n;
}

template <typename TO, int SPLITS, bool WOVEN>
int up(const Args& p, int pieces, cudaStream_t s) {
    int groups[MAX_PARTS], all = 0, parts = WOVEN ? 1 : p.parts.n;
    for (int i = 0, first = 0; i < parts; first = p.parts.end[i++])
        all += groups[i] = ((WOVEN ? p.N : p.parts.end[i]) - first + GROUP - 1) / GROUP;
    // blocks of up to 32 groups (1,024 columns), fewer while the grid would not hold four blocks an SM
    int span = 32;
    while (span > 2 && (long long)p.max_tiles * ((all + span - 1) / span) < 4 * sm_count()) span /= 2;
    int blocks = 0;
    for (int i = 0; i < parts; ++i) blocks += (groups[i] + span - 1) / span;
    const size_t smem = (size_t)SPLITS * TILE * ((WOVEN ? 2 : 1) * p.rank + 8) * 2;
    const size_t align = (size_t)p.base | (size_t)p.out | (size_t)(p.ld_base * sizeof(TO)) | (size_t)(p.ld_out * sizeof(TO));
    static SmemLimit limit;
    cudaError_t e = limit.raise(adapter_up_tc_kernel<TO, SPLITS, WOVEN>, smem);
    if (e != cudaSuccess) return (int)e;
    RFX_LAUNCH((adapter_up_tc_kernel<TO, SPLITS, WOVEN>), dim3(blocks, p.max_tiles), UP_THREADS, smem, s, p, pieces, span,
               (align & 15) == 0 ? 1 : 0);
    return 0;
}

}  // namespace

namespace adapters {

// Whether the tcgen05 form takes these: x, a and b by 16 bytes, ranks in sixteens, the rank rows in tensor memory and
// the low-rank rows in shared memory.
bool prompt_takes(const Args& p) {
    const size_t align = (size_t)p.x | (size_t)p.a | (size_t)p.b | (size_t)(p.ld_x * 2) | (size_t)(p.lda * 2);
    return p.tile == TILE && (align & 15) == 0 && p.K % 8 == 0 && p.K >= BK && p.lda == p.K && p.rank % 16 == 0 &&
           p.parts.n * p.rank <= MAX_W && (p.parts.woven ? 2 : 1) * p.rank <= 256 && p.max_tiles <= 65535;
}

long long prompt_low_floats(int R, int K, int W, int max_tiles) { return (long long)pieces_of(K, max_tiles) * R * W; }

int prompt_form(const Args& p, int dt_out, int* err, cudaStream_t s) {
    const int W = p.parts.n * p.rank, pieces = pieces_of(p.K, p.max_tiles);
    CUtensorMap map_a;
    if (!rfx::tma::make_map_rows64(&map_a, p.a, (long long)p.n * W, p.K, 16)) return RFX_ERR_UNSUPPORTED;
    const int stage = X_BYTES + W * BK * 2;
    // up to two blocks an SM
    int stages = 100 * 1024 / stage;
    if (stages < 2) stages = 2;
    if (stages > 6) stages = 6;
    uint32_t cols = 32;
    while ((int)cols < W) cols *= 2;
    const size_t smem = (size_t)stages * stage + 1024;
    static SmemLimit limit;
    cudaError_t e = limit.raise(adapter_low_tc_kernel, smem);
    if (e != cudaSuccess) return (int)e;
    RFX_LAUNCH(adapter_low_tc_kernel, dim3(p.max_tiles, pieces), LOW_THREADS, smem, s, p, map_a, stages, pieces, cols, err);
    if (dt_out == RFX_DT_F32) return p.parts.woven ? up<float, 3, true>(p, pieces, s) : up<float, 3, false>(p, pieces, s);
    return p.parts.woven ? up<__nv_bfloat16, 2, true>(p, pieces, s) : up<__nv_bfloat16, 2, false>(p, pieces, s);
}

}  // namespace adapters
