// Part of attention_shared.cu: a large group's pages on the fifth-generation tensor cores (tcgen05), head sizes 64 and 128.
//
// The rows of a group and kv head (members x heads of the group) are cut into tiles of 128; a block takes two tiles and a run of the group's pages, two
// pages (128 keys) a turn, fetched once for both tiles by tiled copies (two stages each of keys and values). As in attention_prefill_tc.cu, tensor
// memory holds per tile the scores S [128 x 128] and the output O [128 x D]:
//   warps 0-3, 4-7   a tile's rows, a thread each: bring the queries into shared memory, then turn by turn the row of S, maximum, exponentials,
//                    sum; the weights go back over the scores as bf16, the left operand of the second product
//   warp 8           issues the products: O += P V of a tile as soon as its weights are written, then S = Q K^T of its next turn
//   warp 9           issues the copies
// There is no causal mask: a row sees every key of the run, and only the half turn behind an odd page count is masked. At the end every row leaves its sums,
// unnormalised and in float32, with its reference maximum and its sum of weights; a warp's rows go through the room that their queries had, so that they
// are written 128 bytes or more at a time.
// Blocks without a tile record give their ten warps the records of everything else, at the same time: sequences' own pages and small groups'.
// What bounds it: 16,384 exponentials a tile and turn on the SM's special-function units, beside as many cycles of products at D = 128, and the chain scores,
// exponentials, product of a tile, of which two overlap; a short run, the way to its first scores (plan, queries: 4 to 5 us) and its sums' way out (2.7 us).
// Measured: 250 sequences, 14 heads of 64 over 2, behind 250 pages: the turns of 126 blocks 26 us, 550 TFLOP/s, the operator 35.6; 64 sequences, 28 heads of
// 128 over 4, behind 128 pages, 88 blocks: turns 13 us, the operator 27.0. Tried with the first of them, at 38.4 us then: a warp for each tile's products
// 43.6; that with a page a turn and the next page's scores formed meanwhile 40.4; the tiles' exponentials strictly in turn 39.9.
// Every wait is bounded: one that runs out sets QF_ERR_COPY_TIMEOUT and ends the thread's loop, and the block still frees its tensor memory and returns.
#pragma once
#include "tcgen05.cuh"

#define ST_BM 128              // rows of a tile
#define ST_BK 128              // keys of a turn: two pages
#define ST_THREADS (2 * ST_BM + 64)

// The largest of three: one instruction.
__device__ __forceinline__ float shared_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// What this thread wrote to shared memory is visible to the tensor cores' reads of it that follow a hand-over.
__device__ __forceinline__ void fence_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int D>
__global__ void __launch_bounds__(ST_THREADS, 1)
shared_tiles_kernel(const __grid_constant__ CUtensorMap kv_map, const bf16* __restrict__ q, KvSite<bf16> site, SharedArgs a) {
    constexpr int WARPS = ST_THREADS / 32;
    constexpr int CB = D / 64;                    // blocks of 64 columns in a row of Q, K or V
    constexpr int Q_BLOCK = ST_BM * 128;          // bytes of one [128][64] block of Q
    constexpr int KV_BLOCK = ST_BK * 128;         // bytes of one [128][64] block of two pages' keys or values
    constexpr int PAGE_BYTES = QF_PAGE * 128;     // one page's part of it
    constexpr int Q_BYTES = CB * Q_BLOCK, KV_BYTES = CB * KV_BLOCK;
    constexpr uint32_t TMEM_COLS = 512, O_COL = 256;   // S (and P) of tile t in columns 128 t .., O behind them
    constexpr int PRODUCTS = 8, COPIES = 9;            // the issuing warps
    extern __shared__ __align__(128) unsigned char tc_smem[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tc_smem) + 1023) & ~(uintptr_t)1023);
    unsigned char* q_s = smem;                          // [2][CB][128][64]
    unsigned char* k_s = q_s + 2 * Q_BYTES;             // [2][CB][128][64]
    unsigned char* v_s = k_s + 2 * KV_BYTES;            // [2][CB][128][64]
    __shared__ __align__(8) uint64_t bar_q, bar_k[2], bar_v[2], bar_k_free[2], bar_v_free[2], bar_s[2], bar_p[2], bar_pv[2], bar_end;
    __shared__ uint32_t tmem_base_s;
    __shared__ SharedRecord record_s[WARPS];
    const int warp = threadIdx.x >> 5, t = warp < 8 ? warp >> 2 : 0, row = threadIdx.x & 127;   // row threads: tile t, row `row`
    // Barriers and tensor memory before anything else: beside the end of the kernel before this one. (A block that turns out to have no tile record gives
    // its tensor memory back unused.)
    if (threadIdx.x == 0) {
        mbar_init(&bar_q, 8);
        mbar_init(&bar_end, 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_k[i], 1);
            mbar_init(&bar_v[i], 1);
            mbar_init(&bar_k_free[i], 1);
            mbar_init(&bar_v_free[i], 1);
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_p[i], ST_BM / 32);
            mbar_init(&bar_pv[i], 1);
        }
    }
    if (warp == PRODUCTS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base_s)), "r"(TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    grid_launch_dependents();   // (the block has its tensor memory)
    grid_dependency_wait();
    const int kv_heads = site.kv_heads, kvh = (int)(blockIdx.x % kv_heads);
    const SharedPlan plan = shared_plan<ST_THREADS, true>(a, reinterpret_cast<int*>(tc_smem), D);   // (room that nothing else needs yet)
    if (blockIdx.x == gridDim.x - 1) shared_count_parts<ST_THREADS>(a, plan);
    const int tile_blocks = plan.tiles * kv_heads;
    bool timed_out = false;
    if ((int)blockIdx.x >= tile_blocks) {
        // ---- the other records, a warp each
        const int all = ((int)gridDim.x - tile_blocks) * WARPS;
        unsigned char* const room = tc_smem + (shared_plan_ints(a.n_seqs, a.n_groups) * 4 + 127) / 128 * 128 + warp * (shared_stages(D) * shared_stage_bytes(D));
        for (int task = warp * ((int)gridDim.x - tile_blocks) + (int)blockIdx.x - tile_blocks; task < plan.singles * kv_heads; task += all) {
            shared_records<32, 1>(a, plan, threadIdx.x & 31, 0, task / kv_heads, record_s + warp);
            __syncwarp();
            const SharedRecord rec = record_s[warp];
            __syncwarp();
            SharedSums<D> x;
            shared_warp_staged<D>(q, site, a, rec, task % kv_heads, room, x);
            x.leave_part(a, rec.part);
        }
    } else {
        const SharedRecord rec = shared_tile_record(a, plan, blockIdx.x / kv_heads);
        const int rows = rec.rows - 2 * ST_BM * rec.chunk;   // from the first tile's on
        const int tiles = rows > ST_BM ? 2 : 1;
        const int turns = (rec.p_end - rec.p_begin + 1) / 2, end = rec.p_end * QF_PAGE;   // no key of this run from `end` on
        // the rows' queries, on their way while the block comes together
        int place = -1;
        uint4 query[D / 8];
        if (warp < PRODUCTS) {
            if (t < tiles) place = shared_row(a, rec, kv_heads, kvh, 2 * ST_BM * rec.chunk + ST_BM * t + row);
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {   // a warp's 32 rows, whole rows at a time: piece c of row r
                const int r = (32 * i + (threadIdx.x & 31)) / (D / 8), c = threadIdx.x % (D / 8), from = __shfl_sync(0xffffffffu, place, r);
                query[i] = from < 0 ? make_uint4(0, 0, 0, 0) : reinterpret_cast<const uint4*>(q + (size_t)from * D)[c];
            }
        }
        fence_to_async();   // (the plan's room is the copies' from here on)
        __syncthreads();    // (everyone has read what it wants of the plan)
        // A warp waits as one: the loads and stores of tensor memory and the choice of the issuing lane are collective.
        auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0; };

        if (warp == COPIES) {
            const bool leader = elect_one();
            const int* table_row = site.table + (long long)rec.slot * site.table_stride;
            int keys = 0, values = 0;   // turns whose copies have been asked for
            for (int j = 0; j < turns; ++j) {
                const int stage = j & 1, first = rec.p_begin + 2 * j;
                const uint32_t freed = ((j >> 1) + 1) & 1;   // the turn before last has been read
                int page[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    page[h] = table_row[min(first + h, rec.p_end - 1)];   // (beyond the last page: masked keys, values that nothing reads)
                    if (page[h] < 0) {  // a page that is not held: reported; some held memory is read instead
                        if (leader) atomicOr(a.err, QF_ERR_NO_PAGE);
                        page[h] = 0;
                    }
                }
                if (j >= 2 && !wait_all(&bar_k_free[stage], freed)) {
                    timed_out = true;
                    break;
                }
                // row of the cache seen as one matrix [rows][D]; pages may lie at any distance that is whole rows
                ++keys;
                if (leader) {
                    mbar_expect_tx(&bar_k[stage], KV_BYTES);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int cb = 0; cb < CB; ++cb)
                            tma_load_2d(k_s + stage * KV_BYTES + cb * KV_BLOCK + h * PAGE_BYTES, &kv_map, cb * 64,
                                        (int)((long long)page[h] * (site.page_elems / D) + kvh * QF_PAGE), &bar_k[stage]);
                }
                __syncwarp();
                if (j >= 2 && !wait_all(&bar_v_free[stage], freed)) {
                    timed_out = true;
                    break;
                }
                ++values;
                if (leader) {
                    mbar_expect_tx(&bar_v[stage], KV_BYTES);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int cb = 0; cb < CB; ++cb)
                            tma_load_2d(v_s + stage * KV_BYTES + cb * KV_BLOCK + h * PAGE_BYTES, &kv_map, cb * 64,
                                        (int)((long long)page[h] * (site.page_elems / D) + (kv_heads + kvh) * QF_PAGE), &bar_v[stage]);
                }
                __syncwarp();
            }
            // The block ends, also after a wait that ran out, only when nothing is on its way to its shared memory (long arrived otherwise).
            for (int j = max(keys - 2, 0); j < keys; ++j) timed_out |= !wait_all(&bar_k[j & 1], (j >> 1) & 1);
            for (int j = max(values - 2, 0); j < values; ++j) timed_out |= !wait_all(&bar_v[j & 1], (j >> 1) & 1);
        } else if (warp == PRODUCTS) {
            const bool leader = elect_one();
            // descriptors: an address field counts 16 bytes, so 16 columns of a K-major row (32 bytes) are 2 units
            const uint64_t desc_q = smem_desc_sw128(q_s), desc_k = smem_desc_sw128(k_s), desc_v = smem_desc_mn_sw128(v_s, KV_BLOCK);
            constexpr uint32_t idesc_s = umma_idesc_bf16(ST_BM, ST_BK, false), idesc_pv = umma_idesc_bf16(ST_BM, D, true);
            // S of tile i, turn j; the last tile that reads a turn's keys hands their stage back
            auto issue_s = [&](int i, int j) {
                if (!wait_all(&bar_k[j & 1], (j >> 1) & 1)) return false;
                tc_fence_after();
                if (leader) {
                    const uint64_t dq = desc_q + (uint64_t)(i * (Q_BYTES >> 4)), dk = desc_k + (uint64_t)((j & 1) * (KV_BYTES >> 4));
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                        umma_bf16(tmem + 128 * i, dq + (uint64_t)((ks / 4) * (Q_BLOCK >> 4) + 2 * (ks % 4)),
                                  dk + (uint64_t)((ks / 4) * (KV_BLOCK >> 4) + 2 * (ks % 4)), idesc_s, ks > 0 ? 1u : 0u);
                    umma_commit(&bar_s[i]);
                    if (i == tiles - 1) umma_commit(&bar_k_free[j & 1]);
                }
                __syncwarp();
                return true;
            };
            timed_out = !wait_all(&bar_q, 0);
            for (int i = 0; i < tiles && !timed_out; ++i) timed_out = !issue_s(i, 0);
            for (int j = 0; j < turns && !timed_out; ++j) {
                for (int i = 0; i < tiles && !timed_out; ++i) {
                    if (!wait_all(&bar_v[j & 1], (j >> 1) & 1) || !wait_all(&bar_p[i], j & 1)) {   // every row has written its weights
                        timed_out = true;
                        break;
                    }
                    tc_fence_after();
                    if (leader) {   // values [128 keys][D] as they lie (MN-major), 16 keys are two groups of 8 rows (2048 bytes)
                        const uint64_t dv = desc_v + (uint64_t)((j & 1) * (KV_BYTES >> 4));
                        const int k1 = rec.p_begin + 2 * j + 1 < rec.p_end ? ST_BK / 16 : ST_BK / 32;
#pragma unroll
                        for (int kk = 0; kk < ST_BK / 16; ++kk)
                            if (kk < k1)
                                umma_bf16_tmem_a(tmem + O_COL + 128 * i, tmem + 128 * i + 8 * kk, dv + (uint64_t)(kk * (2048 >> 4)), idesc_pv,
                                                 (j > 0 || kk > 0) ? 1u : 0u);
                        umma_commit(&bar_pv[i]);
                        if (i == tiles - 1) umma_commit(&bar_v_free[j & 1]);
                    }
                    __syncwarp();
                    if (j + 1 < turns && (!wait_all(&bar_pv[i], j & 1) || !issue_s(i, j + 1))) timed_out = true;
                }
            }
            if (leader) umma_commit(&bar_end);   // the block ends when no product of its is at work
            __syncwarp();
            timed_out |= !wait_all(&bar_end, 0);
        } else {
            // ---- the row threads
            {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {   // the 128-byte swizzle: 16-byte chunk c of a row of 64 columns lies at c XOR (row modulo 8)
                    const int r = (warp & 3) * 32 + (32 * i + (threadIdx.x & 31)) / (D / 8), c = threadIdx.x % (D / 8);
                    *reinterpret_cast<uint4*>(q_s + t * Q_BYTES + c / 8 * Q_BLOCK + r * 128 + ((c % 8) ^ (r & 7)) * 16) = query[i];
                }
                fence_to_async();
                __syncwarp();
                if ((threadIdx.x & 31) == 0) mbar_arrive(&bar_q);
            }
            if (t < tiles) {
            const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), s_at = lanes + 128 * t, o_at = lanes + O_COL + 128 * t;
            const float folded = a.scale_log2 > 0.f ? a.scale_log2 : 1.f;
            float m_ref = QF_NEG_BIG, l_run = 0.f;   // the reference maximum of the exponentials, and their sum
            for (int j = 0; j < turns; ++j) {
                if (!wait_all(&bar_s[t], j & 1)) {   // (the product of the turn before is done too: S was issued after it)
                    timed_out = true;
                    break;
                }
                tc_fence_after();
                float s[ST_BK];
                tmem_load_row_128(s_at, s);
                if (!(a.scale_log2 > 0.f)) {   // below, the scale is folded into the exponent, behind the maximum and the mask: above zero only
#pragma unroll
                    for (int i = 0; i < ST_BK; ++i) s[i] *= a.scale_log2;
                }
                const int key0 = (rec.p_begin + 2 * j) * QF_PAGE;
                if (key0 + ST_BK > end) {   // the second page is none: weights of 2^-inf = 0, and the products leave it out
#pragma unroll
                    for (int i = QF_PAGE; i < ST_BK; ++i) s[i] = -INFINITY;
                }
                float mx[4];  // four chains instead of one: the comparisons do not wait for each other
#pragma unroll
                for (int i = 0; i < 4; ++i) mx[i] = s[i];
#pragma unroll
                for (int i = 4; i < ST_BK - 4; i += 8)
#pragma unroll
                    for (int c = 0; c < 4; ++c) mx[c] = shared_max3(mx[c], s[i + c], s[i + 4 + c]);
#pragma unroll
                for (int c = 0; c < 4; ++c) mx[c] = fmaxf(mx[c], s[ST_BK - 4 + c]);
                // (the scores stay unscaled; the scale is folded into the exponent)
                const float m_true = fmaxf(m_ref, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * folded);
                float f_o = 1.0f;
                bool moved = false;
                if (j == 0) {
                    m_ref = m_true;  // nothing to rescale yet: the first products overwrite O
                } else if (m_true - m_ref > 8.0f) {   // (weights stay below 2^8, well inside bf16 and float32)
                    moved = true;
                    f_o = fast_exp2(m_ref - m_true);
                    m_ref = m_true;
                    l_run *= f_o;
                }
                if (__any_sync(0xffffffffu, moved)) {  // the warp's 32 rows of O are loaded and stored together
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t raw[16];
                        tmem_load_16(o_at + c0, raw);
#pragma unroll
                        for (int i = 0; i < 16; ++i) raw[i] = __float_as_uint(__uint_as_float(raw[i]) * f_o);
                        tmem_store_16(o_at + c0, raw);
                    }
                }
                // two neighbouring weights an instruction where the pipes allow it: s * scale - reference, and the sums
                const float2 by = make_float2(folded, folded), less = make_float2(-m_ref, -m_ref);
                float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {   // half of the weights at a time: the first are stored while the others are formed
                    uint32_t packed[32];
#pragma unroll
                    for (int i = 0; i < 64; i += 2) {
                        float2 p = __ffma2_rn(make_float2(s[64 * h + i], s[64 * h + i + 1]), by, less);
                        p.x = fast_exp2(p.x), p.y = fast_exp2(p.y);
                        part[(i >> 1) & 1] = __fadd2_rn(part[(i >> 1) & 1], p);
                        packed[i / 2] = pack_bf16(p.x, p.y);
                    }
                    tmem_store_32(s_at + 32 * h, packed);
                }
                l_run += (part[0].x + part[0].y) + (part[1].x + part[1].y);
                tmem_store_wait();
                tc_fence_before();
                __syncwarp();
                if ((threadIdx.x & 31) == 0) mbar_arrive(&bar_p[t]);
            }
            if (!timed_out && !wait_all(&bar_pv[t], (turns - 1) & 1)) timed_out = true;
            tc_fence_after();
            if (!timed_out) {   // (the loads are collective: every lane takes part, rows that are not there store nothing)
                constexpr int HALF = D / 2, C4 = HALF / 4, AT_ONCE = 32 / C4;   // a row's 16-byte pieces of half its columns, and rows that a warp writes at once
                const int lane = threadIdx.x & 31;
                if (place >= 0) *reinterpret_cast<float2*>(a.part_ml + ((size_t)place * a.most_parts + rec.part) * 2) = make_float2(m_ref, l_run);
                float4* const room = reinterpret_cast<float4*>(q_s + t * Q_BYTES) + (warp & 3) * 32 * C4;   // the warp's 32 rows of [128][HALF] floats
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int c0 = 0; c0 < HALF; c0 += 32) {
                        uint32_t raw[32];
                        tmem_load_32(o_at + h * HALF + c0, raw);
#pragma unroll
                        for (int c = 0; c < 8; ++c)   // piece c of a row lies at c XOR (row modulo 8): neither side meets a bank twice
                            room[lane * C4 + ((c0 / 4 + c) ^ (lane & 7))] = make_float4(__uint_as_float(raw[4 * c]), __uint_as_float(raw[4 * c + 1]),
                                                                                         __uint_as_float(raw[4 * c + 2]), __uint_as_float(raw[4 * c + 3]));
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
                        const int r = r0 + lane / C4, c = lane % C4, to = __shfl_sync(0xffffffffu, place, r);
                        if (to >= 0)
                            *reinterpret_cast<float4*>(a.part_o + ((size_t)to * a.most_parts + rec.part) * D + h * HALF + 4 * c) = room[r * C4 + (c ^ (r & 7))];
                    }
                    __syncwarp();
                }
            }
            }
        }
    }
    if (timed_out) atomicOr(a.err, QF_ERR_COPY_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    if (warp == PRODUCTS)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32  %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
}

template <int D>
static int launch_tiles(const void* q, KvSite<bf16> site, const SharedArgs& a, int most_tiles, cudaStream_t stream) {
    CUtensorMap map = {};
    if (site.page_elems % D) return (int)cudaErrorInvalidValue;
    // The cache of this entry as one matrix of rows of D elements. The map is given more rows than any cache has (its extent only bounds what a copy may
    // address; copies address rows of held pages only).
    if (!qf_make_map_bf16(&map, site.base, 1ll << 31, D, D, QF_PAGE)) return (int)cudaErrorNotSupported;
    constexpr size_t stages = (size_t)(D / 64) * (2 * ST_BM + 4 * ST_BK) * 128 + 1024;
    constexpr size_t smem = 226 * 1024;   // (one block an SM in any case)
    static_assert(SH_TILE_PLAN_INTS * sizeof(int) + 128 + ST_THREADS / 32 * shared_stages(D) * shared_stage_bytes(D) <= smem,
                  "the plan's room, and the stages of the other records' warps");
    static_assert(qf_tmem_fits(512, smem) && stages <= smem && smem <= 227 * 1024, "the rule of tcgen05.cuh");
    auto kernel = shared_tiles_kernel<D>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    // a block to an SM, and no fewer than the records that cannot be cut into fewer, with a few blocks for everything else
    const int least = most_tiles * site.kv_heads + 4, blocks = least > a.sms ? least : a.sms;
    return (int)launch_pdl(kernel, dim3((unsigned)blocks), dim3(ST_THREADS), smem, stream, map, (const bf16*)q, site, a);
}
