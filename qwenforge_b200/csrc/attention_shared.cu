// Decode attention of sequences whose caches begin with the same pages (several answers to one prompt, branches of a search): one new token per
// sequence, grouped heads, paged cache, bf16 with head sizes 32, 64, 96 and 128, and float32 or bf16 of any other size up to 256.
//
// For a query row i (sequence, head) and the keys j <= its position,  o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(s_ij - m_i),
// s_ij = q_i k_j scale log2(e). The sums over a sequence's keys fall into parts, each with a maximum m of its own; parts (m, l, o) join as
//   M = max m,  out = sum 2^(m - M) o / sum 2^(m - M) l.
// The keys of the pages that a group of sequences shares are one part (or, cut into runs, several) of ALL rows of the group at once: they are
// fetched once for members x heads rows, instead of once for every member. The keys behind them are a sequence's own parts, as in
// attention_decode.cu. A last kernel joins each row's parts.
//
// Which block takes which run is worked out on the device from the lengths of the step (`shared_plan_kernel`), so that a captured step can be
// replayed with other lengths; what is shared stands in arrays on the device:
//   entry_pages [n_seqs]  pages that the sequence shares with its group (0: none)
//   members     [n_seqs]  batch entries, group after group;   begin [n_groups + 1]  where each group starts there;   pages [n_groups]
// The plan: header of n_seqs ints (runs of the shared part | runs of the own part << 16), padded to four, then records of eight ints.
//
// Everything is held in float32 but the weights, which enter the second product as bf16 (their rounding, 2^-9 of each, is that of the result).
#include "mma.cuh"

#define SH_PREFIX 1   // record kinds
#define SH_OWN 0

struct SharedRecord {
    int kind;      // SH_OWN, SH_PREFIX, or -1: no such block
    int subject;   // batch entry, or group
    int chunk;     // which rows of it
    int slot;      // whose page table is read
    int p_begin, p_end;
    int limit;     // keys below it are seen by every row
    int part;      // which of a row's parts the block writes
};

// ---- the plan: one block. A group's pages count once per chunk of its rows, a sequence's own pages once per chunk of its heads; the target is the
// pages per block at which all of them fill `slots` blocks once (at least `least`: a page per warp), as in attention_decode.cu.
#define SH_PLAN_THREADS 256
__global__ void __launch_bounds__(SH_PLAN_THREADS)
shared_plan_kernel(const int* __restrict__ cu_q, const int* __restrict__ tok_pos, const int* __restrict__ slots, int n_seqs, const int* __restrict__ entry_pages,
                   const int* __restrict__ members, const int* __restrict__ begin, const int* __restrict__ pages, int n_groups, int kv_heads, int group_heads,
                   int row_chunk, int own_chunk, float row_cost, int blocks, int least, int most_shared, int most_own, int* __restrict__ plan, int n_records) {
    __shared__ int scratch[SH_PLAN_THREADS / 32 + 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto block_total = [&](int v) -> int {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if (lane == 0) scratch[warp] = v;
        __syncthreads();
        int t = 0;
#pragma unroll
        for (int w = 0; w < SH_PLAN_THREADS / 32; ++w) t += scratch[w];
        return t;
    };
    grid_dependency_wait();
    const int own_chunks = (group_heads + own_chunk - 1) / own_chunk;
    auto own_pages = [&](int s) -> int {
        if (s >= n_seqs || slots[s] < 0) return 0;
        return max(0, tok_pos[cu_q[s]] / QF_PAGE + 1 - entry_pages[s]);
    };
    auto group_slot = [&](int g) -> int {   // the first live member's: its pages are everyone's
        for (int i = begin[g]; i < begin[g + 1]; ++i)
            if (slots[members[i]] >= 0) return slots[members[i]];
        return -1;
    };
    auto chunks_of = [&](int g) -> int { return ((begin[g + 1] - begin[g]) * group_heads + row_chunk - 1) / row_chunk; };
    auto cut = [](int n_pages, float target, int most) -> int {   // runs of equal size, none without a page
        if (n_pages <= 0) return 0;
        const int n = min(max((int)ceilf((float)n_pages / target), 1), most);
        const int each = (n_pages + n - 1) / n;
        return (n_pages + each - 1) / each;
    };
    int cost = 0;
    for (int s = tid; s < n_seqs; s += SH_PLAN_THREADS) cost += own_pages(s) * own_chunks;
    for (int g = tid; g < n_groups; g += SH_PLAN_THREADS)
        if (group_slot(g) >= 0) cost += (int)(pages[g] * chunks_of(g) * row_cost);
    cost = block_total(cost);
    float target = fmaxf((float)least, (float)cost * (float)kv_heads / (float)blocks);
    for (int round = 0; round < 16; ++round) {
        int runs = 0;
        for (int s = tid; s < n_seqs; s += SH_PLAN_THREADS) runs += cut(own_pages(s), target, most_own) * own_chunks;
        for (int g = tid; g < n_groups; g += SH_PLAN_THREADS)
            if (group_slot(g) >= 0) runs += cut(pages[g], fmaxf((float)least, target / row_cost), most_shared) * chunks_of(g);
        runs = block_total(runs);
        if ((long long)runs * kv_heads <= blocks) break;
        if (round == 14) target = 3.0e38f;   // one run each: always within the grid
        else target *= fmaxf(1.05f, (float)runs * (float)kv_heads / (float)blocks);
    }
    SharedRecord* records = reinterpret_cast<SharedRecord*>(plan + (n_seqs + 3) / 4 * 4);
    // the records: groups first (their blocks take longest), then sequences, each in rising order
    int before = 0;
    auto place = [&](int n) -> int {   // exclusive prefix sum over the block, and the sum added to `before` for everyone
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        __syncthreads();
        if (lane == 31) scratch[warp] = upto;
        __syncthreads();
        int first = before, all = 0;
#pragma unroll
        for (int w = 0; w < SH_PLAN_THREADS / 32; ++w) {
            if (w < warp) first += scratch[w];
            all += scratch[w];
        }
        before += all;
        return first + upto - n;
    };
    for (int g0 = 0; g0 < n_groups; g0 += SH_PLAN_THREADS) {
        const int g = g0 + tid;
        const int slot = g < n_groups ? group_slot(g) : -1;
        const int runs = slot >= 0 ? cut(pages[g], fmaxf((float)least, target / row_cost), most_shared) : 0, chunks = slot >= 0 ? chunks_of(g) : 0;
        const int first = place(runs * chunks);
        if (runs <= 0) continue;
        const int each = (pages[g] + runs - 1) / runs;
        for (int k = 0; k < runs * chunks; ++k)
            if (first + k < n_records)
                records[first + k] = SharedRecord{SH_PREFIX, g, k / runs, slot, k % runs * each, min((k % runs + 1) * each, pages[g]), pages[g] * QF_PAGE, k % runs};
        for (int i = begin[g]; i < begin[g + 1]; ++i) plan[members[i]] = runs;
    }
    __syncthreads();   // the header's first halves are written
    for (int s0 = 0; s0 < n_seqs; s0 += SH_PLAN_THREADS) {
        const int s = s0 + tid;
        const int mine = own_pages(s), runs = cut(mine, target, most_own);
        const int first = place(runs * own_chunks);
        if (s >= n_seqs) continue;
        const int shared = entry_pages[s] > 0 && slots[s] >= 0 ? plan[s] : 0;
        plan[s] = shared | runs << 16;
        if (runs <= 0) continue;
        const int each = (mine + runs - 1) / runs, from = entry_pages[s];
        for (int k = 0; k < runs * own_chunks; ++k)
            if (first + k < n_records)
                records[first + k] = SharedRecord{SH_OWN, s, k / runs, slots[s], from + k % runs * each, from + min((k % runs + 1) * each, mine),
                                                  tok_pos[cu_q[s]] + 1, shared + k % runs};
    }
    for (int j = before + tid; j < n_records; j += SH_PLAN_THREADS) records[j].kind = -1;
}

// ---- what every kernel of the parts needs
struct SharedArgs {
    const int* cu_q;
    const int* tok_pos;
    const int* slots;
    const int* members;
    const int* begin;
    const int* plan;
    float* part_o;    // [n_seqs * n_heads][most_parts][D]
    float* part_ml;   // [n_seqs * n_heads][most_parts][2]
    int* err;
    int n_seqs, n_heads, most_parts;
    float scale_log2;
};

// Row r of a block: its place in q ([n_seqs * n_heads] rows of D), the keys it sees, or -1 where there is no such row or its entry is padding.
__device__ __forceinline__ int shared_row(const SharedArgs& a, const SharedRecord& rec, int kv_heads, int kvh, int rows, int r, int& limit) {
    const int G = a.n_heads / kv_heads;
    int entry, head;
    limit = 0;
    const int at = rec.chunk * rows + r;
    if (rec.kind == SH_PREFIX) {
        const int i = a.begin[rec.subject] + at / G;
        if (i >= a.begin[rec.subject + 1]) return -1;
        entry = a.members[i];
        head = at % G;
    } else {
        if (at >= G) return -1;
        entry = rec.subject;
        head = at;
    }
    if (a.slots[entry] < 0) return -1;
    limit = a.tok_pos[a.cu_q[entry]] + 1;
    return entry * a.n_heads + kvh * G + head;
}

// ---- bf16 on mma.sync: a block takes one run for up to 16 * MT rows. Each warp works alone on whole pages, in two halves through its own two
// buffers (16-byte asynchronous copies into padded rows), as in attention_decode.cu; the rows' queries lie in shared memory and every fragment of keys
// or values that a warp loads serves all of the block's tiles of 16 rows (one of a sequence's own part, up to MT of a group).
__host__ __device__ constexpr int shared_warps(int d) { return d <= 64 ? 8 : 4; }
template <int D> struct SharedShape {
    static constexpr int WARPS = shared_warps(D), THREADS = 32 * WARPS, LD = D + 8;   // LD: a padded row of keys, values, queries (bf16) or sums (float32)
    static constexpr int PAGE_BYTES = 2 * QF_PAGE * LD * 2;
};

template <int D, int MT>
__global__ void __launch_bounds__(SharedShape<D>::THREADS)
shared_parts_kernel(const bf16* __restrict__ q, KvSite<bf16> site, SharedArgs a) {
    using S = SharedShape<D>;
    constexpr int WARPS = S::WARPS, LD = S::LD, KS = D / 16, NT = D / 8, HALF = QF_PAGE / 2, STAGE = 2 * HALF * LD, ROWS = 16 * MT, CH = D / 8;
    extern __shared__ uint4 smem[];
    unsigned char* pages_s = reinterpret_cast<unsigned char*>(smem);
    bf16* q_s = reinterpret_cast<bf16*>(pages_s + (size_t)WARPS * S::PAGE_BYTES);
    __shared__ float m_s[WARPS * ROWS], l_s[WARPS * ROWS];
    __shared__ int row_at[ROWS], row_limit[ROWS], least_limit;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_launch_dependents();
    grid_dependency_wait();
    const int4* records = reinterpret_cast<const int4*>(a.plan + (a.n_seqs + 3) / 4 * 4) + 2 * (blockIdx.x / site.kv_heads);
    const int4 x = records[0], y = records[1];
    const SharedRecord rec = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    if (rec.kind < 0) return;
    const int kvh = blockIdx.x % site.kv_heads, tiles = rec.kind == SH_PREFIX ? MT : 1;

    bf16* stage0 = reinterpret_cast<bf16*>(pages_s + (size_t)warp * S::PAGE_BYTES);
    const int* table_row = site.table + (long long)rec.slot * site.table_stride;
    const int my_pages = rec.p_begin + warp < rec.p_end ? (rec.p_end - rec.p_begin - warp + WARPS - 1) / WARPS : 0;
    const int n_halves = 2 * my_pages;
    auto half_live = [&](int i, int& page, int& key0) {
        if (i >= n_halves) return false;
        const int p = rec.p_begin + warp + (i >> 1) * WARPS;
        key0 = p * QF_PAGE + (i & 1) * HALF;
        page = __ldg(table_row + p);
        if (page < 0) {
            if (lane == 0 && (i & 1) == 0) atomicOr(a.err, QF_ERR_NO_PAGE);
            return false;
        }
        return key0 < rec.limit;
    };
    auto issue = [&](int i) {
        int page, key0;
        if (half_live(i, page, key0)) {
            bf16* kb = stage0 + (size_t)(i & 1) * STAGE;
            bf16* vb = kb + HALF * LD;
            const bf16* kp = site.base + (long long)page * site.page_elems + ((long long)kvh * QF_PAGE + (i & 1) * HALF) * D;
            const bf16* vp = kp + (long long)site.kv_heads * QF_PAGE * D;
#pragma unroll 4
            for (int j = lane; j < HALF * CH; j += 32) {
                const int r = j / CH, c = (j % CH) * 8;
                cp_async_16(kb + (size_t)r * LD + c, kp + (size_t)r * D + c, true);
                cp_async_16(vb + (size_t)r * LD + c, vp + (size_t)r * D + c, true);
            }
        }
        cp_async_commit();   // one group per half, empty when there is nothing to fetch
    };
    issue(0);

    // ---- the rows and their queries
    if (threadIdx.x == 0) least_limit = rec.limit;
    __syncthreads();
    if (threadIdx.x < ROWS) {
        int limit;
        const int place = threadIdx.x < 16 * tiles ? shared_row(a, rec, site.kv_heads, kvh, 16 * tiles, threadIdx.x, limit) : -1;
        row_at[threadIdx.x] = place;
        row_limit[threadIdx.x] = place < 0 ? rec.limit : limit;   // (a row that is not there sees what all see; nothing is kept of it)
        if (place >= 0 && limit < rec.limit) atomicMin(&least_limit, limit);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * CH; i += S::THREADS) {
        const int r = i / CH, c = i % CH * 8, place = row_at[r];
        uint4 v = make_uint4(0, 0, 0, 0);
        if (place >= 0) v = *reinterpret_cast<const uint4*>(q + (size_t)place * D + c);
        *reinterpret_cast<uint4*>(q_s + (size_t)r * LD + c) = v;
    }
    __syncthreads();

    float o[MT][NT][4];
    float m_run[MT][2], l_run[MT][2];
    int seen[MT][2];   // keys that this lane's rows see
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int i = 0; i < NT; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            m_run[t][r] = QF_NEG_BIG;
            l_run[t][r] = 0.f;
            seen[t][r] = row_limit[16 * t + (lane >> 2) + 8 * r];
        }
    }
    for (int i = 0; i < n_halves; ++i) {
        issue(i + 1);
        int page, key0;
        const bool live = half_live(i, page, key0);
        cp_async_wait<1>();
        __syncwarp();   // each lane waited for its own copies; together the half page is complete
        if (live) {
            bf16* kb = stage0 + (size_t)(i & 1) * STAGE;
            bf16* vb = kb + HALF * LD;
            if (key0 + HALF > rec.limit) {
                // what lies behind a sequence's last position is nobody's: 0 times a NaN left there is not 0
                for (int j = lane; j < HALF * CH; j += 32) {
                    const int r = j / CH, c = (j % CH) * 8;
                    if (key0 + r >= rec.limit) *reinterpret_cast<uint4*>(vb + (size_t)r * LD + c) = make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
            }
            const bool full = key0 + HALF <= least_limit;   // every row sees the half whole
            float s[MT][4][4];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int n = 0; n < 4; ++n) s[t][n][0] = s[t][n][1] = s[t][n][2] = s[t][n][3] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t kf[2][4];
#pragma unroll
                for (int t2 = 0; t2 < 2; ++t2)   // 16 keys each
                    ldmatrix_x4(kf[t2], kb + (size_t)(16 * t2 + (lane >> 4) * 8 + (lane & 7)) * LD + 16 * ks + ((lane >> 3) & 1) * 8);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    if (t >= tiles) break;
                    uint32_t qa[4];
                    ldmatrix_x4(qa, q_s + (size_t)(16 * t + (lane & 15)) * LD + 16 * ks + (lane >> 4) * 8);
#pragma unroll
                    for (int t2 = 0; t2 < 2; ++t2) {
                        mma_bf16_16816(s[t][2 * t2], qa, kf[t2][0], kf[t2][1]);
                        mma_bf16_16816(s[t][2 * t2 + 1], qa, kf[t2][2], kf[t2][3]);
                    }
                }
            }
            uint32_t pa[MT][2][4];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if (t >= tiles) break;
                float mx[2] = {QF_NEG_BIG, QF_NEG_BIG};
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[t][n][e] *= a.scale_log2;
                        if (!full) {
                            const int kj = key0 + 8 * n + 2 * (lane & 3) + (e & 1);
                            if (kj >= seen[t][e >> 1]) s[t][n][e] = QF_NEG_BIG;
                        }
                        mx[e >> 1] = fmaxf(mx[e >> 1], s[t][n][e]);
                    }
                float corr[2], sum[2] = {0.f, 0.f};
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                    const float m_new = fmaxf(m_run[t][r], mx[r]);
                    corr[r] = fast_exp2(m_run[t][r] - m_new);
                    m_run[t][r] = m_new;
                    mx[r] = m_new <= QF_NEG_BIG ? 0.f : m_new;   // a row that has seen no key yet: its weights are 2^(-huge) = 0
                }
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[t][n][e] = fast_exp2(s[t][n][e] - mx[e >> 1]);
                        sum[e >> 1] += s[t][n][e];
                    }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
                    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
                    l_run[t][r] = l_run[t][r] * corr[r] + sum[r];
                }
                if (corr[0] != 1.f || corr[1] != 1.f) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        o[t][nt][0] *= corr[0];
                        o[t][nt][1] *= corr[0];
                        o[t][nt][2] *= corr[1];
                        o[t][nt][3] *= corr[1];
                    }
                }
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    pa[t][kk][0] = pack_bf16(s[t][2 * kk][0], s[t][2 * kk][1]);
                    pa[t][kk][1] = pack_bf16(s[t][2 * kk][2], s[t][2 * kk][3]);
                    pa[t][kk][2] = pack_bf16(s[t][2 * kk + 1][0], s[t][2 * kk + 1][1]);
                    pa[t][kk][3] = pack_bf16(s[t][2 * kk + 1][2], s[t][2 * kk + 1][3]);
                }
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                for (int nt = 0; nt < NT; nt += 2) {
                    uint32_t vf[4];
                    ldmatrix_x4_trans(vf, vb + (size_t)(16 * kk + ((lane >> 3) & 1) * 8 + (lane & 7)) * LD + 8 * nt + (lane >> 4) * 8);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        if (t >= tiles) break;
                        mma_bf16_16816(o[t][nt], pa[t][kk], vf[0], vf[1]);
                        mma_bf16_16816(o[t][nt + 1], pa[t][kk], vf[2], vf[3]);
                    }
                }
            }
        }
        __syncwarp();   // every lane has read this buffer before the copies of half i + 2 overwrite it
    }
    cp_async_wait<0>();

    // ---- the warps' sums come together, 16 rows at a time through the warps' own buffers, in warp order
#pragma unroll
    for (int t = 0; t < MT; ++t)
        if ((lane & 3) == 0) {
            m_s[warp * ROWS + 16 * t + (lane >> 2)] = m_run[t][0];
            m_s[warp * ROWS + 16 * t + (lane >> 2) + 8] = m_run[t][1];
        }
    __syncthreads();
    float* o_w = reinterpret_cast<float*>(pages_s + (size_t)warp * S::PAGE_BYTES);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if (t >= tiles) break;
        float f[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = 16 * t + (lane >> 2) + 8 * r;
            float m_all = m_s[row];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) m_all = fmaxf(m_all, m_s[w * ROWS + row]);
            f[r] = exp2f(m_run[t][r] - m_all);
            if ((lane & 3) == 0) l_s[warp * ROWS + row] = l_run[t][r] * f[r];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int c = 8 * nt + 2 * (lane & 3), r0 = lane >> 2, r1 = r0 + 8;
            *reinterpret_cast<float2*>(o_w + r0 * LD + c) = make_float2(o[t][nt][0] * f[0], o[t][nt][1] * f[0]);
            *reinterpret_cast<float2*>(o_w + r1 * LD + c) = make_float2(o[t][nt][2] * f[1], o[t][nt][3] * f[1]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * (D / 4); i += S::THREADS) {
            const int r = i / (D / 4), c = i % (D / 4) * 4, place = row_at[16 * t + r];
            if (place < 0) continue;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(pages_s + (size_t)w * S::PAGE_BYTES) + r * LD + c);
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
            *reinterpret_cast<float4*>(a.part_o + ((size_t)place * a.most_parts + rec.part) * D + c) = sum;
        }
        __syncthreads();
    }
    if (threadIdx.x < 16 * tiles) {
        const int r = threadIdx.x, place = row_at[r];
        if (place < 0) return;
        float m = m_s[r], l = 0.f;
#pragma unroll
        for (int w = 1; w < WARPS; ++w) m = fmaxf(m, m_s[w * ROWS + r]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) l += l_s[w * ROWS + r];
        *reinterpret_cast<float2*>(a.part_ml + ((size_t)place * a.most_parts + rec.part) * 2) = make_float2(m, l);
    }
}

// ---- any type and head size: float32 arithmetic. A block takes one run for 16 rows; a page's keys, then its values, in shared memory as float32.
#define SH_ROWS 16
#define SH_THREADS 256
template <typename T>
__global__ void __launch_bounds__(SH_THREADS)
shared_parts_generic_kernel(const T* __restrict__ q, KvSite<T> site, SharedArgs a) {
    extern __shared__ float fs[];
    const int D = site.head_dim, LD = (D + 3) / 4 * 4 + 4;
    float* q_s = fs;                              // [16][LD]
    float* kv_s = q_s + SH_ROWS * LD;             // [64][LD]
    float* p_s = kv_s + QF_PAGE * LD;             // [16][64 + 4]
    __shared__ int row_at[SH_ROWS], row_limit[SH_ROWS];
    __shared__ float m_s[SH_ROWS], l_s[SH_ROWS], corr_s[SH_ROWS];
    grid_launch_dependents();
    grid_dependency_wait();
    const int4* records = reinterpret_cast<const int4*>(a.plan + (a.n_seqs + 3) / 4 * 4) + 2 * (blockIdx.x / site.kv_heads);
    const int4 x = records[0], y = records[1];
    const SharedRecord rec = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    if (rec.kind < 0) return;
    const int kvh = blockIdx.x % site.kv_heads, tid = threadIdx.x;
    if (tid < SH_ROWS) {
        int limit;
        row_at[tid] = shared_row(a, rec, site.kv_heads, kvh, SH_ROWS, tid, limit);
        row_limit[tid] = limit;   // (0, and no key, for a row that is not there)
        m_s[tid] = QF_NEG_BIG;
        l_s[tid] = 0.f;
    }
    __syncthreads();
    for (int i = tid; i < SH_ROWS * LD; i += SH_THREADS) {
        const int r = i / LD, c = i % LD;
        q_s[i] = c < D && row_at[r] >= 0 ? Num<T>::to_f(q[(size_t)row_at[r] * D + c]) : 0.f;
    }
    // a thread's outputs: row tid / 16, columns 4 (tid % 16) + 64 u .. + 3
    constexpr int U = 4;   // head sizes up to 256
    float4 o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int my_row = tid / 16, my_col = tid % 16 * 4;
    auto fetch = [&](const T* from, int n_rows) {   // rows of D into kv_s, zeros behind row n_rows and column D
        for (int i = tid; i < QF_PAGE * LD; i += SH_THREADS) {
            const int r = i / LD, c = i % LD;
            kv_s[i] = r < n_rows && c < D ? Num<T>::to_f(from[(size_t)r * D + c]) : 0.f;
        }
    };
    for (int p = rec.p_begin; p < rec.p_end; ++p) {
        const int page = site.table[(long long)rec.slot * site.table_stride + p];
        if (page < 0) {
            if (tid == 0) atomicOr(a.err, QF_ERR_NO_PAGE);
            continue;
        }
        const int key0 = p * QF_PAGE, n_rows = min(QF_PAGE, rec.limit - key0);
        const T* keys = site.base + (long long)page * site.page_elems + (long long)kvh * QF_PAGE * D;
        __syncthreads();
        fetch(keys, n_rows);
        __syncthreads();
        {   // scores: thread = key tid % 64, rows tid / 64 + 4 i
            const int key = tid % 64, r0 = tid / 64;
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            for (int c = 0; c < LD - 4; c += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(kv_s + key * LD + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 q4 = *reinterpret_cast<const float4*>(q_s + (r0 + 4 * i) * LD + c);
                    s[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[i]))));
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) p_s[(r0 + 4 * i) * (QF_PAGE + 4) + key] = key0 + key < row_limit[r0 + 4 * i] ? s[i] * a.scale_log2 : QF_NEG_BIG;
        }
        __syncthreads();
        fetch(keys + (long long)site.kv_heads * QF_PAGE * D, n_rows);
        {   // softmax: 16 lanes a row, four keys each
            float* p4 = p_s + my_row * (QF_PAGE + 4) + my_col;
            float4 v = *reinterpret_cast<float4*>(p4);
            float mx = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float m_old = m_s[my_row], m_new = fmaxf(m_old, mx), from = m_new <= QF_NEG_BIG ? 0.f : m_new;
            v.x = exp2f(v.x - from), v.y = exp2f(v.y - from), v.z = exp2f(v.z - from), v.w = exp2f(v.w - from);
            float sum = (v.x + v.y) + (v.z + v.w);
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            *reinterpret_cast<float4*>(p4) = v;
            __syncwarp();
            if (tid % 16 == 0) {
                const float corr = exp2f(m_old - m_new);
                corr_s[my_row] = corr;
                m_s[my_row] = m_new;
                l_s[my_row] = l_s[my_row] * corr + sum;
            }
        }
        __syncthreads();
        const float corr = corr_s[my_row];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (64 * u + my_col < D) {
                o[u].x *= corr, o[u].y *= corr, o[u].z *= corr, o[u].w *= corr;
                for (int k = 0; k < n_rows; ++k) {
                    const float w = p_s[my_row * (QF_PAGE + 4) + k];
                    const float4 v = *reinterpret_cast<const float4*>(kv_s + k * LD + 64 * u + my_col);
                    o[u].x = fmaf(w, v.x, o[u].x), o[u].y = fmaf(w, v.y, o[u].y), o[u].z = fmaf(w, v.z, o[u].z), o[u].w = fmaf(w, v.w, o[u].w);
                }
            }
    }
    __syncthreads();
    const int place = row_at[my_row];
    if (place < 0) return;
    const size_t part = (size_t)place * a.most_parts + rec.part;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const float v[4] = {o[u].x, o[u].y, o[u].z, o[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (64 * u + my_col + e < D) a.part_o[part * D + 64 * u + my_col + e] = v[e];
    }
    if (tid % 16 == 0) {
        a.part_ml[part * 2] = m_s[my_row];
        a.part_ml[part * 2 + 1] = l_s[my_row];
    }
}

// ---- the parts of a row come together: a thread per output element
template <typename T>
__global__ void __launch_bounds__(256)
shared_join_kernel(SharedArgs a, int D, T* __restrict__ out, const float* __restrict__ sinks) {
    grid_launch_dependents();
    grid_dependency_wait();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)a.n_seqs * a.n_heads * D) return;
    const int row = (int)(i / D), d = (int)(i % D), entry = row / a.n_heads;
    const int runs = a.slots[entry] < 0 ? 0 : (a.plan[entry] & 0xffff) + (a.plan[entry] >> 16);
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (size_t)row * a.most_parts;
    const float* po = a.part_o + (size_t)row * a.most_parts * D + d;
    float top = QF_NEG_BIG, den = 0.f, num = 0.f;
    for (int k = 0; k < runs; ++k) {
        const float2 x = ml[k];
        const float m = fmaxf(top, x.x), keep = exp2f(top - m), w = exp2f(x.x - m);
        den = den * keep + w * x.y;
        num = num * keep + w * po[(size_t)k * D];
        top = m;
    }
    if (sinks && runs > 0) {   // a logit that joins the sum of weights once, with no key and no value
        const float s2 = sinks[row % a.n_heads] * 1.4426950408889634f, m = fmaxf(top, s2), keep = exp2f(top - m);
        den = den * keep + exp2f(s2 - m);
        num *= keep;
    }
    out[i] = Num<T>::from_f(den > 0.f ? num / den : 0.f);
}

// ---------------------------------------------------------------------------------------------------------------- host
static bool shared_fast(int is_bf16, int d) { return is_bf16 && (d == 32 || d == 64 || d == 96 || d == 128); }
// Tiles of 16 rows that a block takes of a group's rows: one or two (four at head size 64 do not fit the registers).
static int shared_tiles(int is_bf16, int d, int most_rows) {
    if (!shared_fast(is_bf16, d)) return 1;
    return most_rows <= 16 ? 1 : 2;
}
template <int D> constexpr size_t shared_smem(int mt) {
    return (size_t)SharedShape<D>::WARPS * SharedShape<D>::PAGE_BYTES + (size_t)16 * mt * SharedShape<D>::LD * 2;
}
static size_t shared_generic_smem(int d) {
    const int ld = (d + 3) / 4 * 4 + 4;
    return (size_t)((SH_ROWS + QF_PAGE) * ld + SH_ROWS * (QF_PAGE + 4)) * sizeof(float);
}

// What sizes the plan and the workspaces. sizes[0]: rows of a block for a group; [1]: rows of a block for a sequence's own part; [2]: pages that a
// run should have at least; [3]: blocks that run at once.
QF_EXPORT int qf_attention_shared_shape(int is_bf16, int head_dim, int most_rows, int* sizes) {
    const int sms = qf_sm_count();
    if (sms <= 0 || head_dim <= 0 || head_dim > 256) return (int)cudaErrorInvalidValue;
    const bool fast = shared_fast(is_bf16, head_dim);
    sizes[0] = 16 * shared_tiles(is_bf16, head_dim, most_rows);
    sizes[1] = 16;
    sizes[2] = fast ? shared_warps(head_dim) : 2;
    sizes[3] = fast ? sms : 2 * sms;
    return 0;
}

QF_EXPORT int qf_attention_shared_plan(const int* cu_q, const int* tok_pos, const int* slots, int n_seqs, const int* entry_pages, const int* members,
                                       const int* begin, const int* pages, int n_groups, int kv_heads, int n_heads, int is_bf16, int head_dim,
                                       int most_rows, int most_shared, int most_own, int* plan, int n_records, cudaStream_t stream) {
    int sizes[4];
    if (kv_heads <= 0 || n_heads % kv_heads || n_records <= 0 || most_shared > 0xffff || most_own > 0x7fff) return (int)cudaErrorInvalidValue;
    const int bad = qf_attention_shared_shape(is_bf16, head_dim, most_rows, sizes);
    if (bad) return bad;
    const float row_cost = sizes[0] <= 16 ? 1.f : 1.4f;
    return (int)launch_pdl(shared_plan_kernel, dim3(1), dim3(SH_PLAN_THREADS), 0, stream, cu_q, tok_pos, slots, n_seqs, entry_pages, members, begin, pages,
                           n_groups, kv_heads, n_heads / kv_heads, sizes[0], sizes[1], row_cost, sizes[3], sizes[2], most_shared, most_own, plan, n_records);
}

template <int D, int MT>
static int launch_parts(const void* q, KvSite<bf16> site, const SharedArgs& a, int n_records, cudaStream_t stream) {
    constexpr size_t smem = shared_smem<D>(MT);
    static_assert(smem <= 227 * 1024 && (size_t)16 * SharedShape<D>::LD * 4 <= (size_t)SharedShape<D>::PAGE_BYTES, "a block's shared memory");
    auto kernel = shared_parts_kernel<D, MT>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    return (int)launch_pdl(kernel, dim3((unsigned)(n_records * site.kv_heads)), dim3(SharedShape<D>::THREADS), smem, stream, (const bf16*)q, site, a);
}

template <typename T>
static int launch_generic(const void* q, KvSite<T> site, const SharedArgs& a, int n_records, cudaStream_t stream) {
    const size_t smem = shared_generic_smem(site.head_dim);
    auto kernel = shared_parts_generic_kernel<T>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    return (int)launch_pdl(kernel, dim3((unsigned)(n_records * site.kv_heads)), dim3(SH_THREADS), smem, stream, (const T*)q, site, a);
}

// The parts and their joining. `plan`: of qf_attention_shared_plan with the same shape, n_records records; part_o, part_ml: n_seqs * n_heads *
// most_parts * head_dim and * 2 floats, most_parts >= most_shared + most_own. `launched` counts the launches.
QF_EXPORT int qf_attention_shared(int is_bf16, const void* q, void* out, const int* cu_q, const int* tok_pos, const int* slots, const int* members,
                                  const int* begin, const int* plan, int n_records, void* base, const int* table, long long page_elems, int table_stride,
                                  int kv_heads, int head_dim, int n_heads, int n_seqs, float scale, int most_rows, int most_parts, float* part_o,
                                  float* part_ml, const float* sinks, int* err, cudaStream_t stream) {
    if (n_seqs <= 0) return 0;
    if (kv_heads <= 0 || n_heads % kv_heads || head_dim <= 0 || head_dim > 256 || n_records <= 0) return (int)cudaErrorInvalidValue;
    const SharedArgs a = {cu_q, tok_pos, slots, members, begin, plan, part_o, part_ml, err, n_seqs, n_heads, most_parts, scale * 1.4426950408889634f};
    int code;
    if (shared_fast(is_bf16, head_dim)) {
        const KvSite<bf16> site{(bf16*)base, table, page_elems, table_stride, kv_heads, head_dim};
        const int mt = shared_tiles(is_bf16, head_dim, most_rows);
#define QF_SH(D, MT) launch_parts<D, MT>(q, site, a, n_records, stream)
        if (head_dim == 32) code = mt == 1 ? QF_SH(32, 1) : QF_SH(32, 2);
        else if (head_dim == 64) code = mt == 1 ? QF_SH(64, 1) : QF_SH(64, 2);
        else if (head_dim == 96) code = mt == 1 ? QF_SH(96, 1) : QF_SH(96, 2);
        else code = mt == 1 ? QF_SH(128, 1) : QF_SH(128, 2);
#undef QF_SH
    } else if (is_bf16) {
        code = launch_generic(q, KvSite<bf16>{(bf16*)base, table, page_elems, table_stride, kv_heads, head_dim}, a, n_records, stream);
    } else {
        code = launch_generic(q, KvSite<float>{(float*)base, table, page_elems, table_stride, kv_heads, head_dim}, a, n_records, stream);
    }
    if (code) return code;
    const unsigned blocks = (unsigned)(((long long)n_seqs * n_heads * head_dim + 255) / 256);
    if (is_bf16) return (int)launch_pdl(shared_join_kernel<bf16>, dim3(blocks), dim3(256), 0, stream, a, head_dim, (bf16*)out, sinks);
    return (int)launch_pdl(shared_join_kernel<float>, dim3(blocks), dim3(256), 0, stream, a, head_dim, (float*)out, sinks);
}
