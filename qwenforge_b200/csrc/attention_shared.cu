// Decode attention of sequences whose caches begin with the same pages (several answers to one prompt, branches of a search): one new token per
// sequence, grouped heads, paged cache, bf16 with head sizes 32, 64, 96 and 128, and float32 or bf16 of any other size up to 256.
//
// For a query row i (sequence, head) and the keys j <= its position,  o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(s_ij - m_i),
// s_ij = q_i k_j scale log2(e). The sums over a sequence's keys fall into parts, each with a maximum m of its own; parts (m, l, o) join as
//   M = max m,  out = sum 2^(m - M) o / sum 2^(m - M) l.
// The keys of the pages that a group of sequences shares are one part (or, cut into runs, several) of ALL rows of the group at once: they are
// fetched once for members x heads rows, instead of once for every member. The keys behind them are a sequence's own parts. A last kernel joins
// each row's parts.
//
// Which block and warp take which run is worked out on the device from the lengths of the step (`shared_plan_kernel`), so that a captured step can
// be replayed with other lengths; what is shared stands in arrays on the device:
//   entry_pages [n_seqs]  pages that the sequence shares with its group (0: none);   entry_group [n_seqs]  its group (-1: none)
//   members     [n_seqs]  batch entries, group after group;   begin [n_groups + 1]  where each group starts there;   pages [n_groups]
//
// Everything is held in float32 but the weights, which enter the second product as bf16 (their rounding, 2^-9 of each, is that of the result).
#include "mma.cuh"

// Record kinds: a sequence's own pages or a group's; with SH_TOGETHER, one of a block's that bring their sums together; none.
#define SH_OWN 0
#define SH_PREFIX 1
#define SH_TOGETHER 2
#define SH_NONE 4

struct __align__(16) SharedRecord {
    int kind;
    int subject;   // batch entry, or group
    int chunk;     // which rows of it: chunk * (rows of a tile) ..
    int slot;      // whose page table is read
    int p_begin, p_end;
    int limit;     // keys below it are seen by every row (a sequence's own part: its length)
    int part;      // which of a row's parts this is
};

// The plan: four counts (units, tile records, 0, 0), then n_seqs ints (a row's shared parts | its own parts << 16) padded to four, then the units (a record
// for each of a block's SH_TEAM warps) and the tile records.
#define SH_TEAM 4
__host__ __device__ constexpr long long shared_plan_records(int n_seqs) { return 4 + (n_seqs + 3) / 4 * 4; }   // (where they begin, in ints)

// ---- the plan: one block. An item is a group's pages or a sequence's own, times its tiles of rows. With X pages x tiles x kv heads in all and `warps`
// warps at once, a warp gets t = max(1, X / warps) pages. Items of up to SH_TEAM t pages are cut into records of t pages for a warp each, every one a part
// of its own; longer ones into runs of up to SH_TEAM t pages for a block, whose warps bring their sums together (SH_TOGETHER; not where a record is a
// whole block's work, `together_warps` 1). A group of `tile_rows`
// rows or more with `tile_pages` pages or more goes to the tensor-core tiles instead (attention_shared_tiles.cuh): pairs of tiles of 128 rows, cut into
// runs of as many turns of two pages as make the records fill the SMs once.
// What bounds it: the latency of a few dependent loads and of the block's barriers; every number is read once and kept in shared memory.
#define SH_PLAN_THREADS 256
#define SH_MAX_SEQS 2048
__global__ void __launch_bounds__(SH_PLAN_THREADS)
shared_plan_kernel(const int* __restrict__ tok_pos, const int* __restrict__ slots, int n_seqs, const int* __restrict__ entry_pages,
                   const int* __restrict__ entry_group, const int* __restrict__ begin, const int* __restrict__ pages, int n_groups, int kv_heads,
                   int group_heads, int row_tile, int warps, int together_warps, int most_shared, int most_own, int tile_rows, int tile_pages, int sms, int* __restrict__ plan,
                   int most_units, int most_tiles) {
    extern __shared__ int plan_s[];
    __shared__ long long sums_s[SH_PLAN_THREADS / 32];
    int* own_s = plan_s;                  // [n_seqs] pages of a sequence's own part
    int* slot_s = own_s + n_seqs;         // [n_groups] a live member's slot (-1: all have ended)
    int* least_s = slot_s + n_groups;     // [n_groups] the fewest keys that a live member sees
    int* rows_s = least_s + n_groups;     // [n_groups]
    int* pages_s = rows_s + n_groups;     // [n_groups]
    int* first_s = pages_s + n_groups;    // [n_groups] the group's first record of its kind
    int* runs_s = first_s + n_groups;     // [n_groups] its parts
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto block_total = [&](long long v) -> long long {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if (lane == 0) sums_s[warp] = v;
        __syncthreads();
        long long t = 0;
#pragma unroll
        for (int w = 0; w < SH_PLAN_THREADS / 32; ++w) t += sums_s[w];
        return t;
    };
    for (int g = tid; g < n_groups; g += SH_PLAN_THREADS) slot_s[g] = -1, least_s[g] = 0x7fffffff;
    __syncthreads();
    grid_dependency_wait();
    const int own_tiles = (group_heads + row_tile - 1) / row_tile;
    auto tiled = [&](int g) -> bool { return rows_s[g] >= tile_rows && pages_s[g] >= tile_pages; };
    auto group_tiles = [&](int g) -> int { return tiled(g) ? (rows_s[g] + 255) / 256 : (rows_s[g] + row_tile - 1) / row_tile; };
    long long sum = 0;   // pages x tiles of this thread's items, and (32 bits up) turns of pairs of tiles
    for (int g = tid; g < n_groups; g += SH_PLAN_THREADS) rows_s[g] = (begin[g + 1] - begin[g]) * group_heads, pages_s[g] = pages[g];
    for (int s = tid; s < n_seqs; s += SH_PLAN_THREADS) {
        const int slot = slots[s], pos = tok_pos[s], g = entry_group[s], n = slot < 0 ? 0 : max(0, pos / QF_PAGE + 1 - entry_pages[s]);
        own_s[s] = n;
        sum += n * own_tiles;
        if (slot >= 0 && g >= 0) {
            atomicMax(slot_s + g, slot);
            atomicMin(least_s + g, pos + 1);
        }
    }
    __syncthreads();
    for (int g = tid; g < n_groups; g += SH_PLAN_THREADS)
        if (slot_s[g] >= 0) sum += tiled(g) ? (long long)((pages_s[g] + 1) / 2 * group_tiles(g)) << 32 : (long long)(pages_s[g] * group_tiles(g));
    sum = block_total(sum);
    const int each = (int)max(1ll, ((sum & 0xffffffff) * kv_heads + warps - 1) / warps), team = together_warps > 1 ? (int)min((long long)each * SH_TEAM, 0x3fffffffll) : 0x3fffffff;
    int stretch = 2;   // turns of a tile record
    if (most_tiles > 0) {
        stretch = (int)max(2ll, ((sum >> 32) * kv_heads + sms - 1) / sms);
        for (int round = 0; round < 16; ++round) {   // (cutting into whole turns may give more records than SMs)
            long long records = 0;
            for (int g = tid; g < n_groups; g += SH_PLAN_THREADS)
                if (slot_s[g] >= 0 && tiled(g)) records += ((pages_s[g] + 1) / 2 + stretch - 1) / stretch * group_tiles(g);
            records = block_total(records) * kv_heads;
            if (records <= sms) break;
            stretch = round == 14 ? 0x3fffffff : (int)max((long long)stretch + 1, stretch * records / sms);
        }
    }
    // parts of an item: no more than there is room for (longer runs then), none without a page; and the pages of each
    auto cut = [&](int n_pages, int unit, int most, int& run) -> int {
        if (n_pages <= 0) return 0;
        const int n = min((n_pages + unit - 1) / unit, most);
        run = (n_pages + n - 1) / n;
        return (n_pages + run - 1) / run;
    };
    auto cut_group = [&](int g, int& run) -> int {
        if (slot_s[g] < 0) return 0;
        if (!tiled(g)) return cut(pages_s[g], pages_s[g] > team ? team : each, most_shared, run);
        const int n = cut((pages_s[g] + 1) / 2, stretch, most_shared, run);
        run *= 2;
        return n;
    };
    // Where every item's records begin: a prefix sum of three counts at once, 21 bits each: runs for a block, tile records, records for a warp.
    constexpr int BLOCKS = 42, TILES = 21, BITS = (1 << 21) - 1;
    long long before = 0;
    auto place = [&](long long mine) -> long long {
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        __syncthreads();
        if (lane == 31) sums_s[warp] = upto;
        __syncthreads();
        long long first = before + upto - mine;
#pragma unroll
        for (int w = 0; w < SH_PLAN_THREADS / 32; ++w) {
            if (w < warp) first += sums_s[w];
            before += sums_s[w];
        }
        return first;
    };
    for (int g0 = 0; g0 < n_groups; g0 += SH_PLAN_THREADS) {
        const int g = g0 + tid;
        int run = 0, parts = 0, shift = 0;
        if (g < n_groups) {
            parts = cut_group(g, run);
            shift = tiled(g) ? TILES : pages_s[g] > team ? BLOCKS : 0;
        }
        const long long first = place(g < n_groups ? (long long)(parts * group_tiles(g)) << shift : 0);
        if (g < n_groups) runs_s[g] = parts, first_s[g] = (int)(first >> shift) & BITS;
    }
    // The sequences' own counts are needed before any warp record can be placed (they lie behind the block's): first the counts, then the records.
    const long long groups_end = before;
    for (int s0 = 0; s0 < n_seqs; s0 += SH_PLAN_THREADS) {
        const int s = s0 + tid;
        int run = 0;
        const int n = s < n_seqs ? own_s[s] : 0;
        const long long parts = cut(n, n > team ? team : each, most_own, run) * own_tiles;
        place(parts << (n > team ? BLOCKS : 0));
    }
    const int blocks = (int)(before >> BLOCKS) & BITS, singles = (int)before & BITS, units = blocks + (singles + SH_TEAM - 1) / SH_TEAM;
    SharedRecord* const records = reinterpret_cast<SharedRecord*>(plan + shared_plan_records(n_seqs));
    SharedRecord* const tiles = records + (size_t)most_units * SH_TEAM;
    if (tid == 0) {
        plan[0] = min(units, most_units);
        plan[1] = min((int)(before >> TILES) & BITS, most_tiles);
    }
    // a run for a block: its warps' shares of the pages; a record for a warp: its place behind all blocks'
    auto write = [&](bool together, int index, SharedRecord r) {
        if (!together) {
            const int at = blocks * SH_TEAM + index;
            if (at < most_units * SH_TEAM) records[at] = r;
            return;
        }
        if (index >= most_units) return;
        const int from = r.p_begin, to = r.p_end, per = (to - from + SH_TEAM - 1) / SH_TEAM;
        r.kind |= SH_TOGETHER;
#pragma unroll
        for (int w = 0; w < SH_TEAM; ++w) {
            r.p_begin = min(from + w * per, to);
            r.p_end = min(from + (w + 1) * per, to);
            records[index * SH_TEAM + w] = r;
        }
    };
    if (tid < SH_TEAM && singles % SH_TEAM && tid >= singles % SH_TEAM)   // the last unit's warps without a record
        write(false, singles / SH_TEAM * SH_TEAM + tid, SharedRecord{SH_NONE, 0, 0, 0, 0, 0, 0, 0});
    for (int g = 0; g < n_groups; ++g) {   // the whole block at a group's records
        int run = 0;
        const int parts = cut_group(g, run), n = parts * group_tiles(g), limit = min(least_s[g], pages_s[g] * QF_PAGE);
        const bool tile = tiled(g), together = !tile && pages_s[g] > team;
        for (int k = tid; k < n; k += SH_PLAN_THREADS) {
            const int part = k % parts;
            const SharedRecord r = {SH_PREFIX, g, k / parts, slot_s[g], part * run, min((part + 1) * run, pages_s[g]), limit, part};
            if (!tile) write(together, first_s[g] + k, r);
            else if (first_s[g] + k < most_tiles) tiles[first_s[g] + k] = r;
        }
    }
    before = groups_end;
    for (int s0 = 0; s0 < n_seqs; s0 += SH_PLAN_THREADS) {
        const int s = s0 + tid;
        int run = 0;
        const int n = s < n_seqs ? own_s[s] : 0, parts = cut(n, n > team ? team : each, most_own, run);
        const bool together = n > team;
        const long long first = place((long long)(parts * own_tiles) << (together ? BLOCKS : 0));
        if (s >= n_seqs) continue;
        const int g = entry_group[s], slot = slots[s], shared = g >= 0 && slot >= 0 ? runs_s[g] : 0, from = entry_pages[s];
        plan[4 + s] = shared | parts << 16;
        const int index = (int)(first >> (together ? BLOCKS : 0)) & BITS;
        for (int k = 0; k < parts * own_tiles; ++k) {
            const int part = k % parts;
            write(together, index + k, SharedRecord{SH_OWN, s, k / parts, slot, from + part * run, from + min((part + 1) * run, n), tok_pos[s] + 1, shared + part});
        }
    }
}

// ---- what every kernel of the parts needs
struct SharedArgs {
    const int* tok_pos;
    const int* slots;
    const int* members;
    const int* begin;
    const int* plan;
    float* part_o;    // [n_seqs * n_heads][most_parts][D]
    float* part_ml;   // [n_seqs * n_heads][most_parts][2]
    int* err;
    int n_seqs, n_heads, most_parts, most_units;
    float scale_log2;
};

// Row `at` of a record's subject: its place in q ([n_seqs * n_heads] rows of D), or -1 where there is no such row. (The rows of a member that has ended
// have a place too: nobody reads what is left there.)
__device__ __forceinline__ int shared_row(const SharedArgs& a, const SharedRecord& rec, int kv_heads, int kvh, int at) {
    const int G = a.n_heads / kv_heads;
    if (!(rec.kind & SH_PREFIX)) return at < G ? rec.subject * a.n_heads + kvh * G + at : -1;
    const int i = a.begin[rec.subject] + at / G;
    return i < a.begin[rec.subject + 1] ? a.members[i] * a.n_heads + kvh * G + at % G : -1;
}
// The keys that the row at a place sees.
__device__ __forceinline__ int shared_seen(const SharedArgs& a, int place) {
    return place < 0 ? 0 : a.tok_pos[place / a.n_heads] + 1;
}

// 16 bytes of shared memory, read where it says so (the compiler would read them once, ahead of the loop, into registers).
__device__ __forceinline__ uint4 load_shared_16(const uint4* p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem_addr(p)));
    return v;
}

// ---- bf16 on mma.sync, straight from memory to registers. A warp takes 16 rows and a run of pages, KEYS keys a step: S = Q K^T, softmax with a running
// maximum, O += P V. Neither product minds the order of what it sums over, nor the second one the order of its columns, so the fragments are cut to
// suit 16-byte loads: lane (g, j) = (lane / 4, lane % 4) holds of key g's row the columns 32 u + 8 j .. + 7 (two k-steps of the first product, Q
// cut alike), and of the values of keys 2 j, 2 j + 1, 2 j + 8, 2 j + 9 the columns E g .. E g + E - 1, E = D / 8, which make the n-tiles' column g. No shared
// memory, no barrier: all of a step's keys and values are on their way at once, the next step's as soon as the registers are free again.
// What bounds it: the latency of memory while a run is short (a page at head size 64 is one step), then the rate at which pages arrive.
__host__ __device__ constexpr int shared_keys(int d) { return d <= 64 ? 64 : 32; }

template <int D>
__global__ void __launch_bounds__(32 * SH_TEAM, 2)
shared_parts_kernel(const bf16* __restrict__ q, KvSite<bf16> site, SharedArgs a) {
    constexpr int KEYS = shared_keys(D), SIX = KEYS / 16, STEPS = QF_PAGE / KEYS, KU = D / 32, E = D / 8, NT = E, LO = D + 4;
    __shared__ __align__(16) float merge_s[SH_TEAM][16][LO];
    __shared__ float m_s[SH_TEAM][16], l_s[SH_TEAM][16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
    grid_launch_dependents();
    grid_dependency_wait();
    const int kv_heads = site.kv_heads, units = a.plan[0] * kv_heads;
    const SharedRecord* records = reinterpret_cast<const SharedRecord*>(a.plan + shared_plan_records(a.n_seqs));
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int kvh = unit % kv_heads;
        const SharedRecord rec = records[unit / kv_heads * SH_TEAM + warp];
        if (rec.kind & SH_NONE) break;   // (the last warps of the last unit)
        const bool prefix = rec.kind & SH_PREFIX;
        const int p0 = rec.p_begin, p1 = rec.p_end, steps = STEPS * (p1 - p0);
        const int bound = prefix ? p1 * QF_PAGE : rec.limit;   // no row sees a key from here on
        const int* table_row = site.table + (long long)rec.slot * site.table_stride;
        int table = 0;   // a lane each the numbers of 32 pages
        uint4 k[2 * SIX][KU];          // n-tile t: key 8 t + g
        uint32_t v[4 * SIX][E / 2];    // of every 16 keys 2 j, 2 j + 1, 2 j + 8, 2 j + 9
        const bf16* k_at = nullptr;    // the step's keys (null: nothing to see there)
        auto find = [&](int i) {
            k_at = nullptr;
            if (i >= steps) return;
            const int n = i / STEPS, half = i % STEPS;
            if (n % 32 == 0 && half == 0) table = p0 + n + lane < p1 ? __ldg(table_row + p0 + n + lane) : 0;
            const int page = __shfl_sync(0xffffffffu, table, n & 31);
            if (page < 0) {
                if (lane == 0 && half == 0) atomicOr(a.err, QF_ERR_NO_PAGE);
                return;
            }
            if ((p0 + n) * QF_PAGE + KEYS * half >= bound) return;
            k_at = site.base + (long long)page * site.page_elems + ((long long)kvh * QF_PAGE + KEYS * half) * D;
        };
        auto load_keys = [&]() {
#pragma unroll
            for (int t = 0; t < 2 * SIX; ++t)
#pragma unroll
                for (int u = 0; u < KU; ++u) k[t][u] = __ldg(reinterpret_cast<const uint4*>(k_at + (8 * t + g) * D + 32 * u + 8 * j));
        };
        auto load_values = [&](const bf16* v_at) {
#pragma unroll
            for (int r = 0; r < 4 * SIX; ++r) {
                const bf16* row = v_at + (r / 4 * 16 + 2 * j + (r & 1) + 8 * (r >> 1 & 1)) * D + E * g;
                if constexpr (E % 8 == 0) {
#pragma unroll
                    for (int u = 0; u < E / 8; ++u) {
                        const uint4 x = __ldg(reinterpret_cast<const uint4*>(row + 8 * u));
                        v[r][4 * u] = x.x, v[r][4 * u + 1] = x.y, v[r][4 * u + 2] = x.z, v[r][4 * u + 3] = x.w;
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < E / 4; ++u) {
                        const uint2 x = __ldg(reinterpret_cast<const uint2*>(row + 4 * u));
                        v[r][2 * u] = x.x, v[r][2 * u + 1] = x.y;
                    }
                }
            }
        };
        const long long to_values = (long long)kv_heads * QF_PAGE * D;
        find(0);
        if (k_at) {
            load_keys();
            load_values(k_at + to_values);
        }
        const int place0 = shared_row(a, rec, kv_heads, kvh, 16 * rec.chunk + g), place1 = shared_row(a, rec, kv_heads, kvh, 16 * rec.chunk + g + 8);
        // the queries' fragments: in registers, or, beyond head size 64, where keys, values and sums fill those, a lane's own 16 bytes at a time out of
        // shared memory (the room that the warp's sums take at the end)
        constexpr bool HELD = D <= 64;
        uint4 q_held[HELD ? KU : 1][2];
        uint4* const q_s = reinterpret_cast<uint4*>(&merge_s[warp][0][0]) + lane;
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int place = r ? place1 : place0;
                const uint4 x = place < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(q + (size_t)place * D + 32 * u + 8 * j);
                if (HELD) q_held[HELD ? u : 0][r] = x;
                else q_s[(2 * u + r) * 32] = x;
            }
        asm volatile("" ::: "memory");   // (the stores stand before the reads below, which the compiler does not see as reads of this)
        float o[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
        float m0 = QF_NEG_BIG, m1 = QF_NEG_BIG, l0 = 0.f, l1 = 0.f;   // rows g and g + 8; the sums are this lane's share
        for (int i = 0; i < steps; ++i) {
            const bool live = k_at != nullptr;
            const int key0 = (p0 + i / STEPS) * QF_PAGE + KEYS * (i % STEPS);
            float s[2 * SIX][4];
            if (live) {
#pragma unroll
                for (int t = 0; t < 2 * SIX; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
                for (int u = 0; u < KU; ++u) {
                    const uint4 x = HELD ? q_held[HELD ? u : 0][0] : load_shared_16(q_s + 2 * u * 32), y = HELD ? q_held[HELD ? u : 0][1] : load_shared_16(q_s + (2 * u + 1) * 32);
                    const uint32_t lo[4] = {x.x, y.x, x.y, y.y}, hi[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
                    for (int t = 0; t < 2 * SIX; ++t) {
                        mma_bf16_16816(s[t], lo, k[t][u].x, k[t][u].y);
                        mma_bf16_16816(s[t], hi, k[t][u].z, k[t][u].w);
                    }
                }
            }
            find(i + 1);
            if (k_at) load_keys();   // (on their way while the softmax and the second product run)
            if (live) {
                float top0 = QF_NEG_BIG, top1 = QF_NEG_BIG;
                if (key0 + KEYS > rec.limit) {   // some row may not see some key; values behind the last one are nobody's (0 times a NaN is not 0)
                    const int see0 = prefix ? min(bound, shared_seen(a, place0)) : bound, see1 = prefix ? min(bound, shared_seen(a, place1)) : bound;
#pragma unroll
                    for (int t = 0; t < 2 * SIX; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[t][e] = key0 + 8 * t + 2 * j + (e & 1) < (e >> 1 ? see1 : see0) ? s[t][e] * a.scale_log2 : QF_NEG_BIG;
#pragma unroll
                    for (int r = 0; r < 4 * SIX; ++r)
                        if (key0 + r / 4 * 16 + 2 * j + (r & 1) + 8 * (r >> 1 & 1) >= bound)
#pragma unroll
                            for (int u = 0; u < E / 2; ++u) v[r][u] = 0u;
                } else {
#pragma unroll
                    for (int t = 0; t < 2 * SIX; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[t][e] *= a.scale_log2;
                }
#pragma unroll
                for (int t = 0; t < 2 * SIX; ++t) top0 = fmaxf(top0, fmaxf(s[t][0], s[t][1])), top1 = fmaxf(top1, fmaxf(s[t][2], s[t][3]));
                top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 1));
                top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 1));
                top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 2));
                top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 2));
                if (__any_sync(0xffffffffu, top0 > m0 || top1 > m1)) {
                    const float n0 = fmaxf(m0, top0), n1 = fmaxf(m1, top1), c0 = fast_exp2(m0 - n0), c1 = fast_exp2(m1 - n1);
                    m0 = n0, m1 = n1;
                    l0 *= c0, l1 *= c1;
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[t][0] *= c0, o[t][1] *= c0, o[t][2] *= c1, o[t][3] *= c1;
                }
                const float from0 = m0 <= QF_NEG_BIG ? 0.f : m0, from1 = m1 <= QF_NEG_BIG ? 0.f : m1;   // (no key seen yet: weights of 2^(-huge) = 0)
#pragma unroll
                for (int x = 0; x < SIX; ++x) {   // 16 keys at a time
#pragma unroll
                    for (int t = 2 * x; t < 2 * x + 2; ++t) {
                        s[t][0] = fast_exp2(s[t][0] - from0), s[t][1] = fast_exp2(s[t][1] - from0);
                        s[t][2] = fast_exp2(s[t][2] - from1), s[t][3] = fast_exp2(s[t][3] - from1);
                        l0 += s[t][0] + s[t][1];
                        l1 += s[t][2] + s[t][3];
                    }
                    const uint32_t p[4] = {pack_bf16(s[2 * x][0], s[2 * x][1]), pack_bf16(s[2 * x][2], s[2 * x][3]),
                                           pack_bf16(s[2 * x + 1][0], s[2 * x + 1][1]), pack_bf16(s[2 * x + 1][2], s[2 * x + 1][3])};
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint32_t pick = t & 1 ? 0x7632u : 0x5410u;
                        mma_bf16_16816(o[t], p, __byte_perm(v[4 * x][t / 2], v[4 * x + 1][t / 2], pick), __byte_perm(v[4 * x + 2][t / 2], v[4 * x + 3][t / 2], pick));
                    }
                }
            }
            if (k_at) load_values(k_at + to_values);
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, d);
            l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        // o[t][0], o[t][1] are row g's columns 2 j E + t and (2 j + 1) E + t: 2 E columns side by side
        auto leave = [&](float* row0, float* row1, float f0, float f1) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < E; t += 4) {
                    const int c = (2 * j + h) * E + t;
                    if (row0) *reinterpret_cast<float4*>(row0 + c) = make_float4(o[t][h] * f0, o[t + 1][h] * f0, o[t + 2][h] * f0, o[t + 3][h] * f0);
                    if (row1) *reinterpret_cast<float4*>(row1 + c) = make_float4(o[t][2 + h] * f1, o[t + 1][2 + h] * f1, o[t + 2][2 + h] * f1, o[t + 3][2 + h] * f1);
                }
        };
        if (!(rec.kind & SH_TOGETHER)) {
            const size_t at0 = (size_t)place0 * a.most_parts + rec.part, at1 = (size_t)place1 * a.most_parts + rec.part;
            leave(place0 < 0 ? nullptr : a.part_o + at0 * D, place1 < 0 ? nullptr : a.part_o + at1 * D, 1.f, 1.f);
            if (j == 0 && place0 >= 0) *reinterpret_cast<float2*>(a.part_ml + at0 * 2) = make_float2(m0, l0);
            if (j == 0 && place1 >= 0) *reinterpret_cast<float2*>(a.part_ml + at1 * 2) = make_float2(m1, l1);
            continue;
        }
        // the warps' sums come together in warp order
        if (j == 0) m_s[warp][g] = m0, m_s[warp][g + 8] = m1;
        __syncthreads();
        float top0 = m_s[0][g], top1 = m_s[0][g + 8];
#pragma unroll
        for (int w = 1; w < SH_TEAM; ++w) top0 = fmaxf(top0, m_s[w][g]), top1 = fmaxf(top1, m_s[w][g + 8]);
        const float f0 = fast_exp2(m0 - top0), f1 = fast_exp2(m1 - top1);
        if (j == 0) l_s[warp][g] = l0 * f0, l_s[warp][g + 8] = l1 * f1;
        leave(merge_s[warp][g], merge_s[warp][g + 8], f0, f1);
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * (D / 4); i += 32 * SH_TEAM) {
            const int r = i / (D / 4), c = i % (D / 4) * 4, place = shared_row(a, rec, kv_heads, kvh, 16 * rec.chunk + r);
            if (place < 0) continue;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < SH_TEAM; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(&merge_s[w][r][c]);
                sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
            }
            const size_t at = (size_t)place * a.most_parts + rec.part;
            *reinterpret_cast<float4*>(a.part_o + at * D + c) = sum;
            if (c == 0) {
                float m = m_s[0][r], l = 0.f;
#pragma unroll
                for (int w = 0; w < SH_TEAM; ++w) m = fmaxf(m, m_s[w][r]), l += l_s[w][r];
                *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m, l);
            }
        }
        __syncthreads();   // (the next unit writes these again)
    }
}

#include "attention_shared_tiles.cuh"

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
    const SharedRecord* records = reinterpret_cast<const SharedRecord*>(a.plan + shared_plan_records(a.n_seqs));
    const int kv_heads = site.kv_heads, units = a.plan[0] * SH_TEAM * kv_heads, tid = threadIdx.x;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {   // (a record is a block's work here)
    const int kvh = unit % kv_heads;
    const SharedRecord rec = records[unit / kv_heads];
    if (rec.kind & SH_NONE) break;
    const int bound = rec.kind & SH_PREFIX ? rec.p_end * QF_PAGE : rec.limit;
    if (tid < SH_ROWS) {
        row_at[tid] = shared_row(a, rec, kv_heads, kvh, SH_ROWS * rec.chunk + tid);
        row_limit[tid] = min(bound, shared_seen(a, row_at[tid]));
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
        const int key0 = p * QF_PAGE, n_rows = min(QF_PAGE, bound - key0);
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
    if (place >= 0) {
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
    __syncthreads();   // (the next unit writes these again)
    }
}

// ---- the parts of a row come together: a thread per V neighbouring output elements, eight parts on their way at once
template <typename T, int V>
__global__ void __launch_bounds__(256)
shared_join_kernel(SharedArgs a, int D, T* __restrict__ out, const float* __restrict__ sinks) {
    grid_launch_dependents();
    grid_dependency_wait();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const int per = D / V;
    if (i >= (long long)a.n_seqs * a.n_heads * per) return;
    const int row = (int)(i / per), d = (int)(i % per) * V, entry = row / a.n_heads;
    const int packed = a.plan[4 + entry], runs = a.slots[entry] < 0 ? 0 : (packed & 0xffff) + (packed >> 16);
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (size_t)row * a.most_parts;
    const float* po = a.part_o + (size_t)row * a.most_parts * D + d;
    float top = QF_NEG_BIG, den = 0.f, num[V];
#pragma unroll
    for (int e = 0; e < V; ++e) num[e] = 0.f;
    for (int k0 = 0; k0 < runs; k0 += 8) {
        float2 x[8];
        float o[8][V];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool in = k0 + k < runs;
            x[k] = in ? ml[k0 + k] : make_float2(QF_NEG_BIG, 0.f);
            if constexpr (V == 4) {
                const float4 v = in ? *reinterpret_cast<const float4*>(po + (size_t)(k0 + k) * D) : make_float4(0.f, 0.f, 0.f, 0.f);
                o[k][0] = v.x, o[k][1] = v.y, o[k][2] = v.z, o[k][3] = v.w;
            } else {
                o[k][0] = in ? po[(size_t)(k0 + k) * D] : 0.f;
            }
        }
        float m = top;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, x[k].x);
        const float keep = exp2f(top - m);
        den *= keep;
#pragma unroll
        for (int e = 0; e < V; ++e) num[e] *= keep;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float w = exp2f(x[k].x - m);
            den = fmaf(w, x[k].y, den);
#pragma unroll
            for (int e = 0; e < V; ++e) num[e] = fmaf(w, o[k][e], num[e]);
        }
        top = m;
    }
    float keep = 1.f;
    if (sinks && runs > 0) {   // a logit that joins the sum of weights once, with no key and no value
        const float s2 = sinks[row % a.n_heads] * 1.4426950408889634f, m = fmaxf(top, s2);
        keep = exp2f(top - m);
        den = den * keep + exp2f(s2 - m);
    }
    const float inv = den > 0.f ? keep / den : 0.f;
    T* to = out + (size_t)row * D + d;
    if constexpr (V == 4 && sizeof(T) == 2)
        *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(num[0] * inv, num[1] * inv), pack_bf16(num[2] * inv, num[3] * inv));
    else if constexpr (V == 4)
        *reinterpret_cast<float4*>(to) = make_float4(num[0] * inv, num[1] * inv, num[2] * inv, num[3] * inv);
    else
        to[0] = Num<T>::from_f(num[0] * inv);
}

// ---------------------------------------------------------------------------------------------------------------- host
static bool shared_fast(int is_bf16, int d) { return is_bf16 && (d == 32 || d == 64 || d == 96 || d == 128); }
static size_t shared_generic_smem(int d) {
    const int ld = (d + 3) / 4 * 4 + 4;
    return (size_t)((SH_ROWS + QF_PAGE) * ld + SH_ROWS * (QF_PAGE + 4)) * sizeof(float);
}

// Where the tiles take over.
#define SH_TILE_ROWS 65
#define SH_TILE_PAGES 8

// What sizes the plan and the workspaces. sizes[0]: rows of a tile; [1]: warps (or blocks, of the kernel for any type) that run at once; [2]: warps of a
// block that bring their sums together; [3]: the most parts of an item; [4], [5]: a group of so many rows and pages goes to the tiles (0: there are none); [6]: SMs.
QF_EXPORT int qf_attention_shared_shape(int is_bf16, int head_dim, int* sizes) {
    const int sms = qf_sm_count();
    if (sms <= 0 || head_dim <= 0 || head_dim > 256) return (int)cudaErrorInvalidValue;
    const bool fast = shared_fast(is_bf16, head_dim);
    sizes[0] = 16;
    sizes[1] = fast ? 2 * SH_TEAM * sms : 2 * sms;
    sizes[2] = fast ? SH_TEAM : 1;
    sizes[3] = 64;
    sizes[4] = fast && (head_dim == 64 || head_dim == 128) ? SH_TILE_ROWS : 0;
    sizes[5] = SH_TILE_PAGES;
    sizes[6] = sms;
    return 0;
}

QF_EXPORT int qf_attention_shared_plan(const int* tok_pos, const int* slots, int n_seqs, const int* entry_pages, const int* entry_group, const int* begin,
                                       const int* pages, int n_groups, int kv_heads, int n_heads, int is_bf16, int head_dim, int most_shared, int most_own,
                                       int* plan, int most_units, int most_tiles, cudaStream_t stream) {
    int sizes[7];
    if (n_seqs <= 0 || n_seqs > SH_MAX_SEQS || n_groups > n_seqs || kv_heads <= 0 || n_heads % kv_heads || most_own <= 0 || most_own > 0x7fff || most_shared > 0xffff ||
        (n_groups > 0 && most_shared <= 0) || most_units <= 0)
        return (int)cudaErrorInvalidValue;
    const int bad = qf_attention_shared_shape(is_bf16, head_dim, sizes);
    if (bad) return bad;
    const size_t smem = (size_t)(n_seqs + 6 * n_groups) * sizeof(int);
    const cudaError_t e = cudaFuncSetAttribute(shared_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 7 * SH_MAX_SEQS * (int)sizeof(int));
    if (e != cudaSuccess) return (int)e;
    return (int)launch_pdl(shared_plan_kernel, dim3(1), dim3(SH_PLAN_THREADS), smem, stream, tok_pos, slots, n_seqs, entry_pages, entry_group, begin, pages,
                           n_groups, kv_heads, n_heads / kv_heads, sizes[0], sizes[1], sizes[2], most_shared, most_own,
                           most_tiles > 0 ? sizes[4] : 0x7fffffff, sizes[5], sizes[6], plan, most_units, most_tiles);
}

template <int D>
static int launch_parts(const void* q, KvSite<bf16> site, const SharedArgs& a, int units, cudaStream_t stream) {
    const int at_once = 2 * qf_sm_count();
    return (int)launch_pdl(shared_parts_kernel<D>, dim3((unsigned)(units < at_once ? units : at_once)), dim3(32 * SH_TEAM), 0, stream, (const bf16*)q, site, a);
}

template <typename T>
static int launch_generic(const void* q, KvSite<T> site, const SharedArgs& a, int units, cudaStream_t stream) {
    const size_t smem = shared_generic_smem(site.head_dim);
    auto kernel = shared_parts_generic_kernel<T>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    const int at_once = 2 * qf_sm_count();
    return (int)launch_pdl(kernel, dim3((unsigned)(units < at_once ? units : at_once)), dim3(SH_THREADS), smem, stream, (const T*)q, site, a);
}

template <typename T>
static int launch_join(const SharedArgs& a, int head_dim, void* out, const float* sinks, cudaStream_t stream) {
    const long long items = (long long)a.n_seqs * a.n_heads * head_dim;
    if (head_dim % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0)
        return (int)launch_pdl(shared_join_kernel<T, 4>, dim3((unsigned)((items / 4 + 255) / 256)), dim3(256), 0, stream, a, head_dim, (T*)out, sinks);
    return (int)launch_pdl(shared_join_kernel<T, 1>, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, a, head_dim, (T*)out, sinks);
}

// The parts and their joining. `plan`: of qf_attention_shared_plan with the same shape; part_o, part_ml: n_seqs * n_heads * most_parts * head_dim and
// * 2 floats, most_parts >= the most shared and own parts of a row together.
QF_EXPORT int qf_attention_shared(int is_bf16, const void* q, void* out, const int* tok_pos, const int* slots, const int* members, const int* begin,
                                  const int* plan, int most_units, int most_tiles, void* base, const int* table, long long page_elems, int table_stride,
                                  int kv_heads, int head_dim, int n_heads, int n_seqs, float scale, int most_parts, float* part_o, float* part_ml,
                                  const float* sinks, int* err, cudaStream_t stream) {
    if (n_seqs <= 0) return 0;
    if (kv_heads <= 0 || n_heads % kv_heads || head_dim <= 0 || head_dim > 256 || most_units <= 0)
        return (int)cudaErrorInvalidValue;
    const SharedArgs a = {tok_pos, slots, members, begin, plan, part_o, part_ml, err, n_seqs, n_heads, most_parts, most_units, scale * 1.4426950408889634f};
    const bool fast = shared_fast(is_bf16, head_dim);
    const long long all = (long long)most_units * kv_heads * (fast ? 1 : SH_TEAM);
    const int units = (int)(all < 0x7fffffff ? all : 0x7fffffff);
    int code;
    if (fast) {
        const KvSite<bf16> site{(bf16*)base, table, page_elems, table_stride, kv_heads, head_dim};
        if (most_tiles > 0) {
            code = head_dim == 64 ? launch_tiles<64>(q, site, a, most_tiles, stream) : head_dim == 128 ? launch_tiles<128>(q, site, a, most_tiles, stream)
                                                                                                         : (int)cudaErrorInvalidValue;
            if (code) return code;
        }
        code = head_dim == 32 ? launch_parts<32>(q, site, a, units, stream) : head_dim == 64 ? launch_parts<64>(q, site, a, units, stream)
             : head_dim == 96 ? launch_parts<96>(q, site, a, units, stream) : launch_parts<128>(q, site, a, units, stream);
    } else if (is_bf16) {
        code = launch_generic(q, KvSite<bf16>{(bf16*)base, table, page_elems, table_stride, kv_heads, head_dim}, a, units, stream);
    } else {
        code = launch_generic(q, KvSite<float>{(float*)base, table, page_elems, table_stride, kv_heads, head_dim}, a, units, stream);
    }
    if (code) return code;
    return is_bf16 ? launch_join<bf16>(a, head_dim, out, sinks, stream) : launch_join<float>(a, head_dim, out, sinks, stream);
}
