// Decode attention of sequences whose caches begin with the same pages (several answers to one prompt, branches of a search): one new token per
// sequence, grouped heads, paged cache, bf16 with head sizes 32, 64, 96 and 128, and float32 or bf16 of any other size up to 256.
//
// For a query row i (sequence, head) and the keys j <= its position,  o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(s_ij - m_i),
// s_ij = q_i k_j scale log2(e). The sums over a sequence's keys fall into parts, each with a maximum m of its own; parts (m, l, o) join as
//   M = max m,  out = sum 2^(m - M) o / sum 2^(m - M) l.
// The keys of the pages that a group of sequences shares are one part (or, cut into runs, several) of ALL rows of the group at once: they are
// fetched once for members x heads rows, instead of once for every member. The keys behind them are a sequence's own parts. A last kernel joins
// each row's parts. A member that stands inside the shared pages does not see all of their keys. No mask would do for it in a product of all rows: what lies
// behind its position may be anything, and a weight of 0 times a NaN is a NaN. So it takes no part in its group, and reads all of its pages as its own; the
// group's records leave sums at its rows' places too, which the join passes over.
//
// Which block and warp takes which run is worked out on the device from the lengths of the step, so that a captured step can be replayed with other
// lengths, and by every block for itself (`shared_plan`: a launch of its own for it took 5 of 11 microseconds of a small call); what is shared stands in
// arrays on the device:
//   entry_pages [n_seqs]  pages that the sequence shares with its group (0: none);   entry_group [n_seqs]  its group (-1: none)
//   members     [n_seqs]  batch entries, group after group;   begin [n_groups + 1]  where each group starts there;   pages [n_groups]
//
// Everything is held in float32 but the weights, which enter the second product as bf16 (their rounding, up to 2^-8 of each, is that of the result).
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
    int limit;     // no key from here on is seen (a sequence's own part: its length); all rows see every key below
    int part;      // which of a row's parts this is
    int begin, rows;   // of a group: its first member's place, and members x heads
    int pad[2];
};
#define SH_TEAM 4            // warps of a block of the parts' kernel
#define SH_MAX_SEQS 2048
#define SH_TILE_PLAN_INTS 12288
// Beside tiles, microseconds (`shared_plan`): a page of 16 rows at head sizes 64 and 128 with ten warps of an SM at work, what a record costs besides, and how
// much longer than the others' blocks a tile's takes to and from its turns. Fitted to the blocks' times of two cases (attention_shared_tiles.cuh): the own pages
// of 250 sequences on 22 SMs 21 to 23 (estimate with the lag: 21), of 64 sequences on 60 SMs 17 (15).
#define SH_PAGE_TIME_64 0.24f
#define SH_PAGE_TIME_128 0.5f
#define SH_RECORD_TIME 0.35f
#define SH_TILE_LAG 4.5f

// What every kernel gets.
struct SharedArgs {
    const int* tok_pos;
    const int* slots;
    const int* entry_pages;
    const int* entry_group;
    const int* members;
    const int* begin;
    const int* pages;
    float* part_o;    // [n_seqs * n_heads][most_parts][D]
    float* part_ml;   // [n_seqs * n_heads][most_parts][2]
    int* part_n;      // [n_seqs] a row's first part | how many there are << 16
    int* err;
    int n_seqs, n_groups, n_heads, kv_heads, most_parts, most_shared, most_own;
    int warps, team, tile_rows, tile_work, sms;   // (see shared_plan; tile_rows 0: no tiles)
    float scale_log2;
};

// n / d rounded down, and up, for 0 <= n < 2^20 and 0 < d, with one = 1 / d in float32: the product is off by one at most.
__device__ __forceinline__ int shared_div(int n, int d, float one) {
    int q = (int)((float)n * one);
    const int r = n - q * d;
    return q + (r < 0 ? -1 : r >= d ? 1 : 0);
}
__device__ __forceinline__ int shared_div(int n, int d) { return shared_div(n, d, __fdividef(1.f, (float)d)); }
__device__ __forceinline__ int shared_div_up(int n, int d, float one) {
    const int q = shared_div(n, d, one);
    return q + (q * d < n);
}
__device__ __forceinline__ int shared_div_up(int n, int d) { return shared_div_up(n, d, __fdividef(1.f, (float)d)); }

// ---- the plan. An item is a group's pages or a sequence's own, times its tiles of 16 rows. A group of `tile_rows` rows or more, and `tile_work` rows x
// pages or more, goes to the tensor-core tiles (attention_shared_tiles.cuh): pairs of tiles of 128 rows, every group's pages cut into runs by its share of the
// work, no more records than the SMs that the tiles get by theirs. Everything else is cut into records of t pages for a warp each, every one a part of its
// own: t = max(1, pages x tiles x kv heads / warps), beside tiles the next larger t that gives no more records than the other SMs have warps (two records
// in a row take a warp twice the time); without tiles an item of more than SH_TEAM t pages goes in runs of up to SH_TEAM t to blocks, whose warps bring
// their sums together (SH_TOGETHER).
// What bounds it: the latency of one round of loads (0.4 us), then of divisions, reductions and half a dozen barriers. Measured from a block's start: with
// two sequences 2.2 us, beside tiles 3.0 to 3.6 (250 and 64 sequences), a tile's block 2.1 to 2.5.
#define SH_ROW_TILE 16
struct SharedPlan {
    int* own;        // [n_seqs] pages of a sequence's own part
    int* own_first;  // [n_seqs] its first record of its kind
    int* slot;       // [n_groups] the slot of a live member that sees all that is shared (-1: there is none)
    int* rows;       // [n_groups]
    int* begin;      // [n_groups]
    int* pages;      // [n_groups]
    int* first;      // [n_groups] the group's first record of its kind
    int* parts;      // [n_groups]
    int own_tiles, each, together;    // (together: items of more pages are blocks' runs)
    float one_each;                   // 1 / each
    float tile_share;                 // parts of a tiled group beyond its first, for every turn
    int blocks, singles, tiles;       // records of each kind
};
__host__ __device__ constexpr int shared_plan_ints(int n_seqs, int n_groups) { return 2 * n_seqs + 6 * n_groups; }
// Whether a sequence at `pos` sees all of the pages that it shares.
__device__ __forceinline__ bool shared_whole(int pos, int shared) { return pos + 1 >= shared * QF_PAGE; }
// What an SM takes for a turn of a pair of tiles, microseconds (126 blocks of 14 turns 26 at head size 64, 88 of 6 13 at 128), and for a page.
__device__ __forceinline__ float shared_turn_time(int d) { return d <= 64 ? 1.8f : 2.1f; }
__device__ __forceinline__ float shared_page_time(int d) { return d <= 64 ? SH_PAGE_TIME_64 : SH_PAGE_TIME_128; }

// An item of n pages: how many parts it is cut into, no more than there is room for, none without a page; run: the pages of each but the last.
__device__ __forceinline__ int shared_cut(const SharedPlan& p, int n, int most, int& run) {
    run = 0;
    if (n <= 0) return 0;
    const bool whole = n > p.together;
    run = whole ? p.together : p.each;
    int parts = shared_div_up(n, run, whole ? p.one_each * (1.f / SH_TEAM) : p.one_each);
    if (parts > most) {
        run = shared_div_up(n, most);
        parts = shared_div_up(n, run);
    }
    return parts;
}
__device__ __forceinline__ bool shared_tiled(const SharedArgs& a, const SharedPlan& p, int g) {
    return a.tile_rows > 0 && p.rows[g] >= a.tile_rows && (float)p.rows[g] * p.pages[g] >= (float)a.tile_work;
}
__device__ __forceinline__ int shared_tiles_of(const SharedArgs& a, const SharedPlan& p, int g) {
    return shared_tiled(a, p, g) ? (p.rows[g] + 255) / 256 : (p.rows[g] + SH_ROW_TILE - 1) / SH_ROW_TILE;
}
__device__ __forceinline__ int shared_cut_group(const SharedArgs& a, const SharedPlan& p, int g, int& run) {
    run = 0;
    if (p.slot[g] < 0) return 0;
    const int n = p.pages[g];
    if (!shared_tiled(a, p, g)) return shared_cut(p, n, a.most_shared, run);
    const int turns = (n + 1) / 2, each = shared_div_up(turns, min(1 + (int)((float)turns * p.tile_share), min(turns, a.most_shared)));
    run = 2 * each;
    return shared_div_up(turns, each);
}
__device__ __forceinline__ int shared_cut_own(const SharedArgs& a, const SharedPlan& p, int s, int& run) {
    return shared_cut(p, p.own[s], a.most_own, run);
}

// By all threads of a block; `room`: shared_plan_ints of shared memory. TILES: of the kernel with tiles, where a block that gets a tile record needs, and
// works out, the tile records only (the grid's last block works out everything).
template <int THREADS, bool TILES>
__device__ __forceinline__ SharedPlan shared_plan(const SharedArgs& a, int* room, int head_dim) {
    constexpr int WARPS = THREADS / 32, SIZES = 6;
    constexpr unsigned ALL = 0xffffffffu;
    __shared__ uint4 sums_s[WARPS];
    __shared__ int2 counts_s[2][WARPS];
    __shared__ int records_s[SIZES];
    SharedPlan p;
    p.own = room, p.own_first = p.own + a.n_seqs;
    p.slot = p.own_first + a.n_seqs, p.rows = p.slot + a.n_groups, p.begin = p.rows + a.n_groups;
    p.pages = p.begin + a.n_groups, p.first = p.pages + a.n_groups, p.parts = p.first + a.n_groups;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group_heads = a.n_heads / a.kv_heads;
    p.own_tiles = (group_heads + SH_ROW_TILE - 1) / SH_ROW_TILE;
    // (everything is asked for before the first barrier: one round trip)
    int slot = -1, pos = 0, group = -1, shared = 0, begin = 0, end = 0, pages = 0;
    if (tid < a.n_seqs) slot = a.slots[tid], pos = a.tok_pos[tid], group = a.entry_group[tid], shared = a.entry_pages[tid];
    if (tid < a.n_groups) begin = a.begin[tid], end = a.begin[tid + 1], pages = a.pages[tid];
    for (int g = tid; g < a.n_groups; g += THREADS) {
        if (g != tid) begin = a.begin[g], end = a.begin[g + 1], pages = a.pages[g];
        p.slot[g] = -1, p.rows[g] = (end - begin) * group_heads, p.begin[g] = begin, p.pages[g] = pages;
    }
    if (a.n_groups > 0) __syncthreads();
    uint4 sum = make_uint4(0, 0, 0, 0);   // of this thread's items: pages x tiles, and tiles; turns of pairs of tiles, and pairs
    for (int s0 = 0; s0 < a.n_seqs; s0 += THREADS) {
        const int s = s0 + tid;
        if (s0 > 0) {
            slot = -1;
            if (s < a.n_seqs) slot = a.slots[s], pos = a.tok_pos[s], group = a.entry_group[s], shared = a.entry_pages[s];
        }
        const bool whole = shared_whole(pos, shared);
        const int n = slot < 0 ? 0 : max(0, pos / QF_PAGE + 1 - (whole ? shared : 0));
        if (s < a.n_seqs) p.own[s] = n;
        sum.x += n * p.own_tiles, sum.y += n > 0 ? p.own_tiles : 0;
        const bool member = slot >= 0 && group >= 0 && whole;
        const unsigned members = __ballot_sync(ALL, member);
        if (members == 0) continue;
        const int teller = __ffs(members) - 1, first = __shfl_sync(ALL, group, teller);
        if (__all_sync(ALL, !member || group == first)) {   // (mostly: a warp's members are of one group)
            const int a_slot = __reduce_max_sync(ALL, member ? slot : -1);
            if (lane == teller) atomicMax(p.slot + first, a_slot);
        } else if (member) {
            atomicMax(p.slot + group, slot);
        }
    }
    if (a.n_groups > 0) __syncthreads();
    for (int g = tid; g < a.n_groups; g += THREADS)
        if (p.slot[g] >= 0 && p.pages[g] > 0) {
            const int tiles = shared_tiles_of(a, p, g);
            if (shared_tiled(a, p, g)) sum.z += (p.pages[g] + 1) / 2 * tiles, sum.w += tiles;
            else sum.x += p.pages[g] * tiles, sum.y += tiles;
        }
    sum = make_uint4(__reduce_add_sync(ALL, sum.x), __reduce_add_sync(ALL, sum.y), __reduce_add_sync(ALL, sum.z), __reduce_add_sync(ALL, sum.w));
    if (lane == 0) sums_s[warp] = sum;
    __syncthreads();
    sum = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        const uint4 x = sums_s[w];
        sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
    }
    const float work = (float)sum.x * a.kv_heads, items = (float)sum.y * a.kv_heads;
    int warps = a.warps;
    p.together = 0x3fffffff, p.tile_share = 0.f;
    p.tiles = 0;
    if constexpr (TILES) {
        const float turns = (float)sum.z * a.kv_heads, pairs = (float)sum.w * a.kv_heads;
        // x SMs for the tiles, so that they end with the others: lag + tile_time / x = page_time / (sms - x)
        const float tile_time = turns * shared_turn_time(head_dim), page_time = work * shared_page_time(head_dim) + items * SH_RECORD_TIME;
        const float half = SH_TILE_LAG * a.sms - tile_time - page_time, x = (half + sqrtf(half * half + 4.f * SH_TILE_LAG * tile_time * a.sms)) / (2.f * SH_TILE_LAG);
        // (by a little less than the quotient, so that no rounding makes it one record more)
        const float shared_sms = work == 0.f ? (float)a.sms : fminf(fmaxf(floorf(x), 1.f), a.sms - 1.f);
        const float sms = turns == 0.f ? 0.f : shared_sms;   // (no tiles this time: what a graph's groups share now may be too little, or they have ended)
        if (turns > 0.f) p.tile_share = fmaxf(sms - pairs, 0.f) / turns * 0.9999f;
        warps = (int)fmaxf((float)gridDim.x - fmaxf(sms, pairs), 1.f) * WARPS;
        for (int g0 = 0; g0 < a.n_groups; g0 += 32) {   // every warp counts for itself
            const int g = g0 + lane;
            int run, parts = 0, mine = 0;
            const bool tiled = g < a.n_groups && shared_tiled(a, p, g);
            if (tiled) parts = shared_cut_group(a, p, g, run), mine = parts * shared_tiles_of(a, p, g);
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(ALL, upto, o);
                if (lane >= o) upto += x;
            }
            if (tiled && warp == 0) p.first[g] = p.tiles + upto - mine, p.parts[g] = parts;
            p.tiles += __shfl_sync(ALL, upto, 31);
        }
        if ((int)blockIdx.x < p.tiles * a.kv_heads && blockIdx.x != gridDim.x - 1) {
            __syncthreads();
            return p;
        }
    }
    p.each = max(1, (int)ceilf(work / (float)warps));
    if (a.team > 1) p.together = p.each * SH_TEAM;
    if (TILES && items <= (float)warps) {   // records for some sizes, a warp for each: the first that gives every record a warp
        for (int c = warp; c < SIZES; c += WARPS) {
            const int each = p.each + c;
            const float one = __fdividef(1.f, (float)each);
            int n = 0;
            for (int s = lane; s < a.n_seqs; s += 32) n += shared_div_up(p.own[s], each, one) * p.own_tiles;
            for (int g = lane; g < a.n_groups; g += 32)
                if (p.slot[g] >= 0 && !shared_tiled(a, p, g)) n += shared_div_up(p.pages[g], each, one) * shared_tiles_of(a, p, g);
            n = __reduce_add_sync(ALL, n);
            if (lane == 0) records_s[c] = n;
        }
        __syncthreads();
        int larger = 0;
        while (larger < SIZES - 1 && records_s[larger] * a.kv_heads > warps) ++larger;
        p.each += larger;
    }
    p.one_each = __fdividef(1.f, (float)p.each);
    // Where the other items' records begin: prefix sums of two counts, records for a warp and blocks' runs.
    int2 before = make_int2(0, 0);
    for (int i0 = 0; i0 < a.n_groups + a.n_seqs; i0 += THREADS) {
        const int i = i0 + tid, s = i - a.n_groups;
        int run, parts = 0;
        int2 mine = make_int2(0, 0);
        bool single = false;
        const bool tiled = TILES && s < 0 && shared_tiled(a, p, i);
        if (s < 0) {
            if (!tiled) {
                parts = shared_cut_group(a, p, i, run);
                single = p.pages[i] <= p.together;
                mine.x = parts * ((p.rows[i] + SH_ROW_TILE - 1) / SH_ROW_TILE);
            }
        } else if (s < a.n_seqs) {
            mine.x = shared_cut_own(a, p, s, run) * p.own_tiles;
            single = p.own[s] <= p.together;
        }
        if (!single) mine = make_int2(0, mine.x);
        int2 upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(ALL, upto.x, o), y = __shfl_up_sync(ALL, upto.y, o);
            if (lane >= o) upto.x += x, upto.y += y;
        }
        int2* const sums = counts_s[i0 / THREADS & 1];   // (the other half may still be read)
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        int2 at = make_int2(before.x + upto.x - mine.x, before.y + upto.y - mine.y);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const int2 x = sums[w];
            if (w < warp) at.x += x.x, at.y += x.y;
            before.x += x.x, before.y += x.y;
        }
        if (s < 0) {
            if (!tiled) p.first[i] = single ? at.x : at.y, p.parts[i] = parts;
        } else if (s < a.n_seqs) p.own_first[s] = single ? at.x : at.y;
    }
    p.singles = before.x, p.blocks = before.y;
    __syncthreads();
    return p;
}

// A record of a group's, the k-th.
__device__ __forceinline__ SharedRecord shared_group_record(const SharedArgs& a, const SharedPlan& p, int g, int k, int kind) {
    int run;
    shared_cut_group(a, p, g, run);
    const int chunk = shared_div(k, p.parts[g]), part = k - chunk * p.parts[g];
    const int end = min((part + 1) * run, p.pages[g]);
    return SharedRecord{SH_PREFIX | kind, g, chunk, p.slot[g], part * run, end, end * QF_PAGE, part, p.begin[g], p.rows[g], {0, 0}};
}
// Tile record `index`, which there is.
__device__ __forceinline__ SharedRecord shared_tile_record(const SharedArgs& a, const SharedPlan& p, int index) {
    int g = 0;
    while (g < a.n_groups - 1 && !(shared_tiled(a, p, g) && index >= p.first[g] && index < p.first[g] + p.parts[g] * shared_tiles_of(a, p, g))) ++g;
    return shared_group_record(a, p, g, index - p.first[g], 0);
}
// Records [index, index + N) of a kind (SH_TOGETHER: blocks' runs; 0: warps' records) into to[N]; by THREADS threads, this one the `tid`-th, which then
// synchronise. Records that there are none of are left as they were.
template <int THREADS, int N>
__device__ __forceinline__ void shared_records(const SharedArgs& a, const SharedPlan& p, int tid, int kind, int index, SharedRecord* to) {
    for (int g = tid; g < a.n_groups; g += THREADS) {
        if (shared_tiled(a, p, g)) continue;
        const int mine = p.pages[g] > p.together ? SH_TOGETHER : 0, n = p.parts[g] * shared_tiles_of(a, p, g), first = p.first[g];
        if (mine != kind || first >= index + N || first + n <= index) continue;
#pragma unroll
        for (int w = 0; w < N; ++w)
            if (index + w >= first && index + w < first + n) to[w] = shared_group_record(a, p, g, index + w - first, kind & SH_TOGETHER);
    }
    for (int s = tid; s < a.n_seqs; s += THREADS) {
        const int mine = p.own[s] > p.together ? SH_TOGETHER : 0, first = p.own_first[s];
        if (mine != kind || first >= index + N) continue;
        int run;
        const int parts = shared_cut_own(a, p, s, run), n = parts * p.own_tiles;
        if (first + n <= index) continue;
        const int pages = a.entry_pages[s], g = a.entry_group[s], shared = g >= 0 ? p.parts[g] : 0, pos = a.tok_pos[s];
        const int slot = a.slots[s], from = shared_whole(pos, pages) ? pages : 0;
#pragma unroll
        for (int w = 0; w < N; ++w) {
            const int k = index + w - first;
            if (k < 0 || k >= n) continue;
            const int chunk = shared_div(k, parts), part = k - chunk * parts;
            to[w] = SharedRecord{SH_OWN | kind, s, chunk, slot, from + part * run, from + min((part + 1) * run, p.own[s]), pos + 1, shared + part, 0, 0, {0, 0}};
        }
    }
}

// Which parts every row has, for whoever joins them: by one block of the parts' kernel.
template <int THREADS>
__device__ __forceinline__ void shared_count_parts(const SharedArgs& a, const SharedPlan& p) {
    for (int s = threadIdx.x; s < a.n_seqs; s += THREADS) {
        int run;
        const int g = a.entry_group[s], slot = a.slots[s], shared = g >= 0 ? p.parts[g] : 0, own = shared_cut_own(a, p, s, run);
        a.part_n[s] = slot < 0 ? 0 : shared_whole(a.tok_pos[s], a.entry_pages[s]) ? (shared + own) << 16 : shared | own << 16;
    }
}

// Row `at` of a record's subject: its place in q ([n_seqs * n_heads] rows of D), or -1 where there is no such row. (The rows of a member that has ended, or
// stands inside the shared pages, have a place too: nobody reads what is left there.)
__device__ __forceinline__ int shared_row(const SharedArgs& a, const SharedRecord& rec, int kv_heads, int kvh, int at) {
    const int G = a.n_heads / kv_heads;
    if (!(rec.kind & SH_PREFIX)) return at < G ? rec.subject * a.n_heads + kvh * G + at : -1;
    const int i = shared_div(at, G);
    return at < rec.rows ? a.members[rec.begin + i] * a.n_heads + kvh * G + at - i * G : -1;
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
// What bounds it: the latency of memory while a run is short (a page at head size 64 is two steps), then the rate at which pages arrive.
// Measured, the operator with plan and join: two sequences, 14 heads of 64 over 2, behind 16 pages 9.4 us; 8 behind 64 pages, up to 300 tokens of their
// own, 10.4 us (its 2.8 MB alone 0.43).
template <int D> struct SharedSums {
    float o[D / 8][4];       // o[t][0], o[t][1]: row g's columns 2 j E + t and (2 j + 1) E + t; o[t][2], o[t][3]: row g + 8's
    float m0, m1, l0, l1;    // rows g and g + 8: maximum and sum of weights
    int place0, place1;      // where they lie in q
    bool by_fragment;        // o[t] holds columns 8 t + 2 j and the next of both rows instead
    // 2 E columns of either row side by side
    __device__ __forceinline__ void leave(float* row0, float* row1, float f0, float f1) const {
        constexpr int E = D / 8;
        const int j = threadIdx.x & 3;
        if (by_fragment) {
#pragma unroll
            for (int t = 0; t < E; ++t) {
                if (row0) *reinterpret_cast<float2*>(row0 + 8 * t + 2 * j) = make_float2(o[t][0] * f0, o[t][1] * f0);
                if (row1) *reinterpret_cast<float2*>(row1 + 8 * t + 2 * j) = make_float2(o[t][2] * f1, o[t][3] * f1);
            }
            return;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < E; t += 4) {
                const int c = (2 * j + h) * E + t;
                if (row0) *reinterpret_cast<float4*>(row0 + c) = make_float4(o[t][h] * f0, o[t + 1][h] * f0, o[t + 2][h] * f0, o[t + 3][h] * f0);
                if (row1) *reinterpret_cast<float4*>(row1 + c) = make_float4(o[t][2 + h] * f1, o[t + 1][2 + h] * f1, o[t + 2][2 + h] * f1, o[t + 3][2 + h] * f1);
            }
    }
    // as a part of its own
    __device__ __forceinline__ void leave_part(const SharedArgs& a, int part) const {
        const size_t at0 = (size_t)place0 * a.most_parts + part, at1 = (size_t)place1 * a.most_parts + part;
        leave(place0 < 0 ? nullptr : a.part_o + at0 * D, place1 < 0 ? nullptr : a.part_o + at1 * D, 1.f, 1.f);
        if ((threadIdx.x & 3) == 0 && place0 >= 0) *reinterpret_cast<float2*>(a.part_ml + at0 * 2) = make_float2(m0, l0);
        if ((threadIdx.x & 3) == 0 && place1 >= 0) *reinterpret_cast<float2*>(a.part_ml + at1 * 2) = make_float2(m1, l1);
    }
};
// Bytes of shared memory that a warp needs for its queries: none where they are held in registers.
__host__ __device__ constexpr int shared_query_bytes(int d) { return d <= 64 ? 0 : 16 * d * 2; }

template <int D, int KEYS>
__device__ __forceinline__ void shared_warp(const bf16* __restrict__ q, const KvSite<bf16>& site, const SharedArgs& a, const SharedRecord& rec, int kvh,
                                            uint4* query_room, SharedSums<D>& out) {
    constexpr int SIX = KEYS / 16, STEPS = QF_PAGE / KEYS, KU = D / 32, E = D / 8, NT = E;
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3, kv_heads = site.kv_heads;
    const int p0 = rec.p_begin, p1 = rec.p_end, steps = STEPS * (p1 - p0), bound = rec.limit;
    const int* table_row = site.table + (long long)rec.slot * site.table_stride;
    int table = 0;   // a lane each the numbers of 32 pages
    uint4 k[2 * SIX][KU];          // n-tile t: key 8 t + g
    uint32_t v[4 * SIX][E / 2];    // of every 16 keys 2 j, 2 j + 1, 2 j + 8, 2 j + 9
    const bf16* k_at = nullptr;    // the step's keys (null: nothing to see there)
    auto find = [&](int i) {
        k_at = nullptr;
        if (i >= steps) return;
        const int n = i / STEPS, part = i % STEPS;
        if (n % 32 == 0 && part == 0) table = p0 + n + lane < p1 ? __ldg(table_row + p0 + n + lane) : 0;
        const int page = __shfl_sync(0xffffffffu, table, n & 31);
        if (page < 0) {
            if (lane == 0 && part == 0) atomicOr(a.err, QF_ERR_NO_PAGE);
            return;
        }
        if ((p0 + n) * QF_PAGE + KEYS * part >= bound) return;
        k_at = site.base + (long long)page * site.page_elems + ((long long)kvh * QF_PAGE + KEYS * part) * D;
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
    const int place0 = out.place0 = shared_row(a, rec, kv_heads, kvh, 16 * rec.chunk + g);
    const int place1 = out.place1 = shared_row(a, rec, kv_heads, kvh, 16 * rec.chunk + g + 8);
    // the queries' fragments: in registers, or, beyond head size 64, where keys, values and sums fill those, a lane's own 16 bytes at a time out of
    // shared memory
    constexpr bool HELD = shared_query_bytes(D) == 0;
    uint4 q_held[HELD ? KU : 1][2];
    uint4* const q_s = query_room + lane;
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
    float(&o)[NT][4] = out.o;
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    float m0 = QF_NEG_BIG, m1 = QF_NEG_BIG, l0 = 0.f, l1 = 0.f;   // (the sums are this lane's share)
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
            if (key0 + KEYS > bound) {   // values behind the last key are nobody's (0 times a NaN is not 0)
#pragma unroll
                for (int t = 0; t < 2 * SIX; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][e] = key0 + 8 * t + 2 * j + (e & 1) < bound ? s[t][e] * a.scale_log2 : QF_NEG_BIG;
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
    out.m0 = m0, out.m1 = m1, out.l0 = l0, out.l1 = l1;
    out.by_fragment = false;
}

// ---- the same work through shared memory, for the warps beside the tiles, of which an SM holds ten with half the registers: stages of 16 keys by 16-byte
// asynchronous copies, so that what is on its way does not take registers. A row's 16-byte pieces are stored at c XOR (row modulo 8): neither the copies
// nor ldmatrix meet a bank twice. Fragments as ldmatrix gives them.
// What bounds it: the latency of a warp's few stages, ten warps an SM. Measured: the own pages of 64 sequences, 28 heads of 128 over 4, 37 MB, on the 60 SMs
// that 88 tile records leave, 17 us, 2.1 TB/s.
__host__ __device__ constexpr int shared_stages(int d) { return d <= 64 ? 4 : 2; }
__host__ __device__ constexpr int shared_stage_bytes(int d) { return 2 * 16 * d * 2; }

template <int D>
__device__ __forceinline__ void shared_warp_staged(const bf16* __restrict__ q, const KvSite<bf16>& site, const SharedArgs& a, const SharedRecord& rec, int kvh,
                                                   unsigned char* room, SharedSums<D>& out) {
    constexpr int STAGES = shared_stages(D), BYTES = shared_stage_bytes(D), C = D / 8, KS = D / 16, NT = D / 8, STEPS = QF_PAGE / 16;
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3, kv_heads = site.kv_heads;
    const int p0 = rec.p_begin, p1 = rec.p_end, bound = rec.limit, steps = (min(bound, p1 * QF_PAGE) - p0 * QF_PAGE + 15) / 16;
    const int* table_row = site.table + (long long)rec.slot * site.table_stride;
    int table = 0;
    auto piece = [&](unsigned char* base, int r, int c) { return base + (r * C + (c ^ (r & 7))) * 16; };
    auto issue = [&](int i) {
        if (i < steps) {
            const int n = i / STEPS;
            if (i % (32 * STEPS) == 0) table = p0 + n + lane < p1 ? __ldg(table_row + p0 + n + lane) : 0;
            const int page = __shfl_sync(0xffffffffu, table, n & 31);
            unsigned char* keys = room + i % STAGES * BYTES;
            if (page < 0 && lane == 0 && i % STEPS == 0) atomicOr(a.err, QF_ERR_NO_PAGE);   // (reported; some held memory is read instead)
            const bf16* from = site.base + (long long)max(page, 0) * site.page_elems + ((long long)kvh * QF_PAGE + 16 * (i % STEPS)) * D;
            const bf16* values = from + (long long)kv_heads * QF_PAGE * D;
#pragma unroll
            for (int x = lane; x < 16 * C; x += 32) {
                cp_async_16(piece(keys, x / C, x % C), from + x * 8, true);
                cp_async_16(piece(keys + BYTES / 2, x / C, x % C), values + x * 8, true);
            }
        }
        cp_async_commit();   // one group per step, empty when there is nothing to fetch
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i);
    const int place0 = out.place0 = shared_row(a, rec, kv_heads, kvh, SH_ROW_TILE * rec.chunk + g);
    const int place1 = out.place1 = shared_row(a, rec, kv_heads, kvh, SH_ROW_TILE * rec.chunk + g + 8);
    uint32_t qa[KS][4];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int place = e & 1 ? place1 : place0;
            qa[ks][e] = place < 0 ? 0u : *reinterpret_cast<const uint32_t*>(q + (size_t)place * D + 16 * ks + 8 * (e >> 1) + 2 * j);
        }
    float(&o)[NT][4] = out.o;
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    float m0 = QF_NEG_BIG, m1 = QF_NEG_BIG, l0 = 0.f, l1 = 0.f;
    for (int i = 0; i < steps; ++i) {
        issue(i + STAGES - 1);
        cp_async_wait<STAGES - 1>();
        __syncwarp();   // each lane waited for its own copies; together the stage is complete
        unsigned char* keys = room + i % STAGES * BYTES;
        unsigned char* values = keys + BYTES / 2;
        const int key0 = p0 * QF_PAGE + 16 * i;
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint32_t kf[4];
            ldmatrix_x4(kf, piece(keys, (lane >> 4) * 8 + (lane & 7), 2 * ks + ((lane >> 3) & 1)));
            mma_bf16_16816(s[0], qa[ks], kf[0], kf[1]);
            mma_bf16_16816(s[1], qa[ks], kf[2], kf[3]);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] *= a.scale_log2;
        if (key0 + 16 > bound) {   // values behind the last key are nobody's (0 times a NaN is not 0)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (key0 + 8 * t + 2 * j + (e & 1) >= bound) s[t][e] = QF_NEG_BIG;
            for (int x = lane; x < 16 * C; x += 32)
                if (key0 + x / C >= bound) *reinterpret_cast<uint4*>(piece(values, x / C, x % C)) = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }
        float top0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), top1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
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
        const float from0 = m0 <= QF_NEG_BIG ? 0.f : m0, from1 = m1 <= QF_NEG_BIG ? 0.f : m1;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t][0] = fast_exp2(s[t][0] - from0), s[t][1] = fast_exp2(s[t][1] - from0);
            s[t][2] = fast_exp2(s[t][2] - from1), s[t][3] = fast_exp2(s[t][3] - from1);
            l0 += s[t][0] + s[t][1];
            l1 += s[t][2] + s[t][3];
        }
        const uint32_t p[4] = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]), pack_bf16(s[1][0], s[1][1]), pack_bf16(s[1][2], s[1][3])};
#pragma unroll
        for (int t = 0; t < NT; t += 2) {
            uint32_t vf[4];
            ldmatrix_x4_trans(vf, piece(values, ((lane >> 3) & 1) * 8 + (lane & 7), t + (lane >> 4)));
            mma_bf16_16816(o[t], p, vf[0], vf[1]);
            mma_bf16_16816(o[t + 1], p, vf[2], vf[3]);
        }
        __syncwarp();   // every lane has read this stage before the copies that come next overwrite it
    }
    cp_async_wait<0>();
    __syncwarp();
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    out.m0 = m0, out.m1 = m1, out.l0 = l0, out.l1 = l1;
    out.by_fragment = true;
}

// Batches without tiles: blocks of SH_TEAM warps, two an SM.
template <int D>
__global__ void __launch_bounds__(32 * SH_TEAM, 2)
shared_parts_kernel(const bf16* __restrict__ q, KvSite<bf16> site, SharedArgs a) {
    // Keys a step: 64 of head size 32, else 32. The operator with 64 / 32, one group of 8 sequences behind 64 pages, 70 tokens each of their own, microseconds:
    // head size 32 8.4 / 9.0, 64 11.4 / 10.4, 96 13.1 / 11.0 (two sequences behind one page: 8.0 / 8.1, 9.1 / 8.6, 12.0 / 9.8, 128 16.1 / 11.9).
    constexpr int KEYS = D <= 32 ? 64 : 32, LO = D + 4, THREADS = 32 * SH_TEAM;
    __shared__ __align__(16) float merge_s[SH_TEAM][16][LO];
    __shared__ float m_s[SH_TEAM][16], l_s[SH_TEAM][16];
    __shared__ SharedRecord record_s[SH_TEAM];
    extern __shared__ int plan_s[];
    static_assert(shared_query_bytes(D) <= (int)sizeof(merge_s[0]), "the queries lie where the sums will");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3, kv_heads = site.kv_heads;
    grid_launch_dependents();
    grid_dependency_wait();
    const SharedPlan plan = shared_plan<THREADS, false>(a, plan_s, D);
    if (blockIdx.x == 0) shared_count_parts<THREADS>(a, plan);
    const int units = (plan.blocks + (plan.singles + SH_TEAM - 1) / SH_TEAM) * kv_heads;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int kvh = unit % kv_heads, index = unit / kv_heads;
        const bool whole = index < plan.blocks;   // a block's run, or a record for each of its warps
        if (threadIdx.x < SH_TEAM) record_s[threadIdx.x].kind = SH_NONE;
        __syncthreads();
        if (whole) shared_records<THREADS, 1>(a, plan, threadIdx.x, SH_TOGETHER, index, record_s);
        else shared_records<THREADS, SH_TEAM>(a, plan, threadIdx.x, 0, (index - plan.blocks) * SH_TEAM, record_s);
        __syncthreads();
        SharedRecord rec = record_s[whole ? 0 : warp];
        __syncthreads();   // (the next unit writes these again)
        if (rec.kind & SH_NONE) continue;   // (the last warps of the last unit)
        if (whole) {   // this warp's share of the pages
            const int from = rec.p_begin, to = rec.p_end, per = (to - from + SH_TEAM - 1) / SH_TEAM;
            rec.p_begin = min(from + warp * per, to);
            rec.p_end = min(rec.p_begin + per, to);
        }
        SharedSums<D> x;
        shared_warp<D, KEYS>(q, site, a, rec, kvh, reinterpret_cast<uint4*>(&merge_s[warp][0][0]), x);
        if (!whole) {
            x.leave_part(a, rec.part);
            continue;
        }
        // the warps' sums come together in warp order
        if (j == 0) m_s[warp][g] = x.m0, m_s[warp][g + 8] = x.m1;
        __syncthreads();
        float top0 = m_s[0][g], top1 = m_s[0][g + 8];
#pragma unroll
        for (int w = 1; w < SH_TEAM; ++w) top0 = fmaxf(top0, m_s[w][g]), top1 = fmaxf(top1, m_s[w][g + 8]);
        const float f0 = fast_exp2(x.m0 - top0), f1 = fast_exp2(x.m1 - top1);
        if (j == 0) l_s[warp][g] = x.l0 * f0, l_s[warp][g + 8] = x.l1 * f1;
        x.leave(merge_s[warp][g], merge_s[warp][g + 8], f0, f1);
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * (D / 4); i += THREADS) {
            const int r = i / (D / 4), c = i % (D / 4) * 4, place = shared_row(a, rec, kv_heads, kvh, 16 * rec.chunk + r);
            if (place < 0) continue;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < SH_TEAM; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(&merge_s[w][r][c]);
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
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

// ---- any type and head size: float32 arithmetic. A block takes a record: 16 rows, a page at a time. Keys and values come in registers, all of a page's in
// flight at once and the next page's while this one's are at work, and go to shared memory as float32 (padded rows: eight keys' 16 bytes meet no bank
// twice). Thread = (key, every fourth row) for the scores, (row, 4 columns of every 64) for the sums.
// What bounds it: shared memory's reads, 5 of 16 bytes for 16 multiply-adds in the first product and 5 for 16 in the second; a short run, latency.
// Measured with the join, float32, head size 64, 14 heads over 2, 12 sequences behind 24 shared pages, each with up to 200 tokens of its own, and one alone: 19.0 us;
// with loads a page late and a key's row read once per query instead, 36.6.
#define SH_ROWS SH_ROW_TILE
#define SH_THREADS 256
// 4 columns from c of a row of D as float32: 16 bytes at once where `wide`, zeros behind the row's end.
template <typename T>
__device__ __forceinline__ float4 shared_four(const T* row, int c, int D, bool wide) {
    if constexpr (sizeof(T) == 4)
        if (wide) return c < D ? __ldg(reinterpret_cast<const float4*>(row + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
    return make_float4(c < D ? Num<T>::to_f(row[c]) : 0.f, c + 1 < D ? Num<T>::to_f(row[c + 1]) : 0.f, c + 2 < D ? Num<T>::to_f(row[c + 2]) : 0.f,
                       c + 3 < D ? Num<T>::to_f(row[c + 3]) : 0.f);
}

// UNITS: head sizes up to 64 UNITS.
template <typename T, int UNITS>
__global__ void __launch_bounds__(SH_THREADS)
shared_parts_generic_kernel(const T* __restrict__ q, KvSite<T> site, SharedArgs a, int wide) {
    extern __shared__ float4 fs[];
    constexpr int EACH = 4 * UNITS;               // fours of a row that a thread brings: columns 4 (tid % 4) + 16 i
    constexpr bool AHEAD = UNITS <= 2;            // beyond, there are no registers for a second page's values
    const int D = site.head_dim, LD = (D + 3) / 4 * 4 + 4;
    float* q_s = reinterpret_cast<float*>(fs);    // [16][LD]
    float* k_s = q_s + SH_ROWS * LD;              // [64][LD]
    float* v_s = k_s + QF_PAGE * LD;              // [64][LD]
    float* p_s = v_s + QF_PAGE * LD;              // [16][64 + 4]
    __shared__ int row_at[SH_ROWS];
    __shared__ float m_s[SH_ROWS], l_s[SH_ROWS], corr_s[SH_ROWS];
    __shared__ SharedRecord record_s;
    grid_launch_dependents();
    grid_dependency_wait();
    const SharedPlan plan = shared_plan<SH_THREADS, false>(a, reinterpret_cast<int*>(p_s + SH_ROWS * (QF_PAGE + 4)), D);
    if (blockIdx.x == 0) shared_count_parts<SH_THREADS>(a, plan);
    const int kv_heads = site.kv_heads, units = plan.singles * kv_heads, tid = threadIdx.x;
    const int their_row = tid / 4, their_col = tid % 4 * 4;   // what this thread brings of a page
    const int key = tid % 64, r0 = tid / 64;                  // its scores: rows r0 + 4 i
    const int my_row = tid / 16, my_col = tid % 16 * 4;       // its sums: columns my_col + 64 u
    const long long to_values = (long long)kv_heads * QF_PAGE * D;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {   // (a record is a block's work here)
        const int kvh = unit % kv_heads;
        shared_records<SH_THREADS, 1>(a, plan, tid, 0, unit / kv_heads, &record_s);
        __syncthreads();
        const SharedRecord rec = record_s;
        const int bound = rec.limit;
        const int* table_row = site.table + (long long)rec.slot * site.table_stride;
        float4 keys[EACH], values[AHEAD ? EACH : 1];
        // A row of a page: null where there is none to read (zeros then): behind the run, behind its last key, a page that is not held.
        auto row_of = [&](int p) -> const T* {
            if (p >= rec.p_end || p * QF_PAGE + their_row >= bound) return nullptr;
            const int page = table_row[p];
            return page < 0 ? nullptr : site.base + (long long)page * site.page_elems + ((long long)kvh * QF_PAGE + their_row) * D;
        };
        auto bring = [&](const T* row, float4* to) {
#pragma unroll
            for (int i = 0; i < EACH; ++i) to[i] = row ? shared_four(row, their_col + 16 * i, D, wide) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        auto put = [&](const float4* from, float* to) {
#pragma unroll
            for (int i = 0; i < EACH; ++i)
                if (their_col + 16 * i < LD - 4) *reinterpret_cast<float4*>(to + their_row * LD + their_col + 16 * i) = from[i];
        };
        const T* row = row_of(rec.p_begin);
        bring(row, keys);
        if (AHEAD) bring(row ? row + to_values : nullptr, values);
        if (tid < SH_ROWS) {
            row_at[tid] = shared_row(a, rec, kv_heads, kvh, SH_ROWS * rec.chunk + tid);
            m_s[tid] = QF_NEG_BIG;
            l_s[tid] = 0.f;
        }
        __syncthreads();
        {
            const int place = row_at[my_row];
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
                if (64 * u + my_col < LD - 4)
                    *reinterpret_cast<float4*>(q_s + my_row * LD + 64 * u + my_col) =
                        place < 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : shared_four(q + (size_t)place * D, 64 * u + my_col, D, wide);
        }
        float4 o[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = rec.p_begin; p < rec.p_end; ++p) {
            const T* here = row;
            const bool missing = table_row[p] < 0;
            if (missing && tid == 0) atomicOr(a.err, QF_ERR_NO_PAGE);
            put(keys, k_s);
            __syncthreads();
            row = row_of(p + 1);
            bring(row, keys);
            {
                float s[4] = {0.f, 0.f, 0.f, 0.f};
                for (int c = 0; c < LD - 4; c += 4) {
                    const float4 k4 = *reinterpret_cast<const float4*>(k_s + key * LD + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 q4 = *reinterpret_cast<const float4*>(q_s + (r0 + 4 * i) * LD + c);
                        s[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[i]))));
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    p_s[(r0 + 4 * i) * (QF_PAGE + 4) + key] = !missing && p * QF_PAGE + key < bound ? s[i] * a.scale_log2 : QF_NEG_BIG;
            }
            if (AHEAD) put(values, v_s);
            else {
                float4 now[AHEAD ? 1 : EACH];
                bring(here ? here + to_values : nullptr, now);
                put(now, v_s);
            }
            __syncthreads();
            if (AHEAD) bring(row ? row + to_values : nullptr, values);
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
                __syncwarp();   // (a row's 16 threads are half a warp: nobody else writes or reads its weights)
                if (tid % 16 == 0) {
                    const float corr = exp2f(m_old - m_new);
                    corr_s[my_row] = corr;
                    m_s[my_row] = m_new;
                    l_s[my_row] = l_s[my_row] * corr + sum;
                }
                __syncwarp();
            }
            const float corr = corr_s[my_row];
#pragma unroll
            for (int u = 0; u < UNITS; ++u) o[u].x *= corr, o[u].y *= corr, o[u].z *= corr, o[u].w *= corr;
#pragma unroll 4
            for (int k0 = 0; k0 < QF_PAGE; k0 += 4) {   // (rows behind the last key are zeros, and so are their weights)
                const float4 w4 = *reinterpret_cast<const float4*>(p_s + my_row * (QF_PAGE + 4) + k0);
                const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int u = 0; u < UNITS; ++u)
                        if (64 * u + my_col < LD - 4) {
                            const float4 v = *reinterpret_cast<const float4*>(v_s + (k0 + e) * LD + 64 * u + my_col);
                            o[u].x = fmaf(w[e], v.x, o[u].x), o[u].y = fmaf(w[e], v.y, o[u].y), o[u].z = fmaf(w[e], v.z, o[u].z), o[u].w = fmaf(w[e], v.w, o[u].w);
                        }
            }
        }
        const int place = row_at[my_row];
        if (place >= 0) {
            const size_t part = (size_t)place * a.most_parts + rec.part;
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const float v[4] = {o[u].x, o[u].y, o[u].z, o[u].w};
                const int c = 64 * u + my_col;
                if (D % 4 == 0 && c < D) *reinterpret_cast<float4*>(a.part_o + part * D + c) = o[u];
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < D) a.part_o[part * D + c + e] = v[e];
            }
            if (tid % 16 == 0) {
                a.part_ml[part * 2] = m_s[my_row];
                a.part_ml[part * 2 + 1] = l_s[my_row];
            }
        }
        __syncthreads();   // (the next unit writes these again)
    }
}

// ---- the parts of a row come together: V neighbouring output elements are a lane's, and of their parts every SPLIT-th, eight on their way at once.
// (No shared memory: the tiles' kernel behind, which wants all of it, may start its blocks beside these.)
// SPLIT 4 up to 256 elements' lanes an SM, else 2. The operator with 4 / 2 / 1, microseconds: 8 sequences, 14 heads of 64 11.2 / 12.2 / 12.8; 48, 16 heads of
// 128 18.2 / 19.6 / 22.0; beyond that, 64, 28 heads of 128 28.4 / 27.2 / 28.8; 250, 14 heads of 64 37.4 / 36.4 / 38.1 (the next call's blocks find room later).
// What bounds it: the latency of three dependent loads and a launch behind the parts; beyond some thousand rows, their bytes.
#define SH_JOIN 128   // threads of a block
template <typename T, int V, int SPLIT>
__global__ void __launch_bounds__(SH_JOIN)
shared_join_kernel(SharedArgs a, int D, T* __restrict__ out, const float* __restrict__ sinks) {
    constexpr int COLUMNS = 32 / SPLIT;
    grid_launch_dependents();
    const int split = (threadIdx.x & 31) / COLUMNS, entry = blockIdx.y, per = D / V, i = blockIdx.x * (SH_JOIN / SPLIT) + threadIdx.x / 32 * COLUMNS + threadIdx.x % COLUMNS;
    const int head = (int)((unsigned)i / (unsigned)per), d = (i - head * per) * V, row = entry * a.n_heads + head;
    const bool there = head < a.n_heads;
    grid_dependency_wait();
    const int packed = there ? a.part_n[entry] : 0, runs = packed >> 16;
    const size_t first = (size_t)row * a.most_parts + (packed & 0xffff);
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first;
    const float* po = a.part_o + first * D + d;
    float top = QF_NEG_BIG, den = 0.f, num[V];
#pragma unroll
    for (int e = 0; e < V; ++e) num[e] = 0.f;
    for (int k0 = split; k0 < runs; k0 += 8 * SPLIT) {
        float2 x[8];
        float o[8][V];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int part = k0 + k * SPLIT;
            const bool in = part < runs;
            x[k] = in ? ml[part] : make_float2(QF_NEG_BIG, 0.f);
            if constexpr (V == 4) {
                const float4 v = in ? *reinterpret_cast<const float4*>(po + (size_t)part * D) : make_float4(0.f, 0.f, 0.f, 0.f);
                o[k][0] = v.x, o[k][1] = v.y, o[k][2] = v.z, o[k][3] = v.w;
            } else {
                o[k][0] = in ? po[(size_t)part * D] : 0.f;
            }
        }
        float m = top;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, x[k].x);
        const float keep = fast_exp2(top - m);
        den *= keep;
#pragma unroll
        for (int e = 0; e < V; ++e) num[e] *= keep;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float w = fast_exp2(x[k].x - m);
            den = fmaf(w, x[k].y, den);
#pragma unroll
            for (int e = 0; e < V; ++e) num[e] = fmaf(w, o[k][e], num[e]);
        }
        top = m;
    }
    const float s2 = sinks && runs > 0 ? sinks[head] * 1.4426950408889634f : -INFINITY;   // a logit that joins the sum of weights once, with no key and no value
    float all = fmaxf(top, s2);
#pragma unroll
    for (int o = COLUMNS; o < 32; o <<= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    const float f = fast_exp2(top - all);
    den *= f;
#pragma unroll
    for (int e = 0; e < V; ++e) num[e] *= f;
#pragma unroll
    for (int o = COLUMNS; o < 32; o <<= 1) {
        den += __shfl_xor_sync(0xffffffffu, den, o);
#pragma unroll
        for (int e = 0; e < V; ++e) num[e] += __shfl_xor_sync(0xffffffffu, num[e], o);
    }
    if (split != 0 || !there) return;
    den += fast_exp2(s2 - all);
    const float inv = den > 0.f ? 1.f / den : 0.f;
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
static size_t shared_generic_smem(int d, int plan_ints) {
    const int ld = (d + 3) / 4 * 4 + 4;
    return (size_t)((SH_ROWS + 2 * QF_PAGE) * ld + SH_ROWS * (QF_PAGE + 4) + plan_ints) * sizeof(float);
}

// Where the tiles take over, unless the plan takes more shared memory than the warps beside them leave. Rows x pages, single warps / tiles, microseconds (one
// group, and 70 tokens of each sequence's own): head size 64, 448 x 16 12.1 / 12.6, 112 x 64 11.2 / 12.8, 168 x 64 14.1 / 14.5, 448 x 64 19.1 / 15.0, 1,792 x 8
// 17.6 / 14.1; head size 128, 70 x 8 13.6 / 13.7, 448 x 2 16.1 / 15.2, 112 x 8 15.6 / 13.8, 56 x 64 16.4 / 15.4, 448 x 16 21.1 / 15.7; 32 x 64 12.9 / 14.9.
#define SH_TILE_ROWS 48
#define SH_TILE_WORK_64 8192
#define SH_TILE_WORK_128 896

// What sizes the launches and the workspaces. sizes[0]: rows of a tile; [1]: warps (or blocks, of the kernel for any type) that run at once; [2]: warps of
// a block that bring their sums together; [3]: the most parts of an item; [4], [5]: a group of so many rows, and rows x pages, goes to the tiles (0: there are
// none), [7] if the plan takes no more than so many ints (2 a sequence, 6 a group); [6]: SMs.
QF_EXPORT int qf_attention_shared_shape(int is_bf16, int head_dim, int* sizes) {
    const int sms = qf_sm_count();
    if (sms <= 0 || head_dim <= 0 || head_dim > 256) return (int)cudaErrorInvalidValue;
    const bool fast = shared_fast(is_bf16, head_dim);
    sizes[0] = SH_ROW_TILE;
    sizes[1] = fast ? 2 * SH_TEAM * sms : 2 * sms;
    sizes[2] = fast ? SH_TEAM : 1;
    sizes[3] = 64;
    sizes[4] = fast && (head_dim == 64 || head_dim == 128) ? SH_TILE_ROWS : 0;
    sizes[5] = head_dim == 64 ? SH_TILE_WORK_64 : SH_TILE_WORK_128;
    sizes[6] = sms;
    sizes[7] = SH_TILE_PLAN_INTS;
    return 0;
}

template <int D>
static int launch_parts(const void* q, KvSite<bf16> site, const SharedArgs& a, int units, cudaStream_t stream) {
    const int at_once = 2 * qf_sm_count(), smem = shared_plan_ints(a.n_seqs, a.n_groups) * (int)sizeof(int);
    auto kernel = shared_parts_kernel<D>;
    if (smem > 8 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_plan_ints(SH_MAX_SEQS, SH_MAX_SEQS) * (int)sizeof(int));
        if (e != cudaSuccess) return (int)e;
    }
    return (int)launch_pdl(kernel, dim3((unsigned)(units < at_once ? units : at_once)), dim3(32 * SH_TEAM), (size_t)smem, stream, (const bf16*)q, site, a);
}

template <typename T, int UNITS>
static int launch_generic(const void* q, KvSite<T> site, const SharedArgs& a, int units, cudaStream_t stream) {
    const size_t smem = shared_generic_smem(site.head_dim, shared_plan_ints(a.n_seqs, a.n_groups));
    if (smem > 227 * 1024) return (int)cudaErrorInvalidValue;
    auto kernel = shared_parts_generic_kernel<T, UNITS>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
    if (e != cudaSuccess) return (int)e;
    const int at_once = 2 * qf_sm_count();
    const bool wide = sizeof(T) == 4 && site.head_dim % 4 == 0 && site.page_elems % 4 == 0 && reinterpret_cast<uintptr_t>(site.base) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(q) % 16 == 0;
    return (int)launch_pdl(kernel, dim3((unsigned)(units < at_once ? units : at_once)), dim3(SH_THREADS), smem, stream, (const T*)q, site, a, (int)wide);
}
template <typename T>
static int launch_generic(const void* q, KvSite<T> site, const SharedArgs& a, int units, cudaStream_t stream) {
    return site.head_dim <= 64 ? launch_generic<T, 1>(q, site, a, units, stream) : site.head_dim <= 128 ? launch_generic<T, 2>(q, site, a, units, stream)
                                                                                                        : launch_generic<T, 4>(q, site, a, units, stream);
}

template <typename T, int V, int SPLIT>
static int launch_join(const SharedArgs& a, int head_dim, void* out, const float* sinks, cudaStream_t stream) {
    const long long items = (long long)a.n_heads * (head_dim / V);
    const dim3 grid((unsigned)((items * SPLIT + SH_JOIN - 1) / SH_JOIN), (unsigned)a.n_seqs);
    return (int)launch_pdl(shared_join_kernel<T, V, SPLIT>, grid, dim3(SH_JOIN), 0, stream, a, head_dim, (T*)out, sinks);
}
template <typename T>
static int launch_join(const SharedArgs& a, int head_dim, void* out, const float* sinks, cudaStream_t stream) {
    if (head_dim % 4 || (reinterpret_cast<uintptr_t>(out) & 15)) return launch_join<T, 1, 1>(a, head_dim, out, sinks, stream);
    const bool few = (long long)a.n_seqs * a.n_heads * head_dim / 4 <= 256ll * a.sms;
    return few ? launch_join<T, 4, 4>(a, head_dim, out, sinks, stream) : launch_join<T, 4, 2>(a, head_dim, out, sinks, stream);
}

// `most_units`, `most_tiles`: bounds of the blocks' runs with the groups of SH_TEAM warps' records, and of the tile records that cannot be cut into fewer, of
// one kv head (0: no group is given to the tiles); `most_shared`, `most_own`: the most parts that a row has room for of each; part_o, part_ml: n_seqs * n_heads * (most_shared +
// most_own) * head_dim and * 2 floats; part_n: n_seqs ints.
QF_EXPORT int qf_attention_shared(int is_bf16, const void* q, void* out, const int* tok_pos, const int* slots, const int* entry_pages,
                                  const int* entry_group, const int* members, const int* begin, const int* pages, int n_groups, int most_units,
                                  int most_tiles, int most_shared, int most_own, void* base, const int* table, long long page_elems, int table_stride,
                                  int kv_heads, int head_dim, int n_heads, int n_seqs, float scale, float* part_o, float* part_ml, int* part_n,
                                  const float* sinks, int* err, cudaStream_t stream) {
    int sizes[8];
    if (n_seqs <= 0 || n_seqs > SH_MAX_SEQS || n_groups > n_seqs || kv_heads <= 0 || n_heads % kv_heads || most_units <= 0 || most_own <= 0 || most_own > 0x7fff ||
        most_shared > 0x7fff - most_own || (n_groups > 0 && most_shared <= 0))
        return (int)cudaErrorInvalidValue;
    const int bad = qf_attention_shared_shape(is_bf16, head_dim, sizes);
    if (bad) return bad;
    const SharedArgs a = {tok_pos, slots, entry_pages, entry_group, members, begin, pages, part_o, part_ml, part_n, err, n_seqs, n_groups, n_heads, kv_heads,
                          most_shared + most_own, most_shared, most_own, sizes[1], most_tiles > 0 ? 1 : sizes[2], most_tiles > 0 ? sizes[4] : 0, sizes[5], sizes[6],
                          scale * 1.4426950408889634f};
    const bool fast = shared_fast(is_bf16, head_dim);
    if (most_tiles > 0 && (!fast || shared_plan_ints(n_seqs, n_groups) > SH_TILE_PLAN_INTS)) return (int)cudaErrorInvalidValue;
    const long long all = (long long)most_units * kv_heads * (fast ? 1 : SH_TEAM);
    const int units = (int)(all < 0x7fffffff ? all : 0x7fffffff);
    int code;
    if (fast) {
        const KvSite<bf16> site{(bf16*)base, table, page_elems, table_stride, kv_heads, head_dim};
        if (most_tiles > 0)
            code = head_dim == 64 ? launch_tiles<64>(q, site, a, most_tiles, stream) : head_dim == 128 ? launch_tiles<128>(q, site, a, most_tiles, stream)
                                                                                                       : (int)cudaErrorInvalidValue;
        else
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
