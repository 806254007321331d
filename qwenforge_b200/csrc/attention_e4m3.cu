// Attention of single tokens, and of short spans of tokens, over a sequence cache of e4m3 codes (the format: e4m3.cuh).
//
//   o = softmax_j(q k_j^T scale) v_j over the keys j that the token sees: max(0, p - window + 1) <= j <= p
//
// The codes are multiplied as float16, in which they are exact, with float32 sums. A page's power of two for the keys is a factor of its scores; that
// for the values is the unit in which a row's sum of outputs is kept while the page adds to it (an exact shift where the next page's differs).
// Queries become float16 behind a power of two per row that brings their largest element to 2^7 .. 2^8: bfloat16 queries lose nothing but
// what lies 2^-31 below that, float32 queries are two such numbers (22 bits) and take two products. Weights are 2^(s - m + 14), at most 2^14
// for the running maximum m: rounded to float16 (2^-12 of each weight, less than the output's own rounding) where the output is bfloat16, two
// numbers where it is float32. Maxima, sums and outputs are float32; for float32 outputs the tensor cores' sums end with a tile (they cut bits off).
//
// A block takes pages of a (sequence, kv head, 16 rows), its warps a page each in turn; a warp looks its next 32 pages and their scales up at once. A row is a query head of the kv head's
// group and a token of the span; 16 of them are the rows of m16n8k16 products, whose columns are keys, then components. No shared memory
// lies on the way of the codes: a lane loads what its fragments hold. For the keys, columns are 8 positions and a lane takes D / 4
// components of one of them, 16 bytes at a time (which components a product's steps go through is free, as long as the queries'
// fragments go through the same). For the values a lane takes D / 8 neighbouring components of the four positions that a step wants
// of it, and byte t of them is its element of the t-th product: a byte permutation puts two positions side by side for the conversion.
// A tile's values are on their way while its scores are formed, the next tile's keys from then on.
//
// Work is shared out on the device, from the lengths (a captured graph replays this launch with others): all pages of all (sequence, kv head,
// 16 rows) in a row, `target` of them to a block, so that one round of blocks does it all. Where every pair's pages can be rounded up to
// whole blocks within that round, they are, and a block has one pair; else blocks begin and end anywhere, and lengths that
// differ leave no SM idle. A pair of several blocks leaves partial results (maximum, sum, output); the block that ends last, by a
// ticket, joins them in their order, sixteen at a time, and the last of those the sixteens.
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "e4m3.cuh"

#define EA_WARPS 4
#define EA_ROWS 16
#define EA_NONE (-3.0e38f)   // the running maximum of a row that has seen nothing

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// what float16 leaves over of two numbers
__device__ __forceinline__ uint32_t pack_rest(float lo, float hi, uint32_t taken) {
    const float2 t = floats_of(taken);
    return pack_half(lo - t.x, hi - t.y);
}
__device__ __forceinline__ uint4 load16(const void* p) {   // (codes are read once: past L1)
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load8(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load4(const void* p) {
    uint32_t v;
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load2(const void* p) {
    uint16_t v;
    asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}

// A row of D components in parts of 128, 64, 32 and 16 that fragments go through one after another.
template <int D> struct Parts {
    // keys: a lane's words (four codes, one step of 16 components each) are D / 16; those of part 64 first
    static constexpr int k64 = D / 64, k32 = (D % 64) / 32, k16 = (D % 32) / 16, k_words = D / 16;
    // values: bytes of a lane from part 128, 64, 32, 16: 16, 8, 4, 2
    static constexpr int v128 = D / 128, v64 = (D % 128) / 64, v32 = (D % 64) / 32, v16 = (D % 32) / 16;
    static constexpr int v_words = 4 * v128 + 2 * v64 + v32 + v16;   // (16 fills half a word)
};
// First component of a lane's key word w (quad column c).
template <int D> __device__ __forceinline__ constexpr int key_component(int w, int c) {
    using P = Parts<D>;
    if (w < 4 * P::k64) return 64 * (w / 4) + 16 * c + 4 * (w % 4);
    w -= 4 * P::k64;
    if (w < 2 * P::k32) return 64 * P::k64 + 8 * c + 4 * w;
    return 64 * P::k64 + 32 * P::k32 + 4 * c;
}
// The component that product t (of D / 8) has in its column n.
template <int D> __device__ __forceinline__ int value_component(int t, int n) {
    using P = Parts<D>;
    int base = 0;
    if (t < 16 * P::v128) return 16 * n + t;
    t -= 16 * P::v128, base += 128 * P::v128;
    if (t < 8 * P::v64) return base + 8 * n + t;
    t -= 8 * P::v64, base += 64 * P::v64;
    if (t < 4 * P::v32) return base + 4 * n + t;
    t -= 4 * P::v32, base += 32 * P::v32;
    return base + 2 * n + t;
}
template <int D> __device__ __forceinline__ void load_key(uint32_t (&w)[D / 16], const unsigned char* row, int c) {
    using P = Parts<D>;
#pragma unroll
    for (int i = 0; i < P::k64; ++i) {
        const uint4 v = load16(row + 64 * i + 16 * c);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
    if constexpr (P::k32 != 0) {
        const uint2 v = load8(row + 64 * P::k64 + 8 * c);
        w[4 * P::k64] = v.x, w[4 * P::k64 + 1] = v.y;
    }
    if constexpr (P::k16 != 0) w[4 * P::k64 + 2 * P::k32] = load4(row + 64 * P::k64 + 32 * P::k32 + 4 * c);
}
template <int D> __device__ __forceinline__ void load_value(uint32_t (&w)[Parts<D>::v_words], const unsigned char* row, int g) {
    using P = Parts<D>;
    int at = 0, o = 0;
    if constexpr (P::v128 != 0) {
        const uint4 v = load16(row + 16 * g);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        at += 128, o += 4;
    }
    if constexpr (P::v64 != 0) {
        const uint2 v = load8(row + at + 8 * g);
        w[o] = v.x, w[o + 1] = v.y;
        at += 64, o += 2;
    }
    if constexpr (P::v32 != 0) {
        w[o] = load4(row + at + 4 * g);
        at += 32, o += 1;
    }
    if constexpr (P::v16 != 0) w[o] = load2(row + at + 2 * g);
}
__device__ __forceinline__ bool holds_nan(uint32_t codes) { return __vcmpeq4(codes & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0; }

template <typename T, int D> struct Shape {
    static constexpr bool TWO = sizeof(T) == 4;                       // float32: queries and weights as two float16 each
    static constexpr int TILE = D <= 64 ? (TWO ? 32 : 64) : (TWO && D > 96 ? 16 : 32);   // positions of a step
    static constexpr int BLOCKS = D <= 32 ? 3 : 2;                    // of an SM
    // floats from a row to the next where warps leave their outputs: product t's column n at 8 t + 8 (t / 4) + n, so that four products of 32 lanes
    // meet 32 banks; rows 8 or 24 banks apart, for the warps' own stores
    static constexpr int ROW = D + 8 * ((D / 8 + 3) / 4), LD = ROW % 32 == 8 || ROW % 32 == 24 ? ROW : ROW + 8;
    static constexpr int SMEM = EA_WARPS * EA_ROWS * LD * 4;
    static constexpr int PART = 32 * Parts<D>::v_words;               // floats of a row of a partial result
};

struct AttendArgs {
    const int *cu_q, *tok_pos, *slots;
    E4m3Site site;
    int n_heads, n_seqs, single, chunks, most_pages, block_slots, window;
    float scale_log2;
    float *part_o, *part_ml;   // [2 * blocks][16][PART], [2 * blocks][16][2]
    int *tickets, *err;        // [4 * blocks]
};

struct Sequence {
    int slot, begin, tokens, first_pos, last_pos, page0, pages;
};
__device__ __forceinline__ Sequence sequence_of(const AttendArgs& a, int s) {
    Sequence r;
    r.begin = a.single ? s : a.cu_q[s];   // (single: every entry has one token)
    r.tokens = a.single ? 1 : a.cu_q[s + 1] - r.begin;
    r.slot = r.tokens > 0 ? a.slots[s] : -1;
    r.first_pos = r.last_pos = r.page0 = r.pages = 0;
    if (r.tokens > 0) {
        r.first_pos = a.tok_pos[r.begin];
        r.last_pos = a.single ? r.first_pos : a.tok_pos[r.begin + r.tokens - 1];
    }
    if (r.slot >= 0) {
        r.page0 = a.window > 0 ? max(0, r.first_pos - a.window + 1) / QF_PAGE : 0;
        r.pages = min(max(r.last_pos / QF_PAGE - r.page0 + 1, 0), a.most_pages);   // (more than the call has said: cut, and reported)
    }
    return r;
}

template <typename T> __device__ __forceinline__ void store4(T* to, const float (&v)[4], int n) {
    if constexpr (sizeof(T) == 4) {
        if (n == 4) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<float2*>(to) = make_float2(v[0], v[1]);
    } else {
        if (n == 4) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
        else *reinterpret_cast<uint32_t*>(to) = pack_bf16(v[0], v[1]);
    }
}

// x * 2^e, e of any size that the result has room for
__device__ __forceinline__ float scaled(float x, int e) { return x * pow2(e / 2) * pow2(e - e / 2); }

#define EA_PAIR_COST 8     // pages whose time a pair's beginning and end take
#define EA_GROUP 16        // partial results that a block joins at once
#define EA_SHARE (EA_WARPS * 32 / EA_ROWS)
#define EA_MOST_GROUPS 64  // ... and groups of them: enough for 1,024 blocks

template <typename T, int D>
__global__ void __launch_bounds__(EA_WARPS * 32, Shape<T, D>::BLOCKS)
attend_e4m3_kernel(const T* __restrict__ q, T* __restrict__ out, const AttendArgs a) {
    using S = Shape<T, D>;
    using P = Parts<D>;
    constexpr bool TWO = S::TWO;
    constexpr int TILE = S::TILE, NT = TILE / 8, KT = TILE / 16, OT = D / 8, KW = P::k_words, VW = P::v_words, LD = S::LD, PART = S::PART;
    constexpr int PER_PAGE = QF_PAGE / TILE, THREADS = EA_WARPS * 32;
    grid_chain_entry();
    extern __shared__ float shared_o[];   // [warps][rows][LD]
    __shared__ float m_s[EA_WARPS][EA_ROWS], l_s[EA_WARPS][EA_ROWS], total_s[EA_ROWS], factor_s[EA_MOST_GROUPS][EA_ROWS];
    __shared__ int ticket_s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const E4m3Site& site = a.site;
    const int KVH = site.kv_heads, G = a.n_heads / KVH, pairs_each = KVH * a.chunks;
    const int q_width = a.n_heads * D, n_blocks = gridDim.x;

    // ---- this block's share (every warp works it out for itself)
    int total = 0, pairs = 0, whole = 0, target = EA_WARPS;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
        const int pages = s0 + lane < a.n_seqs ? sequence_of(a, s0 + lane).pages : 0;
        total += pages;
        pairs += pages > 0;
    }
    total = (int)warp_sum_u32((uint32_t)total) * pairs_each;
    pairs = (int)warp_sum_u32((uint32_t)pairs) * pairs_each;
    target = max(target, (total + a.block_slots - 1) / a.block_slots);
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) whole += s0 + lane < a.n_seqs ? (sequence_of(a, s0 + lane).pages + target - 1) / target : 0;
    whole = (int)warp_sum_u32((uint32_t)whole) * pairs_each;
    // pages of a pair are rounded up to whole units; where blocks may have several pairs, each counts EA_PAIR_COST pages more
    const bool aligned = whole <= a.block_slots;
    const int ahead = aligned ? 0 : EA_PAIR_COST;
    if (aligned) {
        total = whole * target;
    } else {
        total += pairs * ahead;
        target = max(target, (total + a.block_slots - 1) / a.block_slots);
    }
    auto places_of = [&](int pages) { return pages == 0 ? 0 : aligned ? (pages + target - 1) / target * target : pages + ahead; };
    // padding entries: zeros
    for (int s = blockIdx.x; s < a.n_seqs; s += n_blocks) {
        const Sequence r = sequence_of(a, s);
        if (r.slot < 0)
            for (int i = threadIdx.x; i < r.tokens * q_width; i += THREADS) out[(long long)r.begin * q_width + i] = Num<T>::from_f(0.f);
    }
    const int range_begin = blockIdx.x * target, range_end = min(range_begin + target, total);
    if (range_begin >= range_end) return;
    // the sequence in whose pages it begins
    int seq = 0, base = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
        const int mine = s0 + lane < a.n_seqs ? places_of(sequence_of(a, s0 + lane).pages) * pairs_each : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t beyond = __ballot_sync(0xffffffffu, base + upto > range_begin);
        if (beyond) {
            const int who = __ffs(beyond) - 1;
            seq = s0 + who;
            base += __shfl_sync(0xffffffffu, upto - mine, who);
            break;
        }
        base += __shfl_sync(0xffffffffu, upto, 31);
    }

    Sequence r = sequence_of(a, seq);
    int padded = places_of(r.pages);
    for (int at = range_begin; at < range_end;) {
        while (at >= base + padded * pairs_each) {   // (sequences without pages are passed over)
            base += padded * pairs_each;
            r = sequence_of(a, ++seq);
            padded = places_of(r.pages);
        }
        const int y = (at - base) / padded, pair_begin = base + y * padded, kvh = y / a.chunks, chunk = y % a.chunks;
        const int p_begin = r.page0 + max(at - pair_begin - ahead, 0), p_end = r.page0 + min(min(padded, range_end - pair_begin) - ahead, r.pages);
        const bool reports = y == 0 && threadIdx.x == 0 && at == pair_begin;
        at = min(pair_begin + padded, range_end);
        if (reports && r.last_pos / QF_PAGE - r.page0 + 1 > r.pages) atomicOr(a.err, QF_ERR_POSITION_RANGE);
        const int row0 = chunk * EA_ROWS, n_rows = min(EA_ROWS, r.tokens * G - row0);   // rows: token * G + head of the group
        if (n_rows <= 0 || p_begin >= p_end) continue;
        // element 0 of a row's query (and output)
        auto row_at = [&](int row) -> long long {
            const int i = row0 + row;
            return (long long)(r.begin + i / G) * q_width + (long long)(kvh * G + i % G) * D;
        };
        const int my_pages = p_begin + warp < p_end ? (p_end - p_begin - warp + EA_WARPS - 1) / EA_WARPS : 0;
        // what the rows see, lo .. hi - 1: this lane's two, all of them together, every one of them
        const int t_first = row0 / G, t_last = (row0 + n_rows - 1) / G;
        const int first_hi = (t_first == 0 ? r.first_pos : a.tok_pos[r.begin + t_first]) + 1, some_hi = (a.single ? r.first_pos : a.tok_pos[r.begin + t_last]) + 1;
        const int some_lo = a.window > 0 ? max(0, first_hi - a.window) : 0, all_lo = a.window > 0 ? max(0, some_hi - a.window) : 0;
        int lo[2], hi[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = g + 8 * e;
            hi[e] = row >= n_rows ? 0 : t_first == t_last ? first_hi : a.tok_pos[r.begin + (row0 + row) / G] + 1;
            lo[e] = a.window > 0 ? max(0, hi[e] - a.window) : 0;
        }

        // ---- keys of a step: pages p_begin + warp, + EA_WARPS, ..., a tile of one at a time
        const int steps = my_pages * PER_PAGE;
        const long long plane = (long long)KVH * QF_PAGE * D;
        int lane_page = -1, lane_unit = 0;   // of 32 of the warp's pages, one a lane: its number, its scales
        float lane_scale = 0.f;
        int page_next = -1, unit_next = 0;   // of the step whose keys are loaded
        float ks_next = 0.f;
        uint32_t kw[NT][KW];
        auto key0_of = [&](int step) { return (p_begin + warp + step / PER_PAGE * EA_WARPS) * QF_PAGE + step % PER_PAGE * TILE; };
        auto look_up = [&](int from) {   // pages from .. from + 31 of the warp's
            lane_page = -1;
            if (from + lane < my_pages) {
                lane_page = e4m3_page(site, r.slot, (p_begin + warp + (from + lane) * EA_WARPS) * QF_PAGE);
                if (lane_page < 0) {
                    if (y == 0) atomicOr(a.err, QF_ERR_NO_PAGE);
                } else {
                    const float* scales = site.scales + (long long)lane_page * site.page_scales + kvh;
                    lane_scale = scales[0];
                    lane_unit = exponent_of(scales[KVH]);
                }
            }
        };
        auto load_keys = [&](int step) {
            const int key0 = key0_of(step);
            if (step % PER_PAGE == 0) {
                const int i = step / PER_PAGE;
                if (i % 32 == 0) look_up(i);
                page_next = __shfl_sync(0xffffffffu, lane_page, i % 32);
                ks_next = __shfl_sync(0xffffffffu, lane_scale, i % 32);
                unit_next = __shfl_sync(0xffffffffu, lane_unit, i % 32);
            }
            if (page_next < 0 || key0 >= some_hi || key0 + TILE <= some_lo) return;
            const unsigned char* k = site.codes + (long long)page_next * site.page_bytes + ((long long)kvh * QF_PAGE + step % PER_PAGE * TILE + g) * D;
#pragma unroll
            for (int t = 0; t < NT; ++t) load_key<D>(kw[t], k + t * 8 * D, c);
        };
        if (steps > 0) load_keys(0);

        // ---- the queries' fragments
        uint32_t qa[TWO ? 2 : 1][KW][4];
        float by[2];   // scores of a row in base-2 units: product * key scale * by
        {
            float2 x[2][KW][2];
            float top[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = g + 8 * e;
                const T* src = q + (row < n_rows ? row_at(row) : 0);
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    const int d = key_component<D>(w, c);
                    x[e][w][0] = x[e][w][1] = make_float2(0.f, 0.f);
                    if (row < n_rows) {
                        if constexpr (TWO) {
                            const float4 v = *reinterpret_cast<const float4*>(src + d);
                            x[e][w][0] = make_float2(v.x, v.y), x[e][w][1] = make_float2(v.z, v.w);
                        } else {
                            const uint2 v = *reinterpret_cast<const uint2*>(src + d);
                            x[e][w][0] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x));
                            x[e][w][1] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) top[e] = fmaxf(top[e], fmaxf(fabsf(x[e][w][i].x), fabsf(x[e][w][i].y)));
                }
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
                const int up = min(max(exponent_of(top[e]) - 7, -119), 120);
                by[e] = pow2(up) * fabsf(a.scale_log2);
                const float down = copysignf(pow2(-up), a.scale_log2);
#pragma unroll
                for (int w = 0; w < KW; ++w)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float u = x[e][w][i].x * down, v = x[e][w][i].y * down;
                        qa[0][w][2 * i + e] = pack_half(u, v);
                        if constexpr (TWO) qa[1][w][2 * i + e] = pack_rest(u, v, qa[0][w][2 * i + e]);
                    }
            }
        }

        float o[OT][4];
#pragma unroll
        for (int i = 0; i < OT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m_run[2] = {EA_NONE, EA_NONE}, l_run[2] = {0.f, 0.f};   // (l: this lane's columns only)
        int unit_run[2] = {0, 0};                                      // o stands for o * 2^unit_run
        bool begun = false;

        for (int step = 0; step < steps; ++step) {
            const int page = page_next, key0 = key0_of(step), unit_v = unit_next;
            const float ks = ks_next;
            if (page < 0 || key0 >= some_hi || key0 + TILE <= some_lo) {
                if (step + 1 < steps) load_keys(step + 1);
                continue;
            }
            if (!begun) unit_run[0] = unit_run[1] = unit_v;
            begun = true;
            // ---- this tile's values: positions 16 kt + 2 c, + 1, + 8, + 9
            uint32_t vw[KT][4][VW];
            {
                const unsigned char* v = site.codes + (long long)page * site.page_bytes + plane + ((long long)kvh * QF_PAGE + step % PER_PAGE * TILE + 2 * c) * D;
                if (key0 >= some_lo && key0 + TILE <= some_hi) {   // every position is held, and seen by some row
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) load_value<D>(vw[kt][i], v + (16 * kt + (i & 1) + 8 * (i >> 1)) * D, g);
                } else {
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int at = 16 * kt + (i & 1) + 8 * (i >> 1), key = key0 + at + 2 * c;
#pragma unroll
                            for (int w = 0; w < VW; ++w) vw[kt][i][w] = 0u;   // (what lies elsewhere is nobody's, NaN perhaps)
                            if (key >= some_lo && key < some_hi) load_value<D>(vw[kt][i], v + at * D, g);
                        }
                }
            }
            // ---- scores
            float s[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
            for (int w = 0; w < KW; ++w)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint32_t b0 = half2_of_low(kw[t][w]), b1 = half2_of_high(kw[t][w]);
                    if constexpr (TWO) mma_f16_16816(s[t], qa[1][w], b0, b1);
                    mma_f16_16816(s[t], qa[0][w], b0, b1);
                }
            if (step + 1 < steps) load_keys(step + 1);
            // ---- weights. What a row does not see is EA_NONE on the way to the maximum, and has none
            const float by_k[2] = {by[0] * ks, by[1] * ks};
            const bool full = key0 >= all_lo && key0 + TILE <= first_hi;
            auto seen = [&](int t, int e) {
                const int key = key0 + 8 * t + 2 * c + (e & 1);
                return key >= lo[e >> 1] && key < hi[e >> 1];
            };
            float top[2] = {EA_NONE, EA_NONE}, corr[2], shift[2];
            if (full) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[t][e]);
            } else {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (seen(t, e)) top[e >> 1] = fmaxf(top[e >> 1], s[t][e]);
            }
            float m_tile[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
                m_tile[e] = top[e] > EA_NONE ? top[e] * by_k[e] : EA_NONE;
                const float m = fmaxf(m_run[e], m_tile[e]);
                corr[e] = fast_exp2(m_run[e] - m);
                m_run[e] = m;
                shift[e] = 14.f - m;
                l_run[e] *= corr[e];
            }
            uint32_t pa[TWO ? 2 : 1][KT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[t][e] = fast_exp2(fmaf(s[t][e], by_k[e >> 1], shift[e >> 1]));
                    if (!full && !seen(t, e)) s[t][e] = 0.f;
                    l_run[e >> 1] += s[t][e];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    pa[0][t / 2][2 * (t % 2) + e] = pack_half(s[t][2 * e], s[t][2 * e + 1]);
                    if constexpr (TWO) pa[1][t / 2][2 * (t % 2) + e] = pack_rest(s[t][2 * e], s[t][2 * e + 1], pa[0][t / 2][2 * (t % 2) + e]);
                }
            }
            // ---- values. Word w of the four positions of a step holds their elements of the products 4 w .. 4 w + 3
            auto word_products = [&](int kt, int w, auto take, auto add) {
                uint32_t x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = take(vw[kt][i][w], 16 * kt + 2 * c + (i & 1) + 8 * (i >> 1));
                const uint32_t u[2] = {__byte_perm(x[0], x[1], 0x5140), __byte_perm(x[0], x[1], 0x7362)};
                const uint32_t v[2] = {__byte_perm(x[2], x[3], 0x5140), __byte_perm(x[2], x[3], 0x7362)};
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if (P::v16 != 0 && w == VW - 1 && t >= 2) break;
                    add(t, t & 1 ? half2_of_high(u[t / 2]) : half2_of_low(u[t / 2]), t & 1 ? half2_of_high(v[t / 2]) : half2_of_low(v[t / 2]));
                }
            };
            bool apart = false;
            if (!full && t_first != t_last) {   // a NaN that some of the rows do not see must not reach them: 0 * NaN
                bool nan = false;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int w = 0; w < VW; ++w) nan |= holds_nan(vw[kt][i][w]);
                apart = nan;
            }
            const int up0 = unit_run[0] - unit_v, up1 = unit_run[1] - unit_v;
            const bool far = apart || abs(up0) > 30 || abs(up1) > 30;   // (an output is within 2^40 units: 2^14 weights, 448, some thousand pages)
            if (!__any_sync(0xffffffffu, far)) {
                const float f0 = corr[0] * pow2(up0), f1 = corr[1] * pow2(up1);
                unit_run[0] = unit_run[1] = unit_v;
                if constexpr (TWO) {
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        float acc[4][4];
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt)
                            word_products(kt, w, [](uint32_t x, int) { return x; }, [&](int t, uint32_t b0, uint32_t b1) {
                                mma_f16_16816(acc[t], pa[1][kt], b0, b1);
                                mma_f16_16816(acc[t], pa[0][kt], b0, b1);
                            });
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            if (P::v16 != 0 && w == VW - 1 && t >= 2) break;
                            float(&x)[4] = o[4 * w + t];
                            x[0] = fmaf(x[0], f0, acc[t][0]), x[1] = fmaf(x[1], f0, acc[t][1]), x[2] = fmaf(x[2], f1, acc[t][2]), x[3] = fmaf(x[3], f1, acc[t][3]);
                        }
                    }
                } else {
                    if (__any_sync(0xffffffffu, f0 != 1.f || f1 != 1.f)) {
#pragma unroll
                        for (int t = 0; t < OT; ++t) o[t][0] *= f0, o[t][1] *= f0, o[t][2] *= f1, o[t][3] *= f1;
                    }
#pragma unroll
                    for (int w = 0; w < VW; ++w)
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt)
                            word_products(kt, w, [](uint32_t x, int) { return x; }, [&](int t, uint32_t b0, uint32_t b1) { mma_f16_16816(o[4 * w + t], pa[0][kt], b0, b1); });
                }
            } else {
                // scales far apart, or a NaN: a unit in which what was there (2^had at most) and what comes (2^comes) both have room, and token by
                // token, each with the positions that it sees
                int shift_old[2], shift_new[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float most = 0.f;
#pragma unroll
                    for (int t = 0; t < OT; ++t) most = fmaxf(most, fmaxf(fabsf(o[t][2 * e]), fabsf(o[t][2 * e + 1])));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2)) * corr[e];
                    const int had = most > 0.f ? unit_run[e] + exponent_of(most) : -1000;
                    const int comes = unit_v + 30 + (int)fmaxf(m_tile[e] - m_run[e], -800.f);
                    const int unit_both = max(max(had, comes) - 30, -150);
                    shift_old[e] = unit_run[e] - unit_both, shift_new[e] = unit_v - unit_both;
                    unit_run[e] = unit_both;
                }
#pragma unroll
                for (int t = 0; t < OT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[t][e] = ldexpf(o[t][e] * corr[e >> 1], shift_old[e >> 1]);
                for (int token = t_first; token <= t_last; ++token) {
                    const int upto = t_first == t_last ? first_hi : a.tok_pos[r.begin + token] + 1, from = a.window > 0 ? upto - a.window : 0;
                    const bool mine[2] = {(row0 + g) / G == token, (row0 + g + 8) / G == token};
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        float acc[4][4];
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt)
                            word_products(kt, w, [&](uint32_t x, int at) { return key0 + at >= from && key0 + at < upto ? x : 0u; }, [&](int t, uint32_t b0, uint32_t b1) {
                                if constexpr (TWO) mma_f16_16816(acc[t], pa[1][kt], b0, b1);
                                mma_f16_16816(acc[t], pa[0][kt], b0, b1);
                            });
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            if (P::v16 != 0 && w == VW - 1 && t >= 2) break;
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (mine[e >> 1]) o[4 * w + t][e] += ldexpf(acc[t][e], shift_new[e >> 1]);
                        }
                    }
                }
            }
        }

        // ---- the warps' results together: the outputs of each alone, under shares of the whole weight
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 1);
            l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 2);
            if (c == 0) {
                m_s[warp][g + 8 * e] = m_run[e];
                l_s[warp][g + 8 * e] = l_run[e];
            }
            // (l is 2^14 or more: the division comes first, so that nothing leaves float32's range before the result does)
            const float inv = l_run[e] != 0.f ? 1.f / l_run[e] : 0.f;
#pragma unroll
            for (int t = 0; t < OT; ++t)
                *reinterpret_cast<float2*>(&shared_o[(warp * EA_ROWS + g + 8 * e) * LD + 8 * t + 8 * (t / 4) + 2 * c]) =
                    make_float2(scaled(o[t][2 * e] * inv, unit_run[e]), scaled(o[t][2 * e + 1] * inv, unit_run[e]));
        }
        __syncthreads();
        const int live_warps = min(EA_WARPS, p_end - p_begin);   // (the others have seen nothing)
        if (threadIdx.x < EA_ROWS) {
            float m = EA_NONE, l = 0.f, part[EA_WARPS];
            for (int w = 0; w < live_warps; ++w) m = fmaxf(m, m_s[w][threadIdx.x]);
#pragma unroll
            for (int w = 0; w < EA_WARPS; ++w) {
                part[w] = w < live_warps ? fast_exp2(m_s[w][threadIdx.x] - m) * l_s[w][threadIdx.x] : 0.f;
                l += part[w];
            }
            const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
            for (int w = 0; w < EA_WARPS; ++w) factor_s[w][threadIdx.x] = part[w] * inv;
            m_s[0][threadIdx.x] = m;
            total_s[threadIdx.x] = l;
        }
        __syncthreads();
        const int first_block = (pair_begin + ahead) / target, runs = (pair_begin + ahead + r.pages - 1) / target - first_block + 1, run = (int)blockIdx.x - first_block;
        // where run k of this pair leaves its results: a block's first pair in the first of its two places
        auto place_of = [&](int k) { return 2 * (first_block + k) + (pair_begin > (first_block + k) * target ? 1 : 0); };
        // an item: four products' elements of one column and row, neighbours in the output
        auto each_item = [&](auto work) {
            for (int i = threadIdx.x; i < n_rows * VW * 8; i += THREADS) {
                const int row = i / (VW * 8), w = i / 8 % VW, n = i % 8;
                work(i, row, w, n, P::v16 != 0 && w == VW - 1 ? 2 : 4);
            }
        };
        auto give_out = [&](const float (&v)[4], int row, int w, int n, int count) {
            store4(out + row_at(row) + value_component<D>(4 * w, n), v, count);
        };
        each_item([&](int i, int row, int w, int n, int count) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < live_warps; ++k) {
                const float f = factor_s[k][row];
                const float* from = shared_o + (k * EA_ROWS + row) * LD + 40 * w + n;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < count) v[j] = fmaf(f, from[8 * j], v[j]);
            }
            if (runs == 1) give_out(v, row, w, n, count);
            else *reinterpret_cast<float4*>(a.part_o + (long long)place_of(run) * EA_ROWS * PART + i * 4) = make_float4(v[0], v[1], v[2], v[3]);
        });
        if (runs > 1) {
            // joins the results in `count` places (the k-th: place(k)): their sums in total_s, the output by `done`
            auto join = [&](int count, auto place, auto done) {
                __threadfence();
                const int row = threadIdx.x / EA_SHARE, sub = threadIdx.x % EA_SHARE;   // EA_SHARE lanes a row
                float2 x[EA_MOST_GROUPS / EA_SHARE];
                float m = EA_NONE, l = 0.f;
#pragma unroll
                for (int i = 0; i < EA_MOST_GROUPS / EA_SHARE; ++i) {
                    const int k = sub + i * EA_SHARE;
                    x[i] = k < count && row < n_rows ? __ldcg(reinterpret_cast<const float2*>(a.part_ml + (place(k) * EA_ROWS + row) * 2)) : make_float2(EA_NONE, 0.f);
                    m = fmaxf(m, x[i].x);
                }
#pragma unroll
                for (int s = 1; s < EA_SHARE; s <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
#pragma unroll
                for (int i = 0; i < EA_MOST_GROUPS / EA_SHARE; ++i) l += x[i].y = fast_exp2(x[i].x - m) * x[i].y;
#pragma unroll
                for (int s = 1; s < EA_SHARE; s <<= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
                const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
                for (int i = 0; i < EA_MOST_GROUPS / EA_SHARE; ++i)
                    if (sub + i * EA_SHARE < count) factor_s[sub + i * EA_SHARE][row] = x[i].y * inv;
                if (sub == 0) m_s[0][row] = m, total_s[row] = l;
                __syncthreads();
                each_item([&](int i, int row, int w, int n, int items) {
                    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
                    for (int k = 0; k < count; ++k) {
                        const float f = factor_s[k][row];
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(a.part_o + (long long)place(k) * EA_ROWS * PART + i * 4));
                        v[0] = fmaf(f, x.x, v[0]), v[1] = fmaf(f, x.y, v[1]), v[2] = fmaf(f, x.z, v[2]), v[3] = fmaf(f, x.w, v[3]);
                    }
                    done(v, i, row, w, n, items);
                });
            };
            auto leave = [&](int place) {   // maximum and sum
                if (threadIdx.x < n_rows) *reinterpret_cast<float2*>(a.part_ml + (place * EA_ROWS + threadIdx.x) * 2) = make_float2(m_s[0][threadIdx.x], total_s[threadIdx.x]);
            };
            auto last_of = [&](int* ticket, int count) {   // whether all others have left theirs; the counter is then as the next call wants it
                __threadfence();
                __syncthreads();
                if (threadIdx.x == 0) {
                    ticket_s = atomicAdd(ticket, 1);
                    if (ticket_s == count - 1) *ticket = 0;
                }
                __syncthreads();
                return ticket_s == count - 1;
            };
            leave(place_of(run));
            const int group = run / EA_GROUP, groups = (runs + EA_GROUP - 1) / EA_GROUP, members = min(EA_GROUP, runs - group * EA_GROUP);
            const int home = place_of(group * EA_GROUP);
            if (last_of(a.tickets + home, members)) {
                auto member = [&](int k) { return place_of(group * EA_GROUP + k); };
                if (groups == 1) {
                    join(members, member, [&](const float (&v)[4], int, int row, int w, int n, int count) { give_out(v, row, w, n, count); });
                } else {
                    join(members, member, [&](const float (&v)[4], int i, int, int, int, int) {
                        *reinterpret_cast<float4*>(a.part_o + (long long)home * EA_ROWS * PART + i * 4) = make_float4(v[0], v[1], v[2], v[3]);
                    });
                    leave(home);
                    if (last_of(a.tickets + 2 * n_blocks + place_of(0), groups))
                        join(groups, [&](int k) { return place_of(k * EA_GROUP); },
                             [&](const float (&v)[4], int, int row, int w, int n, int count) { give_out(v, row, w, n, count); });
                }
            }
        }
        __syncthreads();   // (the next pair takes the same shared memory)
    }
}

// Blocks that the device holds at once of this shape; 0 where the shape has no kernel.
template <typename T, int D> static int slots_of() {
    static int cached[64];
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
    if (cached[device] == 0) {
        int n = 0;
        if (cudaFuncSetAttribute(attend_e4m3_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<T, D>::SMEM) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attend_e4m3_kernel<T, D>, EA_WARPS * 32, Shape<T, D>::SMEM) != cudaSuccess)
            return 0;
        cached[device] = std::min(n * qf_sm_count(), EA_GROUP * EA_MOST_GROUPS);
    }
    return cached[device];
}
template <typename T, int D> static int attend(const void* q, void* out, AttendArgs& a, int blocks, cudaStream_t stream) {
    if (a.block_slots <= 0 || a.block_slots != slots_of<T, D>()) return (int)cudaErrorInvalidValue;
    return (int)launch_pdl(attend_e4m3_kernel<T, D>, dim3(blocks), dim3(EA_WARPS * 32), Shape<T, D>::SMEM, stream, (const T*)q, (T*)out, a);
}

#define EA_EVERY(T, CALL)               \
    switch (head_dim) {                 \
        case 16: return CALL(T, 16);    \
        case 32: return CALL(T, 32);    \
        case 48: return CALL(T, 48);    \
        case 64: return CALL(T, 64);    \
        case 80: return CALL(T, 80);    \
        case 96: return CALL(T, 96);    \
        case 112: return CALL(T, 112);  \
        case 128: return CALL(T, 128);  \
    }

// Blocks that the current device holds at once for a head size (0: there is no kernel for it): what the workspaces are sized by.
QF_EXPORT int qf_attention_e4m3_slots(int is_bf16, int head_dim) {
#define EA_SLOTS(T, D) slots_of<T, D>()
    if (is_bf16) {
        EA_EVERY(bf16, EA_SLOTS)
    } else {
        EA_EVERY(float, EA_SLOTS)
    }
    return 0;
}

// q, out [tokens][n_heads * head_dim], on 16 bytes; single: every entry has one token; chunks: rows of 16 of the longest span, ceil(tokens * n_heads /
// kv_heads / 16); most_pages: the most pages that a sequence reads; blocks: n_seqs * kv_heads * chunks * ceil(most_pages / 4), block_slots (of
// qf_attention_e4m3_slots) at most. part_o [2 * blocks][16][32 * ceil(head_dim / 32)], part_ml [2 * blocks][16][2]; tickets [4 * blocks], zero before the
// first call and after every call.
QF_EXPORT int qf_attention_e4m3(int is_bf16, const void* q, void* out, const int* cu_q, const int* tok_pos, const int* slots, void* codes, float* scales,
                                const int* table, long long page_bytes, long long page_scales, int table_stride, int columns, int n_slots, int kv_heads,
                                int head_dim, int n_heads, int n_seqs, int single, int chunks, int most_pages, int blocks, int block_slots, float scale, int window,
                                float* part_o, float* part_ml, int* tickets, int* err, cudaStream_t stream) {
    const E4m3Site site{(unsigned char*)codes, scales, table, page_bytes, page_scales, table_stride, columns, n_slots, kv_heads, head_dim};
    if (head_dim <= 0 || head_dim % 16 || kv_heads <= 0 || n_heads <= 0 || n_heads % kv_heads || chunks <= 0 || most_pages <= 0 || columns <= 0 || n_slots <= 0 ||
        page_bytes % 16 || ((uintptr_t)codes | (uintptr_t)q | (uintptr_t)out) % 16 || page_bytes < 2ll * kv_heads * QF_PAGE * head_dim || page_scales < 2ll * kv_heads ||
        blocks <= 0 || blocks > block_slots || window < 0 || (long long)n_seqs * kv_heads * chunks * (most_pages + 2ll * block_slots) > 0x7fffffffll)
        return (int)cudaErrorInvalidValue;
    if (n_seqs <= 0) return 0;
    AttendArgs a{cu_q, tok_pos, slots, site, n_heads, n_seqs, single, chunks, most_pages, block_slots, window, scale * 1.4426950408889634f, part_o, part_ml, tickets, err};
#define EA_ATTEND(T, D) attend<T, D>(q, out, a, blocks, stream)
    if (is_bf16) {
        EA_EVERY(bf16, EA_ATTEND)
    } else {
        EA_EVERY(float, EA_ATTEND)
    }
    return (int)cudaErrorInvalidValue;
}
