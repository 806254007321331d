// Attention of single tokens, and of short spans of tokens, over a sequence cache of e4m3 codes (the format: e4m3.cuh).
//
//   o = softmax_j(q k_j^T scale) v_j over the keys j that the token sees: max(0, p - window + 1) <= j <= p
//
// The codes are multiplied as float16, in which they are exact, with float32 sums. A page's power of two for the keys is a factor of its scores; that
// for the values is the unit in which a row's sum of outputs is kept while the page adds to it (an exact shift where the next page's differs).
// Queries become float16 behind a power of two per row that brings their largest element to 2^7 .. 2^8: bfloat16 queries lose nothing but
// what lies 2^-31 below that, float32 queries are two such numbers (22 bits) and take two products. Weights are 2^(s - m + 14), at most 2^14
// for the running maximum m: rounded to float16 (2^-11 of each weight, an eighth of the output's own rounding) where the output is bfloat16,
// two numbers where it is float32; either ends at 2^-24, so a weight below 2^-28 of the row's largest is kept to 2^-39 of that (where values' scales are far
// apart, of the tile's largest). Maxima, sums and outputs are float32. The tensor cores' additions cut off bits below 2^-23 of a sum; for float32
// outputs their sums end with a tile, for bfloat16 they go on over a warp's pages (2^-14 after 8,000 positions).
//
// A block takes pages of a (sequence, kv head, 8 or 16 rows), its warps a page each in turn; a warp looks its next 32 pages and their scales up
// at once. A row is a query head of the kv head's group and a token of the span. Both products are taken with the cache on the left, whose
// tiles are the tall side of m16n8k16: S^T = K Q^T (16 positions by 8 rows), O^T = V^T P^T (16 components by 8 rows), so that seven or eight heads
// of a group fill a tile, where they would be half of one the other way round, with half the products, exponentials and sums to keep.
// P^T comes out of the first with positions where the second wants rows: eight by eight, the warp transposes it (movmatrix).
// A warp's tiles come through shared memory of its own, the next one on its way while it works on one. For the keys a lane takes D / 4 components
// of one position in eight, 16 bytes at a time (which components a product's steps go through is free, as long as the queries'
// fragments go through the same). For the values a lane takes D / 8 neighbouring components of the four positions that a step wants
// of it, and byte t of them is its element of component column t: a byte permutation puts two positions side by side for the conversion.
//
// Work is shared out on the device, from the lengths (a captured graph replays this launch with others): all pages of all (sequence, kv head,
// rows) in a row, `target` of them to a block, so that one round of blocks does it all. Where every pair's pages can be rounded up to
// whole blocks within that round, they are, and a block has one pair; else blocks begin and end anywhere, and lengths that
// differ leave no SM idle. A pair of several blocks leaves partial results (maximum, sum, output); the block that ends last, by a
// ticket, joins them in their order, sixteen at a time, and the last of those the sixteens.
//
// Microseconds, calls captured one behind another: a chat of 900 tokens, 14 heads over 2 of 64, 7.2; 8 of 4,096 9.0 (8.3 MB); one document of 32,000, 16 over 2 of 128,
// 14.2 (16.4 MB); 64 of up to 8,000, 28 over 4 of 128, 57.5 (272 MB, 4.7 TB/s; a copy has 6.5); 256 of 8,000 each 345 to 360 (2.1 GB, 6 TB/s); 12 spans of up to five
// tokens behind up to 3,000 25.0; float32, 20 of up to 3,500, 16 over 2 of 128, 14.5. Small calls are a chain: the plan from the lengths 2, first loads 1.3, the warps'
// merge 1.3, bringing blocks together 2 to 4. That is no floor: `attention_decode` reads the 16.8 MB of 8 of 4,096 in bfloat16 in 6.8, with a plan that one launch makes
// for all layers of a step. Here every warp goes through all entries' lengths three times, in 32s: 256 / 600 sequences of up to 300 tokens take 23.5 / 36, 28 over 4 of
// 128 40 to 44 / 76, where their bytes are 1.6 / 4.0 and 6.5 / 15. Large calls are bound by memory where lengths are even; ragged ones and spans by the issue of some 550
// instructions a tile of 32 positions, in 8 warps of an SM whose steps wait for their own products, exponentials and conversions. Blocks of 16 rows spill a
// little for some head sizes (bytes stored a thread: bfloat16 128 16; float32 64 68, 112 112, 128 160).
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "e4m3.cuh"

#define EA_WARPS 4
#define EA_DEAD 0x7fffffff   // the exponent of a tile that is not there, or that no row sees
#define EA_NONE (-3.0e38f)   // the running maximum of a row that has seen nothing
// How far (in powers of two) the values' units of a warp's pages may be from the one at which it last measured its outputs before it measures them again. An output is
// within 2^40 units of one page (2^14 weights, 448, some hundred thousand positions), so that with three times this there is room for float32's 2^127 however
// the units fall and rise, and a weight that float16 keeps to 2^-39 only stays far below what its value can make of it. A model's pages are within a few powers of two;
// measuring costs: 64 sequences of up to 8,000 tokens, 28 over 4 of 128, take 273 microseconds with values' scales of 2^-20 to 2^20 at random, for 57.
#define EA_APART 10
// Scores in base 2 up to which a weight's exponent is score - (maximum - 14), in float32: below 2^24 that is within one of 14 at the most, and off by no more than a
// score's own rounding. (From 2^25 on the largest weight could be float16's infinity.) Where the row's largest query component, the page's scale and 448 allow
// larger ones, the maximum is taken off the rounded score first, and the tile goes the way of scales that are far apart (289 microseconds).
#define EA_LARGE 1.6e7f

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
// An 8 x 8 matrix of float16, a row's two neighbours to a lane, with rows and columns exchanged.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// what float16 leaves over of two numbers
__device__ __forceinline__ uint32_t pack_rest(float lo, float hi, uint32_t taken) {
    const float2 t = floats_of(taken);
    return pack_half(lo - t.x, hi - t.y);
}
// A row of D components in parts of 128, 64, 32 and 16 that fragments go through one after another.
template <int D> struct Parts {
    // keys: a lane's words (four codes, one step of 16 components each) are D / 16; those of part 128 first
    static constexpr int k128 = D / 128, k64 = (D % 128) / 64, k32 = (D % 64) / 32, k16 = (D % 32) / 16, k_words = D / 16;
    // values: bytes of a lane from part 128, 64, 32, 16: 16, 8, 4, 2
    static constexpr int v128 = D / 128, v64 = (D % 128) / 64, v32 = (D % 64) / 32, v16 = (D % 32) / 16;
    static constexpr int v_words = 4 * v128 + 2 * v64 + v32 + v16;   // (16 fills half a word)
};
// First component of a lane's key word w (quad column c).
template <int D> __device__ __forceinline__ constexpr int key_component(int w, int c) {
    using P = Parts<D>;
    int base = 0;
    if (w < 8 * P::k128) return 32 * c + 4 * w;
    w -= 8 * P::k128, base += 128 * P::k128;
    if (w < 4 * P::k64) return base + 16 * c + 4 * w;
    w -= 4 * P::k64, base += 64 * P::k64;
    if (w < 2 * P::k32) return base + 8 * c + 4 * w;
    return base + 32 * P::k32 + 4 * c;
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
    int at = 0, o = 0;
    if constexpr (P::k128 != 0) {
        const uint4 u = *reinterpret_cast<const uint4*>(row + 32 * c), v = *reinterpret_cast<const uint4*>(row + 32 * c + 16);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w, w[4] = v.x, w[5] = v.y, w[6] = v.z, w[7] = v.w;
        at += 128, o += 8;
    }
    if constexpr (P::k64 != 0) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + at + 16 * c);
        w[o] = v.x, w[o + 1] = v.y, w[o + 2] = v.z, w[o + 3] = v.w;
        at += 64, o += 4;
    }
    if constexpr (P::k32 != 0) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + at + 8 * c);
        w[o] = v.x, w[o + 1] = v.y;
        at += 32, o += 2;
    }
    if constexpr (P::k16 != 0) w[o] = *reinterpret_cast<const uint32_t*>(row + at + 4 * c);
}
template <int D> __device__ __forceinline__ void load_value(uint32_t (&w)[Parts<D>::v_words], const unsigned char* row, int g) {
    using P = Parts<D>;
    int at = 0, o = 0;
    if constexpr (P::v128 != 0) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + 16 * g);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        at += 128, o += 4;
    }
    if constexpr (P::v64 != 0) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + at + 8 * g);
        w[o] = v.x, w[o + 1] = v.y;
        at += 64, o += 2;
    }
    if constexpr (P::v32 != 0) {
        w[o] = *reinterpret_cast<const uint32_t*>(row + at + 4 * g);
        at += 32, o += 1;
    }
    if constexpr (P::v16 != 0) w[o] = *reinterpret_cast<const uint16_t*>(row + at + 2 * g);
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from)); }
__device__ __forceinline__ void copy16_or_zero(uint32_t to, const void* from, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0));
}
__device__ __forceinline__ bool holds_nan(uint32_t codes) { return __vcmpeq4(codes & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0; }

// NR: eights of rows of a block. Microseconds of the other choices in bfloat16, this one's first (both sides of a pair in turn, pairs at several states of the kernel: its
// own figures are at the head of this file; heads of 64 are 14 over 2, of 128 28 over 4 where it does not say):
// SMALL's tiles and blocks as of the rest of D <= 64: 8 sequences of 4,096 tokens, heads of 64, 9.2 / 12.0, 64 of up to 8,000 24.5 / 25.0, a chat of 900
// 7.7 / 7.4; three stages: 64 of up to 8,000, heads of 128, 58.3 / 60.8, one of 32,000, 16 over 2 of 128, 14.3 / 14.6, spans of five tokens, heads of
// 64, 13.5 / 15.6; tiles of a whole page for heads of 128: 64 of up to 8,000 58.3 / 69, 8 of 2,000 to 4,000 12.0 / 13.7, alone with 2,000 tokens 8.9 / 8.3; three blocks
// to an SM there (168 registers, some spilled): 58.3 / 61.1, one of 32,000 14.6 / 13.5, alone with 8,000 11.6 / 12.8.
template <typename T, int D, int NR> struct Shape {
    static constexpr bool TWO = sizeof(T) == 4;                       // float32: queries and weights as two float16 each
    static constexpr int ROWS = 8 * NR;
    static constexpr bool SMALL = D <= 64 && NR == 1;
    static constexpr int TILE = SMALL ? 32 : D <= 64 ? 64 : TWO && NR > 1 ? 16 : 32;   // positions of a step
    static constexpr int BLOCKS = SMALL ? 3 : 2;                      // of an SM
    static constexpr int STAGES = 2;                                  // tiles of a warp in shared memory: one at work, the others on their way
    static constexpr int PITCH = D / 16 % 2 ? D : D + 16;             // bytes of a staged row: an odd number of 16, so that eight rows meet all banks
    static constexpr int STAGE = 2 * TILE * PITCH;                    // keys, then values
    static constexpr int PART = 32 * Parts<D>::v_words;               // floats of a row of a partial result: items of four
    static constexpr int LD = PART + 4;                               // and where warps leave theirs: rows four banks apart
    // (the outputs, the warps' and the block's with its maxima and sums, take the tiles' place)
    static constexpr int OUTPUTS = (EA_WARPS + 1) * ROWS * LD * 4 + ROWS * 8, TILES = EA_WARPS * STAGES * STAGE, SMEM = TILES > OUTPUTS ? TILES : OUTPUTS;
    static constexpr int SHARE = EA_WARPS * 32 / ROWS;                // lanes that join a row's maxima and sums
};

struct AttendArgs {
    const int *cu_q, *tok_pos, *slots;
    E4m3Site site;
    int n_heads, group, n_seqs, single, chunks, most_pages, block_slots, window, constants, cluster, cluster_log;   // group: query heads of a kv head
    float scale_log2;
    float *part_o, *part_ml;   // [2 * blocks][ROWS][PART], [2 * blocks][ROWS][2]
    int *tickets, *err;        // [4 * blocks]
};

struct Sequence {
    int slot, begin, tokens, first_pos, last_pos, page0, pages, pairs;   // pairs: kv heads times blocks of rows
};
template <int ROWS> __device__ __forceinline__ Sequence sequence_of(const AttendArgs& a, int s) {
    Sequence r;
    const int guess = a.single ? a.tok_pos[s] : 0;   // (single: as many tokens as entries, so most probably one each: all loads at once)
    r.begin = a.cu_q[s];
    r.tokens = a.cu_q[s + 1] - r.begin;
    r.slot = a.slots[s];
    if (r.tokens <= 0) r.slot = -1;
    r.first_pos = r.last_pos = r.page0 = r.pages = 0;
    r.pairs = a.site.kv_heads * min(a.chunks, (int)((unsigned)(r.tokens * a.group + ROWS - 1) / ROWS));
    if (a.single && r.begin == s && r.tokens == 1) {
        r.first_pos = r.last_pos = guess;
    } else if (r.tokens > 0) {
        r.first_pos = a.tok_pos[r.begin];
        r.last_pos = a.tok_pos[r.begin + r.tokens - 1];
    }
    if (r.slot >= 0) {
        r.page0 = a.window > 0 ? max(0, r.first_pos - a.window + 1) / QF_PAGE : 0;
        r.pages = min(max(r.last_pos / QF_PAGE - r.page0 + 1, 0), a.most_pages);   // (more than the call has said: cut, and reported)
    }
    return r;
}

// a / b rounded down, 0 <= a < 2^20 (pages of a sequence): (a + 1/2) / b is at least 1 / (2 b) away from a whole number, its rounding errors less than
// that.
__device__ __forceinline__ int quotient(int a, int b) { return (int)(((float)a + 0.5f) * __frcp_rn((float)b)); }

template <typename T> __device__ __forceinline__ void store4(T* to, const float (&v)[4], int n) {
    if constexpr (sizeof(T) == 4) {
        if (n == 4) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<float2*>(to) = make_float2(v[0], v[1]);
    } else {
        if (n == 4) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
        else *reinterpret_cast<uint32_t*>(to) = pack_bf16(v[0], v[1]);
    }
}

// Pages whose time a pair's beginning and end take. Microseconds with 14 / 0, in turn: 64 sequences of up to 8,000 tokens, 28 heads over 4 of 128, 61 / 74, 12 spans of up to
// five tokens 26 / 47.
#define EA_PAIR_COST 14
#define EA_GROUP 16        // partial results that a block joins at once
#define EA_MOST_GROUPS 64  // ... and groups of them: enough for 1,024 blocks

// Where the results of a pair that begins at pair_begin lie that block `block` leaves: a block's first pair has the first of its two places.
__device__ __forceinline__ int place_in(int pair_begin, int block, int target) { return 2 * block + (pair_begin > block * target ? 1 : 0); }
// Element 0 of the query (and output) of row i (token * group + head of the group) of the kv head kvh.
template <int D> __device__ __forceinline__ long long row_offset(const AttendArgs& a, int begin, int kvh, int i) {
    const int G = a.group, token = i < G ? 0 : i / G;
    return (long long)(begin + token) * a.n_heads * D + (long long)(kvh * G + i - token * G) * D;
}
// Item i of a row, four neighbouring components (two of a part of 16), to its row of the output.
template <typename T, int D> __device__ __forceinline__ void give_out(T* row, const float4& v, int i) {
    const float u[4] = {v.x, v.y, v.z, v.w};
    store4(row + value_component<D>(i / 8 * 4, i % 8), u, Parts<D>::v16 != 0 && i / 8 == Parts<D>::v_words - 1 ? 2 : 4);
}

// Whether this block draws the last of `count` tickets; it then sees what all the others wrote before they drew theirs, and the counter is as the next
// call wants it. (The block's writes come before its first thread's, by the barrier; that thread's draw releases and acquires for all.)
__device__ __forceinline__ bool drew_last(int* ticket, int count, int* ticket_s) {
    __syncthreads();
    if (threadIdx.x == 0) {
        int drawn;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(drawn) : "l"(ticket) : "memory");
        if (drawn == count - 1) *ticket = 0;
        *ticket_s = drawn;
    }
    __syncthreads();
    return *ticket_s == count - 1;
}

struct Pair {
    int begin, first_block, runs, n_rows, row0, kvh, token0;
};
// Joins the results of `count` runs of a pair, run0, run0 + apart, ..., in this order: to the output, or, home >= 0, to the place `home` as one more result.
template <typename T, int D, int NR>
__device__ __forceinline__ void join_parts(T* out, const AttendArgs& a, const Pair& pair, int target, int run0, int apart, int count, int home, float* factor_s) {
    using S = Shape<T, D, NR>;
    constexpr int VW = Parts<D>::v_words, PART = S::PART, ROWS = S::ROWS, THREADS = EA_WARPS * 32, EACH = EA_MOST_GROUPS / S::SHARE;
    auto place = [&](int k) { return place_in(pair.begin, pair.first_block + run0 + k * apart, target); };
    auto part_of = [&](int k, int i) { return __ldcg(reinterpret_cast<const float4*>(a.part_o + (long long)place(k) * ROWS * PART + i * 4)); };
    const int items = pair.n_rows * VW * 8;
    float4 ready[EA_GROUP];   // the first sixteen parts of this thread's first item, on their way beside the statistics
#pragma unroll
    for (int k = 0; k < EA_GROUP; ++k)
        if (k < count && (int)threadIdx.x < items) ready[k] = part_of(k, threadIdx.x);
    const int row = threadIdx.x / S::SHARE, sub = threadIdx.x % S::SHARE;
    float2 x[EACH];
    float m = EA_NONE, l = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int k = sub + i * S::SHARE;
        x[i] = k < count && row < pair.n_rows ? __ldcg(reinterpret_cast<const float2*>(a.part_ml + (place(k) * ROWS + row) * 2)) : make_float2(EA_NONE, 0.f);
        m = fmaxf(m, x[i].x);
    }
#pragma unroll
    for (int i = 1; i < S::SHARE; i <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
#pragma unroll
    for (int i = 0; i < EACH; ++i) l += x[i].y = fast_exp2(x[i].x - m) * x[i].y;
#pragma unroll
    for (int i = 1; i < S::SHARE; i <<= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (sub + i * S::SHARE < count) factor_s[(sub + i * S::SHARE) * ROWS + row] = x[i].y * inv;
    __syncthreads();   // (every result's maximum and sum have been read, and its factor is there)
    if (home >= 0 && sub == 0 && row < pair.n_rows) *reinterpret_cast<float2*>(a.part_ml + (home * ROWS + row) * 2) = make_float2(m, l);
    for (int i = threadIdx.x; i < items; i += THREADS) {
        const int at_row = i / (VW * 8);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < count; k0 += EA_GROUP) {
            if (k0 > 0 || i >= THREADS) {
#pragma unroll
                for (int k = 0; k < EA_GROUP; ++k)
                    if (k0 + k < count) ready[k] = part_of(k0 + k, i);
            }
#pragma unroll
            for (int k = 0; k < EA_GROUP; ++k)
                if (k0 + k < count) {
                    const float f = factor_s[(k0 + k) * ROWS + at_row];
                    v.x = fmaf(f, ready[k].x, v.x), v.y = fmaf(f, ready[k].y, v.y), v.z = fmaf(f, ready[k].z, v.z), v.w = fmaf(f, ready[k].w, v.w);
                }
        }
        if (home >= 0) *reinterpret_cast<float4*>(a.part_o + (long long)home * ROWS * PART + i * 4) = v;
        else give_out<T, D>(out + row_offset<D>(a, pair.token0, pair.kvh, pair.row0 + at_row), v, i % (VW * 8));
    }
}

// Thread-block clusters: all threads of all blocks arrive (what they wrote is then seen by whoever has waited) and wait.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Shared memory of block `rank` of the cluster at the place that is `at` in this one's.
__device__ __forceinline__ uint32_t of_rank(const void* at, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(at)), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 remote4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ float2 remote2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
    return v;
}
// The end of a pair whose runs are clusters: a block puts its warps' results together, the cluster its blocks', each block a share of the items; of
// several clusters the last one to leave a share joins that. No result takes the way through memory where one cluster has the pair.
template <typename T, int D, int NR>
__device__ __forceinline__ void join_cluster(T* out, const AttendArgs& a, float* shared_o, const float* m_s, const float* l_s, int items, int row0, int token0, int kvh,
                                             int rank, int first, int run, int runs, int* ticket_s) {
    using S = Shape<T, D, NR>;
    constexpr int VW = Parts<D>::v_words, LD = S::LD, PART = S::PART, ROWS = S::ROWS, THREADS = EA_WARPS * 32;
    float* block_o = shared_o + EA_WARPS * ROWS * LD;   // [rows][LD], behind the warps' own; then maxima and sums
    float2* block_ml = reinterpret_cast<float2*>(block_o + ROWS * LD);
    for (int i = threadIdx.x; i < items; i += THREADS) {
        const int row = i / (VW * 8), at = row * LD + i % (VW * 8) * 4;
        float m = EA_NONE, l = 0.f, part[EA_WARPS];
#pragma unroll
        for (int k = 0; k < EA_WARPS; ++k) m = fmaxf(m, m_s[k * ROWS + row]);
#pragma unroll
        for (int k = 0; k < EA_WARPS; ++k) l += part[k] = fast_exp2(m_s[k * ROWS + row] - m) * l_s[k * ROWS + row];
        const float inv = l != 0.f ? 1.f / l : 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < EA_WARPS; ++k) {
            const float f = part[k] * inv;
            const float4 x = *reinterpret_cast<const float4*>(&shared_o[k * ROWS * LD + at]);
            v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
        }
        *reinterpret_cast<float4*>(block_o + at) = v;
        if (i % (VW * 8) == 0) block_ml[row] = make_float2(m, l);
    }
    cluster_arrive();
    cluster_wait();
    const int each = (items + a.cluster - 1) >> a.cluster_log, begin = rank * each, end = min(begin + each, items);
    // one of `count` results to the others: their maxima and sums, their items
    auto join = [&](int count, auto ml_of, auto item_of, float2& ml) {
        float2 x[16];
        float4 y[16], v = make_float4(0.f, 0.f, 0.f, 0.f);
        ml = make_float2(EA_NONE, 0.f);
        for (int k0 = 0; k0 < count; k0 += 16) {   // (blocks of a cluster, or clusters of a pair)
            float m = ml.x;
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (k0 + k < count) x[k] = ml_of(k0 + k), y[k] = item_of(k0 + k), m = fmaxf(m, x[k].x);
            const float old = fast_exp2(ml.x - m) * ml.y;
            float l = old;
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (k0 + k < count) l += x[k].y = fast_exp2(x[k].x - m) * x[k].y;
            const float inv = l != 0.f ? 1.f / l : 0.f;
            const float f0 = old * inv;
            v.x *= f0, v.y *= f0, v.z *= f0, v.w *= f0;
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (k0 + k < count) {
                    const float f = x[k].y * inv;
                    v.x = fmaf(f, y[k].x, v.x), v.y = fmaf(f, y[k].y, v.y), v.z = fmaf(f, y[k].z, v.z), v.w = fmaf(f, y[k].w, v.w);
                }
            ml = make_float2(m, l);
        }
        return v;
    };
    auto to_out = [&](const float4& v, int i) { give_out<T, D>(out + row_offset<D>(a, token0, kvh, row0 + i / (VW * 8)), v, i % (VW * 8)); };
    for (int i = begin + threadIdx.x; i < end; i += THREADS) {
        const int row = i / (VW * 8), at = row * LD + i % (VW * 8) * 4;
        float2 ml;
        const float4 v = join(a.cluster, [&](int k) { return remote2(of_rank(block_ml + row, k)); }, [&](int k) { return remote4(of_rank(block_o + at, k)); }, ml);
        if (runs == 1) {
            to_out(v, i);
        } else {
            *reinterpret_cast<float4*>(a.part_o + (long long)(first + run) * ROWS * PART + i * 4) = v;
            // (blocks that share a row leave the same)
            if (i % (VW * 8) == 0 || i == begin) *reinterpret_cast<float2*>(a.part_ml + ((first + run) * ROWS + row) * 2) = ml;
        }
    }
    if (runs == 1) return;
    if (!drew_last(a.tickets + first * a.cluster + rank, runs, ticket_s)) return;
    for (int i = begin + threadIdx.x; i < end; i += THREADS) {
        const int row = i / (VW * 8);
        float2 ml;
        to_out(join(runs, [&](int k) { return __ldcg(reinterpret_cast<const float2*>(a.part_ml + ((first + k) * ROWS + row) * 2)); },
                    [&](int k) { return __ldcg(reinterpret_cast<const float4*>(a.part_o + (long long)(first + k) * ROWS * PART + i * 4)); }, ml),
               i);
    }
}

template <typename T, int D, int NR>
__global__ void __launch_bounds__(EA_WARPS * 32, Shape<T, D, NR>::BLOCKS)
attend_e4m3_kernel(const T* __restrict__ q, T* __restrict__ out, const __grid_constant__ AttendArgs a) {
    using S = Shape<T, D, NR>;
    using P = Parts<D>;
    constexpr bool TWO = S::TWO;
    constexpr int TILE = S::TILE, KT = TILE / 16, DT = D / 16, KW = P::k_words, VW = P::v_words, LD = S::LD, PART = S::PART, ROWS = S::ROWS;
    constexpr int PER_PAGE = QF_PAGE / TILE, THREADS = EA_WARPS * 32, TERMS = TWO ? 2 : 1;
    grid_launch_dependents();
    // `constants`: lengths, slots, page tables and the pages before an entry's first new one are nobody's output, so the kernel ahead is waited for only
    // before the rest is read
    bool waited = !a.constants;
    if (waited) grid_dependency_wait();
    extern __shared__ __align__(16) unsigned char staged[];   // [warps][STAGES][keys, values][TILE][PITCH]; later the outputs, [warps][rows][LD]
    float* shared_o = reinterpret_cast<float*>(staged);
    __shared__ float scale_s[EA_WARPS][S::STAGES];   // of the staged tiles: the keys' scale, the values' exponent
    __shared__ int unit_s[EA_WARPS][S::STAGES];
    __shared__ float m_s[EA_WARPS][ROWS], l_s[EA_WARPS][ROWS], factor_s[EA_MOST_GROUPS * ROWS];
    __shared__ int ticket_s;
    __shared__ Pair left_s[2];
    int n_left = 0;
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    const E4m3Site& site = a.site;
    const int KVH = site.kv_heads, G = a.group;
    const int q_width = a.n_heads * D, n_blocks = gridDim.x;

    // ---- this block's share (every warp works it out for itself; a lane keeps its one of the first 32 sequences)
    Sequence first;
    first.pages = first.pairs = 0;
    if ((int)lane < a.n_seqs) first = sequence_of<ROWS>(a, lane);
    auto pages_of = [&](int s0) {   // (pages, pairs) of this lane's one of 32 sequences
        if (s0 == 0) return make_int2(first.pages, first.pairs);
        if (s0 + (int)lane >= a.n_seqs) return make_int2(0, 0);
        const Sequence x = sequence_of<ROWS>(a, s0 + lane);
        return make_int2(x.pages, x.pairs);
    };
    const int rank = (int)blockIdx.x & (a.cluster - 1), number = (int)blockIdx.x >> a.cluster_log;   // (one of 1, 8 or 16)
    int total = 0, target = EA_WARPS, ahead = 0;
    bool aligned = true;
    if (a.cluster > 1) {   // a cluster takes the part of a block, always whole units; there is one for every pair's every unit
        target = EA_WARPS << a.cluster_log;
        total = 0x7fffffff;
    } else {
        int pairs = 0, whole = 0;
        for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
            const int2 x = pages_of(s0);
            total += x.x * x.y;
            pairs += x.x > 0 ? x.y : 0;
        }
        total = (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
        pairs = (int)__reduce_add_sync(0xffffffffu, (unsigned)pairs);
        if (total > target * a.block_slots) target = (total + a.block_slots - 1) / a.block_slots;
        for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
            const int2 x = pages_of(s0);
            whole += quotient(x.x + target - 1, target) * x.y;
        }
        whole = (int)__reduce_add_sync(0xffffffffu, (unsigned)whole);
        // pages of a pair are rounded up to whole units; where blocks may have several pairs, each counts EA_PAIR_COST pages more
        aligned = whole <= a.block_slots;
        if (aligned) {
            total = whole * target;
        } else {
            ahead = EA_PAIR_COST;
            total += pairs * ahead;
            target = max(target, (total + a.block_slots - 1) / a.block_slots);
        }
    }
    auto places_of = [&](int pages) { return pages == 0 ? 0 : aligned ? quotient(pages + target - 1, target) * target : pages + ahead; };
    const int range_begin = number * target;
    int range_end = min(range_begin + target, total);
    // the sequence in whose pages it begins
    int seq = 0, base = 0;
    Sequence r = first;
    if (range_begin < range_end) {
        for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
            const int2 x = pages_of(s0);
            const int mine = places_of(x.x) * x.y;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if ((int)lane >= o) upto += v;
            }
            const uint32_t beyond = __ballot_sync(0xffffffffu, base + upto > range_begin);
            if (beyond) {
                const int who = __ffs(beyond) - 1;
                seq = s0 + who;
                base += __shfl_sync(0xffffffffu, upto - mine, who);
                if (s0 == 0) {
                    r.slot = __shfl_sync(0xffffffffu, first.slot, who), r.begin = __shfl_sync(0xffffffffu, first.begin, who);
                    r.tokens = __shfl_sync(0xffffffffu, first.tokens, who), r.first_pos = __shfl_sync(0xffffffffu, first.first_pos, who);
                    r.last_pos = __shfl_sync(0xffffffffu, first.last_pos, who), r.page0 = __shfl_sync(0xffffffffu, first.page0, who);
                    r.pages = __shfl_sync(0xffffffffu, first.pages, who), r.pairs = __shfl_sync(0xffffffffu, first.pairs, who);
                } else {
                    r = sequence_of<ROWS>(a, seq);
                }
                break;
            }
            base += __shfl_sync(0xffffffffu, upto, 31);
            if (s0 + 32 >= a.n_seqs) range_end = range_begin;   // (a cluster that nothing is left for)
        }
    }

    int padded = places_of(r.pages);
    for (int at = range_begin; at < range_end;) {
        while (at >= base + padded * r.pairs) {   // (sequences without pages are passed over)
            base += padded * r.pairs;
            r = sequence_of<ROWS>(a, ++seq);
            padded = places_of(r.pages);
        }
        const int y = (at - base) / padded, pair_begin = base + y * padded, kvh = y % KVH, chunk = y / KVH;
        int p_begin = r.page0 + max(at - pair_begin - ahead, 0), p_end = r.page0 + min(min(padded, range_end - pair_begin) - ahead, r.pages);
        const bool reports = y == 0 && threadIdx.x == 0 && at == pair_begin && rank == 0;
        at = min(pair_begin + padded, range_end);
        if (reports && r.last_pos / QF_PAGE - r.page0 + 1 > r.pages) atomicOr(a.err, QF_ERR_POSITION_RANGE);
        if (reports && r.tokens * G > a.chunks * ROWS) atomicOr(a.err, QF_ERR_ROW_RANGE);   // (a span longer than the call has said)
        const int row0 = chunk * ROWS, n_rows = min(ROWS, r.tokens * G - row0);   // rows: token * G + head of the group
        if (n_rows <= 0 || p_begin >= p_end) continue;
        if (a.cluster > 1) {   // this block's share, perhaps none
            const int each = (p_end - p_begin + a.cluster - 1) >> a.cluster_log;
            p_begin += rank * each;
            p_end = min(p_begin + each, p_end);
        }
        auto row_at = [&](int row) { return row_offset<D>(a, r.begin, kvh, row0 + row); };
        const int my_pages = max(p_end - p_begin - (int)warp + EA_WARPS - 1, 0) / EA_WARPS;   // (0 where there are fewer than warps)
        // what the rows see, lo .. hi - 1: this lane's (8 n + 2 c and + 1), all of them together, every one of them
        const int t_first = r.tokens == 1 ? 0 : row0 / G, t_last = r.tokens == 1 ? 0 : (row0 + n_rows - 1) / G;
        const int first_hi = (t_first == 0 ? r.first_pos : a.tok_pos[r.begin + t_first]) + 1, some_hi = (t_last == 0 ? r.first_pos : a.tok_pos[r.begin + t_last]) + 1;
        const int some_lo = a.window > 0 ? max(0, first_hi - a.window) : 0, all_lo = a.window > 0 ? max(0, some_hi - a.window) : 0;
        int lo[NR][2], hi[NR][2];
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 8 * n + 2 * c + e;
                hi[n][e] = row >= n_rows ? 0 : t_first == t_last ? first_hi : a.tok_pos[r.begin + (row0 + row) / G] + 1;
                lo[n][e] = a.window > 0 ? max(0, hi[n][e] - a.window) : 0;
            }

        // ---- pages p_begin + warp, + EA_WARPS, ...: a tile of one at a time, through the warp's own stages
        const unsigned steps = my_pages * PER_PAGE;
        const long long plane = (long long)KVH * QF_PAGE * D;
        int lane_page = -1, lane_unit = 0, page_next = -1, unit_next = 0;   // of 32 of the warp's pages, one a lane: its number, its scales
        float lane_scale = 0.f, scale_next = 0.f;
        const unsigned char* stage0 = staged + warp * S::STAGES * S::STAGE;
        const uint32_t lane_to = smem_addr(stage0) + lane * 16 + lane / (D / 16) * (S::PITCH - D);   // where the lane's first piece of a tile goes
        auto key0_of = [&](unsigned step) { return (p_begin + (int)warp + (int)(step / PER_PAGE) * EA_WARPS) * QF_PAGE + (int)(step % PER_PAGE) * TILE; };
        unsigned fetched = 0, fetch_stage = 0;
        auto fetch = [&]() {   // the next tile (one group of copies, perhaps an empty one)
            if (fetched < steps) {
                const int key0 = key0_of(fetched);
                if (fetched % PER_PAGE == 0) {
                    const int i = fetched / PER_PAGE;
                    if (i % 32 == 0) {   // the next 32 pages
                        lane_page = -1;
                        if (i + (int)lane < my_pages) {
                            lane_page = e4m3_page(site, r.slot, (p_begin + (int)warp + (i + (int)lane) * EA_WARPS) * QF_PAGE);
                            if (lane_page < 0) {
                                if (y == 0) atomicOr(a.err, QF_ERR_NO_PAGE);
                            } else {
                                const float* scales = site.scales + (long long)lane_page * site.page_scales + kvh;
                                lane_scale = scales[0];
                                lane_unit = exponent_of(scales[KVH]);
                            }
                        }
                    }
                    page_next = __shfl_sync(0xffffffffu, lane_page, i % 32);
                    scale_next = __shfl_sync(0xffffffffu, lane_scale, i % 32);
                    unit_next = __shfl_sync(0xffffffffu, lane_unit, i % 32);
                }
                const bool live = page_next >= 0 && key0 < some_hi && key0 + TILE > some_lo;
                if (lane == 0) scale_s[warp][fetch_stage] = scale_next, unit_s[warp][fetch_stage] = live ? unit_next : EA_DEAD;
                if (live) {
                    const unsigned char* k =
                        site.codes + (long long)page_next * site.page_bytes + (kvh * QF_PAGE + (int)(fetched % PER_PAGE) * TILE) * D + lane * 16;
                    const unsigned char* v = k + plane;
                    const uint32_t to = lane_to + fetch_stage * S::STAGE;
                    constexpr int CHUNKS = TILE * D / 16, ROUNDS = (CHUNKS + 31) / 32;
                    // piece i * 32 + lane: its row's number and so its place move by constants where a round has whole rows
                    auto place = [&](int i) -> uint32_t {
                        if constexpr (32 % (D / 16) == 0) return to + i * (512 + 32 / (D / 16) * (S::PITCH - D));
                        else return to + i * 512 + ((unsigned)(i * 32 + lane) / (D / 16) - lane / (D / 16)) * (S::PITCH - D);
                    };
                    if (key0 >= some_lo && key0 + TILE <= some_hi) {
#pragma unroll
                        for (int i = 0; i < ROUNDS; ++i)
                            if (CHUNKS % 32 == 0 || i * 32 + lane < CHUNKS) {
                                copy16(place(i), k + i * 512);
                                copy16(place(i) + TILE * S::PITCH, v + i * 512);
                            }
                    } else {   // zeros where nobody looks, NaN perhaps
#pragma unroll
                        for (int i = 0; i < ROUNDS; ++i)
                            if (CHUNKS % 32 == 0 || i * 32 + lane < CHUNKS) {
                                const int key = key0 + (int)((unsigned)(i * 32 + lane) / (D / 16));
                                copy16_or_zero(place(i), k + i * 512, key >= some_lo && key < some_hi);
                                copy16_or_zero(place(i) + TILE * S::PITCH, v + i * 512, key >= some_lo && key < some_hi);
                            }
                    }
                }
                ++fetched;
                fetch_stage = fetch_stage + 1 == S::STAGES ? 0 : fetch_stage + 1;
            }
            cp_async_commit();
        };
        if (waited) {
#pragma unroll
            for (int i = 0; i < S::STAGES - 1; ++i) fetch();
        }
#pragma unroll 1
        for (int i = waited ? S::STAGES : 0; i < S::STAGES; ++i) {
            if (!waited && (i == S::STAGES - 1 || i >= (int)steps || key0_of(i) / QF_PAGE >= r.first_pos / QF_PAGE)) {
                grid_dependency_wait();
                waited = true;
                if (lane_page >= 0 && p_begin + (int)warp + (int)lane * EA_WARPS >= r.first_pos / QF_PAGE) {   // (scales that were looked up before)
                    const float* scales = site.scales + (long long)lane_page * site.page_scales + kvh;
                    lane_scale = scales[0];
                    lane_unit = exponent_of(scales[KVH]);
                }
            }
            if (i < S::STAGES - 1) fetch();
        }

        // ---- the queries' fragments: lane (g, c) has row g's components of its column
        uint32_t qb[TERMS][NR][KW][2];
        float by[NR][2];   // scores of rows 8 n + 2 c + e in base-2 units: product * key scale * by
        float most_by = 0.f;   // key scale * this is no less than any score: D * 448 * the largest query component * scale
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            float2 x[KW][2];
            float top = 0.f;
            const int row = 8 * n + g;
            const T* src = q + (row < n_rows ? row_at(row) : 0);
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const int d = key_component<D>(w, c);
                x[w][0] = x[w][1] = make_float2(0.f, 0.f);
                if (row < n_rows) {
                    if constexpr (TWO) {
                        const float4 v = *reinterpret_cast<const float4*>(src + d);
                        x[w][0] = make_float2(v.x, v.y), x[w][1] = make_float2(v.z, v.w);
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(src + d);
                        x[w][0] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x));
                        x[w][1] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) top = fmaxf(top, fmaxf(fabsf(x[w][i].x), fabsf(x[w][i].y)));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int up = min(max(exponent_of(top) - 7, -119), 120);
            const float mine = pow2(up) * fabsf(a.scale_log2), down = copysignf(pow2(-up), a.scale_log2);
            by[n][0] = __shfl_sync(0xffffffffu, mine, 8 * c);
            by[n][1] = __shfl_sync(0xffffffffu, mine, 8 * c + 4);
            most_by = fmaxf(most_by, top * fabsf(a.scale_log2));
#pragma unroll
            for (int w = 0; w < KW; ++w)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float u = x[w][i].x * down, v = x[w][i].y * down;
                    qb[0][n][w][i] = pack_half(u, v);
                    if constexpr (TWO) qb[TERMS - 1][n][w][i] = pack_rest(u, v, qb[0][n][w][i]);
                }
        }

        most_by = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most_by))) * (D * 448.f);   // (positive: in their bits' order)

        float o[DT][NR][4];   // components of columns 2 d (0, 1) and 2 d + 1 (2, 3) by rows 2 c, 2 c + 1
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int n = 0; n < NR; ++n) o[d][n][0] = o[d][n][1] = o[d][n][2] = o[d][n][3] = 0.f;
        float m_run[NR][2], l_run[NR][2];   // (l: this lane's positions only)
        int unit_run[NR][2];                // o stands for o * 2^unit_run
#pragma unroll
        for (int n = 0; n < NR; ++n) m_run[n][0] = m_run[n][1] = EA_NONE, l_run[n][0] = l_run[n][1] = 0.f, unit_run[n][0] = unit_run[n][1] = 0;
        bool begun = false;
        int unit_measured = 0;   // of the values at which the outputs were last measured, or begun; far from all where a row's outputs stand far from it

        unsigned stage = S::STAGES - 1;   // (of the step before the first)
        for (unsigned step = 0; step < steps; ++step) {
            cp_async_wait<S::STAGES - 2>();
            __syncwarp();   // (this tile has come for every lane, and every lane is done with the one before it)
            fetch();
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
            const int key0 = key0_of(step), unit_v = unit_s[warp][stage];
            const float ks = scale_s[warp][stage];
            if (unit_v == EA_DEAD) continue;
            if (!begun) {
#pragma unroll
                for (int n = 0; n < NR; ++n) unit_run[n][0] = unit_run[n][1] = unit_v;
                unit_measured = unit_v;
                begun = true;
            }
            const unsigned char* keys = stage0 + stage * S::STAGE + g * S::PITCH;
            // ---- scores: positions 16 t + g (0, 1) and 16 t + 8 + g (2, 3) by rows 2 c, 2 c + 1
            float s[KT][NR][4];
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int n = 0; n < NR; ++n) s[t][n][0] = s[t][n][1] = s[t][n][2] = s[t][n][3] = 0.f;
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                uint32_t kw[2][KW];
                load_key<D>(kw[0], keys + 16 * t * S::PITCH, c);
                load_key<D>(kw[1], keys + (16 * t + 8) * S::PITCH, c);
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    const uint32_t k[4] = {half2_of_low(kw[0][w]), half2_of_low(kw[1][w]), half2_of_high(kw[0][w]), half2_of_high(kw[1][w])};
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        if constexpr (TWO) mma_f16_16816(s[t][n], k, qb[TERMS - 1][n][w][0], qb[TERMS - 1][n][w][1]);
                        mma_f16_16816(s[t][n], k, qb[0][n][w][0], qb[0][n][w][1]);
                    }
                }
            }
            // ---- this tile's values: positions 16 kt + 2 c, + 1, + 8, + 9
            uint32_t vw[KT][4][VW];
            const unsigned char* values = stage0 + stage * S::STAGE + (TILE + 2 * c) * S::PITCH;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) load_value<D>(vw[kt][i], values + (16 * kt + (i & 1) + 8 * (i >> 1)) * S::PITCH, g);
            const bool full = key0 >= all_lo && key0 + TILE <= first_hi;
            // ---- weights. What a row does not see is EA_NONE on the way to the maximum, and has none. Where scales are far apart, or scores may be large, they
            // are those under the tile's own maximum, so that float16 keeps them however far below the row's they lie: their values may be as much larger
            const bool own = abs(unit_measured - unit_v) > EA_APART || !(ks * most_by <= EA_LARGE);
            float corr[NR][2], m_tile[NR][2];
            uint32_t pb[TERMS][KT][NR][2];
            auto weigh = [&](auto whole) {   // (whole: every row sees every position, and the maximum is the running one)
                auto seen = [&](int t, int n, int e) {
                    if (decltype(whole)::value) return true;
                    const int key = key0 + 16 * t + 8 * (e >> 1) + g;
                    return key >= lo[n][e & 1] && key < hi[n][e & 1];
                };
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    float top[2] = {EA_NONE, EA_NONE}, shift[2], by_k[2], sum[2] = {0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < KT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (seen(t, n, e)) top[e & 1] = fmaxf(top[e & 1], s[t][n][e]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        by_k[e] = by[n][e] * ks;
#pragma unroll
                        for (int i = 4; i < 32; i <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], i));
                        m_tile[n][e] = top[e] > EA_NONE ? __fmul_rn(top[e], by_k[e]) : EA_NONE;
                        const float m = fmaxf(m_run[n][e], m_tile[n][e]);
                        corr[n][e] = fast_exp2(m_run[n][e] - m);
                        m_run[n][e] = m;
                        shift[e] = 14.f - m;
                    }
#pragma unroll
                    for (int t = 0; t < KT; ++t) {
                        float(&x)[4] = s[t][n];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float under = __fadd_rn(__fsub_rn(__fmul_rn(x[e], by_k[e & 1]), m_tile[n][e & 1]), 14.f);
                            x[e] = fast_exp2(!decltype(whole)::value && own ? under : fmaf(x[e], by_k[e & 1], shift[e & 1]));
                            if (!seen(t, n, e)) x[e] = 0.f;
                            sum[e & 1] += x[e];
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t most = pack_half(x[2 * h], x[2 * h + 1]);
                            pb[0][t][n][h] = transposed(most);
                            if constexpr (TWO) pb[TERMS - 1][t][n][h] = transposed(pack_rest(x[2 * h], x[2 * h + 1], most));
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float share = !decltype(whole)::value && own ? fast_exp2(__fsub_rn(m_tile[n][e], m_run[n][e])) : 1.f;
                        l_run[n][e] = fmaf(l_run[n][e], corr[n][e], sum[e] * share);
                    }
                }
            };
            if (full && !own) weigh(std::true_type{});
            else weigh(std::false_type{});
            bool by_token = false;   // a NaN that some of the rows do not see must not reach them: 0 * NaN
            if (!full && t_first != t_last) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int w = 0; w < VW; ++w) by_token |= holds_nan(vw[kt][i][w]);
                by_token = __any_sync(0xffffffffu, by_token);
            }
            // ---- values. Word w of the four positions of a step holds their elements of the component columns 4 w .. 4 w + 3
            auto word_products = [&](int kt, int w, auto take, auto add) {
                uint32_t x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = take(vw[kt][i][w], 16 * kt + 2 * c + (i & 1) + 8 * (i >> 1));
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    if (P::v16 != 0 && w == VW - 1 && d >= 1) break;
                    const uint32_t u = __byte_perm(x[0], x[1], d ? 0x7362 : 0x5140), v = __byte_perm(x[2], x[3], d ? 0x7362 : 0x5140);
                    const uint32_t f[4] = {half2_of_low(u), half2_of_high(u), half2_of_low(v), half2_of_high(v)};
                    add(2 * w + d, f);
                }
            };
            if (__builtin_expect(!own && !by_token, 1)) {
                float f[NR][2];
                bool moved = false;
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        f[n][e] = corr[n][e] * pow2(unit_run[n][e] - unit_v);
                        moved |= f[n][e] != 1.f;
                        unit_run[n][e] = unit_v;
                    }
                if constexpr (TWO) {
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        float acc[2][NR][4];
#pragma unroll
                        for (int d = 0; d < 2; ++d)
#pragma unroll
                            for (int n = 0; n < NR; ++n) acc[d][n][0] = acc[d][n][1] = acc[d][n][2] = acc[d][n][3] = 0.f;
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt)
                            word_products(kt, w, [](uint32_t x, int) { return x; }, [&](int d, const uint32_t(&v)[4]) {
#pragma unroll
                                for (int n = 0; n < NR; ++n) {
                                    mma_f16_16816(acc[d & 1][n], v, pb[TERMS - 1][kt][n][0], pb[TERMS - 1][kt][n][1]);
                                    mma_f16_16816(acc[d & 1][n], v, pb[0][kt][n][0], pb[0][kt][n][1]);
                                }
                            });
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            if (P::v16 != 0 && w == VW - 1 && d >= 1) break;
#pragma unroll
                            for (int n = 0; n < NR; ++n)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[2 * w + d][n][e] = fmaf(o[2 * w + d][n][e], f[n][e & 1], acc[d][n][e]);
                        }
                    }
                } else {
                    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int n = 0; n < NR; ++n)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[d][n][e] *= f[n][e & 1];
                    }
#pragma unroll
                    for (int w = 0; w < VW; ++w)
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt)
                            word_products(kt, w, [](uint32_t x, int) { return x; }, [&](int d, const uint32_t(&v)[4]) {
#pragma unroll
                                for (int n = 0; n < NR; ++n) mma_f16_16816(o[d][n], v, pb[0][kt][n][0], pb[0][kt][n][1]);
                            });
                }
            } else {
                // a unit in which what was there (2^had at most) and what comes (2^comes) both have room, and token by token, each with the positions that
                // it sees
                int shift_new[NR][2];
                float share[NR][2];   // of the tile's own weights in the row's, with 2^shift_new
                bool apart = false;
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float most = 0.f;
#pragma unroll
                        for (int d = 0; d < DT; ++d) most = fmaxf(most, fmaxf(fabsf(o[d][n][e]), fabsf(o[d][n][2 + e])));
#pragma unroll
                        for (int i = 4; i < 32; i <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, i));
                        most *= corr[n][e];
                        const int had = most > 0.f ? unit_run[n][e] + exponent_of(most) : -1000;
                        const float below = own ? fmaxf(__fsub_rn(m_tile[n][e], m_run[n][e]), -800.f) : 0.f, whole = floorf(below);
                        share[n][e] = fast_exp2(below - whole);
                        const int comes = unit_v + 30 + (own ? (int)whole : (int)fmaxf(m_tile[n][e] - m_run[n][e], -800.f));
                        const int unit_both = max(max(had, comes) - 30, -150);
                        shift_new[n][e] = unit_v + (int)whole - unit_both;
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int h = 0; h < 2; ++h) o[d][n][2 * h + e] = ldexpf(o[d][n][2 * h + e] * corr[n][e], unit_run[n][e] - unit_both);
                        unit_run[n][e] = unit_both;
                        apart |= abs(unit_both - unit_v) > EA_APART;
                    }
                unit_measured = __any_sync(0xffffffffu, apart) ? 1000 : unit_v;
                for (int token = t_first; token <= t_last; ++token) {
                    const int upto = t_first == t_last ? first_hi : a.tok_pos[r.begin + token] + 1, from = a.window > 0 ? upto - a.window : 0;
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        float acc[2][NR][4];
#pragma unroll
                        for (int d = 0; d < 2; ++d)
#pragma unroll
                            for (int n = 0; n < NR; ++n) acc[d][n][0] = acc[d][n][1] = acc[d][n][2] = acc[d][n][3] = 0.f;
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt)
                            word_products(kt, w, [&](uint32_t x, int at_key) { return key0 + at_key >= from && key0 + at_key < upto ? x : 0u; }, [&](int d, const uint32_t(&v)[4]) {
#pragma unroll
                                for (int n = 0; n < NR; ++n) {
                                    if constexpr (TWO) mma_f16_16816(acc[d & 1][n], v, pb[TERMS - 1][kt][n][0], pb[TERMS - 1][kt][n][1]);
                                    mma_f16_16816(acc[d & 1][n], v, pb[0][kt][n][0], pb[0][kt][n][1]);
                                }
                            });
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            if (P::v16 != 0 && w == VW - 1 && d >= 1) break;
#pragma unroll
                            for (int n = 0; n < NR; ++n)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if ((row0 + 8 * n + 2 * c + (e & 1)) / G == token) o[2 * w + d][n][e] += ldexpf(acc[d][n][e] * share[n][e & 1], shift_new[n][e & 1]);
                        }
                    }
                }
            }
        }

        cp_async_wait<0>();
        __syncthreads();   // (the outputs take the tiles' place)
        // ---- the warps' results together: the outputs of each alone, under shares of the whole weight. An item is four neighbouring components of a row
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 8 * n + 2 * c + e;
#pragma unroll
                for (int i = 4; i < 32; i <<= 1) l_run[n][e] += __shfl_xor_sync(0xffffffffu, l_run[n][e], i);
                if (g == 0) m_s[warp][row] = m_run[n][e], l_s[warp][row] = l_run[n][e];
                // (l is 2^14 or more: the division comes first, so that nothing leaves float32's range before the result does)
                const float inv = l_run[n][e] != 0.f ? 1.f / l_run[n][e] : 0.f;
                const float u1 = pow2(unit_run[n][e] / 2), u2 = pow2(unit_run[n][e] - unit_run[n][e] / 2);
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    auto value = [&](int d, int h) { return d < DT ? o[d][n][2 * h + e] * inv * u1 * u2 : 0.f; };
                    *reinterpret_cast<float4*>(&shared_o[(warp * ROWS + row) * LD + (w * 8 + g) * 4]) =
                        make_float4(value(2 * w, 0), value(2 * w, 1), value(2 * w + 1, 0), value(2 * w + 1, 1));
                }
            }
        __syncthreads();
        const int first_block = (pair_begin + ahead) / target, runs = (pair_begin + ahead + r.pages - 1) / target - first_block + 1, run = number - first_block;
        // where run k of this pair leaves its results: a block's first pair in the first of its two places
        auto place_of = [&](int k) { return place_in(pair_begin, first_block + k, target); };
        const int items = n_rows * VW * 8;
        if (a.cluster > 1) {
            join_cluster<T, D, NR>(out, a, shared_o, &m_s[0][0], &l_s[0][0], items, row0, r.begin, kvh, rank, first_block, run, runs, &ticket_s);
            break;   // (a cluster has one pair)
        }
        for (int i = threadIdx.x; i < items; i += THREADS) {
            const int row = i / (VW * 8);
            float m = EA_NONE, l = 0.f, part[EA_WARPS];
#pragma unroll
            for (int k = 0; k < EA_WARPS; ++k) m = fmaxf(m, m_s[k][row]);
#pragma unroll
            for (int k = 0; k < EA_WARPS; ++k) l += part[k] = fast_exp2(m_s[k][row] - m) * l_s[k][row];   // (a warp without pages: nothing)
            const float inv = l != 0.f ? 1.f / l : 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < EA_WARPS; ++k) {
                const float f = part[k] * inv;
                const float4 x = *reinterpret_cast<const float4*>(&shared_o[(k * ROWS + row) * LD + i % (VW * 8) * 4]);
                v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
            }
            if (runs == 1) {
                give_out<T, D>(out + row_at(row), v, i % (VW * 8));
            } else {
                *reinterpret_cast<float4*>(a.part_o + (long long)place_of(run) * ROWS * PART + i * 4) = v;
                if (i % (VW * 8) == 0) *reinterpret_cast<float2*>(a.part_ml + (place_of(run) * ROWS + row) * 2) = make_float2(m, l);
            }
        }
        if (runs > 1) {
            if (threadIdx.x == 0) left_s[n_left] = {pair_begin, first_block, runs, n_rows, row0, kvh, r.begin};
            ++n_left;   // (two at the most: a block's first pair and its last)
        }
        __syncthreads();   // (the next pair takes the same shared memory)
    }
    if (a.cluster > 1) {   // (no block's shared memory goes while another may read it)
        cluster_arrive();
        cluster_wait();
    }
    // ---- pairs of several blocks: whoever leaves the last of sixteen results joins them, whoever joins the last sixteen joins the sixteens
    for (int k = 0; k < n_left; ++k) {
        const Pair pair = left_s[k];
        const int run = (int)blockIdx.x - pair.first_block, group = run / EA_GROUP, groups = (pair.runs + EA_GROUP - 1) / EA_GROUP;
        const int home = place_in(pair.begin, pair.first_block + group * EA_GROUP, target);
        for (int level = 0; level < 2; ++level) {
            const int count = level == 0 ? min(EA_GROUP, pair.runs - group * EA_GROUP) : groups;
            if (!drew_last(a.tickets + (level == 0 ? home : 2 * n_blocks + place_in(pair.begin, pair.first_block, target)), count, &ticket_s)) break;
            join_parts<T, D, NR>(out, a, pair, target, level == 0 ? group * EA_GROUP : 0, level == 0 ? 1 : EA_GROUP, count, level == 0 && groups > 1 ? home : -1, factor_s);
            if (groups == 1) break;
        }
    }
    if (!waited) grid_dependency_wait();
    // padding entries: zeros
    for (int s = n_blocks - 1 - blockIdx.x; s < a.n_seqs; s += n_blocks) {
        const Sequence x = sequence_of<ROWS>(a, s);
        if (x.slot < 0)
            for (long long i = threadIdx.x; i < (long long)x.tokens * q_width; i += THREADS) out[(long long)x.begin * q_width + i] = Num<T>::from_f(0.f);
    }
}

// Blocks that the device holds at once of this shape; 0 where the shape has no kernel.
template <typename T, int D, int NR> static int slots_of() {
    static int cached[64];
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
    if (cached[device] == 0) {
        int n = 0;
        if (cudaFuncSetAttribute(attend_e4m3_kernel<T, D, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<T, D, NR>::SMEM) != cudaSuccess ||
            cudaFuncSetAttribute(attend_e4m3_kernel<T, D, NR>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attend_e4m3_kernel<T, D, NR>, EA_WARPS * 32, Shape<T, D, NR>::SMEM) != cudaSuccess)
            return 0;
        cached[device] = std::min(n * qf_sm_count(), EA_GROUP * EA_MOST_GROUPS);
    }
    return cached[device];
}
// Clusters of 2^log blocks that the device holds at once.
template <typename T, int D, int NR> static int clusters_of(int log) {
    static int cached[64][5];
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
    int& n = cached[device][log];
    if (n == 0) {
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(1 << log);
        config.blockDim = dim3(EA_WARPS * 32);
        config.dynamicSmemBytes = Shape<T, D, NR>::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1 << log;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        config.attrs = attr;
        config.numAttrs = 1;
        int found = 0;
        if (cudaOccupancyMaxActiveClusters(&found, attend_e4m3_kernel<T, D, NR>, &config) != cudaSuccess || found <= 0) {
            (void)cudaGetLastError();   // (none of this size)
            found = -1;
        }
        n = found;
    }
    return n;
}
template <typename T, int D, int NR> static int attend(const void* q, void* out, AttendArgs& a, int blocks, cudaStream_t stream) {
    if (a.block_slots <= 0 || a.block_slots != slots_of<T, D, NR>()) return (int)cudaErrorInvalidValue;
    // Where clusters have room for every pair at once, they take its pages: eight blocks (sixteen, if that is what a pair's pages want) bring their
    // results together without the way through memory. Microseconds, without clusters / with: one chat of 900 tokens, 14 heads over 2 of 64, 8.3 / 7.7,
    // 8 of 4,096 10.4 / 9.2, 20 of 1,000 10.2 / 8.6; 28 over 4 of 128, 7 of 1,000 11.3 / 9.1, one of 8,000 14.2 / 11.6. More than seven ninths of the device's
    // places are not for clusters, which want theirs side by side: 8 of 300 tokens (256 blocks of 296) 10.6 / 12.3, 4 of 4,000 (256) 12.1 / 15.0, 8 of 1,000 11.5 / 11.5,
    // heads of 64, 12 of 4,096 (384 of 444) 10.6 / 13.0, 11 of up to 4,096 (352) 9.8 / 10.1.
    for (int log = a.most_pages > EA_WARPS * 8 ? 4 : 3; log >= 3 && a.cluster_log == 0; --log) {
        const long long all = (long long)a.n_seqs * a.site.kv_heads * a.chunks * ((a.most_pages + (EA_WARPS << log) - 1) / (EA_WARPS << log));
        if ((all << log) * 9 <= a.block_slots * 7ll && all <= clusters_of<T, D, NR>(log)) a.cluster_log = log, blocks = (int)all << log;
    }
    a.cluster = 1 << a.cluster_log;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(EA_WARPS * 32);
    config.dynamicSmemBytes = Shape<T, D, NR>::SMEM;
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = a.cluster > 1 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&config, attend_e4m3_kernel<T, D, NR>, (const T*)q, (T*)out, a);
}

#define EA_EVERY(T, NR, CALL)               \
    switch (head_dim) {                     \
        case 16: return CALL(T, 16, NR);    \
        case 32: return CALL(T, 32, NR);    \
        case 48: return CALL(T, 48, NR);    \
        case 64: return CALL(T, 64, NR);    \
        case 80: return CALL(T, 80, NR);    \
        case 96: return CALL(T, 96, NR);    \
        case 112: return CALL(T, 112, NR);  \
        case 128: return CALL(T, 128, NR);  \
    }
#define EA_ALL(CALL)                        \
    if (is_bf16 && rows == 8) {             \
        EA_EVERY(bf16, 1, CALL)             \
    } else if (is_bf16 && rows == 16) {     \
        EA_EVERY(bf16, 2, CALL)             \
    } else if (rows == 8) {                 \
        EA_EVERY(float, 1, CALL)            \
    } else if (rows == 16) {                \
        EA_EVERY(float, 2, CALL)            \
    }

// Blocks that the current device holds at once for a head size and blocks of 8 or 16 rows (0: there is no kernel for it): what the workspaces are
// sized by.
QF_EXPORT int qf_attention_e4m3_slots(int is_bf16, int head_dim, int rows) {
#define EA_SLOTS(T, D, NR) slots_of<T, D, NR>()
    EA_ALL(EA_SLOTS)
    return 0;
}

// q, out [n_tokens][n_heads * head_dim], on 16 bytes; single: there are as many tokens as entries, and an entry has one at the most; rows: of a block, 8 or 16; chunks: of the longest span, ceil(tokens *
// n_heads / kv_heads / rows); most_pages: the most pages that a sequence reads; blocks: n_seqs * kv_heads * chunks * ceil(most_pages / 4), block_slots (of
// qf_attention_e4m3_slots) at most. part_o [2 * blocks][rows][32 * ceil(head_dim / 32)], part_ml [2 * blocks][rows][2]; tickets [4 * blocks], zero before the
// first call and after every call.
QF_EXPORT int qf_attention_e4m3(int is_bf16, const void* q, void* out, const int* cu_q, const int* tok_pos, const int* slots, void* codes, float* scales,
                                const int* table, long long page_bytes, long long page_scales, int table_stride, int columns, int n_slots, int kv_heads,
                                int head_dim, int n_heads, int n_seqs, int n_tokens, int single, int rows, int chunks, int most_pages, int blocks, int block_slots, float scale, int window, int constants,
                                float* part_o, float* part_ml, int* tickets, int* err, cudaStream_t stream) {
    const E4m3Site site{(unsigned char*)codes, scales, table, page_bytes, page_scales, table_stride, columns, n_slots, kv_heads, head_dim};
    if (n_seqs <= 0) return 0;
    if (head_dim <= 0 || head_dim % 16 || kv_heads <= 0 || n_heads <= 0 || n_heads % kv_heads || chunks <= 0 || most_pages <= 0 || most_pages >= 1 << 20 || columns <= 0 || n_slots <= 0 ||
        page_bytes % 16 || ((uintptr_t)codes | (uintptr_t)q | (uintptr_t)out) % 16 || page_bytes < 2ll * kv_heads * QF_PAGE * head_dim || page_scales < 2ll * kv_heads ||
        (rows != 8 && rows != 16) || blocks <= 0 || blocks > block_slots || window < 0)
        return (int)cudaErrorInvalidValue;
    // pages of all (sequence, kv head, rows) are counted in 32 bits: an entry has a block of rows for each `rows` of its own and one that is partly empty
    const long long row_blocks = std::min((long long)n_seqs * chunks, (long long)n_tokens * (n_heads / kv_heads) / rows + n_seqs);
    if (row_blocks * kv_heads * (most_pages + 2ll * block_slots) > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    AttendArgs a{cu_q, tok_pos, slots, site, n_heads, n_heads / kv_heads, n_seqs, single, chunks, most_pages, block_slots, window, constants, 1, 0, scale * 1.4426950408889634f, part_o, part_ml, tickets, err};
#define EA_ATTEND(T, D, NR) attend<T, D, NR>(q, out, a, blocks, stream)
    EA_ALL(EA_ATTEND)
    return (int)cudaErrorInvalidValue;
}
