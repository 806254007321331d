// Verification of drafted tokens against a model's logits (float32). With p = softmax(target / T), q = softmax(draft / T):
//   draft d_j is kept while  u_j q_j(d_j) < p_j(d_j);  the token behind the last kept one is  argmax_i r_i / E_i,  r = max(0, p - q) at a refusal
//   (p without d where there are no draft logits) and r = p behind the last draft,  E_i = -ln u_i, u_i the sampler's number for token i of that step,
//   under a seed of its own at a refusal with draft logits: given that d was refused, numbers that d was drawn with are no longer what they were.
// argmax_i r_i / E_i draws i with probability r_i / sum r (independent exponential times of rate r_i: the first to go), so neither r's sum nor a
// running sum over the vocabulary is needed, and a token turns on rounding only where two scores are equal to the last bits.
// T <= 0: kept while it is the row's argmax (lowest id of equals); the next token is the argmax.
//
// Two launches. (1) A block takes VF_CHUNK logits of a row, all of them in registers at once: their maximum, its lowest id, and the sum of the
// exponentials against it. (2) Every block of an entry brings its rows' statistics together (a warp per draft) and decides how many drafts stay; one writes
// what follows. Then they score the tokens of the row behind the kept drafts, chunk after chunk, and the block that draws the entry's last ticket
// picks the best. (That every block decides for itself costs less than a launch between, and than tickets in (1), which hold its blocks up: 48 entries, 346
// rows of 151,936: (1) 32 microseconds, with tickets 49.)
// Measured: those 48 entries 53.3 us: (1) 32, 210 MB at 6.6 TB/s, (2) 21, of which the decision 3.7; one entry of four drafts 10.0; argmaxes of 48 rows
// of 152,064, 7.1.
// What bounds it: memory, in (1); in (2), latency, and of the same rows out of the second-level cache the hash and the logarithm of the tokens that may
// still win.
//
// Decisions are whole numbers, so they are made on sums that are good to more than float32: sums over threads and blocks and the comparison u q < p are
// float64 (of exponentials of 2^-20 or better, so a draft whose u q and p are closer than that may go either way). Scores are formed in float32 with bounds of
// their errors; where two or more tokens may be the best by those, one block forms the row's sums and those tokens' scores again in float64.
#include <float.h>
#include <math.h>

#include "mma.cuh"
#include "random.cuh"

#define VF_THREADS 256
#define VF_EACH 32                             // logits of a thread
#define VF_CHUNK (VF_THREADS * VF_EACH)
#define VR_EACH 8                              // tokens of a thread and chunk in (2)
#define VR_CHUNK (VF_THREADS * VR_EACH)
// Blocks of an SM at once. Tokens of a thread / blocks, one entry of four drafts and 48 of up to seven (the kernel's and (1)'s microseconds, vocabulary of
// 151,936): 8 / 3 10.0 and 53.4; 8 / 4 11.0 and 54.3; 8 / 5 11.6 and 57.0; 4 / 6 11.7 and 58.9; 4 / 8 16.0 and 63.8 (registers spill); 16 / 2 11.2 and 53.3.
#define VR_BLOCKS 3

// What a block has decided.
struct Decision {
    int kept, row, d_row, without;   // the rows of target and draft logits that a token is drawn from (-1: none), the token that is ruled out (-1: none)
    float t_top, d_top, t_log, d_log;   // the rows' maxima, and the base-2 logarithms of their sums
    double t_sum, d_sum;
};
// Of some tokens, the best by the upper bounds of their scores (id 0x7fffffff: none), the next highest upper bound, and the highest lower bound; none of the
// bounds is negative.
struct __align__(16) Contenders {
    float high, second, low;
    int id;
};

struct RowStats {
    float top;       // the largest logit, and its lowest id
    int id;
    double sum;      // of e^((x - top) / T)
};

struct VerifyArgs {
    const float* target;
    const float* draft;      // null: none
    long long t_stride, d_stride;
    const int* drafted;
    const int* first;
    const float* uniforms;
    const long long* seq_ids;
    const int* steps;
    int* accepted;
    int* tokens;
    double* sums;            // [rows + draft rows][chunks]
    float2* tops;            // the same: maximum, its id as bits
    Contenders* best;        // [n][chunks of (2)]
    int* counters;           // [n]
    int rows, total, vocab, n, most, chunks, race_chunks;
    double inv_t;
    float rate;              // log2(e) / T
    unsigned long long seed, redraw_seed;   // redraw_seed: of draws behind a refused draft that has logits
    int sampling;
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// EACH logits of a thread from x[begin ..): fours of neighbours, VF_THREADS fours apart; -infinity from `end` on. at(i): the id of the i-th.
template <int EACH>
__device__ __forceinline__ void load_logits(const float* x, int begin, int end, float (&v)[EACH]) {
    const bool aligned = (reinterpret_cast<uintptr_t>(x + begin) & 15) == 0;
#pragma unroll
    for (int u = 0; u < EACH / 4; ++u) {
        const int i = begin + 4 * (threadIdx.x + u * VF_THREADS);
        if (aligned && i + 4 <= end) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(x + i));
            v[4 * u] = f.x, v[4 * u + 1] = f.y, v[4 * u + 2] = f.z, v[4 * u + 3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * u + e] = i + e < end ? __ldg(x + i + e) : -INFINITY;
        }
    }
}
__device__ __forceinline__ int id_of(int begin, int i) { return begin + 4 * (threadIdx.x + i / 4 * VF_THREADS) + (i & 3); }

// The statistics of a target row and of the draft row beside it (-1: none, a sum of 1) from their chunks', by one warp: every lane gets them. What the
// chunks leave is asked for at once; a chunk's factor 2^((its maximum - the row's) rate) is the hardware's, within 2^-22.
__device__ __forceinline__ void row_stats(const VerifyArgs& a, int row, int d_row, RowStats& t, RowStats& r) {
    const int lane = threadIdx.x & 31, rows[2] = {row, d_row};
    float2 mine[2];
    double part[2] = {0.0, 0.0};
    RowStats s[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const bool in = rows[k] >= 0 && lane < a.chunks;
        mine[k] = in ? __ldcg(a.tops + (size_t)rows[k] * a.chunks + lane) : make_float2(-INFINITY, __int_as_float(0x7fffffff));
        if (in && a.sampling) part[k] = __ldcg(a.sums + (size_t)rows[k] * a.chunks + lane);
        s[k].top = mine[k].x, s[k].id = __float_as_int(mine[k].y);
        for (int c = lane + 32; rows[k] >= 0 && c < a.chunks; c += 32) {   // (32 chunks are 262,144 logits)
            const float2 x = __ldcg(a.tops + (size_t)rows[k] * a.chunks + c);
            if (x.x > s[k].top || (x.x == s[k].top && __float_as_int(x.y) < s[k].id)) s[k].top = x.x, s[k].id = __float_as_int(x.y);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float top = __shfl_xor_sync(0xffffffffu, s[k].top, o);
            const int id = __shfl_xor_sync(0xffffffffu, s[k].id, o);
            if (top > s[k].top || (top == s[k].top && id < s[k].id)) s[k].top = top, s[k].id = id;
        }
    if (a.sampling) {
        double sum[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            sum[k] = mine[k].x > -INFINITY ? part[k] * (double)fast_exp2((mine[k].x - s[k].top) * a.rate) : 0.0;
            for (int c = lane + 32; rows[k] >= 0 && c < a.chunks; c += 32) {
                const float m = __ldcg(a.tops + (size_t)rows[k] * a.chunks + c).x;
                if (m > -INFINITY) sum[k] += __ldcg(a.sums + (size_t)rows[k] * a.chunks + c) * (double)fast_exp2((m - s[k].top) * a.rate);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < 2; ++k) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
        s[0].sum = sum[0], s[1].sum = sum[1];
    }
    if (d_row < 0) s[1] = RowStats{0.f, 0, 1.0};
    t = s[0], r = s[1];
}

// ---- (1) maximum, its lowest id and the sum of exponentials of VF_CHUNK logits of a row. The difference from the maximum, its product with log2(e) / T
// and that factor itself round by 2^-24 each of an exponent, the hardware's exponential by 2^-22: of single weights, some up and some down.
__global__ void __launch_bounds__(VF_THREADS, 4)
verify_rows_kernel(VerifyArgs a) {
    grid_chain_entry();
    __shared__ float top_s[VF_THREADS / 32];
    __shared__ int id_s[VF_THREADS / 32];
    __shared__ double sum_s[VF_THREADS / 32];
    const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* x = row < a.rows ? a.target + row * a.t_stride : a.draft + (row - a.rows) * a.d_stride;
    const int begin = blockIdx.x * VF_CHUNK, end = min(a.vocab, begin + VF_CHUNK);
    float v[VF_EACH];
    load_logits(x, begin, end, v);
    float top = v[0];
#pragma unroll
    for (int i = 1; i < VF_EACH; ++i) top = fmaxf(top, v[i]);
    float most = warp_max(top);
    if (lane == 0) top_s[warp] = most;
    __syncthreads();
    most = top_s[0];
#pragma unroll
    for (int w = 1; w < VF_THREADS / 32; ++w) most = fmaxf(most, top_s[w]);
    int id = 0x7fffffff;
    if (top == most) {
#pragma unroll
        for (int i = VF_EACH - 1; i >= 0; --i)
            if (v[i] == most && id_of(begin, i) < end) id = id_of(begin, i);   // (ids of a thread rise with i)
    }
    double sum = 0.0;
    if (a.sampling && most > -INFINITY) {   // (else no token of the chunk has a weight)
#pragma unroll
        for (int u = 0; u < VF_EACH / 8; ++u) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) s += fast_exp2((v[8 * u + e] - most) * a.rate);   // (-infinity: 0)
            sum += (double)s;
        }
        sum = warp_sum_f64(sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) id = min(id, __shfl_xor_sync(0xffffffffu, id, o));
    if (lane == 0) {
        id_s[warp] = id;
        sum_s[warp] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < VF_THREADS / 32; ++w) {
            id = min(id, id_s[w]);
            sum += sum_s[w];
        }
        const size_t place = (size_t)row * a.chunks + blockIdx.x;
        a.sums[place] = sum;
        a.tops[place] = make_float2(most, __int_as_float(id));
    }
}

// ---- (2) how many drafts of an entry stay, by all threads of a block; false: there is nothing to draw.
__device__ __forceinline__ bool decide(const VerifyArgs& a, int s, bool writes, Decision& made) {
    constexpr int WARPS = VF_THREADS / 32, CACHE = 32;
    __shared__ int kept_s;
    __shared__ RowStats t_s[CACHE], r_s[CACHE], last_s[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int before = 0;   // entries with rows in front of this one: each has a row more than it has drafts
    for (int i = 0; i < s; i += VF_THREADS) {
        const int e = i + threadIdx.x;
        before += __syncthreads_count(e < s && a.first[e + 1] > a.first[e]);
    }
    const int row0 = a.first[s], row1 = a.first[s + 1], count = row1 - row0 - 1, draft0 = row0 - before;
    const bool empty = row1 == row0, wrong = !empty && (row0 < 0 || count < 0 || row1 > a.rows || count > a.most || draft0 < 0 || draft0 + count > a.total);
    int* const tokens = a.tokens + (size_t)s * (a.most + 1);
    if (empty || wrong) {
        if (writes) {
            if (threadIdx.x == 0) a.accepted[s] = wrong ? -1 : 0;
            for (int i = threadIdx.x; i <= a.most; i += VF_THREADS) tokens[i] = -1;
        }
        return false;
    }
    if (threadIdx.x == 0) kept_s = count;
    __syncthreads();
    for (int j = warp; j <= count; j += WARPS) {   // a warp per draft, and one for the row behind the last; the first that is refused ends the kept run
        if (j > __shfl_sync(0xffffffffu, *(volatile int*)&kept_s, 0)) break;
        const int d = j < count ? a.drafted[draft0 + j] : -1;
        const bool known = d >= 0 && d < a.vocab;
        const double u = a.sampling && j < count ? (double)a.uniforms[draft0 + j] : 0.0;
        const float t_logit = a.sampling && known ? a.target[(row0 + j) * a.t_stride + d] : 0.f;
        const float d_logit = a.draft && known ? a.draft[(draft0 + j) * a.d_stride + d] : 0.f;
        RowStats t, r;
        row_stats(a, row0 + j, a.draft && j < count ? a.rows + draft0 + j : -1, t, r);
        bool keep = j == count;
        if (!keep && known) {
            if (!a.sampling) {
                keep = t.id == d;
            } else {
                const double p = exp(((double)t_logit - (double)t.top) * a.inv_t) / t.sum;
                const double q = a.draft ? exp(((double)d_logit - (double)r.top) * a.inv_t) / r.sum : 1.0;
                keep = u * q < p;
            }
        }
        if (lane == 0) {
            if (j < CACHE) t_s[j] = t, r_s[j] = r;
            if (!keep) atomicMin(&kept_s, j);
        }
    }
    __syncthreads();
    const int kept = kept_s;   // (its row has been worked out: no warp leaves out a row up to the lowest refused one)
    const bool refused = kept < count;
    if (kept >= CACHE) {
        if (warp == 0) {
            RowStats t, r;
            row_stats(a, row0 + kept, refused && a.draft ? a.rows + draft0 + kept : -1, t, r);
            if (lane == 0) last_s[0] = t, last_s[1] = r;
        }
        __syncthreads();
    }
    const RowStats t = kept < CACHE ? t_s[kept] : last_s[0], r = kept < CACHE ? r_s[kept] : last_s[1];
    if (writes) {
        for (int i = threadIdx.x; i <= a.most; i += VF_THREADS)
            if (i != kept) tokens[i] = i < kept ? a.drafted[draft0 + i] : -1;
        if (threadIdx.x == 0) {
            a.accepted[s] = kept;
            if (!a.sampling) tokens[kept] = t.id >= a.vocab ? 0 : t.id;
        }
    }
    made = Decision{kept, row0 + kept, refused && a.draft ? draft0 + kept : -1, refused && !a.draft ? a.drafted[draft0 + kept] : -1,
                    t.top, r.top, __log2f((float)t.sum), __log2f((float)r.sum), t.sum, r.sum};
    return a.sampling;
}

// ---- (2) the token behind the kept drafts. A score is r / E. p = 2^((x - top) rate - log2 sum): the difference, the product and the exponent round by 2^-24
// each of a number of bits, 1.3e-7 of p per bit; the sum is good to 2.7e-6 (weights' errors of 1.3e-7 per bit below the maximum, of which a mean has 14 at
// most, the hardware's exponentials, eight additions in float32), its logarithm to 1e-6, the hardware's exponential to 2.4e-7. So p is within 1e-5 of its value, as a
// share, for every token down to 2^-45 of the largest, and none below that has a chance (E is 2^-24 at the least). E = -ln u: near 1 by its series in
// w = 1 - u, which is exact in float32, else by the hardware's logarithm, within 6e-6. So a score lies between (p - q - 1e-5 (p + q)) (1 - 1e-5) / E and the
// same with other signs. A thread, a warp, a block keeps the token with the highest upper bound, the next highest upper bound, and the highest lower bound.
// Where the entry's next highest upper bound is below its highest lower bound, the token with the highest is the best: nearly always, but for models so
// close that what is left of p - q is lost in the slack; else `rescore`. Since E >= w, a token whose upper bound on p - q is below w times the lower bound
// so far cannot win: nearly none needs a logarithm or a division. The bound goes round a warp after every four tokens of its threads, and round the
// block after every chunk.
#define VR_SLACK 1.0e-5f
__device__ __forceinline__ void keep_best(Contenders& x, float high, int id) {
    if (high > x.high || (high == x.high && id < x.id)) {
        x.second = x.high;
        x.high = high, x.id = id;
    } else {
        x.second = fmaxf(x.second, high);
    }
}
// Of all threads of a block, to all of them: bounds that are not negative compare as their bits do, which a warp reduces in one instruction.
__device__ __forceinline__ Contenders of_warp(const Contenders& x) {
    Contenders y;
    const unsigned high = __float_as_uint(x.high), most = __reduce_max_sync(0xffffffffu, high);
    y.high = __uint_as_float(most);
    y.id = __reduce_min_sync(0xffffffffu, high == most ? x.id : 0x7fffffff);
    // (a lane whose best is the warp's best stands in with its second)
    y.second = __uint_as_float(__reduce_max_sync(0xffffffffu, x.id == y.id ? __float_as_uint(x.second) : high));
    y.low = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x.low)));
    return y;
}
__device__ __forceinline__ Contenders of_block(const Contenders& x, Contenders* room) {
    constexpr int WARPS = VF_THREADS / 32;
    const int lane = threadIdx.x & 31;
    const Contenders mine = of_warp(x);
    __syncthreads();
    if (lane == 0) room[threadIdx.x >> 5] = mine;
    __syncthreads();
    Contenders y = {0.f, 0.f, 0.f, 0x7fffffff};
    if (lane < WARPS) y = room[lane];
    return of_warp(y);
}

// r and its slack for one token, r = -1 where its upper bound does not reach: reach = 2^23 / (the highest lower bound so far).
__device__ __forceinline__ bool may_win(const VerifyArgs& a, const Decision& made, bool with_draft, float x, float y, uint32_t bits, float reach, float& r, float& slack) {
    const float p = fast_exp2(fmaf(x - made.t_top, a.rate, -made.t_log));
    const float q = with_draft ? fast_exp2(fmaf(y - made.d_top, a.rate, -made.d_log)) : 0.f;
    r = p - q, slack = (p + q) * VR_SLACK;
    // 2^23 w: 23 bits under the exponent of 2^23 are that number more than themselves. (Behind the vocabulary's end: 0 < 0, or a NaN.)
    return __uint_as_float(0x4b000000u | (8388607u - bits)) - 8388607.5f < (r + slack) * reach;
}
__device__ __forceinline__ float reach_of(float low) {
    return __fdividef(8388608.f * 1.000001f, low);   // (of the quotient's rounding, upwards; infinite as long as there is no bound)
}

// The entry's best token in float64, by all threads of a block: the rows' sums (without a draft row, scores p / E compare without them), then the scores of the
// tokens whose upper bounds reach `low`. The lowest id of equals; 0x7fffffff where no token has a score above 0. 0.35 ms for rows of
// 151,936: of ordinary models about one draw in 10^5 comes here, of models whose logits differ by 10^-4 or less most that follow a refusal (of which there are
// as few as the models are close). Not inlined, so that its registers are not the others'.
__device__ __noinline__ int rescore(const VerifyArgs& a, const Decision& made, const float* t_row, const float* d_row, uint32_t key, float low) {
    constexpr int WARPS = VF_THREADS / 32;
    __shared__ double part_s[2][WARPS];
    __shared__ int id_s[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double sum[2] = {0.0, 0.0};
    if (d_row) {
        for (int i = threadIdx.x; i < a.vocab; i += VF_THREADS) {
            sum[0] += exp(((double)t_row[i] - (double)made.t_top) * a.inv_t);
            sum[1] += exp(((double)d_row[i] - (double)made.d_top) * a.inv_t);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            sum[k] = warp_sum_f64(sum[k]);
            if (lane == 0) part_s[k][warp] = sum[k];
        }
        __syncthreads();
        sum[0] = sum[1] = 0.0;
        for (int w = 0; w < WARPS; ++w) sum[0] += part_s[0][w], sum[1] += part_s[1][w];
        __syncthreads();
    }
    const float reach = reach_of(low);
    double best = 0.0;
    int chosen = 0x7fffffff;
    for (int i = threadIdx.x; i < a.vocab; i += VF_THREADS) {
        float r32, slack;
        const uint32_t bits = token_bits(key, (uint32_t)i);
        if (i == made.without || !may_win(a, made, d_row != nullptr, t_row[i], d_row ? d_row[i] : 0.f, bits, reach, r32, slack)) continue;
        double r = exp(((double)t_row[i] - (double)made.t_top) * a.inv_t);
        if (d_row) r = r / sum[0] - exp(((double)d_row[i] - (double)made.d_top) * a.inv_t) / sum[1];
        const double score = r / -log(((double)bits + 0.5) / 8388608.0);
        if (score > best) best = score, chosen = i;   // (ids of a thread rise)
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double v = __shfl_xor_sync(0xffffffffu, best, o);
        const int i = __shfl_xor_sync(0xffffffffu, chosen, o);
        if (v > best || (v == best && i < chosen)) best = v, chosen = i;
    }
    if (lane == 0) part_s[0][warp] = best, id_s[warp] = chosen;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w)
        if (part_s[0][w] > best || (part_s[0][w] == best && id_s[w] < chosen)) best = part_s[0][w], chosen = id_s[w];
    return chosen;
}

__global__ void __launch_bounds__(VF_THREADS, VR_BLOCKS)
verify_draw_kernel(const __grid_constant__ VerifyArgs a) {
    grid_chain_entry();
    constexpr int WARPS = VF_THREADS / 32;
    __shared__ int low_s, ticket_s;
    __shared__ Contenders best_s[WARPS];
    const int s = blockIdx.y, lane = threadIdx.x & 31;
    const long long seq_id = a.sampling ? a.seq_ids[s] : 0;
    const int step = a.sampling ? a.steps[s] : 0;
    Decision made;
    if (!decide(a, s, blockIdx.x == 0, made)) return;
    const float* t_row = a.target + made.row * a.t_stride;
    const float* d_row = made.d_row >= 0 ? a.draft + made.d_row * a.d_stride : nullptr;
    // (A refused draft may have been drawn with this step's numbers under `seed`: the draw behind it must not depend on those.)
    const uint32_t key = row_key(made.d_row >= 0 ? a.redraw_seed : a.seed, seq_id, step + made.kept);
    if (threadIdx.x == 0) low_s = 0;   // the highest lower bound that a thread has found, as bits of a float32 that is not negative
    __syncthreads();
    Contenders mine = {0.f, 0.f, 0.f, 0x7fffffff};
    float x[VR_EACH], y[VR_EACH], x_next[VR_EACH], y_next[VR_EACH];   // (the next chunk's are on their way while this one's are scored)
    auto load = [&](int begin) {
        const int end = min(a.vocab, begin + VR_CHUNK);
        if (begin >= end) return;
        load_logits(t_row, begin, end, x_next);
        if (d_row) load_logits(d_row, begin, end, y_next);
    };
    load(blockIdx.x * VR_CHUNK);
    for (int begin = blockIdx.x * VR_CHUNK; begin < a.vocab; begin += gridDim.x * VR_CHUNK) {
#pragma unroll
        for (int i = 0; i < VR_EACH; ++i) x[i] = x_next[i], y[i] = y_next[i];
        load(begin + gridDim.x * VR_CHUNK);
        float low = fmaxf(mine.low, __int_as_float(*(volatile int*)&low_s));
        const float before = low;
#pragma unroll
        for (int u = 0; u < VR_EACH; u += 4) {
            const float reach = reach_of(low);
            float r[4], slack[4];
            uint32_t bits[4];
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                bits[e] = token_bits(key, (uint32_t)id_of(begin, u + e));
                if (!may_win(a, made, d_row != nullptr, x[u + e], y[u + e], bits[e], reach, r[e], slack[e])) r[e] = -1.f;
                any |= r[e] > -1.f;
            }
            if (any) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int id = id_of(begin, u + e);
                    if (!(r[e] > -1.f) || id == made.without) continue;
                    const float w = ((float)(8388607u - bits[e]) + 0.5f) * (1.0f / 8388608.0f);
                    const float v = ((float)bits[e] + 0.5f) * (1.0f / 8388608.0f);
                    const float wait = w < 0.03125f ? w * fmaf(w, fmaf(w, fmaf(w, fmaf(w, 0.2f, 0.25f), 0.33333333f), 0.5f), 1.f) : -0.69314718f * __log2f(v);
                    const float per = __fdividef(1.f, wait);
                    low = fmaxf(low, (r[e] - slack[e]) * (1.f - VR_SLACK) * per);
                    keep_best(mine, fmaxf(fmaf(r[e], VR_SLACK, r[e] + slack[e]) * per, 0.f), id);
                }
            }
            low = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(low)));
        }
        mine.low = low;
        if (begin + (int)gridDim.x * VR_CHUNK < a.vocab && lane == 0 && low > before) atomicMax(&low_s, __float_as_int(low));
    }
    mine = of_block(mine, best_s);
    Contenders* all = a.best + (size_t)s * a.race_chunks;
    if (threadIdx.x == 0) {
        all[blockIdx.x] = mine;
        __threadfence();
        ticket_s = atomicAdd(a.counters + s, 1);
    }
    __syncthreads();
    if (ticket_s != (int)gridDim.x - 1) return;
    __threadfence();
    // the entry's last block: what the others have left
    mine = Contenders{0.f, 0.f, 0.f, 0x7fffffff};
    for (int c = threadIdx.x; c < (int)gridDim.x; c += VF_THREADS) {
        const float4 other = __ldcg(reinterpret_cast<const float4*>(all + c));
        keep_best(mine, other.x, __float_as_int(other.w));
        mine.second = fmaxf(mine.second, other.y);
        mine.low = fmaxf(mine.low, other.z);
    }
    mine = of_block(mine, best_s);
    int chosen = mine.id;
    if (mine.second >= mine.low) chosen = rescore(a, made, t_row, d_row, key, mine.low);   // two or more may be the best
    if (threadIdx.x == 0) {
        a.counters[s] = 0;
        a.tokens[(size_t)s * (a.most + 1) + made.kept] = chosen >= a.vocab ? 0 : chosen;
    }
}

// target [rows][t_stride >= vocab] and draft [total][d_stride] (or null) float32; drafted, uniforms [total]; first [n + 1]; accepted [n],
// tokens [n][most + 1]. Workspaces: sums (8 bytes) and tops (8) of (rows + draft rows) x chunks of VF_CHUNK, best (16) of n x chunks of VR_CHUNK,
// counters int32 of n, zero before the first call (the kernels leave them zero).
QF_EXPORT int qf_verify_drafts(const float* target, int rows, int vocab, long long t_stride, const float* draft, long long d_stride, const int* drafted,
                               int total, const int* first, int n, const float* uniforms, float temperature, unsigned long long seed,
                               unsigned long long redraw_seed, const long long* seq_ids, const int* steps, int* accepted, int* tokens, int most,
                               double* sums, void* tops, void* best, int* counters, cudaStream_t stream) {
    static_assert(sizeof(Contenders) == 16, "what the workspaces are sized by");
    if (n <= 0 || vocab <= 0) return 0;
    VerifyArgs a = {};
    a.target = target, a.draft = draft, a.t_stride = t_stride, a.d_stride = d_stride, a.drafted = drafted, a.first = first, a.uniforms = uniforms;
    a.seq_ids = seq_ids, a.steps = steps, a.accepted = accepted, a.tokens = tokens, a.sums = sums, a.tops = (float2*)tops;
    a.best = (Contenders*)best, a.counters = counters, a.rows = rows, a.total = total, a.vocab = vocab, a.n = n;
    a.most = most, a.seed = seed, a.redraw_seed = redraw_seed, a.sampling = temperature > 0.f;
    a.chunks = (vocab + VF_CHUNK - 1) / VF_CHUNK, a.race_chunks = (vocab + VR_CHUNK - 1) / VR_CHUNK;
    if (a.sampling) {
        a.inv_t = 1.0 / (double)temperature;
        a.rate = (float)fmin(1.4426950408889634 * a.inv_t, (double)FLT_MAX);   // (an infinite one times a difference of 0 would be no number)
    }
    const long long all = (long long)rows + (draft ? total : 0);
    if (n > 65535 || all > 65535) return (int)cudaErrorInvalidValue;
    if (all > 0) {
        const cudaError_t e = launch_pdl(verify_rows_kernel, dim3((unsigned)a.chunks, (unsigned)all), dim3(VF_THREADS), 0, stream, a);
        if (e != cudaSuccess) return (int)e;
    }
    // as many blocks to an entry as make all of them run at once
    const int each = a.sampling ? VR_BLOCKS * qf_sm_count() / n : 1;
    return (int)launch_pdl(verify_draw_kernel, dim3((unsigned)(each < 1 ? 1 : each < a.race_chunks ? each : a.race_chunks), (unsigned)n), dim3(VF_THREADS), 0, stream, a);
}
