// Verification of drafted tokens against a model's logits (float32). With p = softmax(target / T), q = softmax(draft / T):
//   draft d_j is kept while  u_j q_j(d_j) < p_j(d_j);  the token behind the last kept one is  argmax_i r_i / E_i,  r = max(0, p - q) at a refusal
//   (p without d where there are no draft logits) and r = p behind the last draft,  E_i = -ln u_i, u_i the sampler's number for token i of that step.
// argmax_i r_i / E_i draws i with probability r_i / sum r (independent exponential times of rate r_i: the first to go), so neither r's sum nor a
// running sum over the vocabulary is needed, and a token turns on rounding only where two scores are equal to the last bits.
// T <= 0: kept while it is the row's argmax (lowest id of equals); the next token is the argmax.
//
// Three launches. (1) A block takes VF_CHUNK logits of a row, all of them in registers at once: their maximum, its lowest id, and the sum of the
// exponentials against it. (2) A block takes an entry: it brings the rows' statistics together (a warp per draft), decides how many drafts stay, and
// writes all outputs but the token that is drawn. (3) A block takes a chunk of the row that follows and scores its tokens; the block that draws the
// entry's last ticket picks the best. (At T <= 0 the second launch writes everything.)
// What bounds it: memory, in (1); in (3), of the same rows out of the second-level cache, the hash and the logarithm of every token.
//
// Decisions are whole numbers, so they are made on sums that are good to more than float32: sums over threads and blocks and the comparison u q < p are
// float64, and of a chunk's scores, formed in float32, those within the error bound of the best are formed again in float64.
#include <float.h>
#include <math.h>

#include "mma.cuh"
#include "random.cuh"

#define VF_THREADS 256
#define VF_EACH 32                             // logits of a thread
#define VF_CHUNK (VF_THREADS * VF_EACH)
#define VR_THREADS 256
#define VR_FEW 8                               // tokens of a thread in (3): few where there are few blocks, many else
#define VR_MANY 32

// What (2) leaves for (3).
struct Decision {
    int kept, row, d_row, without;   // kept -1: nothing to draw; the rows of target and draft logits (-1: none), the token that is ruled out (-1: none)
    float t_top, d_top;
    double t_sum, d_sum;
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
    RowStats* stats;         // [rows + draft rows]
    Decision* decisions;     // [n]
    double2* best;           // [n][race chunks]: score, id
    int* counters;           // [n]
    int rows, total, vocab, n, most, chunks, race_chunks;
    double inv_t;
    float rate;              // log2(e) / T
    unsigned long long seed;
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

// ---- (1) maximum, its lowest id and the sum of exponentials of VF_CHUNK logits of a row. The difference from the maximum, its product with log2(e) / T
// and that factor itself round by 2^-24 each of an exponent, the hardware's exponential by 2^-22: of single weights, some up and some down.
__global__ void __launch_bounds__(VF_THREADS)
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

// A row's statistics from its chunks', by one warp: every lane gets them.
__device__ __forceinline__ RowStats row_stats(const VerifyArgs& a, int row) {
    const int lane = threadIdx.x & 31;
    const float2* tops = a.tops + (size_t)row * a.chunks;
    const double* sums = a.sums + (size_t)row * a.chunks;
    RowStats s = {-INFINITY, 0x7fffffff, 0.0};
    float2 mine = make_float2(-INFINITY, __int_as_float(0x7fffffff));
    double part = 0.0;
    if (lane < a.chunks) mine = tops[lane], part = sums[lane];   // (32 chunks are 262,144 logits: the loop below is for vocabularies beyond)
    s.top = mine.x, s.id = __float_as_int(mine.y);
    for (int c = lane + 32; c < a.chunks; c += 32) {
        const float2 t = tops[c];
        const int id = __float_as_int(t.y);
        if (t.x > s.top || (t.x == s.top && id < s.id)) s.top = t.x, s.id = id;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float top = __shfl_xor_sync(0xffffffffu, s.top, o);
        const int id = __shfl_xor_sync(0xffffffffu, s.id, o);
        if (top > s.top || (top == s.top && id < s.id)) s.top = top, s.id = id;
    }
    if (a.sampling) {
        double sum = mine.x > -INFINITY ? part * exp(((double)mine.x - (double)s.top) * a.inv_t) : 0.0;
        for (int c = lane + 32; c < a.chunks; c += 32) {
            const float m = tops[c].x;
            if (m > -INFINITY) sum += sums[c] * exp(((double)m - (double)s.top) * a.inv_t);
        }
        s.sum = warp_sum_f64(sum);
    }
    return s;
}

// ---- (2) how many drafts of an entry stay
__global__ void __launch_bounds__(VR_THREADS)
verify_decide_kernel(VerifyArgs a) {
    grid_chain_entry();
    constexpr int WARPS = VR_THREADS / 32;
    __shared__ int kept_s;
    const int s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int before = 0;   // entries with rows in front of this one: each has a row more than it has drafts
    for (int i = 0; i < s; i += VR_THREADS) {
        const int e = i + threadIdx.x;
        before += __syncthreads_count(e < s && a.first[e + 1] > a.first[e]);
    }
    const int row0 = a.first[s], row1 = a.first[s + 1], count = row1 - row0 - 1, draft0 = row0 - before;
    const bool empty = row1 == row0, wrong = !empty && (row0 < 0 || count < 0 || row1 > a.rows || count > a.most || draft0 < 0 || draft0 + count > a.total);
    int* const tokens = a.tokens + (size_t)s * (a.most + 1);
    if (empty || wrong) {
        if (threadIdx.x == 0) {
            a.accepted[s] = wrong ? -1 : 0;
            a.decisions[s].kept = -1;
        }
        for (int i = threadIdx.x; i <= a.most; i += VR_THREADS) tokens[i] = -1;
        return;
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
        const RowStats t = row_stats(a, row0 + j);
        RowStats r = {0.f, 0, 1.0};
        if (a.draft && j < count) r = row_stats(a, a.rows + draft0 + j);
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
            a.stats[row0 + j] = t;
            if (a.draft && j < count) a.stats[a.rows + draft0 + j] = r;
            if (!keep) atomicMin(&kept_s, j);
        }
    }
    __syncthreads();
    const int kept = kept_s;   // (its row has been worked out: no warp leaves out a row up to the lowest refused one)
    for (int i = threadIdx.x; i <= a.most; i += VR_THREADS)
        if (i != kept) tokens[i] = i < kept ? a.drafted[draft0 + i] : -1;
    if (threadIdx.x == 0) {
        const RowStats t = a.stats[row0 + kept];
        const bool refused = kept < count;
        a.accepted[s] = kept;
        if (!a.sampling) {
            tokens[kept] = t.id >= a.vocab ? 0 : t.id;
            return;
        }
        RowStats r = {0.f, 0, 1.0};
        if (refused && a.draft) r = a.stats[a.rows + draft0 + kept];
        a.decisions[s] = Decision{kept, row0 + kept, refused && a.draft ? draft0 + kept : -1, refused && !a.draft ? a.drafted[draft0 + kept] : -1,
                                  t.top, r.top, t.sum, r.sum};
    }
}

// ---- (3) the token behind the kept drafts. A score is r / E. p = 2^((x - top) rate - log2 sum): the difference, the product and the exponent round by
// 2^-24 each, of numbers that are at most a few tens for any token with a chance, and the hardware's exponential by 2^-22: p is within 6e-6 of its value
// as a share. E = -ln u: near 1 by its series in w = 1 - u, which is exact in float32, else by the hardware's logarithm, within 6e-6 as well. So a score
// lies between (p - q - 6e-6 (p + q)) (1 - 6e-6) / E and the same with other signs; of a thread's tokens the two with the highest upper bounds are
// kept, and whichever of them reach the block's highest lower bound are scored again in float64.
#define VR_SLACK 6.0e-6f
template <int EACH>
__global__ void __launch_bounds__(VR_THREADS)
verify_draw_kernel(VerifyArgs a) {
    grid_chain_entry();
    constexpr int WARPS = VR_THREADS / 32, CHUNK = VR_THREADS * EACH;
    __shared__ int ticket_s, id_s[WARPS];
    __shared__ float low_s[WARPS];
    __shared__ double best_s[WARPS];
    const int s = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Decision made = a.decisions[s];
    if (made.kept < 0) return;
    const float* t_row = a.target + made.row * a.t_stride;
    const float* d_row = made.d_row >= 0 ? a.draft + made.d_row * a.d_stride : nullptr;
    const int begin = blockIdx.x * CHUNK, end = min(a.vocab, begin + CHUNK);
    float x[EACH], y[EACH];
    load_logits(t_row, begin, end, x);
    if (d_row) load_logits(d_row, begin, end, y);
    const uint32_t key = row_key(a.seed, a.seq_ids[s], a.steps[s] + made.kept);
    const float t_log = (float)log2(made.t_sum), d_log = (float)log2(made.d_sum);
    float high[2] = {-1.f, -1.f}, low = -1.f;
    int high_at[2] = {-1, -1};
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int id = id_of(begin, i);
        const float p = fast_exp2(fmaf(x[i] - made.t_top, a.rate, -t_log));
        const float q = d_row ? fast_exp2(fmaf(y[i] - made.d_top, a.rate, -d_log)) : 0.f;
        const uint32_t bits = token_bits(key, (uint32_t)id);
        const float u = ((float)bits + 0.5f) * (1.0f / 8388608.0f), w = ((float)(8388607u - bits) + 0.5f) * (1.0f / 8388608.0f);
        const float wait = w < 0.03125f ? w * fmaf(w, fmaf(w, fmaf(w, fmaf(w, 0.2f, 0.25f), 0.33333333f), 0.5f), 1.f) : -0.69314718f * __log2f(u);
        const float r = p - q, slack = (p + q) * VR_SLACK, per = __fdividef(1.f, wait);
        const bool in = id < end && id != made.without;
        const float may = in ? fmaf(r, VR_SLACK, r + slack) * per : -1.f;
        if (in) low = fmaxf(low, (r - slack) * (1.f - VR_SLACK) * per);
        if (may > high[0]) {
            high[1] = high[0], high_at[1] = high_at[0];
            high[0] = may, high_at[0] = i;
        } else if (may > high[1]) {
            high[1] = may, high_at[1] = i;
        }
    }
    low = warp_max(fmaxf(low, 0.f));
    if (lane == 0) low_s[warp] = low;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) low = fmaxf(low, low_s[w]);
    double best = -1.0;
    int best_id = 0x7fffffff;
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
        const float reach = k ? high[1] : high[0];
        const int i = k ? high_at[1] : high_at[0];
        if (i < 0 || !(reach >= low)) continue;
        const int id = id_of(begin, i);
        double r = exp(((double)t_row[id] - (double)made.t_top) * a.inv_t) / made.t_sum;
        if (d_row) r = fmax(r - exp(((double)d_row[id] - (double)made.d_top) * a.inv_t) / made.d_sum, 0.0);
        const double score = r / -log(((double)token_bits(key, (uint32_t)id) + 0.5) / 8388608.0);
        if (score > best || (score == best && id < best_id)) best = score, best_id = id;
    }
    auto better = [](double v, int i, double than, int than_i) { return v > than || (v == than && i < than_i); };
    auto warp_best = [&]() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double v = __shfl_xor_sync(0xffffffffu, best, o);
            const int i = __shfl_xor_sync(0xffffffffu, best_id, o);
            if (better(v, i, best, best_id)) best = v, best_id = i;
        }
    };
    warp_best();
    if (lane == 0) best_s[warp] = best, id_s[warp] = best_id;
    __syncthreads();
    if (warp != 0) return;
    best = lane < WARPS ? best_s[lane] : -1.0;
    best_id = lane < WARPS ? id_s[lane] : 0x7fffffff;
    warp_best();
    if (lane == 0) {
        a.best[(size_t)s * a.race_chunks + blockIdx.x] = make_double2(best, (double)best_id);
        __threadfence();
        ticket_s = atomicAdd(a.counters + s, 1);
    }
    __syncwarp();
    if (ticket_s != (int)gridDim.x - 1) return;
    __threadfence();
    best = -1.0;
    best_id = 0x7fffffff;
    for (int c = lane; c < (int)gridDim.x; c += 32) {
        const double2 b = __ldcg(a.best + (size_t)s * a.race_chunks + c);
        if (better(b.x, (int)b.y, best, best_id)) best = b.x, best_id = (int)b.y;
    }
    warp_best();
    if (lane == 0) {
        a.counters[s] = 0;
        a.tokens[(size_t)s * (a.most + 1) + made.kept] = best_id >= a.vocab ? 0 : best_id;
    }
}

// target [rows][t_stride >= vocab] and draft [total][d_stride] (or null) float32; drafted, uniforms [total]; first [n + 1]; accepted [n],
// tokens [n][most + 1]. Workspaces: sums (8 bytes) and tops (8) of (rows + draft rows) x chunks of VF_CHUNK, stats (16) of rows + draft rows, decisions
// (40) of n, best (16) of n x chunks of VR_THREADS * VR_FEW, counters int32 of n, zero before the first call (the kernels leave them zero).
QF_EXPORT int qf_verify_drafts(const float* target, int rows, int vocab, long long t_stride, const float* draft, long long d_stride, const int* drafted,
                               int total, const int* first, int n, const float* uniforms, float temperature, unsigned long long seed,
                               const long long* seq_ids, const int* steps, int* accepted, int* tokens, int most, double* sums, void* tops, void* stats,
                               void* decisions, void* best, int* counters, cudaStream_t stream) {
    static_assert(sizeof(Decision) == 40 && sizeof(RowStats) == 16, "what the workspaces are sized by");
    if (n <= 0 || vocab <= 0) return 0;
    VerifyArgs a = {};
    a.target = target, a.draft = draft, a.t_stride = t_stride, a.d_stride = d_stride, a.drafted = drafted, a.first = first, a.uniforms = uniforms;
    a.seq_ids = seq_ids, a.steps = steps, a.accepted = accepted, a.tokens = tokens, a.sums = sums, a.tops = (float2*)tops, a.stats = (RowStats*)stats;
    a.decisions = (Decision*)decisions, a.best = (double2*)best, a.counters = counters, a.rows = rows, a.total = total, a.vocab = vocab, a.n = n;
    a.most = most, a.seed = seed, a.sampling = temperature > 0.f;
    a.chunks = (vocab + VF_CHUNK - 1) / VF_CHUNK, a.race_chunks = (vocab + VR_THREADS * VR_FEW - 1) / (VR_THREADS * VR_FEW);
    if (a.sampling) {
        a.inv_t = 1.0 / (double)temperature;
        a.rate = (float)(1.4426950408889634 * a.inv_t);
    }
    const long long all = (long long)rows + (draft ? total : 0);
    if (n > 65535 || all > 65535) return (int)cudaErrorInvalidValue;
    cudaError_t e = cudaSuccess;
    if (all > 0) e = launch_pdl(verify_rows_kernel, dim3((unsigned)a.chunks, (unsigned)all), dim3(VF_THREADS), 0, stream, a);
    if (e == cudaSuccess) e = launch_pdl(verify_decide_kernel, dim3((unsigned)n), dim3(VR_THREADS), 0, stream, a);
    if (e != cudaSuccess || !a.sampling) return (int)e;
    // Blocks of 2,048 tokens where they all fit the SMs at once (five to an SM), of 8,192 else.
    const unsigned many = (unsigned)((vocab + VR_THREADS * VR_MANY - 1) / (VR_THREADS * VR_MANY));
    if ((long long)a.race_chunks * n <= 5ll * qf_sm_count())
        return (int)launch_pdl(verify_draw_kernel<VR_FEW>, dim3((unsigned)a.race_chunks, (unsigned)n), dim3(VR_THREADS), 0, stream, a);
    return (int)launch_pdl(verify_draw_kernel<VR_MANY>, dim3(many, (unsigned)n), dim3(VR_THREADS), 0, stream, a);
}
