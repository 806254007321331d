// Verification of drafted tokens against a model's logits (float32). With p = softmax(target / T), q = softmax(draft / T):
//   draft d_j is kept while  u_j q_j(d_j) < p_j(d_j);  the token behind the last kept one is  argmax_i r_i / E_i,  r = max(0, p - q) at a refusal
//   (p without d where there are no draft logits) and r = p behind the last draft,  E_i = -ln u_i, u_i the sampler's number for token i of that step.
// argmax_i r_i / E_i draws i with probability r_i / sum r (independent exponential times of rate r_i: the first to go), so neither r's sum nor a
// running sum over the vocabulary is needed, and a token turns on rounding only where two scores are equal to the last bits.
// T <= 0: kept while it is the row's argmax (lowest id of equals); the next token is the argmax.
//
// Two launches. (1) A block takes VF_CHUNK logits of a row, all of them in registers at once: their maximum, its lowest id, and the sum of the
// exponentials against it. (2) A block takes VR_CHUNK tokens of an entry: it brings the rows' statistics together (a warp per draft), decides how many
// drafts stay, and scores its tokens of the row that follows; the block that draws the entry's last ticket picks the best and writes the outputs.
//
// Decisions are whole numbers, so they are made on sums that are good to more than float32: the argument (x - max) log2(e) / T is formed with its
// rounding errors (two floats), sums over threads and blocks and the comparison u q < p are float64, and of a block's scores, formed in float32,
// those within the error bound of the best are formed again in float64.
#include <float.h>
#include <math.h>

#include "mma.cuh"
#include "random.cuh"

#define VF_THREADS 256
#define VF_EACH 32                             // logits of a thread
#define VF_CHUNK (VF_THREADS * VF_EACH)
#define VR_THREADS 256
#define VR_EACH 8
#define VR_CHUNK (VR_THREADS * VR_EACH)

// log2(e) / T as two floats.
struct Rate {
    float hi, lo;
};

// 2^((x - top) rate) with the errors of the difference and of the product carried along: within 2^-22 of the value plus the hardware exponential's
// own error, whatever the size of the argument.
__device__ __forceinline__ float weight_of(float x, float top, Rate r) {
    const float d = x - top;
    if (!(d > -FLT_MAX)) return 0.f;             // -infinity: no weight (an infinite difference has no rounding error to carry)
    const float back = x - d, e = (x - (d + back)) + (back - top);   // d + e = x - top
    const float y = d * r.hi, low = fmaf(d, r.hi, -y) + fmaf(d, r.lo, e * r.hi);
    return fast_exp2(y) * fmaf(low, 0.6931471805599453f, 1.f);
}

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
    double2* best;           // [n][race chunks]: score, id
    int* counters;           // [n]
    int rows, total, vocab, n, most, chunks, race_chunks;
    double inv_t;
    Rate rate;
    unsigned long long seed;
    int sampling;
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ---- (1) maximum, its lowest id and the sum of exponentials of VF_CHUNK logits of a row
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
    int at[VF_EACH / 4];   // first id of each four
    if ((reinterpret_cast<uintptr_t>(x + begin) & 15) == 0) {
#pragma unroll
        for (int u = 0; u < VF_EACH / 4; ++u) {
            at[u] = begin + 4 * (threadIdx.x + u * VF_THREADS);
            if (at[u] + 4 <= end) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(x + at[u]));
                v[4 * u] = f.x, v[4 * u + 1] = f.y, v[4 * u + 2] = f.z, v[4 * u + 3] = f.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * u + e] = at[u] + e < end ? x[at[u] + e] : -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < VF_EACH / 4; ++u) {
            at[u] = begin + 4 * (threadIdx.x + u * VF_THREADS);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * u + e] = at[u] + e < end ? x[at[u] + e] : -INFINITY;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < VF_EACH; ++i) top = fmaxf(top, v[i]);
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
            if (v[i] == most && at[i / 4] + (i & 3) < end) id = min(id, at[i / 4] + (i & 3));
    }
    double sum = 0.0;
    if (a.sampling) {
#pragma unroll
        for (int u = 0; u < VF_EACH / 4; ++u) {
            const float s = (weight_of(v[4 * u], most, a.rate) + weight_of(v[4 * u + 1], most, a.rate)) +
                            (weight_of(v[4 * u + 2], most, a.rate) + weight_of(v[4 * u + 3], most, a.rate));
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
struct RowStats {
    float top;
    int id;
    double sum;
};
__device__ __forceinline__ RowStats row_stats(const VerifyArgs& a, int row) {
    const int lane = threadIdx.x & 31;
    RowStats s = {-INFINITY, 0x7fffffff, 0.0};
    for (int c = lane; c < a.chunks; c += 32) {
        const float2 t = a.tops[(size_t)row * a.chunks + c];
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
        double sum = 0.0;
        for (int c = lane; c < a.chunks; c += 32) {
            const float m = a.tops[(size_t)row * a.chunks + c].x;
            if (m > -INFINITY) sum += a.sums[(size_t)row * a.chunks + c] * exp(((double)m - (double)s.top) * a.inv_t);
        }
        s.sum = warp_sum_f64(sum);
    }
    return s;
}

// ---- (2) how many drafts stay, and the token behind them
__global__ void __launch_bounds__(VR_THREADS)
verify_choose_kernel(VerifyArgs a) {
    grid_chain_entry();
    constexpr int WARPS = VR_THREADS / 32;
    __shared__ int kept_s, ticket_s, id_s[WARPS];
    __shared__ float low_s[WARPS], t_top, d_top;
    __shared__ double t_sum, d_sum, best_s[WARPS];
    const int s = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int before = 0;   // entries with rows in front of this one: each has a row more than it has drafts
    for (int i = 0; i < s; i += VR_THREADS) {
        const int e = i + threadIdx.x;
        before += __syncthreads_count(e < s && a.first[e + 1] > a.first[e]);
    }
    const int row0 = a.first[s], row1 = a.first[s + 1], count = row1 - row0 - 1, draft0 = row0 - before;
    const bool empty = row1 == row0, wrong = !empty && (row0 < 0 || count < 0 || row1 > a.rows || count > a.most || draft0 < 0 || draft0 + count > a.total);
    if (empty || wrong) {
        if (blockIdx.x == 0) {
            if (threadIdx.x == 0) a.accepted[s] = wrong ? -1 : 0;
            for (int i = threadIdx.x; i <= a.most; i += VR_THREADS) a.tokens[(size_t)s * (a.most + 1) + i] = -1;
        }
        return;
    }
    if (threadIdx.x == 0) kept_s = count;
    __syncthreads();
    for (int j = warp; j < count; j += WARPS) {   // a warp per draft; the first that is refused ends the kept run
        if (j >= __shfl_sync(0xffffffffu, *(volatile int*)&kept_s, 0)) break;
        const int d = a.drafted[draft0 + j];
        const bool known = d >= 0 && d < a.vocab;
        const RowStats t = row_stats(a, row0 + j);
        bool keep;
        if (!a.sampling) {
            keep = known && t.id == d;
        } else {
            const double p = known ? exp(((double)a.target[(row0 + j) * a.t_stride + d] - (double)t.top) * a.inv_t) / t.sum : 0.0;
            double q = 1.0;
            if (a.draft) {
                const RowStats r = row_stats(a, a.rows + draft0 + j);
                q = known ? exp(((double)a.draft[(draft0 + j) * a.d_stride + d] - (double)r.top) * a.inv_t) / r.sum : 1.0;
            }
            keep = known && (double)a.uniforms[draft0 + j] * q < p;
        }
        if (lane == 0 && !keep) atomicMin(&kept_s, j);
    }
    __syncthreads();
    const int kept = kept_s, row = row0 + kept;
    const bool refused = kept < count;
    const int d_row = draft0 + kept;
    auto write = [&](int chosen) {
        for (int i = threadIdx.x; i <= a.most; i += VR_THREADS)
            a.tokens[(size_t)s * (a.most + 1) + i] = i < kept ? a.drafted[draft0 + i] : i == kept ? chosen : -1;
        if (threadIdx.x == 0) a.accepted[s] = kept;
    };
    if (!a.sampling) {   // (one block an entry)
        if (warp == 0) {
            const RowStats t = row_stats(a, row);
            if (lane == 0) id_s[0] = t.id >= a.vocab ? 0 : t.id;
        }
        __syncthreads();
        write(id_s[0]);
        return;
    }
    if (warp == 0) {
        const RowStats t = row_stats(a, row);
        if (lane == 0) t_top = t.top, t_sum = t.sum;
    } else if (warp == 1 && refused && a.draft) {
        const RowStats r = row_stats(a, a.rows + d_row);
        if (lane == 0) d_top = r.top, d_sum = r.sum;
    }
    __syncthreads();
    const float* t_row = a.target + row * a.t_stride;
    const float* d_logits = refused && a.draft ? a.draft + d_row * a.d_stride : nullptr;
    const int without = refused && !a.draft ? a.drafted[d_row] : -1;
    const uint32_t key = row_key(a.seed, a.seq_ids[s], a.steps[s] + kept);
    const float t_inv = (float)(1.0 / t_sum), d_inv = d_logits ? (float)(1.0 / d_sum) : 0.f;
    // the two best of a thread, by the upper bounds of their scores
    float high[2] = {-1.f, -1.f}, low = -1.f;
    int high_id[2] = {-1, -1};
    const int begin = blockIdx.x * VR_CHUNK, end = min(a.vocab, begin + VR_CHUNK);
#pragma unroll
    for (int u = 0; u < VR_EACH; ++u) {
        const int i = begin + threadIdx.x + u * VR_THREADS;
        if (i >= end || i == without) continue;
        const float p = weight_of(t_row[i], t_top, a.rate) * t_inv;
        const float q = d_logits ? weight_of(d_logits[i], d_top, a.rate) * d_inv : 0.f;
        const float uniform = ((float)token_bits(key, (uint32_t)i) + 0.5f) * (1.0f / 8388608.0f);
        const float wait = -logf(uniform);
        // p and q are within 2^-20 of their values, the quotient within 2^-21 more
        const float slack = (p + q) * 2.0e-6f, sure = fmaxf(p - q - slack, 0.f) / wait, may = fmaxf(p - q + slack, 0.f) / wait;
        low = fmaxf(low, sure);
        if (may > high[0]) {
            high[1] = high[0], high_id[1] = high_id[0];
            high[0] = may, high_id[0] = i;
        } else if (may > high[1]) {
            high[1] = may, high_id[1] = i;
        }
    }
    low = warp_max(low);
    if (lane == 0) low_s[warp] = low;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) low = fmaxf(low, low_s[w]);
    double best = -1.0;
    int best_id = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (high_id[k] < 0 || !(high[k] >= low)) continue;
        const int i = high_id[k];
        double r = exp(((double)t_row[i] - (double)t_top) * a.inv_t) / t_sum;
        if (d_logits) r = fmax(r - exp(((double)d_logits[i] - (double)d_top) * a.inv_t) / d_sum, 0.0);
        const double score = r / -log(((double)token_bits(key, (uint32_t)i) + 0.5) / 8388608.0);
        if (score > best || (score == best && i < best_id)) best = score, best_id = i;
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
    if (warp == 0) {
        best = lane < WARPS ? best_s[lane] : -1.0;
        best_id = lane < WARPS ? id_s[lane] : 0x7fffffff;
        warp_best();
        if (lane == 0) {
            a.best[(size_t)s * a.race_chunks + blockIdx.x] = make_double2(best, (double)best_id);
            __threadfence();
            ticket_s = atomicAdd(a.counters + s, 1);
        }
    }
    __syncthreads();
    if (ticket_s != a.race_chunks - 1) return;
    __threadfence();
    if (warp == 0) {
        best = -1.0;
        best_id = 0x7fffffff;
        for (int c = lane; c < a.race_chunks; c += 32) {
            const double2 b = __ldcg(a.best + (size_t)s * a.race_chunks + c);
            if (better(b.x, (int)b.y, best, best_id)) best = b.x, best_id = (int)b.y;
        }
        warp_best();
        if (lane == 0) {
            a.counters[s] = 0;
            id_s[0] = best_id >= a.vocab ? 0 : best_id;
        }
    }
    __syncthreads();
    write(id_s[0]);
}

// Chunks of a row in (1), and of an entry in (2).
QF_EXPORT int qf_verify_chunks(int vocab, int* sizes) {
    sizes[0] = (vocab + VF_CHUNK - 1) / VF_CHUNK;
    sizes[1] = (vocab + VR_CHUNK - 1) / VR_CHUNK;
    return 0;
}

// target [rows][t_stride >= vocab] and draft [total][d_stride] (or null) float32; drafted, uniforms [total]; first [n + 1]; accepted [n],
// tokens [n][most + 1]; sums, tops, best, counters: workspaces of (rows + draft rows) x chunks, n x race chunks and n, counters zero before the
// first call (the kernel leaves them zero).
QF_EXPORT int qf_verify_drafts(const float* target, int rows, int vocab, long long t_stride, const float* draft, long long d_stride, const int* drafted,
                               int total, const int* first, int n, const float* uniforms, float temperature, unsigned long long seed,
                               const long long* seq_ids, const int* steps, int* accepted, int* tokens, int most, double* sums, void* tops, void* best,
                               int* counters, cudaStream_t stream) {
    if (n <= 0 || vocab <= 0) return 0;
    VerifyArgs a = {};
    a.target = target, a.draft = draft, a.t_stride = t_stride, a.d_stride = d_stride, a.drafted = drafted, a.first = first, a.uniforms = uniforms;
    a.seq_ids = seq_ids, a.steps = steps, a.accepted = accepted, a.tokens = tokens, a.sums = sums, a.tops = (float2*)tops, a.best = (double2*)best;
    a.counters = counters, a.rows = rows, a.total = total, a.vocab = vocab, a.n = n, a.most = most, a.seed = seed, a.sampling = temperature > 0.f;
    a.chunks = (vocab + VF_CHUNK - 1) / VF_CHUNK, a.race_chunks = (vocab + VR_CHUNK - 1) / VR_CHUNK;
    if (a.sampling) {
        a.inv_t = 1.0 / (double)temperature;
        const double rate = 1.4426950408889634 * a.inv_t;
        a.rate.hi = (float)rate;
        a.rate.lo = (float)(rate - (double)a.rate.hi);
    }
    const long long all = (long long)rows + (draft ? total : 0);
    if (n > 65535 || all > 65535) return (int)cudaErrorInvalidValue;
    if (all > 0) {
        const cudaError_t e = launch_pdl(verify_rows_kernel, dim3((unsigned)a.chunks, (unsigned)all), dim3(VF_THREADS), 0, stream, a);
        if (e != cudaSuccess) return (int)e;
    }
    return (int)launch_pdl(verify_choose_kernel, dim3(a.sampling ? (unsigned)a.race_chunks : 1u, (unsigned)n), dim3(VR_THREADS), 0, stream, a);
}
