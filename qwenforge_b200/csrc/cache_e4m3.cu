// Writing a sequence cache of e4m3 codes, and reading it back (the format: e4m3.cuh).
//
// ---- Write, behind the q/k/v projection of a step's tokens: x = row + bias; queries and keys rotated (split halves over the first R
// components, as rope_cache.cu, with angles that are as exact at position 30,000 as at 3); queries written out. For every page that gets new
// rows, of each plane and kv head:
//   amax = max |x| over the new rows' finite elements,  e = the least exponent with amax <= 448 * 2^e
//   the page had rows before (the first new one does not begin it): e = max(e, e_old), and where that is more than e_old, those
//   rows' codes become round(code * 2^(e_old - e))
//   new codes = round(x * 2^-e), to nearest even, from float32: one rounding
// A page that is begun takes its exponent from its new rows alone, whatever an earlier holder left there. Rows behind the new ones stay.
//
// A run is a page's new rows. Two kernels, the same in what they write:
//   write_runs     spans of EW_LONG tokens or more: a block takes a run and some of the heads, all its threads one head at a time. A thread has the
//                  same one or two pieces (a row, eight pairs of the rotation) of every head, so their sines and cosines are worked out once
//                  and stay in registers, a key's or value's elements stay there between amax and codes, and the next head's are loaded
//                  meanwhile. One prompt of 8,192 tokens, 28 + 4 + 4 heads of 128 in bfloat16: 38 microseconds, 3.7 TB/s (142 MB, 22 at the
//                  copy's rate). It waits for its loads: 128 registers a thread leave four warps to a scheduler, with one head's rows each on their way; half of the
//                  issue slots are used, and per issue 2.2 warps wait for memory, 0.9 for the instruction before. Twelve float32 prompts of up to
//                  900 tokens, 16 + 2 + 2 heads of 128: 17.4 microseconds, 3.9 TB/s.
//   write_any      single tokens, short spans, and rows or rotations that 16-byte accesses do not fit: a warp a head at a time over all rows of
//                  a run; amax and codes are one warp's business, without a barrier. Sines and cosines come from shared memory, worked
//                  out once per run. A key or value head is read twice, the second time from L1 or L2. One token of one sequence: 3.1
//                  microseconds, of 96 sequences at 28 + 4 + 4 heads of 128 4.5: a chain of loads (position, page, scale), the angle, the
//                  warp's maximum. Spans of 8 tokens of 64 sequences there: 10.1, for 1.4 of bytes: rows are loaded and turned twice, and a warp has a head alone.
#include <algorithm>

#include "e4m3.cuh"

#define EW_WARPS 8

// VEC elements from `p` (8: 16-byte accesses) as float32, with their bias.
template <typename T, int VEC> __device__ __forceinline__ void load_values(const T* p, const T* b, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = Num<T>::to_f(p[0]) + (b ? Num<T>::to_f(b[0]) : 0.f);
    } else {
        constexpr int PER = 16 / sizeof(T);   // elements of an access
        uint4 raw[VEC / PER], braw[VEC / PER];
#pragma unroll
        for (int i = 0; i < VEC / PER; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
        if (b) {
#pragma unroll
            for (int i = 0; i < VEC / PER; ++i) braw[i] = reinterpret_cast<const uint4*>(b)[i];
        }
        const T *x = reinterpret_cast<const T*>(raw), *y = reinterpret_cast<const T*>(braw);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = Num<T>::to_f(x[i]) + (b ? Num<T>::to_f(y[i]) : 0.f);
    }
}
template <typename T, int VEC> __device__ __forceinline__ void store_values(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        p[0] = Num<T>::from_f(v[0]);
    } else {
        constexpr int PER = 16 / sizeof(T);
        uint4 raw[VEC / PER];
        T* x = reinterpret_cast<T*>(raw);
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = Num<T>::from_f(v[i]);
#pragma unroll
        for (int i = 0; i < VEC / PER; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
    }
}
template <int VEC> __device__ __forceinline__ void store_codes(unsigned char* p, const float (&v)[VEC], float by) {
    if constexpr (VEC == 1) {
        *p = (unsigned char)e4m3_pair(v[0] * by, 0.f);
    } else {
        *reinterpret_cast<uint2*>(p) = make_uint2(e4m3_four(v[0] * by, v[1] * by, v[2] * by, v[3] * by), e4m3_four(v[4] * by, v[5] * by, v[6] * by, v[7] * by));
    }
}
// |v|, 0 for infinities and NaN
__device__ __forceinline__ float finite_size(float v) {
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.f;
}

// Codes of rows that a page had, rounded to a larger unit: code * `by`, by <= 1/2 a power of two.
__device__ __forceinline__ void rescale_codes(uint4* codes, int pieces, float by, int first, int step) {
    for (int i = first; i < pieces; i += step) {
        uint4 w = codes[i];
        uint32_t* words = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 lo = floats_of(half2_of_low(words[e])), hi = floats_of(half2_of_high(words[e]));
            words[e] = e4m3_four(lo.x * by, lo.y * by, hi.x * by, hi.y * by);
        }
        codes[i] = w;
    }
}

// Cosine and sine of position * frequency. The angle is taken in turns, position * (frequency / 2 pi) with both factors' rounding errors, so that whole
// turns fall away exactly and an angle of tens of thousands is as good as a small one. What the rest of a turn loses as one float32 (up to 2e-7 in the
// angle, as much as all that comes behind it) turns the result by a first-order step: with it a prompt of 8,192 tokens has one to six of its 8.4 million codes
// off those of the exact rotation, as a rotation by float64 angles has, without it six to seventeen; it costs 0.9 microseconds of 38 there.
struct Turns {
    float most, rest;   // frequency / 2 pi, in two parts
    __device__ __forceinline__ explicit Turns(float frequency) {
        const float inv = 0.15915494f, inv_rest = 6.42063824e-09f;   // 1 / 2 pi, in two parts
        most = frequency * inv;
        rest = fmaf(frequency, inv, -most) + frequency * inv_rest;
    }
    __device__ __forceinline__ float2 at(float position) const {
        const float product = position * most, high = product - rintf(product);
        const float low = fmaf(position, most, -product) + position * rest, part = high + low, lost = low - (part - high);
        float s0, c0;
        sincospif(2.f * part, &s0, &c0);
        const float step = 6.2831853f * lost, s = fmaf(c0, step, s0), c = fmaf(-s0, step, c0);
        return make_float2(c, s);
    }
};

// A run: the rows from token t on, of entry seq, that one page gets.
struct NewRows {
    int t, seq, rows, first_pos;
};
// The number-th run of a step. `single`: an entry's tokens are one (or none), and every token is a run.
__device__ __forceinline__ bool run_of(int number, int single, int n_seqs, const int* cu_q, const int* tok_seq, const int* tok_pos, NewRows& r) {
    if (single) {
        r = NewRows{number, tok_seq[number], 1, tok_pos[number]};
        return true;
    }
    const int lane = threadIdx.x & 31;
    for (int s0 = 0, before = 0; s0 < n_seqs; s0 += 32) {
        int begin = 0, count = 0, first = 0, runs = 0;
        if (s0 + lane < n_seqs) {
            begin = cu_q[s0 + lane];
            count = cu_q[s0 + lane + 1] - begin;
            if (count > 0) {
                first = tok_pos[begin];
                runs = (first + count - 1) / QF_PAGE - first / QF_PAGE + 1;
            }
        }
        int upto = runs;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t beyond = __ballot_sync(0xffffffffu, before + upto > number);
        if (beyond) {
            const int who = __ffs(beyond) - 1, k = number - before - __shfl_sync(0xffffffffu, upto - runs, who);
            begin = __shfl_sync(0xffffffffu, begin, who), count = __shfl_sync(0xffffffffu, count, who), first = __shfl_sync(0xffffffffu, first, who);
            const int from = k == 0 ? 0 : (first / QF_PAGE + k) * QF_PAGE - first;   // tokens of the entry before the run
            r = NewRows{begin + from, s0 + who, min(count - from, QF_PAGE - (first + from) % QF_PAGE), first + from};
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(EW_WARPS * 32)
write_any_kernel(const T* __restrict__ qkv, const T* __restrict__ bias, long long qkv_stride, const int* __restrict__ cu_q, const int* __restrict__ tok_seq,
                 const int* __restrict__ tok_pos, const int* __restrict__ slots, const float* __restrict__ inv_freq, int rot_dim, int n_heads,
                 T* __restrict__ q_out, E4m3Site site, int write_cache, int n_seqs, int single, int most_rows, int constants,
                 int* err) {
    grid_launch_dependents();
    if (!constants) grid_dependency_wait();
    extern __shared__ float2 turn[];   // [rows of a run][rot_dim / 2] cosine, sine
    const int D = site.head_dim, KVH = site.kv_heads, half = rot_dim / 2, pass = D - rot_dim;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int heads = n_heads + 2 * KVH;
    const int h_each = (heads + gridDim.y - 1) / gridDim.y, h_begin = blockIdx.y * h_each, h_end = min(h_begin + h_each, heads);
    NewRows run;
    if (!run_of(blockIdx.x, single, n_seqs, cu_q, tok_seq, tok_pos, run)) {
        grid_dependency_wait();
        return;
    }
    const int t = run.t, first_pos = run.first_pos, at = first_pos % QF_PAGE, seq = single ? min(max(run.seq, 0), n_seqs - 1) : run.seq;
    const int entry_begin = cu_q[seq], entry_end = cu_q[seq + 1], held = slots[seq];
    const bool inside = !single || (seq == run.seq && t >= entry_begin && t < entry_end);   // (or a row behind the last entry's, which nothing becomes of)
    const int slot = write_cache && inside ? held : -1;
    int rows = run.rows;
    if (rows > most_rows || (single && inside && entry_end - entry_begin > 1)) {   // (an entry longer than the call has said: there is no room for its angles.
        if (threadIdx.x == 0 && held >= 0) atomicOr(err, QF_ERR_ROW_RANGE);          // A padding entry may be: nobody asks for its queries)
        rows = min(rows, most_rows);
    }
    const int page = slot >= 0 ? e4m3_page(site, slot, first_pos) : -1;
    if (slot >= 0 && page < 0 && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(err, QF_ERR_NO_PAGE);
    for (int i = threadIdx.x; i < rows * half; i += blockDim.x) turn[i] = Turns(inv_freq[i % half]).at((float)(first_pos + i / half));
    if (!inside) rows = 0;
    __syncthreads();
    if (constants) grid_dependency_wait();   // (what is read from here on may be the output of the kernel ahead)
    for (int h = h_begin + warp; h < h_end; h += EW_WARPS) {
        const bool is_q = h < n_heads, is_v = h >= n_heads + KVH;
        if (!is_q && page < 0) continue;
        const int plane = is_v ? 1 : 0, kvh = is_v ? h - n_heads - KVH : h - n_heads;
        const T* src = qkv + (long long)t * qkv_stride + (long long)h * D;
        const T* b = bias ? bias + (long long)h * D : nullptr;
        unsigned char* codes = is_q ? nullptr : site.codes + (long long)page * site.page_bytes + (long long)(plane * KVH + kvh) * QF_PAGE * D;
        T* q_dst = q_out + (long long)t * n_heads * D + (long long)h * D;
        const int turned = is_v ? 0 : half / VEC, plain = is_v ? D / VEC : pass / VEC, plain0 = is_v ? 0 : rot_dim;
        // one item: VEC pairs of the rotation of a row, then VEC components that pass through
        auto pairs_of = [&](int i, int& row, int& j, float (&a)[VEC], float (&z)[VEC]) {
            row = i / turned, j = (i % turned) * VEC;
            const T* x = src + (long long)row * qkv_stride;
            float x1[VEC], x2[VEC];
            load_values<T, VEC>(x + j, b ? b + j : nullptr, x1);
            load_values<T, VEC>(x + j + half, b ? b + j + half : nullptr, x2);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 cs = turn[row * half + j + e];
                a[e] = x1[e] * cs.x - x2[e] * cs.y;
                z[e] = x2[e] * cs.x + x1[e] * cs.y;
            }
        };
        auto plain_of = [&](int i, int& row, int& j, float (&a)[VEC]) {
            row = i / plain, j = plain0 + (i % plain) * VEC;
            load_values<T, VEC>(src + (long long)row * qkv_stride + j, b ? b + j : nullptr, a);
        };
        int row, j;
        float a[VEC], z[VEC];
        if (is_q) {
            for (int i = lane; i < rows * turned; i += 32) {
                pairs_of(i, row, j, a, z);
                store_values<T, VEC>(q_dst + (long long)row * n_heads * D + j, a);
                store_values<T, VEC>(q_dst + (long long)row * n_heads * D + j + half, z);
            }
            for (int i = lane; i < rows * plain; i += 32) {
                plain_of(i, row, j, a);
                store_values<T, VEC>(q_dst + (long long)row * n_heads * D + j, a);
            }
            continue;
        }
        float amax = 0.f;
        for (int i = lane; i < rows * turned; i += 32) {
            pairs_of(i, row, j, a, z);
#pragma unroll
            for (int e = 0; e < VEC; ++e) amax = fmaxf(amax, fmaxf(finite_size(a[e]), finite_size(z[e])));
        }
        for (int i = lane; i < rows * plain; i += 32) {
            plain_of(i, row, j, a);
#pragma unroll
            for (int e = 0; e < VEC; ++e) amax = fmaxf(amax, finite_size(a[e]));
        }
        float* scale = site.scales + (long long)page * site.page_scales + plane * KVH + kvh;
        int exp = e4m3_exponent(warp_max(amax));
        if (at > 0) {
            const int before = exponent_of(*scale);
            exp = max(exp, before);
            if (exp > before) rescale_codes(reinterpret_cast<uint4*>(codes), at * D / 16, pow2(max(before - exp, -126)), lane, 32);
        }
        const float by = pow2(-exp);
        codes += at * D;
        for (int i = lane; i < rows * turned; i += 32) {
            pairs_of(i, row, j, a, z);
            store_codes<VEC>(codes + row * D + j, a, by);
            store_codes<VEC>(codes + row * D + j + half, z, by);
        }
        for (int i = lane; i < rows * plain; i += 32) {
            plain_of(i, row, j, a);
            store_codes<VEC>(codes + row * D + j, a, by);
        }
        __syncwarp();   // (every lane has read the old scale)
        if (lane == 0) *scale = pow2(exp);
    }
}

#define EW_THREADS 256

// PIECES of a thread: two for heads of more than 64 components, one for the others. Threads whose row lies behind the run work on its last row, whose
// elements change no maximum, and store nothing.
template <typename T, int PIECES>
__global__ void __launch_bounds__(EW_THREADS, 2)
write_runs_kernel(const T* __restrict__ qkv, const T* __restrict__ bias, long long qkv_stride, const int* __restrict__ cu_q, const int* __restrict__ tok_seq,
                  const int* __restrict__ tok_pos, const int* __restrict__ slots, const float* __restrict__ inv_freq, int rot_dim, int n_heads,
                  T* __restrict__ q_out, E4m3Site site, int write_cache, int n_seqs, int constants, int* err) {
    grid_launch_dependents();
    if (!constants) grid_dependency_wait();
    constexpr int WORDS = 8 * sizeof(T) / 16;   // of 16 bytes, of eight elements
    __shared__ float amax_s[2][EW_THREADS / 32];
    const int D = site.head_dim, KVH = site.kv_heads, half = rot_dim / 2;
    const unsigned groups = D / 16, rows_each = EW_THREADS / groups;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = n_heads + 2 * KVH;
    const int h_each = (heads + gridDim.y - 1) / gridDim.y, h_begin = blockIdx.y * h_each, h_end = min(h_begin + h_each, heads);
    NewRows run;
    if (h_begin >= h_end || !run_of(blockIdx.x, 0, n_seqs, cu_q, tok_seq, tok_pos, run)) {
        grid_dependency_wait();
        return;
    }
    const int at = run.first_pos % QF_PAGE, rows = run.rows, slot = write_cache ? slots[run.seq] : -1;
    const int page = slot >= 0 ? e4m3_page(site, slot, run.first_pos) : -1;
    if (slot >= 0 && page < 0 && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(err, QF_ERR_NO_PAGE);
    // this thread's pieces: rows, and of each the same sixteen components, eight here and eight there
    const int g = threadIdx.x % groups;
    const bool turns = 8 * g < half;
    const int a_at = turns ? 8 * g : 16 * g;   // (behind the rotated part: rot_dim + 16 (g - half / 8), and the eight behind that)
    const int b_off = turns ? half : 8;
    // float32 queries: two neighbours' eight elements, four and four by each, are 32 bytes side by side of a store (rows of an even number of threads,
    // whose rotated ones come in twos). One prompt of some thousand tokens, 16 + 2 + 2 heads of 128, 12.4 / 11.4 microseconds, eight of up to 1,000,
    // 14 + 2 + 2 of 64, 10.7 / 9.7
    const bool paired = sizeof(T) == 4 && groups % 2 == 0 && half % 16 == 0;
    bool mine[PIECES];
    int code_at[PIECES];
    const T* src[PIECES];
    T* dst[PIECES];
    float2 turn[PIECES][8];
    uint4 raw[PIECES][2][WORDS];
    auto load = [&]() {   // the next head
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                raw[k][0][i] = reinterpret_cast<const uint4*>(src[k])[i];
                raw[k][1][i] = reinterpret_cast<const uint4*>(src[k] + b_off)[i];
            }
            src[k] += D;
        }
    };
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
        const int place = threadIdx.x / groups + k * rows_each, row = min(place, rows - 1);
        mine[k] = place < rows && threadIdx.x < groups * rows_each;
        code_at[k] = (at + row) * D + a_at;
        src[k] = qkv + (long long)(run.t + row) * qkv_stride + h_begin * D + a_at;
        dst[k] = q_out + ((long long)(run.t + row) * n_heads + h_begin) * D + a_at;
    }
    if (!constants) load();
    if (turns) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const Turns f(inv_freq[a_at + e]);
#pragma unroll
            for (int k = 0; k < PIECES; ++k) turn[k][e] = f.at((float)(run.first_pos + code_at[k] / D - at));
        }
    }
    if (constants) {
        grid_dependency_wait();   // (the rows may be the output of the kernel ahead)
        load();
    }
    int parity = 0;
    for (int h = h_begin; h < h_end; ++h) {
        const bool is_q = h < n_heads, is_v = h >= n_heads + KVH;
        float x[PIECES][2][8];
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const T* v = reinterpret_cast<const T*>(raw[k][i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[k][i][e] = Num<T>::to_f(v[e]);
            }
        if (h + 1 < h_end) load();
        if (bias) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float b[8];
                load_values<T, 8>(bias + h * D + a_at + i * b_off, nullptr, b);
#pragma unroll
                for (int k = 0; k < PIECES; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[k][i][e] += b[e];
            }
        }
        if (!is_v && turns) {
#pragma unroll
            for (int k = 0; k < PIECES; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float u = x[k][0][e], w = x[k][1][e];
                    x[k][0][e] = u * turn[k][e].x - w * turn[k][e].y;
                    x[k][1][e] = w * turn[k][e].x + u * turn[k][e].y;
                }
        }
        if (is_q) {
#pragma unroll
            for (int k = 0; k < PIECES; ++k) {
                bool stored = false;
                if constexpr (sizeof(T) == 4) {
                    if (paired) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float* v = x[k][i];
                            float other[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) other[e] = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[e] : v[4 + e], 1);
                            if (mine[k] && turns) {
                                T* to = dst[k] + i * b_off;
                                const float4 theirs = make_float4(other[0], other[1], other[2], other[3]);
                                *reinterpret_cast<float4*>(lane & 1 ? to - 4 : to) = lane & 1 ? theirs : make_float4(v[0], v[1], v[2], v[3]);
                                *reinterpret_cast<float4*>(lane & 1 ? to + 4 : to + 8) = lane & 1 ? make_float4(v[4], v[5], v[6], v[7]) : theirs;
                            }
                        }
                        stored = turns;
                    }
                }
                if (mine[k] && !stored) {
                    store_values<T, 8>(dst[k], x[k][0]);
                    store_values<T, 8>(dst[k] + b_off, x[k][1]);
                }
                dst[k] += D;
            }
            continue;
        }
        if (page < 0) continue;
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fmaxf(finite_size(x[k][0][e]), finite_size(x[k][1][e])));
        const int place = h - n_heads;   // plane * kv heads + head
        float* scale = site.scales + (long long)page * site.page_scales + place;
        const int before = at > 0 ? exponent_of(*scale) : E4M3_LOW;
        amax = warp_max(amax);
        if (lane == 0) amax_s[parity][warp] = amax;
        __syncthreads();   // (every thread has read the old scale, too)
#pragma unroll
        for (int w = 0; w < EW_THREADS / 32; ++w) amax = fmaxf(amax, amax_s[parity][w]);
        parity ^= 1;
        const int exp = max(e4m3_exponent(amax), before);
        unsigned char* codes = site.codes + (long long)page * site.page_bytes + place * QF_PAGE * D;
        if (at > 0 && exp > before) rescale_codes(reinterpret_cast<uint4*>(codes), at * D / 16, pow2(max(before - exp, -126)), threadIdx.x, EW_THREADS);
        const float by = pow2(-exp);
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
            if (mine[k]) {
                store_codes<8>(codes + code_at[k], x[k][0], by);
                store_codes<8>(codes + code_at[k] + b_off, x[k][1], by);
            }
        if (threadIdx.x == 0) *scale = pow2(exp);
    }
}

// Heads of a block of write_runs, which share its sines and cosines (how many hardly matters to a long prompt: angles are not what it waits for) and make the grid's last
// wave fuller or emptier, which is what the float32 figures show: other numbers of heads and tokens have it elsewhere. Microseconds with 3, 4, 5, 6 and 9 of them: twelve float32 prompts of up to 900 tokens,
// 16 + 2 + 2 heads of 128, 20.0, 21.7, 17.5, 17.5 and 22.0; one of 8,192 in bfloat16, 28 + 4 + 4 heads of 128, 39.3, 36.9, 36.8, 37.4 and 37.3.
#define EW_HEADS 6
// Tokens of the longest span from which write_runs is the faster one. Microseconds, write_any / write_runs, bfloat16, spans of 8, 16 and 32 tokens: 14 + 2 + 2
// heads of 64, 1 sequence 4.0 / 6.6, 5.2 / 6.5, 7.4 / 6.7, 64 sequences 5.9 / 8.4, 8.0 / 8.7, 13.4 / 9.3; 28 + 4 + 4 of 128, 1 sequence 5.8 / 7.2, 8.4 / 7.2,
// 13.7 / 8.3, 64 sequences 10.1 / 13.2, 16.6 / 14.5, 34 / 22.
#define EW_LONG 16

template <typename T>
static int write_launch(const void* qkv, const void* bias, long long qkv_stride, const int* cu_q, const int* tok_seq, const int* tok_pos, const int* slots,
                        const float* inv_freq, int rot_dim, int n_heads, void* q_out, const E4m3Site& site, int write_cache, int n_tokens, int n_seqs, int max_q_len,
                        int constants, int* err, cudaStream_t stream) {
    const int heads = n_heads + 2 * site.kv_heads, single = max_q_len == 1;
    // runs: an entry of n tokens has n / 64 + 2 at the most
    const long long most_runs = n_tokens / QF_PAGE + 2ll * n_seqs;
    const int runs = single || most_runs > n_tokens ? n_tokens : (int)most_runs;
    const bool wide = rot_dim % 16 == 0 && qkv_stride % 8 == 0 && ((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)bias) % 16 == 0;
    if (wide && max_q_len >= EW_LONG) {
        return (int)launch_pdl(site.head_dim > 64 ? write_runs_kernel<T, 2> : write_runs_kernel<T, 1>, dim3(runs, (heads + EW_HEADS - 1) / EW_HEADS), dim3(EW_THREADS), 0,
                               stream, (const T*)qkv, (const T*)bias, qkv_stride, cu_q, tok_seq, tok_pos, slots, inv_freq, rot_dim, n_heads, (T*)q_out, site, write_cache,
                               n_seqs, constants, err);
    }
    const int most_rows = max_q_len < QF_PAGE ? max_q_len : QF_PAGE;
    const size_t smem = (size_t)most_rows * (rot_dim / 2) * sizeof(float2);
    const dim3 grid(runs, (heads + EW_WARPS - 1) / EW_WARPS);
    return (int)(wide ? launch_pdl(write_any_kernel<T, 8>, grid, dim3(EW_WARPS * 32), smem, stream, (const T*)qkv, (const T*)bias, qkv_stride, cu_q, tok_seq, tok_pos,
                                   slots, inv_freq, rot_dim, n_heads, (T*)q_out, site, write_cache, n_seqs, single, most_rows, constants, err)
                      : launch_pdl(write_any_kernel<T, 1>, grid, dim3(EW_WARPS * 32), smem, stream, (const T*)qkv, (const T*)bias, qkv_stride, cu_q, tok_seq, tok_pos,
                                   slots, inv_freq, rot_dim, n_heads, (T*)q_out, site, write_cache, n_seqs, single, most_rows, constants, err));
}

static bool site_fits(const E4m3Site& s) {
    return s.head_dim > 0 && s.head_dim % 16 == 0 && s.kv_heads > 0 && s.columns > 0 && s.n_slots > 0 && s.page_bytes % 16 == 0 &&
           s.page_bytes >= 2ll * s.kv_heads * QF_PAGE * s.head_dim && s.page_scales >= 2ll * s.kv_heads && (uintptr_t)s.codes % 16 == 0;
}

// qkv [n_tokens][qkv_stride]: q heads, then k heads, then v heads; bias as a row, or null; inv_freq null: no rotation. Every entry's tokens
// stand at consecutive positions; max_q_len: the most tokens of an entry that has a slot. q_out [n_tokens][n_heads * head_dim].
QF_EXPORT int qf_rope_cache_write_e4m3(int is_bf16, const void* qkv, const void* bias, long long qkv_stride, const int* cu_q, const int* tok_seq,
                                       const int* tok_pos, const int* slots, const float* inv_freq, int rot_dim, int n_heads, void* q_out, void* codes,
                                       float* scales, const int* table, long long page_bytes, long long page_scales, int table_stride, int columns, int n_slots,
                                       int kv_heads, int head_dim, int write_cache, int n_tokens, int n_seqs, int max_q_len, int constants, int* err, cudaStream_t stream) {
    const E4m3Site site{(unsigned char*)codes, scales, table, page_bytes, page_scales, table_stride, columns, n_slots, kv_heads, head_dim};
    if (!inv_freq) rot_dim = 0;
    if (!site_fits(site) || head_dim > 128 || rot_dim < 0 || rot_dim > head_dim || (rot_dim & 1) || n_heads <= 0 || max_q_len <= 0) return (int)cudaErrorInvalidValue;
    if (n_tokens <= 0 || n_seqs <= 0) return 0;
    return is_bf16 ? write_launch<bf16>(qkv, bias, qkv_stride, cu_q, tok_seq, tok_pos, slots, inv_freq, rot_dim, n_heads, q_out, site, write_cache, n_tokens, n_seqs, max_q_len, constants, err, stream)
                   : write_launch<float>(qkv, bias, qkv_stride, cu_q, tok_seq, tok_pos, slots, inv_freq, rot_dim, n_heads, q_out, site, write_cache, n_tokens, n_seqs, max_q_len, constants, err, stream);
}

// ---- Read back: the rows that a batch's sequences hold (from the first that a window of `window` positions leaves the first new token, 0:
// all; up to the last new token) as values, into a storage of the same shape in another type, at the same page numbers: a page table serves
// both. A block takes one plane and head of a page, and of every `columns_each`-th behind it: with a window few of a sequence's pages are wanted, and blocks
// for all of them would be thousands that find nothing to do (71 sequences of up to 1,676 tokens, 10 planes and heads, a window of 37: 20.4 / 5.1 microseconds). A thread
// reads what becomes 16 bytes, so that a warp's stores are whole lines. Four documents of 68,000 tokens together, 4 heads of 128: 37 microseconds, 5.7 TB/s of
// the 6.5 that a copy has; two of up to 13,777 in float32, 2 heads of 128, 10.1 (14.3 with 16 codes a thread).
template <typename T>
__global__ void __launch_bounds__(256)
read_e4m3_kernel(T* __restrict__ out, long long out_page, const int* __restrict__ cu_q, const int* __restrict__ tok_pos, const int* __restrict__ slots,
                 E4m3Site site, int columns_each, int window, int* err) {
    grid_chain_entry();
    constexpr int N = 16 / sizeof(T), U = 4;   // codes of a piece; pieces of a thread on their way at once
    const int seq = blockIdx.x / columns_each, D = site.head_dim;
    const int slot = slots[seq], begin = cu_q[seq], end = cu_q[seq + 1];
    if (slot < 0 || end <= begin) return;
    const int length = tok_pos[end - 1] + 1, lo = window > 0 ? max(0, tok_pos[begin] - window + 1) : 0;
    for (int column = lo / QF_PAGE + blockIdx.x % columns_each; column * QF_PAGE < length; column += columns_each) {
        const int row0 = max(lo - column * QF_PAGE, 0), row1 = min(length - column * QF_PAGE, QF_PAGE);
        const int page = e4m3_page(site, slot, column * QF_PAGE);
        if (page < 0) {
            if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(err, QF_ERR_NO_PAGE);
            if (column >= site.columns) return;
            continue;
        }
        const float scale = site.scales[(long long)page * site.page_scales + blockIdx.y];
        const unsigned char* codes = site.codes + (long long)page * site.page_bytes + (long long)blockIdx.y * QF_PAGE * D;
        T* to = out + (long long)page * out_page + (long long)blockIdx.y * QF_PAGE * D;
        const int last = row1 * D / N;
        for (int i0 = row0 * D / N + threadIdx.x; i0 < last; i0 += U * 256) {
            uint32_t words[U][N / 4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * 256;
                if (i < last) {
                    if constexpr (N == 8) {
                        const uint2 w = reinterpret_cast<const uint2*>(codes)[i];
                        words[u][0] = w.x, words[u][1] = w.y;
                    } else {
                        words[u][0] = reinterpret_cast<const uint32_t*>(codes)[i];
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * 256;
                if (i < last) {
                    float v[N];
#pragma unroll
                    for (int e = 0; e < N / 4; ++e) {
                        const float2 a = floats_of(half2_of_low(words[u][e])), b = floats_of(half2_of_high(words[u][e]));
                        v[4 * e] = a.x * scale, v[4 * e + 1] = a.y * scale, v[4 * e + 2] = b.x * scale, v[4 * e + 3] = b.y * scale;
                    }
                    if constexpr (N == 8)
                        reinterpret_cast<uint4*>(to)[i] = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
                    else
                        reinterpret_cast<float4*>(to)[i] = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
        }
    }
}

// out [pages][2][kv_heads][QF_PAGE][head_dim], out_page elements from a page to the next; pages_each: the most pages of a sequence.
QF_EXPORT int qf_cache_read_e4m3(int is_bf16, void* out, long long out_page, const int* cu_q, const int* tok_pos, const int* slots, void* codes, float* scales,
                                 const int* table, long long page_bytes, long long page_scales, int table_stride, int columns, int n_slots, int kv_heads,
                                 int head_dim, int n_seqs, int pages_each, int window, int* err, cudaStream_t stream) {
    const E4m3Site site{(unsigned char*)codes, scales, table, page_bytes, page_scales, table_stride, columns, n_slots, kv_heads, head_dim};
    if (!site_fits(site) || pages_each <= 0 || 2 * kv_heads > 65535 || (long long)n_seqs * pages_each > 0x7fffffffll || (uintptr_t)out % 16 || out_page % 8 ||
        out_page < 2ll * kv_heads * QF_PAGE * head_dim)
        return (int)cudaErrorInvalidValue;
    if (n_seqs <= 0) return 0;
    int columns_each = window > 0 && window / QF_PAGE + 3 < pages_each ? window / QF_PAGE + 3 : pages_each;   // (a window's pages and a short span's)
    // And where there would be rounds of blocks that write less than 16 KB each, fewer of them with more: 44 sequences of up to 3,709 tokens, 2 heads of 16,
    // 11.1 / 8.5 microseconds (float32 14.4 / 11.8), 64 of up to 4,000, 2 of 64, 23.8 / 20.6.
    const long long rounds = (long long)n_seqs * columns_each * 2 * kv_heads / (8 * qf_sm_count());
    const int most = 16384 / (QF_PAGE * head_dim * (is_bf16 ? 2 : 4));
    if (rounds > 1 && most > 1) columns_each = (columns_each + std::min((int)rounds, most) - 1) / std::min((int)rounds, most);
    const dim3 grid(n_seqs * columns_each, 2 * kv_heads), block(256);
    return (int)(is_bf16 ? launch_pdl(read_e4m3_kernel<bf16>, grid, block, 0, stream, (bf16*)out, out_page, cu_q, tok_pos, slots, site, columns_each, window, err)
                         : launch_pdl(read_e4m3_kernel<float>, grid, block, 0, stream, (float*)out, out_page, cu_q, tok_pos, slots, site, columns_each, window, err));
}
