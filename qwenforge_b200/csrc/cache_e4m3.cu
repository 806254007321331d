// Writing a sequence cache of e4m3 codes, and reading it back (the format: e4m3.cuh).
//
// ---- Write, behind the q/k/v projection of a step's tokens: x = row + bias; queries and keys rotated (split halves over the first R
// components, as rope_cache.cu; the product position * frequency with its rounding error, so that an angle of tens of thousands is
// as exact as a small one); queries written out. For every page that gets new rows, of each plane and kv head:
//   amax = max |x| over the new rows' finite elements,  e = the least exponent with amax <= 448 * 2^e
//   the page had rows before (the first new one does not begin it): e = max(e, e_old), and where that is more than e_old, those
//   rows' codes become round(code * 2^(e_old - e))
//   new codes = round(x * 2^-e), to nearest even, from float32: one rounding
// A page that is begun takes its exponent from its new rows alone, whatever an earlier holder left there. Rows behind the new ones stay.
//
// A run is a page's new rows. Two kernels, the same in what they write:
//   write_runs     spans of EW_LONG tokens or more: a block takes the runs that begin among 64 of the step's tokens and some of the heads, all its
//                  threads one head at a time. A thread has the same one or two pieces (a row, eight pairs of the rotation) of every head, so
//                  their sines and cosines are worked out once and stay in registers, a key's or value's elements stay there between amax and
//                  codes, and the next head's are loaded meanwhile.
//   write_any      single tokens, short spans, and rows or rotations that 16-byte accesses do not fit: a warp a head at a time over all rows of
//                  a run; amax and codes are one warp's business, without a barrier. Sines and cosines come from shared memory, worked
//                  out once per run. A key or value head is read twice, the second time from L1 or L2.
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

template <typename T, int VEC>
__global__ void __launch_bounds__(EW_WARPS * 32)
write_any_kernel(const T* __restrict__ qkv, const T* __restrict__ bias, long long qkv_stride, const int* __restrict__ cu_q, const int* __restrict__ tok_seq,
                  const int* __restrict__ tok_pos, const int* __restrict__ slots, const float* __restrict__ inv_freq, int rot_dim, int n_heads,
                  T* __restrict__ q_out, E4m3Site site, int write_cache, int n_tokens, int share, int most_rows, int* err) {
    grid_chain_entry();
    extern __shared__ float2 turn[];   // [rows of a run][rot_dim / 2] cosine, sine
    const int D = site.head_dim, KVH = site.kv_heads, half = rot_dim / 2, pass = D - rot_dim;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int heads = n_heads + 2 * KVH;
    const int h_each = (heads + gridDim.y - 1) / gridDim.y, h_begin = blockIdx.y * h_each, h_end = min(h_begin + h_each, heads);
    const int t_begin = blockIdx.x * share, t_end = min(t_begin + share, n_tokens);
    for (int t = t_begin; t < t_end; ++t) {
        const int seq = tok_seq[t], first_pos = tok_pos[t];
        if (t != cu_q[seq] && first_pos % QF_PAGE != 0) continue;   // (the run began at an earlier token)
        const int slot = write_cache ? slots[seq] : -1, at = first_pos % QF_PAGE;
        int rows = min(cu_q[seq + 1] - t, QF_PAGE - at);
        if (rows > most_rows) {   // (an entry longer than the call has said: there is no room for its angles)
            if (threadIdx.x == 0) atomicOr(err, QF_ERR_ROW_RANGE);
            rows = most_rows;
        }
        const int page = slot >= 0 ? e4m3_page(site, slot, first_pos) : -1;
        if (slot >= 0 && page < 0 && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(err, QF_ERR_NO_PAGE);
        __syncthreads();
        for (int i = threadIdx.x; i < rows * half; i += blockDim.x) {
            const float p = (float)(first_pos + i / half), f = inv_freq[i % half];
            const float angle = p * f, rest = fmaf(p, f, -angle);
            float s, c;
            sincosf(angle, &s, &c);
            turn[i] = make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
        }
        __syncthreads();
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
}

#define EW_THREADS 256
#define EW_PIECES 2   // of a thread: 64 rows of up to eight pieces

template <typename T>
__global__ void __launch_bounds__(EW_THREADS, 2)
write_runs_kernel(const T* __restrict__ qkv, const T* __restrict__ bias, long long qkv_stride, const int* __restrict__ cu_q, const int* __restrict__ tok_seq,
                  const int* __restrict__ tok_pos, const int* __restrict__ slots, const float* __restrict__ inv_freq, int rot_dim, int n_heads,
                  T* __restrict__ q_out, E4m3Site site, int write_cache, int n_tokens, int* err) {
    grid_chain_entry();
    constexpr int RAW = 16 * sizeof(T) / 16;   // 16-byte words of a piece: eight elements here, eight there
    __shared__ float amax_s[2][EW_THREADS / 32];
    const int D = site.head_dim, KVH = site.kv_heads, half = rot_dim / 2, groups = D / 16;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = n_heads + 2 * KVH;
    const int h_each = (heads + gridDim.y - 1) / gridDim.y, h_begin = blockIdx.y * h_each, h_end = min(h_begin + h_each, heads);
    const int t0 = blockIdx.x * QF_PAGE;
    int parity = 0;
    for (int part = 0; part < QF_PAGE; part += 32) {
        // tokens at which a run begins
        bool begins = false;
        if (t0 + part + lane < n_tokens) begins = tok_pos[t0 + part + lane] % QF_PAGE == 0 || t0 + part + lane == cu_q[tok_seq[t0 + part + lane]];
        for (uint32_t left = __ballot_sync(0xffffffffu, begins); left; left &= left - 1) {
            const int t = t0 + part + __ffs(left) - 1, seq = tok_seq[t], first_pos = tok_pos[t], at = first_pos % QF_PAGE;
            const int slot = write_cache ? slots[seq] : -1, rows = min(cu_q[seq + 1] - t, QF_PAGE - at);
            const int page = slot >= 0 ? e4m3_page(site, slot, first_pos) : -1;
            if (slot >= 0 && page < 0 && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(err, QF_ERR_NO_PAGE);
            // this thread's pieces: a row, the places of its two eights in a head, and their turn
            int row[EW_PIECES], a_at[EW_PIECES], b_at[EW_PIECES];
            bool turns[EW_PIECES];
            float cosine[EW_PIECES][8], sine[EW_PIECES][8];
#pragma unroll
            for (int k = 0; k < EW_PIECES; ++k) {
                const unsigned i = threadIdx.x + k * EW_THREADS, g = i % (unsigned)groups;
                row[k] = i / (unsigned)groups;
                turns[k] = 8 * (int)g < half;
                a_at[k] = turns[k] ? 8 * g : 16 * g;   // (rot_dim + 16 (g - half / 8) behind the rotated part)
                b_at[k] = turns[k] ? 8 * g + half : 16 * g + 8;
                if (row[k] < rows && turns[k]) {
                    const float p = (float)(first_pos + row[k]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float f = inv_freq[8 * g + e], angle = p * f, rest = fmaf(p, f, -angle);
                        float s, c;
                        sincosf(angle, &s, &c);
                        cosine[k][e] = fmaf(-s, rest, c);
                        sine[k][e] = fmaf(c, rest, s);
                    }
                }
            }
            uint4 raw[EW_PIECES][RAW];
            auto load = [&](int h) {
#pragma unroll
                for (int k = 0; k < EW_PIECES; ++k)
                    if (row[k] < rows) {
                        const T* src = qkv + (long long)(t + row[k]) * qkv_stride + (long long)h * D;
#pragma unroll
                        for (int i = 0; i < RAW / 2; ++i) {
                            raw[k][i] = reinterpret_cast<const uint4*>(src + a_at[k])[i];
                            raw[k][RAW / 2 + i] = reinterpret_cast<const uint4*>(src + b_at[k])[i];
                        }
                    }
            };
            if (h_begin < h_end) load(h_begin);
            for (int h = h_begin; h < h_end; ++h) {
                const bool is_q = h < n_heads, is_v = h >= n_heads + KVH;
                const int kvh = is_v ? h - n_heads - KVH : h - n_heads;
                float x[EW_PIECES][16], amax = 0.f;
#pragma unroll
                for (int k = 0; k < EW_PIECES; ++k) {
                    if (row[k] >= rows) continue;
                    const T* v = reinterpret_cast<const T*>(raw[k]);
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[k][e] = Num<T>::to_f(v[e]);
                    if (bias) {
                        float b[8];
#pragma unroll
                        for (int part16 = 0; part16 < 2; ++part16) {
                            load_values<T, 8>(bias + (long long)h * D + (part16 ? b_at[k] : a_at[k]), nullptr, b);
#pragma unroll
                            for (int e = 0; e < 8; ++e) x[k][8 * part16 + e] += b[e];
                        }
                    }
                    if (!is_v && turns[k]) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float u = x[k][e], w = x[k][8 + e];
                            x[k][e] = u * cosine[k][e] - w * sine[k][e];
                            x[k][8 + e] = w * cosine[k][e] + u * sine[k][e];
                        }
                    }
                }
                if (h + 1 < h_end) load(h + 1);
                if (is_q) {
#pragma unroll
                    for (int k = 0; k < EW_PIECES; ++k)
                        if (row[k] < rows) {
                            T* dst = q_out + ((long long)(t + row[k]) * n_heads + h) * D;
                            store_values<T, 8>(dst + a_at[k], *reinterpret_cast<const float(*)[8]>(&x[k][0]));
                            store_values<T, 8>(dst + b_at[k], *reinterpret_cast<const float(*)[8]>(&x[k][8]));
                        }
                    continue;
                }
                if (page < 0) continue;
#pragma unroll
                for (int k = 0; k < EW_PIECES; ++k)
                    if (row[k] < rows) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) amax = fmaxf(amax, finite_size(x[k][e]));
                    }
                float* scale = site.scales + (long long)page * site.page_scales + (is_v ? KVH : 0) + kvh;
                const int before = at > 0 ? exponent_of(*scale) : E4M3_LOW;
                amax = warp_max(amax);
                if (lane == 0) amax_s[parity][warp] = amax;
                __syncthreads();   // (every thread has read the old scale, too)
#pragma unroll
                for (int w = 0; w < EW_THREADS / 32; ++w) amax = fmaxf(amax, amax_s[parity][w]);
                parity ^= 1;
                const int exp = max(e4m3_exponent(amax), before);
                unsigned char* codes = site.codes + (long long)page * site.page_bytes + (long long)((is_v ? KVH : 0) + kvh) * QF_PAGE * D;
                if (at > 0 && exp > before) rescale_codes(reinterpret_cast<uint4*>(codes), at * D / 16, pow2(max(before - exp, -126)), threadIdx.x, EW_THREADS);
                const float by = pow2(-exp);
#pragma unroll
                for (int k = 0; k < EW_PIECES; ++k)
                    if (row[k] < rows) {
                        unsigned char* dst = codes + (at + row[k]) * D;
                        store_codes<8>(dst + a_at[k], *reinterpret_cast<const float(*)[8]>(&x[k][0]), by);
                        store_codes<8>(dst + b_at[k], *reinterpret_cast<const float(*)[8]>(&x[k][8]), by);
                    }
                if (threadIdx.x == 0) *scale = pow2(exp);
            }
        }
    }
}

#ifndef EW_HEADS
#define EW_HEADS 6   // heads of a block of write_runs
#endif
#ifndef EW_LONG
#define EW_LONG 16   // tokens of the longest span from which write_runs is the faster one (@LONG@)
#endif

template <typename T>
static int write_launch(const void* qkv, const void* bias, long long qkv_stride, const int* cu_q, const int* tok_seq, const int* tok_pos, const int* slots,
                        const float* inv_freq, int rot_dim, int n_heads, void* q_out, const E4m3Site& site, int write_cache, int n_tokens, int max_q_len, int* err,
                        cudaStream_t stream) {
    const int heads = n_heads + 2 * site.kv_heads, slices = (heads + EW_WARPS - 1) / EW_WARPS;
    const int share = max_q_len > 1 ? 16 : 1;
    const int most_rows = max_q_len < QF_PAGE ? max_q_len : QF_PAGE;
    const size_t smem = (size_t)most_rows * (rot_dim / 2) * sizeof(float2);
    const bool wide = rot_dim % 16 == 0 && qkv_stride % 8 == 0 && ((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)bias) % 16 == 0;
    if (wide && max_q_len >= EW_LONG) {
        const int pieces = (heads + EW_HEADS - 1) / EW_HEADS;
        return (int)launch_pdl(write_runs_kernel<T>, dim3((n_tokens + QF_PAGE - 1) / QF_PAGE, pieces), dim3(EW_THREADS), 0, stream, (const T*)qkv, (const T*)bias, qkv_stride,
                               cu_q, tok_seq, tok_pos, slots, inv_freq, rot_dim, n_heads, (T*)q_out, site, write_cache, n_tokens, err);
    }
    const dim3 grid((n_tokens + share - 1) / share, slices);
    return (int)(wide ? launch_pdl(write_any_kernel<T, 8>, grid, dim3(EW_WARPS * 32), smem, stream, (const T*)qkv, (const T*)bias, qkv_stride, cu_q, tok_seq,
                                   tok_pos, slots, inv_freq, rot_dim, n_heads, (T*)q_out, site, write_cache, n_tokens, share, most_rows, err)
                      : launch_pdl(write_any_kernel<T, 1>, grid, dim3(EW_WARPS * 32), smem, stream, (const T*)qkv, (const T*)bias, qkv_stride, cu_q, tok_seq,
                                   tok_pos, slots, inv_freq, rot_dim, n_heads, (T*)q_out, site, write_cache, n_tokens, share, most_rows, err));
}

static bool site_fits(const E4m3Site& s) {
    return s.head_dim > 0 && s.head_dim % 16 == 0 && s.kv_heads > 0 && s.columns > 0 && s.n_slots > 0 && s.page_bytes % 16 == 0 &&
           s.page_bytes >= 2ll * s.kv_heads * QF_PAGE * s.head_dim && s.page_scales >= 2ll * s.kv_heads && (uintptr_t)s.codes % 16 == 0;
}

// qkv [n_tokens][qkv_stride]: q heads, then k heads, then v heads; bias as a row, or null; inv_freq null: no rotation. Every entry's tokens
// stand at consecutive positions; max_q_len: the most tokens of an entry. q_out [n_tokens][n_heads * head_dim].
QF_EXPORT int qf_rope_cache_write_e4m3(int is_bf16, const void* qkv, const void* bias, long long qkv_stride, const int* cu_q, const int* tok_seq,
                                       const int* tok_pos, const int* slots, const float* inv_freq, int rot_dim, int n_heads, void* q_out, void* codes,
                                       float* scales, const int* table, long long page_bytes, long long page_scales, int table_stride, int columns, int n_slots,
                                       int kv_heads, int head_dim, int write_cache, int n_tokens, int max_q_len, int* err, cudaStream_t stream) {
    const E4m3Site site{(unsigned char*)codes, scales, table, page_bytes, page_scales, table_stride, columns, n_slots, kv_heads, head_dim};
    if (!inv_freq) rot_dim = 0;
    if (!site_fits(site) || head_dim > 128 || rot_dim < 0 || rot_dim > head_dim || (rot_dim & 1) || n_heads <= 0 || max_q_len <= 0) return (int)cudaErrorInvalidValue;
    if (n_tokens <= 0) return 0;
    return is_bf16 ? write_launch<bf16>(qkv, bias, qkv_stride, cu_q, tok_seq, tok_pos, slots, inv_freq, rot_dim, n_heads, q_out, site, write_cache, n_tokens, max_q_len, err, stream)
                   : write_launch<float>(qkv, bias, qkv_stride, cu_q, tok_seq, tok_pos, slots, inv_freq, rot_dim, n_heads, q_out, site, write_cache, n_tokens, max_q_len, err, stream);
}

// ---- Read back: the rows that a batch's sequences hold (from the first that a window of `window` positions leaves the first new token, 0:
// all; up to the last new token) as values, into a storage of the same shape in another type, at the same page numbers: a page table serves
// both. A block takes one plane and head of a page.
template <typename T>
__global__ void __launch_bounds__(256)
read_e4m3_kernel(T* __restrict__ out, long long out_page, const int* __restrict__ cu_q, const int* __restrict__ tok_pos, const int* __restrict__ slots,
                 E4m3Site site, int pages_each, int window, int* err) {
    grid_chain_entry();
    const int seq = blockIdx.x / pages_each, column = blockIdx.x % pages_each, D = site.head_dim;
    const int slot = slots[seq], begin = cu_q[seq], end = cu_q[seq + 1];
    if (slot < 0 || end <= begin) return;
    const int length = tok_pos[end - 1] + 1, lo = window > 0 ? max(0, tok_pos[begin] - window + 1) : 0;
    const int row0 = max(lo - column * QF_PAGE, 0), row1 = min(length - column * QF_PAGE, QF_PAGE);
    if (row0 >= row1) return;
    const int page = e4m3_page(site, slot, column * QF_PAGE);
    if (page < 0) {
        if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(err, QF_ERR_NO_PAGE);
        return;
    }
    const float scale = site.scales[(long long)page * site.page_scales + blockIdx.y];
    const unsigned char* codes = site.codes + (long long)page * site.page_bytes + (long long)blockIdx.y * QF_PAGE * D;
    T* to = out + (long long)page * out_page + (long long)blockIdx.y * QF_PAGE * D;
    for (int i = row0 * D / 16 + threadIdx.x; i < row1 * D / 16; i += blockDim.x) {
        const uint4 w = reinterpret_cast<const uint4*>(codes)[i];
        const uint32_t* words = reinterpret_cast<const uint32_t*>(&w);
        T v[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 a = floats_of(half2_of_low(words[e])), b = floats_of(half2_of_high(words[e]));
            v[4 * e] = Num<T>::from_f(a.x * scale);
            v[4 * e + 1] = Num<T>::from_f(a.y * scale);
            v[4 * e + 2] = Num<T>::from_f(b.x * scale);
            v[4 * e + 3] = Num<T>::from_f(b.y * scale);
        }
#pragma unroll
        for (int e = 0; e < (int)sizeof(T); ++e) reinterpret_cast<uint4*>(to + 16ll * i)[e] = reinterpret_cast<const uint4*>(v)[e];
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
    const dim3 grid(n_seqs * pages_each, 2 * kv_heads), block(256);
    return (int)(is_bf16 ? launch_pdl(read_e4m3_kernel<bf16>, grid, block, 0, stream, (bf16*)out, out_page, cu_q, tok_pos, slots, site, pages_each, window, err)
                         : launch_pdl(read_e4m3_kernel<float>, grid, block, 0, stream, (float*)out, out_page, cu_q, tok_pos, slots, site, pages_each, window, err));
}
