// A sequence cache in 8 bits. Storage of one schedule entry: a byte per element, [pages][2 (k, v)][kv_heads][QF_PAGE][head_dim] codes of
// e4m3 (a sign, four bits of exponent, three of mantissa, largest value 448, no infinities), and a float32 power of two per page, plane and
// kv head, [pages][2][kv_heads]: an element stands for code * 2^e. With a power of two for a scale the product is exact in bfloat16 and
// float32, the codes alone are exact in float16 (what the tensor cores multiply), and a page whose scale grows keeps its older codes'
// values but for those that fall below the smallest normal code (2^-6 of the larger unit).
#pragma once
#include "mma.cuh"

struct E4m3Site {
    unsigned char* codes;
    float* scales;
    const int* table;        // [n_slots][table_stride] page ids, -1 where none is held
    long long page_bytes;    // codes from a page to the next, at least 2 * kv_heads * QF_PAGE * head_dim
    long long page_scales;   // scales from a page to the next, at least 2 * kv_heads
    int table_stride, columns, n_slots;
    int kv_heads, head_dim;
};

// The page that holds position `pos` of `slot`; -1 where none does.
__device__ __forceinline__ int e4m3_page(const E4m3Site& s, int slot, int pos) {
    const int column = pos / QF_PAGE;
    if (slot >= s.n_slots || pos < 0 || column >= s.columns) return -1;
    return s.table[(long long)slot * s.table_stride + column];
}

// Exponents of scales: at the low end a page's smallest value 2^-9 * 2^e is still a normal bfloat16, at the high end its largest is finite.
#define E4M3_LOW (-112)
#define E4M3_HIGH 119

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float scale) { return (int)((__float_as_uint(scale) >> 23) & 255u) - 127; }

// The least e with amax <= 448 * 2^e = 1.75 * 2^(e + 8): the exponent of amax, one more where its mantissa is above 1.75 (the addition
// carries into the exponent from there on).
__device__ __forceinline__ int e4m3_exponent(float amax) {
    const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
    return min(max(e, E4M3_LOW), E4M3_HIGH);
}

// Two values to two codes, `lo` in the low byte: to nearest, ties to even; what is too large, infinities among it, to +-448; NaN to NaN.
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_four(float a, float b, float c, float d) { return e4m3_pair(a, b) | (e4m3_pair(c, d) << 16); }

// The two codes in the low / high half of a word as two float16 (exact).
__device__ __forceinline__ uint32_t half2_of_low(uint32_t codes) {
    uint32_t r;
    asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(r) : "r"(codes));
    return r;
}
__device__ __forceinline__ uint32_t half2_of_high(uint32_t codes) {
    uint32_t r;
    asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi;\n}\n" : "=r"(r) : "r"(codes));
    return r;
}
__device__ __forceinline__ float2 floats_of(uint32_t half2) {
    float2 f;
    asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %2;\n cvt.f32.f16 %0, lo;\n cvt.f32.f16 %1, hi;\n}\n" : "=f"(f.x), "=f"(f.y) : "r"(half2));
    return f;
}
