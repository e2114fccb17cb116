// The 4-bit weights of the int4 kernels: a packed word holds 8 codes of one column, the
// code of row 8kp+j at bits 4j..4j+3, two's complement (-8..7); the weight is code * S of
// its 128-row group.
//
// A code's nibble with its top bit flipped is code + 8 (0..15); put in the low mantissa
// bits of a power of two it reads as that power + code + 8, and one subtraction leaves the
// code exactly, in fp16 and bf16.  Only codes go through the 16-bit types: the scale is
// applied to fp32 sums of a group, so no weight is ever rounded.
#pragma once
#include "common.cuh"
#include "digit_common.cuh"

namespace ternocl {
namespace int4 {

constexpr int kRowsPerWord = 8;
constexpr int kWordsPerGroup = kGS / kRowsPerWord;  // 16 word rows per scale group

// two codes at bits 0..3 of the halves of x -> half2 / bf16x2 of them
template <class DT>
__device__ __forceinline__ uint32_t low_pair(uint32_t x) {
    // fp16: 1024 + code + 8 (10 mantissa bits); bf16: 128 + code + 8 (7 mantissa bits)
    constexpr uint32_t magic = DT::kBF16 ? 0x43084308u : 0x64086408u;
    constexpr uint32_t bias = magic;  // 136 or 1032
    uint32_t r, v;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;\n" : "=r"(r) : "r"(x), "n"(0x000F000Fu), "r"(magic));  // (x & m) ^ magic
    if constexpr (DT::kBF16) asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(v) : "r"(r), "r"(bias));
    else asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(v) : "r"(r), "r"(bias));
    return v;
}

// two codes at bits 4..7 of the halves of x: fp16 reads 1024 + 16 (code + 8), times 1/16
// minus 72; bf16 has too few mantissa bits for that and shifts first
template <class DT>
__device__ __forceinline__ uint32_t high_pair(uint32_t x) {
    if constexpr (DT::kBF16) {
        return low_pair<DT>(x >> 4);
    } else {
        uint32_t r, v;
        asm("lop3.b32 %0, %1, %2, %3, 0x6A;\n" : "=r"(r) : "r"(x), "n"(0x00F000F0u), "r"(0x64806480u));
        asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(v) : "r"(r), "r"(0x2C002C00u), "r"(0xD480D480u));
        return v;
    }
}

// the four pairs of a word: out[p] = (row p, row p + 4)
template <class DT>
__device__ __forceinline__ void word_pairs(uint32_t x, uint32_t (&out)[4]) {
    const uint32_t y = x >> 8;
    out[0] = low_pair<DT>(x);
    out[1] = high_pair<DT>(x);
    out[2] = low_pair<DT>(y);
    out[3] = high_pair<DT>(y);
}

// ---- the integer form: int8 weights and fixed-point activation digits ---------------
//
// The low (high) nibbles of a word's four bytes are rows 0,2,4,6 (1,3,5,7); moved to the top
// of their bytes they read as int8 16 * code, two operations for four weights.  With 2^e
// such that |A| * 2^e < 2^22 (digit_common.cuh), i = round(A * 2^e) is split into three
// balanced base-256 digits, i = d0 + 256 d1 + 65536 d2 with d in [-128, 127]: adding
// 0x808080 makes them the bytes of a positive number, and flipping each top bit makes those
// bytes signed.  A group's dots |sum 16 code d| <= 128 * 128 * 128 = 2^21 are exact, and read
// as floats from the accumulator's start pattern (below 2^22).
__device__ __forceinline__ uint32_t even_rows(uint32_t x) { return (x << 4) & 0xF0F0F0F0u; }
__device__ __forceinline__ uint32_t odd_rows(uint32_t x) { return x & 0xF0F0F0F0u; }

__device__ __forceinline__ void imma(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                     uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 2^-e / 16 (the weights are 16 x code); NaN when the maximum is Inf or NaN
template <class DT>
__device__ __forceinline__ float inverse_scale(uint32_t mx_bits, int e) {
    const bool bad = DT::kBF16 ? mx_bits >= 0x7F80u : mx_bits >= 0x7C00u;
    return bad ? __int_as_float(0x7FC00000) : __int_as_float((127 - e - 4) << 23);
}

// the 8 activations of a word (v: packed pairs, rows in order) -> per digit plane d its even
// and its odd rows' bytes, out[d] = (rows 0,2,4,6 | rows 1,3,5,7)
template <class DT>
__device__ __forceinline__ void word_digits(const uint4 v, int e, uint2 (&out)[3]) {
    const float up = __int_as_float((127 + e) << 23);  // 2^e
    const uint32_t h2[4] = {v.x, v.y, v.z, v.w};
    uint32_t x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint16_t h = (uint16_t)((k & 1) ? h2[k / 2] >> 16 : h2[k / 2] & 0xFFFFu);
        // bits of 1.5 * 2^23 + i -> the bytes of i + 0x808080, top bits flipped
        const uint32_t b = __float_as_uint(fmaf(DT::tof(h), up, digit::kMagic));
        x[k] = (b + (0x00808080u - digit::kMagicBits)) ^ 0x00808080u;
    }
    uint32_t r[2][3];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
        const uint32_t p01 = __byte_perm(x[o], x[o + 2], 0x5140), p23 = __byte_perm(x[o + 4], x[o + 6], 0x5140);
        const uint32_t q01 = __byte_perm(x[o], x[o + 2], 0x7362), q23 = __byte_perm(x[o + 4], x[o + 6], 0x7362);
        r[o][0] = __byte_perm(p01, p23, 0x5410);
        r[o][1] = __byte_perm(p01, p23, 0x7632);
        r[o][2] = __byte_perm(q01, q23, 0x5410);
    }
#pragma unroll
    for (int d = 0; d < 3; ++d) out[d] = make_uint2(r[0][d], r[1][d]);
}

// max |value| of 8 packed activations, as magnitude bits
__device__ __forceinline__ uint32_t absmax_bits(const uint4 v) {
    uint32_t mx = __vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu);
    mx = __vmaxu2(mx, __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
    return max(mx & 0xFFFFu, mx >> 16);
}

}  // namespace int4
}  // namespace ternocl
