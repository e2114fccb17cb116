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

}  // namespace int4
}  // namespace ternocl
