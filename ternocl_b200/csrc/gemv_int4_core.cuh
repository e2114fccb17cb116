// The core of the int4 decode GEMVs (gemv_int4.cu, moe_decode_int4.cu): one warp multiplies up
// to 8 activation rows with 32 columns of consecutive 128-row groups.
//
// Lane (g, t) loads, per group, 16 bytes of words (columns 4g .. 4g+3) of the word rows 4c + t
// (c = 0..3) and the four columns' scales, one group ahead of the one it multiplies, straight
// into registers.  A word decodes into four half2 of rows (p, p+4) (int4_common.cuh), two A
// registers for each of two mma.sync m16n8k16: the 16 columns of a block are the MMA's rows,
// the activation rows its columns.  Lane (g, t) reads its B registers, row g's activations of
// the same K rows, from L1.  Products of codes and DT activations are exact in the MMA's fp32
// sums; a group's sum is scaled by S in fp32.
//
// For one row there is an integer form with a third of the instructions: a word is two
// A registers of mma.sync m16n8k32 s8 x s8 (its even and odd rows as 16 * code, three
// operations for eight weights), against digit planes of the activations.  With 2^e such that
// |A| * 2^e < 2^30 in a group, i = A * 2^e is split into four balanced base-256 digits,
// i = d0 + 256 d1 + 65536 d2 + 2^24 d3 with d in [-128, 127]: adding 0x80808080 makes them the bytes
// of an unsigned number, and flipping each top bit makes those bytes signed.  The planes are
// the first four of the MMA's eight n-columns; a group's dots (|sum 16 code d| <=
// 128 * 128 * 128 = 2^21) are exact, read as floats from the accumulator's start pattern and
// scaled by 2^-e and S in fp32.  Every i is exact: a group whose exponents are too far apart for
// that (bf16: more than 2^22, fp16: 2^19) or that holds an Inf or a NaN is multiplied in 16 bits
// after the others, its words read again.  That is 1 group in 10,000 of normal values, 1 in
// 1,000 of products of them in bf16.  (At M = 1 in the integer form, at M = 2 in 16 bits:
// 4096x28672 14.2 and 18.1 us, 5120x248320 129 and 147.)
#pragma once
#include "common.cuh"
#include "digit_common.cuh"
#include "int4_common.cuh"

namespace ternocl {
namespace int4 {

// Weights of consecutive groups of one matrix, as a lane reads them.
struct WordStream {
    const uint32_t *wp;  // next group: word row t, column 4g
    const uint16_t *sp;
    size_t row4, n;  // four word rows, a scale row (elements)
    uint4 w[4];  // the group read last
    uint2 s;

    __device__ __forceinline__ void width(int N) {
        row4 = (size_t)4 * N;
        n = N;
    }
    // to group `grp` of the matrix (B [K/8, N], S [K/128, N]); a lane whose columns lie behind N
    // reads column 0 (and its results are not stored)
    __device__ __forceinline__ void seek(const uint32_t *B, const uint16_t *S, int N, int grp, int n0, int lane) {
        const int col = n0 + 4 * (lane >> 2) < N ? n0 + 4 * (lane >> 2) : 0;
        wp = B + ((size_t)grp * kWordsPerGroup + (lane & 3)) * N + col;
        sp = S + (size_t)grp * N + col;
    }
    // the next group's words into L2.  Loads into registers before the digits are staged would share
    // scoreboards with the activations' and hold them up: 14336x4096 11.5 us, so 11.1.
    __device__ __forceinline__ void prefetch() const {
#pragma unroll
        for (int c = 0; c < 4; ++c) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(wp + c * row4));
    }
    // (one load in a loop, whatever moved the pointers: a second one in a branch of its own kept
    // the compiler from overlapping it with the arithmetic)
    __device__ __forceinline__ void load() {
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = ldg_stream128(wp + c * row4);
        s = ldg_stream64(sp);
        wp += 4 * row4;
        sp += n;
    }
};

// acc += factor * (ng groups (>= 1; the first is read) x the rows): acc[b][c] is
// column 4g + 2b + (c >> 1) of row 2t + (c & 1).  `arow`: row g's activations of the first
// group's K row 8t on; not read where !rowok.
template <class DT>
__device__ __forceinline__ void multiply(WordStream &st, const uint16_t *arow, bool rowok, int ng, float factor,
                                         float (&acc)[2][4]) {
    for (int i = 0; i < ng; ++i) {
        // the rows first: a wait for them must not wait for the next group's weights
        uint4 x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            x[c] = make_uint4(0u, 0u, 0u, 0u);
            if (rowok) x[c] = __ldg(reinterpret_cast<const uint4 *>(arow + 32 * c));
        }
        arow += kGS;
        const uint4 w[4] = {st.w[0], st.w[1], st.w[2], st.w[3]};
        const uint2 s4 = st.s;
        if (i + 1 < ng) st.load();
        float part[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t d0[4], d1[4], d2[4], d3[4];
            word_pairs<DT>(w[c].x, d0);
            word_pairs<DT>(w[c].y, d1);
            word_pairs<DT>(w[c].z, d2);
            word_pairs<DT>(w[c].w, d3);
            // rows (0, 4) and (1, 5), then (2, 6) and (3, 7), as the words decode
            const uint32_t bb[2][2] = {{__byte_perm(x[c].x, x[c].z, 0x5410), __byte_perm(x[c].x, x[c].z, 0x7632)},
                                       {__byte_perm(x[c].y, x[c].w, 0x5410), __byte_perm(x[c].y, x[c].w, 0x7632)}};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t a0[4] = {d0[2 * s], d1[2 * s], d0[2 * s + 1], d1[2 * s + 1]};
                const uint32_t a1[4] = {d2[2 * s], d3[2 * s], d2[2 * s + 1], d3[2 * s + 1]};
                mma16816<DT>(part[0], a0, bb[s]);
                mma16816<DT>(part[1], a1, bb[s]);
            }
        }
        const float s[4] = {DT::tof((uint16_t)(s4.x & 0xffffu)) * factor, DT::tof((uint16_t)(s4.x >> 16)) * factor,
                            DT::tof((uint16_t)(s4.y & 0xffffu)) * factor, DT::tof((uint16_t)(s4.y >> 16)) * factor};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[b][k] = fmaf(part[b][k], s[2 * b + (k >> 1)], acc[b][k]);
    }
}

// ---- the integer form ------------------------------------------------------------------
constexpr int kStage = 16;  // groups whose digit planes a warp holds
constexpr int kPlanes = 4;
// bytes of a plane: 128 per group; the 16 more put the planes of two neighbouring lanes' rows
// on the two 16-byte halves of every 32 bytes (conflict-free 16-byte reads)
__host__ __device__ constexpr int plane_bytes(int groups) { return (groups < kStage ? groups : kStage) * 128 + 16; }

__device__ __forceinline__ uint32_t even_rows(uint32_t x) { return (x << 4) & 0xF0F0F0F0u; }
__device__ __forceinline__ uint32_t odd_rows(uint32_t x) { return x & 0xF0F0F0F0u; }

__device__ __forceinline__ void imma(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                     uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// of 8 packed activations: max |value| in the high half, 0xFFFF - (min non-zero |value| - 1) in
// the low half (0 if there is none), as magnitude bits
__device__ __forceinline__ uint32_t extent(const uint4 v) {
    const uint32_t m[4] = {v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu, v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu};
    const uint32_t mx = __vmaxu2(__vmaxu2(m[0], m[1]), __vmaxu2(m[2], m[3]));
    uint32_t mn = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)  // 0x8000 - magnitude, 0x8000 itself for 0 -> 0
        mn = __vmaxu2(mn, (0x80008000u - m[k]) & 0x7FFF7FFFu);
    return (max(mx & 0xFFFFu, mx >> 16) << 16) | max(mn & 0xFFFFu, mn >> 16);
}

// the 8 activations of a word (v: packed pairs, rows in order) -> per digit plane d its even
// and its odd rows' bytes, out[d] = (rows 0,2,4,6 | rows 1,3,5,7)
template <class DT>
__device__ __forceinline__ void word_digits(const uint4 v, float up, uint2 (&out)[4]) {
    const uint32_t h2[4] = {v.x, v.y, v.z, v.w};
    uint32_t x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint16_t h = (uint16_t)((k & 1) ? h2[k / 2] >> 16 : h2[k / 2] & 0xFFFFu);
        x[k] = (uint32_t)__float2int_rn(DT::tof(h) * up) + 0x80808080u;
    }
    uint32_t r[2][4];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
        const uint32_t p01 = __byte_perm(x[o], x[o + 2], 0x5140), p23 = __byte_perm(x[o + 4], x[o + 6], 0x5140);
        const uint32_t q01 = __byte_perm(x[o], x[o + 2], 0x7362), q23 = __byte_perm(x[o + 4], x[o + 6], 0x7362);
        r[o][0] = __byte_perm(p01, p23, 0x5410) ^ 0x80808080u;
        r[o][1] = __byte_perm(p01, p23, 0x7632) ^ 0x80808080u;
        r[o][2] = __byte_perm(q01, q23, 0x5410) ^ 0x80808080u;
        r[o][3] = __byte_perm(q01, q23, 0x7632) ^ 0x80808080u;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) out[d] = make_uint2(r[0][d], r[1][d]);
}

// An activation row of up to kStage groups as digit planes in the warp's shared memory.
template <class DT>
struct DigitRow {
    char *planes;
    int pbytes;   // of a plane
    float *step;  // [kStage]: 2^-e / 16 (the weights are 16 x code) of every group, 0 of those left out; then left()

    // shared memory of a warp whose stages have `groups` groups at most
    __host__ __device__ static constexpr int bytes(int groups) { return kPlanes * plane_bytes(groups) + kStage * 4 + 16; }
    __device__ __forceinline__ DigitRow(char *mem, int groups) {
        pbytes = plane_bytes(groups);
        planes = mem;
        step = reinterpret_cast<float *>(mem + kPlanes * pbytes);
    }

    // Two passes over the activations, whose exponents meet in between (in the planes' memory): all loads of a pass
    // are on their way together.
    __device__ __forceinline__ void stage(const uint16_t *a0, int ng, int lane) {
        constexpr int kMant = DT::kBF16 ? 7 : 10, kBias = DT::kBF16 ? 127 : 15;
        const uint4 *a = reinterpret_cast<const uint4 *>(a0);
        uint32_t *ext = reinterpret_cast<uint32_t *>(planes);
        __syncwarp();  // the planes' last readers are through
#pragma unroll 2
        for (int u = lane; u < 16 * ng; u += 32) ext[u] = extent(__ldg(a + u));  // word row u
        __syncwarp();
        // two lanes per group
        uint32_t r = 0;
        if (lane < 2 * ng) {
            const uint4 x = reinterpret_cast<const uint4 *>(ext)[2 * lane], y = reinterpret_cast<const uint4 *>(ext)[2 * lane + 1];
            r = __vmaxu2(__vmaxu2(__vmaxu2(x.x, x.y), __vmaxu2(x.z, x.w)), __vmaxu2(__vmaxu2(y.x, y.y), __vmaxu2(y.z, y.w)));
        }
        r = __vmaxu2(r, __shfl_xor_sync(0xffffffffu, r, 1));
        // exponents of the largest and the smallest value (a subnormal has the lowest one's)
        const int mx = (int)(r >> 16), mn = 0x8000 - (int)(r & 0xFFFFu);
        const int top = max(mx >> kMant, 1), low = max(mn >> kMant, 1);
        const int e = 29 + kBias - top;  // |value| < 2^(top - kBias + 1)
        // the last bit of the smallest counts 1 or more; 2^e and 2^-e / 16 are normal fp32
        const bool exact = top - low <= 29 - kMant && top < (DT::kBF16 ? 255 : 31) && e <= 122;
        const unsigned out = __ballot_sync(0xffffffffu, !exact && mx != 0) & 0x55555555u;
        if ((lane & 1) == 0 && lane < 2 * ng) step[lane / 2] = exact && mx != 0 ? __int_as_float((123 - e) << 23) : 0.0f;
        if (lane == 0) step[kStage] = __uint_as_float(out);
        __syncwarp();
#pragma unroll 1
        for (int u = lane; u < 16 * ng; u += 32) {
            const int s = __float_as_int(step[u / 16]);  // 2^e has the exponent 250 - that of 2^(-4 - e)
            uint2 d[kPlanes];
            word_digits<DT>(__ldg(a + u), s ? __int_as_float((250 << 23) - s) : 0.0f, d);
            char *dst = planes + (u / 16) * 128 + (u & 3) * 32 + ((u >> 2) & 3) * 8;
#pragma unroll
            for (int k = 0; k < kPlanes; ++k) *reinterpret_cast<uint2 *>(dst + k * pbytes) = d[k];
        }
        __syncwarp();
    }
    // the groups that stage() left out: bit 2i for group i.  (Kept in shared memory: the loops over the
    // groups have no register for it.)
    __device__ __forceinline__ unsigned left() const {
        return __float_as_uint(*reinterpret_cast<volatile float *>(step + kStage));
    }

    // acc += (staged group i) x w, scaled by s4 * factor: acc[b][c] is column 4g + 2b + (c >> 1),
    // plane 2t + (c & 1)
    __device__ __forceinline__ void group(const uint4 (&w)[4], const uint2 s4, float factor, int i, int lane,
                                          float (&acc)[2][4]) const {
        const int g = lane >> 2, t = lane & 3;
        const char *b0 = planes + (g < kPlanes ? g : 0) * pbytes + t * 32 + i * 128;
        const uint32_t mask = g < kPlanes ? 0xffffffffu : 0u;
        const float f = step[i], zero = -digit::kMagic * f;
        int32_t d[2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c) d[b][c] = (int32_t)digit::kMagicBits;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 v = *reinterpret_cast<const uint4 *>(b0 + 16 * h);
            const uint32_t b[4] = {v.x & mask, v.y & mask, v.z & mask, v.w & mask};
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint4 x = w[2 * h + q];
                imma(d[0], even_rows(x.x), even_rows(x.y), odd_rows(x.x), odd_rows(x.y), b[2 * q], b[2 * q + 1]);
                imma(d[1], even_rows(x.z), even_rows(x.w), odd_rows(x.z), odd_rows(x.w), b[2 * q], b[2 * q + 1]);
            }
        }
        const float s[4] = {DT::tof((uint16_t)(s4.x & 0xFFFFu)) * factor, DT::tof((uint16_t)(s4.x >> 16)) * factor,
                            DT::tof((uint16_t)(s4.y & 0xFFFFu)) * factor, DT::tof((uint16_t)(s4.y >> 16)) * factor};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                acc[b][c] = fmaf(fmaf(__int_as_float(d[b][c]), f, zero), s[2 * b + (c >> 1)], acc[b][c]);
    }

    // acc += factor * (a group that stage() left out) in 16 bits, as plane 0: `st` at that group,
    // `a` its activations
    __device__ __forceinline__ static void left_out(WordStream &st, const uint16_t *a, float factor, int lane,
                                                    float (&acc)[2][4]) {
        st.load();
        multiply<DT>(st, a + 8 * (lane & 3), lane < 4, 1, factor, acc);
    }

    // total[j] += acc's planes at column 4g + j, in the lanes with t = 0
    __device__ __forceinline__ static void finish(const float (&acc)[2][4], float (&total)[4]) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float r = acc[b][2 * c] + 256.0f * acc[b][2 * c + 1];  // planes 0, 1 here and 2, 3 at t = 1
                total[2 * b + c] += r + 65536.0f * __shfl_down_sync(0xffffffffu, r, 1);
            }
    }
};

}  // namespace int4
}  // namespace ternocl
