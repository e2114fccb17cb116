// int4 product for a few rows (9 to 24):
//
//   C[m,n] = DT(epi( sum_g S[g,n] * sum_{k in g} A[m,k] * code(k,n) ))
//
// Between the GEMV, whose CTAs would read the activations once per 32 columns, and the tcgen05
// GEMM, whose decoded 16-bit operand crosses shared memory twice (48 KB of traffic per 4 KB of
// words, 375 cycles a step whatever the rows): here a word decodes into registers as in
// gemv_int4_core.cuh and is used for R blocks of 8 rows at once.  A CTA owns 256 columns of
// all rows (8R at most) and a K range (split over a thread-block cluster); warp w owns 32 of the columns, streams
// their words into registers one group ahead, and all warps share the activations of a group,
// staged in the words' pair order in one of two buffers in shared memory.  The sums leave through
// shared memory, so that stores and the other CTAs' shares (distributed shared memory, in split
// order) are whole rows.
//
// ~180 instructions decode a group of 32 columns, ~55 more multiply a block of 8 rows.  No unit is full: on
// 5376x64512 at M = 24 L1's data pipe is at 55 %, the tensor pipe at 40 %, DRAM at 29 %, and an instruction
// issues in 47 % of the cycles; the 4 warps per scheduler that 128 registers leave wait for the
// tensor pipe (a third of their stalls), for fixed latencies and at the group's barrier.
// Measured on B200 (bf16, CUDA graph): 5376x21504 M=9 22.7-26.8 us, M=16 23.5-24.2 us (on the tcgen05 GEMM
// 31.0 and 31.6), M=24 28.7 us (33.0); floor 9.4 us, the words once.
#include <cuda_runtime.h>

#include "common.cuh"
#include "gemv_common.cuh"
#include "gemv_int4_core.cuh"
#include "launch.h"

namespace ternocl {

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kTileCols = kWarps * 32;
constexpr int kActRow = kGS * 2 + 64;   // bytes of a staged row: 64 mod 128, 16-byte reads conflict-free

struct RParams {  // M <= 8R
    const uint16_t *A;
    const uint32_t *B;
    const uint16_t *S;
    void *C;
    const uint16_t *Other;
    const void *Bias;
    int M, N, K;
};

template <int R>
struct Smem {
    static constexpr int act = 0;  // two buffers of 8R rows
    static constexpr int out = 2 * 8 * R * kActRow;
    static constexpr int total = out + 8 * R * kTileCols * 4;
};

template <int R, class DT, int POSTOP, bool OUT_F32>
__global__ void __launch_bounds__(kThreads, 2) gemm_int4_rows_kernel(const RParams p) {
    using SM = Smem<R>;
    extern __shared__ __align__(128) char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    const int G = p.K / kGS, SK = gridDim.y, sk = blockIdx.y;
    const int rows = min(8 * R, p.M);  // (M; the bound, told to the compiler, is worth 2 us at M = 24)
    const int g0 = (int)((long long)G * sk / SK), ng = (int)((long long)G * (sk + 1) / SK) - g0;
    const int n0 = blockIdx.x * kTileCols, ns = n0 + warp * 32;

    int4::WordStream st;
    st.width(p.N);
    st.seek(p.B, p.S, p.N, g0, ns, lane);
    st.load();
    pdl_wait();  // the weights are on their way; the activations are the previous kernel's

    // a group's activations: word w of row r as unit 16r + w, pairs (j, j+4) of each word
    constexpr int kUnits = (8 * R * 16 + kThreads - 1) / kThreads;
    uint4 next[kUnits];
    auto fetch = [&](int grp) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int x = u * kThreads + tid, r = x >> 4;
            next[u] = make_uint4(0u, 0u, 0u, 0u);
            if (r < rows)
                next[u] = __ldg(reinterpret_cast<const uint4 *>(p.A + (size_t)r * p.K + (size_t)grp * kGS) + (x & 15));
        }
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int x = u * kThreads + tid, r = x >> 4;
            const uint4 v = next[u];
            uint4 o;
            o.x = __byte_perm(v.x, v.z, 0x5410);
            o.y = __byte_perm(v.x, v.z, 0x7632);
            o.z = __byte_perm(v.y, v.w, 0x5410);
            o.w = __byte_perm(v.y, v.w, 0x7632);
            if (r < 8 * R)
                *reinterpret_cast<uint4 *>(smem + SM::act + (buf * 8 * R + r) * kActRow + (x & 15) * 16) = o;
        }
    };
    fetch(g0);
    stage(0);
    __syncthreads();

    float acc[R][2][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[r][b][k] = 0.0f;
    for (int i = 0; i < ng; ++i) {
        if (i + 1 < ng) fetch(g0 + i + 1);
        const uint4 w[4] = {st.w[0], st.w[1], st.w[2], st.w[3]};
        const uint2 s4 = st.s;
        if (i + 1 < ng) st.load();
        float part[R][2][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) part[r][b][k] = 0.0f;
        const char *act = smem + SM::act + ((i & 1) * 8 * R + g) * kActRow + t * 16;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t d0[4], d1[4], d2[4], d3[4];
            int4::word_pairs<DT>(w[c].x, d0);
            int4::word_pairs<DT>(w[c].y, d1);
            int4::word_pairs<DT>(w[c].z, d2);
            int4::word_pairs<DT>(w[c].w, d3);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint4 x = *reinterpret_cast<const uint4 *>(act + r * 8 * kActRow + c * 64);
                const uint32_t bb[2][2] = {{x.x, x.y}, {x.z, x.w}};
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint32_t a0[4] = {d0[2 * s], d1[2 * s], d0[2 * s + 1], d1[2 * s + 1]};
                    const uint32_t a1[4] = {d2[2 * s], d3[2 * s], d2[2 * s + 1], d3[2 * s + 1]};
                    mma16816<DT>(part[r][0], a0, bb[s]);
                    mma16816<DT>(part[r][1], a1, bb[s]);
                }
            }
        }
        const float s[4] = {DT::tof((uint16_t)(s4.x & 0xffffu)), DT::tof((uint16_t)(s4.x >> 16)),
                            DT::tof((uint16_t)(s4.y & 0xffffu)), DT::tof((uint16_t)(s4.y >> 16))};
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[r][b][k] = fmaf(part[r][b][k], s[2 * b + (k >> 1)], acc[r][b][k]);
        if (i + 1 < ng) stage((i + 1) & 1);  // (its last readers passed the barrier below)
        __syncthreads();
    }
    pdl_launch_dependents();

    // sums [8R][256]: lane (g, t) holds columns 4g + 2b + {0, 1} of rows 8r + 2t + {0, 1}
    float *out = reinterpret_cast<float *>(smem + SM::out);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float4 *>(out + (8 * r + 2 * t + h) * kTileCols + warp * 32 + 4 * g) =
                make_float4(acc[r][0][h], acc[r][0][2 + h], acc[r][1][h], acc[r][1][2 + h]);
    __syncthreads();
    if (SK > 1) gemv::cluster_sync_all();
    const int r0 = rows * sk / SK, r1 = rows * (sk + 1) / SK;
    for (int x = r0 * 32 + tid; x < r1 * 32; x += kThreads) {  // 8 columns of a row
        const int r = x >> 5, n = n0 + 8 * (x & 31);
        if (n >= p.N) continue;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const float *src = out + r * kTileCols + 8 * (x & 31);
        for (int q = 0; q < SK; ++q) {
            float4 lo, hi;
            if (SK > 1) {
                lo = gemv::ld_dsmem_f4(gemv::smem_u32(src), (uint32_t)q);
                hi = gemv::ld_dsmem_f4(gemv::smem_u32(src + 4), (uint32_t)q);
            } else {
                lo = *reinterpret_cast<const float4 *>(src);
                hi = *reinterpret_cast<const float4 *>(src + 4);
            }
            v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
            v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
        }
        const size_t at = (size_t)r * p.N + n;
        uint4 o = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (POSTOP == 1 || POSTOP == 2) o = *reinterpret_cast<const uint4 *>(p.Other + at);
        const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float e;
            if constexpr (POSTOP == 1 || POSTOP == 2) e = DT::tof((uint16_t)((k & 1) ? ow[k / 2] >> 16 : ow[k / 2] & 0xFFFFu));
            else e = epi_in<DT, POSTOP, OUT_F32>(p.Other, p.Bias, at, n + k);
            v[k] = epi<POSTOP, OUT_F32>(v[k], e);
        }
        if constexpr (OUT_F32) {
            float4 *dst = reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.C) + at);
            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = (uint32_t)DT::fromf(v[2 * k]) | ((uint32_t)DT::fromf(v[2 * k + 1]) << 16);
            *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(p.C) + at) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    if (SK > 1) gemv::cluster_sync_all();  // every CTA's sums stay until all have read them
}

template <int R>
cudaError_t launch(const GemvArgs &a, int sms) {
    const RParams p{(const uint16_t *)a.A, a.B, (const uint16_t *)a.S, a.C, (const uint16_t *)a.Other, a.Bias,
                    a.M, a.N, a.K};
    const int G = a.K / kGS, cols = (a.N + kTileCols - 1) / kTileCols;
    // K split: the rounds of two CTAs per SM it takes, per group, and ~2 groups' time for a CTA's ends
    int sk = 1;
    long long best = 1LL << 60;
    for (int s = 1; s <= 8 && s <= G; ++s) {
        const long long rounds = ((long long)cols * s + 2 * sms - 1) / (2 * sms);
        const long long cost = rounds * ((G + s - 1) / s + 2);
        if (cost < best) {
            best = cost;
            sk = s;
        }
    }
    return dispatch_epilogue<GemvArgs>(a, [&](auto dt, auto po, auto of) -> cudaError_t {
        using DT = typename decltype(dt)::type;
        auto kern = gemm_int4_rows_kernel<R, DT, decltype(po)::value, decltype(of)::value>;
        const cudaError_t e = ensure_smem(kern, Smem<R>::total);
        if (e != cudaSuccess) return e;
        return launch_kernel_cluster(kern, dim3(cols, sk), dim3(kThreads), (size_t)Smem<R>::total, a.stream,
                                     dim3(1, sk, 1), p);
    });
}

}  // namespace

cudaError_t int4_rows_launch(const GemvArgs &a, int sms) {
    return a.M <= 16 ? launch<2>(a, sms) : launch<3>(a, sms);
}

}  // namespace ternocl
