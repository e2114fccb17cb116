// int4 decode GEMV (small M):
//
//   C[m,n] = DT(epi( sum_g S[g,n] * sum_{k in g} A[m,k] * code(B[k,n]) ))
//
// Weight layout B uint32 [K/8, N] (int4_common.cuh).  On the skeleton of gemv_common.cuh:
// thread (g, q) streams, per 128-row group, the words of rows kp = 16grp + 4c + q
// (c = 0..3) and columns n0+4g .. n0+4g+3 plus those columns' scales.  A word decodes into
// four half2 of rows (p, p+4), two A registers for each of two mma.sync m16n8k16 (the 16
// columns of a block are the MMA's rows, up to 8 activation rows its columns); the
// activations are staged in the words' pair order.  Products of codes and DT activations
// are exact in the MMA's fp32 sums; a group's sum is scaled by S in fp32.
#include <cuda_runtime.h>

#include "gemv_common.cuh"
#include "int4_common.cuh"
#include "launch.h"

namespace ternocl {

namespace {

struct Int4Policy {
    static constexpr int kWords16 = 4;
    static constexpr int kWordRegs = kWords16;
    static constexpr bool kSharedSlots = false;
    using AccurateEpilogueTag = void;
    __device__ static void read_words(const char *stage, int tid, int nthreads, uint4 *w) {
#pragma unroll
        for (int c = 0; c < kWords16; ++c) w[c] = reinterpret_cast<const uint4 *>(stage)[c * nthreads + tid];
    }
    static constexpr bool kContiguousCols = true;
    static constexpr int kActGroupBytes = 16 * 16;  // 16 words x 8 activations
    static constexpr int kExtraGroupBytes = 0;
    static constexpr int kActBytesPerK = 2;  // DT activations
    static constexpr int kActPadBytes = 64;  // row stride = 64 mod 128: 16-byte reads conflict-free
    __device__ static int thread_col0(int g) { return 4 * g; }
    __device__ static bool copy_ok(int N, int n0, int g) { return n0 + 4 * g < N; }
    __device__ static int thread_col(int g, int i) { return 4 * g + i; }
    __device__ static const uint32_t *word_ptr(const gemv::Params &p, int grp, int g, int q, int n0) {
        return p.B + (size_t)(grp * int4::kWordsPerGroup + q) * p.N + n0 + 4 * g;
    }
    __device__ static size_t group_stride(const gemv::Params &p) { return (size_t)int4::kWordsPerGroup * p.N; }
    __device__ static size_t chunk_stride(const gemv::Params &p) { return (size_t)4 * p.N; }
    __host__ __device__ static size_t extra_smem(int, int) { return 0; }

    // rows [mb, mb+rows) x words [16cg0, 16(cg0+ng)), each word's activations as pairs (j, j+4)
    template <class DT>
    __device__ static void stage(const gemv::Params &p, char *act, int stride, char *, int mb, int rows, int cg0,
                                 int ng) {
        const int nw = ng * int4::kWordsPerGroup;
        for (int it = threadIdx.x; it < rows * nw; it += blockDim.x) {
            const int m = it / nw, w = it - m * nw;
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(
                p.A + (size_t)(mb + m) * p.K + (size_t)(cg0 * int4::kWordsPerGroup + w) * 8));
            uint4 o;
            o.x = __byte_perm(v.x, v.z, 0x5410);  // rows 0, 4
            o.y = __byte_perm(v.x, v.z, 0x7632);  // rows 1, 5
            o.z = __byte_perm(v.y, v.w, 0x5410);  // rows 2, 6
            o.w = __byte_perm(v.y, v.w, 0x7632);  // rows 3, 7
            *reinterpret_cast<uint4 *>(act + (size_t)m * stride + (size_t)w * 16) = o;
        }
    }

    template <class DT>
    __device__ static void compute(const uint4 w[4], uint2 sc, const char *arow, bool rowok, int q, const char *,
                                   float acc[2][4], int) {
        float part[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint4 b = make_uint4(0u, 0u, 0u, 0u);
            if (rowok) b = *reinterpret_cast<const uint4 *>(arow + (4 * c + q) * 16);
            uint32_t d0[4], d1[4], d2[4], d3[4];
            int4::word_pairs<DT>(w[c].x, d0);
            int4::word_pairs<DT>(w[c].y, d1);
            int4::word_pairs<DT>(w[c].z, d2);
            int4::word_pairs<DT>(w[c].w, d3);
            const uint32_t bb[2][2] = {{b.x, b.y}, {b.z, b.w}};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t a0[4] = {d0[2 * s], d1[2 * s], d0[2 * s + 1], d1[2 * s + 1]};
                const uint32_t a1[4] = {d2[2 * s], d3[2 * s], d2[2 * s + 1], d3[2 * s + 1]};
                mma16816<DT>(part[0], a0, bb[s]);
                mma16816<DT>(part[1], a1, bb[s]);
            }
        }
        const float s0 = DT::tof((uint16_t)(sc.x & 0xffffu)), s1 = DT::tof((uint16_t)(sc.x >> 16));
        const float s2 = DT::tof((uint16_t)(sc.y & 0xffffu)), s3 = DT::tof((uint16_t)(sc.y >> 16));
        acc[0][0] += part[0][0] * s0;
        acc[0][1] += part[0][1] * s0;
        acc[0][2] += part[0][2] * s1;
        acc[0][3] += part[0][3] * s1;
        acc[1][0] += part[1][0] * s2;
        acc[1][1] += part[1][1] * s2;
        acc[1][2] += part[1][2] * s3;
        acc[1][3] += part[1][3] * s3;
    }

    // C fragment: block b, c0/c1 = (row g -> column 4g+2b, activation rows 2q, 2q+1),
    // c2/c3 = (row g+8 -> column 4g+2b+1)
    __device__ static void thread_values(const float acc[2][4], float v[8]) {
        v[0] = acc[0][0]; v[1] = acc[0][2]; v[2] = acc[1][0]; v[3] = acc[1][2];
        v[4] = acc[0][1]; v[5] = acc[0][3]; v[6] = acc[1][1]; v[7] = acc[1][3];
    }
};

template <int W, class DT, int POSTOP, bool OUT_F32>
cudaError_t launch_w(const GemvArgs &a) {
    gemv::Params p = gemv::gemv_params_impl(a);
    const int G = a.K / kGS;
    const int max_ng = (G + a.SK - 1) / a.SK;
    const int rows = a.M < 8 ? a.M : 8;
    const size_t smem = gemv::smem_bytes<Int4Policy, W>(rows, max_ng * kGS);
    auto kern = gemv::gemv_kernel<Int4Policy, W, DT, POSTOP, OUT_F32>;
    if (smem > 48 * 1024) {
        cudaError_t e = ensure_smem(kern, smem);
        if (e != cudaSuccess) return e;
    }
    dim3 grid((a.N + 31) / 32, a.SK, (a.M + 7) / 8);
    return launch_kernel_cluster(kern, grid, dim3(W * 32), smem, a.stream, dim3(1, a.cluster ? a.SK : 1, 1), p);
}

template <class DT, int POSTOP, bool OUT_F32>
cudaError_t launch_t(const GemvArgs &a) {
    if (a.warps >= 8) return launch_w<8, DT, POSTOP, OUT_F32>(a);
    return launch_w<4, DT, POSTOP, OUT_F32>(a);
}

}  // namespace

size_t int4_gemv_smem(int M, int K, int SK, int warps) {
    const int G = K / kGS;
    const int max_ng = (G + SK - 1) / SK;
    return gemv::smem_bytes_w<Int4Policy>(warps, M < 8 ? M : 8, max_ng * kGS);
}

cudaError_t int4_gemv_launch(const GemvArgs &a) {
    return dispatch_epilogue<GemvArgs>(a, [&](auto dt, auto po, auto of) {
        using DT = typename decltype(dt)::type;
        return launch_t<DT, decltype(po)::value, decltype(of)::value>(a);
    });
}

}  // namespace ternocl
