// int4 decode GEMV (small M):
//
//   C[m,n] = DT(epi( sum_g S[g,n] * sum_{k in g} A[m,k] * code(B[k,n]) ))
//
// M >= 3: a CTA owns 32 columns, up to 8 activation rows and a K range, which its W warps (and
// SK CTAs of a cluster) split by 128-row groups (gemv_int4_core.cuh); the partial sums meet in
// gemv::finish, in a fixed order.
//
// M <= 2: the same on the integer form, for ranges of up to kStage groups per warp.
//
// Bound by HBM, with issue close behind (the 16-bit form needs 314 instructions per group and
// warp, the integer one ~110).  Weights go straight to registers: no ring in shared memory
// leaves ~24 resident warps per SM with 2 KB each in flight, and a warp nothing to wait for
// before its first words (on the cp.async ring of gemv_common.cuh 5120x248320 at M = 2 took
// 223 us, 2.9 TB/s).  Reading further ahead (2 to 4 groups at 80 to 128 registers) measured
// the same or slower, and so did CTAs that walk several strips with the planes kept and the
// next strip's words on their way (134 against 130 us).
// Measured on B200 (bf16, CUDA graph, us; floor = words and scales at 6.45 TB/s): 4096x4096 M=1 4.45
// (1.3), M=8 5.65; 4096x28672 M=1 17.1 (9.4), M=8 20.2; 5376x21504 M=1 15.6 (9.3), M=8 17.3;
// 14336x4096 M=1 10.9 (4.7); 5120x248320 M=1 126 (102), M=8 156.  ncu, 5120x124160 M=1
// (profiles/int4_gemv_gemm.md): DRAM reads = words + scales, issue 54 % busy, 256 instructions
// per group and warp with a CTA's ends counted in.
#include <cuda_runtime.h>

#include "gemv_common.cuh"
#include "gemv_int4_core.cuh"
#include "launch.h"

namespace ternocl {

namespace {

struct Int4Cols {
    using AccurateEpilogueTag = void;
    static constexpr bool kContiguousCols = true;
    __device__ static int thread_col(int g, int i) { return 4 * g + i; }
};

template <int W, class DT, int POSTOP, bool OUT_F32>
__global__ void __launch_bounds__(W * 32, 24 / W) gemv_int4_kernel(const gemv::Params p) {
    extern __shared__ __align__(128) char smem[];  // [W][32][8] partial sums
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 32, mb = blockIdx.z * 8;
    const int G = p.K / kGS, sk = blockIdx.y;
    const int cg0 = (int)((long long)G * sk / p.SK), ng = (int)((long long)G * (sk + 1) / p.SK) - cg0;
    const int g0 = cg0 + ng * warp / W, g1 = cg0 + ng * (warp + 1) / W;
    const bool rowok = mb + g < p.M;
    float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    int4::WordStream st;
    st.width(p.N);
    if (g0 < g1) {
        st.seek(p.B, p.S, p.N, g0, n0, lane);
        st.load();
    }
    pdl_wait();  // the weights are on their way; the activations are the previous kernel's
    if (g0 < g1)
        int4::multiply<DT>(st, p.A + (size_t)(rowok ? mb + g : 0) * p.K + (size_t)g0 * kGS + 8 * t, rowok, g1 - g0, 1.0f,
                           acc);
    pdl_launch_dependents();
    float v[8] = {acc[0][0], acc[0][2], acc[1][0], acc[1][2], acc[0][1], acc[0][3], acc[1][1], acc[1][3]};
    gemv::finish<Int4Cols, W, DT, POSTOP, OUT_F32>(p, smem, v, n0 + 4 * g < p.N);
}

template <int W, int ROWS, class DT, int POSTOP, bool OUT_F32>
__global__ void __launch_bounds__(W * 32, 24 / W) gemv_int4_digit_kernel(const gemv::Params p, int pbytes) {
    extern __shared__ __align__(128) char smem[];  // [W][32][8] partial sums, then the warps' planes
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2;
    const int n0 = blockIdx.x * 32;
    const int G = p.K / kGS, sk = blockIdx.y;
    const int cg0 = (int)((long long)G * sk / p.SK), cng = (int)((long long)G * (sk + 1) / p.SK) - cg0;
    const int g0 = cg0 + cng * warp / W, ng = cg0 + cng * (warp + 1) / W - g0;
    int4::WordStream st;
    st.width(p.N);
    if (ng > 0) {
        st.seek(p.B, p.S, p.N, g0, n0, lane);
        st.load();
    }
    pdl_wait();  // the weights are on their way; the activations are the previous kernel's
    int4::DigitRows<ROWS, DT> rows;
    rows.pbytes = pbytes;
    rows.planes = smem + W * 1024 + warp * 3 * ROWS * pbytes;
    rows.stage(p.A + (size_t)g0 * kGS, p.K, ng, lane);
    float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int i = 0; i < ng; ++i) {
        const uint4 w[4] = {st.w[0], st.w[1], st.w[2], st.w[3]};
        const uint2 s4 = st.s;
        if (i + 1 < ng) st.load();
        rows.group(w, s4, 1.0f, i, lane, acc);
    }
    pdl_launch_dependents();
    float total[4] = {0.f, 0.f, 0.f, 0.f};
    if (ng > 0) rows.finish(acc, lane, total);  // (ng is the same for the whole warp)
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = total[j];                                                                     // row 2t
        v[4 + j] = ROWS == 2 ? __shfl_down_sync(0xffffffffu, total[j], 2) : 0.0f;  // row 2t + 1: from lane t = 2
    }
    gemv::finish<Int4Cols, W, DT, POSTOP, OUT_F32>(p, smem, v, n0 + 4 * g < p.N);
}

template <int W, int ROWS, class DT, int POSTOP, bool OUT_F32>
cudaError_t launch_digit(const GemvArgs &a, int most) {
    const gemv::Params p = gemv::gemv_params_impl(a);
    auto kern = gemv_int4_digit_kernel<W, ROWS, DT, POSTOP, OUT_F32>;
    const int pbytes = int4::plane_bytes(most);
    const size_t smem = (size_t)W * (1024 + 3 * ROWS * pbytes);
    const cudaError_t e = ensure_smem(kern, smem);
    if (e != cudaSuccess) return e;
    return launch_kernel_cluster(kern, dim3((a.N + 31) / 32, a.SK), dim3(W * 32), smem, a.stream,
                                 dim3(1, a.cluster ? a.SK : 1, 1), p, pbytes);
}

template <int W, class DT, int POSTOP, bool OUT_F32>
cudaError_t launch_w(const GemvArgs &a) {
    const int G = a.K / kGS, most = ((G + a.SK - 1) / a.SK + W - 1) / W;  // groups of any warp
    if (a.M == 1 && most <= int4::kStage) return launch_digit<W, 1, DT, POSTOP, OUT_F32>(a, most);
    if (a.M == 2 && most <= int4::kStage) return launch_digit<W, 2, DT, POSTOP, OUT_F32>(a, most);
    const gemv::Params p = gemv::gemv_params_impl(a);
    auto kern = gemv_int4_kernel<W, DT, POSTOP, OUT_F32>;
    const dim3 grid((a.N + 31) / 32, a.SK, (a.M + 7) / 8);
    return launch_kernel_cluster(kern, grid, dim3(W * 32), (size_t)W * 1024, a.stream,
                                 dim3(1, a.cluster ? a.SK : 1, 1), p);
}

}  // namespace

cudaError_t int4_gemv_launch(const GemvArgs &a) {
    return dispatch_epilogue<GemvArgs>(a, [&](auto dt, auto po, auto of) {
        using DT = typename decltype(dt)::type;
        constexpr int PO = decltype(po)::value;
        constexpr bool F32 = decltype(of)::value;
        if (a.warps >= 8) return launch_w<8, DT, PO, F32>(a);
        return launch_w<4, DT, PO, F32>(a);
    });
}

}  // namespace ternocl
