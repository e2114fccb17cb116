// int4 decode GEMV (small M):
//
//   C[m,n] = DT(epi( sum_g S[g,n] * sum_{k in g} A[m,k] * code(B[k,n]) ))
//
// M >= 2: a CTA owns 32 columns, up to 8 activation rows and a K range, which its W warps (and
// SK CTAs of a cluster) split by 128-row groups (gemv_int4_core.cuh); the partial sums meet in
// gemv::finish, in a fixed order.
//
// M = 1: the same on the integer form, for ranges of up to kStage groups per warp.  (With the digits
// of two rows it was slower than the 16-bit form: 4096x28672 M=2 21.1 against 18-20 us, 4096x4096
// 5.5 / 5.1, 14336x4096 12.8 / 11.9, 5120x34816 25.9 / 25.2, 5120x248320 149 / 145-149.)
//
// Grouped by expert, with 8 rows per expert or fewer on average: the M >= 2 form on the rows of one
// expert in blocks of 8.
//
// What bounds it: L1's data pipe is the busiest unit (76 % of the time at M = 1, 79 % at M = 8 on
// 5120x124160, where DRAM is at 60 and 53 % of its peak and an instruction issues in 54 and 63 % of the
// cycles); a group of a warp takes 236 instructions at M = 1 (the product ~110, the rest staging and
// a CTA's ends) and 297 at M = 8.  Weights go straight to registers: no ring in shared memory
// leaves 24 to 28 resident warps per SM with 2 KB each in flight, and a warp nothing to wait for
// before its first words (on the cp.async ring of gemv_common.cuh 5120x248320 at M = 2 took
// 223 us, 2.9 TB/s).  Reading further ahead (2 to 4 groups at 80 to 128 registers) measured
// the same or slower, and so did CTAs that walk several strips with the planes kept and the
// next strip's words on their way (134 against 130 us).
// Measured on B200 (bf16, CUDA graph, us; floor = words and scales at 6.45 TB/s): 4096x4096 M=1 4.3
// (1.3), M=8 5.0-5.3; 4096x28672 M=1 14.1 (9.4), M=8 17.4; 5376x21504 M=1 15.3 (9.3), M=8 16.8;
// 14336x4096 M=1 11.2 (4.7), M=8 12.1; 5120x248320 M=1 121-129 (102), M=2 145-149, M=8 148-155.
// Grouped, 536 rows x 2048 x 768 over 128 experts 28.6 us (floor 16.4; 46 us on the tcgen05 kernel,
// whose tiles would hold 4 rows), 128 rows 18.2 (10.5).
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

// warps on an SM, at 72 registers: 7 CTAs of 4 warps, or 3 of 8
constexpr int kResident = 28;

template <int W, class DT, int POSTOP, bool OUT_F32>
__global__ void __launch_bounds__(W * 32, kResident / W) gemv_int4_kernel(const gemv::Params p) {
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

template <int W, class DT, int POSTOP, bool OUT_F32>
__global__ void __launch_bounds__(W * 32, kResident / W)
    gemv_int4_digit_kernel(const gemv::Params p, int most) {  // most: groups of any warp
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
        st.prefetch();
    }
    pdl_wait();  // the weights are on their way; the activations are the previous kernel's
    int4::DigitRow<DT> row(smem + W * 1024 + warp * int4::DigitRow<DT>::bytes(most), most);
    row.stage(p.A + (size_t)g0 * kGS, ng, lane);
    if (ng > 0) st.load();
    float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int i = 0; i < ng; ++i) {
        const uint4 w[4] = {st.w[0], st.w[1], st.w[2], st.w[3]};
        const uint2 s4 = st.s;
        if (i + 1 < ng) st.load();
        row.group(w, s4, 1.0f, i, lane, acc);
    }
    for (unsigned left = row.left(); left; left &= left - 1) {
        const int grp = g0 + (__ffs(left) - 1) / 2;
        st.seek(p.B, p.S, p.N, grp, n0, lane);
        row.left_out(st, p.A + (size_t)grp * kGS, 1.0f, lane, acc);
    }
    pdl_launch_dependents();
    float total[4] = {0.f, 0.f, 0.f, 0.f};
    if (ng > 0) row.finish(acc, total);  // (ng is the same for the whole warp)
    float v[8] = {total[0], total[1], total[2], total[3], 0.f, 0.f, 0.f, 0.f};  // row 2t (of t = 0)
    gemv::finish<Int4Cols, W, DT, POSTOP, OUT_F32>(p, smem, v, n0 + 4 * g < p.N);
}

// ---- the grouped product for a few rows per expert ----------------------------------------
// CTA (x, y): 32 columns of expert y's first 8 rows; y >= E: of the (y - E)-th of the further blocks of
// 8 rows, counted over the experts, most of which do not exist.
struct GroupedParams {
    const int *meta;
    const uint16_t *A;
    const uint32_t *B;
    const uint16_t *S;
    void *C;
    const uint16_t *Other;
    int M, N, K, E;
};

template <int W, class DT, int POSTOP, bool OUT_F32>
__global__ void __launch_bounds__(W * 32, kResident / W) gemv_int4_grouped_kernel(const GroupedParams p) {
    __shared__ __align__(16) float red[W][32][8];  // partial sums
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 32, G = p.K / kGS;
    pdl_wait();  // meta comes from the routing kernel
    int e = blockIdx.y, block = 0;
    auto first = [&](int x) { return min(max(p.meta[x], 0), p.M); };
    auto count = [&](int x) { return x < p.E ? max(first(x + 1) - first(x), 0) : 0; };
    if (e >= p.E) {
        int want = e - p.E, e0 = 0;
        for (;; e0 += 32) {
            if (e0 >= p.E) return;  // (every warp finds the same)
            const int own = max(count(e0 + lane) - 1, 0) / 8;
            int incl = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            const unsigned past = __ballot_sync(0xffffffffu, incl > want);
            if (past) {
                const int l = __ffs(past) - 1;
                e = e0 + l;
                block = 1 + want - __shfl_sync(0xffffffffu, incl - own, l);
                break;
            }
            want -= __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    const int rows = min(count(e) - 8 * block, 8), row0 = first(e) + 8 * block;
    if (rows <= 0) return;
    const int g0 = G * warp / W, g1 = G * (warp + 1) / W;
    float acc[2][4] = {};
    if (g0 < g1) {
        int4::WordStream st;
        st.width(p.N);
        st.seek(p.B, p.S, p.N, e * G + g0, n0, lane);
        st.load();
        int4::multiply<DT>(st, p.A + (size_t)(row0 + (g < rows ? g : 0)) * p.K + (size_t)g0 * kGS + 8 * t, g < rows,
                           g1 - g0, 1.0f, acc);
    }
    pdl_launch_dependents();
    *reinterpret_cast<float4 *>(&red[warp][lane][0]) = make_float4(acc[0][0], acc[0][2], acc[1][0], acc[1][2]);
    *reinterpret_cast<float4 *>(&red[warp][lane][4]) = make_float4(acc[0][1], acc[0][3], acc[1][1], acc[1][3]);
    __syncthreads();
    // columns c, c + 1 of row m: lane (c / 4, m / 2)'s
    for (int m = tid >> 4; m < rows; m += 2 * W) {
        const int c = 2 * (tid & 15);
        if (n0 + c >= p.N) break;
        float v0 = 0.0f, v1 = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 x = *reinterpret_cast<const float2 *>(&red[w][c / 4 * 4 + m / 2][(m & 1) * 4 + (c & 3)]);
            v0 += x.x;
            v1 += x.y;
        }
        epi_store2<DT, POSTOP, OUT_F32, OUT_F32>(p.C, p.Other, nullptr, p.N, row0 + m, n0 + c, v0, v1);
    }
}

template <int W, class DT, int POSTOP, bool OUT_F32>
cudaError_t launch_digit(const GemvArgs &a, int most) {
    const gemv::Params p = gemv::gemv_params_impl(a);
    auto kern = gemv_int4_digit_kernel<W, DT, POSTOP, OUT_F32>;
    const size_t smem = (size_t)W * (1024 + int4::DigitRow<DT>::bytes(most));
    const cudaError_t e = ensure_smem(kern, smem);
    if (e != cudaSuccess) return e;
    return launch_kernel_cluster(kern, dim3((a.N + 31) / 32, a.SK), dim3(W * 32), smem, a.stream,
                                 dim3(1, a.cluster ? a.SK : 1, 1), p, most);
}

template <int W, class DT, int POSTOP, bool OUT_F32>
cudaError_t launch_w(const GemvArgs &a) {
    const int G = a.K / kGS, most = ((G + a.SK - 1) / a.SK + W - 1) / W;  // groups of any warp
    if (a.M == 1 && most <= int4::kStage) return launch_digit<W, DT, POSTOP, OUT_F32>(a, most);
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

// 4 warps split K, or 2 where that left a warp fewer than 4 groups.  With 4 and with 2 warps, 128 experts,
// us: K 768 (2048 columns) 536 rows 37.8 / 29.2, 128 rows 22.1 / 19.1; K 1024 (1024) 536 rows 22.9 / 21.1; K 1536
// (1024) 29.4 / 29.0 and 18.6 / 19.7; K 2048 (768) 28.3 / 27.9 and 17.9 / 21.4; K 4096 (768) 50.6 / 50.8 and
// 31.8 / 41.1.
cudaError_t int4_gemv_grouped_launch(const GemvArgs &a, const int *meta, int E) {
    const GroupedParams p{meta, (const uint16_t *)a.A, a.B, (const uint16_t *)a.S, a.C, (const uint16_t *)a.Other,
                          a.M, a.N, a.K, E};
    return dispatch_epilogue<GemvArgs>(a, [&](auto dt, auto po, auto of) {
        using DT = typename decltype(dt)::type;
        constexpr int PO = decltype(po)::value;
        constexpr bool F32 = decltype(of)::value;
        const dim3 grid((a.N + 31) / 32, E + a.M / 8);
        if (a.K / kGS >= 16) return launch_kernel(gemv_int4_grouped_kernel<4, DT, PO, F32>, grid, dim3(128), 0, a.stream, p);
        return launch_kernel(gemv_int4_grouped_kernel<2, DT, PO, F32>, grid, dim3(64), 0, a.stream, p);
    });
}

}  // namespace ternocl
