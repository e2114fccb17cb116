// int4 MoE decode GEMVs: moe_decode.cu's products with 4-bit weights (int4_common.cuh),
//
//   gate_up   H[g, n] = DT(silu(x_t . gate_e[:, n]) * (x_t . up_e[:, n])),  x_t = X[g / topk]
//   down_sum  O[t, n] = DT(sum_j RW[g] * (H[g] . down_e[:, n])),  g = t*topk + j
//
// with e = ids[g] and every expert's weights stacked: B [E, K/8, N], S [E, K/128, N].
//
// A CTA owns 32 columns of one routed row (gate_up: of both matrices, whose dots meet in
// the CTA for the SwiGLU; down_sum: of one token, its K running over the topk experts side by
// side) over the whole K; its W warps split the 128-row groups, multiply them in the integer
// form of gemv_int4_core.cuh and are summed in warp order.  A gate_up warp multiplies its
// groups of both matrices with the same digit planes.
//
// An expert id outside [0, E) contributes zero, whatever its activations, and sets bit 1 of the device error word.
//
// Bound by latency for one token (ids, then words, then one or two groups per warp).  For several no unit is
// full: at 9 tokens L1's data pipe is at 56 % (down_sum 45 %), DRAM at 38 % (28 %), and the 4 warps per
// scheduler that 128 registers leave wait for loads most of the time; tokens that share an expert read
// its words again, from L2.  Measured on B200 (K 2048, N 768 and back, 128 experts, top-8, CUDA
// graph): gate_up 1 token 6.2-6.7 us (floor 2.0: every touched expert's words once), 9 tokens 25.2 us
// (14.2); down_sum 6.3-6.6 us (1.0) and 15.1 us (7.1).
#include <cuda_runtime.h>

#include "common.cuh"
#include "gemv_int4_core.cuh"
#include "launch.h"
#include "tc_common.cuh"

namespace ternocl {

namespace {

constexpr int kCols = 32;
// Units (a group of a matrix) a warp has on their way.  Two at 128 registers (16 resident warps)
// measured best: 4 spill, and with 24 warps at 80 registers 2 do.
constexpr int kAhead = 2;
enum Mode { kGateUp = 0, kDownSum = 1 };

struct MParams {
    const int *ids;
    const uint16_t *A;         // X [T, K] (gate_up) or H [G, K] (down_sum)
    const uint32_t *B0, *B1;   // gate / up, or down
    const uint16_t *S0, *S1;
    const uint16_t *RW;        // [G]
    uint16_t *out;             // H [G, N] or O [T, N]
    int N, K, topk, E, strips;
};

template <int MODE>
constexpr int kMats = MODE == kGateUp ? 2 : 1;

template <int W, int MODE, class DT>
__global__ void __launch_bounds__(W * 32, 16 / W) moe_decode_int4_kernel(const MParams p) {
    constexpr int NM = kMats<MODE>;
    extern __shared__ __align__(128) char smem[];  // the warps' planes
    __shared__ __align__(16) float red[W][NM][kCols];  // (written 16 bytes at a time)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int z = blockIdx.x / p.strips;  // routed row (gate_up) or token (down_sum)
    const int n0 = (blockIdx.x - z * p.strips) * kCols;
    const int G = p.K / kGS;
    const int all = MODE == kGateUp ? G : p.topk * G;
    const int g0 = (int)((long long)all * warp / W), ng = (int)((long long)all * (warp + 1) / W) - g0;
    const int most = (all + W - 1) / W;  // groups of any warp
    int4::DigitRow<DT> row(smem + warp * int4::DigitRow<DT>::bytes(most), most);

    pdl_wait();  // ids and activations come from the kernels before

    const uint16_t *a0 = p.A + (size_t)(MODE == kGateUp ? z / p.topk : z * p.topk) * p.K + (size_t)g0 * kGS;
    float total[NM][4];
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) total[m][j] = 0.0f;
    // the next kAhead (matrix, group) units are on their way
    uint4 w[kAhead][4];
    uint2 sc[kAhead];
    float factor[kAhead];
    bool bad_id = false;
    auto expert = [&](int slot) {
        const int e = p.ids[slot];
        bad_id |= e < 0 || e >= p.E;
        return e >= 0 && e < p.E ? e : -1;
    };
    const int col = n0 + 4 * (lane >> 2) < p.N ? n0 + 4 * (lane >> 2) : 0;  // (columns behind N are not stored)
    const size_t row4 = (size_t)4 * p.N;
    // group lg of expert e's matrix m into slot k
    auto load = [&](int k, int m, int e, int lg) {
        const size_t grp = (size_t)e * G + lg;
        const uint32_t *wp = (m ? p.B1 : p.B0) + (grp * int4::kWordsPerGroup + (lane & 3)) * p.N + col;
#pragma unroll
        for (int c = 0; c < 4; ++c) w[k][c] = ldg_stream128(wp + c * row4);
        sc[k] = ldg_stream64((m ? p.S1 : p.S0) + grp * p.N + col);
    };
    int4::WordStream st;  // to prefetch, and of the groups that the digits leave out
    st.width(p.N);
    auto prefetch = [&](int m, int e, int lg) {
        st.seek(m ? p.B1 : p.B0, m ? p.S1 : p.S0, p.N, e * G + lg, n0, lane);
        st.prefetch();
    };
    if constexpr (MODE == kGateUp) {
        const int e = expert(z);
        for (int c0 = 0; c0 < ng && e >= 0; c0 += int4::kStage) {
            const int nc = min(int4::kStage, ng - c0);
            // unit u: group u / 2 of the stage, of the gate (u even) or the up matrix
            auto unit = [&](int k, int u) {
                if (u < 2 * nc) load(k, k & 1, e, g0 + c0 + (u >> 1));
            };
            prefetch(0, e, g0 + c0);
            prefetch(1, e, g0 + c0);
            row.stage(a0 + (size_t)c0 * kGS, nc, lane);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) unit(k, k);
            float acc[2][2][4];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[m][b][c] = 0.0f;
            for (int u0 = 0; u0 < 2 * nc; u0 += kAhead)
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    if (u0 + k >= 2 * nc) break;
                    row.group(w[k], sc[k], 1.0f, (u0 + k) >> 1, lane, acc[k & 1]);
                    unit(k, u0 + k + kAhead);
                }
            for (unsigned left = row.left(); left; left &= left - 1) {
                const int i = c0 + (__ffs(left) - 1) / 2;
#pragma unroll 1
                for (int m = 0; m < 2; ++m) {
                    st.seek(m ? p.B1 : p.B0, m ? p.S1 : p.S0, p.N, e * G + g0 + i, n0, lane);
                    if (m) row.left_out(st, a0 + (size_t)i * kGS, 1.0f, lane, acc[1]);
                    else row.left_out(st, a0 + (size_t)i * kGS, 1.0f, lane, acc[0]);
                }
            }
            row.finish(acc[0], total[0]);
            row.finish(acc[1], total[NM - 1]);
        }
    } else {
        // the token's experts side by side: a group's expert changes every G groups
        int lg = g0 % G, slot = z * p.topk + g0 / G, e = ng > 0 ? expert(slot) : -1;
        float f = ng > 0 ? DT::tof(p.RW[slot]) : 0.0f;
        for (int c0 = 0; c0 < ng; c0 += int4::kStage) {
            const int nc = min(int4::kStage, ng - c0);
            auto unit = [&](int k, int u) {
                if (u >= nc) return;
                if (lg == G) {
                    lg = 0;
                    ++slot;
                    e = expert(slot);
                    f = DT::tof(p.RW[slot]);
                }
                factor[k] = f;
                if (e >= 0) {
                    load(k, 0, e, lg);
                } else {  // contributes zero
#pragma unroll
                    for (int c = 0; c < 4; ++c) w[k][c] = make_uint4(0u, 0u, 0u, 0u);
                    sc[k] = make_uint2(0u, 0u);
                    factor[k] = 0.0f;
                }
                ++lg;
            };
            if (e >= 0 && lg < G) prefetch(0, e, lg);  // (the next chunk may start at an expert's end)
            row.stage(a0 + (size_t)c0 * kGS, nc, lane);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) unit(k, k);
            float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            for (int u0 = 0; u0 < nc; u0 += kAhead)
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    if (u0 + k >= nc) break;
                    row.group(w[k], sc[k], factor[k], u0 + k, lane, acc);
                    unit(k, u0 + k + kAhead);
                }
            for (unsigned left = row.left(); left; left &= left - 1) {
                const int i = c0 + (__ffs(left) - 1) / 2, at = z * p.topk + (g0 + i) / G, e1 = p.ids[at];
                if (e1 < 0 || e1 >= p.E) continue;
                st.seek(p.B0, p.S0, p.N, e1 * G + (g0 + i) % G, n0, lane);
                row.left_out(st, a0 + (size_t)i * kGS, DT::tof(p.RW[at]), lane, acc);
            }
            row.finish(acc, total[0]);
        }
    }
    if ((lane & 3) == 0) {
#pragma unroll
        for (int m = 0; m < NM; ++m)
            *reinterpret_cast<float4 *>(&red[warp][m][lane]) =
                make_float4(total[m][0], total[m][1], total[m][2], total[m][3]);
    }
    if (bad_id && lane == 0) atomicOr(&tc::g_device_error, 2u);
    pdl_launch_dependents();
    __syncthreads();
    if (warp != 0) return;
    float v[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
        v[m] = 0.0f;
        for (int w = 0; w < W; ++w) v[m] += red[w][m][lane];
    }
    const int n = n0 + lane;
    if (n < p.N) p.out[(size_t)z * p.N + n] = DT::fromf(MODE == kGateUp ? epi<1>(v[0], v[NM - 1]) : v[0]);
}

template <int W, int MODE, class DT>
cudaError_t launch_w(const MParams &p, int rows, cudaStream_t st) {
    auto kern = moe_decode_int4_kernel<W, MODE, DT>;
    const int all = (MODE == kGateUp ? 1 : p.topk) * (p.K / kGS);
    const size_t smem = (size_t)W * int4::DigitRow<DT>::bytes((all + W - 1) / W);  // <= 67 KB
    const cudaError_t e = ensure_smem(kern, smem);
    if (e != cudaSuccess) return e;
    return launch_kernel(kern, dim3((unsigned)p.strips * (unsigned)rows), dim3(W * 32), smem, st, p);
}

// 8 warps split K while the CTAs fill the SMs less than twice, else 4, whose longer ranges spend
// less on their ends: gate_up (K 2048, N 768, top-8) 1 token 6.2 against 7.3 us, 2 tokens 10.1
// against 8.6, 9 tokens 31.2 against 25.3; down_sum 4 tokens 8.9 against 11.6, 9 tokens 16.9
// against 15.4.
template <int MODE>
cudaError_t launch(const MParams &p, int rows, int sms, int dtype, cudaStream_t st) {
    const bool many = (long long)rows * p.strips >= 2LL * sms;
    if (dtype == TERNOCL_BF16)
        return many ? launch_w<4, MODE, BF16>(p, rows, st) : launch_w<8, MODE, BF16>(p, rows, st);
    return many ? launch_w<4, MODE, F16>(p, rows, st) : launch_w<8, MODE, F16>(p, rows, st);
}

}  // namespace

cudaError_t moe_decode_gate_up_int4_launch(const int *ids, const void *X, const uint32_t *Bg, const void *Sg,
                                           const uint32_t *Bu, const void *Su, void *H, int G, int N, int K, int topk,
                                           int E, int dtype, int sms, cudaStream_t st) {
    const MParams p{ids, (const uint16_t *)X, Bg, Bu, (const uint16_t *)Sg, (const uint16_t *)Su, nullptr,
                    (uint16_t *)H, N, K, topk, E, (N + kCols - 1) / kCols};
    return launch<kGateUp>(p, G, sms, dtype, st);
}

cudaError_t moe_decode_down_sum_int4_launch(const int *ids, const void *H, const void *RW, const uint32_t *B,
                                            const void *S, void *O, int T, int N, int K, int topk, int E, int dtype,
                                            int sms, cudaStream_t st) {
    const MParams p{ids, (const uint16_t *)H, B, B, (const uint16_t *)S, (const uint16_t *)S, (const uint16_t *)RW,
                    (uint16_t *)O, N, K, topk, E, (N + kCols - 1) / kCols};
    return launch<kDownSum>(p, T, sms, dtype, st);
}

cudaError_t read_device_error_moe_decode_int4(unsigned *out, int reset) { return tc::read_tu_error(out, reset); }

}  // namespace ternocl
