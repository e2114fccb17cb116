// int4 MoE decode GEMVs: moe_decode.cu's products with 4-bit weights (int4_common.cuh),
//
//   gate_up   H[g, n] = DT(silu(x_t . gate_e[:, n]) * (x_t . up_e[:, n])),  x_t = X[g / topk]
//   down_sum  O[t, n] = DT(sum_j RW[g] * (H[g] . down_e[:, n])),  g = t*topk + j
//
// with e = ids[g] and every expert's weights stacked: B [E, K/8, N], S [E, K/128, N].
//
// A CTA owns 32 columns of one routed row (gate_up: of both matrices, whose dots meet in
// the CTA for the SwiGLU; down_sum: of one token, its K running over the topk experts) over
// the whole K; its W warps split the 128-row groups and are summed in warp order.  A warp
// streams its groups' words (16 rows x 128 bytes) and scales through a ring in shared memory
// and turns its activations into int8 digit planes, kChunk groups at a time: a chunk has one
// exponent, and its sums are scaled back into the warp's totals at its end, so the shared
// memory does not grow with K.  The dots are mma.sync m16n8k32 s8 x s8, three of the eight
// n-columns being the digit planes of the row.
//
// An expert id outside [0, E) contributes zero and sets bit 1 of the device error word.
#include <cuda_runtime.h>

#include "common.cuh"
#include "gemv_common.cuh"
#include "int4_common.cuh"
#include "launch.h"
#include "tc_common.cuh"

namespace ternocl {

namespace {

constexpr int kCols = 32;
constexpr int kRowBytes = kCols * 4;
constexpr int kWordBytes = int4::kWordsPerGroup * kRowBytes;  // 2 KB
constexpr int kScaleBytes = kCols * 2;
constexpr int kStageBytes = kWordBytes + kScaleBytes;
constexpr int kRingBytes = gemv::kStages * kStageBytes;
constexpr int kChunk = 8;  // groups per digit staging
// 128 bytes per group; the 16 more put the planes of two neighbouring lanes' rows on the
// two 16-byte halves of every 32 bytes (conflict-free 16-byte reads)
constexpr int kPlane = kChunk * 128 + 16;

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

template <int W, int MODE>
constexpr size_t smem_bytes() {
    return (size_t)W * (kRingBytes + 3 * kPlane + kMats<MODE> * kCols * 4);
}

template <int W, int MODE, class DT>
__global__ void __launch_bounds__(W * 32) moe_decode_int4_kernel(const MParams p) {
    constexpr int NM = kMats<MODE>;
    extern __shared__ __align__(128) char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    const int z = blockIdx.x / p.strips;  // routed row (gate_up) or token (down_sum)
    const int n0 = (blockIdx.x - z * p.strips) * kCols;
    const int G = p.K / kGS;
    const int ng = MODE == kGateUp ? 2 * G : p.topk * G;
    const int wg0 = (int)((long long)ng * warp / W), nwg = (int)((long long)ng * (warp + 1) / W) - wg0;
    char *ring = smem + warp * kRingBytes;
    char *planes = smem + W * kRingBytes + warp * 3 * kPlane;
    float *red = reinterpret_cast<float *>(smem + W * (kRingBytes + 3 * kPlane));  // [W][NM][32]

    pdl_wait();  // ids and activations come from the kernels before

    // group grp -> its matrix (gate_up) or expert slot (down_sum) and its group there
    auto part = [&](int grp, int &lg) {
        const int i = grp / G;
        lg = grp - i * G;
        return i;
    };
    auto expert = [&](int slot) {
        const int e = p.ids[MODE == kGateUp ? z : z * p.topk + slot];
        return e >= 0 && e < p.E ? e : -1;
    };
    auto act = [&](int grp) -> const uint16_t * {
        if (MODE == kGateUp) {
            int lg;
            part(grp, lg);
            return p.A + (size_t)(z / p.topk) * p.K + (size_t)lg * kGS;
        }
        return p.A + (size_t)z * p.topk * p.K + (size_t)grp * kGS;  // the token's rows side by side
    };

    const int col = n0 + 4 * (lane & 7);  // N % 16 == 0: 4-column pieces are whole
    const bool copies = col < p.N;
    const bool scales = lane < 4 && n0 + 8 * lane < p.N;
    int issued = 0;
    auto issue = [&]() {
        if (issued < nwg) {
            char *st = ring + (issued & (gemv::kStages - 1)) * kStageBytes;
            int lg;
            const int i = part(wg0 + issued, lg);
            const int e = expert(i);
            if (e >= 0) {
                const uint32_t *B = (MODE == kGateUp && i ? p.B1 : p.B0) +
                                    ((size_t)e * (p.K / int4::kRowsPerWord) + lg * int4::kWordsPerGroup) * p.N;
                const uint16_t *S = (MODE == kGateUp && i ? p.S1 : p.S0) + ((size_t)e * G + lg) * p.N;
                if (copies) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int r = 4 * c + (lane >> 3);
                        gemv::cp_async16(st + r * kRowBytes + 16 * (lane & 7), B + (size_t)r * p.N + col);
                    }
                }
                if (scales) gemv::cp_async16(st + kWordBytes + 16 * lane, S + n0 + 8 * lane);
            }
        }
        gemv::cp_async_commit();
        ++issued;
    };
#pragma unroll
    for (int i = 0; i < gemv::kStages - 1; ++i) issue();

    float total[NM][2][4];
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c) total[m][b][c] = 0.0f;
    const char *bsrc = g < 3 ? planes + g * kPlane + t * 32 : nullptr;
    bool bad_id = false;

    for (int c0 = 0; c0 < nwg; c0 += kChunk) {
        const int nc = min(kChunk, nwg - c0);
        // ---- the chunk's activations -> digit planes (16 word rows per group) ----
        uint32_t mx = 0;
        uint4 v[kChunk / 2];
#pragma unroll
        for (int i = 0; i < kChunk / 2; ++i) {
            const int u = 32 * i + lane;  // word row of the chunk
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (u < 16 * nc) v[i] = __ldg(reinterpret_cast<const uint4 *>(act(wg0 + c0 + u / 16) + 8 * (u % 16)));
            mx = max(mx, int4::absmax_bits(v[i]));
        }
        mx = __reduce_max_sync(0xffffffffu, mx);
        const int e = digit::exponent_for<DT>(mx);
        const float rs = int4::inverse_scale<DT>(mx, e);
        __syncwarp();  // the previous chunk's planes have been read
#pragma unroll
        for (int i = 0; i < kChunk / 2; ++i) {
            const int u = 32 * i + lane;
            if (u < 16 * nc) {
                uint2 d[3];
                int4::word_digits<DT>(v[i], e, d);
                char *dst = planes + (u / 16) * 128 + (u & 3) * 32 + ((u >> 2) & 3) * 8;
#pragma unroll
                for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2 *>(dst + k * kPlane) = d[k];
            }
        }
        __syncwarp();

        float acc[NM][2][4];
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[m][b][c] = 0.0f;

        for (int i = c0; i < c0 + nc; ++i) {
            gemv::cp_async_wait<gemv::kStages - 2>();
            __syncwarp();  // the lanes' copies of this stage are visible to the whole warp
            const char *st = ring + (i & (gemv::kStages - 1)) * kStageBytes;
            int lg;
            const int slot = part(wg0 + i, lg);
            const int ex = expert(slot);
            bad_id |= ex < 0;
            if (ex >= 0) {
                float gf = 1.0f;
                if (MODE == kDownSum) gf = DT::tof(p.RW[z * p.topk + slot]);
                int32_t d[2][4];
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int c = 0; c < 4; ++c) d[b][c] = (int32_t)digit::kMagicBits;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4 b = make_uint4(0u, 0u, 0u, 0u);
                    if (bsrc) b = *reinterpret_cast<const uint4 *>(bsrc + (i - c0) * 128 + 16 * h);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint4 w = *reinterpret_cast<const uint4 *>(st + (8 * h + 4 * q + t) * kRowBytes + 16 * g);
                        const uint32_t be = q ? b.z : b.x, bo = q ? b.w : b.y;
                        int4::imma(d[0], int4::even_rows(w.x), int4::even_rows(w.y), int4::odd_rows(w.x),
                                   int4::odd_rows(w.y), be, bo);
                        int4::imma(d[1], int4::even_rows(w.z), int4::even_rows(w.w), int4::odd_rows(w.z),
                                   int4::odd_rows(w.w), be, bo);
                    }
                }
                const uint2 s4 = *reinterpret_cast<const uint2 *>(st + kWordBytes + 8 * g);
                const float s[4] = {DT::tof((uint16_t)(s4.x & 0xFFFFu)) * gf, DT::tof((uint16_t)(s4.x >> 16)) * gf,
                                    DT::tof((uint16_t)(s4.y & 0xFFFFu)) * gf, DT::tof((uint16_t)(s4.y >> 16)) * gf};
#pragma unroll
                for (int m = 0; m < NM; ++m) {
                    if (NM > 1 && m != slot) continue;
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            acc[m][b][c] =
                                fmaf(__int_as_float(d[b][c]) - digit::kMagic, s[2 * b + (c >> 1)], acc[m][b][c]);
                }
            }
            __syncwarp();  // every lane is done with this stage before it is refilled
            issue();
        }
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int c = 0; c < 4; ++c) total[m][b][c] = fmaf(acc[m][b][c], rs, total[m][b][c]);
    }
    gemv::cp_async_wait<0>();
    if (bad_id && lane == 0) atomicOr(&tc::g_device_error, 2u);
    pdl_launch_dependents();
    __syncwarp();

    // ---- digit planes -> column values of this warp: tb[mat][plane][col] in its ring ----
    float(*tb)[8][kCols] = reinterpret_cast<float(*)[8][kCols]>(ring);
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c) tb[m][2 * t + (c & 1)][4 * g + 2 * b + (c >> 1)] = total[m][b][c];
    __syncwarp();
#pragma unroll
    for (int m = 0; m < NM; ++m)
        red[(warp * NM + m) * kCols + lane] =
            (tb[m][0][lane] + 256.0f * tb[m][1][lane]) + 65536.0f * tb[m][2][lane];
    __syncthreads();
    if (warp != 0) return;
    float v[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
        v[m] = 0.0f;
        for (int w = 0; w < W; ++w) v[m] += red[(w * NM + m) * kCols + lane];
    }
    const int n = n0 + lane;
    if (n < p.N) p.out[(size_t)z * p.N + n] = DT::fromf(MODE == kGateUp ? epi<1>(v[0], v[NM - 1]) : v[0]);
}

template <int W, int MODE, class DT>
cudaError_t launch_w(const MParams &p, int rows, cudaStream_t st) {
    auto kern = moe_decode_int4_kernel<W, MODE, DT>;
    constexpr size_t smem = smem_bytes<W, MODE>();
    cudaError_t e = ensure_smem(kern, smem);
    if (e != cudaSuccess) return e;
    return launch_kernel(kern, dim3((unsigned)p.strips * (unsigned)rows), dim3(W * 32), smem, st, p);
}

template <int MODE>
cudaError_t launch(const MParams &p, int rows, int dtype, cudaStream_t st) {
    const int ng = (MODE == kGateUp ? 2 : p.topk) * (p.K / kGS);
    if (dtype == TERNOCL_BF16)
        return ng >= 16 ? launch_w<8, MODE, BF16>(p, rows, st) : launch_w<4, MODE, BF16>(p, rows, st);
    return ng >= 16 ? launch_w<8, MODE, F16>(p, rows, st) : launch_w<4, MODE, F16>(p, rows, st);
}

}  // namespace

cudaError_t moe_decode_gate_up_int4_launch(const int *ids, const void *X, const uint32_t *Bg, const void *Sg,
                                           const uint32_t *Bu, const void *Su, void *H, int G, int N, int K, int topk,
                                           int E, int dtype, cudaStream_t st) {
    const MParams p{ids, (const uint16_t *)X, Bg, Bu, (const uint16_t *)Sg, (const uint16_t *)Su, nullptr,
                    (uint16_t *)H, N, K, topk, E, (N + kCols - 1) / kCols};
    return launch<kGateUp>(p, G, dtype, st);
}

cudaError_t moe_decode_down_sum_int4_launch(const int *ids, const void *H, const void *RW, const uint32_t *B,
                                            const void *S, void *O, int T, int N, int K, int topk, int E, int dtype,
                                            cudaStream_t st) {
    const MParams p{ids, (const uint16_t *)H, B, B, (const uint16_t *)S, (const uint16_t *)S, (const uint16_t *)RW,
                    (uint16_t *)O, N, K, topk, E, (N + kCols - 1) / kCols};
    return launch<kDownSum>(p, T, dtype, st);
}

cudaError_t read_device_error_moe_decode_int4(unsigned *out, int reset) { return tc::read_tu_error(out, reset); }

}  // namespace ternocl
