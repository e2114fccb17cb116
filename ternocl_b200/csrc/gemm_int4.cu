// int4 GEMM on the 5th-generation tensor cores (tcgen05), dense and grouped by expert:
//
//   C[m,n] = DT(epi( sum_g S[g,n] * D_g[m,n] )),   D_g[m,n] = sum_{k in g} A[m,k] * code(k,n)
//
// A weight code * S does not fit DT (3 + 8 or 3 + 11 significant bits), so a GEMM on
// dequantised weights would round every weight.  Here the codes alone are the MMA operand
// (exact in DT), every 128-row group has an accumulator of its own in TMEM, and its sums are
// scaled by S and added up in fp32 registers: the GEMV's arithmetic, nothing rounded before
// the output.
//
// The weights are the MMA's M operand (128 columns n of C) and the activation rows its N
// operand (up to MT): then a TMEM lane is a column n, a thread scales its whole lane by one
// S[g,n], the N extent follows the rows that are there, and the accumulated tile's rows are
// stored 32 consecutive columns per warp.
//
// CTA: 128 columns x MT rows, groups [G sk/SK, G (sk+1)/SK) of a K split over a
// thread-block cluster.  Roles:
//   warp 0      TMA producer: per group two boxes of A (MT rows x 64, 128-byte swizzle) and
//               one box of packed words (16 word rows x 128 columns);
//   warp 1      TMEM allocation and the MMA issuer: per group 2 x 4 tcgen05.mma kind::f16
//               (M=128, N=rows rounded up to 16, K=16) into one of kAccBufs accumulators;
//   4 NT warps  decode (NT teams of 4): a team turns every NT-th half group (8 word rows) into
//               a K=64 slice of the M operand, MN-major: one lane makes one 8 x 8 core
//               matrix out of 8 words (8 columns of one word row);
//   NP warps    promotion: tcgen05.ld of a finished group, acc += S * D_g, then the epilogue.
// With SK > 1 the CTAs of a cluster leave their sums in shared memory and each adds up a
// share of the rows in split order over distributed shared memory (deterministic).
// Every mbarrier wait is bounded (tc::mbar_wait); on a timeout the roles skip ahead, the
// producer waits (bounded) for its copies in flight, and TMEM is freed.
#include <cuda.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "gemv_common.cuh"
#include "int4_common.cuh"
#include "launch.h"
#include "tc_common.cuh"

namespace ternocl {
namespace gemm4 {

constexpr int BN = 128;                        // columns of C per CTA (the MMA's M)
constexpr int kHalf = 64;                      // K rows of a decode stage
constexpr int kDecLBO = 128;                   // next 8 K rows
constexpr int kDecSBO = kHalf / 8 * 128 + 16;  // next 8 columns; the pad spreads the stores over the banks
constexpr int kDecStageBytes = BN / 8 * kDecSBO;
constexpr int kPackBytes = int4::kWordsPerGroup * BN * 4;  // 8 KB
constexpr int kMetaTile = 128;                 // rows of a tile in moe_route's meta

template <int MT_>
struct Cfg {
    static constexpr int MT = MT_;
    static constexpr int NT = MT >= 128 ? 2 : 1;         // decode teams of 4 warps
    static constexpr int NP = MT >= 128 ? 8 : 4;         // promotion warps
    static constexpr int kWarps = 2 + 4 * NT + NP;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kCols = MT * 4 / NP;            // accumulator columns per promotion thread
    static constexpr int kLoads = 3;
    static constexpr int kDecs = MT >= 128 ? 5 : 3;
    static constexpr int kAccBufs = MT >= 128 ? 4 : 2;
    static constexpr int kTmemCols = MT * kAccBufs;
    static constexpr int kABytes = MT * kGS * 2;
    static constexpr int kCtasPerSm = MT >= 128 ? 1 : 2;
    // shared memory: decoded stages first, then 1024-byte aligned A stages
    static constexpr int dec = 0;
    static constexpr int a = (kDecs * kDecStageBytes + 1023) / 1024 * 1024;
    static constexpr int pack = a + kLoads * kABytes;
    static constexpr int bars = pack + kLoads * kPackBytes;
    static constexpr int total = bars + 256 + 1024;  // + alignment slack
    static_assert(total <= 227 * 1024, "shared memory");
    static_assert(MT * BN * 4 <= bars, "the split's sums reuse the stages");
    static_assert(kTmemCols * kCtasPerSm <= 512, "TMEM");
};

struct Params {
    const uint16_t *S;
    void *C;
    const uint16_t *Other;
    const void *Bias;
    int M, N, K, SK;
    const int *meta;  // grouped: [E+1 row offsets | E+1 row-tile offsets], else null
    int E;
};

// 8 words (columns 8nb..8nb+7 of one word row) -> the core matrix rows out[r] (K row r, the 8
// columns as 4 half2): two columns' halves side by side decode together
template <class DT>
__device__ __forceinline__ void decode8(const uint4 w0, const uint4 w1, uint4 (&out)[8]) {
    const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    uint32_t d[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t z = __byte_perm(w[2 * i], w[2 * i + 1], h ? 0x7632u : 0x5410u);  // rows 4h .. 4h+3
            const uint32_t y = z >> 8;
            d[i][4 * h] = int4::low_pair<DT>(z);
            d[i][4 * h + 1] = int4::high_pair<DT>(z);
            d[i][4 * h + 2] = int4::low_pair<DT>(y);
            d[i][4 * h + 3] = int4::high_pair<DT>(y);
        }
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) out[r] = make_uint4(d[0][r], d[1][r], d[2][r], d[3][r]);
}

__device__ __forceinline__ float ld_dsmem_f32(uint32_t local_addr, uint32_t rank) {
    uint32_t remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(local_addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(remote));
    return v;
}

// element (m, n) through the epilogue
template <class DT, int POSTOP, bool OUT_F32>
__device__ __forceinline__ void store(const Params &p, int m, int n, float v) {
    const size_t i = (size_t)m * p.N + n;
    v = epi<POSTOP, OUT_F32>(v, epi_in<DT, POSTOP, OUT_F32>(p.Other, p.Bias, i, n));
    if constexpr (OUT_F32) reinterpret_cast<float *>(p.C)[i] = v;
    else reinterpret_cast<uint16_t *>(p.C)[i] = DT::fromf(v);
}

template <int MT, class DT, int POSTOP, bool OUT_F32>
__global__ void __launch_bounds__(Cfg<MT>::kThreads, Cfg<MT>::kCtasPerSm)
    gemm_int4_kernel(const Params p, const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB) {
    using C = Cfg<MT>;
    extern __shared__ __align__(1024) char smem_raw[];
    char *smem = smem_raw + ((1024u - (tc::smem_addr(smem_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n0 = blockIdx.x * BN;
    const int G = p.K / kGS;
    int m0 = blockIdx.y * MT, m_end = p.M, expert = 0;
    if (p.meta) {
        // the expert of this 128-row tile: the last one whose first tile is <= it
        pdl_wait();
        constexpr int kSub = MT < kMetaTile ? kMetaTile / MT : 1;
        const int tile = blockIdx.y / kSub, E = p.E;
        if (tile >= p.meta[2 * E + 1]) return;
        int lo = 0, hi = E - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (p.meta[E + 1 + mid] <= tile) lo = mid;
            else hi = mid - 1;
        }
        expert = lo;
        m0 = p.meta[lo] + (tile - p.meta[E + 1 + lo]) * kMetaTile + (blockIdx.y % kSub) * MT;
        m_end = p.meta[lo + 1];
        if (m0 >= m_end) return;
    }
    const int rows = min(MT, m_end - m0);
    const int g0 = (int)((long long)G * blockIdx.z / p.SK), g1 = (int)((long long)G * (blockIdx.z + 1) / p.SK);
    const int ng = g1 - g0;

    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::bars);
    uint64_t *load_empty = full + C::kLoads;
    uint64_t *dec_full = load_empty + C::kLoads;
    uint64_t *dec_empty = dec_full + C::kDecs;
    uint64_t *acc_full = dec_empty + C::kDecs;
    uint64_t *acc_empty = acc_full + C::kAccBufs;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + C::kAccBufs);
    static_assert((2 * C::kLoads + 2 * C::kDecs + 2 * C::kAccBufs) * 8 + 4 <= 256, "barriers");

    if (tid == 0) {
        for (int s = 0; s < C::kLoads; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&load_empty[s], 1 + 8);  // the MMAs, and 4 decode warps for each half
        }
        for (int d = 0; d < C::kDecs; ++d) {
            tc::mbar_init(&dec_full[d], 4);
            tc::mbar_init(&dec_empty[d], 1);
        }
        for (int b = 0; b < C::kAccBufs; ++b) {
            tc::mbar_init(&acc_full[b], 1);
            tc::mbar_init(&acc_empty[b], C::NP);
        }
        tc::fence_mbar_init();
    }
    if (warp == 1) tc::tmem_alloc(tmem_slot, C::kTmemCols);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    // promotion threads: column n (TMEM lane) and rows jbase .. jbase + kCols - 1 of the tile
    const int pw = warp - (2 + 4 * C::NT);
    const int quad = warp & 3;
    const int jbase = pw >= 4 ? C::kCols : 0;
    const int n = n0 + 32 * quad + lane;
    float acc[C::kCols];

    if (warp == 0) {
        // ---------------- producer ----------------
        if (lane == 0) {
            if (!p.meta) pdl_wait();
            int issued = 0;
            for (int i = 0; i < ng; ++i) {
                const int s = i % C::kLoads;
                if (i >= C::kLoads && !tc::mbar_wait(&load_empty[s], ((i / C::kLoads) - 1) & 1)) break;
                tc::mbar_expect_tx(&full[s], C::kABytes + kPackBytes);
                const int grp = g0 + i;
                tc::tma_load_2d(smem + C::pack + s * kPackBytes, &tmB, n0,
                                expert * (p.K / int4::kRowsPerWord) + grp * int4::kWordsPerGroup, &full[s]);
                char *a = smem + C::a + s * C::kABytes;
                tc::tma_load_2d(a, &tmA, grp * kGS, m0, &full[s]);
                tc::tma_load_2d(a + C::kABytes / 2, &tmA, grp * kGS + kHalf, m0, &full[s]);
                ++issued;
            }
            // copies still in flight must land before the block can exit
            for (int i = issued < C::kLoads ? 0 : issued - C::kLoads; i < issued; ++i)
                tc::mbar_wait(&full[i % C::kLoads], (i / C::kLoads) & 1);
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (lane == 0) {
            // M operand MN-major (bit 15), N operand K-major
            const uint32_t idesc = tc::idesc_f16(DT::kBF16, BN, (rows + 15) & ~15) | (1u << 15);
            bool ok = true;
            for (int i = 0; i < ng && ok; ++i) {
                const int s = i % C::kLoads, b = i % C::kAccBufs;
                if (!tc::mbar_wait(&full[s], (i / C::kLoads) & 1)) break;
                if (i >= C::kAccBufs && !tc::mbar_wait(&acc_empty[b], ((i / C::kAccBufs) - 1) & 1)) break;
                const uint32_t act = tc::smem_addr(smem + C::a + s * C::kABytes);
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    const int x = 2 * i + h, d = x % C::kDecs;
                    if (!tc::mbar_wait(&dec_full[d], (x / C::kDecs) & 1)) {
                        ok = false;
                        break;
                    }
                    tc::fence_after_sync();
                    const uint32_t w = tc::smem_addr(smem + C::dec + d * kDecStageBytes);
#pragma unroll
                    for (int kk = 0; kk < kHalf / 16; ++kk)
                        tc::mma_ss_f16(tmem + b * MT, tc::sdesc_kmajor_noswz(w + kk * 2 * kDecLBO, kDecLBO, kDecSBO),
                                       tc::sdesc_kmajor_sw128(act + h * (C::kABytes / 2) + kk * 32), idesc,
                                       (h | kk) != 0);
                    tc::mma_commit(&dec_empty[d]);
                }
                if (!ok) break;
                tc::mma_commit(&load_empty[s]);
                tc::mma_commit(&acc_full[b]);
            }
        }
    } else if (warp < 2 + 4 * C::NT) {
        // ---------------- decode ----------------
        const int team = (warp - 2) >> 2;
        const int task = ((warp - 2) & 3) * 32 + lane;  // 8 word rows x 16 column blocks
        const int wr = task >> 4, nb = task & 15;
        // two 16-byte chunks per lane, read in the other order by every second four lanes, so
        // that both reads of a quarter-warp touch 8 distinct 16-byte bank groups
        const int sw = (nb >> 2) & 1;
        for (int x = team; x < 2 * ng; x += C::NT) {
            const int i = x >> 1, s = i % C::kLoads, d = x % C::kDecs;
            if (!tc::mbar_wait(&full[s], (i / C::kLoads) & 1)) break;
            const uint4 *src = reinterpret_cast<const uint4 *>(smem + C::pack + s * kPackBytes +
                                                               ((x & 1) * 8 + wr) * (BN * 4) + nb * 32);
            const uint4 c0 = src[sw], c1 = src[sw ^ 1];
            uint4 out[8];
            decode8<DT>(sw ? c1 : c0, sw ? c0 : c1, out);
            if (x >= C::kDecs && !tc::mbar_wait(&dec_empty[d], ((x / C::kDecs) - 1) & 1)) break;
            char *dst = smem + C::dec + d * kDecStageBytes + nb * kDecSBO + wr * 128;
#pragma unroll
            for (int r = 0; r < 8; ++r) *reinterpret_cast<uint4 *>(dst + r * 16) = out[r];
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive(&dec_full[d]);
                tc::mbar_arrive(&load_empty[s]);
            }
        }
    } else {
        // ---------------- promotion ----------------
#pragma unroll
        for (int j = 0; j < C::kCols; ++j) acc[j] = 0.0f;
        const bool nok = n < p.N;
        const uint16_t *sp = p.S + ((size_t)expert * G + g0) * p.N + (nok ? n : 0);
        constexpr int kAhead = 4;  // scales are requested this many groups early
        float sc[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) sc[k] = k < ng ? DT::tof(__ldg(sp + (size_t)k * p.N)) : 0.0f;
        for (int i = 0; i < ng; ++i) {
            const int b = i % C::kAccBufs;
            const float s = sc[0];
#pragma unroll
            for (int k = 0; k + 1 < kAhead; ++k) sc[k] = sc[k + 1];
            sc[kAhead - 1] = i + kAhead < ng ? DT::tof(__ldg(sp + (size_t)(i + kAhead) * p.N)) : 0.0f;
            if (!tc::mbar_wait(&acc_full[b], (i / C::kAccBufs) & 1)) break;
            tc::fence_after_sync();
            const uint32_t taddr = tmem + ((uint32_t)(32 * quad) << 16) + (uint32_t)(b * MT + jbase);
#pragma unroll
            for (int c = 0; c < C::kCols; c += 16) {
                if (jbase + c < rows) {  // warp-uniform
                    float v[16];
                    tc::tmem_ld<16>(taddr + c, v);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[c + j] = fmaf(v[j], s, acc[c + j]);
                }
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&acc_empty[b]);
        }
        if (p.SK == 1) {
            pdl_wait();
            if (nok) {
#pragma unroll
                for (int j = 0; j < C::kCols; ++j)
                    if (jbase + j < rows) store<DT, POSTOP, OUT_F32>(p, m0 + jbase + j, n, acc[j]);
            }
            pdl_launch_dependents();
        }
    }
    if (p.SK > 1) {
        // the split's sums [rows][128] in the stages, which the MMAs have finished reading
        __syncthreads();
        float *part = reinterpret_cast<float *>(smem);
        if (warp >= 2 + 4 * C::NT) {
#pragma unroll
            for (int j = 0; j < C::kCols; ++j)
                if (jbase + j < rows) part[(jbase + j) * BN + 32 * quad + lane] = acc[j];
        }
        gemv::cluster_sync_all();
        pdl_wait();
        const int r0 = rows * (int)blockIdx.z / p.SK, r1 = rows * ((int)blockIdx.z + 1) / p.SK;
        for (int x = r0 * BN + tid; x < r1 * BN; x += C::kThreads) {
            const uint32_t la = tc::smem_addr(part + x);
            float v = 0.0f;
            for (int r = 0; r < p.SK; ++r) v += ld_dsmem_f32(la, (uint32_t)r);
            if (n0 + x % BN < p.N) store<DT, POSTOP, OUT_F32>(p, m0 + x / BN, n0 + x % BN, v);
        }
        pdl_launch_dependents();
        gemv::cluster_sync_all();  // every CTA's sums stay until all have read them
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, C::kTmemCols);
    }
}

template <int MT>
cudaError_t launch(const GemvArgs &a, const int *meta, int E) {
    using C = Cfg<MT>;
    CUtensorMap mapA, mapB;
    cudaError_t e = tc::make_map_sw128(
        &mapA, a.A, a.dtype == TERNOCL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
        a.M, a.K, MT);
    if (e != cudaSuccess) return e;
    e = tc::make_map_plain(&mapB, a.B, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, (meta ? E : 1) * (a.K / int4::kRowsPerWord),
                           a.N, int4::kWordsPerGroup, BN);
    if (e != cudaSuccess) return e;
    const Params p{(const uint16_t *)a.S, a.C, (const uint16_t *)a.Other, a.Bias, a.M, a.N, a.K, a.SK, meta, E};
    return dispatch_epilogue<GemvArgs>(a, [&](auto dt, auto po, auto of) -> cudaError_t {
        using DT = typename decltype(dt)::type;
        auto kern = gemm_int4_kernel<MT, DT, decltype(po)::value, decltype(of)::value>;
        cudaError_t err = ensure_smem(kern, C::total);
        if (err != cudaSuccess) return err;
        const int strips = (a.N + BN - 1) / BN;
        // grouped: every expert adds at most one partial 128-row tile
        const int tiles = meta ? ((a.M + kMetaTile - 1) / kMetaTile + E) * (MT < kMetaTile ? kMetaTile / MT : 1)
                               : (a.M + MT - 1) / MT;
        return launch_kernel_cluster(kern, dim3(strips, tiles, a.SK), dim3(C::kThreads), (size_t)C::total, a.stream,
                                     dim3(1, 1, a.SK), p, mapA, mapB);
    });
}

}  // namespace gemm4

cudaError_t int4_gemm_launch(const GemvArgs &a, int sms, const int *meta, int E) {
    GemvArgs b = a;
    // activation rows per CTA: what the rows (grouped: an expert's average) fill
    const long long per = meta ? (a.M + E - 1) / E : a.M;
    const int MT = per <= 32 ? 32 : per <= 64 ? 64 : 128;
    // K split over a cluster while the tiles leave SMs without work
    const long long tiles = (long long)((a.N + gemm4::BN - 1) / gemm4::BN) * ((a.M + MT - 1) / MT);
    int sk = 1;
    if (!meta)
        while (sk < 8 && 2 * sk <= a.K / kGS && tiles * 2 * sk <= sms) sk *= 2;
    b.SK = sk;
    return MT == 32 ? gemm4::launch<32>(b, meta, E) : MT == 64 ? gemm4::launch<64>(b, meta, E)
                                                               : gemm4::launch<128>(b, meta, E);
}

cudaError_t read_device_error_gemm_int4(unsigned *out, int reset) { return tc::read_tu_error(out, reset); }

}  // namespace ternocl
