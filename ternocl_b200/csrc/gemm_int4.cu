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
// S[g,n], and the N extent follows the rows that are there.
//
// Persistent CTAs walk tiles of 128 columns x MT rows; a step is half a group (K = 64).  At
// MT = 256 two CTAs of a cluster work as a pair on 256 columns x 256 rows (cta_group::2):
// each holds its own columns' weights and half of the rows' activations, and every MMA
// reads both halves, so the activations cross from L2 once for 256 columns.  Roles:
//   warp 0      the activations of a step: TMA boxes of 64 rows x 64 (128-byte swizzle);
//   warp 1      the MMA issuer (of a pair: the first CTA's): per step 4 tcgen05.mma kind::f16
//               (M=128 a CTA, N=rows rounded up, K=16) into one of kAccBufs accumulators;
//   warp 2      the packed words of a step: one TMA box of 8 word rows x 128 columns;
//   warp 3      TMEM allocation, and with few rows the MMAs of every other group;
//   4 NT warps  decode, NT teams of 4 that take the steps in turn: one lane makes one 8 x 8 core
//               matrix of the M operand (MN-major) out of 8 words;
//   NP warps    promotion: tcgen05.ld of a finished group, acc += S * D_g (f32x2), and at the
//               tile's end the epilogue, while the other roles run on into the next tile.
// The tiles of the last round, when they would leave CTAs without work, are split along K over
// the CTAs of a cluster: these leave their sums in shared memory and each adds up a share of
// the rows in split order over distributed shared memory.
//
// What bounds it: for many rows the MMAs (1024 of ~1220 cycles a group at MT = 256; a single CTA
// per tile was bound by the latency of its activations, 36 KB a step: 1380 cycles) and at short K
// the epilogue, of which the other roles hide two groups; for few rows shared memory, which a
// decoded step crosses twice (48 KB, 375 cycles).  Chains of waits decided the rest: a step's
// decode takes ~1000 cycles from its words' arrival to the MMA, so NT teams keep NT steps in
// flight, every stage has one barrier that says "filled" and one that says "free", and the
// MMA issuer waits once per step.  Measured on B200 (bf16, CUDA graph): 14336x4096 M=2047 with
// a residual 193-204 us in runs of some ms, 222 us = 1080 TFLOP/s over a second of load (1605 MHz under
// the power cap; floor 140 us at the burst peak), 4096x4096 M=2048 56-62 us; few rows 5376x21504 M=32 33.6 us
// (9.5), M=64 40.9 (9.8), M=128 48.9 (17.2), M=512 112 (69); 4096x4096 M=64 12.0, M=512 24.3 (10.0); grouped
// 32768 rows x 768 x 2048 over 128 experts with SwiGLU 175 us (floor 60), 12.5 rows per expert 53, 24 62,
// 48 72 us (17.5, 18.8, 21.5).
// Every mbarrier wait is bounded (tc::mbar_wait); on a timeout the roles stop, the producers
// wait (bounded) for their copies in flight, and TMEM is freed.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "gemv_common.cuh"
#include "int4_common.cuh"
#include "launch.h"
#include "tc_common.cuh"

namespace ternocl {
namespace gemm4 {

constexpr int BN = 128;                        // columns of C per tile (the MMA's M)
constexpr int kStepK = 64;                     // K rows of a step
constexpr int kDecLBO = 128;                   // next 8 K rows
constexpr int kDecSBO = kStepK / 8 * 128 + 16; // next 8 columns; the pad spreads the stores over the banks
constexpr int kDecBytes = BN / 8 * kDecSBO;    // 16640
constexpr int kWordBytes = kStepK / int4::kRowsPerWord * BN * 4;  // 4 KB
constexpr int kMaxExperts = 1024;
// an epilogue block: 8 rows x 128 fp32 columns, the right half 16 words further on (a warp's
// 16 + 16 columns then lie in different banks)
constexpr int kOutRow = BN + 16, kOutRows = 8, kOutBytes = kOutRows * kOutRow * 4;

// Threads, rings and register shares by the rows of a tile; one CTA per SM.  kRegs*: setmaxnreg
// values (0: not used), whose sum over the warps stays within what the block launches with.
// Few rows leave shared memory for words, to cover the ~1.2 us that they take from HBM, and two
// MMA issuers, since a step's MMAs then take less than the ~330 cycles that one issuer spends on it.
//
// A wait for a barrier's parity tells a pass from the one before only for a role that sees every
// pass of the slot, or whose earlier waits imply the pass before.  One issuer does the steps in
// order, so a decode team at step x, which has waited for step x - NT's slot, knows that step
// x - 2 kSteps is done if NT <= kSteps.  Two issuers do not, so there every slot has one team
// and one issuer: kSteps and kWords are multiples of NT and kSteps of 4.
template <int MT_>
struct Cfg;
template <>
struct Cfg<256> {
    static constexpr int MT = 256, NT = 2, NP = 8, kSteps = 5, kWords = 6, kAccBufs = 2, kIssuers = 1;
    static constexpr int kRegsPromote = 168, kRegsOther = 48;
};
template <>
struct Cfg<128> {
    static constexpr int MT = 128, NT = 3, NP = 8, kSteps = 4, kWords = 16, kAccBufs = 4, kIssuers = 1;
    static constexpr int kRegsPromote = 112, kRegsOther = 64;
};
template <>
struct Cfg<64> {
    static constexpr int MT = 64, NT = 4, NP = 4, kSteps = 4, kWords = 28, kAccBufs = 4, kIssuers = 2;
    static constexpr int kRegsPromote = 112, kRegsOther = 72;
};
template <>
struct Cfg<32> {
    static constexpr int MT = 32, NT = 4, NP = 4, kSteps = 8, kWords = 12, kAccBufs = 4, kIssuers = 2;
    static constexpr int kRegsPromote = 0, kRegsOther = 0;
};

template <int MT>
struct Plan : Cfg<MT> {
    using C = Cfg<MT>;
    static constexpr int kWarps = 4 + 4 * C::NT + C::NP;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kCols = MT * 4 / C::NP;  // accumulator columns per promotion thread
    static constexpr int kTmemCols = MT * C::kAccBufs;
    static constexpr int kBoxRows = MT < 64 ? MT : 64;
    static constexpr int kBoxBytes = kBoxRows * kStepK * 2;
    static constexpr bool kPair = MT == 256;      // two CTAs share the activations
    static constexpr int kCtas = kPair ? 2 : 1;
    static constexpr int kABytes = MT / kCtas * kStepK * 2;
    static constexpr int kLaunchRegs = 65536 / kThreads / 8 * 8;
    static_assert(C::kRegsPromote * C::NP * 32 + C::kRegsOther * (kWarps - C::NP) * 32 <= kLaunchRegs * kThreads,
                  "register shares");
    // shared memory: 1024-byte aligned A stages first
    static constexpr int a = 0;
    static constexpr int dec = a + C::kSteps * kABytes;
    static constexpr int words = dec + C::kSteps * kDecBytes;
    static constexpr int bars = words + C::kWords * kWordBytes;
    static constexpr int first = bars + 640;  // grouped: first tile of every expert
    // the epilogue's blocks: two of 8 rows for every 4 promotion warps
    static constexpr int out = (first + (kMaxExperts + 1) * 4 + 15) / 16 * 16;
    static constexpr int total = out + C::NP / 4 * 2 * kOutBytes + 1024;  // + alignment slack
    static_assert(total <= 227 * 1024, "shared memory");
    static_assert(kPair || MT * BN * 4 <= words, "the split's sums reuse the stages");
    static_assert(C::NT <= C::kSteps && C::NT <= C::kWords, "decode teams");
    static_assert(C::kIssuers == 1 || (C::kSteps % C::NT == 0 && C::kWords % C::NT == 0 && C::kSteps % 4 == 0 &&
                                       C::kAccBufs % 2 == 0),
                  "two issuers: a slot belongs to one team and one issuer");
    static_assert(kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM");
    static_assert((2 * C::kSteps + 2 * C::kWords + 2 * C::kAccBufs) * 8 + 4 <= 640, "barriers");
};

struct Params {
    const uint16_t *S;
    void *C;
    const uint16_t *Other;
    const void *Bias;
    int M, N, K, strips;
    int cluster;  // CTAs that may share a tile of the last round (a pair: 2, which share every tile)
    const int *meta;  // grouped: E+1 row offsets (moe_route's meta), else null
    int E;
};

// a ring's slot and the parity of its current pass
template <int R>
struct Ring {
    int i = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void advance(int by = 1) {
        i += by;
        if (i >= R) {
            i -= R;
            parity ^= 1u;
        }
    }
};

// One lane of a converged warp.  A branch on elect.sync tells the compiler that a single lane
// runs it: under `lane == 0` it wraps every tcgen05 instruction, whose operands are uniform
// registers, in a loop over the lanes, ~100 cycles each (2400 for the 8 MMAs of a group).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}

template <int R>
__device__ __forceinline__ void regs_inc() {
    if constexpr (R > 0) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_dec() {
    if constexpr (R > 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(R));
}

__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Column of the tile that row r of the M operand holds: a core matrix's 8 rows are 4 columns
// of the tile's left half and 4 of its right half, so that a decode lane's two 16-byte reads
// of words are both conflict-free.
__device__ __forceinline__ int column_of(int r) { return 4 * (r >> 3) + (r & 3) + ((r & 4) << 4); }

// K rows 4h .. 4h+3 of the core matrix of 8 words (w0: columns 0-3, w1: 4-7): two columns'
// halves side by side decode together
template <class DT>
__device__ __forceinline__ void decode_half(const uint4 w0, const uint4 w1, int h, uint4 (&out)[4]) {
    const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    uint32_t d[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t z = __byte_perm(w[2 * i], w[2 * i + 1], h ? 0x7632u : 0x5410u);
        const uint32_t y = z >> 8;
        d[i][0] = int4::low_pair<DT>(z);
        d[i][1] = int4::high_pair<DT>(z);
        d[i][2] = int4::low_pair<DT>(y);
        d[i][3] = int4::high_pair<DT>(y);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) out[r] = make_uint4(d[0][r], d[1][r], d[2][r], d[3][r]);
}

// element i = m * N + n, e = its epilogue operand
template <class DT, int POSTOP, bool OUT_F32>
__device__ __forceinline__ void store(const Params &p, size_t i, float v, float e) {
    v = epi<POSTOP, OUT_F32>(v, e);
    if constexpr (OUT_F32) reinterpret_cast<float *>(p.C)[i] = v;
    else reinterpret_cast<uint16_t *>(p.C)[i] = DT::fromf(v);
}

// ---- what a pair's CTAs do through the first one ------------------------------------------
__device__ __forceinline__ uint32_t in_first_cta(const void *p) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(r) : "r"(tc::smem_addr(p)));
    return r;
}
// Arrive on the barrier that the MMA issuer waits for.  Before it the arriving warp has made its
// shared-memory stores visible to the async proxy (decode) or ordered its TMEM loads (promotion),
// and the issuer touches that memory through MMAs only; a .release.cluster here would flush
// all of the warp's memory operations first (~1300 cycles a step, a third of the GEMM's time).
template <bool PAIR>
__device__ __forceinline__ void arrive_at_issuer(uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(in_first_cta(bar)) : "memory");
    else tc::mbar_arrive(bar);
}
// TMA load into this CTA's shared memory, counted on the issuer's barrier
template <bool PAIR>
__device__ __forceinline__ void load_rows(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
            "%3}], [%4];\n" ::"r"(tc::smem_addr(dst)),
            "l"(map), "r"(x), "r"(y), "r"(in_first_cta(bar))
            : "memory");
    else tc::tma_load_2d(dst, map, x, y, bar);
}
template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
    else tc::mma_ss_f16(d, a, b, idesc, accumulate);
}
// arrive on *bar (of both CTAs of a pair) when the MMAs issued so far are through
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
                tc::smem_addr(bar)),
            "h"((uint16_t)3)
            : "memory");
    else tc::mma_commit(bar);
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t ncols) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc::smem_addr(slot)),
                     "r"(ncols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::);
    } else {
        tc::tmem_alloc(slot, ncols);
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_dealloc(uint32_t base, uint32_t ncols) {
    if constexpr (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(base), "r"(ncols));
    else tc::tmem_dealloc(base, ncols);
}

struct Tile {
    int n0, m0, rows, expert;
    int g0, ng;  // the groups of this CTA
};

// The CTA's tiles: `full` rounds of one tile per CTA (or pair), then the rest, `split` CTAs of a
// cluster per tile.
struct Schedule {
    int index, stride;       // of the CTA (or pair) among all
    int full, split, items;  // items: the CTA's tiles
    int rest;                // first tile of the last round
    __device__ __forceinline__ Schedule(int ntiles, int unit, int units, int cluster, int groups) {
        index = unit;
        stride = units;
        full = ntiles / units;
        rest = full * units;
        const int left = ntiles - rest;
        split = 1;
        while (2 * split <= cluster && 2 * split * left <= units && 2 * split <= groups) split *= 2;
        if (left == 0) split = 1;
        items = full + (unit / split < left ? 1 : 0);
    }
};

// tile of item k: row tile t / strips, column strip t % strips (neighbours share their rows)
template <int MT>
__device__ __forceinline__ Tile tile_of(const Params &p, const int *first, const Schedule &s, int k, int rank) {
    const int G = p.K / kGS;
    const bool last = k == s.full;
    const int t = last ? s.rest + s.index / s.split : k * s.stride + s.index;
    const int sk = last ? s.index % s.split : 0, n = last ? s.split : 1;
    const int r = t / p.strips;
    Tile ti;
    ti.g0 = (int)((long long)G * sk / n);
    ti.ng = (int)((long long)G * (sk + 1) / n) - ti.g0;
    ti.n0 = ((t - r * p.strips) * Plan<MT>::kCtas + rank) * BN;
    ti.expert = 0;
    ti.m0 = r * MT;
    int end = p.M;
    if (p.meta) {
        int lo = 0, hi = p.E - 1;  // the last expert whose first tile is <= r
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= r) lo = mid;
            else hi = mid - 1;
        }
        ti.expert = lo;
        const int row0 = min(max(p.meta[lo], 0), p.M);
        end = min(max(p.meta[lo + 1], row0), p.M);
        ti.m0 = row0 + (r - first[lo]) * MT;
    }
    ti.rows = min(MT, end - ti.m0);
    return ti;
}

template <int MT, class DT, int POSTOP, bool OUT_F32>
__global__ void __launch_bounds__(Plan<MT>::kThreads, 1)
    gemm_int4_kernel(const Params p, const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB) {
    using C = Plan<MT>;
    extern __shared__ __align__(1024) char smem_raw[];
    char *smem = smem_raw + ((1024u - (tc::smem_addr(smem_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int G = p.K / kGS;
    constexpr bool PAIR = C::kPair;
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;  // in the pair; the first one issues the MMAs

    uint64_t *ready = reinterpret_cast<uint64_t *>(smem + C::bars);  // a step's operands are in place
    uint64_t *done = ready + C::kSteps;                              // its MMAs have read them
    uint64_t *words_full = done + C::kSteps;
    uint64_t *words_empty = words_full + C::kWords;
    uint64_t *acc_full = words_empty + C::kWords;
    uint64_t *acc_empty = acc_full + C::kAccBufs;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + C::kAccBufs);
    int *first = reinterpret_cast<int *>(smem + C::first);

    if (tid == 0) {
        for (int s = 0; s < C::kSteps; ++s) {
            // the (first) CTA's activations and the decode team's warps (of both CTAs)
            tc::mbar_init(&ready[s], 1 + 4 * C::kCtas);
            tc::mbar_init(&done[s], 1);
        }
        for (int s = 0; s < C::kWords; ++s) {
            tc::mbar_init(&words_full[s], 1);
            tc::mbar_init(&words_empty[s], 4);
        }
        for (int b = 0; b < C::kAccBufs; ++b) {
            tc::mbar_init(&acc_full[b], 1);
            tc::mbar_init(&acc_empty[b], C::NP * C::kCtas);
        }
        tc::fence_mbar_init();
    }
    if (warp == 3) tmem_alloc<PAIR>(tmem_slot, C::kTmemCols);
    if (p.meta) {
        pdl_wait();  // meta comes from the routing kernel
        if (warp == 0) {
            int sum = 0;
            for (int e0 = 0; e0 < p.E; e0 += 32) {
                const int e = e0 + lane;
                int x = 0;
                if (e < p.E) {
                    const int lo = min(max(p.meta[e], 0), p.M), hi = min(max(p.meta[e + 1], lo), p.M);
                    x = (hi - lo + MT - 1) / MT;
                }
                int incl = x;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += y;
                }
                if (e < p.E) first[e] = sum + incl - x;
                sum += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (lane == 0) first[p.E] = sum;
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (PAIR) gemv::cluster_sync_all();  // the other CTA's barriers are initialised
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const int ntiles = (p.meta ? first[p.E] : (p.M + MT - 1) / MT) * p.strips;
    const Schedule sched(ntiles, blockIdx.x / C::kCtas, gridDim.x / C::kCtas, PAIR ? 1 : p.cluster, G);

    // promotion threads: row r of the M operand (a column of C) and the tile's activation rows
    // jbase .. jbase + kCols - 1
    const int pw = warp - (4 + 4 * C::NT);
    const int quad = warp & 3;
    const int jbase = (pw >> 2) * C::kCols;
    const int col = column_of(32 * quad + lane);

    if (warp < 4) {
        regs_dec<C::kRegsOther>();
        if (warp == 0) {
            // ---------------- activations ----------------
            pdl_wait();
            Ring<C::kSteps> q;
            bool ok = true;
            for (int k = 0; k < sched.items && ok; ++k) {
                const Tile ti = tile_of<MT>(p, first, sched, k, rank);
                // a pair's CTA holds half of the MMA's N rows
                const int nrows = PAIR ? (ti.rows + 31) / 32 * 16 : ti.rows;
                const int boxes = (nrows + C::kBoxRows - 1) / C::kBoxRows;
                for (int x = 0; x < 2 * ti.ng; ++x, q.advance()) {
                    if (!tc::mbar_wait(&done[q.i], q.parity ^ 1u)) {
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        if (rank == 0) tc::mbar_expect_tx(&ready[q.i], C::kCtas * boxes * C::kBoxBytes);
                        char *a = smem + C::a + q.i * C::kABytes;
                        for (int b = 0; b < boxes; ++b)
                            load_rows<PAIR>(a + b * C::kBoxBytes, &tmA, ti.g0 * kGS + x * kStepK,
                                            ti.m0 + rank * nrows + b * C::kBoxRows, &ready[q.i]);
                    }
                    __syncwarp();
                }
            }
            if (!ok && rank == 0) {  // copies still in flight must land before the blocks can exit
                for (int s = 0; s < C::kSteps; ++s) {
                    q.advance();
                    tc::mbar_wait(&ready[q.i], q.parity ^ 1u);
                }
            }
        } else if ((warp == 1 || (C::kIssuers == 2 && warp == 3)) && rank == 0) {
            // ---------------- MMA issuer ----------------
            Ring<C::kSteps> q;
            Ring<C::kAccBufs> b;
            bool ok = true;
            int c = 0;  // groups over all tiles
            for (int k = 0; k < sched.items && ok; ++k) {
                const Tile ti = tile_of<MT>(p, first, sched, k, rank);
                // M operand MN-major (bit 15), N operand K-major
                const int nrows = PAIR ? (ti.rows + 31) & ~31 : (ti.rows + 15) & ~15;
                const uint32_t idesc = tc::idesc_f16(DT::kBF16, BN * C::kCtas, nrows) | (1u << 15);
                for (int i = 0; i < ti.ng && ok; ++i, ++c, b.advance()) {
                    if (C::kIssuers == 2 && (c & 1) != (warp >> 1)) {
                        q.advance(2);
                        continue;
                    }
                    if (!tc::mbar_wait(&acc_empty[b.i], b.parity ^ 1u)) {
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (!tc::mbar_wait(&ready[q.i], q.parity)) {
                            ok = false;
                            break;
                        }
                        tc::fence_after_sync();
                        const uint64_t w = tc::sdesc_kmajor_noswz(tc::smem_addr(smem + C::dec + q.i * kDecBytes),
                                                                  kDecLBO, kDecSBO);
                        const uint64_t v = tc::sdesc_kmajor_sw128(tc::smem_addr(smem + C::a + q.i * C::kABytes));
                        if (elect_one()) {
                            // (addresses stay below 2^18: a step along K adds to the address field only)
#pragma unroll
                            for (int kk = 0; kk < kStepK / 16; ++kk)
                                mma<PAIR>(tmem + b.i * MT, w + (uint64_t)(kk * 2 * kDecLBO / 16), v + (uint64_t)(kk * 2),
                                          idesc, (h | kk) != 0);
                            commit<PAIR>(&done[q.i]);
                            if (h) commit<PAIR>(&acc_full[b.i]);
                        }
                        __syncwarp();
                        q.advance();
                    }
                }
            }
        } else if (warp == 2) {
            // ---------------- packed words (weights: read before the previous kernel ends) ----------------
            Ring<C::kWords> q;
            bool ok = true;
            for (int k = 0; k < sched.items && ok; ++k) {
                const Tile ti = tile_of<MT>(p, first, sched, k, rank);
                const int row0 = (ti.expert * G + ti.g0) * int4::kWordsPerGroup;
                for (int x = 0; x < 2 * ti.ng; ++x, q.advance()) {
                    if (!tc::mbar_wait(&words_empty[q.i], q.parity ^ 1u)) {
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        tc::mbar_expect_tx(&words_full[q.i], kWordBytes);
                        tc::tma_load_2d(smem + C::words + q.i * kWordBytes, &tmB, ti.n0,
                                        row0 + x * (kStepK / int4::kRowsPerWord), &words_full[q.i]);
                    }
                    __syncwarp();
                }
            }
            if (!ok) {
                for (int s = 0; s < C::kWords; ++s) {
                    q.advance();
                    tc::mbar_wait(&words_full[q.i], q.parity ^ 1u);
                }
            }
        }
    } else if (warp < 4 + 4 * C::NT) {
        // ---------------- decode ----------------
        regs_dec<C::kRegsOther>();
        const int team = (warp - 4) >> 2;
        const int task = ((warp - 4) & 3) * 32 + lane;  // 8 word rows x 16 column blocks
        const int wr = task >> 4, nb = task & 15;
        const char *src0 = smem + C::words + wr * (BN * 4) + nb * 16;
        char *dst0 = smem + C::dec + nb * kDecSBO + wr * 128;
        Ring<C::kWords> qw;
        Ring<C::kSteps> q;
        qw.advance(team);
        q.advance(team);
        bool ok = true;
        int x = team;  // steps over all tiles; each team takes every NT-th
        for (int k = 0; k < sched.items && ok; ++k) {
            const Tile ti = tile_of<MT>(p, first, sched, k, rank);
            for (; x < 2 * ti.ng; x += C::NT, qw.advance(C::NT), q.advance(C::NT)) {
                if (!tc::mbar_wait(&words_full[qw.i], qw.parity)) {
                    ok = false;
                    break;
                }
                const char *src = src0 + qw.i * kWordBytes;
                const uint4 w0 = *reinterpret_cast<const uint4 *>(src);
                const uint4 w1 = *reinterpret_cast<const uint4 *>(src + 256);
                uint4 out[4];
                decode_half<DT>(w0, w1, 0, out);
                if (!tc::mbar_wait(&done[q.i], q.parity ^ 1u)) {
                    ok = false;
                    break;
                }
                char *dst = dst0 + q.i * kDecBytes;
#pragma unroll
                for (int r = 0; r < 4; ++r) *reinterpret_cast<uint4 *>(dst + r * 16) = out[r];
                decode_half<DT>(w0, w1, 1, out);
#pragma unroll
                for (int r = 0; r < 4; ++r) *reinterpret_cast<uint4 *>(dst + 64 + r * 16) = out[r];
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (elect_one()) {
                    arrive_at_issuer<PAIR>(&ready[q.i]);
                    tc::mbar_arrive(&words_empty[qw.i]);
                }
                __syncwarp();
            }
            x -= 2 * ti.ng;
        }
    } else {
        // ---------------- promotion and epilogue ----------------
        regs_inc<C::kRegsPromote>();
        // the scales of the next kAhead groups are on their way, as loaded: converting or moving
        // one before its group would wait for it
        constexpr int kAhead = 4;
        constexpr int kLd = MT == 32 ? 16 : 32;  // accumulator columns per round of loads
        uint16_t sc[kAhead];
        const uint16_t *sp = nullptr;
        auto scales_of = [&](int k) {
            const Tile ti = tile_of<MT>(p, first, sched, k, rank);
            const int n = ti.n0 + col;
            sp = p.S + ((size_t)ti.expert * G + ti.g0) * p.N + (n < p.N ? n : 0);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) sc[j] = __ldg(sp + (size_t)min(j, ti.ng - 1) * p.N);
        };
        if (sched.items > 0) scales_of(0);
        Ring<C::kAccBufs> b;
        bool ok = true;  // (a warp whose wait timed out still meets the others at their barriers)
        for (int k = 0; k < sched.items; ++k) {
            const Tile ti = tile_of<MT>(p, first, sched, k, rank);
            uint64_t acc[C::kCols / 2];
#pragma unroll
            for (int j = 0; j < C::kCols / 2; ++j) acc[j] = 0ull;
            for (int i0 = 0; i0 < ti.ng && ok; i0 += kAhead) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const int i = i0 + j;
                    if (i >= ti.ng) break;
                    if (!tc::mbar_wait(&acc_full[b.i], b.parity)) {
                        ok = false;
                        break;
                    }
                    tc::fence_after_sync();
                    const float s1 = DT::tof(sc[j]);
                    const uint64_t s = pack2(s1, s1);
                    sc[j] = __ldg(sp + (size_t)min(i + kAhead, ti.ng - 1) * p.N);
                    const uint32_t taddr = tmem + ((uint32_t)(32 * quad) << 16) + (uint32_t)(b.i * MT + jbase);
#pragma unroll
                    for (int c = 0; c < C::kCols; c += kLd) {
                        if (jbase + c < ti.rows) {  // warp-uniform
                            float v[kLd];
                            tc::tmem_ld<16>(taddr + c, *reinterpret_cast<float(*)[16]>(&v[0]));
                            if constexpr (kLd == 32)
                                tc::tmem_ld<16>(taddr + c + 16, *reinterpret_cast<float(*)[16]>(&v[16]));
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int l = 0; l < kLd; l += 2)
                                acc[(c + l) / 2] = fma2(pack2(v[l], v[l + 1]), s, acc[(c + l) / 2]);
                        }
                    }
                    tc::fence_before_sync();
                    __syncwarp();
                    if (elect_one()) arrive_at_issuer<PAIR>(&acc_empty[b.i]);
                    __syncwarp();
                    b.advance();
                }
            }
            if (!PAIR && k == sched.full && sched.split > 1) {
                // its sums [rows][128] go into the stages, whose last readers (the MMAs of the last
                // group) are through, and are joined below
                float *part = reinterpret_cast<float *>(smem);
#pragma unroll
                for (int j = 0; j < C::kCols; j += 2) {
                    float v0, v1;
                    unpack2(acc[j / 2], v0, v1);
                    part[(jbase + j) * BN + col] = v0;
                    part[(jbase + j + 1) * BN + col] = v1;
                }
                break;
            }
            if (k + 1 < sched.items) scales_of(k + 1);
            pdl_wait();
            // 16 rows at a time through shared memory, so that a thread takes 8 columns of two rows
            // (storing TMEM lanes directly, 2 bytes a lane, took 20,000-31,000 cycles a tile)
            char *blocks = smem + C::out + (pw >> 2) * 2 * kOutBytes;
            const int th = (pw & 3) * 32 + lane, row = th >> 4, cb = th & 15;
            const int on = ti.n0 + 8 * cb, sw = (cb >> 2) & 1;
            constexpr bool kOther = POSTOP == 1 || POSTOP == 2;
            uint4 other[2];
            auto fetch = [&](int c) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int m = jbase + (c + h) * kOutRows + row;
                    if (kOther && m < ti.rows && on < p.N)
                        other[h] = __ldg(reinterpret_cast<const uint4 *>(p.Other + (size_t)(ti.m0 + m) * p.N + on));
                }
            };
            fetch(0);
#pragma unroll
            for (int c = 0; c < C::kCols / kOutRows; c += 2) {
                if (jbase + c * kOutRows >= ti.rows) continue;  // the same for the four warps that share the blocks
                if (c) asm volatile("bar.sync %0, 128;\n" ::"r"(1 + (pw >> 2)) : "memory");  // read by all
#pragma unroll
                for (int j = 0; j < 2 * kOutRows; j += 2) {
                    float *mine = reinterpret_cast<float *>(blocks + (j / kOutRows) * kOutBytes) + col +
                                  ((col >> 6) << 4) + (j % kOutRows) * kOutRow;
                    float v0, v1;
                    unpack2(acc[(c * kOutRows + j) / 2], v0, v1);
                    mine[0] = v0;
                    mine[kOutRow] = v1;
                }
                asm volatile("bar.sync %0, 128;\n" ::"r"(1 + (pw >> 2)) : "memory");
                float v[2][8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 *src = reinterpret_cast<const float4 *>(blocks + h * kOutBytes) +
                                        (row * kOutRow + 8 * cb + ((cb >> 3) << 4)) / 4;
                    const float4 x0 = src[sw], x1 = src[sw ^ 1];
                    const float4 lo = sw ? x1 : x0, hi = sw ? x0 : x1;
                    v[h][0] = lo.x, v[h][1] = lo.y, v[h][2] = lo.z, v[h][3] = lo.w;
                    v[h][4] = hi.x, v[h][5] = hi.y, v[h][6] = hi.z, v[h][7] = hi.w;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        float e;
                        if constexpr (kOther) {
                            const uint32_t ow[4] = {other[h].x, other[h].y, other[h].z, other[h].w};
                            e = DT::tof((uint16_t)((k & 1) ? ow[k / 2] >> 16 : ow[k / 2] & 0xFFFFu));
                        } else {
                            e = on < p.N ? epi_in<DT, POSTOP, OUT_F32>(p.Other, p.Bias, 0, on + k) : 0.0f;
                        }
                        v[h][k] = epi<POSTOP, OUT_F32>(v[h][k], e);
                    }
                }
                fetch(c + 2);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int m = jbase + (c + h) * kOutRows + row;
                    if (!ok || m >= ti.rows || on >= p.N) continue;
                    const size_t i = (size_t)(ti.m0 + m) * p.N + on;
                    if constexpr (OUT_F32) {
                        float4 *dst = reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.C) + i);
                        dst[0] = make_float4(v[h][0], v[h][1], v[h][2], v[h][3]);
                        dst[1] = make_float4(v[h][4], v[h][5], v[h][6], v[h][7]);
                    } else {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            w[k] = (uint32_t)DT::fromf(v[h][2 * k]) | ((uint32_t)DT::fromf(v[h][2 * k + 1]) << 16);
                        *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(p.C) + i) =
                            make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            // the next tile writes the blocks again
            asm volatile("bar.sync %0, 128;\n" ::"r"(1 + (pw >> 2)) : "memory");
        }
        pdl_launch_dependents();
        regs_dec<C::kRegsOther>();  // every warp goes on with the same share
    }
    if (!PAIR && sched.split > 1) {
        __syncthreads();
        gemv::cluster_sync_all();
        if (sched.items > sched.full) {
            pdl_wait();
            const Tile ti = tile_of<MT>(p, first, sched, sched.full, rank);
            const float *part = reinterpret_cast<const float *>(smem);
            // the cluster's CTAs from `base` on share the tile
            const int sk = sched.index % sched.split, base = (int)(blockIdx.x % p.cluster) - sk;
            const int r0 = ti.rows * sk / sched.split, r1 = ti.rows * (sk + 1) / sched.split;
            for (int x = r0 * BN + tid; x < r1 * BN; x += C::kThreads) {
                const uint32_t la = tc::smem_addr(part + x);
                float v = 0.0f;
                for (int r = 0; r < sched.split; ++r) v += gemv::ld_dsmem_f1(la, (uint32_t)(base + r));
                const int n = ti.n0 + x % BN;
                const size_t i = (size_t)(ti.m0 + x / BN) * p.N + n;
                if (n < p.N) store<DT, POSTOP, OUT_F32>(p, i, v, epi_in<DT, POSTOP, OUT_F32>(p.Other, p.Bias, i, n));
            }
        }
        gemv::cluster_sync_all();  // every CTA's sums stay until all have read them
    }
    tc::fence_before_sync();
    __syncthreads();
    if (PAIR) gemv::cluster_sync_all();  // neither CTA leaves while the other may use its memory
    if (warp == 3) {
        tc::fence_after_sync();
        tmem_dealloc<PAIR>(tmem, C::kTmemCols);
    }
}

// CTAs that fit the GPU at once in clusters of 1 << c (asked once per device and configuration)
template <int MT>
int resident(int c, int sms) {
    using C = Plan<MT>;
    static std::atomic<int> known[64][4];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sms;
    int n = known[dev][c].load();
    if (n == 0) {
        auto kern = gemm_int4_kernel<MT, F16, 0, false>;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 1u << c;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.gridDim = dim3(sms / (1 << c) * (1 << c));
        cfg.blockDim = dim3(C::kThreads);
        cfg.dynamicSmemBytes = C::total;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (ensure_smem(kern, C::total) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) != cudaSuccess)
            clusters = 0;
        (void)cudaGetLastError();
        n = clusters > 0 ? std::min(clusters << c, sms) : sms / (1 << c) * (1 << c);
        known[dev][c].store(n);
    }
    return n;
}

template <int MT>
cudaError_t launch(const GemvArgs &a, int sms, const int *meta, int E) {
    using C = Plan<MT>;
    CUtensorMap mapA, mapB;
    cudaError_t e = tc::make_map_sw128(
        &mapA, a.A, a.dtype == TERNOCL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
        a.M, a.K, C::kBoxRows);
    if (e != cudaSuccess) return e;
    e = tc::make_map_plain(&mapB, a.B, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, (meta ? E : 1) * (a.K / int4::kRowsPerWord),
                           a.N, kStepK / int4::kRowsPerWord, BN);
    if (e != cudaSuccess) return e;
    const int strips = (a.N + BN * C::kCtas - 1) / (BN * C::kCtas), G = a.K / kGS;
    // grouped: an upper bound, every expert adds at most one partial tile
    const long long tiles = ((long long)(a.M + MT - 1) / MT + (meta ? E : 0)) * strips;
    // Cluster size: what makes the rounds over the tiles fewest, in sixteenths of a round (a split
    // tile costs 1/16 more for its join).  Larger clusters leave some SMs out.  Grouped, the tiles are
    // only counted on the GPU: clusters of 2, which fill it.
    int cl = C::kPair || meta ? 1 : 0, units = C::kPair ? sms / 2 : sms / 2 * 2;
    if (!C::kPair && !meta) {
        long long best = 1LL << 60;
        for (int c = 0; c < 4; ++c) {
            const int n = resident<MT>(c, sms), u = (int)std::min<long long>(n, (tiles << c));
            if (u < (1 << c)) continue;
            const long long full = tiles / u, left = tiles - full * u;
            int split = 1;
            while (2 * split <= (1 << c) && 2 * split * left <= u && 2 * split <= G) split *= 2;
            const long long cost = 16 * full + (left ? 16 / split + (split > 1) : 0);
            if (cost < best) {
                best = cost;
                cl = c;
                units = u;
            }
        }
    }
    const int cluster = 1 << cl;
    if (C::kPair || meta) units = (int)std::min<long long>(units, (tiles + cluster - 1) / cluster * cluster);
    else units = (units + cluster - 1) / cluster * cluster;
    const Params p{(const uint16_t *)a.S, a.C, (const uint16_t *)a.Other, a.Bias, a.M, a.N, a.K, strips, cluster, meta, E};
    return dispatch_epilogue<GemvArgs>(a, [&](auto dt, auto po, auto of) -> cudaError_t {
        using DT = typename decltype(dt)::type;
        auto kern = gemm_int4_kernel<MT, DT, decltype(po)::value, decltype(of)::value>;
        if (C::kRegsPromote > 0 && !smem_attr_known((const void *)kern, C::total)) {
            // the register shares are drawn from what the block launches with
            cudaFuncAttributes fa;
            const cudaError_t fe = cudaFuncGetAttributes(&fa, kern);
            if (fe != cudaSuccess) return fe;
            if (fa.numRegs != C::kLaunchRegs) return cudaErrorInvalidConfiguration;
        }
        cudaError_t err = ensure_smem(kern, C::total);
        if (err != cudaSuccess) return err;
        return launch_kernel_cluster(kern, dim3(units * C::kCtas), dim3(C::kThreads), (size_t)C::total, a.stream,
                                     dim3(cluster, 1, 1), p, mapA, mapB);
    });
}

}  // namespace gemm4

cudaError_t int4_gemm_launch(const GemvArgs &a, int sms, const int *meta, int E) {
    // activation rows per tile: what the rows (grouped: an expert's average) fill
    const long long per = meta ? (a.M + E - 1) / E : a.M;
    // Up to 24 rows by gemm_int4_rows.cu where its 256-column tiles, split 8 ways, fill the SMs: 5376x21504
    // at M = 16 23.5 against 31.6 us here, at M = 24 28.5 against 33.0; 4096x6144 at M = 16 10.9 against 12.5;
    // 14336x4096 at M = 16 23.4 against 17.2.
    if (!meta && a.M <= kInt4RowsMaxM && (long long)((a.N + 255) / 256) * 8 >= sms) return int4_rows_launch(a, sms);
    // Grouped, up to 8 rows per expert on average by gemv_int4.cu (K 2048, 768 columns, 128 experts: 1 row
    // each 18.0 against 35.1 us here, 4 28.5 / 46.3, 8 39.3 / 52.1, 12.5 55.7 / 53.1; K 4096, 14336 columns, 8
    // experts: 6 rows 60 / 87, 12 rows 108 / 93).
    if (meta && per <= kInt4GemvMaxM) return int4_gemv_grouped_launch(a, meta, E);
    int MT = per <= 32 ? 32 : per <= 64 ? 64 : per <= 128 ? 128 : 256;
    const long long strips = (a.N + gemm4::BN - 1) / gemm4::BN;
    if (MT == 256 && !meta) {
        // a pair of CTAs takes a group of 256 x 256 in ~1.5 times a CTA's 128 x 128
        const long long pairs = (strips + 1) / 2 * ((a.M + 255) / 256), singles = strips * ((a.M + 127) / 128);
        const long long pair_waves = (2 * pairs + sms - 1) / sms, waves = (singles + sms - 1) / sms;
        if (3 * pair_waves > 2 * waves) MT = 128;
    }
    return MT == 32    ? gemm4::launch<32>(a, sms, meta, E)
           : MT == 64  ? gemm4::launch<64>(a, sms, meta, E)
           : MT == 128 ? gemm4::launch<128>(a, sms, meta, E)
                       : gemm4::launch<256>(a, sms, meta, E);
}

cudaError_t read_device_error_gemm_int4(unsigned *out, int reset) { return tc::read_tu_error(out, reset); }

}  // namespace ternocl
