// The experts' choice of a mixture-of-experts layer, from router logits l[T, E]:
//
//   s = softmax(l) or sigmoid(l)          score
//   c = s + b                             what the experts are chosen by (b: balance bias)
//   group score = sum of a group's group_top (1 or 2) largest c;  the topk_group best
//   groups stay;  the topk largest c of those groups give ids, in descending order;
//   w = s[ids], divided by its sum if renormalize, times scale, -> RW
//
// Ties go to the lowest index.  An expert whose logit is NaN or -inf, or whose bias is, is
// masked: it is left out of the softmax, comes after every other expert of the kept groups
// (lowest index first) and weighs 0, so ids always holds topk distinct valid experts; a
// group with fewer than group_top unmasked experts comes after all others.  A logit of
// +inf counts as the largest finite fp32.
//
// The choice is discrete, so it is made on 64-bit scores: in 32 bits two experts whose
// scores differ by less than 2^-24 would tie, which a few tokens of a long prompt meet.
// Without a bias the scores rise with the logits, and the logits themselves are compared
// (exactly).  A choice value becomes an unsigned key that orders as the value does, with
// 1 for masked experts and 0 for experts that cannot be taken.
//
// One warp per token: lane l holds experts l, l + 32, ..; each of the topk steps is a
// local maximum and three warp reductions (the key's high word, its low word, the index).
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include "common.cuh"
#include "launch.h"

namespace ternocl {
namespace {

constexpr int kWarps = 4;  // tokens per CTA
constexpr unsigned kAll = 0xffffffffu;
typedef unsigned long long u64;

struct TopkParams {
    const void *logits;
    const float *bias;  // or null
    int *ids;
    void *RW;
    int T, E, topk, scoring, n_group, topk_group, group_top, renorm;
    float scale;
    int logits_dtype, rw_dtype;
};

__device__ __forceinline__ float load_logit(const TopkParams &p, size_t i) {
    if (p.logits_dtype == TERNOCL_FP32) return reinterpret_cast<const float *>(p.logits)[i];
    const uint16_t h = reinterpret_cast<const uint16_t *>(p.logits)[i];
    return p.logits_dtype == TERNOCL_BF16 ? BF16::tof(h) : F16::tof(h);
}

// orders as the value does (-0 as +0); every value but NaN maps to a key > 1
__device__ __forceinline__ u64 order_key(double v) {
    const long long b = __double_as_longlong(v + 0.0);
    return b < 0 ? ~(u64)b : (u64)b | (1ull << 63);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}

// the warp's largest key, and the lowest index that holds it
__device__ __forceinline__ void warp_best(u64 key, unsigned idx, u64 &best, unsigned &at) {
    const unsigned hi = (unsigned)(key >> 32), lo = (unsigned)key;
    const unsigned mh = __reduce_max_sync(kAll, hi);
    const unsigned ml = __reduce_max_sync(kAll, hi == mh ? lo : 0u);
    at = __reduce_min_sync(kAll, hi == mh && lo == ml ? idx : 0xffffffffu);
    best = ((u64)mh << 32) | ml;
}

template <int IPL>  // experts per lane
__global__ void __launch_bounds__(kWarps * 32) moe_topk_kernel(const TopkParams p) {
    extern __shared__ double sm[];  // [kWarps][E] choice values (groups only)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * kWarps + warp;
    pdl_wait();
    if (t >= p.T) return;  // whole warps; no CTA-wide barrier below

    float l[IPL];
    bool open[IPL];  // unmasked
    float mx = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        const int e = i * 32 + lane;
        l[i] = 0.0f;
        open[i] = false;
        if (e < p.E) {
            const float x = load_logit(p, (size_t)t * p.E + e);
            l[i] = fminf(x, FLT_MAX);  // (a NaN becomes FLT_MAX and is masked)
            open[i] = x >= -FLT_MAX;
            if (p.bias) open[i] = open[i] && p.bias[e] >= -FLT_MAX;
            if (open[i]) mx = fmaxf(mx, l[i]);
        }
    }
    double s[IPL];
    if (p.scoring == TERNOCL_SCORE_SOFTMAX) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, o));
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            s[i] = open[i] ? exp((double)l[i] - (double)mx) : 0.0;
            sum += s[i];
        }
        sum = warp_sum(sum);
#pragma unroll
        for (int i = 0; i < IPL; ++i) s[i] = open[i] ? s[i] / sum : 0.0;
    } else {
#pragma unroll
        for (int i = 0; i < IPL; ++i) s[i] = open[i] ? 1.0 / (1.0 + exp(-(double)l[i])) : 0.0;
    }

    u64 key[IPL];
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        const int e = i * 32 + lane;
        key[i] = e >= p.E ? 0ull : !open[i] ? 1ull : order_key(p.bias ? s[i] + (double)p.bias[e] : (double)l[i]);
    }

    if (p.n_group > 1 && p.topk_group < p.n_group) {
        double *c = sm + (size_t)warp * p.E;
        const int per = p.E / p.n_group;
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            const int e = i * 32 + lane;
            if (e < p.E) c[e] = open[i] ? (p.bias ? s[i] + (double)p.bias[e] : s[i]) : -INFINITY;
        }
        __syncwarp();
        u64 gkey = 0ull;  // lane = group (n_group <= 32)
        if (lane < p.n_group) {
            double b1 = -INFINITY, b2 = -INFINITY;
            for (int j = 0; j < per; ++j) {
                const double v = c[lane * per + j];
                if (v > b1) {
                    b2 = b1;
                    b1 = v;
                } else if (v > b2) {
                    b2 = v;
                }
            }
            const bool whole = (p.group_top == 2 ? b2 : b1) > -INFINITY;
            gkey = whole ? order_key(p.group_top == 2 ? b1 + b2 : b1) : 1ull;
        }
        unsigned kept = 0;
        for (int j = 0; j < p.topk_group; ++j) {
            u64 best;
            unsigned at;
            warp_best(gkey, lane, best, at);
            kept |= 1u << at;
            if (lane == (int)at) gkey = 0ull;
        }
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            const int e = i * 32 + lane;
            if (e < p.E && !((kept >> (e / per)) & 1u)) key[i] = 0ull;
        }
    }

    int my_id = 0;
    double my_w = 0.0;
    for (int j = 0; j < p.topk; ++j) {
        u64 bk = 0ull;
        unsigned be = 0xffffffffu;
        double bs = 0.0;
#pragma unroll
        for (int i = 0; i < IPL; ++i)
            if (key[i] > bk) {
                bk = key[i];
                be = i * 32 + lane;
                bs = s[i];
            }
        u64 best;
        unsigned at;
        warp_best(bk, be, best, at);
        const double w = __shfl_sync(kAll, bs, at & 31);
        if (lane == j) {
            my_id = (int)at;
            my_w = w;
        }
#pragma unroll
        for (int i = 0; i < IPL; ++i)
            if ((unsigned)(i * 32 + lane) == at) key[i] = 0ull;
    }
    pdl_launch_dependents();
    if (p.renorm) {
        const double sum = warp_sum(my_w);
        my_w = sum > 0.0 ? my_w / sum : 0.0;
    }
    if (lane < p.topk) {
        const size_t o = (size_t)t * p.topk + lane;
        const float w = (float)(my_w * (double)p.scale);
        p.ids[o] = my_id;
        if (p.rw_dtype == TERNOCL_FP32) reinterpret_cast<float *>(p.RW)[o] = w;
        else reinterpret_cast<uint16_t *>(p.RW)[o] = p.rw_dtype == TERNOCL_BF16 ? BF16::fromf(w) : F16::fromf(w);
    }
}

}  // namespace

cudaError_t moe_topk_launch(const MoeTopkArgs &a) {
    const TopkParams p{a.logits, a.bias, a.ids, a.RW, a.T, a.E, a.topk, a.scoring, a.n_group, a.topk_group,
                       a.group_top, a.renorm, a.scale, a.logits_dtype, a.rw_dtype};
    const dim3 grid((unsigned)((a.T + kWarps - 1) / kWarps)), block(kWarps * 32);
    const size_t smem = a.n_group > 1 ? (size_t)kWarps * a.E * sizeof(double) : 0;  // <= 32 KB
    const int ipl = (a.E + 31) / 32;
    if (ipl <= 1) return launch_kernel(moe_topk_kernel<1>, grid, block, smem, a.stream, p);
    if (ipl <= 2) return launch_kernel(moe_topk_kernel<2>, grid, block, smem, a.stream, p);
    if (ipl <= 4) return launch_kernel(moe_topk_kernel<4>, grid, block, smem, a.stream, p);
    if (ipl <= 8) return launch_kernel(moe_topk_kernel<8>, grid, block, smem, a.stream, p);
    if (ipl <= 16) return launch_kernel(moe_topk_kernel<16>, grid, block, smem, a.stream, p);
    return launch_kernel(moe_topk_kernel<32>, grid, block, smem, a.stream, p);
}

}  // namespace ternocl
