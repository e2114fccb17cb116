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
// The choice is discrete and defined on 64-bit scores: in 32 bits two experts whose scores
// differ by less than 2^-24 would tie, which a few tokens of a long prompt meet.  Without a
// bias the scores rise with the logits, and the logits themselves are compared, exactly.
// Else the choice is first made on fp32 scores, one expert past topk, and stands if every gap
// between neighbours exceeds what fp32 can be off by; a token that fails the test (1 in 100
// or fewer on random logits, and exact ties) is done again in 64 bits, and so is one that
// chooses a score below 2^-100.  The weights of the other tokens are made in fp32 too, within 2^-19 of
// themselves by the bound below: far less than half a step of the 16-bit types.
//
// A segment of 32 or 16 lanes per token: lane l holds experts IPL l .. IPL l + IPL - 1, so that
// a group is a few neighbouring lanes.  A value becomes an unsigned key that orders as the value
// does, with 1 for masked experts and 0 for experts that cannot be taken; each of the topk
// steps is a local maximum, the segment's maximum, and the lowest lane that holds it.
//
// Bound by latency (topk dependent steps) for few tokens, where a warp per token reduces with one
// instruction.  For many it is the steps' arithmetic and their dependences: an instruction issues in 60 %
// of the cycles (57 % with groups), the ALU pipe is busy for 50 %, DRAM for 4 %.  That one instruction
// (REDUX) takes an SM ~19 cycles, so there two tokens share a warp and reduce with shuffles.
// Measured on B200 (GPU time in a CUDA graph): 16381 tokens of 128 bf16 logits, softmax, top-8
// 11.7 us (0.78 us of HBM time), 1 token 2.8 us; sigmoid with a bias, 8 of 256 experts in 4 of 8
// groups: 1 token 5.3 us, 16384 tokens 40-42 us (2.7); groups that are not a power of two of whole lanes,
// 64 bits throughout: 6 of 160 experts in 3 of 8 groups, 1 token 8.6 us, 16384 tokens 71 us (1.7).
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include "common.cuh"
#include "launch.h"

namespace ternocl {
namespace {

constexpr int kWarps = 4;
constexpr unsigned kAll = 0xffffffffu;
typedef unsigned long long u64;
// From here on two tokens share a warp: 16384 softmax tokens of 128 experts 13.1 -> 11.7 us; below,
// fewer warps cost more than the cheaper reductions give (2048 tokens 4.1 -> 4.8 us).
constexpr int kPairTokens = 2048;

struct TopkParams {
    const void *logits;
    const float *bias;  // or null
    int *ids;
    void *RW;
    int T, E, topk, scoring, n_group, topk_group, group_top, renorm;
    float scale;
    int logits_dtype, rw_dtype;
    int vec;  // rows can be read in 4-element pieces
};

template <int IPL>
__device__ __forceinline__ void load_logits(const TopkParams &p, bool vec, size_t row, int lane, float (&l)[IPL]) {
    const size_t i0 = row * p.E + (size_t)lane * IPL;
    if (p.logits_dtype == TERNOCL_FP32) {
        const float *src = reinterpret_cast<const float *>(p.logits) + i0;
        if (IPL % 4 == 0 && vec) {
            if (lane * IPL < p.E) {
#pragma unroll
                for (int i = 0; i < IPL / 4; ++i) {
                    const float4 v = __ldg(reinterpret_cast<const float4 *>(src) + i);
                    l[4 * i] = v.x, l[4 * i + 1] = v.y, l[4 * i + 2] = v.z, l[4 * i + 3] = v.w;
                }
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < IPL; ++i)
            if (lane * IPL + i < p.E) l[i] = __ldg(src + i);
        return;
    }
    const bool bf = p.logits_dtype == TERNOCL_BF16;
    const uint16_t *src = reinterpret_cast<const uint16_t *>(p.logits) + i0;
    if (IPL % 4 == 0 && vec) {
        if (lane * IPL < p.E) {
#pragma unroll
            for (int i = 0; i < IPL / 4; ++i) {
                const uint2 v = __ldg(reinterpret_cast<const uint2 *>(src) + i);
                const uint32_t w[2] = {v.x, v.y};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint16_t h = (uint16_t)((k & 1) ? w[k / 2] >> 16 : w[k / 2] & 0xFFFFu);
                    l[4 * i + k] = bf ? BF16::tof(h) : F16::tof(h);
                }
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < IPL; ++i)
        if (lane * IPL + i < p.E) l[i] = bf ? BF16::tof(__ldg(src + i)) : F16::tof(__ldg(src + i));
}

// keys that order as the values do (-0 as +0); every value but NaN maps to a key > 1
__device__ __forceinline__ u64 order_key(double v) {
    const long long b = __double_as_longlong(v + 0.0);
    return b < 0 ? ~(u64)b : (u64)b | (1ull << 63);
}
__device__ __forceinline__ unsigned order_key(float v) {
    const int b = __float_as_int(v + 0.0f);
    return b < 0 ? ~(unsigned)b : (unsigned)b | 0x80000000u;
}

// over the L lanes of a segment
template <int L, class F>
__device__ __forceinline__ F seg_sum(F v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
template <int L>
__device__ __forceinline__ float seg_max(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
    return v;
}
template <int L>
__device__ __forceinline__ unsigned seg_max(unsigned v) {
    if constexpr (L == 32) {
        return __reduce_max_sync(kAll, v);
    } else {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kAll, v, o));
        return v;
    }
}
// the lowest lane of this lane's segment where `is` holds (some lane's does)
template <int L>
__device__ __forceinline__ int seg_first(bool is) {
    unsigned m = __ballot_sync(kAll, is);
    if constexpr (L < 32) m &= ((1u << L) - 1u) << (threadIdx.x & 31 & ~(L - 1));
    return __ffs(m) - 1;
}

// The best keys in turn (their experts are struck out); lane j of the segment gets the j-th one
// and its expert.  Lanes hold ascending experts: of equal keys the lowest lane's first one wins.
template <int L, int IPL>
__device__ __forceinline__ void take(unsigned (&key)[IPL], int steps, int &id, unsigned &its_key) {
    const int lane = threadIdx.x & 31, sl = lane & (L - 1);
    for (int j = 0; j < steps; ++j) {
        unsigned bk = key[0];
        int bi = 0;
#pragma unroll
        for (int i = 1; i < IPL; ++i)
            if (key[i] > bk) {
                bk = key[i];
                bi = i;
            }
        const unsigned m = seg_max<L>(bk);
        const int owner = seg_first<L>(bk == m);
        const int at = __shfl_sync(kAll, sl * IPL + bi, owner);
        if (sl == j) {
            id = at;
            its_key = m;
        }
#pragma unroll
        for (int i = 0; i < IPL; ++i)
            if (lane == owner && i == bi) key[i] = 0;
    }
}
// the same for keys that hold their expert, as 1024 - expert in the low 11 bits
template <int L, int IPL>
__device__ __forceinline__ void take_indexed(unsigned (&key)[IPL], int steps, int &id, unsigned &its_key) {
    const int sl = threadIdx.x & (L - 1);
    for (int j = 0; j < steps; ++j) {
        unsigned bk = key[0];
#pragma unroll
        for (int i = 1; i < IPL; ++i) bk = max(bk, key[i]);
        const unsigned m = seg_max<L>(bk);
        if (sl == j) {
            id = 1024 - (int)(m & 2047u);
            its_key = m;
        }
#pragma unroll
        for (int i = 0; i < IPL; ++i) key[i] = key[i] == m ? 0u : key[i];
    }
}
// the lowest index that holds the warp's largest key
__device__ __forceinline__ unsigned warp_best(u64 key, unsigned idx) {
    const unsigned hi = (unsigned)(key >> 32), lo = (unsigned)key;
    const unsigned mh = __reduce_max_sync(kAll, hi);
    const unsigned ml = __reduce_max_sync(kAll, hi == mh ? lo : 0u);
    return __reduce_min_sync(kAll, hi == mh && lo == ml ? idx : 0xffffffffu);
}

__device__ __forceinline__ float logit_at(const TopkParams &p, size_t i) {
    if (p.logits_dtype == TERNOCL_FP32) return __ldg(reinterpret_cast<const float *>(p.logits) + i);
    const uint16_t h = __ldg(reinterpret_cast<const uint16_t *>(p.logits) + i);
    return p.logits_dtype == TERNOCL_BF16 ? BF16::tof(h) : F16::tof(h);
}

__device__ __forceinline__ void put(const TopkParams &p, int t, int j, int id, float w) {
    const size_t o = (size_t)t * p.topk + j;
    p.ids[o] = id;
    if (p.rw_dtype == TERNOCL_FP32) reinterpret_cast<float *>(p.RW)[o] = w;
    else reinterpret_cast<uint16_t *>(p.RW)[o] = p.rw_dtype == TERNOCL_BF16 ? BF16::fromf(w) : F16::fromf(w);
}

// l[] of the lane's experts (+inf clamped), the unmasked ones as bits, and their largest
template <int L, int IPL>
__device__ __forceinline__ void read_token(const TopkParams &p, int t, float (&l)[IPL], unsigned &open, float &mx) {
    const int sl = threadIdx.x & (L - 1);
#pragma unroll
    for (int i = 0; i < IPL; ++i) l[i] = -INFINITY;
    load_logits<IPL>(p, p.vec && p.E % IPL == 0, t, sl, l);
    open = 0;
    mx = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        const int e = sl * IPL + i;
        bool o = l[i] >= -FLT_MAX;
        if (p.bias && e < p.E) o = o && __ldg(p.bias + e) >= -FLT_MAX;
        l[i] = fminf(l[i], FLT_MAX);  // (a NaN becomes FLT_MAX and is masked)
        if (o) {
            open |= 1u << i;
            mx = fmaxf(mx, l[i]);
        }
    }
    if (p.scoring == TERNOCL_SCORE_SOFTMAX) mx = seg_max<L>(mx);
}

// token t in 64 bits throughout, by the whole warp; c: [E] in shared memory
template <int IPL>
__device__ __forceinline__ void exact_token(const TopkParams &p, int t, double *c) {
    const int lane = threadIdx.x & 31;
    float l[IPL], mx;
    unsigned open;
    read_token<32, IPL>(p, t, l, open, mx);
    double s[IPL];
    if (p.scoring == TERNOCL_SCORE_SOFTMAX) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            s[i] = (open >> i) & 1u ? exp((double)l[i] - (double)mx) : 0.0;
            sum += s[i];
        }
        sum = seg_sum<32>(sum);
#pragma unroll
        for (int i = 0; i < IPL; ++i) s[i] = (open >> i) & 1u ? s[i] / sum : 0.0;
    } else {
#pragma unroll
        for (int i = 0; i < IPL; ++i) s[i] = (open >> i) & 1u ? 1.0 / (1.0 + exp(-(double)l[i])) : 0.0;
    }
    u64 key[IPL];
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        const int e = lane * IPL + i;
        key[i] = e >= p.E ? 0ull
                 : !((open >> i) & 1u) ? 1ull
                                       : order_key(p.bias ? s[i] + (double)p.bias[e] : (double)l[i]);
    }
    if (p.topk_group < p.n_group) {
        const int per = p.E / p.n_group;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            const int e = lane * IPL + i;
            if (e < p.E) c[e] = !((open >> i) & 1u) ? -INFINITY : p.bias ? s[i] + (double)p.bias[e] : s[i];
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
            const unsigned at = warp_best(gkey, lane);
            kept |= 1u << at;
            if (lane == (int)at) gkey = 0ull;
        }
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            const int e = lane * IPL + i;
            if (e < p.E && !((kept >> (e / per)) & 1u)) key[i] = 0ull;
        }
    }
    int id = 0;
    double w = 0.0;
    for (int j = 0; j < p.topk; ++j) {
        u64 bk = 0ull;
        unsigned be = 0xffffffffu;
        double bs = 0.0;
#pragma unroll
        for (int i = 0; i < IPL; ++i)
            if (key[i] > bk) {
                bk = key[i];
                be = lane * IPL + i;
                bs = s[i];
            }
        const unsigned at = warp_best(bk, be);
        const double x = __shfl_sync(kAll, bs, (int)(at / IPL) & 31);
        if (lane == j) {
            id = (int)at;
            w = x;
        }
#pragma unroll
        for (int i = 0; i < IPL; ++i)
            if (lane * IPL + i == (int)at) key[i] = 0ull;
    }
    if (p.renorm) {
        const double sum = seg_sum<32>(w);  // (lanes from topk on hold 0)
        w = sum > 0.0 ? w / sum : 0.0;
    }
    if (lane < p.topk) put(p, t, lane, id, (float)(w * (double)p.scale));
}

template <int L, int IPL>  // lanes per token, experts per lane
__global__ void __launch_bounds__(kWarps * 32) moe_topk_kernel(const TopkParams p) {
    extern __shared__ double sm[];  // [kWarps][E] 64-bit choice values (groups only)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sl = lane & (L - 1);
    const int tw = (blockIdx.x * kWarps + warp) * (32 / L);  // the warp's first token
    pdl_wait();
    if (tw >= p.T) return;  // whole warps; no CTA-wide barrier below
    const int t = min(tw + lane / L, p.T - 1);

    const bool grouped = p.topk_group < p.n_group;
    const int per = p.E / p.n_group, span = per / IPL;  // lanes per group where groups are whole lanes
    const bool softmax = p.scoring == TERNOCL_SCORE_SOFTMAX;
    // groups that are not a power of two of whole lanes are compared in 64 bits only
    const bool lanes_ok = !grouped || (per % IPL == 0 && (span & (span - 1)) == 0);
    bool sure = lanes_ok;
    if (lanes_ok) {
        float l[IPL], mx;
        unsigned open;
        read_token<L, IPL>(p, t, l, open, mx);
        int id = 0;
        float w = 0.0f;
        // What fp32 can be off by, in units of u = 2^-24.  A sigmoid: expf 2 ulp (4 u), a sum and a quotient,
        // 6 u s.  A softmax: expf 4 u, its argument 0.4 u (|x - mx| is off by itself times u, and
        // d exp(-d) < 0.37); of the sum, expf 4 u, the arguments 4.5 u (the mean of |x - mx| weighted by
        // the terms, of 1024 experts), 10 additions (pairwise in a lane, then over lanes); the quotient and the
        // product: 24.5 u s + 0.4 u, taken as 32 u s + 0.5 u.  c is off by u |c| more.
        float inv = 1.0f;  // softmax: 1 / sum over the experts (renormalised weights alone do without)
        if (softmax && (p.bias || grouped || !p.renorm)) {
            float term[IPL];
#pragma unroll
            for (int i = 0; i < IPL; ++i) term[i] = (open >> i) & 1u ? expf(l[i] - mx) : 0.0f;
#pragma unroll
            for (int o = IPL / 2; o > 0; o >>= 1)
#pragma unroll
                for (int i = 0; i < o; ++i) term[i] += term[i + o];
            inv = 1.0f / seg_sum<L>(term[0]);
        }
        auto score = [&](float x) { return softmax ? expf(x - mx) * inv : 1.0f / (1.0f + expf(-x)); };
        const bool indexed = !p.bias && p.logits_dtype != TERNOCL_FP32;
        float c[IPL];
        unsigned key[IPL];
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            const bool o = (open >> i) & 1u;
            const int e = sl * IPL + i;
            c[i] = 0.0f;
            if (o && (p.bias || grouped)) c[i] = score(l[i]) + (p.bias ? __ldg(p.bias + e) : 0.0f);
            key[i] = e >= p.E ? 0u : !o ? 1u : order_key(p.bias ? c[i] : l[i]);
            // a 16-bit logit has 19 high bits as fp32 (1 + 8 + 10 of fp16's mantissa); below them the expert
            if (indexed && e < p.E) key[i] = (o ? key[i] >> 13 << 11 : 0u) | (unsigned)(1024 - e);
        }
        if (grouped) {
            float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
            for (int i = 0; i < IPL; ++i) {
                const float v = (open >> i) & 1u ? c[i] : -INFINITY;
                b2 = fmaxf(b2, fminf(b1, v));
                b1 = fmaxf(b1, v);
            }
            for (int o = 1; o < span; o <<= 1) {
                const float v1 = __shfl_xor_sync(kAll, b1, o), v2 = __shfl_xor_sync(kAll, b2, o);
                b2 = fmaxf(fminf(b1, v1), fmaxf(b2, v2));
                b1 = fmaxf(b1, v1);
            }
            const bool real = sl * IPL < p.E;
            const bool whole = (p.group_top == 2 ? b2 : b1) > -INFINITY;
            const float total = p.group_top == 2 ? b1 + b2 : b1;
            const unsigned gkey = !real ? 0u : whole ? order_key(total) : 1u;
            bool kept = false;
            for (int j = 0; j < p.topk_group; ++j) {
                const unsigned k = kept ? 0u : gkey;
                const int first = seg_first<L>(k == seg_max<L>(k));
                if ((lane - first) / span == 0 && lane >= first) kept = true;
            }
            // the least kept score against the best of the others: two groups' scores (a softmax's sum to 1 at
            // most, four sigmoids) are off by 34 u; their c by |b1| + |b2| <= |total| + 2 * 16 u each, with larger
            // opposites left to 64 bits; the totals by |total| u: less than 128 u + 16 u max |total|
            if (p.group_top == 2 && real && b1 > 0.0f && b2 < -16.0f) sure = false;
            const unsigned lo = ~seg_max<L>(kept && real ? ~gkey : 0u);
            const unsigned hi = seg_max<L>(!kept && real ? gkey : 0u);
            if (lo > 1u && hi > 1u) {  // (masked groups are ordered by index)
                const float a = __int_as_float(lo >> 31 ? lo & 0x7fffffffu : ~lo);
                const float b = __int_as_float(hi >> 31 ? hi & 0x7fffffffu : ~hi);
                sure = sure && a - b > 0x1p-17f + 0x1p-20f * fmaxf(fabsf(a), fabsf(b));
            }
#pragma unroll
            for (int i = 0; i < IPL; ++i)
                if (!kept) key[i] = 0u;
        }
        unsigned its = 0u;
        const int steps = min(p.topk + (p.bias ? 1 : 0), L);
        if (indexed) take_indexed<L, IPL>(key, steps, id, its);
        else take<L, IPL>(key, steps, id, its);
        if (indexed ? its >= 2048u : its > 1u) {  // unmasked
            const float x = fminf(logit_at(p, (size_t)t * p.E + id), FLT_MAX);
            w = score(x);
            if (softmax) {
                // d = x - mx is off by up to |d| u, which the weight would be off by: what the subtraction
                // rounded away, times w (beyond 128 the token is computed in 64 bits)
                const float d = x - mx, b = d - x;
                if (d > -128.0f) w = fmaf(w, (x - (d - b)) - (mx + b), w);
            }
            // scores near the end of fp32's range (a sigmoid far below 0, a softmax's far below its largest)
            // would lose bits or vanish, and with them the weights that they are divided into
            if (sl < p.topk && w < 0x1p-100f) sure = false;
        }
        if (p.bias) {
            // neighbours in the order (and the first one left out; at topk = 32 the rest's best)
            unsigned next = __shfl_down_sync(kAll, its, 1);
            float ws = __shfl_down_sync(kAll, w, 1);
            if (p.topk == L) {
                unsigned bk = 0u;
#pragma unroll
                for (int i = 0; i < IPL; ++i) bk = max(bk, key[i]);
                bk = seg_max<L>(bk);
                if (sl == L - 1) {
                    next = bk;
                    ws = 1.0f;  // (not known here, at most 1)
                }
            }
            if (sl < p.topk && its > 1u && next > 1u) {
                const float a = __int_as_float(its >> 31 ? its & 0x7fffffffu : ~its);
                const float b = __int_as_float(next >> 31 ? next & 0x7fffffffu : ~next);
                const float rel = softmax ? 0x1p-19f : 0x1p-20f;
                sure = sure && a - b > rel * (w + ws) + 0x1p-22f + 0x1p-22f * fmaxf(fabsf(a), fabsf(b));
            }
        }
        if (p.renorm) {
            const float sum = seg_sum<L>(sl < p.topk ? w : 0.0f);
            w = sum > 0.0f ? w / sum : 0.0f;
        }
        if (sl < p.topk && tw + lane / L < p.T) put(p, t, sl, id, w * p.scale);
    }
    const unsigned unsure = __ballot_sync(kAll, !sure);
    if (unsure) {
        __syncwarp();  // (the 64-bit results replace what other lanes have written)
#pragma unroll 1
        for (int h = 0; h < 32 / L; ++h)
            if (tw + h < p.T && (L == 32 || ((unsure >> (h * L)) & ((1u << (L & 31)) - 1u))))
                exact_token<(IPL * L + 31) / 32>(p, tw + h, sm + (size_t)warp * p.E);
    }
    pdl_launch_dependents();
}

}  // namespace

cudaError_t moe_topk_launch(const MoeTopkArgs &a) {
    TopkParams p{a.logits, a.bias, a.ids, a.RW, a.T, a.E, a.topk, a.scoring, a.n_group, a.topk_group,
                 a.group_top, a.renorm, a.scale, a.logits_dtype, a.rw_dtype, 0};
    const size_t smem = a.topk_group < a.n_group ? (size_t)kWarps * a.E * sizeof(double) : 0;  // <= 32 KB
    p.vec = (uintptr_t)a.logits % (a.logits_dtype == TERNOCL_FP32 ? 16 : 8) == 0;
    auto run = [&](auto lanes, auto ipl) {
        constexpr int L = decltype(lanes)::value, IPL = decltype(ipl)::value;
        constexpr int tokens = kWarps * (32 / L);
        return launch_kernel(moe_topk_kernel<L, IPL>, dim3((unsigned)((a.T + tokens - 1) / tokens)), dim3(kWarps * 32),
                             smem, a.stream, p);
    };
    auto with = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        const int ipl = (a.E + L - 1) / L;
        if (ipl <= 1) return run(lanes, std::integral_constant<int, 1>{});
        if (ipl <= 2) return run(lanes, std::integral_constant<int, 2>{});
        if (ipl <= 4) return run(lanes, std::integral_constant<int, 4>{});
        if (ipl <= 8) return run(lanes, std::integral_constant<int, 8>{});
        if (ipl <= 16) return run(lanes, std::integral_constant<int, 16>{});
        return run(lanes, std::integral_constant<int, 32>{});
    };
    if (a.T >= kPairTokens && a.E <= 512 && a.topk < 16) return with(std::integral_constant<int, 16>{});
    return with(std::integral_constant<int, 32>{});
}

}  // namespace ternocl
