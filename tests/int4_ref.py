"""Plain 64-bit implementations of the int4 products and of the experts' choice, and the error bounds that
the kernels' arithmetic implies (test infrastructure)."""
import numpy as np
import torch

GS = 128


def weights(gen, *shape, dtype, device="cuda"):
    """Random packed weights int32 [..., K/8, N] (every code value) and scales [..., K/128, N]."""
    *lead, K, N = shape
    B = torch.randint(-2 ** 31, 2 ** 31, (*lead, K // 8, N), generator=gen, device=device, dtype=torch.int64)
    S = torch.rand(*lead, K // GS, N, generator=gen, device=device) * 0.04 + 0.01
    return B.to(torch.int32), S.to(dtype)


def codes64(B):
    """float64 codes [..., K, N] of packed words: row 8i + j at bits 4j, two's complement."""
    w = B.long() & 0xFFFFFFFF
    c = torch.stack([(w >> (4 * j)) & 15 for j in range(8)], dim=-2)
    c = torch.where(c > 7, c - 16, c)
    return c.reshape(*B.shape[:-2], B.shape[-2] * 8, B.shape[-1]).double()


def matrix64(B, S):
    return codes64(B) * S.double().repeat_interleave(GS, dim=-2)


def sigmoid64(v):
    """The library's sigmoid: 0 up to -10 (common/epilogue.hpp:34)."""
    return torch.where(v <= -10.0, torch.zeros_like(v), 1.0 / (1.0 + torch.exp(-v)))


def epilogue64(v, d, postop, other, bias, rounded):
    """(value, error bound) of the epilogue of v with error d.  The kernels' sigmoid of a value that is
    rounded to 16 bits is off by up to 4e-6 of itself (__expf: 2 ulp and |x| 2^-23.5 for |x| <= 17, beyond which
    exp(-x) no longer counts; __fdividef: 2 ulp), else by 2^-21; |d(v sigmoid(v))/dv| <= 1.1, |sigmoid'| <= 1/4; an fp32
    operation 2^-24 of its result."""
    es = 4e-6 if rounded else 2.0 ** -21
    if postop == 1:
        s, o = sigmoid64(v), other.double()
        r = v * s * o
        d = 1.1 * d * o.abs() + (es + 2.0 ** -22) * r.abs()
        # either side of the step at -10 is right for a value that may lie on it
        d = d + torch.where((v + 10.0).abs() <= d + 1e-5, 10.1 * 4.6e-5 * o.abs(), 0.0)
        return r, d
    if postop in (2, 3):
        r = v + (other if postop == 2 else bias).double()
        return r, d + 2.0 ** -24 * r.abs()
    if postop == 4:
        r = sigmoid64(v)
        return r, 0.25 * d + es * r.abs() + torch.where((v + 10.0).abs() <= d + 1e-5, 4.6e-5, 0.0)
    return v, d


def product64(A, W, digits):
    """A @ W in 64 bits and the bound of the kernels' sum: 128 products of a group and then the groups (and up to
    16 warps and 8 splits) are added in fp32, each addition off by at most 2^-23 of the sum of magnitudes
    (tensor cores may truncate).  With activation digits a group's sums are exact; an activation is off by
    half a step of its row's largest (2^-23 of it), and the digit planes' magnitudes exceed the
    activation's by at most 3 * 2^-7 of the largest."""
    A, W = A.double(), W.double()
    groups = A.shape[-1] // GS
    mag = A.abs() @ W.abs()
    if digits:
        most = A.abs().amax(dim=-1, keepdim=True) * W.abs().sum(dim=-2)
        return A @ W, (groups + 24) * 2.0 ** -23 * (mag + 2.0 ** -5 * most) + 2.0 ** -23 * most
    return A @ W, (GS + groups + 24) * 2.0 ** -23 * mag


def check(got, want, bound, what=""):
    """Every element of `got` within `bound` of `want` plus the rounding of its type (half a step: eps / 2 of
    the value, or of the smallest normal one), for values inside the type's range."""
    info = torch.finfo(got.dtype)
    want, bound = want.to(got.device), bound.to(got.device)
    allowed = bound + (want.abs() + bound) * (info.eps / 2) + info.tiny * info.eps
    err = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all()), what + ": not finite"
    assert bool((want.abs() + bound < info.max).all()), what + ": the case leaves the type's range"
    worst = (err / allowed).max().item() if err.numel() else 0.0
    assert worst <= 1.0, "%s: error %.3g times the bound" % (what, worst)
    return worst


def topk64(logits, topk, bias=None, scoring="softmax", n_group=1, topk_group=1, group_top=1, renormalize=True,
           scale=1.0):
    """(ids, weights float64) by the definition, one token at a time."""
    x = np.asarray(logits, np.float64)
    T, E = x.shape
    ids = np.zeros((T, topk), np.int32)
    w = np.zeros((T, topk))
    per = E // n_group
    big = float(np.finfo(np.float32).max)
    for t in range(T):
        masked = np.isnan(x[t]) | (x[t] == -np.inf)
        if bias is not None:
            b = np.asarray(bias, np.float64)
            masked |= np.isnan(b) | (b == -np.inf)
        l = np.where(masked, 0.0, np.minimum(x[t], big))
        s = np.zeros(E)
        if (~masked).any():
            if scoring == "softmax":
                e = np.where(masked, 0.0, np.exp(np.where(masked, -np.inf, l) - l[~masked].max()))
                s = e / e.sum()
            else:
                with np.errstate(over="ignore"):
                    s = np.where(masked, 0.0, 1.0 / (1.0 + np.exp(-l)))
        c = s if bias is None else s + np.where(masked, 0.0, b)
        order = l if bias is None else c
        kept = list(range(n_group))
        if topk_group < n_group:
            score = []
            for g in range(n_group):
                best = sorted((c[e] for e in range(g * per, (g + 1) * per) if not masked[e]), reverse=True)[:group_top]
                score.append(sum(best) if len(best) == group_top else -np.inf)
            kept = sorted(range(n_group), key=lambda g: (-score[g], g))[:topk_group]
        allowed = [e for g in kept for e in range(g * per, (g + 1) * per)]
        allowed.sort(key=lambda e: (masked[e], 0.0 if masked[e] else -order[e], e))
        ids[t] = allowed[:topk]
        w[t] = s[ids[t]]
        if renormalize:
            total = w[t].sum()
            w[t] = w[t] / total if total > 0 else 0.0
    return ids, w * scale
