"""4-bit weights on the GPU: the linear layer (GEMV and tcgen05 GEMM), the grouped GEMM and the MoE decode
GEMVs against 64-bit products, element by element within the bounds of their arithmetic (int4_ref.py)."""
import numpy as np
import pytest
import torch

from int4_ref import check, codes64, epilogue64, matrix64, product64, sigmoid64, topk64, weights

pytestmark = pytest.mark.gpu
DT = {0: torch.float16, 1: torch.bfloat16}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def activations(g, M, K, dtype):
    """Normal values with outlier channels (a few far larger than the rest)."""
    a = torch.randn(M, K, generator=g, device="cuda")
    a[:, :: max(1, K // 3)] *= 20.0
    return a.to(dtype)


def linear_case(tl, seed, M, K, N, bf16, postop, out_f32, algo):
    g = gen(seed)
    dt = DT[bf16]
    A = activations(g, M, K, dt)
    B, S = weights(g, K, N, dtype=dt)
    S = (S / K ** 0.5).to(dt)
    other = torch.randn(M, N, generator=g, device="cuda").to(dt) if postop in (1, 2) else None
    bias = torch.randn(N, generator=g, device="cuda").to(torch.float32 if out_f32 else dt) if postop == 3 else None
    C = tl.int4_upcvt(A, B, S, postop=postop, out_f32=out_f32, other=other, bias=bias, algo=algo)
    v, d = product64(A, matrix64(B, S), digits=False)
    vd, dd = product64(A, matrix64(B, S), digits=True)
    want, bound = epilogue64(v, torch.maximum(d, dd), postop, other, bias, not out_f32)
    assert C.dtype == (torch.float32 if out_f32 else dt) and C.shape == (M, N)
    check(C, want, bound, "M=%d K=%d N=%d" % (M, K, N))


@pytest.mark.parametrize("algo", [1, 2], ids=["gemv", "gemm"])
@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("M,K,N", [(1, 128, 16), (1, 4096, 272), (2, 384, 48), (3, 1152, 144), (7, 256, 4096),
                                   (8, 2048, 176), (9, 128, 2400), (17, 640, 208), (33, 512, 112), (65, 384, 272),
                                   (129, 256, 144), (200, 1280, 400)])
def test_linear_shapes(cuda, tl, algo, bf16, M, K, N):
    linear_case(tl, M + K + N, M, K, N, bf16, 0, bool((M + K // 128) & 1), algo)
    assert tl.device_error() == 0


@pytest.mark.parametrize("algo,M", [(1, 1), (1, 5), (2, 5), (2, 40), (2, 300)])
@pytest.mark.parametrize("postop", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("out_f32", [False, True])
def test_linear_epilogues(cuda, tl, algo, M, postop, out_f32):
    for bf16 in (0, 1):
        linear_case(tl, 7 * M + postop, M, 640, 208, bf16, postop, out_f32, algo)
    assert tl.device_error() == 0


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("M", [1, 2, 8, 24, 64, 700])
def test_linear_auto_long_k(cuda, tl, bf16, M):
    linear_case(tl, M, M, 14336, 304, bf16, 0, True, 0)
    assert tl.device_error() == 0


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("algo,M", [(1, 1), (1, 2), (1, 8), (2, 32), (2, 64), (2, 256)])
def test_linear_reads_every_code_exactly(cuda, tl, bf16, algo, M):
    """One-hot activation rows pick single weights: code * S, exact in fp32."""
    K, N = 256, 272
    B, S = weights(gen(3), K, N, dtype=DT[bf16])
    W = matrix64(B, S).float()
    for k0 in range(0, K, M):
        A = torch.zeros(M, K, device="cuda", dtype=DT[bf16])
        A[torch.arange(M), torch.arange(k0, k0 + M)] = 1.0
        C = tl.int4_upcvt(A, B, S, out_f32=True, algo=algo)
        assert torch.equal(C, W[k0:k0 + M]), k0
    assert tl.device_error() == 0


@pytest.mark.parametrize("algo,M", [(1, 8), (2, 8), (2, 130)])
def test_linear_rows_do_not_touch_each_other(cuda, tl, algo, M):
    g = gen(4)
    A = activations(g, M, 512, torch.float16)
    B, S = weights(g, 512, 144, dtype=torch.float16)
    C = tl.int4_upcvt(A, B, S, out_f32=True, algo=algo)
    for bad in (float("nan"), float("inf"), 65504.0):
        A2 = A.clone()
        A2[3, 77] = bad
        C2 = tl.int4_upcvt(A2, B, S, out_f32=True, algo=algo)
        keep = torch.arange(M, device="cuda") != 3
        assert torch.equal(C[keep], C2[keep])
        if bad != 65504.0:
            nonzero = (codes64(B)[77] != 0)
            assert not bool(torch.isfinite(C2[3][nonzero]).any())


def test_linear_zero_rows_and_empty(cuda, tl):
    B, S = weights(gen(5), 256, 64, dtype=torch.bfloat16)
    for M in (1, 40):
        A = torch.zeros(M, 256, device="cuda", dtype=torch.bfloat16)
        assert not bool(tl.int4_upcvt(A, B, S).any())
    assert tl.int4_upcvt(torch.zeros(0, 256, device="cuda", dtype=torch.bfloat16), B, S).shape == (0, 64)


@pytest.mark.parametrize("M", [1, 4, 20, 300])
def test_linear_is_reproducible_and_captured(cuda, tl, M):
    """Equal bits from every call, on another stream and from a replayed graph on new inputs."""
    g = gen(6)
    B, S = weights(g, 1024, 400, dtype=torch.bfloat16)
    A1, A2 = activations(g, M, 1024, torch.bfloat16), activations(g, M, 1024, torch.bfloat16)
    want1, want2 = tl.int4_upcvt(A1, B, S), tl.int4_upcvt(A2, B, S)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = tl.int4_upcvt(A2, B, S)
    handed = tl.int4_upcvt(A1, B, S, stream=side)
    side.synchronize()
    assert torch.equal(on_side, want2) and torch.equal(handed, want1)
    A, C = A1.clone(), torch.empty_like(want1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tl.int4_upcvt(A, B, S, out=C)
    for src, want in ((A2, want2), (A1, want1)):
        A.copy_(src)
        C.zero_()
        graph.replay()
        assert torch.equal(C, want)


def test_linear_under_pdl(cuda, tl):
    """Chained calls with programmatic dependent launch: each reads what the one before wrote."""
    g = gen(7)
    B, S = weights(g, 512, 512, dtype=torch.float16)
    S = (S / 512 ** 0.5).to(torch.float16)
    for M in (1, 8, 50):
        x = activations(g, M, 512, torch.float16)
        want = x
        for _ in range(6):
            want = tl.int4_upcvt(want, B, S)
        old = tl.set_option(tl.OPT_PDL, 1)
        try:
            got = x
            for _ in range(6):
                got = tl.int4_upcvt(got, B, S)
        finally:
            tl.set_option(tl.OPT_PDL, old)
        assert torch.equal(got, want), M


# ---------------------------------------------------------------------------------- experts
def routing(g, T, topk, E):
    return torch.argsort(torch.rand(T, E, generator=g, device="cuda"), dim=1)[:, :topk].to(torch.int32).reshape(-1)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("T,topk,E,K,N", [(1, 1, 1, 128, 16), (1, 8, 16, 2048, 768), (3, 4, 8, 384, 272),
                                          (11, 2, 6, 1152, 48), (2, 3, 5, 14336, 32)])
def test_gate_up(cuda, tl, bf16, T, topk, E, K, N):
    g, dt = gen(T + K), DT[bf16]
    X, ids = activations(g, T, K, dt), routing(g, T, topk, E)
    (Bg, Sg), (Bu, Su) = weights(g, E, K, N, dtype=dt), weights(g, E, K, N, dtype=dt)
    Sg, Su = (Sg / K ** 0.5).to(dt), (Su / K ** 0.5).to(dt)
    H = tl.moe_decode_gate_up_int4(ids, X, Bg, Sg, Bu, Su, E, topk)
    for r, e in enumerate(ids.tolist()):
        x = X[r // topk][None]
        vg, dg = product64(x, matrix64(Bg[e], Sg[e]), True)
        vu, du = product64(x, matrix64(Bu[e], Su[e]), True)
        want, bound = epilogue64(vg, dg, 1, vu, None, True)
        check(H[r][None], want, bound + 1.1 * (vg.abs() + dg) * du, "row %d" % r)
    assert tl.device_error() == 0


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("T,topk,E,K,N", [(1, 1, 1, 128, 16), (1, 8, 16, 768, 2048), (4, 3, 8, 384, 272),
                                          (9, 2, 5, 1152, 48), (2, 8, 9, 4096, 32)])
def test_down_sum(cuda, tl, bf16, T, topk, E, K, N):
    g, dt = gen(T + K), DT[bf16]
    H, ids = activations(g, T * topk, K, dt), routing(g, T, topk, E)
    RW = torch.rand(T * topk, generator=g, device="cuda").to(dt)
    B, S = weights(g, E, K, N, dtype=dt)
    S = (S / K ** 0.5).to(dt)
    O = tl.moe_decode_down_sum_int4(ids, H, RW, B, S, E, topk)
    for t in range(T):
        # the experts' rows side by side are one long row; a scale times RW is one more rounding
        rows = range(t * topk, (t + 1) * topk)
        W = torch.cat([matrix64(B[ids[r]], S[ids[r]]) * RW[r].double() for r in rows])
        v, d = product64(H[list(rows)].reshape(1, -1), W, True)
        check(O[t][None], v, d + 2.0 ** -23 * (H[list(rows)].reshape(1, -1).double().abs() @ W.abs()), "token %d" % t)
    assert tl.device_error() == 0


def test_decode_bad_expert_ids_contribute_zero(cuda, tl):
    g = gen(9)
    T, topk, E, K, N = 2, 3, 4, 256, 64
    X, ids = activations(g, T, K, torch.float16), routing(g, T, topk, E)
    B, S = weights(g, E, K, N, dtype=torch.float16)
    Bd, Sd = weights(g, E, N * 2, K, dtype=torch.float16)  # K of the way back: 128
    S[0], Sd[0] = float("nan"), float("nan")  # what a bad id must not read
    good = torch.tensor([1, 2, 3, 3, 1, 2], dtype=torch.int32, device="cuda")
    H = tl.moe_decode_gate_up_int4(good, X, B, S, B, S, E, topk)
    Hd = activations(g, T * topk, 128, torch.float16)
    RW = torch.rand(T * topk, generator=g, device="cuda").half()
    tl.device_error(reset=True)
    for bad in (-1, E, 2 ** 31 - 1, -2 ** 31):
        ids = good.clone()
        ids[4] = bad
        H2 = tl.moe_decode_gate_up_int4(ids, X, B, S, B, S, E, topk)
        O2 = tl.moe_decode_down_sum_int4(ids, Hd, RW, Bd, Sd, E, topk)
        assert tl.device_error(reset=True) == 2
        assert not bool(H2[4].any())
        keep = torch.arange(T * topk, device="cuda") != 4
        assert torch.equal(H2[keep], H[keep])
        RW0 = RW.clone()
        RW0[4] = 0
        assert torch.equal(O2, tl.moe_decode_down_sum_int4(good, Hd, RW0, Bd, Sd, E, topk))
    assert tl.device_error() == 0


@pytest.mark.parametrize("T,topk,K", [(1, 6, 128), (3, 8, 384), (40, 8, 128), (1, 3, 4096)])
def test_down_sum_ignores_the_activations_of_bad_ids(cuda, tl, T, topk, K):
    """Left-out rows (another device's experts, say) may hold anything: NaN, Inf, or values so large that
    sharing a fixed-point scale with them would wipe the others out."""
    g, E, N = gen(T * K), 5, 144
    H, ids = activations(g, T * topk, K, torch.bfloat16), torch.randint(0, E, (T * topk,), generator=g, device="cuda",
                                                                       dtype=torch.int32)
    B, S = weights(g, E, K, N, dtype=torch.bfloat16)
    RW = torch.rand(T * topk, generator=g, device="cuda").bfloat16()
    ids[1::2] = -1
    H[1::2] = 0
    want = tl.moe_decode_down_sum_int4(ids, H, RW, B, S, E, topk)
    assert bool(want.isfinite().all()) and bool(want.any())
    for v in (float("nan"), float("inf"), 3e38):
        H[1::2] = v
        assert torch.equal(tl.moe_decode_down_sum_int4(ids, H, RW, B, S, E, topk), want), v
    assert tl.device_error(reset=True) == 2


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("T,topk,E,K,N,postop,out_f32", [
    (1, 1, 1, 128, 16, 0, True), (5, 2, 4, 256, 144, 1, False), (40, 4, 8, 640, 272, 2, True),
    (300, 2, 3, 384, 128, 0, False), (600, 1, 2, 256, 48, 4, True), (9, 8, 64, 256, 112, 1, True)])
def test_grouped_gemm(cuda, tl, bf16, T, topk, E, K, N, postop, out_f32):
    g, dt = gen(T + K + N), DT[bf16]
    G = T * topk
    ids = routing(g, T, topk, E)
    meta, perm, inv = tl.moe_route(ids, E)
    A = activations(g, G, K, dt)
    B, S = weights(g, E, K, N, dtype=dt)
    S = (S / K ** 0.5).to(dt)
    other = torch.randn(G, N, generator=g, device="cuda").to(dt) if postop in (1, 2) else None
    C = tl.moe_gemm_int4(meta, A, B, S, E, postop=postop, out_f32=out_f32, other=other)
    first = meta[:E + 1].tolist()
    for e in range(E):
        lo, hi = first[e], first[e + 1]
        if hi > lo:
            v, d = product64(A[lo:hi], matrix64(B[e], S[e]), False)
            want, bound = epilogue64(v, d, postop, None if other is None else other[lo:hi], None, not out_f32)
            check(C[lo:hi], want, bound, "expert %d" % e)
    assert tl.device_error() == 0


@pytest.mark.parametrize("counts", [[0, 0, 5], [128, 0, 129, 1, 0, 256, 127], [0, 300, 0], [33, 31, 32, 0, 64]])
def test_grouped_gemm_segments_and_rows_behind_them(cuda, tl, counts):
    """Experts without rows, segments around the tile sizes, and rows behind the last segment untouched."""
    g = gen(sum(counts))
    E, K, N, extra = len(counts), 256, 144, 7
    G = sum(counts) + extra
    A = activations(g, G, K, torch.bfloat16)
    B, S = weights(g, E, K, N, dtype=torch.bfloat16)
    rows = np.concatenate([[0], np.cumsum(counts)])
    tiles = np.concatenate([[0], np.cumsum([(c + 127) // 128 for c in counts])])
    meta = torch.tensor(np.concatenate([rows, tiles]), dtype=torch.int32, device="cuda")
    C = torch.full((G, N), -7.0, device="cuda")
    tl.moe_gemm_int4(meta, A, B, S, E, out_f32=True, out=C)
    for e in range(E):
        lo, hi = int(rows[e]), int(rows[e + 1])
        if hi > lo:
            check(C[lo:hi], *product64(A[lo:hi], matrix64(B[e], S[e]), False), "expert %d" % e)
    assert bool((C[G - extra:] == -7.0).all())
    assert tl.device_error() == 0


@pytest.mark.parametrize("K,N", [(384, 144), (2176, 48)])
@pytest.mark.parametrize("counts", [[0] * 70 + [200] + [0, 1, 7, 8, 9, 16, 17] * 4 + [0], [8, 9, 0, 7], [1] * 40,
                                    [0] * 31 + [60] + [33] + [0] * 31, [0, 0, 0, 24]])
def test_grouped_gemm_few_rows_per_expert(cuda, tl, counts, K, N):
    """Up to 8 rows per expert on average, unevenly: blocks of 8 rows beyond an expert's first, experts
    beyond a warp's lanes, rows before the first segment and behind the last untouched."""
    g = gen(sum(counts) + K)
    E, before, behind = len(counts), 3, 5
    G = before + sum(counts) + behind
    A = activations(g, G, K, torch.float16)
    A[:before] = A[G - behind:] = float("nan")
    B, S = weights(g, E, K, N, dtype=torch.float16)
    S = (S / K ** 0.5).half()
    other = torch.randn(G, N, generator=g, device="cuda").half()
    rows = before + np.concatenate([[0], np.cumsum(counts)])
    tiles = np.concatenate([[0], np.cumsum([(c + 127) // 128 for c in counts])])
    meta = torch.tensor(np.concatenate([rows, tiles]), dtype=torch.int32, device="cuda")
    C = torch.full((G, N), -7.0, device="cuda", dtype=torch.float16)
    tl.moe_gemm_int4(meta, A, B, S, E, postop=2, other=other, out=C)
    for e in range(E):
        lo, hi = int(rows[e]), int(rows[e + 1])
        if hi > lo:
            v, d = product64(A[lo:hi], matrix64(B[e], S[e]), False)
            want, bound = epilogue64(v, d, 2, other[lo:hi], None, True)
            check(C[lo:hi], want, bound, "expert %d" % e)
    assert bool((C[:before] == -7.0).all()) and bool((C[G - behind:] == -7.0).all())
    assert tl.device_error() == 0


def test_expert_weights_beyond_32_bit_offsets(cuda, tl):
    """The last expert's words start behind 4 GiB."""
    E, K, N = 1024, 4096, 2048
    B = torch.zeros(E, K // 8, N, dtype=torch.int32, device="cuda")
    S = torch.zeros(E, K // 128, N, dtype=torch.float16, device="cuda")
    g = gen(10)
    B[-1], S[-1] = weights(g, K, N, dtype=torch.float16)
    S[-1] /= 64
    X = activations(g, 1, K, torch.float16)
    ids = torch.tensor([E - 1], dtype=torch.int32, device="cuda")
    W = matrix64(B[-1], S[-1])
    v, d = product64(X, W, True)
    one = torch.ones(1, dtype=torch.float16, device="cuda")
    check(tl.moe_decode_down_sum_int4(ids, X, one, B, S, E, 1), v, d + 2.0 ** -23 * (X.double().abs() @ W.abs()))
    H = tl.moe_decode_gate_up_int4(ids, X, B, S, B, S, E, 1)
    want, bound = epilogue64(v, d, 1, v, None, True)
    check(H, want, bound + 1.1 * (v.abs() + d) * d)
    meta, _, _ = tl.moe_route(ids, E)
    v, d = product64(X, W, False)
    check(tl.moe_gemm_int4(meta, X, B, S, E, out_f32=True), v, d)
    assert tl.device_error() == 0


# ------------------------------------------------------------------------- the run of them together
@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("T", [1, 6, 150])
def test_layer_from_logits(cuda, tl, bf16, T):
    """Router logits -> ids and weights -> the experts' layer, for prompts and for single tokens, against 64 bits;
    and the ternary layers take the same ids and weights."""
    import ternocl_b200.torch_ops  # noqa: F401
    g, dt = gen(T), DT[bf16]
    E, topk, H, I = 16, 4, 512, 256
    X = torch.randn(T, H, generator=g, device="cuda").to(dt)
    logits = torch.randn(T, E, generator=g, device="cuda")
    bias = 0.1 * torch.randn(E, generator=g, device="cuda")
    (Bg, Sg), (Bu, Su) = weights(g, E, H, I, dtype=dt), weights(g, E, H, I, dtype=dt)
    Bd, Sd = weights(g, E, I, H, dtype=dt)
    Sg, Su, Sd = (Sg / 16).to(dt), (Su / 16).to(dt), (Sd / 16).to(dt)
    how = dict(bias=bias, scoring="sigmoid", n_group=4, topk_group=2, group_top=2, renormalize=True, scale=2.5)
    ids, RW = torch.ops.ternocl.moe_topk(logits, topk, dtype=dt, **how)
    want_ids, want_w = topk64(logits.cpu().numpy(), topk, **{**how, "bias": bias.cpu().numpy()})
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    outs = [torch.ops.ternocl.moe_prefill_int4(X, ids, RW, Bg, Sg, Bu, Su, Bd, Sd, E, topk)]
    if T <= 6:
        outs.append(torch.ops.ternocl.moe_decode_int4(X, ids, RW, Bg, Sg, Bu, Su, Bd, Sd, E, topk))
    x, eps = X.double(), torch.finfo(dt).eps / 2
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    for t in range(T):
        for j in range(topk):
            e = int(ids[t, j])
            vg, dg = product64(x[t:t + 1], matrix64(Bg[e], Sg[e]), True)
            vu, du = product64(x[t:t + 1], matrix64(Bu[e], Su[e]), True)
            dg, du = 64 * dg, 64 * du + eps * vu.abs()  # (the GEMM's sums, and up rounded to DT)
            h, dh = epilogue64(vg, dg, 1, vu, None, True)
            dh = dh + 1.1 * (vg.abs() + dg) * du
            dh = dh + eps * (h.abs() + dh)  # H rounded to DT
            Wd, w = matrix64(Bd[e], Sd[e]), RW[t, j].double()
            want[t] += w * (h @ Wd)[0]
            bound[t] += w * (dh @ Wd.abs() + 300 * 2.0 ** -23 * (h.abs() @ Wd.abs()))[0]
    for O in outs:
        check(O, want, bound, "T=%d" % T)
    # the ternary experts' layer on the same routing runs
    B2 = torch.randint(0, 2, (E, H // 16, I), generator=g, device="cuda", dtype=torch.int32)
    D2 = torch.randint(0, 2, (E, I // 16, H), generator=g, device="cuda", dtype=torch.int32)
    O2 = torch.ops.ternocl.moe_prefill(X, ids, RW, B2, Sg, B2, Su, D2, Sd, E, topk)
    assert bool(torch.isfinite(O2).all())
    assert tl.device_error() == 0


def test_custom_operators(cuda, tl):
    import ternocl_b200.torch_ops  # noqa: F401
    g = gen(12)
    B, S = weights(g, 512, 256, dtype=torch.float16)
    A = torch.randn(2, 3, 512, generator=g, device="cuda").half()
    C = torch.ops.ternocl.int4_linear(A, B, S)
    assert torch.equal(C.reshape(6, 256), tl.int4_upcvt(A.reshape(6, 512), B, S))
    logits = torch.randn(2, 3, 32, generator=g, device="cuda")
    ids, RW = torch.ops.ternocl.moe_topk(logits, 4)
    ids2, RW2 = tl.moe_topk(logits.reshape(6, 32), 4)
    assert torch.equal(ids.reshape(6, 4), ids2) and torch.equal(RW.reshape(6, 4), RW2)
    for op, args in ((torch.ops.ternocl.int4_linear.default, (A, B, S)),
                     (torch.ops.ternocl.moe_topk.default, (logits, 4))):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


def test_custom_operators_without_tokens(cuda, tl):
    import ternocl_b200.torch_ops  # noqa: F401
    g, E, topk, H, I = gen(2), 4, 2, 256, 128
    X = torch.empty(0, H, dtype=torch.float16, device="cuda")
    ids, RW = torch.ops.ternocl.moe_topk(torch.empty(0, E, device="cuda"), topk, dtype=torch.float16)
    assert ids.shape == RW.shape == (0, topk)
    up, down = weights(g, E, H, I, dtype=torch.float16), weights(g, E, I, H, dtype=torch.float16)
    for op in (torch.ops.ternocl.moe_prefill_int4, torch.ops.ternocl.moe_decode_int4):
        O = op(X, ids, RW, *up, *up, *down, E, topk)
        assert O.shape == X.shape and O.dtype == X.dtype
    assert torch.ops.ternocl.int4_linear(X, up[0][0], up[1][0]).shape == (0, I)


# ------------------------------------------------------------- every kernel and schedule of the linear layer
@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("M,K,N", [
    (9, 128, 4864), (16, 640, 5008), (17, 256, 4880), (24, 1280, 9232),  # 9 to 24 rows, many columns
    (25, 640, 19216), (64, 1280, 19200), (40, 256, 38416),               # a full round of tiles and a split one
    (100, 384, 19216), (300, 256, 19344),
    (512, 640, 8208), (700, 384, 16400), (257, 1152, 37904),             # CTA pairs, odd strips among them
    (1, 17408, 7136), (2, 17408, 7136), (8, 4096, 7136)])                # long ranges per warp
def test_linear_kernels(cuda, tl, bf16, M, K, N):
    linear_case(tl, M + K + N, M, K, N, bf16, 2 if M % 2 else 1, bool(K & 128), 0)
    assert tl.device_error() == 0


@pytest.mark.parametrize("M", [9, 20])
@pytest.mark.parametrize("postop", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("out_f32", [False, True])
def test_linear_epilogues_of_few_rows(cuda, tl, M, postop, out_f32):
    linear_case(tl, M + postop, M, 384, 4912, postop & 1, postop, out_f32, 0)
    linear_case(tl, M + postop, 30 * M, 256, 16400, postop & 1, postop, out_f32, 0)
    assert tl.device_error() == 0


def test_linear_calls_on_two_streams_at_once(cuda, tl):
    """Nothing is shared between calls that overlap: the same results as one after the other."""
    g = gen(13)
    cases = []
    for M, K, N in ((1, 4096, 8192), (16, 1024, 8192), (64, 1024, 4096), (600, 512, 8192)):
        B, S = weights(g, K, N, dtype=torch.float16)
        cases.append((activations(g, M, K, torch.float16), B, (S / K ** 0.5).half()))
    want = [tl.int4_upcvt(*c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] += [tl.int4_upcvt(*c) for c in (cases if k else cases[::-1])]
    torch.cuda.synchronize()
    for k in range(2):
        for i, C in enumerate(got[k]):
            assert torch.equal(C, want[i % 4 if k else 3 - i % 4])
    assert tl.device_error() == 0


def test_linear_residual_in_place(cuda, tl):
    """C may be Other itself (the residual's own buffer)."""
    g = gen(14)
    for M, N in ((1, 512), (6, 512), (16, 5120), (40, 512), (300, 8192)):
        A = activations(g, M, 512, torch.bfloat16)
        B, S = weights(g, 512, N, dtype=torch.bfloat16)
        x = torch.randn(M, N, generator=g, device="cuda").bfloat16()
        want = tl.int4_upcvt(A, B, S, postop=2, other=x)
        tl.int4_upcvt(A, B, S, postop=2, other=x, out=x)
        assert torch.equal(x, want), (M, N)


def test_functions_refuse_what_does_not_fit(cuda, tl):
    g = gen(15)
    B, S = weights(g, 256, 64, dtype=torch.float16)
    A = activations(g, 2, 256, torch.float16)
    ok = tl.int4_upcvt(A, B, S)
    for bad in (dict(A=A.float()), dict(A=A[:, :128].contiguous()), dict(A=A.t()), dict(B=B.long()), dict(B=B[:-1]),
                dict(B=B[:, ::2]), dict(S=S.bfloat16()), dict(S=S[:1]), dict(S=S.cpu()), dict(A=A[0])):
        with pytest.raises((ValueError, TypeError, IndexError)):
            tl.int4_upcvt(**{"A": A, "B": B, "S": S, **bad})
    for bad in (dict(postop=1), dict(postop=2, other=ok.float()), dict(postop=2, other=ok[:1]), dict(postop=3),
                dict(postop=3, bias=ok[0].float()), dict(out=ok.float()), dict(out=ok[:1]), dict(out_f32=True, out=ok)):
        with pytest.raises((ValueError, TypeError)):
            tl.int4_upcvt(A, B, S, **bad)
    with pytest.raises(tl.TernoclError):
        tl.int4_upcvt(A, B, S, postop=7)
    buf = torch.zeros(2 * 64 + 4, dtype=torch.float16, device="cuda")
    with pytest.raises(tl.TernoclError):  # 8-byte aligned only
        tl.int4_upcvt(A, B, S, out=buf[4:132].view(2, 64))
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    Be, Se = B[None], S[None]
    with pytest.raises(ValueError):
        tl.moe_decode_gate_up_int4(ids[:3], A, Be, Se, Be, Se, 1, 2)
    with pytest.raises(ValueError):
        tl.moe_decode_gate_up_int4(ids, A, Be, Se, Be, Se, 2, 2)
    with pytest.raises(ValueError):
        tl.moe_decode_down_sum_int4(ids[:2], A, torch.ones(3, device="cuda").half(), Be, Se, 1, 2)
    with pytest.raises(ValueError):
        tl.moe_gemm_int4(ids, A, Be, Se, 2)
    with pytest.raises(tl.TernoclError):
        tl.moe_gemm_int4(ids, A, Be, Se, 1, postop=3)
