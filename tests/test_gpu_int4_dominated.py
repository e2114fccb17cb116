"""Activations of very different sizes in a few rows: every product is as exact as a 16-bit MMA with fp32 sums
makes it (int4_ref.product64 without digits), in columns too whose weights leave the large ones out."""
import pytest
import torch

from int4_ref import check, codes64, epilogue64, matrix64, product64, weights

pytestmark = pytest.mark.gpu
DT = {0: torch.float16, 1: torch.bfloat16}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def dominated(g, M, K, dtype, large, small=0.01):
    """Values around `small`, one of `large` in every row (and one in between)."""
    a = small * torch.randn(M, K, generator=g, device="cuda")
    at = torch.randint(0, K, (M, 2), generator=g, device="cuda")
    a.scatter_(1, at, torch.tensor([(large * small) ** 0.5, large], device="cuda").expand(M, 2))
    return a.to(dtype)


def some_zero_codes(g, B):
    """Half of the codes 0."""
    keep = torch.randint(0, 2, (*B.shape, 8), generator=g, device="cuda")
    mask = (keep * (15 << (4 * torch.arange(8, device="cuda")))).sum(-1)
    return (B.long() & mask).to(torch.int32)


def check_in_range(got, want, bound, what):
    """check() of the elements that the type can hold (2000 x 7 x 0.05 of a gate times as much of an up is 4.9e5,
    beyond fp16's 65504)."""
    fits = (want.abs() + bound) * (1.0 + torch.finfo(got.dtype).eps) < torch.finfo(got.dtype).max
    check(got[fits], want[fits], bound[fits], what)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("large", [20.0, 2000.0, 60000.0])
@pytest.mark.parametrize("M,K,N", [(1, 128, 272), (1, 4096, 528), (1, 17408, 144), (1, 17408, 7136), (2, 128, 272),
                                   (2, 4096, 528), (2, 17408, 144)])
def test_linear(cuda, tl, bf16, large, M, K, N):
    g, dt = gen(K), DT[bf16]
    A = dominated(g, M, K, dt, large)
    B, S = weights(g, K, N, dtype=dt)
    B = some_zero_codes(g, B)
    C = tl.int4_upcvt(A, B, S, out_f32=True)
    check(C, *product64(A, matrix64(B, S), False), "large %g" % large)
    rows = A.abs().amax(1, keepdim=True) == A.abs()
    assert bool((codes64(B)[rows.any(0)] == 0).any()) and tl.device_error() == 0


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("weight", [0.0, 2.0 ** -14])
@pytest.mark.parametrize("T,topk,K", [(64, 8, 128), (1, 5, 768), (64, 8, 768), (1, 3, 4096)])
def test_down_sum_of_one_expert_with_a_large_row(cuda, tl, bf16, weight, T, topk, K):
    """A token's rows of H each in values of one size, the first's 2^20 times the others' and weighing (almost)
    nothing: the others' products keep their bits."""
    g, dt, E, N = gen(T * K), DT[bf16], 5, 144
    H = torch.randint(1, 128, (T * topk, K), generator=g, device="cuda").double()
    H *= torch.where(torch.rand(H.shape, generator=g, device="cuda") < 0.5, 1.0, -1.0) * 2.0 ** -14
    H[::topk] *= 2.0 ** 20
    H = H.to(dt)
    ids = torch.randint(0, E, (T * topk,), generator=g, device="cuda", dtype=torch.int32)
    RW = torch.rand(T * topk, generator=g, device="cuda").to(dt)
    RW[::topk] = weight
    B, S = weights(g, E, K, N, dtype=dt)
    O = tl.moe_decode_down_sum_int4(ids, H, RW, B, S, E, topk)
    for t in range(T):
        rows = range(t * topk, (t + 1) * topk)
        W = torch.cat([matrix64(B[ids[r]], S[ids[r]]) * RW[r].double() for r in rows])
        check(O[t][None], *product64(H[list(rows)].reshape(1, -1), W, False), "token %d" % t)
    assert tl.device_error() == 0


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("large", [20.0, 2000.0])
@pytest.mark.parametrize("T,topk,K,N", [(1, 4, 128, 48), (2, 3, 2048, 272), (40, 2, 640, 272)])
def test_experts(cuda, tl, bf16, large, T, topk, K, N):
    """gate_up and down_sum on such rows, every expert's weights half zeros."""
    g, dt, E = gen(K), DT[bf16], 4
    ids = torch.argsort(torch.rand(T, E, generator=g, device="cuda"), dim=1)[:, :topk].to(torch.int32).reshape(-1)
    (Bg, Sg), (Bu, Su) = weights(g, E, K, N, dtype=dt), weights(g, E, K, N, dtype=dt)
    Bg, Bu = some_zero_codes(g, Bg), some_zero_codes(g, Bu)
    X, H = dominated(g, T, K, dt, large), dominated(g, T * topk, K, dt, large)
    got = tl.moe_decode_gate_up_int4(ids, X, Bg, Sg, Bu, Su, E, topk)
    RW = torch.rand(T * topk, generator=g, device="cuda").to(dt)
    O = tl.moe_decode_down_sum_int4(ids, H, RW, Bg, Sg, E, topk)
    for t in range(T):
        rows = list(range(t * topk, (t + 1) * topk))
        for r in rows:
            vg, dg = product64(X[t][None], matrix64(Bg[ids[r]], Sg[ids[r]]), False)
            vu, du = product64(X[t][None], matrix64(Bu[ids[r]], Su[ids[r]]), False)
            want, bound = epilogue64(vg, dg, 1, vu, None, True)
            check_in_range(got[r][None], want, bound + 1.1 * (vg.abs() + dg) * du, "row %d" % r)
        W = torch.cat([matrix64(Bg[ids[r]], Sg[ids[r]]) * RW[r].double() for r in rows])
        check(O[t][None], *product64(H[rows].reshape(1, -1), W, False), "token %d" % t)
    assert tl.device_error() == 0


def wide(g, M, K, bf16):
    """Groups of every kind side by side: values of one size, zeros, exponents from one end of the type to the
    other, the lowest ones only (subnormals), a few values among zeros."""
    low, high = (-60, 20) if bf16 else (-24, 10)
    a = torch.randn(M, K // 128, 128, generator=g, device="cuda").double()
    kind = torch.randint(0, 6, (M, K // 128, 1), generator=g, device="cuda")
    scale = torch.randint(low, high, a.shape, generator=g, device="cuda").double()
    a = torch.where(kind == 1, torch.zeros_like(a), a)
    a = torch.where(kind == 2, a * 2.0 ** scale, a)
    a = torch.where(kind == 3, a * 2.0 ** (-130 if bf16 else -22), a)
    a = torch.where((kind == 4) & (torch.rand(a.shape, generator=g, device="cuda") < 0.97), torch.zeros_like(a), a)
    return a.reshape(M, K).to(DT[bf16])


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("K,N", [(128, 48), (2048, 272), (16384, 144), (17408, 7136)])
def test_linear_of_every_kind_of_group(cuda, tl, bf16, K, N):
    g, dt = gen(K), DT[bf16]
    for seed in range(4):
        A = wide(g, 1, K, bf16)
        B, S = weights(g, K, N, dtype=dt)
        check(tl.int4_upcvt(A, B, S, out_f32=True), *product64(A, matrix64(B, S), False), "try %d" % seed)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("T,topk,K", [(1, 1, 2048), (3, 4, 640), (30, 4, 2176)])
def test_experts_of_every_kind_of_group(cuda, tl, bf16, T, topk, K):
    """down_sum, some experts left out; gate_up with an up matrix that passes the gate's sums on."""
    g, dt, E, N = gen(K), DT[bf16], 5, 144
    H = wide(g, T * topk, K, bf16)
    ids = torch.randint(-1, E, (T * topk,), generator=g, device="cuda", dtype=torch.int32)
    RW = torch.rand(T * topk, generator=g, device="cuda").to(dt)
    B, S = weights(g, E, K, N, dtype=dt)
    O = tl.moe_decode_down_sum_int4(ids, H, RW, B, S, E, topk)
    for t in range(T):
        rows = list(range(t * topk, (t + 1) * topk))
        W = torch.cat([matrix64(B[ids[r]], S[ids[r]]) * (RW[r].double() if ids[r] >= 0 else 0.0) for r in rows])
        check(O[t][None], *product64(H[rows].reshape(1, -1), W, False), "token %d" % t)
    ids, X, up = ids.clamp(min=0), wide(g, T, K, bf16), weights(g, E, K, N, dtype=dt)
    tl.device_error(reset=True)
    S2 = (S / 2 ** 10).to(dt)
    got = tl.moe_decode_gate_up_int4(ids, X, B, S2, *up, E, topk)
    for r, e in enumerate(ids.tolist()):
        vg, dg = product64(X[r // topk][None], matrix64(B[e], S2[e]), False)
        vu, du = product64(X[r // topk][None], matrix64(up[0][e], up[1][e]), False)
        want, bound = epilogue64(vg, dg, 1, vu, None, True)
        check_in_range(got[r][None], want, bound + 1.1 * (vg.abs() + dg) * du, "row %d" % r)
    assert tl.device_error() == 0


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_one_row_with_a_value_that_is_not_finite(cuda, tl, bf16, bad):
    """It reaches every column whose weight there is not 0."""
    g, dt, K, N = gen(1), DT[bf16], 4096, 272
    B, S = weights(g, K, N, dtype=dt)
    A = torch.randn(1, K, generator=g, device="cuda").to(dt)
    A[0, 777] = bad
    C = tl.int4_upcvt(A, B, S, out_f32=True)
    assert not bool(torch.isfinite(C[0][codes64(B)[777] != 0]).any())
