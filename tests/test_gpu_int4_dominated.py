"""Activations of very different sizes in a few rows: every product is as exact as a 16-bit MMA with fp32 sums
makes it (int4_ref.product64 without digits), in columns too whose weights leave the large ones out."""
import pytest
import torch

from int4_ref import check, codes64, matrix64, product64, weights

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


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("large", [20.0, 2000.0, 60000.0])
@pytest.mark.parametrize("M,K,N", [(2, 128, 272), (2, 4096, 528), (2, 17408, 144)])
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
