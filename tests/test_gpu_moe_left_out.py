"""Routed rows whose expert id lies outside [0, E) (another device's experts, say): what the routing writes for
them, and that the prefill layers, as the decode ones, take them as contributing nothing."""
import numpy as np
import pytest
import torch

from int4_ref import check, epilogue64, matrix64, product64, weights

pytestmark = pytest.mark.gpu
BAD = (-1, None, 2 ** 31 - 1, -2 ** 31)  # None: E itself


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def some_left_out(rng, T, topk, E):
    """ids [T, topk] with bad ones among them, the last token's all bad."""
    ids = np.stack([rng.permutation(E)[:topk] for _ in range(T)]).astype(np.int64)
    for k, bad in enumerate(BAD):
        ids.reshape(-1)[k::11] = E if bad is None else bad
    ids[-1] = -1
    return ids.astype(np.int32)


def route_by_hand(ids, E, rows_per_tile):
    ids = ids.reshape(-1)
    valid = (ids >= 0) & (ids < E)
    count = np.bincount(ids[valid], minlength=E)
    rows = np.concatenate([[0], np.cumsum(count)])
    tiles = np.concatenate([[0], np.cumsum((count + rows_per_tile - 1) // rows_per_tile)])
    perm, inv = np.full(ids.size, -1), np.full(ids.size, -1)
    order = np.argsort(np.where(valid, ids.astype(np.int64), 2 ** 40), kind="stable")[:rows[-1]]
    perm[:rows[-1]] = order
    inv[order] = np.arange(rows[-1])
    return np.concatenate([rows, tiles]), perm, inv


@pytest.mark.parametrize("T,topk,E", [(5, 4, 8), (128, 8, 16), (129, 8, 16), (700, 6, 256), (1, 1, 1)])
def test_route_gather_combine(cuda, tl, T, topk, E):
    """One CTA (up to 1024 rows) and one CTA per 1024 rows."""
    ids = some_left_out(np.random.default_rng(T), T, topk, E)
    G = T * topk
    tl.device_error(reset=True)
    meta, perm, inv = tl.moe_route(torch.from_numpy(ids.reshape(-1)).cuda(), E)
    assert tl.device_error(reset=True) == 2
    for got, want in zip((meta, perm, inv), route_by_hand(ids, E, tl.moe_rows_per_tile())):
        assert np.array_equal(got.cpu().numpy(), want)
    g = gen(T)
    X = torch.randn(T, 256, generator=g, device="cuda").half()
    token = (perm.long() // topk).clamp(min=0)
    want = torch.where((perm >= 0)[:, None], X[token], torch.zeros_like(X[:1]))
    assert torch.equal(tl.moe_gather(X, perm, topk), want)
    SAt, Xq = tl.int8_quant_a(X)
    Xsq, SA = tl.moe_gather_q(Xq, SAt, perm, topk)
    assert torch.equal(Xsq, torch.where((perm >= 0)[:, None], Xq[token], torch.zeros_like(Xq[:1])))
    assert torch.equal(SA[:, :G], torch.where((perm >= 0)[None], SAt[:, token], torch.zeros_like(SAt[:, :1])))
    Y = torch.randn(G, 64, generator=g, device="cuda")
    Y[int(meta[E]):] = float("nan")  # rows of no expert
    RW = torch.rand(G, generator=g, device="cuda").half()
    O = tl.moe_combine(Y, inv, torch.where(inv >= 0, RW, torch.full_like(RW, float("nan"))), T, topk)
    y = torch.where((inv >= 0)[:, None], Y[inv.long().clamp(min=0)].nan_to_num().double(), 0.0)
    terms = (RW.double()[:, None] * y).view(T, topk, 64)
    check(O, terms.sum(1), (topk + 1) * 2.0 ** -24 * terms.abs().sum(1))
    assert not bool(O[-1].any())


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("T", [6, 150, 700])
def test_int4_layers(cuda, tl, bf16, T):
    """Prompt and single-token layers against 64 bits with the left-out rows not there."""
    import ternocl_b200.torch_ops  # noqa: F401
    g, dt = gen(T), torch.bfloat16 if bf16 else torch.float16
    E, topk, H, I = 16, 4, 512, 256
    ids = some_left_out(np.random.default_rng(T), T, topk, E)
    X = torch.randn(T, H, generator=g, device="cuda").to(dt)
    RW = torch.rand(T, topk, generator=g, device="cuda").to(dt)
    (Bg, Sg), (Bu, Su) = weights(g, E, H, I, dtype=dt), weights(g, E, H, I, dtype=dt)
    Bd, Sd = weights(g, E, I, H, dtype=dt)
    Sg, Su, Sd = (Sg / 16).to(dt), (Su / 16).to(dt), (Sd / 16).to(dt)
    args = (X, torch.from_numpy(ids).cuda(), RW, Bg, Sg, Bu, Su, Bd, Sd, E, topk)
    outs = [torch.ops.ternocl.moe_prefill_int4(*args)]
    if T <= 6:
        outs.append(torch.ops.ternocl.moe_decode_int4(*args))
    assert tl.device_error(reset=True) == 2
    x, eps = X.double(), torch.finfo(dt).eps / 2
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    Wg, Wu, Wd = matrix64(Bg, Sg), matrix64(Bu, Su), matrix64(Bd, Sd)
    for e in range(E):
        t, j = (torch.from_numpy(a).cuda() for a in np.nonzero(ids == e))
        vg, dg = product64(x[t], Wg[e], True)
        vu, du = product64(x[t], Wu[e], True)
        dg, du = 64 * dg, 64 * du + eps * vu.abs()  # (the GEMM's sums, and up rounded to the type)
        h, dh = epilogue64(vg, dg, 1, vu, None, True)
        dh = dh + 1.1 * (vg.abs() + dg) * du
        dh = dh + eps * (h.abs() + dh)  # H rounded to the type
        w = RW[t, j].double()[:, None]
        want.index_add_(0, t, w * (h @ Wd[e]))
        bound.index_add_(0, t, w * (dh @ Wd[e].abs() + 300 * 2.0 ** -23 * (h.abs() @ Wd[e].abs())))
    for O in outs:
        check(O, want, bound, "T=%d" % T)
        assert not bool(O[-1].any())


@pytest.mark.parametrize("int8", [False, True])
def test_ternary_layer(cuda, tl, int8):
    """The ternary prompt layer: bit for bit as if the left-out rows went to one more expert and weighed nothing
    (the others' rows then stand in the same places)."""
    import ternocl_b200.torch_ops  # noqa: F401
    g = gen(3)
    T, E, topk, H, I = 300, 8, 4, 512, 256
    ids = some_left_out(np.random.default_rng(3), T, topk, E)
    valid = (ids >= 0) & (ids < E)
    X = torch.randn(T, H, generator=g, device="cuda").half()
    RW = torch.rand(T, topk, generator=g, device="cuda").half()
    B, D = (torch.randint(-2 ** 31, 2 ** 31, (E + 1, n // 16, m), generator=g, device="cuda").to(torch.int32)
            for n, m in ((H, I), (I, H)))
    S, Sd = (torch.rand(E + 1, n // 128, m, generator=g, device="cuda").half() / 64 for n, m in ((H, I), (I, H)))
    run = torch.ops.ternocl.moe_prefill
    got = run(X, torch.from_numpy(ids).cuda(), RW, B[:E], S[:E], B[:E], S[:E], D[:E], Sd[:E], E, topk, int8)
    assert tl.device_error(reset=True) == 2
    stand_in = torch.from_numpy(np.where(valid, ids, E).astype(np.int32)).cuda()
    RW0 = torch.where(torch.from_numpy(valid).cuda(), RW, torch.zeros_like(RW))
    want = run(X, stand_in, RW0, B, S, B, S, D, Sd, E + 1, topk, int8)
    assert torch.equal(got, want) and bool(got.any()) and not bool(got[-1].any())
    assert tl.device_error() == 0


@pytest.mark.parametrize("T", [2, 150, 2000])
def test_layers_without_any_row(cuda, tl, T):
    """Every id left out: zeros from each layer, whatever the unused rows hold."""
    import ternocl_b200.torch_ops  # noqa: F401
    g = gen(T)
    E, topk, H, I = 4, 2, 256, 128
    X = torch.full((T, H), float("nan"), device="cuda").half()
    ids = torch.full((T, topk), -1, dtype=torch.int32, device="cuda")
    RW = torch.ones(T, topk, device="cuda").half()
    up, down = weights(g, E, H, I, dtype=torch.float16), weights(g, E, I, H, dtype=torch.float16)
    ops = torch.ops.ternocl
    for O in (ops.moe_prefill_int4(X, ids, RW, *up, *up, *down, E, topk),
              ops.moe_decode_int4(X, ids, RW, *up, *up, *down, E, topk)):
        assert bool((O == 0).all())
    up2, down2 = (up[0][:, ::2].contiguous(), up[1]), (down[0][:, ::2].contiguous(), down[1])
    for int8 in (False, True):
        assert bool((ops.moe_prefill(X, ids, RW, *up2, *up2, *down2, E, topk, int8) == 0).all())
    assert tl.device_error(reset=True) == 2
