"""The 4-bit experts' layers from router logits as a server runs them: with programmatic dependent launch, captured
into a graph and replayed on new inputs, and on two streams at once: the bits of plain calls."""
import pytest
import torch

from int4_ref import weights

pytestmark = pytest.mark.gpu
E, TOPK, H, I = 16, 4, 512, 256


def layer(T, X, logits, bias, up, gate, down):
    ops = torch.ops.ternocl
    ids, RW = ops.moe_topk(logits, TOPK, bias=bias, scoring="sigmoid", n_group=4, topk_group=2, group_top=2,
                           dtype=X.dtype)
    op = ops.moe_decode_int4 if T <= 6 else ops.moe_prefill_int4
    return op(X, ids, RW, *gate, *up, *down, E, TOPK)


def case(T, seed, dtype=torch.bfloat16):
    import ternocl_b200.torch_ops  # noqa: F401
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    X = torch.randn(T, H, generator=g, device="cuda").to(dtype)
    logits = torch.randn(T, E, generator=g, device="cuda")
    bias = 0.1 * torch.randn(E, generator=g, device="cuda")
    mats = []
    for k, n in ((H, I), (H, I), (I, H)):
        B, S = weights(g, E, k, n, dtype=dtype)
        mats.append((B, (S / 16).to(dtype)))
    return [X, logits, bias, *mats]


@pytest.mark.parametrize("T", [1, 6, 20, 150, 1100])
def test_layer_under_pdl(cuda, tl, T):
    args = case(T, T)
    x = want = args[0]
    for _ in range(4):
        want = layer(T, want, *args[1:])
    old = tl.set_option(tl.OPT_PDL, 1)
    try:
        for _ in range(4):
            x = layer(T, x, *args[1:])
    finally:
        tl.set_option(tl.OPT_PDL, old)
    assert torch.equal(x, want) and bool(x.any())
    assert tl.device_error() == 0


@pytest.mark.parametrize("T", [1, 6, 20, 150, 1100])
@pytest.mark.parametrize("pdl", [0, 1])
def test_layer_captured(cuda, tl, T, pdl):
    a, b = case(T, 2 * T + 1), case(T, 2 * T + 1)
    b[0], b[1] = b[0].flip(0).contiguous() * 0.5, b[1].flip(1).contiguous()
    want = [layer(T, *a), layer(T, *b)]
    X, logits = torch.zeros_like(a[0]), torch.zeros_like(a[1])
    old = tl.set_option(tl.OPT_PDL, pdl)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(T, X, logits, *a[2:])
    finally:
        tl.set_option(tl.OPT_PDL, old)
    for src, w in ((a, want[0]), (b, want[1]), (a, want[0])):
        X.copy_(src[0])
        logits.copy_(src[1])
        out.zero_()
        graph.replay()
        assert torch.equal(out, w)
    assert tl.device_error() == 0


def test_layers_on_two_streams_at_once(cuda, tl):
    cases = [(T, case(T, T)) for T in (1, 6, 150, 1100)]
    want = [layer(T, *c) for T, c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] += [(i, layer(cases[i][0], *cases[i][1])) for i in (range(4) if k else (3, 2, 1, 0))]
    torch.cuda.synchronize()
    for i, out in got[0] + got[1]:
        assert torch.equal(out, want[i])
    assert tl.device_error() == 0
