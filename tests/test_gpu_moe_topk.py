"""The experts' choice on the GPU against its 64-bit definition (int4_ref.topk64): ids equal, weights within
the rounding of their type (the kernel computes them in 64 bits or with a few fp32 operations: 2^-20)."""
import itertools

import numpy as np
import pytest
import torch

from int4_ref import topk64

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def run(tl, logits, topk, dtype=torch.float32, **how):
    ids, w = tl.moe_topk(logits, topk, dtype=dtype, **how)
    T, E = logits.shape
    assert ids.shape == w.shape == (T, topk) and ids.dtype == torch.int32 and w.dtype == dtype
    if how.get("bias") is not None:
        how = {**how, "bias": how["bias"].cpu().numpy()}
    want_ids, want_w = topk64(logits.double().cpu().numpy(), topk, **how)
    got = ids.cpu().numpy()
    assert np.array_equal(got, want_ids), np.argwhere((got != want_ids).any(1))[:4]
    err = np.abs(w.double().cpu().numpy() - want_w)
    info = torch.finfo(dtype)
    assert np.all(err <= np.abs(want_w) * (info.eps / 2 + 2.0 ** -20) + info.tiny * info.eps), err.max()


@pytest.mark.parametrize("T,E,topk", [(1, 1, 1), (1, 8, 8), (5, 31, 4), (3, 33, 32), (130, 64, 6), (77, 100, 1),
                                      (9, 128, 8), (64, 256, 8), (7, 500, 17), (6, 1024, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_shapes(cuda, tl, T, E, topk, scoring, biased):
    g = torch.Generator(device="cuda")
    g.manual_seed(T + E)
    for k, dtype in enumerate(TYPES):
        logits = (2.0 * torch.randn(T, E, generator=g, device="cuda")).to(dtype)
        bias = 0.1 * torch.randn(E, generator=g, device="cuda") if biased else None
        run(tl, logits, topk, dtype=TYPES[(k + E) % 3], bias=bias, scoring=scoring, renormalize=bool(k & 1),
            scale=[1.0, 2.5][k & 1])


@pytest.mark.parametrize("E,n_group,topk_group,topk", [(8, 2, 1, 4), (256, 8, 4, 8), (160, 8, 3, 6), (96, 32, 5, 12),
                                                        (64, 4, 4, 9), (60, 3, 2, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_top", [1, 2])
def test_groups(cuda, tl, E, n_group, topk_group, topk, scoring, group_top):
    g = torch.Generator(device="cuda")
    g.manual_seed(E)
    for biased in (False, True):
        logits = 2.0 * torch.randn(41, E, generator=g, device="cuda")
        bias = 0.1 * torch.randn(E, generator=g, device="cuda") if biased else None
        run(tl, logits, topk, bias=bias, scoring=scoring, n_group=n_group, topk_group=topk_group, group_top=group_top)


def test_ties_go_to_the_lowest_index(cuda, tl):
    for E, dtype in itertools.product((7, 64, 300), TYPES):
        g = torch.Generator(device="cuda")
        g.manual_seed(E)
        logits = torch.randint(-2, 3, (50, E), generator=g, device="cuda").to(dtype)
        logits[0] = 0.0
        logits[1, ::2] = -0.0
        logits[1, 1::2] = 0.0
        for scoring in ("softmax", "sigmoid"):
            run(tl, logits, min(E, 9), scoring=scoring)
            run(tl, logits, min(E, 9), scoring=scoring, bias=torch.zeros(E, device="cuda"))
    run(tl, torch.zeros(3, 32, device="cuda"), 5, n_group=8, topk_group=2, group_top=2, scoring="sigmoid")


def test_masked_and_extreme_logits(cuda, tl):
    inf, nan = float("inf"), float("nan")
    E = 24
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    base = torch.randn(12, E, generator=g, device="cuda")
    base[0] = -inf                       # a row with nothing
    base[1] = nan
    base[2, 3:] = -inf                   # fewer unmasked than topk
    base[3, 5] = nan
    base[4, 7] = inf
    base[5, 2] = base[5, 9] = inf
    base[6] = torch.finfo(torch.float32).min
    base[7] = torch.linspace(-3e38, 3e38, E)
    base[8] = 1e4 * base[8]
    base[9, ::2] = -inf
    bias = torch.zeros(E, device="cuda")
    bias[4], bias[6], bias[8] = -inf, nan, 0.3
    for scoring, renorm in itertools.product(("softmax", "sigmoid"), (False, True)):
        run(tl, base, 8, scoring=scoring, renormalize=renorm)
        run(tl, base[:8], 8, scoring=scoring, renormalize=renorm, n_group=4, topk_group=2, group_top=2)
        run(tl, base[:6], 8, scoring=scoring, renormalize=renorm, bias=bias)
        run(tl, base[:6], 8, scoring=scoring, renormalize=renorm, bias=bias, n_group=6, topk_group=3, group_top=1)
    run(tl, base[:6].half(), 8, dtype=torch.float16)
    for value in (inf, -inf):
        b = torch.zeros(E, device="cuda")
        b[11] = value
        run(tl, torch.randn(5, E, generator=g, device="cuda"), 4, bias=b, scoring="sigmoid")


def test_near_ties_are_told_apart(cuda, tl):
    """Choice values that differ by a few 2^-40 of themselves (equal in 32 bits) keep their 64-bit order."""
    E = 64
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    logits = torch.randn(200, E, generator=g, device="cuda")
    for scoring in ("softmax", "sigmoid"):
        x = logits.double()
        s = torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)
        # the bias that makes the first row's choice values 1 up to the bias's own rounding to 32 bits
        run(tl, logits, 8, bias=(1.0 - s[0]).float(), scoring=scoring)
        # one fp32 step between neighbouring logits
        step = torch.full((4, E), 1.25, device="cuda").view(torch.int32) + torch.randperm(E, device="cuda").int()
        run(tl, step.view(torch.float32), 8, scoring=scoring)
        run(tl, step.view(torch.float32), 8, bias=torch.full((E,), 0.5, device="cuda"), scoring=scoring)


def test_long_batches_streams_and_graphs(cuda, tl):
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    logits = torch.randn(5003, 256, generator=g, device="cuda")
    bias = 0.05 * torch.randn(256, generator=g, device="cuda")
    how = dict(bias=bias, scoring="sigmoid", n_group=8, topk_group=4, group_top=2)
    run(tl, logits, 8, **how)
    ids, w = tl.moe_topk(logits, 8, dtype=torch.bfloat16, **how)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ids2, w2 = tl.moe_topk(logits, 8, dtype=torch.bfloat16, **how)
    side.synchronize()
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    x, i3, w3 = torch.zeros_like(logits), torch.empty_like(ids), torch.empty_like(w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tl.moe_topk(x, 8, ids=i3, out=w3, **how)
    x.copy_(logits)
    graph.replay()
    assert torch.equal(ids, i3) and torch.equal(w, w3)
    assert tl.moe_topk(logits[:0], 8, **how)[0].shape == (0, 8)


@pytest.mark.parametrize("E,topk,scoring,biased,groups", [
    (128, 8, "softmax", False, {}), (128, 15, "sigmoid", True, {}), (16, 4, "softmax", True, {}),
    (500, 6, "softmax", False, {}), (9, 9, "sigmoid", True, {}), (257, 16, "softmax", True, {}),
    (256, 8, "softmax", True, dict(n_group=8, topk_group=4, group_top=2)),
    (96, 6, "sigmoid", False, dict(n_group=12, topk_group=3, group_top=1)),
    (384, 8, "sigmoid", True, dict(n_group=3, topk_group=2, group_top=2))])
def test_many_tokens(cuda, tl, E, topk, scoring, biased, groups):
    """Batches long enough for the form with two tokens per warp (an odd number of them)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(E)
    for dtype in TYPES:
        logits = (2.0 * torch.randn(2051, E, generator=g, device="cuda")).to(dtype)
        logits[5] = float("-inf")
        logits[6, : E // 2] = float("nan")
        logits[7, 3] = float("inf")
        logits[-1] = 0.5
        bias = 0.1 * torch.randn(E, generator=g, device="cuda") if biased else None
        run(tl, logits, topk, bias=bias, scoring=scoring, renormalize=dtype != torch.float16, **groups)


@pytest.mark.parametrize("T,E", [(70, 1024), (70, 512), (2050, 512), (2050, 300)])
def test_near_ties_behind_a_sum_of_many_small_terms(cuda, tl, T, E):
    """A softmax of one large and 31 small terms, each below half a step of the running sum in 32 bits: an expert
    whose choice value lies within the sum of what those additions lose comes out as in 64 bits."""
    g = torch.Generator(device="cuda")
    g.manual_seed(E)
    logits = torch.full((T, E), -100.0, device="cuda")
    logits[:, 0] = 0.0
    logits[:, 1:32] = -15.9 - 3.0 * torch.rand(T, 31, generator=g, device="cuda")
    logits[0, 1:32] = float(np.log(2.0 ** -24))
    logits[1, 1:32] = -16.62
    bias = torch.full((E,), -5.0, device="cuda")
    bias[0], bias[100] = -1.0, -1.5e-6
    for renorm in (False, True):
        run(tl, logits, 1, bias=bias, renormalize=renorm)
        run(tl, logits, 3, bias=bias, renormalize=renorm)
    bias = torch.zeros(E, device="cuda")
    bias[40] = 1.0 - 33 * 2.0 ** -24
    run(tl, logits, 1, bias=bias, renormalize=False)


@pytest.mark.parametrize("T", [300, 2500])
@pytest.mark.parametrize("per", [2, 4])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_group_scores_whose_biases_cancel(cuda, tl, T, per, scoring):
    """Groups whose two best biases are 1000 and -1000: their scores are small and of what 32 bits lose of the
    two choice values."""
    g = torch.Generator(device="cuda")
    g.manual_seed(per)
    n_group = 4
    logits = 2e-4 * torch.randn(T, per * n_group, generator=g, device="cuda")
    bias = torch.full((n_group, per), float("-inf"), device="cuda")
    bias[:, 0] = 1000.0 + 0.25 * torch.arange(n_group)
    bias[:, 1] = -bias[:, 0]
    run(tl, logits, 2, bias=bias.reshape(-1), scoring=scoring, n_group=n_group, topk_group=1, group_top=2)


@pytest.mark.parametrize("T", [5, 2100])
def test_chosen_scores_at_the_end_of_32_bits(cuda, tl, T):
    """All chosen scores so small that 32 bits hold them as 0 or with few bits: their ratios are the weights."""
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    for E, groups in ((24, {}), (32, dict(n_group=8, topk_group=3, group_top=2))):
        noise = torch.rand(T, E, generator=g, device="cuda")
        for level in (-70.0, -88.0, -89.0, -100.0, -104.0, -150.0, -700.0):
            for dtype in TYPES:  # sigmoids far below 0
                logits = (level + noise).to(dtype)
                run(tl, logits, 8, scoring="sigmoid", **groups)
                run(tl, logits, 8, scoring="sigmoid", bias=torch.rand(E, generator=g, device="cuda"), **groups)
        logits = torch.full((T, 8), -100.0, device="cuda")
        assert bool((tl.moe_topk(logits, 8, scoring="sigmoid", scale=2.0)[1] == 0.25).all())


@pytest.mark.parametrize("T", [5, 2100])
@pytest.mark.parametrize("below", [50.0, 90.0, 110.0, 600.0])
def test_chosen_scores_far_below_the_softmax_maximum(cuda, tl, T, below):
    """A bias, or the choice of groups, leaves out the row's largest logit."""
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    E = 16
    # whole multiples of 1/8, so that every difference is exact in 32 bits
    logits = -below + 0.125 * torch.randint(0, 16, (T, E), generator=g, device="cuda")
    logits[:, 0] = 0.0
    bias = torch.rand(E, generator=g, device="cuda")
    bias[0] = -10.0
    for renorm in (False, True):
        run(tl, logits, 4, bias=bias, renormalize=renorm)
        # group 0 has no second unmasked expert
        alone = logits.clone()
        alone[:, 1:4] = float("-inf")
        run(tl, alone, 4, n_group=4, topk_group=2, group_top=2, renormalize=renorm)
        run(tl, alone, 4, bias=bias, n_group=4, topk_group=2, group_top=2, renormalize=renorm)


@pytest.mark.parametrize("T", [5, 2100])
@pytest.mark.parametrize("E,biased", [(64, False), (64, True), (600, False)])
def test_weights_of_logits_far_apart(cuda, tl, T, E, biased):
    """Logits tens below the largest one: their difference to it is rounded in 32 bits, their weight is not off by
    that rounding."""
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    logits = 65.0 * torch.rand(T, E, generator=g, device="cuda")
    bias = torch.rand(E, generator=g, device="cuda") if biased else None
    for renorm in (False, True):
        run(tl, logits, 12, bias=bias, renormalize=renorm)
        run(tl, logits - 1000.0, 12, bias=bias, renormalize=renorm)
