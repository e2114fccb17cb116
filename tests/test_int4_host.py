"""4-bit weights and the experts' choice without a GPU: the packer, what the C ABI and the Python functions
refuse, and the custom operators' shapes."""
import ctypes

import numpy as np
import pytest
import torch

import ternocl_b200 as tl
import ternocl_b200.torch_ops  # noqa: F401
from int4_ref import codes64, topk64


def test_pack_round_trip_and_refusals():
    rng = np.random.default_rng(0)
    codes = rng.integers(-8, 8, (128, 48))
    words = tl.int4_pack(codes)
    assert words.shape == (16, 48) and words.dtype == np.uint32
    assert np.array_equal(codes64(torch.from_numpy(words.view(np.int32))).numpy(), codes)
    assert tl.int4_pack(np.arange(8).reshape(8, 1))[0, 0] == 0x76543210
    for bad in (8, -9):
        with pytest.raises(ValueError):
            tl.int4_pack(np.full((8, 1), bad))
    L = tl.lib()
    c8 = np.full((8, 2), 9, np.int8)
    out = np.zeros((1, 2), np.uint32)
    assert L.ternocl_int4_pack(c8.ctypes.data, 8, 2, out.ctypes.data) == 2
    assert L.ternocl_int4_pack(c8.ctypes.data, 7, 2, out.ctypes.data) == 1
    assert L.ternocl_int4_pack(None, 8, 2, out.ctypes.data) == 2


def test_pack_refuses_codes_that_are_not_integers():
    for codes in (np.full((128, 16), 1.5), np.zeros((128, 16), bool), torch.zeros(128, 16)):
        with pytest.raises(TypeError):
            tl.int4_pack(codes)


def test_sizes_that_would_leave_32_bits_are_refused():
    """Refused on the host, before any pointer is read."""
    L, p = tl.lib(), ctypes.c_void_p(64)
    N, T = 2 ** 31 - 16, 2 ** 31 - 1
    assert L.ternocl_int4_upcvt(p, p, p, p, None, None, 1, N, 128, 0, 0, 0, 0, None) == 1
    assert L.ternocl_moe_gemm_int4(p, p, p, p, p, None, 1, N, 128, 1, 0, 0, 0, None) == 1
    assert L.ternocl_moe_decode_gate_up_int4(p, p, p, p, p, p, p, 1, N, 128, 1, 1, 0, None) == 1
    assert L.ternocl_moe_decode_down_sum_int4(p, p, p, p, p, p, 1, N, 128, 1, 1, 0, None) == 1
    assert L.ternocl_moe_topk(p, None, p, p, T, 1, 1, 0, 1, 1, 1, 0, 1.0, 2, 2, None) == 1


def test_c_abi_refusals():
    L = tl.lib()
    p, q = ctypes.c_void_p(64), ctypes.c_void_p(66)  # never dereferenced
    f = L.ternocl_int4_upcvt

    def linear(A=p, B=p, S=p, C=p, other=None, bias=None, M=1, N=48, K=128, dtype=0, postop=0, f32=0, algo=0):
        return f(A, B, S, C, other, bias, M, N, K, dtype, postop, f32, algo, None)

    assert linear(N=40) == 1 and linear(K=100) == 1 and linear(M=-1) == 1 and linear(N=0) == 1
    assert linear(M=524281) == 1
    assert linear(dtype=2) == 2 and linear(postop=5) == 2 and linear(algo=3) == 2 and linear(f32=2) == 2
    assert linear(A=None) == 2 and linear(A=q) == 2 and linear(B=q) == 2 and linear(S=q) == 2 and linear(C=q) == 2
    assert linear(postop=1) == 2 and linear(postop=2) == 2 and linear(postop=3) == 2
    assert linear(M=0) == 0
    g = L.ternocl_moe_gemm_int4
    assert g(None, p, p, p, p, None, 1, 48, 128, 4, 0, 0, 0, None) == 2
    assert g(p, p, p, p, p, None, 1, 48, 128, 0, 0, 0, 0, None) == 2
    assert g(p, p, p, p, p, None, 1, 48, 128, 1025, 0, 0, 0, None) == 2
    assert g(p, p, p, p, p, None, 1, 48, 128, 4, 0, 3, 0, None) == 2
    assert g(p, p, p, p, p, None, 1, 48, 100, 4, 0, 0, 0, None) == 1
    assert g(p, p, p, p, p, None, (1 << 20) + 1, 48, 128, 4, 0, 0, 0, None) == 1
    u = L.ternocl_moe_decode_gate_up_int4
    assert u(p, p, p, p, p, p, p, 5, 48, 128, 2, 4, 0, None) == 1  # G % topk
    assert u(p, p, p, p, p, p, p, 4, 40, 128, 2, 4, 0, None) == 1
    assert u(p, p, p, p, p, p, p, 4, 48, 128, 2, 0, 0, None) == 1
    assert u(p, q, p, p, p, p, p, 4, 48, 128, 2, 4, 0, None) == 2
    assert u(p, p, p, p, p, p, p, 4, 48, 128, 2, 4, 2, None) == 2
    assert u(p, p, p, p, p, p, p, 2 ** 30, 2 ** 20, 128, 2, 4, 0, None) == 1
    d = L.ternocl_moe_decode_down_sum_int4
    assert d(p, p, None, p, p, p, 4, 48, 128, 2, 4, 0, None) == 2
    assert d(p, p, p, p, p, p, 4, 48, 120, 2, 4, 0, None) == 1
    assert d(p, p, p, p, p, p, 2 ** 30, 48, 128, 2 ** 20, 4, 0, None) == 1


def test_topk_refusals():
    L = tl.lib()
    p, q = ctypes.c_void_p(64), ctypes.c_void_p(65)

    def f(logits=p, bias=None, ids=p, RW=p, T=1, E=64, topk=4, scoring=0, n_group=1, topk_group=1, group_top=1,
          renorm=1, scale=1.0, ldt=2, wdt=2):
        return L.ternocl_moe_topk(logits, bias, ids, RW, T, E, topk, scoring, n_group, topk_group, group_top, renorm,
                                  scale, ldt, wdt, None)

    assert f(T=0) == 0
    for bad in (dict(T=-1), dict(E=0), dict(E=1025), dict(topk=0), dict(topk=33), dict(E=3), dict(n_group=0),
                dict(n_group=33), dict(n_group=5), dict(n_group=8, topk_group=9), dict(topk_group=0),
                dict(n_group=32, topk_group=1), dict(group_top=3), dict(group_top=0),
                dict(n_group=32, E=32, topk=1, group_top=2)):
        assert f(**bad) == 1, bad
    for bad in (dict(scoring=2), dict(renorm=2), dict(ldt=3), dict(wdt=-1), dict(logits=None), dict(ids=None),
                dict(RW=None), dict(logits=q), dict(RW=q), dict(bias=q)):
        assert f(**bad) == 2, bad


def test_python_refuses_host_tensors_and_unknown_scoring():
    A, B, S = torch.zeros(1, 128).half(), torch.zeros(16, 16, dtype=torch.int32), torch.zeros(1, 16).half()
    with pytest.raises(ValueError):
        tl.int4_upcvt(A, B, S)
    with pytest.raises(ValueError):
        tl.moe_topk(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError):
        tl.moe_topk(torch.zeros(2, 8), 2, scoring="relu")
    with pytest.raises(TypeError):
        tl.moe_topk(torch.zeros(2, 8, dtype=torch.float64), 2)


def test_custom_operator_shapes():
    m = "meta"
    A = torch.empty(3, 5, 4096, dtype=torch.bfloat16, device=m)
    B, S = torch.empty(512, 6144, dtype=torch.int32, device=m), torch.empty(32, 6144, dtype=torch.bfloat16, device=m)
    C = torch.ops.ternocl.int4_linear(A, B, S, 0, True)
    assert C.shape == (3, 5, 6144) and C.dtype == torch.float32
    ids, RW = torch.ops.ternocl.moe_topk(torch.empty(3, 5, 64, device=m), 6, dtype=torch.float16)
    assert ids.shape == RW.shape == (3, 5, 6) and ids.dtype == torch.int32 and RW.dtype == torch.float16
    X, ids = torch.empty(9, 2048, dtype=torch.float16, device=m), torch.empty(9, 8, dtype=torch.int32, device=m)
    W = torch.empty(1, device=m)
    for op in (torch.ops.ternocl.moe_prefill_int4, torch.ops.ternocl.moe_decode_int4):
        assert op(X, ids, W, W, W, W, W, W, W, 16, 8).shape == X.shape


def test_prefill_layer_refuses_routing_that_does_not_fit():
    """Refused before anything is launched: ids and weights that are too few, too many or of another type would be
    read as other memory or as other numbers."""
    T, E, topk, H, I = 6, 4, 2, 256, 128
    X = torch.zeros(T, H).half()
    ids, RW = torch.zeros(T, topk, dtype=torch.int32), torch.zeros(T, topk).half()
    up = torch.zeros(E, H // 8, I, dtype=torch.int32), torch.zeros(E, H // 128, I).half()
    down = torch.zeros(E, I // 8, H, dtype=torch.int32), torch.zeros(E, I // 128, H).half()
    wide = torch.zeros(E, I // 8, 2 * H, dtype=torch.int32), torch.zeros(E, I // 128, 2 * H).half()
    op = torch.ops.ternocl.moe_prefill_int4
    for kind, what, args in (
            (ValueError, "entries", (ids[:-1], RW)), (ValueError, "entries", (ids.repeat(2, 1), RW)),
            (ValueError, "entries", (ids, RW[:, :1])), (ValueError, "entries", (ids, RW.repeat(1, 2))),
            (TypeError, "int32", (ids.long(), RW)), (TypeError, "int32", (ids, RW.float())),
            (TypeError, "int32", (ids, RW.bfloat16()))):
        with pytest.raises(kind, match=what):
            op(X, *args, *up, *up, *down, E, topk)
    with pytest.raises(ValueError, match="entries"):
        op(X, ids[:, :0], RW[:, :0], *up, *up, *down, E, 0)
    with pytest.raises(ValueError, match="lead back"):
        op(X, ids, RW, *up, *up, *wide, E, topk)


def test_prefill_layer_runs_on_the_device_of_its_inputs(monkeypatch):
    """Every launch of the layer, also when another device is current."""
    current, entered = [None], []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)
            current[0] = self.device

        def __exit__(self, *_):
            current[0] = None

    T, E, topk, H, I = 6, 4, 2, 256, 128
    X = torch.zeros(T, H).half()

    def stub(out):
        def f(*args, **kw):
            assert current[0] == X.device
            return out
        return f

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(tl, "moe_route", stub((None, None, None)))
    for name in ("moe_gather", "moe_gemm_int4"):
        monkeypatch.setattr(tl, name, stub(X))
    monkeypatch.setattr(tl, "moe_combine", stub(X.clone()))
    up = torch.zeros(E, H // 8, I, dtype=torch.int32), torch.zeros(E, H // 128, I).half()
    down = torch.zeros(E, I // 8, H, dtype=torch.int32), torch.zeros(E, I // 128, H).half()
    ids, RW = torch.zeros(T, topk, dtype=torch.int32), torch.zeros(T, topk).half()
    torch.ops.ternocl.moe_prefill_int4(X, ids, RW, *up, *up, *down, E, topk)
    assert entered == [X.device]


def test_reference_choice_by_hand():
    """The 64-bit definition on a case small enough to do by hand."""
    ids, w = topk64([[0.0, 1.0, 1.0, -1.0]], 2, scoring="sigmoid", renormalize=False)
    assert ids.tolist() == [[1, 2]] and np.allclose(w, 1 / (1 + np.exp(-1.0)))
    ids, w = topk64([[0.0, 1.0, 2.0, 3.0]], 2, bias=[9.0, 0, 0, 0], n_group=2, topk_group=1)
    assert ids.tolist() == [[0, 1]]  # the first group holds the best biased score
    e = np.exp([0.0, 1.0])
    assert np.allclose(w[0], e / e.sum())
    ids, w = topk64([[np.nan, -np.inf, 5.0]], 3)
    assert ids.tolist() == [[2, 0, 1]] and np.allclose(w, [[1, 0, 0]])
