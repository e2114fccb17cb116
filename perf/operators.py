"""Cases of the 4-bit-weight and routing operators: their inputs, plain forms and 64-bit definitions.

Five operators: the experts' choice from router logits (moe_topk), the product with 4-bit weights and
scales per 128 rows (int4_upcvt), and the same product inside a mixture-of-experts layer: one row per
routed pair for single tokens (moe_decode_gate_up_int4, moe_decode_down_sum_int4) and over rows sorted
by expert for prompts (moe_gemm_int4).

`own` false: run() computes in elementary torch operations, in 32 bits (64 for the choice of the
experts, where 32 would turn near values into ties), rounded once at the end.  `own` true: run()
makes the calls a user makes of ternocl_b200.
"""
import math

import numpy as np
import torch

own = False

GROUP = 128  # weight rows that share a scale
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one token's routing: 256 experts in 8 groups, sigmoid scores with a balance bias (latency)
        dict(name="topk token", op="topk", T=1, E=256, topk=8, scoring="sigmoid", bias=True, n_group=8,
             topk_group=4, group_top=2, renorm=True, scale=2.5, logits="fp32", dtype="bf16"),
        # a long prompt batch's routing: 128 experts, softmax, 16-bit logits (many equal ones)
        dict(name="topk prompts", op="topk", T=16381, E=128, topk=8, scoring="softmax", bias=False, n_group=1,
             topk_group=1, group_top=1, renorm=True, scale=1.0, logits="bf16", dtype="fp16"),
        # one token through an 8B model's joined gate and up projection
        dict(name="int4 token", op="int4", M=1, K=4096, N=28672, dtype="bf16", postop=0, out_f32=False),
        # a decode batch through a 27B model's gate projection, SwiGLU fused
        dict(name="int4 batch", op="int4", M=24, K=5376, N=21504, dtype="fp16", postop=1, out_f32=False),
        # two streams' logits from a 27B model's output head, in fp32
        dict(name="int4 head", op="int4", M=2, K=5120, N=248320, dtype="bf16", postop=0, out_f32=True),
        # a ragged prompt through an 8B model's down projection, residual fused
        dict(name="int4 prompt", op="int4", M=2047, K=14336, N=4096, dtype="bf16", postop=2, out_f32=False),
        # one token through the experts: gate and up of its 8 experts of 128
        dict(name="gate_up token", op="gate_up", T=1, topk=8, E=128, K=2048, N=768, dtype="fp16"),
        # a small decode batch of the same layer
        dict(name="gate_up batch", op="gate_up", T=9, topk=8, E=128, K=2048, N=768, dtype="bf16"),
        # the way back of the same layer
        dict(name="down_sum token", op="down_sum", T=1, topk=8, E=128, K=768, N=2048, dtype="bf16"),
        dict(name="down_sum batch", op="down_sum", T=9, topk=8, E=128, K=768, N=2048, dtype="fp16"),
        # a larger decode batch's routed rows, a few for each expert
        dict(name="moe_gemm batch", op="moe_gemm", T=67, topk=8, E=128, K=2048, N=768, dtype="bf16", postop=0,
             out_f32=False),
        # a prompt's routed rows through the gate projection, SwiGLU fused
        dict(name="moe_gemm prompt", op="moe_gemm", T=4096, topk=8, E=128, K=2048, N=768, dtype="fp16", postop=1,
             out_f32=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["topk", "int4", "int4", "gate_up", "down_sum", "moe_gemm"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "topk":
        n_group = rng.choice([1, 1, 2, 4, 8])
        per = _log(rng, 4 if n_group > 1 else 8, 512 // n_group)
        topk_group = rng.randint(1, n_group)
        return dict(op=op, T=_log(rng, 1, 16384), E=per * n_group, topk=rng.randint(1, min(16, per * topk_group)),
                    scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, n_group=n_group,
                    topk_group=topk_group, group_top=rng.choice([1, 2]), renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), logits=rng.choice(["fp32", "bf16", "fp16"]),
                    dtype=rng.choice(["fp16", "bf16", "fp32"]))
    if op == "int4":
        M = _log(rng, 1, 2048)
        K = GROUP * _log(rng, 1, 112)
        N = 16 * _log(rng, 1, max(1, min(4096, int(2.3e11 / (2.0 * M * K * 16)))))
        return dict(op=op, M=M, K=K, N=N, dtype=dtype, postop=rng.randint(0, 4), out_f32=rng.random() < 0.3)
    E = _log(rng, 2, 160)
    topk = rng.randint(1, min(8, E))
    K = GROUP * _log(rng, 1, 16)
    N = 16 * _log(rng, 1, 128)
    if op == "moe_gemm":
        return dict(op=op, T=_log(rng, 1, 4096), topk=topk, E=E, K=K, N=min(N, 768), dtype=dtype,
                    postop=rng.choice([0, 1, 2, 4]), out_f32=rng.random() < 0.4)
    return dict(op=op, T=_log(rng, 1, 12), topk=topk, E=E, K=K, N=N, dtype=dtype)


# ----------------------------------------------------------------------------------- the inputs
def _weights(g, shape, dtype):
    """Packed 4-bit weights int32 [..., K/8, N] (row 8i+j at bits 4j) and scales [..., K/128, N]:
    rounded normal values as of weights divided by a group's largest over 7."""
    *lead, K, N = shape
    B = torch.zeros(*lead, K // 8, N, dtype=torch.int32, device="cuda")
    for j in range(8):
        code = torch.empty_like(B, dtype=torch.float32).normal_(0.0, 2.6, generator=g).round_().clamp_(-8, 7)
        B |= (code.to(torch.int32) & 15) << (4 * j)
    S = torch.rand(*lead, K // GROUP, N, generator=g, device="cuda") * 0.02 + 0.01
    return B, (S * (4096.0 / K) ** 0.5).to(dtype)


def _activations(g, rows, K, dtype):
    """Normal values whose channels differ in size, a few of them by much."""
    channel = torch.exp(0.5 * torch.randn(K, generator=g, device="cuda"))
    return (0.3 * torch.randn(rows, K, generator=g, device="cuda") * channel).to(dtype)


def _ids(g, T, topk, E):
    """Different experts for each token, some experts more often than others."""
    popular = 0.5 * torch.randn(E, generator=g, device="cuda")
    noise = -torch.log(-torch.log(torch.rand(T, E, generator=g, device="cuda").clamp_(1e-6, 1 - 1e-6)))
    return torch.argsort(popular + noise, dim=1, descending=True, stable=True)[:, :topk].to(torch.int32).reshape(-1)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 12345)
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "topk":
        s["logits"] = (1.5 * torch.randn(c["T"], c["E"], generator=g, device="cuda")).to(DTYPES[c["logits"]])
        s["bias"] = 0.05 * torch.randn(c["E"], generator=g, device="cuda") if c["bias"] else None
        return s
    K, N = c["K"], c["N"]
    if c["op"] == "int4":
        M = c["M"]
        s["A"] = _activations(g, M, K, dt)
        s["B"], s["S"] = _weights(g, (K, N), dt)
        s["other"] = torch.randn(M, N, generator=g, device="cuda").to(dt) if c["postop"] in (1, 2) else None
        s["bias"] = (torch.randn(N, generator=g, device="cuda").to(torch.float32 if c["out_f32"] else dt)
                     if c["postop"] == 3 else None)
        return s
    E, T, topk = c["E"], c["T"], c["topk"]
    ids = _ids(g, T, topk, E)
    if c["op"] == "gate_up":
        s["ids"], s["X"] = ids, _activations(g, T, K, dt)
        s["Bg"], s["Sg"] = _weights(g, (E, K, N), dt)
        s["Bu"], s["Su"] = _weights(g, (E, K, N), dt)
        return s
    if c["op"] == "down_sum":
        s["ids"], s["H"] = ids, _activations(g, T * topk, K, dt)
        w = torch.rand(T, topk, generator=g, device="cuda") + 0.05
        s["RW"] = (w / w.sum(1, keepdim=True)).to(dt).reshape(-1)
        s["B"], s["S"] = _weights(g, (E, K, N), dt)
        return s
    G = T * topk
    s["A"] = _activations(g, G, K, dt)
    s["B"], s["S"] = _weights(g, (E, K, N), dt)
    s["other"] = torch.randn(G, N, generator=g, device="cuda").to(dt) if c["postop"] in (1, 2) else None
    # the routing's plan: row and 128-row-tile offsets of the experts
    count = torch.bincount(ids.long(), minlength=E)
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    tiles = (count + 127) // 128
    s["meta"] = torch.cat([zero, count.cumsum(0), zero, tiles.cumsum(0)]).to(torch.int32)
    s["most"] = int(count.max())
    return s


# ------------------------------------------------------------------------------- the plain forms
def _dequant(B, S):
    """fp32 [..., K, N] of packed weights and scales."""
    shift = torch.arange(0, 32, 4, dtype=torch.int32, device=B.device).view(8, 1)
    code = (((B.unsqueeze(-2) >> shift) & 15) ^ 8) - 8  # [..., K/8, 8, N]
    w = code.to(torch.float32).view(*S.shape[:-1], GROUP, S.shape[-1]) * S.to(torch.float32).unsqueeze(-2)
    return w.view(*B.shape[:-2], B.shape[-2] * 8, B.shape[-1])


def _sigmoid(v):
    """The library's: 0 up to -10."""
    return torch.where(v <= -10.0, torch.zeros_like(v), 1.0 / (1.0 + torch.exp(-v)))


def _epilogue(v, postop, other, bias):
    if postop == 1:
        return v * _sigmoid(v) * other.to(v.dtype)
    if postop == 2:
        return v + other.to(v.dtype)
    if postop == 3:
        return v + bias.to(v.dtype)
    return _sigmoid(v) if postop == 4 else v


def _plain_topk(s):
    c = s["case"]
    T, E, k, n_group = c["T"], c["E"], c["topk"], c["n_group"]
    x = s["logits"].double()
    if c["scoring"] == "softmax":
        e = torch.exp(x - x.max(1, keepdim=True).values)
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    choice = score + s["bias"].double() if s["bias"] is not None else score
    order = choice if s["bias"] is not None else x
    if n_group > 1:
        best = torch.sort(choice.view(T, n_group, E // n_group), dim=2, descending=True).values
        total = best[:, :, :c["group_top"]].sum(2)
        kept = torch.sort(total, dim=1, descending=True, stable=True).indices[:, :c["topk_group"]]
        keep = torch.zeros(T, n_group, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        order = order.masked_fill(~keep.repeat_interleave(E // n_group, dim=1), -math.inf)
    ids = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :k]
    w = score.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return ids.to(torch.int32), (w * c["scale"]).to(DTYPES[c["dtype"]])


def _plain(s):
    c = s["case"]
    dt = torch.float32 if c.get("out_f32") else DTYPES[c["dtype"]]
    if c["op"] == "topk":
        return _plain_topk(s)
    if c["op"] == "int4":
        v = s["A"].float() @ _dequant(s["B"], s["S"])
        return _epilogue(v, c["postop"], s["other"], s["bias"]).to(dt)
    T, topk, N = c["T"], c["topk"], c["N"]
    if c["op"] == "gate_up":
        e = s["ids"].long()
        x = s["X"].float().repeat_interleave(topk, dim=0).unsqueeze(1)
        gate = torch.bmm(x, _dequant(s["Bg"][e], s["Sg"][e])).squeeze(1)
        up = torch.bmm(x, _dequant(s["Bu"][e], s["Su"][e])).squeeze(1)
        return (gate * _sigmoid(gate) * up).to(dt)
    if c["op"] == "down_sum":
        e = s["ids"].long()
        y = torch.bmm(s["H"].float().unsqueeze(1), _dequant(s["B"][e], s["S"][e])).squeeze(1)
        return (y * s["RW"].float().unsqueeze(1)).view(T, topk, N).sum(1).to(dt)
    # the experts' rows side by side, each expert's padded to the most of any
    E, most = c["E"], s["most"]
    first = s["meta"][:E + 1].long()
    row = first[:E, None] + torch.arange(most, device=first.device)
    there = row < first[1:, None]
    x = s["A"].float()[row.clamp(max=T * topk - 1)]
    v = torch.bmm(x, _dequant(s["B"], s["S"]))[there]
    return _epilogue(v, c["postop"], s["other"], None).to(dt)


def run(state):
    s = state
    if not own:
        return _plain(s)
    import ternocl_b200 as tl
    c = s["case"]
    if c["op"] == "topk":
        return tl.moe_topk(s["logits"], c["topk"], bias=s["bias"], scoring=c["scoring"], n_group=c["n_group"],
                           topk_group=c["topk_group"], group_top=c["group_top"], renormalize=c["renorm"],
                           scale=c["scale"], dtype=DTYPES[c["dtype"]])
    if c["op"] == "int4":
        return tl.int4_upcvt(s["A"], s["B"], s["S"], postop=c["postop"], out_f32=c["out_f32"], other=s["other"],
                             bias=s["bias"])
    if c["op"] == "gate_up":
        return tl.moe_decode_gate_up_int4(s["ids"], s["X"], s["Bg"], s["Sg"], s["Bu"], s["Su"], c["E"], c["topk"])
    if c["op"] == "down_sum":
        return tl.moe_decode_down_sum_int4(s["ids"], s["H"], s["RW"], s["B"], s["S"], c["E"], c["topk"])
    return tl.moe_gemm_int4(s["meta"], s["A"], s["B"], s["S"], c["E"], postop=c["postop"], out_f32=c["out_f32"],
                            other=s["other"])


# ------------------------------------------------------------------------------ bytes and flops
def work(case):
    c = case
    if c["op"] == "topk":
        inb = 4 if c["logits"] == "fp32" else 2
        outb = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": c["T"] * (c["E"] * inb + c["topk"] * (4 + outb)) + (4 * c["E"] if c["bias"] else 0),
                "flops": 4 * c["T"] * c["E"]}
    K, N = c["K"], c["N"]
    matrix = K * N // 2 + K // GROUP * N * 2
    outb = 4 if c.get("out_f32") else 2
    if c["op"] == "int4":
        M = c["M"]
        other = M * N * 2 if c["postop"] in (1, 2) else 0
        return {"bytes": matrix + M * K * 2 + M * N * outb + other, "flops": 2 * M * N * K}
    G, E = c["T"] * c["topk"], c["E"]
    # distinct experts that uniformly routed tokens touch
    touched = E * (1.0 - (1.0 - c["topk"] / E) ** c["T"])
    if c["op"] == "gate_up":
        return {"bytes": int(2 * touched * matrix) + c["T"] * K * 2 + G * N * 2, "flops": 4 * G * N * K}
    if c["op"] == "down_sum":
        return {"bytes": int(touched * matrix) + G * K * 2 + c["T"] * N * 2, "flops": 2 * G * N * K}
    other = G * N * 2 if c["postop"] in (1, 2) else 0
    return {"bytes": int(touched * matrix) + G * K * 2 + G * N * outb + other, "flops": 2 * G * N * K}


# -------------------------------------------------------------------- the definitions in 64 bits
def _matrix64(B, S):
    """float64 [K, N]: byte b of a word holds rows 2b (low nibble) and 2b+1 (high nibble)."""
    kw, N = B.shape
    byte = B.contiguous().view(torch.uint8).view(kw, N, 4).permute(0, 2, 1).to(torch.int16)
    pair = torch.stack([byte % 16, byte // 16], dim=2)  # [kw, 4, 2, N]
    value = torch.where(pair > 7, pair - 16, pair).reshape(kw * 8, N).double()
    return value * S.double().repeat_interleave(GROUP, dim=0)


def _end64(v, postop, other, bias):
    gate = torch.sigmoid(v) * (v > -10.0)
    if postop == 1:
        return v * gate * other.double()
    if postop == 2:
        return v + other.double()
    if postop == 3:
        return v + bias.double()
    return gate if postop == 4 else v


def _exact_topk(c, s):
    x = s["logits"].double().cpu().numpy()
    T, E = x.shape
    if c["scoring"] == "softmax":
        z = x - x.max(axis=1, keepdims=True)
        score = np.exp(z - np.log(np.exp(z).sum(axis=1, keepdims=True)))
    else:
        score = 0.5 * (1.0 + np.tanh(0.5 * x))
    choice = score if s["bias"] is None else score + s["bias"].double().cpu().numpy()
    order = x if s["bias"] is None else choice
    per = E // c["n_group"]
    allowed = np.ones((T, E), bool)
    if c["n_group"] > 1:
        grouped = -np.sort(-choice.reshape(T, c["n_group"], per), axis=2)[:, :, :c["group_top"]].sum(axis=2)
        rank = np.argsort(np.argsort(-grouped, axis=1, kind="stable"), axis=1, kind="stable")
        allowed = np.repeat(rank < c["topk_group"], per, axis=1)
    ids = np.argsort(np.where(allowed, -order, np.inf), axis=1, kind="stable")[:, :c["topk"]]
    w = np.take_along_axis(score, ids, axis=1)
    if c["renorm"]:
        w = w / w.sum(axis=1, keepdims=True)
    return ids.astype(np.int32), w * c["scale"]


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "topk":
        return _exact_topk(c, s)
    if c["op"] == "int4":
        out = []
        x = s["A"].double()
        for n in range(0, c["N"], 16384):
            end = min(c["N"], n + 16384)
            cut = lambda t: None if t is None else t[..., n:end]  # noqa: E731
            v = x @ _matrix64(s["B"][:, n:end], s["S"][:, n:end])
            out.append(_end64(v, c["postop"], cut(s["other"]), cut(s["bias"])))
        return torch.cat(out, dim=1)
    T, topk = c["T"], c["topk"]
    if c["op"] == "moe_gemm":
        out = []
        first = s["meta"][:c["E"] + 1].tolist()
        for e in range(c["E"]):
            lo, hi = first[e], first[e + 1]
            if hi > lo:
                v = s["A"][lo:hi].double() @ _matrix64(s["B"][e], s["S"][e])
                out.append(_end64(v, c["postop"], None if s["other"] is None else s["other"][lo:hi], None))
        return torch.cat(out, dim=0)
    rows = []
    for r, e in enumerate(s["ids"].tolist()):
        if c["op"] == "gate_up":
            x = s["X"][r // topk].double()
            gate = x @ _matrix64(s["Bg"][e], s["Sg"][e])
            rows.append(_end64(gate, 1, x @ _matrix64(s["Bu"][e], s["Su"][e]), None))
        else:
            rows.append(s["RW"][r].double() * (s["H"][r].double() @ _matrix64(s["B"][e], s["S"][e])))
    out = torch.stack(rows)
    return out if c["op"] == "gate_up" else out.view(T, topk, c["N"]).sum(dim=1)
