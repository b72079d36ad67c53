"""The operators of the transformer encoder whose speed is measured: attention over packed sequences,
the product of 8-bit integers, and the residual norm that feeds it.  What each case is, how its inputs
are made, one pass of it, its plain form and its exact result.

The encoder stands in front of the CRF head: a layer is a projection of the tokens to Q, K and V, the
rotary embedding of Q and K, attention within each chunk or read, a projection back, and a norm of the
sum with the residual; the tokens of every projection are held in 8 bits with a scale each.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# An attention case: "S" sequences of queries between "q_min" and "q_max" long and keys between "k_min"
# and "k_max" ("k_min" 0: as many keys as queries), the lengths drawn from "lens"; "left"/"right" how many keys before and behind
# its own place a query sees (-1: all), places counted from the sequences' common end.  "layout": "qkv" (Q,
# K and V side by side in one tensor, as a projection leaves them), "rows" (three tensors) or "cache" (keys
# and values in a tensor with room for "k_max" tokens a sequence, of which some are used).
# A product case: "M" tokens, "N" channels, "K" deep; "tokens": "i8" (already in 8 bits) or a type, whose
# tokens are brought to 8 bits first.
# A norm case: "rows" rows of "width", "norm" "layer" or "rms", "residual" or not; "N" above 0: its result in 8 bits goes
# through a product with that many channels as well.


def _attention(name, dtype, S, q_min, q_max, k_min, k_max, Hq, Hkv, D, left, right, layout, lens=1):
    return {"name": name, "op": "attention", "dtype": dtype, "S": S, "q_min": q_min, "q_max": q_max, "k_min": k_min,
            "k_max": k_max, "Hq": Hq, "Hkv": Hkv, "D": D, "left": left, "right": right, "layout": layout, "lens": lens}


def _product(name, dtype, M, N, K, tokens="i8", bias=True):
    return {"name": name, "op": "product", "dtype": dtype, "M": M, "N": N, "K": K, "tokens": tokens, "bias": bias}


def _norm(name, dtype, rows, width, norm, residual=True, bias=False, N=0):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "width": width, "norm": norm, "residual": residual,
            "bias": bias, "N": N}


def listed():
    return [
        # the encoder's batch: 32 chunks of 1666 frames, every frame sees its neighbourhood to both sides
        _attention("att_encoder_window", "fp16", 32, 1666, 1666, 0, 0, 8, 8, 64, 128, 128, "qkv"),
        # reads of different lengths packed into one tensor, every frame of a read sees the whole read
        _attention("att_packed_reads", "fp16", 24, 200, 2047, 0, 0, 8, 8, 64, -1, -1, "qkv"),
        # one long prompt, causal, four query heads to a key head
        _attention("att_prompt_8192", "bf16", 1, 8192, 8192, 0, 0, 32, 8, 128, -1, 0, "rows"),
        # a server's step: 64 sequences, one new token each, against what a cache holds of them
        _attention("att_tokens_64", "bf16", 64, 1, 1, 1024, 8192, 32, 8, 128, -1, 0, "cache"),
        # one new token of one sequence: nothing but latency
        _attention("att_token_1", "fp16", 1, 1, 1, 4097, 4097, 8, 8, 64, -1, 0, "rows"),
        # the encoder's projection to Q, K and V: 32 x 1666 frames
        _product("mm_encoder_qkv", "fp16", 53312, 1536, 512),
        # a large product, bound by the arithmetic
        _product("mm_8192", "bf16", 8192, 8192, 8192),
        # a batch of odd sizes, tokens brought to 8 bits on the way
        _product("mm_ragged", "bf16", 1003, 2501, 1237, tokens="bf16"),
        # one token through a projection: the weights are read once
        _product("mm_token_1", "fp16", 1, 4096, 4096, tokens="fp16"),
        # the end of a layer: residual and norm of the encoder's batch
        _norm("norm_encoder", "fp16", 53312, 512, "rms"),
        # the same in front of a projection: norm, tokens in 8 bits, product
        _norm("norm_product", "fp16", 53312, 512, "layer", bias=True, N=2048),
        # a handful of tokens of a wide model
        _norm("norm_7_wide", "bf16", 7, 5120, "rms"),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "product", "norm"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "product":
        N, K = _between(rng, 8, 8192), _between(rng, 16, 8192)
        M = _between(rng, 1, min(50000, int(5e11 / (N * K))))
        return {k: v for k, v in _product("", dtype, M, N, K, rng.choice(["i8", dtype]), rng.random() < 0.5).items() if k != "name"}
    if op == "norm":
        rows, width = _between(rng, 1, 50000), _between(rng, 16, 5120)
        N = rng.choice([0, 0, _between(rng, 64, 2048)])
        c = _norm("", dtype, rows, width, rng.choice(["layer", "rms"]), rng.random() < 0.7, rng.random() < 0.5, N)
        return {k: v for k, v in c.items() if k != "name"}
    D = rng.choice([32, 64, 64, 80, 96, 128, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    Hq = Hkv * rng.choice([1, 1, 2, 4, 5])
    lens = rng.randrange(1 << 20)
    if rng.random() < 0.35:  # new tokens against a cache
        S, q_max, k_max = _between(rng, 1, 64), rng.choice([1, 1, 1, 2, 5]), _between(rng, 16, 8192)
        c = _attention("", dtype, S, 1, q_max, max(1, k_max // 8), k_max, Hq, Hkv, D, -1, 0, rng.choice(["cache", "rows"]), lens)
    else:
        S = _between(rng, 1, 32)
        most = min(8192, int(math.sqrt(1.2e9 / (S * Hq))))  # the plain form holds every score
        q_max = _between(rng, 1, most)
        left, right = rng.choice([(-1, 0), (-1, 0), (-1, -1), (128, 128), (_between(rng, 1, 1000), _between(rng, 1, 1000)), (255, 0)])
        c = _attention("", dtype, S, max(1, q_max // rng.choice([1, 4, 50])), q_max, 0, 0, Hq, Hkv, D, left, right,
                       rng.choice(["qkv", "rows"]), lens)
    return {k: v for k, v in c.items() if k != "name"}


def _lengths(case):
    r = random.Random(case["lens"])
    q = [r.randint(case["q_min"], case["q_max"]) for _ in range(case["S"])]
    k = [r.randint(max(case["k_min"], n), max(case["k_max"], n)) for n in q] if case["k_min"] else list(q)
    return q, k


def _starts(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(dt)

    def whole(*shape):
        """8-bit values as a quantised weight's or token's: a row's largest is 127."""
        x = torch.randn(shape, generator=g, device=DEV)
        return torch.round(x * (127.0 / x.abs().amax(-1, keepdim=True))).to(torch.int8)

    def padded(x):
        """The same rows, each on a 16-byte boundary, as they are kept for the product."""
        at = torch.zeros((x.shape[0], (x.shape[1] + 15) // 16 * 16), dtype=torch.int8, device=DEV)
        at[:, : x.shape[1]] = x
        return at[:, : x.shape[1]]

    def weights(N, K):
        return {"w": padded(whole(N, K)), "w_scale": torch.rand(N, generator=g, device=DEV) * 0.02 / math.sqrt(K) + 0.005 / math.sqrt(K)}

    s = dict(case)
    if case["op"] == "attention":
        q_len, k_len = _lengths(case)
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        rows = sum(q_len)
        if case["layout"] == "qkv":
            qkv = normal(rows, Hq + 2 * Hkv, D)
            s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv], qkv[:, Hq + Hkv :]
        else:
            room = case["S"] * case["k_max"] if case["layout"] == "cache" else sum(k_len)
            s["q"], s["k"], s["v"] = normal(rows, Hq, D), normal(room, Hkv, D), normal(room, Hkv, D)
        s["q_start"] = torch.from_numpy(_starts(q_len)).to(DEV)
        if case["layout"] == "cache":
            s["k_start"] = torch.arange(case["S"] + 1, dtype=torch.int32, device=DEV) * case["k_max"]
            s["k_used"] = torch.tensor(k_len, dtype=torch.int32, device=DEV)
        else:
            s["k_start"], s["k_used"] = torch.from_numpy(_starts(k_len)).to(DEV), None
        s["longest_q"], s["longest_k"] = max(q_len), max(k_len)
    elif case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        if case["tokens"] == "i8":
            s["x"], s["x_scale"] = padded(whole(M, K)), torch.rand(M, generator=g, device=DEV) * 0.04 + 0.005
        else:
            s["x"] = normal(M, K)
        s |= weights(N, K)
        s["b"] = normal(N, scale=0.2) if case["bias"] else None
    else:
        rows, width = case["rows"], case["width"]
        s["x"] = normal(rows, width)
        s["r"] = normal(rows, width, scale=1.5) if case["residual"] else None
        s["weight"] = 1 + normal(width, scale=0.2)
        s["b"] = normal(width, scale=0.1) if case["bias"] else None
        if case["N"]:
            s |= weights(case["N"], width)
    return s


ALPHA = 2.4  # the residual's factor of a deep post-norm encoder
EPS = 1e-5


def run(s):
    if own:
        import openfish_b200 as of
        if s["op"] == "attention":
            return of.attention(s["q"], s["k"], s["v"], s["q_start"], s["k_start"], s["longest_q"], s["longest_k"], k_used=s["k_used"],
                                window=(s["left"], s["right"]))
        if s["op"] == "product":
            x, x_scale = (s["x"], s["x_scale"]) if s["tokens"] == "i8" else of.quantize_i8(s["x"])
            return of.matmul_i8(x, x_scale, s["w"], s["w_scale"], bias=s["b"], dtype=TYPES[s["dtype"]])
        if not s["N"]:
            return of.norm(s["x"], s["norm"], s["weight"], s["b"], eps=EPS, residual=s["r"], residual_scale=ALPHA)
        y, x, x_scale = of.norm(s["x"], s["norm"], s["weight"], s["b"], eps=EPS, residual=s["r"], residual_scale=ALPHA, quantize=True)
        return y, of.matmul_i8(x, x_scale, s["w"], s["w_scale"], dtype=TYPES[s["dtype"]])
    if s["op"] == "attention":
        return _plain_attention(s)
    if s["op"] == "product":
        x, x_scale = (s["x"], s["x_scale"]) if s["tokens"] == "i8" else _plain_tokens(s["x"].float())
        return _plain_product(x, x_scale, s)
    y = s["x"].float()
    if s["r"] is not None:
        y = y + ALPHA * s["r"].float()
    if s["norm"] == "layer":
        y = y - y.mean(1, keepdim=True)
    y = y * torch.rsqrt((y * y).mean(1, keepdim=True) + EPS) * s["weight"].float()
    if s["b"] is not None:
        y = y + s["b"].float()
    if not s["N"]:
        return y.to(s["x"].dtype)
    x, x_scale = _plain_tokens(y)
    return y.to(s["x"].dtype), _plain_product(x, x_scale, dict(s, b=None))


def _plain_tokens(x):
    """Tokens in 8 bits: a row's largest value is 127 steps."""
    top = x.abs().amax(1, keepdim=True)
    return torch.round(x * torch.where(top > 0, 127.0 / top, 0.0)).to(torch.int8), (top / 127.0)[:, 0]


def _plain_product(x, x_scale, s):
    y = (x.float() @ s["w"].float().t()) * x_scale[:, None] * s["w_scale"][None, :]
    if s["b"] is not None:
        y = y + s["b"].float()
    return y.to(TYPES[s["dtype"]])


def _plain_attention(s):
    """Every sequence padded to the longest, all scores at once."""
    S, Hq, Hkv, D = s["S"], s["Hq"], s["Hkv"], s["D"]
    q_start, k_start = s["q_start"].long(), s["k_start"].long()
    q_len = q_start[1:] - q_start[:-1]
    k_len = k_start[1:] - k_start[:-1] if s["k_used"] is None else s["k_used"].long()
    i = torch.arange(s["longest_q"], device=DEV)
    j = torch.arange(s["longest_k"], device=DEV)
    q_at = (q_start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    k_at = (k_start[:-1, None] + j).clamp(max=s["k"].shape[0] - 1)
    q = s["q"][q_at].float().view(S, -1, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, -1, D)
    k = s["k"][k_at].float().permute(0, 2, 3, 1)
    v = s["v"][k_at].float().permute(0, 2, 1, 3)
    p = (q @ k).mul_(1.0 / math.sqrt(D)).view(S, Hq, i.numel(), j.numel())
    place = i[None, :, None] + (k_len - q_len)[:, None, None]
    seen = j[None, None, :] < k_len[:, None, None]
    if s["left"] >= 0:
        seen = seen & (j[None, None, :] >= place - s["left"])
    if s["right"] >= 0:
        seen = seen & (j[None, None, :] <= place + s["right"])
    p.masked_fill_(~seen[:, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(S, Hkv, -1, j.numel()) @ v).view(S, Hq, -1, D) / torch.where(total > 0, total, 1.0)
    there = i[None, :] < q_len[:, None]
    return o.permute(0, 2, 1, 3)[there].to(s["q"].dtype)


def work(case):
    e = 2
    if case["op"] == "attention":
        q_len, k_len = _lengths(case)
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        pairs = 0
        for n, m in zip(q_len, k_len):
            place = np.arange(n, dtype=np.int64) + m - n
            lo = np.maximum(place - case["left"], 0) if case["left"] >= 0 else np.zeros(n, np.int64)
            hi = np.minimum(place + case["right"], m - 1) if case["right"] >= 0 else np.full(n, m - 1)
            pairs += int(np.maximum(hi - lo + 1, 0).sum())
        return {"bytes": e * D * (2 * Hq * sum(q_len) + 2 * Hkv * sum(k_len)), "flops": 4.0 * D * Hq * pairs}
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * (K + 4 if case["tokens"] == "i8" else e * K) + N * (K + 4 + e * case["bias"]) + e * M * N, "flops": 2.0 * M * N * K}
    rows, width, N = case["rows"], case["width"], case["N"]
    return {"bytes": e * rows * width * (2 + case["residual"]) + e * width * (1 + case["bias"]) + N * (width + 4) + e * rows * N,
            "flops": rows * width * (8.0 + 2.0 * N)}


def exact(case, seed):
    """The definitions in 64 bits, a sequence and a key head at a time."""
    s = prepare(case, seed)
    if case["op"] == "attention":
        q_len, k_len = _lengths(case)
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        group = case["Hq"] // case["Hkv"]
        q_at = np.concatenate([[0], np.cumsum(q_len)])
        k_at = np.concatenate([[0], np.cumsum(k_len)]) if case["layout"] != "cache" else np.arange(case["S"] + 1) * case["k_max"]
        for n, (ql, kl) in enumerate(zip(q_len, k_len)):
            gap = torch.arange(kl, device=DEV)[None, :] - torch.arange(ql, device=DEV)[:, None] - (kl - ql)
            hidden = torch.zeros_like(gap, dtype=torch.bool)
            if case["left"] >= 0:
                hidden |= gap < -case["left"]
            if case["right"] >= 0:
                hidden |= gap > case["right"]
            rows = slice(int(q_at[n]), int(q_at[n]) + ql)
            keys = slice(int(k_at[n]), int(k_at[n]) + kl)
            for h in range(case["Hkv"]):
                k, v = s["k"][keys, h].double(), s["v"][keys, h].double()
                for m in range(h * group, (h + 1) * group):
                    z = torch.einsum("qd,kd->qk", s["q"][rows, m].double(), k) / math.sqrt(case["D"])
                    z[hidden] = -math.inf
                    out[rows, m] = torch.nan_to_num(torch.softmax(z, 1), nan=0.0) @ v
        return out

    def tokens(y):
        step = torch.linalg.vector_norm(y, math.inf, dim=1) / 127
        return torch.round(y / torch.where(step > 0, step, 1.0)[:, None]), step

    def product(x, x_scale, bias):
        y = torch.einsum("mk,nk->mn", x, s["w"].double() * s["w_scale"].double()[:, None]) * x_scale[:, None]
        return y if bias is None else y + bias.double()

    if case["op"] == "product":
        x, x_scale = (s["x"].double(), s["x_scale"].double()) if case["tokens"] == "i8" else tokens(s["x"].double())
        return product(x, x_scale, s["b"])
    y = s["x"].double()
    if case["residual"]:
        y = torch.add(y, s["r"].double(), alpha=ALPHA)
    if case["norm"] == "layer":
        y = (y - y.mean(1, keepdim=True)) / torch.sqrt(y.var(1, unbiased=False, keepdim=True) + EPS)
    else:
        y = y / torch.sqrt(y.pow(2).mean(1, keepdim=True) + EPS)
    y = y * s["weight"].double()
    if case["bias"]:
        y = y + s["b"].double()
    return y if not case["N"] else (y, product(*tokens(y), None))
