"""The encoder's operators as a layer uses them: tokens in 8 bits, the projection to Q, K and V, the rotary embedding of Q and
K, attention within every chunk, the projection back, the sum with the residual and its norm."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def tables(T, half):
    angle = torch.arange(T, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    return torch.sin(angle).float(), torch.cos(angle).float()


def layer(of, x, p, lens, T, window, out=None):
    """One layer on x [tokens][width] fp16, chunks of room T, of which lens are used.  The result, and what it came by."""
    H, D = p["H"], p["D"]
    tokens = x.shape[0]
    xq, xs = of.quantize_i8(x)
    qkv = of.matmul_i8(xq, xs, *p["qkv"], bias=p["b"])
    of.rotary_emb_gpu(qkv, *p["tables"], tokens // T, T, 2 * H, D, D // 2, T * 3 * H * D, 3 * H * D, D)
    heads = qkv.view(tokens, 3, H, D)
    att = torch.zeros(tokens, H, D, dtype=x.dtype, device="cuda")
    of.attention(heads[:, 0], heads[:, 1], heads[:, 2], p["starts"], p["starts"], T, T, q_used=lens, k_used=lens, window=window, out=att)
    aq, a_s = of.quantize_i8(att.view(tokens, H * D))
    back = of.matmul_i8(aq, a_s, *p["back"])
    return of.norm(back, "rms", p["g"], residual=x, residual_scale=p["alpha"], out=out), qkv, att, back


def weights(of, H, D, B, T, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = H * D
    make = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    p = {"H": H, "D": D, "alpha": 2.4, "g": (1 + 0.1 * make(width)).half(), "b": (0.1 * make(3 * width)).half(), "tables": tables(T, D // 2),
         "starts": torch.arange(B + 1, dtype=torch.int32, device="cuda") * T,
         "w_qkv": (make(3 * width, width) / math.sqrt(width)).half(), "w_back": (make(width, width) / math.sqrt(width)).half()}
    p["qkv"], p["back"] = of.quantize_i8(p["w_qkv"]), of.quantize_i8(p["w_back"])
    return p, make(B * T, width).half()


@pytest.mark.parametrize("B,T,H,D,window", [(3, 200, 4, 32, (16, 16)), (2, 333, 8, 64, (128, 127)), (2, 130, 2, 128, (-1, -1))])
def test_a_layer_against_its_steps_in_64_bits(native_lib, B, T, H, D, window):
    p, x = weights(native_lib, H, D, B, T, 1)
    used = [T] + [T // 2 + 3 * n for n in range(B - 1)]
    lens = torch.tensor(used, dtype=torch.int32, device="cuda")
    y, qkv, att, back = layer(native_lib, x, p, lens, T, window)
    # every step from what the step before it really gave (so that roundings to 8 bits, which may tip over, are not compared)
    wq, ws = p["qkv"]
    xq, xs = native_lib.quantize_i8(x)
    proj = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double() + p["b"].double()
    half, width = D // 2, H * D
    q = proj.view(B, T, 3, H, D).clone()
    sin, cos = (t.double()[None, :, None, None, :] for t in p["tables"])
    a, b = q[:, :, :2, :, :half].clone(), q[:, :, :2, :, half:].clone()
    q[:, :, :2, :, :half], q[:, :, :2, :, half:] = a * cos - b * sin, b * cos + a * sin
    # fp16 after the product and after the rotation: half a step each, of the pair's length
    length = torch.sqrt(a.square() + b.square())
    bound = torch.zeros_like(q)
    bound[:, :, :2] = 2.5 * 2.0 ** -11 * torch.cat([length, length], -1)
    bound[:, :, 2] = 1.1 * 2.0 ** -11 * q[:, :, 2].abs()
    assert ((qkv.view_as(q).double() - q).abs() <= bound + 2.0 ** -20).all()
    heads = qkv.view(B, T, 3, H, D).double()
    for n in range(B):
        L = used[n]
        z = torch.einsum("ihd,jhd->hij", heads[n, :L, 0], heads[n, :L, 1]) / math.sqrt(D)
        gap = torch.arange(L, device="cuda")[None, :] - torch.arange(L, device="cuda")[:, None]
        hidden = torch.zeros_like(gap, dtype=torch.bool)
        if window[0] >= 0:
            hidden = (gap < -window[0]) | (gap > window[1])
        w = torch.softmax(z.masked_fill(hidden, -math.inf), 2)
        want = torch.einsum("hij,jhd->ihd", w, heads[n, :L, 2])
        weight = torch.einsum("hij,jhd->ihd", w, heads[n, :L, 2].abs())
        off = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -18 * (1 + z.abs().max())) * weight * 1.001 + L * 2.0 ** -17 * heads[n, :L, 2].abs().max()
        got = att.view(B, T, H, D)[n]
        assert ((got[:L].double() - want).abs() <= off).all()
        assert (got[L:] == 0).all()
    s = back.double() + p["alpha"] * x.double()
    want = s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-5) * p["g"].double()
    assert ((y.double() - want).abs() <= 2.0 ** -11 * want.abs() * 1.01 + 2.0 ** -19).all()
    # and the layer as a whole near the one without 8 bits: steps of 1/127 of a row's largest, in three products
    q16 = x.double() @ p["w_qkv"].double().t() + p["b"].double()
    assert (proj - q16).norm() / q16.norm() < 0.03
    native_lib.encoder_wait()


def test_a_layer_captured_into_a_graph(native_lib):
    # all but the rotary embedding (whose call waits for its kernel) in one graph, replayed on other inputs
    B, T, H, D = 4, 300, 8, 64
    p, x = weights(native_lib, H, D, B, T, 2)
    lens = torch.full((B,), T, dtype=torch.int32, device="cuda")

    def step(out):
        q, s = native_lib.quantize_i8(x)
        qkv = native_lib.matmul_i8(q, s, *p["qkv"], bias=p["b"]).view(B * T, 3, H, D)
        att = native_lib.attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], p["starts"], p["starts"], T, T, k_used=lens, window=(128, 128))
        _, q, s = native_lib.norm(att.view(B * T, H * D), "none", quantize=True)
        return native_lib.norm(native_lib.matmul_i8(q, s, *p["back"]), "rms", p["g"], residual=x, residual_scale=p["alpha"], out=out)

    out = torch.empty_like(x)
    step(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    for seed in (3, 4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").half())
        graph.replay()
        want = step(torch.empty_like(x))
        assert torch.equal(out, want)
    native_lib.encoder_wait()


def test_one_token_at_a_time_gives_what_the_whole_prompt_gives(native_lib):
    # a causal prompt at once, and the same tokens one by one against the keys so far
    T, H, Hkv, D = 150, 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(T, n, D, generator=g, device="cuda").half() for n in (H, Hkv, Hkv))
    starts = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    whole = native_lib.attention(q, k, v, starts, starts, T, T, causal=True)
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    used = torch.empty(1, dtype=torch.int32, device="cuda")
    for t in range(T):
        used.fill_(t + 1)
        got = native_lib.attention(q[t : t + 1], k, v, one, starts, 1, T, k_used=used, causal=True)
        # each is within a rounding of the weights and of itself of the same number
        assert ((got - whole[t]).abs().double() <= 4 * 2.0 ** -11 * v[: t + 1].abs().max().double()).all()
