"""The product of 8-bit integers against its definition in 64 bits: the sums are exact, what is left are the scales' and
the result's roundings."""
import math

import pytest
import torch

from encoder_util import HALF, TINY, close

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def rows8(rows, depth, seed, pad=0, fill=77):
    """int8 rows on 16-byte boundaries; what lies behind a row is not zero."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    at = torch.full((rows, (depth + 15) // 16 * 16 + pad), fill, dtype=torch.int8, device="cuda")
    at[:, :depth] = torch.randint(-128, 128, (rows, depth), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    return at[:, :depth]


def scales(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(n, generator=g, device="cuda") * 2e-3 + 1e-4


def check(of, x, w, dtype, bias=None, out=None, xs=None, ws=None):
    xs = scales(x.shape[0], 3) if xs is None else xs
    ws = scales(w.shape[0], 4) if ws is None else ws
    product = (x.double() @ w.double().t()) * (xs.double()[:, None] * ws.double()[None, :])
    want = product if bias is None else product + bias.double()
    got = of.matmul_i8(x, xs, w, ws, bias, dtype, out)
    # a sum beyond 2^24 is rounded to fp32, the scales' product, the scaled sum and the sum with the bias each once
    fp32 = 2.0 ** -24 * (4 * product.abs() + want.abs())
    u = HALF[dtype]
    assert close(got, want, u * want.abs() + (1 + u) * fp32 + TINY[dtype])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 8, 16), (2, 3, 5), (1, 4096, 4096), (3, 1001, 333), (7, 129, 127), (8, 128, 128), (9, 64, 4097),
                                   (16, 512, 512), (17, 300, 1000), (31, 2048, 96), (64, 1536, 512), (100, 250, 31), (127, 127, 129), (128, 256, 128),
                                   (129, 257, 257), (200, 7, 2000), (333, 512, 48), (500, 1000, 1237), (1024, 1024, 1024), (2049, 96, 160), (5000, 264, 80)])
def test_sizes(native_lib, dtype, M, N, K):
    check(native_lib, rows8(M, K, 1), rows8(N, K, 2), dtype)
    b = torch.randn(N, device="cuda").to(dtype)
    check(native_lib, rows8(M, K, 5), rows8(N, K, 6), dtype, b)


@pytest.mark.parametrize("M,N,K", [(1, 640, 640), (5, 200, 200), (40, 640, 1040), (700, 520, 640)])
def test_strides(native_lib, M, N, K):
    x, w = rows8(M, K, 1, pad=48), rows8(N, K, 2, pad=16)
    for extra, offset in ((0, 0), (8, 8), (3, 0), (1, 1), (5, 3)):
        base = torch.randn(M * (N + extra) + 16, device="cuda").half()
        before = base.clone()
        out = base[offset : offset + M * (N + extra)].view(M, N + extra)[:, :N]
        check(native_lib, x, w, torch.float16, torch.randn(N + 1, device="cuda").half()[1:], out)
        touched = torch.zeros_like(base, dtype=torch.bool)
        touched[offset : offset + M * (N + extra)].view(M, N + extra)[:, :N] = True
        assert torch.equal(base[~touched], before[~touched])


@pytest.mark.parametrize("M", [1, 6, 33, 150])
def test_the_deepest_sums_stay_exact(native_lib, M):
    # every product 2^14: the sum is 131071 * 2^14, just inside 32 bits
    K = 131071
    x = torch.full((M, (K + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = torch.full((40, (K + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :K]
    one = torch.ones(40, device="cuda")
    got = native_lib.matmul_i8(x, torch.full((M,), 2.0 ** -20, device="cuda"), w, one, dtype=torch.bfloat16)
    assert (got.float() == torch.tensor(K * 2.0 ** -6).bfloat16().float()).all()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_scales_that_are_no_numbers_stay_in_their_rows(native_lib, M):
    x, w, xs, ws = rows8(M, 256, 1), rows8(300, 256, 2), scales(M, 3), scales(300, 4)
    xs[0] = math.nan
    ws[7] = math.inf
    got = native_lib.matmul_i8(x, xs, w, ws)
    assert torch.isnan(got[0]).all() and torch.isinf(got[1:, 7]).all()
    rest = [n for n in range(300) if n != 7]
    assert torch.isfinite(got[1:][:, rest]).all()
    assert torch.equal(got[1:][:, rest], native_lib.matmul_i8(x, scales(M, 3), w, scales(300, 4))[1:][:, rest])


def test_no_rows(native_lib):
    out = native_lib.matmul_i8(rows8(4, 64, 1)[:0], scales(0, 1), rows8(5, 64, 2), scales(5, 2))
    assert out.shape == (0, 5)


@pytest.mark.parametrize("M,N,K", [(1, 500, 2000), (24, 640, 4096), (300, 640, 640)])
def test_captured_and_on_two_streams_at_once(native_lib, M, N, K):
    x, w, xs, ws = rows8(M, K, 1), rows8(N, K, 2), scales(M, 3), scales(N, 4)
    x2 = rows8(M, K, 9)
    want, want2 = native_lib.matmul_i8(x, xs, w, ws), native_lib.matmul_i8(x2, xs, w, ws)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = [[native_lib.matmul_i8(t, xs, w, ws, stream=s) for t, s in zip((x, x2), side)] for _ in range(20)]
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, want) and torch.equal(b, want2) for a, b in got)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        native_lib.matmul_i8(x, xs, w, ws, out=out)
    x.copy_(x2)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want2)


def test_from_tokens_to_product(native_lib):
    # the two calls as they are used together: within the steps of 8 bits of the product of what went in
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w = (torch.randn(n, 600, generator=g, device="cuda").half() for n in (77, 130))
    (xq, xs), (wq, ws) = native_lib.quantize_i8(x), native_lib.quantize_i8(w)
    got = native_lib.matmul_i8(xq, xs, wq, ws).double()
    want = x.double() @ w.double().t()
    # |x w - xq wq| <= |dx||w| + |x||dw| + |dx||dw| with |dx| <= xs / 2, |dw| <= ws / 2 (and 2^-10 of room for fp16 and fp32)
    dx, dw = 0.5 * xs.double()[:, None], 0.5 * ws.double()[:, None]
    off = dx * w.double().abs().sum(1)[None, :] + x.double().abs().sum(1)[:, None] * dw.t() + 600 * dx * dw.t()
    assert ((got - want).abs() <= off * 1.001 + 2.0 ** -11 * got.abs() + 1e-6).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(64, 4096, 4096), (9, 4096, 4097), (128, 4090, 8000), (100, 1024, 4096), (129, 1003, 3999), (16, 64, 131071), (64, 256, 16384), (37, 321, 16000),
                                   (128, 512, 2048), (300, 70, 5000), (64, 1100, 130000), (12, 1, 9999)])
def test_few_tiles_and_much_depth(native_lib, dtype, M, N, K):
    for pad, bias in ((0, False), (16, True)):
        x, w = rows8(M, K, 1, pad), rows8(N, K, 2, pad)
        got = check(native_lib, x, w, dtype, torch.randn(N, device="cuda").to(dtype) if bias else None)
        # results that go off the 16-byte boundaries, and nothing beside them
        wide = torch.full((M, N + 5), 7.0, dtype=dtype, device="cuda")
        if not bias:
            assert torch.equal(check(native_lib, x, w, dtype, out=wide[:, 3 : N + 3]), got)
            assert (wide[:, :3] == 7).all() and (wide[:, N + 3 :] == 7).all()
    # sums at the ends of 32 bits
    x.fill_(-128)
    w.fill_(-128)
    check(native_lib, x, w, dtype, xs=torch.full((M,), 2.0 ** -20, device="cuda"), ws=torch.full((N,), 2.0 ** -10, device="cuda"))


def test_few_tiles_captured_and_on_two_streams(native_lib):
    x, w = rows8(64, 4096, 1), rows8(1024, 4096, 2)
    x2, xs, ws = rows8(64, 4096, 5), scales(64, 3), scales(1024, 4)
    want = [native_lib.matmul_i8(t, xs, w, ws) for t in (x, x2)]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = [[native_lib.matmul_i8(t, xs, w, ws, stream=s) for t, s in zip((x, x2), side)] for _ in range(30)]
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, v) for pair in got for g, v in zip(pair, want))
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want[0])
    with torch.cuda.graph(graph):
        native_lib.matmul_i8(x, xs, w, ws, out=out)
    x.copy_(x2)
    graph.replay()
    assert torch.equal(out, want[1])
    native_lib.encoder_wait()
