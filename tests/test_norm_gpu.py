"""Residual, norm and 8-bit tokens against their definition in 64 bits."""
import math

import pytest
import torch

from encoder_util import HALF, TINY, close, norm_reference

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def make(rows, width, dtype, seed=0, scale=1.0, at=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, width, generator=g, device="cuda") * scale + at).to(dtype)


def check(of, x, kind, weight=None, bias=None, eps=1e-5, residual=None, residual_scale=1.0, out=None):
    y, bound = norm_reference(x, kind, weight, bias, eps, residual, residual_scale)
    got, q, scale = of.norm(x, kind, weight, bias, eps, residual, residual_scale, out=out, quantize=True)
    u = HALF[x.dtype]
    assert close(got, y, u * y.abs() + (1 + u) * bound + TINY[x.dtype])
    # the codes: half a step, and what y is off by (twice: once in the largest value, which the step is made of)
    step = y.abs().amax(1) / 127
    off = bound.amax(1)
    assert close(scale, step, off / 127 + 2.0 ** -22 * step + 2.0 ** -149)
    held = q.double() * scale.double()[:, None]
    assert ((held - y).abs() <= 0.5 * step[:, None] + 2 * off[:, None] + 2.0 ** -20 * y.abs() + 2.0 ** -140).all()
    assert q.abs().max() <= 127 and (q.abs().amax(1)[step > 0] == 127).all()
    return got, q, scale


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["layer", "rms", "none"])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (5, 8), (2, 31), (65, 128), (33, 255), (9, 256), (300, 512), (17, 520), (4, 1000), (3, 1024),
                                        (5, 1032), (2, 4095), (3, 4096), (7, 5120), (2, 8192), (2, 8200), (1, 16385), (2, 32761), (2, 32768)])
def test_widths(native_lib, dtype, kind, rows, width):
    x, r = make(rows, width, dtype, 1), make(rows, width, dtype, 2, 1.5)
    w, b = (None, None) if kind == "none" else (make(1, width, dtype, 3, 0.2, 1.0)[0], make(1, width, dtype, 4, 0.1)[0])
    check(native_lib, x, kind, w, b, residual=r, residual_scale=2.4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weight,bias,residual", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (1, 1, 0), (0, 0, 1)])
def test_what_may_be_left_out(native_lib, dtype, weight, bias, residual):
    x = make(40, 200, dtype, 5, 3.0, 2.0)
    w = make(1, 200, dtype, 6, 0.2, 1.0)[0] if weight else None
    b = make(1, 200, dtype, 7)[0] if bias else None
    r = make(40, 200, dtype, 8) if residual else None
    for kind in ("layer", "rms"):
        got, q, scale = check(native_lib, x, kind, w, b, 1e-3, r, -0.5)
        assert torch.equal(native_lib.norm(x, kind, w, b, 1e-3, r, -0.5), got)
        none, q2, scale2 = native_lib.norm(x, kind, w, b, 1e-3, r, -0.5, out=False, quantize=True)
        assert none is None and torch.equal(q, q2) and torch.equal(scale, scale2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [64, 72, 100, 2048, 2056])
def test_strides_and_offsets(native_lib, dtype, width):
    # rows further apart than their width, and starts off the 16-byte boundary
    for offset, stride in ((0, width + 8), (1, width + 8), (8, width + 9), (3, 2 * width + 1)):
        base, rbase, obase = (make(1, 12 * stride + 64, dtype, n)[0] for n in (1, 2, 3))
        x, r, o = (t[offset : offset + 12 * stride].view(12, stride)[:, :width] for t in (base, rbase, obase))
        before = obase.clone()
        check(native_lib, x, "layer", residual=r, out=o)
        touched = torch.zeros_like(obase, dtype=torch.bool)
        touched[offset : offset + 12 * stride].view(12, stride)[:, :width] = True
        assert torch.equal(obase[~touched], before[~touched])
    same = make(1, width, dtype, 9).expand(30, width)  # one row read thirty times
    got, q, _ = check(native_lib, same, "rms")
    assert (got == got[0]).all() and (q == q[0]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 3, 7, 9, 15, 101, 250, 511, 1021, 1023, 2001, 4099, 8191, 8193, 32767])
@pytest.mark.parametrize("kind", ["layer", "rms", "none"])
def test_odd_widths_next_to_rows_that_hold_no_numbers(native_lib, dtype, width, kind):
    # rows without room between them: what is read around a row is its neighbours', and has no part in it
    x, r = make(9, width, dtype, 1), make(9, width, dtype, 2)
    w, b = (None, None) if kind == "none" else (make(1, width, dtype, 3, 0.2, 1.0)[0], make(1, width, dtype, 4)[0])
    clean, q, scale = check(native_lib, x, kind, w, b, residual=r, residual_scale=0.5)
    x[::2], r[::2] = math.nan, math.inf
    got, q2, scale2 = native_lib.norm(x, kind, w, b, residual=r, residual_scale=0.5, quantize=True)
    assert torch.equal(got[1::2], clean[1::2]) and torch.equal(q[1::2], q2[1::2]) and torch.equal(scale[1::2], scale2[1::2])
    assert torch.isnan(scale2[::2]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [96, 101, 6000])
def test_in_place(native_lib, dtype, width):
    x, r = make(50, width, dtype, 1), make(50, width, dtype, 2)
    want = native_lib.norm(x, "layer", residual=r)
    x2, r2 = x.clone(), r.clone()
    assert torch.equal(native_lib.norm(x2, "layer", residual=r, out=x2), want)
    assert torch.equal(native_lib.norm(x, "layer", residual=r2, out=r2), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_constants_and_no_numbers(native_lib, dtype):
    x = make(8, 512, dtype, 3)
    x[1] = 0
    x[2] = 4
    x[3, 17] = math.inf
    x[4, 100] = math.nan
    x[5, 511] = -math.inf
    x[6] = 6e-8 if dtype == torch.float16 else 1e-38
    for kind in ("layer", "rms", "none"):
        y, q, scale = native_lib.norm(x, kind, quantize=True)
        assert torch.isnan(scale[3:6]).all() and (q[3:6] == 0).all()
        assert (q[1] == 0).all() and scale[1] == 0 and (y[1] == 0).all()
        if kind != "none":
            assert torch.isnan(y[4]).all()
        keep = [0, 1, 2, 7] + ([6] if kind == "none" else [])
        check(native_lib, x[keep], kind)
    check(native_lib, x[2:3], "layer")  # no deviation at all: zeros
    assert (native_lib.norm(x[2:3], "layer") == 0).all()
    # a large mean and a small deviation: nothing cancels but what the sums cost
    check(native_lib, make(16, 700, dtype, 4, 0.5, 100.0), "layer", eps=0.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_go_to_the_even_step(native_lib, dtype):
    # 127 steps to 127: every value its own code, every half between two codes to the even one
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 125.5]], device="cuda").to(dtype)
    q, scale = native_lib.quantize_i8(x)
    want = torch.round(x.float())
    assert torch.equal(q.float(), want) and scale.item() == 1.0


def test_no_rows_and_many(native_lib):
    assert native_lib.norm(torch.empty(0, 16, device="cuda", dtype=torch.float16), "rms").shape == (0, 16)
    q, scale = native_lib.quantize_i8(torch.empty(0, 16, device="cuda", dtype=torch.float16))
    assert q.shape == (0, 16) and scale.shape == (0,)
    check(native_lib, make(40007, 72, torch.float16, 5), "rms")


def test_offsets_beyond_32_bits(native_lib):
    # 2^31 elements between the first and the last row
    stride = 1 << 29
    base = torch.empty(4 * stride + 64, dtype=torch.float16, device="cuda")
    x = base[: 5 * stride].as_strided((5, 64), (stride, 1)) if base.numel() >= 5 * stride else base.as_strided((5, 64), (stride, 1))
    x.copy_(make(5, 64, torch.float16, 6))
    check(native_lib, x, "layer")


def test_captured_and_on_another_stream(native_lib):
    x, r = make(64, 512, torch.float16, 1), make(64, 512, torch.float16, 2)
    want = native_lib.norm(x, "layer", residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = native_lib.norm(x, "layer", residual=r, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        native_lib.norm(x, "layer", residual=r, out=out)
    x.copy_(make(64, 512, torch.float16, 3))
    graph.replay()
    assert torch.equal(out, native_lib.norm(x, "layer", residual=r))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1032, 1040, 1536, 2504, 4088, 8184, 8192, 8200, 9000, 9001, 12289, 16384, 16392, 20001, 24576])
def test_wide_rows_in_turn(native_lib, dtype, width):
    # more rows than blocks are launched for, and a few; in place
    for rows in (5, 1500):
        x, r = make(rows, width, dtype, 1), make(rows, width, dtype, 2)
        w, b = make(1, width, dtype, 3, 0.2, 1.0)[0], make(1, width, dtype, 4, 0.1)[0]
        got, q, scale = check(native_lib, x, "layer", w, b, residual=r, residual_scale=2.4)
        again = native_lib.norm(x, "layer", w, b, residual=r, residual_scale=2.4, out=x, quantize=True)
        assert torch.equal(again[0], got) and torch.equal(again[1], q) and torch.equal(again[2], scale)
