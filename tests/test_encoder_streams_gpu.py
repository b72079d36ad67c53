"""The encoder's operators on streams that are not their tensors' own: memory that is given back while a call still
waits to run, and the rotary embedding behind work on a side stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu
LONG = 300_000_000  # cycles: 0.15 s or more, for which a stream is kept busy


def calls(of):
    """(name, inputs, call) of every operator; call(inputs, stream)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    half = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    whole = lambda *s: torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    start = torch.arange(5, dtype=torch.int32, device="cuda") * 1000
    return [
        ("norm", {"x": half(4000, 512), "residual": half(4000, 512), "weight": half(512)},
         lambda t, stream: of.norm(t["x"], "rms", t["weight"], residual=t["residual"], quantize=True, stream=stream)),
        ("quantize", {"x": half(4000, 512)}, lambda t, stream: of.quantize_i8(t["x"], stream=stream)),
        ("matmul", {"x": whole(4000, 512), "w": whole(1024, 512), "xs": torch.rand(4000, generator=g, device="cuda"),
                    "ws": torch.rand(1024, generator=g, device="cuda"), "b": half(1024)},
         lambda t, stream: (of.matmul_i8(t["x"], t["xs"], t["w"], t["ws"], bias=t["b"], stream=stream),)),
        ("attention", {"q": half(4000, 8, 64), "k": half(4000, 2, 64), "v": half(4000, 2, 64), "start": start,
                       "used": torch.tensor([1000, 7, 0, 555], dtype=torch.int32, device="cuda")},
         lambda t, stream: (of.attention(t["q"], t["k"], t["v"], t["start"], t["start"], 1000, 1000, k_used=t["used"], stream=stream),)),
    ]


@pytest.mark.parametrize("which", range(4))
def test_inputs_may_be_given_back_once_the_call_returns(native_lib, which):
    _, inputs, call = calls(native_lib)[which]
    want = [w.clone() for w in call(inputs, None)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
    got = call(inputs, side)
    shapes = {n: (t.shape, t.dtype) for n, t in inputs.items()}
    inputs.clear()
    fresh = [torch.full(s, 3, dtype=d, device="cuda") for _ in range(2) for s, d in shapes.values()]  # into their places, if those are free
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del fresh


@pytest.mark.parametrize("which", range(4))
def test_results_may_be_given_back_while_they_are_read(native_lib, which):
    _, inputs, call = calls(native_lib)[which]
    want = [w.clone() for w in call(inputs, None)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = list(call(inputs, side))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(LONG)
    copies = [t.clone() for t in got]  # behind the pause
    shapes = [(t.shape, t.dtype) for t in got]
    got.clear()
    with torch.cuda.stream(side):
        fresh = [torch.full(s, 3, dtype=d, device="cuda") for _ in range(2) for s, d in shapes]
    for a, b in zip(copies, want):
        assert torch.equal(a, b)
    del fresh


def test_rotary_on_what_a_side_stream_makes(native_lib):
    # the embedding runs on the legacy default stream, which torch's side streams do not wait for nor are waited for by
    T, H, D = 500, 8, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    first, then = (torch.randn(T, 3 * H, D, generator=g, device="cuda").half() for _ in range(2))
    angle = torch.rand(T, D // 2, generator=g, device="cuda")
    sin, cos = torch.sin(angle), torch.cos(angle)
    args = (1, T, 2 * H, D, D // 2, T * 3 * H * D, 3 * H * D, D)
    want = then.clone()
    native_lib.rotary_emb_gpu(want, sin, cos, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
        first.copy_(then)
        native_lib.rotary_emb_gpu(first, sin, cos, *args)
        got = first.clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
