"""What the Python calls of the encoder's operators refuse on a GPU, and that nothing is left behind by it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def cuda(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def starts(*at):
    return torch.tensor(at, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("error,change", [
    (TypeError, dict(q="float32")), (TypeError, dict(q="2d")), (TypeError, dict(k="cpu")), (TypeError, dict(v="bf16")),
    (ValueError, dict(k="dim")), (ValueError, dict(v="rows")), (ValueError, dict(q="strided")), (TypeError, dict(q_start="int64")),
    (ValueError, dict(k_start="longer")), (ValueError, dict(k_used="longer")), (TypeError, dict(k_used="int64")), (ValueError, dict(out="shape")),
    (TypeError, dict(out="float32"))])
def test_attention_refuses_what_is_no_such_tensor(native_lib, error, change):
    a = dict(q=cuda(6, 4, 64), k=cuda(9, 2, 64), v=cuda(9, 2, 64), q_start=starts(0, 6), k_start=starts(0, 9), max_q=6, max_k=9)
    for name, how in change.items():
        x = a.get(name)
        a[name] = {"float32": lambda: cuda(6, 4, 64, dtype=torch.float32), "2d": lambda: x[0], "cpu": lambda: x.cpu(), "bf16": lambda: x.bfloat16(),
                   "dim": lambda: cuda(9, 2, 32), "rows": lambda: cuda(8, 2, 64), "strided": lambda: cuda(6, 4, 128)[:, :, ::2], "int64": lambda: starts(0, 6).long(),
                   "longer": lambda: starts(0, 4, 9), "shape": lambda: cuda(6, 4, 32)}.get(how, lambda: how)()
    with pytest.raises(error):
        native_lib.attention(**a)


@pytest.mark.parametrize("change", [dict(heads=3), dict(window=(-2, 0)), dict(window=(0, -2)), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(dim=60),
                                    dict(dim=136), dict(max_q=-1), dict(shift=1)])
def test_attention_refuses_what_it_cannot_serve(native_lib, change):
    dim, heads = change.pop("dim", 64), change.pop("heads", 2)
    q, k = cuda(6, 4, dim), cuda(9 * heads * dim + 8)[change.pop("shift", 0):][: 9 * heads * dim].view(9, heads, dim)
    max_q = change.pop("max_q", 6)
    out = torch.full_like(q, 7)
    with pytest.raises(native_lib.OpenfishError):
        native_lib.attention(q, k, k, starts(0, 6), starts(0, 9), max_q, 9, out=out, **change)
    assert (out == 7).all()


def test_products_and_norms_refuse(native_lib):
    x, w = cuda(4, 64, dtype=torch.int8), cuda(5, 64, dtype=torch.int8)
    xs, ws = cuda(4, dtype=torch.float32), cuda(5, dtype=torch.float32)
    for error, call in ((ValueError, lambda: native_lib.matmul_i8(x, xs, cuda(5, 32, dtype=torch.int8), ws)), (ValueError, lambda: native_lib.matmul_i8(x, ws, w, ws)),
                        (TypeError, lambda: native_lib.matmul_i8(x, xs.half(), w, ws)), (TypeError, lambda: native_lib.matmul_i8(x.half(), xs, w, ws)),
                        (TypeError, lambda: native_lib.matmul_i8(x, xs, w, ws, bias=cuda(5).float())), (TypeError, lambda: native_lib.matmul_i8(x, xs, w, ws, dtype=torch.float32)),
                        (ValueError, lambda: native_lib.matmul_i8(x, xs, w, ws, out=cuda(4, 6))),
                        (TypeError, lambda: native_lib.matmul_i8(x, xs, w, ws, dtype=torch.bfloat16, out=cuda(4, 5))),
                        (native_lib.OpenfishError, lambda: native_lib.matmul_i8(cuda(4, 65, dtype=torch.int8)[:, 1:], xs, w, ws)),
                        (native_lib.OpenfishError, lambda: native_lib.matmul_i8(cuda(4, 60, dtype=torch.int8), xs, cuda(5, 60, dtype=torch.int8), ws)),
                        (TypeError, lambda: native_lib.norm(cuda(4, 64, dtype=torch.float32), "rms")), (TypeError, lambda: native_lib.norm(cuda(4, 4, 4), "rms")),
                        (ValueError, lambda: native_lib.norm(cuda(4, 64), "rms", weight=cuda(63))), (TypeError, lambda: native_lib.norm(cuda(4, 64), "rms", weight=cuda(64).float())),
                        (ValueError, lambda: native_lib.norm(cuda(4, 64), "rms", residual=cuda(4, 63))), (ValueError, lambda: native_lib.norm(cuda(4, 128)[:, ::2], "rms")),
                        (native_lib.OpenfishError, lambda: native_lib.norm(cuda(4, 64), "none", weight=cuda(64))),
                        (native_lib.OpenfishError, lambda: native_lib.norm(cuda(4, 64), "rms", eps=-1.0)),
                        (native_lib.OpenfishError, lambda: native_lib.norm(cuda(2, 40000), "rms"))):
        with pytest.raises(error):
            call()
    assert native_lib.norm(cuda(4, 64), "rms").shape == (4, 64)  # a call after all those
    native_lib.encoder_wait()


def test_inputs_that_want_gradients(native_lib):
    # the results are plain tensors, whatever the inputs want
    x = cuda(4, 64).requires_grad_()
    assert not native_lib.norm(x, "rms").requires_grad
