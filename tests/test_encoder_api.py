"""The encoder's entry points without a GPU: struct layouts, refusals, calls with nothing to do."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARGUMENT, LAYOUT, SHAPE, TOO_LONG = 1, 2, 3, 9
P = 1 << 20  # an address that is never followed


@pytest.fixture()
def lib(native_lib):
    L = native_lib.lib()
    L.set_openfish_log_level(0)
    yield L
    L.set_openfish_log_level(4)


@pytest.mark.parametrize("struct,mirror", [("openfish_b200_attention_t", "AttentionArgs"), ("openfish_b200_matmul_i8_t", "MatmulI8Args"),
                                           ("openfish_b200_norm_t", "NormArgs")])
def test_struct_layouts_match_the_header(native_lib, tmp_path, struct, mirror):
    m = getattr(native_lib.encoder, mirror)
    names = [f[0] for f in m._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"openfish_b200.h\"\nint main(void) {\n    printf(\"%%zu\", sizeof(%s));\n%s    return 0;\n}\n" % (
        struct, "".join("    printf(\" %%zu %%zu\", offsetof(%s, %s), sizeof(((%s *)0)->%s));\n" % (struct, n, struct, n) for n in names)))
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(m)] + [v for n in names for v in (getattr(m, n).offset, getattr(m, n).size)]


def attention(of, **change):
    a = of.encoder.AttentionArgs(dtype=0, head_dim=64, q_heads=8, kv_heads=4, sequences=2, max_q=10, max_k=20, window_left=-1, window_right=0,
                                 scale=0.125, q_rows=20, k_rows=40, q_start=P, k_start=P, q=P, k=P, v=P, out=P, q_stride_row=512,
                                 q_stride_head=64, k_stride_row=256, k_stride_head=64, v_stride_row=256, v_stride_head=64,
                                 out_stride_row=512, out_stride_head=64)
    for n, v in change.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), ARGUMENT), (dict(dtype=-1), ARGUMENT), (dict(head_dim=0), SHAPE), (dict(head_dim=60), SHAPE), (dict(head_dim=136), SHAPE),
    (dict(q_heads=0), SHAPE), (dict(kv_heads=0), SHAPE), (dict(kv_heads=3), SHAPE), (dict(q_heads=-8, kv_heads=-4), SHAPE),
    (dict(sequences=-1), SHAPE), (dict(max_q=-1), SHAPE), (dict(max_k=-1), SHAPE), (dict(q_rows=-1), SHAPE), (dict(k_rows=-1), SHAPE),
    (dict(q_rows=1 << 31), TOO_LONG), (dict(k_rows=1 << 31), TOO_LONG), (dict(max_q=1 << 30), TOO_LONG), (dict(max_k=(1 << 31) - 1), TOO_LONG),
    (dict(sequences=1 << 30), TOO_LONG), (dict(scale=0.0), ARGUMENT), (dict(scale=-1.0), ARGUMENT), (dict(scale=float("nan")), ARGUMENT),
    (dict(scale=float("inf")), ARGUMENT), (dict(window_left=-2), ARGUMENT), (dict(window_right=-2), ARGUMENT),
    (dict(q_start=None), ARGUMENT), (dict(k_start=None), ARGUMENT), (dict(q=None), ARGUMENT), (dict(k=None), ARGUMENT), (dict(v=None), ARGUMENT),
    (dict(out=None), ARGUMENT), (dict(q_start=P + 2), LAYOUT), (dict(k_used=P + 1), LAYOUT), (dict(q=P + 8), LAYOUT), (dict(k=P + 2), LAYOUT),
    (dict(v=P + 4), LAYOUT), (dict(out=P + 8), LAYOUT), (dict(q_stride_row=500), LAYOUT), (dict(k_stride_row=0), LAYOUT),
    (dict(k_stride_row=-256), LAYOUT), (dict(v_stride_head=63), LAYOUT), (dict(out_stride_row=516), LAYOUT), (dict(v_stride_row=1 << 39), LAYOUT)])
def test_attention_refuses(native_lib, lib, change, status):
    lib.openfish_b200_attention(None, C.byref(attention(native_lib, **change)))
    assert lib.openfish_b200_last_status() == status, lib.openfish_b200_error_text()


@pytest.mark.parametrize("change", [dict(sequences=0), dict(q_rows=0), dict(max_q=0), dict(sequences=0, q_start=None, q=None, out=None)])
def test_attention_with_nothing_to_do(native_lib, lib, change):
    a = attention(native_lib, **change)
    assert lib.openfish_b200_attention_workspace(C.byref(a)) == 0
    lib.openfish_b200_attention(None, C.byref(a))
    assert lib.openfish_b200_last_status() == 0


def matmul(of, **change):
    a = of.encoder.MatmulI8Args(dtype=1, cols=100, depth=60, rows=50, x=P, w=P, x_scale=P, w_scale=P, out=P, x_stride=64, w_stride=64, out_stride=100)
    for n, v in change.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(dtype=7), ARGUMENT), (dict(rows=-1), SHAPE), (dict(cols=0), SHAPE), (dict(depth=0), SHAPE), (dict(depth=131072, x_stride=131072, w_stride=131072), TOO_LONG),
    (dict(rows=(1 << 30) + 1), TOO_LONG), (dict(cols=(1 << 30) + 1), TOO_LONG), (dict(x=None), ARGUMENT), (dict(w=None), ARGUMENT), (dict(x_scale=None), ARGUMENT),
    (dict(w_scale=None), ARGUMENT), (dict(out=None), ARGUMENT), (dict(x=P + 8), LAYOUT), (dict(w=P + 1), LAYOUT), (dict(x_stride=60), LAYOUT),
    (dict(x_stride=48), LAYOUT), (dict(w_stride=72), LAYOUT), (dict(w_stride=0), LAYOUT), (dict(x_scale=P + 2), LAYOUT), (dict(bias=P + 1), LAYOUT),
    (dict(out=P + 1), LAYOUT), (dict(out_stride=99), LAYOUT)])
def test_matmul_i8_refuses(native_lib, lib, change, status):
    lib.openfish_b200_matmul_i8(None, C.byref(matmul(native_lib, **change)))
    assert lib.openfish_b200_last_status() == status, lib.openfish_b200_error_text()


def norm(of, **change):
    a = of.encoder.NormArgs(dtype=0, kind=1, width=100, eps=1e-5, residual_scale=1.0, rows=10, x=P, out=P, x_stride=100, out_stride=100, q_stride=112)
    for n, v in change.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), ARGUMENT), (dict(kind=3), ARGUMENT), (dict(kind=-1), ARGUMENT), (dict(rows=-1), SHAPE), (dict(width=0), SHAPE), (dict(width=32769), TOO_LONG),
    (dict(eps=-1.0), ARGUMENT), (dict(eps=float("nan")), ARGUMENT), (dict(kind=0, weight=P), ARGUMENT), (dict(kind=0, bias=P), ARGUMENT),
    (dict(x=None), ARGUMENT), (dict(out=None), ARGUMENT), (dict(q=P), ARGUMENT), (dict(x=P + 1), LAYOUT), (dict(residual=P + 1), LAYOUT),
    (dict(out=P + 1), LAYOUT), (dict(out_stride=96), LAYOUT), (dict(q=P, q_scale=P, q_stride=64), LAYOUT), (dict(q=P, q_scale=P + 2), LAYOUT)])
def test_norm_refuses(native_lib, lib, change, status):
    lib.openfish_b200_norm(None, C.byref(norm(native_lib, **change)))
    assert lib.openfish_b200_last_status() == status, lib.openfish_b200_error_text()


def test_no_arguments_and_no_rows(native_lib, lib):
    for f in (lib.openfish_b200_attention, lib.openfish_b200_matmul_i8, lib.openfish_b200_norm):
        f(None, None)
        assert lib.openfish_b200_last_status() == ARGUMENT
    assert lib.openfish_b200_attention_workspace(None) == 0 and lib.openfish_b200_last_status() == ARGUMENT
    lib.openfish_b200_matmul_i8(None, C.byref(matmul(native_lib, rows=0, x=None, out=None)))
    assert lib.openfish_b200_last_status() == 0
    lib.openfish_b200_norm(None, C.byref(norm(native_lib, rows=0, x=None, out=None)))
    assert lib.openfish_b200_last_status() == 0


def test_host_tensors_are_refused(native_lib):
    import torch
    x = torch.zeros(4, 64, dtype=torch.float16)
    q = torch.zeros(4, 64, dtype=torch.int8)
    starts = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError):
        native_lib.norm(x, "rms")
    with pytest.raises(ValueError):
        native_lib.norm(x, "batch")
    with pytest.raises(TypeError):
        native_lib.quantize_i8(x)
    with pytest.raises(TypeError):
        native_lib.matmul_i8(q, torch.ones(4), q, torch.ones(4))
    with pytest.raises(TypeError):
        native_lib.attention(x[:, None], x[:, None], x[:, None], starts, starts, 4, 4)


@pytest.mark.parametrize("change,status", [
    (dict(out_stride_row=448), LAYOUT), (dict(out_stride_head=56), LAYOUT), (dict(out_stride_row=64, out_stride_head=64), LAYOUT), (dict(q_heads=4, out_stride_row=248), LAYOUT),
    (dict(out_stride_row=64, out_stride_head=64 * 19), LAYOUT), (dict(out_stride_row=56, out_stride_head=56 * 20), LAYOUT), (dict(kv_heads=1, q_heads=1, out_stride_row=56), LAYOUT),
    (dict(q_rows=1, out_stride_head=56), LAYOUT)])
def test_attention_refuses_results_that_share_places(native_lib, lib, change, status):
    lib.openfish_b200_attention(None, C.byref(attention(native_lib, **change)))
    assert lib.openfish_b200_last_status() == status, lib.openfish_b200_error_text()
    assert b"overlap" in lib.openfish_b200_error_text()


@pytest.mark.parametrize("pack,args", [("_pack_attention", "AttentionArgs"), ("_pack_matmul_i8", "MatmulI8Args"), ("_pack_norm", "NormArgs")])
@pytest.mark.parametrize("number", [1 << 31, 1 << 70, 2.5, None])
def test_numbers_that_no_field_holds_are_refused(native_lib, pack, args, number):
    fields = [0] * len(getattr(native_lib.encoder, args)._fields_)
    assert len(getattr(native_lib.encoder, pack)(*fields)) == C.sizeof(getattr(native_lib.encoder, args))
    fields[1] = number
    with pytest.raises(ValueError):
        getattr(native_lib.encoder, pack)(*fields)


def test_results_that_share_places_beyond_64_bits(native_lib, lib):
    # 10^9 heads, 2^38 elements apart, in rows no further apart
    a = attention(native_lib, q_heads=10 ** 9, kv_heads=1, sequences=1, max_q=1, q_stride_head=64, out_stride_row=1 << 38, out_stride_head=1 << 38)
    lib.openfish_b200_attention(None, C.byref(a))
    assert lib.openfish_b200_last_status() == LAYOUT and b"overlap" in lib.openfish_b200_error_text()
