"""What the host layer of the encoder's operators makes of a CUDA side that fails or has given up waiting.  The layer is built over
one made for the purpose; no GPU is involved."""
import ctypes as C
import os
import subprocess

import pytest

from openfish_b200 import encoder

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
P = 1 << 20  # an address that is never followed
CUDA, DEVICE_WAIT = 6, 7


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("fake_encoder") / "libfake.so")
    csrc = os.path.join(ROOT, "openfish_b200", "csrc")
    subprocess.run(["gcc", "-O1", "-fPIC", "-shared", "-std=gnu11", "-I", os.path.join(ROOT, "include"), "-I", csrc, "-o", so,
                    os.path.join(csrc, "openfish_api.c"), os.path.join(csrc, "encoder_api.c"),
                    os.path.join(HERE, "host_model", "failing_backend.c"), os.path.join(HERE, "host_model", "fake_encoder.c")], check=True)
    L = C.CDLL(so)
    L.openfish_b200_set_error_mode(1)
    L.set_openfish_log_level(0)
    L.openfish_b200_error_text.restype = C.c_char_p
    encoder.declare(L)
    return L


def value(lib, name):
    return C.c_int.in_dll(lib, name)


ATTENTION = dict(dtype=0, head_dim=64, q_heads=8, kv_heads=4, sequences=2, max_q=10, max_k=20, window_left=-1, window_right=0, scale=0.125,
                 q_rows=20, k_rows=40, q_start=P, k_start=P, q=P, k=P, v=P, out=P, q_stride_row=512, q_stride_head=64, k_stride_row=256,
                 k_stride_head=64, v_stride_row=256, v_stride_head=64, out_stride_row=512, out_stride_head=64)
CALLS = [("openfish_b200_attention", encoder.AttentionArgs, ATTENTION),
         ("openfish_b200_matmul_i8", encoder.MatmulI8Args, dict(dtype=1, cols=100, depth=60, rows=50, x=P, w=P, x_scale=P, w_scale=P, out=P,
                                                                x_stride=64, w_stride=64, out_stride=100)),
         ("openfish_b200_norm", encoder.NormArgs, dict(dtype=0, kind=1, width=100, eps=1e-5, rows=10, x=P, out=P, x_stride=100, out_stride=100))]


@pytest.mark.parametrize("name,struct,fields", CALLS)
def test_a_call_that_fails_is_an_error(lib, name, struct, fields):
    value(lib, "fake_fails").value = 0
    getattr(lib, name)(None, C.byref(struct(**fields)))
    assert lib.openfish_b200_last_status() == 0
    value(lib, "fake_fails").value = 1
    getattr(lib, name)(None, C.byref(struct(**fields)))
    value(lib, "fake_fails").value = 0
    assert lib.openfish_b200_last_status() == CUDA and b"the backend says no" in lib.openfish_b200_error_text()


@pytest.mark.parametrize("gave_up", [(0, 0), (1, 0), (0, 1), (1, 1)])
def test_kernels_that_gave_up_are_reported(lib, gave_up):
    flags = (C.c_int * 2).in_dll(lib, "fake_gave_up")
    flags[:] = gave_up
    lib.openfish_b200_encoder_wait(None)
    assert lib.openfish_b200_last_status() == (DEVICE_WAIT if any(gave_up) else 0)
    flags[:] = (0, 0)
    value(lib, "fake_fails").value = 1
    lib.openfish_b200_encoder_wait(None)
    value(lib, "fake_fails").value = 0
    assert lib.openfish_b200_last_status() == CUDA


@pytest.mark.parametrize("workspace,room,served", [(0, 0, False), (P, 999, False), (P + 8, 1000, False), (P, 1000, True), (P, 2000, True)])
def test_a_workspace_that_is_too_small_is_refused(lib, workspace, room, served):
    C.c_size_t.in_dll(lib, "fake_workspace").value = 1000
    before = value(lib, "fake_calls").value
    a = encoder.AttentionArgs(**ATTENTION, workspace=workspace, workspace_bytes=room)
    assert lib.openfish_b200_attention_workspace(C.byref(a)) == 1000
    lib.openfish_b200_attention(None, C.byref(a))
    C.c_size_t.in_dll(lib, "fake_workspace").value = 0
    assert lib.openfish_b200_last_status() == (0 if served else 1)
    assert value(lib, "fake_calls").value == before + served


def test_a_refused_call_reaches_no_kernel(lib):
    before = value(lib, "fake_calls").value
    for name, struct, fields in CALLS:
        getattr(lib, name)(None, C.byref(struct(**dict(fields, dtype=9))))
        assert lib.openfish_b200_last_status() == 1
    assert value(lib, "fake_calls").value == before
