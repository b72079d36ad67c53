"""Numbers at the limits of what the encoder's entry points take, without a GPU: calls that are refused, or have nothing to do."""
import ctypes as C

import pytest

P = 1 << 20  # an address that is never followed
ARGUMENT = 1


@pytest.fixture()
def lib(native_lib):
    L = native_lib.lib()
    L.set_openfish_log_level(0)
    yield L
    L.set_openfish_log_level(4)


# the kernels count in powers of two: scale * log2(e) has to be an fp32 number as well
@pytest.mark.parametrize("scale,status", [(3.4e38, ARGUMENT), (2.4e38, ARGUMENT), (2.3e38, 0), (1e-45, 0)])
def test_a_scale_beyond_what_the_exponential_takes(native_lib, lib, scale, status):
    a = native_lib.encoder.AttentionArgs(dtype=0, head_dim=64, q_heads=8, kv_heads=4, sequences=0, max_q=10, max_k=20, window_left=-1, window_right=0,
                                         scale=scale, q_rows=20, k_rows=40, q_start=P, k_start=P, q=P, k=P, v=P, out=P, q_stride_row=512,
                                         q_stride_head=64, k_stride_row=256, k_stride_head=64, v_stride_row=256, v_stride_head=64,
                                         out_stride_row=512, out_stride_head=64)
    lib.openfish_b200_attention(None, C.byref(a))
    assert lib.openfish_b200_last_status() == status
    assert lib.openfish_b200_attention_workspace(C.byref(a)) == 0
    assert lib.openfish_b200_last_status() == status
