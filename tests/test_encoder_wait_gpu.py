"""The way from a wait that runs out in the encoder's kernels to the host's error, without anything being wrong: one block waits a
millisecond for a barrier that nothing completes."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

pytestmark = pytest.mark.gpu


def told(of, stream=None):
    try:
        of.encoder_wait(stream)
    except of.OpenfishError as e:
        assert e.status == 7  # OPENFISH_B200_ERR_DEVICE_WAIT
        return True
    return False


def use(of):
    x = torch.randn(40, 64, device="cuda").half()
    q, s = of.quantize_i8(x)
    of.matmul_i8(q, s, q, s)
    start = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    return of.attention(x[:, None], x[:, None], x[:, None], start, start, 40, 40)


@pytest.mark.parametrize("kernels", [1, 2, 3])
def test_a_wait_that_runs_out_is_reported_once(native_lib, kernels):
    use(native_lib)
    assert not told(native_lib)
    for limit in (1000, 200):
        assert native_lib.selfcheck_encoder_wait(kernels, limit) == 0
        assert told(native_lib) and not told(native_lib)
    use(native_lib)
    assert not told(native_lib)


def test_a_wait_on_another_stream(native_lib):
    side = torch.cuda.Stream()
    assert native_lib.selfcheck_encoder_wait(3, 300, side) == 0
    side.synchronize()
    assert told(native_lib) and not told(native_lib, side)


def test_every_thread_is_told(native_lib):
    one, two, late = (ThreadPoolExecutor(1) for _ in range(3))
    for t in (one, two):
        t.submit(use, native_lib).result()
        assert not t.submit(told, native_lib).result()
    assert one.submit(native_lib.selfcheck_encoder_wait, 1, 300).result() == 0
    torch.cuda.synchronize()
    assert two.submit(told, native_lib).result()  # the other one's look takes nothing away
    assert one.submit(told, native_lib).result()
    late.submit(use, native_lib).result()  # (what has been reported by its first call is no concern of its kernels)
    assert [t.submit(told, native_lib).result() for t in (one, two, late)] == [False, False, False]
    assert told(native_lib) and not told(native_lib)


def test_what_it_refuses(native_lib):
    for kernels in (0, 4, -1):
        assert native_lib.selfcheck_encoder_wait(kernels) == 1  # OPENFISH_B200_ERR_ARGUMENT
    assert not told(native_lib)
