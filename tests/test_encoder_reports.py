"""Who is told that a kernel of the encoder's operators has given up waiting: the host's part, built without a GPU.  The
device counts; every thread hears of what is new to it."""
import ctypes as C
import os
import subprocess
import threading

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture()
def host(tmp_path):
    so = str(tmp_path / "libreports.so")
    subprocess.run(["g++", "-O2", "-fPIC", "-shared", "-std=c++17", "-o", so, os.path.join(HERE, "host_model", "reports.cpp"), "-lpthread"], check=True)
    return C.CDLL(so)


def elsewhere(f, *args):
    """f's result from a thread of its own."""
    got = []
    t = threading.Thread(target=lambda: got.append(f(*args)))
    t.start()
    t.join()
    return got[0]


class Thread:
    """A thread that does one thing after the other as it is told."""

    def __init__(self):
        from concurrent.futures import ThreadPoolExecutor
        self.pool = ThreadPoolExecutor(1)

    def __call__(self, f, *args):
        return self.pool.submit(f, *args).result()


def test_a_thread_is_told_once(host):
    assert host.take(0, 0) == 0
    assert host.take(0, 1) == 1 and host.take(0, 1) == 0
    assert host.take(0, 5) == 1 and host.take(0, 5) == 0


def test_devices_are_apart(host):
    assert host.take(3, 1) == 1 and host.take(4, 0) == 0 and host.take(4, 2) == 1 and host.take(3, 1) == 0
    assert host.take(64, 0) == 0 and host.take(64, 1) == 1  # beyond the list: whatever there is


def test_one_thread_s_look_takes_no_other_s_report(host):
    a, b = Thread(), Thread()
    a(host.begin, 0)
    b(host.begin, 0)
    assert b(host.take, 0, 1) == 1  # (a kernel of a's)
    assert a(host.take, 0, 1) == 1
    assert a(host.take, 0, 1) == 0 and b(host.take, 0, 1) == 0


def test_a_new_thread_hears_of_what_is_new(host):
    assert host.take(0, 2) == 1
    late = Thread()
    late(host.begin, 0)
    assert late(host.take, 0, 2) == 0
    assert late(host.take, 0, 3) == 1
    assert elsewhere(host.take, 0, 3) == 0  # one that only looks: what nobody has been told yet
    assert elsewhere(host.take, 0, 4) == 1


def test_a_device_that_was_reset_counts_anew(host):
    assert host.take(0, 3) == 1 and host.take(0, 0) == 0 and host.take(0, 1) == 1
    assert elsewhere(host.take, 0, 1) == 0
