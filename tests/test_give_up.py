"""What a block of the matrix kernels does about its copies when one of its waits has run out, built for the host: none may be under way
when the block ends, however far each block of a pair has come."""
import ctypes as C
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("give_up") / "libgive_up.so")
    subprocess.run(["g++", "-O2", "-fPIC", "-shared", "-o", so, os.path.join(HERE, "host_model", "give_up.cpp")], check=True)
    return C.CDLL(so)


@pytest.mark.parametrize("ring", [2, 5, 7])
def test_no_copy_is_under_way_when_a_block_ends(host, ring):
    # from nothing issued to a ring ahead of what has been read, in the first rounds of the ring and later ones
    for read in range(3 * ring):
        for mine in range(read, read + ring + 1):
            assert host.copies_left(ring, read, mine, mine, 0) == 0, (read, mine)


@pytest.mark.parametrize("ring", [2, 5, 7])
def test_no_copy_is_under_way_when_a_pair_ends(host, ring):
    # either block may be ahead of the other
    for read in range(3 * ring):
        for mine in range(read, read + ring + 1):
            for theirs in range(read, read + ring + 1):
                assert host.copies_left(ring, read, mine, theirs, 1) == 0, (read, mine, theirs)
