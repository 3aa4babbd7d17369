"""The 8-bit layer's host-side bookkeeping (csrc/layer_host.h) with fakes of the CUDA calls behind it."""
import ctypes as C
import itertools
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "hostcheck", "layer_host.cpp")
INC = os.path.join(ROOT, "intel_gaudi3_software_b200", "csrc")


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("host") / "liblayer_host.so")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-Wall", "-fPIC", "-shared", "-I" + INC, "-o", so, SRC])
    return C.CDLL(so)


def holds(host, times, failures, answer, instead):
    results, forgotten = (C.c_int * times)(), C.c_int()
    asked = host.hc_device_holds(times, failures, answer, instead, results, C.byref(forgotten))
    return list(results), asked, forgotten.value


def test_an_answer_is_asked_for_once(host):
    assert holds(host, 3, 0, 74, -1) == ([74, 74, 74], 1, 0)
    assert holds(host, 3, 0, 0, -1) == ([0, 0, 0], 1, 0)       # none fit: an answer too
    assert holds(host, 2, 0, 0, 37) == ([37, 37], 1, 0)


def test_a_failed_question_is_asked_again_and_its_error_cleared(host):
    assert holds(host, 4, 2, 74, -1) == ([-1, -1, 74, 74], 3, 2)


def test_a_number_instead_of_a_failed_answer_stays(host):
    """The gradient's workspace is asked for and used by two calls: both have to see the same number."""
    assert holds(host, 3, 1, 74, 18) == ([18, 18, 18], 1, 1)


@pytest.mark.parametrize("takes,fails,mark_status,marks,status", [(0, 0, 0, 0, 0), (0, 1, 0, 0, -3), (1, 0, 0, 1, 0), (1, 1, 0, 1, -3), (1, 0, -7, 1, -7)])
def test_the_use_of_scratch_memory_is_marked_once_on_every_way_out(host, takes, fails, mark_status, marks, status):
    got = C.c_int()
    assert host.hc_use_mark(takes, fails, mark_status, C.byref(got)) == marks and got.value == status


def test_rows_lie_apart_only_where_no_byte_is_shared(host):
    """Against the set of bytes of each tensor: never yes where they share one, and yes for column ranges of one matrix."""
    rng = random.Random(3)

    def apart(a, na, b, nb, strides):
        return host.hc_rows_lie_apart(C.c_uint64(a), C.c_uint64(na), C.c_uint64(b), C.c_uint64(nb), (C.c_uint64 * len(strides))(*strides), len(strides))

    def cells(at, n, dims):
        return {at + sum(i * s for i, (_, s) in zip(index, dims)) + k for index in itertools.product(*(range(c) for c, _ in dims)) for k in range(n)}

    yes = 0
    for _ in range(4000):
        pitch = rng.choice([8, 12, 16, 24])
        a, b, na, nb = rng.randrange(100, 130), rng.randrange(100, 130), rng.randrange(1, 14), rng.randrange(1, 14)
        da, db = ([(rng.randrange(2, 5), pitch * rng.choice([1, 1, 2])), (rng.randrange(2, 4), pitch * rng.choice([1, 3, 4]))] for _ in range(2))
        if apart(a, na, b, nb, [s for _, s in da + db]):
            yes += 1
            assert not cells(a, na, da) & cells(b, nb, db)
    assert yes > 100
    for lo, hi in ((0, 40), (40, 0)):      # the two halves of rows of 80 bytes, either way round; one byte more is too much
        assert apart(1000 + lo, 40, 1000 + hi, 40, [80, 0, 80]) and not apart(1000 + lo, 41, 1000 + hi, 40, [80, 80])
        assert apart(1000 + lo, 40, 1000 + hi + 800, 40, [80, 160])
    assert not apart(1000, 4, 1100, 4, [0, 0])
