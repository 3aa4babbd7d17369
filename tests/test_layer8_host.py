"""The 8-bit layer's host-side bookkeeping (csrc/layer_host.h) with fakes of the CUDA calls behind it."""
import ctypes as C
import os
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
