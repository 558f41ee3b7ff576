"""The table of shared-memory limits behind the library's launches, without a device: a limit belongs to one kernel on one
device, and it only ever grows; and what the calls about
a device say where there is none."""
import ctypes as C
import threading

import pytest

import pufferlean_b200 as plb

SET = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_size_t)


@pytest.fixture(scope="module")
def raise_smem():
    f = plb.lib().pl_test_raise_smem
    f.argtypes = [C.c_int, C.c_void_p, C.c_size_t, SET]
    f.restype = C.c_int
    return f


def test_limit_belongs_to_the_device(raise_smem):
    """A kernel that may use its memory on one device is set on the next one too, once on each."""
    calls = []
    on = SET(lambda k, n: calls.append((k, n)) or 0)
    for device in (60, 61, 60, 61):
        assert raise_smem(device, 0x1000, 200000, on) == 0
    assert calls == [(0x1000, 200000)] * 2
    assert raise_smem(60, 0x2000, 200000, on) == 0 and len(calls) == 3


def test_failed_limit_is_not_remembered(raise_smem):
    calls = []
    assert raise_smem(62, 0x1000, 100, SET(lambda k, n: calls.append(n) or -3)) == -3
    assert raise_smem(62, 0x1000, 100, SET(lambda k, n: calls.append(n) or 0)) == 0
    assert calls == [100, 100]


def test_limit_never_falls(raise_smem):
    """Two threads that ask for different sizes of one kernel: no call lowers what an earlier one was promised."""
    limit, seen = [0], []

    def put(k, n):
        seen.append((limit[0], n))
        limit[0] = n
        return 0

    on = SET(put)

    def go(sizes):
        for n in sizes * 50:
            assert raise_smem(59, 0x7000, n, on) == 0
            assert limit[0] >= n

    threads = [threading.Thread(target=go, args=(s,)) for s in ([53248, 51200], [51200, 73728, 50000])]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert limit[0] == 73728 and all(b > a for a, b in seen)


def test_full_table_still_sets(raise_smem):
    calls = []
    on = SET(lambda k, n: calls.append(k) or 0)
    for k in range(1, 300):
        assert raise_smem(63, k, 64, on) == 0
    assert raise_smem(63, 299, 64, on) == 0 and raise_smem(63, 5, 64, on) == 0
    assert calls == list(range(1, 300)) + [299]


def test_get_device_refuses_null():
    assert plb.lib().pl_get_device(None) == -1


def test_device_check_needs_a_device():
    if plb.device_count() == 0:
        assert plb.lib().pl_device_check() == -6 and plb.lib().pl_last_error()
    else:
        assert plb.lib().pl_device_check() == 0
