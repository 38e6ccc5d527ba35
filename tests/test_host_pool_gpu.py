"""Packet pools from mi_cksum_host_alloc (mi.page_buffer): batches inside a
registered range are read in place over PCIe -- through the drop-in service (up
to 64 datagrams), one dispatch, or the whole grid -- and the host's writes
between calls are seen; batches outside it are staged.  Against the oracle."""
import threading

import numpy as np
import pytest

import libunsod_amd as mi
from libunsod_amd import synth
from libunsod_amd._lib import load
from oracle.pyoracle import Oracle

pytestmark = pytest.mark.gpu
ORC = Oracle("port")
STRIDE, FIRST, L = 2176, 142, 1500
LAY = dict(stride=STRIDE, first_off=FIRST, fixed_len=L)
OLAY = dict(stride=STRIDE, first_off=FIRST, fixed_flen=L)


def _pool(n, seed):
    b = synth.build_ipv4_batch(n, L, stride=STRIDE, first_off=FIRST, seed=seed)
    pool = mi.page_buffer(b["buf"].size)
    pool[:] = b["buf"]
    ORC.ipv4_finalize_batch(pool, n, **OLAY)
    return pool


def _in_place(buf):
    lib = load()
    lib.mi__reg_table_lookup.restype = np.ctypeslib.ctypes.c_uint64
    lib.mi__reg_table_lookup.argtypes = [np.ctypeslib.ctypes.c_void_p, np.ctypeslib.ctypes.c_uint64]
    return lib.mi__reg_table_lookup(buf.ctypes.data, buf.nbytes) != 0


@pytest.mark.parametrize("n", [1, 64, 65, 600, 5000])
def test_host_writes_between_bursts_are_seen(n):
    """The same slots rewritten by the host, 12 bursts in a row: each verify sees
    this burst's bytes, in place and staged alike."""
    pool = _pool(n, seed=n)
    rng = np.random.default_rng(n)
    mi.host_register(pool)
    try:
        assert _in_place(pool)
        for burst in range(12):
            pick = rng.choice(n, min(n, 1 + burst % 3), replace=False)
            at = FIRST + pick.astype(np.int64) * STRIDE + rng.integers(20, L, pick.size)
            pool[at] ^= 0x21
            want = ORC.ipv4_verify_batch(pool, n, **OLAY)
            for staged in (False, True):
                ip, l4, st, bad = mi.ipv4_verify_host(pool, n, staged=staged, **LAY)
                assert np.array_equal(ip, want[0]) and np.array_equal(l4, want[1]), (burst, staged)
                assert np.array_equal(st, want[2]) and bad == int((want[2] != 0).sum()) > 0, (burst, staged)
            pool[at] ^= 0x21
    finally:
        mi.host_unregister(pool)
    ip, l4, st, bad = mi.ipv4_verify_host(pool, n, **LAY)
    assert bad == 0 and not st.any() and not ip.any() and not l4.any()


def test_a_range_of_a_block():
    """Part of a block registered: a batch inside it goes in place, one that
    reaches past it is staged; both right.  Ranges of one block come and go."""
    n = 400
    pool = _pool(n, seed=77)
    pool[FIRST + 250 * STRIDE + 99] ^= 1
    half = (pool.nbytes // 2) & ~4095
    front, back = pool[:half], pool[half:]
    mi.host_register(front)
    try:
        k = (half - FIRST - L) // STRIDE  # the slots wholly inside the front
        for buf, cnt, where in ((front, k, True), (pool, n, False)):
            assert _in_place(buf) == where
            want = ORC.ipv4_verify_batch(pool, cnt, **OLAY)
            ip, l4, st, bad = mi.ipv4_verify_host(buf, cnt, **LAY)
            assert np.array_equal(l4, want[1]) and np.array_equal(st, want[2]) and bad == int((want[2] != 0).sum())
        mi.host_register(back)
        mi.host_unregister(back)
        with pytest.raises(mi.MiCksumError) as e:
            mi.host_register(pool)  # shares pages with the front
        assert e.value.rc == -17
    finally:
        mi.host_unregister(front)


def test_pools_of_several_threads():
    """Threads with a pool each, alive side by side: registered, verified in
    place, unregistered and freed while the others' calls run."""
    errors = []

    def work(t):
        try:
            for r in range(4):
                n = (8, 200)[r % 2]
                pool = _pool(n, seed=100 * t + r)
                pool[FIRST + (n // 2) * STRIDE + 50] ^= 2
                want = ORC.ipv4_verify_batch(pool, n, **OLAY)
                mi.host_register(pool)
                try:
                    for _ in range(3):
                        ip, l4, st, bad = mi.ipv4_verify_host(pool, n, **LAY)
                        if bad != 1 or not np.array_equal(l4, want[1]) or not np.array_equal(st, want[2]):
                            errors.append((t, r, bad))
                finally:
                    mi.host_unregister(pool)
        except Exception as e:  # noqa: BLE001 -- reported below
            errors.append((t, repr(e)))

    ts = [threading.Thread(target=work, args=(t,)) for t in range(8)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in ts) and not errors, errors[:5]
