"""What the library's host code does when a HIP call fails: over a runtime of
host memory (tests/hip_stub.cpp), on the CPU."""
import pytest

import stubbed

import libunsod_amd as mi

pytestmark = pytest.mark.skipif(mi.device_count() > 0, reason="the stub runtime stands in for a missing GPU")


@pytest.fixture(scope="module")
def so(tmp_path_factory):
    return stubbed.build(tmp_path_factory.mktemp("hip_stub"))


# every entry point that launches: (name, the call)
LAUNCHES = r'''
n = 64
b = batch(n)
o16, o8, o32 = np.zeros(2 * n, np.uint16), np.zeros(n, np.uint8), np.zeros(2 * n, np.uint32)
p16, p8, p32 = o16.ctypes.data, o8.ctypes.data, o32.ctypes.data
seg_off, seg_len = (np.arange(n) * 2176).astype(np.uint64), np.full(n, 1500, np.int32)
pkt_seg, clen, skip = np.arange(n + 1, dtype=np.uint32), np.full(n, 1500, np.int32), np.zeros(n, np.int32)
cb = _lib.ChainBatchC(b.base, b.bytes, seg_off.ctypes.data, seg_len.ctypes.data, pkt_seg.ctypes.data, n, 0,
                      clen.ctypes.data, skip.ctypes.data, None, None, None, 1500, n)
tb = tx_batch(8)
one = (C.c_void_p * 1)
st1 = one(p8)
rep, trep = C.c_void_p(), C.c_void_p()
assert lib.mi_cksum_repeat_create(C.byref(b), 1, None, None, st1, 1, C.byref(rep)) == 0, err()
assert lib.mi_cksum_tx_repeat_create(C.byref(tb), 1, st1, 1, C.byref(trep)) == 0, err()
us = C.c_float()
lens = np.full(n, 1500, np.uint32)
classes = batch(n, lens=lens)
dense = batch(n, L=46, stride=64)
tight = batch(n, L=100, stride=128)
entries = {
    "verify": lambda: lib.mi_cksum_ipv4_verify(C.byref(b), p16, None, p8, None, None),
    "verify, length classes": lambda: lib.mi_cksum_ipv4_verify(C.byref(classes), p16, None, p8, None, None),
    "verify, 64-byte slots": lambda: lib.mi_cksum_ipv4_verify(C.byref(dense), p16, None, p8, None, None),
    "verify, flat run": lambda: lib.mi_cksum_ipv4_verify(C.byref(tight), p16, None, p8, None, None),
    "verify_multi": lambda: lib.mi_cksum_ipv4_verify_multi(C.byref(b), 1, None, None, st1, None, None),
    "rx_offload": lambda: lib.mi_cksum_rx_offload(C.byref(b), p32, None, None, None),
    "span": lambda: lib.mi_cksum_span_batch(C.byref(b), 0, None, p16, None),
    "chain": lambda: lib.mi_cksum_chain_batch(C.byref(cb), p16, None),
    "finalize": lambda: lib.mi_cksum_ipv4_finalize(C.byref(b), None),
    "finalize, flat run": lambda: lib.mi_cksum_ipv4_finalize(C.byref(tight), None),
    "synth": lambda: lib.mi_cksum_synth_ipv4(C.byref(b), 1, None),
    "tx_copy": lambda: lib.mi_cksum_tx_copy(C.byref(tb), p8, None),
    "tx_copy_host": lambda: lib.mi_cksum_tx_copy_host(C.byref(tb), p8, 0),
    "verify_host": lambda: lib.mi_cksum_ipv4_verify_host(C.byref(b), p16, None, p8, None),
    "verify_repeat": lambda: lib.mi_cksum_ipv4_verify_repeat(C.byref(b), 1, None, None, st1, 3, 2, 0, None, None),
    "repeat_run": lambda: lib.mi_cksum_repeat_run(rep, 3, 0, None),
    "repeat_run, timed": lambda: lib.mi_cksum_repeat_run(rep, 3, 1, C.byref(us)),
    "tx repeat_run": lambda: lib.mi_cksum_repeat_run(trep, 3, 0, None),
}
for name, call in entries.items():  # once each: contexts, staging and the first-use queries are set up
    assert call() == 0, (name, err())
stub.stub_set_last(0)
'''


def test_an_earlier_error_is_not_the_launchs(so):
    """An error that some other call of the thread left behind is not reported
    by the next launch, whose kernel was enqueued, and stays there for the code
    that left it (a later failing call overwrites it: chain and TX calls ask the
    runtime for the extent of tables it does not know)."""
    stubbed.run(so, LAUNCHES + r'''
for name, call in entries.items():
    stub.stub_set_last(INVALID)
    before, errors = calls("hipLaunchKernel") + calls("hipExtLaunchKernel"), stub.stub_errors()
    assert call() == 0, (name, err())
    assert calls("hipLaunchKernel") + calls("hipExtLaunchKernel") > before, name
    assert stub.stub_last() == (INVALID if stub.stub_errors() == errors else 0), name
''')


def test_a_failed_launch_is_reported(so):
    """A launch that fails is: -EIO, with the launch named, from every entry point."""
    stubbed.run(so, LAUNCHES + r'''
for name, call in entries.items():
    fn = "hipExtLaunchKernel" if name == "repeat_run, timed" else "hipLaunchKernel"
    fail(fn, err=700)
    assert call() == EIO, name
    assert "stub error 700" in err() and "aunch" in err(), (name, err())
    assert call() == 0, (name, err())
''')


# every entry point that talks to the runtime, each on a thread of its own
# (thread contexts start empty: the first call allocates), once for every
# runtime call it makes with that call failing
SWEEP = r'''
import threading

n = 64
o16, o8, o32 = np.zeros(2 * n, np.uint16), np.zeros(n, np.uint8), np.zeros(2 * n, np.uint32)
p16, p8, p32 = o16.ctypes.data, o8.ctypes.data, o32.ctypes.data
st1 = (C.c_void_p * 1)(p8)
lens = np.full(n, 1500, np.uint32)
seg_off, seg_len = (np.arange(n) * 2176).astype(np.uint64), np.full(n, 1500, np.int32)
pkt_seg, skip = np.arange(n + 1, dtype=np.uint32), np.zeros(n, np.int32)
b, big, mixed, tb = batch(n), batch(4 * n, stride=4096), batch(n, lens=lens), tx_batch(8)
cb = _lib.ChainBatchC(b.base, b.bytes, seg_off.ctypes.data, seg_len.ctypes.data, pkt_seg.ctypes.data, n, 0,
                      seg_len.ctypes.data, skip.ctypes.data, None, None, None, 1500, n)
B = C.byref(b)
for f in ("mi__scalar_staging",):
    getattr(lib, f).restype, getattr(lib, f).argtypes = C.c_void_p, [C.c_size_t]


def created(tx=False):
    h = C.c_void_p()
    rc = (lib.mi_cksum_tx_repeat_create(C.byref(tb), 1, st1, 2, C.byref(h)) if tx else
          lib.mi_cksum_repeat_create(B, 1, None, None, st1, 2, C.byref(h)))
    assert (rc == 0) == bool(h), "a handle with an error"
    return rc, h


def whole(tx=False):  # a handle's life
    rc, h = created(tx)
    if rc == 0:
        rc = lib.mi_cksum_repeat_run(h, 3, 0, None) or lib.mi_cksum_repeat_run(h, 3, 1 | 0x200, C.byref(C.c_float()))
        lib.mi_cksum_repeat_destroy(h)
    return rc


def registered(call):
    rc = lib.mi_cksum_host_register(b.base, b.bytes)
    if rc == 0:
        rc = call()
        r2 = lib.mi_cksum_host_unregister(b.base)
        rc = rc or r2
    return rc


us8 = (C.c_float * 8)()
us = C.cast(us8, C.POINTER(C.c_float))
chunked = lambda **k: lib.mi_cksum_ipv4_verify_host(C.byref(k.get("b", b)), p16, p16 + 2 * n, p8, C.byref(C.c_uint32()))
entries = {
    "init": lambda: lib.mi_cksum_init(0),
    "set_busy_wait": lambda: lib.mi_cksum_set_busy_wait(1),
    "verify": lambda: lib.mi_cksum_ipv4_verify(B, p16, None, p8, None, None),
    "verify_multi": lambda: lib.mi_cksum_ipv4_verify_multi(B, 1, None, None, st1, None, None),
    "chain": lambda: lib.mi_cksum_chain_batch(C.byref(cb), p16, None),
    "finalize": lambda: lib.mi_cksum_ipv4_finalize(B, None),
    "synth": lambda: lib.mi_cksum_synth_ipv4(B, 1, None),
    "tx_copy": lambda: lib.mi_cksum_tx_copy(C.byref(tb), p8, None),
    "tx_copy_host": lambda: lib.mi_cksum_tx_copy_host(C.byref(tb), p8, 0),
    "verify_host": chunked,
    "verify_host, lengths": lambda: chunked(b=mixed),
    "rx_offload_host": lambda: lib.mi_cksum_rx_offload_host(B, p32, p32 + 4 * n, C.byref(C.c_uint32())),
    "verify_host, registered": lambda: registered(chunked),
    "verify_repeat": lambda: lib.mi_cksum_ipv4_verify_repeat(B, 1, None, None, st1, 3, 2, 1, None, us),
    "verify_repeat, per pass": lambda: lib.mi_cksum_ipv4_verify_repeat(B, 1, None, None, st1, 3, 2, 2, us, None),
    "verify_repeat, graph": lambda: lib.mi_cksum_ipv4_verify_repeat(B, 1, None, None, st1, 3, 2, 0x101, None, us),
    "repeat handle": whole,
    "tx repeat handle": lambda: whole(True),
    "drop-in staging": lambda: 0 if lib.mi__scalar_staging(100) else -1,
}


def in_thread(f):
    out = []

    def go():
        try:
            out.append(f())
        except BaseException as e:
            out.append(e)
    t = threading.Thread(target=go)
    t.start()
    t.join()
    if isinstance(out[0], BaseException):
        raise out[0]
    return out[0]


def counts_of(call):
    def probe():
        stub.stub_reset()
        rc = call()
        return rc, dict((k, int(v)) for k, v in (ln.split() for ln in stub.stub_counts().decode().splitlines()))
    return in_thread(probe)


stub.stub_counts.restype = C.c_char_p
# HIP launches alone, and MI_CKSUM_HOST_CHUNK makes host batches several chunks
assert os.environ["MI_CKSUM_HOST_CHUNK"] == "20000"
in_thread(lambda: [f() for f in entries.values()])  # per-process first-use queries


def sweep(check):
    done = 0
    for name, call in entries.items():
        rc, counts = counts_of(call)
        assert rc == 0, (name, rc, err())
        for fn, k in counts.items():
            for nth in range(1, k + 1):
                def one():
                    stub.stub_reset()
                    fail(fn, nth, NOMEM)
                    check((name, fn, nth), call, call())
                    stub.stub_reset()
                in_thread(one)
                done += 1
    return done
'''


def test_no_failure_leaves_the_last_error(so):
    """Whatever runtime call fails, the thread's last error is clear when the
    library returns: the failure is in its return code, or was recovered from."""
    stubbed.run(so, SWEEP + r'''
def check(where, call, rc):
    assert stub.stub_last() == 0, (where, rc, stub.stub_last())


assert sweep(check) > 200
''', MI_CKSUM_HOST_CHUNK="20000")


def test_no_error_return_leaves_work_in_flight(so):
    """Whatever runtime call fails, a call that runs on the library's own streams
    returns with nothing on them: a host-memory batch (several chunks), a
    back-to-back submission, a handle's run."""
    stubbed.run(so, SWEEP + r'''
def check(where, call, rc):
    assert stub.stub_pending(1) == 0, (where, rc)


assert sweep(check) > 200
''', MI_CKSUM_HOST_CHUNK="20000")


def test_what_cannot_be_waited_for_is_not_freed(so):
    """A host batch fails and its streams cannot be synchronized: the buffers
    that its kernels may still use are neither freed nor used again, and the
    next call works with others."""
    stubbed.run(so, SWEEP + r'''
for name in ("verify_host", "verify_host, lengths", "rx_offload_host", "tx_copy_host", "verify_host, registered"):
    def one():
        call = entries[name]
        assert call() == 0, err()
        live = stub.stub_live()
        fail("hipLaunchKernel")
        stub.stub_fail_from(b"hipStreamSynchronize", 1 + (name not in ("tx_copy_host", "verify_host, registered")), INVALID)
        assert call() == EIO, name
        stub.stub_reset()
        assert stub.stub_live() == live, name
        assert call() == 0, (name, err())
        assert stub.stub_live() > live and calls("hipFree") + calls("hipHostFree") == 0, name
    in_thread(one)
''', MI_CKSUM_HOST_CHUNK="20000")


def test_an_error_inside_a_capture_ends_it(so):
    """A back-to-back submission as a graph whose recording fails leaves no
    stream capturing and no graph behind, and the next submission works."""
    stubbed.run(so, SWEEP + r'''
import time

entries = {"verify_repeat, graph": entries["verify_repeat, graph"]}
leaked = [0]  # graphs whose destruction was made to fail


def check(where, call, rc):
    assert not stub.stub_capturing(), (where, rc, err())
    t0 = time.monotonic()  # (the previous thread's context goes just after the thread)
    while stub.stub_graphs() > leaked[0] + 1 and time.monotonic() < t0 + 1.0:
        time.sleep(0.001)
    leaked[0] += where[1] == "hipGraphDestroy"
    assert stub.stub_graphs() <= leaked[0] + 1, (where, stub.stub_graphs())
    stub.stub_reset()
    assert call() == 0 and stub.stub_pending(1) == 0, (where, err())


assert sweep(check) > 20
''', MI_CKSUM_HOST_CHUNK="20000")


def test_a_call_after_a_failed_one_works(so):
    """Whatever runtime call fails while a context is set up or regrown, a
    smaller and then the same call after it work: on the library's own streams,
    in buffers that are there and large enough, nothing freed twice."""
    body = r'''
big = batch(4 * n, stride=4096)
o16, o8, o32 = np.zeros(8 * n, np.uint16), np.zeros(4 * n, np.uint8), np.zeros(8 * n, np.uint32)
p16, p8, p32 = o16.ctypes.data, o8.ctypes.data, o32.ctypes.data
blens = np.full(4 * n, 1500, np.uint32)
bmixed, btb = batch(4 * n, lens=blens), tx_batch(64)
bad = C.byref(C.c_uint32())
sized = {  # name: (a small call, a larger one)
    "verify_host": [lambda x=x: lib.mi_cksum_ipv4_verify_host(C.byref(x), p16, p16 + 8 * n, p8, bad) for x in (b, big)],
    "verify_host, lengths": [lambda x=x: lib.mi_cksum_ipv4_verify_host(C.byref(x), p16, None, p8, bad)
                             for x in (mixed, bmixed)],
    "rx_offload_host": [lambda x=x: lib.mi_cksum_rx_offload_host(C.byref(x), p32, p32 + 16 * n, bad) for x in (b, bmixed)],
    "tx_copy_host": [lambda x=x: lib.mi_cksum_tx_copy_host(C.byref(x), p8, 0) for x in (tb, btb)],
    "verify_repeat": [lambda k=k: lib.mi_cksum_ipv4_verify_repeat(B, 1, None, None, st1, 3, k, 1, None, us)
                      for k in (1, 4)],
    "verify_repeat, graph": [lambda k=k: lib.mi_cksum_ipv4_verify_repeat(B, 1, None, None, st1, 3, k, 0x101, None, us)
                             for k in (1, 4)],
}
memsets = os.environ.get("MI_CKSUM_DEAL") == "1"
for name, (small, large) in sized.items():
    for first in (None, small):  # a fresh context; one that has to grow
        def grown():
            if first:
                assert first() == 0, err()
            stub.stub_reset()
            assert large() == 0, err()
            return dict((k, int(v)) for k, v in (ln.split() for ln in stub.stub_counts().decode().splitlines()))
        for fn, k in in_thread(grown).items():
            for nth in range(1, k + 1):
                def one():
                    if first:
                        assert first() == 0, err()
                    stub.stub_reset()
                    fail(fn, nth, NOMEM)
                    before = stub.stub_pending(0)
                    rc = large()
                    stub.stub_reset()
                    for again in (small, large):
                        assert again() == 0, (name, bool(first), fn, nth, rc, err())
                    assert stub.stub_pending(0) == before, (name, fn, nth, "the default stream")
                    if memsets and name == "verify_repeat" and fn == "hipMemset" and rc:
                        assert calls("hipMemset") == 1, "the counters were never cleared"
                in_thread(one)
assert stub.stub_bad_copies() == 0 and stub.stub_bad_frees() == 0
'''
    stubbed.run(so, SWEEP + body, MI_CKSUM_HOST_CHUNK="20000")
    stubbed.run(so, SWEEP + body, MI_CKSUM_HOST_CHUNK="20000", MI_CKSUM_DEAL="1")


def test_a_result_block_without_a_device_address_is_not_kept(so):
    """The drop-ins' result block: a failed address query is asked again by the
    next call, whose kernel would otherwise store through a null address."""
    stubbed.run(so, r'''
hdr = (C.c_uint8 * 20)(*bytes.fromhex("450000730000400040110000c0a80001c0a800c7"))
lib.mi_cksum_set_dropin_mode(1)
assert lib.in_cksum_hdr(hdr) in (0x61b8, 0xb861)  # (no kernel runs here: answered by the host fold)
import threading
seen = []


def go():
    lib.in_cksum_hdr.restype = C.c_uint
    for k in range(2):
        stub.stub_reset()
        fail("hipHostGetDevicePointer", 2 if k == 0 else 99)
        lib.in_cksum_hdr(hdr)
        seen.append((calls("hipHostGetDevicePointer"), calls("hipLaunchKernel")))


t = threading.Thread(target=go)
t.start()
t.join()
# first call: staging, then the block, refused: no kernel; second: the block again, a kernel
assert seen == [(2, 0), (1, 1)], seen
''')


def test_a_refused_registration_leaves_the_staged_way(so):
    """Page-locking refused: a distinct code and a clean state, and the batch
    that follows is verified through staging."""
    stubbed.run(so, r'''
n = 64
b = batch(n)
o16, o8 = np.zeros(2 * n, np.uint16), np.zeros(n, np.uint8)
verify = lambda: lib.mi_cksum_ipv4_verify_host(C.byref(b), o16.ctypes.data, None, o8.ctypes.data, None)
for code, want in ((INVALID, -95), (NOMEM, ENOMEM), (712, -17)):  # 712: hipErrorHostMemoryAlreadyRegistered
    fail("hipHostRegister", err=code)
    assert lib.mi_cksum_host_register(b.base, b.bytes) == want, err()
    assert "hipHostRegister" in err() and stub.stub_last() == 0
    assert lib.mi__reg_table_count() == 0 and lib.mi_cksum_host_unregister(b.base) == -2
    before = calls("hipMemcpy2DAsync")
    assert verify() == 0, err()
    assert calls("hipMemcpy2DAsync") > before  # staged
assert lib.mi_cksum_host_register(b.base, b.bytes) == 0, err()
before = calls("hipMemcpy2DAsync")
assert verify() == 0 and calls("hipMemcpy2DAsync") == before  # in place
assert lib.mi_cksum_host_unregister(b.base) == 0 and stub.stub_registered() == 0
''')


def test_host_blocks(so):
    """mi_cksum_host_alloc: zero-filled pages whose ranges are registered without
    the runtime, read in place while they are and staged after; the refusals; no
    block is freed under a registered range or leaked by a failed call."""
    stubbed.run(so, r'''
EINVAL, ENOENT, EBUSY, EEXIST = -22, -2, -16, -17
p = C.c_void_p()


def alloc(n):
    p = C.c_void_p(1)
    rc = lib.mi_cksum_host_alloc(n, C.byref(p))
    return rc, p.value or 0


assert lib.mi_cksum_host_alloc(4096, None) == EINVAL
for bad in (0, 2**64 - 1, 2**64 - 4095):
    assert alloc(bad) == (EINVAL, 0), bad
live = stub.stub_live()
fail("hipHostMalloc", err=NOMEM)
assert alloc(4096) == (ENOMEM, 0)
fail("hipHostGetDevicePointer")
assert alloc(4096) == (EIO, 0) and stub.stub_live() == live and stub.stub_last() == 0
assert lib.mi_cksum_host_free(None) == 0 and lib.mi_cksum_host_free(4096) == ENOENT

n = 64
size = 142 + n * 2176 + 64
rc, a = alloc(size)
assert rc == 0 and a % 4096 == 0
assert not np.ctypeslib.as_array((C.c_uint8 * size).from_address(a)).any()
end = a + ((size + 4095) & ~4095)
b = _lib.PktBatchC(a, size, None, 2176, 142, None, 1500, n, 1500, 0)
st = np.zeros(n, np.uint8)


def staged():  # does a verify of the block go through staging?
    before = calls("hipMemcpy2DAsync")
    assert lib.mi_cksum_ipv4_verify_host(C.byref(b), None, None, st.ctypes.data, None) == 0, err()
    return calls("hipMemcpy2DAsync") > before


assert staged()  # a block is not a registered range
assert lib.mi_cksum_host_register(a, end - a + 1) == EINVAL  # one byte past the block's last page
assert lib.mi_cksum_host_register(a - 1, 4096) == EINVAL
assert lib.mi__reg_table_count() == 0 and staged()
assert lib.mi_cksum_host_register(a, size) == 0 and not staged()
assert lib.mi_cksum_host_register(a + 4096, 10) == EEXIST
assert lib.mi_cksum_host_free(a) == EBUSY and lib.mi_cksum_host_free(a + 4096) == ENOENT
assert not staged()  # still there
assert lib.mi_cksum_host_unregister(a + 1) == ENOENT and lib.mi_cksum_host_unregister(a) == 0
assert staged() and lib.mi_cksum_host_unregister(a) == ENOENT
# two ranges of one block, pages apart; the GPU address is the block's plus the offset
lib.mi__reg_table_lookup.restype, lib.mi__reg_table_lookup.argtypes = C.c_uint64, [C.c_void_p, C.c_uint64]
assert lib.mi_cksum_host_register(a, 4096) == 0 and lib.mi_cksum_host_register(a + 8192 + 32, 100) == 0
assert lib.mi__reg_table_lookup(a + 16, 64) == a + 16 and lib.mi__reg_table_lookup(a + 8192 + 64, 32) == a + 8192 + 64
assert lib.mi__reg_table_lookup(a + 4096, 16) == 0
assert lib.mi_cksum_host_unregister(a) == 0 and lib.mi_cksum_host_free(a) == EBUSY
assert lib.mi_cksum_host_unregister(a + 8192 + 32) == 0
assert calls("hipHostRegister") == calls("hipHostUnregister") == 0
live = stub.stub_live()
assert lib.mi_cksum_host_free(a) == 0 and stub.stub_live() == live - 1
assert lib.mi_cksum_host_free(a) == ENOENT and stub.stub_bad_frees() == 0
''')


def test_page_buffer_frees_its_block(so):
    """mi.page_buffer with a device: the block goes with the last array over it,
    not while a view lives or a range is registered."""
    stubbed.run(so, r'''
import gc
import types

# the package's api module over the stubbed library
pkg = types.ModuleType("libunsod_amd")
pkg.__path__ = [os.path.join(ROOT, "libunsod_amd")]
sys.modules["libunsod_amd"] = pkg
sys.modules["libunsod_amd._lib"] = _lib
_lib._lib = lib
import importlib
api = importlib.import_module("libunsod_amd.api")

live = stub.stub_live()
a = api.page_buffer(5000)
assert a.nbytes == 5000 and a.ctypes.data % 4096 == 0 and a.flags.writeable and not a.any()
assert stub.stub_live() == live + 1
v = a[100:200].reshape(10, 10)
del a
gc.collect()
v[:] = 7
assert stub.stub_live() == live + 1
del v
gc.collect()
assert stub.stub_live() == live
assert api.page_buffer(0).nbytes == 0
gc.collect()
assert stub.stub_live() == live
a = api.page_buffer(100)
api.host_register(a)
p = a.ctypes.data
del a
gc.collect()
assert stub.stub_live() == live + 1  # registered: kept
assert lib.mi_cksum_host_unregister(p) == 0 and lib.mi_cksum_host_free(p) == 0 and stub.stub_live() == live
stub.stub_fail_from(b"hipGetDevice", 1, 100)  # no usable device: pages of its own all the same
allocs = calls("hipHostMalloc")
a = api.page_buffer(5000)
assert a.nbytes == 5000 and a.ctypes.data % 4096 == 0 and a.flags.writeable and calls("hipHostMalloc") == allocs
''')
