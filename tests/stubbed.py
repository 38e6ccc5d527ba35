"""Runs libmicksum.so over tests/hip_stub.cpp, a HIP runtime of host memory, in
a child process: what the host code does when a runtime call fails, without a
GPU.  ``run(body)`` executes Python source there with these names defined:

  lib        the library, its signatures declared
  stub       the stub runtime (fail, last, set_last, pending, ... below)
  batch      (n, L=1500, host memory) -> mi_pkt_batch of fixed slots, its buffer
  tx_batch   (n) -> mi_tx_batch of single-segment frames, its arrays kept alive
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))

PRELUDE = r'''
import ctypes as C, importlib.util, os, sys
import numpy as np

ROOT, STUB = sys.argv[1], sys.argv[2]
stub = C.CDLL(STUB, mode=C.RTLD_GLOBAL)  # ahead of the library: its symbols win
stub.stub_fail.argtypes = stub.stub_fail_from.argtypes = [C.c_char_p, C.c_int, C.c_int]
spec = importlib.util.spec_from_file_location("_lib", os.path.join(ROOT, "libunsod_amd", "_lib.py"))
_lib = importlib.util.module_from_spec(spec)
spec.loader.exec_module(_lib)
lib = C.CDLL(_lib.LIB_PATH)
for _n, (_r, _a) in _lib.SIGNATURES.items():
    if hasattr(lib, _n):
        getattr(lib, _n).restype, getattr(lib, _n).argtypes = _r, _a
INVALID, NOMEM = 1, 2  # hipErrorInvalidValue, hipErrorOutOfMemory
EIO, ENOMEM = -5, -12


def fail(name, nth=1, err=INVALID):
    stub.stub_fail(name.encode(), nth, err)


def calls(name):
    return stub.stub_calls(name.encode())


def err():
    return lib.mi_cksum_strerror().decode()


def pages(nbytes):
    import mmap
    return np.frombuffer(mmap.mmap(-1, (nbytes + 4095) & ~4095), np.uint8)


def batch(n=64, L=1500, stride=2176, lens=None, flags=0):
    buf = pages(142 + n * stride + 64)
    b = _lib.PktBatchC(buf.ctypes.data, buf.nbytes, None, stride, 142, None, L, n, L, flags)
    if lens is not None:
        b.lens = lens.ctypes.data
        b.max_len = int(lens.max())
    b._keep = (buf, lens)
    return b


def tx_batch(n=8, L=200, room=2048):
    src, dst = pages(n * 256), pages(n * 2176)
    a = dict(seg_off=(np.arange(n) * 256).astype(np.uint64), seg_len=np.full(n, L, np.int32),
             pkt_seg=np.arange(n + 1, dtype=np.uint32), pkt_len=np.full(n, L, np.uint32))
    b = _lib.TxBatchC()
    b.src, b.src_bytes, b.dst, b.dst_bytes = src.ctypes.data, src.nbytes, dst.ctypes.data, dst.nbytes
    for k, v in a.items():
        setattr(b, k, v.ctypes.data)
    b.dst_stride, b.dst_first, b.room, b.l3_off, b.n, b.max_len = 2176, 0, room, 14, n, L
    b._keep = (src, dst, a)
    return b
'''


def build(outdir) -> str:
    so = os.path.join(str(outdir), "libhipstub.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wall", "-Wno-unused-function",
                    "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", os.path.join(HERE, "hip_stub.cpp"), "-o", so],
                   check=True)
    return so


def run(so: str, body: str, **env) -> None:
    p = subprocess.run([sys.executable, "-c", PRELUDE + body, os.path.dirname(HERE), so], capture_output=True,
                       text=True, timeout=120, env=dict(os.environ, MI_CKSUM_HOST_AQL="0", **env))
    assert p.returncode == 0, p.stdout + p.stderr
