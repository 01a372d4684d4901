"""The runtime's host side without a GPU: a child process in which a stand-in for HIP (host_models/recording_hip.cpp) takes the library's calls, launches
nothing and keeps a record of allocations and launches.  Pointers that the runtime is given there are no memory."""
import functools
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

PRELUDE = """
import ctypes
hip = ctypes.CDLL(%r, mode=ctypes.RTLD_GLOBAL)
hip.recording_memory.argtypes = [ctypes.c_uint64]
hip.recording_held.restype = hip.recording_allocations.restype = ctypes.c_uint64
hip.recording_launches.restype = hip.recording_kernels.restype = ctypes.c_char_p
from tiramisu_amd import runtime
w = runtime.wrappers()
def launches():
    "(kernel, workgroups, threads) of every launch since the last call"
    return [(k, int(b), int(t)) for k, b, t in (line.rsplit(" ", 2) for line in hip.recording_launches().decode().splitlines())]
"""


@functools.lru_cache(maxsize=None)
def _stand_in():
    folder = tempfile.TemporaryDirectory()
    so = os.path.join(folder.name, "librecording_hip.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wno-return-type-c-linkage", "-o", so, os.path.join(HERE, "host_models", "recording_hip.cpp")], check=True)
    return so, folder


def run(code):
    """What `code` prints in such a process (``w``: the runtime's library, ``hip``: the stand-in), and the finished process itself."""
    r = subprocess.run([sys.executable, "-c", PRELUDE % _stand_in()[0] + code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    return r.stdout, r


def printed(code):
    out, r = run(code)
    assert r.returncode == 0, r.stdout + r.stderr
    return out
