"""The library's host code on a stand-in for the CUDA runtime (host_runtime.c): what calls leave
behind for each other, and failed allocations.  No kernel runs, so none of this needs a GPU."""
import glob
import importlib.util
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "zonos2.cpp_b200")
P = 1 << 20   # an address that is never read


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The Python mirror on the library's objects, linked with the stand-in."""
    import ctypes as C
    subprocess.run(["make", "-C", PKG], check=True, capture_output=True)
    folder = tmp_path_factory.mktemp("host")
    obj, so = str(folder / "host_runtime.o"), str(folder / "libhost.so")
    subprocess.run(["gcc", "-c", "-fPIC", "-O1", os.path.join(HERE, "host_runtime.c"), "-o", obj], check=True)
    # -Bsymbolic: torch may have put the real runtime's names into the global scope
    subprocess.run(["g++", "-shared", "-Wl,-Bsymbolic", "-o", so, *glob.glob(os.path.join(PKG, "_build", "*.o")), obj,
                    "-ldl", "-lpthread"], check=True)
    spec = importlib.util.spec_from_file_location("zonos2cu_on_host", os.path.join(PKG, "zonos2cu.py"))
    z = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = z   # its dataclasses look their module up
    spec.loader.exec_module(z)
    z.LIB_PATH = so
    z.lib().fake_launched.restype = C.c_char_p
    return z


def _verify(z, n_cb, n_streams=2):
    import ctypes as C
    p = z.SampleParams()
    return z.lib().zonos2cu_verify_drafts(P, n_streams, 3, n_cb, 1024, 1024, C.byref(p), P, P, None, P, None, 0, None,
                                          None, -1, P, P, None, None)


def test_a_call_leaves_other_threads_shared_memory_alone(host):
    """A kernel's limit of shared memory belongs to all host threads: a call with few codebooks may
    not lower it between another thread's set-up and launch."""
    L = host.lib()
    for n_streams in (2, 2000):          # either of the kernels for up to nine codebooks
        assert _verify(host, 9, n_streams) == 0
        before = [L.fake_smem_limit(b"verify_kernel", i) for i in (0, 1)]
        assert _verify(host, 1, n_streams) == 0
        assert [L.fake_smem_limit(b"verify_kernel", i) for i in (0, 1)] == before
    assert _verify(host, 16) == 0
    before = L.fake_smem_limit(b"verify_kernel", 1)
    assert _verify(host, 10) == 0
    assert L.fake_smem_limit(b"verify_kernel", 1) == before
