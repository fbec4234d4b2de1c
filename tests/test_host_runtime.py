"""The library's host code on a stand-in for the CUDA runtime (host_runtime.c): what calls leave
behind for each other, and failed allocations.  No kernel runs, so none of this needs a GPU."""
import glob
import importlib.util
import os
import subprocess
import sys

import numpy as np
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


@pytest.mark.parametrize("batch", [3, 100])
@pytest.mark.parametrize("n_cb,vocab", [(65535, 1), (65536, 1), (1, 1024 * 65535), (1, 1024 * 65535 + 1)])
def test_adapters_past_a_grids_limits(host, batch, n_cb, vocab):
    """More codebooks, or parts of one, than a launch grid has rows for."""
    z = host
    assert z.lib().zonos2cu_head_adapters(P, z.BF16, vocab, n_cb, vocab, 8, P, batch, 15.0, P, P, None, 2, 8, P, P,
                                          1 << 30, P, None) == 0


S, CB, V, DIM, N, RANK = 2, 2, 1024, 2048, 3, 16


def _context(z):
    ctx = z.Context(0, S, CB, V, DIM, 0, seed=1)
    ctx.set_head(np.zeros((CB * V, DIM), np.uint16), z.BF16, V)
    return ctx


def _adapters(ctx, z):
    ctx.set_adapters(np.zeros((N, RANK, DIM), np.uint16), np.zeros((N, CB * V, RANK), np.uint16), V, z.BF16)


def _step(ctx, z):
    """A step's status and the kernels that it launches."""
    import ctypes as C
    L, p = z.lib(), z.SampleParams()
    L.fake_forget()
    codes = np.zeros((S, CB), np.int32)
    rc = L.zonos2cu_ctx_step(ctx.h, P, z.BF16, C.byref(p), -1, codes.ctypes.data, None, None, None)
    return rc, [L.fake_launched(i).decode() for i in range(L.fake_launches())]


def test_failed_adapters_leave_head_and_norm(host):
    """Whichever allocation of set_adapters fails: no adapters, and a step is the normed head's."""
    z, failures = host, 0
    gamma = np.ones(DIM, np.float32)
    for earlier in (False, True):
        for n in range(1, 20):
            ctx = _context(z)
            ctx.set_out_norm(gamma, 1e-5)
            want = _step(ctx, z)
            assert want[0] == 0 and any("rms" in k for k in want[1]), want
            if earlier:
                _adapters(ctx, z)
                assert any("adapter" in k for k in _step(ctx, z)[1])
            z.lib().fake_fail_alloc(n)
            try:
                _adapters(ctx, z)
                done = True
            except z.Zonos2cuError as e:
                done = False
                assert e.code == z.ENOMEM
            z.lib().fake_fail_alloc(0)
            if not done:
                failures += 1
                rc, kernels = _step(ctx, z)
                assert rc == 0 and any("rms" in k for k in kernels) and not any("adapter" in k for k in kernels), (n, kernels)
            ctx.close()
            if done:
                break
    assert failures >= 8   # A, B, scale, work and the folded A, twice


@pytest.mark.parametrize("adapters", [False, True])
def test_failed_norm_is_not_stepped_over(host, adapters):
    """Whichever allocation of set_out_norm fails: a step is the one before the call or refused, and
    setting the norm again, or off, mends it."""
    z, gamma, refused = host, np.ones(DIM, np.float32), 0
    for n in range(1, 20):
        ctx = _context(z)
        if adapters:
            _adapters(ctx, z)
        want = _step(ctx, z)[1]
        z.lib().fake_fail_alloc(n)
        try:
            ctx.set_out_norm(gamma, 1e-5)
            done = True
        except z.Zonos2cuError as e:
            done = False
            assert e.code == z.ENOMEM
        z.lib().fake_fail_alloc(0)
        rc, kernels = _step(ctx, z)
        if done:
            assert rc == 0 and any("rms" in k for k in kernels)
            ctx.close()
            break
        # the first step of a context draws its generators' numbers first
        assert rc == z.ESTATE and not kernels or rc == 0 and kernels == [k for k in want if "draw" not in k], (n, rc, kernels)
        if rc:
            refused += 1
            ctx.set_out_norm(enable=False)
            assert _step(ctx, z)[0] == 0
        ctx.set_out_norm(gamma, 1e-5)
        rc, kernels = _step(ctx, z)
        assert rc == 0 and any("rms" in k for k in kernels)
        ctx.close()
    assert refused == (2 if adapters else 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("earlier", [False, True])
def test_failed_head_is_not_stepped_with(host, dtype, earlier):
    """Whichever allocation of set_head fails, the logits' and the f32 norm's among them: no head."""
    import ctypes as C
    z, L = host, host.lib()
    code, t = (z.F32, np.float32) if dtype == "f32" else (z.BF16, np.uint16)
    p, codes = z.SampleParams(), np.zeros((S, CB), np.int32)
    W = np.zeros((CB * V, DIM), t)

    def step():
        return L.zonos2cu_ctx_step(ctx.h, P, code, C.byref(p), -1, codes.ctypes.data, None, None, None)

    failures = 0
    for n in range(1, 20):
        ctx = z.Context(0, S, CB, V, DIM, 0, seed=1)
        if earlier:   # a head of the other type, and the norm
            ctx.set_head(np.zeros((CB * V, DIM), np.uint16), z.BF16, V)
        ctx.set_out_norm(None, 1e-5)
        L.fake_fail_alloc(n)
        try:
            ctx.set_head(W, code, V)
            done = True
        except z.Zonos2cuError as e:
            done = False
            assert e.code == z.ENOMEM
        L.fake_fail_alloc(0)
        assert step() == (0 if done else z.ESTATE), n
        failures += not done
        ctx.set_head(W, code, V)
        assert step() == 0
        ctx.close()
        if done:
            break
    # the head; without an earlier one the logits, with it the f32 norm's rows
    assert failures == (2 if dtype == "f32" or not earlier else 1)


def test_contexts_free_what_they_allocate(host):
    z = host
    ctx = _context(z)
    _adapters(ctx, z)
    ctx.close()
    before = z.lib().fake_live_allocs()
    for n in range(1, 12):
        ctx = _context(z)
        z.lib().fake_fail_alloc(n)
        try:
            ctx.set_out_norm(np.ones(DIM, np.float32), 1e-5)
            ctx.set_cfg(1.5)
            _adapters(ctx, z)
        except z.Zonos2cuError:
            pass
        z.lib().fake_fail_alloc(0)
        ctx.close()
        assert z.lib().fake_live_allocs() == before, n
