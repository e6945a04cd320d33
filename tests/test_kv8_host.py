"""Argument checks, error paths and launch order of the 8-bit K/V cache's C entries, without a GPU: thk_kv8.cpp on host stand-ins."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, HIP, OOM, STATE = -1, -2, -3, -4


@pytest.fixture(scope="module")
def lib(tmp_path_factory, thk):
    out = str(tmp_path_factory.mktemp("kv8") / "libkv8host.so")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-w", "-D__HIP_PLATFORM_AMD__", f"-I{rocm}/include", os.path.join(ROOT, "tests", "kv8_host_stub.cpp"),
                           os.path.join(ROOT, "token-hawk_amd", "csrc", "thk_kv8.cpp"), "-o", out])
    so = C.CDLL(out)
    for name, (res, args) in thk._capi.SIGNATURES.items():
        if name.startswith("thk_kv8"):
            getattr(so, name).restype, getattr(so, name).argtypes = res, args
    so.stub_ctx.restype = C.c_void_p
    so.stub_error.restype = so.stub_log.restype = C.c_char_p
    so.stub_error.argtypes = [C.c_void_p]
    return so


class Env:
    def __init__(self, lib, device=0):
        self.lib = lib
        lib.stub_set(0, 0, 0, 0)
        self.ctx = lib.stub_ctx(device)

    def create(self, *args):
        h = C.c_void_p()
        rc = self.lib.thk_kv8_create(self.ctx, *args, C.byref(h))
        assert (rc == 0) == bool(h.value)
        self.rc = rc
        return h

    @property
    def err(self):
        return self.lib.stub_error(self.ctx).decode()


@pytest.fixture
def env(lib):
    e = Env(lib)
    lib.stub_log()
    return e


P = 0x1000      # an address, 16-byte aligned; the stand-ins never touch it


def test_null_handles(thk):
    """The product library itself, no device needed."""
    lib = thk._capi.load()
    h = C.c_void_p()
    assert lib.thk_kv8_create(None, 16, 4, 4, 64, C.byref(h)) == INVALID
    assert lib.thk_kv8_destroy(None) == 0 and lib.thk_kv8_bytes(None) == 0 and lib.thk_kv8_n_ctx(None) == 0
    assert lib.thk_kv8_append(None, P, P, 0, 1) == lib.thk_kv8_read(None, 0, 1, P, P) == INVALID
    assert lib.thk_kv8_attn_decode(None, P, 1, None, None, P) == lib.thk_kv8_attn_prefill(None, P, 0, 1, None, None, P) == INVALID
    assert lib.thk_kv8_evict(None, 1, 1, 0, 0, P, None, None, P) == INVALID


@pytest.mark.parametrize("args,text", [((0, 4, 4, 64), "n_ctx"), ((-5, 4, 4, 64), "n_ctx"), (((1 << 26) + 1, 4, 4, 64), "n_ctx"), ((1 << 62, 4, 4, 64), "n_ctx"), ((16, 0, 4, 64), "heads"),
                                       ((16, 4, 0, 64), "heads"), ((16, 4, 3, 64), "heads"), ((16, 2, 4, 64), "heads"), ((16, 1025, 1025, 64), "heads"), ((16, 4, -4, 64), "heads"),
                                       ((16, 4, 4, 96), "head dim"), ((16, 4, 4, 512), "head dim")])
def test_create_refuses(env, args, text):
    env.create(*args)
    assert env.rc == INVALID and text in env.err and env.lib.stub_log() == b""


def test_create_failures(env, lib):
    lib.stub_set(0, 0, 1, 0)
    env.create(16, 4, 4, 64)
    assert env.rc == OOM and "hipMalloc" in env.err
    lib.stub_set(0, 1, 0, 0)
    env.create(16, 4, 4, 64)
    assert env.rc == STATE and "captured" in env.err
    assert lib.thk_kv8_create(env.ctx, 16, 4, 4, 64, None) == INVALID


def test_size_of_a_cache(env, lib):
    """A quarter of the f32 cache, and little beside it."""
    h = env.create(16384, 32, 32, 128)
    codes = 2 * 32 * 16384 * 128
    assert codes < lib.thk_kv8_bytes(h) < codes * 1.07 and lib.thk_kv8_n_ctx(h) == 16384
    assert lib.thk_kv8_destroy(h) == 0


@pytest.mark.parametrize("n_ctx", [100])
def test_refusals(env, lib, n_ctx):
    kv, to, wide = env.create(n_ctx, 8, 4, 64), env.create(50, 8, 4, 64), env.create(n_ctx, 8, 8, 64)
    other = Env(lib)
    far = other.create(n_ctx, 8, 4, 64)
    lib.stub_log()
    big = 1 << 62
    for rc, text in [(lambda: lib.thk_kv8_append(kv, None, P, 0, 1), "bad arguments"), (lambda: lib.thk_kv8_append(kv, P, None, 0, 1), "bad arguments"),
                     (lambda: lib.thk_kv8_append(kv, P, P, -1, 1), "bad arguments"), (lambda: lib.thk_kv8_append(kv, P, P, 0, 0), "bad arguments"),
                     (lambda: lib.thk_kv8_append(kv, P, P, 100, 1), "outside"), (lambda: lib.thk_kv8_append(kv, P, P, 1, big), "outside"), (lambda: lib.thk_kv8_append(kv, P, P, big, big), "outside"),
                     (lambda: lib.thk_kv8_append(kv, P + 4, P, 0, 1), "aligned"), (lambda: lib.thk_kv8_append(kv, P, P + 8, 0, 1), "aligned"),
                     (lambda: lib.thk_kv8_read(kv, 0, 1, None, None), "bad arguments"), (lambda: lib.thk_kv8_read(kv, 99, 2, P, P), "outside"), (lambda: lib.thk_kv8_read(kv, 0, 1, P + 4, P), "aligned"),
                     (lambda: lib.thk_kv8_attn_decode(kv, P, 0, None, None, P), "outside"), (lambda: lib.thk_kv8_attn_decode(kv, P, 101, None, None, P), "outside"),
                     (lambda: lib.thk_kv8_attn_decode(kv, None, 1, None, None, P), "null"), (lambda: lib.thk_kv8_attn_decode(kv, P, 1, None, None, None), "null"),
                     (lambda: lib.thk_kv8_attn_decode(kv, P, 1, P, None, P), "go together"), (lambda: lib.thk_kv8_attn_decode(kv, P, 1, None, P, P), "go together"),
                     (lambda: lib.thk_kv8_attn_decode(kv, P + 4, 1, None, None, P), "aligned"), (lambda: lib.thk_kv8_attn_decode(kv, P, 1, P, P + 4, P), "aligned"),
                     (lambda: lib.thk_kv8_attn_prefill(kv, P, -1, 1, None, None, P), "outside"), (lambda: lib.thk_kv8_attn_prefill(kv, P, 0, 0, None, None, P), "outside"),
                     (lambda: lib.thk_kv8_attn_prefill(kv, P, 50, 51, None, None, P), "outside"), (lambda: lib.thk_kv8_attn_prefill(kv, P, big, big, None, None, P), "outside"),
                     (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, P, kv, None, P), "same cache"), (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, P, wide, None, P), "differ"),
                     (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, P, far, None, P), "different contexts"), (lambda: lib.thk_kv8_evict(kv, 101, 20, 0, 0, P, to, None, P), "T=101"),
                     (lambda: lib.thk_kv8_evict(kv, 0, 0, 0, 0, P, to, None, P), "T=0"), (lambda: lib.thk_kv8_evict(kv, 100, 51, 0, 0, P, to, None, P), "n_keep=51"),
                     (lambda: lib.thk_kv8_evict(kv, 30, 31, 0, 0, P, to, None, P), "n_keep=31"), (lambda: lib.thk_kv8_evict(kv, 100, 20, 10, 11, P, to, None, P), "exceed"),
                     (lambda: lib.thk_kv8_evict(kv, 100, 20, -1, 0, P, to, None, P), "exceed"), (lambda: lib.thk_kv8_evict(kv, 100, 20, big, big, P, to, None, P), "exceed"),
                     (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, None, to, None, P), "null"), (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, P, to, None, None), "null"),
                     (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, P, to, P, P), "mass_out"), (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, P, to, None, P + 1584), "overlap"),
                     (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, P, to, P + 640, 3 * P), "overlap"), (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, P, to, 3 * P, 3 * P + 16), "overlap"),
                     (lambda: lib.thk_kv8_read(kv, 0, 9, P, P + 9 * 1024 - 16), "overlap"), (lambda: lib.thk_kv8_attn_decode(kv, P, 5, None, None, P), "q and out"),
                     (lambda: lib.thk_kv8_attn_prefill(kv, P, 0, 2, None, None, P + 2 * 2048 - 16), "q and out"), (lambda: lib.thk_kv8_attn_decode(kv, P, 5, 8 * P, 8 * P + 16, 4 * P), "not the same"),
                     (lambda: lib.thk_kv8_attn_decode(kv, P, 5, 8 * P, 8 * P, 8 * P + 1200), "weights overlap"), (lambda: lib.thk_kv8_attn_decode(kv, P, 5, 8 * P, P + 16, 4 * P), "weights overlap"),
                     (lambda: lib.thk_kv8_evict(kv, 100, 20, 0, 0, P + 4, to, None, P), "aligned")]:
        assert rc() == INVALID and text in env.err, (text, env.err)
    assert lib.stub_log() == b""                       # nothing was launched
    assert lib.thk_kv8_evict(kv, 100, 20, 0, 0, P, None, None, P) == INVALID
    for h in (kv, to, wide, far):
        assert lib.thk_kv8_destroy(h) == 0


def test_launches_run_on_the_contexts_device_and_errors_come_back(lib):
    env = Env(lib, device=3)
    lib.stub_set(1, 0, 0, 0)
    kv, to = env.create(5000, 8, 4, 64), env.create(50, 8, 4, 64)
    lib.stub_log()
    assert lib.thk_kv8_append(kv, P, P, 7, 20) == 0 and lib.thk_kv8_evict(kv, 100, 20, 4, 5, 64 * P, to, 2 * P, P) == 0
    assert lib.stub_log() == b"3:append 7 20;3:select 4 100 20 4 5 5000 50;3:move 20;" and lib.stub_device() == 1
    lib.stub_set(1, 1, 0, 0)                           # inside a capture: the calls themselves are allowed, freeing the cache is not
    assert lib.thk_kv8_append(kv, P, P, 0, 1) == 0 and lib.thk_kv8_destroy(kv) == STATE and "captured" in env.err
    lib.stub_set(1, 0, 0, 1)
    for call in (lambda: lib.thk_kv8_append(kv, P, P, 0, 1), lambda: lib.thk_kv8_read(kv, 0, 1, P, None), lambda: lib.thk_kv8_attn_decode(kv, P, 1, None, None, 4 * P),
                 lambda: lib.thk_kv8_attn_prefill(kv, P, 0, 2, 64 * P, 64 * P, 4 * P), lambda: lib.thk_kv8_evict(kv, 100, 20, 4, 5, 64 * P, to, None, P)):
        assert call() == HIP and lib.stub_device() == 1
    lib.stub_set(1, 0, 0, 0)
    assert lib.thk_kv8_destroy(kv) == 0 and lib.thk_kv8_destroy(to) == 0 and lib.stub_device() == 1


@pytest.mark.parametrize("shape", [(1, 1, 1, 64), (64, 8, 8, 64), (512, 32, 32, 128), (512, 32, 8, 128), (2048, 40, 40, 128), (4096, 32, 8, 128), (16384, 32, 32, 128), (131072, 64, 8, 256)])
def test_size_is_that_of_its_calls(env, lib, shape):
    """Codes, scales, the open blocks' rows, and a workspace for no more rows and parts than calls on a cache of this length can have."""
    n_ctx, H, Hkv, D = shape
    h = env.create(*shape)
    n = -(-n_ctx // 128) * 128
    cache = 2 * Hkv * n * D + 2 * Hkv * n // 16 * 4 + 2 * Hkv * 16 * D * 4
    cut = -(-n_ctx // 64) > (4 if D == 256 else 8)                     # more than a tile of 64 for every wave of a workgroup: parts
    rows = 8192 if n_ctx > 32768 else 4096 if cut else 0
    work = min(n_ctx, 2048) * H * 8 + rows * (D * 4 + 8) + 512 * 4 + (H * n * 4 if H // Hkv <= 16 else 0)
    assert cache + work <= lib.thk_kv8_bytes(h) <= cache + work + 6 * 256
    assert lib.thk_kv8_destroy(h) == 0


@pytest.mark.parametrize("shape,percent", [((512, 32, 32, 128), 30), ((512, 32, 8, 128), 34), ((2048, 40, 40, 128), 30), ((16384, 32, 32, 128), 27)])
def test_size_against_the_f32_cache(env, lib, shape, percent):
    """By the sum above: 29.4, 32.9, 29.5 and 26.0 % of the f32 cache."""
    n_ctx, _, Hkv, D = shape
    h = env.create(*shape)
    assert lib.thk_kv8_bytes(h) * 100 < percent * 2 * 4 * n_ctx * Hkv * D
    assert lib.thk_kv8_destroy(h) == 0


@pytest.mark.parametrize("D", [64, 128, 256])
def test_calls_fit_the_workspace(env, lib, D):
    """Every size of cache and call: the parts and row statistics of a launch lie inside the cache's memory (the stand-in launch checks it)."""
    far = 1 << 40
    for n_ctx in (1, 16, 63, 64, 65, 257, 513, 1025, 5000, 33000, 131072):
        for H, Hkv in ((1, 1), (8, 8), (32, 8), (17, 1), (40, 40), (64, 2), (256, 128), (257, 257), (600, 600), (1024, 1)):
            kv = env.create(n_ctx, H, Hkv, D)
            for M in (1, 2, 3, 16, 17, 31, 64, 100, 257, 1000, 2048, 2049):
                for T in {M, (M + n_ctx) // 2, n_ctx}:
                    if M <= T <= n_ctx:
                        for mass in (None, far):
                            assert lib.thk_kv8_attn_prefill(kv, 2 * far, T - M, M, mass, mass, 3 * far) == 0, (n_ctx, H, Hkv, M, T)
            assert lib.thk_kv8_destroy(kv) == 0
            lib.stub_log()
