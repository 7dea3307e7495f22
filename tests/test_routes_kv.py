"""The rule that chooses the form of attention over a paged cache and its parts, on the
CPU: which sizes take which, that parts cover all keys, and that the GPU tests' sizes
reach every form.  tests/c_abi/kv_routes.cpp asks the library, with 256 compute units."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

import minirun_hip as M

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if shutil.which(hipcc) is None:
        pytest.skip("no hipcc")
    M.load()
    out = str(tmp_path_factory.mktemp("routes") / "libkvroutes.so")
    lib = os.path.dirname(M.LIB_PATH)
    r = subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O1", "-std=c++17", "-fPIC", "-shared",
                        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                        "-I", os.path.join(ROOT, "minirun-app_amd", "csrc"), "-I", os.path.join(ROOT, "include"),
                        os.path.join(ROOT, "tests", "c_abi", "kv_routes.cpp"), "-o", out, "-L", lib, "-lminirun_hip",
                        f"-Wl,-rpath,{lib}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    fn = C.CDLL(out).route_kv
    fn.argtypes = [C.c_long] + [C.c_int] * 6 + [C.c_long, C.c_int, C.c_void_p]

    def ask(queries, keys, kv_heads, group, dim=128, batch=1, window=0, cus=256):
        """queries: of a sequence on average, or None for one each without offsets."""
        got = (C.c_int * 4)()
        fn(batch if queries is None else batch * queries, batch, queries is not None, kv_heads, group, dim, window, keys, cus, got)
        return tuple(got)

    return ask


# queries, keys, key heads, group, further sizes; many queries?, rows of a tile, parts, keys of a part
TABLE = [
    ((None, 500, 4, 8), {}, (0, 16, 1, 512)), ((None, 4000, 4, 8), {}, (0, 16, 32, 128)),
    ((None, 131072, 8, 8), {}, (0, 16, 94, 1408)), ((None, 131072, 8, 8), dict(dim=64), (0, 16, 128, 1024)), ((None, 12000, 4, 8), dict(batch=64), (0, 16, 8, 1536)),
    ((None, 4000, 8, 8), dict(batch=64), (0, 16, 1, 4032)), ((None, 10 ** 7, 1, 8), {}, (0, 16, 1022, 9792)),
    ((3, 6000, 4, 8), dict(batch=32), (0, 32, 4, 1536)), ((3, 6000, 4, 8), dict(batch=32, dim=256), (0, 32, 3, 2048)),
    ((8, 3000, 8, 8), dict(batch=64), (0, 64, 1, 3008)), ((5, 2000, 4, 8), dict(dim=256), (1, 128, 16, 128)),
    ((9, 2000, 4, 8), {}, (1, 256, 16, 128)), ((512, 16000, 4, 8), {}, (1, 256, 4, 4032)),
    ((100, 600, 4, 8), dict(batch=16), (1, 256, 1, 640)), ((4096, 5096, 8, 8), {}, (1, 256, 1, 5120)),
    ((2048, 10 ** 6, 1, 1), {}, (1, 256, 32, 31296)), ((None, 30000, 4, 8), dict(window=400), (0, 16, 1, 448)),
    ((16, 250, 4, 8), {}, (1, 256, 1, 256)), ((16, 400, 4, 8), {}, (1, 256, 4, 128)), ((512, 512, 8, 4), {}, (1, 256, 1, 512)),
]


def test_which_sizes_take_which_form(route):
    for args, more, want in TABLE:
        assert route(*args, **more) == want, (args, more)


def test_parts_cover_the_keys(route):
    rng = random.Random(3)
    for _ in range(3000):
        log = lambda hi: int(2 ** rng.uniform(0, hi))
        q, keys, batch = rng.choice([None, log(12)]), log(30) - 1, log(9)
        kvh, group, dim, cus = log(5), log(6), 32 * rng.randint(1, 8), rng.choice([1, 64, 256, 304])
        prompt, rows, splits, chunk = route(q, keys, kvh, group, dim, batch, 0, cus)
        assert chunk % 64 == 0 and 1 <= splits <= 1024 and rows in ((128, 256) if prompt else (16, 32, 64))
        assert (splits == 1 or (splits - 1) * chunk < keys <= splits * chunk) and (dim <= 128 or rows in (16, 32, 128))


def test_gpu_tests_reach_every_form(route):
    """The sizes of tests/test_gpu_kv_attention.py: whole and in parts."""
    one = [route(None, 500, 2, 4, d)[:3] for d in (32, 64, 96, 128, 160, 256)]
    assert one == [(0, 16, 1)] * 6 and route(None, 200, 1, 130)[:3] == (1, 256, 1)
    assert route(2, 40, 2, 4)[:3] == (0, 16, 1) and route(5, 100, 2, 4)[:3] == (0, 32, 1) and route(12, 130, 2, 4)[:3] == (0, 64, 1)
    assert [route(55, 129, 2, 4, d)[:3] for d in (64, 128, 192)] == [(1, 256, 1), (1, 256, 1), (1, 128, 1)]
    for d, rows in ((64, (16, 64, 256)), (128, (16, 64, 256)), (256, (16, 128, 128))):
        got = route(None, 3008, 2, 2, d, 3), route(14, 1516, 2, 8, d, 3) if d > 128 else route(7, 1516, 2, 8, d, 3), route(58, 3008, 1, 4, d, 3)
        assert tuple(g[1] for g in got) == rows and all(g[2] > 1 for g in got)
