"""The rules that choose a kernel for a product with MXFP4 weights, on the CPU:
which sizes take which kernel, and that the GPU tests' sizes reach all of them.
tests/c_abi/mxfp4_routes.cpp asks the library, with 256 compute units."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import minirun_hip as M
import test_gpu_mxfp4_mm as mm
import test_gpu_mxfp4_tiles as large

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256
KINDS = {"bf16": 0, "f32": 1, "mxfp4": 2}
FEW, MID, TILES = range(3)


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if shutil.which(hipcc) is None:
        pytest.skip("no hipcc")
    M.load()
    out = str(tmp_path_factory.mktemp("routes") / "libmxfp4routes.so")
    lib = os.path.dirname(M.LIB_PATH)
    r = subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O1", "-std=c++17", "-fPIC", "-shared",
                        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                        "-I", os.path.join(ROOT, "minirun-app_amd", "csrc"), "-I", os.path.join(ROOT, "include"),
                        os.path.join(ROOT, "tests", "c_abi", "mxfp4_routes.cpp"), "-o", out, "-L", lib, "-lminirun_hip",
                        f"-Wl,-rpath,{lib}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    fn = C.CDLL(out).route_mxfp4

    def ask(kind, rows, out_features, in_features, experts=0, per_token=1):
        got = (C.c_int * 5)()
        fn(KINDS[kind], rows, out_features, in_features, experts, per_token, CUS, got)
        return tuple(got)

    return ask


# kernel, weight rows and rows of x of a workgroup, waves, stages
MATRIX = {
    "bf16": [
        (1, 300, 544, (FEW, 16, 2, 2, 1)), (2, 7168, 2048, (FEW, 16, 2, 4, 1)), (1, 7168, 16384, (FEW, 16, 2, 8, 1)),
        (16, 576, 1024, (FEW, 16, 16, 4, 1)), (96, 576, 7168, (FEW, 16, 16, 8, 1)), (64, 1536, 7168, (FEW, 32, 16, 8, 1)),
        (100, 2048, 12608, (FEW, 64, 16, 8, 1)), (100, 2048, 1024, (FEW, 32, 16, 4, 1)), (100, 4096, 512, (FEW, 64, 16, 4, 1)),
        (150, 4096, 4096, (FEW, 64, 48, 4, 1)), (600, 1536, 12608, (FEW, 64, 64, 3, 1)), (16, 33000, 1536, (MID, 128, 16, 4, 2)),
        (20, 33000, 1536, (MID, 128, 32, 4, 2)), (600, 24576, 1536, (TILES, 128, 128, 4, 2)),
        (4096, 24576, 1536, (TILES, 256, 256, 4, 2)),
    ],
    "f32": [
        (1, 1536, 7168, (FEW, 64, 1, 4, 1)), (64, 2048, 2048, (FEW, 32, 16, 4, 1)), (5, 24576, 1536, (MID, 128, 16, 4, 1)),
        (37, 24576, 1536, (MID, 256, 16, 4, 1)), (4096, 4096, 4096, (MID, 256, 16, 4, 1)),
    ],
    "mxfp4": [
        (16, 4096, 4096, (FEW, 16, 16, 8, 1)), (16, 7168, 4096, (FEW, 32, 16, 8, 1)), (200, 1024, 4096, (FEW, 64, 16, 8, 1)),
        (200, 1024, 1024, (FEW, 32, 16, 4, 1)), (100, 4096, 1024, (FEW, 64, 32, 8, 1)), (600, 1024, 2048, (FEW, 64, 32, 4, 1)),
        (150, 4096, 4096, (FEW, 64, 64, 8, 1)), (600, 2048, 12608, (FEW, 64, 64, 4, 1)), (16, 24576, 1536, (MID, 64, 16, 2, 1)),
        (100, 12000, 1024, (MID, 128, 32, 4, 1)), (400, 7168, 16384, (TILES, 128, 128, 4, 2)),
        (300, 24576, 1536, (TILES, 128, 128, 4, 1)), (4096, 7168, 16384, (TILES, 256, 256, 4, 2)),
    ],
}


def test_neighbouring_sizes_take_the_same_kernel(route):
    """17 to 64 tokens of bf16 on weights of more than 16384 rows: one kernel, whatever
    the number of tokens or the row's length."""
    took = {route("bf16", t, n, k) for t in range(17, 65) for n in (16400, 20480, 24576, 33000, 65536)
            for k in (512, 1536, 2016, 2048, 2080, 4096, 7168)}
    assert took == {(MID, 128, 32, 4, 2)}


EXPERTS = {
    "bf16": [
        (8, 8, 128, 768, 2048, (FEW, 16, 2, 4, 1)), (768, 8, 128, 2048, 768, (MID, 128, 16, 4, 1)),
        (192, 8, 32, 1536, 7168, (MID, 128, 16, 4, 2)), (2432, 8, 128, 2048, 768, (MID, 128, 32, 4, 1)),
        (416, 8, 32, 264, 512, (MID, 128, 32, 4, 2)), (32768, 8, 128, 768, 2048, (TILES, 128, 128, 4, 2)),
    ],
    "f32": [
        (8, 8, 128, 768, 2048, (MID, 64, 16, 4, 1)), (24, 8, 32, 768, 2048, (MID, 128, 16, 4, 1)),
        (1536, 8, 128, 768, 2048, (MID, 256, 16, 4, 1)),
    ],
    "mxfp4": [
        (8, 8, 128, 768, 2048, (FEW, 16, 16, 4, 1)), (1152, 8, 128, 2048, 768, (MID, 64, 16, 2, 1)),
        (2048, 8, 128, 2048, 768, (MID, 64, 32, 2, 1)), (32768, 8, 128, 768, 2048, (TILES, 128, 128, 4, 1)),
        (8192, 8, 32, 1536, 7168, (TILES, 128, 128, 4, 2)),
    ],
}


@pytest.mark.parametrize("kind", KINDS)
def test_kernel_of_a_matrix_product(route, kind):
    assert [(t, n, k, route(kind, t, n, k)) for t, n, k, _ in MATRIX[kind]] == MATRIX[kind]


@pytest.mark.parametrize("kind", KINDS)
def test_kernel_of_an_expert_product(route, kind):
    got = [(r, per, e, n, k, route(kind, r, n, k, e, per)) for r, per, e, n, k, _ in EXPERTS[kind]]
    assert got == EXPERTS[kind]


@pytest.mark.parametrize("kind", KINDS)
def test_the_gpu_tests_reach_every_kernel(route, kind):
    """Every kernel and tile that a search over sizes finds is one that some whole
    numbers in test_gpu_mxfp4_mm.py or test_gpu_mxfp4_tiles.py go through."""
    def key(rows, n, k, *experts):
        # large tiles have a form of their own for rows that end in a part of a stage
        r = route(kind, rows, n, k, *experts)
        return r + (r[0] == TILES and k % (256 if kind == "mxfp4" else 128) != 0,)

    matrix = {key(t, n, k) for n, k in mm.SHAPES for t in mm.TOKENS} | {key(t, n, k) for t, n, k in mm.WIDE}
    experts = {key(t * per, n, k, e, per) for t, per, e, n, k in mm.EXPERTS + large.EXPERTS}
    rows = [1, 2, 3, 16, 17, 33, 48, 64, 65, 100, 128, 200, 300, 600, 1000, 2000, 4096]
    outs = [16, 64, 273, 576, 1024, 1536, 2048, 4096, 7168, 12000, 16385, 24576, 33000]
    ins = [32, 512, 1024, 2048, 4128, 7168, 16384]
    found = {key(t, n, k) for t in rows for n in outs for k in ins}
    assert found <= matrix, found - matrix
    found = {key(r * 8, n, k, e, 8) for r in rows for e in (1, 8, 60, 128, 256) for n in outs[2:9] for k in ins}
    assert found <= experts, found - experts
