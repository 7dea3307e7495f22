"""Wait states in the built library's own code, read from its disassembly.

The loads from global memory to LDS are inline assembly, in front of which the
compiler keeps none of the wait states that the hardware asks of software: one
between a scalar write of m0 and the load, five between a vector instruction's
write of a scalar register and a load that reads it (a descriptor or base that
v_readlane brings back from a spill, or v_readfirstlane has just made).  So each
such load has them directly in front of it, where no path round them leads: s_nop
n waits n + 1 states."""
import os
import re
import shutil
import subprocess

import pytest

import minirun_hip as M

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """The instructions of each kernel of the library, in order."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    M.load()
    d = tmp_path_factory.mktemp("code")
    shutil.copy(M.LIB_PATH, d)
    run = lambda *a: subprocess.run([OBJDUMP, *a], cwd=d, capture_output=True, text=True, check=True).stdout
    run("--offloading", os.path.basename(M.LIB_PATH))
    found = {}
    for f in sorted(os.listdir(d)):
        if "gfx950" not in f:
            continue
        code = None
        for line in run("-d", "--no-show-raw-insn", f).splitlines():
            start = re.match(r"[0-9a-f]+ <(\S+)>:", line)
            if start:
                code = found.setdefault((f, start.group(1)), [])
            elif code is not None and line.startswith("\t"):
                code.append(line.split("//")[0].strip())
    return found


def is_dma(op):
    return re.match(r"global_load_lds_|(buffer_load_\S+ .*\blds\b)", op) is not None


def test_loads_to_lds_are_found(kernels):
    names = {name for (_, name), code in kernels.items() if any(map(is_dma, code))}
    for part in ("mla_decode", "skinny", "affine_gemm", "mxfp4_few", "mxfp4_mid", "mxfp4_gemm"):
        assert any(part in n for n in names), part


def test_every_load_to_lds_brings_its_wait_states(kernels):
    bad = {}
    for (_, name), code in kernels.items():
        for before, op in zip([""] + code, code):
            if not is_dma(op):
                continue
            need = 5 if re.search(r"\bs(\d+|\[)", op.split(None, 1)[1]) else 1
            nop = re.match(r"s_nop (\d+)$", before)
            if (int(nop.group(1)) + 1 if nop else 0) < need:
                bad.setdefault(name, []).append(f"{before} | {op}")
    assert not bad, f"{len(bad)} kernels, e.g. " + "; ".join(f"{k}: {v[0]} ({len(v)})" for k, v in list(bad.items())[:4])
