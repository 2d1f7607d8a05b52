"""What the built library's kernels must not hold, read from their disassembly (the library is built here
from the sources; ROCm's llvm-objdump is needed)."""
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """The instructions of every kernel and device function of the library, by name."""
    from gwn_amd import _lib
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    at = tmp_path_factory.mktemp("code")
    shutil.copy(_lib.LIB_PATH, at / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=at, check=True, stdout=subprocess.DEVNULL)
    found = {}
    for f in sorted(at.glob("lib.so.*gfx950*")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", f.name], cwd=at, check=True,
                              stdout=subprocess.PIPE, text=True).stdout
        now = []
        for line in text.splitlines():
            if line.endswith(">:"):
                now = found.setdefault(line[line.index("<") + 1:-2], [])
            elif line[:1] in " \t" and line.strip():
                now.append(line.split("//")[0].strip())
    assert len(found) > 100 and any("gemm_kernel" in k for k in found)
    return found


def test_no_packed_fp32(kernels):
    """hipcc's packed fp32 instructions have given wrong values on gfx950: every source is built without."""
    bad = sorted(k for k, code in kernels.items() if any(re.match(r"v_pk_(add|mul|fma)_f32", i) for i in code))
    assert not bad


def test_tile_loads_to_lds_have_m0_to_themselves(kernels):
    """gemm_kernel's loads to LDS are assembly that sets m0 (which the compiler lets no assembly clobber): nothing
    else in these kernels names it."""
    n = 0
    for k, code in kernels.items():
        if "gemm_kernel" in k and any(i.endswith("offen lds") for i in code):
            n += 1
            for a, b, c in zip(code, code[1:], code[2:]):
                if re.search(r"\bm0\b", a):
                    assert a.startswith("s_mov_b32 m0,") and b.startswith("s_nop") and c.endswith("offen lds"), (k, a)
    assert n >= 60


def test_tile_loads_wait_for_scalar_results(kernels):
    """Five states pass in these loads' assembly, which the compiler's hazard handling does not look into, before
    they take scalar registers that a vector instruction may have written right before."""
    for k, code in kernels.items():
        if "gemm_kernel" in k:
            for a, b in zip(code, code[1:]):
                if b.endswith("offen lds"):
                    assert a.startswith("s_nop") and int(a.split()[1], 0) >= 3, (k, a)


def test_no_memsets():
    """Memory is cleared by kernels: a memset that a captured graph records has left wrong values on later replays,
    and every entry may be captured."""
    from gwn_amd import _lib
    names = subprocess.run(["nm", "-D", "--undefined-only", _lib.LIB_PATH], check=True, stdout=subprocess.PIPE,
                           text=True).stdout
    assert "hipLaunchKernel" in names and "hipMemset" not in names
