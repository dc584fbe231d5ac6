"""The products' kernels as the compiler writes them. Their matrix instructions are inline asm, so the compiler neither
knows that their results may not be read at once nor that the accumulators should stay where they are: what it made of
that is looked at here, without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

from spanqr_amd import _lib

SOURCE = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc", "loss.hip")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """name -> its instructions, of every instance of the products' kernel"""
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    out = str(tmp_path_factory.mktemp("listing") / "loss.s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-S", "--cuda-device-only", "-o", out, SOURCE], check=True, capture_output=True)
    text = open(out).read()
    found = {}
    for m in re.finditer(r"^(_ZN\w*k_product\w*):", text, re.M):
        body = text[m.end():text.index(".Lfunc_end", m.end())]
        lines = [line.split(";")[0].strip() for line in body.split("\n")]
        found[m.group(1)] = [line for line in lines if line and not line.startswith(".cfi")]
    assert len(found) == 18   # three products, three tiles, two types
    return found


def test_the_last_result_is_waited_for(kernels):
    for name, code in kernels.items():
        last = max(k for k, line in enumerate(code) if line.startswith("v_mfma"))
        assert code[last + 1:last + 3] == ["s_nop 15", "s_nop 3"], name


def test_accumulators_stay_in_the_loop(kernels):
    for name, code in kernels.items():
        at = [k for k, line in enumerate(code) if line.startswith("v_mfma")]
        loop = code[at[0]:at[-1]]
        assert not [line for line in loop if "accvgpr" in line or line.startswith("scratch")], name
        if "ELi256E" in name:   # its results are in accumulation registers, the others' in ordinary ones
            assert all(" a[" in code[k] for k in at), name
        # what a matrix instruction writes is touched by matrix instructions alone
        written = {code[k].split()[1].rstrip(",") for k in at}
        sums = {f"{r[0]}{i}" for r in written for i in range(*[int(x) + d for x, d in zip(r[2:-1].split(":"), (0, 1))])}
        for line in loop:
            if not line.startswith("v_mfma") and line.startswith(("v_", "ds_read")):
                assert line.split()[1].rstrip(",") not in sums, (name, line)
