"""Compiler resource report of the rotary, scored attention and decoding kernels
with the flags of the library's build (CPU only): no scratch memory but for the exceptions
below, and the waves per SIMD that their tilings assume."""
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

import test_kernel_resources as build

# Backward at D = 128, at the register limit: up to 36 bytes, two 16-byte reloads per step
# with a cap or a bias (faster all the same than the kernels that held document ids as a
# run-time case and had none: 632 against 665 us with a cap at B2 H16/4 S4096).
ALLOWED_SCRATCH = re.compile(r"sattn_bwd_kernel<mi::(BF16|F16), 128, (true, \w+|false, true), false>|"
                             r"sattn_bwd_kernel<mi::F32, 128, \w+, false, true>")
SOURCES = ("rotary.hip", "sattn_fwd.hip", "sattn_bwd.hip", "decode.hip")


@pytest.fixture(scope="module")
def reports(tmp_path_factory):
    demangle = shutil.which("llvm-cxxfilt") or shutil.which("c++filt")
    if not shutil.which(build.HIPCC) or demangle is None:
        pytest.skip("hipcc or a C++ demangler is not available")
    tmp = str(tmp_path_factory.mktemp("resources"))
    with ThreadPoolExecutor(len(SOURCES)) as ex:
        res = dict(zip(SOURCES, ex.map(lambda s: build._report(s, tmp), SOURCES)))
    names = [n for r in res.values() for n in r]
    pretty = subprocess.run([demangle], input="\n".join(names), capture_output=True, text=True).stdout
    mapping = dict(zip(names, pretty.splitlines()))
    return {src: {mapping[n]: v for n, v in r.items()} for src, r in res.items()}


def test_no_scratch(reports):
    for src, kernels in reports.items():
        assert kernels, src
        bad = {n: r["ScratchSize"] for n, r in kernels.items()
               if r["ScratchSize"] > (36 if ALLOWED_SCRATCH.search(n) else 0)}
        assert not bad, bad


def test_occupancy(reports):
    def least(src, pattern):
        found = [r["Occupancy"] for n, r in reports[src].items() if re.search(pattern, n)]
        assert found, pattern
        return min(found)

    assert least("rotary.hip", r"rotary_vec_kernel<\d, \d+, 0,") == 8
    assert least("rotary.hip", r"rotary_grad_vec_kernel") >= 3
    assert least("sattn_fwd.hip", r"sattn_fwd_kernel<mi::(BF16|F16)") >= 2
    assert least("sattn_bwd.hip", r"sattn_bwd_kernel<mi::(BF16|F16)") >= 2
