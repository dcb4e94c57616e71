"""bench.py says whether committed hardware counters are of the kernels in this tree: same sources, same compile flags."""
import hashlib
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import bench  # noqa: E402

CSRC = os.path.join(ROOT, "vllm-v0.1.0_amd", "csrc")


def sources():
    return {n: hashlib.sha256(open(os.path.join(CSRC, n), "rb").read()).hexdigest()[:16] for n in ("pa_decode.hip", "pa_common.h")}


def test_sources_alone_do_not_make_the_kernels_the_same():
    table = {"_kernel_sources_sha16": sources()}
    assert bench.pmc_sources_unchanged(table) is None       # compiled with what flags is not recorded
    assert bench.pmc_sources_unchanged({}) is None
    table["_kernel_flags_sha16"] = "0" * 16
    assert bench.pmc_sources_unchanged(table) is False
    table["_kernel_flags_sha16"] = bench.kernel_flags_sha16()
    assert bench.pmc_sources_unchanged(table) is True
    table["_kernel_sources_sha16"]["pa_decode.hip"] = "0" * 16
    assert bench.pmc_sources_unchanged(table) is False
    del table["_kernel_flags_sha16"]
    assert bench.pmc_sources_unchanged(table) is False


def test_the_hash_goes_by_flags():
    with open(os.path.join(CSRC, "Makefile")) as f:
        text = f.read()
    now = bench.kernel_flags_sha16(text)
    assert now == bench.kernel_flags_sha16()
    assert bench.kernel_flags_sha16(text.replace("$(NO_PACKED_F32)", "")) != now
    assert bench.kernel_flags_sha16(text.replace("-packed-fp32-ops", "+packed-fp32-ops")) != now
    assert bench.kernel_flags_sha16(text.replace("-O3", "-O2")) != now
    assert bench.kernel_flags_sha16(text.replace("-Wno-unused-function", "-Wno-unused")) != now     # on a continued line
    assert bench.kernel_flags_sha16(text + "\nother: build/another.o\n\techo $(X)\n") == now
