"""What the compiler made of the language-model kernels' accesses past the
caches: it merges branches that differ in that alone, and drops it, and no
result shows it.  Needs no GPU."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not on PATH")


def wide_accesses(source):
    """kernel -> [(load or store, past the caches?)] of its 16-byte accesses"""
    cmd = ["hipcc", "-O3", "-std=c++17", "--offload-arch=gfx950", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "neon_amd", "csrc"), "-S",
           os.path.join(ROOT, "neon_amd", "csrc", source + ".hip"), "-o", "-", "--offload-device-only"]
    out = subprocess.run(cmd, capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-2000:]
    kernels, at = {}, None
    for line in out.stdout.splitlines():
        label = re.match(r"(_Z\w+):", line)
        if label:
            at = kernels.setdefault(label.group(1), [])
        access = re.search(r"global_(load|store)_dwordx4.*", line)
        if access and at is not None:
            at.append((access.group(1), re.search(r"\bnt\b", access.group(0)) is not None))
    return kernels


def test_distillation_of_large_rows_goes_past_the_caches():
    kernels = wide_accesses("distill")
    for name, stores in (("distill_rows_lse_kernel", False), ("distill_rows_bprop_kernel", True)):
        for past in (False, True):
            found = [a for k, a in kernels.items() if name in k and "Lb%dE" % past in k]
            assert len(found) == 3                                        # storage types
            for accesses in found:
                # (the loop behind the whole batches reads through the caches in any case)
                assert (past and ("load", True) in accesses) or (not past and ("load", True) not in accesses)
                if stores:
                    assert {a for a in accesses if a[0] == "store"} == {("store", past)}
    for k, accesses in kernels.items():
        if "_cols_" in k:
            assert not [a for a in accesses if a[1]]


def test_layer_norm_of_large_rows_stores_past_the_caches():
    kernels = wide_accesses("layernorm")
    found = [a for k, a in kernels.items() if "ln_rows_fprop_kernel" in k or "ln_rows_bprop_kernel" in k]
    assert len(found) == 36                                                  # threads and vectors per row, types
    for accesses in found:
        assert ("store", True) in accesses and ("store", False) in accesses and ("load", True) not in accesses
