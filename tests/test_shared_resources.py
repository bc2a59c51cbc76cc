"""Register budget of the kernels of a shared prefix and of the head norms with rotation (CPU: compiles the device code
only): no instantiation spills, and the prefix's kernels keep the waves per SIMD that their rounds of workgroups count on."""
import os
import re
import subprocess

import pytest

from test_kernel_resources import CSRC, HIPCC


def compiled(name, out):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    cmd = [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-Xclang",
           "-target-feature", "-Xclang", "-packed-fp32-ops", "-mllvm", "-amdgpu-mfma-vgpr-form=1",
           "--cuda-device-only", "-c", "-o", str(out), "-Rpass-analysis=kernel-resource-usage", os.path.join(CSRC, name)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    kernels, at = {}, None
    for line in r.stderr.splitlines():
        m = re.search(r"remark: Function Name: (\S+)", line)
        if m:
            at = kernels.setdefault(m.group(1), {})
            continue
        m = re.search(r"remark:\s+(VGPRs|ScratchSize \[bytes/lane\]|Occupancy \[waves/SIMD\]): (\d+)", line)
        if m and at is not None:
            at[m.group(1).split(" ")[0]] = int(m.group(2))
    return kernels


@pytest.mark.parametrize("source,kernel,count,waves", [
    ("tt_shared.hip", "attn_shared_kernel", 14, 2),  # head dims 64, 96, 128 with 4 or 8 waves and 256, FP32 and FP16 metadata
    ("tt_shared.hip", "attn_shared_few_kernel", 6, 1),  # head dims 64, 96, 128, FP32 and FP16 metadata
    ("tt_rope.hip", "qk_norm_rope_kernel", 13, 4),   # nine pairs of types, four of 16 bits with four heads too
])
def test_no_spills(tmp_path, source, kernel, count, waves):
    found = {k: v for k, v in compiled(source, tmp_path / "x.o").items() if kernel in k}
    assert len(found) == count, sorted(found)
    for k, v in found.items():
        assert v["ScratchSize"] == 0, (k, v)
        assert v["Occupancy"] >= waves, (k, v)
