"""Every kernel is compiled without packed fp32 instructions."""
import os
import re
import shutil
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hy-video-prfl_amd")


@pytest.mark.skipif(not shutil.which("make"), reason="needs make")
def test_no_object_is_built_with_packed_fp32():
    plan = subprocess.run(["make", "-C", PKG, "-n", "-B"], check=True, capture_output=True, text=True).stdout
    lines = [x for x in plan.splitlines() if re.search(r" -c csrc/\w+\.hip", x)]
    names = {re.search(r" -c csrc/(\w+)\.hip", x).group(1) for x in lines}
    assert names == {f[:-4] for f in os.listdir(os.path.join(PKG, "csrc")) if f.endswith(".hip")}
    for x in lines:
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in x, x


def test_no_source_writes_packed_fp32_by_hand():
    for f in os.listdir(os.path.join(PKG, "csrc")):
        with open(os.path.join(PKG, "csrc", f)) as src:
            code = re.sub(r"//[^\n]*", "", src.read())
        assert not re.search(r"v_pk_(add|mul|fma)_f32", code), f
