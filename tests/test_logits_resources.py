"""The kernels on logits use no scratch memory (read from the gfx950 assembly, no GPU needed): a row in registers that
spills is slower, and a register spilled where part of a wave is masked off comes back wrong in the others."""
import os
import re
import shutil
import subprocess

import pytest

from silogic_amd import _build


@pytest.mark.parametrize("name,kernels", [("select", 20), ("distill", 5)])
def test_no_scratch(name, kernels, tmp_path):
    try:
        hipcc = _build._hipcc()
    except RuntimeError as e:   # no ROCm toolchain on this host
        pytest.skip(str(e))
    if not shutil.which(hipcc) and not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    out = tmp_path / "k.s"
    subprocess.run([hipcc] + _build.FLAGS + ["--cuda-device-only", "-S", os.path.join(_build.CSRC, name + ".hip"), "-o",
                                             str(out)], check=True, capture_output=True)
    text = out.read_text()
    sizes = re.findall(r"\.private_segment_fixed_size: (\d+)", text)
    spills = re.findall(r"\.vgpr_spill_count: +(\d+)", text)
    assert len(sizes) == len(spills) >= kernels
    assert set(sizes) == set(spills) == {"0"}, (sizes, spills)
