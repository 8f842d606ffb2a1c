"""No kernel of the rotated append, the page summaries, the selection or the attention over selected pages spills registers
(checked on the CPU from the compiler's own metadata)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("source,some", [("rotary.hip", "rotate_kernel"), ("sparse.hip", "selected_kernel")])
def test_kernels_do_not_spill_vgprs(source, some, tmp_path):
    out = tmp_path / "kernels.s"
    subprocess.run([HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "--cuda-device-only", "-S", os.path.join(ROOT, "lia.rs_amd", "csrc", source), "-o",
                    str(out)], check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    spills = {}
    for block in out.read_text().split("  - .agpr_count:")[1:]:
        name, count = re.search(r"\.name:\s+(\S+)", block), re.search(r"\.vgpr_spill_count:\s+(\d+)", block)
        if name and count:
            spills[name.group(1)] = int(count.group(1))
    assert any(some in k for k in spills)
    assert not {k: v for k, v in spills.items() if v}
