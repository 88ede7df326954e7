"""The log-probability and gradient-list kernels keep their registers: compiled with the
library's own flags none of them uses scratch memory."""
import os
import re
import shutil
import subprocess

import pytest

from bindcraft2_amd import build


@pytest.mark.skipif(not shutil.which(build.HIPCC), reason="no hipcc")
@pytest.mark.parametrize("src", ["logprobs.hip", "optim.hip"])
def test_no_scratch(tmp_path, src):
    asm = tmp_path / "device.s"
    subprocess.run([build.HIPCC, "-x", "hip", *build.FLAGS, *build.EXTRA.get(src, []), "-w", "-S",
                    "--cuda-device-only", "-I", build.CSRC, os.path.join(build.CSRC, src), "-o", str(asm)],
                   check=True)
    use = dict(re.findall(r"^\s+\.name:\s+(\S+)\s+\.private_segment_fixed_size: (\d+)", asm.read_text(), re.M))
    assert use and not any(map(int, use.values())), {k: v for k, v in use.items() if int(v)}
