"""The kernels of rows that a group of lanes holds are those that a call can
reach: one vector a lane only forward (with alternatives) and for rows shorter
than a vector; and what takes no alternatives carries no code for them."""
import os
import re
import shutil
import subprocess

import pytest

from bindcraft2_amd import build


@pytest.mark.skipif(not shutil.which(build.HIPCC), reason="no hipcc")
def test_row_kernels(tmp_path):
    asm = tmp_path / "device.s"
    subprocess.run([build.HIPCC, "-x", "hip", *build.FLAGS, "-w", "-S", "--cuda-device-only", "-I", build.CSRC,
                    os.path.join(build.CSRC, "logprobs.hip"), "-o", str(asm)], check=True)
    kernel = re.compile(r"^\S*lp_rows_kernelI(\w+?)Li(\d+)ELi(\d+)ELi(\d+)ELi(\d+)EE\S*:\s(.*?)^; codeLenInByte",
                        re.M | re.S)
    found = {(t, *map(int, rest)): body for t, *rest, body in kernel.findall(asm.read_text())}
    types = {k[0] for k in found}
    assert len(types) == 3
    want = set()
    for t in types:
        n = 4 if t == "f" else 8
        for mode in (1, 2, 3):
            want |= {(t, 1, 8, 1, mode)} | {(t, n, w, 2, mode) for w in (4, 8, 16, 32, 64)}
        want |= {(t, n, w, 1, 1) for w in (4, 8, 16, 32, 64)}
    assert set(found) == want, set(found) ^ want
    # the largest key of a group, and the moving up of a wave's list
    chooses = re.compile(r"v_max3?_u32|wave_shr:1")
    for (t, n, w, nv, mode), body in found.items():
        assert bool(chooses.search(body)) == (mode == 1 and (nv == 1 or w == 64)), (t, n, w, nv, mode)
