"""The paged attention kernels' assembly, compiled with the Makefile's flags: the
MFMA operand tuples are intact (tests/mfma_operands.py), and nothing of the
kernels goes to scratch."""
import os
import shutil
import subprocess

import pytest

import mfma_operands
from test_mfma_operands import CSRC, FLAGS, HIPCC


@pytest.mark.skipif(not os.path.exists(HIPCC) and not shutil.which("hipcc"), reason="no hipcc")
@pytest.mark.parametrize("source,kernels", [("paged_decode.hip", 6), ("paged_prefill.hip", 12)])
def test_paged_kernels_keep_their_operands(tmp_path, source, kernels):
    out = tmp_path / "k.s"
    run = subprocess.run([HIPCC, *FLAGS, os.path.join(CSRC, source), "-o", str(out)],
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    text = out.read_text()
    found = 0
    for name, lines in mfma_operands.functions(text):
        count, bad = mfma_operands.check_function(lines)
        assert not bad, (name, bad[:3])
        found += count > 0
    assert found == kernels  # one or two per heads of a group
    spills = [line.split()[-1] for line in text.splitlines() if ".vgpr_spill_count:" in line]
    assert len(spills) >= kernels and set(spills) == {"0"}
