"""The block-scaled product's kernels in assembly, compiled with the Makefile's flags: the MFMA
operand tuples are intact (tests/mfma_operands.py), what goes to scratch is known, and loads into
LDS come in the order that their waits count on."""
import os
import re
import shutil
import subprocess

import pytest

import mfma_operands
from test_mfma_operands import CSRC, FLAGS, HIPCC

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) and not shutil.which("hipcc"), reason="no hipcc")


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    out = tmp_path_factory.mktemp("mx") / "mx_gemm.s"
    run = subprocess.run([HIPCC, *FLAGS, os.path.join(CSRC, "mx_gemm.hip"), "-o", str(out)],
                         capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]
    return out.read_text()


def two_halves(origins):
    """Eight registers of 8-bit rows: two 16-byte reads from LDS, four registers each."""
    return (len(origins) == 8 and all(kind == "load" and text.startswith("ds_read_b128") for kind, text in origins) and
            len(set(origins[:4])) == 1 and len(set(origins[4:])) == 1)


def test_operands(listing):
    found = 0
    for name, lines in mfma_operands.functions(listing):
        count, bad = mfma_operands.check_function(lines)
        bad = [b for b in bad if not two_halves(b[1])]
        assert not bad, (name, bad[:3])
        found += count > 0
    assert found == 78  # 3 epilogues of 6 rows, 8 streamed and 12 tile forms


def test_a_mixed_half_is_seen():
    text = """
	ds_read_b128 v[8:11], v1
	ds_read_b128 v[12:15], v2
	ds_read_b128 v[4:7], v3
	v_mfma_scale_f32_32x32x64_f8f6f4 v[20:35], v[4:7], v[8:15], v[20:35], v40, v41 op_sel_hi:[0,0,0] cbsz:4
""".splitlines()
    count, bad = mfma_operands.check_function(text)
    assert count == 1 and all(two_halves(b[1]) for b in bad)
    for spoiled in ("\tds_read_b32 v13, v50", "\tv_mov_b32_e32 v9, v50"):
        _, bad = mfma_operands.check_function(text[:4] + [spoiled] + text[4:])
        assert not all(two_halves(b[1]) for b in bad)


def parameters(name):
    return tuple(map(int, re.findall(r"Li(\d+)E", name)))


def test_scratch(listing):
    """256 x 256 with 8-bit rows and a residual has 128 sums a lane beside residuals read ahead, and keeps 12
    registers in scratch; nothing else does."""
    spilled, name = {}, None
    for line in listing.splitlines():
        key, _, value = line.strip().partition(":")
        if key == ".name" and value.strip().startswith("_Z"):
            name = value.strip()
        elif key == ".vgpr_spill_count":
            spilled[name] = int(value)
    assert len(spilled) == 78
    over = {parameters(n): v for n, v in spilled.items() if v}
    assert set(over) <= {(8, 1, 256, 256, 4, 2, 1, 128, 3)} and sum(over.values()) <= 12


def test_scales_are_asked_for_before_rows(listing):
    """A step that ends a group loads scales that the next step reads, if that is the last of K. Its wait
    leaves out as many loads as a step has of rows: the scales have to come first."""
    ends = 0
    for name, lines in mfma_operands.functions(listing):
        if "tile_kernel" not in name:
            continue
        bits, _, bm, bn, wm, wn, parts, step, stages = parameters(name)
        if parts != 1 or stages != 3:
            continue
        rows = (bm * step * bits // 8 + bn * step // 2) // 1024 // (wm * wn)
        scales = -(-(bm + bn) // 64 // (wm * wn))
        for part in "\n".join(lines).split("s_barrier")[1:]:
            part = part.split(".Lmeet")[0].split("s_waitcnt vmcnt(0)")[0]
            # address ranges: of a block of scales, of A, of W
            ranges = re.findall(r"buffer_load_dwordx4 \S+ (s\[\d+:\d+\]).* lds", part)
            if len(ranges) <= rows:
                continue
            w = bn * step // 2 // 1024 // (wm * wn)
            assert len(ranges) == rows + scales
            assert len(set(ranges[-w:])) == 1 and ranges[-w - 1] != ranges[-1], name
            if scales == 1:  # (two blocks, of 192 x 192, may have A's registers before it has them)
                assert len(set(ranges[1:-w])) == 1 and ranges[0] != ranges[1], name
            ends += 1
    assert ends == 36 + 6
