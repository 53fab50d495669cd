"""The flags that the shipped library is built with: no packed fp32 arithmetic in any kernel, and the hand-issued weight
loads stay untouched by the compiler under these flags too."""
import os
import re
import subprocess
import sys

import pytest

from tests.conftest import ROOT


def test_no_packed_fp32_and_a_clean_ring_in_the_shipped_build(tmp_path):
    import __graft_entry__ as g
    if not os.path.exists(g.HIPCC):
        pytest.skip("no hipcc here")
    asm, act = tmp_path / "camal.s", tmp_path / "act.s"
    jobs = [subprocess.Popen([g.HIPCC, *g.HIPCC_FLAGS, "-S", "--cuda-device-only", "-o", str(out), src], stderr=subprocess.DEVNULL)
            for src, out in zip(g.SRCS, (asm, act))]
    assert [j.wait() for j in jobs] == [0, 0]
    text = asm.read_text()
    assert not re.findall(r"v_pk_(?:add|mul|fma)_f32", text + act.read_text())
    assert "v_mfma_f32_16x16x32_bf16" in text
    sys.path.insert(0, os.path.join(ROOT, "tools"))
    import check_ring
    assert check_ring.check(str(asm)) == []
    assert check_ring.check.kernels_seen > 100
