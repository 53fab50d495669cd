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
    out = [tmp_path / f"{i}.s" for i in range(len(g.SRCS))]
    jobs = [subprocess.Popen([g.HIPCC, *g.HIPCC_FLAGS, "-S", "--cuda-device-only", "-o", str(o), src], stderr=subprocess.DEVNULL)
            for src, o in zip(g.SRCS, out)]
    assert [j.wait() for j in jobs] == [0] * len(jobs)
    asm = out[0]
    text = asm.read_text()
    assert not re.findall(r"v_pk_(?:add|mul|fma)_f32", "".join(o.read_text() for o in out))
    assert "v_mfma_f32_16x16x32_bf16" in text
    sys.path.insert(0, os.path.join(ROOT, "tools"))
    import check_ring
    assert check_ring.check(str(asm)) == []
    assert check_ring.check.kernels_seen > 100
