"""Build-time audit of the 8-bit attention kernels' assembly (no GPU needed): no result of a matrix
instruction is touched before its wait states are over, on any path (hipcc has been seen to miss that
across a basic block's end), no vector-register spills, no packed-f32 arithmetic."""
import importlib.util
import os
import re
import subprocess

import pytest

import mfma_waits

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("nvllm_build", os.path.join(ROOT, "nano-vllm-rs_amd", "build.py"))
build = importlib.util.module_from_spec(spec)
spec.loader.exec_module(build)


def test_the_walk_follows_branches(tmp_path):
    """the walk itself: a read behind a fall-through, one behind a branch, and the same with enough waits"""
    text = """f:
\tv_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]
\ts_cbranch_scc1 .LBB0_2
\t%s
\tv_accvgpr_read_b32 v9, a3
.LBB0_2:
\t%s
\tv_add_f32_e32 v1, v1, v2
\tv_accvgpr_read_b32 v9, a0
\ts_endpgm
.Lfunc_end0:
"""
    for a, b, n in (("s_nop 0", "s_nop 7", 1), ("s_nop 7", "s_nop 0", 1), ("s_nop 7", "s_nop 7", 0)):
        p = tmp_path / "f.s"
        p.write_text(text % (a, b))
        assert len(mfma_waits.audit(str(p))["f"]) == n


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("source", ["paged_attn_kv8.hip"])
def test_assembly(tmp_path, source):
    out = str(tmp_path / "k.s")
    flags = [f for f in build.FLAGS if f != "-fPIC"]
    r = subprocess.run([build.HIPCC] + flags + ["-x", "hip", "--cuda-device-only", "-S",
                                                os.path.join(build.CSRC, source), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    found = mfma_waits.audit(out)
    assert len(found) >= 16 and not {n: b for n, b in found.items() if b}
    text = open(out).read()
    assert set(re.findall(r"\.vgpr_spill_count:\s*(\d+)", text)) == {"0"}
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
