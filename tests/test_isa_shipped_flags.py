"""Audits of the assembly that the library ships: every HIP source compiled with the flags of the build (no GPU needed).

What test_k1_asm_audit and test_kv8_isa_audit look at in one source or under flags of their own is looked at here in
all of them: wait states behind matrix instructions, packed-f32 arithmetic (some of its forms return wrong values on
this part), spills, and the register and LDS-DMA rules of the two kernels that own registers by name."""
import importlib.util
import os
import re
import subprocess
import sys

import pytest

import mfma_waits

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("nvllm_build", os.path.join(ROOT, "nano-vllm-rs_amd", "build.py"))
build = importlib.util.module_from_spec(spec)
spec.loader.exec_module(build)

HIP = [s for s in build.SOURCES if s.endswith(".hip")]
#: kernels with matrix instructions in each source that has them
MATRIX = {"flash_attn_mfma.hip": 8, "paged_attn.hip": 20, "paged_attn_mid.hip": 2, "paged_attn_kv8.hip": 18}


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    """source -> (path of its assembly, what the compiler says of its kernels' resources)"""
    if not os.path.exists(build.HIPCC):
        pytest.skip("hipcc not installed")
    at = tmp_path_factory.mktemp("asm")
    flags = [f for f in build.FLAGS if f != "-fPIC"] + ["-x", "hip", "--cuda-device-only", "-S"]
    jobs = {}
    for s in HIP:
        out = str(at / (s + ".s"))
        jobs[s] = out, subprocess.Popen([build.HIPCC] + flags + ["-Rpass-analysis=kernel-resource-usage",
                                         os.path.join(build.CSRC, s), "-o", out], stderr=subprocess.PIPE, text=True)
    done = {}
    for s, (out, p) in jobs.items():
        _, said = p.communicate()
        assert p.returncode == 0, said
        done[s] = out, said
    return done


@pytest.mark.parametrize("source", HIP)
def test_no_packed_f32(assembly, source):
    assert not re.search(r"v_pk_(add|mul|fma)_f32", open(assembly[source][0]).read())


@pytest.mark.parametrize("source", HIP)
def test_matrix_results_are_waited_for(assembly, source):
    found = mfma_waits.audit(assembly[source][0])
    assert len(found) == MATRIX.get(source, 0) and not {n: b for n, b in found.items() if b}


@pytest.mark.parametrize("source", [s for s in HIP if s != "flash_attn_mfma.hip"])
def test_no_vector_register_spills(assembly, source):
    counts = re.findall(r"\.vgpr_spill_count:\s*(\d+)", open(assembly[source][0]).read())
    assert counts and set(counts) == {"0"}


def test_flash_kernel(assembly):
    """its named accumulators, its LDS-DMA statements, its spills (none, but for the lane constants that the chained
    variants keep in scratch between items)"""
    r = subprocess.run([sys.executable, os.path.join(ROOT, "scripts", "k1_lab", "check_asm.py"),
                        assembly["flash_attn_mfma.hip"][0]], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "inside step loops: 0" in r.stdout
    spills = {l.split()[2]: int(l.split()[1]) for l in r.stdout.splitlines() if l.startswith("spills ")}
    assert len(spills) == MATRIX["flash_attn_mfma.hip"] + 1
    for name, n in spills.items():
        assert n <= (24 if re.search(r"flash_attn_mfma_kernelILb1ELb[01]ELb0ELb1", name) else 0), (name, n)


def test_mid_kernel(assembly):
    """two workgroups a CU: at most 256 registers and 80 KiB of LDS; one write of M0 in front of each request's four
    pieces, behind the s_nop that lets a descriptor settle"""
    path, said = assembly["paged_attn_mid.hip"]
    assert max(int(x) for x in re.findall(r"VGPRs: (\d+)", said)) <= 256
    assert set(re.findall(r"LDS Size \[bytes/block\]: (\d+)", said)) == {"81920"}
    assert set(re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", said)) == {"0"}
    lines = [l.strip() for l in open(path) if l.startswith("\t") and not l.strip().startswith((".", ";"))]
    dma = [i for i, l in enumerate(lines) if l.startswith("buffer_load_dwordx4") and l.endswith("lds")]
    m0 = [i for i, l in enumerate(lines) if re.search(r"\bm0\b", l)]
    assert len(dma) == 128 and len(m0) == 32
    for i in m0:
        assert lines[i].startswith("s_mov_b32 m0") and lines[i - 1].startswith("s_nop 4")
        assert lines[i + 1].startswith("s_nop 0") and [k for k in dma if i < k < i + 6] == list(range(i + 2, i + 6))
        offs = [re.search(r"offset:(\d+)", lines[k]) for k in range(i + 2, i + 6)]
        assert [int(o.group(1)) if o else 0 for o in offs] == [1024 * j for j in range(4)]
