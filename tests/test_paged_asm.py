"""CPU check of the paged-cache kernels' gfx950 assembly.

No loop that holds a barrier leaves through an exec-mask exit (the lanes of a wave
could run different iterations around one barrier), the attention loops keep their
accumulators in registers, and V's transposed reads and the loads into LDS are the
instructions the design counts on.
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from tests.asm_barrier_scan import scan

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"),
                                reason="hipcc not installed")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    from altxs_amd.build import common_flags, hipcc

    d = tmp_path_factory.mktemp("asm")
    out = {}
    for src in ("paged_attn.hip", "rope.hip"):
        s = d / (src + ".s")
        r = subprocess.run([hipcc(), *common_flags(), "--cuda-device-only", "-S",
                            os.path.join(ROOT, "altxs_amd", "csrc", src), "-o", str(s)], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-2000:]
        out[src] = s.read_text()
    return out


@pytest.mark.parametrize("src", ["paged_attn.hip", "rope.hip"])
def test_no_divergent_loop_around_barriers(asm, src):
    rep = scan(asm[src])
    assert rep
    assert not {k: v for k, v in rep.items() if v}


def test_attention_keeps_its_registers(asm):
    spills = {m[0]: int(m[1]) for m in re.findall(r"\.symbol:\s+(\S*attn_\w+_kernel\S*)\.kd.*?\.vgpr_spill_count:\s+(\d+)",
                                                 asm["paged_attn.hip"], re.S)}
    assert len(spills) == 30  # (few, many) x 3 types x 2 head sizes x bias, fold x 3 x 2
    assert max(spills.values()) <= 8, {k: v for k, v in spills.items() if v > 8}


def test_chunk_loops_keep_their_scalars(asm):
    """Scalar registers spill into vector lanes, which the loops then read back every tile."""
    spills = {m[1]: int(m[0]) for m in re.findall(r"\.sgpr_spill_count:\s+(\d+)\s+\.symbol:\s+(\S*attn_many_kernel\S*)\.kd",
                                                 asm["paged_attn.hip"])}
    assert len(spills) == 12 and max(spills.values()) <= 12, spills


def test_instructions(asm):
    for kernel, wanted in (("attn_many_kernelIDF16bLi64ELb0E", ("ds_read_b64_tr_b16", "global_load_lds_dwordx4",
                                                               "v_mfma_f32_16x16x32_bf16", "s_load_dword")),
                           ("attn_few_kernelIDF16_Li128ELb1E", ("ds_read_b64_tr_b16", "global_load_lds_dwordx4",
                                                               "v_mfma_f32_16x16x32_f16")),
                           ("attn_few_kernelIfLi64ELb0E", ("v_mfma_f32_16x16x4_f32",))):
        name = re.search(r"^(\S*%s\S*):" % kernel, asm["paged_attn.hip"], re.M)[1]
        body = asm["paged_attn.hip"].split(name + ":")[1].split(".Lfunc_end")[0]
        for ins in wanted:
            assert ins in body, (kernel, ins)
        assert "v_pk_fma_f32" not in body and "v_pk_mul_f32" not in body and "v_pk_add_f32" not in body
