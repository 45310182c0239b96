"""What the compiler gives the kernels whose speed depends on the workgroups a CU
holds: registers and scratch from its resource remarks (no device needed)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "npu880-mtk-npu-llm-runtime_amd")
HIPCC = "/opt/rocm/bin/hipcc"


def _resources(source):
    """{kernel: (waves per SIMD, scratch bytes)} with the Makefile's own flags."""
    r = subprocess.run(["make", "-s", "-C", PKG, "print-flags"], capture_output=True, text=True, timeout=60, check=True)
    out = subprocess.run([HIPCC, *r.stdout.split(), "--cuda-device-only", "-Rpass-analysis=kernel-resource-usage", "-c",
                          os.path.join(PKG, "csrc", source), "-o", os.devnull],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    got = {}
    for part in out.stderr.split("Function Name: ")[1:]:
        num = {k: int(re.search(re.escape(k) + r": (\d+)", part).group(1))
               for k in ("ScratchSize [bytes/lane]", "Occupancy [waves/SIMD]")}
        got[part.split()[0]] = (num["Occupancy [waves/SIMD]"], num["ScratchSize [bytes/lane]"])
    return got


@pytest.mark.skipif(not shutil.which(HIPCC), reason="no hipcc")
def test_rmsnorm_four_workgroups_per_cu():
    """Every width of the RMSNorm producer leaves registers for four workgroups
    of 256 threads (a wave on each SIMD) per CU, without scratch."""
    rms = {k: v for k, v in _resources("qmm_quant.hip").items() if "rmsnorm_q8k_kernel" in k}
    assert len(rms) == 5
    for name, (waves, scratch) in rms.items():
        assert waves >= 4 and scratch == 0, (name, waves, scratch)


@pytest.mark.skipif(not shutil.which(HIPCC), reason="no hipcc")
def test_attention_keeps_its_loops_out_of_scratch(tmp_path):
    """The attention's loops over tiles (inside the one over pieces or row tiles) touch no scratch: what is
    spilled, at most 32 bytes of a lane, is read between pieces. Two workgroups of four waves a CU, one
    where 128 rows of 256 values take all of its registers."""
    flags = subprocess.run(["make", "-s", "-C", PKG, "print-attn-flags"], capture_output=True, text=True, timeout=60, check=True).stdout
    asm = tmp_path / "attn.s"
    out = subprocess.run([HIPCC, *flags.split(), "--cuda-device-only", "-Rpass-analysis=kernel-resource-usage", "-S",
                          os.path.join(PKG, "csrc", "qmm_attn.hip"), "-o", str(asm)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    kernels = {}
    for part in out.stderr.split("Function Name: ")[1:]:
        waves, scratch = (int(re.search(re.escape(k) + r": (\d+)", part).group(1)) for k in ("Occupancy [waves/SIMD]", "ScratchSize [bytes/lane]"))
        kernels[part.split()[0]] = waves, scratch
    wide = re.compile(r"attn_(split_kernelILi256ELi128|tile_kernelILi256)")
    assert sum("attn_split_kernel" in k or "attn_tile_kernel" in k for k in kernels) > 20
    for name, (waves, scratch) in kernels.items():
        assert waves >= (1 if wide.search(name) else 2) and scratch <= 32, (name, waves, scratch)
    name, depth, loops = "", 0, 0
    for line in asm.read_text().splitlines():
        if re.match(r"_Z\S+:", line):
            name, depth = line.split(":")[0], 0
        elif line.startswith((".LBB", "; %bb.")):  # a block: the loops it is in follow as comments
            depth = 0
        if ";" in line:
            depth = max([depth] + [int(d) for d in re.findall(r"Depth[= ]+(\d+)", line)])
            loops = max(loops, depth)
        assert not (depth >= 2 and "scratch_" in line.split(";")[0]), (name, line)
    assert loops >= 2
