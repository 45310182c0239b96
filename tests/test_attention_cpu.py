"""The host side of the cache append and the attention, without a device: the
tiles a row block attends to, the clamping of what the batch arrays hold, and
every refusal (tests/attn_caller.cpp); null contexts through the library."""
import os
import subprocess

import qmm_hip

HERE = os.path.dirname(os.path.abspath(__file__))


def test_tiles_clamps_and_refusals(tmp_path):
    exe = str(tmp_path / "attn_caller")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                        os.path.join(HERE, "attn_caller.cpp"), "-o", exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.stdout + r.stderr)[-2000:]


def test_null_context():
    lib = qmm_hip.load_library()
    assert lib.qmm_kv_append(None, None, None, None) == qmm_hip.QMM_EINVAL
    assert lib.qmm_paged_attention(None, None, None, None, None) == qmm_hip.QMM_EINVAL
    assert lib.qmm_attention_workspace_bytes(None, None, None, None) == 0
    assert lib.qmm_attention_workspace_create(None, 0, None) == qmm_hip.QMM_EINVAL
    assert lib.qmm_attention_workspace_destroy(None, None) == qmm_hip.QMM_EINVAL
    assert lib.qmm_rope_create(None, None, None) == qmm_hip.QMM_EINVAL
    assert lib.qmm_rope_destroy(None, None) == qmm_hip.QMM_EINVAL
