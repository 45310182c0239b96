"""How calls of the attention are launched (tests/attn_plan_caller.cpp), without a device."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_launches(tmp_path):
    """A workspace serves calls of any length and batch as one of their own would, a small one never leaves
    fewer workgroups than none, and shared work can always be counted."""
    exe = str(tmp_path / "attn_plan_caller")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                        os.path.join(HERE, "attn_plan_caller.cpp"), "-o", exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.stdout + r.stderr)[-2000:]
