"""Inline assembly in the kernels' sources. The compiler knows nothing of what it
reads: an instruction of it that takes an MFMA's result gets no wait states, and
now and then a stale value. So no vector arithmetic stands in it (no device needed)."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "npu880-mtk-npu-llm-runtime_amd", "csrc")


def _statements(text):
    """The texts of all asm statements, strings joined."""
    for m in re.finditer(r"\b(?:__)?asm(?:__)?(?:\s+volatile)?\s*\(((?:\s*\"(?:[^\"\\]|\\.)*\")*)", text):
        yield " ".join(re.findall(r'"((?:[^"\\]|\\.)*)"', m.group(1)))


def test_no_vector_arithmetic():
    found, seen = [], 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*"))):
        for body in _statements(open(path).read()):
            seen += 1
            if re.search(r"\bv_[a-z]", body):
                found.append((os.path.basename(path), body))
    assert seen >= 10, "the sources' asm statements were not found"
    assert not found, found
