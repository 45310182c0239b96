"""The host side of the layers with a carried state and of the beam search,
without a device: rows and slots, sizes, every refusal (tests/state_caller.cpp);
null contexts through the library; the oracles against other forms of the same."""
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

import qmm_hip
import state_ref as R
from test_resources import HIPCC, PKG, _resources

HERE = os.path.dirname(os.path.abspath(__file__))


def test_clamps_sizes_and_refusals(tmp_path):
    exe = str(tmp_path / "state_caller")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                        os.path.join(HERE, "state_caller.cpp"), "-o", exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.stdout + r.stderr)[-2000:]


def test_null_context():
    lib = qmm_hip.load_library()
    assert lib.qmm_short_conv(None, None, None) == qmm_hip.QMM_EINVAL
    assert lib.qmm_gated_delta(None, None, None, None) == qmm_hip.QMM_EINVAL
    assert lib.qmm_gated_delta_workspace_bytes(None, None, None) == 0
    assert lib.qmm_beam_select(None, None, None) == qmm_hip.QMM_EINVAL
    assert lib.qmm_beam_workspace_bytes(None, None) == 0
    assert lib.qmm_copy_slots(None, None, 0, None, None, 0) == qmm_hip.QMM_EINVAL


def test_rule_by_groups_is_the_rule_by_tokens():
    """The oracle of the delta rule, token by token, against its form by groups of tokens in 64 bits."""
    b = R.States([23], seed=1)
    DK, DV, HV, C = 8, 8, 2, 5
    q, k = (b.rows(DK).reshape(-1, 1, DK) for _ in range(2))
    v, a, bt = b.rows(HV * DV).reshape(-1, HV, DV), b.rows(HV), b.rows(HV)
    rate, dt, pool = np.array([-0.5, -3], np.float32), np.zeros(HV, np.float32), b.pool(HV, DK, DV)
    out, tol, after, after_tol = R.delta(b, q, k, v, a, bt, rate, dt, 0.3, 1e-6, pool, of=HV)
    unit = [x[:, 0].astype(np.float64) / np.sqrt((x[:, 0].astype(np.float64) ** 2).sum(-1, keepdims=True) + 1e-6) for x in (q, k)]
    for h in range(HV):
        g = rate[h] * np.log1p(np.exp(a[:, h].astype(np.float64)))
        beta = 1 / (1 + np.exp(-bt[:, h].astype(np.float64)))
        S = pool[b.slot_in[0], h].astype(np.float64)
        for t in range(0, 23, C):
            r = slice(t, min(t + C, 23))
            G, kk, qq = np.cumsum(g[r]), unit[1][r], unit[0][r] * 0.3
            D = np.tril(np.exp(G[:, None] - G[None]))
            A = np.tril(beta[r, None] * (kk @ kk.T) * D, -1)
            d = np.linalg.solve(np.eye(len(G)) + A, beta[r, None] * (v[r, h] - np.exp(G)[:, None] * (kk @ S)))
            assert np.allclose(np.exp(G)[:, None] * (qq @ S) + (np.tril(qq @ kk.T) * D) @ d, out[r, h], rtol=1e-10, atol=1e-12)
            S = np.exp(G[-1]) * S + (kk * np.exp(G[-1] - G)[:, None]).T @ d
        assert np.allclose(S, after[b.slot_out[0], h], rtol=1e-10, atol=1e-12)
    assert (tol[:23] < 1e-3).all() and (after_tol[b.slot_out[0]] < 1e-2).all()


def test_selection_is_the_sorted_vocabulary():
    """The oracle of the selection against a sort of all continuations."""
    rng = np.random.default_rng(3)
    x = rng.integers(-4, 4, (5, 40)).astype(np.float32)
    x[2, ::3] = -np.inf
    s = rng.integers(-3, 0, 5).astype(np.float64)
    total = s[:, None] + x - np.log(np.exp(x.astype(np.float64)).sum(1, keepdims=True))
    ended = np.array([0, 1, 0, 0, 0])
    total[1], total[1, 7] = -np.inf, s[1]
    order = sorted((-total[b, j], b, -x[b, j] if b != 1 else j != 7, j) for b in range(5) for j in range(40))[:30]
    t, p, y, _ = R.select(x, s, ended, 7, 30)
    assert [(int(b), int(j)) for b, j in zip(p, t)] == [(o[1], o[3]) for o in order]
    assert np.allclose(y, [-o[0] for o in order], rtol=1e-12)


@pytest.mark.skipif(not shutil.which(HIPCC), reason="no hipcc")
@pytest.mark.parametrize("source", ["qmm_delta.hip", "qmm_state.hip", "qmm_beam.hip"])
def test_no_scratch(source):
    """No kernel spills (the walk in halves 32 bytes of a lane, between its start and its loop over groups); a token at a time and
    one group leave registers for two to four workgroups of a CU."""
    kernels = _resources(source)
    assert kernels
    for name, (waves, scratch) in kernels.items():
        assert scratch <= (32 if "delta_walk_kernelILi128ELi4ELb1" in name else 0), (name, scratch)
        if "delta_step" in name or "delta_group" in name:
            assert waves >= (3 if "delta_step_kernelILi128ELi128ELb0" in name else 4), (name, waves)


@pytest.mark.skipif(not shutil.which(HIPCC), reason="no hipcc")
def test_walk_keeps_its_loop_out_of_scratch(tmp_path):
    flags = subprocess.run(["make", "-s", "-C", PKG, "print-flags"], capture_output=True, text=True, timeout=60, check=True).stdout
    asm = tmp_path / "delta.s"
    r = subprocess.run([HIPCC, *flags.split(), "--cuda-device-only", "-S", os.path.join(PKG, "csrc", "qmm_delta.hip"), "-o", str(asm)],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    name, depth, products = "", 0, 0
    for line in asm.read_text().splitlines():
        if re.match(r"_Z\S+:", line):
            name, depth = line.split(":")[0], 0
        elif line.startswith((".LBB", "; %bb.")):  # a block: the loops it is in follow as comments
            depth = 0
        if ";" in line:
            depth = max([depth] + [int(d) for d in re.findall(r"Depth[= ]+(\d+)", line)])
        code = line.split(";")[0]
        products += "delta_walk" in name and depth >= 1 and "v_mfma" in code
        assert not (depth >= 1 and "scratch_" in code), (name, line)
    assert products >= 6 * 40


def test_limits_and_workspaces(tmp_path):
    """tests/state_limits.cpp"""
    exe = str(tmp_path / "state_limits")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                        os.path.join(HERE, "state_limits.cpp"), "-o", exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.stdout + r.stderr)[-2000:]
