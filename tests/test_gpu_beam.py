"""qmm_beam_select against the definition in 64 bits, and qmm_copy_slots."""
import numpy as np
import pytest

import qmm_hip
import state_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu


def beam_case(ctx, logits, score, ended, K, beams, gap=0, offset=0, end_token=0, ws=None):
    """logits [items * beams][vocab]"""
    rows, V = logits.shape
    items = rows // beams
    say(f"beam items={items} beams={beams} vocab={V} keep={K} gap={gap} offset={offset}")
    x = np.full(offset + rows * (V + gap), np.nan, np.float32)
    x[offset:].reshape(rows, V + gap)[:, :V] = logits
    bufs = [ctx.upload(x), ctx.upload(np.full((items, K), -5, np.int32)), ctx.upload(np.full((items, K), -5, np.int32)),
            ctx.upload(np.full((items, K), 5, np.float32))]
    sb = ctx.upload(score.astype(np.float32)) if score is not None else None
    eb = ctx.upload(ended.astype(np.int32)) if ended is not None else None
    a = qmm_hip.BeamArgs(int(bufs[0]) + 4 * offset, V + gap, V, items, beams, int(sb) if sb else None, int(eb) if eb else None, end_token, K,
                         int(bufs[1]), int(bufs[2]), int(bufs[3]))
    ctx.beam_select(a, ws or ctx.beam_workspace(a))
    ctx.sync()
    token, parent = (ctx.d2h(b, np.int32, (items, K)) for b in bufs[1:3])
    out = ctx.d2h(bufs[3], np.float32, (items, K))
    for u in bufs + [u for u in (sb, eb) if u]:
        ctx.free(u)
    for i in range(items):
        part = slice(i * beams, (i + 1) * beams)
        t, p, total, certain = R.select(logits[part], np.zeros(beams) if score is None else score[part], None if ended is None else ended[part],
                                        end_token, K)
        assert certain.mean() > 0.5 or K < 4
        assert np.array_equal(token[i][certain], t[certain]) and np.array_equal(parent[i][certain], p[certain]), (i, token[i], t, parent[i], p)
        fine = np.isfinite(total)
        # the sum of exponentials: 40 roundings; the total rounded once, its parts before that in 64 bits
        assert np.array_equal(out[i][~fine], total[~fine].astype(np.float32))
        assert (np.abs(out[i][fine] - total[fine]) <= 40 * R.U + R.U * np.abs(total[fine])).all()
    return token, parent, out


def _logits(rows, V, seed=0, spread=2.5):
    return (np.random.default_rng(seed).standard_normal((rows, V)) * spread).astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 5, 63, 64, 65, 2047, 2048, 2049, 4100, 30011, 151936])
@pytest.mark.parametrize("beams,K", [(1, 1), (4, 8), (3, 7)])
def test_vocabularies(ctx, V, beams, K):
    rng = np.random.default_rng(V)
    beam_case(ctx, _logits(2 * beams, V, V), rng.uniform(-30, -20, 2 * beams), None, min(K, beams * V), beams, gap=V % 5)


@pytest.mark.parametrize("K", [1, 2, 16, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("beams", [1, 5, 64])
def test_keep(ctx, beams, K):
    rng = np.random.default_rng(K)
    beam_case(ctx, _logits(beams, 9001, K), rng.uniform(-3, 0, beams), None, K, beams)
    beam_case(ctx, _logits(beams, 70 if K <= 32 else 100, K), rng.uniform(-3, 0, beams), rng.random(beams) < 0.3, K, beams, end_token=64)


def test_many_slices(ctx):
    """More lists than lanes, and fewer than kept ones."""
    for V, K in ((150000, 64), (300001, 16), (262144, 5), (60000, 40)):
        beam_case(ctx, _logits(2, V, V), None, None, K, 2)


@pytest.mark.parametrize("offset,gap", [(0, 0), (1, 0), (2, 1), (3, 3), (4, 4)])
def test_alignment(ctx, offset, gap):
    beam_case(ctx, _logits(6, 5003, offset), np.zeros(6), None, 6, 3, gap, offset)


def test_ties_go_to_the_lower_beam_and_token(ctx):
    rng = np.random.default_rng(1)
    x = rng.integers(-3, 3, (8, 6000)).astype(np.float32)
    beam_case(ctx, x, np.repeat([-1.0, -2.0], 4), None, 64, 4)
    beam_case(ctx, np.zeros((8, 4500), np.float32), np.zeros(8), None, 33, 8)
    one = _logits(1, 5000, 3)
    t, p, _ = beam_case(ctx, np.repeat(one, 5, 0), np.zeros(5), None, 10, 5)  # beams alike: in their order
    assert np.array_equal(p[0], np.tile(np.arange(5), 2))
    z = np.zeros((2, 100), np.float32)
    z[:, ::2] = -0.0
    beam_case(ctx, z, None, None, 20, 2)


def test_ruled_out_tokens(ctx):
    rng = np.random.default_rng(2)
    x = _logits(8, 9000, 2)
    x[rng.random(x.shape) < 0.9995] = -np.inf
    beam_case(ctx, x, rng.uniform(-3, 0, 8), None, 32, 4)
    x[3] = -np.inf  # a beam with nothing left
    x[4:] = -np.inf  # an item with nothing left
    beam_case(ctx, x, rng.uniform(-3, 0, 8), None, 16, 4)
    beam_case(ctx, np.full((3, 70), np.finfo(np.float32).min, np.float32), None, None, 5, 3)
    low = _logits(3, 5000, 6)
    low[:, 100:] = np.finfo(np.float32).min  # masked by the type's lowest value
    beam_case(ctx, low, None, None, 64, 3)


def test_no_numbers(ctx):
    x = _logits(4, 3001, 4)
    x[0, 5], x[0, 6], x[1, 7], x[2] = np.nan, np.inf, -np.nan, np.nan
    s = np.array([-1.0, np.nan, -2.0, np.inf])
    beam_case(ctx, x, s, None, 20, 4)
    beam_case(ctx, x, np.full(4, -np.inf), None, 9, 4)


def test_ended_beams(ctx):
    x = _logits(8, 4000, 5)
    x[1] = np.nan  # (not read)
    for e in (0, 3, 3999):
        beam_case(ctx, x, np.linspace(-9, -1, 8), np.array([0, 1, 0, 1, 1, 1, 1, 1]), 12, 4, end_token=e)
    beam_case(ctx, x, np.full(8, -np.inf), np.ones(8), 12, 4, end_token=9)
    beam_case(ctx, x[:4, :3], np.linspace(-9, -1, 4), np.array([1, 0, 1, 0]), 12, 4, end_token=1)


def test_best_tokens_side_by_side(ctx):
    """Values that all lie in a few lanes or lists: candidates by the thousand."""
    x = _logits(2, 150001, 7)
    x[:, :4096] += 100
    x[0] = np.sort(x[0])
    beam_case(ctx, x, None, None, 64, 2)
    y = np.zeros((1, 140000), np.float32)
    y[0, :131072].reshape(64, 2048)[:, :64] = 50 + _logits(64, 64, 8)  # 64 lists of 64 good ones each
    beam_case(ctx, y, None, None, 64, 1)
    y[0, :131072].reshape(64, 2048)[:, :64] = 50 + 100 * np.arange(64)[:, None] + _logits(64, 64, 8)
    beam_case(ctx, y, None, None, 64, 1)
    y[0, :131072].reshape(64, 2048)[:, :64] = 50 + np.where(np.arange(64) == 63, 0, 1)[None] * (1 + np.abs(_logits(64, 64, 8)))
    beam_case(ctx, y, None, None, 64, 1)


@pytest.mark.parametrize("n_pools,pairs,size", [(1, 1, 16), (3, 7, 4096 + 16), (70, 2, 48), (2, 5, 70000 * 16), (129, 1, 32)])
def test_copies(ctx, n_pools, pairs, size):
    say(f"copy pools={n_pools} pairs={pairs} bytes={size}")
    rng = np.random.default_rng(n_pools)
    slots = 2 * pairs + 3
    pools = [rng.integers(0, 255, (slots, size), np.uint8) for _ in range(n_pools)]
    order = rng.permutation(slots)
    src, dst = order[:pairs][rng.integers(0, pairs, pairs)], order[pairs:2 * pairs]
    src = np.concatenate([src, [order[-1], -1, slots, order[-1], 2 ** 31 - 1]]).astype(np.int32)  # (the last ones copy nothing)
    dst = np.concatenate([dst, [slots, order[-1], order[-1], order[-1], -2 ** 31]]).astype(np.int32)
    bufs = [ctx.upload(p) for p in pools]
    sb, db = ctx.upload(src), ctx.upload(dst)
    ctx.copy_slots([qmm_hip.SlotPool(int(b), size, slots) for b in bufs], sb, db, len(src))
    ctx.sync()
    for p, b in zip(pools, bufs):
        p[dst[:pairs]] = p[src[:pairs]]
        assert np.array_equal(ctx.d2h(b, np.uint8, p.shape), p)
    for u in [*bufs, sb, db]:
        ctx.free(u)


def test_copies_of_pools_of_several_sizes(ctx):
    rng = np.random.default_rng(1)
    sizes, slots = [16, 40000, 0, 1 << 20], [9, 4, 5, 3]
    pools = [rng.integers(0, 255, (n, s), np.uint8) for s, n in zip(sizes, slots)]
    src, dst = np.array([0, 2, 5], np.int32), np.array([1, 3, 6], np.int32)
    bufs = [ctx.upload(p) if p.size else ctx.malloc(16) for p in pools]
    sb, db = ctx.upload(src), ctx.upload(dst)
    ctx.copy_slots([qmm_hip.SlotPool(int(b), s, n) for b, s, n in zip(bufs, sizes, slots)], sb, db, 3)
    ctx.copy_slots([], sb, db, 3)
    ctx.sync()
    for p, b, n in zip(pools, bufs, slots):
        for i, j in zip(src, dst):
            if i < n and j < n:
                p[j] = p[i]
        if p.size:
            assert np.array_equal(ctx.d2h(b, np.uint8, p.shape), p)
    for u in [*bufs, sb, db]:
        ctx.free(u)


@pytest.mark.parametrize("V,gap", [(5003, 0), (5001, 0), (5002, 1), (9002, 0), (50257, 0), (2047, 0), (3, 0)])
def test_beams_alike_at_any_alignment(ctx, V, gap):
    """Rows of the same bits at the four places that a row may have in 16 B: the same totals, bit for bit, so the lower beam first."""
    one = _logits(1, V, V)
    K = min(10, 5 * V)
    t, p, total = beam_case(ctx, np.repeat(one, 10, 0), None, None, K, 5, gap)
    assert np.array_equal(p, np.tile(np.arange(5), (2, 2))[:, :K]) and np.array_equal(t[0], t[1])
    assert len({x.tobytes() for x in total.reshape(-1, 5)}) == K // 5
    for offset in (1, 2, 3):  # the same item elsewhere
        again = beam_case(ctx, np.repeat(one, 10, 0), None, None, K, 5, gap, offset)
        assert all(x.tobytes() == y.tobytes() for x, y in zip(again, (t, p, total)))
