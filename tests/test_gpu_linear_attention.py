"""qmm_short_conv and qmm_gated_delta against their formulas in 64 bits: ragged
batches, carried states in the same or other slots, strided rows; rows and slots
that nobody holds keep their bits."""
import numpy as np
import pytest

import qmm_hip
import state_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu


def _conv_case(ctx, news, channels=64, width=4, bias=False, silu=True, slots=None, gap=0, extra=0, hints=True, seed=0):
    say(f"conv news={news} C={channels} W={width} bias={bias} silu={silu} slots={slots} gap={gap}")
    b = R.States(news, slots, seed, extra, gap=gap)
    x, pool = b.rows(channels), b.pool(width - 1, channels)
    w = b.rng.uniform(-1, 1, (channels, width)).astype(np.float32)
    bi = b.rng.uniform(-1, 1, channels).astype(np.float32) if bias else None
    b.upload(ctx, hints)
    xb, wb, pb, bb = ctx.upload(x), ctx.upload(w), ctx.upload(pool), ctx.upload(bi) if bias else None
    ob = ctx.upload(np.full((b.M, channels + gap), 7.0, np.float32))
    ctx.short_conv(b.batch, qmm_hip.ConvArgs(int(xb), channels + gap, channels, width, int(wb), int(bb) if bias else None, int(pb),
                                             int(silu), int(ob), channels + gap))
    ctx.sync()
    out, after = ctx.d2h(ob, np.float32, (b.M, channels + gap)), ctx.d2h(pb, np.float32, pool.shape)
    for u in [xb, wb, pb, bb, ob, *b.bufs]:
        if u is not None:
            ctx.free(u)
    ref, tol, ref_pool = R.conv(b, x, w, bi, pool, silu)
    assert (out[:, channels:] == 7).all() and (out[b.held:] == 7).all(), "written past the rows"
    R.within(out[:b.held, :channels], ref[:b.held], tol[:b.held], "rows")
    assert np.array_equal(after.view(np.uint32), ref_pool.view(np.uint32)), "carried inputs are copies, other slots as they were"


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("news", [[1], [0], [2, 1, 0, 3], [15, 16, 17], [4, 5, 31, 32, 33, 100]], ids=str)
def test_conv_lengths(ctx, news, width):
    _conv_case(ctx, news, width=width, bias=width == 3, silu=width != 2, seed=width)


@pytest.mark.parametrize("channels", [4, 60, 1020, 1024, 1028, 8192])
def test_conv_channels(ctx, channels):
    _conv_case(ctx, [3, 1, 18], channels, gap=4, extra=2, seed=channels)


@pytest.mark.parametrize("news", [[1, 1], [2, 5], [40, 3]], ids=str)
def test_conv_slots(ctx, news):
    """In place; new sequences; states not kept; slots outside the pool; no hint, and a wrong one."""
    _conv_case(ctx, news, slots=[(1, 1), (0, 0)])
    _conv_case(ctx, news, slots=[(-1, 1), (0, -1)], hints=False)
    _conv_case(ctx, news, slots=[(-7, 0), (-2 ** 31, 2)])


def test_conv_wrong_hint_and_no_slots(ctx):
    b = R.States([70, 3], seed=3).upload(ctx)
    x, w = b.rows(8), np.ones((8, 4), np.float32)
    xb, wb, ob = ctx.upload(x), ctx.upload(w), ctx.upload(np.zeros((b.M, 8), np.float32))
    b.batch.max_new = 1
    b.batch.slot_in = b.batch.slot_out = None
    ctx.short_conv(b.batch, qmm_hip.ConvArgs(int(xb), 8, 8, 4, int(wb), None, None, 0, int(ob), 8))
    ctx.sync()
    b.slot_in[:] = b.slot_out[:] = -1
    ref, tol, _ = R.conv(b, x, w, None, b.pool(3, 8), False)
    R.within(ctx.d2h(ob, np.float32, (b.M, 8)), ref, tol, "rows")


# -------------------------------------------------------------- delta rule
def delta_case(ctx, news, HK=1, of=2, DK=128, DV=128, gamma=True, gate=True, slots=None, gap=0, extra=0, hints=True, seed=0, ws=True,
               spread=1.0, decay=(0.0, 1.0), state_spread=0.3, alike=0.0, stream=None, repeat=1, eps=1e-6):
    say(f"delta news={news} H={HK}x{of} D={DK},{DV} gamma={gamma} gate={gate} slots={slots} gap={gap} ws={ws} spread={spread} decay={decay}")
    b = R.States(news, slots, seed, extra, gap=gap)
    HV, M = HK * of, b.M
    kw, vw = HK * DK, HV * DV
    qkv = b.rows(2 * kw + vw)
    if alike:  # keys that lie close together: the steps of a group hang on each other
        base = b.rng.standard_normal(DK).astype(np.float32)
        for h in range(HK):
            part = qkv[:b.held, kw + h * DK:kw + (h + 1) * DK]
            part[:] = alike * base + (1 - alike) * part
    qkv[:b.held, 2 * kw:2 * kw + vw] *= np.float32(spread)
    ab = b.rows(2 * HV, gap=3)
    rate = -b.rng.uniform(*decay, HV).astype(np.float32)
    dt = b.rng.uniform(-2, 1, HV).astype(np.float32)
    pool = b.pool(HV, DK, DV, spread=state_spread * spread)
    z = b.rows(vw) if gate else None
    gm = b.rng.uniform(0.5, 1.5, DV).astype(np.float32) if gamma else None
    b.upload(ctx, hints)
    up = {n: ctx.upload(x) for n, x in (("qkv", qkv), ("ab", ab), ("rate", rate), ("dt", dt), ("pool", pool), ("z", z), ("gm", gm)) if x is not None}
    at = {n: int(x) for n, x in up.items()}
    ob = ctx.upload(np.full((M, vw + gap), 7.0, np.float32))
    W = 2 * kw + vw + gap
    args = qmm_hip.DeltaArgs(q=at["qkv"], k=at["qkv"] + 4 * kw, q_stride=W, k_stride=W, v=at["qkv"] + 8 * kw, v_stride=W, qk_heads=HK,
                             v_heads=HV, key_dim=DK, value_dim=DV, a=at["ab"], b=at["ab"] + 4 * HV, a_stride=2 * HV + 3,
                             b_stride=2 * HV + 3, rate=at["rate"], dt_bias=at["dt"], scale=DK ** -0.5, qk_eps=eps, state=at["pool"],
                             z=at.get("z"), z_stride=vw + gap, gamma=at.get("gm"), gamma_eps=1e-6, out=int(ob), out_stride=vw + gap)
    w = ctx.gated_delta_workspace(b.batch, args) if ws else None
    for _ in range(repeat):
        ctx.gated_delta(b.batch, args, w)
    ctx.sync()
    out, after = ctx.d2h(ob, np.float32, (M, vw + gap)), ctx.d2h(up["pool"], np.float32, pool.shape)
    for u in [ob, *up.values(), *b.bufs]:
        ctx.free(u)
    if w:
        w.free()
    ref, tol, ref_pool, pool_tol = R.delta(
        b, qkv[:, :kw].reshape(M, HK, DK), qkv[:, kw:2 * kw].reshape(M, HK, DK), qkv[:, 2 * kw:2 * kw + vw].reshape(M, HV, DV),
        ab[:, :HV], ab[:, HV:2 * HV], rate, dt, DK ** -0.5, eps, pool, None if z is None else z[:, :vw], gm, 1e-6, of)
    assert (out[:, vw:] == 7).all() and (out[b.held:] == 7).all(), "written past the rows"
    R.within(out[:b.held, :vw], ref[:b.held].reshape(-1, vw), tol[:b.held].reshape(-1, vw), "rows")
    R.within(after, ref_pool, pool_tol, "states")
    written = [i for *_, i in b.sequences() if i >= 0]
    rest = np.setdiff1d(np.arange(b.n_slots), written)
    assert np.array_equal(after[rest].view(np.uint32), pool[rest].view(np.uint32)), "other slots were written"
    return out, after


@pytest.mark.parametrize("ws", [False, True])
@pytest.mark.parametrize("news", [[1], [0], [1, 0, 1, 1], [2, 7, 8, 9], [16, 17, 1], [31, 32, 33], [63, 64, 65, 0, 5], [130, 200]], ids=str)
def test_delta_lengths(ctx, news, ws):
    delta_case(ctx, news, ws=ws, seed=len(news))


@pytest.mark.parametrize("ws", [False, True])
@pytest.mark.parametrize("HK,of", [(1, 1), (2, 3), (5, 2)])
@pytest.mark.parametrize("DK,DV", [(64, 64), (64, 128), (128, 64), (128, 128)])
def test_delta_heads(ctx, DK, DV, HK, of, ws):
    delta_case(ctx, [40, 1, 33], HK, of, DK, DV, gamma=of != 3, gate=of != 2, gap=4, extra=3, ws=ws, seed=DK + DV + of)


@pytest.mark.parametrize("ws", [False, True])
@pytest.mark.parametrize("news", [[1, 1], [3, 9], [70, 2]], ids=str)
def test_delta_slots(ctx, news, ws):
    """In place; new sequences; states that are not kept; slots outside the pool; without hints."""
    delta_case(ctx, news, slots=[(1, 1), (0, 0)], ws=ws)
    delta_case(ctx, news, slots=[(-1, 1), (0, -1)], ws=ws, hints=False)
    delta_case(ctx, news, slots=[(-2 ** 31, -5), (-1, 0)], ws=ws, gamma=False, gate=False)


@pytest.mark.parametrize("ws", [False, True])
@pytest.mark.parametrize("spread", [1e-12, 1e-3, 6e4])
def test_delta_sizes_of_values(ctx, spread, ws):
    """Values and states of any size that the inputs may have, beside rows of another size."""
    delta_case(ctx, [50, 70], spread=spread, gamma=False, gate=False, ws=ws)


@pytest.mark.parametrize("ws", [False, True])
@pytest.mark.parametrize("decay", [(0.0, 1e-6), (20.0, 200.0), (5e3, 1e4)])
def test_delta_decays(ctx, decay, ws):
    """Almost none; a state that a few tokens forget; one that each token forgets."""
    delta_case(ctx, [97, 3, 64], decay=decay, gamma=False, ws=ws)


@pytest.mark.parametrize("ws", [False, True])
@pytest.mark.parametrize("alike", [0.9, 0.999, 1.0])
def test_delta_keys_alike(ctx, alike, ws):
    delta_case(ctx, [100, 33], alike=alike, decay=(0.0, 0.01), gamma=False, ws=ws)


def test_delta_same_bits(ctx):
    for news in ([1, 1, 5], [300, 70]):
        a, b = delta_case(ctx, news, HK=2, seed=5), delta_case(ctx, news, HK=2, seed=5)
        assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(a, b))


@pytest.mark.parametrize("DK,DV", [(64, 64), (64, 128), (128, 64), (128, 128)])
def test_delta_many_heads(ctx, DK, DV):
    """More heads than compute units: a workgroup has all columns of one."""
    rng = np.random.default_rng(DK + DV)
    news = [int(n) for n in rng.integers(0, 70, 33)] + [100]
    delta_case(ctx, news, 3, 3, DK, DV, gap=4, extra=2, seed=DV)
    delta_case(ctx, news, 3, 3, DK, DV, gamma=False, gate=False, slots=[(i, i) for i in range(34)], seed=DK)


@pytest.mark.parametrize("DK,DV,of", [(64, 64, 65), (64, 128, 33), (128, 64, 65), (128, 128, 33)])
def test_delta_long_many_heads(ctx, DK, DV, of):
    """Heads that fill the compute units, of sequences long enough for three launches, one of them not a multiple of a group."""
    delta_case(ctx, [201], 2, of, DK, DV, gap=4, extra=2, seed=DV)


@pytest.mark.parametrize("ws", [False, True])
@pytest.mark.parametrize("hint", [1, 9, 40, 1000])
def test_delta_wrong_hints(ctx, hint, ws):
    """Sequences longer than the host knew, and shorter: a choice of launch only."""
    delta_case(ctx, [70, 0, 1, 33, 260], 2, 2, hints=hint, ws=ws, slots=[(0, 0), (1, 1), (2, 2), (3, 4), (5, 5)])


@pytest.mark.parametrize("DK,DV", [(64, 64), (64, 128), (128, 64), (128, 128)])
def test_delta_halves(ctx, DK, DV):
    """Sequences that are walked in halves beside others that are not: an even and an odd number of groups, a last group of one
    token, the shortest ones; states in place, new, not kept."""
    kw = dict(gap=4, extra=3, ws=True, seed=DK + DV)
    delta_case(ctx, [1025, 0, 481, 480, 1, 700, 33], 1, 2, DK, DV, **kw)
    delta_case(ctx, [640, 511, 512, 40, 900], 1, 3, DK, DV, gamma=False, slots=[(0, 0), (-1, 2), (3, -1), (4, 4), (5, 6)], **kw)
    delta_case(ctx, [3000], 2, 2, DK, DV, gate=False, hints=False, **kw)


@pytest.mark.parametrize("decay", [(0.0, 1e-6), (0.0, 0.01), (20.0, 200.0)])
@pytest.mark.parametrize("alike", [0.0, 0.999, 1.0])
def test_delta_halves_of_all_kinds(ctx, decay, alike):
    delta_case(ctx, [1600, 560], alike=alike, decay=decay, spread=100.0, ws=True)
    delta_case(ctx, [1600, 560], alike=alike, decay=decay, spread=1e-3, state_spread=10.0, gamma=False, gate=False, ws=True)


@pytest.mark.parametrize("news", [[3, 1], [30, 9], [200, 40], [700]], ids=str)
def test_delta_decays_past_fp32(ctx, news):
    """Log decays that overflow, beside heads that forget little: a state is forgotten, and no infinity meets another."""
    delta_case(ctx, news, 2, 2, decay=(1e38, 3e38))
    delta_case(ctx, news, 2, 2, decay=(100.0, 1e7))


@pytest.mark.parametrize("news", [[3, 1], [30, 9], [200, 40], [700, 2]], ids=str)
@pytest.mark.parametrize("which", ["q", "k", "v", "a", "b", "state"])
def test_delta_no_number_shows(ctx, which, news):
    """A NaN is in its own head's output of the token and in the state after it; a query's in no state."""
    rng = np.random.default_rng(3)
    HK, HV, D, m, n = 2, 4, 64, sum(news), len(news)
    say(f"delta NaN in {which} news={news}")
    x = {"q": rng.standard_normal((m, HK, D)), "k": rng.standard_normal((m, HK, D)), "v": rng.standard_normal((m, HV, D)),
         "a": rng.standard_normal((m, HV)), "b": rng.standard_normal((m, HV)), "state": rng.standard_normal((n, HV, D, D))}
    x = {i: y.astype(np.float32) for i, y in x.items()}
    row, h = (0 if which == "state" else 1), 1  # (head 1 reads key head 0)
    x[which][(0, h, 5, 7) if which == "state" else (row, 0, 5) if which in "qk" else (row, h, 7) if which == "v" else (row, h)] = np.nan
    up = {i: ctx.upload(y) for i, y in x.items()}
    up.update(starts=ctx.upload(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)), slots=ctx.upload(np.arange(n, dtype=np.int32)),
              rate=ctx.upload(np.full(HV, -0.1, np.float32)), dt=ctx.upload(np.zeros(HV, np.float32)), out=ctx.upload(np.zeros((m, HV, D), np.float32)))
    at = {i: int(u) for i, u in up.items()}
    batch = qmm_hip.StateBatch(n, m, at["starts"], at["slots"], at["slots"], n, max(news))
    args = qmm_hip.DeltaArgs(q=at["q"], k=at["k"], q_stride=HK * D, k_stride=HK * D, v=at["v"], v_stride=HV * D, qk_heads=HK, v_heads=HV, key_dim=D,
                             value_dim=D, a=at["a"], b=at["b"], a_stride=HV, b_stride=HV, rate=at["rate"], dt_bias=at["dt"], scale=1.0, qk_eps=1e-6,
                             state=at["state"], out=at["out"], out_stride=HV * D)
    ws = ctx.gated_delta_workspace(batch, args)
    ctx.gated_delta(batch, args, ws)
    ctx.sync()
    out, state = np.isnan(ctx.d2h(up["out"], np.float32, (m, HV, D))), np.isnan(ctx.d2h(up["state"], np.float32, (n, HV, D, D)))
    ws.free()
    for u in up.values():
        ctx.free(u)
    mine = [0, 1] if which in "qk" else [h]
    rest = [i for i in range(HV) if i not in mine]
    column = 7 if which in ("v", "state") else slice(None)
    assert out[row, mine][:, column].all()
    if which == "q":
        assert not state.any() and not out[2:].any() and not out[0].any()
    else:
        assert state[0, mine][:, :, column].all()
    assert not out[:, rest].any() and not state[:, rest].any() and not out[news[0]:].any() and not state[1:].any()


@pytest.mark.parametrize("n", [2, 63, 64, 65, 130])
def test_delta_many_sequences(ctx, n):
    """Sequences in the order of their lengths, up to 64 of them; equal lengths and empty ones among them."""
    rng = np.random.default_rng(n)
    news = [int(x) for x in rng.choice([0, 1, 31, 33, 64, 65, 97], n - 1)] + [330]
    delta_case(ctx, news, 1, 1, 64, 64, seed=n)


@pytest.mark.parametrize("hint", [True, 1])
@pytest.mark.parametrize("DK,DV", [(64, 64), (64, 128), (128, 64), (128, 128)])
def test_delta_large_batches(ctx, DK, DV, hint):
    """More workgroups than three a CU, with states of more than 32 MB in all and less; some read no state, some keep none."""
    rng = np.random.default_rng(DK + 2 * DV)
    news = [int(n) for n in rng.integers(0, 9 if hint is True else 3, 270)] + ([] if hint is True else [19, 1])
    slots = [(i if i % 5 else -1, i if i % 7 else -1) for i in range(len(news))]
    delta_case(ctx, news, 1, 3, DK, DV, slots=slots, hints=hint, seed=DV)
