"""qmm_paged_attention where roundings and launch choices could show."""
import numpy as np
import pytest

import qmm_hip
from attn_ref import F16_HALF, F32_HALF, Batch, attend, check_rows, queries, run_attention
from gpu_util import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,new,group,hint", [
    (19000, 1, 4, 19000),     # tokens split over workgroups
    (2000, 1, 4, 2000),
    (500, 1, 4, 500),         # one workgroup
    (19000, 1, 4, 1 << 21),   # loads of whole lines
    (6000, 30, 4, 6000),      # 128 rows, split
    (400, 40, 4, 400),        # 128 rows, whole
])
def test_flat_tail_behind_a_strong_key(ctx, q8, D, n, new, group, hint):
    """One key takes nearly all of the weight and has no value; what is left is the many others', each
    1.4 * 2^-24 of it. Weights keep all of an fp16's bits down to 2^-29 of the largest, so the sum is
    right to its own size, whatever the number of tokens."""
    b = Batch([(n, new)], 1, D, 64, q8, seed=n + D, max_pages=max(hint, n) // 64 + 1)
    q = np.ones((b.M, group * D), np.float16)
    scale = 1.0 / D
    score = np.log(2.0 ** 24 / 1.4)  # of the first key; 0 of the others
    p, t = b.cells(0)
    b.k[p, :, t] = 0
    b.v[p, :, :, t] = 127 if q8 else 1
    b.v[p[0], :, :, t[0]] = 0
    if q8:
        b.ks[p, :, t], b.vs[p, :, t] = 1.0, 1 / np.float32(127)
        b.k[p[0], :, t[0]], b.ks[p[0], :, t[0]] = 127, np.float32(score / 127)
    else:
        b.k[p[0], :, t[0]] = score
    say(f"flat tail n={n} new={new} D={D} q8={q8} hint={hint}")
    b.upload(ctx, new, hint)
    got = run_attention(ctx, b, q, group, scale, out_type=qmm_hip.TYPE_F32).astype(np.float64)
    b.free()
    k, v = b.dense(0)
    first = np.exp(-(k[0, 0] @ q[0, :D].astype(np.float64)) * scale)
    for i in range(new):
        tail = (n - new + i) * first
        ref = tail / (1 + tail) * v[0, 1, 0]
        # the first score: D products of equal size summed in fp32, and its product with the scale in base 2; the
        # exponential; each weight's rounding (2^-25 of 2^15 at the largest, 8-bit of 2^9); the output's
        e = 2 * (D + 8) * F32_HALF * score + F16_HALF + (n / 8 + 32) * F32_HALF
        small = n * 2.0 ** -25 * 2.0 ** -(9 if q8 else 15)
        tol = 1.01 * (F16_HALF * (ref + 2.0 ** -14) + e * ref + small)
        d = np.abs(got[i] - ref).max()
        assert d <= tol, f"row {i}: off by {d:.3g} of {ref:.3g}, bound {tol:.3g}"


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,new", [(200, 60), (200, 2), (3000, 60), (3000, 1)])
def test_scales_of_hidden_cells(ctx, D, n, new):
    """8-bit: what scale a cell has that no row sees changes no bit of any row."""
    window, got = 20, []
    for hidden in (0.0, 0.1, 0.3, 0.7, 5.0, 3e38, np.inf, np.nan):
        b = Batch([(n, new)], 1, D, 16, True, seed=D)
        p, t = b.cells(0)
        seen = n - new - window + 1  # the first token of any row's window
        b.vs[p, :, t] *= np.float32(2.0 ** -20)  # (weights with few bits: a change of their exponent shows)
        b.vs[p[:seen], :, t[:seen]] = hidden
        say(f"hidden scale {hidden} n={n} new={new} D={D}")
        b.upload(ctx, new, n)
        got.append(run_attention(ctx, b, queries(b, 4), 4, D ** -0.5, window, out_type=qmm_hip.TYPE_F32))
        b.free()
        assert np.isfinite(got[-1]).all() and (got[-1] != 0).any()
        assert np.array_equal(got[0].view(np.uint32), got[-1].view(np.uint32)), f"hidden scales of {hidden} reached a row"


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens", [[(700, 1)] * 3, [(100, 20), (2000, 1)], [(90, 90)]])
def test_hints_change_the_order_of_sums_only(ctx, lens, q8):
    """Hints choose the launch: the results agree to the roundings of sums in another order."""
    outs = []
    for hints in ((0, 0), (1, 64), (1, 1), (2, 100000), (max(n for _, n in lens), max(n for n, _ in lens))):
        b = Batch(lens, 2, 64, 16, q8, seed=11)
        q = queries(b, 4)
        b.upload(ctx, *hints)
        say(f"hints {hints} lens={lens} q8={q8}")
        outs.append(run_attention(ctx, b, q, 4, 0.125).astype(np.float64))
        b.free()
    ref, tol = attend(b, q, 4, 0.125)
    for o in outs:
        check_rows(o, ref, tol, b.held_rows)
        assert (np.abs(o - outs[0]) <= 2 * tol).all()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,new", [(300, 1), (9000, 1), (200, 40), (9000, 40)])
def test_scores_past_the_digits_of_a_float(ctx, n, new, D, sign, q8):
    """Scores of 2^16 to 2^26 (or their negatives), far apart: a row is the value of its one largest score.
    Where 24 bits end above the point, no rounding of the maximum makes a weight overflow."""
    b = Batch([(n, new)], 1, D, 64, q8, seed=n + D)
    rng = np.random.default_rng(D + new)
    p, t = b.cells(0)
    best = rng.integers(0, n - new + 1)  # (every row sees it)
    size = np.full(n, 0.5 if sign > 0 else 1.0)
    size[best] = 1.0 if sign > 0 else 0.5
    if q8:
        b.k[p, :, t], b.ks[p, :, t] = 64 * sign, size[:, None].astype(np.float32)
        b.vs[p, :, t] = 0.9995
    else:
        b.k[p, :, t] = (64 * sign * size)[:, None, None]
    v = b.dense(0)[1][0, best]
    # q . k scale = 64 D q scale, in base 2 times log2 e: spread over 2^16 .. 2^26, with all digits
    group = 4
    q = (2.0 ** rng.uniform(0, 10, (new, group))).astype(np.float16)
    scale = 2.0 ** 16 / (64 * D * 1.4427)
    say(f"scores of up to 2^26, sign {sign} n={n} new={new} D={D} q8={q8}")
    b.upload(ctx, new, n)
    got = run_attention(ctx, b, np.repeat(q, D, 1), group, scale).astype(np.float64)
    b.free()
    assert np.isfinite(got).all(), f"{np.count_nonzero(~np.isfinite(got))} values are no numbers"
    # one weight, of fp16 over the unrounded sum; its product with the scale; the output
    tol = (2 * F16_HALF + 2.0 ** -20) * np.abs(v) + F16_HALF * 2.0 ** -14
    assert (np.abs(got.reshape(new, group, D) - v) <= tol).all()


@pytest.mark.parametrize("q8", [False, True])
def test_workspace_of_another_call(ctx, q8):
    """One made for a prompt serves single tokens, drafts and both together: the bits of a workspace of
    their own, as they run on as many workgroups."""
    prompt = Batch([(700, 700)], 2, 128, 64, q8, seed=61).upload(ctx, 700, 700)
    q = queries(prompt, 4)
    args = qmm_hip.AttentionArgs(1 << 20, q.shape[1], 8, 0.1, 0, 0, 1 << 20, qmm_hip.TYPE_F16, q.shape[1])  # (not run)
    ws = ctx.attention_workspace(prompt.batch, prompt.cache, args)
    prompt.free()
    for lens in ([(9000, 1)], [(5000, 7), (3000, 3)], [(4000, 60), (6000, 1), (2500, 2)]):
        b = Batch(lens, 2, 128, 64, q8, seed=62).upload(ctx, max(n for _, n in lens), max(n for n, _ in lens))
        q = queries(b, 4)
        say(f"a prompt's workspace for {lens} q8={q8}")
        got = run_attention(ctx, b, q, 4, 0.1, ws=ws)
        own = run_attention(ctx, b, q, 4, 0.1)
        none = run_attention(ctx, b, q, 4, 0.1, workspace=False)
        b.free()
        ref, tol = attend(b, q, 4, 0.1)
        for o in (got, none):
            check_rows(o, ref, tol, b.held_rows)
        assert np.array_equal(got.view(np.uint16), own.view(np.uint16))
        assert not np.array_equal(got.view(np.uint16), none.view(np.uint16)), "work was not shared"
    ws.free()


def test_workspace_of_refused_arguments(ctx):
    """No workspace for a call that the attention refuses, with its reason; one for a call of no rows."""
    b = Batch([(20, 1)], 2, 64, 16, seed=50).upload(ctx, 1, 20)
    make = lambda **kw: qmm_hip.AttentionArgs(**{**dict(  # noqa: E731
        q=1 << 20, q_stride=256, q_heads=4, scale=0.1, out=1 << 20, out_type=qmm_hip.TYPE_F16, out_stride=256), **kw})
    say("workspaces of refused arguments")
    for kw, why in ((dict(q_heads=3), "q_heads"), (dict(scale=0.0), "scale"), (dict(window=-1), "window"), (dict(q_stride=8), "stride")):
        with pytest.raises(qmm_hip.QmmError, match=why):
            ctx.attention_workspace(b.batch, b.cache, make(**kw))
    ctx.attention_workspace(b.batch, b.cache, make()).free()
    b.batch.n_rows = 0
    ctx.attention_workspace(b.batch, b.cache, make(q=None, out=None)).free()
    b.free()


def test_rows_claimed_past_any_count(ctx):
    """Row starts that fall, so that 256 sequences of 2^21 tokens claim all 1024 rows: more work than can be
    counted is not begun, and the next call is as always."""
    S, H, P, D, M, group = 512, 3, 1024, 64, 1024, 16
    b = Batch([(3000, 1)], H, D, P, seed=63).upload(ctx, 1, 3000)
    q = queries(b, group)
    want = run_attention(ctx, b, q, group, 0.125)
    starts = np.zeros(S + 1, np.int32)
    starts[1::2] = M
    up = [ctx.upload(a) for a in (starts, np.full(S, 2 ** 31 - 1, np.int32), np.full((S, 2048), -1, np.int32),
                                  np.zeros((M, H * group * D), np.float16), np.full((M, H * group * D), 7, np.float16))]
    batch = qmm_hip.KvBatch(S, M, int(up[0]), int(up[1]), int(up[2]), 2048, 1, 2 ** 21)
    width = H * group * D
    args = qmm_hip.AttentionArgs(int(up[3]), width, H * group, 0.125, 0, 0, int(up[4]), qmm_hip.TYPE_F16, width)
    ws = ctx.attention_workspace(batch, b.cache, args)
    say("rows claimed past any count")
    ctx.paged_attention(batch, b.cache, args, ws)
    ctx.sync()
    assert (ctx.d2h(up[4], np.float16, (M, width)) == 7).all()
    got = run_attention(ctx, b, q, group, 0.125, ws=ws)
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16))
    ws.free()
    for x in up:
        ctx.free(x)
    b.free()


@pytest.mark.parametrize("q8", [False, True])
def test_captured_prompts_and_single_tokens(q8):
    """A call of both kernels and their joins, captured and replayed with other lengths, rows and queries,
    eager calls of the same context and workspace between: the eager bits each time."""
    group, D, P, H = 4, 64, 64, 2
    with qmm_hip.Context(0) as c:
        b = Batch([(5000, 60), (6000, 1), (2500, 2)], H, D, P, q8, seed=65, max_pages=100).upload(c, 60, 6400)
        b.pages[:, :] = b.pages[:, :1]  # (any length is held: the same page again)
        c.h2d(b.bufs["pages"], b.pages)
        width, rng = H * group * D, np.random.default_rng(4)
        qb = c.upload(queries(b, group))
        outs = [c.upload(np.zeros((b.M, width), np.float16)) for _ in range(2)]
        args = [qmm_hip.AttentionArgs(int(qb), width, H * group, 0.125, 0, 0, int(o), qmm_hip.TYPE_F16, width) for o in outs]
        ws = c.attention_workspace(b.batch, b.cache, args[0])
        c.sync()
        c.graph_begin()
        c.paged_attention(b.batch, b.cache, args[0], ws)
        g = c.graph_end()
        for rep in range(5):
            new = [(60, 1, 2), (1, 61, 1), (20, 20, 23), (0, 0, 63), (63, 0, 0)][rep]
            c.h2d(b.bufs["row_start"], np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
            c.h2d(b.bufs["kv_len"], rng.integers(64, 6400, 3).astype(np.int32))
            c.h2d(qb, (rng.standard_normal((b.M, width)) * 2).astype(np.float16))
            for o in outs:
                c.h2d(o, np.full((b.M, width), np.nan, np.float16))
            say(f"captured prompts and single tokens, replay {rep} new={new} q8={q8}")
            c.graph_launch(g)
            c.paged_attention(b.batch, b.cache, args[1], ws)  # (in stream order behind it)
            c.sync()
            one, two = (c.d2h(o, np.float16, (b.M, width)) for o in outs)
            assert np.isfinite(two).all() and np.array_equal(one.view(np.uint16), two.view(np.uint16)), rep
        c.graph_destroy(g)
        ws.free()
        for x in (qb, *outs):
            c.free(x)
        b.free()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("new", [1, 300])
def test_largest_sequence(ctx, new, q8):
    """A sequence of 2^31 - 256 tokens, of whose pages only the last is there: its new rows are appended (by
    20 workgroups in turn where nothing is known of their number) and attended to, with a window and (one
    row) over all of its 2^25 tiles."""
    D, P, group, cap = 64, 1024, 4, 2 ** 31 - 256
    b = Batch([(P, new)], 1, D, P, q8, seed=71, spare_pages=0)
    table = np.full((1, 2 ** 21), -1, np.int32)
    table[0, -1] = 0
    b.pages, b.max_pages, b.kv_len = table, 2 ** 21, np.array([2 ** 31 - 1], np.int32)  # (the length is clamped)
    b.upload(ctx)
    rng = np.random.default_rng(72)
    x = rng.standard_normal((new, 2 * D)).astype(np.float32)
    xb = ctx.upload(x)
    say(f"largest sequence new={new} q8={q8}")
    ctx.kv_append(b.batch, b.cache, qmm_hip.KvRows(k=int(xb), k_stride=2 * D, v=int(xb) + 4 * D, v_stride=2 * D))
    ctx.sync()
    slots = cap % P  # of the last page
    near = Batch([(slots, new)], 1, D, P, q8, seed=71, spare_pages=0)  # the same page as a short sequence
    near.pages = np.zeros((1, 1), np.int32)
    for n in ("k", "v") + (("ks", "vs") if q8 else ()):
        kept = getattr(b, n)
        got = ctx.d2h(b.bufs[n], kept.dtype, kept.shape)
        axis = 3 if n == "v" else 2
        old = np.delete(kept, np.s_[slots - new:slots], axis)
        assert np.array_equal(np.delete(got, np.s_[slots - new:slots], axis).view(np.uint8), old.view(np.uint8)), f"other cells of {n}"
        setattr(near, n, got)
    k, v = (a[0, -new:] for a in near.dense(0))
    half = np.abs(x.reshape(new, 2, D)).max(2).T[..., None] * ((0.5 + 2.0 ** -14) / 127 if q8 else F16_HALF)
    assert (np.abs(k - x[:, :D]) <= half[0]).all() and (np.abs(v - x[:, D:]) <= half[1]).all()
    q = queries(b, group)
    for window, sinks in ((100, 0), (500, 0), (0, 0)):
        if window == 0 and new > 1:
            continue
        say(f"largest sequence: window {window}")
        ref, tol = attend(near, q, group, 0.125, window, sinks)
        check_rows(run_attention(ctx, b, q, group, 0.125, window, sinks), ref, tol, new)
    ctx.free(xb)
    b.free()
