"""qmm_paged_attention against plain attention in 64 bits: cache types, head
sizes and groups, page sizes, lengths from none to long, several new rows,
windows with first tokens, and cells that hold no numbers."""
import numpy as np
import pytest

import qmm_hip
from attn_ref import Batch, attend, check_rows, queries, run_attention
from gpu_util import say

pytestmark = pytest.mark.gpu


def _check(ctx, b, group, window=0, sinks=0, seed=1, **kw):
    q = queries(b, group, seed)
    scale = b.D ** -0.5
    say(f"attention lens={b.lens} H={b.H}x{group} D={b.D} P={b.P} q8={b.q8} window={window}/{sinks} {kw}")
    hints = kw.pop("hints", True)
    b.upload(ctx, *((max(n for _, n in b.lens), max(n for n, _ in b.lens)) if hints else (0, 0)))
    try:
        got = run_attention(ctx, b, q, group, scale, window, sinks, **kw)
    finally:
        b.free()
    ref, tol = attend(b, q, group, scale, window, sinks)
    check_rows(got, ref, tol, b.held_rows)
    return got


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group,heads", [(1, 3), (4, 2), (7, 1), (17, 1)])
def test_single_tokens(ctx, q8, D, group, heads):
    lens = [(n, 1) for n in (1, 2, 15, 16, 17, 63, 64, 65, 300, 513)]
    _check(ctx, Batch(lens, heads, D, 16, q8, seed=D + group), group)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_pages(ctx, q8, page):
    _check(ctx, Batch([(1, 1), (129, 1), (257, 1), (1030, 1), (64, 1)], 2, 128, page, q8, seed=page), 4)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens", [
    [(5, 5), (70, 3), (200, 8)],          # a few rows
    [(40, 9), (1, 1), (0, 0), (333, 16)],  # up to 64 rows; a sequence of no tokens
    [(130, 130), (70, 33), (257, 1)],     # prompts and single tokens together
    [(300, 270)],                         # one prompt behind a past
])
def test_several_rows(ctx, q8, D, lens):
    _check(ctx, Batch(lens, 2, D, 32, q8, seed=len(lens) + D), 4)


@pytest.mark.parametrize("group", [1, 3, 5, 8])
@pytest.mark.parametrize("new", [2, 11, 65])
def test_groups_of_several_rows(ctx, group, new):
    _check(ctx, Batch([(new + 60, new), (new, new)], 1, 64, 16, seed=group), group)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 1), (50, 4), (64, 64), (64, 70), (100, 130), (200, 0), (100000, 4)])
def test_window(ctx, q8, window, sinks):
    lens = [(400, 1), (7, 7), (330, 19), (64, 1), (260, 150)]
    _check(ctx, Batch(lens, 2, 64, 16, q8, seed=window + sinks), 2, window, sinks)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("new", [1, 6, 80])
def test_pages_outside_a_window_are_not_read(ctx, q8, new):
    """What no row sees may be gone: page ids of none, or pages that hold no numbers."""
    n, window, sinks, P = 500, 70, 5, 16
    for how in ("none", "poison"):
        b = Batch([(n, new)], 2, 64, P, q8, seed=new)
        q = queries(b, 2)
        ref, tol = attend(b, q, 2, 0.125, window, sinks)
        first = n - new - window + 1  # the first token of any row's window
        for t in range(sinks, first):
            page, slot = b.pages[0, t // P], t % P
            if q8:
                b.ks[page, :, slot] = np.nan
                b.vs[page, :, slot] = 3e38
            else:
                b.k[page, :, slot] = np.inf
                b.v[page, :, :, slot] = np.nan
        if how == "none":
            lo, hi = -(-sinks // P), first // P
            b.pages[0, lo:hi] = np.array([-1, b.n_pages, -2 ** 31, 2 ** 31 - 1], np.int64)[np.arange(hi - lo) % 4]
        say(f"cells outside a window: {how} q8={q8} new={new}")
        b.upload(ctx, new, n)
        got = run_attention(ctx, b, q, 2, 0.125, window, sinks)
        b.free()
        check_rows(got, ref, tol, b.held_rows)


@pytest.mark.parametrize("new", [2, 4, 9, 70])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf, "mixed"])
def test_a_value_reaches_only_the_rows_that_see_it(ctx, new, what):
    """No number in a new token's values: earlier rows are as if it were not there, later ones hold it."""
    b = Batch([(100 + new, new), (new, new)], 1, 64, 16, seed=new)
    rng = np.random.default_rng(new)
    for s in range(b.S):
        p, t = b.cells(s)
        for j in (b.lens[s][0] - 1, b.lens[s][0] - 1 - new // 2):
            d = rng.choice(64, 9, replace=False)
            b.v[p[j], 0, d, t[j]] = rng.choice([np.nan, np.inf, -np.inf], 9) if what == "mixed" else what
    _check(ctx, b, 2)


@pytest.mark.parametrize("q8", [False, True])
def test_keys_that_are_no_numbers(ctx, q8):
    """A key of NaN: NaN in the rows that see it, and in no other."""
    b = Batch([(90, 5)], 1, 64, 16, q8, seed=3)
    p, t = b.cells(0)
    if q8:
        b.ks[p[87], 0, t[87]] = np.nan
    else:
        b.k[p[87], 0, t[87], 5] = np.nan
    got = _check(ctx, b, 2)
    assert np.isfinite(got[:2].astype(np.float32)).all() and np.isnan(got[2:].astype(np.float32)).all()


def test_far_apart_value_scales(ctx):
    """8-bit values whose scales differ by up to 2^30: each row's sum keeps its own range."""
    b = Batch([(200, 1), (70, 6)], 2, 64, 16, True, seed=9)
    b.vs *= np.float32(2.0) ** b.rng.integers(-30, 1, b.vs.shape)
    b.poison()
    _check(ctx, b, 4)


def test_large_scores(ctx):
    """Scores of hundreds: one key takes nearly all; and all keys the same."""
    b = Batch([(300, 1), (80, 7)], 2, 128, 16, seed=4, spread=30.0)
    _check(ctx, b, 2)
    b = Batch([(300, 1)], 1, 64, 16, seed=5)
    b.k[:] = 0
    b.poison()
    _check(ctx, b, 2)


def test_rows_that_see_nothing(ctx):
    """Rows at negative places, sequences without tokens, and pages that are all invalid give zeros."""
    b = Batch([(50, 2), (20, 3), (33, 1)], 2, 64, 16, seed=6)
    q = queries(b, 2)
    b.kv_len[1] = 1      # three rows, one token: two rows have no place
    b.pages[2, :] = -1   # nothing to read
    b.upload(ctx, 3, 50)
    got = run_attention(ctx, b, q, 2, 0.125)
    b.free()
    assert (got[2:4] == 0).all() and (got[5] == 0).all()
    b.lens[1], b.lens[2] = (1, 1), (0, 0)
    b.row_start = np.array([0, 2, 2, 2], np.int32)
    first = Batch.dense  # rows of sequence 0, and the last row of sequence 1 over its one token
    ref, tol = attend(b, q, 2, 0.125)
    check_rows(got, ref, tol, 2)
    k, v = first(b, 1)
    one = np.repeat(v[:, 0], 2, 0).reshape(-1)
    assert np.abs(got[4] - one).max() <= 2.0 ** -11 * np.abs(one).max() * 2


@pytest.mark.parametrize("new", [1, 3, 40])
def test_some_pages_invalid(ctx, new):
    """A page that is none hides its tokens and nothing else."""
    b = Batch([(150, new)], 1, 64, 16, seed=7)
    q = queries(b, 2)
    ref_v = b.dense(0)
    gone = [1, 4, 7]
    keep = np.array([j for j in range(150) if j // 16 not in gone])
    b.pages[0, gone] = [-1, b.n_pages, 2 ** 31 - 1]
    b.upload(ctx, new, 150)
    got = run_attention(ctx, b, q, 2, 0.125)
    b.free()
    k, v = ref_v
    for i in range(new):
        j = keep[keep <= 150 - new + i]
        for h in range(2):
            x = k[0][j] @ q[i, h * 64:(h + 1) * 64].astype(np.float64) * 0.125
            w = np.exp(x - x.max())
            w /= w.sum()
            assert np.abs(got[i, h * 64:(h + 1) * 64] - w @ v[0][j]).max() <= 2 ** -10 * (w @ np.abs(v[0][j])).max() + 1e-5


def test_bad_batch_arrays_are_clamped(ctx):
    """Lengths and row starts past what the tensors hold, and below none."""
    b = Batch([(40, 3), (64, 2)], 1, 64, 16, seed=8, extra_rows=2)
    q = queries(b, 2)
    b.kv_len = np.array([-5, 2 ** 31 - 1], np.int32)  # no tokens; all its max_pages hold
    b.row_start = np.array([-7, 3, 2 ** 31 - 1], np.int32)  # rows 0..3 and 3..7
    b.held_rows = b.M
    b.upload(ctx, 3, 64)
    got = run_attention(ctx, b, q, 2, 0.125)
    b.free()
    assert (got[:3] == 0).all()
    b.lens, b.row_start = [(0, 0), (64, 4)], np.array([0, 3, 7], np.int32)
    ref, tol = attend(b, q, 2, 0.125)
    check_rows(got[3:], ref[3:], tol[3:], 4)


@pytest.mark.parametrize("lens", [[(700, 1)] * 3, [(100, 20), (2000, 1)], [(90, 90)]])
def test_hints_change_nothing(ctx, lens):
    """No hints, and hints below the truth (a graph replayed with other lengths)."""
    q8 = False
    outs = []
    for hints in ((0, 0), (1, 64), (1, 1), (2, 100000)):
        b = Batch(lens, 2, 64, 16, q8, seed=11, extra_rows=3)
        q = queries(b, 4)
        b.upload(ctx, *hints)
        say(f"hints {hints} lens={lens}")
        outs.append(run_attention(ctx, b, q, 4, 0.125))
        b.free()
        ref, tol = attend(b, q, 4, 0.125)
        check_rows(outs[-1], ref, tol, b.held_rows)


@pytest.mark.parametrize("q8", [False, True])
def test_outputs_strides_and_no_workspace(ctx, q8):
    lens = [(900, 1), (300, 5), (77, 40)]
    mk = lambda: Batch(lens, 2, 128, 16, q8, seed=12, extra_rows=2)  # noqa: E731
    a = _check(ctx, mk(), 4)
    f = _check(ctx, mk(), 4, out_type=qmm_hip.TYPE_F32, pad=3)
    n = sum(r for _, r in lens)
    assert np.array_equal(a[:n].astype(np.float32), f[:n]), "F32 outputs are the same values"
    _check(ctx, mk(), 4, workspace=False)
    _check(ctx, mk(), 4, hints=False)


def test_results_do_not_vary(ctx):
    """The same call twice gives the same bits (splits are joined in order)."""
    b = Batch([(3000, 1), (1500, 2)], 2, 128, 16, seed=13)
    q = queries(b, 4)
    b.upload(ctx, 2, 3000)
    one = run_attention(ctx, b, q, 4, 0.1)
    two = run_attention(ctx, b, q, 4, 0.1, repeat=5)
    b.free()
    assert np.array_equal(one.view(np.uint16), two.view(np.uint16))


def test_small_workspace(ctx):
    """A workspace for fewer splits, or for none."""
    b = Batch([(2000, 1)], 1, 64, 16, seed=14)
    q = queries(b, 4)
    ref, tol = attend(b, q, 4, 0.125)
    b.upload(ctx, 1, 2000)
    for n in (0, 1000, 30000):
        import ctypes
        h = ctypes.c_void_p()
        assert ctx.lib.qmm_attention_workspace_create(ctx._h, n, ctypes.byref(h)) == 0
        ws = qmm_hip._Handle(ctx, h.value, "qmm_attention_workspace_destroy")
        check_rows(run_attention(ctx, b, q, 4, 0.125, ws=ws), ref, tol, 1)
        ws.free()
    b.free()


@pytest.mark.parametrize("q8", [False, True])
def test_long_sequence(ctx, q8):
    b = Batch([(20011, 1)], 1, 128, 64, q8, seed=15)
    _check(ctx, b, 4)
