"""qmm_kv_append against its formulas in 64 bits: norms, both rotation styles,
several position axes, strided rows, both cache types, ragged batches; cells
and rows that are not written keep their bits."""
import numpy as np
import pytest

import qmm_hip
from attn_ref import F16_HALF, Batch, turned
from gpu_util import say

pytestmark = pytest.mark.gpu


def _case(ctx, lens, heads, group, D, P, q8=False, norm=True, rot=None, style="half", axes=1, far=None, base=1e4, scale=1.0,
          freq=None, with_q=True, gap=0, extra_rows=0, seed=0, spoil=None, eps=1e-6, hints=True, spread=1.0):
    b = Batch(lens, heads, D, P, q8, seed=seed, extra_rows=extra_rows)
    rng = np.random.default_rng(seed + 100)
    HQ, M = heads * group, b.M
    rot = D if rot is None else rot
    width = (HQ + 2 * heads) * D + gap
    x = (rng.standard_normal((M, width)) * spread).astype(np.float32)
    gq, gk = (rng.uniform(0.5, 1.5, D).astype(np.float32) for _ in range(2)) if norm else (None, None)
    pos = None
    if far is not None or axes > 1:
        pos = (rng.integers(0, 50, (axes, M)) + (far or 0)).astype(np.int32)
    axis = [j % axes for j in range(rot // 2)]
    f = np.array(freq) if freq is not None else base ** (-2.0 * np.arange(rot // 2) / rot) if rot else None
    if spoil:
        spoil(b)
    say(f"append lens={lens} H={heads}x{group} D={D} P={P} q8={q8} norm={norm} rot={rot} {style} axes={axes} far={far}")
    b.upload(ctx, *((max(n for _, n in b.lens), 0) if hints else (0, 0)))
    xb = ctx.upload(x)
    extra = {n: ctx.upload(a) for n, a in (("gq", gq), ("gk", gk), ("pos", pos)) if a is not None}
    qo = ctx.upload(np.full((M, HQ * D + 4), 9.0, np.float16))
    rope = ctx.rope(rot, style, base, freq, axes, axis, scale) if rot else None
    a = int(xb)
    rows = qmm_hip.KvRows(q=a if with_q else None, q_stride=width, q_heads=HQ if with_q else 0, k=a + 4 * HQ * D, k_stride=width,
                          v=a + 4 * (HQ + heads) * D, v_stride=width, q_gamma=int(extra["gq"]) if norm else None,
                          k_gamma=int(extra["gk"]) if norm else None, eps=eps, rope=rope.handle if rope else None,
                          pos=int(extra["pos"]) if pos is not None else None, pos_stride=M,
                          q_out=int(qo) if with_q else None, q_out_stride=HQ * D + 4)
    ctx.kv_append(b.batch, b.cache, rows)
    ctx.sync()
    got = {"q": ctx.d2h(qo, np.float16, (M, HQ * D + 4)), "k": ctx.d2h(b.bufs["k"], b.k.dtype, b.k.shape),
           "v": ctx.d2h(b.bufs["v"], b.v.dtype, b.v.shape)}
    if q8:
        got["ks"], got["vs"] = (ctx.d2h(b.bufs[n], np.float32, b.ks.shape) for n in ("ks", "vs"))
    for buf in [xb, qo, *extra.values()]:
        ctx.free(buf)
    b.free()
    # what should be there
    written = np.zeros((b.n_pages, P), bool)
    q_rows = np.zeros(M, bool)
    for s in range(b.S):
        n, new = int(b.kv_len[s]), int(b.row_start[s + 1] - b.row_start[s])
        for i in range(new):
            r, p = int(b.row_start[s]) + i, n - new + i
            at = pos[:, r] if pos is not None else np.full(axes, p)
            parts = np.split(x[r, :(HQ + 2 * heads) * D].reshape(-1, D), [HQ, HQ + heads])
            args = (eps, at, rot, style, f, axis, scale)
            q_rows[r] = with_q
            if with_q:
                ref, err = turned(parts[0], gq, *args)
                tol = F16_HALF * (np.abs(ref) + 2.0 ** -14) + 1.01 * err
                d = np.abs(got["q"][r, :HQ * D].reshape(HQ, D).astype(np.float64) - ref)
                assert (d <= tol).all(), f"row {r}: query off by {(d - tol).max():.3g} over its bound"
            page = b.pages[s, p // P] if 0 <= p < b.max_pages * P else -1
            if not 0 <= page < b.n_pages:
                continue
            written[page, p % P] = True
            ref, err = turned(parts[1], gk, *args)
            for name, ref, err, cells in (("k", ref, err, got["k"][page, :, p % P]),
                                          ("v", parts[2].astype(np.float64), np.zeros((heads, D)), got["v"][page, :, :, p % P])):
                if not q8:
                    tol = F16_HALF * (np.abs(ref) + 2.0 ** -14) + 1.01 * err
                    have = cells.astype(np.float64)
                else:
                    sc = got[name + "s"][page, :, p % P].astype(np.float64)[:, None]
                    want = np.abs(ref).max(1, keepdims=True) / 127
                    assert (np.abs(sc - want) <= 2.0 ** -22 * want + 1.01 * err.max() / 127).all(), "scale"
                    have = cells * sc
                    # half a step of the code, its quotient's last bits, and the largest value's own error
                    tol = sc * (0.5 + 127 * 2.0 ** -22) + 2.02 * err.max(1, keepdims=True) + 2.0 ** -22 * np.abs(ref)
                    assert np.abs(cells.astype(int)).max(initial=0) <= 127
                d = np.abs(have - ref)
                assert (d <= tol).all(), f"row {r}: {name} off by {(d - tol).max():.3g} over its bound"
    bits = lambda z: z.view(np.uint8 if z.dtype == np.int8 else np.uint16)  # noqa: E731
    assert np.array_equal(bits(got["k"]).transpose(0, 2, 1, 3)[~written], bits(b.k).transpose(0, 2, 1, 3)[~written]), "other keys"
    assert np.array_equal(bits(got["v"]).transpose(0, 3, 1, 2)[~written], bits(b.v).transpose(0, 3, 1, 2)[~written]), "other values"
    if q8:
        for n in ("ks", "vs"):
            assert np.array_equal(got[n].view(np.uint32).transpose(0, 2, 1)[~written],
                                  getattr(b, n).view(np.uint32).transpose(0, 2, 1)[~written]), "other scales"
    assert (got["q"][~q_rows] == 9).all() and (got["q"][:, HQ * D:] == 9).all(), "q_out past its rows"
    return got, b


RAGGED = [(1, 1), (17, 17), (40, 3), (300, 1), (64, 64), (5, 0), (100, 33)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("style", ["half", "pairs"])
def test_ragged_batch(ctx, q8, D, style):
    _case(ctx, RAGGED, 2, 4, D, 16, q8, style=style, seed=D, extra_rows=2)


@pytest.mark.parametrize("D,rot", [(64, 64), (128, 32), (256, 64), (256, 256), (64, 8), (128, 24)])
@pytest.mark.parametrize("style", ["half", "pairs"])
def test_part_of_a_head(ctx, D, rot, style):
    _case(ctx, [(9, 4), (33, 2)], 3, 1, D, 32, rot=rot, style=style, norm=False, seed=rot)


@pytest.mark.parametrize("far", [0, 100000, 2 ** 31 - 60])
@pytest.mark.parametrize("axes", [1, 2, 3])
def test_positions(ctx, far, axes):
    """Several axes, and positions where a 32-bit angle has lost all its digits."""
    _case(ctx, [(60, 20), (7, 7)], 2, 2, 128, 64, axes=axes, far=far, base=1e6, seed=axes)


def test_own_frequencies_and_scale(ctx):
    freq = np.random.default_rng(5).uniform(-1, 1, 32)
    _case(ctx, [(12, 5)], 1, 2, 64, 16, freq=freq, scale=1.25, seed=5)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("lens", [[(16, 16)], [(15, 15)], [(200, 129)], [(37, 21), (1040, 30)]])
def test_pages(ctx, q8, page, lens):
    _case(ctx, lens, 1, 1, 64, page, q8, norm=False, rot=0, seed=page)


@pytest.mark.parametrize("heads,group", [(1, 1), (3, 5), (9, 1), (20, 1)])
def test_heads(ctx, heads, group):
    _case(ctx, [(3, 2), (50, 1)], heads, group, 128, 16, seed=heads)


def test_keys_and_values_only(ctx):
    _case(ctx, RAGGED, 2, 4, 64, 16, with_q=False, gap=8)


def test_without_hints(ctx):
    _case(ctx, RAGGED, 2, 2, 64, 16, hints=False, seed=1)


def test_many_rows(ctx):
    """Enough rows for one workgroup each."""
    _case(ctx, [(1100, 1100)], 2, 3, 64, 128, seed=2)


def test_rows_without_a_cell(ctx):
    """Pages that are none, places before the first: the queries are there, the cache is as it was."""
    def spoil(b):
        b.pages[0, 1], b.pages[1, 0] = -1, b.n_pages
        b.kv_len[2] = 2  # four new rows, two of them at negative places

    _case(ctx, [(40, 30), (10, 10), (20, 4)], 2, 2, 64, 16, spoil=spoil, seed=3)


def test_zero_and_tiny_rows_of_an_8_bit_cache(ctx):
    """Rows of zeros, and of values too small for a scale: codes and scales of 0."""
    got, b = _case(ctx, [(4, 4)], 1, 1, 64, 16, True, norm=False, rot=0, spread=0.0)
    p, t = b.cells(0)
    for n in ("k", "v"):
        assert (got[n + "s"][p, :, t] == 0).all()


def test_append_twice_is_the_same(ctx):
    one, _ = _case(ctx, RAGGED, 2, 2, 64, 16, seed=21)
    two, _ = _case(ctx, RAGGED, 2, 2, 64, 16, seed=21)
    for n in one:
        assert np.array_equal(one[n].view(np.uint16), two[n].view(np.uint16))
