"""qmm_kv_append at the ends of its numbers: values that are no numbers, rows at
the smallest scale of an 8-bit cache, and what the attention makes of them."""
import numpy as np
import pytest

import qmm_hip
from attn_ref import Batch, queries, run_attention
from gpu_util import say

pytestmark = pytest.mark.gpu


def _append(ctx, b, x, norm=False):
    """k and v of all heads, side by side in x [M][2 * heads * dim]; the cache afterwards."""
    width, W = 2 * b.H * b.D, b.H * b.D
    xb, g = ctx.upload(x), ctx.upload(np.ones(b.D, np.float32))
    ctx.kv_append(b.batch, b.cache, qmm_hip.KvRows(k=int(xb), k_stride=width, v=int(xb) + 4 * W, v_stride=width, eps=1e-6,
                                                   k_gamma=int(g) if norm else None))
    ctx.sync()
    got = {n: ctx.d2h(b.bufs[n], getattr(b, n).dtype, getattr(b, n).shape) for n in ("k", "v") + (("ks", "vs") if b.q8 else ())}
    ctx.free(xb)
    ctx.free(g)
    return got


# a whole group of 8 slots, parts of one, and single tokens
LENS = [(16, 16), (29, 7), (40, 1), (19, 19)]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("what", [np.nan, -np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("norm", [False, True])
def test_no_numbers_into_an_8_bit_cache(ctx, D, what, norm):
    """A value that is no number makes its token's head one: a scale of NaN over codes of 0. The heads
    and tokens beside it are as without it."""
    H, P = 3, 16
    rng = np.random.default_rng(D)
    clean = Batch(LENS, H, D, P, True, seed=D).upload(ctx, 19, 40)
    x = rng.standard_normal((clean.M, 2 * H * D)).astype(np.float32)
    say(f"8-bit append of {what} D={D} norm={norm}")
    want = _append(ctx, clean, x, norm)
    clean.free()
    hit = {"k": [], "v": []}  # (row, head)
    for r in range(0, clean.M, 3):
        part, h, d = ("k", "v")[r // 3 % 2], int(rng.integers(H)), int(rng.integers(D))
        x[r, ((part == "v") * H + h) * D + d] = what
        hit[part].append((r, h))
    b = Batch(LENS, H, D, P, True, seed=D).upload(ctx, 19, 40)
    got = _append(ctx, b, x, norm)
    b.free()
    at = {}
    for s, (n, new) in enumerate(b.lens):
        p, t = b.cells(s)
        for i in range(new):
            at[b.row_start[s] + i] = p[n - new + i], t[n - new + i]
    for part, axes in (("k", (0, 1, 2, 3)), ("v", (0, 1, 3, 2))):
        codes, kept = got[part].transpose(axes), np.ones((b.n_pages, H, P), bool)
        for r, h in hit[part]:
            page, slot = at[r]
            kept[page, h, slot] = False
            assert np.isnan(got[part + "s"][page, h, slot]), f"row {r} head {h}: {part} has a scale of {got[part + 's'][page, h, slot]}"
            assert (codes[page, h, slot] == 0).all()
        assert np.array_equal(codes[kept], want[part].transpose(axes)[kept])
        assert np.array_equal(got[part + "s"].view(np.uint32)[kept], want[part + "s"].view(np.uint32)[kept])


@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("part", ["k", "v"])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("new", [4, 40])
def test_rows_that_see_an_appended_no_number(ctx, q8, what, part, new):
    """Append, then attend: the rows before that token hold numbers, those that see it do not."""
    H, D = 2, 64
    b = Batch([(70, new)], H, D, 16, q8, seed=new).upload(ctx, new, 70)
    rng = np.random.default_rng(9)
    x = rng.standard_normal((new, 2 * H * D)).astype(np.float32)
    x[new // 2, (part == "v") * H * D + 7] = what  # head 0
    say(f"append of {what} in {part}, then attention: q8={q8} new={new}")
    _append(ctx, b, x)
    q = np.abs(queries(b, 2)) + np.float16(0.5)  # (a key of +inf scores +inf: NaN from inf - inf)
    got = run_attention(ctx, b, q, 2, 0.125).astype(np.float32)
    b.free()
    first, second = got[:, :2 * D], got[:, 2 * D:]
    assert np.isfinite(first[:new // 2]).all() and np.isfinite(second).all()
    spoiled = ~np.isfinite(first[new // 2:])
    assert spoiled.all() if q8 or part == "k" else (spoiled[:, 7::D].all() and spoiled.sum() == spoiled[:, 7::D].size)


def test_no_numbers_into_an_fp16_cache(ctx):
    """They stay what and where they are."""
    H, D = 2, 64
    b = Batch(LENS, H, D, 16, seed=2).upload(ctx, 19, 40)
    x = np.random.default_rng(2).standard_normal((b.M, 2 * H * D)).astype(np.float32)
    x[3, 5], x[9, H * D + 70], x[20, 64], x[30, H * D + 1] = np.nan, np.inf, -np.inf, np.nan
    say("fp16 append of no numbers")
    got = _append(ctx, b, x)
    b.free()
    want = x.astype(np.float16)
    for s, (n, new) in enumerate(b.lens):
        p, t = b.cells(s)
        for i in range(new):
            page, slot, r = p[n - new + i], t[n - new + i], b.row_start[s] + i
            assert np.array_equal(got["k"][page, :, slot].reshape(-1), want[r, :H * D], equal_nan=True)
            assert np.array_equal(got["v"][page, :, :, slot].reshape(-1), want[r, H * D:], equal_nan=True)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_smallest_scales_of_an_8_bit_cache(ctx, D):
    """Largest values just below 2^-100: codes and scale of 0. From 2^-100 on: codes up to 127."""
    H = 2
    b = Batch(LENS, H, D, 16, True, seed=D).upload(ctx, 19, 40)
    rng = np.random.default_rng(D)
    x = rng.uniform(-0.9, 0.9, (b.M, 2 * H, D))
    edge = np.nextafter(np.float32(2.0 ** -100), np.float32(0))
    x *= 2.0 ** -100
    x[:, :, D // 2] = np.where((np.arange(b.M) % 2 == 0)[:, None], edge, np.float32(-2.0 ** -100))
    say(f"smallest scales D={D}")
    got = _append(ctx, b, x.reshape(b.M, -1).astype(np.float32))
    b.free()
    for s, (n, new) in enumerate(b.lens):
        p, t = b.cells(s)
        for i in range(new):
            page, slot, r = p[n - new + i], t[n - new + i], b.row_start[s] + i
            for codes, scale, ref in ((got["k"][page, :, slot], got["ks"][page, :, slot], x[r, :H]),
                                      (got["v"][page, :, :, slot], got["vs"][page, :, slot], x[r, H:])):
                if r % 2 == 0:
                    assert (codes == 0).all() and (scale == 0).all()
                else:
                    assert (codes[:, D // 2] == -127).all() and (np.abs(scale * 127 / 2.0 ** -100 - 1) < 2.0 ** -22).all()
                    # half a step of the code, and its quotient's last bits
                    assert np.abs(codes * scale[:, None].astype(np.float64) - ref).max() <= scale.max() * (0.5 + 127 * 2.0 ** -22)


@pytest.mark.parametrize("q8", [False, True])
def test_many_sequences_without_hints(ctx, q8):
    """4096 sequences of 16 rows with max_new not known: each could have all 65536, and 2^24 workgroups of
    values would be more than a launch has."""
    S, D, rng = 4096, 64, np.random.default_rng(3)
    b = Batch([(16 + int(n), 16) for n in rng.integers(0, 3, S)], 1, D, 32, q8, seed=5).upload(ctx)
    x = rng.standard_normal((b.M, 2 * D)).astype(np.float32)
    say(f"{S} sequences without hints q8={q8}")
    got = _append(ctx, b, x)
    b.free()
    page = np.repeat(b.pages[:, 0], 16)
    slot = (b.kv_len[:, None] - 16 + np.arange(16)).reshape(-1)
    for codes, scale, ref in ((got["k"][page, 0, slot], "ks", x[:, :D]), (got["v"][page, 0, :, slot], "vs", x[:, D:])):
        if not q8:
            assert np.array_equal(codes, ref.astype(np.float16))
        else:
            s = got[scale][page, 0, slot].astype(np.float64)[:, None]
            assert (np.abs(codes * s - ref) <= s * (0.5 + 127 * 2.0 ** -22)).all()
