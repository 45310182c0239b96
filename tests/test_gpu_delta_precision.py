"""How many bits the delta rule keeps where a column's values or its state change their size: states that decay over the second
half of a prompt, small values after large ones, values of any size. The rule in 64 bits; errors are compared with the size that the
results have there, not with the largest that ever was. And what a workspace without the place for second halves gives."""
import ctypes as C

import numpy as np
import pytest

import qmm_hip
import state_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu


def run(ctx, news, x, rate, state, ws=True, hint=None, gamma=None, eps=1e-6):
    """One call on rows x = {q, k, v, a, b} ([rows][heads][..]; scale 1, no bias of the steps), states in place: (rows, states). ws:
    a workspace of its own; an int: smaller by so many bytes."""
    m, HK, DK = x["q"].shape
    HV, DV = x["v"].shape[1:]
    n = len(news)
    up = {i: ctx.upload(np.ascontiguousarray(y, np.float32)) for i, y in x.items()}
    up.update(starts=ctx.upload(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)), slots=ctx.upload(np.arange(n, dtype=np.int32)),
              rate=ctx.upload(np.asarray(rate, np.float32)), dt=ctx.upload(np.zeros(HV, np.float32)),
              out=ctx.upload(np.zeros((m, HV, DV), np.float32)), state=ctx.upload(np.asarray(state, np.float32)))
    if gamma is not None:
        up["gamma"] = ctx.upload(np.asarray(gamma, np.float32))
    at = {i: int(u) for i, u in up.items()}
    batch = qmm_hip.StateBatch(n, m, at["starts"], at["slots"], at["slots"], n, max(news) if hint is None else hint)
    args = qmm_hip.DeltaArgs(q=at["q"], k=at["k"], q_stride=HK * DK, k_stride=HK * DK, v=at["v"], v_stride=HV * DV, qk_heads=HK, v_heads=HV,
                             key_dim=DK, value_dim=DV, a=at["a"], b=at["b"], a_stride=HV, b_stride=HV, rate=at["rate"], dt_bias=at["dt"],
                             scale=1.0, qk_eps=eps, state=at["state"], gamma=at.get("gamma"), gamma_eps=0.0, out=at["out"],
                             out_stride=HV * DV)
    w = ctx.gated_delta_workspace(batch, args) if ws else None
    if w and ws is not True:
        w.free()
        h = C.c_void_p()
        ctx._call("qmm_attention_workspace_create", ctx._h, ctx.lib.qmm_gated_delta_workspace_bytes(ctx._h, C.byref(batch), C.byref(args)) - ws, C.byref(h))
        w = qmm_hip._Handle(ctx, h.value, "qmm_attention_workspace_destroy")
    ctx.gated_delta(batch, args, w)
    ctx.sync()
    got = ctx.d2h(up["out"], np.float32, (m, HV, DV)), ctx.d2h(up["state"], np.float32, state.shape)
    if w:
        w.free()
    for u in up.values():
        ctx.free(u)
    return got


def exact(news, x, rate, state, gamma=None, eps=1e-6):
    """The same in 64 bits; and what the state's columns' lengths were after every token [rows][heads][DV]."""
    x = {i: np.asarray(y, np.float32).astype(np.float64) for i, y in x.items()}
    of = x["v"].shape[1] // x["q"].shape[1]
    unit = lambda y: np.repeat(y / np.sqrt((y * y).sum(-1, keepdims=True) + np.float64(np.float32(eps))), of, 1)  # noqa: E731
    q, k = unit(x["q"]), unit(x["k"])
    decay = np.exp(np.asarray(rate, np.float32).astype(np.float64) * np.log1p(np.exp(x["a"])))
    beta = 1 / (1 + np.exp(-x["b"]))
    S, r = np.asarray(state, np.float32).astype(np.float64), 0
    out, size = np.zeros(x["v"].shape), np.zeros(x["v"].shape)
    for s, n in enumerate(news):
        for r in range(r, r + n):
            S[s] *= decay[r][:, None, None]
            S[s] += k[r][:, :, None] * (beta[r][:, None] * (x["v"][r] - (S[s] * k[r][:, :, None]).sum(1)))[:, None]
            out[r] = (S[s] * q[r][:, :, None]).sum(1)
            size[r] = np.sqrt((S[s] ** 2).sum(1))
        r += 1
    if gamma is not None:
        out = out / np.sqrt((out ** 2).mean(-1, keepdims=True)) * np.asarray(gamma, np.float32)
    return out, S, size


def rows(m, HK, of, DK, DV, seed):
    g = np.random.default_rng(seed)
    return {"q": g.standard_normal((m, HK, DK)), "k": g.standard_normal((m, HK, DK)), "v": g.standard_normal((m, HK * of, DV)),
            "a": g.standard_normal((m, HK * of)), "b": g.standard_normal((m, HK * of))}, g


def rms(x, axis=None):
    return np.sqrt(np.mean(np.square(x), axis))


def mean_error(n):
    """A bound of the rms error of n tokens' steps, relative to the state: a step has six operands (k twice, S, T, the values, D) that are
    2^-22 off or less, and sums in fp32, two more; roundings of either sign, so the steps' errors add as squares."""
    return 8 * 2.0 ** -22 * np.sqrt(n)


WAYS = {"halves": dict(), "walk": dict(beside=3), "one launch": dict(ws=False), "tokens": dict(hint=1)}


def on_way(ctx, way, news, x, rate, state, **kw):
    """The call on one of its ways. `beside`: short sequences that take the halves from the long one (there are then too many heads)."""
    how = dict(WAYS[way])
    n, m = how.pop("beside", 0), sum(news)
    if n:
        HV = x["v"].shape[1]
        n = 64 // HV + 1
        x = {i: np.concatenate([y, np.ones((n, *y.shape[1:]))]) for i, y in x.items()}
        state = np.concatenate([state, np.zeros((n, *state.shape[1:]))])
    got = run(ctx, news + [1] * n, x, rate, state, **how, **kw)
    return got[0][:m], got[1][:len(news)]


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("gamma", [False, True])
@pytest.mark.parametrize("lost", [10, 20, 25, 30])
@pytest.mark.parametrize("DK,DV", [(64, 128), (128, 128), (128, 64)])
def test_state_decays_over_the_second_half(ctx, DK, DV, lost, gamma, way):
    """A large state in the middle of a prompt, forgotten by e^-lost to its end, and next to nothing added: what is left of it keeps its
    bits, in rows and in the state."""
    say(f"delta precision: decays DK={DK} DV={DV} lost={lost} gamma={gamma} way={way}")
    n = 640
    x, g = rows(n, 1, 2, DK, DV, DK + lost)
    x["a"][:n // 2] = -40.0  # no decay
    x["a"][n // 2:] = 0.0
    x["v"][n // 2:] *= 1e-30
    x["b"] -= 3.0  # (small steps: the first state is there to the end)
    rate = np.full(2, -lost / (n / 2) / np.log(2.0))
    state = 300.0 * g.standard_normal((1, 2, DK, DV))
    w = g.uniform(0.5, 1.5, DV) if gamma else None
    out, after = on_way(ctx, way, [n], x, rate, state, gamma=w)
    ref, ref_after, _ = exact([n], x, rate, state, w)
    for part in (slice(0, n // 2), slice(n // 2, 500), slice(500, 600), slice(600, n)):
        off = rms((out[part] - ref[part]) / rms(ref[part], -1)[..., None])
        assert off <= mean_error(n), (part, off, mean_error(n))
    off = rms((after - ref_after) / rms(ref_after, (2, 3))[..., None, None])
    assert off <= mean_error(n), (off, mean_error(n))


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("size", [1e-15, 1e-20, 1e-25, 1e-28])
@pytest.mark.parametrize("D", [64, 128])
def test_values_of_any_size(ctx, D, size, way):
    """Values and states of one size, however small: as far as fp32 has all its bits for what they sum to, none are lost."""
    say(f"delta precision: size={size} D={D} way={way}")
    n = 600
    x, g = rows(n, 1, 2, D, D, D)
    x["v"] *= size
    state = size * g.standard_normal((1, 2, D, D))
    rate = np.array([-0.01, -1.0])
    out, after = on_way(ctx, way, [n], x, rate, state)
    ref, ref_after, _ = exact([n], x, rate, state)
    for h in range(2):
        assert rms(out[:, h] - ref[:, h]) <= mean_error(n) * rms(ref[:, h])
        assert rms(after[:, h] - ref_after[:, h]) <= mean_error(n) * rms(ref_after[:, h])


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("large,small", [(1e4, 1e-25), (6e4, 1e-20), (1e10, 1e-25)])
def test_values_change_their_size_at_once(ctx, large, small, way):
    """Values and a state of one size, all forgotten within a token, and then values of another: no infinity meets a zero. The token
    is the first of a group, so the state before the group is large, and its operands are never finer than 2^-39 of it: 2^-33 of what the
    state and the values before sum to, a token of the group (see state_ref.delta), which stays in the state as nothing decays
    afterwards. A group of zeros between leaves the next ones all their bits. (1e10 is more than the rows may hold: nothing but finite
    numbers is asked for there.)"""
    n, D, first = 576, 64, 288
    for zeros in (0, 32):
        say(f"delta precision: from {large} to {small} zeros={zeros} way={way}")
        x, g = rows(n, 1, 1, D, D, 7)
        x["v"][:first] *= large
        x["v"][first:] *= small
        x["v"][first - zeros:first] = 0.0
        x["a"][:] = -40.0
        x["a"][first - zeros] = 300.0  # e^-300 once
        state = large * g.standard_normal((1, 1, D, D))
        out, after = on_way(ctx, way, [n], x, np.array([-1.0]), state)
        ref, ref_after, _ = exact([n], x, np.array([-1.0]), state)
        assert np.isfinite(out).all() and np.isfinite(after).all()
        if large > 65520:
            continue
        assert rms(out[:first - zeros] - ref[:first - zeros]) <= mean_error(n) * rms(ref[:first - zeros])
        held = 0.0 if zeros else np.abs(x["v"][:first]).sum(0).max() + np.abs(state).sum(2).max()
        for part in (slice(first, first + 32), slice(first + 32, n)):
            assert rms(out[part] - ref[part]) <= mean_error(n) * rms(ref[part]) + 32 * 2.0 ** -33 * held, (zeros, part)
        assert rms(after - ref_after) <= mean_error(n) * rms(ref_after) + 32 * 2.0 ** -33 * held, zeros


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("large", [32, 256, 600])
@pytest.mark.parametrize("D", [64, 128])
def test_small_values_after_large_ones(ctx, D, large, way):
    """Nothing decays, but every value is written over within D tokens (unit vectors in turn as keys, steps of 1): once no large one is
    left, the small ones keep their bits. A row of the state is as its last writing left it."""
    say(f"delta precision: small after large D={D} large={large} way={way}")
    n = large + 5 * D + 61
    x, _ = rows(n, 1, 1, D, D, D + large)
    x["k"] = np.eye(D)[np.arange(n) % D][:, None]
    x["b"][:], x["a"][:] = 40.0, -40.0
    x["v"][:large] *= 6e4
    x["v"][large:] *= 1e-3
    state = np.zeros((1, 1, D, D))
    out, after = on_way(ctx, way, [n], x, np.full(1, -1.0), state, eps=1e-12)
    ref, ref_after, size = exact([n], x, np.full(1, -1.0), state, eps=1e-12)
    # a large value's own error, 2^-22 of it and more, goes as it is written over, and what that leaves the next time
    part = slice(large + 4 * D, n)
    off = rms(out[part] - ref[part]) / rms(ref[part])
    assert off <= mean_error(D), (off, mean_error(D))
    assert rms(after - ref_after) <= mean_error(D) * rms(ref_after)


@pytest.mark.parametrize("DK,DV", [(64, 64), (128, 128)])
def test_workspace_without_room_for_halves(ctx, DK, DV):
    """One that holds the groups still makes three launches of a long prompt: the bits of the walk in one, which short sequences
    beside it leave."""
    say(f"delta: workspace without halves D={DK},{DV}")
    n = 700
    x, g = rows(n, 1, 2, DK, DV, DK)
    state, rate = g.standard_normal((1, 2, DK, DV)), np.array([-0.1, -1.0])
    out, after = run(ctx, [n], x, rate, state, ws=1024)
    for a, b in zip((out, after), on_way(ctx, "walk", [n], x, rate, state)):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    for a, b in zip((out, after), on_way(ctx, "halves", [n], x, rate, state)):
        assert rms(a - b) <= 2 * mean_error(n) * rms(b)


@pytest.mark.parametrize("hint", [1, 8, 9, 40])
def test_a_sequence_follows_the_hint_and_not_its_neighbours(ctx, hint):
    """max_new decides how all of a call's sequences are computed; under the same one a sequence has the same bits alone."""
    say(f"delta: neighbours hint={hint}")
    news, D = [1, 0, 5, 8, 30, 64, 1], 64
    x, g = rows(sum(news), 1, 2, D, D, 11)
    state, rate = g.standard_normal((len(news), 2, D, D)), np.array([-0.1, -1.0])
    out, after = run(ctx, news, x, rate, state, ws=False, hint=hint)
    r = 0
    for i, n in enumerate(news):
        if n:
            alone, alone_after = run(ctx, [n], {k: y[r:r + n] for k, y in x.items()}, rate, state[i:i + 1], ws=False, hint=hint if hint < 9 or n > 8 else 0)
            if hint < 9 or n > 8:
                assert np.array_equal(alone.view(np.uint32), out[r:r + n].view(np.uint32))
                assert np.array_equal(alone_after.view(np.uint32), after[i:i + 1].view(np.uint32))
            else:  # (alone the host knows that the rows are few)
                assert rms(alone - out[r:r + n]) <= 2 * mean_error(n) * rms(alone)
        r += n


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("alike", [0.0, 0.9, 1.0])
@pytest.mark.parametrize("decay", [1e-6, 0.01, 1.0])
def test_mean_error_of_long_prompts(ctx, decay, alike, way):
    """The rms error of a long prompt's rows, also of its last ones, and of its state: a worst case for each token adds up to
    a third of the values there, a lost low part of one operand (2^-11) to a hundredth and less."""
    say(f"delta precision: mean error decay={decay} alike={alike} way={way}")
    n, D = 1600, 64
    x, g = rows(n, 1, 2, D, D, 5)
    x["k"] = alike * g.standard_normal(D) + (1 - alike) * x["k"]
    state, rate = g.standard_normal((1, 2, D, D)), np.array([-decay, -decay / 3])
    out, after = on_way(ctx, way, [n], x, rate, state)
    ref, ref_after, _ = exact([n], x, rate, state)
    for h in range(2):
        for part in (slice(0, 400), slice(400, 1200), slice(1200, 1590), slice(1590, n)):
            off = rms(out[part, h] - ref[part, h]) / rms(ref[part, h])
            assert off <= mean_error(n), (h, part, off)
        assert rms(after[0, h] - ref_after[0, h]) <= mean_error(n) * rms(ref_after[0, h]), h
