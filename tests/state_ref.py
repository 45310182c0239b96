"""The short convolution, the gated delta rule and a beam search's selection in 64
bits, batches over pools whose unused slots and rows hold no numbers, and the
bounds the kernels' outputs are held to."""
import numpy as np

import qmm_hip

U = 2.0 ** -24  # half a step of fp32, relative
NO_NUMBERS = np.array([np.nan, np.inf, -np.inf, 3e38], np.float32)


def _sigmoid(x):
    return np.where(x > 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))


class States:
    """Sequences of `news` new rows. `slots`: per sequence (slot read, slot written), -1: none; default: a slot of its own
    read and another written. Slots nobody reads and rows nobody holds hold no numbers."""

    def __init__(self, news, slots=None, seed=0, extra_rows=0, spare=2, gap=0):
        self.rng = np.random.default_rng(seed)
        self.news, self.S, self.gap = list(news), len(news), gap
        if slots is None:
            order = self.rng.permutation(2 * self.S + spare)
            slots = [(order[i], order[self.S + i]) for i in range(self.S)]
            self.n_slots = 2 * self.S + spare
        else:
            self.n_slots = max([0] + [x for p in slots for x in p]) + 1 + spare
        self.slot_in = np.array([p[0] for p in slots], np.int32)
        self.slot_out = np.array([p[1] for p in slots], np.int32)
        self.row_start = np.concatenate([[0], np.cumsum(self.news)]).astype(np.int32)
        self.held = int(self.row_start[-1])
        self.M = self.held + extra_rows

    def rows(self, width, spread=1.0, gap=None):
        """Random rows [M][width + gap]; no numbers in the gap and behind the last sequence."""
        gap = self.gap if gap is None else gap
        x = self.rng.choice(NO_NUMBERS, (self.M, width + gap))
        x[:self.held, :width] = (self.rng.standard_normal((self.held, width)) * spread).astype(np.float32)
        return x

    def pool(self, *shape, spread=1.0):
        """A pool of slots, those that are read with numbers."""
        p = self.rng.choice(NO_NUMBERS, (self.n_slots, *shape))
        for i in self.slot_in:
            if 0 <= i < self.n_slots:
                p[i] = (self.rng.standard_normal(shape) * spread).astype(np.float32)
        return p

    def upload(self, ctx, hints=True):
        """hints: the longest sequence's new rows; False: none; a number: that."""
        self.bufs = [ctx.upload(a) for a in (self.row_start, self.slot_in, self.slot_out)]
        self.batch = qmm_hip.StateBatch(self.S, self.M, *(int(b) for b in self.bufs), self.n_slots,
                                        max([0] + self.news) if hints is True else int(hints))
        return self

    def sequences(self):
        """(number, first row, new rows, slot read or -1, slot written or -1)"""
        for s, n in enumerate(self.news):
            ok = [int(x) if 0 <= x < self.n_slots else -1 for x in (self.slot_in[s], self.slot_out[s])]
            yield s, int(self.row_start[s]), n, *ok


# ------------------------------------------------------------- convolution
def conv(b, x, w, bias, pool, silu):
    """(rows, bound, pool after) of the short convolution; x [M][>= channels], w [channels][width]."""
    Ch, W = w.shape
    out, tol, after = np.zeros((b.M, Ch)), np.zeros((b.M, Ch)), pool.copy()
    for _, r0, n, i, o in b.sequences():
        past = pool[i].astype(np.float64) if i >= 0 else np.zeros((W - 1, Ch))
        seq = np.concatenate([past, x[r0:r0 + n, :Ch].astype(np.float64)])
        for t in range(n):
            terms = seq[t:t + W] * w.T.astype(np.float64)
            y = terms.sum(0) + (0 if bias is None else bias.astype(np.float64))
            e = (W + 1) * U * (np.abs(terms).sum(0) + (0 if bias is None else np.abs(bias)))  # W products added one by one
            if silu:  # |silu'| <= 1.1; an exponential (of a product, 2^-24 of |y| off), a sum, a reciprocal, a product
                e = 1.1 * e + np.abs(y * _sigmoid(y)) * (8 + np.abs(y)) * U
                y = y * _sigmoid(y)
            out[r0 + t], tol[r0 + t] = y, 1.01 * e + 1e-37
        if o >= 0:
            after[o] = seq[n:].astype(np.float32)
    return out, tol, after


# -------------------------------------------------------------- delta rule
def delta(b, q, k, v, a, bt, rate, dt, scale, eps, pool, z=None, gamma=None, gamma_eps=0.0, of=1):
    """(rows, bound, pool after, its bound) of the gated delta rule, token by token. q, k: [M][qk heads][DK]; v: [M][heads][DV].

    The bound: a step is S <- e^g (S - beta k (S'k)') + beta k v', which makes no column longer than it was and
    adds |v| at most, so the errors of the steps add up, each shrunk by the decays after it. One step's error in a
    column is at most C 2^-24 (|S column| + |v|): sums of DK products (DK), unit vectors (DK / 4 of a sum
    of squares, a root, two products), a decay exp(g) that is (|g| + 8) 2^-24 off, operands of 22 bits (16
    in units of 2^-24), and a few products; C = 1.5 DK + 64 + |g|. An output adds one more such sum.

    Operands of groups of 32 tokens have a smallest step, too. A column is scaled so that b, what its state's values and the
    group's sum to in size, is 2^14 or more, and the low part of a pair is a multiple of 2^-24: at most 2^-39 b off; matrices
    of values up to 1 are at most 2^-39 off. For a token, 2^-39 b of its value, sqrt(DK) 2^-39 b of k.S and
    2^-39 (the sum of 32 values, each at most b) of T's row are another value for the rule, whose effect does not grow;
    the state's own update takes factors 2^4 smaller, 2^-35 b. Together less than 2^-33 b a token. An output adds sqrt(DK) 2^-39 b of q.S,
    and P's row like T's and the 32 values that it meets: less than 2^-32 b. (Columns below 2^-46 count as that.) It
    shows only in values that are 2^-16 times smaller than others of their column and group."""
    M, HV, DV = v.shape
    DK = q.shape[2]
    out, tol = np.zeros((M, HV, DV)), np.zeros((M, HV, DV))
    after, after_tol = pool.astype(np.float64), np.zeros(pool.shape)
    unit = lambda x: x / np.sqrt((x * x).sum(-1, keepdims=True) + eps)  # noqa: E731
    for _, r0, n, i, o in b.sequences():
        S = pool[i].astype(np.float64) if i >= 0 else np.zeros((HV, DK, DV))
        err, held = np.zeros((HV, DV)), np.abs(S).sum(1)
        for r in range(r0, r0 + n):
            if (r - r0) % 32 == 0:
                group = np.abs(v[r:min(r + 32, r0 + n)].astype(np.float64)).sum(0)
                held = np.maximum(held + group, 2.0 ** -46)  # (more than b: without decays)
            kk, qq = (np.repeat(unit(x[r].astype(np.float64)), of, 0) for x in (k, q))
            x = a[r].astype(np.float64) + dt
            g = np.minimum(rate.astype(np.float64) * (np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))), 0)
            beta, decay = _sigmoid(bt[r].astype(np.float64)), np.exp(g)
            C = (1.5 * DK + 64 + np.minimum(-g, 100))[:, None] * U
            size = np.linalg.norm(S, axis=1) + np.abs(v[r])
            S = S * decay[:, None, None]
            d = beta[:, None] * (v[r] - np.einsum("hkv,hk->hv", S, kk))
            S = S + kk[:, :, None] * d[:, None, :]
            err = err * decay[:, None] + C * size + 2.0 ** -33 * held
            y = np.einsum("hkv,hk->hv", S, qq) * scale
            e = scale * (err + C * np.linalg.norm(S, axis=1) + 2.0 ** -32 * held)
            if gamma is not None:
                rms = np.sqrt((y * y).mean(1, keepdims=True) + gamma_eps)
                e = (e + np.abs(y) * np.sqrt((e * e).mean(1, keepdims=True)) / rms) / rms * np.abs(gamma)
                y = y / rms * gamma
                e = e + (DV / 4 + 16) * U * np.abs(y)
            if z is not None:
                zz = z[r].reshape(HV, DV).astype(np.float64)
                f = zz * _sigmoid(zz)
                y, e = y * f, e * np.abs(f) + (10 + np.abs(zz)) * U * np.abs(y * f)
            out[r], tol[r] = y, 1.01 * e + 1e-37
        if o >= 0:
            after[o], after_tol[o] = S, np.broadcast_to(1.01 * err[:, None, :] + 1e-37, S.shape)
    return out, tol, after, after_tol


def within(got, ref, tol, what):
    """Elementwise |got - ref| <= tol; the same bits of what is no number, or untouched (tol 0)."""
    got, ref = got.astype(np.float64), ref.astype(np.float64)
    with np.errstate(invalid="ignore"):
        off = ~((np.abs(got - ref) <= tol) | (got == ref) | (np.isnan(got) & np.isnan(ref)))
    assert not off.any(), f"{what}: {off.sum()} of {off.size} values past their bound, first at {np.argwhere(off)[0].tolist()}: " \
                          f"{got[off][0]!r}, not {ref[off][0]!r} +- {np.broadcast_to(tol, off.shape)[off][0]:.3g}"


# -------------------------------------------------------------------- beams
def select(logits, score, ended, end_token, n_keep):
    """One item's selection in 64 bits: (token, parent, total, certain). Not certain: a candidate of another beam is nearer than the
    sums of exponentials in fp32 allow to tell (40 roundings of 2^-24 each), so the two may change places."""
    B, V = logits.shape
    x = np.where(logits < np.inf, logits, -np.inf).astype(np.float32) + np.float32(0)
    score = np.where(score < np.inf, score, -np.inf).astype(np.float64)
    found = []
    for b in range(B):
        if ended is not None and ended[b] and score[b] > -np.inf:
            order = np.concatenate([[end_token], np.delete(np.arange(min(V, n_keep + 1)), end_token) if end_token <= n_keep else
                                    np.arange(min(V, n_keep + 1))])[:min(n_keep, V)]
            total = np.where(np.arange(len(order)) == 0, score[b], -np.inf)
        elif score[b] == -np.inf or x[b].max() == -np.inf or (ended is not None and ended[b]):
            order = np.arange(min(V, n_keep))
            total = np.full(len(order), -np.inf)
        else:
            order = np.argsort(-x[b].astype(np.float64), kind="stable")[:n_keep]
            top = np.float64(x[b].max())
            lse = top + np.log(np.exp(x[b].astype(np.float64) - top).sum())
            total = score[b] + (x[b][order].astype(np.float64) - lse)
        found += [(-t, b, i, int(j)) for i, (j, t) in enumerate(zip(order, total))]
    found.sort()
    near = 40 * U
    kept = found[:n_keep]
    certain = [not any(o[1] != c[1] and np.isfinite(o[0]) and np.isfinite(c[0]) and abs(o[0] - c[0]) < near and o[0] != c[0]
                       for o in found[max(0, i - 3):i + 4]) for i, c in enumerate(kept)]
    return (np.array([c[3] for c in kept]), np.array([c[1] for c in kept]), -np.array([c[0] for c in kept]), np.array(certain))
