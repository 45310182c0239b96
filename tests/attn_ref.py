"""Plain attention and cache append in 64 bits, batches with poisoned cells, and
the bounds the kernels' outputs are held to."""
import ctypes as C

import numpy as np

import qmm_hip

F16_HALF = 2.0 ** -11   # half a step of fp16, relative; below 2^-14 half a step is 2^-25
F32_HALF = 2.0 ** -24
NO_NUMBER = np.array([0x7e00, 0x7c00, 0xfc00, 0xfdff], np.uint16)  # NaN, inf, -inf, -NaN


class Batch:
    """Sequences of (length, new rows) over shuffled pages; the rest of the cache holds no numbers."""

    def __init__(self, lens, heads, dim, page, q8=False, seed=0, extra_rows=0, spare_pages=2, spread=1.0, max_pages=None):
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.H, self.D, self.P, self.q8 = list(lens), heads, dim, page, q8
        self.S = len(self.lens)
        held = [-(-n // page) for n, _ in self.lens]
        self.n_pages = sum(held) + spare_pages
        self.max_pages = max_pages or max(max(held, default=1), 1)
        order = rng.permutation(self.n_pages).astype(np.int32)
        # entries past a sequence's end: valid ids of other pages, or none
        self.pages = rng.choice(np.array([-1, 0, self.n_pages - 1, self.n_pages, 2 ** 31 - 1], np.int64),
                                (self.S, self.max_pages)).astype(np.int32)
        at = 0
        for s, h in enumerate(held):
            self.pages[s, :h] = order[at:at + h]
            at += h
        self.row_start = np.concatenate([[0], np.cumsum([n for _, n in self.lens])]).astype(np.int32)
        self.kv_len = np.array([n for n, _ in self.lens], np.int32)
        self.held_rows = int(self.row_start[-1])
        self.M = self.held_rows + extra_rows
        # per sequence [heads, length, dim]
        shape = (self.n_pages, heads, page, dim)
        if q8:
            self.k = rng.integers(-127, 128, shape).astype(np.int8)
            self.v = rng.integers(-127, 128, (self.n_pages, heads, dim, page)).astype(np.int8)
            self.ks = rng.uniform(0.3, 1.7, shape[:3]).astype(np.float32) / np.float32(73) * np.float32(spread)
            self.vs = (rng.uniform(0.3, 1.7, shape[:3]) / 73).astype(np.float32)
        else:
            self.k = (rng.standard_normal(shape) * spread).astype(np.float16)
            self.v = rng.standard_normal((self.n_pages, heads, dim, page)).astype(np.float16)
            self.ks = self.vs = None
        self.poison()

    def cells(self, s):
        """(pages, slots) of the sequence's tokens."""
        t = np.arange(self.lens[s][0])
        return self.pages[s, t // self.P], t % self.P

    def poison(self):
        """No numbers in every cell that no sequence holds."""
        free = np.ones((self.n_pages, self.P), bool)
        for s in range(self.S):
            free[self.cells(s)] = False
        p, t = np.nonzero(free)
        if self.q8:
            bad = np.array([np.nan, np.inf, -np.inf, 3e38], np.float32)
            self.ks[p, :, t] = self.rng.choice(bad, (len(p), self.H))
            self.vs[p, :, t] = self.rng.choice(bad, (len(p), self.H))
        else:
            self.k.view(np.uint16)[p, :, t] = self.rng.choice(NO_NUMBER, (len(p), self.H, self.D))
            self.v.view(np.uint16)[p, :, :, t] = self.rng.choice(NO_NUMBER, (len(p), self.H, self.D))

    def dense(self, s):
        """The sequence's keys and values in 64 bits: [heads, length, dim]."""
        p, t = self.cells(s)
        k, v = self.k[p, :, t].astype(np.float64), self.v[p, :, :, t].astype(np.float64)
        if self.q8:
            k, v = k * self.ks[p, :, t].astype(np.float64)[..., None], v * self.vs[p, :, t].astype(np.float64)[..., None]
        return k.transpose(1, 0, 2), v.transpose(1, 0, 2)

    def upload(self, ctx, max_new=0, max_kv=0):
        self.ctx = ctx
        self.bufs = {n: ctx.upload(getattr(self, n)) for n in ("k", "v", "row_start", "kv_len", "pages")}
        if self.q8:
            self.bufs["ks"], self.bufs["vs"] = ctx.upload(self.ks), ctx.upload(self.vs)
        a = {n: int(b) for n, b in self.bufs.items()}
        self.batch = qmm_hip.KvBatch(self.S, self.M, a["row_start"], a["kv_len"], a["pages"], self.max_pages, max_new, max_kv)
        self.cache = qmm_hip.KvCache(qmm_hip.KV_Q8 if self.q8 else qmm_hip.KV_F16, self.P, self.n_pages, self.H, self.D,
                                     a["k"], a["v"], a.get("ks"), a.get("vs"))
        return self

    def free(self):
        for b in self.bufs.values():
            self.ctx.free(b)


def attend(b, q, group, scale, window=0, sinks=0):
    """(rows, bound) in 64 bits, [M, heads * group * dim] of the rows the sequences hold.

    The kernel's roundings, to the first order: the scores are fp32 sums (of D products, in any order, of
    size at most sum|q k| scale), their exponentials off by a few units, the sums of weights and products
    fp32; a weight is rounded to fp16 (half a step, 2^-25 where it is below 2^-14 of the row's largest),
    and the output once more."""
    D, G, HQ = b.D, group, b.H * group
    out, tol = np.zeros((b.M, HQ * D)), np.zeros((b.M, HQ * D))
    for s, (n, new) in enumerate(b.lens):
        if not new:
            continue
        k, v = b.dense(s)
        for i in range(new):
            p = n - new + i
            if p < 0:
                continue
            j = np.arange(p + 1)
            j = j[(j > p - window) | (j < sinks)] if window else j
            r = b.row_start[s] + i
            for h in range(HQ):
                qq = q[r, h * D:(h + 1) * D].astype(np.float64)
                kk, vv = k[h // G][j], v[h // G][j]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = kk @ qq * scale
                    w = np.exp(x - x.max())
                    top = 1 / w.sum()
                    w *= top
                    o = w @ vv
                    size = w @ np.abs(vv)
                    e_score = 2 * (D + 8) * F32_HALF * (np.abs(kk) @ np.abs(qq)).max() * scale
                    e = e_score + F16_HALF + (len(j) / 8 + 32) * F32_HALF
                    out[r, h * D:(h + 1) * D] = o
                    small = len(j) * 2.0 ** -25 * top * np.where(np.isfinite(vv), np.abs(vv), 0).max()  # (others' rows are no numbers)
                    tol[r, h * D:(h + 1) * D] = 1.01 * (F16_HALF * (np.abs(o) + 2.0 ** -14) + e * size + small)
    return out, tol


def run_attention(ctx, b, q, group, scale, window=0, sinks=0, out_type=qmm_hip.TYPE_F16, workspace=True, pad=0,
                  sentinel=7.0, repeat=1, ws=None):
    """The library's outputs [M, heads * group * dim], rows and columns past them checked to be untouched."""
    width = b.H * group * b.D
    qb = ctx.upload(np.concatenate([q, np.full((b.M, 8 * pad), np.nan, np.float16)], 1) if pad else q)
    dt = np.float16 if out_type == qmm_hip.TYPE_F16 else np.float32
    ob = ctx.upload(np.full((b.M, width + 4 * pad), sentinel, dt))
    a = qmm_hip.AttentionArgs(int(qb), width + 8 * pad, b.H * group, scale, window, sinks, int(ob), out_type, width + 4 * pad)
    ws = ws or (ctx.attention_workspace(b.batch, b.cache, a) if workspace else None)
    for _ in range(repeat):
        ctx.paged_attention(b.batch, b.cache, a, ws)
    ctx.sync()
    o = ctx.d2h(ob, dt, (b.M, width + 4 * pad))
    ctx.free(qb)
    ctx.free(ob)
    assert (o[:, width:] == sentinel).all(), "columns past the rows were written"
    assert (o[b.held_rows:] == sentinel).all(), "rows behind the last sequence were written"
    return o[:, :width]


def check_rows(got, ref, tol, rows):
    """Elementwise |got - ref| <= tol; what is no number in one is the same in the other."""
    got, ref, tol = got[:rows].astype(np.float64), ref[:rows], tol[:rows]
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), "NaN at other places"
    assert np.array_equal(got[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)]), "other infinities"
    d = np.abs(got[fine] - ref[fine]) - tol[fine]
    assert not d.size or d.max() <= 0, f"{np.count_nonzero(d > 0)} of {d.size} values off, by up to {d.max():.3g} over their bound"


def queries(b, group, seed=1, spread=2.0):
    return (np.random.default_rng(seed).standard_normal((b.M, b.H * group * b.D)) * spread).astype(np.float16)


# ------------------------------------------------------------------ append
def turned(x, gamma, eps, pos, rot, style, freq, axis, scale):
    """Head norm and rotation of one row's heads [heads, dim] in 64 bits, and the bound of its fp32 arithmetic."""
    D = x.shape[1]
    x = x.astype(np.float64)
    if gamma is not None:
        x = x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * gamma.astype(np.float64)
    # norm: a sum of D squares, a root, a quotient and two products
    err = (D / 2 + 16) * F32_HALF * np.abs(x) if gamma is not None else np.zeros_like(x)
    if rot:
        t = np.array([float(pos[a]) for a in axis]) * freq
        one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if style == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        a, b = x[:, one].copy(), x[:, two].copy()
        # angle off by half a step of a float in [-1/2, 1/2] turns (2^-25 * 2 pi), sine and cosine by a few
        # steps, four products and sums
        e = (abs(scale) * (2.0 ** -22 + 16 * F32_HALF)) * (np.abs(a) + np.abs(b))
        ea = abs(scale) * (err[:, one] + err[:, two])
        x[:, one], x[:, two] = (a * np.cos(t) - b * np.sin(t)) * scale, (b * np.cos(t) + a * np.sin(t)) * scale
        err[:, one], err[:, two] = e + ea, e + ea
    return x, err


def host(x):
    return C.c_void_p(x.ctypes.data)
