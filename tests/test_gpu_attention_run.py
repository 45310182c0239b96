"""The attention of a layer as it is used: projections, append, attention and
output projection one after the other; captured and replayed; on other streams
and two at once; caches and batches at their largest; refusals of the C ABI."""
import ctypes as C

import numpy as np
import pytest

import qmm_hip
import synth
from attn_ref import Batch, attend, check_rows, queries, run_attention, turned
from gpu_util import say
from oracle import TYPE_Q4_K

pytestmark = pytest.mark.gpu


class Layer:
    """One layer's attention over a cache of its own: weights, buffers, and its calls in order."""

    def __init__(self, ctx, n_seqs, rows, q8, H=2, G=4, D=64, P=16, pages=24, window=0, hints=(0, 0), seed=0):
        self.ctx, self.S, self.rows, self.H, self.HQ, self.D, self.P, self.q8 = ctx, n_seqs, rows, H, H * G, D, P, q8
        self.window, self.seed, self.hints = window, seed, hints
        self.K = K = self.HQ * D  # hidden size
        self.width = (self.HQ + 2 * H) * D
        self.bufs = []
        self.wq = [self._keep(ctx.weight_upload(synth.weights(TYPE_Q4_K, n * D, K, seed=seed + i), TYPE_Q4_K, n * D, K))
                   for i, n in enumerate((self.HQ, H, H))]
        self.wo = self._keep(ctx.weight_upload(synth.weights(TYPE_Q4_K, K, K, seed=seed + 5), TYPE_Q4_K, K, K))
        rng = np.random.default_rng(seed)
        self.gamma = rng.uniform(0.5, 1.5, (2, D)).astype(np.float32)
        self.x, self.proj, self.q = (self._new((rows, n), t) for n, t in ((K, np.float32), (self.width, np.float32), (K, np.float16)))
        self.att, self.y = (self._new((rows, K), np.float32) for _ in range(2))
        self.n_pages = n_seqs * pages
        self.ids = rng.permutation(self.n_pages).reshape(n_seqs, pages).astype(np.int32)
        one, cell = (np.int8 if q8 else np.float16), (self.n_pages, H, P, D)
        self.k, self.v = self._new(cell, one), self._new((self.n_pages, H, D, P), one)
        self.ks, self.vs = (self._new(cell[:3], np.float32) if q8 else None for _ in range(2))
        self.row_start, self.kv_len = self._new(n_seqs + 1, np.int32), self._new(n_seqs, np.int32)
        self.page_ids, self.g = self._put(self.ids), [self._put(g) for g in self.gamma]
        self.rope = ctx.rope(D, "half", 1e4)
        self.cache = qmm_hip.KvCache(qmm_hip.KV_Q8 if q8 else qmm_hip.KV_F16, P, self.n_pages, H, D, int(self.k[0]), int(self.v[0]),
                                     *(int(b[0]) if b else None for b in (self.ks, self.vs)))
        self.args = qmm_hip.AttentionArgs(int(self.q[0]), K, self.HQ, D ** -0.5, window, 2 if window else 0, int(self.att[0]),
                                          qmm_hip.TYPE_F32, K)
        self.ws = ctx.attention_workspace(self.batch(rows), self.cache, self.args)

    def _keep(self, b):
        self.bufs.append(b)
        return b

    def _put(self, a):
        return self._keep(self.ctx.upload(np.ascontiguousarray(a)))

    def _new(self, shape, dtype):
        return self._put(np.zeros(shape, dtype)), shape, dtype

    def get(self, what):
        return self.ctx.d2h(what[0], what[2], what[1] if isinstance(what[1], tuple) else (what[1],))

    def batch(self, m):
        return qmm_hip.KvBatch(self.S, m, int(self.row_start[0]), int(self.kv_len[0]), int(self.page_ids), self.ids.shape[1], *self.hints)

    def set(self, x, lens):
        """The next step's inputs: rows, and (length, new rows) of each sequence."""
        self.ctx.h2d(self.x[0], x)
        self.ctx.h2d(self.row_start[0], np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32))
        self.ctx.h2d(self.kv_len[0], np.array([n for n, _ in lens], np.int32))

    def attention(self, m, args=None):
        self.ctx.paged_attention(self.batch(m), self.cache, args or self.args, self.ws)

    def append(self, m):
        D, a = self.D, int(self.proj[0])
        self.ctx.kv_append(self.batch(m), self.cache, qmm_hip.KvRows(
            q=a, q_stride=self.width, q_heads=self.HQ, k=a + 4 * self.HQ * D, k_stride=self.width, v=a + 4 * (self.HQ + self.H) * D,
            v_stride=self.width, q_gamma=int(self.g[0]), k_gamma=int(self.g[1]), eps=1e-6, rope=self.rope.handle,
            q_out=int(self.q[0]), q_out_stride=self.K))

    def project(self, m):
        at = int(self.proj[0])
        tasks = []
        for w, n in zip(self.wq, (self.HQ, self.H, self.H)):
            tasks.append(qmm_hip.MatrixTask(w, TYPE_Q4_K, n * self.D, self.K, at, self.width))
            at += 4 * n * self.D
        self.ctx.gemm_multi_dispatch(self.x[0], m, self.K, tasks)

    def output(self, m):
        self.ctx.gemm_multi_dispatch(self.att[0], m, self.K, [qmm_hip.MatrixTask(self.wo, TYPE_Q4_K, self.K, self.K, self.y[0])])

    def step(self, m):
        self.project(m)
        self.append(m)
        self.attention(m)
        self.output(m)

    def free(self):
        self.ws.free()
        self.rope.free()
        for b in self.bufs:
            self.ctx.free(b)


class View(Batch):
    """A layer's cache as the device holds it, for the plain attention."""

    def __init__(self, layer, lens):
        self.lens, self.H, self.D, self.P, self.q8, self.S = lens, layer.H, layer.D, layer.P, layer.q8, layer.S
        self.pages = layer.ids
        self.row_start = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32)
        self.held_rows = self.M = int(self.row_start[-1])
        self.k, self.v = layer.get(layer.k), layer.get(layer.v)
        if self.q8:
            self.ks, self.vs = layer.get(layer.ks), layer.get(layer.vs)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("window", [0, 24])
def test_prompt_then_single_tokens(ctx, q8, window):
    """A ragged prompt and three decode steps, each step's four calls with no wait between them; every
    stage against plain arithmetic on what the stage before it left."""
    layer = Layer(ctx, 3, 140, q8, window=window, seed=31)
    lens = [(70, 70), (5, 5), (61, 61)]
    for it in range(4):
        m = sum(n for _, n in lens)
        say(f"layer step {it} lens={lens} q8={q8} window={window}")
        layer.set(synth.activations(m, layer.K, seed=60 + it), lens)
        layer.step(m)
        ctx.sync()
        proj, q = layer.get(layer.proj)[:m], layer.get(layer.q)[:m]
        view = View(layer, lens)
        # the append: its queries, and the new tokens in the cache
        freq, r = 1e4 ** (-2.0 * np.arange(layer.D // 2) / layer.D), 0
        for s, (n, new) in enumerate(lens):
            k, v = view.dense(s)
            for i in range(new):
                parts = np.split(proj[r].reshape(-1, layer.D), [layer.HQ, layer.HQ + layer.H])
                rot = [layer.D, "half", freq, [0] * (layer.D // 2), 1.0]
                (rq, eq), (rk, ek) = (turned(p, g, 1e-6, [n - new + i], *rot) for p, g in zip(parts, layer.gamma))
                assert (np.abs(q[r].reshape(rq.shape) - rq) <= 2.0 ** -11 * (np.abs(rq) + 2.0 ** -14) + 1.01 * eq).all()
                for got, ref, err in ((k, rk, ek), (v, parts[2].astype(np.float64), 0 * ek)):
                    half = np.abs(ref).max(1, keepdims=True) / 127 * (0.5 + 127 * 2.0 ** -22) if q8 else 2.0 ** -11 * (np.abs(ref) + 2.0 ** -14)
                    assert (np.abs(got[:, n - new + i] - ref) <= half + 2.02 * err.max(1, keepdims=True) + 2.0 ** -22 * np.abs(ref)).all()
                r += 1
        ref, tol = attend(view, q, layer.HQ // layer.H, layer.D ** -0.5, window, 2 if window else 0)
        att = layer.get(layer.att)[:m]
        check_rows(att, ref, tol, m)
        # the output projection: the same bits as a call of its own on those rows
        y = layer.get(layer.y)[:m]
        ctx.h2d(layer.att[0], att)
        layer.output(m)
        ctx.sync()
        assert np.array_equal(y, layer.get(layer.y)[:m])
        lens = [(n + 1, 1) for n, _ in lens]
    layer.free()


@pytest.mark.parametrize("q8", [False, True])
def test_captured_steps(q8):
    """Append and attention of one token per sequence captured once, and replayed over growing lengths
    (other page counts than at the capture) with eager work between: the eager calls' bits each time."""
    with qmm_hip.Context(0) as c, qmm_hip.Context(0) as e:
        mine, other = (Layer(x, 4, 4, q8, P=64, pages=40, hints=(1, 2560), seed=33) for x in (c, e))
        start = [60, 700, 1, 2200]
        for layer in (mine, other):  # a past of values that are not all zeros
            for name in ("k", "v"):
                b = getattr(layer, name)
                rng = np.random.default_rng(7)
                layer.ctx.h2d(b[0], rng.integers(-100, 100, b[1]).astype(np.int8) if q8 else rng.standard_normal(b[1]).astype(np.float16))
            for b in (layer.ks, layer.vs) if q8 else ():
                layer.ctx.h2d(b[0], np.full(b[1], 0.01, np.float32))
        mine.set(synth.activations(4, mine.K, seed=1), [(n, 1) for n in start])
        mine.project(4)
        c.sync()
        c.graph_begin()
        mine.append(4)
        mine.attention(4)
        g = c.graph_end()
        for rep in range(4):
            lens = [(n + rep * 37, 1) for n in start]
            say(f"captured step {rep} lens={lens} q8={q8}")
            x = synth.activations(4, mine.K, seed=70 + rep)
            for layer in (mine, other):
                layer.set(x, lens)
                layer.project(4)
            c.h2d(mine.att[0], np.full(mine.att[1], np.nan, np.float32))
            c.sync()
            c.graph_launch(g)
            c.sync()
            other.append(4)
            other.attention(4)
            e.sync()
            for name in ("q", "k", "v", "att") + (("ks", "vs") if q8 else ()):
                assert np.array_equal(mine.get(getattr(mine, name)).view(np.uint8), other.get(getattr(other, name)).view(np.uint8)), (rep, name)
            mine.output(4)  # eager work of the same context
            c.sync()
        c.graph_destroy(g)
        mine.free()
        other.free()


def test_two_graphs_share_a_workspace():
    """In stream order one workspace serves both: nothing is kept in it between calls."""
    with qmm_hip.Context(0) as c:
        layer = Layer(c, 2, 2, False, P=64, pages=40, hints=(1, 2560), seed=35)
        rng = np.random.default_rng(8)
        for b in (layer.k, layer.v):
            c.h2d(b[0], rng.standard_normal(b[1]).astype(np.float16))
        c.h2d(layer.q[0], rng.standard_normal(layer.q[1]).astype(np.float16))
        layer.set(np.zeros(layer.x[1], np.float32), [(2500, 1), (1900, 1)])
        out2 = layer._new(layer.att[1], np.float32)
        a = layer.args
        wide = qmm_hip.AttentionArgs(a.q, a.q_stride, a.q_heads, a.scale, 900, 3, int(out2[0]), a.out_type, a.out_stride)
        layer.attention(2)
        layer.attention(2, wide)
        c.sync()
        want = layer.get(layer.att), layer.get(out2)
        graphs = []
        for args in (a, wide):
            c.graph_begin()
            layer.attention(2, args)
            graphs.append(c.graph_end())
        for rep in range(3):
            say(f"two graphs, one workspace, {rep}")
            for b in (layer.att, out2):
                c.h2d(b[0], np.full(b[1], np.nan, np.float32))
            for g in graphs if rep % 2 else graphs[::-1]:
                c.graph_launch(g)
            c.sync()
            assert np.array_equal(layer.get(layer.att), want[0]) and np.array_equal(layer.get(out2), want[1]), rep
        for g in graphs:
            c.graph_destroy(g)
        layer.free()


def test_what_a_graph_uses_outlives_its_handle():
    """A workspace and a rotation destroyed while a graph that used them lives: the replays go on."""
    with qmm_hip.Context(0) as c:
        layer = Layer(c, 2, 2, False, P=64, pages=40, hints=(1, 2560), seed=37)
        rng = np.random.default_rng(9)
        for b in (layer.k, layer.v):
            c.h2d(b[0], rng.standard_normal(b[1]).astype(np.float16))
        layer.set(synth.activations(2, layer.K, seed=3), [(2501, 1), (900, 1)])
        layer.project(2)
        layer.append(2)
        layer.attention(2)
        c.sync()
        want = layer.get(layer.att), layer.get(layer.k)
        say("handles destroyed under a living graph")
        c.graph_begin()
        h = C.c_void_p()
        assert c.status_of("qmm_attention_workspace_create", 4096, C.byref(h)) == qmm_hip.QMM_EINVAL
        with pytest.raises(qmm_hip.QmmError):
            c.rope(64)
        layer.append(2)
        layer.attention(2)
        g = c.graph_end()
        nbytes = c.lib.qmm_attention_workspace_bytes(c._h, C.byref(layer.batch(2)), C.byref(layer.cache), C.byref(layer.args))
        layer.ws.free()
        layer.rope.free()
        fill = [c.upload(np.full(n // 4, np.nan, np.float32)) for n in (nbytes, 2048, nbytes, 2048)]
        for rep in range(3):
            c.h2d(layer.att[0], np.full(layer.att[1], np.nan, np.float32))
            c.graph_launch(g)
            c.sync()
            assert np.array_equal(layer.get(layer.att), want[0]) and np.array_equal(layer.get(layer.k).view(np.uint16), want[1].view(np.uint16)), rep
        c.graph_destroy(g)
        for b in fill:
            c.free(b)
        layer.free()


def test_two_at_once(ctx):
    """Two contexts, and two streams of one context, with a workspace for each: nothing is shared."""
    hip = ctx.lib  # (its own dependency answers for the runtime's calls)
    b = Batch([(3000, 1), (2000, 2)], 2, 128, 16, seed=41)
    q = queries(b, 4)
    ref, tol = attend(b, q, 4, 0.1)
    width = b.H * 4 * b.D
    b.upload(ctx, 2, 3000)
    want = run_attention(ctx, b, q, 4, 0.1)
    check_rows(want, ref, tol, b.held_rows)
    qb = ctx.upload(q)
    outs = [ctx.upload(np.zeros((b.M, width), np.float16)) for _ in range(3)]
    args = [qmm_hip.AttentionArgs(int(qb), width, b.H * 4, 0.1, 0, 0, int(o), qmm_hip.TYPE_F16, width) for o in outs]
    own = ctx.lib.qmm_get_stream(ctx._h)
    stream = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    with qmm_hip.Context(0) as two:
        ws = [c.attention_workspace(b.batch, b.cache, args[0]) for c in (ctx, two, ctx)]
        say("two contexts and a stream of another's")
        ctx.sync()
        for _ in range(20):
            ctx.paged_attention(b.batch, b.cache, args[0], ws[0])
            two.paged_attention(b.batch, b.cache, args[1], ws[1])
            ctx._call("qmm_set_stream", ctx._h, stream)
            ctx.paged_attention(b.batch, b.cache, args[2], ws[2])
            ctx._call("qmm_set_stream", ctx._h, None)
        two.sync()
        assert hip.hipStreamSynchronize(stream) == 0
        ctx.sync()
        assert ctx.lib.qmm_get_stream(ctx._h) == own
        for o in outs:
            assert np.array_equal(ctx.d2h(o, np.float16, (b.M, width)).view(np.uint16), want.view(np.uint16))
        for w in ws:
            w.free()
    assert hip.hipStreamDestroy(stream) == 0
    for x in (qb, *outs):
        ctx.free(x)
    b.free()


@pytest.mark.parametrize("q8", [False, True])
def test_far_pages(ctx, q8):
    """A cache of more than 2^32 bytes (2^31 values) in each half: the last pages' cells, and the same bits
    as a small cache gives."""
    P, H, D, total = 64, 8, 128, 70000 if q8 else 36000
    lens = [(150, 1), (190, 70)]
    b = Batch(lens, H, D, P, q8, seed=43)
    q = queries(b, 2)
    b.upload(ctx, 70, 190)
    want = run_attention(ctx, b, q, 2, 0.09)
    b.free()
    say(f"far pages q8={q8}")
    ids = total - 1 - 17 * np.arange(b.n_pages)  # far apart, from the end
    big = {}
    for n, per in (("k", H * P * D * b.k.itemsize), ("v", H * P * D * b.k.itemsize)) + ((("ks", H * P * 4), ("vs", H * P * 4)) if q8 else ()):
        assert n in ("ks", "vs") or int(ids.min()) * per >= 2 ** 32
        big[n] = ctx.malloc(total * per)
        for i, at in enumerate(ids):
            ctx.h2d(big[n], getattr(b, n)[i], int(at) * per)
    inside = (b.pages >= 0) & (b.pages < b.n_pages)
    far = Batch(lens, H, D, P, q8, seed=43)
    far.pages = np.where(inside, ids[np.where(inside, b.pages, 0)], -1).astype(np.int32)
    far.k = far.v = far.ks = far.vs = np.zeros(4, np.float32)  # (uploaded by upload(), not used)
    far.n_pages = total
    far.upload(ctx, 70, 190)
    far.cache = qmm_hip.KvCache(qmm_hip.KV_Q8 if q8 else qmm_hip.KV_F16, P, total, H, D, int(big["k"]), int(big["v"]),
                                int(big["ks"]) if q8 else None, int(big["vs"]) if q8 else None)
    got = run_attention(ctx, far, q, 2, 0.09)
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16))
    # appending the same rows to both caches writes the same cells
    x = np.random.default_rng(44).standard_normal((b.M, 3 * H * D)).astype(np.float32)
    xb = ctx.upload(x)
    b.upload(ctx, 70, 190)
    for w in (b, far):
        ctx.kv_append(w.batch, w.cache, qmm_hip.KvRows(k=int(xb), k_stride=3 * H * D, v=int(xb) + 4 * H * D, v_stride=3 * H * D))
    ctx.sync()
    for n in ("k", "v") + (("ks", "vs") if q8 else ()):
        small = getattr(b, n)
        near = ctx.d2h(b.bufs[n], small.dtype, small.shape)
        per = small[0].nbytes
        for i, at in enumerate(ids):
            assert np.array_equal(ctx.d2h(big[n], small.dtype, small[0].shape, int(at) * per).view(np.uint8), near[i].view(np.uint8)), (n, i)
    b.free()
    far.free()
    for x in (xb, *big.values()):
        ctx.free(x)


@pytest.mark.parametrize("lens,heads,group,D", [
    ([(1 + 7 * (i % 60), 1) for i in range(600)], 1, 2, 64),                    # more sequences than share work
    ([(40 + i % 9, i % 4) for i in range(300)], 3, 4, 64),                      # sequences without new tokens between
    ([(2500, 1), (30, 1)], 1, 130, 64),                                         # one head, more rows of a token than a tile
    ([(700, 1), (90, 3)], 2, 40, 128),
    ([(1200, 2)], 1, 33, 256),
])
def test_wide_batches(ctx, lens, heads, group, D):
    b = Batch(lens, heads, D, 16, seed=len(lens) + group, extra_rows=2)
    q = queries(b, group)
    say(f"wide: {len(lens)} sequences H={heads}x{group} D={D}")
    ref, tol = attend(b, q, group, D ** -0.5)
    for hints in ((max(n for _, n in lens), max(n for n, _ in lens)), (0, 0)):
        b.upload(ctx, *hints)
        check_rows(run_attention(ctx, b, q, group, D ** -0.5), ref, tol, b.held_rows)
        b.free()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("P", [16, 32, 64, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1100, 3)])
def test_calls_announced_as_large(ctx, q8, D, P, window, sinks):
    """Few rows with hints of long sequences: the loads for caches of more than 96 MB, over ragged lengths,
    pages of every size and cells that hold no numbers; in shares, and (many heads) without."""
    for lens, heads, longest in (([(n, 1 + n % 4) for n in (4, 15, 16, 65, 127, 300, 511, 1500)], 1, 1 << 17),
                                 ([(1500 if i % 40 == 9 else 5 + 37 * i % 400, 1) for i in range(130)], 2, 2000)):
        b = Batch(lens, heads, D, P, q8, seed=D + P, max_pages=longest // P)
        group = 4 if heads == 1 else 3
        q = queries(b, group)
        if not q8:  # a new token's values: the rows before it do not see them
            p, t = b.cells(3)
            b.v[p[-1], 0, 5, t[-1]] = np.nan
            b.v[p[-2], 0, 7, t[-2]] = np.inf
        say(f"announced as large: {len(lens)} sequences D={D} P={P} q8={q8} window={window}")
        ref, tol = attend(b, q, group, D ** -0.5, window, sinks)
        b.upload(ctx, max(n for _, n in lens), longest)
        one = run_attention(ctx, b, q, group, D ** -0.5, window, sinks)
        b.free()
        check_rows(one, ref, tol, b.held_rows)


@pytest.mark.parametrize("new", [1, 9, 60])
def test_value_scales_of_all_sizes(ctx, new):
    """8-bit values from 2^-60 to 2^8 between the tokens, in rising, falling and mixed order; and all zero."""
    for how in ("rise", "fall", "mix", "zero"):
        b = Batch([(300, new), (64, min(new, 30))], 1, 64, 16, True, seed=47)
        for s in range(b.S):
            p, t = b.cells(s)
            e = np.linspace(-60, 8, len(p))
            e = e[::-1] if how == "fall" else b.rng.permutation(e) if how == "mix" else e
            b.vs[p, :, t] = 0 if how == "zero" else 2.0 ** np.floor(e)[:, None]
        q = queries(b, 4)
        say(f"value scales {how} new={new}")
        ref, tol = attend(b, q, 4, 0.125)
        b.upload(ctx, new, 300)
        check_rows(run_attention(ctx, b, q, 4, 0.125), ref, tol, b.held_rows)
        b.free()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 256])
def test_workspaces_of_any_size(ctx, q8, D):
    """Draft rows and single tokens over long sequences with room for any number of workers: the same
    values to rounding, from none that share to all."""
    for lens, group in (([(2500, 9), (700, 13)], 8), ([(2500, 1), (1900, 1)], 8), ([(1500, 30), (1100, 1), (900, 2)], 8)):
        b = Batch(lens, 1, D, 16, q8, seed=53)
        q = queries(b, group)
        ref, tol = attend(b, q, group, D ** -0.5)
        b.upload(ctx, max(n for _, n in lens), 2500)
        rows = 128 if lens[0][1] > 1 else 16
        each = 2 * rows * (D * 4 + 8) + 32
        for workers in (1, 2, 3, 5, 7, 8, 9, 13, 15, 17, 26, 31, 100):
            say(f"workspace for {workers} workers, lens={lens} D={D} q8={q8}")
            h = C.c_void_p()
            ctx._call("qmm_attention_workspace_create", ctx._h, (workers + 1) * each, C.byref(h))
            ws = qmm_hip._Handle(ctx, h.value, "qmm_attention_workspace_destroy")
            check_rows(run_attention(ctx, b, q, group, D ** -0.5, ws=ws), ref, tol, b.held_rows)
            ws.free()
        b.free()


@pytest.mark.parametrize("new", [4, 20])
def test_rows_claimed_twice(ctx, new):
    """Row starts that fall: two sequences (the same one twice) claim all rows, one between them none."""
    b = Batch([(3000, new)], 2, 64, 16, seed=59)
    q = queries(b, 4)
    ref, tol = attend(b, q, 4, 0.125)
    b.S, b.pages, b.kv_len = 3, np.repeat(b.pages, 3, 0), np.array([3000, 77, 3000], np.int32)
    b.row_start = np.array([0, new, 0, new], np.int32)
    say(f"rows claimed twice, new={new}")
    b.upload(ctx, new, 3000)
    got = run_attention(ctx, b, q, 4, 0.125)
    b.free()
    check_rows(got, ref, tol, new)


def test_refusals(ctx):
    """Bad calls return a status and a reason, and launch nothing."""
    b = Batch([(20, 1)], 2, 64, 16, seed=50).upload(ctx, 1, 20)
    q, out = ctx.upload(queries(b, 2)), ctx.upload(np.full((1, 256), 5.0, np.float16))
    x = ctx.upload(np.zeros((1, 512), np.float32))
    say("refusals")

    def changed(base, **kw):
        new = type(base)(*[getattr(base, f[0]) for f in base._fields_])
        for n, v in kw.items():
            setattr(new, n, v)
        return new

    args = qmm_hip.AttentionArgs(int(q), 256, 4, 0.125, 0, 0, int(out), qmm_hip.TYPE_F16, 256)
    rows = qmm_hip.KvRows(q=int(x), q_stride=512, q_heads=4, k=int(x) + 1024, k_stride=512, v=int(x) + 1536, v_stride=512,
                          q_out=int(out), q_out_stride=256)
    att = lambda batch=b.batch, cache=b.cache, a=args: ctx.status_of(  # noqa: E731
        "qmm_paged_attention", C.byref(batch), C.byref(cache), C.byref(a), None)
    app = lambda batch=b.batch, cache=b.cache, r=rows: ctx.status_of(  # noqa: E731
        "qmm_kv_append", C.byref(batch), C.byref(cache), C.byref(r))
    for kw in (dict(head_dim=96), dict(page_tokens=24), dict(page_tokens=8), dict(type=9), dict(k=None), dict(v=b.cache.v + 8),
               dict(n_heads=0), dict(n_pages=-1)):
        assert att(cache=changed(b.cache, **kw)) and ctx.last_error(), kw
        assert app(cache=changed(b.cache, **kw)), kw
    for kw in (dict(n_seqs=-1), dict(n_rows=-1), dict(row_start=None), dict(pages=None), dict(kv_len=None), dict(max_pages=0),
               dict(n_seqs=1 << 23)):
        assert att(batch=changed(b.batch, **kw)) and app(batch=changed(b.batch, **kw)), kw
    for kw in (dict(q=None), dict(q=int(q) + 2), dict(q_stride=128), dict(q_heads=5), dict(scale=0.0), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(window=-1), dict(sinks=-1), dict(out=None), dict(out=int(out) + 2), dict(out_type=77),
               dict(out_stride=4)):
        assert att(a=changed(args, **kw)), kw
    for kw in (dict(k=None), dict(v=None), dict(k=int(x) + 4), dict(q_stride=100), dict(q_out=None), dict(q_heads=5), dict(eps=-1.0),
               dict(q_out_stride=8)):
        assert app(r=changed(rows, **kw)), kw
    far = ctx.rope(128)
    assert app(r=changed(rows, rope=far.handle)), "more turned values than a head has"
    far.free()
    for bad in (dict(rot_dim=12), dict(rot_dim=512), dict(rot_dim=64, base=0.0), dict(rot_dim=64, n_axes=4),
                dict(rot_dim=64, pair_axis=[3] * 32, n_axes=2)):
        with pytest.raises(qmm_hip.QmmError):
            ctx.rope(**bad)
    assert att(batch=changed(b.batch, n_seqs=0)) == 0 and app(batch=changed(b.batch, n_rows=0)) == 0
    ctx.sync()
    assert (ctx.d2h(out, np.float16, (1, 256)) == 5.0).all()
    for y in (q, out, x):
        ctx.free(y)
    b.free()
