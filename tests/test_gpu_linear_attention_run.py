"""Layers with carried states and the beam search as they are used: a prompt, then
decoding with beams that change parents, each stage checked; captured and
replayed; two at once; one workspace for all; a sequence that is spoilt; tensors
past 2^32 bytes; what is refused."""
import ctypes as C

import numpy as np
import pytest

import qmm_hip
import state_ref as R
import synth
from gpu_util import say
from oracle import TYPE_Q4_K

pytestmark = pytest.mark.gpu

K, HK, HV, D, W, V = 256, 2, 4, 64, 4, 5003
QK, VW = HK * D, HV * D
CH = 2 * QK + VW


class Layer:
    """A layer of linear attention between a projection and an LM head, with pools of states, and its calls in order."""

    def __init__(self, ctx, rows, n_slots, items, beams, seed=0):
        self.ctx, self.rows, self.n_slots, self.items, self.beams = ctx, rows, n_slots, items, beams
        rng = np.random.default_rng(seed)
        self.held = []
        self.w = [self.keep(ctx.weight_upload(synth.weights(TYPE_Q4_K, n, k, seed=seed + i), TYPE_Q4_K, n, k))
                  for i, (n, k) in enumerate([(CH, K), (VW, K), (2 * HV, K), (K, VW), (V, K)])]
        self.par = {"filter": rng.uniform(-1, 1, (CH, W)), "rate": -rng.uniform(0.01, 1, HV), "dt": rng.uniform(-2, 1, HV),
                    "gamma": rng.uniform(0.5, 1.5, D)}
        self.par = {n: x.astype(np.float32) for n, x in self.par.items()}
        self.p = {n: self.keep(ctx.upload(x)) for n, x in self.par.items()}
        self.shape = {"x": (rows, K), "mix": (rows, CH), "z": (rows, VW), "ab": (rows, 2 * HV), "seq": (rows, CH), "att": (rows, VW),
                      "y": (rows, K), "past": (n_slots, W - 1, CH), "S": (n_slots, HV, D, D), "logits": (items * beams, V),
                      "total": (items, beams), "score": (items * beams,)}
        self.whole = {"row_start": (rows + 1,), "slot_in": (rows,), "slot_out": (rows,), "token": (items, beams), "parent": (items, beams),
                      "src": (n_slots,), "dst": (n_slots,)}
        self.b = {n: self.keep(ctx.upload(np.zeros(s, np.float32))) for n, s in self.shape.items()}
        self.b.update({n: self.keep(ctx.upload(np.zeros(s, np.int32))) for n, s in self.whole.items()})
        at = {n: int(b) for n, b in {**self.b, **self.p}.items()}
        self.conv = qmm_hip.ConvArgs(at["mix"], CH, CH, W, at["filter"], None, at["past"], 1, at["seq"], CH)
        self.delta = qmm_hip.DeltaArgs(
            q=at["seq"], k=at["seq"] + 4 * QK, q_stride=CH, k_stride=CH, v=at["seq"] + 8 * QK, v_stride=CH, qk_heads=HK, v_heads=HV, key_dim=D,
            value_dim=D, a=at["ab"], b=at["ab"] + 4 * HV, a_stride=2 * HV, b_stride=2 * HV, rate=at["rate"], dt_bias=at["dt"], scale=D ** -0.5,
            qk_eps=1e-6, state=at["S"], z=at["z"], z_stride=VW, gamma=at["gamma"], gamma_eps=1e-6, out=at["att"], out_stride=VW)
        self.sel = qmm_hip.BeamArgs(at["logits"], V, V, items, beams, at["score"], None, 0, beams, at["token"], at["parent"], at["total"])
        self.pools = [qmm_hip.SlotPool(at[n], int(np.prod(self.shape[n][1:])) * 4, n_slots) for n in ("past", "S")]
        batch = qmm_hip.StateBatch(rows, rows, at["row_start"], at["slot_in"], at["slot_out"], n_slots, 0)
        lib = ctx.lib  # one workspace: the larger of the two that are asked for
        n = max(lib.qmm_gated_delta_workspace_bytes(ctx._h, C.byref(batch), C.byref(self.delta)), lib.qmm_beam_workspace_bytes(ctx._h, C.byref(self.sel)))
        assert n > 0
        h = C.c_void_p()
        ctx._call("qmm_attention_workspace_create", ctx._h, n, C.byref(h))
        self.ws = qmm_hip._Handle(ctx, h.value, "qmm_attention_workspace_destroy")

    def keep(self, b):
        self.held.append(b)
        return b

    def get(self, *names):
        got = [self.ctx.d2h(self.b[n], *((np.float32, self.shape[n]) if n in self.shape else (np.int32, self.whole[n]))) for n in names]
        return got[0] if len(got) == 1 else got

    def put(self, **values):
        for n, x in values.items():
            self.ctx.h2d(self.b[n], np.ascontiguousarray(x, np.float32 if n in self.shape else np.int32))

    def batch(self, seqs, m, hint=0):
        return qmm_hip.StateBatch(seqs, m, *(int(self.b[n]) for n in ("row_start", "slot_in", "slot_out")), self.n_slots, hint)

    def project(self, m):
        self.ctx.gemm_multi_dispatch(self.b["x"], m, K, [qmm_hip.MatrixTask(w, TYPE_Q4_K, n, K, int(self.b[to]), n)
                                                         for w, n, to in zip(self.w, (CH, VW, 2 * HV), ("mix", "z", "ab"))])

    def attend(self, seqs, m, hint=0):
        self.ctx.short_conv(self.batch(seqs, m, hint), self.conv)
        self.ctx.gated_delta(self.batch(seqs, m, hint), self.delta, self.ws)

    def head(self, m, last=None):
        self.ctx.gemm_multi_dispatch(self.b["att"], m, VW, [qmm_hip.MatrixTask(self.w[3], TYPE_Q4_K, K, VW, int(self.b["y"]), K)])
        for i, r in enumerate(range(m) if last is None else last):  # (of a prompt, the last row)
            self.ctx.gemm_multi_dispatch(int(self.b["y"]) + 4 * K * r, 1, K, [qmm_hip.MatrixTask(self.w[4], TYPE_Q4_K, V, K, int(self.b["logits"]) + 4 * V * i, V)])

    def select(self, beams=None):
        a = qmm_hip.BeamArgs.from_buffer_copy(self.sel)
        if beams:
            a.n_beams = beams
        self.ctx.beam_select(a, self.ws)

    def free(self):
        self.ws.free()
        for b in self.held:
            self.ctx.free(b)


def check_attend(layer, news, slots, past, S):
    """Both calls, against the formulas on what the projection left and the states before."""
    b = R.States(news, slots)
    b.n_slots, m = layer.n_slots, sum(news)
    mix, z, ab, seq, att = (x[:m] for x in layer.get("mix", "z", "ab", "seq", "att"))
    ref, tol, after = R.conv(b, mix, layer.par["filter"], None, past, True)
    R.within(seq, ref, tol, "convolution")
    assert np.array_equal(layer.get("past").view(np.uint32), after.view(np.uint32))
    ref, tol, after, after_tol = R.delta(
        b, seq[:, :QK].reshape(m, HK, D), seq[:, QK:2 * QK].reshape(m, HK, D), seq[:, 2 * QK:].reshape(m, HV, D), ab[:, :HV], ab[:, HV:],
        layer.par["rate"], layer.par["dt"], D ** -0.5, 1e-6, S, z, layer.par["gamma"], 1e-6, HV // HK)
    R.within(att, ref.reshape(m, VW), tol.reshape(m, VW), "delta rule")
    R.within(layer.get("S"), after, after_tol, "states")


def check_select(layer, beams, score):
    logits, token, parent, total = layer.get("logits", "token", "parent", "total")
    for i in range(layer.items):
        rows = logits[i * beams:(i + 1) * beams]
        t, p, ref, certain = R.select(rows, score[i * beams:(i + 1) * beams], None, 0, layer.beams)
        assert np.array_equal(token[i][certain], t[certain]) and np.array_equal(parent[i][certain], p[certain])
        assert (np.abs(total[i] - ref) <= 40 * R.U + R.U * np.abs(ref)).all()
    return token, parent, total


@pytest.mark.parametrize("copies", [False, True])
def test_decoding_with_beams(ctx, copies):
    """Two prompts, their best tokens, then steps of three beams each. Heirs read their parent's slots and write their own of the
    other half, or the slots are copied first and worked on in place. Every stage against its formula."""
    items, beams, news = 2, 3, [70, 33]
    layer = Layer(ctx, sum(news), 2 * items * beams + items, items, beams, seed=51)
    table = synth.activations(V, K, seed=52)
    m = sum(news)
    prompt = 2 * items * beams  # its slots
    layer.put(x=table[np.random.default_rng(3).integers(0, V, m)], row_start=np.concatenate([[0], np.cumsum(news)]), slot_in=[-1] * items,
              slot_out=[prompt + i for i in range(items)])
    past, S = layer.get("past", "S")
    say(f"beams: prompts copies={copies}")
    layer.project(m)
    layer.attend(items, m, max(news))
    layer.head(m, np.cumsum(news) - 1)
    layer.select(1)
    ctx.sync()
    check_attend(layer, news, [(-1, prompt + i) for i in range(items)], past, S)
    token, parent, total = check_select(layer, 1, np.zeros(items))
    own = [[prompt + i] * beams for i in range(items)]  # each beam's slot
    n = items * beams
    for step in range(5):
        say(f"beams: step {step} copies={copies}")
        read = [own[i][parent[i][j]] for i in range(items) for j in range(beams)]
        write = [(step % 2) * n + j for j in range(n)]
        layer.put(x=np.concatenate([table[token.ravel()], np.zeros((m - n, K), np.float32)]), row_start=np.arange(n + 1), score=total.ravel(),
                  slot_in=write if copies else read, slot_out=write, src=read, dst=write)
        past, S = layer.get("past", "S")
        layer.project(n)
        if copies:
            ctx.copy_slots(layer.pools, layer.b["src"], layer.b["dst"], n)
            for pool in (past, S):
                pool[write] = pool[read]
        layer.attend(n, n, 1)
        layer.head(n)
        layer.select()
        ctx.sync()
        check_attend(layer, [1] * n, [(w if copies else r, w) for r, w in zip(read, write)], past, S)
        score = total.ravel()
        token, parent, total = check_select(layer, beams, score)
        own = [[write[i * beams + j] for j in range(beams)] for i in range(items)]
    layer.free()


OUT = ("seq", "att", "past", "S", "token", "parent", "total")


@pytest.mark.parametrize("news,hint", [([1] * 6, 1), ([12, 16, 0, 9, 1, 16], 16), ([150, 0, 70, 33, 1, 40], 150),
                                       ([700, 0, 520, 33, 1, 40], 700)], ids=["tokens", "drafts", "prompts", "halves"])
def test_captured_steps(news, hint):
    """All calls but the projections, captured once and replayed with other rows, lengths, slots and logits, and eager work
    between: the eager calls' bits each time."""
    n, m = len(news), sum(news)
    with qmm_hip.Context(0) as c, qmm_hip.Context(0) as e:
        mine, other = (Layer(x, m, 20, 2, 3, seed=53) for x in (c, e))

        def calls(layer):
            layer.ctx.copy_slots(layer.pools, layer.b["src"], layer.b["dst"], 3)
            layer.attend(n, m, hint)
            layer.select()

        mine.put(x=synth.activations(m, K, seed=1), row_start=np.concatenate([[0], np.cumsum(news)]))
        mine.project(m)
        c.sync()
        c.graph_begin()
        calls(mine)
        g = c.graph_end()
        rng = np.random.default_rng(54)
        for rep in range(4):
            say(f"captured {news} replay {rep}")
            now = list(rng.permutation(news))
            slots = rng.permutation(20)
            past, S = (rng.standard_normal(mine.shape[k]).astype(np.float32) * 0.3 for k in ("past", "S"))
            for layer in (mine, other):
                layer.put(x=synth.activations(m, K, seed=70 + rep), row_start=np.concatenate([[0], np.cumsum(now)]), slot_in=slots[:n],
                          slot_out=slots[n:2 * n] if rep % 2 else slots[:n], src=slots[:3], dst=slots[2 * n:2 * n + 3], past=past, S=S,
                          logits=rng.standard_normal((6, V)) if layer is mine else mine.get("logits"), score=np.arange(6) * -0.1,
                          att=np.full((m, VW), np.nan, np.float32))
                layer.project(m)
            c.sync()
            c.graph_launch(g)
            c.sync()
            calls(other)
            e.sync()
            for name in OUT:
                assert np.array_equal(mine.get(name).view(np.uint32), other.get(name).view(np.uint32)), (rep, name)
            mine.head(4)  # eager work of the same context
            mine.select()
            c.sync()
        c.graph_destroy(g)
        mine.free()
        other.free()


def test_graphs_share_a_workspace():
    """In stream order one workspace serves prompts and selections of two graphs, in either order; and it outlives its handle."""
    with qmm_hip.Context(0) as c:
        news, m = [150, 70], 220
        layer = Layer(c, m, 4, 1, 64, seed=55)
        rng = np.random.default_rng(56)
        layer.put(x=synth.activations(m, K, seed=2), row_start=[0, 150, 220], slot_in=[0, 1], slot_out=[2, 3], past=rng.standard_normal(layer.shape["past"]),
                  S=rng.standard_normal(layer.shape["S"]), logits=rng.standard_normal(layer.shape["logits"]))
        layer.project(m)
        layer.attend(2, m, 150)
        layer.select()
        c.sync()
        want = layer.get(*OUT)
        graphs = []
        for call in (lambda: layer.attend(2, m, 150), layer.select):
            c.graph_begin()
            call()
            graphs.append(c.graph_end())
        for rep in range(4):
            say(f"two graphs, one workspace, {rep}")
            if rep == 2:
                layer.ws.free()
                fill = c.upload(np.full(1 << 20, np.nan, np.float32))
            layer.put(att=np.full(layer.shape["att"], np.nan), seq=np.full(layer.shape["seq"], np.nan), token=np.zeros((1, 64)), parent=np.zeros((1, 64)))
            for g in graphs if rep % 2 else graphs[::-1]:
                c.graph_launch(g)
            c.sync()
            assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(layer.get(*OUT), want)), rep
        for g in graphs:
            c.graph_destroy(g)
        c.free(fill)
        layer.free()


def test_two_at_once(ctx):
    """Two contexts, and a stream of another's, each with its own tensors and workspace: nothing is shared."""
    hip, stream = ctx.lib, C.c_void_p()  # (its own dependency answers for the runtime's calls)
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    with qmm_hip.Context(0) as two:
        m = 220
        layers = [Layer(c, m, 4, 1, 64, seed=57) for c in (ctx, two, ctx)]
        rng = np.random.default_rng(58)
        fill = {n: rng.standard_normal(layers[0].shape[n]) for n in ("past", "S", "logits")}
        for layer in layers:
            layer.put(x=synth.activations(m, K, seed=3), row_start=[0, 150, 220], slot_in=[0, 1], slot_out=[2, 3], **fill)
            layer.project(m)
            layer.ctx.sync()
        layers[0].attend(2, m, 150)
        layers[0].select()
        ctx.sync()
        want = layers[0].get(*OUT)
        say("two contexts and a stream of another's")
        for _ in range(20):
            for layer, s in zip(layers, (None, None, stream)):
                layer.ctx._call("qmm_set_stream", layer.ctx._h, s)
                layer.attend(2, m, 150)
                layer.select()
        ctx._call("qmm_set_stream", ctx._h, None)
        two.sync()
        assert hip.hipStreamSynchronize(stream) == 0
        ctx.sync()
        for layer in layers:
            assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(layer.get(*OUT), want))
            layer.free()
    assert hip.hipStreamDestroy(stream) == 0


@pytest.mark.parametrize("hint", [1, 20, 150])
@pytest.mark.parametrize("what", ["mix", "z", "ab", "S", "past"])
def test_spoilt_sequence(ctx, what, hint):
    """No numbers in one sequence's rows or states: the others' bits are those of a run without, on each path."""
    news, m = [37, 30, 5, 41], 113
    layer = Layer(ctx, m, 8, 1, 1, seed=59)
    rng = np.random.default_rng(60)
    fill = {n: rng.standard_normal(layer.shape[n]).astype(np.float32) for n in ("past", "S", "mix", "z", "ab")}
    got = []
    for bad in (False, True):
        if bad:
            lo = 1 if what in ("S", "past") else 37
            fill[what][lo:1 + lo if lo == 1 else 67:7] = np.nan
            fill[what][lo + (0 if lo == 1 else 3)] = np.inf
        say(f"spoilt {what if bad else 'nothing'} hint={hint}")
        layer.put(row_start=np.concatenate([[0], np.cumsum(news)]), slot_in=[0, 1, 2, 3], slot_out=[4, 5, 6, 7], **fill)
        layer.attend(4, m, hint)
        ctx.sync()
        got.append(layer.get("seq", "att", "past", "S"))
    rows, slots = np.r_[0:37, 67:113], [0, 2, 3, 4, 6, 7]
    for (a, b), keep in zip(zip(*got), (rows, rows, slots, slots)):
        assert np.array_equal(a[keep].view(np.uint32), b[keep].view(np.uint32))
        assert np.isfinite(a[keep]).all()
    layer.free()


@pytest.mark.parametrize("what", ["mix", "z", "ab", "S", "past"])
def test_spoilt_sequence_of_halves(ctx, what):
    """The same where sequences are walked in halves: the middle one's second half."""
    news, m = [600, 700, 555], 1855
    layer = Layer(ctx, m, 6, 1, 1, seed=69)
    rng = np.random.default_rng(70)
    fill = {n: rng.standard_normal(layer.shape[n]).astype(np.float32) for n in ("past", "S", "mix", "z", "ab")}
    got = []
    for bad in (False, True):
        if bad:
            fill[what][1 if what in ("S", "past") else slice(600 + 500, 600 + 503)] = np.nan
        say(f"spoilt {what if bad else 'nothing'} in halves")
        layer.put(row_start=[0, 600, 1300, 1855], slot_in=[0, 1, 2], slot_out=[3, 4, 5], **fill)
        layer.attend(3, m, 700)
        ctx.sync()
        got.append(layer.get("seq", "att", "past", "S"))
    rows, slots = np.r_[0:600, 1300:1855], [0, 2, 3, 5]
    for (a, b), keep in zip(zip(*got), (rows, rows, slots, slots)):
        assert np.array_equal(a[keep].view(np.uint32), b[keep].view(np.uint32)) and np.isfinite(a[keep]).all()
    layer.free()


@pytest.mark.parametrize("starts", [[0, 50, 20, 400], [-5, 2 ** 31 - 1, -2 ** 31, 30], [90, 10, 60, 60], [200, 300, 400, 500]], ids=str)
@pytest.mark.parametrize("hint", [1, 20, 150])
def test_row_starts_out_of_order(ctx, starts, hint):
    """Clamped to the rows: nothing else is read or written (two sequences may share rows, whose values mean nothing)."""
    rows, m = 120, 100
    layer = Layer(ctx, rows, 6, 1, 1, seed=61)
    rng = np.random.default_rng(62)
    fill = {n: rng.standard_normal(layer.shape[n]).astype(np.float32) for n in ("past", "S", "mix", "z", "ab")}
    say(f"row starts {starts} hint={hint}")
    layer.put(row_start=starts, slot_in=[0, 1, 2], slot_out=[3, 4, 5], seq=np.full((rows, CH), 7), att=np.full((rows, VW), 7), **fill)
    layer.attend(3, m, hint)
    ctx.sync()
    seq, att, past, S = layer.get("seq", "att", "past", "S")
    held = np.zeros(rows, bool)
    for s in range(3):
        a = min(max(starts[s], 0), m)
        held[a:min(max(starts[s + 1], a), m)] = True
    assert (seq[~held] == 7).all() and (att[~held] == 7).all()
    assert np.array_equal(past[:3], fill["past"][:3]) and np.array_equal(S[:3], fill["S"][:3])
    layer.free()


def test_tensors_past_32_bits(ctx):
    """Rows, states, logits and slots beyond 2^32 bytes: the bits of small tensors."""
    # convolution and delta rule: far slots, rows far apart
    m, slots = 105, 70000
    layer = Layer(ctx, m, 4, 1, 1, seed=63)
    rng = np.random.default_rng(64)
    fill = {n: rng.standard_normal(layer.shape[n]).astype(np.float32) for n in ("past", "S", "mix", "z", "ab")}
    layer.put(row_start=[0, 100, 105], slot_in=[0, 1], slot_out=[2, 3], **fill)
    for hint in (1, 20, 100):
        layer.attend(2, m, hint)
        ctx.sync()
        seq, att, past, S = layer.get("seq", "att", "past", "S")
        say(f"past 32 bits: states, hint={hint}")
        pool = {n: ctx.malloc(slots * int(np.prod(layer.shape[n][1:])) * 4) for n in ("past", "S")}
        ids = [slots - 1, slots - 9, slots - 3, slots - 30]
        assert min(ids) * layer.pools[1].slot_bytes >= 2 ** 32
        for n, p in pool.items():
            for i in range(2):
                ctx.h2d(p, fill[n][i], ids[i] * fill[n][0].nbytes)
        layer.put(slot_in=ids[:2], slot_out=ids[2:], seq=np.zeros((m, CH)), att=np.zeros((m, VW)))
        batch = qmm_hip.StateBatch(2, m, int(layer.b["row_start"]), int(layer.b["slot_in"]), int(layer.b["slot_out"]), slots, hint)
        conv, delta = (type(a).from_buffer_copy(a) for a in (layer.conv, layer.delta))
        conv.state, delta.state = int(pool["past"]), int(pool["S"])
        ctx.short_conv(batch, conv)
        ctx.gated_delta(batch, delta, layer.ws)
        ctx.sync()
        assert np.array_equal(layer.get("seq"), seq) and np.array_equal(layer.get("att"), att)
        for n, p, want in (("past", pool["past"], past), ("S", pool["S"], S)):
            for i in (2, 3):
                assert np.array_equal(ctx.d2h(p, np.float32, want[i].shape, ids[i] * want[i].nbytes), want[i]), (n, i)
        for p in pool.values():
            ctx.free(p)
        layer.put(slot_in=[0, 1], slot_out=[2, 3], seq=np.zeros((m, CH)), att=np.zeros((m, VW)))
        for stride in ((1 << 24) - 4, 25 << 20):  # the longest that groups of rows are read at, and past it: a token at a time
            say(f"past 32 bits: rows of stride {stride}, hint={hint}")
            wide = ctx.malloc(((m - 1) * stride + CH) * 4)
            for r in range(m):
                ctx.h2d(wide, seq[r], r * stride * 4)
            delta = type(layer.delta).from_buffer_copy(layer.delta)
            delta.q, delta.k, delta.v = (int(wide) + 4 * o for o in (0, QK, 2 * QK))
            delta.q_stride = delta.k_stride = delta.v_stride = stride
            ctx.gated_delta(layer.batch(2, m, hint), delta, layer.ws)
            ctx.sync()
            got = layer.get("att")
            if hint == 1 or stride < 1 << 24:
                assert np.array_equal(got, att) and np.array_equal(layer.get("S"), S)
            else:
                check_close(layer, seq, fill, got)
            ctx.free(wide)
    layer.free()


def check_close(layer, seq, fill, got):
    b = R.States([100, 5], [(0, 2), (1, 3)])
    b.n_slots = 4
    ref, tol, after, after_tol = R.delta(
        b, seq[:, :QK].reshape(-1, HK, D), seq[:, QK:2 * QK].reshape(-1, HK, D), seq[:, 2 * QK:].reshape(-1, HV, D), fill["ab"][:, :HV],
        fill["ab"][:, HV:], layer.par["rate"], layer.par["dt"], D ** -0.5, 1e-6, fill["S"], fill["z"], layer.par["gamma"], 1e-6, HV // HK)
    R.within(got, ref.reshape(-1, VW), tol.reshape(-1, VW), "rows")
    R.within(layer.get("S")[2:], after[2:], after_tol[2:], "states")


def test_selection_and_copies_past_32_bits(ctx):
    say("past 32 bits: logits")
    items, beams, V1, stride, keep = 130, 64, 700, 150001, 9
    rng = np.random.default_rng(65)
    x, score = rng.standard_normal((beams, V1)).astype(np.float32), rng.uniform(-3, 0, beams).astype(np.float32)
    rows = items * beams
    assert (rows - beams) * stride * 4 >= 2 ** 32
    big = ctx.malloc(rows * stride * 4)
    for b in range(beams):
        ctx.h2d(big, x[b], (rows - beams + b) * stride * 4)
    sb = ctx.upload(np.tile(score, items))
    out = [ctx.upload(np.zeros((items, keep), t)) for t in (np.int32, np.int32, np.float32)]
    a = qmm_hip.BeamArgs(int(big), stride, V1, items, beams, int(sb), None, 0, keep, *(int(o) for o in out))
    ws = ctx.beam_workspace(a)
    ctx.beam_select(a, ws)
    ctx.sync()
    t, p, total, certain = R.select(x, score, None, 0, keep)
    token, parent, got = (ctx.d2h(o, d, (items, keep))[-1] for o, d in zip(out, (np.int32, np.int32, np.float32)))
    assert np.array_equal(token[certain], t[certain]) and np.array_equal(parent[certain], p[certain])
    assert (np.abs(got - total) <= 40 * R.U + R.U * np.abs(total)).all()
    ws.free()
    for u in (big, sb, *out):
        ctx.free(u)
    say("past 32 bits: slots")
    size, n = (1 << 30) + 4096, 6
    pool = ctx.malloc(size * n)
    piece = rng.integers(0, 255, 4096, np.uint8)
    places = [0, size - 4096, 1 << 29]
    for at in places:
        ctx.h2d(pool, piece, at + size)
    src, dst = ctx.upload(np.array([1], np.int32)), ctx.upload(np.array([5], np.int32))
    ctx.copy_slots([qmm_hip.SlotPool(int(pool), size, n)], src, dst, 1)
    ctx.sync()
    for at in places:
        assert np.array_equal(ctx.d2h(pool, np.uint8, 4096, 5 * size + at), piece)
    for u in (pool, src, dst):
        ctx.free(u)


def test_workspaces_too_small(ctx):
    """The selection refuses and writes nothing; the delta rule needs none."""
    layer = Layer(ctx, 220, 4, 1, 64, seed=67)
    rng = np.random.default_rng(68)
    layer.put(x=synth.activations(220, K, seed=4), row_start=[0, 150, 220], slot_in=[0, 1], slot_out=[2, 3], S=rng.standard_normal(layer.shape["S"]),
              logits=rng.standard_normal(layer.shape["logits"]), token=np.full((1, 64), -7))
    n = ctx.lib.qmm_beam_workspace_bytes(ctx._h, C.byref(layer.sel))
    h = C.c_void_p()
    ctx._call("qmm_attention_workspace_create", ctx._h, n - 1, C.byref(h))
    small = qmm_hip._Handle(ctx, h.value, "qmm_attention_workspace_destroy")
    say("workspaces too small")
    for ws in (None, small.handle):
        assert ctx.status_of("qmm_beam_select", C.byref(layer.sel), ws) == qmm_hip.QMM_ENOMEM
    ctx.sync()
    assert (layer.get("token") == -7).all()
    layer.project(220)
    got = []
    for ws in (None, small):
        ctx.short_conv(layer.batch(2, 220, 150), layer.conv)
        ctx.gated_delta(layer.batch(2, 220, 150), layer.delta, ws)
        ctx.sync()
        got.append(layer.get("att", "S"))
    assert n - 1 < ctx.lib.qmm_gated_delta_workspace_bytes(ctx._h, C.byref(layer.batch(2, 220, 150)), C.byref(layer.delta))
    assert all(np.array_equal(x, y) for x, y in zip(*got))
    small.free()
    layer.free()
