"""What the engine's linear-attention layers and beam search need beside the projections, for timing.

A case's "kind":
  conv   qmm_short_conv: the causal convolution of a few taps over every channel of the fused q / k / v projection, with
         SiLU; outputs the rows and the inputs carried to the next call
  delta  qmm_gated_delta: the gated delta rule over single tokens, drafts and prompts, with the output norm and gate or
         without; outputs the rows and the new states
  beam   qmm_beam_select: the best continuations of every item's beams over the vocabulary; outputs tokens, parents, scores
  copy   qmm_copy_slots: beams reordered, their states or their last cache pages copied in all layers; outputs the pools
"seqs" sequences have "new_lo".."new_hi" new tokens; their states are read from one set of slots and written to another,
as a program does that may have to go back (drafts) or whose beams change parents.

Projections are N(0, 1) with one channel in a hundred eight times larger; decay rates 1..16 with steps of 0.001..0.1 as
trained models start from; logits N(0, 2.5) around a bias of the vocabulary's.
"""
import ctypes
import math
import os
import sys

import torch

own = False
DEV = "cuda"
EPS = 1e-6
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _named(name, c, kw):
    c.update(kw)
    return {"name": name, **c} if name else c


def _conv(name, **kw):
    return _named(name, {"kind": "conv", "seqs": 1, "new_lo": 1, "new_hi": 1, "channels": 8192, "width": 4, "bias": False}, kw)


def _delta(name, **kw):
    return _named(name, {"kind": "delta", "seqs": 1, "new_lo": 1, "new_hi": 1, "qk_heads": 16, "v_heads": 32, "key_dim": 128,
                         "value_dim": 128, "fresh": 0.0, "gated": True}, kw)


def _beam(name, **kw):
    return _named(name, {"kind": "beam", "items": 1, "beams": 4, "vocab": 151936, "keep": 8, "masked": 0.0, "ended": 0.0,
                         "first": False}, kw)


def _copy(name, **kw):
    return _named(name, {"kind": "copy", "pools": 16, "slots": 64, "pairs": 8, "slot_bytes": 32768}, kw)


def listed():
    return [
        # a step of a small serving batch
        _conv("conv_tokens", seqs=16),
        # ragged prompts, one of them the first part of a longer one
        _conv("conv_prompts", seqs=5, new_lo=333, new_hi=1900),
        # one decoded token of one user: the smallest call (launch and latency)
        _delta("delta_token"),
        # a step of a serving batch: its states read and written
        _delta("delta_batch", seqs=64),
        # draft tokens to verify: a few rows per sequence
        _delta("delta_drafts", seqs=8, new_lo=5, new_hi=16),
        # ragged prompts without a past, the norm and gate left to the caller
        _delta("delta_prompts", seqs=6, new_lo=129, new_hi=1500, fresh=1.0, gated=False),
        # one short prompt: little to share between the compute units
        _delta("delta_prompt_short", new_lo=417, new_hi=417, fresh=1.0),
        # one long prompt: the largest
        _delta("delta_prompt_long", new_lo=8192, new_hi=8192, fresh=1.0),
        # one user's beams
        _beam("beam_one"),
        # a batch of them, some beams ended
        _beam("beam_batch", items=16, beams=8, keep=16, ended=0.15),
        # the last pages of eight beams in the attention layers: keys and values of 8 layers
        _copy("copy_pages", pools=16, slots=96, pairs=8, slot_bytes=32768),
        # the recurrent states of four beams in 24 layers
        _copy("copy_states", pools=24, slots=8, pairs=4, slot_bytes=2097152),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.random()
    if kind < 0.2:
        seqs = _log_int(rng, 1, 96)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, 8000 // seqs))
        return _conv(None, seqs=seqs, new_lo=max(1, new // 3), new_hi=new, channels=4 * _log_int(rng, 16, 2560),
                     width=rng.choice([2, 3, 4, 4]), bias=rng.random() < 0.4)
    if kind < 0.7:
        qk_heads = rng.choice([1, 2, 4, 8, 16])
        shape = {"qk_heads": qk_heads, "v_heads": qk_heads * rng.choice([1, 2, 2, 3]), "key_dim": rng.choice([64, 128, 128]),
                 "value_dim": rng.choice([64, 128, 128]), "fresh": rng.choice([0.0, 0.3, 1.0]), "gated": rng.random() < 0.6}
        if shape["v_heads"] > 32:
            shape["v_heads"] = 32
        form = rng.random()
        if form < 0.35:  # single tokens
            return _delta(None, seqs=_log_int(rng, 1, 96), **shape)
        if form < 0.55:  # drafts
            new = rng.randint(2, 24)
            return _delta(None, seqs=_log_int(rng, 1, 16), new_lo=rng.randint(1, new), new_hi=new, **shape)
        seqs = rng.randint(1, 6)
        new = _log_int(rng, 25, 8000 // seqs)
        return _delta(None, seqs=seqs, new_lo=max(1, new // 3), new_hi=new, **shape)
    if kind < 0.87:
        beams, items = rng.choice([1, 2, 3, 4, 5, 8, 16]), _log_int(rng, 1, 16)
        vocab = _log_int(rng, 1000, 250000 if items * beams <= 64 else 100000)
        return _beam(None, items=items, beams=beams, vocab=vocab, keep=rng.choice([1, beams, 2 * beams, 2 * beams + 1]),
                     masked=rng.choice([0.0, 0.0, 0.5, 0.999]), ended=rng.choice([0.0, 0.3]), first=rng.random() < 0.2)
    pairs = _log_int(rng, 1, 64)
    pools = rng.randint(1, 40)
    size = 16 * _log_int(rng, 64, max(64, min(131072, 25000000 // (pairs * pools))))
    return _copy(None, pools=pools, slots=2 * pairs + rng.randint(0, 9), pairs=pairs, slot_bytes=size)


def _news(case):
    """New tokens of every sequence: from lo to hi, both among them, in no order."""
    n, lo, hi = case["seqs"], case["new_lo"], case["new_hi"]
    return [hi] if n == 1 else [lo + (hi - lo) * ((1013 * i + 3) % n) // (n - 1) for i in range(n)]


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 43)

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    def uniform(lo, hi, *shape):
        return torch.empty(*shape, device=DEV).uniform_(lo, hi, generator=g)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    s = {"case": case}
    if case["kind"] == "beam":
        R, V = case["items"] * case["beams"], case["vocab"]
        s["logits"] = 2.5 * randn(R, V) + 1.5 * randn(V)
        if case["masked"]:  # tokens that a grammar rules out
            s["logits"].masked_fill_(torch.rand(R, V, device=DEV, generator=g) < case["masked"], -math.inf)
        s["score"] = uniform(-30.0, -20.0, R)
        if case["first"]:  # the first step: all beams are alike, the first one alone counts
            s["logits"].copy_(s["logits"].reshape(case["items"], -1, V)[:, :1].repeat(1, case["beams"], 1).reshape(R, V))
            s["score"].reshape(case["items"], -1)[:, 1:] = -math.inf
        s["ended"] = (torch.rand(R, device=DEV, generator=g) < case["ended"]).to(torch.int32)
        n = case["items"], case["keep"]
        s["token"], s["parent"] = (torch.zeros(n, dtype=torch.int32, device=DEV) for _ in range(2))
        s["score_out"] = torch.zeros(n, device=DEV)
        return s
    if case["kind"] == "copy":
        s["pools"] = [randn(case["slots"], case["slot_bytes"] // 4) for _ in range(case["pools"])]
        order = torch.randperm(case["slots"], device=DEV, generator=g)
        parent = torch.randint(0, case["pairs"], (case["pairs"],), device=DEV, generator=g)  # (a good beam has several heirs)
        s["src"] = order[:case["pairs"]][parent].to(torch.int32)
        s["dst"] = order[case["pairs"]:2 * case["pairs"]].to(torch.int32)
        return s
    news, S = _news(case), case["seqs"]
    M = sum(news)
    s["news"], s["rows"] = news, M
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    s["row_start"], s["max_new"] = ints(starts), max(news)
    s["slot_out"] = ints([S + (5 * i + 1) % S if S % 5 else S + i for i in range(S)])
    if case["kind"] == "conv":
        Ch, W = case["channels"], case["width"]
        s["slot_in"] = ints(list(range(S)))
        s["x"] = randn(M, Ch) * torch.where(torch.rand(Ch, device=DEV, generator=g) < 0.01, 8.0, 1.0)
        s["weight"] = uniform(-0.5, 0.5, Ch, W)
        s["bias"] = uniform(-0.5, 0.5, Ch) if case["bias"] else None
        s["state"] = randn(2 * S, W - 1, Ch)
        s["out"] = torch.zeros(M, Ch, device=DEV)
        return s
    HK, HV, DK, DV = case["qk_heads"], case["v_heads"], case["key_dim"], case["value_dim"]
    s["slot_in"] = torch.where(torch.rand(S, device=DEV, generator=g) < case["fresh"], -1, torch.arange(S, device=DEV)).to(torch.int32)
    width = 2 * HK * DK + HV * DV  # one row of the convolution's output: q, k, v side by side
    x = randn(M, width) * torch.where(torch.rand(width, device=DEV, generator=g) < 0.01, 8.0, 1.0)
    s["qkv"] = x * torch.sigmoid(x)
    s["ab"] = randn(M, 2 * HV)  # decay and step of every head, from one projection
    s["rate"] = -uniform(1.0, 16.0, HV)
    s["dt_bias"] = torch.log(torch.expm1(torch.exp(uniform(math.log(1e-3), math.log(0.1), HV))))
    s["state"] = 0.3 * randn(2 * S, HV, DK, DV)
    s["out"] = torch.zeros(M, HV * DV, device=DEV)
    if case["gated"]:
        s["z"], s["gamma"] = randn(M, HV * DV), uniform(0.5, 1.5, DV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s["call"] = _calls(s)
    return s


# ---------------------------------------------------- the framework's calls
_ctx = None


def _context():
    """The program's one context (it lives as long as the process)."""
    global _ctx
    if _ctx is None:
        pkg = os.path.join(_ROOT, "npu880-mtk-npu-llm-runtime_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import qmm_hip
        _ctx = qmm_hip.Context(0)
    return _ctx


def _calls(s):
    """The entry point and its arguments, as a program's call site holds them."""
    ctx = _context()
    import qmm_hip
    case, kind, ref = s["case"], s["case"]["kind"], ctypes.byref

    def at(name):
        return s[name].data_ptr() if s.get(name) is not None else None

    if kind == "beam":
        args = qmm_hip.BeamArgs(logits=at("logits"), stride=case["vocab"], vocab=case["vocab"], n_items=case["items"],
                                n_beams=case["beams"], score=at("score"), ended=at("ended"), end_token=case["vocab"] - 2,
                                n_keep=case["keep"], token=at("token"), parent=at("parent"), score_out=at("score_out"))
        ws = s["workspace"] = ctx.beam_workspace(args)
        s["keep"] = args
        call = (ctx.lib.qmm_beam_select, (ctx._h, ref(args), ws.handle))
    elif kind == "copy":
        pools = (qmm_hip.SlotPool * case["pools"])(*[(p.data_ptr(), case["slot_bytes"], case["slots"]) for p in s["pools"]])
        s["keep"] = pools
        call = (ctx.lib.qmm_copy_slots, (ctx._h, pools, case["pools"], at("src"), at("dst"), case["pairs"]))
    else:
        batch = qmm_hip.StateBatch(n_seqs=case["seqs"], n_rows=s["rows"], row_start=at("row_start"), slot_in=at("slot_in"),
                                   slot_out=at("slot_out"), n_slots=2 * case["seqs"], max_new=s["max_new"])
        if kind == "conv":
            Ch = case["channels"]
            args = qmm_hip.ConvArgs(x=at("x"), x_stride=Ch, channels=Ch, width=case["width"], weight=at("weight"), bias=at("bias"),
                                    state=at("state"), silu=1, out=at("out"), out_stride=Ch)
            call = (ctx.lib.qmm_short_conv, (ctx._h, ref(batch), ref(args)))
        else:
            HK, HV, DK, DV = case["qk_heads"], case["v_heads"], case["key_dim"], case["value_dim"]
            base, width = at("qkv"), s["qkv"].shape[1]
            args = qmm_hip.DeltaArgs(q=base, q_stride=width, k=base + 4 * HK * DK, k_stride=width, v=base + 8 * HK * DK, v_stride=width,
                                     qk_heads=HK, v_heads=HV, key_dim=DK, value_dim=DV, a=at("ab"), a_stride=2 * HV,
                                     b=at("ab") + 4 * HV, b_stride=2 * HV, rate=at("rate"), dt_bias=at("dt_bias"),
                                     scale=1 / math.sqrt(DK), qk_eps=EPS, state=at("state"), z=at("z"), z_stride=HV * DV,
                                     gamma=at("gamma"), gamma_eps=EPS, out=at("out"), out_stride=HV * DV)
            ws = s["workspace"] = ctx.gated_delta_workspace(batch, args)
            call = (ctx.lib.qmm_gated_delta, (ctx._h, ref(batch), ref(args), ws.handle))
        s["keep"] = batch, args
    torch.cuda.synchronize()  # the inputs were made on another stream than the library's
    return call


def run(state):
    case = state["case"]
    if own:
        entry, args = state["call"]
        rc = entry(*args)
        if rc:
            raise RuntimeError("qmm status %d: %s" % (rc, _context().last_error()))
    else:
        {"conv": _plain_conv, "delta": _plain_delta, "beam": _plain_beam, "copy": _plain_copy}[case["kind"]](state)
    if case["kind"] == "beam":
        return state["token"], state["parent"], state["score_out"]
    return state["pools"] if case["kind"] == "copy" else (state["out"], state["state"][case["seqs"]:])


# ------------------------------------------------------------- plain forms
def _start_states(s):
    """The states that the sequences start from: of their slots, or zeros."""
    slot = s["slot_in"].long()
    fresh = (slot < 0).reshape([-1] + [1] * (s["state"].dim() - 1))
    return torch.where(fresh, 0.0, s["state"][slot.clamp(min=0)])


def _padded(s):
    """Rows as [sequence, place]: the row's index, and whether there is one."""
    start = s["row_start"].long()
    place = torch.arange(s["max_new"], device=DEV)
    there = place < (start[1:] - start[:-1])[:, None]
    return torch.where(there, start[:-1, None] + place, 0), there


def _plain_conv(s):
    case = s["case"]
    W, M = case["width"], s["rows"]
    start = s["row_start"].long()
    row = torch.arange(M, device=DEV)
    seq = torch.searchsorted(start[1:].contiguous(), row, right=True)
    place, new = row - start[seq], start[1:] - start[:-1]
    # every sequence's carried inputs, then its rows, all one after another
    first = start[:-1] + (W - 1) * torch.arange(case["seqs"], device=DEV)
    tap = torch.arange(W - 1, device=DEV)
    x = torch.empty(M + case["seqs"] * (W - 1), case["channels"], device=DEV)
    x[first[:, None] + tap] = _start_states(s)
    at = first[seq] + W - 1 + place
    x[at] = s["x"]
    y = sum(x[at - (W - 1 - i)] * s["weight"][:, i] for i in range(W))
    if s["bias"] is not None:
        y = y + s["bias"]
    s["out"].copy_(y / (1 + torch.exp(-y)))
    s["state"][s["slot_out"].long()] = x[(first + new)[:, None] + tap]


def _unit(x, heads, dim):
    x = x.reshape(*x.shape[:-1], heads, dim)
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)


def _plain_delta(s):
    """By chunks of up to 64 tokens: with G the sums of the log decays, A = tril(beta k k' exp(Gi - Gj), -1) and
    T = (I + A)^-1 beta, a chunk's steps are D = T (v - exp(G) k S); its rows exp(G) q S + tril(q k' exp(Gi - Gj)) D."""
    case = s["case"]
    HK, HV, DK, DV, S = case["qk_heads"], case["v_heads"], case["key_dim"], case["value_dim"], case["seqs"]
    row, there = _padded(s)
    C = min(64, s["max_new"])
    N = -(-s["max_new"] // C)

    def chunks(x, heads):  # [M, heads, ...] -> [S, heads, N, C, ...], zeros where there is no row
        x = torch.where(there.reshape(*there.shape, *[1] * (x.dim() - 1)), x[row], 0.0)
        x = torch.cat([x, x.new_zeros(S, N * C - x.shape[1], *x.shape[2:])], 1)
        return x.reshape(S, N, C, heads, *x.shape[3:]).movedim(3, 1).contiguous()

    q, k, v = s["qkv"].split([HK * DK, HK * DK, HV * DV], 1)
    q = chunks(_unit(q, HK, DK) * (1 / math.sqrt(DK)), HK).repeat_interleave(HV // HK, 1)
    k = chunks(_unit(k, HK, DK), HK).repeat_interleave(HV // HK, 1)
    v = chunks(v.reshape(-1, HV, DV), HV)
    a, b = s["ab"].split(HV, 1)
    step = a.double() + s["dt_bias"].double()
    log_decay = s["rate"].double() * (step.clamp(min=0) + torch.log1p(torch.exp(-step.abs())))
    G = chunks(log_decay, HV).cumsum(-1)  # (64 bits: differences of long sums)
    beta = chunks(1 / (1 + torch.exp(-b)), HV)
    i = torch.arange(C, device=DEV)
    decay = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(i[:, None] < i, -math.inf)).float()
    kt = k.transpose(-1, -2).contiguous()
    A = torch.matmul(k, kt) * decay * beta[..., None]
    P = torch.matmul(q, kt) * decay
    T = torch.zeros_like(A)
    for r in range(C):  # forward substitution, all chunks and heads at once
        T[..., r, :] = -torch.matmul(A[..., r:r + 1, :r].contiguous(), T[..., :r, :])[..., 0, :] if r else 0.0
        T[..., r, r] = 1.0
    T = T * beta[..., None, :]
    grow, left = torch.exp(G).float(), torch.exp(G[..., -1:] - G).float()
    state = _start_states(s)
    out = torch.empty_like(v)
    for n in range(N):
        kn, g = k[:, :, n], grow[:, :, n, :, None]
        D = torch.matmul(T[:, :, n], v[:, :, n] - g * torch.matmul(kn, state))
        out[:, :, n] = g * torch.matmul(q[:, :, n], state) + torch.matmul(P[:, :, n], D)
        state = g[:, :, -1:] * state + torch.matmul(kt[:, :, n], left[:, :, n, :, None] * D)
    s["state"][s["slot_out"].long()] = state
    out = out.movedim(1, 3).reshape(S, N * C, HV, DV)[:, :s["max_new"]][there]
    if case["gated"]:
        z = s["z"].reshape(-1, HV, DV)
        out = out * torch.rsqrt((out * out).mean(-1, keepdim=True) + EPS) * s["gamma"] * (z / (1 + torch.exp(-z)))
    s["out"].copy_(out.reshape(-1, HV * DV))


def _plain_beam(s):
    case = s["case"]
    V, K, B = case["vocab"], case["keep"], case["beams"]
    x, score = s["logits"], s["score"].double()
    top = x.amax(-1, keepdim=True)
    ended = s["ended"] != 0
    void = (top[:, 0] == -math.inf) & ~ended | (s["score"] == -math.inf)  # no continuation but at -inf
    total = torch.exp((x - torch.where(top == -math.inf, 0.0, top)).double()).sum(-1)
    lse = top[:, 0].double() + torch.log(total)
    lse = torch.where(ended | void, 0.0, lse)
    token = torch.arange(V, device=DEV)
    x = torch.where(ended[:, None], torch.where(token == V - 2, 0.0, -math.inf), x)
    x = torch.where(void[:, None], -math.inf, x)
    # one order for values and places: the float's bits as a whole number, the lower place first
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 32) + (V - token)
    n = min(K, V)
    best = torch.topk(key, n, -1).indices  # (keys are all different)
    total = score[:, None] + (x.gather(1, best).double() - lse[:, None])
    total, order = torch.sort(total.reshape(-1, B * n), dim=-1, descending=True, stable=True)
    order = order[:, :K]
    s["parent"].copy_(order // n)
    s["token"].copy_(best.reshape(-1, B * n).gather(1, order))
    s["score_out"].copy_(total[:, :K])


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for p in s["pools"]:
        p[dst] = p[src]


# -------------------------------------------------------------------- costs
def work(case):
    if case["kind"] == "beam":
        R = case["items"] * case["beams"]  # ended beams' logits are not read; three operations a logit
        return {"bytes": 4 * R * case["vocab"] * (1 - case["ended"]) + 12 * case["items"] * case["keep"], "flops": 3 * R * case["vocab"]}
    if case["kind"] == "copy":
        return {"bytes": 2 * case["pools"] * case["pairs"] * case["slot_bytes"], "flops": 0}
    M, S = sum(_news(case)), case["seqs"]
    if case["kind"] == "conv":
        Ch, W = case["channels"], case["width"]
        return {"bytes": 4 * Ch * (2 * M + W + case["bias"] + 2 * S * (W - 1)), "flops": (2 * W + 4) * M * Ch}
    HK, HV, DK, DV = case["qk_heads"], case["v_heads"], case["key_dim"], case["value_dim"]
    row = 2 * HK * DK + HV * DV * (3 if case["gated"] else 2) + 2 * HV
    # a token decays a head's state, asks it twice and adds to it: 7 operations a value
    return {"bytes": 4 * (M * row + S * HV * DK * DV * (2 - case["fresh"])), "flops": 7 * M * HV * DK * DV}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "copy":
        pools = [p.double() for p in s["pools"]]
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            for p in pools:
                p[b] = p[a]
        return pools
    if case["kind"] == "beam":
        B, K, V = case["beams"], case["keep"], case["vocab"]
        found = torch.zeros(case["items"], K, dtype=torch.float64, device=DEV)
        for item in range(case["items"]):
            rows = slice(item * B, item * B + B)
            x = s["logits"][rows].double()
            total = s["score"][rows].double()[:, None] + torch.log_softmax(x, -1)
            total = torch.where(torch.isnan(total), -math.inf, total)
            for b in s["ended"][rows].nonzero()[:, 0].tolist():
                total[b] = -math.inf
                total[b, V - 2] = s["score"][item * B + b].double()
            found[item] = torch.topk(total.reshape(-1), K).values
        return None, None, found
    starts, into = s["row_start"].tolist(), s["slot_out"].tolist()
    new_states = s["state"].double()
    if case["kind"] == "conv":
        out = torch.zeros(s["rows"], case["channels"], dtype=torch.float64, device=DEV)
        for n, slot in enumerate(s["slot_in"].tolist()):
            x = torch.cat([s["state"][slot].double(), s["x"][starts[n]:starts[n + 1]].double()])
            y = torch.nn.functional.conv1d(x.t()[None], s["weight"].double()[:, None], None if s["bias"] is None else s["bias"].double(),
                                           groups=case["channels"])[0].t()
            out[starts[n]:starts[n + 1]] = y * torch.sigmoid(y)
            new_states[into[n]] = x[x.shape[0] - case["width"] + 1:]
        return out, new_states[case["seqs"]:]
    # the rule itself, token by token: S <- exp(g) S; S <- S + beta k (v - S'k)'; o = S'q
    HK, HV, DK, DV, S, T = case["qk_heads"], case["v_heads"], case["key_dim"], case["value_dim"], case["seqs"], s["max_new"]
    if T * S * HV * DK * DV > 6e9:
        return None
    x, of = s["qkv"].double(), HV // HK

    def unit(y):
        y = y.reshape(-1, HK, 1, DK).expand(-1, HK, of, DK).reshape(-1, HV, DK)
        return y / torch.sqrt((y ** 2).sum(-1, keepdim=True) + EPS)

    q, k, v = unit(x[:, :HK * DK]) / DK ** 0.5, unit(x[:, HK * DK:2 * HK * DK]), x[:, 2 * HK * DK:].reshape(-1, HV, DV)
    ab = s["ab"].double()
    decay = torch.exp(s["rate"].double() * torch.nn.functional.softplus(ab[:, :HV] + s["dt_bias"].double(), threshold=40.0))
    beta = torch.sigmoid(ab[:, HV:])
    state = torch.stack([s["state"][i].double() if i >= 0 else torch.zeros_like(new_states[0]) for i in s["slot_in"].tolist()])
    out = torch.zeros(s["rows"], HV, DV, dtype=torch.float64, device=DEV)
    by_len = sorted(range(S), key=lambda n: -s["news"][n])
    state, begin = state[by_len], torch.tensor([starts[n] for n in by_len], device=DEV)
    for t in range(T):
        live = sum(s["news"][n] > t for n in by_len)  # the longer sequences are in front
        r = begin[:live] + t
        S0 = state[:live]
        S0 *= decay[r][..., None, None]
        d = beta[r][..., None] * (v[r] - (S0 * k[r][..., None]).sum(-2))
        S0 += k[r][..., None] * d[..., None, :]
        out[r] = (S0 * q[r][..., None]).sum(-2)
    for n, st in zip(by_len, state):
        new_states[into[n]] = st
    if case["gated"]:
        z = s["z"].double().reshape(-1, HV, DV)
        out = out / torch.sqrt((out ** 2).mean(-1, keepdim=True) + EPS) * s["gamma"].double() * z * torch.sigmoid(z)
    return out.reshape(-1, HV * DV), new_states[S:]
