"""Performance cases of the operators that keep a state per sequence, and of those that let sequences branch.

A case is one call of one operator:
  append   a gated delta layer's projections of the new tokens: causal convolution behind each sequence's last inputs, SiLU,
           normalised queries and keys, decays and write strengths (`hq.delta_append`)
  delta    the recurrence S' = e^g S + k (beta (v - e^g S^T k))^T, o = scale S'^T q over the new tokens of many sequences, each
           from its stored state, with the output's norm and gate (`hq.delta`)
  copy     pages of a cache copied in every layer: the last pages of forked sequences, or a pool's pages moved together
           (`hq.kv_copy`)
  beam     the best continuations of groups of beams from their logits and scores (`hq.beam`)
`listed()` names the fixed cases, `draw()` gives more of the same ranges. With `own` false, `run` computes the operators
in elementary torch operations; with it true, it makes the library's calls.

Head layouts are those of the repository's 32-layer hybrid: 16 key and 32 value heads of 128 over a convolution of 4 taps in
its 24 delta layers, 4 kv heads of 256 in its 8 attention layers; vocabularies 32000 and 151936.

`lens` names the sequences of a case by their new tokens; those with a "+" go on from a stored state, the others begin.
"""
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda:0"
EPS = 1e-6


def _hq():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hilbert-pruned-8b_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import hq
    hq.device_init(0)
    return hq


# ------------------------------------------------------------------------------------ cases
def append(name, lens, k_heads=16, v_heads=32, k_dim=128, v_dim=128, taps=4, type="f32"):
    return dict(name=name, kind="append", lens=lens, k_heads=k_heads, v_heads=v_heads, k_dim=k_dim, v_dim=v_dim, taps=taps, type=type)


def delta(name, lens, k_heads=16, v_heads=32, k_dim=128, v_dim=128, gate="f32"):
    return dict(name=name, kind="delta", lens=lens, k_heads=k_heads, v_heads=v_heads, k_dim=k_dim, v_dim=v_dim, gate=gate)


def copy(name, moves, pages, partial, kv_heads=4, head_dim=256, layers=8, page=64, layout="pos"):
    return dict(name=name, kind="copy", moves=moves, pages=pages, partial=partial, kv_heads=kv_heads, head_dim=head_dim, layers=layers,
                page=page, layout=layout)


def beam(name, groups, beams, vocab, k, type="f32", masked=False, ended=False, first=False):
    return dict(name=name, kind="beam", groups=groups, beams=beams, vocab=vocab, k=k, type=type, masked=masked, ended=ended, first=first)


PROMPTS = "6001 4096 2500 1777 1024 513 300 129 37 7"


def listed():
    return [
        # sixteen sequences decoded together: launch and latency
        append("append_decode16", " ".join(["1+"] * 16)),
        # a pass of prompt chunks of three requests
        append("append_chunks2048", "1000 548+ 500+"),
        # one token of one sequence: the smallest call
        delta("delta_token", "1+", gate="none"),
        # 64 sequences decoded together
        delta("delta_decode64", " ".join(["1+"] * 64)),
        # sixteen sequences whose five drafted tokens are checked
        delta("delta_drafts16", " ".join(["5+"] * 16), gate="f16"),
        # a chunk of one long prompt
        delta("delta_chunk2048", "2048+", gate="none"),
        # whole prompts of different lengths packed into one call: the largest
        delta("delta_prompts16384", PROMPTS),
        # 32 sequences branch off: their last pages, part full, in every attention layer
        copy("copy_fork32", 32, 300, True),
        # a pool's pages moved together after sequences have left it
        copy("copy_compact192", 192, 500, False),
        # four beams of the small vocabulary
        beam("beam1x4", 1, 4, 32000, 8),
        # sixteen requests of eight beams, some of them ended, part of the vocabulary barred
        beam("beam16x8", 16, 8, 151936, 16, "f16", masked=True, ended=True),
        # 64 requests of eight beams
        beam("beam64x8", 64, 8, 151936, 16),
    ]


MOST_TOKENS = 16384 * 32 * 128 * 128  # tokens x value heads x k_dim x v_dim of a drawn delta call
MOST_COPY = 192 * 8 * 64 * 4 * 256    # moves x layers x positions x kv heads x head_dim of a drawn copy


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "delta", "delta", "delta", "copy", "beam"])
    if kind == "copy":
        kv, hd, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128, 256])
        layers = _log_int(rng, 1, 32)
        most = max(1, min(400, MOST_COPY // (layers * page * kv * hd)))
        moves = _log_int(rng, 1, most)
        return dict(kind=kind, moves=moves, pages=2 * moves + rng.randint(0, moves), partial=rng.random() < 0.5, kv_heads=kv, head_dim=hd,
                    layers=layers, page=page, layout=rng.choice(["pos", "head"]))
    if kind == "beam":
        beams = rng.randint(1, 16)
        groups = _log_int(rng, 1, 512 // beams)
        return dict(kind=kind, groups=groups, beams=beams, vocab=rng.choice([32000, 151936, _log_int(rng, 1000, 150000)]),
                    k=min(64, rng.choice([beams, 2 * beams, 2 * beams + 1])), type=rng.choice(["f16", "f32"]), masked=rng.random() < 0.3,
                    ended=rng.random() < 0.3, first=rng.random() < 0.2)
    k_heads = rng.choice([1, 2, 4, 8, 16, 16])
    v_heads = k_heads * rng.choice([1, 2, 2, 4 if k_heads < 16 else 2])
    k_dim, v_dim = rng.choice([(128, 128), (128, 128), (64, 64), (96, 192), (256, 256), (64, 128)])
    n = _log_int(rng, 1, 64)
    form = rng.choice(["decode", "few", "prompt", "mixed"])
    lens = []
    for i in range(n):
        if form == "decode" or (form == "mixed" and i):
            new = 1
        elif form == "few":
            new = rng.randint(2, 9)
        else:
            new = _log_int(rng, 1, max(16, 8192 // n))
        lens.append((new, form == "decode" or rng.random() < 0.5))
    while sum(a for a, _ in lens) * v_heads * k_dim * v_dim > MOST_TOKENS:
        lens = [(max(1, a // 2), c) for a, c in lens]
    case = dict(kind=kind, lens=" ".join(f"{a}{'+' if c else ''}" for a, c in lens), k_heads=k_heads, v_heads=v_heads, k_dim=k_dim, v_dim=v_dim)
    if kind == "append":
        return dict(case, taps=rng.choice([2, 4, 4, 4]), type=rng.choice(["f16", "f32"]))
    return dict(case, gate=rng.choice(["none", "f16", "f32"]))


# ------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _lens(case):
    return [(int(p.rstrip("+")), p.endswith("+")) for p in case["lens"].split()]


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype) * std


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _type(name):
    return torch.float16 if name == "f16" else torch.float32


def _channels(case):
    return 2 * case["k_heads"] * case["k_dim"] + case["v_heads"] * case["v_dim"]


def _slots(case):
    """Slots of the states: sequence i's stored one is i (-1: it begins), the one behind its new tokens goes to n + i."""
    n = len(_lens(case))
    return [i if c else -1 for i, (_, c) in enumerate(_lens(case))], [n + i for i in range(n)]


def _gates(g, T, H):
    """The rows that decays and write strengths come from, and their layer's parameters as layers are initialised: time steps
    of 0.001 .. 0.1, decay rates of 1 .. 16."""
    dt = torch.exp(_rand(g, H) * math.log(100) + math.log(1e-3))
    return _randn(g, T, H), _randn(g, T, H), torch.log(1 + 15 * _rand(g, H)), dt + torch.log(-torch.expm1(-dt))


def _append_inputs(case, seed):
    g = _gen(seed)
    T, n, c, H = sum(a for a, _ in _lens(case)), len(_lens(case)), _channels(case), case["v_heads"]
    a, b, a_log, dt = _gates(g, T, H)
    dt_ = _type(case["type"])
    return {"x": _randn(g, T, c).to(dt_), "a": a.to(dt_), "b": b.to(dt_), "a_log": a_log, "dt_bias": dt,
            "w": _randn(g, c, case["taps"], std=0.5), "conv": _randn(g, 2 * n, case["taps"] - 1, c)}


def _delta_inputs(case, seed):
    g = _gen(seed)
    T, n = sum(a for a, _ in _lens(case)), len(_lens(case))
    hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    x = _randn(g, T, _channels(case))
    x = x / (1 + torch.exp(-x))
    qk = x[:, :2 * hk * dk].view(T, 2 * hk, dk)  # (a view: the queries and keys of x are normalised in place)
    qk /= torch.sqrt(qk.square().sum(-1, keepdim=True) + EPS)
    a, b, a_log, dt = _gates(g, T, hv)
    y = a + dt
    s = {"qkv": x.half(), "decay": -torch.exp(a_log) * (torch.clamp(y, min=0) + torch.log1p(torch.exp(-y.abs()))), "beta": 1 / (1 + torch.exp(-b)),
         "s": _randn(g, 2 * n, hv, dk, dv, std=0.2)}
    if case["gate"] != "none":
        s["norm"], s["z"] = 1 + _randn(g, dv, std=0.1), _randn(g, T, hv * dv).to(_type(case["gate"]))
    return s


def _copy_inputs(case, seed):
    g = _gen(seed)
    inner = (case["page"], case["kv_heads"]) if case["layout"] == "pos" else (case["kv_heads"], case["page"])
    caches = [_randn(g, case["pages"], *inner, case["head_dim"], dtype=torch.float16) for _ in range(2 * case["layers"])]
    n = case["moves"]
    order = torch.randperm(case["pages"], generator=g, device=DEV).cpu().numpy().astype(np.uint32)
    part = torch.randint(1, case["page"] + 1, (n,), generator=g, device=DEV).cpu().numpy().astype(np.int32)
    return caches, order[:n].copy(), order[n:2 * n].copy(), part if case["partial"] else None


def _beam_inputs(case, seed):
    g = _gen(seed)
    G, B, V = case["groups"], case["beams"], case["vocab"]
    x = _randn(g, G * B, V, std=2.5)
    # a few likely tokens in every row, as a trained model's distribution has
    x.scatter_add_(1, torch.randint(0, V, (G * B, 8), generator=g, device=DEV), 4 + 6 * _rand(g, G * B, 8))
    if case["masked"]:
        x.masked_fill_(_rand(g, G * B, V) < 0.3, -math.inf)
    score = -5 - 20 * _rand(g, G, B)
    if case["first"]:
        score[:, 1:] = -math.inf  # a request's first step: one beam has begun
    s = {"x": x.to(_type(case["type"])), "score": score}
    if case["ended"]:
        s["done"] = (_rand(g, G, B) < 0.2).to(torch.uint8)
    return s


def prepare(case, seed):
    st = {"case": case}
    kind = case["kind"]
    if kind == "copy":
        st["caches"], st["src"], st["dst"], st["part"] = _copy_inputs(case, seed)
        page, kv, hd = case["page"], case["kv_heads"], case["head_dim"]
        if own:
            hq = st["hq"] = _hq()
            strides = (page * kv * hd, kv * hd, hd) if case["layout"] == "pos" else (page * kv * hd, hd, page * hd)
            st["kvs"] = [hq.KvCache(hq.KV_F16, case["pages"], page, kv, hd, st["caches"][2 * i].data_ptr(), st["caches"][2 * i + 1].data_ptr(), strides)
                         for i in range(case["layers"])]
        else:
            n = st["part"] if case["partial"] else np.full(case["moves"], page)
            i = np.repeat(np.arange(case["moves"]), n)
            at = [st["src"][i].astype(np.int64), st["dst"][i].astype(np.int64), np.concatenate([np.arange(m) for m in n])]
            st["at"] = [torch.from_numpy(a).to(DEV) for a in at]
        return st
    if kind == "beam":
        st.update(_beam_inputs(case, seed))
        if own:
            n = case["groups"], case["k"]
            st.update(hq=_hq(), out=torch.empty(n, device=DEV), token=torch.empty(n, device=DEV, dtype=torch.int32), beam=torch.empty(n, device=DEV, dtype=torch.int32))
        return st
    st.update(_append_inputs(case, seed) if kind == "append" else _delta_inputs(case, seed))
    lens = [a for a, _ in _lens(case)]
    src, dst = _slots(case)
    T, hv = sum(lens), case["v_heads"]
    if own:
        hq = st["hq"] = _hq()
        st["states"] = hq.States(case["k_heads"], hv, case["k_dim"], case["v_dim"], case.get("taps", 1), 2 * len(lens),
                                 st["s"].data_ptr() if kind == "delta" else None, st["conv"].data_ptr() if kind == "append" else None)
        # the step's sequences and slots, which every layer of a model shares
        st["scan"] = hq.Scan(len(lens), T)
        st["scan"].set(st["states"], lens, src, dst)
        if kind == "append":
            st.update(qkv=torch.empty(T, _channels(case), device=DEV, dtype=torch.float16), decay=torch.empty(T, hv, device=DEV), beta=torch.empty(T, hv, device=DEV))
        else:
            st["out"] = torch.empty(T, hv * case["v_dim"], device=DEV, dtype=torch.float16)
    else:
        # padded rows [sequences, longest]: the token of each place, and which places hold one
        at, most = np.cumsum([0] + lens[:-1]), max(lens)
        tok = at[:, None] + np.minimum(np.arange(most), np.array(lens)[:, None] - 1)
        st["tok"] = torch.from_numpy(tok).to(DEV)
        st["on"] = torch.from_numpy(np.arange(most) < np.array(lens)[:, None]).to(DEV)
        st["row"] = torch.from_numpy(np.concatenate([i * most + np.arange(m) for i, m in enumerate(lens)])).to(DEV)
        st["begins"] = torch.tensor([s < 0 for s in src], device=DEV)
        st["lens"] = lens
    return st


# ------------------------------------------------------------------------------------ plain forms
def _silu(x):
    return x / (1 + torch.exp(-x))


def _append_plain(st):
    case, n = st["case"], len(st["lens"])
    taps, w = case["taps"], st["w"]
    x = st["x"].float()
    old = st["conv"][:n].masked_fill(st["begins"][:, None, None], 0)
    out, at = torch.empty_like(x), 0
    for i, m in enumerate(st["lens"]):
        rows = torch.cat([old[i], x[at:at + m]])  # the inputs before the first new token, and the new ones
        out[at:at + m] = sum(rows[j:j + m] * w[:, j] for j in range(taps))
        st["conv"][n + i] = rows[m:]
        at += m
    out = _silu(out)
    T, c = out.shape[0], 2 * case["k_heads"] * case["k_dim"]
    qk = out[:, :c].reshape(T, 2 * case["k_heads"], case["k_dim"])
    qk = qk * torch.rsqrt(qk.square().sum(-1, keepdim=True) + EPS)
    y = st["a"].float() + st["dt_bias"]
    decay = -torch.exp(st["a_log"]) * (torch.clamp(y, min=0) + torch.log1p(torch.exp(-y.abs())))
    beta = 1 / (1 + torch.exp(-st["b"].float()))
    return {"qkv": torch.cat([qk.reshape(T, c), out[:, c:]], 1).half(), "decay": decay, "beta": beta, "conv": st["conv"]}


def _delta_plain(st):
    case = st["case"]
    n, hk, hv, dk, dv = len(st["lens"]), case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    rep, scale = hv // hk, 1 / math.sqrt(dk)
    x = st["qkv"].float()[st["tok"]]  # [sequences, longest, channels]
    L = x.shape[1]
    q, k = (x[..., i * hk * dk:(i + 1) * hk * dk].reshape(n, L, hk, dk).repeat_interleave(rep, 2) for i in range(2))
    v = x[..., 2 * hk * dk:].reshape(n, L, hv, dv)
    keep = torch.exp(st["decay"][st["tok"]]).masked_fill(~st["on"][..., None], 1)
    beta = st["beta"][st["tok"]].masked_fill(~st["on"][..., None], 0)
    s = st["s"][:n].masked_fill(st["begins"][:, None, None, None], 0)
    out = torch.empty(n, L, hv, dv, device=DEV)
    for t in range(L):
        s = s * keep[:, t, :, None, None]
        kt = k[:, t, :, :, None]
        u = (v[:, t] - (s * kt).sum(2)) * beta[:, t, :, None]
        s = s + kt * u[:, :, None]
        out[:, t] = (s * q[:, t, :, :, None]).sum(2)
    st["s"][n:] = s
    o = out.reshape(n * L, hv, dv)[st["row"]] * scale
    if case["gate"] != "none":
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * st["norm"] * _silu(st["z"].float()).reshape(-1, hv, dv)
    return {"out": o.reshape(-1, hv * dv).half(), "s": st["s"]}


def _copy_plain(st):
    src, dst, slot = st["at"]
    for c in st["caches"]:
        if st["case"]["layout"] == "pos":
            c[dst, slot] = c[src, slot]
        else:
            c[dst, :, slot] = c[src, :, slot]
    return {"caches": st["caches"]}


def _beam_plain(st):
    case = st["case"]
    G, B, V, k = case["groups"], case["beams"], case["vocab"], case["k"]
    best = []
    for i in range(G):
        # in 64 bits: sums of unlike rows are compared
        x = st["x"][i * B:(i + 1) * B].double()
        m = x.amax(-1, keepdim=True)
        s = st["score"][i].double()[:, None]
        val = s + (x - m - torch.log(torch.exp(x - m).sum(-1, keepdim=True)))
        if case["ended"]:
            ended = st["done"][i] != 0
            val = val.masked_fill(ended[:, None], -math.inf)
            val[:, 0] = torch.where(ended, s[:, 0], val[:, 0])  # an ended beam goes on as it is, with token 0
        top, at = torch.sort(val.reshape(-1), descending=True, stable=True)  # ties: the lowest beam, then the lowest token
        best.append((top[:k], at[:k]))
    top, at = torch.stack([b[0] for b in best]), torch.stack([b[1] for b in best])
    none = top == -math.inf
    return {"score": top.float(), "token": (at % V).masked_fill(none, -1).to(torch.int32), "beam": (at // V).masked_fill(none, -1).to(torch.int32)}


def run(st):
    case, kind = st["case"], st["case"]["kind"]
    if not own:
        return {"append": _append_plain, "delta": _delta_plain, "copy": _copy_plain, "beam": _beam_plain}[kind](st)
    hq = st["hq"]
    if kind == "append":
        hq.delta_append(st["scan"], st["states"], st["x"].data_ptr(), st["w"].data_ptr(), st["a"].data_ptr(), st["b"].data_ptr(),
                        st["a_log"].data_ptr(), st["dt_bias"].data_ptr(), st["qkv"].data_ptr(), st["decay"].data_ptr(), st["beta"].data_ptr(),
                        f32=case["type"] == "f32", eps=EPS)
        return {"qkv": st["qkv"], "decay": st["decay"], "beta": st["beta"], "conv": st["conv"]}
    if kind == "delta":
        p, c, hk = st["qkv"].data_ptr(), _channels(case), case["k_heads"] * case["k_dim"]
        g = {}
        if case["gate"] != "none":
            g = dict(norm=st["norm"].data_ptr(), gate=st["z"].data_ptr(), gate_f32=case["gate"] == "f32", eps=EPS)
        hq.delta(st["scan"], st["states"], p, p + 2 * hk, p + 4 * hk, st["decay"].data_ptr(), st["beta"].data_ptr(), st["out"].data_ptr(),
                 1 / math.sqrt(case["k_dim"]), qk_stride=c, v_stride=c, **g)
        return {"out": st["out"], "s": st["s"]}
    if kind == "copy":
        hq.kv_copy(st["kvs"], st["src"], st["dst"], st["part"])
        return {"caches": st["caches"]}
    hq.beam(st["x"].data_ptr(), case["groups"], case["beams"], case["vocab"], st["score"].data_ptr(), case["k"], st["out"].data_ptr(),
            st["token"].data_ptr(), st["beam"].data_ptr(), f32=case["type"] == "f32", done=st["done"].data_ptr() if case["ended"] else None,
            done_token=0)
    return {"score": st["out"], "token": st["token"], "beam": st["beam"]}


def work(case):
    kind = case["kind"]
    if kind == "copy":
        # a partial page holds half of one in the mean
        pos = case["moves"] * ((case["page"] + 1) / 2 if case["partial"] else case["page"])
        return {"bytes": int(pos * case["layers"] * 2 * case["kv_heads"] * case["head_dim"] * 2 * 2), "flops": 0}
    if kind == "beam":
        n, b = case["groups"] * case["beams"], 2 if case["type"] == "f16" else 4
        return {"bytes": n * case["vocab"] * b + n * 5 + case["groups"] * case["k"] * 12, "flops": 3 * n * case["vocab"]}
    lens, c, hv = _lens(case), _channels(case), case["v_heads"]
    T, n, going = sum(a for a, _ in lens), len(lens), sum(c for _, c in lens)
    if kind == "append":
        b = 2 if case["type"] == "f16" else 4
        return {"bytes": T * (c * (b + 2) + hv * (2 * b + 8)) + c * case["taps"] * 4 + (n + going) * (case["taps"] - 1) * c * 4,
                "flops": T * c * (2 * case["taps"] + 8)}
    state = hv * case["k_dim"] * case["v_dim"]
    row = c * 2 + hv * case["v_dim"] * (2 + {"none": 0, "f16": 2, "f32": 4}[case["gate"]]) + hv * 8
    return {"bytes": T * row + (n + going) * state * 4, "flops": 6 * T * state}


# ------------------------------------------------------------------------------------ float64
def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    taps, hk, dk = case["taps"], case["k_heads"], case["k_dim"]
    x, n = s["x"].double(), len(_lens(case))
    T = x.shape[0]
    conv, acc = s["conv"].double(), torch.zeros_like(x)
    t0 = 0
    for i, (m, goes) in enumerate(_lens(case)):
        for back in range(taps):  # the input `back` tokens before each
            col = s["w"][:, taps - 1 - back].double()
            if m > back:
                acc[t0 + back:t0 + m] += col * x[t0:t0 + m - back]
            for t in range(min(back, m)):
                if goes:
                    acc[t0 + t] += col * conv[i, taps - 1 + t - back]
        for j in range(taps - 1):
            t = m - (taps - 1) + j
            conv[n + i, j] = x[t0 + t] if t >= 0 else (conv[i, t + taps - 1] if goes else 0)
        t0 += m
    y = acc * torch.sigmoid(acc)
    qk = y[:, :2 * hk * dk].reshape(T, 2 * hk, dk)
    y[:, :2 * hk * dk] = (qk / (qk.pow(2).sum(-1, keepdim=True) + EPS).sqrt()).reshape(T, -1)
    return {"qkv": y, "decay": -s["a_log"].double().exp() * torch.nn.functional.softplus(s["a"].double() + s["dt_bias"].double(), threshold=1e9),
            "beta": torch.sigmoid(s["b"].double()), "conv": conv}


def _exact_delta(case, seed):
    """Chunk by chunk: within one, (I + A) U = beta (V - e^G K S) with A_ij = beta_i e^(G_i - G_j) k_i k_j below the diagonal and
    G the sums of the log decays."""
    s = _delta_inputs(case, seed)
    hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    n, T = len(_lens(case)), s["qkv"].shape[0]
    states, out = s["s"].double(), torch.empty(hv, T, dv, device=DEV, dtype=torch.float64)
    head = torch.arange(hv, device=DEV) // (hv // hk)
    x = s["qkv"].double()
    q, k = (x[:, i * hk * dk:(i + 1) * hk * dk].reshape(T, hk, dk)[:, head].transpose(0, 1).contiguous() for i in range(2))
    v = x[:, 2 * hk * dk:].reshape(T, hv, dv).transpose(0, 1).contiguous()
    g, beta = s["decay"].double().T.contiguous(), s["beta"].double().T.contiguous()
    t0 = 0
    for i, (m, goes) in enumerate(_lens(case)):
        S = states[i].clone() if goes else torch.zeros(hv, dk, dv, device=DEV, dtype=torch.float64)
        for c0 in range(t0, t0 + m, 128):
            r = slice(c0, min(c0 + 128, t0 + m))
            G = g[:, r].cumsum(-1)
            kt = k[:, r].transpose(1, 2).contiguous()
            w = torch.exp((G[:, :, None] - G[:, None, :]).tril()).tril()
            A = (beta[:, r, None] * w * torch.bmm(k[:, r].contiguous(), kt)).tril(-1)
            rhs = beta[:, r, None] * (v[:, r] - G.exp()[..., None] * torch.bmm(k[:, r].contiguous(), S))
            U = torch.linalg.solve_triangular(A, rhs, upper=False, unitriangular=True)
            out[:, r] = G.exp()[..., None] * torch.bmm(q[:, r].contiguous(), S) + torch.bmm(w * torch.bmm(q[:, r].contiguous(), kt), U)
            S = G[:, -1:, None].exp() * S + torch.bmm(kt, torch.exp(G[:, -1:] - G)[..., None] * U)
        states[n + i] = S
        t0 += m
    o = out.transpose(0, 1) / math.sqrt(dk)
    if case["gate"] != "none":
        z = s["z"].double().reshape(T, hv, dv)
        o = o / (o.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["norm"].double() * z * torch.sigmoid(z)
    return {"out": o.reshape(T, hv * dv), "s": states}


def _exact_copy(case, seed):
    caches, src, dst, part = _copy_inputs(case, seed)
    for c in caches:
        x = c if case["layout"] == "pos" else c.transpose(1, 2)
        for i, (a, b) in enumerate(zip(src.tolist(), dst.tolist())):
            m = case["page"] if part is None else int(part[i])
            x[b, :m] = x[a, :m]
    return {"caches": [c.double() for c in caches]}


def _exact_beam(case, seed):
    s = _beam_inputs(case, seed)
    B, k = case["beams"], case["k"]
    r = {n: [] for n in ("score", "token", "beam")}
    for i in range(case["groups"]):
        found = []
        for j in range(B):
            base = float(s["score"][i, j])
            if case["ended"] and int(s["done"][i, j]):
                found += [(-base, j, 0)] if base > -math.inf else []
                continue
            row = s["x"][i * B + j].double()
            lp = torch.log_softmax(row, 0)
            kth = torch.topk(row, min(k, row.numel())).values[-1]
            at = torch.nonzero(row >= kth)[:, 0]
            found += [(-(base + p), j, t) for t, p in zip(at.tolist(), lp[at].tolist()) if base + p > -math.inf]
        found = (sorted(found) + [(math.inf, -1, -1)] * k)[:k]
        r["score"].append([-f[0] for f in found]), r["beam"].append([f[1] for f in found]), r["token"].append([f[2] for f in found])
    return {"score": torch.tensor(r["score"], dtype=torch.float64, device=DEV), "token": torch.tensor(r["token"], dtype=torch.int32, device=DEV),
            "beam": torch.tensor(r["beam"], dtype=torch.int32, device=DEV)}


def exact(case, seed):
    return {"append": _exact_append, "delta": _exact_delta, "copy": _exact_copy, "beam": _exact_beam}[case["kind"]](case, seed)
