"""Performance cases of the operators of a serving loop: many sequences share one paged cache of keys and values.

A case is one call of one operator:
  append    rotary positions of the new tokens' queries and keys (one axis, or time, height and width), and their keys
            and values written into the pages of their sequences (`hq.rope_append`)
  attention the new tokens' queries over the cached positions of their sequences (`hq.attention`)
  logprobs  log probabilities of given tokens, entropy and the likeliest alternatives of rows of logits (`hq.logprobs`)
`listed()` names the fixed cases, `draw()` gives more of the same ranges. With `own` false, `run` computes the operators
in elementary torch operations in 32 bits; with it true, it makes the library's calls.

Head layouts are those of the repository's models: 8 heads of 64 (the 4-layer Llama), 32 / 8 of 128 (query width 4096,
key width 1024) and 16 / 4 of 256 with an output gate; vocabularies 32000 and 151936.

`lens` names the sequences of a case as "new@total" pairs: the last `new` of `total` positions are the call's tokens.
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
def append(name, lens, heads, kv_heads, head_dim, type="f32", rot=None, norm=False, axes=1, page=64, layout="pos"):
    return dict(name=name, kind="append", lens=lens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, type=type,
                rot=rot or head_dim, norm=norm, axes=axes, page=page, layout=layout)


def attention(name, lens, heads, kv_heads, head_dim, cache="f16", page=64, layout="pos", gate=False):
    return dict(name=name, kind="attention", lens=lens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, cache=cache,
                page=page, layout=layout, gate=gate)


def logprobs(name, rows, vocab, type="f32", ids=1, top=0, masked=False):
    return dict(name=name, kind="logprobs", rows=rows, vocab=vocab, type=type, ids=ids, top=top, masked=masked)


def _ragged(n, lo, hi, new=1):
    """n sequences of totals spread evenly over the logarithm of lo .. hi."""
    tot = [int(round(lo * (hi / lo) ** (i / max(n - 1, 1)))) for i in range(n)]
    return " ".join(f"{new}@{max(t, new)}" for t in tot)


PROMPTS = " ".join(f"{n}@{n}" for n in (6001, 4096, 2500, 1777, 1024, 513, 300, 129, 37, 7))


def listed():
    return [
        # sixteen sequences decoded together, one new token each: launch and latency
        append("append_decode16", _ragged(16, 100, 4000), 32, 8, 128),
        # a pass of prompt chunks of three requests, with q/k RMSNorm
        append("append_chunks2048", "1000@1000 548@4097 500@9001", 32, 8, 128, norm=True),
        # an image and text prompt: positions on three axes, 64 of each head's 256 dims rotated, fp16 projections
        append("append_image8191", "8191@8191", 16, 4, 256, "f16", rot=64, norm=True, axes=3, layout="head"),
        # one token of the small model behind a cached context: the smallest call
        attention("token_at1000", "1@1001", 8, 8, 64, page=16),
        # 64 sequences decoded together, their lengths spread over 200 .. 8192
        attention("decode64", _ragged(64, 200, 8192), 32, 8, 128),
        # eight long sequences decoded from an 8-bit cache
        attention("decode8_long_q8", _ragged(8, 20000, 40000), 32, 8, 128, cache="q8", page=128, layout="head"),
        # heads of 256 with the output gate: a chunk of a prompt together with 30 decoded sequences
        attention("mixed31_gated", "1000@3001 " + _ragged(30, 100, 5000), 16, 4, 256, page=32, gate=True),
        # a chunk of new tokens behind a long context
        attention("chunk512_at32k", "512@32768", 32, 8, 128),
        # whole prompts of different lengths packed into one call: the largest
        attention("prompts16384", PROMPTS, 32, 8, 128),
        # the next token's scores of the small model
        logprobs("logprobs1", 1, 32000, ids=4, top=5),
        # sixteen decoded sequences, part of the vocabulary barred, with twenty alternatives
        logprobs("logprobs16_top20", 16, 151936, "f16", ids=1, top=20, masked=True),
        # a prompt's tokens scored, with eight options each
        logprobs("logprobs512", 512, 151936, "f32", ids=8, top=5),
    ]


MOST_PAIRS = 32 * 128 * 31_800_000  # heads x head_dim x (query, position) pairs of a drawn attention call
MOST_CACHE = 140_000 * 8 * 128      # positions x kv heads x head_dim of a drawn cache


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([1, 2, 4, 8]), kv, head_dim


def _pairs(lens):
    return sum(n * t - n * (n - 1) // 2 for n, t in lens)


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "logprobs"])
    page, layout = rng.choice([16, 32, 64, 128, 256]), rng.choice(["pos", "head"])
    if kind == "logprobs":
        return dict(kind=kind, rows=_log_int(rng, 1, 512), vocab=rng.choice([32000, 151936, _log_int(rng, 1000, 150000)]),
                    type=rng.choice(["f16", "f32"]), ids=rng.randint(1, 8), top=rng.choice([0, 1, 5, 20]), masked=rng.random() < 0.3)
    heads, kv, hd = _heads(rng)
    if kind == "append":
        n = _log_int(rng, 1, 64)
        lens = []
        for _ in range(n):
            new = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, 8192 // n))
            lens.append((new, new + (0 if rng.random() < 0.4 else _log_int(rng, 1, 4000))))
        rot = rng.choice([hd, hd, hd // 2])
        return dict(kind=kind, lens=" ".join(f"{a}@{b}" for a, b in lens), heads=heads, kv_heads=kv, head_dim=hd,
                    type=rng.choice(["f16", "f32"]), rot=rot, norm=rng.random() < 0.5, axes=rng.choice([1, 1, 3]), page=page, layout=layout)
    form = rng.choice(["decode", "decode", "few", "chunk", "prompt", "mixed"])
    n = _log_int(rng, 1, 64) if form in ("decode", "few") else _log_int(rng, 1, 12)
    lens = []
    for i in range(n):
        if form == "decode" or (form == "mixed" and i):
            new, behind = 1, _log_int(rng, 1, 16384)
        elif form == "few":
            new, behind = rng.randint(2, 9), _log_int(rng, 1, 16384)
        elif form == "prompt":
            new, behind = _log_int(rng, 1, 4096), 0
        else:
            new, behind = _log_int(rng, 16, 2048), _log_int(rng, 1, 16384)
        lens.append((new, new + behind))
    while _pairs(lens) * heads * hd > MOST_PAIRS or sum(t for _, t in lens) * kv * hd > MOST_CACHE:
        lens = [(max(1, a // 2), max(1, a // 2) + (b - a) // 2) for a, b in lens]
    return dict(kind=kind, lens=" ".join(f"{a}@{b}" for a, b in lens), heads=heads, kv_heads=kv, head_dim=hd,
                cache=rng.choice(["f16", "q8"]), page=page, layout=layout, gate=rng.random() < 0.2)


# ------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _lens(case):
    return [tuple(int(x) for x in p.split("@")) for p in case["lens"].split()]


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype) * std


def _pages(case, g):
    """The page table [sequences, most pages] of a pool whose pages the sequences hold in no order, and the pool's pages."""
    need = [(t + case["page"] - 1) // case["page"] for _, t in _lens(case)]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device=DEV)[:sum(need)].cpu().numpy().astype(np.uint32)
    table = np.zeros((len(need), max(need)), np.uint32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pool


def _cache_shape(case, pool):
    inner = (case["page"], case["kv_heads"]) if case["layout"] == "pos" else (case["kv_heads"], case["page"])
    return (pool, *inner, case["head_dim"])


def _where(case):
    """Of every new token: its sequence and its position there."""
    seq, pos = [], []
    for s, (n, t) in enumerate(_lens(case)):
        seq += [s] * n
        pos += range(t - n, t)
    return np.array(seq, np.int64), np.array(pos, np.int64)


def _positions(case):
    """Positions [axes, tokens]: one axis is the place in the sequence; on three, images of 24 x 32 patches stand between
    texts of 256 tokens (a text's axes agree; an image has one time, and its rows and columns)."""
    _, pos = _where(case)
    if case["axes"] == 1:
        return pos[None]
    out = []
    for n, t in _lens(case):
        row, start = np.zeros((3, t), np.int64), 0
        i = 0
        while i < t:
            text = min(256, t - i)
            row[:, i:i + text] = start + np.arange(text)
            i, start = i + text, start + text
            img = min(24 * 32, t - i)
            p = np.arange(img)
            row[0, i:i + img], row[1, i:i + img], row[2, i:i + img] = start, start + p // 32, start + p % 32
            i, start = i + img, start + (32 if img else 0)
        out.append(row[:, t - n:])
    return np.concatenate(out, 1)


def _axis_of(case):
    """The axis of each of the rot / 2 frequencies: in turn time, height, width."""
    return (np.arange(case["rot"] // 2) % case["axes"]).astype(np.uint8)


def _table(n, rot):
    """Cosines and sines [n positions, rot / 2, 2] as a program computes them once for its model."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def _append_inputs(case, seed):
    g = _gen(seed)
    h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    dt = torch.float16 if case["type"] == "f16" else torch.float32
    T = sum(n for n, _ in _lens(case))
    pages, pool = _pages(case, g)
    pos = _positions(case)
    s = {"rows": _randn(g, T, (h + 2 * kv) * hd).to(dt),  # [q | k | v] rows of one product
         "kc": _randn(g, *_cache_shape(case, pool), dtype=torch.float16),
         "vc": _randn(g, *_cache_shape(case, pool), dtype=torch.float16),
         "table": _table(int(pos.max()) + 1, case["rot"])}
    if case["norm"]:
        s["qn"], s["kn"] = 1 + _randn(g, hd, std=0.1), 1 + _randn(g, hd, std=0.1)
    return s, pages, pool, pos


def _quantize(x):
    """8-bit codes and one fp16 scale for every position and kv head (the last axis)."""
    d = (x.float().abs().amax(-1) / 127).clamp_min(1e-7).half()
    return (x.float() / d.float()[..., None]).round().clamp(-127, 127).to(torch.int8), d


def _attention_inputs(case, seed):
    g = _gen(seed)
    h, hd = case["heads"], case["head_dim"]
    T = sum(n for n, _ in _lens(case))
    pages, pool = _pages(case, g)
    # queries and keys whose scores spread as trained models' do (standard deviation 2)
    s = {"q": _randn(g, T, h, hd, std=2.0).half(),
         "kc": _randn(g, *_cache_shape(case, pool), dtype=torch.float16),
         "vc": _randn(g, *_cache_shape(case, pool), dtype=torch.float16)}
    if case["cache"] == "q8":
        # scales lie [pages, kv heads, positions of the page]
        for n in ("k", "v"):
            s[n + "c"], d = _quantize(s[n + "c"])
            s[n + "s"] = (d.transpose(1, 2) if case["layout"] == "pos" else d).contiguous()
    if case["gate"]:
        s["qg"] = _randn(g, T, h, 2 * hd).half()  # the projection's rows: [query | gate] of each head
    return s, pages, pool


def _logprobs_inputs(case, seed):
    g = _gen(seed)
    M, V = case["rows"], case["vocab"]
    x = _randn(g, M, V, std=2.5)
    # a few likely tokens in every row, as a trained model's distribution has
    x.scatter_add_(1, torch.randint(0, V, (M, 8), generator=g, device=DEV), 4 + 6 * torch.rand(M, 8, generator=g, device=DEV))
    if case["masked"]:
        x.masked_fill_(torch.rand(M, V, generator=g, device=DEV) < 0.3, -math.inf)
    x = x.to(torch.float16 if case["type"] == "f16" else torch.float32)
    return x, torch.randint(0, V, (M, case["ids"]), generator=g, device=DEV)


def prepare(case, seed):
    st = {"case": case}
    if case["kind"] == "logprobs":
        x, ids = _logprobs_inputs(case, seed)
        st.update(x=x, ids=ids.to(torch.int32))
        if own:
            M, k = case["rows"], case["top"]
            st.update(hq=_hq(), logp=torch.empty(M, case["ids"], device=DEV), entropy=torch.empty(M, device=DEV),
                      top=torch.empty(M, k, device=DEV, dtype=torch.int32), top_logp=torch.empty(M, k, device=DEV))
        return st
    if case["kind"] == "append":
        s, pages, pool, pos = _append_inputs(case, seed)
    else:
        s, pages, pool = _attention_inputs(case, seed)
    st.update(s)
    lens, h, kv, hd, page = _lens(case), case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    T = sum(n for n, _ in lens)
    if case["kind"] == "append" and case["axes"] > 1:
        st["pos"] = torch.from_numpy(pos.astype(np.int32)).to(DEV)
    if own:
        hq = st["hq"] = _hq()
        strides = (page * kv * hd, kv * hd, hd) if case["layout"] == "pos" else (page * kv * hd, hd, page * hd)
        q8 = case.get("cache") == "q8"
        st["kv"] = hq.KvCache(hq.KV_Q8 if q8 else hq.KV_F16, pool, page, kv, hd, st["kc"].data_ptr(), st["vc"].data_ptr(), strides,
                              st["ks"].data_ptr() if q8 else None, st["vs"].data_ptr() if q8 else None)
        # the step's sequences and pages, which every layer of a model shares
        st["batch"] = hq.Batch(len(lens), T, pages.shape[1])
        st["batch"].set(st["kv"], h, [n for n, _ in lens], [t for _, t in lens], pages)
        st["out"] = torch.empty(T, h, hd, device=DEV, dtype=torch.float16)
    else:
        seq, where = _where(case)
        st["page"] = torch.from_numpy(pages[seq, where // page].astype(np.int64)).to(DEV)
        st["slot"] = torch.from_numpy(where % page).to(DEV)
        st["where"] = torch.from_numpy(pos if case["kind"] == "append" else where[None]).to(DEV)
        st["pages"] = [torch.from_numpy(pages[i, :(t + page - 1) // page].astype(np.int64)).to(DEV) for i, (_, t) in enumerate(lens)]
        if case["kind"] == "append":
            st["axis"] = torch.from_numpy(_axis_of(case).astype(np.int64)).to(DEV)
    return st


# ------------------------------------------------------------------------------------ plain forms
def _rotate_plain(x, cs, half):
    a, b = x[..., :half], x[..., half:2 * half]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def _append_plain(st):
    case = st["case"]
    h, kv, hd, half = case["heads"], case["kv_heads"], case["head_dim"], case["rot"] // 2
    T = st["rows"].shape[0]
    x = st["rows"].float().reshape(T, h + 2 * kv, hd)
    q, k, v = x[:, :h], x[:, h:h + kv], x[:, h + kv:]
    if case["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * st["qn"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * st["kn"]
    cs = st["table"][st["where"][st["axis"]].T, torch.arange(half, device=DEV)]  # [tokens, rot / 2, 2]
    q, k = _rotate_plain(q, cs, half).half(), _rotate_plain(k, cs, half).half()
    for cache, new in ((st["kc"], k), (st["vc"], v.half())):
        if case["layout"] == "pos":
            cache[st["page"], st["slot"]] = new
        else:
            cache[st["page"], :, st["slot"]] = new
    return {"q": q, "k": st["kc"], "v": st["vc"]}


def _sequence(st, name, s, total):
    """Keys or values [kv heads, positions, head_dim] of sequence s, as floats."""
    case = st["case"]
    x = st[name + "c"][st["pages"][s]].float()
    if case["layout"] == "pos":
        x = x.transpose(1, 2)
    if case["cache"] == "q8":
        x = x * st[name + "s"][st["pages"][s]].float()[..., None]
    return x.transpose(0, 1).reshape(case["kv_heads"], -1, case["head_dim"])[:, :total]


def _attention_plain(st):
    case = st["case"]
    h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    rep, scale = h // kv, 1 / math.sqrt(hd)
    out = torch.empty(st["q"].shape, device=DEV, dtype=torch.float16)
    at = 0
    for s, (n, t) in enumerate(_lens(case)):
        k, v = _sequence(st, "k", s, t), _sequence(st, "v", s, t)
        step = max(1, (1 << 28) // (t * h))  # rows at a time, so that the scores fit
        for r0 in range(0, n, step):
            r = slice(at + r0, at + min(n, r0 + step))
            m = r.stop - r.start
            q = st["q"][r].float().reshape(m, kv, rep, hd).permute(1, 2, 0, 3).reshape(kv, rep * m, hd)
            x = torch.bmm(q, k.transpose(1, 2).contiguous()).reshape(kv, rep, m, t) * scale
            limit = t - n + r0 + torch.arange(m, device=DEV)
            x = x.masked_fill(torch.arange(t, device=DEV) > limit[:, None], -math.inf)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            x = x / x.sum(-1, keepdim=True)
            y = torch.bmm(x.reshape(kv, rep * m, t), v.contiguous()).reshape(kv, rep, m, hd).permute(2, 0, 1, 3).reshape(m, h, hd)
            if case["gate"]:
                y = y / (1 + torch.exp(-st["qg"][r][..., hd:].float()))
            out[r] = y.half()
        at += n
    return {"out": out}


def _logprobs_plain(st):
    x = st["x"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lp = x - m - torch.log(z)
    ent = -(e / z * lp.masked_fill(e == 0, 0)).sum(-1)
    r = {"logp": lp.gather(1, st["ids"].long()), "entropy": ent}
    k = st["case"]["top"]
    if k:
        _, at = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lowest token first
        at = at[:, :k].contiguous()
        r["top"], r["top_logp"] = at.to(torch.int32), lp.gather(1, at)
    return r


def run(st):
    case = st["case"]
    if not own:
        return {"append": _append_plain, "attention": _attention_plain, "logprobs": _logprobs_plain}[case["kind"]](st)
    hq = st["hq"]
    if case["kind"] == "logprobs":
        k = case["top"]
        hq.logprobs(st["x"].data_ptr(), case["rows"], case["vocab"], f32=case["type"] == "f32", ids=st["ids"].data_ptr(),
                    n_ids=case["ids"], top_k=k, logp=st["logp"].data_ptr(), entropy=st["entropy"].data_ptr(),
                    top_ids=st["top"].data_ptr() if k else None, top_logp=st["top_logp"].data_ptr() if k else None)
        r = {"logp": st["logp"], "entropy": st["entropy"]}
        return dict(r, top=st["top"], top_logp=st["top_logp"]) if k else r
    h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        x, size = st["rows"], st["rows"].element_size()
        p, row = x.data_ptr(), x.shape[1]
        hq.rope_append(st["batch"], st["kv"], p, p + h * hd * size, p + (h + kv) * hd * size, st["out"].data_ptr(),
                       st["table"].data_ptr(), st["table"].shape[0], case["rot"], f32=case["type"] == "f32", q_stride=row, kv_stride=row,
                       positions=st["pos"].data_ptr() if case["axes"] > 1 else None, axis=_axis_of(case) if case["axes"] > 1 else None,
                       q_norm=st["qn"].data_ptr() if case["norm"] else None, k_norm=st["kn"].data_ptr() if case["norm"] else None, eps=EPS)
        return {"q": st["out"], "k": st["kc"], "v": st["vc"]}
    g = {}
    if case["gate"]:
        g = dict(gate=st["qg"].data_ptr() + 2 * hd, gate_stride=2 * h * hd, gate_head_stride=2 * hd)
    hq.attention(st["batch"], st["kv"], st["q"].data_ptr(), st["out"].data_ptr(), 1 / math.sqrt(hd), **g)
    return {"out": st["out"]}


def work(case):
    if case["kind"] == "logprobs":
        M, V, b = case["rows"], case["vocab"], 2 if case["type"] == "f16" else 4
        return {"bytes": M * V * b + M * (case["ids"] * 8 + 4 + case["top"] * 8), "flops": 4 * M * V}
    lens, h, kv, hd = _lens(case), case["heads"], case["kv_heads"], case["head_dim"]
    T = sum(n for n, _ in lens)
    if case["kind"] == "append":
        b = 2 if case["type"] == "f16" else 4
        return {"bytes": T * (h + 2 * kv) * hd * (b + 2) + T * case["rot"] * 4 + (12 * T if case["axes"] > 1 else 0),
                "flops": T * (h + kv) * (3 * case["rot"] + (4 * hd if case["norm"] else 0))}
    b = 2 if case["cache"] == "f16" else 1 + 2 / hd
    return {"bytes": 2 * sum(t for _, t in lens) * kv * hd * b + T * h * hd * (6 if case["gate"] else 4),
            "flops": 4 * h * hd * _pairs(lens)}


# ------------------------------------------------------------------------------------ float64
def _exact_append(case, seed):
    s, pages, _, pos = _append_inputs(case, seed)
    h, kv, hd, half = case["heads"], case["kv_heads"], case["head_dim"], case["rot"] // 2
    rows = s["rows"].double()
    T = rows.shape[0]
    cos, sin = (torch.empty(T, 1, half, device=DEV, dtype=torch.float64) for _ in range(2))
    t64 = s["table"].double()
    for i, a in enumerate(_axis_of(case)):
        at = t64[torch.from_numpy(pos[a]).to(DEV), i]
        cos[:, 0, i], sin[:, 0, i] = at[:, 0], at[:, 1]

    def turned(x, n, w):
        x = x.reshape(T, n, hd)
        if case["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
        y = x.clone()
        y[..., :half] = cos * x[..., :half] - sin * x[..., half:2 * half]
        y[..., half:2 * half] = sin * x[..., :half] + cos * x[..., half:2 * half]
        return y

    new = {"k": turned(rows[:, h * hd:(h + kv) * hd], kv, s.get("kn")), "v": rows[:, (h + kv) * hd:].reshape(T, kv, hd)}
    seq, where = _where(case)
    page, slot = torch.from_numpy(pages[seq, where // case["page"]].astype(np.int64)).to(DEV), torch.from_numpy(where % case["page"]).to(DEV)
    r = {"q": turned(rows[:, :h * hd], h, s.get("qn"))}
    for n in ("k", "v"):
        r[n] = s[n + "c"].double()
        x = r[n] if case["layout"] == "pos" else r[n].transpose(1, 2)
        x[page, slot] = new[n]
    return r


def _exact_attention(case, seed):
    s, pages, _ = _attention_inputs(case, seed)
    h, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    rep = h // kv
    out = torch.empty(s["q"].shape, device=DEV, dtype=torch.float64)
    at = 0
    for i, (n, t) in enumerate(_lens(case)):
        j = np.arange(t)
        p, o = torch.from_numpy(pages[i, j // page].astype(np.int64)).to(DEV), torch.from_numpy(j % page).to(DEV)
        for g in range(kv):
            kw = {}
            for name in ("k", "v"):
                x = (s[name + "c"][p, o, g] if case["layout"] == "pos" else s[name + "c"][p, g, o]).double()
                kw[name] = x * s[name + "s"][p, g, o].double()[:, None] if case["cache"] == "q8" else x
            kt = kw["k"].T.contiguous() / math.sqrt(hd)
            for e in range(g * rep, g * rep + rep):
                for r0 in range(0, n, 4096):
                    m = min(4096, n - r0)
                    x = s["q"][at + r0:at + r0 + m, e].double() @ kt
                    if n > 1:
                        x += torch.full((m, t), -math.inf, device=DEV, dtype=torch.float64).triu(t - n + r0 + 1)
                    out[at + r0:at + r0 + m, e] = torch.softmax(x, -1) @ kw["v"]
        at += n
    if case["gate"]:
        out = out * torch.sigmoid(s["qg"][..., hd:].double())
    return {"out": out}


def _exact_logprobs(case, seed):
    x, ids = _logprobs_inputs(case, seed)
    r = {k: [] for k in ("logp", "entropy", "top", "top_logp")}
    for i in range(case["rows"]):
        row = x[i].double()
        lp = torch.log_softmax(row, 0)
        r["logp"].append(lp[ids[i]])
        seen = lp[row > -math.inf]
        r["entropy"].append(-(seen.exp() * seen).sum())
        if case["top"]:
            # by value, then by token
            kth = torch.topk(row, case["top"]).values[-1]
            c = torch.nonzero(row >= kth)[:, 0].cpu().numpy()
            c = c[np.lexsort((c, -row[torch.from_numpy(c).to(DEV)].cpu().numpy()))][:case["top"]]
            r["top"].append(torch.from_numpy(c).to(DEV))
            r["top_logp"].append(lp[r["top"][-1]])
    r = {k: torch.stack(v) for k, v in r.items() if v}
    if case["top"]:
        r["top"] = r["top"].to(torch.int32)
    return r


def exact(case, seed):
    return {"append": _exact_append, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["kind"]](case, seed)
