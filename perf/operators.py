"""The operators of a prompt pass, as measured: the paged cache's writer, the attention of new tokens over the paged
cache, the product in 8-bit integers, and the log probabilities of given tokens.

`own = False` computes their plain forms (elementary torch operations in fp32, rounded once at the end); `own = True`
makes the calls that a user makes of byteprof_b200. `exact` gives the same outputs in float64, written apart.
"""

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16


# ---- the cases ----------------------------------------------------------------------------------------
def listed():
    return [
        # one decoded patch of the 16-head global model: the smallest write, latency alone
        {"name": "append one token", "op": "append", "seqs": 1, "new": 1, "ctx": 700, "nh": 16, "nkv": 16, "hd": 128,
         "page": 16, "ragged": False},
        # a prompt's chunk of a grouped-head model: 4099 rows of q, k and v through the norms, the rotation, the pages
        {"name": "append 4099 rows", "op": "append", "seqs": 3, "new": 4099, "ctx": 1000, "nh": 32, "nkv": 8,
         "hd": 128, "page": 64, "ragged": True},
        # one stream's next token at the largest patch count of the byte decoder's cache
        {"name": "attend one token", "op": "attend", "seqs": 1, "new": 1, "ctx": 1023, "nh": 16, "nkv": 16, "hd": 128,
         "page": 16, "ragged": False},
        # a serving batch, a token each, lengths of all sizes, grouped heads: the cache is read once
        {"name": "attend 64 streams", "op": "attend", "seqs": 64, "new": 64, "ctx": 8191, "nh": 32, "nkv": 8,
         "hd": 128, "page": 64, "ragged": True},
        # verifying a few drafted tokens of one long stream
        {"name": "attend 5 drafts", "op": "attend", "seqs": 1, "new": 5, "ctx": 30001, "nh": 16, "nkv": 16, "hd": 128,
         "page": 32, "ragged": False},
        # prompts of several users packed into one call, nothing cached yet
        {"name": "attend 9 prompts", "op": "attend", "seqs": 9, "new": 6151, "ctx": 0, "nh": 32, "nkv": 8, "hd": 64,
         "page": 16, "ragged": True},
        # a chunk of a long prompt over what is cached of it: the largest
        {"name": "attend chunk of 4096", "op": "attend", "seqs": 1, "new": 4096, "ctx": 20480, "nh": 16, "nkv": 16,
         "hd": 128, "page": 128, "ragged": False},
        # one token through the MLP's up-projection: the weights are read once
        {"name": "int8 one row", "op": "int8", "m": 1, "k": 2048, "n": 8192},
        # an odd number of prompt rows through the down-projection
        {"name": "int8 509 rows", "op": "int8", "m": 509, "k": 8192, "n": 2048},
        # a long prompt through gate and up at once
        {"name": "int8 8192 rows", "op": "int8", "m": 8192, "k": 2048, "n": 16384},
        # the token just decoded, with twenty alternatives, as a server reports it
        {"name": "logprobs one row", "op": "logprobs", "rows": 1, "vocab": 100352, "top": 20, "dtype": "fp32"},
        # scoring a text: every token's log probability, a few alternatives
        {"name": "logprobs 1500 rows", "op": "logprobs", "rows": 1500, "vocab": 100352, "top": 5, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "int8", "logprobs"])
    if op in ("append", "attend"):
        nkv = rng.choice([1, 2, 4, 5, 8, 16])
        c = {"op": op, "nkv": nkv, "nh": nkv * rng.choice([1, 1, 2, 3, 4, 7, 8]), "hd": rng.choice([64, 128]),
             "page": rng.choice([8, 16, 32, 64, 128, 256])}
        seqs = _log(rng, 1, 96)
        if op == "append":
            c.update(seqs=seqs, new=max(seqs, _log(rng, 1, 4096)), ctx=_log(rng, 1, 4000), ragged=rng.random() < 0.7)
            while c["new"] * (c["nh"] + 2 * nkv) * c["hd"] > 4096 * 48 * 128:
                c["nh"], c["new"] = nkv, max(seqs, c["new"] // 2)
        elif rng.random() < 0.5:  # a token each
            c.update(seqs=seqs, new=seqs, ctx=_log(rng, 1, 16000), ragged=rng.random() < 0.7)
            while seqs * c["ctx"] * nkv * c["hd"] > 64 * 8192 * 8 * 128:
                c["ctx"] //= 2
        else:  # chunks
            seqs = min(seqs, 16)
            c.update(seqs=seqs, new=max(seqs, _log(rng, 2, 4096)), ctx=rng.choice([0, _log(rng, 1, 16000)]),
                     ragged=rng.random() < 0.7)
            # the padded plain form holds seqs x nh x new x (ctx + new) scores
            while seqs * c["nh"] * c["new"] * (c["ctx"] + c["new"]) * 128 > 4096 * 24576 * 16 * 128:
                c["new"], c["ctx"] = max(seqs, c["new"] // 2), c["ctx"] // 2
        return c
    if op == "int8":
        c = {"op": op, "m": _log(rng, 1, 8192), "k": 16 * _log(rng, 4, 512), "n": _log(rng, 1, 100352)}
        while c["m"] * c["k"] * c["n"] > 8192 * 2048 * 16384 or c["n"] * c["k"] > 1 << 28:
            c["n"] = max(1, c["n"] // 2)
        return c
    c = {"op": op, "rows": _log(rng, 1, 4096), "vocab": _log(rng, 2, 131072), "top": rng.choice([0, 1, 5, 20, 32]),
         "dtype": rng.choice(["fp32", "bf16"])}
    c["top"] = min(c["top"], c["vocab"])
    while c["rows"] * c["vocab"] > 700 * 100352:
        c["rows"] //= 2
    return c


# ---- inputs -------------------------------------------------------------------------------------------
def _lengths(case):
    """New rows and cached lengths of each sequence, on the host (the program knows them): the case's own."""
    s, new, ctx = case["seqs"], case["new"], case["ctx"]
    g = torch.Generator().manual_seed(s + 97 * new + 31 * ctx)
    if not case["ragged"] or s == 1:
        n = [new // s + (1 if i < new % s else 0) for i in range(s)]
        before = [ctx] * s
    else:
        extra = torch.rand(s, generator=g)
        extra = (extra / extra.sum() * (new - s)).floor().long().tolist()
        n = [1 + e for e in extra]
        n[0] += new - sum(n)
        before = (torch.rand(s, generator=g) * (ctx + 1)).floor().long().tolist()
        before[-1] = ctx
    return n, before


def _paged(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n, before = _lengths(case)
    kv = [a + b for a, b in zip(n, before)]
    page, nkv, hd = case["page"], case["nkv"], case["hd"]
    need = [-(-x // page) for x in kv]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed + 1))
    table = torch.full((len(n), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c].int()
        at += c
    starts = torch.tensor([0] + n).cumsum(0).int()
    st = {"case": case, "pages": table.to(DEV), "q_start": starts.to(DEV),
          "kv_len": torch.tensor(kv, dtype=torch.int32).to(DEV), "max_new": max(n), "max_kv": max(kv)}
    for name in ("k_pages", "v_pages"):
        st[name] = torch.randn(pool, page, nkv, hd, generator=g, device=DEV, dtype=torch.float32).to(BF16)
    return st, g


def prepare(case, seed):
    op = case["op"]
    if op == "append":
        st, g = _paged(case, seed)
        nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
        st["qkv"] = torch.randn(case["new"], (nh + 2 * nkv) * hd, generator=g, device=DEV).to(BF16)
        st["q_norm"] = (1 + 0.02 * torch.randn(nh * hd, generator=g, device=DEV)).to(BF16)
        st["k_norm"] = (1 + 0.02 * torch.randn(nkv * hd, generator=g, device=DEV)).to(BF16)
        inv = 500000.0 ** (-torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
        ang = torch.arange(st["max_kv"], dtype=torch.float64)[:, None] * inv
        st["cos"], st["sin"] = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
        return st
    if op == "attend":
        st, g = _paged(case, seed)
        # q and k have unit mean square behind their norms; a learnt norm weight sharpens the scores
        st["q"] = (2 * torch.randn(case["new"], case["nh"], case["hd"], generator=g, device=DEV)).to(BF16)
        return st
    g = torch.Generator(device=DEV).manual_seed(seed)
    if op == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        w = (torch.randn(n, k, generator=g, device=DEV) * 0.02).to(BF16).float()
        scale = (w.abs().amax(1) / 127).to(BF16)
        wq = torch.round(w / scale.float()[:, None]).clamp(-127, 127).to(torch.int8)
        # a few channels run hot, as hidden states do
        hot = 1 + 9 * (torch.rand(k, generator=g, device=DEV) < 0.01).float()
        x = (torch.randn(m, k, generator=g, device=DEV) * hot).to(BF16)
        return {"case": case, "x": x, "w": wq, "w_scale": scale}
    r, v = case["rows"], case["vocab"]
    logits = (3 * torch.randn(r, v, generator=g, device=DEV)).to(torch.float32 if case["dtype"] == "fp32" else BF16)
    return {"case": case, "logits": logits, "ids": torch.randint(0, v, (r,), generator=g, device=DEV)}


# ---- the framework's calls ----------------------------------------------------------------------------
def _own(st):
    case = st["case"]
    if case["op"] in ("append", "attend"):
        cache = st.get("cache")
        if cache is None:  # the handle that a program keeps beside its pages
            from byteprof_b200.optim.paged import PagedCache
            cache = st["cache"] = PagedCache(st["k_pages"], st["v_pages"])
        if case["op"] == "append":
            q = cache.append(st["qkv"], case["nh"], st["pages"], st["q_start"], st["kv_len"], st["q_norm"],
                             st["k_norm"], st["cos"], st["sin"], eps=1e-6)
            return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
        return cache.attend(st["q"], st["pages"], st["q_start"], st["kv_len"])
    if case["op"] == "int8":
        from byteprof_b200.quant.int8 import int8_linear
        return int8_linear(st["x"], st["w"], st["w_scale"])
    from byteprof_b200.optim.decode_ops import token_logprobs
    return _named(token_logprobs(st["logits"], st["ids"], case["top"]))


def _named(r):
    out = {"logprob": r[0], "entropy": r[1]}
    if r[2] is not None:
        out.update(top_logprob=r[2], top_id=r[3])
    return out


# ---- the plain forms ----------------------------------------------------------------------------------
def _row_places(st):
    """(sequence, index in it, position) of every packed row."""
    t = torch.arange(st["case"]["new"], device=DEV)
    start = st["q_start"].long()
    s = torch.searchsorted(start[1:], t, right=True)
    i = t - start[s]
    n = start[s + 1] - start[s]
    return s, i, st["kv_len"].long()[s] - n + i


def _norm_rope(x, w, cos, sin):
    """[T, heads, hd] fp32: RMS over all heads, the weight, the rotation of the two halves."""
    t, heads, hd = x.shape
    f = x.reshape(t, heads * hd)
    f = f * torch.rsqrt((f * f).mean(1, keepdim=True) + 1e-6) * w.float()
    a, b = f.view(t, heads, hd).split(hd // 2, dim=2)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], dim=2)


def _append(st):
    c = st["case"]
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    s, _, pos = _row_places(st)
    x = st["qkv"].float().view(c["new"], nh + 2 * nkv, hd)
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = _norm_rope(x[:, :nh], st["q_norm"], cos, sin)
    k = _norm_rope(x[:, nh:nh + nkv], st["k_norm"], cos, sin)
    slot = st["pages"].long()[s, pos // c["page"]] * c["page"] + pos % c["page"]
    st["k_pages"].view(-1, nkv, hd)[slot] = k.to(BF16)
    st["v_pages"].view(-1, nkv, hd)[slot] = x[:, nh + nkv:].to(BF16)
    return {"q": q.to(BF16), "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _attend(st):
    c = st["case"]
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    g, seqs, mq, mk = nh // nkv, c["seqs"], st["max_new"], st["max_kv"]
    j = torch.arange(mk, device=DEV)
    slot = st["pages"].long().clamp_min(0)[:, j // page] * page + j % page
    k = st["k_pages"].view(-1, nkv, hd)[slot].float().permute(0, 2, 3, 1)
    v = st["v_pages"].view(-1, nkv, hd)[slot].float().permute(0, 2, 1, 3)
    start, kv = st["q_start"].long(), st["kv_len"].long()
    i = torch.arange(mq, device=DEV)
    q = st["q"][(start[:-1, None] + i).clamp_max(c["new"] - 1)].float().view(seqs, mq, nkv, g, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, nkv, g * mq, hd)
    score = torch.matmul(q * hd ** -0.5, k).view(seqs, nkv, g, mq, mk)
    last = kv[:, None] - (start[1:] - start[:-1])[:, None] + i
    score.masked_fill_((j > last[:, :, None])[:, None, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(seqs, nkv, g * mq, mk), v).view(seqs, nkv, g, mq, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    s, i, _ = _row_places(st)
    return o[s, :, :, i].reshape(c["new"], nh, hd).to(BF16)


def _int8(st):
    x, w = st["x"].float(), st["w"].float()
    scale = (x.abs().amax(1, keepdim=True) / 127).clamp_min(1e-12)
    q = torch.round(x / scale).clamp(-127, 127)
    return (torch.matmul(q, w.t()) * scale * st["w_scale"].float()).to(BF16)


def _logprobs(st):
    x, top = st["logits"].float(), st["case"]["top"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    p = e / total
    entropy = (p * (lse - (x - m))).sum(1)
    lp = (x.gather(1, st["ids"][:, None]) - m - lse)[:, 0]
    if not top:
        return _named((lp, entropy, None, None))
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    return _named((lp, entropy, value[:, :top] - m - lse, index[:, :top]))


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "attend": _attend, "int8": _int8, "logprobs": _logprobs}[state["case"]["op"]](state)


# ---- what each has to read, write and compute ---------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "append":
        width = (case["nh"] + 2 * case["nkv"]) * case["hd"]
        return {"bytes": case["new"] * width * 4, "flops": case["new"] * width * 6}
    if op == "attend":
        n, before = _lengths(case)
        seen = sum(a * b + a * (a + 1) // 2 for a, b in zip(n, before))
        keys = sum(n) + sum(before)
        return {"bytes": keys * case["nkv"] * case["hd"] * 4 + case["new"] * case["nh"] * case["hd"] * 4,
                "flops": 4 * seen * case["nh"] * case["hd"]}
    if op == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * 2 + n * k + n * 2 + m * n * 2, "flops": 2 * m * n * k}
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 12 * case["top"]),
            "flops": 6 * case["rows"] * case["vocab"]}


# ---- the definitions in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("append", "attend"):
        start, kv, table = st["q_start"].tolist(), st["kv_len"].tolist(), st["pages"].long()
        nh, nkv, hd, page = case["nh"], case["nkv"], case["hd"], case["page"]
    if op == "append":
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        q_out = torch.zeros(case["new"], nh, hd, dtype=torch.float64, device=DEV)
        for s in range(case["seqs"]):
            a, b = start[s], start[s + 1]
            pos = torch.arange(kv[s] - (b - a), kv[s], device=DEV)
            rows = st["qkv"][a:b].double()
            got = []
            for part, weight in ((rows[:, :nh * hd], st["q_norm"]), (rows[:, nh * hd:(nh + nkv) * hd], st["k_norm"])):
                y = part / torch.sqrt(part.pow(2).sum(1, keepdim=True) / part.shape[1] + 1e-6) * weight.double()
                y = y.view(b - a, -1, 2, hd // 2)
                z = torch.complex(y[:, :, 0], y[:, :, 1]) * torch.complex(st["cos"][pos].double(),
                                                                          st["sin"][pos].double())[:, None]
                got.append(torch.cat([z.real, z.imag], dim=2))
            q_out[a:b] = got[0]
            kp[table[s, pos // page], pos % page] = got[1]
            vp[table[s, pos // page], pos % page] = rows[:, (nh + nkv) * hd:].view(b - a, nkv, hd)
        return {"q": q_out, "k_pages": kp, "v_pages": vp}
    if op == "attend":
        out = torch.zeros(case["new"], nh, hd, dtype=torch.float64, device=DEV)
        for s in range(case["seqs"]):
            a, b = start[s], start[s + 1]
            at = torch.arange(kv[s], device=DEV)
            keys = st["k_pages"][table[s, at // page], at % page].double()
            vals = st["v_pages"][table[s, at // page], at % page].double()
            hidden = at[None] > torch.arange(kv[s] - (b - a), kv[s], device=DEV)[:, None]
            for h in range(nh):
                x = st["q"][a:b, h].double() @ keys[:, h // (nh // nkv)].t() / hd ** 0.5
                out[a:b, h] = torch.softmax(x.masked_fill(hidden, float("-inf")), 1) @ vals[:, h // (nh // nkv)]
        return out
    if op == "int8":
        x = st["x"].double()
        peak = x.abs().amax(1, keepdim=True).clamp_min(127e-12)
        q = torch.round(127 * x / peak)
        y = torch.empty(case["m"], case["n"], dtype=torch.float64, device=DEV)
        for a in range(0, case["n"], 4096):
            y[:, a:a + 4096] = q @ st["w"][a:a + 4096].double().t()
        return y * (peak / 127) * st["w_scale"].double()
    lp, ent, tl, ti = [], [], [], []
    for r in range(0, case["rows"], 256):
        z = torch.log_softmax(st["logits"][r:r + 256].double(), 1)
        lp.append(z.gather(1, st["ids"][r:r + 256, None])[:, 0])
        ent.append(-(z.exp() * z).sum(1))
        if case["top"]:
            v, i = torch.sort(z, dim=1, descending=True, stable=True)
            tl.append(v[:, :case["top"]])
    return _named((torch.cat(lp), torch.cat(ent), torch.cat(tl) if tl else None, None))
