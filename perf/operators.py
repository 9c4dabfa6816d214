"""Work of the batched decode operators over paged key-value caches, at the sizes that users meet.

Three operators make one step of a batch of sequences whose caches live in pages:

* ``append``: rotate the new queries and keys by their positions and write keys and values into
  the pages of their sequences;
* ``attention``: attention of the step's new tokens (one per sequence when decoding, up to 16 when
  a draft is verified) over each sequence's pages;
* ``logprobs``: log probabilities of given tokens under the step's logits, with the entropy of
  each row and its most likely alternatives.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU, ``run`` computes it in
plain torch operations (``own = False``) or through the package (``own = True``), ``work`` counts
the bytes and operations no implementation can do without, and ``exact`` is the same result in 64
bits, written from the definition.
"""

import math

import torch

own = False

VOCAB = 151936  # the vocabulary of the repository's configurations


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _attention(name, **kw):
    case = {"name": name, "op": "attention", "b": 1, "t": 1, "heads": 16, "kv_heads": 4, "dim": 128, "page": 64,
            "length": 2048, "ragged": False, "idle": False, "kv": "bf16", "window": 0}
    case.update(kw)
    return case


def _append(name, **kw):
    case = {"name": name, "op": "append", "b": 1, "t": 1, "heads": 16, "kv_heads": 4, "dim": 128, "rot": 32,
            "page": 64, "length": 2048, "ragged": False, "idle": False, "kv": "bf16", "gated": False}
    case.update(kw)
    return case


def _logprobs(name, **kw):
    case = {"name": name, "op": "logprobs", "rows": 1, "vocab": VOCAB, "pad": 0, "top": 0, "dtype": "bf16",
            "masked": False}
    case.update(kw)
    return case


def listed():
    return [
        # one sequence of the hybrid model (16 query / 4 kv heads) at its 2048-token cache: the
        # smallest decode call, where latency counts
        _attention("attention one sequence"),
        # a batch of the dense model (40 / 8 heads) with caches of different lengths up to 4096 and
        # idle slots, as a server's batch has them; small pages
        _attention("attention batch ragged", b=32, heads=40, kv_heads=8, page=16, length=4096, ragged=True, idle=True),
        # a few very long documents
        _attention("attention long context", b=2, heads=40, kv_heads=8, page=64, length=131071),
        # a draft of 7 tokens and the last emitted one verified for every sequence of a batch
        _attention("attention verify", b=8, t=8, length=4095, page=48, ragged=True),
        # a cache held in 8 bits, twice as many sequences in the same memory
        _attention("attention 8-bit cache", b=64, heads=40, kv_heads=8, page=32, length=4096, ragged=True, kv="e4m3"),
        # one new token for every sequence of a batch of the dense model
        _append("append decode", b=32, heads=40, kv_heads=8, rot=128, page=16, length=4096, ragged=True, idle=True),
        # a prompt of the dense model goes into its pages at once
        _append("append prompt", t=8191, heads=40, kv_heads=8, rot=128, length=0),
        # drafts of the hybrid model into 8-bit pages, queries interleaved with their gates
        _append("append verify 8-bit", b=16, t=8, page=32, length=131001, ragged=True, kv="e4m3", gated=True),
        # the token just decoded and its 20 most likely alternatives
        _logprobs("logprobs one row", top=20),
        # the rows of a verified draft, 5 alternatives each, over f32 logits (after penalties)
        _logprobs("logprobs verify", rows=16, top=5, dtype="f32", masked=True),
        # a batch of rows with the alternatives a serving API returns at most
        _logprobs("logprobs batch", rows=509, top=20),
        # scoring a text: every token's log probability and entropy, no alternatives; rows that
        # start at odd addresses
        _logprobs("logprobs scoring", rows=1024, vocab=VOCAB - 1, pad=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "logprobs"])
    if op == "logprobs":
        vocab = _log_int(rng, 1000, VOCAB)
        dtype = rng.choice(["bf16", "f32"])
        rows = _log_int(rng, 1, max(1, min(4096, 75_000_000 // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, 3, 64]), "top": rng.choice([0, 1, 5, 20, 32]),
                "dtype": dtype, "masked": rng.random() < 0.3}
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    kv = rng.choice(["bf16", "bf16", "e4m3"])
    b = _log_int(rng, 1, 96)
    case = {"op": op, "b": b, "t": 1, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "length": 1,
            "ragged": rng.random() < 0.6, "idle": rng.random() < 0.3, "kv": kv}
    if op == "attention":
        case["t"] = rng.choice([1, 1, 1, 2, 5, 8, 16])
        wide = max(1, case["t"] * heads // kv_heads // 32)  # many rows per key cost operations, not bytes
        case["length"] = _log_int(rng, 1, max(1, min(131072, 200_000_000 // (b * kv_heads * dim * wide))))
        case["window"] = rng.choice([0, 0, 0, 500, 4000])
    else:
        case["rot"] = rng.choice([0, 32, 64, dim])
        case["t"] = _log_int(rng, 1, max(1, min(8192, 20_000_000 // (b * (heads + 2 * kv_heads) * dim))))
        case["length"] = _log_int(rng, 1, max(1, min(131072, 20_000_000 // (b * kv_heads * dim))))
        case["gated"] = rng.random() < 0.3
    return case


def _steps(case):
    """Per sequence: tokens in the cache before the step, and new tokens (0: an idle slot)."""
    b, t, n = case["b"], case["t"], case["length"]
    lengths = [n - (i * i * 37 + i * 101) % max(1, n // 2) if case["ragged"] else n for i in range(b)]
    counts = [0 if case["idle"] and i % 8 == 5 else (max(1, t - i % 3) if case["ragged"] else t) for i in range(b)]
    return lengths, counts


def work(case):
    if case["op"] == "logprobs":
        size = 2 if case["dtype"] == "bf16" else 4
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": n * v * size + n * (4 + 8 + 8 * k), "flops": 5 * n * v}
    lengths, counts = _steps(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    size = 2 if case["kv"] == "bf16" else 1
    if case["op"] == "append":
        new = sum(counts)
        read = new * (hq + 2 * hk) * d * 2
        return {"bytes": read + case["b"] * case["t"] * hq * d * 2 + new * 2 * hk * d * size,
                "flops": 3 * new * (hq + hk) * case["rot"]}
    seen = keys = 0
    for n, c in zip(lengths, counts):
        first = max(0, n - case["window"] + 1) if case["window"] else 0
        keys += (n + c - first) if c else 0
        seen += sum(min(n + i + 1, case["window"] or n + i + 1) for i in range(c))
    io = case["b"] * case["t"] * hq * (2 * d * 2 + 4)
    return {"bytes": keys * hk * d * 2 * size + io, "flops": 4 * seen * hq * d}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    if case["op"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        logits = normal(n, v + case["pad"], dtype=dtype, std=2.5)[:, :v]
        if case["masked"]:  # a grammar or a bad-words list rules most of the vocabulary out
            logits.masked_fill_(torch.rand(n, v, generator=gen, device=dev) < 0.9, -math.inf)
        tokens = torch.randint(0, v, (n,), generator=gen, device=dev, dtype=torch.int32)
        return {"case": case, "logits": logits, "tokens": tokens}

    lengths, counts = _steps(case)
    b, t, hq, hk, d, page = (case[k] for k in ("b", "t", "heads", "kv_heads", "dim", "page"))
    width = (max(lengths) + t + page - 1) // page
    # pages are handed out in no particular order, with some to spare
    pages = b * width + 3
    table = torch.randperm(pages, generator=gen, device=dev)[:b * width].to(torch.int32).view(b, width)
    state = {"case": case, "table": table, "k_scale": None, "v_scale": None, "counts": None,
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev)}
    if case["ragged"] or case["idle"]:
        state["counts"] = torch.tensor(counts, dtype=torch.int32, device=dev)
    pool = [normal(pages, hk, page, d) for _ in range(2)]
    if case["kv"] == "e4m3":  # calibrated per head: what the cache holds is the value over its scale
        for name in ("k_scale", "v_scale"):
            state[name] = 0.01 + 0.02 * torch.rand(hk, generator=gen, device=dev)
        pool = [(x.float() / state[s][:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
                for x, s in zip(pool, ("k_scale", "v_scale"))]
    state["k_pages"], state["v_pages"] = pool
    if case["op"] == "attention":
        state["q"] = normal(b, t, hq, d)
        state["window"] = case["window"] or None
        return state
    # the step's fused projection: queries (each followed by its gate in a gated model), keys, values
    per = 2 * d if case["gated"] else d
    rows = normal(b, t, hq * per + 2 * hk * d)
    state["q"] = rows[..., :hq * per].unflatten(-1, (hq, per))[..., :d]
    state["k"] = rows[..., hq * per:hq * per + hk * d].unflatten(-1, (hk, d))
    state["v"] = rows[..., hq * per + hk * d:].unflatten(-1, (hk, d))
    half = case["rot"] // 2
    state["inv_freq"] = None
    if half:
        state["inv_freq"] = 1e6 ** (-torch.arange(half, device=dev, dtype=torch.float32) / half)
    return state


# ---------------------------------------------------------------------------------------------
# the plain forms and the package's calls
# ---------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        from skinny_mlx_b200 import logprobs, paged

        if op == "logprobs":
            r = logprobs.token_logprobs(state["logits"], state["tokens"], top_n=state["case"]["top"])
            return {"logprobs": r.logprobs, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_ids": r.top_ids}
        if op == "attention":
            o, lse = paged.attention(state["q"], state["k_pages"], state["v_pages"], state["table"], state["lengths"],
                                     counts=state["counts"], window=state["window"], k_scale=state["k_scale"],
                                     v_scale=state["v_scale"], return_lse=True)
            return {"o": o, "lse": lse}
        q = paged.append(state["q"], state["k"], state["v"], state["k_pages"], state["v_pages"], state["table"],
                         state["lengths"], state["inv_freq"], counts=state["counts"], k_scale=state["k_scale"],
                         v_scale=state["v_scale"])
        return {"q": q, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}
    return {"logprobs": _plain_logprobs, "attention": _plain_attention, "append": _plain_append}[op](state)


def _plain_logprobs(state):
    x = state["logits"].float() + 0.0  # (-0 and 0 are one value)
    n, v = x.shape
    top = state["case"]["top"]
    m = x.amax(-1, keepdim=True)
    lse = m + (x - m).exp().sum(-1, keepdim=True).log()
    y = x - lse
    p = y.exp()
    entropy = -(p * torch.where(p > 0, y, 0.0)).sum(-1)
    logprobs = y.gather(1, state["tokens"].long()[:, None])[:, 0]
    # the order of the values, ties to the lowest index, as one whole number per logit
    bits = x.view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = order * 2 ** 32 + (v - 1 - torch.arange(v, device=x.device))
    ids = v - 1 - (key.topk(top, dim=-1).values & 0xFFFFFFFF)
    return {"logprobs": logprobs, "entropy": entropy, "top_logprobs": y.gather(1, ids), "top_ids": ids.to(torch.int32)}


def _cached(pages, table, scale):
    """[b, kv head, position, dim] f32 of every sequence's pages, in order."""
    x = pages.view(torch.uint8)[table.long()].view(torch.float8_e4m3fn).float() * scale[:, None, None] \
        if scale is not None else pages[table.long()].float()
    b, w, h, page, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, w * page, d)


def _plain_attention(state):
    q = state["q"].float()
    b, t, hq, d = q.shape
    hk = state["k_pages"].shape[1]
    dev = q.device
    k = _cached(state["k_pages"], state["table"], state["k_scale"])
    v = _cached(state["v_pages"], state["table"], state["v_scale"])
    new = torch.arange(t, device=dev)
    counts = state["counts"] if state["counts"] is not None else torch.full((b,), t, device=dev)
    at = (state["lengths"][:, None] + new)[:, :, None]                     # [b, t, 1] a query's position
    j = torch.arange(k.shape[2], device=dev)
    seen = (j <= at) & (new < counts[:, None])[:, :, None]
    if state["window"] is not None:
        seen &= j > at - state["window"]
    seen = seen.repeat_interleave(hq // hk, 1)[:, None]                     # rows (t, head in the group)
    s = q.view(b, t, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d) @ k.transpose(2, 3)
    s = torch.where(seen, s * (1.0 / math.sqrt(d)), -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.where(seen, (s - torch.where(m == -math.inf, 0.0, m)).exp(), 0.0)
    z = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(z == 0, 1.0, z)
    lse = m + z.log()
    back = lambda x: x.view(b, hk, t, hq // hk, -1).permute(0, 2, 1, 3, 4).reshape(b, t, hq, -1)
    return {"o": back(o).to(torch.bfloat16), "lse": back(lse)[..., 0].contiguous()}


def _plain_append(state):
    q, k, v = state["q"].float(), state["k"].float(), state["v"].float()
    b, t = q.shape[:2]
    dev = q.device
    page = state["k_pages"].shape[2]
    new = torch.arange(t, device=dev)
    at = state["lengths"][:, None].long() + new
    real = torch.ones(b, t, dtype=torch.bool, device=dev)
    if state["counts"] is not None:
        real = new < state["counts"][:, None]
    if state["inv_freq"] is not None:
        ang = at.double()[..., None] * state["inv_freq"].double()
        cos, sin = ang.cos().float()[:, :, None], ang.sin().float()[:, :, None]
        half = cos.shape[-1]

        def turn(x):
            x1, x2 = x[..., :half], x[..., half:2 * half]
            return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin, x[..., 2 * half:]], -1)

        q, k = turn(q), turn(k)
    where = state["table"].long().gather(1, at // page)
    slot = at % page
    for x, pages, scale in ((k, state["k_pages"], state["k_scale"]), (v, state["v_pages"], state["v_scale"])):
        if scale is not None:
            x = (x / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            pages = pages.view(torch.uint8)
        else:
            x = x.to(torch.bfloat16)
        pages[where, :, slot] = torch.where(real[..., None, None], x, pages[where, :, slot])
    q = torch.where(real[..., None, None], q, 0.0)
    return {"q": q.to(torch.bfloat16), "k_pages": state["k_pages"], "v_pages": state["v_pages"]}


# ---------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "logprobs":
        rows = []
        for x, tok in zip(state["logits"], state["tokens"]):
            y = torch.log_softmax(x.double(), 0)
            values, ids = torch.sort(x.double(), descending=True, stable=True)
            p = y.exp()
            rows.append((y[tok.long()], -torch.special.xlogy(p, p).sum(), y[ids[:case["top"]]], ids[:case["top"]]))
        lp, ent, top, ids = (torch.stack(c) for c in zip(*rows))
        return {"logprobs": lp, "entropy": ent, "top_logprobs": top, "top_ids": ids}
    lengths, counts = _steps(case)
    b, t, hq, hk, d, page = (case[n] for n in ("b", "t", "heads", "kv_heads", "dim", "page"))
    table = state["table"].long()
    scales = [torch.ones(hk, device=table.device) if state[n] is None else state[n] for n in ("k_scale", "v_scale")]
    scales = [s.double()[:, None, None] for s in scales]
    if case["op"] == "attention":
        o = torch.zeros(b, t, hq, d, dtype=torch.float64, device=table.device)
        lse = torch.full((b, t, hq), -math.inf, dtype=torch.float64, device=table.device)
        for i in range(b):
            kv = [pool[table[i]].transpose(0, 1).reshape(hk, -1, d).double() * s
                  for pool, s in zip((state["k_pages"], state["v_pages"]), scales)]
            for c in range(counts[i]):
                end = lengths[i] + c + 1
                beg = max(0, end - case["window"]) if case["window"] else 0
                k, v = (x[:, beg:end] for x in kv)
                s = torch.einsum("hrd,hnd->hrn", state["q"][i, c].double().view(hk, -1, d), k) / math.sqrt(d)
                o[i, c] = (torch.softmax(s, -1) @ v).reshape(hq, d)
                lse[i, c] = torch.logsumexp(s, -1).reshape(hq)
        return {"o": o, "lse": lse}
    half = case["rot"] // 2
    q_out = torch.zeros(b, t, hq, d, dtype=torch.float64, device=table.device)
    pools = [state["k_pages"].double(), state["v_pages"].double()]
    for i in range(b):
        c = counts[i]
        if not c:
            continue
        at = lengths[i] + torch.arange(c, device=table.device)
        q, k, v = (state[n][i, :c].double() for n in "qkv")
        if half:
            turn = torch.polar(torch.ones(c, half, dtype=torch.float64, device=table.device),
                               at.double()[:, None] * state["inv_freq"].double())[:, None]
            for x in (q, k):
                z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
                x[..., :half], x[..., half:2 * half] = z.real, z.imag
        q_out[i, :c] = q
        for x, pool, s in zip((k, v), pools, scales):
            pool[table[i, at // page], :, at % page] = x / s[:, :, 0]
    return {"q": q_out, "k_pages": pools[0], "v_pages": pools[1]}
