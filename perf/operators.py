"""Cases of the speculative decoding step: attention of a few drafted tokens of every request over the paged
cache, temperature / top-p sampling, and the verification of drafted tokens against the target's distribution."""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2}


# ---- cases ---------------------------------------------------------------------------------------------------------------
def _chunk(name, batch, kv_lo, kv_hi, new_lo, new_hi, hq, hkv, d, page, dtype):
    c = {"op": "chunk", "batch": batch, "kv_lo": kv_lo, "kv_hi": kv_hi, "new_lo": new_lo, "new_hi": new_hi, "hq": hq,
         "hkv": hkv, "d": d, "page": page, "dtype": dtype}
    return dict(c, name=name) if name else c


def _sample(name, rows, vocab, dtype, temps, top_p, probs):
    c = {"op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temps": temps, "top_p": top_p, "probs": probs}
    return dict(c, name=name) if name else c


def _verify(name, batch, n_lo, n_hi, vocab, dtype, temps, top_p, probs):
    c = {"op": "verify", "batch": batch, "n_lo": n_lo, "n_hi": n_hi, "vocab": vocab, "dtype": dtype, "temps": temps,
         "top_p": top_p, "probs": probs}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one conversation with a long context: four drafted tokens and the last sampled one
        _chunk("chunk_one_long", 1, 65536, 65536, 5, 5, 32, 8, 128, 16, "bfloat16"),
        # a pipeline microbatch of a 64-head model, each request with its own number of drafts
        _chunk("chunk_microbatch", 128, 512, 4096, 1, 8, 64, 8, 128, 16, "bfloat16"),
        # two short chats: launch and merge latency
        _chunk("chunk_two_short", 2, 90, 110, 2, 4, 8, 2, 64, 16, "float16"),
        # long re-reads of a cached prefix (a tool's answer, a continued document)
        _chunk("chunk_long_new", 16, 3000, 8192, 100, 257, 32, 8, 128, 16, "bfloat16"),
        # the small fp32 configuration that results are checked on
        _chunk("chunk_fp32", 4, 100, 300, 3, 3, 8, 2, 64, 16, "float32"),
        # one interactive request
        _sample("sample_one", 1, 128256, "bfloat16", "fixed", "nucleus", False),
        # a microbatch whose requests bring their own parameters, greedy ones among them
        _sample("sample_microbatch", 128, 128256, "bfloat16", "mixed", "mixed", False),
        # all sequences of a large offline job, plain temperature sampling
        _sample("sample_offline", 1024, 128256, "bfloat16", "fixed", "one", False),
        # a draft model's step: its probabilities are kept for the verification
        _sample("sample_draft_probs", 64, 32003, "float32", "fixed", "nucleus", True),
        # a few interactive requests with four drafts each
        _verify("verify_interactive", 4, 4, 4, 128256, "bfloat16", "fixed", "one", True),
        # a microbatch with ragged drafts and mixed parameters
        _verify("verify_microbatch", 128, 0, 7, 128256, "bfloat16", "mixed", "mixed", True),
        # drafts looked up in the prompt (no draft distribution), odd vocabulary
        _verify("verify_lookup", 64, 1, 8, 32003, "float16", "mixed", "nucleus", False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk", "sample", "verify"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "chunk":
        hkv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 5, 8])
        d = rng.choice([64, 128])
        small = dtype == "float32"  # the type that results are checked in, on small models
        new_hi = _log(rng, 1, 32 if small else 200)
        hi = max(_log(rng, 40, 4000 if small else 60000), new_hi)
        batch = max(1, min(_log(rng, 1, 128), (60000 if small else 250000) // hi, 3000 // new_hi))
        return _chunk(None, batch, rng.randint(max(1, hi // 8), hi), hi, rng.randint(1, new_hi), new_hi, hkv * group, hkv, d,
                      rng.choice([8, 16, 16, 32]), dtype)
    vocab = _log(rng, 1000, 131072)
    temps, top_p = rng.choice(["fixed", "mixed"]), rng.choice(["one", "nucleus", "mixed"])
    if op == "sample":
        return _sample(None, min(_log(rng, 1, 512), 60000000 // vocab), vocab, dtype, temps, top_p, rng.random() < 0.3)
    n_hi = rng.randint(1, 8)
    return _verify(None, _log(rng, 1, 100), rng.randint(0, n_hi), n_hi, vocab, dtype, temps, top_p, rng.random() < 0.7)


# ---- what is in hand before the call ---------------------------------------------------------------------------------------
def _spread(lo, hi, n, gen):
    return torch.randint(lo, hi + 1, (n,), generator=gen).tolist()


def _chunk_lengths(case):
    """Cache length and new tokens of every request: a matter of the case, so that outputs of all seeds have one shape."""
    gen = torch.Generator().manual_seed(case["batch"])
    lens = _spread(case["kv_lo"], case["kv_hi"], case["batch"], gen)
    return lens, [min(n, m) for n, m in zip(_spread(case["new_lo"], case["new_hi"], case["batch"], gen), lens)]


def _cumsum(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _logits(rows, vocab, dtype, g):
    # a heavy-tailed vocabulary: exponential scores give Zipf-like probabilities; the last entries are padding that no
    # token owns
    x = torch.empty(rows, vocab, device=DEV).exponential_(generator=g).mul_(1.3)
    x += 0.5 * torch.randn(rows, vocab, device=DEV, generator=g)
    x[:, vocab - vocab // 200:] = -math.inf
    return x.to(dtype)


def _params(case, n, gen):
    temps = {"fixed": [0.8], "mixed": [0.0, 0.6, 0.8, 1.0, 1.2]}[case["temps"]]
    top_p = {"one": [1.0], "nucleus": [0.9, 0.95], "mixed": [1.0, 0.95, 0.9, 0.8]}[case["top_p"]]
    pick = lambda v: torch.tensor([v[i] for i in _spread(0, len(v) - 1, n, gen)], dtype=torch.float32, device=DEV)
    return pick(temps), pick(top_p)


def prepare(case, seed):
    g, gen = torch.Generator(device=DEV).manual_seed(seed), torch.Generator().manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"op": case["op"]}
    if case["op"] == "chunk":
        b, ps = case["batch"], case["page"]
        lens, new = _chunk_lengths(case)
        pages = [-(-n // ps) for n in lens]
        total = sum(pages)
        pool = total + total // 8 + 1
        qo, kvp = _cumsum(new), _cumsum(pages)
        s.update(lens=_i32(lens), new=_i32(new), pages_of=_i32(pages), qo=_i32(qo), kv_indptr=_i32(kvp),
                 last=_i32([(n - 1) % ps + 1 for n in lens]), max_new=max(new), max_pages=max(pages), batch=b,
                 kv_indices=torch.randperm(pool, generator=gen)[:total].to(torch.int32).to(DEV),
                 pages=torch.empty(pool, 2, ps, case["hkv"], case["d"], dtype=dtype, device=DEV).normal_(generator=g),
                 q=torch.empty(qo[-1], case["hq"], case["d"], dtype=dtype, device=DEV).normal_(generator=g))
        if own:  # the step's plan: one for all layers of the model
            from deserve_b200 import ops
            s["wrapper"] = ops.BatchChunkWithPagedKVCacheWrapper(torch.empty(256 << 20, dtype=torch.uint8, device=DEV))
            s["wrapper"].begin_forward(s["qo"], s["kv_indptr"], s["kv_indices"], s["last"], case["hq"], case["hkv"], case["d"],
                                       ps, dtype, qo_indptr_host=s["qo"].cpu().numpy(), kv_indptr_host=s["kv_indptr"].cpu().numpy())
            s["lse"] = torch.empty(qo[-1], case["hq"], dtype=torch.float32, device=DEV)
        return s
    if case["op"] == "sample":
        n = case["rows"]
        s["logits"] = _logits(n, case["vocab"], dtype, g)
        s["temperature"], s["top_p"] = _params(case, n, gen)
        s["uniform"] = torch.rand(n, device=DEV, generator=g)
        s["probs"] = torch.empty(n, case["vocab"], device=DEV) if case["probs"] else None
        return s
    b = case["batch"]
    rows = [n + 1 for n in _spread(case["n_lo"], case["n_hi"], b, gen)]
    indptr = _cumsum(rows)
    nnz = indptr[-1]
    s["logits"] = _logits(nnz, case["vocab"], dtype, g)
    s["temperature"], s["top_p"] = _params(case, b, gen)
    s["uniform"] = torch.rand(nnz, device=DEV, generator=g)
    s["indptr"] = _i32(indptr)
    s["batch"], s["max_rows"] = b, max(rows)
    owner = torch.repeat_interleave(torch.arange(b, device=DEV), torch.tensor(rows, device=DEV))
    # the draft model sees nearly the same scores; each draft is drawn from its distribution
    t = s["temperature"][owner, None]
    z = s["logits"].float() / torch.where(t > 0, t, torch.ones_like(t))
    z += 0.7 * torch.randn(z.shape, device=DEV, generator=g)
    q = torch.softmax(torch.where(t > 0, z, z * 1e4), dim=1)
    noise = torch.empty_like(q).exponential_(generator=g)
    drafted = torch.argmax(q / noise, dim=1).to(torch.int32)  # a draw from every row of q
    del noise, z
    s["tokens"] = torch.cat([drafted[-1:], drafted[:-1]])  # row j of a request proposes the token at j + 1
    s["draft_probs"] = q if case["probs"] else None
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        from deserve_b200 import ops
        if s["op"] == "chunk":
            return {"out": s["wrapper"].forward(s["q"], s["pages"], lse=s["lse"]), "lse": s["lse"]}
        if s["op"] == "sample":
            tokens = ops.sample_top_p(s["logits"], s["temperature"], s["top_p"], s["uniform"], probs=s["probs"])
            return {"tokens": tokens} if s["probs"] is None else {"tokens": tokens, "probs": s["probs"]}
        accepted, tokens = ops.verify_draft(s["logits"], s["tokens"], s["indptr"], s["uniform"], s["temperature"], s["top_p"],
                                            draft_probs=s["draft_probs"])
        return {"accepted": accepted, "tokens": tokens}
    return {"chunk": _plain_chunk, "sample": _plain_sample, "verify": _plain_verify}[s["op"]](s)


def _plain_chunk(s):
    """Every request padded to the longest, products in fp32."""
    q, pages = s["q"], s["pages"]
    _, _, ps, hkv, d = pages.shape
    b, hq = s["batch"], q.shape[1]
    group = hq // hkv
    at = torch.arange(s["max_pages"], device=DEV)
    live = at[None] < s["pages_of"][:, None]
    ids = s["kv_indices"][torch.where(live, s["kv_indptr"][:-1, None] + at, 0)].long()
    length = s["max_pages"] * ps
    k = pages[ids, 0].reshape(b, length, hkv, d).permute(0, 2, 3, 1).float()
    v = pages[ids, 1].reshape(b, length, hkv, d).permute(0, 2, 1, 3).float()
    t, j = torch.arange(length, device=DEV), torch.arange(s["max_new"], device=DEV)
    v = torch.where((t[None] < s["lens"][:, None])[:, None, :, None], v, 0.0)
    row = torch.where(j[None] < s["new"][:, None], s["qo"][:-1, None] + j, 0)
    qp = q[row].float().view(b, -1, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    x = (qp @ k) / math.sqrt(d)
    seen = t[None, None] <= (s["lens"] - s["new"])[:, None, None] + j[None, :, None]
    seen = seen[:, None].expand(b, hkv, s["max_new"], length).repeat_interleave(group, dim=2)
    x = torch.where(seen, x, -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(dim=-1, keepdim=True)
    o = (e @ v) / total
    lse = (top + torch.log(total)).squeeze(-1)
    o = o.view(b, hkv, -1, group, d).permute(0, 2, 1, 3, 4).reshape(b, -1, hq, d)
    lse = lse.view(b, hkv, -1, group).permute(0, 2, 1, 3).reshape(b, -1, hq)
    keep = j[None] < s["new"][:, None]
    return {"out": o[keep].to(q.dtype), "lse": lse[keep]}


def _plain_probs(logits, temperature, top_p):
    """Kept probabilities of every row, in 64 bits: the order of the running sums must not decide a token."""
    x = logits.double()
    greedy = temperature[:, None] <= 0
    z = x / torch.where(greedy, 1.0, temperature.double()[:, None])
    w = torch.exp(z - z.amax(dim=1, keepdim=True))
    first = torch.zeros_like(w).scatter_(1, logits.argmax(dim=1, keepdim=True), 1.0)
    w = torch.where(greedy, first, w)
    ranked, order = torch.sort(logits, dim=1, descending=True, stable=True)
    ws = torch.where(greedy, w, w.gather(1, order))
    before = torch.cumsum(ws, dim=1) - ws
    keep = (before <= top_p.double()[:, None] * w.sum(dim=1, keepdim=True)) | (top_p[:, None] >= 1) | greedy
    keep = torch.where(greedy, keep, torch.empty_like(keep).scatter_(1, order, keep))
    w = torch.where(keep, w, 0.0)
    return w / w.sum(dim=1, keepdim=True)


def _plain_draw(w, u):
    """First index whose running sum exceeds u times the whole."""
    c = torch.cumsum(w, dim=1)
    return (c <= u.double()[:, None] * c[:, -1:]).sum(dim=1)


def _plain_sample(s):
    p = _plain_probs(s["logits"], s["temperature"], s["top_p"])
    tokens = _plain_draw(p, s["uniform"]).to(torch.int32)
    return {"tokens": tokens} if s["probs"] is None else {"tokens": tokens, "probs": p.float()}


def _plain_verify(s):
    begin, end = s["indptr"][:-1].long(), s["indptr"][1:].long()
    nnz, vocab = s["logits"].shape
    r = torch.arange(nnz, device=DEV)
    owner = torch.searchsorted(end, r, right=True)
    p = _plain_probs(s["logits"], s["temperature"][owner], s["top_p"][owner])
    draft = s["tokens"][(r + 1) % nnz].long()
    px = p.gather(1, draft[:, None]).squeeze(1)
    qx = torch.ones_like(px) if s["draft_probs"] is None else s["draft_probs"].gather(1, draft[:, None]).squeeze(1).double()
    ok = (s["uniform"].double() * qx < px) & (r + 1 < end[owner])
    j = torch.arange(s["max_rows"], device=DEV)
    okp = ok[torch.clamp(begin[:, None] + j, max=nnz - 1)] & (j[None] < (end - begin)[:, None])
    accepted = torch.cumprod(okp.long(), dim=1).sum(dim=1)
    at = begin + accepted
    rejected = (at + 1 < end)[:, None]
    if s["draft_probs"] is None:
        q = torch.zeros(len(at), vocab, dtype=torch.float64, device=DEV).scatter_(1, draft[at][:, None], 1.0)
    else:
        q = s["draft_probs"][at].double()
    rest = torch.clamp(p[at] - torch.where(rejected, q, 0.0), min=0.0)
    rest = torch.where(rest.sum(dim=1, keepdim=True) > 0, rest, p[at])
    return {"accepted": accepted.to(torch.int32), "tokens": _plain_draw(rest, s["uniform"][end - 1]).to(torch.int32)}


# ---- bytes and operations of one pass ---------------------------------------------------------------------------------------
def work(case):
    es = SIZES[case["dtype"]]
    if case["op"] == "chunk":
        lens, new = _chunk_lengths(case)
        seen = sum(n * m - n * (n - 1) // 2 for n, m in zip(new, lens))
        return {"bytes": sum(lens) * 2 * case["hkv"] * case["d"] * es + sum(new) * case["hq"] * (2 * case["d"] * es + 4),
                "flops": 4 * seen * case["hq"] * case["d"]}
    vocab = case["vocab"]
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (vocab * (es + (4 if case["probs"] else 0)) + 16), "flops": 4 * case["rows"] * vocab}
    rows = case["batch"] * (1 + (case["n_lo"] + case["n_hi"]) / 2)
    return {"bytes": rows * (vocab * es + 12) + (case["batch"] * vocab * 4 if case["probs"] and case["n_hi"] else 0),
            "flops": 4 * rows * vocab}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "chunk":
        return _exact_chunk(s)
    if case["op"] == "sample":
        rows = [_exact_row(s["logits"][i], float(s["temperature"][i]), float(s["top_p"][i])) for i in range(len(s["logits"]))]
        u = s["uniform"].tolist()
        got = {"tokens": torch.tensor([_exact_draw(p, x) for p, x in zip(rows, u)], dtype=torch.int32)}
        return got if s["probs"] is None else dict(got, probs=torch.stack(rows))
    accepted, tokens = [], []
    indptr, u, tok = s["indptr"].tolist(), s["uniform"].tolist(), s["tokens"].tolist()
    temps, tops = s["temperature"].tolist(), s["top_p"].tolist()
    for i, (a, b) in enumerate(zip(indptr[:-1], indptr[1:])):
        r = a
        while True:
            p = _exact_row(s["logits"][r], temps[i], tops[i])
            if r == b - 1:
                break
            x = tok[r + 1]
            if s["draft_probs"] is None:
                q = torch.zeros_like(p)
                q[x] = 1.0
            else:
                q = s["draft_probs"][r].double()
            if not u[r] * float(q[x]) < float(p[x]):
                left = (p - q).clamp_(min=0)
                p = left if float(left.sum()) > 0 else p
                break
            r += 1
        accepted.append(r - a)
        tokens.append(_exact_draw(p, u[b - 1]))
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "tokens": torch.tensor(tokens, dtype=torch.int32)}


def _exact_row(logits, temperature, top_p):
    x = logits.double()
    if temperature <= 0:
        p = torch.zeros_like(x)
        p[int((x == x.max()).nonzero()[0])] = 1.0
        return p
    x = x / temperature
    p = torch.softmax(x, dim=0)
    if top_p >= 1:
        return p
    order = torch.argsort(x, descending=True, stable=True)
    ranked = p[order]
    below = torch.cat([ranked.new_zeros(1), ranked.cumsum(0)[:-1]])
    p = torch.zeros_like(p).index_copy_(0, order, ranked * (below <= top_p))
    return p / p.sum()


def _exact_draw(p, u):
    c = p.cumsum(0)
    return int(torch.searchsorted(c, u * c[-1:], right=True))


def _exact_chunk(s):
    pages, q = s["pages"], s["q"]
    _, _, ps, hkv, d = pages.shape
    qo, kvp, lens = s["qo"].tolist(), s["kv_indptr"].tolist(), s["lens"].tolist()
    group = q.shape[1] // hkv
    out, lse = torch.empty(q.shape, dtype=torch.float64, device=DEV), torch.empty(q.shape[:2], dtype=torch.float64, device=DEV)
    for i, n in enumerate(lens):
        kv = pages[s["kv_indices"][kvp[i]: kvp[i + 1]].long()].double()
        k, v = (kv[:, x].reshape(-1, hkv, d)[:n].repeat_interleave(group, dim=1).transpose(0, 1) for x in (0, 1))
        rows = q[qo[i]: qo[i + 1]].double().transpose(0, 1)
        x = rows @ k.transpose(1, 2) * d ** -0.5
        m = rows.shape[1]
        hidden = torch.arange(n, device=DEV)[None] > torch.arange(n - m, n, device=DEV)[:, None]
        x.masked_fill_(hidden, -math.inf)
        lse[qo[i]: qo[i + 1]] = torch.logsumexp(x, dim=-1).T
        out[qo[i]: qo[i + 1]] = (torch.softmax(x, dim=-1) @ v).transpose(0, 1)
    return {"out": out, "lse": lse}
