"""The paged-cache and sampling operators: their cases, inputs, plain forms and exact values.

Four operators that one serving step uses together, on a pool of pages that holds the q8 key/value
cache (rows of kv_heads * head_dim codes, one byte each with bias 128, and one f16 scale for every 64):

- append:    RMS norm of each query and key head, rotary positions, queries out, the new key and
             value rows quantized into the sequences' pages;
- attention: the batch's tokens, one to many for each sequence, over their sequence's pages, causal;
- read:      the batch's key and value rows out of the pages as the values that they stand for;
- sample:    temperature, top-k, top-p and min-p over a row of logits, from a given uniform number.

`run` computes them in their plain form, or, where `own` is true, through the framework.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 64  # values that share a scale
BIAS = 128  # the code that stands for zero
THETA = 1000000.0
EPS = 1e-6


# ---- cases ----


def listed():
    shape = dict(heads=16, kv_heads=8, head_dim=128)  # both released decoders
    return [
        # One clip a third of the way through its transcript: what a single decoding stream waits for.
        dict(name="attention 1x1 over 301", op="attention", type="f32", page=16, seqs=1, query=1, context=301, mix=1, **shape),
        # A full batch of streams, long clips, contexts of every length: the decoding step of a busy server.
        dict(name="attention 64x1 over 4096", op="attention", type="f32", page=64, seqs=64, query=1, context=4096, mix=2, **shape),
        # Prompt chunks of 64 positions beside streams that only decode, small pages, a 16-bit model.
        dict(name="attention 24x64 over 1237", op="attention", type="bf16", page=16, seqs=24, query=64, context=1237, mix=3, **shape),
        # A prompt of an odd length on top of a shared prefix, the engine's own type.
        dict(name="attention 2x391 over 2047", op="attention", type="f32", page=64, seqs=2, query=391, context=2047, mix=4, **shape),
        # Long clips prefilled at once: the largest call.
        dict(name="attention 4x1500 over 4096", op="attention", type="bf16", page=128, seqs=4, query=1500, context=4096, mix=5, **shape),
        # One decoding step's rows of a small batch.
        dict(name="append 8x1", op="append", type="f32", page=16, seqs=8, query=1, context=200, mix=6, **shape),
        # A whole batch of prompts at once.
        dict(name="append 64x391", op="append", type="bf16", page=64, seqs=64, query=391, context=391, mix=7, **shape),
        # One prompt's rows handed to something that wants them in 32 bits.
        dict(name="read 1x391", op="read", type="f32", page=16, seqs=1, query=391, context=391, mix=8, **shape),
        # Every stream's rows, as 16-bit values.
        dict(name="read 64x2850", op="read", type="bf16", page=64, seqs=64, query=2850, context=2850, mix=9, **shape),
        # One stream's next token.
        dict(name="sample 1x151936", op="sample", type="f32", rows=1, vocab=151936, mix=10),
        # A full batch's next tokens, every setting of the filters among the rows.
        dict(name="sample 64x151936", op="sample", type="f32", rows=64, vocab=151936, mix=11),
        # 16-bit logits, where many tokens tie, and a vocabulary of an odd size.
        dict(name="sample 16x32003", op="sample", type="bf16", rows=16, vocab=32003, mix=12),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "append", "read", "sample"))
    kind = rng.choice(("f32", "f16", "bf16"))
    mix = rng.randrange(1 << 20)
    if op == "sample":
        return dict(op=op, type=kind, rows=_spread(rng, 1, 64), vocab=_spread(rng, 500, 151936), mix=mix)
    heads, kv_heads, head_dim = rng.choice(((16, 8, 128), (16, 8, 128), (16, 16, 64), (14, 2, 64), (12, 4, 128), (8, 1, 128), (5, 5, 64)))
    case = dict(op=op, type=kind, page=rng.choice((8, 16, 24, 64, 128, 256)), heads=heads, kv_heads=kv_heads, head_dim=head_dim, mix=mix)
    if op == "attention":
        context = _spread(rng, 8, 8192)
        query = rng.choice((1, 1, _spread(rng, 2, 16), _spread(rng, 16, 1500)))
        query = min(query, context)
        # No more work than the largest listed cases, whose sequences average about half of their longest one: the
        # scores of the long prompts, the cache of the full batch.
        most = min(64, (2 * 16 * 1500 * 4096) // (heads * query * context), (32 * 4096 * 1024) // (context * kv_heads * head_dim))
        return dict(case, seqs=_spread(rng, 1, max(1, most)), query=query, context=context)
    query = _spread(rng, 1, 2850 if op == "read" else 1500)
    most = min(64, (32 * 391 * 1024 if op == "append" else 32 * 2850 * 1024) // (query * kv_heads * head_dim))
    return dict(case, seqs=_spread(rng, 1, max(1, most)), query=query, context=query if op == "read" else query + rng.randrange(500))


def _lengths(case):
    """The tokens and the context of each sequence: the first has the most of both, the others anything down to one
    token and down to a quarter of the longest context."""
    r = np.random.RandomState(case["mix"])
    n = case["seqs"]
    query = r.randint(max(1, case["query"] // 8), case["query"] + 1, n)
    context = r.randint(max(1, case["context"] // 4), case["context"] + 1, n)
    query[0], context[0] = case["query"], case["context"]
    return query, np.maximum(context, query)


# ---- inputs ----


def _quantized(x):
    """q8 of rows in groups of 64, as the cache holds them: f16 scales (amax / 128), codes round(x / scale) + 128."""
    g = x.reshape(x.shape[0], -1, GROUP)
    scales = (g.abs().amax(-1) / 128).half()
    s = scales.float()[..., None]
    y = g / torch.where(s == 0, torch.ones_like(s), s)
    codes = torch.where(s == 0, torch.zeros_like(y), torch.trunc(y + torch.where(y >= 0, 0.5, -0.5)).clamp(-128, 127))
    return scales, (codes + BIAS).to(torch.uint8).reshape(x.shape)


def _prepare_paged(case, g, dev):
    query, context = _lengths(case)
    page, heads, kv_heads, dim = case["page"], case["heads"], case["kv_heads"], case["head_dim"]
    need = -(-context // page)
    pages = int(need.sum()) + 3  # a few that no sequence holds
    width = kv_heads * dim
    dtype = TYPES[case["type"]]
    where = np.random.RandomState(case["mix"] + 1).permutation(pages)[: int(need.sum())]  # pages are handed out in no order
    table = np.zeros((case["seqs"], int(need.max())), np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = where[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(query)]).astype(np.int32)
    tokens = int(starts[-1])
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    rand = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    state = dict(case=case, starts=put(starts), context=put(context.astype(np.int32)), table=put(table), tokens=tokens)
    # Keys and queries as a norm with weights leaves them, values of the size that a value projection gives.
    k_norm = 1 + 0.25 * rand(dim)
    q_norm = 1.4 + 0.25 * rand(dim)
    for name, row in (("k", rand(pages * page, kv_heads, dim) * k_norm), ("v", rand(pages * page, kv_heads, dim) * 0.7)):
        state[name + "_scales"], state[name + "_codes"] = _quantized(row.reshape(-1, width))
        del row
    if case["op"] == "attention":
        state["q"] = (rand(tokens, heads, dim) * q_norm).to(dtype)
    elif case["op"] == "append":
        # One row for each token from the joint projection: queries, keys, values.
        rows = (rand(tokens, (heads + 2 * kv_heads) * dim) * 1.3).to(dtype)
        state["q"] = rows[:, : heads * dim].unflatten(1, (heads, dim))
        state["k"] = rows[:, heads * dim: (heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
        state["v"] = rows[:, (heads + kv_heads) * dim:].unflatten(1, (kv_heads, dim))
        state["q_norm"], state["k_norm"] = q_norm, k_norm
        angle = torch.arange(int(context.max()), dtype=torch.float64, device=dev)[:, None] * THETA ** (
            -torch.arange(dim // 2, dtype=torch.float64, device=dev) / (dim // 2))
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    if own:  # the handles that a program makes once for its pool and once for a batch, and uses in every layer
        from qwenscriber_b200 import paged

        state["cache"] = paged.PagedCache(state["k_scales"], state["k_codes"], state["v_scales"], state["v_codes"],
                                          page_size=page, kv_heads=kv_heads, head_dim=dim)
        state["batch"] = paged.PagedBatch(state["starts"], state["context"], state["table"], tokens=tokens,
                                          max_query=int(query.max()), max_context=int(context.max()))
    return state


def _prepare_sample(case, g, dev):
    rows, vocab = case["rows"], case["vocab"]
    # A language model's logits: a wide body and a few tokens that stand out.
    logits = 2.2 * torch.randn(rows, vocab, generator=g, device=dev)
    likely = torch.randint(0, vocab, (rows, 12), generator=g, device=dev)
    logits.scatter_add_(1, likely, 9 + 2.5 * torch.randn(rows, 12, generator=g, device=dev))
    r = np.random.RandomState(case["mix"])
    put = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device=dev)  # noqa: E731
    # Requests with settings of their own: one in eight takes the best token, some leave a filter out.
    temperature = np.where(np.arange(rows) % 8 == 5, 0.0, r.uniform(0.3, 1.3, rows))
    return dict(
        case=case, logits=logits.to(TYPES[case["type"]]), uniform=torch.rand(rows, generator=g, device=dev),
        temperature=put(temperature, torch.float32), top_k=put(r.choice([0, 0, 1, 20, 50, 400], rows), torch.int32),
        top_p=put(np.where(r.rand(rows) < 0.3, 1.0, r.uniform(0.5, 0.99, rows)), torch.float32),
        min_p=put(np.where(r.rand(rows) < 0.6, 0.0, r.uniform(0.001, 0.1, rows)), torch.float32))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    return _prepare_sample(case, g, dev) if case["op"] == "sample" else _prepare_paged(case, g, dev)


# ---- plain forms ----


def _token_places(st):
    """Of each token of the batch: its sequence, its position there, and its row of the pool."""
    starts, tokens, page = st["starts"].long(), st["tokens"], st["case"]["page"]
    t = torch.arange(tokens, device=starts.device)
    s = torch.searchsorted(starts, t, right=True) - 1
    pos = st["context"].long()[s] - starts[s + 1] + t
    row = st["table"].long()[s, pos // page] * page + pos % page
    return s, pos, row


def _values(scales, codes, kv_heads, dim):
    """What rows of the cache stand for, in 32 bits."""
    v = (codes.float() - BIAS).unflatten(-1, (-1, GROUP)) * scales.float()[..., None]
    return v.flatten(-2).unflatten(-1, (kv_heads, dim))


def _plain_attention(st):
    c = st["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    share = heads // kv_heads
    context, starts = st["context"].long(), st["starts"].long()
    query = starts[1:] - starts[:-1]
    most, longest = c["query"], c["context"]
    pos = torch.arange(longest, device=context.device)
    held = pos < context[:, None]
    row = torch.where(held, st["table"].long()[:, pos // page] * page + pos % page, 0)
    keys = _values(st["k_scales"][row], st["k_codes"][row], kv_heads, dim)
    values = _values(st["v_scales"][row], st["v_codes"][row], kv_heads, dim)
    i = torch.arange(most, device=context.device)
    token = torch.where(i < query[:, None], starts[:-1, None] + i, 0)
    q = st["q"].float()[token]  # [seqs, most, heads, dim]
    q = q.unflatten(2, (kv_heads, share)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = q @ keys.permute(0, 2, 3, 1) * (1 / math.sqrt(dim))
    scores = scores.unflatten(2, (share, most))
    seen = pos <= (context - query)[:, None, None] + i[:, None]
    scores.masked_fill_(~(seen & held[:, None])[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    out = scores.flatten(2, 3) @ values.permute(0, 2, 1, 3)
    out = out.unflatten(2, (share, most)) / total
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)  # [seqs, most, heads, dim]
    return out[i < query[:, None]].to(st["q"].dtype)


def _turned(x, weight, cos, sin):
    """RMS norm over a head's values, then the rotation of the pairs (d, d + half)."""
    x = x.float()
    x = x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * weight
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _plain_append(st):
    c = st["case"]
    _, pos, row = _token_places(st)
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    q = _turned(st["q"], st["q_norm"], cos, sin).to(st["q"].dtype)
    for name, x in (("k", _turned(st["k"], st["k_norm"], cos, sin)), ("v", st["v"].float())):
        scales, codes = _quantized(x.flatten(1))
        st[name + "_scales"][row] = scales
        st[name + "_codes"][row] = codes
    k, v = (_values(st[n + "_scales"][row], st[n + "_codes"][row], c["kv_heads"], c["head_dim"]).half() for n in "kv")
    return {"q": q, "k": k, "v": v}


def _plain_read(st):
    c = st["case"]
    _, _, row = _token_places(st)
    k, v = (_values(st[n + "_scales"][row], st[n + "_codes"][row], c["kv_heads"], c["head_dim"]).to(TYPES[c["type"]]) for n in "kv")
    return {"k": k, "v": v}


def _plain_sample(st):
    x = st["logits"].float()
    best = x.amax(-1, keepdim=True)
    greedy = st["temperature"] <= 0
    heat = torch.where(greedy, 1.0, st["temperature"])[:, None]
    w = ((x - best) / heat).exp()
    down, index = x.sort(dim=-1, descending=True, stable=True)  # ties: the lowest index first
    wd = w.gather(1, index)
    rank = torch.arange(x.shape[1], device=x.device)
    k, p = st["top_k"][:, None], st["top_p"][:, None]
    keep = (k <= 0) | (rank < k)
    mass = (wd * keep).cumsum(-1)
    keep &= (p >= 1) | (mass - wd < p * mass[:, -1:])  # up to the token that reaches p
    keep &= wd >= st["min_p"][:, None]
    keep[:, 0] = True
    kept = torch.zeros_like(keep).scatter_(1, index, keep)
    mass = (w * kept).cumsum(-1)
    token = (mass <= st["uniform"][:, None] * mass[:, -1:]).sum(-1)  # the first whose sum passes the number
    last = (kept * (rank + 1)).amax(-1) - 1
    token = torch.where(greedy, index[:, 0], torch.minimum(token, last))
    logprob = (x.gather(1, token[:, None]) - best) / heat - w.sum(-1, keepdim=True).log()
    return {"token": token.int(), "logprob": logprob[:, 0]}


def run(state):
    case = state["case"]
    if not own:
        return {"attention": _plain_attention, "append": _plain_append, "read": _plain_read, "sample": _plain_sample}[case["op"]](state)
    from qwenscriber_b200 import paged, sampling

    if case["op"] == "attention":
        return paged.attention(state["cache"], state["batch"], state["q"])
    if case["op"] == "append":
        q = paged.append(state["cache"], state["batch"], state["q"], state["k"], state["v"], state["cos"], state["sin"],
                         q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS)
        # The rows that the call wrote, as the values that they stand for.
        k, v = paged.read(state["cache"], state["batch"], torch.float16)
        return {"q": q, "k": k, "v": v}
    if case["op"] == "read":
        k, v = paged.read(state["cache"], state["batch"], TYPES[case["type"]])
        return {"k": k, "v": v}
    token, logprob = sampling.sample(state["logits"], state["uniform"], temperature=state["temperature"],
                                     top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    return {"token": token, "logprob": logprob}


# ---- what a pass cannot do without ----


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 28, "flops": 3 * n}  # difference, exponential, sum
    query, context = _lengths(case)
    tokens, heads, kv_heads, dim = int(query.sum()), case["heads"], case["kv_heads"], case["head_dim"]
    row = kv_heads * dim + kv_heads * dim // GROUP * 2  # a key or value row of the cache
    if case["op"] == "attention":
        pairs = int((query * (context - query) + query * (query + 1) // 2).sum())
        return {"bytes": 2 * int(context.sum()) * row + 2 * tokens * heads * dim * size, "flops": 4 * dim * heads * pairs}
    if case["op"] == "append":  # the rows in, the queries and the cache's rows out, and these as values
        given = (heads + 2 * kv_heads) * dim * size + heads * dim * size
        return {"bytes": tokens * (given + 4 * row + 2 * kv_heads * dim * 2) + 2 * int(context.max()) * dim * 2,
                "flops": tokens * (10 * (heads + kv_heads) + 3 * 2 * kv_heads) * dim}
    return {"bytes": tokens * 2 * (row + kv_heads * dim * size), "flops": tokens * 4 * kv_heads * dim}


# ---- the same from the definitions, in 64 bits ----


def _exact_rows(st, s, first, last):
    """Positions first..last-1 of sequence s: rows of the pool."""
    page = st["case"]["page"]
    pos = np.arange(first, last)
    table = st["table"][s].cpu().numpy().astype(np.int64)
    return torch.from_numpy(table[pos // page] * page + pos % page).to(st["table"].device)


def _exact_cache(st, name, rows):
    c = st["case"]
    scale = st[name + "_scales"][rows].double().repeat_interleave(GROUP, dim=1)
    return ((st[name + "_codes"][rows].double() - 128.0) * scale).view(len(rows), c["kv_heads"], c["head_dim"])


def _exact_attention(st, query, context):
    c = st["case"]
    share = c["heads"] // c["kv_heads"]
    outs, at = [], 0
    for s, (n, length) in enumerate(zip(query.tolist(), context.tolist())):
        rows = _exact_rows(st, s, 0, length)
        k, v = _exact_cache(st, "k", rows), _exact_cache(st, "v", rows)
        q = st["q"][at:at + n].double()
        at += n
        out = torch.empty(n, c["heads"], c["head_dim"], dtype=torch.float64, device=q.device)
        hidden = torch.arange(length, device=q.device)[None] > torch.arange(length - n, length, device=q.device)[:, None]
        for h in range(c["heads"]):
            score = torch.einsum("nd,ld->nl", q[:, h], k[:, h // share]) / c["head_dim"] ** 0.5
            score[hidden] = -math.inf
            out[:, h] = torch.softmax(score, -1) @ v[:, h // share]
        outs.append(out)
    return torch.cat(outs)


def _exact_append(st, query, context):
    c = st["case"]
    pos = np.concatenate([np.arange(l - n, l) for n, l in zip(query, context)])
    half = c["head_dim"] // 2
    # The rotation tables are inputs: what they hold, not the angles that they came from.
    cos, sin = (st[n].double().cpu()[torch.from_numpy(pos)].to(st[n].device).unsqueeze(1) for n in ("cos", "sin"))

    def turn(x, w):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / c["head_dim"] + EPS).sqrt() * w.double()
        y = torch.empty_like(x)
        y[..., :half] = x[..., :half] * cos - x[..., half:] * sin
        y[..., half:] = x[..., half:] * cos + x[..., :half] * sin
        return y

    def through(x):
        flat = x.reshape(len(x), -1, GROUP)
        scale = (flat.abs().max(-1, keepdim=True).values / 128).half().double()
        code = flat / scale
        code = (torch.sign(code) * torch.floor(code.abs() + 0.5)).clamp(-128, 127)
        return torch.where(scale == 0, 0.0, code * scale).reshape(x.shape)

    return {"q": turn(st["q"], st["q_norm"]), "k": through(turn(st["k"], st["k_norm"])), "v": through(st["v"].double())}


def _exact_read(st, query, context):
    rows = torch.cat([_exact_rows(st, s, l - n, l) for s, (n, l) in enumerate(zip(query.tolist(), context.tolist()))])
    return {"k": _exact_cache(st, "k", rows), "v": _exact_cache(st, "v", rows)}


def _exact_sample(st):
    tokens, logs = [], []
    for r in range(st["case"]["rows"]):
        x = st["logits"][r].double().cpu().numpy()
        heat, k, p, least, u = (float(st[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
        greedy = heat <= 0
        z = x / (1.0 if greedy else heat)
        logp = z - (z.max() + math.log(np.exp(z - z.max()).sum()))
        order = np.lexsort((np.arange(len(x)), -x))
        if k > 0:
            order = order[: int(k)]
        prob = np.exp(logp[order] - logp[order[0]])
        if p < 1:
            before = np.concatenate([[0.0], np.cumsum(prob)[:-1]])
            order, prob = order[before < p * prob.sum()], prob[before < p * prob.sum()]
        order = order[(prob >= np.float64(least)) | (np.arange(len(order)) == 0)] if len(order) else order
        chosen = np.sort(order)
        mass = np.cumsum(np.exp(logp[chosen] - logp.max()))
        token = int(np.argmax(x)) if greedy else int(chosen[min(np.searchsorted(mass, u * mass[-1], side="right"), len(chosen) - 1)])
        tokens.append(token)
        logs.append(logp[token])
    return {"token": torch.tensor(tokens, dtype=torch.int32), "logprob": torch.tensor(logs, dtype=torch.float64)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    query, context = _lengths(case)
    return {"attention": _exact_attention, "append": _exact_append, "read": _exact_read}[case["op"]](st, query, context)
