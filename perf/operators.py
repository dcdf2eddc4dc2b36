"""The serving operators over a paged KV cache, and the cases they are timed on.

Three operators that make up one serving step next to the projections and the LM head:

``append``   K (rotated for its position) and V of new tokens into a paged cache
             (``Context.paged_append``);
``attend``   causal attention of each sequence's new tokens -- one token or a chunk -- over
             its pages, q rotated on the way (``Context.paged_attention``);
``sample``   one token per row of logits by temperature, top-k, top-p and min-p from a
             given uniform number (``Context.sample``).

With ``own`` false, ``run`` computes them in elementary torch operations; with ``own`` true it
makes the framework's calls.  ``exact`` gives the same outputs from the definitions in
64 bits.  The shapes are the two that the contexts are built for: 12 / 2 heads of 128 (6 query
heads per KV head) and 14 / 2 heads of 64 (7 per KV head).
"""
import math
import random

import numpy as np
import torch

own = False

THETA = 1e6
VOCAB = 151936  # rows of the framework's LM heads
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_GROUP = {128: 6, 64: 7}  # query heads per KV head, by head_dim


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _cache_case(op, dtype, head_dim, layout, page, n_seq, n_chunk, new_lo, new_hi, ctx_lo, ctx_hi,
                lengths, n_kv=2):
    """Of n_seq sequences the first n_chunk bring new_lo..new_hi new tokens, the others one;
    before them ctx_lo..ctx_hi rows are cached.  `lengths` seeds these numbers."""
    return {"op": op, "dtype": dtype, "head_dim": head_dim, "n_kv": n_kv, "layout": layout,
            "page": page, "n_seq": n_seq, "n_chunk": n_chunk, "new_lo": new_lo, "new_hi": new_hi,
            "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "lengths": lengths}


def _sample_case(dtype, rows, vocab, settings):
    return {"op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "settings": settings}


def listed():
    cases = [
        # One decode step of 64 sequences writing its keys and values: the latency of a launch.
        ("append_decode_f32", _cache_case("append", "f32", 128, "hnd", 16, 64, 0, 1, 1, 256, 2048,
                                          1)),
        # Eight prompts' chunks written at once, in 16 bits, heads innermost in a page.
        ("append_chunks_bf16", _cache_case("append", "bf16", 128, "nhd", 64, 8, 8, 256, 2048, 0,
                                           8192, 2)),
        # One request at the end of the server's 4096-row context: the smallest attention.
        ("attend_single_f32", _cache_case("attend", "f32", 128, "hnd", 16, 1, 0, 1, 1, 4095, 4095,
                                          3)),
        # One request over the long single sequence of the benchmark, fp32 as it runs there.
        ("attend_long_f32", _cache_case("attend", "f32", 128, "hnd", 128, 1, 0, 1, 1, 32767, 32767,
                                        4)),
        # A full batch of ordinary requests (the benchmark's 64 sequences of 256 to 8192 rows).
        ("attend_batch_bf16", _cache_case("attend", "bf16", 128, "hnd", 64, 64, 0, 1, 1, 255, 8191,
                                          5)),
        # A chunk of a long prompt behind what is cached of it.
        ("attend_chunk_bf16", _cache_case("attend", "bf16", 128, "hnd", 32, 1, 1, 512, 512, 7680,
                                          7680, 6)),
        # Four whole prompts of odd lengths in the 0.5B shape, nothing cached before them.
        ("attend_prompts_f16", _cache_case("attend", "f16", 64, "nhd", 16, 4, 4, 1500, 2500, 0, 0,
                                           7)),
        # A continuous batch: prompt chunks of three new requests beside 45 running ones.
        ("attend_mixed_bf16", _cache_case("attend", "bf16", 128, "hnd", 16, 48, 3, 200, 700, 1,
                                          6000, 8)),
        # Short prompts behind cached prefixes with the fp32 cache of the decode path.
        ("attend_chunk_f32", _cache_case("attend", "f32", 128, "hnd", 32, 2, 2, 96, 256, 500, 2000,
                                         9)),
        # One request's next token from the LM head's row of logits.
        ("sample_row_f32", _sample_case("f32", 1, VOCAB, "chat")),
        # A batch of requests, each with its own settings.
        ("sample_batch_f32", _sample_case("f32", 64, VOCAB, "mixed")),
        # A large batch with 16-bit logits (many ties) over an odd vocabulary.
        ("sample_batch_bf16", _sample_case("bf16", 192, 50257, "mixed")),
    ]
    return [dict(case, name=name) for name, case in cases]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "chunk", "chunk", "mixed",
                       "sample", "sample", "sample"])
    if kind == "sample":
        rows = _log_int(rng, 1, 192)
        vocab = _log_int(rng, 1000, min(VOCAB, 9000000 // rows))
        return _sample_case(rng.choice(["f32", "bf16", "f16"]), rows, vocab,
                            rng.choice(["chat", "mixed"]))
    dtype = rng.choice(["f32", "bf16", "f16"])
    head_dim = rng.choice([128, 128, 64])
    layout = rng.choice(["hnd", "nhd"])
    page = rng.choice([16, 32, 64, 128, 256])
    n_kv = rng.choice([1, 2, 2, 4])
    seed = rng.randrange(1 << 30)

    def case(op, *shape):
        return _cache_case(op, dtype, head_dim, layout, page, *shape, seed, n_kv=n_kv)

    if kind == "append":
        n_seq = _log_int(rng, 1, 64)
        n_chunk = rng.choice([0, n_seq, rng.randint(0, n_seq)])
        hi = _log_int(rng, 2, max(2, min(2048, 8192 // max(n_chunk, 1))))
        ctx = _log_int(rng, 16, max(16, min(32768, 65536 // n_seq)))
        return case("append", n_seq, n_chunk, max(1, hi // 4), hi, 0, ctx)
    if kind == "decode":
        n_seq = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 1, max(16, min(65536, 131072 // (n_seq * n_kv))))
        return case("attend", n_seq, 0, 1, 1, rng.choice([0, ctx // 8, ctx]), ctx)
    n_seq = _log_int(rng, 1, 4) if kind == "chunk" else _log_int(rng, 4, 48)
    n_chunk = n_seq if kind == "chunk" else rng.randint(1, 3)
    hi = _log_int(rng, 2, 700 if dtype != "f32" else 200)
    ctx = _log_int(rng, 1, 4000 if dtype != "f32" else 1500)
    return case("attend", n_seq, n_chunk, max(1, hi // 3), hi, 0, ctx)


def _plan(case):
    """New tokens and total rows (after the append) of each sequence."""
    r = random.Random(case["lengths"])
    new, total = [], []
    for s in range(case["n_seq"]):
        n = r.randint(case["new_lo"], case["new_hi"]) if s < case["n_chunk"] else 1
        new.append(n)
        total.append(n + r.randint(case["ctx_lo"], case["ctx_hi"]))
    return new, total


def _heads(case):
    return _GROUP[case["head_dim"]] * case["n_kv"], case["n_kv"], case["head_dim"]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        # one read of the logits; a difference, a scale and an exponential per logit
        return {"bytes": n * _DTYPES[case["dtype"]].itemsize + case["rows"] * 24, "flops": 3 * n}
    new, total = _plan(case)
    n_q, n_kv, d = _heads(case)
    size = _DTYPES[case["dtype"]].itemsize
    tokens = sum(new)
    if case["op"] == "append":
        return {"bytes": tokens * 2 * n_kv * d * 2 * size, "flops": tokens * n_kv * d * 3}
    keys = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    return {"bytes": sum(total) * 2 * n_kv * d * size + tokens * n_q * d * 2 * size,
            "flops": keys * n_q * d * 4}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _prepare_sample(case, g):
    rows, vocab = case["rows"], case["vocab"]
    # Logits as a head gives them: a broad bulk, a few dozen candidates well above it, and in
    # every fourth row the tokens that a grammar forbids at minus infinity.
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.2
    hot = torch.randint(0, vocab, (rows, 48), generator=g, device="cuda")
    lift = -4.0 * torch.log1p(-torch.rand(rows, 48, generator=g, device="cuda"))
    x.scatter_add_(1, hot, lift + 4.0)
    banned = torch.rand(rows, vocab, generator=g, device="cuda") < 0.3
    banned &= (torch.arange(rows, device="cuda") % 4 == 3)[:, None]
    x.masked_fill_(banned, -math.inf)
    st = {"logits": x.to(_DTYPES[case["dtype"]])}
    u = torch.rand(5, rows, generator=g, device="cuda")
    if case["settings"] == "chat":
        st["temperature"] = torch.full((rows,), 0.7, device="cuda")
        st["top_k"] = torch.full((rows,), 40, dtype=torch.int32, device="cuda")
        st["top_p"] = torch.full((rows,), 0.95, device="cuda")
        st["min_p"] = torch.full((rows,), 0.05, device="cuda")
    else:
        # each request has its own: one in eight greedy; each filter on in about half of them
        kind = torch.arange(rows, device="cuda") % 8
        st["temperature"] = torch.where(kind == 7, 0.0, 0.5 + u[0])
        k = (1.0 + u[1] * u[1] * (vocab / 4)).to(torch.int32)
        st["top_k"] = torch.where(kind % 2 == 1, k, torch.zeros_like(k))
        st["top_p"] = torch.where(kind // 2 % 2 == 1, 0.5 + 0.5 * u[2], torch.ones_like(u[2]))
        st["min_p"] = torch.where(kind // 4 % 2 == 1, 0.1 * u[3], torch.zeros_like(u[3]))
    st["uniform"] = u[4].contiguous()
    st["tokens"] = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "sample":
        st = _prepare_sample(case, g)
        head_dim, n_kv = 128, 2
    else:
        new, total = _plan(case)
        n_q, n_kv, head_dim = _heads(case)
        dt, page = _DTYPES[case["dtype"]], case["page"]
        counts = [-(-t // page) for t in total]
        n_pages = sum(counts)
        hnd = case["layout"] == "hnd"
        shape = (n_pages, n_kv, page, head_dim) if hnd else (n_pages, page, n_kv, head_dim)
        st = {"new": new, "total": total, "page": page, "hnd": hnd, "n_kv": n_kv, "n_q": n_q}
        st["k_pages"] = torch.randn(shape, generator=g, device="cuda").to(dt)
        st["v_pages"] = torch.randn(shape, generator=g, device="cuda").to(dt)
        # the pool's pages are handed out in any order
        perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        st["page_table"] = torch.full((len(new), max(counts)), -1, dtype=torch.int32,
                                      device="cuda")
        at = 0
        for s, n in enumerate(counts):
            st["page_table"][s, :n] = perm[at:at + n]
            at += n
        st["n_tokens"] = sum(new)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        st["starts"] = starts
        one = max(new) == 1
        st["q_starts"] = None if one else torch.tensor(starts, dtype=torch.int32, device="cuda")
        st["seq_lens"] = torch.tensor(total, dtype=torch.int32, device="cuda")
        st["max_new"], st["max_len"] = max(new), max(total)
        # position and sequence of every new token, one after another
        st["pos"] = torch.cat([torch.arange(t - n, t) for n, t in zip(new, total)]).cuda()
        st["seq"] = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
        # rows of the qkv projection: q | k | v heads of one token after another; queries
        # somewhat longer than keys, so that the softmax has a few dominant keys
        qkv = torch.randn(st["n_tokens"], (n_q + 2 * n_kv) * head_dim, generator=g, device="cuda")
        qkv[:, :n_q * head_dim] *= 1.5
        st["qkv"] = qkv.to(dt)
        st["out"] = torch.zeros(st["n_tokens"], n_q * head_dim, dtype=dt, device="cuda")
    st["op"], st["head_dim"] = case["op"], head_dim
    if own:
        import __graft_entry__
        pkg = __graft_entry__.load_package()
        ctx = pkg.Context(n_heads_q=_GROUP[head_dim] * n_kv, n_heads_kv=n_kv, head_dim=head_dim,
                          rope_theta=THETA, device=torch.cuda.current_device())
        st["ctx"] = ctx
        if case["op"] != "sample":
            st["kv"] = pkg.paged_kv_of(st["k_pages"], st["v_pages"], st["page_table"],
                                       layout=case["layout"])
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if own:
        ctx = state["ctx"]
        if op == "append":
            ctx.paged_append(state["kv"], len(state["new"]), state["n_tokens"], state["q_starts"],
                             state["seq_lens"], state["qkv"])
            return state["k_pages"], state["v_pages"]
        if op == "attend":
            ctx.paged_attention(state["kv"], len(state["new"]), state["n_tokens"],
                                state["q_starts"], state["seq_lens"], state["max_new"],
                                state["max_len"], state["qkv"], state["out"])
            return state["out"]
        rows, vocab = state["logits"].shape
        ctx.sample(rows, vocab, state["logits"], state["temperature"], state["top_k"],
                   state["top_p"], state["min_p"], state["uniform"], state["tokens"])
        return state["tokens"]
    if op == "append":
        return _plain_append(state)
    if op == "attend":
        return _plain_attend(state)
    return _plain_sample(state)


def _rotate(x, pos):
    """x [tokens, heads, d] in fp32: pairs (i, i + d/2) turned by pos * theta^(-2i/d); the
    angles in 64 bits, reduced to one turn before they are rounded."""
    d = x.shape[-1]
    i = torch.arange(d // 2, device=x.device, dtype=torch.float64)
    angle = pos.double()[:, None] * THETA ** (-2.0 * i / d)
    angle = torch.remainder(angle, 2.0 * math.pi)
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([a * c - b * s, a * s + b * c], dim=-1)


def _plain_append(st):
    n_q, n_kv, d, page = st["n_q"], st["n_kv"], st["head_dim"], st["page"]
    rows = st["qkv"].view(st["n_tokens"], n_q + 2 * n_kv, d)
    pos = st["pos"]
    pages = st["page_table"][st["seq"], pos // page].long()
    k = _rotate(rows[:, n_q:n_q + n_kv].float(), pos).to(st["qkv"].dtype)
    v = rows[:, n_q + n_kv:]
    if st["hnd"]:
        st["k_pages"][pages, :, pos % page] = k
        st["v_pages"][pages, :, pos % page] = v
    else:
        st["k_pages"][pages, pos % page] = k
        st["v_pages"][pages, pos % page] = v
    return st["k_pages"], st["v_pages"]


def _gather(st, pages, s):
    """Cache rows [0, total[s]) of sequence s as [n_kv, rows, d]."""
    n = -(-st["total"][s] // st["page"])
    x = pages[st["page_table"][s, :n].long()]
    if st["hnd"]:
        x = x.transpose(1, 2)  # [pages, page, n_kv, d]
    return x.reshape(n * st["page"], st["n_kv"], st["head_dim"])[:st["total"][s]].transpose(0, 1)


def _plain_attend(st):
    n_q, n_kv, d = st["n_q"], st["n_kv"], st["head_dim"]
    group = n_q // n_kv
    rows = st["qkv"].view(st["n_tokens"], n_q + 2 * n_kv, d)
    q = _rotate(rows[:, :n_q].float(), st["pos"]) * (1.0 / math.sqrt(d))
    for s, (n, t) in enumerate(zip(st["new"], st["total"])):
        at = st["starts"][s]
        k = _gather(st, st["k_pages"], s).float()
        v = _gather(st, st["v_pages"], s).float()
        qs = q[at:at + n].view(n, n_kv, group, d).permute(1, 2, 0, 3).reshape(n_kv, group * n, d)
        x = torch.bmm(qs, k.transpose(1, 2)).view(n_kv, group, n, t)
        if n > 1:
            last = torch.arange(t - n, t, device="cuda")
            hidden = torch.arange(t, device="cuda")[None, :] > last[:, None]
            x.masked_fill_(hidden, -math.inf)
        x = torch.exp(x - x.amax(dim=-1, keepdim=True))
        norm = x.sum(dim=-1, keepdim=True)
        o = torch.bmm(x.view(n_kv, group * n, t), v).view(n_kv, group, n, d) / norm
        st["out"][at:at + n] = o.permute(2, 0, 1, 3).reshape(n, n_q * d).to(st["out"].dtype)
    return st["out"]


def _plain_sample(st):
    """Weights and sums in 64 bits: a cumulative sum over a vocabulary needs them next to the
    border that the uniform number or top-p picks out."""
    x = st["logits"].float()
    rows, vocab = x.shape
    top, first = x.max(dim=1, keepdim=True)
    greedy = st["temperature"] <= 0
    t = torch.where(greedy, 1.0, st["temperature"]).double()[:, None]
    w = torch.exp((x.double() - top.double()) / t)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(vocab, device=x.device)[None, :]
    k = st["top_k"].long()[:, None]
    keep = (k <= 0) | (rank < k)
    ws = torch.where(keep, ws, 0.0)
    before = torch.cumsum(ws, dim=1) - ws
    p = st["top_p"].double()[:, None]
    keep &= (p >= 1) | (before < p * ws.sum(dim=1, keepdim=True))
    keep &= ws >= st["min_p"].double()[:, None]
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    c = torch.cumsum(kept, dim=1)
    target = st["uniform"].double()[:, None] * c[:, -1:]
    token = ((c <= target) | (kept == 0)).to(torch.int8).argmin(dim=1)
    st["tokens"][:] = torch.where(greedy, order[:, 0], token).to(torch.int32)
    return st["tokens"]


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _turn64(x, positions):
    """RoPE as a product of complex numbers: x [heads, tokens, d] in 64 bits."""
    d = x.shape[-1]
    freq = torch.tensor([THETA ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64,
                        device=x.device)
    angle = torch.outer(positions.to(torch.float64), freq)
    z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous())
    z = z * torch.polar(torch.ones_like(angle), angle)
    return torch.cat((z.real, z.imag), dim=-1)


def _exact_append(st):
    n_q, n_kv, d, page = st["n_q"], st["n_kv"], st["head_dim"], st["page"]
    k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
    rows = st["qkv"].double()
    table = st["page_table"].cpu()
    for s, (n, t) in enumerate(zip(st["new"], st["total"])):
        part = rows[st["starts"][s]:st["starts"][s] + n].view(n, -1, d).transpose(0, 1)
        k = _turn64(part[n_q:n_q + n_kv], torch.arange(t - n, t, device="cuda"))
        v = part[n_q + n_kv:]
        for p in range((t - n) // page, (t - 1) // page + 1):
            lo, hi = max(p * page, t - n), min(p * page + page, t)
            src = slice(lo - (t - n), hi - (t - n))
            dst = slice(lo - p * page, hi - p * page)
            for pages, x in ((k_pages, k), (v_pages, v)):
                one = pages[int(table[s, p])]
                if st["hnd"]:
                    one[:, dst] = x[:, src]
                else:
                    one[dst] = x[:, src].transpose(0, 1)
    return k_pages, v_pages


def _exact_attend(st):
    n_q, n_kv, d, page = st["n_q"], st["n_kv"], st["head_dim"], st["page"]
    group = n_q // n_kv
    out = torch.zeros(st["n_tokens"], n_q * d, dtype=torch.float64, device="cuda")
    for s, (n, t) in enumerate(zip(st["new"], st["total"])):
        at = st["starts"][s]
        ids = st["page_table"][s, :-(-t // page)].long()
        where = torch.arange(t - n, t, device="cuda")
        for h in range(n_kv):
            k, v = ((x[ids, h] if st["hnd"] else x[ids, :, h]).reshape(-1, d)[:t].double()
                    for x in (st["k_pages"], st["v_pages"]))
            for j in range(h * group, (h + 1) * group):
                q = _turn64(st["qkv"][at:at + n, j * d:(j + 1) * d].double()[None], where)[0]
                score = torch.mm(q, k.T) / math.sqrt(d)
                score += torch.triu(torch.full_like(score, -math.inf), diagonal=t - n + 1)
                out[at:at + n, j * d:(j + 1) * d] = torch.mm(torch.softmax(score, dim=1), v)
    return out


def _exact_sample(st):
    logits = st["logits"].double().cpu().numpy()
    names = ("temperature", "top_k", "top_p", "min_p", "uniform")
    tokens = []
    for x, t, k, p, m, u in zip(logits, *(st[n].double().cpu().numpy() for n in names)):
        if t <= 0:
            tokens.append(int(np.argmax(x)))
            continue
        w = np.exp((x - x.max()) / t)
        ids = np.lexsort((np.arange(x.size), -x))  # by logit, then by index
        if k >= 1:
            ids = ids[:int(k)]
        if p < 1:
            mass = np.cumsum(w[ids])
            n = int(np.searchsorted(mass, p * mass[-1], side="left")) + 1
            ids = ids[:max(1, min(n, ids.size))]
        ids = np.concatenate((ids[:1], ids[1:][w[ids[1:]] >= m]))
        ids.sort()
        mass = np.cumsum(w[ids])
        n = int(np.searchsorted(mass, u * mass[-1], side="right"))
        live = np.flatnonzero(w[ids])
        tokens.append(int(ids[min(n, live[-1])]))
    return torch.tensor(tokens, dtype=torch.int32)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"append": _exact_append, "attend": _exact_attend,
            "sample": _exact_sample}[case["op"]](st)
