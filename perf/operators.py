"""Speed cases of the operators that serve several samples of one prompt: attention over a paged
cache whose rows share a prefix, the page table kept on the device, and token log-probabilities.

``run`` computes them in plain torch operations (``own`` false) or through the package (``own``
true).  Shapes: the verify and draft steps of the engine's benchmark models (32 / 8 and 16 / 8 heads
of 128, k = 4 and 8 drafts, 151936 tokens of vocabulary), its 128-token pages, and batches, prompts
and vocabularies around them.
"""
import math
import pathlib
import sys

import torch

own = False

ROOT = pathlib.Path(__file__).resolve().parent.parent
PAGE = 128                       # tokens per page of the paged cache
VOCAB = 151936
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _package():
    """This repository's package on the path (it lives in a folder that is no module name)."""
    p = str(ROOT / "adaptive-specdec_b200")
    if p not in sys.path:
        sys.path.insert(0, p)


# ---- cases --------------------------------------------------------------------------------------

def _attn(name, rows, qlen, hq, hkv, groups, pages, suffix, dim=128, dtype="bf16"):
    return {"name": name, "op": "prefix_attention", "rows": rows, "qlen": qlen, "hq": hq, "hkv": hkv,
            "dim": dim, "groups": groups, "pages_lo": pages[0], "pages_hi": pages[1],
            "suffix_lo": suffix[0], "suffix_hi": suffix[1], "dtype": dtype}


def _logp(name, rows, vocab, dtype, temperature, top, pad=0):
    return {"name": name, "op": "token_logprobs", "rows": rows, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "top": top, "pad": pad}


def _pages(name, rows, width, lo, hi, new, ragged):
    return {"name": name, "op": "page_table", "rows": rows, "width": width, "lo": lo, "hi": hi,
            "new": new, "ragged": ragged}


def listed():
    return [
        # two samples of a one-page prompt, the first decoding step: nothing but latency
        _attn("attn_pair", 2, 1, 32, 8, 1, (1, 1), (1, 9)),
        # a draft step of the small model at the engine benchmark's batch, half a thousand prompt tokens
        _attn("attn_draft", 32, 1, 16, 8, 1, (4, 4), (1, 300)),
        # a verify step of 64 samples under one long system prompt (k = 4)
        _attn("attn_verify", 64, 5, 32, 8, 1, (64, 64), (16, 1024)),
        # eight prompts of different lengths with ragged numbers of samples, k = 8 drafts
        _attn("attn_groups", 45, 9, 32, 8, 8, (0, 32), (1, 700)),
        # many samples under a very long document (k = 4)
        _attn("attn_long", 128, 5, 32, 8, 1, (128, 128), (64, 512)),
        # fp32 rows of a small model with heads of 64
        _attn("attn_fp32", 8, 3, 8, 2, 2, (2, 2), (1, 200), dim=64, dtype="fp32"),
        # the token that one request's step emitted
        _logp("logp_one", 1, VOCAB, "bf16", 1.0, 0),
        # every position of a verify round of 64 rows (k = 4), five alternatives each
        _logp("logp_verify", 320, VOCAB, "bf16", 0.7, 5),
        # fp32 logits of an odd vocabulary, many alternatives
        _logp("logp_odd", 33, 32003, "fp32", 1.0, 20),
        # scoring a prompt
        _logp("logp_prompt", 2048, VOCAB, "bf16", 1.0, 1),
        # pages and slots of a verify round of 64 rows: the last round's pages back, this round's out
        _pages("pages_round", 64, 66, 512, 8192, 5, 0),
        # pages and slots of 512 prompts of very different lengths
        _pages("pages_prompts", 512, 66, 0, 0, 8192, 1),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prefix_attention", "prefix_attention", "token_logprobs", "token_logprobs", "page_table"])
    if kind == "token_logprobs":
        vocab = rng.choice([VOCAB, 32003, _log_between(rng, 40, 260000)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        rows = _log_between(rng, 1, min(4096, max(2, 300_000_000 // vocab)))
        return _drawn(_logp("", rows, vocab, dtype, rng.choice([1.0, 0.7, 1.5]), rng.choice([0, 1, 5, 20, 32]),
                            rng.choice([0, 0, 1, 8])))
    if kind == "page_table":
        rows = _log_between(rng, 1, 2048)
        if rng.random() < 0.5:
            return _drawn(_pages("", rows, 66, 1, _log_between(rng, 2, 8192), rng.randint(1, 17), 0))
        return _drawn(_pages("", rows, 66, 0, 0, _log_between(rng, 8, min(8192, 4_000_000 // rows)), 1))
    if rng.random() < 0.15:
        rows = _log_between(rng, 1, 16)
        lo, hi = sorted((rng.randint(0, 3), rng.randint(0, 3)))
        return _drawn(_attn("", rows, rng.randint(1, 5), 8, rng.choice([1, 2, 8]), rng.randint(1, min(3, rows)), (lo, hi),
                            (1, rng.randint(2, 300)), dim=rng.choice([64, 128]), dtype="fp32"))
    hq, hkv = rng.choice([(32, 8), (32, 8), (16, 8), (8, 8), (16, 2)])
    rows, qlen = _log_between(rng, 1, 192), rng.choice([1, 2, 3, 5, 9, 13])
    hi = _log_between(rng, 1, 128)
    lo = rng.choice([hi, 0, hi // 2])
    suffix_hi = _log_between(rng, 2, 1500)
    case = _drawn(_attn("", rows, qlen, hq, hkv, rng.randint(1, min(8, rows)), (lo, hi),
                        (rng.randint(1, suffix_hi), suffix_hi)))
    top = listed()[4]
    most_flops, most_keys = work(top)["flops"], _keys(top)
    while work(case)["flops"] > most_flops or _keys(case) > most_keys:
        case["rows"] = max(1, case["rows"] // 2)
        case["groups"] = min(case["groups"], case["rows"])
    return case


def _drawn(case):
    del case["name"]
    return case


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _groups(case):
    """(first row of each group and the end, prefix pages of each group): uneven groups."""
    rows, n = case["rows"], case["groups"]
    cut = [rows * i * (i + 3) // (n * (n + 3)) for i in range(n + 1)]
    cut = [max(c, i) for i, c in enumerate(cut)]
    return cut[:-1] + [rows], _spread(case["pages_lo"], case["pages_hi"], n)


def _suffixes(case):
    return _spread(case["suffix_lo"], case["suffix_hi"], case["rows"])


def _keys(case):
    """Keys that the rows see, counted per row, times the bytes of their 32-bit copies."""
    cut, pages = _groups(case)
    width = max(pages) + -(-(case["suffix_hi"] + case["qlen"]) // PAGE) + 1
    return case["rows"] * width * case["hkv"] * case["dim"]


def work(case):
    if case["op"] == "prefix_attention":
        e = 4 if case["dtype"] == "fp32" else 2
        cut, pages = _groups(case)
        rows, qlen, d, hq, hkv = case["rows"], case["qlen"], case["dim"], case["hq"], case["hkv"]
        own_keys = sum(_suffixes(case)) + rows * qlen
        shared = sum(pages) * PAGE
        seen = sum((b - a) * p * PAGE for a, b, p in zip(cut, cut[1:], pages)) + own_keys
        return {"bytes": e * (2 * d * hkv * (shared + own_keys) + 2 * rows * qlen * hq * d),
                "flops": 4 * seen * qlen * hq * d}
    if case["op"] == "token_logprobs":
        e = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * e + 24 + 12 * case["top"]), "flops": 6 * case["rows"] * case["vocab"]}
    tokens = _tokens(case)
    pages = tokens // PAGE + case["rows"]
    return {"bytes": case["rows"] * 8 * 4 + tokens * 8 + pages * 16, "flops": tokens}


def _tokens(case):
    """Tokens that a page-table call maps (ragged: every row another number, from one to `new`)."""
    return sum(_spread(1, case["new"], case["rows"])) if case["ragged"] else case["rows"] * case["new"]


# ---- inputs -------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op, rows = case["op"], case["rows"]
    state = {"op": op}
    mix = lambda values: torch.tensor(values, device=dev)[torch.randperm(len(values), generator=g, device=dev)]  # noqa: E731
    if op == "prefix_attention":
        d, hq, hkv, qlen, dt = case["dim"], case["hq"], case["hkv"], case["qlen"], TYPES[case["dtype"]]
        cut, pages = _groups(case)
        suffix = mix(_suffixes(case))                       # tokens of each row's own before this step
        sizes = torch.tensor([b - a for a, b in zip(cut, cut[1:])], device=dev)
        group = torch.repeat_interleave(torch.arange(len(pages), device=dev), sizes, output_size=rows)
        shared = torch.tensor(pages, device=dev)[group]
        lengths = shared * PAGE + suffix
        width = max(pages) + -(-(case["suffix_hi"] + qlen) // PAGE)
        # one page of the pool for each shared page and each page of a row's own, in random places
        n_shared = sum(pages)
        mine = -(-(suffix + qlen) // PAGE)
        n_pages = n_shared + rows * (width + 1)
        place = torch.randperm(n_pages, generator=g, device=dev)
        first = torch.cumsum(torch.tensor([0] + pages, device=dev), 0)
        col = torch.arange(width, device=dev).view(1, -1)
        at = torch.where(col < shared.view(-1, 1), first[group].view(-1, 1) + col,
                         n_shared + torch.arange(rows, device=dev).view(-1, 1) * (width + 1) + col - shared.view(-1, 1))
        table = torch.where(col < (shared + mine).view(-1, 1), place[at.clamp(0, n_pages - 1)], -1)
        # keys with a few strong channels and values with a bias, as trained layers have
        k = torch.randn(n_pages, hkv, PAGE, d, generator=g, device=dev, dtype=torch.float32)
        k += 2.0 * torch.randn(1, hkv, 1, d, generator=g, device=dev)
        state["k"] = k.to(dt)
        v = torch.randn(n_pages, hkv, PAGE, d, generator=g, device=dev, dtype=torch.float32, out=k)
        v += 0.5 * torch.randn(1, hkv, 1, d, generator=g, device=dev)
        state["v"] = v.to(dt)
        # queries as a projection writes them: [rows, qlen, heads, dim] seen head first
        state["q"] = torch.randn(rows, qlen, hq, d, generator=g, device=dev).to(dt).transpose(1, 2)
        state["lengths"] = lengths
        state["table"] = table.to(torch.int32).contiguous()
        state["starts"] = torch.tensor(cut, dtype=torch.int32, device=dev)
        state["pages"] = torch.tensor(pages, dtype=torch.int32, device=dev)
    elif op == "token_logprobs":
        vocab, dt = case["vocab"], TYPES[case["dtype"]]
        # a spread of logits under a Zipf prior, another order of the vocabulary for each row
        x = torch.randn(rows, vocab + case["pad"], generator=g, device=dev) * 3.0
        prior = -1.1 * torch.log(torch.arange(1, vocab + case["pad"] + 1, device=dev, dtype=torch.float32))
        shift = torch.randint(0, vocab, (rows, 1), generator=g, device=dev)
        order = torch.randperm(vocab + case["pad"], generator=g, device=dev).view(1, -1)
        x += prior[(order + shift) % (vocab + case["pad"])]
        state["logits"] = x.to(dt)[:, :vocab]
        # half of the tokens are likely ones, half are any
        likely = state["logits"].argmax(-1)
        anyone = torch.randint(0, vocab, (rows,), generator=g, device=dev)
        state["ids"] = torch.where(torch.rand(rows, generator=g, device=dev) < 0.5, likely, anyone)
        state["temperature"], state["top"] = case["temperature"], min(case["top"], vocab)
    else:
        width = case["width"]
        if case["ragged"]:
            lengths = torch.zeros(rows, dtype=torch.long, device=dev)
            new = mix(_spread(1, case["new"], rows))
        else:
            lengths = mix(_spread(case["lo"], case["hi"], rows))
            new = case["new"]
        n_pages = rows * width
        place = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
        owned = -(-lengths // PAGE)
        col = torch.arange(width, device=dev).view(1, -1)
        at = torch.arange(rows, device=dev).view(-1, 1) * width + col
        mapped = col < owned.view(-1, 1)
        state["table"] = torch.where(mapped, place[at], -1).to(torch.int32).contiguous()
        state["owned"] = owned.to(torch.int32)
        # a quarter of the rows hold their first page for somebody else
        held = torch.rand(rows, generator=g, device=dev) < 0.25
        state["shared"] = torch.minimum(owned, held.long()).to(torch.int32)
        rest = place[torch.where(~mapped.view(-1), at.view(-1), 0)]
        left = torch.sort(torch.where(mapped.view(-1), 1, 0), stable=True)[1]
        state["free"] = torch.where(torch.arange(n_pages, device=dev) < (~mapped).sum(), rest[left], -1).to(torch.int32)
        state["n_free"] = (~mapped).sum().to(torch.int32).view(1)
        state["err"] = torch.zeros(1, dtype=torch.int32, device=dev)
        state["lengths"], state["new"], state["tokens"] = lengths, new, _tokens(case)
    return state


# ---- one pass -----------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"prefix_attention": _attention, "token_logprobs": _logprobs, "page_table": _table}[state["op"]](state)


def _run_own(s):
    _package()
    if s["op"] == "prefix_attention":
        from specdec.attention import prefix_attention
        return prefix_attention(s["q"], s["k"], s["v"], s["lengths"], s["table"], s["starts"], s["pages"])
    if s["op"] == "token_logprobs":
        from specdec.sampling import token_logprobs
        r = token_logprobs(s["logits"], s["ids"], temperature=s["temperature"], top_n=s["top"])
        out = {"logprob": r.logprob, "rank": r.rank, "entropy": r.entropy}
        return out | {"top_ids": r.top_ids, "top_logprobs": r.top_logprobs} if s["top"] else out
    from specdec.kvcache import DevicePageTable
    t = DevicePageTable.over(s["table"], s["owned"], s["shared"], s["free"], s["n_free"], s["err"])
    t.trim(s["lengths"])
    slots, starts = t.reserve(s["lengths"], s["new"], max_tokens=s["tokens"])
    return {"table": s["table"], "owned": s["owned"], "free": s["free"], "n_free": s["n_free"], "err": s["err"],
            "slots": slots, "starts": starts}


def _attention(s):
    """Every row over its own pages: query j of row b sees the keys s <= lengths[b] + j."""
    q, table, lengths = s["q"], s["table"].long().clamp_min(0), s["lengths"]
    rows, hq, qlen, d = q.shape
    hkv, width = s["k"].shape[1], table.shape[1]
    by_head = lambda pool: pool[table].permute(0, 2, 1, 3, 4).reshape(rows, hkv, width * PAGE, d).float()  # noqa: E731
    qg = q.float().reshape(rows, hkv, (hq // hkv) * qlen, d)
    scores = torch.matmul(qg, by_head(s["k"]).transpose(-1, -2)).view(rows, hkv, hq // hkv, qlen, width * PAGE)
    scores *= d ** -0.5
    last = lengths.view(-1, 1) + torch.arange(qlen, device=q.device)
    hidden = torch.arange(width * PAGE, device=q.device) > last.view(rows, 1, 1, qlen, 1)
    scores.masked_fill_(hidden, -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(rows, hkv, -1, width * PAGE), by_head(s["v"])).view(rows, hkv, hq // hkv, qlen, d) / total
    return o.view(rows, hq, qlen, d).transpose(1, 2).contiguous().to(q.dtype)


def _logprobs(s):
    """Ranks and alternatives by falling logit, of equal ones the lowest id first."""
    x, ids, n = s["logits"].float(), s["ids"].view(-1, 1), s["top"]
    y = x / s["temperature"]
    below = y - y.amax(-1, keepdim=True)
    e = below.exp()
    z = e.sum(-1, keepdim=True)
    logz = z.log()
    own_x = x.gather(1, ids)
    earlier = torch.arange(x.shape[1], device=x.device).view(1, -1) < ids
    rank = 1 + ((x > own_x) | ((x == own_x) & earlier)).sum(-1)
    entropy = logz - (below * e).sum(-1, keepdim=True) / z
    out = {"logprob": (below.gather(1, ids) - logz).view(-1), "rank": rank, "entropy": entropy.view(-1)}
    if n:
        top = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :n].contiguous()
        out |= {"top_ids": top, "top_logprobs": below.gather(1, top) - logz}
    return out


def _table(s):
    """Pages past each row's tokens go back, then pages for its new tokens come out, first to last."""
    table, free, n_free, lengths, width = s["table"], s["free"], s["n_free"], s["lengths"], s["table"].shape[1]
    rows, dev = table.shape[0], table.device
    col = torch.arange(width, device=dev).view(1, -1)
    # back: the last page of the last row ends lowest on the stack
    owned = s["owned"].long()
    keep = torch.minimum(torch.maximum(-(-lengths // PAGE), s["shared"].long()), owned)
    gone = ((col >= keep.view(-1, 1)) & (col < owned.view(-1, 1))).view(-1)
    order = torch.cumsum(gone, 0)
    spare = torch.cat([free, free.new_zeros(1)])
    at = torch.where(gone, n_free + order[-1] - order, free.numel())
    spare.index_put_((at,), table.view(-1))
    free.copy_(spare[:-1])
    table.copy_(torch.where(gone.view(rows, width), -1, table))
    n_free += order[-1].to(torch.int32)
    # out: the top of the stack goes to the first row's first missing page
    new = torch.full_like(lengths, s["new"]) if isinstance(s["new"], int) else s["new"]
    need = -(-(lengths + new) // PAGE)
    short = (need - keep).clamp_min(0)
    fits = (need <= width).all() & (short.sum() <= n_free)
    short *= fits
    missing = ((col >= keep.view(-1, 1)) & (col < (keep + short).view(-1, 1))).view(-1)
    taken = torch.cumsum(missing, 0)
    page = free[(n_free - taken).clamp_min(0)]
    table.copy_(torch.where(missing, page, table.view(-1)).view(rows, width))
    s["owned"].copy_(keep + short)
    n_free -= short.sum().to(torch.int32)
    starts = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    token = torch.arange(s["tokens"], device=dev)
    row = torch.searchsorted(starts[1:], token, right=True).clamp_max(rows - 1)
    place = lengths[row] + token - starts[row]
    slots = table[row, place // PAGE].long() * PAGE + place % PAGE
    slots = torch.where((token < starts[-1]) & fits, slots, -1)
    return {"table": table, "owned": s["owned"], "free": free, "n_free": n_free, "err": s["err"], "slots": slots,
            "starts": starts.to(torch.int32)}


# ---- the definitions in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prefix_attention":
        q, k, v, table = s["q"], s["k"], s["v"], s["table"].tolist()
        rows, hq, qlen, d = q.shape
        hkv = k.shape[1]
        out = torch.empty(rows, qlen, hq, d, dtype=torch.float64, device=q.device)
        for b, n in enumerate(s["lengths"].tolist()):
            pages = torch.tensor(table[b][:-(-(n + qlen) // PAGE)], device=q.device)
            kb = torch.cat(list(k[pages].double()), 1)[:, :n + qlen]       # [kv heads, keys, dim]
            vb = torch.cat(list(v[pages].double()), 1)[:, :n + qlen]
            for j in range(qlen):
                w = torch.einsum("hgd,hsd->hgs", q[b, :, j].double().view(hkv, hq // hkv, d), kb[:, :n + j + 1])
                w = torch.softmax(w / math.sqrt(d), -1)
                out[b, j] = torch.einsum("hgs,hsd->hgd", w, vb[:, :n + j + 1]).reshape(hq, d)
        return out
    if case["op"] == "token_logprobs":
        outs = []
        for x, t in zip(s["logits"].split(64), s["ids"].split(64)):
            lp = torch.log_softmax(x.double() / case["temperature"], -1)
            got = [lp.gather(1, t.view(-1, 1)).view(-1), -(lp.exp() * lp).sum(-1)]
            if s["top"]:
                got.append(torch.topk(lp, s["top"], -1)[0])
            outs.append(got)
        got = [torch.cat(c) for c in zip(*outs)]
        out = {"logprob": got[0], "rank": None, "entropy": got[1]}
        return out | {"top_ids": None, "top_logprobs": got[2]} if s["top"] else out
    return None
