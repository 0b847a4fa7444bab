"""Speed cases of the operators for trees of drafted tokens and constrained logits: attention of a
tree's nodes over the cache, the accepted path with the compaction of the cache behind it, and
penalties, biases and grammar masks on the logits of every node.

``run`` computes them in plain torch operations (``own`` false) or through the package (``own``
true).  Shapes: the engine's benchmark models (32 / 8 heads and 36 layers, 16 / 8 heads and 28 layers,
heads of 128, 151936 tokens of vocabulary), its 128-token pages, and batches, trees and contexts
around them.
"""
import math
import pathlib
import random
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

def _attn(name, rows, nodes, first, hq, hkv, lengths, paged, ragged, dim=128, dtype="bf16"):
    return {"name": name, "op": "tree_attention", "rows": rows, "nodes": nodes, "first": first, "hq": hq, "hkv": hkv,
            "dim": dim, "len_lo": lengths[0], "len_hi": lengths[1], "paged": paged, "ragged": ragged, "dtype": dtype}


def _commit(name, rows, nodes, depth, layers, hkv, lengths, paged, dim=128, dtype="bf16"):
    return {"name": name, "op": "tree_commit", "rows": rows, "nodes": nodes, "depth": depth, "layers": layers,
            "hkv": hkv, "dim": dim, "len_lo": lengths[0], "len_hi": lengths[1], "paged": paged, "dtype": dtype}


def _logits(name, rows, nodes, tree, vocab, dtype, penalties, biases, mask, pad=0):
    return {"name": name, "op": "process_logits", "rows": rows, "nodes": nodes, "tree": tree, "vocab": vocab,
            "dtype": dtype, "penalties": penalties, "biases": biases, "mask": mask, "pad": pad}


def listed():
    return [
        # one request, a small tree behind a short prompt: nothing but latency
        _attn("attn_one", 1, 8, 0, 32, 8, (40, 40), 0, 0),
        # the small model drafts the third level of a tree (nodes 5 to 12) for the engine benchmark's batch
        _attn("attn_level", 32, 13, 5, 16, 8, (512, 700), 1, 0),
        # a verify step of trees of 26 nodes at the lengths of the serving sweep, contiguous cache
        _attn("attn_verify", 32, 26, 0, 32, 8, (128, 4096), 0, 0),
        # trees of 64 nodes, each row another one with some nodes missing, long contexts, paged
        _attn("attn_wide", 64, 64, 0, 32, 8, (512, 8192), 1, 1),
        # one long document, as many key heads as query heads, an odd number of nodes
        _attn("attn_document", 2, 33, 0, 8, 8, (30011, 30011), 0, 1),
        # fp32 rows of a small model with heads of 64
        _attn("attn_fp32", 8, 9, 0, 8, 2, (1, 460), 1, 0, dim=64, dtype="fp32"),
        # the accepted path of one request's tree into the small model's cache
        _commit("commit_one", 1, 8, 4, 28, 8, (40, 40), 0),
        # the same for 32 rows of the large model, contiguous cache
        _commit("commit_round", 32, 26, 5, 36, 8, (60, 200), 0),
        # 64 rows, wide trees, paged
        _commit("commit_paged", 64, 64, 8, 36, 8, (1, 150), 1),
        # penalties on the logits of a draft step of one request
        _logits("logits_step", 1, 1, 0, VOCAB, "bf16", 1, 0, 0),
        # every position of a verify round of 64 rows (k = 4): penalties, some biases and a grammar
        _logits("logits_verify", 64, 5, 0, VOCAB, "bf16", 1, 16, 1),
        # every node of 32 trees; fp32 logits of an odd vocabulary are among the drawn cases
        _logits("logits_tree", 32, 26, 1, VOCAB, "bf16", 1, 0, 1),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree_attention", "tree_attention", "tree_commit", "process_logits", "process_logits"])
    if op == "process_logits":
        vocab = rng.choice([VOCAB, 32003, _log_between(rng, 40, 260000)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        nodes = rng.choice([1, 2, 5, 9, 26, 64])
        most = 126_000_000 // (vocab * nodes * (2 if dtype == "fp32" else 1))
        rows = _log_between(rng, 1, max(1, min(256, most)))
        penalties, mask = rng.choice([(0, 1), (1, 0), (1, 1)])
        return _drawn(_logits("", rows, nodes, rng.randint(0, 1), vocab, dtype, penalties, rng.choice([0, 1, 16, 300]),
                              mask, rng.choice([0, 0, 1, 8])))
    if op == "tree_commit":
        rows, nodes, layers = _log_between(rng, 1, 64), rng.randint(2, 64), rng.choice([1, 28, 36])
        hkv, dim, dtype = rng.choice([1, 2, 8]), rng.choice([64, 128]), rng.choice(["bf16", "bf16", "fp32"])
        hi = _log_between(rng, 2, 150)
        return _drawn(_commit("", rows, nodes, rng.randint(1, min(8, nodes - 1)), layers, hkv, (rng.randint(1, hi), hi),
                              rng.randint(0, 1), dim, dtype))
    if rng.random() < 0.15:
        nodes, hi = rng.randint(1, 16), _log_between(rng, 1, 600)
        return _drawn(_attn("", _log_between(rng, 1, 16), nodes, rng.randrange(nodes), 8, rng.choice([1, 2, 8]),
                            (rng.randint(0, hi), hi), rng.randint(0, 1), rng.randint(0, 1), dim=rng.choice([64, 128]),
                            dtype="fp32"))
    hq, hkv = rng.choice([(32, 8), (32, 8), (16, 8), (8, 8), (16, 2)])
    rows, nodes = _log_between(rng, 1, 128), _log_between(rng, 1, 100)
    hi = _log_between(rng, 1, 30000)
    case = _drawn(_attn("", rows, nodes, rng.choice([0, 0, rng.randrange(nodes)]), hq, hkv,
                        (rng.choice([hi, 0, hi // 2]), hi), rng.randint(0, 1), rng.randint(0, 1)))
    top = next(c for c in listed() if c["name"] == "attn_wide")
    while work(case)["flops"] > work(top)["flops"] or _cells(case) > _cells(top):
        case["rows"] = max(1, case["rows"] // 2)
        if case["rows"] == 1:
            case["len_hi"] = case["len_hi"] // 2 + 1
            case["len_lo"] = min(case["len_lo"], case["len_hi"])
    return case


def _drawn(case):
    del case["name"]
    return case


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _cells(case):
    """Elements of the keys of all rows, counted at the longest row."""
    return case["rows"] * (case["len_hi"] + case["nodes"]) * case["hkv"] * case["dim"]


def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def work(case):
    rows, e = case["rows"], _size(case)
    if case["op"] == "tree_attention":
        base, q = sum(_spread(case["len_lo"], case["len_hi"], rows)), case["nodes"] - case["first"]
        hq, hkv, d = case["hq"], case["hkv"], case["dim"]
        return {"bytes": e * (2 * d * hkv * (base + rows * case["nodes"]) + 2 * rows * q * hq * d),
                "flops": 4 * (base + 3 * rows) * q * hq * d}
    if case["op"] == "tree_commit":
        # about half of an accepted path is not where it belongs
        moved = rows * max(1, case["depth"] // 2)
        return {"bytes": 2 * moved * case["layers"] * 2 * case["hkv"] * case["dim"] * e + rows * case["nodes"] * 20,
                "flops": rows * case["nodes"]}
    n = rows * case["nodes"] * case["vocab"]
    return {"bytes": 2 * n * e + (2 * rows * case["vocab"] if case["penalties"] else 0) + (n // 8 if case["mask"] else 0),
            "flops": 4 * n}


# ---- inputs -------------------------------------------------------------------------------------

def _parents(rng, nodes, depth, missing):
    """Parents of a random tree in breadth-first order, -1 for the root and -2 for nodes that it lacks."""
    parents, level = [-1], [0]
    there = nodes - (rng.randint(0, nodes // 4) if missing else 0)
    for i in range(1, nodes):
        # (the youngest of the nodes that may still have children, or any)
        open_ = [j for j in range(i) if level[j] < depth and parents[j] > -2]
        p = rng.choice(open_[-max(1, len(open_) // 2):]) if i < there else -2
        parents.append(p)
        level.append(level[p] + 1 if p >= 0 else 0)
    return parents


def _masks(parents):
    """Ancestor bits (the node's own among them) as int32 words [trees, nodes, words], for lists of parents."""
    words = -(-len(parents[0]) // 32)
    out = []
    for tree in parents:
        bits = []
        for i, p in enumerate(tree):
            bits.append(0 if p < -1 else (1 << i) | (bits[p] if p >= 0 else 0))
        out.append([[((b >> (32 * w)) & 0xFFFFFFFF) for w in range(words)] for b in bits])
    m = torch.tensor(out, dtype=torch.int64)
    return torch.where(m >= 1 << 31, m - (1 << 32), m).to(torch.int32)


def _pool(rows, width, g, dev):
    """(pages, block table [rows, width]) of a pool with every row's pages in random places."""
    n = rows * width
    place = torch.randperm(n, generator=g, device=dev)
    return n, place.view(rows, width).to(torch.int32).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    rows, nodes, dt = case["rows"], case["nodes"], TYPES[case["dtype"]]
    state = {"op": case["op"]}
    mix = lambda values: torch.tensor(values, device=dev)[torch.randperm(len(values), generator=g, device=dev)]  # noqa: E731
    if case["op"] == "tree_attention":
        d, hq, hkv, first = case["dim"], case["hq"], case["hkv"], case["first"]
        depth = max(1, min(8, nodes // 2))
        trees = [_parents(rng, nodes, depth, case["ragged"]) for _ in range(rows if case["ragged"] else 1)]
        state["masks"] = _masks(trees).to(dev)
        base = mix(_spread(case["len_lo"], case["len_hi"], rows))
        state["lengths"] = base + first
        capacity = case["len_hi"] + nodes + 3
        if case["paged"]:
            width = -(-capacity // PAGE)
            n, state["table"] = _pool(rows, width, g, dev)
            shape = (n, hkv, PAGE, d)
        else:
            state["table"] = None
            shape = (rows, hkv, capacity, d)
        # keys with a few strong channels and values with a bias, as trained layers have
        k = torch.randn(shape, generator=g, device=dev, dtype=torch.float32)
        k += 2.0 * torch.randn(1, hkv, 1, d, generator=g, device=dev)
        state["k"] = k.to(dt)
        v = torch.randn(shape, generator=g, device=dev, dtype=torch.float32, out=k)
        v += 0.5 * torch.randn(1, hkv, 1, d, generator=g, device=dev)
        state["v"] = v.to(dt)
        # queries as a projection writes them: [rows, nodes, heads, dim] seen head first
        state["q"] = torch.randn(rows, nodes - first, hq, d, generator=g, device=dev).to(dt).transpose(1, 2)
        state["first"] = first
    elif case["op"] == "tree_commit":
        d, hkv, layers = case["dim"], case["hkv"], case["layers"]
        trees = [_parents(rng, nodes, case["depth"], 0) for _ in range(rows)]
        state["masks"] = _masks(trees).to(dev)
        # siblings hold different tokens; two times out of three the target model agrees with one of the children
        tokens = [rng.sample(range(VOCAB), nodes) for _ in range(rows)]
        choices = []
        for tree, t in zip(trees, tokens):
            children = [[j for j in range(nodes) if tree[j] == i] for i in range(nodes)]
            choices.append([t[rng.choice(c)] if c and rng.random() < 0.67 else rng.randrange(VOCAB) for c in children])
        state["tokens"], state["choices"] = torch.tensor(tokens, device=dev), torch.tensor(choices, device=dev)
        state["after"] = mix(_spread(case["len_lo"], case["len_hi"], rows)) + nodes
        state["lengths"] = state["after"].clone()
        state["most"] = case["depth"] + 1
        capacity = case["len_hi"] + nodes + 3
        if case["paged"]:
            n, state["table"] = _pool(rows, -(-capacity // PAGE), g, dev)
            shape = (layers, n, hkv, PAGE, d)
        else:
            state["table"] = None
            shape = (layers, rows, hkv, capacity, d)
        state["k"] = torch.empty(shape, dtype=dt, device=dev).normal_(generator=g)
        state["v"] = torch.empty(shape, dtype=dt, device=dev).normal_(generator=g)
    else:
        vocab = case["vocab"]
        # a spread of logits under a Zipf prior, another order of the vocabulary for each row
        x = torch.empty(rows, nodes, vocab + case["pad"], device=dev, dtype=dt)
        prior = -1.1 * torch.log(torch.arange(1, vocab + case["pad"] + 1, device=dev, dtype=torch.float32))
        order = torch.randperm(vocab + case["pad"], generator=g, device=dev)
        for b in range(rows):
            y = torch.randn(nodes, vocab + case["pad"], generator=g, device=dev) * 3.0
            x[b] = y + prior[(order + rng.randrange(vocab)) % (vocab + case["pad"])] + 6.0
        state["logits"] = x[..., :vocab]
        state["masks"] = _masks([_parents(rng, nodes, 8, 0)]).to(dev) if case["tree"] else None
        # tokens that were written before are likely to be drafted again
        likely = state["logits"][:, 0].topk(min(vocab, 64), dim=-1)[1]
        pick = torch.randint(0, likely.shape[1], (rows, nodes), generator=g, device=dev)
        state["tokens"] = likely.gather(1, pick)
        state["history"] = state["repetition"] = state["presence"] = state["frequency"] = None
        if case["penalties"]:
            # a prompt of 1500 tokens and 400 written ones, a quarter of these likely ones
            prompt = torch.randint(0, vocab, (rows, 1500), generator=g, device=dev)
            wrote = torch.randint(0, vocab, (rows, 400), generator=g, device=dev)
            at = torch.randint(0, likely.shape[1], (rows, 100), generator=g, device=dev)
            wrote[:, :100] = likely.gather(1, at)
            count = torch.zeros(rows, vocab, dtype=torch.int32, device=dev)
            count.scatter_add_(1, wrote, torch.ones_like(wrote, dtype=torch.int32))
            seen = torch.zeros(rows, vocab, dtype=torch.bool, device=dev).scatter_(1, prompt, True)
            # low 15 bits: times written; the sign bit: in the prompt
            state["history"] = torch.where(seen, count - 32768, count).to(torch.int16)
            state["repetition"] = mix(_spread(100, 130, rows)).float() / 100
            state["presence"] = mix(_spread(0, 60, rows)).float() / 100
            state["frequency"] = mix(_spread(-10, 40, rows)).float() / 100
        state["bias"] = None
        if case["biases"]:
            n = min(case["biases"], vocab)
            ids = torch.rand(rows, vocab, generator=g, device=dev).topk(n, dim=-1)[1]
            state["bias"] = (ids, torch.randn(rows, n, generator=g, device=dev) * 5.0)
        state["mask"] = None
        if case["mask"]:
            # a bit for each token: some positions allow a handful of tokens, some nearly all, some a part
            words = -(-vocab // 32)
            full = torch.randint(-2 ** 31, 2 ** 31, (rows, nodes, words), generator=g, device=dev, dtype=torch.int64)
            kind = torch.randint(0, 3, (rows, nodes, 1), generator=g, device=dev)
            bit = torch.randint(0, 31, full.shape, generator=g, device=dev)
            rare = torch.rand(full.shape, generator=g, device=dev) < 0.002
            few = torch.where(rare, 1 << bit, 0)
            state["mask"] = torch.where(kind == 0, few, torch.where(kind == 1, -1 - few, full)).to(torch.int32)
    return state


# ---- one pass -----------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"tree_attention": _attention, "tree_commit": _accept_commit, "process_logits": _process}[state["op"]](state)


def _run_own(s):
    _package()
    if s["op"] == "tree_attention":
        from specdec.attention import tree_attention
        return tree_attention(s["q"], s["k"], s["v"], s["lengths"], s["masks"], first=s["first"], block_table=s["table"])
    if s["op"] == "tree_commit":
        from specdec.kvcache import commit_tree
        from specdec.tree import tree_accept
        s["lengths"].copy_(s["after"])                       # the verify forward advanced the cache
        r = tree_accept(s["tokens"], s["choices"], s["masks"], max_path=s["most"])
        commit_tree(s["k"].unbind(0), s["v"].unbind(0), s["lengths"], r.path, r.n_acc, s["tokens"].shape[1],
                    block_table=s["table"])
        return {"k": s["k"], "v": s["v"], "lengths": s["lengths"], "n_acc": r.n_acc, "y": r.y, "path": r.path}
    from specdec.sampling import process_logits
    return process_logits(s["logits"], s["tokens"], s["masks"], history=s["history"], repetition=s["repetition"],
                          presence=s["presence"], frequency=s["frequency"], bias=s["bias"], allowed=s["mask"])


def _bits(masks):
    """Ancestor words [trees, nodes, words] as truth values [trees, nodes, nodes]."""
    n = torch.arange(masks.shape[1], device=masks.device)
    return ((masks[:, :, n // 32] >> (n % 32)) & 1).bool()


def _attention(s):
    """Node i of row b, in slot base + i, sees the slots below base and those of its ancestors and itself."""
    q, lengths, first = s["q"], s["lengths"], s["first"]
    rows, hq, qlen, d = q.shape
    hkv = s["k"].shape[1]
    if s["table"] is None:
        by_head = lambda cache: cache.float()  # noqa: E731
    else:
        table = s["table"].long()
        by_head = lambda pool: pool[table].permute(0, 2, 1, 3, 4).reshape(rows, hkv, -1, d).float()  # noqa: E731
    qg = q.float().reshape(rows, hkv, (hq // hkv) * qlen, d)
    scores = torch.matmul(qg, by_head(s["k"]).transpose(-1, -2))
    keys = scores.shape[-1]
    scores = scores.view(rows, hkv, hq // hkv, qlen, keys)
    scores *= d ** -0.5
    tree = _bits(s["masks"])[:, first:].expand(rows, -1, -1)                       # [rows, qlen, nodes]
    there = tree.any(-1, keepdim=True)
    at = torch.arange(keys, device=q.device).view(1, 1, -1) - (lengths - first).view(-1, 1, 1)
    seen = tree.gather(2, at.clamp(0, tree.shape[2] - 1).expand(rows, qlen, -1)) & (at >= 0) & (at < tree.shape[2])
    seen = (seen | (at < 0)) & there
    scores.masked_fill_(~seen.view(rows, 1, 1, qlen, keys), -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = scores.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(rows, hkv, -1, keys), by_head(s["v"])).view(rows, hkv, hq // hkv, qlen, d)
    o = torch.where(total > 0, o / total, 0.0)
    return o.view(rows, hq, qlen, d).transpose(1, 2).contiguous().to(q.dtype)


def _accept_commit(s):
    """The path from the root along children that hold their parent's choice, moved to the slots behind the row's tokens."""
    tokens, choices, lengths, most = s["tokens"], s["choices"], s["lengths"], s["most"]
    rows, nodes = tokens.shape
    dev = tokens.device
    lengths.copy_(s["after"])
    tree = _bits(s["masks"]).expand(rows, -1, -1)
    index = torch.arange(nodes, device=dev)
    above = tree & (index.view(-1, 1) > index)                                     # ancestors without the node
    parent = torch.where(above, index, -1).amax(-1)                                # the youngest of them
    fits = (parent >= 0) & (tokens == choices.gather(1, parent.clamp_min(0)))
    twin = (parent.unsqueeze(2) == parent.unsqueeze(1)) & fits.unsqueeze(1) & (index < index.view(-1, 1))
    fits &= ~twin.any(-1)                                                          # an older sibling holds it, too
    fits[:, 0] = True
    on = (fits.unsqueeze(1) | ~tree).all(-1) & tree[:, :, 0]
    order = torch.sort(torch.where(on, index, nodes), dim=-1)[0][:, :most]
    path = torch.where(order < nodes, order, -1).to(torch.int32)
    n_acc = (path >= 0).sum(-1) - 1
    y = choices.gather(1, path.long().gather(1, n_acc.view(-1, 1))).view(-1)
    base = lengths - nodes
    to = base.view(-1, 1) + torch.arange(most, device=dev)
    frm = torch.where(path >= 0, base.view(-1, 1) + path, to)
    row = torch.arange(rows, device=dev).view(-1, 1)
    for cache in (s["k"], s["v"]):
        if s["table"] is None:
            cache[:, row, :, to] = cache[:, row, :, frm]
        else:
            t = s["table"].long()
            cache[:, t[row, to // PAGE], :, to % PAGE] = cache[:, t[row, frm // PAGE], :, frm % PAGE]
    lengths.copy_(base + 1 + n_acc)
    return {"k": s["k"], "v": s["v"], "lengths": lengths, "n_acc": n_acc, "y": y, "path": path}


def _path_counts(s, dtype):
    """Times that each token stands on the way to each node, [rows, nodes, vocab]."""
    rows, nodes, vocab = s["logits"].shape
    dev = s["tokens"].device
    tree = torch.ones(1, nodes, nodes, dtype=torch.bool, device=dev).tril() if s["masks"] is None else _bits(s["masks"])
    c = torch.zeros(rows, nodes, vocab, dtype=dtype, device=dev)
    return c.scatter_add_(2, s["tokens"].unsqueeze(1).expand(rows, nodes, nodes), tree.expand(rows, -1, -1).to(dtype))


def _process(s):
    """Penalties by what the row and the node's path hold, then biases, then the tokens that the grammar allows."""
    x = s["logits"].float()
    rows, nodes, vocab = x.shape
    if s["history"] is not None:
        h = s["history"].unsqueeze(1)
        per_row = lambda t: t.view(-1, 1, 1)  # noqa: E731
        c = _path_counts(s, torch.float32)
        c += h & 0x7FFF
        wrote = c > 0
        r = per_row(s["repetition"])
        x = torch.where(wrote | (h < 0), torch.where(x > 0, x / r, x * r), x)
        x -= c * per_row(s["frequency"])
        x -= wrote * per_row(s["presence"])
    if s["bias"] is not None:
        ids, values = s["bias"]
        x = x.scatter_add(2, ids.unsqueeze(1).expand(-1, nodes, -1), values.unsqueeze(1).expand(-1, nodes, -1))
    if s["mask"] is not None:
        t = torch.arange(vocab, device=x.device)
        x = x.masked_fill(((s["mask"][:, :, t // 32] >> (t % 32).to(torch.int32)) & 1) == 0, -math.inf)
    return x.to(s["logits"].dtype)


# ---- the definitions in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "tree_commit":
        return None
    s = prepare(case, seed)
    if case["op"] == "tree_attention":
        q, k, v, first = s["q"], s["k"], s["v"], s["first"]
        rows, hq, qlen, d = q.shape
        hkv = k.shape[1]
        masks = s["masks"].tolist()
        out = torch.zeros(rows, qlen, hq, d, dtype=torch.float64, device=q.device)
        for b, n in enumerate((s["lengths"] - first).tolist()):
            tree = masks[b if len(masks) > 1 else 0]
            nodes = len(tree)
            if s["table"] is None:
                kb, vb = k[b, :, :n + nodes].double(), v[b, :, :n + nodes].double()
            else:
                pages = s["table"][b, :-(-(n + nodes) // PAGE)].long()
                kb, vb = (torch.cat(list(x[pages].double()), 1)[:, :n + nodes] for x in (k, v))
            sees = torch.zeros(qlen, n + nodes, dtype=torch.bool)
            for j in range(qlen):
                word = tree[first + j]
                path = [a for a in range(nodes) if word[a // 32] >> (a % 32) & 1]
                if path:
                    sees[j, :n] = True
                    sees[j, [n + a for a in path]] = True
            live = sees.any(-1).to(q.device)
            w = torch.einsum("hgjd,hsd->hgjs", q[b].double().view(hkv, hq // hkv, qlen, d), kb) / math.sqrt(d)
            w = torch.softmax(w.masked_fill(~sees.to(q.device), -math.inf), -1)
            o = torch.einsum("hgjs,hsd->jhgd", w, vb).reshape(qlen, hq, d)
            out[b] = torch.where(live.view(-1, 1, 1), o, 0.0)
        return out
    x = s["logits"]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    tree = None if s["masks"] is None else s["masks"][0].tolist()
    for b in range(x.shape[0]):
        for i in range(x.shape[1]):
            z = x[b, i].double()
            if s["history"] is not None:
                h = s["history"][b].long()
                way = [a for a in range(x.shape[1]) if (a <= i if tree is None else tree[i][a // 32] >> (a % 32) & 1)]
                c = torch.remainder(h, 32768) + torch.bincount(s["tokens"][b, way], minlength=h.numel())
                r = s["repetition"][b].double()
                z = torch.where((c > 0) | (h < 0), torch.where(z > 0, z / r, z * r), z)
                z = z - s["frequency"][b].double() * c - s["presence"][b].double() * (c > 0)
            if s["bias"] is not None:
                z = z.index_add(0, s["bias"][0][b], s["bias"][1][b].double())
            if s["mask"] is not None:
                bits = (s["mask"][b, i].long().view(-1, 1) >> torch.arange(32, device=x.device)) & 1
                z = torch.where(bits.reshape(-1)[:z.numel()] == 1, z, -math.inf)
            out[b, i] = z
    return out
