"""Ancestor bits, the accepted path and the cache behind it, against plain loops.  All results
are whole numbers or copies: exact."""
import pytest
import torch

from specdec import _lib as L
from specdec import attention as A
from specdec.kvcache import PAGE, PagedRaggedCache, RaggedCache, commit_tree
from specdec.tree import TREE_MAX, tree_accept, tree_masks, tree_of_widths

gpu = pytest.mark.gpu
DEV = "cuda"


def _masks_plain(tree):
    """Sets of a tree's ancestors (with the node), empty for absent ones, and the depths."""
    sees, depth = [], []
    for i, p in enumerate(tree):
        ok = p == -1 or (0 <= p < i and sees[p])
        sees.append(({i} | (sees[p] if p >= 0 else set())) if ok else set())
        depth.append(depth[p] + 1 if ok and p >= 0 else 0)
    return sees, depth


def _sets(masks):
    return [[{32 * w + k for w, word in enumerate(node) for k in range(32) if word >> k & 1}
             for node in tree] for tree in masks.tolist()]


def _random_parents(n, g):
    """Any earlier node, now and then a root, an absent node or nonsense."""
    out = [-1]
    for i in range(1, n):
        k = int(torch.randint(0, 20, (1,), generator=g))
        out.append(-1 if k == 0 else -2 if k == 1 else i if k == 2 else 1000 if k == 3
                   else int(torch.randint(0, i, (1,), generator=g)))
    return out


@gpu
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 100, TREE_MAX])
def test_masks(n):
    g = torch.Generator().manual_seed(n)
    trees = [_random_parents(n, g) for _ in range(5)] + [list(range(-1, n - 1)), [-1] * n, [-2] * n]
    got = tree_masks(torch.tensor(trees), device=DEV)
    want = [_masks_plain(t) for t in trees]
    assert got.masks.shape == (8, n, -(-n // 32)) and got.masks.dtype == torch.int32
    assert _sets(got.masks) == [w[0] for w in want]
    assert got.depths.tolist() == [w[1] for w in want]
    one = tree_masks(trees[0], device=DEV)
    assert torch.equal(one.masks, got.masks[0]) and torch.equal(one.depths, got.depths[0])
    strided = torch.tensor(trees, dtype=torch.int32, device=DEV).t().contiguous().t()
    assert torch.equal(tree_masks(strided).masks, got.masks)


def test_tree_of_widths():
    assert tree_of_widths([]) == ([-1], [0, 1])
    assert tree_of_widths([2, 1]) == ([-1, 0, 0, 1, 2], [0, 1, 3, 5])
    parents, starts = tree_of_widths((3, 2))
    assert parents == [-1, 0, 0, 0, 1, 1, 2, 2, 3, 3] and starts == [0, 1, 4, 10]
    for bad in ([0], [2, -1], [16, 16]):
        with pytest.raises(ValueError):
            tree_of_widths(bad)


def _walk(tree, tokens, choices, most, alive):
    sees, _ = _masks_plain(tree)
    parent = [max(s - {i}, default=-1) if s else -1 for i, s in enumerate(sees)]
    path = [0]
    while alive and len(path) < most:
        nxt = [i for i in range(len(tree)) if sees[i] and parent[i] == path[-1]
               and tokens[i] == choices[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path


def _random_tree(n, depth, g):
    par, lev = [-1], [0]
    for i in range(1, n):
        opts = [j for j in range(i) if lev[j] < depth and par[j] > -2]
        p = opts[int(torch.randint(0, len(opts), (1,), generator=g))]
        if int(torch.randint(0, 10, (1,), generator=g)) == 0:
            p = -2
        par.append(p)
        lev.append(lev[p] + 1 if p >= 0 else 0)
    return par


@gpu
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("n", [1, 2, 13, 32, 33, 64, 150, TREE_MAX])
def test_accept(n, shared):
    """Few different tokens, so that paths are long and siblings alike."""
    g = torch.Generator().manual_seed(n)
    B = 40
    trees = [_random_tree(n, 12, g) for _ in range(1 if shared else B)]
    tokens = torch.randint(0, 3, (B, n), generator=g)
    choices = torch.randint(0, 3, (B, n), generator=g) + (torch.rand(B, n, generator=g) < .05) * 2 ** 40
    alive = torch.rand(B, generator=g) < 0.8
    masks = tree_masks(torch.tensor(trees), device=DEV).masks
    for most, live in ((None, None), (1, None), (3, alive), (n + 2, alive)):
        r = tree_accept(tokens.to(DEV), choices.to(DEV), masks,
                        alive=None if live is None else live.to(DEV), max_path=most)
        P = n if most is None else most
        assert r.path.shape == (B, P) and r.path.dtype == torch.int32
        for b in range(B):
            want = _walk(trees[0 if shared else b], tokens[b].tolist(), choices[b].tolist(), P,
                         live is None or bool(live[b]))
            assert r.path[b].tolist() == want + [-1] * (P - len(want))
            assert int(r.n_acc[b]) == len(want) - 1
            assert int(r.y[b]) == int(choices[b, want[-1]])


@gpu
def test_accept_takes_views_and_other_integers():
    g = torch.Generator().manual_seed(0)
    par = _random_tree(9, 4, g)
    masks = tree_masks(par, device=DEV).masks
    tokens = torch.randint(0, 2, (6, 9), generator=g).to(DEV)
    choices = torch.randint(0, 2, (6, 9), generator=g).to(DEV)
    want = tree_accept(tokens, choices, masks)
    wide = torch.zeros(6, 20, dtype=torch.long, device=DEV)
    wide[:, 3:12] = tokens
    turned = choices.t().contiguous().t()
    for a, b in ((wide[:, 3:12], turned), (tokens.int(), choices.short())):
        got = tree_accept(a, b, masks)
        assert all(torch.equal(x, y) for x, y in zip(want, got))


def _commit_plain(caches, lengths, path, n_acc, nodes, capacity):
    """caches: lists of [B, H, C, D] tensors on the CPU, changed in place."""
    out = lengths.clone()
    for b in range(len(lengths)):
        base, n = int(lengths[b]) - nodes, int(n_acc[b]) + 1
        p = path[b].tolist()
        if base < 0 or int(lengths[b]) > capacity or not 1 <= n <= min(nodes, len(p)):
            continue
        if any(not j <= p[j] < nodes or (j and p[j] <= p[j - 1]) for j in range(n)):
            continue
        for c in caches:
            c[b, :, base:base + n] = c[b, :, [base + x for x in p[:n]]].clone()
        out[b] = base + n
    return out


@gpu
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("dtype,heads,d", [(torch.bfloat16, 8, 128), (torch.float16, 2, 64),
                                           (torch.float32, 3, 20), (torch.bfloat16, 1, 7),
                                           (torch.float32, 2, 1), (torch.bfloat16, 5, 6)])
@pytest.mark.parametrize("nodes", [1, 2, 13, 64, TREE_MAX])
def test_commit(nodes, dtype, heads, d, paged):
    g = torch.Generator().manual_seed(nodes)
    B, layers = 9, 3
    base = torch.randint(0, 300, (B,), generator=g)
    base[0], base[1], base[2] = 0, 127, 128
    width = -(-(int(base.max()) + nodes) // PAGE)
    cap = width * PAGE if paged else int(base.max()) + nodes + 1
    keys = [torch.randn(B, heads, cap, d, generator=g).to(dtype) for _ in range(layers)]
    vals = [torch.randn(B, heads, cap, d, generator=g).to(dtype) for _ in range(layers)]
    n_acc = torch.tensor([min(nodes - 1, (5 * b) % (nodes + 3)) for b in range(B)])
    path = torch.full((B, nodes), -1)
    for b in range(B):
        n = int(n_acc[b])
        rest = torch.randperm(nodes - 1, generator=g)[:n].sort()[0] + 1
        path[b, :n + 1] = torch.cat([torch.zeros(1, dtype=torch.long), rest])
    lengths = base + nodes
    place = torch.randperm(B * width + 2, generator=g)[:B * width].view(B, width)

    def send(c):
        if not paged:
            return c.to(DEV)
        pool = torch.zeros(B * width + 2, heads, PAGE, d, dtype=dtype)
        pool[place.view(-1)] = c.view(B, heads, width, PAGE, d).transpose(1, 2).reshape(-1, heads, PAGE, d)
        return pool.to(DEV)

    def back(p):
        if not paged:
            return p.cpu()
        return p.cpu()[place.view(-1)].view(B, width, heads, PAGE, d).transpose(1, 2).reshape(
            B, heads, cap, d)
    gk, gv = [send(k) for k in keys], [send(v) for v in vals]
    glen = lengths.to(DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    table = place.to(torch.int32).to(DEV) if paged else None
    commit_tree(gk, gv, glen, path.to(torch.int32).to(DEV), n_acc.to(DEV), nodes, block_table=table,
                err=err)
    want = _commit_plain(keys + vals, lengths, path, n_acc, nodes, cap)
    assert int(err) == 0
    assert torch.equal(glen.cpu(), want) and torch.equal(want, base + 1 + n_acc)
    for a, b in zip(gk + gv, keys + vals):
        assert torch.equal(back(a).view(torch.uint8), b.contiguous().view(torch.uint8))


@gpu
@pytest.mark.parametrize("paged", [False, True])
def test_commit_leaves_wrong_rows_alone(paged):
    """Rows out of range, paths that do not rise, missing pages: flagged, the others committed."""
    B, nodes, cap = 8, 6, 2 * PAGE
    g = torch.Generator().manual_seed(1)
    k = [torch.randn(B, 2, cap, 8, generator=g)]
    v = [torch.randn(B, 2, cap, 8, generator=g)]
    lengths = torch.tensor([20, 5, cap + 1, 30, 40, 50, 60, 70])
    path = torch.tensor([[0, 2, 5]] * B)
    path[3] = torch.tensor([0, 2, 2])
    path[4] = torch.tensor([0, 3, 6])
    path[5] = torch.tensor([1, 0, 3])
    n_acc = torch.tensor([2, 2, 2, 2, 2, 2, 3, 1])        # row 6: more than the path holds
    place = torch.arange(2 * B).view(B, 2)
    def send(c):
        return (c.view(B, 2, 2, PAGE, 8).transpose(1, 2).reshape(-1, 2, PAGE, 8) if paged else c).to(DEV)
    def back(p):
        return p.cpu().view(B, 2, 2, PAGE, 8).transpose(1, 2).reshape(B, 2, cap, 8) if paged else p.cpu()
    gk, gv = [send(k[0])], [send(v[0])]
    glen, err = lengths.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    commit_tree(gk, gv, glen, path.to(torch.int32).to(DEV), n_acc.to(DEV), nodes, err=err,
                block_table=place.to(torch.int32).to(DEV) if paged else None)
    want = _commit_plain(k + v, lengths, path, n_acc, nodes, cap)
    assert torch.equal(glen.cpu(), want) and int(err) == 1 + 32
    assert want.tolist() == [17, 5, cap + 1, 30, 40, 50, 60, 66]
    for a, b in zip(gk + gv, k + v):
        assert torch.equal(back(a), b)
    if paged:
        table = place.to(torch.int32)
        table[0, 0], table[7, 0] = -1, 10 ** 6
        err.zero_()
        glen.copy_(lengths)
        before = gk[0].clone()
        commit_tree(gk, gv, glen, path.to(torch.int32).to(DEV), n_acc.to(DEV), nodes, err=err,
                    block_table=table.to(DEV))
        assert int(err) == 1 + 2 + 32
        assert torch.equal(back(gk[0])[0], back(before)[0]) and torch.equal(back(gk[0])[7], back(before)[7])


@gpu
def test_commit_of_more_buffers_than_one_launch_takes():
    g = torch.Generator().manual_seed(2)
    k = [torch.randn(1, 1, 9, 4, generator=g) for _ in range(150)]
    v = [torch.randn(1, 1, 9, 4, generator=g) for _ in range(150)]
    gk, gv = [x.to(DEV) for x in k], [x.to(DEV) for x in v]
    path, n = torch.tensor([[0, 2, 4]]), torch.tensor([2])
    lengths = torch.tensor([8])
    glen = lengths.to(DEV)
    commit_tree(gk, gv, glen, path.to(torch.int32).to(DEV), n.to(DEV), 6)
    want = _commit_plain(k + v, lengths, path, n, 6, 9)
    assert torch.equal(glen.cpu(), want)
    for a, b in zip(gk + gv, k + v):
        assert torch.equal(a.cpu(), b)


@gpu
def test_caches_commit_and_flag():
    """RaggedCache.commit_tree, contiguous and paged, and positions of a tree's nodes."""
    g = torch.Generator().manual_seed(3)
    parents, starts = tree_of_widths([2, 2])
    masks, depths = tree_masks(parents, device=DEV)
    for make in (lambda: RaggedCache(2, 3, 300, DEV, attn_impl="specdec_b200"),
                 lambda: PagedRaggedCache(2, 3, 300, DEV),
                 lambda: PagedRaggedCache(2, 3, 300, DEV, device_pages=True)):
        c = make()
        n = len(parents)
        seqs = [[torch.randn(3, 2, 126 + n, 16, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
                for _ in range(2)]
        for part in (slice(0, 126), slice(126, 126 + n)):
            if isinstance(c, PagedRaggedCache):
                c.reserve(part.stop - part.start)
            if part.start:
                c.set_tree(masks, depths)
                assert c.positions(n).tolist() == [[126 + d for d in depths.tolist()]] * 3
            for layer, (k, v) in zip(c.layers, seqs):
                layer.update(k[:, :, part], v[:, :, part])
            c.advance(part.stop - part.start)
        path = torch.tensor([[0, 1, 4], [0, 2, -1], [0, 2, 6]], dtype=torch.int32, device=DEV)
        c.commit_tree(path, torch.tensor([2, 1, 2], device=DEV), n)
        c.check_errors()
        assert c.lengths.tolist() == [129, 128, 129] and c.tree is None
        table = getattr(c, "block_table", None)
        for layer, (k, v) in zip(c.layers, seqs):
            for buf, full in ((layer.keys, k), (layer.values, v)):
                for b, p in enumerate(path.tolist()):
                    p = [x for x in p if x >= 0]
                    for j, x in enumerate(p):
                        slot = 126 + j
                        got = buf[b, :, slot] if table is None else \
                            buf[int(table[b, slot // PAGE]), :, slot % PAGE]
                        assert torch.equal(got, full[b, :, 126 + x])
        c.commit_tree(path.flip(1).contiguous(), torch.tensor([2, 2, 2], device=DEV), 7)
        with pytest.raises(RuntimeError, match="rising"):
            c.check_errors()
        assert c.lengths.tolist() == [129, 128, 129]


@gpu
def test_accept_and_commit_replay():
    """Captured once, replayed on other trees and tokens in the same buffers."""
    g = torch.Generator().manual_seed(4)
    B, n, cap = 4, 12, 60
    def fresh():
        trees = [_random_tree(n, 5, g) for _ in range(B)]
        return (trees, torch.randint(0, 2, (B, n), generator=g), torch.randint(0, 2, (B, n), generator=g),
                torch.randint(0, 40, (B,), generator=g) + n, torch.randn(B, 2, cap, 8, generator=g))
    def parents(trees):
        return torch.tensor(trees, dtype=torch.int32)
    t0 = fresh()
    bufs = [parents(t0[0]).to(DEV)] + [x.to(DEV) for x in t0[1:]] + [t0[4].to(DEV)]

    def body():
        m = tree_masks(bufs[0]).masks
        r = tree_accept(bufs[1], bufs[2], m, max_path=6)
        commit_tree([bufs[4]], [bufs[5]], bufs[3], r.path, r.n_acc, n)
        return r
    body()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        r = body()
    for _ in range(3):
        trees, tok, cho, lens, k = fresh()
        for b, x in zip(bufs, (parents(trees), tok, cho, lens, k, k)):
            b.copy_(x)
        gr.replay()
        paths = [_walk(t, a, c, 6, True) for t, a, c in zip(trees, tok.tolist(), cho.tolist())]
        assert r.path.tolist() == [p + [-1] * (6 - len(p)) for p in paths]
        plain = torch.tensor([p + [-1] * (6 - len(p)) for p in paths])
        want = _commit_plain([k], lens, plain, torch.tensor([len(p) - 1 for p in paths]), n, cap)
        assert torch.equal(bufs[3].cpu(), want) and torch.equal(bufs[4].cpu(), k)
        assert torch.equal(bufs[5].cpu(), k)


@gpu
def test_refusals():
    masks = tree_masks([-1, 0, 0], device=DEV).masks
    tok = torch.zeros(2, 3, dtype=torch.long, device=DEV)
    for args, kw in (((tok, tok[:, :2], masks), {}), ((tok.float(), tok, masks), {}),
                     ((tok, tok, masks.long()), {}), ((tok, tok, masks[:2]), {}),
                     ((tok[0], tok[0], masks), {}), ((tok, tok.cpu(), masks), {}),
                     ((tok, tok, masks), dict(max_path=0)),
                     ((tok, tok, masks), dict(alive=torch.ones(3, dtype=torch.bool, device=DEV)))):
        with pytest.raises(L.SpecdecError):
            tree_accept(*args, **kw)
    for bad in (torch.zeros(2, 3), torch.zeros(1, 1, 3, dtype=torch.long),
                torch.zeros(TREE_MAX + 1, dtype=torch.long), torch.zeros(2, 0, dtype=torch.long)):
        with pytest.raises(L.SpecdecError):
            tree_masks(bad, device=DEV)
    k = torch.zeros(2, 1, 20, 8, device=DEV)
    lens, n = torch.tensor([5, 5], device=DEV), torch.zeros(2, dtype=torch.long, device=DEV)
    path = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    good = ([k], [k.clone()], lens, path, n, 3)
    for i, x in ((0, []), (0, [k, k]), (1, [k.half()]), (1, [k[:, :, :10]]), (2, lens.int()), (2, lens[:1]),
                 (3, path.long()), (3, path[:1]), (3, path[:, :0]), (4, n[:1]), (4, n.float()), (5, 0),
                 (5, TREE_MAX + 1), (0, [k.double()]), (0, [k.cpu()])):
        args = list(good)
        args[i] = x
        with pytest.raises(L.SpecdecError):
            commit_tree(*args)
    with pytest.raises(L.SpecdecError):
        commit_tree(*good, block_table=torch.zeros(2, 1, dtype=torch.int32, device=DEV))
    with pytest.raises(L.SpecdecError):
        RaggedCache(1, 1, 10, DEV).set_tree(masks, masks)


@gpu
def test_a_buffer_that_is_there_twice_is_refused():
    """Two threads would move the same bytes."""
    k, v = torch.zeros(2, 1, 20, 8, device=DEV), torch.zeros(2, 1, 20, 8, device=DEV)
    lens, n = torch.tensor([5, 5], device=DEV), torch.zeros(2, dtype=torch.long, device=DEV)
    path = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    for keys, values in (([k], [k]), ([k, k], [v, torch.zeros_like(v)])):
        with pytest.raises(L.SpecdecError):
            commit_tree(keys, values, lens, path, n, 3)
    assert lens.tolist() == [5, 5]


def test_refused_on_the_host():
    lib = L.lib()
    assert lib.sd_tree_masks(None, 0, 1, 4, 16, 16, None) == -22
    assert lib.sd_tree_masks(16, 4, 1, TREE_MAX + 1, 16, 16, None) == -95
    assert lib.sd_tree_masks(16, 4, -1, 4, 16, 16, None) == -22
    assert lib.sd_tree_masks(None, 0, 0, 4, None, None, None) == 0
    for kw in (dict(B=-1), dict(N=0), dict(P=0), dict(tok=None), dict(y=None)):
        a = {**dict(tok=16, B=1, N=4, P=4, y=16), **kw}
        assert lib.sd_tree_accept(a["tok"], 4, 16, 4, 16, 0, None, a["B"], a["N"], a["P"], 16, 16,
                                  a["y"], None) == -22
    assert lib.sd_tree_accept(16, 4, 16, 4, 16, 0, None, 1, TREE_MAX + 1, 4, 16, 16, 16, None) == -95
    import ctypes
    bufs = (ctypes.c_void_p * 2)(16, 32)
    ok = dict(bufs=bufs, n=2, bt=None, bts=0, npg=0, lens=16, path=16, plen=4, nacc=16, N=4, B=1, H=1,
              C=64, D=8, e=2)

    def call(**kw):
        a = {**ok, **kw}
        return lib.sd_kv_commit_tree(a["bufs"], a["n"], a["bt"], a["bts"], a["npg"], a["lens"],
                                     a["path"], 4, a["plen"], a["nacc"], a["N"], a["B"], a["H"],
                                     a["C"], a["D"], a["e"], None, None)
    for kw in (dict(bufs=None), dict(n=-1), dict(lens=None), dict(path=None), dict(plen=0),
               dict(nacc=None), dict(N=0), dict(B=-1), dict(H=0), dict(C=0), dict(D=0), dict(e=8),
               dict(bt=16, bts=0, npg=1), dict(bufs=(ctypes.c_void_p * 2)(16, None)),
               dict(bufs=(ctypes.c_void_p * 2)(16, 33))):
        assert call(**kw) == -22, kw
    assert call(N=TREE_MAX + 1) == -95 and call(bt=16, bts=2 ** 25, npg=1) == -95
    assert call(B=0) == 0
    for f in (lambda: tree_masks([-1, 0]),
              lambda: tree_accept(torch.zeros(1, 1).long(), torch.zeros(1, 1).long(),
                                  torch.zeros(1, 1, dtype=torch.int32)),
              lambda: commit_tree([torch.zeros(1, 1, 1, 1)], [torch.zeros(1, 1, 1, 1)],
                                  torch.zeros(1).long(), torch.zeros(1, 1, dtype=torch.int32),
                                  torch.zeros(1).long(), 1)):
        with pytest.raises(L.SpecdecError):
            f()


@gpu
@pytest.mark.parametrize("make", ["contiguous", "paged", "device pages"])
@pytest.mark.parametrize("end", ["reset", "rollback", "rollback on the device", "set_lengths", "commit"])
def test_a_tree_ends_with_its_round(make, end):
    """A tree's forward that is not committed: what follows is a chain again, its positions by
    place and every query behind the keys before it."""
    g = torch.Generator().manual_seed(7)
    masks, depths = tree_masks([-1, 0, 0, 1], device=DEV)
    c = RaggedCache(1, 2, 256, DEV, attn_impl="specdec_b200") if make == "contiguous" else \
        PagedRaggedCache(1, 2, 256, DEV, device_pages=make == "device pages")
    x = [torch.randn(2, 2, 20, 16, generator=g).to(DEV) for _ in range(3)]

    def forward(part):
        n = part.stop - part.start
        if make != "contiguous":
            c.reserve(n)
        assert c.attn_mask(n, torch.float32) is None
        pos = c.positions(n)
        keys, values = c.layers[0].update(x[1][:, :, part], x[2][:, :, part])
        out, _ = A.hf_attention(None, x[0][:, :, part], keys, values, None, scaling=0.25)
        c.advance(n)
        return pos, out
    forward(slice(0, 6))
    c.set_tree(masks, depths)
    forward(slice(6, 10))
    base = 6
    if end == "reset":
        c.reset()
        base = 0
    elif end == "rollback":
        c.rollback(4)
    elif end == "rollback on the device":
        c.rollback(torch.tensor([4, 4], device=DEV))
    elif end == "commit":
        c.commit(torch.tensor([0, 0], device=DEV), 4)
    else:
        c.set_lengths([6, 6])
    assert c.tree is None
    pos, out = forward(slice(12, 15))
    assert pos.tolist() == [[base, base + 1, base + 2]] * 2
    k, v = (torch.cat([t[:, :, :base], t[:, :, 12:15]], 2).double() for t in x[1:])
    s = torch.einsum("bhqd,bhkd->bhqk", x[0][:, :, 12:15].double(), k) * 0.25
    s.masked_fill_(torch.ones(3, base + 3, dtype=torch.bool, device=DEV).triu(base + 1), -torch.inf)
    want = torch.einsum("bhqk,bhkd->bqhd", s.softmax(-1), v)
    # fp32: at most 9 keys of |v| < 5, scores of 16 terms; 2^-18 for the powers of two
    assert float((out.double() - want).abs().max()) <= 5 * 2.0 ** -16


@gpu
@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_masks_of_parents_of_every_integer_type(dtype):
    """(In an unsigned type no node is a root: 255 and 254 are no earlier nodes, so all are absent.)"""
    trees = [[-1, 0, 0, 1, -2, 4, 2, 100, 3], [-1, -1, -2, 1, 0, 3, 5, 5, 8]]
    parents = torch.tensor(trees).to(dtype)
    want = [_masks_plain(t) for t in parents.tolist()]
    got = tree_masks(parents, device=DEV)
    assert _sets(got.masks) == [w[0] for w in want] and got.depths.tolist() == [w[1] for w in want]


@gpu
@pytest.mark.parametrize("device_pages", [False, True])
def test_a_released_row_leaves_the_others_their_tree(device_pages):
    masks, depths = tree_masks([-1, 0, 0, 1], device=DEV)
    c = PagedRaggedCache(1, 2, 256, DEV, device_pages=device_pages)
    c.reserve(6)
    c.advance(6)
    c.set_tree(masks, depths)
    c.release([1])
    assert c.tree is not None
    assert c.positions(4).tolist() == [[6, 7, 7, 8], [0, 1, 1, 2]]
