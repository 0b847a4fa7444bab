"""tree_attention against its definition in 64 bits.

Tolerances, from the arithmetic.  With weights p_s = exp(score_s - m), l = sum p,
o = sum p v / l, and A = sum p |v| / l (per output element):
  scores: a float32 dot product of D terms is off by at most (D + 4) u times scale
    sum |q k| (u = 2^-24; products of bf16 values are exact), which moves a weight by
    that much relative: at most e_s = (D + 4) u max_s(scale sum |q k|) for every key;
    beyond 2^20 (base 2) the scaled score is rounded by itself, u |score| more;
    a power of two is good to 2^-18 (the approximation to 2^-21, the polynomial of
    degree 4 to 2.7e-6), and its argument s - m to 2 u (|s| + |m|): with |s| <= max
    |score| that is 6 u max|score| in all;
  sums: at most 3 + (keys / 32 + 128) additions deep in any order the kernels use,
    (keys / 32 + 200) u relative, for l and for o;
  bf16: each weight is rounded once, 2^-8 relative of p, and the output 2^-8 of o.
So |error| <= A (2 (e_s + 6 u max|s| + 2^-18) + 2 (keys / 32 + 200) u [+ 2^-8]) [+ 2^-8 |o|].
"""
import math

import pytest
import torch

from specdec import _lib as L
from specdec import attention as A
from specdec.tree import TREE_MAX, tree_masks

gpu = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
PAGE = 128


def _parents(n, g, depth=8, missing=0):
    """A random tree in breadth-first order; its last `missing` nodes are not there."""
    par, lev = [-1], [0]
    for i in range(1, n):
        opts = [j for j in range(i) if lev[j] < depth and par[j] > -2]
        p = opts[int(torch.randint(0, len(opts), (1,), generator=g))] if i < n - missing else -2
        par.append(p)
        lev.append(lev[p] + 1 if p >= 0 else 0)
    return par


def _bits(parents):
    """Truth values [T, N, N] of parents [T][N]: what each node sees of its tree."""
    out = torch.zeros(len(parents), len(parents[0]), len(parents[0]), dtype=torch.bool)
    for t, tree in enumerate(parents):
        for i, p in enumerate(tree):
            if p >= -1 and (p < 0 or out[t, p, p]):
                if p >= 0:
                    out[t, i] = out[t, p]
                out[t, i, i] = True
    return out


def _case(bases, parents, hq, hkv, d, dtype, first=0, paged=False, qlen=None, seed=0, slack=5,
          scale_q=1.0):
    """Caches with NaN wherever nobody looks, and the call's arguments."""
    g = torch.Generator().manual_seed(seed)
    B, N = len(bases), len(parents[0])
    qlen = N - first if qlen is None else qlen
    bits = _bits(parents).expand(B, N, N)
    cap = max(bases) + N + slack
    width = -(-cap // PAGE)
    cap = width * PAGE if paged else cap
    k = torch.full((B, hkv, cap, d), math.nan)
    v = torch.full((B, hkv, cap, d), math.nan)
    for b, n in enumerate(bases):
        k[b, :, :n + N] = torch.randn(hkv, n + N, d, generator=g) * 1.5
        v[b, :, :n + N] = torch.randn(hkv, n + N, d, generator=g) + 0.5
        nobody = ~bits[b].any(0)                       # absent nodes: nobody sees their slots
        k[b, :, n:n + N][:, nobody] = math.nan
        v[b, :, n:n + N][:, nobody] = math.inf
    k, v = k.to(dtype).to(DEV), v.to(dtype).to(DEV)
    q = (torch.randn(B, qlen, hq, d, generator=g) * scale_q).to(dtype).to(DEV).transpose(1, 2)
    table = None
    if paged:
        place = torch.randperm(B * width + 3, generator=g)[:B * width].view(B, width)
        pool_k = torch.full((B * width + 3, hkv, PAGE, d), math.nan, dtype=dtype, device=DEV)
        pool_v = pool_k.clone()
        at = place.to(DEV).view(-1)
        pool_k[at] = k.view(B, hkv, width, PAGE, d).transpose(1, 2).reshape(-1, hkv, PAGE, d)
        pool_v[at] = v.view(B, hkv, width, PAGE, d).transpose(1, 2).reshape(-1, hkv, PAGE, d)
        used = torch.tensor([-(-(n + N) // PAGE) for n in bases]).view(-1, 1)
        table = torch.where(torch.arange(width) < used, place, -1).to(torch.int32).to(DEV)
        args = (q, pool_k, pool_v)
    else:
        args = (q, k, v)
    lengths = torch.tensor([n + first for n in bases], device=DEV)
    masks = tree_masks(torch.tensor(parents), device=DEV).masks
    return args + (lengths, masks), dict(first=first, block_table=table), (k, v, bits, bases)


def _check(call, kw, ref, scale=None, out=None):
    q, _, _, lengths, masks = call
    k, v, bits, bases = ref
    got = A.tree_attention(*call, scale=scale, out=out, **kw)
    _compare(got, q, ref, kw["first"], scale)
    return got


def _compare(got, q, ref, first, scale=None):
    k, v, bits, bases = ref
    B, hq, qlen, d = q.shape
    hkv, N = k.shape[1], bits.shape[1]
    sc = d ** -0.5 if scale is None else scale
    assert got.shape == (B, qlen, hq, d) and got.dtype == q.dtype
    for b, n in enumerate(bases):
        kb, vb = k[b, :, :n + N].double(), v[b, :, :n + N].double()
        sees = torch.ones(qlen, n + N, dtype=torch.bool)
        sees[:, n:] = bits[b, first:first + qlen]
        there = bits[b, first:first + qlen].any(-1)
        sees[~there] = False
        sees, there = sees.to(DEV), there.to(DEV)
        seen = sees.any(0)
        kb, vb = kb[:, seen], vb[:, seen]
        sees = sees[:, seen]
        qb = q[b].double().view(hkv, hq // hkv, qlen, d)
        s = torch.einsum("hgjd,hsd->hgjs", qb, kb) * sc
        sab = torch.einsum("hgjd,hsd->hgjs", qb.abs(), kb.abs()) * sc
        o = torch.zeros(qlen, hkv, hq // hkv, d, dtype=torch.float64, device=DEV)
        av = torch.zeros_like(o)
        big = e_s = 0.0
        if sees.shape[1]:
            p = torch.softmax(s.masked_fill(~sees, -math.inf), -1)
            p = torch.where(there.view(-1, 1), p, 0.0)
            o = torch.einsum("hgjs,hsd->jhgd", p, vb)
            av = torch.einsum("hgjs,hsd->jhgd", p, vb.abs())
            big, e_s = float(s.abs().max()), float(sab.max()) * (d + 4) * U
        rel = 2 * (e_s + 6 * U * big + 2.0 ** -18) + 2 * ((n + N) / 32 + 200) * U
        tol = av * (rel + (2.0 ** -8 if q.dtype == torch.bfloat16 else 0))
        tol = tol + o.abs() * (2.0 ** -8 if q.dtype == torch.bfloat16 else U) + 1e-37
        diff = (got[b].double().view(qlen, hkv, hq // hkv, d) - o).abs()
        assert bool(torch.isfinite(diff).all()), f"row {b}: not finite"
        assert bool((diff <= tol).all()), f"row {b}: {float((diff / tol).max())} of the tolerance"
        assert not bool(got[b][~there].any()), "an absent node is 0"


BASES = [0, 1, 31, 64, 100, 127, 128, 129, 255, 300, 511, 640]


@gpu
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("dtype,hq,hkv,d", [
    (torch.bfloat16, 8, 2, 128), (torch.bfloat16, 4, 4, 128), (torch.bfloat16, 16, 2, 128),
    (torch.float32, 8, 2, 64), (torch.float32, 4, 4, 128), (torch.bfloat16, 6, 2, 64),
    (torch.float32, 3, 1, 20), (torch.bfloat16, 2, 1, 33)])
@pytest.mark.parametrize("n", [1, 7, 33])
def test_every_border_of_tiles_and_words(dtype, hq, hkv, d, n, paged):
    g = torch.Generator().manual_seed(n)
    parents = [_parents(n, g, missing=min(n - 1, b % 3)) for b in range(len(BASES))]
    _check(*_case(BASES, parents, hq, hkv, d, dtype, paged=paged, seed=n))


@gpu
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8), (16, 2)])
@pytest.mark.parametrize("n", [2, 16, 31, 32, 48, 64, 65, 97, 128, 200, TREE_MAX])
def test_numbers_of_nodes(hq, hkv, n):
    g = torch.Generator().manual_seed(n)
    bases = [0, 90, 200, 1037]
    _check(*_case(bases, [_parents(n, g)], hq, hkv, 128, torch.bfloat16, paged=n % 2 == 0, seed=n))


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("first,qlen", [(0, 1), (1, 4), (5, 8), (12, 1), (3, 10)])
def test_level_by_level(dtype, d, first, qlen):
    """Nodes first .. first + qlen of a tree whose earlier nodes are in the cache."""
    g = torch.Generator().manual_seed(first)
    bases = [0, 126, 250, 400]
    call, kw, ref = _case(bases, [_parents(13, g)], 16, 8, d, dtype, first=first, qlen=qlen,
                          paged=True)
    _check(call, kw, ref)


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 32)])
def test_rows_without_a_tree_and_empty_rows(dtype, d):
    """Absent nodes, whole rows of them, over empty and filled caches."""
    parents = [[-1, 0, 0, 1], [-2, -2, -2, -2], [-1, -2, 1, 0], [-2, -1, 1, -1], [-2] * 4]
    call, kw, ref = _case([130, 260, 0, 7, 0], parents, 4, 2, d, dtype, paged=True)
    got = _check(call, kw, ref)
    assert not bool(got[1].any()) and not bool(got[4].any())


@gpu
@pytest.mark.parametrize("bases", [[5000] * 3, [12, 9000, 1], [0, 0, 20000]])
def test_long_rows_are_split_and_joined(bases):
    g = torch.Generator().manual_seed(3)
    for n, hq, hkv in ((5, 8, 2), (40, 16, 4), (64, 32, 8)):
        _check(*_case(bases, [_parents(n, g)], hq, hkv, 128, torch.bfloat16, paged=True, seed=n))


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_many_rows(dtype, d):
    g = torch.Generator().manual_seed(4)
    bases = [int(x) for x in torch.randint(0, 900, (700,), generator=g)]
    _check(*_case(bases, [_parents(9, g)], 4, 2, d, dtype, paged=True))


@gpu
@pytest.mark.parametrize("scale_q", [1e3, 1e7, 1e12])
def test_scores_of_every_size(scale_q):
    """One key takes all the weight; far scores must not become NaN or lose it."""
    g = torch.Generator().manual_seed(5)
    call, kw, ref = _case([200, 700], [_parents(12, g)], 8, 2, 128, torch.bfloat16)
    q, k = call[0], ref[0]
    # scores that float32 separates: keys on one axis, spaced by a quarter of their size
    k.zero_()
    call[1].copy_(k)
    axis = torch.tensor([1.0, -1.0, 0.5, 2.0, -0.25, 0.125], dtype=torch.bfloat16, device=DEV)
    call[1][..., 0] = axis[torch.arange(k.shape[2], device=DEV) % 6]
    call[1][:, :, 37, 0] = 4.0
    ref[0].copy_(call[1])
    qq = torch.zeros_like(q)
    qq[..., 0] = scale_q
    got = A.tree_attention(qq, *call[1:], **kw)
    want = ref[1][:, :, 37].repeat_interleave(4, 1).unsqueeze(1).expand_as(got)
    assert torch.equal(got, want)


@gpu
def test_infinite_and_nan_keys_that_are_seen():
    """As the formula: a NaN score makes its rows NaN, a key of -inf scores weighs nothing."""
    call, kw, ref = _case([150], [[-1, 0, 0]], 2, 1, 128, torch.bfloat16)
    call[0].fill_(1.0)
    call[1][0, 0, 10] = -math.inf
    got = A.tree_attention(*call, **kw)
    ref[0][0, 0, 10] = 0
    ref[1][0, 0, 10] = 0
    rest = A.tree_attention(call[0], call[1].clone().index_fill_(2, torch.tensor([10], device=DEV),
                                                                -1e30), *call[2:], **kw)
    assert bool(torch.isfinite(got).all()) and torch.allclose(got, rest, rtol=2 ** -7, atol=1e-6)
    call[1][0, 0, 151] = math.nan                       # node 1's own key
    got = A.tree_attention(*call, **kw)
    assert bool(got[0, 1].isnan().all())
    assert bool(torch.isfinite(got[0, 0]).all()) and bool(torch.isfinite(got[0, 2]).all())


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_strides_scale_and_given_output(dtype, d):
    g = torch.Generator().manual_seed(6)
    call, kw, ref = _case([70, 300], [_parents(6, g)], 8, 2, d, dtype)
    q = call[0]
    wide = torch.zeros(2, 8, 6, d + 16, dtype=dtype, device=DEV)
    wide[..., 8:d + 8] = q
    out = torch.full((2, 8, 9, d), 7.0, dtype=dtype, device=DEV).transpose(1, 2)   # [2, 9, 8, d]
    view = out[:, 2:8]
    got = _check((wide[..., 8:d + 8],) + call[1:], kw, ref, scale=0.3, out=view)
    assert got.data_ptr() == view.data_ptr()
    assert bool((out[:, :2] == 7).all()) and bool((out[:, 8:] == 7).all())
    odd = torch.zeros(2 * 8 * 6 * d + 3, dtype=dtype, device=DEV)[3:].view(2, 8, 6, d)
    odd.copy_(q)                                        # 2 bytes past an aligned address
    _check((odd,) + call[1:], kw, ref)
    with pytest.raises(L.SpecdecError):
        A.tree_attention(q.transpose(0, 1), *call[1:], **kw)


@gpu
@pytest.mark.parametrize("hq,hkv", [(32, 8), (4, 4), (16, 2)])
@pytest.mark.parametrize("n,first", [(1, 0), (9, 4), (33, 0), (64, 0), (65, 2), (TREE_MAX, 0)])
@pytest.mark.parametrize("bases", [[0, 90, 129, 1037], [3000, 9000]])
def test_heads_of_64(hq, hkv, n, first, bases):
    g = torch.Generator().manual_seed(n)
    parents = [_parents(n, g, missing=min(n - 1, b % 3)) for b in range(len(bases))]
    _check(*_case(bases, parents, hq, hkv, 64, torch.bfloat16, first=first, paged=n % 2 == 0, seed=n))


@gpu
@pytest.mark.parametrize("scale_q", [1e3, 1e7, 1e12])
def test_scores_of_every_size_with_heads_of_64(scale_q):
    g = torch.Generator().manual_seed(19)
    for n, hq in ((12, 8), (70, 16)):
        _check(*_case([40, 700], [_parents(n, g)], hq, 2, 64, torch.bfloat16, scale_q=scale_q))


@gpu
@pytest.mark.parametrize("bases", [[70, 300], [2000, 5000]])
def test_outputs_that_no_wide_store_reaches(bases):
    """Rows of an output that start 2 bytes past aligned addresses: whole and joined items."""
    g = torch.Generator().manual_seed(16)
    call, kw, ref = _case(bases, [_parents(7, g)], 8, 2, 128, torch.bfloat16)
    room = torch.full((2, 7, 8, 131), 7.0, dtype=torch.bfloat16, device=DEV)
    _check(call, kw, ref, out=room[..., 1:129])
    assert bool((room[..., 0] == 7).all()) and bool((room[..., 129:] == 7).all())


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_broadcast_queries_and_masks(dtype, d):
    """One query for all heads, nodes or rows, one row of masks for all rows."""
    g = torch.Generator().manual_seed(17)
    call, kw, ref = _case([9, 150], [_parents(5, g)], 8, 2, d, dtype)
    q, k, v, lengths, masks = call
    for x in (q[:1].expand(2, -1, -1, -1), q[:, :1].expand(-1, 8, -1, -1), q[:, :, :1].expand(-1, -1, 5, -1)):
        _check((x, k, v, lengths, masks.expand(2, -1, -1)), kw, ref)


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_any_stride_of_dimensions_of_one(d):
    g = torch.Generator().manual_seed(20)
    call, kw, ref = _case([33], [_parents(6, g)], 1, 1, d, torch.bfloat16)
    q = call[0]
    assert q.shape == (1, 1, 6, d)
    rows = q[0, 0].contiguous()
    _check((rows.as_strided((1, 1, 6, d), (3, 5, d, 1)),) + call[1:], kw, ref)
    call, kw, ref = _case([33, 200], [[-1]], 4, 2, d, torch.bfloat16)
    q = call[0].contiguous()
    _check((q.as_strided((2, 4, 1, d), (4 * d, d, 7, 1)),) + call[1:], kw, ref)


@gpu
@pytest.mark.parametrize("hq,hkv", [(5, 1), (71, 1), (128, 1), (129, 1), (40, 8), (192, 3)])
@pytest.mark.parametrize("n", [1, 3, 20])
def test_head_groups_of_every_size(hq, hkv, n):
    g = torch.Generator().manual_seed(n)
    _check(*_case([0, 60, 900], [_parents(n, g)], hq, hkv, 128, torch.bfloat16, paged=n == 3, seed=n))


@gpu
def test_caches_smaller_than_a_tile():
    g = torch.Generator().manual_seed(18)
    for n, base in ((1, 0), (2, 3), (9, 1)):
        _check(*_case([base], [_parents(n, g)], 2, 1, 128, torch.bfloat16, slack=0))


@gpu
def test_masks_that_are_no_tree_and_bits_past_the_nodes():
    """Any bits are followed; the ones from N on are ignored."""
    call, kw, ref = _case([140], [[-1, 0, 1, 0, 3]], 4, 2, 128, torch.bfloat16)
    bits = ref[2].clone()
    bits[0, 4] = torch.tensor([False, True, False, True, True])
    masks = call[4].clone()
    masks[0, 4, 0] = 0b11010
    masks[0, 2, 0] |= -32                                # bits 5 to 31
    got = A.tree_attention(*call[:4], masks, **kw)
    _compare(got, call[0], (ref[0], ref[1], bits, ref[3]), 0)
    dead = call[4].clone()
    dead[0, 1, 0] = -32                                  # nothing but bits from N on: absent
    assert not bool(A.tree_attention(*call[:4], dead, **kw)[0, 1].any())


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_wrong_lengths_and_tables_read_nothing_out_of_bounds(dtype, d):
    """Lengths past the capacity or below the fed nodes, pages outside the pool: any
    values come out, and nothing faults."""
    g = torch.Generator().manual_seed(8)
    call, kw, _ = _case([70, 300, 5], [_parents(6, g)], 8, 2, d, dtype, paged=True)
    lengths = torch.tensor([-5, 10 ** 12, 3 * PAGE], device=DEV)
    A.tree_attention(*call[:3], lengths, call[4], **kw)
    table = kw["block_table"].clone()
    table[1] = torch.tensor([-7, 10 ** 9, 2], dtype=torch.int32, device=DEV)[:table.shape[1]]
    A.tree_attention(*call, first=0, block_table=table)
    call, kw, _ = _case([70, 300, 5], [_parents(6, g)], 8, 2, d, dtype)
    A.tree_attention(*call[:3], lengths, call[4], **kw)
    torch.cuda.synchronize()


@gpu
def test_the_same_result_on_every_run_stream_and_replay():
    g = torch.Generator().manual_seed(9)
    call, kw, ref = _case([900, 20, 3000, 0], [_parents(30, g)], 16, 4, 128, torch.bfloat16,
                          paged=True)
    first = _check(call, kw, ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(A.tree_attention(*call, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    graphs, res = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res.append(A.tree_attention(*call, **kw))
        graphs.append(gr)
    # other lengths and another tree in the same buffers: the graphs follow them
    bases = [10, 2500, 64, 129]
    call2, kw2, ref2 = _case(bases, [_parents(30, g, depth=3)], 16, 4, 128, torch.bfloat16,
                             paged=True, seed=1, slack=505)
    assert call2[1].shape == call[1].shape
    for a, b in zip(call + (kw["block_table"],), call2 + (kw2["block_table"],)):
        a.copy_(b)
    for _ in range(2):
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    for r in res:
        _compare(r, call2[0], ref2, 0)


@gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("bases", [[40, 7], [3000, 9000]])
def test_inputs_that_kernels_before_it_or_another_stream_still_write(bases, captured):
    """The kernel starts beside the end of the one before it, and reads nothing until that and
    whatever its stream waits for are done."""
    g = torch.Generator().manual_seed(21)
    call, kw, ref = _case(bases, [_parents(9, g)], 8, 2, 128, torch.bfloat16)
    q, k, v, lengths, masks = call
    src = [t.clone() for t in (q, k, v, lengths, masks)]
    live = [torch.zeros_like(t) for t in src]
    side = torch.cuda.Stream()
    main = torch.cuda.Stream()

    def body():
        cur = torch.cuda.current_stream()
        side.wait_stream(cur)
        with torch.cuda.stream(side):
            torch.cuda._sleep(400000)
            live[1].copy_(src[1])
            live[4].copy_(src[4])
        live[2].copy_(src[2])
        cur.wait_stream(side)
        first = A.tree_attention(src[0], live[1], live[2], src[3], live[4], **kw)
        torch.cuda._sleep(400000)
        live[0].copy_(src[0])
        live[3].copy_(src[3])
        second = A.tree_attention(live[0], live[1], live[2], live[3], live[4], **kw)
        third = A.tree_attention(second.transpose(1, 2), live[1], live[2], live[3], live[4], **kw)
        for t in live:
            t.zero_()                                  # the calls have read them
        return first, second, third

    main.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(main):
        if captured:
            body()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=main):
                outs = body()
            for _ in range(3):
                for t in live:
                    t.zero_()
                graph.replay()
        else:
            outs = body()
    torch.cuda.synchronize()
    for got in outs[:2]:
        _compare(got, q, ref, kw["first"])
    assert torch.equal(outs[0], outs[1])
    _compare(outs[2], outs[1].transpose(1, 2), ref, kw["first"])


@gpu
def test_chains_match_verify_attention():
    """A chain of drafts is the tree that verify_attention computes."""
    n = 5
    call, kw, ref = _case([40, 700, 128], [list(range(-1, n - 1))], 32, 8, 128, torch.bfloat16)
    q, k, v, lengths, masks = call
    want = A.verify_attention(q, k.nan_to_num(0.0), v.nan_to_num(0.0), lengths).double()
    got = A.tree_attention(*call, **kw).double()
    # both round weights and outputs once: 2^-8 each of A <= max |v| and of the output
    assert bool(((got - want).abs() <= 4 * 2.0 ** -8 * 6.0).all())
    _compare(got.to(torch.bfloat16), q, ref, 0)


@gpu
def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements: the last row's keys lie behind them."""
    B, hkv, d = 3, 8, 128
    cap = 2 ** 31 // (2 * hkv * d) + 64                  # rows 0 and 1 fill 2^31 elements
    k = torch.zeros(B, hkv, cap, d, dtype=torch.bfloat16, device=DEV)
    assert k.numel() > 2 ** 31
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(10)
    n, N = 300, 6
    k[2, :, :n + N] = torch.randn(hkv, n + N, d, generator=g).to(torch.bfloat16)
    v[2, :, :n + N] = torch.randn(hkv, n + N, d, generator=g).to(torch.bfloat16)
    par = [_parents(N, g)]
    q = torch.randn(B, 16, N, d, generator=g).to(torch.bfloat16).to(DEV)
    masks = tree_masks(torch.tensor(par), device=DEV).masks
    got = A.tree_attention(q, k, v, torch.tensor([0, 1, n], device=DEV), masks)
    _compare(got[2:], q[2:], (k[2:, :, :n + N], v[2:, :, :n + N], _bits(par), [n]), 0)


@gpu
def test_refusals():
    call, kw, _ = _case([20, 30], [[-1, 0, 0, 1]], 4, 2, 128, torch.bfloat16)
    q, k, v, lengths, masks = call
    bad = [
        (q.half(), k.half(), v.half(), lengths, masks),
        (q, k.float(), v.float(), lengths, masks),
        (q, k[:, :, :, :64], v[:, :, :, :64], lengths, masks),
        (q, k[:1], v[:1], lengths, masks),
        (q, k, v, lengths[:1], masks),
        (q, k, v, lengths, masks.long()),
        (q, k, v, lengths, masks[:, :2]),                # fewer nodes than queries
        (q, k, v, lengths, torch.zeros(2, 4, 2, dtype=torch.int32, device=DEV)),
        (q, k, v, lengths, torch.zeros(3, 4, 1, dtype=torch.int32, device=DEV)),
        (q, k, v, lengths, torch.zeros(1, TREE_MAX + 1, 9, dtype=torch.int32, device=DEV)),
        (q, k, v, lengths.cpu(), masks),
        (q[:, :3], k, v, lengths, masks),                # heads that do not divide
    ]
    for args in bad:
        with pytest.raises(L.SpecdecError):
            A.tree_attention(*args)
    for more in (dict(first=1), dict(first=-1), dict(scale=0.0), dict(scale=math.nan),
                 dict(out=torch.empty(2, 4, 4, 64, dtype=torch.bfloat16, device=DEV)),
                 dict(block_table=torch.zeros(2, 1, dtype=torch.int32, device=DEV))):
        with pytest.raises(L.SpecdecError):
            A.tree_attention(*call, **more)
    wide = torch.zeros(1, 2, 1, 160, device=DEV)
    with pytest.raises(L.SpecdecError):                  # head sizes past 128
        A.tree_attention(wide, wide, wide, lengths[:1], masks[:, :1])
    assert A.tree_attention(q[:0], k[:0], v[:0], lengths[:0], masks).shape == (0, 4, 4, 128)
    assert A.tree_attention(q[:, :, :0], k, v, lengths, masks).shape == (2, 0, 4, 128)


def test_refused_on_the_host():
    """No GPU is touched: the C entry refuses before any launch."""
    lib = L.lib()
    ok = dict(q=16, k=16, v=16, bt=None, bts=0, npg=0, lens=16, masks=16, mbs=0, N=8, first=0, B=1,
              Hq=4, Hkv=2, D=128, C=256, qlen=8, scale=0.1, out=16, dtype=2, ws=None, nws=0)

    def call(**kw):
        a = {**ok, **kw}
        return lib.sd_tree_attn(a["q"], 8, 8, 8, a["k"], a["v"], a["bt"], a["bts"], a["npg"],
                                a["lens"], a["masks"], a["mbs"], a["N"], a["first"], a["B"],
                                a["Hq"], a["Hkv"], a["D"], a["C"], a["qlen"], a["scale"], a["out"],
                                8, 8, 8, a["dtype"], a["ws"], a["nws"], None)
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(lens=None), dict(masks=None),
               dict(out=None), dict(Hq=3), dict(Hkv=0), dict(D=0), dict(first=1), dict(qlen=9),
               dict(first=-1), dict(scale=0.0), dict(scale=float("nan")), dict(C=0), dict(B=-1),
               dict(bt=16, bts=0, npg=4), dict(bt=16, bts=4, npg=0)):
        assert call(**kw) == -22, kw
    for kw in (dict(dtype=1), dict(N=TREE_MAX + 1), dict(D=160), dict(C=2 ** 31 - 1),
               dict(bt=16, bts=2 ** 25, npg=1)):
        assert call(**kw) == -95, kw
    assert call(B=0) == 0 and call(qlen=0) == 0
    with pytest.raises(L.SpecdecError):
        A.tree_attention(*[torch.zeros(1, 1, 1, 8)] * 3, torch.zeros(1).long(),
                         torch.ones(1, 1, dtype=torch.int32))


def test_outputs_that_overlap_themselves_are_refused_on_the_host():
    """Rows, nodes or heads of the output that share entries (refused before any launch)."""
    lib = L.lib()

    def call(obs, oqs, ohs, B=2, qlen=3, Hq=4, dtype=0):
        return lib.sd_tree_attn(1 << 20, 96, 8, 32, 1 << 21, 1 << 22, None, 0, 0, 1 << 23, 1 << 24, 0, 4, 0,
                                B, Hq, 2, 8, 64, qlen, 0.1, 1 << 25, obs, oqs, ohs, dtype, None, 0, None)
    for strides in ((0, 32, 8), (96, 0, 8), (96, 32, 0), (96, 32, 7), (96, 24, 8), (88, 32, 8), (-88, 32, 8)):
        assert call(*strides) == -22, strides
    assert call(0, 8, 8, B=1, qlen=2, Hq=2) == -22


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_outputs_that_overlap_themselves_are_refused(dtype, d):
    g = torch.Generator().manual_seed(22)
    call, kw, ref = _case([70, 300], [_parents(6, g)], 8, 2, d, dtype)
    for i, shape in enumerate(((1, 6, 8, d), (2, 1, 8, d), (2, 6, 1, d))):
        with pytest.raises(L.SpecdecError):
            A.tree_attention(*call, out=torch.empty(shape, dtype=dtype, device=DEV).expand(2, 6, 8, d), **kw)
    room = torch.empty(2 * 6 * 8 * d, dtype=dtype, device=DEV)
    with pytest.raises(L.SpecdecError):
        A.tree_attention(*call, out=room.as_strided((2, 6, 8, d), (5 * 8 * d, 8 * d, d, 1)), **kw)
    for order in ((0, 1, 2, 3), (2, 1, 0, 3), (1, 2, 0, 3)):     # any order of the dimensions
        out = torch.empty([(2, 6, 8, d)[i] for i in order], dtype=dtype, device=DEV)
        back = [order.index(i) for i in range(4)]
        _check(call, kw, ref, out=out.permute(back))


@gpu
@pytest.mark.parametrize("n", [40, 70])
@pytest.mark.parametrize("paged", [False, True])
def test_a_tree_on_an_empty_cache_is_a_tree(n, paged):
    """Through the caches, with a cap on the padding given, too: no causal shortcut."""
    from specdec.kvcache import PagedRaggedCache, RaggedCache
    g = torch.Generator().manual_seed(n)
    masks, depths = tree_masks(_parents(n, g), device=DEV)
    c = PagedRaggedCache(1, 2, 128, DEV) if paged else RaggedCache(1, 2, 128, DEV, attn_impl="specdec_b200")
    if paged:
        c.reserve(n)
    c.set_tree(masks, depths)
    q, k, v = (torch.randn(2, h, n, 128, generator=g).to(torch.bfloat16).to(DEV) for h in (4, 2, 2))
    c.attn_mask(n, torch.bfloat16, valid=torch.tensor([n, n], device=DEV))
    keys, values = c.layers[0].update(k, v)
    out, _ = A.hf_attention(None, q, keys, values, None, scaling=0.125)
    want = A.tree_attention(q, keys, values, c.lengths, masks, scale=0.125,
                            block_table=c.block_table if paged else None)
    assert torch.equal(out, want)
