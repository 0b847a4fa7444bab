"""prefix_attention against its definition in 64 bits.

Tolerance, bf16 heads of 128.  With w_s the exact softmax weights and A =
sum_s w_s |v_s| (per output element): the kernel rounds each unnormalised
weight to bf16 (relative 2^-8 at most) but sums the unrounded ones, which moves
the output by at most 2^-8 A; the final rounding adds 2^-8 of the result.
Scores are float32 sums of 128 exact products, so a weight is off by at most
2 * 128 * 2^-24 * scale * sum |q k| relative (numerator and denominator):
2^-10 with scale * sum |q k| <= 64, as all cases here have.  The exponentials
(2^-22) and the float32 accumulation are far below.  So
|out - exact| <= 2^-8 |exact| + (2^-8 + 2^-10) A.
fp32 (CUDA-core path): the same 2^-10 for the scores bounds it; 2^-9 A leaves
the exponential and the sums their part.  bf16 of other head sizes takes that
path too, with float32 weights: 2^-9 A and 2^-8 of the result's own rounding,
within the bf16 bound above.
"""
import ctypes
import math

import pytest
import torch

from specdec import _lib as L
from specdec import attention as A
from specdec.kvcache import PAGE

gpu = pytest.mark.gpu
DEV = "cuda"


def _case(sizes, pages, suffix, qlen, hq, hkv, D=128, dt=torch.bfloat16, seed=0, lone=0, width=0,
          stale=float("nan")):
    """Groups of `sizes` rows sharing `pages` pages each, then `lone` rows of no
    group; row b holds pages * PAGE + suffix[b] tokens before this step.  Every
    pool slot that no row may see holds `stale`."""
    g = torch.Generator().manual_seed(seed)
    B = sum(sizes) + lone
    shared = [p for n, p in zip(sizes, pages) for _ in range(n)] + [0] * lone
    lens = [p * PAGE + s for p, s in zip(shared, suffix)]
    live = [n + qlen for n in lens]
    W = max(max(-(-n // PAGE) for n in live), width, 1)
    group = [i for i, n in enumerate(sizes) for _ in range(n)]
    n_pages = sum(pages) + sum(-(-n // PAGE) - p for n, p in zip(live, shared)) + 3
    ids = torch.randperm(n_pages, generator=g).tolist()
    front = [[ids.pop() for _ in range(p)] for p in pages]
    bt = torch.full((B, W), -1, dtype=torch.int32)
    for b in range(B):
        row = list(front[group[b]]) if b < len(group) else []
        row += [ids.pop() for _ in range(-(-live[b] // PAGE) - len(row))]
        bt[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    k = torch.full((n_pages, hkv, PAGE, D), stale)
    v = torch.full((n_pages, hkv, PAGE, D), stale)
    for b in range(B):
        for s in range(0, live[b], PAGE):
            n = min(PAGE, live[b] - s)
            p = int(bt[b, s // PAGE])
            k[p, :, :n] = torch.randn(hkv, n, D, generator=g)
            v[p, :, :n] = torch.randn(hkv, n, D, generator=g) + 0.3
    q = torch.randn(B, qlen, hq, D, generator=g)
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(q=q.to(dt).to(DEV).transpose(1, 2), k=k.to(dt).to(DEV), v=v.to(dt).to(DEV),
                lens=torch.tensor(lens, device=DEV), bt=bt.to(DEV), starts=i32(starts),
                pages=i32(list(pages)))


def _definition(c, valid=None, scale=None):
    """(out, A) in float64 on the CPU, row by row."""
    q, k, v = c["q"].cpu().double(), c["k"].cpu().double(), c["v"].cpu().double()
    B, hq, qlen, D = q.shape
    hkv = k.shape[1]
    sc = D ** -0.5 if scale is None else scale
    out, mag = torch.zeros(B, qlen, hq, D).double(), torch.zeros(B, qlen, hq, D).double()
    bt, lens = c["bt"].cpu(), c["lens"].tolist()
    for b in range(B):
        for j in range(qlen):
            n = lens[b] + j + 1
            n = n if valid is None else max(0, min(n, valid[b]))
            if n == 0:
                continue
            pg = bt[b, :-(-n // PAGE)].long()
            kb = k[pg].permute(1, 0, 2, 3).reshape(hkv, -1, D)[:, :n]
            vb = v[pg].permute(1, 0, 2, 3).reshape(hkv, -1, D)[:, :n]
            qq = q[b, :, j].view(hkv, hq // hkv, D)
            w = torch.softmax(torch.einsum("hgd,hsd->hgs", qq, kb) * sc, -1)
            out[b, j] = torch.einsum("hgs,hsd->hgd", w, vb).reshape(hq, D)
            mag[b, j] = torch.einsum("hgs,hsd->hgd", w, vb.abs()).reshape(hq, D)
    return out, mag


def _run(c, **kw):
    return A.prefix_attention(c["q"], c["k"], c["v"], c["lens"], c["bt"], c["starts"], c["pages"],
                              **kw)


def _check(c, valid=None, scale=None):
    val = None if valid is None else torch.tensor(valid, device=DEV)
    got = _run(c, valid=val, scale=scale)
    want, mag = _definition(c, valid, scale)
    g = got.cpu().double()
    assert bool(g.isfinite().all())
    if got.dtype == torch.bfloat16:
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * mag
    else:
        tol = 2.0 ** -9 * mag
    bad = (g - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), ((g - want).abs() / tol.clamp_min(1e-30)).max())
    return got


@gpu
@pytest.mark.parametrize("hq,hkv,qlen", [(32, 8, 1), (32, 8, 5), (16, 8, 3), (8, 8, 1), (8, 1, 4),
                                         (16, 1, 2), (32, 1, 1), (4, 2, 9), (32, 8, 13)])
def test_heads_and_queries(hq, hkv, qlen):
    _check(_case([3, 2], [2, 1], [0, 5, 130, 127, 300], qlen, hq, hkv, seed=qlen))


@gpu
@pytest.mark.parametrize("sizes,pages", [([2], [1]), ([7], [9]), ([64], [3]), ([1, 1], [2, 2]),
                                         ([3, 1, 5], [0, 4, 2]), ([20, 30], [5, 0]),
                                         ([2] * 12, [1, 2, 3] * 4)])
def test_groups(sizes, pages):
    n = sum(sizes)
    _check(_case(sizes, pages, [(37 * b) % 290 for b in range(n)], 2, 8, 2, seed=n))


@gpu
@pytest.mark.parametrize("rows", [1, 15, 16, 17, 31, 32, 33, 47, 48, 64, 65])
def test_rows_around_the_tile_bounds(rows):
    """8 query rows per batch row and kv head: one tile up to 16 rows, then pairs."""
    _check(_case([rows], [4], [b % 5 for b in range(rows)], 4, 4, 2, seed=rows))


@gpu
@pytest.mark.parametrize("pages", [1, 2, 3, 5, 40, 67])
@pytest.mark.parametrize("rows,hkv", [(3, 1), (40, 2)])
def test_long_prefixes_split_over_the_machine(pages, rows, hkv):
    """Few rows and heads: a prefix is split over many CTAs and joined again."""
    _check(_case([rows], [pages], [1 + b % 3 for b in range(rows)], 1, 8 * hkv, hkv, seed=pages))


@gpu
def test_rows_of_no_group_and_no_groups_at_all():
    _check(_case([2, 3], [2, 3], [9, 200, 0, 1, 127, 50, 400], 3, 8, 2, lone=2))
    c = _case([], [], [9, 200], 3, 8, 2, lone=2)
    assert c["pages"].numel() == 0
    _check(c)


@gpu
def test_rows_shorter_than_the_prefix():
    """Empty, short and just-long-enough rows in a group: cut lengths."""
    c = _case([6], [3], [0, 10, 20, 0, 5, 130], 4, 8, 2, stale=0.0)
    c["lens"] = torch.tensor([0, 3 * PAGE - 1, 3 * PAGE - 2, 100, 3 * PAGE - 5, 3 * PAGE + 130],
                             device=DEV)
    _check(c)


@gpu
def test_caps():
    """valid: nothing, inside the prefix, at its end, inside the row's own keys."""
    c = _case([4, 3], [2, 1], [10, 140, 3, 0, 60, 200, 7], 5, 8, 4)
    _check(c, valid=[0, 100, 2 * PAGE, 2 * PAGE + 2, 1, PAGE + 130, 10 ** 6])
    out = _run(c, valid=torch.zeros(7, dtype=torch.long, device=DEV))
    assert bool((out == 0).all())


@gpu
def test_matches_verify_attention():
    c = _case([16, 9], [6, 11], [(61 * b) % 500 for b in range(25)], 5, 32, 8, stale=0.0)
    got = _run(c).float()
    want = A.verify_attention(c["q"], c["k"], c["v"], c["lens"], block_table=c["bt"]).float()
    # both round weights and result to bf16: twice the tolerance of one
    _, mag = _definition(c)
    assert bool(((got - want).abs().cpu() <= 2 * (2.0 ** -7 + 2.0 ** -10) * mag).all())


F32, BF16 = torch.float32, torch.bfloat16


@gpu
@pytest.mark.parametrize("D,dt", [(64, F32), (128, F32), (64, BF16), (8, F32), (1, F32), (33, F32),
                                  (100, F32), (72, BF16), (30, BF16)])
def test_other_shapes_row_by_row(D, dt):
    _check(_case([3, 2], [1, 2], [5, 0, 130, 44, 17], 3, 8, 2, D=D, dt=dt))


@gpu
@pytest.mark.parametrize("hq,hkv,qlen,dt", [(8, 8, 1, F32), (6, 2, 7, F32), (4, 1, 40, F32),
                                            (256, 1, 1, BF16), (64, 1, 1, BF16)])
def test_rows_of_a_head_over_several_blocks(hq, hkv, qlen, dt):
    _check(_case([2], [1], [5, 9], qlen, hq, hkv, dt=dt))


@gpu
@pytest.mark.parametrize("rows,suffix", [(1, 2500), (2, 31), (2, 2049), (40, 300), (1, 0)])
def test_row_by_row_clusters(rows, suffix):
    """One to eight CTAs on a row, more groups of keys than they have warps."""
    _check(_case([], [], [suffix + 3 * b for b in range(rows)], 2, 4, 2, D=64, dt=F32, lone=rows,
                 width=24))


@gpu
def test_row_by_row_masks_nan_and_repeats():
    c = _case([3], [1], [100, 3, 250], 4, 4, 2, D=64, dt=F32)
    _check(c, valid=[0, 5, 300])
    _check(c, valid=[1, 128, 129], scale=0.5)
    want = _run(c)
    assert torch.equal(want, _run(c))
    q = c["q"].clone()
    q[1, 2, 3] = math.nan
    got = _run(dict(c, q=q))
    assert bool(got[1, 3, 2].isnan().all())
    got[1, 3, 2] = want[1, 3, 2]
    assert torch.equal(got, want)
    q = torch.empty(3, 4, 4, 65, device=DEV)[..., 1:]        # rows off the 16-byte bounds
    q.copy_(c["q"])
    assert torch.equal(_run(dict(c, q=q)), want)
    k = torch.empty(c["k"].numel() + 1, device=DEV)[1:].view(c["k"].shape)
    k.copy_(c["k"])
    _check(dict(c, k=k))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _run(c)
    c["lens"].add_(-3)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, _run(c)) and not torch.equal(out, want)


@gpu
def test_scale_and_large_scores():
    """Scores of hundreds: the running maximum moves often, most weights vanish."""
    c = _case([10], [5], [3 * b for b in range(10)], 2, 8, 2)
    _check(c, scale=0.5)
    c["q"] = c["q"] * 8.0
    _check(c, scale=0.088)


@gpu
def test_rising_scores_move_the_maximum_on_every_page():
    c = _case([9], [12], [50] * 9, 2, 8, 1)
    ramp = torch.arange(c["bt"].shape[1], device=DEV).float()
    for b in range(9):
        for j, p in enumerate(c["bt"][b].tolist()):
            if p >= 0:
                c["k"][p, :, :, 0] = (6.0 * ramp[j]).to(torch.bfloat16)
    c["q"][..., 0] = 8.0
    _check(c)


@gpu
def test_query_and_output_layouts():
    """q as [B, H, L, D], q off its alignment, a strided output whose gaps stay."""
    c = _case([5], [2], [5, 9, 1, 0, 130], 3, 8, 2)
    want = _check(c)
    c2 = dict(c, q=c["q"].contiguous())
    assert torch.equal(_run(c2), want)
    flat = torch.zeros(c["q"].numel() + 1, dtype=torch.bfloat16, device=DEV)
    flat[1:] = c["q"].contiguous().view(-1)
    assert torch.equal(_run(dict(c, q=flat[1:].view(c["q"].shape))), want)
    for pad in (8, 3):
        big = torch.full((5, 3, 8, 128 + pad), 7.0, dtype=torch.bfloat16, device=DEV)
        got = _run(c, out=big[..., :128])
        assert torch.equal(got, want) and bool((big[..., 128:] == 7.0).all())


@gpu
def test_nan_and_inf_of_one_row_stay_there():
    c = _case([6], [3], [20 * b + 1 for b in range(6)], 2, 8, 2)
    want = _run(c)
    q = c["q"].clone()
    q[2, 3, 1] = math.nan
    got = _run(dict(c, q=q))
    assert bool(got[2, 1, 3].isnan().all())
    got[2, 1, 3] = want[2, 1, 3]
    assert torch.equal(got, want)
    v = c["v"].clone()
    p = int(c["bt"][4, 3])                                   # row 4's own page
    v[p, 1, 5] = math.inf
    got = _run(dict(c, v=v))
    assert bool(got[4, :, 4:].isinf().all())
    got[4, :, 4:] = want[4, :, 4:]
    assert torch.equal(got, want)


@gpu
def test_a_short_row_does_not_meet_masked_values():
    """A NaN among prefix keys that a short row does not see leaves that row finite."""
    c = _case([3], [2], [5, 6, 7], 1, 4, 1, stale=0.0)
    c["lens"][1] = PAGE + 3
    want = _run(c)
    c["v"][int(c["bt"][0, 1]), 0, 100] = math.nan
    got = _run(c)
    assert torch.equal(got[1], want[1]) and bool(got[0].isnan().all()) and bool(got[2].isnan().all())


@gpu
def test_overlapping_groups_and_wild_arrays():
    """Group arrays out of order or out of range share less, not wrongly."""
    c = _case([8], [2], [3 * b for b in range(8)], 2, 8, 2, stale=0.0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for starts, pages in (([0, 5, 2, 8], [2, 2, 2]), ([-4, 100], [2]), ([0, 8], [-3]),
                          ([8, 0], [2]), ([0, 3, 3, 8], [2, 1, 1])):
        _check(dict(c, starts=i32(starts), pages=i32(pages)))


@gpu
def test_repeats_bit_for_bit_on_streams_and_in_graphs():
    a = _case([30], [20], [(61 * b) % 300 for b in range(30)], 5, 32, 8)
    b = _case([4, 5], [3, 7], [(17 * b) % 200 for b in range(9)], 1, 16, 8, seed=1)
    wa, wb = _run(a), _run(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(3):
        with torch.cuda.stream(s1):
            ra = _run(a)
        with torch.cuda.stream(s2):
            rb = _run(b)
        outs.append((ra, rb))
    torch.cuda.synchronize()
    assert all(torch.equal(x, wa) and torch.equal(y, wb) for x, y in outs)
    # graphs follow the lengths, the table and the group arrays on the device
    lens, pages = a["lens"].clone(), a["pages"].clone()
    a2 = dict(a, lens=lens, pages=pages)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        ra = _run(a2)
    with torch.cuda.graph(g2):
        rb = _run(b)
    pages.zero_()
    g1.replay()
    g2.replay()
    torch.cuda.synchronize()
    unshared = ra.clone()
    pages.copy_(a["pages"])
    g1.replay()
    torch.cuda.synchronize()
    assert torch.equal(ra, wa) and torch.equal(rb, wb)
    assert not torch.equal(unshared, wa)                     # another order of sums
    lens.fill_(20 * PAGE)
    g1.replay()
    torch.cuda.synchronize()
    assert torch.equal(ra, _run(a2))


@gpu
def test_refusals():
    c = _case([2], [1], [5, 9], 1, 4, 1)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan),
                dict(valid=torch.zeros(3, dtype=torch.long, device=DEV)),
                dict(out=torch.empty(2, 1, 4, 64, dtype=torch.bfloat16, device=DEV))):
        with pytest.raises(L.SpecdecError):
            _run(c, **bad)
    for key, bad in (("starts", c["starts"].long()), ("starts", c["starts"][:1]),
                     ("bt", c["bt"].long()), ("bt", c["bt"][:1]), ("k", c["k"].float()),
                     ("k", c["k"][:, :, :64]), ("lens", c["lens"][:1]), ("q", c["q"].half()),
                     ("q", c["q"].cpu())):
        with pytest.raises(L.SpecdecError):
            _run(dict(c, **{key: bad}))
    empty = {k: (v[:0] if k in ("q", "lens", "bt") else v) for k, v in c.items()}
    assert _run(empty).shape == (0, 1, 4, 128)


def test_refusals_on_cpu():
    z = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(L.SpecdecError):
        A.prefix_attention(z, z, z, i.long(), i.view(1, 1), i, i[:0])


def test_arguments_are_checked_before_any_launch():
    lib = L.lib()
    n, d = ctypes.c_void_p(0), ctypes.c_void_p(4096)

    def call(q=d, k=d, bt=d, bts=4, pages=9, lens=d, starts=d, G=1, B=2, Hq=8, Hkv=2, D=128, ql=3,
             scale=0.1, dtype=2, ws=d, nws=1 << 40, qs=1024):
        return lib.sd_prefix_attn(q, qs, 128, 1024, k, d, bt, bts, pages, lens, n, starts, d, G, B,
                                  Hq, Hkv, D, ql, scale, d, 0, 0, 0, dtype, ws, nws, n)
    assert call(B=0) == 0 and call(ql=0) == 0
    assert call(B=-1) == -22 and call(q=n) == -22 and call(bt=n) == -22 and call(lens=n) == -22
    assert call(starts=n) == -22 and call(Hq=7) == -22 and call(bts=0) == -22 and call(pages=0) == -22
    assert call(scale=0.0) == -22 and call(scale=float("nan")) == -22 and call(G=-1) == -22
    assert call(dtype=1) == -95 and call(bts=1 << 25) == -95
    assert call(pages=1 << 30) == -95
    assert call(q=ctypes.c_void_p(4104)) == -22 and call(qs=1027) == -22
    assert call(k=ctypes.c_void_p(4104)) == -22
    assert call(ws=n) == -28 and call(nws=100) == -28 and call(ws=ctypes.c_void_p(4112)) == -28
    size = lib.sd_prefix_attn_workspace_bytes
    assert size(64, 1, 32, 8, 128, 66, 5, 2) > 0 and size(64, 1, 32, 7, 128, 66, 5, 2) == 0
    assert size(64, 1, 32, 8, 64, 66, 5, 2) == 0 and call(D=136) == -95 and call(D=256, dtype=0) == -95


@gpu
@pytest.mark.parametrize("hq,hkv,qlen", [(4, 1, 40), (8, 2, 33), (32, 1, 5), (128, 1, 2), (8, 8, 129),
                                         (6, 2, 100)])
def test_more_query_rows_than_a_chunk(hq, hkv, qlen):
    """More than 128 query rows of a kv head: the own ranges take them in chunks, the
    last one shorter."""
    _check(_case([2, 1], [2, 1], [5, 126, 300], qlen, hq, hkv, seed=qlen))
    _check(_case([3], [1], [0, 60, 200], qlen, hq, hkv, seed=qlen), valid=[0, PAGE + 70, 10 ** 6])


@gpu
@pytest.mark.parametrize("sizes,pages", [([200], [2]), ([3] * 70, [1, 0, 2, 1, 3] * 14),
                                         ([2] * 330, [1] * 330), ([1100], [1]),
                                         ([2] * 520 + [40], [1, 0] * 260 + [2]),
                                         ([1] * 1030 + [5], [1] * 1030 + [1])])
def test_many_rows_and_groups(sizes, pages):
    """Past the plan's 1024 rows or groups at a time, past the threads of the kernels
    that look for a CTA's first row or group."""
    n = sum(sizes)
    _check(_case(sizes, pages, [(7 * b) % 130 for b in range(n)], 1, 2, 1, seed=n, stale=0.0))


@gpu
@pytest.mark.parametrize("scale", [1e4, 1e7, 3e8, 1e10, 1e20, 1e30])
@pytest.mark.parametrize("shift", [0.0, -60.0])
def test_scores_beyond_what_a_float_resolves(scale, shift):
    """Scores of 1e5 to 1e31, all of one sign in the second form: the largest takes
    the whole weight.  A float32 score of 128 products is off by at most 128 *
    2^-24 of their magnitudes' sum (1.5e-3 of scale here, with |q k| sums of 200): rows
    whose two largest scores are nearer than 4e-3 may give either and are left out."""
    c = _case([7, 3], [2, 1], [5, 130, 0, 44, 300, 9, 77, 12, 1, 200], 2, 8, 2, seed=3)
    c["k"][..., 0] = torch.where(c["k"][..., 0].isnan(), c["k"][..., 0], shift / 8.0)
    c["q"][..., 0] = 8.0
    got = _run(c, scale=scale).cpu().double()
    q, k, v = c["q"].cpu().double(), c["k"].cpu().double(), c["v"].cpu().double()
    seen = 0
    for b, n in enumerate(c["lens"].tolist()):
        for j in range(2):
            pg = c["bt"][b, :-(-(n + j + 1) // PAGE)].long().cpu()
            kb = k[pg].permute(1, 0, 2, 3).reshape(2, -1, 128)[:, :n + j + 1]
            vb = v[pg].permute(1, 0, 2, 3).reshape(2, -1, 128)[:, :n + j + 1]
            s = torch.einsum("hgd,hsd->hgs", q[b, :, j].view(2, 4, 128), kb)
            top, at = s.topk(2, -1)
            for h in range(2):
                for g in range(4):
                    if float(top[h, g, 0] - top[h, g, 1]) < 4e-3 + 20.0 / scale:
                        continue
                    want = vb[h, at[h, g, 0]]
                    tol = (2.0 ** -7 + 2.0 ** -10) * want.abs()
                    assert bool(((got[b, j, 4 * h + g] - want).abs() <= tol).all()), (b, j, h, g)
                    seen += 1
    assert seen > 120
