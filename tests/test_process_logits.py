"""process_logits and TokenHistory against their definition in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, every step rounds once to float32, a
product and the following subtraction perhaps together): the scaled logit is off by
u |x1|, frequency * c by u |f c|, each of the two subtractions and the bias
addition by u times its result, the sum of M biases by M u sum |b|:
  |error| <= u (|x1| + |f c| + 3 (|x1| + |f c| + |p| + sum |b|) + M sum |b|), then half a step of the
output type.  Untouched entries, -inf and masks are exact.
"""
import math

import pytest
import torch

from specdec import _lib as L
from specdec.sampling import BIAS_MAX, TokenHistory, process_logits
from specdec.tree import TREE_MAX, tree_masks

gpu = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _bits(parents):
    n = len(parents)
    out = torch.zeros(n, n, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            out[i] = out[p]
        out[i, i] = True
    return out


def _plain(x, tokens, sees, hist, rep, pres, freq, bias, allowed):
    """(result, error bound before the output's rounding) in float64; sees [B or 1, L, N]."""
    B, Lq, V = x.shape
    z = x.double()
    zero = torch.zeros((), dtype=torch.float64)
    tol = torch.zeros_like(z)
    if hist is not None:
        h = hist.long().view(B, 1, V)
        c = (h % 32768).expand(B, Lq, V).clone()
        if tokens is not None:
            for b in range(B):
                for l in range(Lq):
                    for i in torch.nonzero(sees[b if sees.shape[0] > 1 else 0, l]).view(-1).tolist():
                        t = int(tokens[b, i])
                        if 0 <= t < V:
                            c[b, l, t] += 1
        col = lambda t, d: (torch.full((B,), d) if t is None else t).double().view(B, 1, 1)  # noqa: E731
        r, p, f = col(rep, 1.0), col(pres, 0.0), col(freq, 0.0)
        hit = (c > 0) | (h < 0)
        x1 = torch.where(hit, torch.where(z > 0, z / r, z * r), z)
        z = torch.where(hit, x1 - f * c - p * (c > 0), z)
        tol += torch.where(hit, U * (4 * x1.abs() + 4 * (f * c).abs() + 3 * p.abs()), zero)
    if bias is not None:
        ids, val = bias
        add, mag, cnt = torch.zeros_like(z), torch.zeros_like(z), torch.zeros_like(z)
        for b in range(B):
            bb = b if ids.shape[0] > 1 else 0
            for t, w in zip(ids[bb].tolist(), val[bb].tolist()):
                if 0 <= t < V:
                    add[b, :, t] += w
                    mag[b, :, t] += abs(w)
                    cnt[b, :, t] += 1
        z = z + add
        tol += U * ((3 + cnt) * mag + torch.where(cnt > 0, z.abs(), zero))
    if allowed is not None:
        bit = torch.arange(V)
        on = (allowed.long()[..., bit // 32] >> (bit % 32)) & 1
        z = torch.where(on.expand(B, Lq, V) == 1, z, torch.tensor(-math.inf, dtype=torch.float64))
    return z, torch.where(torch.isfinite(tol), tol, zero)


def _check(got, z, tol, dtype):
    got = got.cpu().double()
    nan = z.isnan()
    assert torch.equal(got.isnan(), nan)
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    fin = torch.isfinite(z)
    big = torch.finfo(dtype).max
    over = fin & (z.abs() > big * (1 - half))            # may round to infinity
    assert torch.equal(got[~fin & ~nan], z[~fin & ~nan])
    fin &= ~over
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    lim = tol + half * (z.abs() + tol) + (tiny / 2 if dtype == torch.float16 else 0.0)
    d = (got - z).abs()
    assert bool((d[fin] <= lim[fin]).all()), float((d[fin] / (lim[fin] + 1e-300)).max())


def _inputs(B, Lq, V, N, dtype, seed, pad=0, hist_pad=0, tree=False, M=0, one_bias=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, Lq, V + pad, generator=g) * 4).to(dtype)
    tokens = torch.randint(-1, V + 1, (B, N), generator=g) if N else None
    if N:
        tokens[:, N // 2:] = tokens[:, :N - N // 2]       # the same token twice on a path
    parents = [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, N)]
    sees = (_bits(parents) if tree else torch.ones(N, N).tril().bool())[N - Lq:].unsqueeze(0) if N else None
    hist = torch.zeros(B, V + hist_pad, dtype=torch.int16)
    for b in range(B):
        w = torch.randint(0, V, (max(1, V // 8),), generator=g)
        hist[b, :V] += torch.bincount(w, minlength=V).to(torch.int16)
        hist[b, torch.randint(0, V, (max(1, V // 6),), generator=g)] |= -32768
        hist[b, int(torch.randint(0, V, (1,), generator=g))] = 32767
    par = [torch.rand(B, generator=g) + 0.6, torch.randn(B, generator=g), torch.randn(B, generator=g) * .3]
    bias = None
    if M:
        nb = 1 if one_bias else B
        bias = (torch.randint(-1, V + 1, (nb, M), generator=g), torch.randn(nb, M, generator=g) * 5)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (B, Lq, -(-V // 32)), generator=g).to(torch.int32)
    allowed[0, 0] = 0                                    # a row with nothing left
    if B > 1:
        allowed[1, -1] = -1                              # and one with everything
    return x, tokens, parents, sees, hist, par, bias, allowed


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,Lq,V,N,tree,M,pad,hist_pad", [
    (1, 1, 1, 1, False, 1, 0, 0), (2, 1, 40, 1, False, 0, 0, 0), (3, 5, 1000, 5, False, 7, 0, 0),
    (2, 4, 2049, 9, True, 300, 1, 3), (1, 1, 151936, 1, False, 16, 0, 0), (2, 3, 32003, 64, True, 0, 0, 5),
    (4, 2, 8192, 2, False, BIAS_MAX, 8, 8), (1, 1, 7, TREE_MAX, True, 0, 0, 0),
    (5, 9, 4104, 40, True, 33, 0, 0)])
def test_against_the_definition(dtype, B, Lq, V, N, tree, M, pad, hist_pad):
    x, tokens, parents, sees, hist, par, bias, allowed = _inputs(B, Lq, V, N, dtype, V, pad, hist_pad,
                                                                tree, M, M % 2 == 1)
    gx, gh = x.to(DEV)[..., :V], hist.to(DEV)[:, :V]
    masks = tree_masks(parents, device=DEV).masks if tree else None
    gb = None if bias is None else tuple(t.to(DEV) for t in bias)
    gp = dict(zip(("repetition", "presence", "frequency"), (t.to(DEV) for t in par)))
    kept = gx.clone()
    for use_hist, use_bias, use_mask in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 0, 0)):
        b = bias if use_bias else None
        z, tol = _plain(x[..., :V], tokens, sees, hist[:, :V] if use_hist else None, *par, b,
                        allowed if use_mask else None)
        got = process_logits(gx, tokens.to(DEV), masks, bias=gb if use_bias else None,
                             allowed=allowed.to(DEV) if use_mask else None,
                             **(dict(history=gh, **gp) if use_hist else {}))
        assert got.shape == (B, Lq, V) and got.dtype == dtype and got.is_contiguous()
        _check(got, z, tol, dtype)
        assert torch.equal(gx, kept)
    # in place, and into a view
    z, tol = _plain(x[..., :V], tokens, sees, hist[:, :V], *par, bias, allowed)
    wide = torch.full((B, Lq, V + 9), 3.0, dtype=dtype, device=DEV)
    _check(process_logits(gx, tokens.to(DEV), masks, history=gh, bias=gb, allowed=allowed.to(DEV),
                          out=wide[..., 4:V + 4], **gp), z, tol, dtype)
    assert bool((wide[..., :4] == 3).all()) and bool((wide[..., V + 4:] == 3).all())
    same = process_logits(gx, tokens.to(DEV), masks, history=gh, bias=gb, allowed=allowed.to(DEV),
                          out=gx, **gp)
    assert same is gx
    _check(gx, z, tol, dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [40, 2049, 20001])
def test_every_alignment_of_input_output_and_history(dtype, V):
    x, tokens, parents, sees, hist, par, bias, allowed = _inputs(2, 3, V, 4, dtype, V, M=5)
    gb, allowed_d = tuple(t.to(DEV) for t in bias), allowed.to(DEV)
    gp = dict(zip(("repetition", "presence", "frequency"), (t.to(DEV) for t in par)))
    z, tol = _plain(x, tokens, sees, hist, *par, bias, allowed)
    for a, c, h in ((0, 1, 1), (1, 0, 2), (3, 3, 8), (5, 2, 0), (8, 7, 5)):
        room = torch.full((2, 3, V + 16), 3.0, dtype=dtype, device=DEV)
        room_h = torch.full((2, V + 16), 77, dtype=torch.int16, device=DEV)
        room[..., a:a + V], room_h[:, h:h + V] = x.to(DEV), hist.to(DEV)
        out = torch.full((2, 3, V + 16), 3.0, dtype=dtype, device=DEV)
        kw = dict(history=room_h[:, h:h + V], bias=gb, allowed=allowed_d, **gp)
        _check(process_logits(room[..., a:a + V], tokens.to(DEV), out=out[..., c:c + V], **kw), z, tol, dtype)
        assert bool((out[..., :c] == 3).all()) and bool((out[..., c + V:] == 3).all())
        view = room[..., a:a + V]
        _check(process_logits(view, tokens.to(DEV), out=view, **kw), z, tol, dtype)
        assert bool((room[..., :a] == 3).all()) and bool((room[..., a + V:] == 3).all())


@gpu
def test_outputs_over_other_logits_are_refused():
    wide = torch.randn(4, 3, 64, device=DEV)
    for logits, out in ((wide[:2], wide[1:3]), (wide[::2], wide[1::2])):
        before = wide.clone()
        with pytest.raises(L.SpecdecError):
            process_logits(logits, out=out)
        assert torch.equal(wide, before)
    flat = torch.randn(2 * 3 * 64 + 8, device=DEV)
    with pytest.raises(L.SpecdecError):
        process_logits(flat[:384].view(2, 3, 64), out=flat[4:388].view(2, 3, 64))


@gpu
def test_shared_masks_numbers_and_missing_tokens():
    """One mask for all rows or positions, numbers for the penalties, no drafted tokens."""
    x, tokens, _, _, hist, par, _, allowed = _inputs(3, 4, 515, 4, torch.float32, 0)
    gx, gh = x.to(DEV), hist.to(DEV)
    for a in (allowed[:1], allowed[:, :1], allowed[:1, :1], allowed):
        z, tol = _plain(x, None, None, hist, torch.full((3,), 1.3), None, torch.full((3,), 0.25), None, a)
        got = process_logits(gx, history=TokenHistory.over(gh), repetition=1.3, frequency=0.25,
                             allowed=a.to(DEV))
        _check(got, z, tol, torch.float32)
    strided = torch.zeros(3, 8, 40, dtype=torch.int32, device=DEV)[:, ::2, 10:27]
    strided.copy_(allowed)
    z, tol = _plain(x, None, None, None, None, None, None, None, allowed)
    _check(process_logits(gx, allowed=strided), z, tol, torch.float32)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_and_nan(dtype):
    """Masked places win over everything; others follow the formula."""
    V = 640
    x = torch.zeros(1, 1, V, dtype=dtype)
    x[0, 0, :6] = torch.tensor([math.inf, -math.inf, math.nan, torch.finfo(dtype).max,
                                torch.finfo(dtype).min, -0.0])
    hist = torch.zeros(1, V, dtype=torch.int16)
    hist[0, :6] = 3
    hist[0, 100:] = -32768
    allowed = torch.full((1, 1, V // 32), -1, dtype=torch.int32)
    x[0, 0, 40:80] = math.nan
    allowed[0, 0, 1] = 0                                 # 32 to 63
    par = [torch.tensor([1.5]), torch.tensor([0.5]), torch.tensor([0.25])]
    z, tol = _plain(x, None, None, hist, *par, None, allowed)
    got = process_logits(x.to(DEV), history=hist.to(DEV), allowed=allowed.to(DEV),
                         **dict(zip(("repetition", "presence", "frequency"), (p.to(DEV) for p in par))))
    _check(got, z, tol, dtype)
    assert bool((got[0, 0, 40:64] == -math.inf).all()) and bool(got[0, 0, 64:80].isnan().all())


@gpu
def test_chain_positions_of_the_last_tokens():
    """L < N: the logits are those of the last L nodes (a draft model's step)."""
    V = 50
    x = torch.zeros(1, 1, V)
    tokens = torch.tensor([[7, 9, 7, 12]])
    got = process_logits(x.to(DEV), tokens.to(DEV), history=TokenHistory(1, V, DEV), frequency=1.0)
    want = torch.zeros(V)
    want[7], want[9], want[12] = -2, -1, -1
    assert torch.equal(got.cpu().view(-1), want)
    masks = tree_masks([-1, 0, 0, 2], device=DEV).masks   # node 3 hangs on 2 and 0
    got = process_logits(x.to(DEV), tokens.to(DEV), masks, history=TokenHistory(1, V, DEV), frequency=1.0)
    want[9] = 0
    assert torch.equal(got.cpu().view(-1), want)


@gpu
def test_offsets_past_32_bits():
    B, Lq, V = 2, 120, 9_000_000
    x = torch.zeros(B, Lq, V, dtype=torch.bfloat16, device=DEV)
    assert x.numel() > 2 ** 31
    x[1, 119] = 1.0
    hist = TokenHistory(B, V, DEV)
    hist.append(torch.tensor([[0], [V - 1]], device=DEV))
    process_logits(x, history=hist, presence=2.0, out=x)
    assert float(x[1, 119, V - 1]) == -1.0 and float(x[1, 119, V - 2]) == 1.0
    assert float(x[0, 0, 0]) == -2.0 and int((x[0, 5] != 0).sum()) == 1


@gpu
def test_history():
    B, V = 3, 77
    h = TokenHistory(B, V, DEV)
    assert h.counts.shape == (B, V) and not bool(h.counts.any())
    ids = torch.tensor([[5, 5, 76, -1], [0, 1, 2, 3], [9, 9, 9, 9]], device=DEV)
    h.add_prompt(ids, torch.tensor([4, 2, 0], device=DEV))
    h.append(ids, torch.tensor([3, 4, 2], device=DEV))
    h.append(ids[:, :1].int())
    want = torch.zeros(B, V, dtype=torch.int64)
    want[0, 5], want[0, 76] = 3 - 32768, 1 - 32768
    want[1, 0], want[1, 1], want[1, 2], want[1, 3] = 2 - 32768, 1 - 32768, 1, 1
    want[2, 9] = 3
    assert torch.equal(h.counts.cpu().long(), want)
    path = torch.tensor([[0, 2, -1], [0, 3, 1], [0, 50, 1]], dtype=torch.int32, device=DEV)
    h.append(ids, torch.tensor([3, 2, 3], device=DEV), path=path)
    want[0, 5] += 1
    want[0, 76] += 1
    want[1, 0] += 1
    want[1, 3] += 1
    want[2, 9] += 2
    assert torch.equal(h.counts.cpu().long(), want)
    two = h.repeat_interleave(2)
    assert torch.equal(two.counts.cpu().long(), want.repeat_interleave(2, 0))
    h.reset([1])
    want[1] = 0
    assert torch.equal(h.counts.cpu().long(), want)
    h.reset()
    assert not bool(h.counts.any())
    many = torch.full((B, 40000), 11, device=DEV)         # counts stop at 32767
    h.append(many)
    h.add_prompt(many[:, :1])
    assert h.counts[:, 11].tolist() == [-1] * B and int((h.counts != 0).sum()) == B
    assert bool((h.counts[:, 11].long() % 32768 == 32767).all())


@gpu
def test_replays_and_streams():
    V = 3000
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, V, generator=g).to(DEV)
    tok = torch.randint(0, V, (2, 3), generator=g).to(DEV)
    h = TokenHistory(2, V, DEV)
    n = torch.tensor([3, 1], device=DEV)
    process_logits(x, tok, history=h, frequency=0.5)
    rep = torch.tensor([1.2, 0.9], device=DEV)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = process_logits(x, tok, history=h, repetition=rep)
        h.append(tok, n)
    hist = torch.zeros(2, V, dtype=torch.int16)
    for _ in range(3):
        x.copy_(torch.randn(2, 3, V, generator=g))
        tok.copy_(torch.randint(0, 9, (2, 3), generator=g))
        gr.replay()
        z, tol = _plain(x.cpu(), tok.cpu(), torch.ones(3, 3).tril().bool().unsqueeze(0), hist, rep.cpu(),
                        None, None, None, None)
        _check(out, z, tol, torch.float32)
        for b, k in enumerate(n.tolist()):
            for t in tok[b, :k].tolist():
                hist[b, t] += 1
        assert torch.equal(h.counts.cpu(), hist)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = process_logits(x, tok, history=h, repetition=rep)
    side.synchronize()
    assert torch.equal(again, process_logits(x, tok, history=h, repetition=rep))


@gpu
def test_refusals():
    x = torch.zeros(2, 3, 64, device=DEV)
    tok = torch.zeros(2, 3, dtype=torch.long, device=DEV)
    h = TokenHistory(2, 64, DEV)
    masks = tree_masks([-1, 0, 0], device=DEV).masks
    ids, val = torch.zeros(2, 1, dtype=torch.long, device=DEV), torch.zeros(2, 1, device=DEV)
    mask = torch.zeros(2, 3, 2, dtype=torch.int32, device=DEV)
    bad = [
        ((x[0],), {}), ((x.double(),), {}), ((x.transpose(1, 2),), {}), ((x, tok[:, :2]), {}),
        ((x, tok.float()), {}), ((x, tok[:1]), {}), ((x, tok.cpu()), {}), ((x,), dict(masks=masks)),
        ((x, tok, masks[:2]), {}), ((x, torch.zeros(2, TREE_MAX + 1, dtype=torch.long, device=DEV)), {}),
        ((x,), dict(repetition=1.2)), ((x,), dict(history=TokenHistory(2, 63, DEV))),
        ((x,), dict(history=h.counts.int())), ((x,), dict(history=h, presence=torch.zeros(3, device=DEV))),
        ((x,), dict(bias=(ids, val[:1]))), ((x,), dict(bias=(ids.float(), val))),
        ((x,), dict(bias=(ids.expand(2, 1).repeat(1, BIAS_MAX + 1), val.repeat(1, BIAS_MAX + 1)))),
        ((x,), dict(allowed=mask.long())), ((x,), dict(allowed=mask[..., :1])),
        ((x,), dict(allowed=mask[:, :2])), ((x,), dict(out=torch.zeros(2, 3, 63, device=DEV))),
        ((x,), dict(out=torch.zeros(2, 3, 64, dtype=torch.bfloat16, device=DEV))),
    ]
    for args, kw in bad:
        with pytest.raises(L.SpecdecError):
            process_logits(*args, **kw)
    assert process_logits(x[:0]).shape == (0, 3, 64) and process_logits(x[:, :0]).shape == (2, 0, 64)
    for f in (lambda: h.append(tok[:1]), lambda: h.append(tok.float()), lambda: h.append(tok, tok),
              lambda: h.append(tok, path=tok), lambda: h.append(tok.cpu()),
              lambda: TokenHistory.over(h.counts.int()), lambda: TokenHistory.over(h.counts[0])):
        with pytest.raises(L.SpecdecError):
            f()


def test_refused_on_the_host():
    lib = L.lib()
    ok = dict(x=16, dt=0, B=1, L=1, V=8, tok=None, N=0, first=0, ids=None, val=None, M=0, out=16)

    def call(**kw):
        a = {**ok, **kw}
        return lib.sd_process_logits(a["x"], 8, 8, a["dt"], a["B"], a["L"], a["V"], a["tok"], 4, None, 0,
                                     a["N"], a["first"], None, 0, None, None, None, a["ids"], a["val"], 0,
                                     a["M"], None, 0, 0, a["out"], 8, 8, None)
    for kw in (dict(x=None), dict(out=None), dict(dt=7), dict(B=-1), dict(V=0), dict(N=4), dict(M=3),
               dict(tok=16, N=4, first=4), dict(first=-1)):
        assert call(**kw) == -22, kw
    assert call(tok=16, N=TREE_MAX + 1) == -95
    assert call(ids=16, val=16, M=BIAS_MAX + 1) == -95
    assert call(B=0) == 0
    assert lib.sd_history_add(None, 8, 8, 16, 4, 4, None, 0, None, 4, 1, 0, None) == -22
    assert lib.sd_history_add(16, 8, 8, 16, 4, 3, None, 0, None, 4, 1, 0, None) == -22
    assert lib.sd_history_add(16, 8, 8, 16, 4, 4, None, 0, None, 0, 1, 0, None) == 0
    for f in (lambda: process_logits(torch.zeros(1, 1, 4)), lambda: TokenHistory(1, 4, "cpu"),
              lambda: TokenHistory.over(torch.zeros(1, 4, dtype=torch.int16))):
        with pytest.raises(L.SpecdecError):
            f()


def _out_strides(**kw):
    """rc of a call whose output has these sizes and strides (refused before any launch)."""
    a = dict(x=1 << 20, xbs=64, xps=8, B=1, L=1, V=8, out=1 << 24, bs=8, ps=8)
    a.update(kw)
    return L.lib().sd_process_logits(a["x"], a["xbs"], a["xps"], 0, a["B"], a["L"], a["V"], None, 0,
                                     None, 0, 0, 0, None, 0, None, None, None, None, None, 0, 0, None,
                                     0, 0, a["out"], a["bs"], a["ps"], None)


def test_outputs_that_overlap_themselves_are_refused_on_the_host():
    """Rows or positions of the output that share entries: several CTAs would write them."""
    same = dict(x=1 << 24)                               # in place
    for kw in (dict(B=2, bs=0), dict(L=2, ps=0), dict(B=2, bs=7), dict(L=2, ps=7), dict(B=2, bs=-7),
               dict(B=2, L=3, bs=16, ps=8), dict(B=3, L=2, bs=8, ps=16), dict(B=2, L=2, bs=12, ps=8),
               dict(B=2, bs=0, xbs=0, **same), dict(L=4, ps=0, xps=0, **same),
               dict(B=2, L=2, bs=8, ps=8, xbs=8, xps=8, **same)):
        assert _out_strides(**kw) == -22, kw


@gpu
def test_outputs_that_overlap_themselves_are_refused():
    x = torch.randn(3, 2, 40, device=DEV)
    room = torch.zeros(400, device=DEV)
    for out in (room[:80].view(1, 2, 40).expand(3, -1, -1), room[:120].view(3, 1, 40).expand(-1, 2, -1),
                room.as_strided((3, 2, 40), (60, 40, 1)), room.as_strided((3, 2, 40), (40, 39, 1))):
        with pytest.raises(L.SpecdecError):
            process_logits(x, out=out)
    for same in (x[:1].expand(3, -1, -1), x[:, :1].expand(-1, 2, -1)):
        before = x.clone()
        with pytest.raises(L.SpecdecError):
            process_logits(same, out=same)
        assert torch.equal(x, before)
        assert torch.equal(process_logits(same), same)   # (as an input they are good)
    turned = torch.zeros(2, 3, 40, device=DEV).transpose(0, 1)
    assert torch.equal(process_logits(x, out=turned), x)
    one = room.as_strided((1, 2, 40), (0, 50, 1))        # the stride of a single row is any
    assert torch.equal(process_logits(x[:1], out=one), x[:1])
