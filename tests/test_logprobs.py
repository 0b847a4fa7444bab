"""token_logprobs against its definition in 64 bits.

Tolerances, from the kernel's arithmetic.  u = 2^-24.  Every exponent is
d = fma(x, c, -R) held at -256 against a float reference R that cancels, and c =
log2(e) / T rounded: |error of d| <= 3 u |d|, plus 2^-22 relative for ex2.approx; the terms' weights 2^d make the
mean of that 3 ln2 u D, where D = sum |d| 2^d / z (the entropy's second part in
bits).  Sums of positive terms lose u relative per add: a thread adds at most
V / 512 + 8 terms one after another into each of two sums (a part has a step of
1024 units of 16 bytes or more; 2 V / 512 for fp32), moves them to a larger
reference a few times (3 u each, at most 20 here) and the joins add 5 + 8 + 7 + 7
more: K = 150 + V / 256 covers both types.
  log z: absolute error of that relative error, plus u |log z| for logf.
  logprob = (x - m) / T - log z: u |x - m| / T + u |log z| more.
  entropy = log z + ln2 D': D' carries the same relative errors as z plus one
  product per term, twice in the quotient.
With E(z) = 2^-22 + K u + 3 u D: |logprob| is within E + 3 u (|x-m|/T + |log
z|), |entropy| within 3 E (1 + D).  Ranks and ids are exact.
"""
import math

import pytest
import torch

from specdec import _lib as L
from specdec import sampling as S

gpu = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _definition(x, ids, T, n):
    """(logprob, rank, entropy, top_ids, top_logprobs) in float64 on the CPU."""
    x = x.detach().cpu().double()
    ids = ids.cpu().long()
    V = x.shape[-1]
    y = x / T
    lp = torch.log_softmax(y, -1)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    ent = torch.where(lp.isnan().any(-1), torch.full_like(ent, math.nan), ent)
    nan = x.isnan()
    key = torch.where(nan, torch.full_like(x, math.inf), x)
    # by (NaN first, value falling, id rising): two stable sorts
    by_value = torch.sort(key, dim=-1, descending=True, stable=True)[1]
    order = torch.gather(by_value, -1, torch.sort(
        torch.gather(nan.int(), -1, by_value), dim=-1, descending=True, stable=True)[1])
    place = torch.empty_like(order)
    place.scatter_(-1, order, torch.arange(V).expand_as(order).contiguous())
    ok = (ids >= 0) & (ids < V)
    at = ids.clamp(0, V - 1).unsqueeze(-1)
    logprob = torch.where(ok, lp.gather(-1, at).squeeze(-1), torch.full(ids.shape, math.nan,
                                                                       dtype=torch.float64))
    # what a float32 cannot hold (a lowest-value mask under T < 1) is -inf there
    lp = torch.where(lp < -torch.finfo(torch.float32).max, torch.full_like(lp, -math.inf), lp)
    logprob = torch.where(logprob < -torch.finfo(torch.float32).max,
                          torch.full_like(logprob, -math.inf), logprob)
    rank = torch.where(ok, place.gather(-1, at).squeeze(-1) + 1, torch.zeros_like(ids))
    top = order[..., :n]
    return logprob, rank, ent, top, lp.gather(-1, top), x, y


def _bounds(x, T):
    """(allowance of log z, D, |log z|) per row, from the module's derivation."""
    y = x.detach().cpu().double() / T
    m = y.amax(-1, keepdim=True)
    m = torch.where(m.isfinite(), m, torch.zeros_like(m))
    d = (y - m).clamp_min(-700.0)
    w = d.exp()
    z = w.sum(-1)
    D = (-d * w).sum(-1) / z / math.log(2.0)
    return 2.0 ** -22 + (150 + x.shape[-1] / 256) * U + 3 * U * D, D, z.log().abs()


def _check(x, ids, T, n):
    got = S.token_logprobs(x, ids, temperature=T, top_n=n)
    lp, rank, ent, top, tlp, xd, y = _definition(x, ids, T, n)
    ez, D, lz = _bounds(x, T)
    m = y.amax(-1)
    g = got.logprob.cpu().double()
    assert g.shape == lp.shape
    ok = lp.isfinite()
    assert torch.equal(ok, g.isfinite()) and torch.equal(lp.isnan(), g.isnan())
    assert torch.equal(lp[~ok & ~lp.isnan()], g[~ok & ~lp.isnan()])
    at = ids.cpu().long().clamp(0, x.shape[-1] - 1).unsqueeze(-1)
    dist = (m - y.gather(-1, at).squeeze(-1)).abs()
    tol = ez + 3 * U * (dist + lz)
    assert bool(((g - lp).abs()[ok] <= tol[ok]).all()), ((g - lp).abs()[ok] / tol[ok]).max()
    assert torch.equal(got.rank.cpu(), rank)
    e = got.entropy.cpu().double()
    fin = ent.isfinite()
    assert torch.equal(fin, e.isfinite())
    tol_e = 3 * ez * (1 + D)
    assert bool(((e - ent).abs()[fin] <= tol_e[fin]).all()), ((e - ent).abs()[fin] / tol_e[fin]).max()
    if n == 0:
        assert got.top_ids is None and got.top_logprobs is None
        return got
    assert torch.equal(got.top_ids.cpu(), top)
    t = got.top_logprobs.cpu().double()
    fin = tlp.isfinite()
    assert torch.equal(fin, t.isfinite()) and torch.equal(tlp.isnan(), t.isnan())
    tol_t = (ez + 3 * U * lz).unsqueeze(-1) + 3 * U * (m.unsqueeze(-1) - y.gather(-1, top)).abs()
    assert bool(((t - tlp).abs()[fin] <= tol_t[fin]).all())
    return got


def _logits(rows, V, dt, seed, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(*rows, V, generator=g, device=DEV) * scale
    ids = torch.randint(0, V, rows, generator=g, device=DEV)
    return x.to(dt), ids


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,n", [(1, 1), (2, 0), (7, 7), (32, 5), (33, 32), (255, 20), (2048, 3),
                                 (4097, 1), (32003, 20), (151936, 5)])
def test_against_the_definition(dt, V, n):
    x, ids = _logits((3,), V, dt, V + n)
    _check(x, ids, 1.0, n)
    _check(x, x.argmax(-1), 0.7, n)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,n", [(3, 0), (31, 31), (40, 32), (300, 32), (512, 20), (513, 32),
                                 (1000, 5), (1024, 32), (1025, 32), (1500, 32), (2047, 20)])
def test_small_vocabularies(dt, V, n):
    """A warp per row, and rows with fewer units than threads."""
    x, ids = _logits((37,), V, dt, 7 * V + n)
    x[0] = 0.0                                               # every entry on the list
    x[1] = -math.inf
    x[2, V // 2:] = -math.inf
    x[3, V - 1] = math.nan
    x[4, 0] = math.inf
    x[5] = -1.0
    x[5, V // 3:] = 1.0
    x[6, :-1] = torch.finfo(dt).min
    _check(x, ids, 1.0, n)
    _check(x[:, 1:], ids.clamp(max=V - 2), 0.3, min(n, V - 1))
    _check(x[:5].view(5, 1, V).expand(5, 3, V), ids[:15].view(5, 3), 2.0, n)


@gpu
@pytest.mark.parametrize("rows", [(1,), (150,), (700,), (5, 3), (2, 2, 3)])
def test_batches_and_shapes(rows):
    x, ids = _logits(rows, 5001, torch.bfloat16, 1)
    got = _check(x, ids, 1.3, 4)
    assert got.logprob.shape == rows and got.top_ids.shape == rows + (4,)


@gpu
def test_a_single_row_without_batch_and_an_empty_batch():
    x, ids = _logits((1,), 999, torch.bfloat16, 2)
    a = S.token_logprobs(x[0], ids[0], top_n=3)
    b = S.token_logprobs(x, ids, top_n=3)
    assert a.logprob.shape == () and torch.equal(a.logprob, b.logprob[0])
    assert torch.equal(a.top_ids, b.top_ids[0])
    e = S.token_logprobs(x[:0], ids[:0], top_n=3)
    assert e.logprob.shape == (0,) and e.top_ids.shape == (0, 3)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_strides_and_alignments(dt):
    """Rows at every offset within 16 bytes, verify-shaped slices, a strided id tensor."""
    g = torch.Generator(device=DEV).manual_seed(3)
    wide = (torch.randn(4, 6, 9013, generator=g, device=DEV) * 3).to(dt)
    for off in (0, 1, 3, 5):
        x = wide[:, 1:5, off:off + 8999]
        ids = torch.randint(0, 8999, (4, 8), generator=g, device=DEV)[:, ::2]
        _check(x, ids, 1.0, 6)
    _check(wide[:, 0, :9013], torch.zeros(4, dtype=torch.int32, device=DEV), 1.0, 2)
    row = wide[0, 0].expand(3, 9013)                       # one row, three times
    _check(row, torch.tensor([0, 9012, 77], device=DEV), 1.0, 2)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_entries(dt):
    """-inf and the type's lowest value as masks, most of the vocabulary masked."""
    x, ids = _logits((6,), 40000, dt, 4)
    x[0, 5:] = -math.inf
    x[1, :39990] = -math.inf
    x[2, ::2] = torch.finfo(dt).min
    x[3, 1:] = torch.finfo(dt).min
    x[4, 100:30000] = -math.inf
    ids[0], ids[1], ids[2], ids[3], ids[4] = 3, 39999, 4, 0, 200
    got = _check(x, ids, 0.7, 32)
    assert float(got.logprob[4]) == -math.inf
    # one live entry: its exponent is fma(m, c, -R) with R = m c rounded, |m c| u at
    # most, and the sum rounds to 1; never above 0
    near = float(x[3, 0].abs()) / 0.7 * U
    assert -near <= float(got.logprob[3]) <= 0.0 <= float(got.entropy[3]) <= near


@gpu
def test_rows_without_a_finite_entry_and_with_nan_or_inf():
    x, ids = _logits((5,), 20011, torch.bfloat16, 5)
    x[0] = -math.inf
    x[1, 70] = math.nan
    x[2, 9] = math.inf
    x[3, [3, 20000]] = math.nan
    ids[3] = 20000
    got = _check(x, ids, 1.0, 5)
    assert bool(got.logprob[:4].isnan().all()) and bool(got.entropy[:4].isnan().all())
    assert bool(got.logprob[4].isfinite())
    assert got.top_ids[3, :2].tolist() == [3, 20000]


@gpu
@pytest.mark.parametrize("V", [300, 40000, 151936])
def test_ties_go_to_the_lowest_id(V):
    """Flat rows (every entry equal), two-valued rows, and signed zeros."""
    x = torch.zeros(5, V, dtype=torch.bfloat16, device=DEV)
    x[1] = -2.5
    x[2, V // 2:] = 1.0
    x[3, ::3] = -0.0
    x[4, V - 40:] = 1.0
    ids = torch.tensor([V - 1, 0, V // 2 + 1, 1, 0], device=DEV)
    got = _check(x, ids, 1.0, 32)
    assert got.rank.tolist() == [V, 1, 2, 2, 41]
    assert got.top_ids[0].tolist() == list(range(32))


@gpu
def test_a_run_of_falling_logits():
    """Sorted logits: every alternative sits in one 16-byte unit."""
    V = 30000
    x = torch.linspace(12, -12, V, device=DEV).repeat(3, 1)
    x[1] = x[1].flip(0)
    x[2] = x[2].roll(V // 2)
    _check(x, torch.tensor([0, 0, 5], device=DEV), 1.0, 32)


@gpu
def test_padding_ids():
    x, _ = _logits((4,), 12000, torch.bfloat16, 6)
    ids = torch.tensor([-1, 12000, 11999, 2 ** 40], device=DEV)
    got = _check(x, ids, 1.0, 2)
    assert got.rank.tolist()[:2] == [0, 0] and got.rank.tolist()[3] == 0


@gpu
@pytest.mark.parametrize("T", [1e-3, 0.05, 30.0, 1e6])
def test_temperatures_and_offsets(T):
    """Nearly one-hot to flat; logits far from 0 (a common offset changes nothing)."""
    x, ids = _logits((4,), 20000, torch.float32, 11)
    x[1] += 5000.0
    x[2] -= 70000.0
    _check(x, ids, T, 4)
    _check(x, x.argmax(-1), T, 4)


@gpu
def test_sums_to_to_probs_and_repeats_bit_for_bit():
    x, ids = _logits((64, 5), 151936, torch.bfloat16, 7)
    a = S.token_logprobs(x, ids, temperature=0.7, top_n=20)
    p = S.to_probs(x[:2], 0.7)
    lp = S.gather_prob(p, ids[:2]).log()
    assert bool(((a.logprob[:2] - lp).abs() <= 1e-4).all())
    b = S.token_logprobs(x, ids, temperature=0.7, top_n=20)
    for u, v in zip(a, b):
        assert torch.equal(u, v)


@gpu
def test_streams_and_graphs():
    """Two streams at once, and two captured graphs replayed in turn on new inputs."""
    x, ids = _logits((48,), 60000, torch.bfloat16, 8)
    y, idy = _logits((7,), 32003, torch.bfloat16, 9)
    want_x, want_y = S.token_logprobs(x, ids, top_n=5), S.token_logprobs(y, idy, top_n=9)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(3):
        with torch.cuda.stream(s1):
            a = S.token_logprobs(x, ids, top_n=5)
        with torch.cuda.stream(s2):
            b = S.token_logprobs(y, idy, top_n=9)
        outs.append((a, b))
    torch.cuda.synchronize()
    for a, b in outs:
        assert all(torch.equal(u, v) for u, v in zip(a, want_x))
        assert all(torch.equal(u, v) for u, v in zip(b, want_y))
    bx, by = torch.zeros_like(x), torch.zeros_like(y)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        a = S.token_logprobs(bx, ids, top_n=5)
    with torch.cuda.graph(g2):
        b = S.token_logprobs(by, idy, top_n=9)
    bx.copy_(x)
    by.copy_(y)
    for _ in range(2):
        g1.replay()
        g2.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(a, want_x))
    assert all(torch.equal(u, v) for u, v in zip(b, want_y))


@gpu
def test_refusals():
    x, ids = _logits((4,), 1000, torch.bfloat16, 10)
    for bad in (dict(top_n=33), dict(top_n=-1), dict(temperature=0.0), dict(temperature=-1.0),
                dict(temperature=1e-7), dict(temperature=1e7), dict(temperature=math.inf), dict(temperature=math.nan)):
        with pytest.raises(L.SpecdecError):
            S.token_logprobs(x, ids, **bad)
    with pytest.raises(L.SpecdecError):
        S.token_logprobs(x[:, :20], ids, top_n=21)             # more alternatives than entries
    with pytest.raises(L.SpecdecError):
        S.token_logprobs(x, ids[:3])
    with pytest.raises(L.SpecdecError):
        S.token_logprobs(x, ids.float())
    with pytest.raises(L.SpecdecError):
        S.token_logprobs(x.double(), ids)
    with pytest.raises(L.SpecdecError):
        S.token_logprobs(x.t(), torch.zeros(1000, dtype=torch.long, device=DEV))
    with pytest.raises(L.SpecdecError):
        S.token_logprobs(x.cpu(), ids.cpu())


def test_refusals_on_cpu():
    with pytest.raises(L.SpecdecError):
        S.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))


def test_arguments_are_checked_before_any_launch():
    import ctypes
    lib = L.lib()
    n, d = ctypes.c_void_p(0), ctypes.c_void_p(4096)

    def call(x=d, dtype=2, ids=d, B=2, Lr=3, V=100, T=1.0, top=0, out=d, tops=n):
        return lib.sd_token_logprobs(x, 0, 0, dtype, ids, 0, B, Lr, V, T, top, out, d, d, tops, tops,
                                     n)
    assert call(B=0) == 0 and call(Lr=0) == 0                  # nothing to do
    assert call(B=-1) == -22 and call(x=n) == -22 and call(ids=n) == -22 and call(out=n) == -22
    assert call(V=0) == -22 and call(dtype=3) == -22
    assert call(T=0.0) == -22 and call(T=float("nan")) == -22 and call(T=float("inf")) == -22
    assert call(top=-1) == -22 and call(top=5) == -22          # alternatives without their outputs
    assert call(top=101, tops=d) == -22                        # more than V
    assert call(top=33, tops=d) == -95
    assert call(V=(1 << 20) + 1) == -95
    assert call(x=ctypes.c_void_p(4097)) == -22                # not aligned to its type


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [40, 700, 1024, 1500, 20000, 151936])
@pytest.mark.parametrize("T", [1e-6, 1e-5, 0.01, 1e6])
def test_large_logits_at_any_temperature(dt, V, T):
    """Products x log2(e) / T far beyond what a float32 resolves: only differences
    of logits count.  Few distinct values, so that rows have ties at the maximum."""
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randint(-3, 4, (7, V), generator=g, device=DEV).float()
    x[1] += 5000.0
    x[2] -= 5000.0
    x[3] += 65504.0 - 3.0
    x[4] = (x[4] * 16.0 - 40000.0)
    x[5] = 65504.0
    x[6, V // 2:] = -65504.0
    ids = torch.randint(0, V, (7,), generator=g, device=DEV)
    x = x.to(dt)
    _check(x, ids, T, 5)
    _check(x, x.argmax(-1), T, 0)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [40, 700, 1500, 20000, 151936])
@pytest.mark.parametrize("T", [0.7, 1.0, 1.5])
def test_finite_masks(dt, V, T):
    """Masks of every size down to the type's lowest value, over most of a row and
    over all of it; entries at both ends of the type."""
    x, ids = _logits((9,), V, dt, V)
    lo, hi = torch.finfo(dt).min, torch.finfo(dt).max
    for r, mask in enumerate((-1e4, -1e9, -1e10, -3e20, -1e30, lo)):
        x[r, 7:] = max(mask, lo)
    x[6] = lo                                                  # nothing but masks: uniform
    x[7] = hi
    x[7, ::2] = lo
    x[8, V // 3:] = max(-1e30, lo)
    x[8, V // 2:] = lo
    x[8, :V // 3] = -math.inf
    ids[:6] = 3
    got = _check(x, ids, T, 6)
    assert abs(float(got.logprob[6]) + math.log(V)) < 1e-4
    _check(x, x.argmax(-1), T, 0)


@gpu
@pytest.mark.parametrize("rows", [1, 30, 100, 150, 500])
def test_large_rows_among_others_in_parts_and_whole(rows):
    """Rows of one and of several CTAs: a part's maximum may be far above the others'."""
    V = 40000
    x, ids = _logits((rows,), V, torch.float32, rows)
    x[::3] *= 1e6
    x[0, V - 5:] = 3e38
    x[0, :V // 2] = -3e38
    _check(x, ids, 0.5, 3)


@gpu
@pytest.mark.parametrize("rows", [18, 19, 137, 138, 139, 142, 148, 149, 296, 297])
def test_rows_around_the_bounds_of_the_split(rows):
    """Eight, four and two parts, whole rows with a rest in halves."""
    x, ids = _logits((rows,), 17001, torch.bfloat16, rows)
    _check(x, ids, 0.8, 3)
