"""Several samples per prompt: the device page table, the forked cache, the
shared-prefix attention and the token log-probabilities together.

Cache comparisons are exact.  fp32 tiny models attend row by row whether rows
share or not, with the same float32 sums in another order (some 1e-6 of scale), so
their greedy tokens are equal, too, unless two logits are that close.  The
log-probability comparisons are between two fp32 forwards of the same 2-layer
model (other batch sizes, or the engine's and a plain teacher-forced one): float32 rounding through
about 10 dependent matrix products of widths up to 64 and logits of order 1 is
within 10 * 64 * 2^-24 * 4 = 1.6e-4 of scale; 1e-3 is asserted.
"""
import copy

import pytest
import torch
from transformers import Qwen3Config, Qwen3ForCausalLM

from specdec import _lib as L
from specdec import attention as A
from specdec.engine import SamplingConfig, SpecDecodeEngine
from specdec.kvcache import PAGE, DevicePageTable, PagedRaggedCache, PageTable
from tests.tiny_models import VOCAB, TinyTok, tiny_pair_noisy

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def _filled(lens, n_pages, H=2, D=128, layers=2, seed=0):
    """A device-paged cache with `lens` random tokens per row."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, P = len(lens), max(lens)
    c = PagedRaggedCache(layers, B, 1024, DEV, n_pages=n_pages, device_pages=True)
    c.reserve_prefill(P, torch.tensor(lens))
    kv = [(torch.randn(B, H, P, D, generator=g, device=DEV).bfloat16(),
           torch.randn(B, H, P, D, generator=g, device=DEV).bfloat16()) for _ in range(layers)]
    for lay, (k, v) in zip(c.layers, kv):
        lay.update(k, v)
    c.set_lengths(torch.tensor(lens))
    c.check_errors()
    return c, kv


def test_device_pages_prefill_like_the_host_tables():
    lens = [5, 300, 128, 257]
    c, kv = _filled(lens, 40)
    h = PagedRaggedCache(2, 4, 1024, DEV, n_pages=40)
    h.reserve_prefill(300, torch.tensor(lens))
    for lay, (k, v) in zip(h.layers, kv):
        lay.update(k, v)
    h.set_lengths(torch.tensor(lens))
    assert torch.equal(c.block_table, h.block_table)
    for a, b in zip(c.layers, h.layers):
        assert torch.equal(a.keys[:39], b.keys[:39]) and torch.equal(a.values[:39], b.values[:39])
    for _ in range(30):
        for x in (c, h):
            x.reserve(9)
            x.layers[0].update(kv[0][0][:, :, :9], kv[0][1][:, :, :9])
            x.advance(9)
        assert torch.equal(c.block_table, h.block_table)
    c.check_errors()
    assert c.free_pages == h.free_pages
    c.release([1, 3])
    h.release([1, 3])
    assert c.free_pages == h.free_pages and c.lengths.tolist() == h.lengths.tolist()
    c.reset()
    assert c.free_pages == 39 and bool((c.block_table == -1).all())


def test_fork_shares_full_pages_and_copies_the_last():
    lens = [5, 300, 128, 257]
    c, kv = _filled(lens, 60)
    want = [[A.gather_pages(p, c.block_table, 512).clone() for p in (l.keys, l.values)]
            for l in c.layers]
    old = c.block_table.clone()
    free = c.free_pages
    f = c.fork([3, 1, 2, 4])
    src = [0] * 3 + [1] + [2] * 2 + [3] * 4
    assert f.lengths.tolist() == [lens[s] for s in src]
    assert f.prefix[0].tolist() == [0, 4, 6] + [10] * 7      # rows that share nothing in one group
    assert f.prefix[1].tolist() == [0, 1, 2] + [0] * 6
    for l, w in zip(f.layers, want):
        for pool, ww in zip((l.keys, l.values), w):
            got = A.gather_pages(pool, f.block_table, 512)
            for b, s in enumerate(src):
                assert torch.equal(got[b, :, :lens[s]], ww[s, :, :lens[s]])
    bt = f.block_table.tolist()
    for b, s in enumerate(src):
        full = lens[s] // PAGE
        assert bt[b][:full] == old[s, :full].tolist()
    private = [p for b, s in enumerate(src) for p in bt[b][lens[s] // PAGE:] if p >= 0]
    assert len(set(private)) == len(private) == 3 + 1 + 4      # rows of 5, 300 and 257 tokens
    assert f.free_pages == free + 3 - 8                        # three copied-from pages came back
    assert bool((c.block_table == -1).all()) and c.lengths.tolist() == [0] * 4
    # a row's own tokens do not reach its neighbours
    f.reserve(7)
    k = torch.randn(10, 2, 7, 128, device=DEV).bfloat16()
    f.layers[0].update(k, k)
    f.advance(7)
    f.check_errors()
    got = A.gather_pages(f.layers[0].keys, f.block_table, 512)
    for b, s in enumerate(src):
        assert torch.equal(got[b, :, :lens[s]], want[0][0][s, :, :lens[s]])
        assert torch.equal(got[b, :, lens[s]:lens[s] + 7], k[b])
    f.release([0, 9])
    assert f.pages.owned[[0, 9]].tolist() == [0, 0] and f.lengths[[0, 9]].tolist() == [0, 0]
    f.reset()
    assert f.free_pages == 59


def test_forked_rows_attend_like_unforked_ones():
    """The shared-prefix attention on a fork against the plain one on the same table."""
    c, _ = _filled([260, 5, 700], 80, H=2)
    f = c.fork([6, 3, 8])
    f.reserve(4)
    k = torch.randn(17, 2, 4, 128, device=DEV).bfloat16()
    f.layers[0].update(k, k)
    _same_attention(f, 4, 1)


def _same_attention(f, qlen, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B = f.batch_size
    q = torch.randn(B, 8, qlen, 128, generator=g, device=DEV).bfloat16()
    k, v = f.layers[0].keys, f.layers[0].values
    got = A.prefix_attention(q, k, v, f.lengths, f.block_table, *f.prefix).float()
    want = A.verify_attention(q, k, v, f.lengths, block_table=f.block_table).float()
    mag = A.verify_attention(q, k, v.abs(), f.lengths, block_table=f.block_table).float()
    # weights and results are rounded to bf16 on both sides: 4 * 2^-8 of sum w |v|
    assert bool(((got - want).abs() <= 2.0 ** -6 * mag * 1.02).all())


def test_released_rows_of_a_fork_leave_their_group():
    """A released row (the group's first too) that grows again holds other
    pages and other keys than the group it was in."""
    c, _ = _filled([260, 300], 80, H=2)
    f = c.fork([6, 4])
    held = f.prefix[0].data_ptr(), f.prefix[1].data_ptr()
    f.release([0, 3, 9])
    # six runs for five places: one of the two least savings is given up
    assert f.prefix[0].tolist() == [0, 4, 6, 9, 10, 10]
    assert f.prefix[1].tolist() == [0, 2, 2, 0, 0]
    with pytest.raises(L.SpecdecError):
        f.release([10])
    with pytest.raises(L.SpecdecError):
        f.release([-1])
    assert held == (f.prefix[0].data_ptr(), f.prefix[1].data_ptr())
    g = torch.Generator(device=DEV).manual_seed(3)
    for _ in range(3):                                 # past the 256 tokens that the others share
        f.reserve(100)
        k = torch.randn(10, 2, 100, 128, generator=g, device=DEV).bfloat16()
        f.layers[0].update(k, k)
        f.advance(100)
    f.reserve(4)
    k = torch.randn(10, 2, 4, 128, generator=g, device=DEV).bfloat16()
    f.layers[0].update(k, k)
    f.check_errors()
    _same_attention(f, 4, 5)
    f.release(range(10))
    assert f.prefix[1].tolist() == [0] * 5 and f.pages.owned.tolist() == [0] * 10


def test_a_forked_row_does_not_grow_inside_its_shared_pages():
    c, _ = _filled([260, 300], 80, H=2)
    f = c.fork([2, 2])
    f.rollback([0, 5, 0, 44])                          # rows of 260, 255, 300 and 256 tokens
    owned, free = f.pages.owned.clone(), f.free_pages
    f.reserve(200)
    assert torch.equal(f.pages.owned, owned) and f.free_pages == free
    with pytest.raises(RuntimeError, match="shares"):
        f.check_errors()
    f.reserve(0)                                       # nothing is written
    f.set_lengths(torch.tensor([260, 256, 300, 256]))
    f.reserve(200)
    f.check_errors()


def test_fork_refusals():
    c, _ = _filled([5, 300], 8)                                # 4 pages used, 3 left
    with pytest.raises(L.SpecdecError):
        c.fork([1])
    with pytest.raises(L.SpecdecError):
        c.fork([1, 0])
    bt, free = c.block_table.clone(), c.free_pages
    with pytest.raises(L.SpecdecError):
        c.fork([2, 2])                                         # four private pages wanted
    assert torch.equal(c.block_table, bt) and c.free_pages == free
    f = c.fork([1, 2])
    assert f.lengths.tolist() == [5, 300, 300]
    h = PagedRaggedCache(1, 2, 256, DEV)
    with pytest.raises(L.SpecdecError):
        h.fork([1, 1])


@pytest.fixture(scope="module")
def engine():
    target, draft = tiny_pair_noisy(noise=4.0)
    return SpecDecodeEngine(target, draft, TinyTok(), device=DEV, capacity=512)


def _prompts(P=150):
    torch.manual_seed(0)
    return torch.randint(0, VOCAB, (3, P)), torch.tensor([P, 7, P - 20])


@pytest.mark.parametrize("k", [1, 4])
def test_greedy_samples_equal_the_single_one(engine, k):
    ids, plen = _prompts()
    sp = SamplingConfig(temperature=0.0)
    one, st1 = engine.generate(ids, plen, 40, sampling=sp, k_fixed=k, logprobs=2)
    out, st = engine.generate(ids, plen, 40, sampling=sp, k_fixed=k, n=3, logprobs=2)
    assert len(out) == 9 and st.batch == 9
    for b in range(9):
        m = min(len(out[b]), len(one[b // 3]))
        assert m >= 40 and out[b][:40] == one[b // 3][:40]
        # the projections' GEMMs run on 9 rows here and on 3 there, in another
        # order of float32 sums: two forwards of the module's bound (sorted
        # alternatives move by no more than their values)
        for x, y in zip(st.logprobs[b][:40], st1.logprobs[b // 3][:40]):
            assert abs(x - y) < 1e-3
        for x, y in zip(st.top_logprobs[b][:40], st1.top_logprobs[b // 3][:40]):
            assert all(abs(p - q) < 1e-3 for (_, p), (_, q) in zip(x, y))


def _teacher_logprobs(model, prompt, tokens):
    """log softmax of a plain forward at the tokens' positions (eager attention)."""
    m = copy.deepcopy(model)
    from specdec import fused_attention as FA
    from specdec import fused_layers as FL
    FA.uninstall(m)
    FL.uninstall(m)
    m.set_attn_implementation("eager")
    seq = torch.tensor([prompt + tokens], device=DEV)
    with torch.no_grad():
        lp = torch.log_softmax(m(input_ids=seq).logits[0].double(), -1)
    at = torch.arange(len(prompt) - 1, len(prompt) + len(tokens) - 1, device=DEV)
    return lp[at]


@pytest.mark.parametrize("T", [0.0, 1.0])
def test_logprobs_of_the_emitted_tokens(engine, T):
    ids, plen = _prompts(40)
    out, st = engine.generate(ids, plen, 30, sampling=SamplingConfig(temperature=T, top_p=0.9),
                              k_fixed=3, n=2, seed=5, logprobs=3)
    for b, toks in enumerate(out):
        assert len(st.logprobs[b]) == len(toks) == len(st.top_logprobs[b])
        prompt = ids[b // 2, :int(plen[b // 2])].tolist()
        lp = _teacher_logprobs(engine.target, prompt, toks)
        want = lp[torch.arange(len(toks)), torch.tensor(toks, device=DEV)]
        got = torch.tensor(st.logprobs[b], device=DEV).double()
        assert bool(((got - want).abs() < 1e-3).all())
        for alts, row in zip(st.top_logprobs[b], lp):
            assert len(alts) == 3 and all(abs(p - float(row[i])) < 1e-3 for i, p in alts)
            assert alts[0][1] >= alts[1][1] >= alts[2][1]
    if T == 0.0:
        assert all(a[0][0] == t for b in range(6) for a, t in zip(st.top_logprobs[b], out[b]))


def test_samples_differ_and_repeat_for_a_seed(engine):
    ids, plen = _prompts(30)
    sp = SamplingConfig(temperature=1.0)
    a, _ = engine.generate(ids, plen, 24, sampling=sp, k_fixed=3, n=4, seed=11)
    b, _ = engine.generate(ids, plen, 24, sampling=sp, k_fixed=3, n=4, seed=11)
    assert a == b
    assert len({tuple(x) for x in a[:4]}) > 1
    ar, st = engine.generate_autoregressive(ids, plen, 8, sampling=SamplingConfig(), logprobs=0)
    assert [len(x) for x in st.logprobs] == [len(x) for x in ar] and st.top_logprobs == []


def _bf16_pair():
    cfg = Qwen3Config(vocab_size=VOCAB, hidden_size=64, intermediate_size=128, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                      max_position_embeddings=1024, tie_word_embeddings=True)
    torch.manual_seed(3)
    target = Qwen3ForCausalLM(cfg).eval().to(torch.bfloat16).to(DEV)
    return target, copy.deepcopy(target)


def test_bf16_samples_share_their_prompt():
    """Heads of 128 in bf16 take the shared path (fused layers, CUDA graphs): the
    draft equals the target, so nearly every draft is accepted, and every
    log-probability is the one of its own sequence."""
    target, draft = _bf16_pair()
    eng = SpecDecodeEngine(target, draft, TinyTok(), device=DEV, capacity=1024)
    torch.manual_seed(1)
    ids = torch.randint(0, VOCAB, (2, 400))
    plen = torch.tensor([400, 290])
    out, st = eng.generate(ids, plen, 60, sampling=SamplingConfig(temperature=1.0), k_fixed=4, n=8,
                           seed=2, logprobs=1)
    assert len(out) == 16 and all(len(x) >= 60 for x in out)
    assert st.acceptance_rate > 0.9
    for b in (0, 7, 8, 15):
        prompt = ids[b // 8, :int(plen[b // 8])].tolist()
        lp = _teacher_logprobs(eng.target, prompt, out[b])
        want = lp[torch.arange(len(out[b])), torch.tensor(out[b], device=DEV)]
        got = torch.tensor(st.logprobs[b], device=DEV).double()
        # bf16 logits of order 1 (2^-8 each), activations rounded a dozen times
        assert bool(((got - want).abs() < 0.1).all())


def test_a_pool_that_runs_out_raises(engine):
    ids, plen = _prompts(30)
    small = SpecDecodeEngine(engine.target, engine.draft, TinyTok(), device=DEV, capacity=512,
                             kv_pages=3 + 6 + 1)
    with pytest.raises(L.SpecdecError):
        small.generate(ids, plen, 200, sampling=SamplingConfig(), k_fixed=3, n=2)


def test_bad_arguments(engine):
    ids, plen = _prompts(10)
    for bad in (dict(n=0), dict(logprobs=-1), dict(logprobs=VOCAB + 1)):
        with pytest.raises(ValueError):
            engine.generate(ids, plen, 4, **bad)


def test_rows_without_their_pages_do_not_fork(engine):
    """A prefill that found too few pages: nothing went to the sink for it, and the
    fork raises, also when somebody has read the flag in between."""
    lens = [700, 5]
    c = PagedRaggedCache(1, 2, 1024, DEV, n_pages=6, device_pages=True)
    c.reserve_prefill(700, torch.tensor(lens))                 # seven pages wanted, five free
    assert c.block_table[0, :6].tolist() == [-1] * 6 and c.block_table[1, 0] == -1
    assert c.block_table[1, 1:6].tolist() == [c.pages.sink] * 5
    k = torch.randn(2, 2, 700, 128, device=DEV).bfloat16()
    c.layers[0].update(k, k)
    c.set_lengths(torch.tensor(lens))
    assert int(c._err) & 6 == 6                                # no pages, slots without one
    with pytest.raises(L.SpecdecError, match="exhausted"):
        c.fork([2, 1])
    with pytest.raises(L.SpecdecError, match="without a page"):
        c.fork([2, 1])
    assert c.free_pages == 5 and bool((c.block_table == -1).all())
    # the same from the engine: two pages are enough for the samples' own tokens,
    # not for the prompt's 384
    small = SpecDecodeEngine(engine.target, engine.draft, TinyTok(), device=DEV, capacity=512,
                             kv_pages=3)
    torch.manual_seed(0)
    ids = torch.randint(0, VOCAB, (1, 384))
    with pytest.raises(L.SpecdecError, match="exhausted"):
        small.generate(ids, torch.tensor([384]), 8, sampling=SamplingConfig(), k_fixed=3, n=2)


def test_a_row_rolled_back_into_its_shared_pages_does_not_fork():
    """Its neighbours still read those pages: they are not its to give or to split."""
    c, _ = _filled([300, 5], 40, H=2)
    f = c.fork([2, 1])
    f.rollback([170, 0, 0])                                    # rows of 130, 300 and 5 tokens
    bt, free, owned = f.block_table.clone(), f.free_pages, f.pages.owned.clone()
    with pytest.raises(L.SpecdecError, match="shares"):
        f.fork([1, 1, 1])
    assert torch.equal(f.block_table, bt) and f.free_pages == free
    assert torch.equal(f.pages.owned, owned) and f.lengths.tolist() == [130, 300, 5]
    f.release([0])                                             # a row without tokens may
    h = f.fork([1, 2, 1])
    used = [p for p in h.block_table.flatten().tolist() if p >= 0]
    assert len(set(used)) == 2 + 2 + 1 and h.free_pages == 39 - 5


@pytest.mark.parametrize("order", [[range(7)], [[0], [1, 2], [3], [4, 5, 6]], [[6], [5, 0, 2], [4, 1], [3]],
                                   [[3, 3], [0, 1, 2, 0], [5, 4], [6, 6, 6]]])
def test_the_last_row_of_a_prompt_gives_its_pages_back(order):
    c, _ = _filled([260, 5, 700], 30, H=2)                     # 2, 0 and 5 shared pages
    f = c.fork([3, 1, 3])
    f.reserve(200)
    f.check_errors()
    left = set(range(7))
    for rows in order:
        held = set(f.block_table[sorted(left)].flatten().tolist()) - {-1}
        f.release(rows)
        left -= set(rows)
        now = set(f.block_table[sorted(left)].flatten().tolist()) - {-1}
        assert now <= held and f.free_pages == 29 - len(now)
        assert not now & set(f.pages.free[:f.free_pages].tolist())
        f.release(rows)                                        # a second time: nothing to give
        assert f.free_pages == 29 - len(now)
    assert f.free_pages == 29 and sorted(f.pages.free[:29].tolist()) == list(range(29))
    # every page is handed out once again
    f.reserve(4 * PAGE)
    f.check_errors()
    got = f.block_table[:, :4].flatten().tolist()
    assert len(set(got)) == 28 and -1 not in got


def test_pages_of_a_fork_of_a_fork_come_back_once():
    c, _ = _filled([260, 300], 60, H=2)
    f = c.fork([2, 1])
    f.reserve(300)
    k = torch.randn(3, 2, 300, 128, device=DEV).bfloat16()
    f.layers[0].update(k, k)
    f.advance(300)                                             # rows of 560, 560 and 600 tokens
    h = f.fork([2, 3, 1])                                      # rows 0 to 4 hold the first two pages
    h.check_errors()
    h.reserve(100)
    free = [h.free_pages]
    for rows in ([1], [0], [2, 4], [3], [5]):
        h.release(rows)
        free.append(h.free_pages)
        used = set(h.block_table.flatten().tolist()) - {-1}
        assert free[-1] == 59 - len(used) and not used & set(h.pages.free[:free[-1]].tolist())
    # own page(s) of 560 + 100 tokens past four shared ones: 2; a source row's own two
    # full pages leave with its last reader, the prompt's two with the last of all
    assert [b - a for a, b in zip(free, free[1:])] == [2, 4, 4, 6, 6]


def test_rows_released_before_a_fork_leave_their_pages_to_the_others():
    c, _ = _filled([300, 5], 40, H=2)
    f = c.fork([2, 1])
    f.release([0])
    h = f.fork([1, 2, 1])
    h.release([0, 3, 1])
    assert h.free_pages == 39 - 3                              # row 2 still reads the prompt
    h.release([2])
    assert h.free_pages == 39
