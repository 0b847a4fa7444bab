"""Generation with trees of drafted tokens and with constrained logits, on tiny models.

Greedy speculative decoding gives the tokens of greedy autoregressive decoding whatever
the drafts are, so trees and constraints are checked token for token; at a temperature
the tokens follow the target's distribution, which the enumerated marginals of a tiny
vocabulary check.  Tiny fp32 models take the CUDA-core attention, the bf16 pair of
head size 128 the tensor cores.
"""
import copy
import math

import numpy as np
import pytest
import torch
from transformers import Qwen3Config, Qwen3ForCausalLM

from oracle import sampling_oracle as O
from specdec.engine import SamplingConfig, SpecDecodeEngine
from specdec.kvcache import PagedRaggedCache, RaggedCache
from specdec.sampling import TokenHistory, process_logits
from specdec.tree import tree_masks, tree_of_widths
from tests.tiny_models import VOCAB, TinyTok, tiny_pair, tiny_pair_noisy

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
TREES = [(1,), (3,), (2, 2), (4, 2, 1), (1, 1, 1, 1), ()]


@pytest.fixture(scope="module")
def pair():
    return tiny_pair_noisy(noise=4.0)


def _prompts():
    torch.manual_seed(0)
    ids = torch.randint(0, VOCAB, (4, 6))
    return ids, torch.tensor([6, 5, 4, 6])


def _cut(rows, n):
    return [r[:n] for r in rows]


@pytest.mark.parametrize("tree", TREES)
@pytest.mark.parametrize("kind", ["contiguous", "paged", "eager"])
def test_greedy_trees_are_autoregressive(pair, tree, kind):
    eng = SpecDecodeEngine(*pair, TinyTok(), device=DEV, capacity=160, paged_kv=kind == "paged",
                           cuda_graphs=kind != "eager")
    ids, plen = _prompts()
    sp = SamplingConfig(temperature=0.0)
    ar, _ = eng.generate_autoregressive(ids, plen, 24, sampling=sp)
    out, st = eng.generate(ids, plen, 24, sampling=sp, tree=tree)
    assert _cut(out, 24) == _cut(ar, 24)
    assert st.rounds > 0 and st.k_history[0] == len(tree)
    if tree:
        assert 0 < st.alpha_conditional < 1


def test_wider_trees_accept_more(pair):
    """The children of a node are the draft's likeliest: a wider tree holds the narrower."""
    eng = SpecDecodeEngine(*pair, TinyTok(), device=DEV, capacity=160)
    ids, plen = _prompts()
    sp = SamplingConfig(temperature=0.0)
    rounds = [eng.generate(ids[:1], plen[:1], 24, sampling=sp, tree=t)[1].rounds
              for t in ((1, 1), (2, 1), (8, 1), (8, 8))]
    assert rounds == sorted(rounds, reverse=True) and rounds[-1] < rounds[0]


def test_several_samples_and_logprobs_on_trees(pair):
    eng = SpecDecodeEngine(*pair, TinyTok(), device=DEV, capacity=160)
    ids, plen = _prompts()
    sp = SamplingConfig(temperature=0.0)
    ar, sa = eng.generate_autoregressive(ids, plen, 16, sampling=sp, logprobs=2)
    out, st = eng.generate(ids, plen, 16, sampling=sp, tree=(3, 2), n=2, logprobs=2)
    assert len(out) == 8
    for b in range(8):
        assert out[b][:16] == ar[b // 2][:16]
        assert len(st.logprobs[b]) == len(out[b]) == len(st.top_logprobs[b])
        # two forwards of the same fp32 model, in other orders of addition
        np.testing.assert_allclose(st.logprobs[b][:16], sa.logprobs[b // 2][:16], atol=1e-4)
        assert [t[0][0] for t in st.top_logprobs[b][:16]] == out[b][:16]


def _bf16_pair():
    cfg = Qwen3Config(vocab_size=300, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                      num_attention_heads=8, num_key_value_heads=2, head_dim=128,
                      max_position_embeddings=2048, tie_word_embeddings=True)
    torch.manual_seed(2)
    target = Qwen3ForCausalLM(cfg).eval()
    draft = copy.deepcopy(target)
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        for p in draft.parameters():
            p.add_(torch.randn(p.shape, generator=g) * 0.7 * p.std().clamp_min(1e-3))
    return target.to(DEV, torch.bfloat16), draft.to(DEV, torch.bfloat16)


@pytest.mark.parametrize("paged", [False, True])
def test_tree_forward_matches_chains_on_tensor_cores(paged):
    """Every node's hidden state is that of a chain forward over its path (bf16, heads of
    128, a prompt of several pages): the differences are those of two orders of
    accumulation, held to a tenth of the spread between different nodes."""
    target, _ = _bf16_pair()
    eng = SpecDecodeEngine(target, target, TinyTok(), device=DEV, capacity=512)
    parents, _ = tree_of_widths((3, 2, 1))
    N = len(parents)
    masks, depths = tree_masks(parents, device=DEV)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 300, (2, 250), generator=g).to(DEV)
    plen = torch.tensor([250, 130], device=DEV)
    tok = torch.randint(0, 300, (2, N), generator=g).to(DEV)

    def fresh():
        c = PagedRaggedCache(2, 2, 512, DEV) if paged else RaggedCache(2, 2, 512, DEV, attn_impl="specdec_b200")
        eng._prefill(target, c, ids, plen)
        if paged:
            c.reserve(N)
        return c
    with torch.inference_mode():
        c = fresh()
        c.set_tree(masks, depths)
        got = eng._forward(target, c, tok).float()
        for leaf in range(N):
            path = [leaf]
            while parents[path[0]] >= 0:
                path.insert(0, parents[path[0]])
            c = fresh()
            want = eng._forward(target, c, tok[:, path]).float()[:, -1]
            near = (got[:, leaf] - want).norm(dim=-1)
            far = (got[:, leaf].unsqueeze(1) - got).norm(dim=-1)
            far = torch.where(torch.arange(N, device=DEV) == leaf, math.inf, far).amin(-1)
            assert bool((near < 0.1 * far).all()), (leaf, near / far)


def test_tree_decoding_on_tensor_cores():
    """bf16 heads of 128: two accumulation orders may part greedy rows where two logits are
    next to each other, so each emitted token is held to be within rounding of the best."""
    target, draft = _bf16_pair()
    eng = SpecDecodeEngine(target, draft, TinyTok(), device=DEV, capacity=640, paged_kv=True)
    g = torch.Generator().manual_seed(5)
    ids, plen = torch.randint(0, 300, (3, 200), generator=g), torch.tensor([200, 128, 37])
    out, st = eng.generate(ids, plen, 20, sampling=SamplingConfig(temperature=0.0), tree=(4, 2, 2))
    assert st.accepted > 0
    with torch.inference_mode():
        for b in range(3):
            seq = torch.cat([ids[b, :plen[b]], torch.tensor(out[b][:20])]).to(DEV).view(1, -1)
            lg = target(input_ids=seq).logits[0].float()
            for j, t in enumerate(out[b][:20]):
                row = lg[int(plen[b]) - 1 + j]
                # bf16 logits (half a step each way) from hidden states of two bf16 forwards
                assert float(row.max() - row[t]) <= 8 * 2.0 ** -8 * float(row.abs().max()), (b, j)


@torch.inference_mode()
@pytest.mark.parametrize("tree,constrained", [((3, 2), False), ((2,), True)])
def test_tree_sampling_is_lossless(tree, constrained):
    """The second token's histogram against the enumerated marginal (total variation 0.02, as
    for chains: 81920 draws of 16 tokens leave about sqrt(16 / (2 pi 81920)) = 0.006)."""
    target, draft = tiny_pair()
    eng = SpecDecodeEngine(target, draft, TinyTok(), device=DEV, capacity=64)
    kw = dict(repetition_penalty=1.4, frequency_penalty=0.3, presence_penalty=0.2,
              logit_bias={3: 0.5}, allowed_tokens=list(range(1, VOCAB))) if constrained else {}
    sp = SamplingConfig(temperature=1.0, top_p=0.9, **kw)
    torch.manual_seed(0)
    prompt = torch.randint(0, VOCAB, (1, 5))

    def probs(written):
        seq = torch.cat([prompt[0], torch.tensor(written, dtype=torch.long)]).view(1, -1).to(DEV)
        x = target(input_ids=seq).logits[0, -1].float().cpu().double()
        if constrained:
            c = torch.bincount(torch.tensor(written, dtype=torch.long), minlength=VOCAB)
            seen = (c > 0) | (torch.bincount(prompt[0], minlength=VOCAB) > 0)
            x = torch.where(seen, torch.where(x > 0, x / 1.4, x * 1.4), x)
            x = x - 0.3 * c - 0.2 * (c > 0)
            x[3] += 0.5
            x[0] = -math.inf
        return O.to_probs_row(x.float().numpy(), 1.0, 0.9)
    p0 = probs([])
    marg = sum(p0[t] * probs([t]) for t in range(VOCAB) if p0[t] > 0)
    B = 2048
    ids, plen = prompt.expand(B, -1).contiguous(), torch.full((B,), 5, dtype=torch.long)
    first, second = [], []
    for r in range(40):
        out, _ = eng.generate(ids, plen, max_new_tokens=2, sampling=sp, tree=tree, seed=r)
        first += [o[0] for o in out]
        second += [o[1] for o in out]
    tv = [0.5 * np.abs(np.bincount(t, minlength=VOCAB) / len(t) - p).sum()
          for t, p in ((first, p0), (second, marg))]
    assert max(tv) < 0.02, tv


CONSTRAINTS = [dict(repetition_penalty=1.5), dict(frequency_penalty=0.7, presence_penalty=0.4),
               dict(repetition_penalty=0.8, frequency_penalty=-0.2, logit_bias={2: 1.0, 5: -100.0},
                    allowed_tokens=[1, 2, 3, 5, 8, 9, 12]),
               dict(logit_bias={7: 2.0}), dict(allowed_tokens=[4, 6])]


@pytest.mark.parametrize("kw", CONSTRAINTS)
@pytest.mark.parametrize("cuda_graphs", [True, False])
def test_constraints_hold_for_chains_trees_and_no_drafts(pair, kw, cuda_graphs):
    """Speculation changes nothing: chains and trees give what one token at a time gives, and
    that is the plain formula applied to the target's logits."""
    target, _ = pair
    eng = SpecDecodeEngine(*pair, TinyTok(), device=DEV, capacity=160, cuda_graphs=cuda_graphs)
    ids, plen = _prompts()
    sp = SamplingConfig(temperature=0.0, **kw)
    ar, _ = eng.generate_autoregressive(ids, plen, 20, sampling=sp)
    for how in (dict(k_fixed=1), dict(k_fixed=4), dict(tree=(2, 2, 1))):
        out, _ = eng.generate(ids, plen, 20, sampling=sp, **how)
        assert _cut(out, 20) == _cut(ar, 20), how
    # (beside: the engine is not left constrained)
    none = SamplingConfig(temperature=0.0)
    free, _ = eng.generate(ids, plen, 20, sampling=none, k_fixed=4)
    assert _cut(free, 20) == _cut(eng.generate_autoregressive(ids, plen, 20, sampling=none)[0], 20)
    if "allowed_tokens" in kw:
        assert all(t in kw["allowed_tokens"] for row in ar for t in row)
    with torch.inference_mode():
        b, written = 1, ar[1][:20]
        seq = torch.cat([ids[b, :plen[b]], torch.tensor(written)]).to(DEV).view(1, -1)
        lg = target(input_ids=seq).logits[:, int(plen[b]) - 1:-1]
        h = TokenHistory(1, VOCAB, DEV)
        h.add_prompt(ids[b:b + 1, :plen[b]].to(DEV))
        for j, t in enumerate(written):
            x = lg[0, j].double().cpu()
            c = torch.bincount(torch.tensor(written[:j], dtype=torch.long), minlength=VOCAB)
            seen = (c > 0) | (torch.bincount(ids[b, :plen[b]], minlength=VOCAB) > 0)
            r = kw.get("repetition_penalty", 1.0)
            x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
            x = x - kw.get("frequency_penalty", 0.0) * c - kw.get("presence_penalty", 0.0) * (c > 0)
            for tok, v in kw.get("logit_bias", {}).items():
                x[tok] += v
            if "allowed_tokens" in kw:
                x[[i for i in range(VOCAB) if i not in kw["allowed_tokens"]]] = -math.inf
            # fp32 forwards of other shapes: within 1e-4 of the best
            assert float(x.max() - x[t]) < 1e-4


def test_several_samples_with_penalties(pair):
    eng = SpecDecodeEngine(*pair, TinyTok(), device=DEV, capacity=160)
    ids, plen = _prompts()
    sp = SamplingConfig(temperature=0.0, repetition_penalty=1.5, frequency_penalty=0.4)
    ar, _ = eng.generate_autoregressive(ids, plen, 16, sampling=sp)
    for how in (dict(k_fixed=3), dict(tree=(2, 1))):
        out, _ = eng.generate(ids, plen, 16, sampling=sp, n=2, **how)
        assert all(out[b][:16] == ar[b // 2][:16] for b in range(8)), how


@pytest.mark.parametrize("paged", [False, True])
def test_rows_that_are_done_do_not_grow_and_the_capacity_is_enough(pair, paged):
    """A row that ends after a few tokens waits for the others with the length it has, and the
    smallest capacity that is not refused gives the same tokens."""
    ids, plen = _prompts()
    sp, tree, new = SamplingConfig(temperature=0.0), (3, 2), 40
    nodes = len(tree_of_widths(tree)[0])
    need = int(plen.max()) + new + len(tree) + nodes
    eng = SpecDecodeEngine(*pair, TinyTok(), device=DEV, capacity=need, paged_kv=paged)
    free, _ = eng.generate(ids, plen, new, sampling=sp, tree=tree)
    caches = []
    make = eng._mk_cache
    eng._mk_cache = lambda *a, **k: caches.append(make(*a, **k)) or caches[-1]
    eng.eos_ids = {free[0][3]}
    out, st = eng.generate(ids, plen, new, sampling=sp, tree=tree)
    for b in range(4):
        cut = next((i + 1 for i, t in enumerate(free[b][:new]) if t in eng.eos_ids), new)
        assert out[b][:cut] == free[b][:cut] and len(out[b]) == cut
        for c in caches:
            assert int(c.lengths[b]) <= int(plen[b]) + cut + len(tree)
    assert len(out[0]) <= 4 and st.rounds > 4
    small = SpecDecodeEngine(*pair, TinyTok(), device=DEV, capacity=need - 1, paged_kv=paged)
    with pytest.raises(ValueError, match="capacity"):
        small.generate(ids, plen, new, sampling=sp, tree=tree)


def test_refusals(pair):
    eng = SpecDecodeEngine(*pair, TinyTok(), device=DEV, capacity=160)
    ids, plen = _prompts()
    for kw in (dict(tree=(2,), k_fixed=3), dict(tree=(0,)), dict(tree=(VOCAB + 1,)),
               dict(tree=(16, 16)), dict(tree=(2, -1))):
        with pytest.raises(ValueError):
            eng.generate(ids, plen, 8, **kw)
    for bad in (dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0),
                dict(repetition_penalty=math.inf), dict(allowed_tokens=[]),
                dict(allowed_tokens=[VOCAB]), dict(logit_bias={i: 1.0 for i in range(2000)}),
                dict(logit_bias={VOCAB: 1.0}), dict(logit_bias={-1: 1.0})):
        with pytest.raises(ValueError):
            eng.generate(ids, plen, 8, sampling=SamplingConfig(**bad), k_fixed=2)
    with pytest.raises(Exception):
        process_logits(torch.zeros(1, 1, 4, device=DEV), repetition=1.0)


@pytest.mark.parametrize("cuda_graphs", [True, False])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_constraints_with_a_draft_head_of_another_type(cuda_graphs, temperature):
    """A draft head that gives float32 logits of a bf16 model: the draft's logits end in bf16,
    rounded once from the same float32 values, so the tokens are those of its own head."""
    target, draft = _bf16_pair()
    g = torch.Generator().manual_seed(6)
    ids, plen = torch.randint(0, 300, (3, 40), generator=g), torch.tensor([40, 12, 33])
    for kw in ({}, dict(repetition_penalty=1.2, frequency_penalty=0.1, logit_bias={5: 1.0})):
        sp = SamplingConfig(temperature=temperature, **kw)
        runs = []
        for head in (None, lambda hidden, tokens: draft.lm_head(hidden).float()):
            draft.specdec_head = head
            eng = SpecDecodeEngine(target, draft, TinyTok(), device=DEV, capacity=256,
                                   cuda_graphs=cuda_graphs)
            runs.append(eng.generate(ids, plen, 12, sampling=sp, k_fixed=3, seed=1)[0])
        assert runs[0] == runs[1]
