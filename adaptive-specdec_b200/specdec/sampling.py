"""Sampling transforms and rejection sampling on B200 kernels.

Drop-in for the reference's specdec/sampling.py (to_probs, sample_from_probs,
residual_probs, gather_prob at lines 34-95), with the same names, argument
meaning and output dtypes, plus the two fused entry points the engine uses:

* ``verify_sample`` -- one launch sequence for engine.py:282-303: to_probs on
  the k+1 target and k draft vectors, the accept test, and the residual or
  bonus draw;
* ``draft_sample``  -- one draft step, engine.py:250-251 and :256;

and ``token_logprobs`` (no counterpart in the reference): log-probability, rank
and entropy for given tokens, with the largest alternatives, for callers that
rank several samples of one prompt; and ``process_logits`` with ``TokenHistory``:
penalties for repeated tokens, biases and grammar masks on the logits of a draft or
verify forward, the drafted tokens before each position counted in.

Draws are inverse-CDF with uniforms: either passed in (``u=...``) or drawn
from ``generator`` on the device.  Given the same uniforms, results match the
reference's arithmetic as restated in oracle/sampling_oracle.py.

Tie rule at the top-p boundary: among equal probabilities, lower vocabulary
index first (the reference's ``torch.sort`` is unstable, so any order is a
valid reading of it; this one is deterministic).
"""
from typing import NamedTuple, Optional

import torch

from specdec import _lib as L
from specdec.tree import TREE_MAX, check_masks

__all__ = ["to_probs", "sample_from_probs", "residual_probs", "gather_prob",
           "verify_sample", "verify_sample_probs", "draft_sample", "TokenLogprobs",
           "token_logprobs", "TokenHistory", "process_logits"]

TOP_N_MAX = 32             # SD_TOPN_MAX
LOGPROBS_MAX_V = 1 << 20   # SD_LOGPROBS_MAX_V
BIAS_MAX = 1024            # SD_BIAS_MAX


def _knobs(temperature, top_p, top_k):
    T = 0.0 if temperature is None or temperature <= 0.0 else float(temperature)
    tp = 1.0 if top_p is None else float(top_p)
    tk = 0 if not top_k else int(top_k)
    return T, tp, tk


def _rows(x):
    """View x [..., V] as [N, V] with unit stride along V."""
    V = x.shape[-1]
    x2 = x.reshape(-1, V)
    if x2.stride(-1) != 1 or (x2.shape[0] > 1 and x2.stride(0) < V):
        x2 = x2.contiguous()
    return x2


def to_probs(logits, temperature=1.0, top_p=1.0, top_k=0):
    """Logits -> float32 probabilities over the full vocabulary.

    Same contract as reference specdec/sampling.py:34-67: temperature <= 0 is a
    one-hot at the first maximum; otherwise softmax(logits / T), then top-k
    (ties at the k-th value kept), then top-p (smallest prefix of the sorted
    probabilities reaching top_p, first entry always kept), renormalised.
    """
    L.require_cuda(logits)
    T, tp, tk = _knobs(temperature, top_p, top_k)
    x = _rows(logits)
    n, V = x.shape
    out = torch.empty((n, V), dtype=torch.float32, device=x.device)
    code = L.dtype_code(x.dtype)
    lib = L.lib()
    with torch.cuda.device(x.device):
        ws = L.workspaces.get(lib.sd_sampling_workspace_bytes(n, n, V, code), x.device)
        L.check(lib.sd_to_probs(L.ptr(x), x.stride(0), code, n, V, T, tp, tk, L.ptr(out),
                                out.stride(0), L.ptr(ws), ws.numel(), L.stream_ptr(x.device)),
                "to_probs")
    return out.reshape(logits.shape)


def sample_from_probs(probs, generator=None, u=None):
    """Inverse-CDF draw per row: probs [..., V] -> ids [...] (int64).

    Replaces reference specdec/sampling.py:70-74 (torch.multinomial).  The
    uniforms are ``u`` if given, else drawn from ``generator`` on the device.
    """
    L.require_cuda(probs)
    p = _rows(probs.float())
    n, V = p.shape
    if u is None:
        u = torch.rand(n, generator=generator, device=p.device)
    u = u.reshape(-1).float().contiguous()
    out = torch.empty(n, dtype=torch.long, device=p.device)
    with torch.cuda.device(p.device):
        L.check(L.lib().sd_sample_from_probs(L.ptr(p.contiguous()), n, V, L.ptr(u), L.ptr(out),
                                             L.stream_ptr(p.device)), "sample_from_probs")
    return out.reshape(probs.shape[:-1])


def residual_probs(p, q):
    """norm((p - q)_+), p itself where that sums to <= 1e-9 (sampling.py:77-90)."""
    L.require_cuda(p, q)
    p2 = _rows(p.float()).contiguous()
    q2 = _rows(q.float()).contiguous()
    n, V = p2.shape
    out = torch.empty_like(p2)
    with torch.cuda.device(p2.device):
        L.check(L.lib().sd_residual_probs(L.ptr(p2), L.ptr(q2), n, V, L.ptr(out),
                                          L.stream_ptr(p2.device)), "residual_probs")
    return out.reshape(p.shape)


def gather_prob(probs, ids):
    """probs [..., V], ids [...] -> probs at ids (sampling.py:93-95)."""
    L.require_cuda(probs, ids)
    p2 = _rows(probs.float()).contiguous()
    i2 = ids.reshape(-1).long().contiguous()
    out = torch.empty(i2.shape[0], dtype=torch.float32, device=p2.device)
    with torch.cuda.device(p2.device):
        L.check(L.lib().sd_gather_prob(L.ptr(p2), p2.shape[0], p2.shape[1], L.ptr(i2), L.ptr(out),
                                       L.stream_ptr(p2.device)), "gather_prob")
    return out.reshape(ids.shape)


def _vocab_rows(x, name):
    if x.stride(-1) != 1:
        raise L.SpecdecError(f"{name} must be contiguous along the vocabulary")
    return x


def verify_sample(target_logits, draft_logits, draft_ids, u_acc, u_res, temperature=1.0,
                  top_p=1.0, top_k=0, alive=None, return_probs=False):
    """The fused verify round (reference engine.py:282-303).

    target_logits [B, k+1, V] (p_1..p_{k+1}), draft_logits [B, k, V] (q_1..q_k;
    ignored when temperature <= 0), draft_ids [B, k], u_acc [B, k] and u_res [B]
    float uniforms, alive [B] bool or None.  Returns (n_acc [B], y [B]) int64,
    plus (p_i(x_i), q_i(x_i)) [B, k] float32 when return_probs.
    """
    L.require_cuda(target_logits, draft_ids, u_acc, u_res)
    B, k1, V = target_logits.shape
    k = k1 - 1
    greedy = temperature is None or temperature <= 0.0
    T, tp, tk = _knobs(temperature, top_p, top_k)
    tgt = _vocab_rows(target_logits, "target_logits")
    if greedy:
        drf = None
        dbs = dps = 0
    else:
        L.require_cuda(draft_logits)
        drf = _vocab_rows(draft_logits, "draft_logits")
        if drf.shape != (B, k, V) or drf.dtype != tgt.dtype:
            raise L.SpecdecError("draft_logits must be [B, k, V] with the target's dtype")
        dbs, dps = drf.stride(0), drf.stride(1)
    xs = draft_ids.long()
    if xs.stride(-1) != 1:
        xs = xs.contiguous()
    ua = u_acc.float()
    if ua.stride(-1) != 1:
        ua = ua.contiguous()
    ur = u_res.float().contiguous()
    al = None if alive is None else alive.to(torch.uint8).contiguous()
    dev = tgt.device
    n_acc = torch.empty(B, dtype=torch.long, device=dev)
    y = torch.empty(B, dtype=torch.long, device=dev)
    px = torch.empty(B, k, dtype=torch.float32, device=dev) if return_probs else None
    qx = torch.empty(B, k, dtype=torch.float32, device=dev) if return_probs else None
    code = L.dtype_code(tgt.dtype)
    lib = L.lib()
    nvec = B * (k + 1) if greedy else B * (2 * k + 1)
    with torch.cuda.device(dev):
        ws = L.workspaces.get(lib.sd_sampling_workspace_bytes(B, nvec, V, code), dev)
        L.check(lib.sd_verify_sample(L.ptr(tgt), tgt.stride(0), tgt.stride(1), L.ptr(drf), dbs,
                                     dps, code, L.ptr(xs), xs.stride(0), L.ptr(ua), ua.stride(0),
                                     L.ptr(ur), L.ptr(al), B, k, V, T, tp, tk, L.ptr(n_acc),
                                     L.ptr(y), L.ptr(px), L.ptr(qx), L.ptr(ws), ws.numel(),
                                     L.stream_ptr(dev)), "verify_sample")
    if return_probs:
        return n_acc, y, px, qx
    return n_acc, y


def verify_sample_probs(target_logits, draft_probs, draft_ids, u_acc, u_res, temperature=1.0,
                        top_p=1.0, top_k=0, alive=None, return_probs=False):
    """The fused verify round with the draft distributions given as
    probabilities: q_i = draft_probs[:, i] (fp32 [B, k, V], used as given),
    as a serving engine's rejection sampler holds them.  Otherwise as
    ``verify_sample``: to_probs (temperature, top-p, top-k) on the target
    logits [B, k+1, V], the accept test u < min(1, p(x)/max(q(x), 1e-10)), the
    residual draw from norm((p - q)+) at the first rejection or the bonus draw
    from p_k (reference engine.py:282-303).  Returns (n_acc, y) int64, plus
    (p_i(x_i), q_i(x_i)) when return_probs.
    """
    L.require_cuda(target_logits, draft_ids, u_acc, u_res)
    B, k1, V = target_logits.shape
    k = k1 - 1
    T, tp, tk = _knobs(temperature, top_p, top_k)
    tgt = _vocab_rows(target_logits, "target_logits")
    q = None
    if T > 0.0:
        L.require_cuda(draft_probs)
        if draft_probs.shape != (B, k, V) or draft_probs.dtype != torch.float32:
            raise L.SpecdecError("draft_probs must be float32 [B, k, V]")
        q = _vocab_rows(draft_probs, "draft_probs")
    xs = draft_ids.long()
    if xs.stride(-1) != 1:
        xs = xs.contiguous()
    ua = u_acc.float()
    if ua.stride(-1) != 1:
        ua = ua.contiguous()
    ur = u_res.float().contiguous()
    al = None if alive is None else alive.to(torch.uint8).contiguous()
    dev = tgt.device
    n_acc = torch.empty(B, dtype=torch.long, device=dev)
    y = torch.empty(B, dtype=torch.long, device=dev)
    px = torch.empty(B, k, dtype=torch.float32, device=dev) if return_probs else None
    qx = torch.empty(B, k, dtype=torch.float32, device=dev) if return_probs else None
    code = L.dtype_code(tgt.dtype)
    lib = L.lib()
    with torch.cuda.device(dev):
        ws = L.workspaces.get(lib.sd_sampling_workspace_bytes(B, B * (k + 1), V, code), dev)
        L.check(lib.sd_verify_sample_qprobs(
            L.ptr(tgt), tgt.stride(0), tgt.stride(1), code, L.ptr(q),
            0 if q is None else q.stride(0), 0 if q is None else q.stride(1), L.ptr(xs),
            xs.stride(0), L.ptr(ua), ua.stride(0), L.ptr(ur), L.ptr(al), B, k, V, T, tp, tk,
            L.ptr(n_acc), L.ptr(y), L.ptr(px), L.ptr(qx), L.ptr(ws), ws.numel(),
            L.stream_ptr(dev)), "verify_sample_probs")
    if return_probs:
        return n_acc, y, px, qx
    return n_acc, y


def draft_sample(logits, u, temperature=1.0, top_p=1.0, top_k=0):
    """x ~ to_probs(logits) by inverse CDF with uniforms u; returns (x, q(x)).

    logits [B, V] (row stride free, vocabulary contiguous), u [B].
    """
    L.require_cuda(logits, u)
    x2 = _vocab_rows(logits, "logits")
    if x2.dim() != 2:
        raise L.SpecdecError("draft_sample expects [B, V] logits")
    B, V = x2.shape
    T, tp, tk = _knobs(temperature, top_p, top_k)
    uu = u.reshape(-1).float().contiguous()
    x = torch.empty(B, dtype=torch.long, device=x2.device)
    qx = torch.empty(B, dtype=torch.float32, device=x2.device)
    code = L.dtype_code(x2.dtype)
    lib = L.lib()
    with torch.cuda.device(x2.device):
        ws = L.workspaces.get(lib.sd_sampling_workspace_bytes(B, B, V, code), x2.device)
        L.check(lib.sd_draft_sample(L.ptr(x2), x2.stride(0), code, B, V, L.ptr(uu), T, tp, tk,
                                    L.ptr(x), L.ptr(qx), L.ptr(ws), ws.numel(),
                                    L.stream_ptr(x2.device)), "draft_sample")
    return x, qx


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns (shapes: those of ``ids``; top_* have one
    more dimension of top_n entries and are None without alternatives)."""
    logprob: torch.Tensor                   # float32
    rank: torch.Tensor                      # int64, 1 = the largest logit
    entropy: torch.Tensor                   # float32, natural log
    top_ids: Optional[torch.Tensor]         # int64
    top_logprobs: Optional[torch.Tensor]    # float32


def token_logprobs(logits, ids, temperature=1.0, top_n=0):
    """Log-probabilities of ``ids`` under softmax(logits / temperature).

    logits [..., V] (bf16 / fp16 / fp32, vocabulary contiguous, other strides
    free up to three dimensions), ids [...] integer, temperature in [1e-6, 1e6].  Per position: the
    token's log-probability, its rank by (logit falling, id rising; 1 = first),
    the entropy of the distribution, and with ``top_n`` > 0 the first top_n ids
    in that order with their log-probabilities.  No top-p / top-k applies.  An
    id outside [0, V) (padding) gets logprob NaN and rank 0.  A row with a NaN or
    a +inf, or with nothing above -inf, has NaN log-probabilities and entropy.
    One pass over the logits (sd_token_logprobs), no host synchronisation.
    """
    dev, shape, dims = logits.device, ids.shape, logits.dim()
    if not logits.is_cuda or ids.device != dev:
        L.require_cuda(logits, ids)
        raise L.SpecdecError("logits and ids must be on one device")
    if dims < 1 or shape != logits.shape[:-1]:
        raise L.SpecdecError(f"token_logprobs needs one id per row: logits {tuple(logits.shape)}, "
                             f"ids {tuple(shape)}")
    if ids.dtype != torch.long:
        if ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
            raise L.SpecdecError(f"ids must be integers, got {ids.dtype}")
        ids = ids.long()
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return token_logprobs(logits, ids, temperature, top_n)
    code, V, n, T = L.dtype_code(logits.dtype), logits.shape[-1], int(top_n), float(temperature)
    if not 1 <= V <= LOGPROBS_MAX_V:
        raise L.SpecdecError(f"the vocabulary must have 1 to {LOGPROBS_MAX_V} entries, got {V}")
    if not 0 <= n <= min(V, TOP_N_MAX):
        raise L.SpecdecError(f"top_n must be between 0 and min(V, {TOP_N_MAX}), got {n}")
    if not 1e-6 <= T <= 1e6:
        raise L.SpecdecError(f"temperature must be between 1e-6 and 1e6, got {temperature}")
    # rows (b, l) with strides (bs, ps), their ids with stride ids_bs over b
    if V == 1:
        logits = logits.contiguous()
    x = _vocab_rows(logits, "logits")
    if dims == 2:
        B, Lr, bs, ps, ids_bs = shape[0], 1, x.stride(0), 0, ids.stride(0)
    elif dims == 3:
        (B, Lr), (bs, ps, _) = shape, x.stride()
        if Lr > 1 and ids.stride(1) != 1:
            ids = ids.contiguous()
        ids_bs = ids.stride(0)
    else:
        x = x.reshape(-1, V)
        if x.stride(1) != 1:                       # what reshape makes of a single row or entry
            x = x.contiguous()
        ids = ids.reshape(-1)
        B, Lr, bs, ps, ids_bs = x.shape[0], 1, x.stride(0), 0, ids.stride(0)
    if dims in (2, 3) and ids.is_contiguous():
        # (empty_like costs half of an empty with a torch.Size)
        logprob = torch.empty_like(ids, dtype=torch.float32)
        rank, entropy = torch.empty_like(ids), torch.empty_like(logprob)
    else:
        logprob = torch.empty(shape, dtype=torch.float32, device=dev)
        rank = torch.empty(shape, dtype=torch.long, device=dev)
        entropy = torch.empty(shape, dtype=torch.float32, device=dev)
    top_ids = top_lp = None
    if n:
        top_ids = ids.new_empty(*shape, n)
        top_lp = torch.empty_like(top_ids, dtype=torch.float32)
    L.check(L.lib().sd_token_logprobs(
        x.data_ptr(), bs, ps, code, ids.data_ptr(), ids_bs, B, Lr, V, T, n, logprob.data_ptr(),
        rank.data_ptr(), entropy.data_ptr(), L.address(top_ids), L.address(top_lp),
        L.stream_of(dev)), "token_logprobs")
    return TokenLogprobs(logprob, rank, entropy, top_ids, top_lp)


class TokenHistory:
    """Which tokens each row's prompt holds and how often it has written each.

    ``counts`` [B, V] int16 on the device: the low 15 bits count the written
    tokens (up to 32767), the sign bit marks the prompt's.  ``process_logits`` reads
    it; ``add_prompt`` and ``append`` add to it.  Both are stream ordered, never
    synchronise and can be captured into CUDA graphs.
    """

    def __init__(self, batch_size, vocab_size, device):
        B, V = int(batch_size), int(vocab_size)
        dev = torch.device(device)
        if B < 0 or V < 1:
            raise L.SpecdecError(f"a history needs rows and a vocabulary, got {B} x {V}")
        if dev.type != "cuda":
            raise L.SpecdecError("TokenHistory keeps its counts on the GPU (no CPU fallback)")
        # (rows of whole 16-byte units)
        self._bind(torch.zeros(B, -(-V // 8) * 8, dtype=torch.int16, device=dev)[:, :V])

    def _bind(self, counts):
        self.counts, self.device = counts, counts.device
        self.B, self.V = counts.shape

    @classmethod
    def over(cls, counts):
        """A history over counts [B, V] int16 that the caller holds (no copy)."""
        if not counts.is_cuda:
            raise L.SpecdecError("TokenHistory keeps its counts on the GPU (no CPU fallback)")
        if counts.dtype != torch.int16 or counts.dim() != 2 or counts.shape[1] < 1 \
                or (counts.stride(1) != 1 and counts.shape[1] > 1) \
                or (counts.shape[0] > 1 and counts.stride(0) < counts.shape[1]):
            raise L.SpecdecError("counts must be int16 [B, V] with contiguous rows")
        self = cls.__new__(cls)
        self._bind(counts)
        return self

    def _add(self, ids, counts, path, prompt):
        dev = self.device
        if ids.device != dev or ids.dim() != 2 or ids.shape[0] != self.B:
            raise L.SpecdecError(f"ids must be [{self.B}, n] on {dev}")
        if ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
            raise L.SpecdecError(f"ids must be integers, got {ids.dtype}")
        n = ids.shape[1]
        ids = ids.long() if ids.dtype != torch.long else ids
        if ids.stride(1) != 1 and n > 1:
            ids = ids.contiguous()
        if counts is not None:
            if counts.device != dev or counts.numel() != self.B or counts.is_floating_point():
                raise L.SpecdecError(f"counts must be integers [{self.B}] on {dev}")
            counts = counts.reshape(-1).long().contiguous()
        path_bs = 0
        if path is not None:
            if path.device != dev or path.dtype != torch.int32 or path.dim() != 2 \
                    or path.shape[0] != self.B or (path.stride(1) != 1 and path.shape[1] > 1):
                raise L.SpecdecError(f"path must be int32 [{self.B}, P] on {dev}")
            path_bs = path.stride(0)
        with L.on_device(dev):
            L.check(L.lib().sd_history_add(
                self.counts.data_ptr(), self.counts.stride(0), self.V, ids.data_ptr(),
                ids.stride(0), n, L.address(path), path_bs, L.address(counts),
                n if path is None else path.shape[1], self.B, int(prompt), L.stream_of(dev)),
                "history_add")

    def add_prompt(self, ids, lengths=None):
        """Marks the first lengths[b] (default: all) of ids [B, n] as prompt tokens."""
        self._add(ids, lengths, None, True)

    def append(self, ids, counts=None, path=None):
        """Counts the first counts[b] (default: all) of ids [B, n] as written; with
        ``path`` [B, P] int32 (``tree_accept``'s) the tokens ids[b, path[b, i]], i <
        counts[b], instead.  Ids outside [0, V) are padding."""
        self._add(ids, counts, path, False)

    def repeat_interleave(self, n):
        """A history with n copies of every row, side by side."""
        return TokenHistory.over(self.counts.repeat_interleave(int(n), 0))

    def reset(self, rows=None):
        """Forgets every row, or the given ones."""
        if rows is None:
            self.counts.zero_()
        else:
            self.counts[rows] = 0


def _per_row(x, B, dev, name):
    """A float32 [B] tensor of a number or a tensor; None stays None."""
    if x is None:
        return None
    if not torch.is_tensor(x):
        return torch.full((B,), float(x), dtype=torch.float32, device=dev)
    if x.device != dev or x.numel() != B:
        raise L.SpecdecError(f"{name} must be a number or [{B}] on {dev}")
    return x if x.dtype == torch.float32 and x.is_contiguous() else x.reshape(-1).float().contiguous()


def process_logits(logits, tokens=None, masks=None, history=None, repetition=None, presence=None,
                   frequency=None, bias=None, allowed=None, out=None):
    """Penalties, biases and a grammar mask on the logits of a draft or verify forward.

    logits [B, L, V] (bf16 / fp16 / fp32, vocabulary contiguous) are those of the
    last L of N drafted tokens ``tokens`` [B, N] (N >= L): a chain, or with ``masks``
    (``tree_masks``) a tree.  Position l is node N - L + l; what stands before it is
    the row's ``history`` (a TokenHistory or its counts; without this forward's
    tokens) and the tokens of its path, itself included.  Per entry, in float32 and
    rounded once:

      c = times written + times on the path;  s = c > 0 or in the prompt
      s:      x = x / repetition if x > 0 else x * repetition
              x = x - frequency * c
      c > 0:  x = x - presence
              x = x + bias            bias = (ids [B or 1, M], values [B or 1, M])
      bit t % 32 of allowed[b, l, t // 32] is 0:  x = -inf

    ``repetition``, ``presence`` and ``frequency`` are numbers or float [B] tensors and
    need ``history``; ``allowed`` int32 [B or 1, L or 1, ceil(V / 32)].  Ids outside
    [0, V) are padding, biases of one id add up; at most BIAS_MAX per row and
    TREE_MAX tokens (made for some dozens of biases: with M of them and N tokens a
    position's time grows by (M + N)^2).  repetition > 0.  Returns a new tensor, or
    ``out`` ([B, L, V]): the logits themselves, or memory outside the span from their
    first to their last entry; anything else is refused, and so is an ``out`` whose
    rows share entries (an expanded tensor).  One launch, no synchronisation.
    """
    dev = logits.device
    if not logits.is_cuda:
        L.require_cuda(logits)
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return process_logits(logits, tokens, masks, history, repetition, presence, frequency,
                                  bias, allowed, out)
    if logits.dim() != 3:
        raise L.SpecdecError(f"process_logits expects [B, L, V] logits, got {tuple(logits.shape)}")
    code = L.dtype_code(logits.dtype)
    B, Lq, V = logits.shape
    if V < 1:
        raise L.SpecdecError("the vocabulary must have at least one entry")
    if V > 1:
        _vocab_rows(logits, "logits")
    N = first = tokens_bs = mask_bs = 0
    hist = None
    if history is not None:
        hist = history.counts if isinstance(history, TokenHistory) else \
            TokenHistory.over(history).counts
        if hist.shape != (B, V) or hist.device != dev:
            raise L.SpecdecError(f"history is {tuple(hist.shape)} on {hist.device}, the logits "
                                 f"{tuple(logits.shape)} on {dev}")
        repetition = _per_row(repetition, B, dev, "repetition")
        presence = _per_row(presence, B, dev, "presence")
        frequency = _per_row(frequency, B, dev, "frequency")
    elif repetition is not None or presence is not None or frequency is not None:
        raise L.SpecdecError("repetition, presence and frequency need a history")
    if tokens is not None:
        if tokens.device != dev or tokens.dim() != 2 or tokens.shape[0] != B or \
                tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
            raise L.SpecdecError(f"tokens must be integers [{B}, N] on {dev}")
        N = tokens.shape[1]
        if not Lq <= N <= TREE_MAX:
            raise L.SpecdecError(f"{Lq} positions of {N} drafted tokens (at most {TREE_MAX})")
        if tokens.dtype != torch.long:
            tokens = tokens.long()
        if N > 1 and tokens.stride(1) != 1:
            tokens = tokens.contiguous()
        tokens_bs, first = tokens.stride(0), N - Lq
    if masks is not None:
        if tokens is None or masks.device != dev:
            raise L.SpecdecError(f"masks need tokens, and to be on {dev}")
        mask_bs, n = check_masks(masks, B, "process_logits")
        if n != N:
            raise L.SpecdecError(f"process_logits: {N} tokens per row, but masks of {n} nodes")
    ids = values = None
    M = bias_bs = 0
    if bias is not None:
        ids, values = bias
        if ids.device != dev or values.device != dev or ids.dim() != 2 or ids.shape != values.shape \
                or ids.shape[0] not in (1, B) or ids.is_floating_point():
            raise L.SpecdecError(f"bias must be (integer ids, values), both [{B} or 1, M] on {dev}")
        M = ids.shape[1]
        if M > BIAS_MAX:
            raise L.SpecdecError(f"at most {BIAS_MAX} biases per row, got {M}")
        ids, values = ids.long().contiguous(), values.float().contiguous()
        bias_bs = M if ids.shape[0] == B else 0
    allowed_bs = allowed_ps = 0
    if allowed is not None:
        words = -(-V // 32)
        if allowed.device != dev or allowed.dtype != torch.int32 or allowed.dim() != 3 \
                or allowed.shape[0] not in (1, B) or allowed.shape[1] not in (1, Lq) \
                or allowed.shape[2] != words or (words > 1 and allowed.stride(2) != 1):
            raise L.SpecdecError(f"allowed must be int32 [{B} or 1, {Lq} or 1, {words}] on {dev}")
        allowed_bs = allowed.stride(0) if allowed.shape[0] == B else 0
        allowed_ps = allowed.stride(1) if allowed.shape[1] == Lq else 0
    if out is None:
        out = torch.empty(B, Lq, V, dtype=logits.dtype, device=dev)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev \
            or (V > 1 and out.stride(2) != 1):
        raise L.SpecdecError(f"out must be {tuple(logits.shape)} of {logits.dtype} on {dev}, "
                             "contiguous along the vocabulary")
    L.check(L.lib().sd_process_logits(
        logits.data_ptr(), logits.stride(0), logits.stride(1), code, B, Lq, V, L.address(tokens),
        tokens_bs, L.address(masks), mask_bs, N, first, L.address(hist),
        0 if hist is None else hist.stride(0), L.address(repetition), L.address(presence),
        L.address(frequency), L.address(ids), L.address(values), bias_bs, M, L.address(allowed),
        allowed_bs, allowed_ps, out.data_ptr(), out.stride(0), out.stride(1), L.stream_of(dev)),
        "process_logits")
    return out
