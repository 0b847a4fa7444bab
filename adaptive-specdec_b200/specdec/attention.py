"""Verify attention over the ragged cache, and its transformers hook.

``verify_attention`` is the Python face of sd_verify_attn: grouped-query
attention where query j of row b reads cache slots s <= lengths[b] + j (and
s < valid[b] in a right-padded prefill).  It replaces the reference's HF SDPA
over ``_RaggedLayer.update``'s max-width view plus the additive mask
(specdec/kvcache.py:61-74 and :138-162, called at specdec/engine.py:274): each
row reads only its own live keys.  ``prefix_attention`` is the same over a paged
cache whose rows share their first pages (sd_prefix_attn), ``tree_attention`` that
of a drafted tree's nodes (sd_tree_attn).

``register()`` installs it as the transformers attention implementation
"specdec_b200" (with a mask function that builds no mask); a model loaded with
``attn_implementation="specdec_b200"`` and run against a
``RaggedCache(..., attn_impl="specdec_b200")`` then attends through the kernel.
"""
import torch

from specdec import _lib as L
from specdec.tree import check_masks

IMPL = "specdec_b200"
PREFILL_SDPA_MIN = 64          # prefills longer than this (fresh cache) use torch SDPA
SD_PAGE = 128                  # SD_KV_PAGE (kvcache.PAGE)
_ATTN_DTYPES = {torch.bfloat16: 2, torch.float32: 0}


class _WS:
    def __init__(self):
        self.t = {}

    def get(self, n, device):
        key = (device.index, torch.cuda.current_stream(device).cuda_stream)
        cur = self.t.get(key)
        if cur is None or cur.numel() < n:
            cur = torch.empty(max(int(n), 1 << 20), dtype=torch.uint8, device=device)
            self.t[key] = cur
        return cur


_ws = _WS()


def verify_attention(q, k_cache, v_cache, lengths, valid=None, scale=None, out=None,
                     block_table=None):
    """q [B, Hq, qlen, D], caches [B, Hkv, C, D] -> out [B, qlen, Hq, D].

    ``lengths`` [B] int64 on the device are the lengths before this forward's
    advance (the new keys were already appended at lengths[b] + j).  With
    ``block_table`` [B, W] int32 the caches are page pools
    [n_pages, Hkv, PAGE, D] (PagedRaggedCache) and C = W * PAGE.
    """
    L.require_cuda(q, k_cache, v_cache, lengths)
    if q.dtype not in _ATTN_DTYPES or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise L.SpecdecError(f"verify_attention supports bf16 / fp32, got {q.dtype}")
    B, Hq, qlen, D = q.shape
    if block_table is not None:
        return _verify_attention_paged(q, k_cache, v_cache, lengths, valid, scale, out,
                                       block_table)
    _, Hkv, C, _ = k_cache.shape
    if q.stride(-1) != 1:
        q = q.contiguous()
    kc = k_cache if k_cache.is_contiguous() else k_cache.contiguous()
    vc = v_cache if v_cache.is_contiguous() else v_cache.contiguous()
    if out is None:
        out = torch.empty(B, qlen, Hq, D, dtype=q.dtype, device=q.device)
    sc = float(scale) if scale is not None else D ** -0.5
    lens = lengths.to(torch.long).contiguous()
    val = None if valid is None else valid.to(q.device, torch.long).contiguous()
    lib = L.lib()
    with torch.cuda.device(q.device):
        nws = lib.sd_verify_attn_workspace_bytes(B, Hq, Hkv, D, C, qlen)
        ws = _ws.get(nws, q.device)
        L.check(lib.sd_verify_attn(L.ptr(q), q.stride(0), q.stride(1), q.stride(2), L.ptr(kc),
                                   L.ptr(vc), L.ptr(lens), L.ptr(val), B, Hq, Hkv, D, C, qlen, sc,
                                   L.ptr(out), out.stride(0), out.stride(1), out.stride(2),
                                   _ATTN_DTYPES[q.dtype], L.ptr(ws), ws.numel(),
                                   L.stream_ptr(q.device)), "verify_attn")
    return out


def _verify_attention_paged(q, kpool, vpool, lengths, valid, scale, out, bt):
    from specdec.kvcache import PAGE
    B, Hq, qlen, D = q.shape
    npages, Hkv, page, _ = kpool.shape
    if page != PAGE or vpool.shape != kpool.shape or not (kpool.is_contiguous()
                                                          and vpool.is_contiguous()):
        raise L.SpecdecError("paged caches must be contiguous [n_pages, Hkv, PAGE, D] pools")
    if bt.dtype != torch.int32 or bt.dim() != 2 or bt.shape[0] != B or not bt.is_contiguous():
        raise L.SpecdecError("block_table must be a contiguous [B, W] int32 tensor")
    W = bt.shape[1]
    if q.stride(-1) != 1:
        q = q.contiguous()
    if out is None:
        out = torch.empty(B, qlen, Hq, D, dtype=q.dtype, device=q.device)
    sc = float(scale) if scale is not None else D ** -0.5
    lens = lengths.to(torch.long).contiguous()
    val = None if valid is None else valid.to(q.device, torch.long).contiguous()
    lib = L.lib()
    with torch.cuda.device(q.device):
        nws = lib.sd_verify_attn_workspace_bytes(B, Hq, Hkv, D, W * PAGE, qlen)
        ws = _ws.get(nws, q.device)
        L.check(lib.sd_verify_attn_paged(
            L.ptr(q), q.stride(0), q.stride(1), q.stride(2), L.ptr(kpool), L.ptr(vpool), L.ptr(bt),
            W, npages, L.ptr(lens), L.ptr(val), B, Hq, Hkv, D, qlen, sc, L.ptr(out), out.stride(0),
            out.stride(1), out.stride(2), _ATTN_DTYPES[q.dtype], L.ptr(ws), ws.numel(),
            L.stream_ptr(q.device)), "verify_attn_paged")
    return out


def prefix_attention(q, k_pool, v_pool, lengths, block_table, group_starts, prefix_pages,
                     valid=None, scale=None, out=None):
    """``verify_attention`` over a paged cache whose rows share pages in front.

    q [B, Hq, qlen, D], pools [n_pages, Hkv, PAGE, D], ``lengths`` [B] and
    ``block_table`` [B, W] int32 as in ``verify_attention`` -> out [B, qlen, Hq,
    D].  Group g is the rows ``group_starts[g]`` .. ``group_starts[g + 1]`` (int32
    [G + 1] on the device, rising) whose first ``prefix_pages[g]`` (int32 [G])
    table entries are equal: samples of one prompt, requests under one system
    prompt.  Their keys are read once for the group instead of once per row.
    The result is ``verify_attention``'s but for the order of the float32 sums.
    Both group arrays live on the device, so a captured call follows them.
    bf16 heads of 128 share; other shapes (D <= 128) are computed row by row.
    Slots that no query of a row sees may hold anything.  In the slots of this
    step's own queries V has to be finite: a NaN there reaches the row's earlier
    queries, too.
    """
    dev, dt = q.device, q.dtype
    if not q.is_cuda:
        L.require_cuda(q)
    if k_pool.device != dev or v_pool.device != dev or lengths.device != dev \
            or block_table.device != dev or group_starts.device != dev \
            or prefix_pages.device != dev or (valid is not None and valid.device != dev) \
            or (out is not None and out.device != dev):
        raise L.SpecdecError("prefix_attention needs every tensor on one CUDA device")
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return prefix_attention(q, k_pool, v_pool, lengths, block_table, group_starts,
                                    prefix_pages, valid, scale, out)
    if q.dim() != 4 or k_pool.dim() != 4:
        raise L.SpecdecError("prefix_attention needs q [B, Hq, qlen, D] and pools "
                             "[n_pages, Hkv, PAGE, D]")
    if dt not in _ATTN_DTYPES or k_pool.dtype != dt or v_pool.dtype != dt:
        raise L.SpecdecError(f"prefix_attention supports bf16 / fp32, got {dt}")
    B, Hq, qlen, D = q.shape
    npages, Hkv, page, Dk = k_pool.shape
    if page != SD_PAGE or Dk != D or v_pool.shape != k_pool.shape or not (
            k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise L.SpecdecError("paged caches must be contiguous [n_pages, Hkv, PAGE, D] pools")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B \
            or not block_table.is_contiguous():
        raise L.SpecdecError("block_table must be a contiguous [B, W] int32 tensor")
    G = prefix_pages.numel()
    if group_starts.dtype != torch.int32 or prefix_pages.dtype != torch.int32 or \
            group_starts.numel() != G + 1 or not (group_starts.is_contiguous()
                                                  and prefix_pages.is_contiguous()):
        raise L.SpecdecError("group_starts [G + 1] and prefix_pages [G] must be contiguous int32")
    if lengths.numel() != B or (valid is not None and valid.numel() != B):
        raise L.SpecdecError(f"lengths and valid need one entry per row ({B})")
    sc = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < sc < 3e38:
        raise L.SpecdecError(f"scale must be positive and finite, got {scale}")
    qb, qh, ql, qd = q.stride()
    if qd != 1 or (dt == torch.bfloat16 and D == 128 and (
            q.data_ptr() % 16 or qb % 8 or qh % 8 or ql % 8)):
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        qb, qh, ql, qd = q.stride()
    if lengths.dtype != torch.long or not lengths.is_contiguous():
        lengths = lengths.long().contiguous()
    if valid is not None and (valid.dtype != torch.long or not valid.is_contiguous()):
        valid = valid.long().contiguous()
    if out is None:
        out = q.new_empty(B, qlen, Hq, D)
        ob, ol, oh = qlen * Hq * D, Hq * D, D
    else:
        if out.shape != (B, qlen, Hq, D) or out.dtype != dt or (D > 1 and out.stride(3) != 1):
            raise L.SpecdecError(f"out must be {(B, qlen, Hq, D)} of {dt}, contiguous along D")
        ob, ol, oh, _ = out.stride()
    if B == 0 or qlen == 0:
        return out
    W, code = block_table.shape[1], _ATTN_DTYPES[dt]
    # a fresh buffer per call: calls on several streams and calls captured into
    # different graphs never share one
    nws = L.workspace_bytes("sd_prefix_attn_workspace_bytes", B, G, Hq, Hkv, D, W, qlen, code)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev)
    L.check(L.lib().sd_prefix_attn(
        q.data_ptr(), qb, qh, ql, k_pool.data_ptr(), v_pool.data_ptr(), block_table.data_ptr(),
        W, npages, lengths.data_ptr(), L.address(valid), group_starts.data_ptr(),
        prefix_pages.data_ptr(), G, B, Hq, Hkv, D, qlen, sc, out.data_ptr(), ob, ol, oh, code,
        ws.data_ptr(), nws, L.stream_of(dev)), "prefix_attn")
    return out


def tree_attention(q, k_cache, v_cache, lengths, masks, first=0, scale=None, out=None,
                   block_table=None):
    """Attention of the nodes of a drafted tree over the cache (``specdec.tree``).

    q [B, Hq, qlen, D], caches [B, Hkv, C, D] (or, with ``block_table`` [B, W]
    int32, page pools [n_pages, Hkv, PAGE, D]) -> out [B, qlen, Hq, D].  Query j is
    node ``first`` + j of the row's tree; ``lengths`` [B] are the lengths before this
    forward's advance (so with ``first`` = 0 the row's tokens, and ``first`` more when
    the tree is fed level by level).  It reads the slots s < lengths[b] - first and
    those of its ancestors and itself, lengths[b] - first + a for every bit a of
    ``masks`` [N, W] or [B, N, W] (``tree_masks``).  A node without a bit gives 0.
    Slots that no node sees may hold anything; V has to be finite in the slots that
    some of the row's nodes see and others do not.  bf16 and fp32.  ``out`` lies in
    memory of its own, contiguous along D; one whose heads share entries (an
    expanded tensor) is refused.
    """
    dev, dt = q.device, q.dtype
    if not q.is_cuda:
        L.require_cuda(q)
    if k_cache.device != dev or v_cache.device != dev or lengths.device != dev \
            or masks.device != dev or (block_table is not None and block_table.device != dev) \
            or (out is not None and out.device != dev):
        raise L.SpecdecError("tree_attention needs every tensor on one CUDA device")
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return tree_attention(q, k_cache, v_cache, lengths, masks, first, scale, out,
                                  block_table)
    if q.dim() != 4 or k_cache.dim() != 4:
        raise L.SpecdecError("tree_attention needs q [B, Hq, qlen, D] and caches [B, Hkv, C, D] "
                             "or pools [n_pages, Hkv, PAGE, D]")
    if dt not in _ATTN_DTYPES or k_cache.dtype != dt or v_cache.dtype != dt:
        raise L.SpecdecError(f"tree_attention supports bf16 / fp32, got {dt}")
    B, Hq, qlen, D = q.shape
    n0, Hkv, C, Dk = k_cache.shape
    if Dk != D or v_cache.shape != k_cache.shape or not (k_cache.is_contiguous()
                                                         and v_cache.is_contiguous()):
        raise L.SpecdecError("K and V caches must be contiguous, of one shape, with q's head size")
    W = npages = 0
    if block_table is not None:
        if C != SD_PAGE:
            raise L.SpecdecError("paged caches must be [n_pages, Hkv, PAGE, D] pools")
        if block_table.dtype != torch.int32 or block_table.dim() != 2 or \
                block_table.shape[0] != B or not block_table.is_contiguous():
            raise L.SpecdecError("block_table must be a contiguous [B, W] int32 tensor")
        W, npages = block_table.shape[1], n0
        C = W * SD_PAGE
    elif n0 != B:
        raise L.SpecdecError(f"a cache of {n0} rows for {B} rows of queries")
    mask_bs, N = check_masks(masks, B, "tree_attention")
    first = int(first)
    if not 0 <= first <= N - qlen:
        raise L.SpecdecError(f"nodes {first} to {first + qlen - 1} of a tree of {N}")
    if lengths.numel() != B:
        raise L.SpecdecError(f"lengths needs one entry per row ({B})")
    sc = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < sc < 3e38:
        raise L.SpecdecError(f"scale must be positive and finite, got {scale}")
    qb, qh, ql, qd = q.stride()
    if qd != 1 or (dt == torch.bfloat16 and D in (64, 128) and (
            q.data_ptr() % 16 or any(n > 1 and (x % 8 or not x) for n, x in zip(q.shape, (qb, qh, ql))))):
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        qb, qh, ql, qd = q.stride()
    if lengths.dtype != torch.long or not lengths.is_contiguous():
        lengths = lengths.long().contiguous()
    if out is None:
        out = q.new_empty(B, qlen, Hq, D)
        ob, ol, oh = qlen * Hq * D, Hq * D, D
    else:
        if out.shape != (B, qlen, Hq, D) or out.dtype != dt or (D > 1 and out.stride(3) != 1):
            raise L.SpecdecError(f"out must be {(B, qlen, Hq, D)} of {dt}, contiguous along D")
        ob, ol, oh, _ = out.stride()
    if B == 0 or qlen == 0:
        return out
    code = _ATTN_DTYPES[dt]
    # a fresh buffer per call: calls on several streams and calls captured into
    # different graphs never share one
    nws = L.workspace_bytes("sd_tree_attn_workspace_bytes", B, Hq, Hkv, D, C, qlen, code)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    L.check(L.lib().sd_tree_attn(
        q.data_ptr(), qb, qh, ql, k_cache.data_ptr(), v_cache.data_ptr(), L.address(block_table),
        W, npages, lengths.data_ptr(), masks.data_ptr(), mask_bs, N, first, B, Hq, Hkv, D, C, qlen,
        sc, out.data_ptr(), ob, ol, oh, code, L.address(ws), nws, L.stream_of(dev)), "tree_attn")
    return out


def gather_pages(pool, block_table, n):
    """The first n slots of every row of a page pool as [B, Hkv, n, D]."""
    from specdec.kvcache import PAGE
    npg = -(-n // PAGE)
    idx = block_table[:, :npg].long().clamp_min(0)
    B = idx.shape[0]
    g = pool[idx]                                     # [B, npg, Hkv, PAGE, D]
    return g.permute(0, 2, 1, 3, 4).reshape(B, pool.shape[1], npg * PAGE, pool.shape[3])[:, :, :n]


def hf_attention(module, query, key, value, attention_mask, dropout=0.0, scaling=None, **kwargs):
    """transformers AttentionInterface function for RaggedCache buffers."""
    cache = getattr(key, "_sd_cache", None)
    if cache is not None:
        bt, prefix = getattr(cache, "block_table", None), getattr(cache, "prefix", None)
        if cache.tree is not None:                  # a drafted tree: nodes see their ancestors
            masks, _, first = cache.tree
            return tree_attention(query, key, value, cache.lengths, masks, first, scaling,
                                  block_table=bt), None
        q_len = query.shape[2]
        if (cache.valid is not None and q_len > PREFILL_SDPA_MIN and cache._host_valid
                and int(cache._host.max()) == 0):
            # right-padded prefill of a fresh cache (every row at length 0):
            # plain causal attention over the q new keys; a real token i < valid[b]
            # only sees keys s <= i, so the padding never reaches it.  Prefill is
            # outside the verify round; torch's SDPA (flash / cuDNN) runs it.
            if bt is not None:
                ks, vs = gather_pages(key, bt, q_len), gather_pages(value, bt, q_len)
            else:
                ks, vs = key[:, :, :q_len], value[:, :, :q_len]
            out = torch.nn.functional.scaled_dot_product_attention(
                query, ks, vs, is_causal=True, scale=scaling, enable_gqa=True)
            return out.transpose(1, 2), None
        if prefix is not None:                      # a forked cache: rows share their prompt's pages
            return prefix_attention(query, key, value, cache.lengths, bt, *prefix,
                                    valid=cache.valid, scale=scaling), None
        out = verify_attention(query, key, value, cache.lengths, valid=cache.valid, scale=scaling,
                               block_table=bt)
        return out, None
    # a forward without a RaggedCache: causal self-attention over the given
    # K/V, i.e. the same kernel with every row starting at length 0
    if attention_mask is not None and attention_mask.dim() == 4 and not bool(
            (attention_mask == 0).all()):
        raise L.SpecdecError("specdec_b200 attention without a RaggedCache supports plain "
                             "causal masks only")
    if key.shape[2] != query.shape[2]:
        raise L.SpecdecError("specdec_b200 attention without a RaggedCache needs q_len == kv_len")
    lens = torch.zeros(query.shape[0], dtype=torch.long, device=query.device)
    out = verify_attention(query, key.contiguous(), value.contiguous(), lens, scale=scaling)
    return out, None


def _no_mask(*args, **kwargs):
    return None


def register():
    """Register the kernel as attention implementation "specdec_b200"."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface
    AttentionInterface.register(IMPL, hf_attention)
    AttentionMaskInterface.register(IMPL, _no_mask)
    return IMPL
