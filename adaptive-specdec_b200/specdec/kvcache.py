"""A KV cache whose rows roll back independently, in O(1), on the device.

Drop-in for the reference's specdec/kvcache.py (RaggedCache, kvcache.py:
98-202): same constructor, same geometry and mutation methods, and the
transformers ``Cache`` interface.  What changes is where the bookkeeping runs:

* ``lengths`` is device-resident and authoritative.  advance / rollback /
  commit are one tiny kernel each (sd_kv_lengths_update / sd_kv_commit): no
  data movement and no host synchronisation, also when the counts are a CUDA
  tensor (the reference copies them to the host, kvcache.py:183-185).
* a host mirror of the lengths is kept whenever the host knows them (int or
  list arguments), so ``max_len`` / ``kv_len_for`` stay sync-free on those
  paths; after a device-side rollback it is refreshed lazily, once.
* ``layers[i].update`` appends the new K/V rows at each row's own offset with
  one kernel (sd_kv_append), replacing the two scatters of kvcache.py:61-74.

Two attention modes:

* ``attn_impl="specdec_b200"`` (what the engine uses): ``update`` returns the
  full [B, Hkv, C, D] buffers and the registered attention function reads only
  each row's live keys with the verify-attention kernel (sd_verify_attn);
* the default mode returns [:, :, :max_len+q] views exactly like the reference,
  for use with stock attention implementations and ``attn_mask``.

Invariant (the reference's, kvcache.py:17-21): after a rollback the cache is
indistinguishable from one that only ever processed the accepted prefix.

``PagedRaggedCache`` keeps the same interface over pages of PAGE tokens
drawn from one pool per layer, so that memory follows each row's own length
rather than the widest row's (the reference pads every row to the capacity,
kvcache.py:98-116).  Its page bookkeeping runs on the host (``PageTable``) or, with
``device_pages=True``, on the device (``DevicePageTable``): pages then follow the
device lengths without a host copy of them, and ``fork`` makes several rows of
one prompt that share its pages.
"""
from array import array

import numpy as np
import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from specdec import _lib as L
from specdec.tree import TREE_MAX

__all__ = ["RaggedCache", "PagedRaggedCache", "DevicePageTable", "commit_tree", "PAGE"]

_BAD_PATH = "RaggedCache: a committed path was not a rising list of the tree's nodes"

PAGE = 128            # tokens per page (SD_KV_PAGE): one K/V tile of the verify attention


def commit_tree(keys, values, lengths, path, n_acc, nodes, block_table=None, err=None):
    """Commit a tree round in every layer: the accepted path's K and V move to the
    slots behind the row's tokens, ``lengths`` follow.

    keys / values: the layers' caches, lists of [B, Hkv, C, D] or, with
    ``block_table`` [B, W] int32, of pools [n_pages, Hkv, PAGE, D]; 2- or 4-byte
    types.  ``lengths`` [B] int64 are those after the forward over ``nodes`` tree
    nodes (base + nodes) and become base + 1 + n_acc; ``path`` [B, P] int32 and
    ``n_acc`` [B] are ``specdec.tree.tree_accept``'s.  A row whose slots would leave
    the cache, or whose path is not strictly rising below ``nodes``, stays as it
    was and sets bit 0 or 5 of ``err`` ([1] int32); a slot without a page is not
    moved (bit 1).  No host synchronisation.
    """
    keys, values = list(keys), list(values)
    dev = lengths.device
    if not lengths.is_cuda:
        L.require_cuda(lengths)
    B = lengths.numel()
    if lengths.dtype != torch.long or not lengths.is_contiguous():
        raise L.SpecdecError("lengths must be contiguous int64 (they are updated in place)")
    if path.device != dev or path.dtype != torch.int32 or path.dim() != 2 or path.shape[0] != B \
            or path.shape[1] < 1 or (path.shape[1] > 1 and path.stride(1) != 1):
        raise L.SpecdecError(f"path must be int32 [{B}, P] on {dev}")
    if n_acc.device != dev or n_acc.numel() != B or n_acc.is_floating_point():
        raise L.SpecdecError(f"n_acc must be integers [{B}] on {dev}")
    if n_acc.dtype != torch.long or not n_acc.is_contiguous():
        n_acc = n_acc.long().contiguous()
    N = int(nodes)
    if not 1 <= N <= TREE_MAX:
        raise L.SpecdecError(f"a tree has 1 to {TREE_MAX} nodes, got {nodes}")
    if err is not None and (err.device != dev or err.dtype != torch.int32 or err.numel() != 1):
        raise L.SpecdecError(f"err must be int32 [1] on {dev}")
    bufs = keys + values
    if not bufs or len(keys) != len(values):
        raise L.SpecdecError(f"commit_tree needs K and V of every layer, got {len(keys)} and "
                             f"{len(values)}")
    shape, dt, e = bufs[0].shape, bufs[0].dtype, bufs[0].element_size()
    if len(shape) != 4 or e not in (2, 4):
        raise L.SpecdecError("caches must be [B, Hkv, C, D] or [n_pages, Hkv, PAGE, D] of a 2- or "
                             "4-byte type")
    index = dev.index
    for t in bufs:                                   # (two per layer: what a call costs most)
        if t.dtype is not dt or t.get_device() != index or not t.is_contiguous() or t.shape != shape:
            raise L.SpecdecError("every layer's K and V must be contiguous, of one shape, type and "
                                 f"device ({dev})")
    n0, H, C, D = shape
    W = npages = 0
    if block_table is not None:
        if block_table.device != dev or block_table.dtype != torch.int32 or block_table.dim() != 2 \
                or block_table.shape[0] != B or not block_table.is_contiguous():
            raise L.SpecdecError(f"block_table must be contiguous int32 [{B}, W] on {dev}")
        W, npages = block_table.shape[1], n0
        if C != PAGE:
            raise L.SpecdecError("paged caches must be [n_pages, Hkv, PAGE, D] pools")
    elif n0 != B:
        raise L.SpecdecError(f"caches of {n0} rows for {B} lengths")
    ptrs = array("Q", map(torch.Tensor.data_ptr, bufs))
    if len(set(ptrs)) != len(ptrs) and bufs[0].numel():
        raise L.SpecdecError("a buffer stands twice among the layers' K and V")
    with L.on_device(dev):
        L.check(L.lib().sd_kv_commit_tree(
            ptrs.buffer_info()[0], len(bufs), L.address(block_table), W, npages, lengths.data_ptr(),
            path.data_ptr(), path.stride(0), path.shape[1], n_acc.data_ptr(), N, B, H, C, D, e,
            L.address(err), L.stream_of(dev)), "kv_commit_tree")


class _RaggedLayer(CacheLayerMixin):
    """One layer's preallocated [B, Hkv, C, D] K and V buffers."""

    is_sliding = False
    is_compileable = False

    def __init__(self, parent):
        super().__init__()
        self.parent = parent
        self.keys = None
        self.values = None
        self.is_initialized = False

    def lazy_initialization(self, key_states, value_states=None):
        p = self.parent
        b, h, _, d = key_states.shape
        self.dtype, self.device = key_states.dtype, key_states.device
        self.keys = torch.zeros(b, h, p.capacity, d, dtype=self.dtype, device=self.device)
        self.values = torch.zeros(b, h, p.capacity, d, dtype=self.dtype, device=self.device)
        self.keys._sd_cache = p
        self.values._sd_cache = p
        self.is_initialized = True

    def update(self, key_states, value_states, *args, **kwargs):
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        p = self.parent
        b, h, q, d = key_states.shape
        # offsets are the lengths BEFORE this forward; the parent advances once,
        # after every layer has written (kvcache.py:63-66)
        L.require_cuda(key_states, value_states, p.lengths)
        ks, vs = key_states, value_states
        if ks.stride(-1) != 1:
            ks = ks.contiguous()
        if vs.stride() != ks.stride():
            vs = vs.contiguous()
            ks = ks.contiguous()
        code = L.dtype_code(ks.dtype)
        with torch.cuda.device(ks.device):
            L.check(L.lib().sd_kv_append(L.ptr(self.keys), L.ptr(self.values), L.ptr(ks), L.ptr(vs),
                                         ks.stride(0), ks.stride(1), ks.stride(2), L.ptr(p.lengths),
                                         b, h, p.capacity, d, q, code, L.ptr(p._err),
                                         L.stream_ptr(ks.device)), "kv_append")
        p._last_q = q
        if p.attn_impl == "specdec_b200":
            return self.keys, self.values
        kv_len = p.kv_len_for(q)
        return self.keys[:, :, :kv_len, :], self.values[:, :, :kv_len, :]

    def get_mask_sizes(self, query_length, layer_idx=None):
        return self.parent.get_mask_sizes(query_length, layer_idx)

    def get_seq_length(self):
        return self.parent.get_seq_length() if self.is_initialized else 0

    def get_max_cache_shape(self):
        return self.parent.capacity


class RaggedCache(Cache):
    """Per-row-length KV cache with O(1), device-side rollback.

    Usage per forward (as the reference):
        pos  = cache.positions(q)                  # [B, q] RoPE positions
        mask = cache.attn_mask(q, dtype, valid)    # only for stock attention
        out  = model(input_ids, position_ids=pos, attention_mask=mask,
                     past_key_values=cache, cache_position=cache.cache_position(q))
        cache.advance(q)                           # exactly once per forward
    """

    _layer_cls = _RaggedLayer

    def __init__(self, n_layers, batch_size, capacity, device, attn_impl=None):
        self.capacity = int(capacity)
        self.batch_size = int(batch_size)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise L.SpecdecError("RaggedCache keeps its lengths on the GPU (no CPU fallback)")
        self.attn_impl = attn_impl
        self.lengths = torch.zeros(self.batch_size, dtype=torch.long, device=self.device)
        self._err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._host = torch.zeros(self.batch_size, dtype=torch.long)
        self._host_valid = True
        self.valid = None           # optional [B] cap for right-padded prefill
        self.tree = None            # (masks, depths, first node) of a drafted tree's forward
        self._last_q = 0
        super().__init__(layers=[self._layer_cls(self) for _ in range(n_layers)])

    # ---- host mirror -----------------------------------------------------
    def _mirror(self):
        if not self._host_valid:
            self._host = self.lengths.to("cpu")
            self._host_valid = True
        return self._host

    def invalidate_host(self):
        """Forget the host mirror (the next host read syncs once).  Steps that
        are replayed from CUDA graphs change the device lengths only."""
        self._host_valid = False

    @property
    def lengths_cpu(self):
        return self._mirror()

    @property
    def max_len(self):
        return int(self._mirror().max()) if self.batch_size else 0

    @property
    def _uniform(self):
        h = self._mirror()
        return bool(int(h.min()) == int(h.max()))

    # ---- geometry ----------------------------------------------------------
    def kv_len_for(self, q):
        """Width of the key/value window the stock attention path reads."""
        return self.max_len + q

    def positions(self, q):
        """RoPE positions [B, q]: each row continues from its own length (a tree's
        nodes by their depth)."""
        if self.tree is not None:
            _, depths, first = self.tree
            return (self.lengths.view(-1, 1) - first) + depths[..., first:first + q]
        ar = torch.arange(q, device=self.device).view(1, q)
        return self.lengths.view(-1, 1) + ar

    def cache_position(self, q):
        """Shared 1-D cache_position, consistent with the widest row.

        Only mask construction reads it; the kernel path builds no mask, so
        there it is arange(q) and needs no host copy of the lengths.
        """
        if self.attn_impl == "specdec_b200":
            return torch.arange(q, device=self.device)
        m = self.max_len
        return torch.arange(m, m + q, device=self.device)

    def attn_mask(self, q, dtype, valid=None):
        """Additive mask [B, 1, q, kv_len] (0 = attend) for stock attention.

        Same rule as the reference (kvcache.py:138-162): s <= lengths[b] + j,
        and s < valid[b] when given; None when all rows are level and there is
        no padding.  The kernel attention path needs no mask.
        """
        if self.attn_impl == "specdec_b200":
            self.valid = valid
            return None
        if valid is None and self._uniform:
            return None
        kv_len = self.kv_len_for(q)
        s = torch.arange(kv_len, device=self.device).view(1, 1, kv_len)
        j = torch.arange(q, device=self.device).view(1, q, 1)
        allowed = s <= (self.lengths.view(-1, 1, 1) + j)
        if valid is not None:
            allowed = allowed & (s < valid.to(self.device).view(-1, 1, 1))
        neg = torch.finfo(dtype).min
        return torch.where(allowed, 0.0, neg).to(dtype).unsqueeze(1)

    # ---- mutation ----------------------------------------------------------
    def _update(self, delta, q, sign):
        with torch.cuda.device(self.device):
            L.check(L.lib().sd_kv_lengths_update(L.ptr(self.lengths), L.ptr(delta), int(q), sign,
                                                 self.batch_size, self.capacity, L.ptr(self._err),
                                                 L.stream_ptr(self.device)), "kv lengths")

    def advance(self, q):
        """Call once per forward, after the model has run."""
        q = int(q)
        if self._host_valid and int(self._host.max()) + q > self.capacity:
            raise RuntimeError("RaggedCache.advance beyond capacity")
        self._update(None, q, +1)
        if self._host_valid:
            self._host += q
        self.valid = None

    def set_lengths(self, lengths):
        self.valid = self.tree = None
        t = torch.as_tensor(lengths, dtype=torch.long)
        if t.is_cuda:
            self.lengths.copy_(t)
            self._host_valid = False
        else:
            self._host = t.clone()
            self._host_valid = True
            self.lengths.copy_(t, non_blocking=False)

    def set_host_lengths(self, lengths):
        """Tell the cache its device lengths, as the caller read them back
        (no device work): host-side geometry and page reservations then need
        no sync of their own."""
        self._host = torch.as_tensor(lengths, dtype=torch.long).reshape(-1).clone()
        self._host_valid = True

    def rollback(self, n):
        """Drop the last n[b] tokens of row b.  O(1): no copy, no allocation.

        int / list: checked on the host (RuntimeError below zero, as the
        reference, kvcache.py:188-189).  CUDA tensor: applied on the device
        with no sync; a row that would go below zero is left unchanged and
        flagged, and the next check_errors() raises.
        """
        if torch.is_tensor(n) and n.is_cuda:
            d = n.to(torch.long).reshape(-1).contiguous()
            self._update(d, 0, -1)
            self._host_valid = False
            self.tree = None
            return
        if isinstance(n, int):
            n_cpu = torch.full((self.batch_size,), n, dtype=torch.long)
        elif torch.is_tensor(n):
            n_cpu = n.detach().to("cpu", torch.long).reshape(-1)
        else:
            n_cpu = torch.as_tensor(list(n), dtype=torch.long)
        h = self._mirror()
        if bool(((h - n_cpu) < 0).any()):
            raise RuntimeError("RaggedCache.rollback below zero")
        self._update(n_cpu.to(self.device, non_blocking=True), 0, -1)
        self._host = h - n_cpu
        self.tree = None

    def commit(self, n_acc, k):
        """Verify-round commit: lengths -= k - n_acc (device n_acc, no sync)."""
        with torch.cuda.device(self.device):
            L.check(L.lib().sd_kv_commit(L.ptr(self.lengths), L.ptr(n_acc.to(torch.long)), int(k),
                                         self.batch_size, L.ptr(self._err),
                                         L.stream_ptr(self.device)), "kv commit")
        self._host_valid = False
        self.tree = None

    # ---- trees of drafted tokens ---------------------------------------------
    def set_tree(self, masks=None, depths=None, first=0):
        """The next forwards are over nodes first, first + 1, ... of a drafted tree
        (``specdec.tree.tree_masks``) whose earlier nodes the cache already holds.
        They are over chains again once the round ends, in commit_tree, commit,
        rollback, set_lengths or reset, or by a call without arguments.  Only the
        kernel attention path (attn_impl "specdec_b200") knows trees."""
        if masks is None:
            self.tree = None
            return
        if self.attn_impl != "specdec_b200":
            raise L.SpecdecError("trees of drafted tokens need the specdec_b200 attention")
        self.tree = (masks, depths, int(first))

    def commit_tree(self, path, n_acc, nodes):
        """Tree-round commit, after a forward over ``nodes`` tree nodes and its
        advance: every layer keeps the accepted path behind the row's tokens,
        lengths go from base + nodes to base + 1 + n_acc (``commit_tree``)."""
        live = [layer for layer in self.layers if layer.is_initialized]
        commit_tree([x.keys for x in live], [x.values for x in live], self.lengths, path, n_acc,
                    nodes, block_table=getattr(self, "block_table", None), err=self._err)
        self._host_valid = False
        self.tree = None

    def check_errors(self):
        """Raise if any device-side update was refused (syncs once)."""
        e = int(self._err.item())
        if e:
            self._err.zero_()
            if e & 32:
                raise RuntimeError(_BAD_PATH)
            raise RuntimeError("RaggedCache: a length update left [0, capacity]")

    # ---- Cache interface ---------------------------------------------------
    def get_seq_length(self, layer_idx: int = 0):
        # On the kernel path transformers only feeds this to mask construction,
        # which the registered mask function skips: answer from the host mirror
        # when it is valid and never read the device lengths back (so forwards
        # stay free of host syncs and can be graph-captured).
        if self.attn_impl == "specdec_b200":
            return int(self._host.max()) if self._host_valid and self.batch_size else 0
        return self.max_len

    def get_mask_sizes(self, query_length, layer_idx=0):
        # transformers 5.x passes an int query length; older callers pass the
        # cache_position tensor (the reference's signature, kvcache.py:76-78).
        # The kernel path builds no mask, so it needs no (host) max length.
        q = query_length if isinstance(query_length, int) else int(query_length.shape[0])
        if self.attn_impl == "specdec_b200":
            return q, 0
        return self.kv_len_for(q), 0

    def reset(self):
        self.lengths.zero_()
        self.tree = None
        self._host = torch.zeros(self.batch_size, dtype=torch.long)
        self._host_valid = True
        self._err.zero_()
        for layer in self.layers:
            if layer.is_initialized:
                layer.keys.zero_()
                layer.values.zero_()


class _PagedLayer(_RaggedLayer):
    """One layer's K and V page pools [n_pages, Hkv, PAGE, D]."""

    def lazy_initialization(self, key_states, value_states=None):
        p = self.parent
        _, h, _, d = key_states.shape
        self.dtype, self.device = key_states.dtype, key_states.device
        self.keys = torch.zeros(p.n_pages, h, PAGE, d, dtype=self.dtype, device=self.device)
        self.values = torch.zeros(p.n_pages, h, PAGE, d, dtype=self.dtype, device=self.device)
        self.keys._sd_cache = p
        self.values._sd_cache = p
        self.is_initialized = True

    def update(self, key_states, value_states, *args, **kwargs):
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        p = self.parent
        b, h, q, d = key_states.shape
        L.require_cuda(key_states, value_states, p.lengths)
        ks, vs = key_states, value_states
        if ks.stride(-1) != 1:
            ks = ks.contiguous()
        if vs.stride() != ks.stride():
            vs, ks = vs.contiguous(), ks.contiguous()
        with torch.cuda.device(ks.device):
            L.check(L.lib().sd_kv_append_paged(
                L.ptr(self.keys), L.ptr(self.values), L.ptr(ks), L.ptr(vs), ks.stride(0),
                ks.stride(1), ks.stride(2), L.ptr(p.block_table), p.pages_per_row, p.n_pages,
                L.ptr(p.lengths), b, h, d, q, L.dtype_code(ks.dtype), L.ptr(p._err),
                L.stream_ptr(ks.device)), "kv_append_paged")
        p._last_q = q
        return self.keys, self.values


class PageTable:
    """Host-side page bookkeeping of a PagedRaggedCache (no device state).

    ``bt`` [B, pages_per_row] int32 holds row b's pages in slot order (-1 =
    none); pages [0, n_pages - 1) are handed out from a free stack, page
    n_pages - 1 is the sink that a right-padded prefill writes its padding
    to.  Every method returns True when ``bt`` changed.
    """

    def __init__(self, batch_size, pages_per_row, n_pages):
        if n_pages < 2:
            raise L.SpecdecError("a page pool needs at least two pages (one is the sink)")
        self.B, self.W, self.n_pages = int(batch_size), int(pages_per_row), int(n_pages)
        self.sink = self.n_pages - 1
        self.bt = np.full((self.B, self.W), -1, dtype=np.int32)
        self.owned = np.zeros(self.B, dtype=np.int64)              # real pages per row
        self.free = list(range(self.sink - 1, -1, -1))             # stack, page 0 on top

    def grow(self, need):
        """Give row b pages until it owns need[b] (slots [0, need[b] * PAGE))."""
        need = np.asarray(need, dtype=np.int64)
        if int(need.max(initial=0)) > self.W:
            raise RuntimeError("KV pages beyond the row capacity")
        short = np.maximum(need - self.owned, 0)
        total = int(short.sum())
        if total == 0:
            return False
        if total > len(self.free):
            raise L.SpecdecError(f"KV page pool exhausted: {total} pages wanted, "
                                 f"{len(self.free)} free of {self.n_pages - 1}")
        for b in np.nonzero(short)[0]:
            o = int(self.owned[b])
            for j in range(o, o + int(short[b])):
                self.bt[b, j] = self.free.pop()
            self.owned[b] = o + int(short[b])
        return True

    def reserve(self, lengths, q):
        """Pages for slots [0, lengths[b] + q) of every row."""
        lens = np.asarray(lengths, dtype=np.int64)
        return self.grow(-(-(lens + int(q)) // PAGE))

    def reserve_prefill(self, lengths, P, plen):
        """Real pages for [0, lengths[b] + plen[b]), the sink for the rest of
        [0, lengths[b] + P)."""
        lens = np.asarray(lengths, dtype=np.int64)
        pl = np.asarray(plen, dtype=np.int64)
        top = -(-(lens + int(P)) // PAGE)
        if int(top.max(initial=0)) > self.W:
            raise RuntimeError("KV pages beyond the row capacity")
        self.grow(-(-(lens + np.minimum(pl, int(P))) // PAGE))
        for b in range(self.B):
            o = int(self.owned[b])
            if top[b] > o:
                self.bt[b, o:top[b]] = self.sink
        return True

    def unsink(self):
        hit = self.bt == self.sink
        if not hit.any():
            return False
        self.bt[hit] = -1
        return True

    def release(self, rows):
        """Return the pages of the given rows to the free stack."""
        changed = False
        for b in (int(r) for r in rows):
            o = int(self.owned[b])
            self.free.extend(int(x) for x in self.bt[b, :o][::-1])
            changed = changed or o > 0 or bool((self.bt[b] >= 0).any())
            self.bt[b, :] = -1
            self.owned[b] = 0
        return changed

    def reset(self):
        self.bt[:] = -1
        self.owned[:] = 0
        self.free = list(range(self.sink - 1, -1, -1))
        return True

    def check(self):
        """Invariant: every handed-out page belongs to exactly one row slot."""
        used = self.bt[(self.bt >= 0) & (self.bt != self.sink)]
        assert len(set(used.tolist())) == used.size, "a page is owned twice"
        assert used.size + len(self.free) == self.n_pages - 1, "pages lost"
        for b in range(self.B):
            o = int(self.owned[b])
            assert (self.bt[b, :o] >= 0).all() and (self.bt[b, :o] != self.sink).all()


class DevicePageTable:
    """Page bookkeeping on the device: PageTable's page order, by device lengths.

    ``block_table`` [B, W] int32 (-1 = none), ``owned`` [B] pages of each row,
    ``shared`` [B] leading pages that the row reads but does not give back,
    ``free`` [n_pages] a stack of ``n_free`` [1] free pages, ``err`` [1] sticky
    error bits.  ``reserve`` and ``trim`` are stream ordered, never
    synchronise the host and can be captured into CUDA graphs; a call that
    cannot serve every row changes nothing and sets bits of ``err``
    (``check_errors``).  The stack starts with page 0 on top; the last page is
    kept out of it as the sink of right-padded prefills (``sink``).
    """

    ERRORS = {1: "a row's length left [0, capacity]", 2: "a slot was written without a page",
              4: "page pool exhausted", 8: "more new tokens than max_tokens",
              16: "a new token below a row's floor of shared pages",
              32: "a committed path was not a rising list of the tree's nodes"}

    def __init__(self, batch_size, pages_per_row, n_pages, device, err=None, stack=None):
        B, W, n = int(batch_size), int(pages_per_row), int(n_pages)
        if n < 2:
            raise L.SpecdecError("a page pool needs at least two pages (one is the sink)")
        if B < 1 or W < 1:
            raise L.SpecdecError("a page table needs at least one row and one page per row")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise L.SpecdecError("DevicePageTable keeps its state on the GPU (no CPU fallback)")
        if stack is None:
            free = torch.arange(n - 2, -2, -1, dtype=torch.int32, device=dev)
            n_free = torch.full((1,), n - 1, dtype=torch.int32, device=dev)
        else:
            free, n_free = stack                   # another table's: one pool for both
        self._bind(torch.full((B, W), -1, dtype=torch.int32, device=dev),
                   torch.zeros(B, dtype=torch.int32, device=dev),
                   torch.zeros(B, dtype=torch.int32, device=dev), free, n_free,
                   torch.zeros(1, dtype=torch.int32, device=dev) if err is None else err)

    def _bind(self, block_table, owned, shared, free, n_free, err):
        self.block_table, self.owned, self.shared = block_table, owned, shared
        self.free, self.n_free, self.err = free, n_free, err
        self.B, self.W = block_table.shape
        self.n_pages = free.numel()
        self.sink = self.n_pages - 1
        self.device = block_table.device

    @classmethod
    def over(cls, block_table, owned, shared, free, n_free, err):
        """A table over state that the caller holds (no copies)."""
        dev, i32 = block_table.device, torch.int32
        if not block_table.is_cuda:
            raise L.SpecdecError("DevicePageTable keeps its state on the GPU (no CPU fallback)")
        if block_table.dtype != i32:
            raise L.SpecdecError("a page table's state is int32 on one CUDA device")
        for t in (owned, shared, free, n_free, err):
            if t.dtype != i32 or t.device != dev:
                raise L.SpecdecError("a page table's state is int32 on one CUDA device")
            if not t.is_contiguous():
                raise L.SpecdecError("owned, shared, free, n_free and err must be contiguous")
        if block_table.dim() != 2 or block_table.stride(1) != 1:
            raise L.SpecdecError("block_table must be [B, W] with contiguous rows")
        B = block_table.shape[0]
        if owned.numel() != B or shared.numel() != B or n_free.numel() != 1 or err.numel() != 1:
            raise L.SpecdecError(f"owned and shared need {B} entries, n_free and err one")
        if B == 0 or block_table.shape[1] == 0 or free.numel() == 0:
            raise L.SpecdecError("a page table needs at least one row, one page per row and a pool")
        self = cls.__new__(cls)
        self._bind(block_table, owned, shared, free, n_free, err)
        return self

    def _rows(self, t, name):
        if t.device != self.device or t.numel() != self.B or t.is_floating_point():
            raise L.SpecdecError(f"{name} must be an integer [B] tensor on {self.device}")
        return t if t.dtype == torch.long and t.is_contiguous() else t.long().contiguous()

    def reserve(self, lengths, new, max_tokens=None, slot_map=True, floor=None):
        """Pages for ``new`` more tokens of every row past ``lengths`` [B].

        ``new`` is one int for all rows or an integer [B] tensor; with a tensor
        ``max_tokens`` bounds their sum (the size of ``slots``).  Returns
        (slots [max_tokens] int64, starts [B + 1] int32): token i of row b goes
        to pool slot slots[starts[b] + i] = page * PAGE + offset; slots behind
        the last token are -1.  ``slot_map=False`` leaves the map out: (None,
        starts).  With ``floor`` [B] int32 (``shared``, for rows that must not
        write what others read) a new token of row b in its first floor[b]
        pages is an error.
        """
        lens = self._rows(lengths, "lengths")
        if not slot_map:
            max_tokens = 0
        if torch.is_tensor(new):
            if max_tokens is None:
                raise L.SpecdecError("max_tokens is needed with per-row token counts")
            add, each, total = self._rows(new, "new"), 0, int(max_tokens)
        else:
            add, each = None, int(new)
            if not 0 <= each < 1 << 31:
                raise L.SpecdecError(f"new tokens must be in [0, 2^31), got {each}")
            total = self.B * each if max_tokens is None else int(max_tokens)
        if floor is not None and (floor.dtype != torch.int32 or floor.device != self.device
                                  or floor.numel() != self.B or not floor.is_contiguous()):
            raise L.SpecdecError(f"floor must be a contiguous int32 [B] tensor on {self.device}")
        if not 0 <= total < 1 << 31:
            raise L.SpecdecError(f"max_tokens must be in [0, 2^31), got {total}")
        dev = self.device
        # (an empty map still has an address: NULL means no map)
        slots = torch.empty(max(total, 1), dtype=torch.long, device=dev) if slot_map else None
        starts = torch.empty(self.B + 1, dtype=torch.int32, device=dev)
        nws = L.workspace_bytes("sd_pages_workspace_bytes", self.B)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        with L.on_device(dev):
            L.check(L.lib().sd_pages_reserve(
                self.block_table.data_ptr(), self.block_table.stride(0), self.W,
                self.owned.data_ptr(), self.free.data_ptr(), self.n_pages, self.n_free.data_ptr(),
                lens.data_ptr(), L.address(add), each, L.address(floor), self.B, L.address(slots),
                total, starts.data_ptr(), self.err.data_ptr(), ws.data_ptr(), nws, L.stream_of(dev)),
                "pages_reserve")
        return (slots[:total] if slot_map and total == 0 else slots), starts

    def trim(self, lengths):
        """Give back every row's pages past its ``lengths`` [B] tokens (never
        its shared ones); a trim after a reserve restores the stack."""
        lens = self._rows(lengths, "lengths")
        with L.on_device(self.device):
            L.check(L.lib().sd_pages_trim(
                self.block_table.data_ptr(), self.block_table.stride(0), self.W,
                self.owned.data_ptr(), self.shared.data_ptr(), self.free.data_ptr(), self.n_pages,
                self.n_free.data_ptr(), lens.data_ptr(), self.B, self.err.data_ptr(),
                L.stream_of(self.device)), "pages_trim")

    def reset(self):
        """Every page back on the stack, page 0 on top (of this table's pool)."""
        self.block_table.fill_(-1)
        self.owned.zero_()
        self.shared.zero_()
        n = self.n_pages
        self.free.copy_(torch.arange(n - 2, -2, -1, dtype=torch.int32, device=self.device))
        self.n_free.fill_(n - 1)
        self.err.zero_()

    def check_errors(self):
        """Raise if a call could not be done (syncs once)."""
        e = int(self.err.item())
        if e:
            self.err.zero_()
            raise RuntimeError("DevicePageTable: " + "; ".join(
                text for bit, text in self.ERRORS.items() if e & bit))


class PagedRaggedCache(RaggedCache):
    """RaggedCache whose rows own pages of PAGE tokens from a shared pool.

    Row b's slot s lives in page ``block_table[b, s // PAGE]`` of every
    layer's pool.  Pages are handed out on the host, before the forwards that
    need them: ``reserve(q)`` gives each row the pages for its next q tokens
    (one small host-to-device copy of the table when anything changed; no
    host sync while the host mirror of the lengths is valid), and
    ``reserve_prefill(P, plen)`` does the same for a right-padded prefill,
    pointing the padding past each row's own prompt at a shared sink page
    that nothing reads.  Pages stay with their row after a rollback (the row
    grows back into them); ``release(rows)`` and ``reset()`` return them.
    A slot written without a page sets the device error flag (bit 1).

    With ``device_pages`` the bookkeeping is a DevicePageTable: ``reserve``
    follows the device lengths with no host copy of them, a pool that runs out
    sets the error flag instead of raising, and ``fork`` makes several rows
    of each prompt that share its pages.  ``prefix`` (group starts, shared
    pages) then tells the attention which rows share what.  A forked row may
    not be rolled back into its shared pages and then grow: ``reserve`` sets
    the error flag (bit 16) and hands out nothing.

    Only the kernel attention path (attn_impl "specdec_b200") reads paged
    layers.
    """

    _layer_cls = _PagedLayer

    def __init__(self, n_layers, batch_size, capacity, device, attn_impl="specdec_b200",
                 n_pages=None, device_pages=False, _stack=None):
        if attn_impl != "specdec_b200":
            raise L.SpecdecError("PagedRaggedCache is read by the specdec_b200 attention only")
        self.pages_per_row = -(-int(capacity) // PAGE)
        super().__init__(n_layers, batch_size, self.pages_per_row * PAGE, device, attn_impl)
        self.n_pages = int(n_pages) if n_pages is not None else \
            self.batch_size * self.pages_per_row + 1
        self.device_pages = bool(device_pages)
        self.prefix = None
        # (rows that read them, first column, end) of the table columns whose pages
        # several rows of a fork share.  A row's runs follow one another from
        # column 0, and the readers of a later one read the earlier ones too.
        self._shared_runs = []
        if self.device_pages:
            self.pages = DevicePageTable(self.batch_size, self.pages_per_row, self.n_pages,
                                         self.device, err=self._err, stack=_stack)
            self.block_table = self.pages.block_table
            return
        self.pages = PageTable(self.batch_size, self.pages_per_row, self.n_pages)
        self.block_table = torch.full((self.batch_size, self.pages_per_row), -1,
                                      dtype=torch.int32, device=self.device)

    # ---- pages -------------------------------------------------------------
    @property
    def free_pages(self):
        return int(self.pages.n_free) if self.device_pages else len(self.pages.free)

    def _push(self, changed=True):
        if changed:
            self.block_table.copy_(torch.from_numpy(self.pages.bt))

    def _columns(self):
        return torch.arange(self.pages_per_row, device=self.device).view(1, -1)

    def reserve(self, q):
        """Pages for the next q tokens of every row (call before the forward)."""
        if self.device_pages:
            # (rows of a fork must not write the pages that they share)
            self.pages.reserve(self.lengths, int(q), slot_map=False,
                               floor=None if self.prefix is None else self.pages.shared)
            return
        self._push(self.pages.reserve(self._mirror().numpy(), q))

    def reserve_prefill(self, P, plen):
        """Pages for a right-padded prefill of P tokens with prompt lengths
        plen (real pages for each row's prompt, the sink for its padding)."""
        if self.device_pages:
            pl = torch.as_tensor(plen).to(self.device, torch.long).reshape(-1).clamp(max=int(P))
            self.pages.reserve(self.lengths, pl, slot_map=False,
                               floor=None if self.prefix is None else self.pages.shared)
            # only the padding goes to the sink: where the pool ran out, the prompt's
            # columns stay -1, so that writes there are flagged
            need = (self.lengths + pl + PAGE - 1) // PAGE
            top = (self.lengths + int(P) + PAGE - 1) // PAGE
            col = self._columns()
            pad = (col >= need.view(-1, 1)) & (col < top.view(-1, 1)) & (self.block_table < 0)
            self.block_table.masked_fill_(pad, self.pages.sink)
            return
        pl = torch.as_tensor(plen).to("cpu", torch.long).reshape(-1).numpy()
        self._push(self.pages.reserve_prefill(self._mirror().numpy(), P, pl))

    def release(self, rows):
        """Return the pages of the given rows to the pool (their lengths go to 0).
        Shared pages of a forked row stay with the rows that still read them and
        go back with the last of these; the row itself leaves its group."""
        rows = [int(r) for r in rows]
        if self.device_pages:
            if rows and not 0 <= min(rows) <= max(rows) < self.batch_size:
                raise L.SpecdecError(f"rows must be in [0, {self.batch_size}), got {rows}")
            at = torch.tensor(rows, dtype=torch.long, device=self.device)
            own = self._last_readers(rows)             # shared pages that are the row's now
            if own:
                self.pages.shared[list(own)] = torch.tensor(list(own.values()), dtype=torch.int32,
                                                            device=self.device)
            keep = self.pages.owned.long() * PAGE
            keep[at] = 0
            self.pages.trim(keep)
            self.lengths[at] = 0
            self.block_table[at] = -1
            self.pages.owned[at] = 0
            self.pages.shared[at] = 0
            if self.prefix is not None:
                gone = set(rows)
                self._set_groups([
                    (a, b, 0 if a in gone else p)
                    for first, end, p in self._groups
                    for a, b in self._runs(first, end, gone)])
            if self._host_valid:
                self._host[rows] = 0
            return
        h = self._mirror().clone()
        h[rows] = 0
        self.pages.release(rows)
        tree = self.tree
        self.set_lengths(h)
        self.tree = tree                             # (the other rows' round goes on)
        self._push()

    def _last_readers(self, rows):
        """Take `rows` out of the shared runs: {row: first column that nobody else reads}."""
        own = {}
        for r in rows:
            for readers, first, _ in self._shared_runs:
                if r in readers:
                    readers.remove(r)
                    if not readers:
                        own[r] = min(own.get(r, first), first)
        self._shared_runs = [run for run in self._shared_runs if run[0]]
        return own

    @staticmethod
    def _runs(first, end, gone):
        """[first, end) as runs without the rows of `gone` and these rows one by one."""
        out, a = [], first
        for r in range(first, end):
            if r in gone:
                out += ([(a, r)] if a < r else []) + [(r, r + 1)]
                a = r + 1
        return out + ([(a, end)] if a < end else [])

    def _set_groups(self, groups):
        """The groups (first row, end, shared pages) behind ``prefix``.  Its
        tensors keep their size and addresses, so that captured graphs follow a
        release: twice the first groups and one (groups behind the last are
        empty).  Runs that share nothing are one group; past the room, the
        groups that save least stop sharing."""
        B = self.batch_size
        if self.prefix is None:
            room = min(B, 2 * len(groups) + 1)
            self.prefix = (torch.empty(room + 1, dtype=torch.int32, device=self.device),
                           torch.empty(room, dtype=torch.int32, device=self.device))
        room = self.prefix[1].numel()
        while True:
            runs = []
            for a, b, p in groups:
                p = p if b - a > 1 else 0
                if runs and p == 0 and runs[-1][2] == 0:
                    runs[-1] = (runs[-1][0], b, 0)
                else:
                    runs.append((a, b, p))
            if len(runs) <= room:
                break
            least = min((r for r in runs if r[2]), key=lambda r: (r[1] - r[0] - 1) * r[2])
            groups = [(a, b, 0 if (a, b, p) == least else p) for a, b, p in runs]
        self._groups, n = runs, len(runs)
        starts = [r[0] for r in runs] + [B] * (room + 1 - n)
        pages = [r[2] for r in runs] + [0] * (room - n)
        for t, v in zip(self.prefix, (starts, pages)):
            t.copy_(torch.tensor(v, dtype=torch.int32))

    def fork(self, counts):
        """counts[b] rows for each row b, which share the full pages of row b;
        its last, partly filled page is copied to each.  Returns the new cache
        (rows of one source row side by side) over the same pools; this cache
        is left empty and must not be used further.  The shared pages go back
        with the last of their rows that the new cache releases, or its ``reset``.
        Raises what this cache's error flag holds (a prefill that found no
        pages), when a row holds tokens without a page, and when a forked row was
        rolled back into the pages it shares (its neighbours read them).
        Synchronises (error checks)."""
        if not self.device_pages:
            raise L.SpecdecError("fork needs device_pages=True")
        counts = [int(c) for c in counts]
        if len(counts) != self.batch_size or min(counts) < 1:
            raise L.SpecdecError(f"fork needs one positive count per row ({self.batch_size})")
        self.check_errors()
        need = (self.lengths.view(-1, 1) + PAGE - 1) // PAGE
        if bool(((self._columns() < need) & (self.block_table < 0)).any()):
            raise L.SpecdecError("fork: a row holds tokens without a page")
        if bool((self.lengths < self.pages.shared * PAGE).any()):
            raise L.SpecdecError("fork: a row was rolled back into the pages it shares")
        host = self._mirror().clone()
        src = torch.repeat_interleave(torch.arange(self.batch_size), torch.tensor(counts))
        new = PagedRaggedCache(len(self.layers), len(src), self.capacity, self.device,
                               n_pages=self.n_pages, device_pages=True,
                               _stack=(self.pages.free, self.pages.n_free))
        lens, full = host[src], host[src] // PAGE
        srcd, fulld = src.to(self.device), full.to(self.device)
        table = torch.where(new._columns() < fulld.view(-1, 1), self.block_table[srcd], -1)
        new.block_table.copy_(table)
        new.pages.owned.copy_(fulld)
        new.pages.shared.copy_(fulld)
        new.set_lengths(lens)
        new.pages.reserve(new.lengths, 0, slot_map=False)
        new.check_errors()
        part = torch.nonzero(lens % PAGE).view(-1).to(self.device)
        old_page = self.block_table[srcd[part], fulld[part]].long()
        new_page = new.block_table[part, fulld[part]].long()
        for a, b in zip(self.layers, new.layers):
            if not a.is_initialized:
                continue
            for pool in (a.keys, a.values):
                pool[new_page] = pool[old_page]
            b.dtype, b.device, b.is_initialized = a.dtype, a.device, True
            b.keys, b.values = a.keys[:], a.values[:]
            b.keys._sd_cache = b.values._sd_cache = new
        ends = torch.tensor(counts).cumsum(0).tolist()
        rows = [set(range(e - n, e)) for n, e in zip(counts, ends)]
        new._shared_runs = [(set().union(*(rows[r] for r in readers)), first, end)
                            for readers, first, end in self._shared_runs]
        for b, n in enumerate((host // PAGE).tolist()):
            first = max((end for readers, _, end in self._shared_runs if b in readers), default=0)
            if first < n:
                new._shared_runs.append((rows[b], first, n))
        # the copies are taken: the partly filled source pages go back
        self.pages.shared.copy_(host // PAGE)
        self.pages.trim(self.lengths // PAGE * PAGE)
        self.block_table.fill_(-1)
        self.pages.owned.zero_()
        self.pages.shared.zero_()
        self.set_lengths(torch.zeros(self.batch_size, dtype=torch.long))
        self.prefix = None
        self._shared_runs = []
        new._set_groups(list(zip([0] + ends[:-1], ends, (host // PAGE).tolist())))
        return new

    def set_lengths(self, lengths):
        super().set_lengths(lengths)
        if self.device_pages:
            self.block_table.masked_fill_(self.block_table == self.pages.sink, -1)
            return
        self._push(self.pages.unsink())

    def reset(self):
        super().reset()
        self.prefix = None
        self._shared_runs = []
        if self.device_pages:
            self.pages.reset()
            return
        self._push(self.pages.reset())

    def check_errors(self):
        e = int(self._err.item())
        if e:
            self._err.zero_()
            if e & 4:
                raise L.SpecdecError("KV page pool exhausted")
            if e & 32:
                raise RuntimeError(_BAD_PATH)
            if e & 16:
                raise RuntimeError("PagedRaggedCache: a forked row was rolled back into the pages "
                                   "it shares and would write them")
            if e & 2:
                raise RuntimeError("PagedRaggedCache: a slot was written without a page "
                                   "(reserve() before the forward)")
            raise RuntimeError("RaggedCache: a length update left [0, capacity]")

    @property
    def kv_bytes(self):
        """Bytes held by the K and V pools of the initialised layers."""
        return sum(2 * l.keys.numel() * l.keys.element_size() for l in self.layers
                   if l.is_initialized)
