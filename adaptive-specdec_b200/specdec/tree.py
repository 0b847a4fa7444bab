"""Trees of drafted tokens: ancestor bits and the accepted path.

The reference drafts chains; a tree offers the target model several
continuations per step and keeps the longest that it agrees with.  A tree of N
nodes is verified in ONE forward: node i is input position i, its key and value
go to cache slot base + i (base: the row's tokens before the forward), its rotary
position is base + depth(i), and it attends to the cache and to its ancestors
(``specdec.attention.tree_attention``).  Node 0 is the root: the token that the
last round emitted (``pending``), whose logits decide between its children.

  tree_masks(parents)              ancestor bits and depths, once per tree
  tree_attention(q, ..., masks)    each layer's attention
  process_logits(logits, tokens, masks, ...)   penalties along each node's path
  tree_accept(tokens, choices, masks)          the accepted path and the next token
  commit_tree(...) / RaggedCache.commit_tree   the path's K and V to the row's end

``choices[b, i]`` is what the target draws behind node i from its own
distribution (``draft_sample`` on node i's logits; at temperature 0 the argmax).
A child is accepted when it holds its parent's choice, so every emitted token is a
draw from the target's distribution whatever the drafts were: the round is
lossless for trees of any origin.
"""
from typing import NamedTuple

import torch

from specdec import _lib as L

__all__ = ["TREE_MAX", "tree_masks", "tree_of_widths", "TreePath", "tree_accept"]

TREE_MAX = 256            # SD_TREE_MAX


class TreeMasks(NamedTuple):
    masks: torch.Tensor       # int32 [N, W] or [B, N, W]
    depths: torch.Tensor      # int32 [N] or [B, N]


def tree_masks(parents, device=None):
    """Ancestor bits and depths of trees.

    parents [N] (one tree for every row) or [B, N], integers: the parent of each
    node, which comes before its child; -1 for a root, any other negative number
    for a node that is not there (a row's tree may be smaller than the widest).
    Children of an absent node are absent, too.  ``device`` is needed for a list or
    a CPU tensor.  Returns (masks [.., N, ceil(N / 32)] int32: bit a of node i says
    that a is i or one of its ancestors; depths [.., N] int32: 0 for a root or an
    absent node).  At most TREE_MAX nodes.  Stream ordered.
    """
    if not torch.is_tensor(parents):
        parents = torch.tensor(parents, dtype=torch.int64)
    if parents.is_floating_point() or parents.is_complex() or parents.dtype == torch.bool:
        raise L.SpecdecError(f"parents must be integers, got {parents.dtype}")
    if parents.dim() not in (1, 2):
        raise L.SpecdecError(f"parents must be [N] or [B, N], got {tuple(parents.shape)}")
    if device is not None:
        parents = parents.to(device)
    if not parents.is_cuda:
        raise L.SpecdecError("tree_masks needs a CUDA device (no CPU fallback)")
    p = parents if parents.dim() == 2 else parents.unsqueeze(0)
    if p.dtype != torch.int32:
        p = p.long().clamp(-2, TREE_MAX).to(torch.int32)     # (8 bits do not hold the limits)
    if p.stride(1) != 1:
        p = p.contiguous()
    T, N = p.shape
    if not 1 <= N <= TREE_MAX:
        raise L.SpecdecError(f"a tree has 1 to {TREE_MAX} nodes, got {N}")
    W = -(-N // 32)
    masks = torch.empty(*parents.shape, W, dtype=torch.int32, device=p.device)
    depths = torch.empty(parents.shape, dtype=torch.int32, device=p.device)
    with L.on_device(p.device):
        L.check(L.lib().sd_tree_masks(p.data_ptr(), p.stride(0), T, N, masks.data_ptr(),
                                      depths.data_ptr(), L.stream_of(p.device)), "tree_masks")
    return TreeMasks(masks, depths)


def tree_of_widths(widths):
    """Parents of the tree whose nodes on level d have widths[d] children each:
    (parents list in breadth-first order, first node of each level and the end)."""
    parents, starts = [-1], [0, 1]
    for w in widths:
        if int(w) < 1:
            raise ValueError(f"every level needs at least one child per node, got {list(widths)}")
        parents += [p for p in range(starts[-2], starts[-1]) for _ in range(int(w))]
        starts.append(len(parents))
        if len(parents) > TREE_MAX:
            raise ValueError(f"the tree of widths {list(widths)} has more than {TREE_MAX} nodes")
    return parents, starts


def check_masks(masks, rows, name):
    """(words between rows' trees, N) of masks [N, W], [1, N, W] or [rows, N, W]."""
    if masks.dtype != torch.int32 or masks.dim() not in (2, 3):
        raise L.SpecdecError(f"{name}: masks must be int32 [N, W] or [B, N, W]")
    N, W = masks.shape[-2:]
    if not masks.is_contiguous() and ((W > 1 and masks.stride(-1) != 1)
                                      or (N > 1 and masks.stride(-2) != W)):
        raise L.SpecdecError(f"{name}: the words of a tree's masks must lie together")
    if not 1 <= N <= TREE_MAX or W != -(-N // 32):
        raise L.SpecdecError(f"{name}: a tree of N nodes (1 to {TREE_MAX}) has ceil(N / 32) words "
                             f"per node, got {tuple(masks.shape)}")
    if masks.dim() == 2 or masks.shape[0] == 1:
        return 0, N
    if masks.shape[0] != rows:
        raise L.SpecdecError(f"{name}: masks for {masks.shape[0]} trees, but {rows} rows")
    return masks.stride(0), N


class TreePath(NamedTuple):
    """What ``tree_accept`` returns."""
    n_acc: torch.Tensor       # int64 [B]: accepted drafts
    y: torch.Tensor           # int64 [B]: the token behind the path
    path: torch.Tensor        # int32 [B, max_path]: nodes from the root on, -1 behind


def _ids(t, shape, name):
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool or t.shape != shape:
        raise L.SpecdecError(f"{name} must be integers {tuple(shape)}, got {t.dtype} "
                             f"{tuple(t.shape)}")
    if t.dtype != torch.long:
        t = t.long()
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def tree_accept(tokens, choices, masks, alive=None, max_path=None):
    """The accepted path of each row's tree.

    tokens [B, N]: the drafted token of each node (node 0's is not looked at);
    choices [B, N]: the target's draw behind each node; masks as ``tree_masks``
    gives them.  From node 0 on, the path goes to the first child (lowest index) that
    holds its parent's choice, up to ``max_path`` nodes (default N; the tree's
    greatest depth + 1 is enough).  ``alive`` [B] bool: a row that is False stays at
    node 0.  Returns TreePath(n_acc, y, path): the row emits tokens[path[1:n_acc + 1]]
    and then y, the choice at the path's last node.  No host synchronisation.
    """
    if not (tokens.is_cuda and choices.is_cuda and masks.is_cuda):
        L.require_cuda(tokens, choices, masks)
    dev = tokens.device
    if choices.device != dev or masks.device != dev or (alive is not None and alive.device != dev):
        raise L.SpecdecError("tree_accept needs every tensor on one CUDA device")
    if tokens.dim() != 2:
        raise L.SpecdecError(f"tokens must be [B, N], got {tuple(tokens.shape)}")
    B, N = tokens.shape
    mask_bs, n = check_masks(masks, B, "tree_accept")
    if n != N:
        raise L.SpecdecError(f"tree_accept: {N} tokens per row, but masks of {n} nodes")
    tokens, choices = _ids(tokens, (B, N), "tokens"), _ids(choices, (B, N), "choices")
    P = N if max_path is None else int(max_path)
    if P < 1:
        raise L.SpecdecError(f"max_path must be at least 1, got {max_path}")
    if alive is not None:
        if alive.shape != (B,):
            raise L.SpecdecError(f"alive must be [{B}], got {tuple(alive.shape)}")
        alive = alive.to(torch.uint8).contiguous()
    path = torch.empty(B, P, dtype=torch.int32, device=dev)
    out = torch.empty(2, B, dtype=torch.long, device=dev)
    n_acc, y = out[0], out[1]
    with L.on_device(dev):
        L.check(L.lib().sd_tree_accept(
            tokens.data_ptr(), tokens.stride(0), choices.data_ptr(), choices.stride(0),
            masks.data_ptr(), mask_bs, L.address(alive), B, N, P, path.data_ptr(),
            n_acc.data_ptr(), y.data_ptr(), L.stream_of(dev)), "tree_accept")
    return TreePath(n_acc, y, path)
