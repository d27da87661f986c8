"""Several drafted tokens at a time over a layer's cache, and caches that give up keys.

    softmax_tree_step(q, k, v, cache, parents, ...)   a softmax layer's attention of a tree of drafted tokens; a single token
                                                      with capped scores or a distance bias is a tree of one
    dilution_tree_step(q, k, v, cache, parents)       the dilution operator's: each node's bids meet the demand of the cached
                                                      tokens and of its ancestors, as a chain of decode steps would
    tree_accept(cache, draft, path)                   the accepted branch joins the cache: rows, demand and length
    evict_cache(cache, keep, ...)                     the keys that were bid for least leave the cache

A cache is the model's dict {"k", "v", "len"[, "committed"]} that the decode steps take.  Tree steps only read it, so a
draft that is rejected leaves nothing behind.  With a tree {x: parent of x}, node x sees the cached keys, its ancestors and
itself, and stands at position len + depth(x) (depth 0 follows the last cached token):

    p_x       = softmax over those keys of the scores
    demand_x  = committed + sum of p_a over the ancestors a of x                 (dilution)
    share_x   = p_x / (demand_x + p_x + eps);   out_x = (share_x / (sum share_x + eps)) V
"""

from __future__ import annotations

import functools
import math

import torch

from . import _lib
from . import kernels as K
from .masked import _CODE, _DIMS, aligned, check_slopes, check_softcap, on_device

MAX_NODES = 64


@functools.lru_cache(maxsize=256)
def _scratch_bytes(*sizes) -> int:
    return _lib.load().dilution_tree_scratch_bytes(*sizes)


def _cache(cache, batch, heads, dim, dtype, device):
    """(k, v, capacity, length) of a cache whose rows the kernels read by their addresses."""
    k, v, length = cache["k"], cache["v"], cache["len"]
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or shape[0] != batch or shape[1] != heads or shape[3] != dim:
        raise ValueError("the caches are (batch, key heads, capacity, head_dim), like the drafted keys")
    if k.dtype != dtype or v.dtype != dtype or k.device != device or v.device != device:
        raise ValueError("the caches must have the drafted tokens' dtype and device")
    capacity = shape[2]
    if not 0 <= length <= capacity or capacity < 1:
        raise ValueError(f"length {length} outside cache capacity {capacity}")
    k, v = K._cache_rows(k, batch, heads, capacity, dim), K._cache_rows(v, batch, heads, capacity, dim)
    if (k.data_ptr() | v.data_ptr()) % 16:
        raise RuntimeError("the caches must start on a 16-byte boundary")
    return k, v, capacity, length


def _demand(x, batch, heads, capacity, device, name="committed"):
    if x.dtype != torch.float32 or x.device != device or tuple(x.shape) != (batch, heads, capacity) or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape {(batch, heads, capacity)}")
    return x


def _indices(x, batch, name, device):
    """(int32 tensor on the device, stride between sequences, the host's copy or None) of a list, (N,) or (B, N)."""
    host = None
    if isinstance(x, torch.Tensor) and x.is_cuda and x.dtype == torch.int32 and x.is_contiguous() and x.device == device:
        shape = x.shape
        if len(shape) == 1:
            return x, 0, None
        if len(shape) == 2 and shape[0] == batch:
            return x, shape[1], None
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        x = torch.as_tensor(x)
        if x.numel() == 0:
            x = x.to(torch.int64)
        if x.dtype in (torch.int32, torch.int64):
            host = x.tolist()
        x = x.to(device)
    if x.dtype not in (torch.int32, torch.int64) or x.dim() not in (1, 2) or (x.dim() == 2 and x.shape[0] != batch):
        raise ValueError(f"{name} must be whole numbers, (nodes,) for all sequences or (batch, nodes)")
    if x.device != device:
        raise ValueError(f"{name} must be on q's device (or on the host)")
    stride = x.shape[1] if x.dim() == 2 else 0
    if x.dtype == torch.int64:                 # (what lies outside every tree may not wrap into one)
        x = x.clamp(-1, MAX_NODES)
    return x.to(torch.int32).contiguous(), stride, host


def _trees(host):
    return host if host and isinstance(host[0], list) else [host]


def _draft(q, k, v, cache, parents):
    """The checks that both tree steps share, and the draft that tree_accept takes."""
    if not q.is_cuda:
        raise RuntimeError("tree steps need CUDA tensors (no CPU fallback in this backend)")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:]:
        raise ValueError("q is (batch, heads, nodes, head_dim), k and v the same with as many heads as the cache")
    batch, heads, nodes, dim = q.shape
    kv_heads = k.shape[1]
    if kv_heads < 1 or heads % kv_heads or batch < 1:
        raise ValueError(f"{kv_heads} key heads do not divide {heads} query heads")
    if q.dtype not in _CODE or k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be all float32 or all bfloat16, on one device")
    if dim not in _DIMS:
        raise ValueError(f"head_dim {dim} not in {_DIMS}")
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, not {nodes}")
    parents, stride, host = _indices(parents, batch, "parents", q.device)
    if parents.shape[-1] != nodes:
        raise ValueError(f"{parents.shape[-1]} parents for {nodes} nodes")
    if host is not None and any(not -1 <= up < x for tree in _trees(host) for x, up in enumerate(tree)):
        raise ValueError("a node's parent is an earlier node, or -1")
    kc, vc, capacity, length = _cache(cache, batch, kv_heads, dim, q.dtype, q.device)
    pos_dev = cache.get("pos_dev")
    draft = dict(q=aligned(q), k=aligned(k), v=aligned(v), parents=parents, parent_stride=stride, tree=host, len=length,
                 softcap=0.0, slopes=None, lse=torch.empty(batch, heads, nodes, device=q.device, dtype=torch.float32))
    sizes = (batch, heads, kv_heads, nodes, dim, capacity, length)
    return draft, sizes, (kc, vc), pos_dev


def _buffers(sizes, pos_dev, like, out, scratch):
    batch, heads, kv_heads, nodes, dim, capacity, length = sizes
    if out is None:
        out = torch.empty(like.shape, device=like.device, dtype=like.dtype)
    elif out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor like q")
    need = _scratch_bytes(batch, kv_heads, heads // kv_heads, nodes, capacity if pos_dev is not None else length, dim)
    if scratch is None or scratch.numel() * scratch.element_size() < need or scratch.data_ptr() % 16 or not scratch.is_contiguous() \
            or scratch.device != like.device:
        scratch = torch.empty(need, device=like.device, dtype=torch.uint8)
    return out, scratch


def softmax_tree_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: dict, parents, softcap: float | None = None,
                      slopes: torch.Tensor | None = None, out: torch.Tensor | None = None,
                      scratch: torch.Tensor | None = None):
    """Softmax attention of a tree of drafted tokens over a cache.  Returns (out, draft).

    q: (B, H, N, D), N <= 64; k, v: (B, H_kv, N, D) of the drafted tokens, rotated for their positions len + depth where
    the layer rotates; cache: {"k", "v", "len"} with H_kv heads.  parents: (N,), or (B, N) for a tree of each sequence: the
    earlier node that a node follows, -1 for the last cached token (a device tensor is not checked: any other number counts
    as -1).  softcap and slopes as in softmax_attention, by the distance of the positions (no slopes over a cache that keys
    were evicted from).  out and scratch are optional buffers.  out: (B, H, N, D) in q's dtype; draft is for tree_accept, and
    refers to q, k, v and parents: they stay as they are until then.  The cache is only read; with cache["pos_dev"] its
    length is read from the device, so that the step can be recorded into a CUDA graph.
    """
    draft, sizes, (kc, vc), pos_dev = _draft(q, k, v, cache, parents)
    batch, heads, kv_heads, nodes, dim, capacity, length = sizes
    draft["softcap"], draft["slopes"] = check_softcap(softcap), check_slopes(slopes, heads, q.device)
    if slopes is not None and cache.get("evicted"):
        raise ValueError("a cache that keys were evicted from does not know its keys' positions, which slopes need")
    lib = _lib.load()
    out, scratch = _buffers(sizes, pos_dev, q, out, scratch)
    with on_device(q.device):
        _lib.check(lib.dilution_tree_softmax(
            draft["q"].data_ptr(), draft["k"].data_ptr(), draft["v"].data_ptr(), kc.data_ptr(), vc.data_ptr(), _CODE[q.dtype], batch,
            kv_heads, heads // kv_heads, nodes, capacity, length, K._ptr(pos_dev), dim, 1.0 / math.sqrt(dim), draft["softcap"],
            K._ptr(draft["slopes"]), draft["parents"].data_ptr(), draft["parent_stride"], draft["lse"].data_ptr(), out.data_ptr(),
            scratch.data_ptr(), K._stream(q.device)), "dilution_tree_softmax")
    return out, draft


def dilution_tree_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: dict, parents,
                       out: torch.Tensor | None = None, scratch: torch.Tensor | None = None):
    """The dilution operator for a tree of drafted tokens over a cache with its demand.  Returns (out, draft).

    As softmax_tree_step, with as many key heads as query heads and cache["committed"] (B, H, capacity) fp32.  Every node's
    row is what dilution_decode_append_step gives at the end of its branch; the demand itself is not advanced, which
    tree_accept does for the branch that is accepted.
    """
    draft, sizes, (kc, vc), pos_dev = _draft(q, k, v, cache, parents)
    batch, heads, kv_heads, nodes, dim, capacity, length = sizes
    if kv_heads != heads:
        raise ValueError("a dilution layer has as many key heads as query heads")
    if cache.get("committed") is None:
        raise ValueError("a dilution layer's cache holds the committed demand of its keys")
    committed = _demand(cache["committed"], batch, heads, capacity, q.device)
    lib = _lib.load()
    out, scratch = _buffers(sizes, pos_dev, q, out, scratch)
    with on_device(q.device):
        _lib.check(lib.dilution_tree_dilute(
            draft["q"].data_ptr(), draft["k"].data_ptr(), draft["v"].data_ptr(), kc.data_ptr(), vc.data_ptr(), _CODE[q.dtype], batch,
            heads, nodes, capacity, length, K._ptr(pos_dev), dim, 1.0 / math.sqrt(dim), K.EPS, committed.data_ptr(),
            draft["parents"].data_ptr(), draft["parent_stride"], draft["lse"].data_ptr(), out.data_ptr(), scratch.data_ptr(),
            K._stream(q.device)), "dilution_tree_dilute")
    return out, draft


def tree_accept(cache: dict, draft: dict, path, out: torch.Tensor | None = None):
    """The nodes `path` of a draft join the cache that it was drafted over; returns the advanced demand, or None.

    path: (A,), or (B, A) for each sequence its own: the accepted nodes, each the parent of the next.  Their keys and values
    go to the cache's rows len .. len + A - 1, cache["len"] grows by A, and cache["committed"], if the cache has it, advances
    by their bids (for a softmax layer: by their attention weights, summed over the heads that share a key head), in place
    or into `out`, a buffer like it whose rows behind the new length are left as they are.  On a host tensor or a list
    the path is checked against the tree; on the device an index outside the tree counts as its nearest node.  With
    cache["pos_dev"] the caller advances that count (a cache that GraphedDecode steps is closed there first).
    """
    q = draft["q"]
    batch, heads, nodes, dim = q.shape
    kv_heads = draft["k"].shape[1]
    kc, vc, capacity, length = _cache(cache, batch, kv_heads, dim, q.dtype, q.device)
    pos_dev = cache.get("pos_dev")
    if pos_dev is None and length != draft["len"]:
        raise ValueError(f"the draft was made over {draft['len']} keys, the cache holds {length}")
    path, stride, host = _indices(path, batch, "path", q.device)
    accepted = path.shape[-1]
    if accepted > nodes:
        raise ValueError(f"{accepted} accepted nodes of {nodes}")
    if length + accepted > capacity:
        raise ValueError("accepted tokens past the cache capacity (context_length)")
    if host is not None:
        for row, nodes_taken in enumerate(_trees(host)):
            if any(not 0 <= x < nodes for x in nodes_taken):
                raise ValueError(f"path leaves the tree of {nodes} nodes")
            if draft["tree"] is not None:
                trees = _trees(draft["tree"])
                for tree in [trees[row]] if len(trees) > 1 and len(_trees(host)) > 1 else trees:
                    if any(tree[x] != up for x, up in zip(nodes_taken, [-1, *nodes_taken])):
                        raise ValueError("path must be a branch of the tree: each node the parent of the next")
    committed = cache.get("committed")
    if committed is not None:
        committed = _demand(committed, batch, kv_heads, capacity, q.device)
        out = committed if out is None else _demand(out, batch, kv_heads, capacity, q.device, "out")
    elif out is not None:
        raise ValueError("the cache keeps no demand that out could receive")
    if accepted == 0:
        if out is not committed:
            out[:, :, :length].copy_(committed[:, :, :length])
        return out
    lib = _lib.load()
    with on_device(q.device):
        _lib.check(lib.dilution_tree_accept(
            q.data_ptr(), draft["k"].data_ptr(), draft["v"].data_ptr(), kc.data_ptr(), vc.data_ptr(), _CODE[q.dtype], batch, kv_heads,
            heads // kv_heads, nodes, capacity, length, K._ptr(pos_dev), dim, 1.0 / math.sqrt(dim), draft["softcap"],
            K._ptr(draft["slopes"]), draft["parents"].data_ptr(), draft["parent_stride"], draft["lse"].data_ptr(), path.data_ptr(), stride,
            accepted, K._ptr(committed), K._ptr(out), K._stream(q.device)), "dilution_tree_accept")
    cache["len"] = length + accepted
    return out


def evict_cache(cache: dict, keep: int, recent: int = 0, sinks: int = 0, scores: torch.Tensor | None = None,
                capacity: int | None = None) -> dict:
    """A cache with the `keep` keys of each (batch, head) row that were bid for most; the given one is only read.

    The first `sinks` keys and the last `recent` stay whatever they are; of those between, the ones of the highest
    cache["committed"] (or `scores`, (B, H, at least len) fp32, for caches without it), equal ones by position, NaN above
    every number.  They stay in their order.  Returns {"k", "v", "len": keep, "committed" if the cache has it, "index":
    (B, H, keep) int32 positions that stayed, "evicted": how many tokens the cache has lost in all}, with room for
    `capacity` tokens (the cache's own by default), zeros behind the kept ones.  The next token's position is len + evicted,
    which the cached steps of this library's layers rotate by.
    """
    k = cache["k"]
    if not k.is_cuda:
        raise RuntimeError("evict_cache needs CUDA tensors (no CPU fallback in this backend)")
    if k.dim() != 4 or k.dtype not in _CODE:
        raise ValueError("the caches are (batch, heads, capacity, head_dim), float32 or bfloat16")
    if cache.get("pos_dev") is not None:
        raise ValueError("a cache whose length is on the device cannot be cut; close the recorded decode first")
    batch, heads, _, dim = k.shape
    if dim not in _DIMS:
        raise ValueError(f"head_dim {dim} not in {_DIMS}")
    kc, vc, old, length = _cache(cache, batch, heads, dim, k.dtype, k.device)
    if not 1 <= keep <= length:
        raise ValueError(f"keep {keep} of {length} keys")
    if recent < 0 or sinks < 0 or recent + sinks > keep:
        raise ValueError(f"{recent} recent and {sinks} first keys do not fit the {keep} that stay")
    capacity = old if capacity is None else capacity
    if capacity < keep:
        raise ValueError(f"capacity {capacity} below the {keep} keys that stay")
    committed = cache.get("committed")
    if committed is not None:
        committed = _demand(committed, batch, heads, old, k.device)
    if scores is None:
        if committed is None:
            raise ValueError("a cache without committed demand needs scores")
        scores = committed
    if scores.dim() != 3 or scores.shape[:2] != (batch, heads) or scores.shape[2] < length or scores.dtype != torch.float32 \
            or scores.device != k.device:
        raise ValueError(f"scores must be float32, ({batch}, {heads}, at least {length})")
    scores = scores.contiguous()
    kept = {x: torch.empty(batch, heads, capacity, dim, device=k.device, dtype=k.dtype) for x in ("k", "v")}
    kept["len"] = keep
    if committed is not None:
        kept["committed"] = torch.empty(batch, heads, capacity, device=k.device, dtype=torch.float32)
    kept["index"] = torch.empty(batch, heads, keep, device=k.device, dtype=torch.int32)
    kept["evicted"] = cache.get("evicted", 0) + length - keep
    lib = _lib.load()
    with on_device(k.device):
        _lib.check(lib.dilution_evict(
            kc.data_ptr(), vc.data_ptr(), K._ptr(committed), _CODE[k.dtype], batch * heads, old, length, dim, scores.data_ptr(),
            scores.shape[2], keep, recent, sinks, capacity, kept["k"].data_ptr(), kept["v"].data_ptr(),
            K._ptr(kept.get("committed")), kept["index"].data_ptr(), K._stream(k.device)), "dilution_evict")
    return kept
