"""Cached keys and values that are not finite under tree steps: what they reach, what stays as it was, and how long it takes."""

from __future__ import annotations

import pytest
import torch

from conftest import load_package, seeded
from oracle import operators_oracle as O
from test_gpu_trees import DEV, TREE, TYPES, case, within

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("heads,length", [(2, 150), (40, 150), (2, 9000)])
@pytest.mark.parametrize("at", [0, 77, 149])
def test_an_infinite_key(at, heads, length, dtype, dim):
    """Scores of +inf make no number of a node, and of the nodes that come after it in a dilution layer; scores of -inf are a key that is not
    there."""
    lib = load_package()
    q, k, v, cache = case(1, heads, heads, len(TREE), dim, length, dtype)
    short = {x: torch.cat((cache[x][:, :, :at], cache[x][:, :, at + 1:]), 2) for x in ("k", "v", "committed")}
    cache["k"][:, :, at, 3] = INF
    below = q[0, :, :, 3] < 0
    line = below.clone()
    for x, up in enumerate(TREE):
        if up >= 0:
            line[:, x] &= line[:, up]
    some = [0, 1]
    for name, step, good in (("softmax", lib.softmax_tree_step, below), ("dilution", lib.dilution_tree_step, line)):
        out, draft = step(q, k, v, cache, TREE)
        assert torch.equal(torch.isfinite(out[0]), good[..., None].expand_as(out[0])), name
        assert torch.equal(torch.isfinite(draft["lse"][0]), below), name
        want, off = O.tree_nodes(q[:, some], k[:, some], v[:, some], short["k"][:, some], short["v"][:, some], length - 1, TREE,
                                 committed=short["committed"][:, some] if name == "dilution" else None)[:2]
        keep = good[None, some]
        within(out[:, some][keep], want[keep], off[keep])


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("heads", [2, 40])
@pytest.mark.parametrize("value", [INF, -INF, float("nan")])
def test_a_value(value, heads, dtype, dim):
    """One feature of a cached value: the nodes' other features are as they were, and so are lse and the bids."""
    lib = load_package()
    q, k, v, cache = case(1, heads, heads, len(TREE), dim, 150, dtype)
    for step in (lib.softmax_tree_step, lib.dilution_tree_step):
        clean, draft = step(q, k, v, cache, TREE)
        bad = dict(cache, v=cache["v"].clone())
        bad["v"][:, :, 60, 3] = value
        out, other = step(q, k, v, bad, TREE)
        assert torch.equal(out[..., 3], torch.full_like(out[..., 3], value)) or value != value and out[..., 3].isnan().all()
        rest = [x for x in range(dim) if x != 3]
        # (a softmax step's rows are computed again, in another order)
        u = 2 * (2.0 ** -8 if dtype == torch.bfloat16 else (150 + len(TREE) + dim + 64) * 2.0 ** -24)
        spread = 2 * cache["v"][:, :, :150].double().abs().amax()
        assert ((out - clean)[..., rest].double().abs() <= u * spread).all()
        assert ((draft["lse"] - other["lse"]).abs() <= 2.0 ** -18 * draft["lse"].abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("nodes", [12, 64])
@pytest.mark.parametrize("where,value", [("k", INF), ("k", float("nan")), ("v", INF)])
def test_they_take_no_long_time(where, value, nodes):
    """16384 keys: a warp walks over them once for each of its nodes (12 nodes: 16 warps; 64: four each), under 0.25 us a key (0.09 of it
    on one B200; one key at a time took 0.35)."""
    lib = load_package()
    tree = list(range(-1, nodes - 1))
    q, k, v = (seeded((1, 8, nodes, 64), s).to(DEV, torch.bfloat16) for s in range(3))
    cache = {x: seeded((1, 8, 16384 + 64, 64), s).to(DEV, torch.bfloat16) for s, x in ((3, "k"), (4, "v"))}
    cache.update(len=16384, committed=torch.ones(1, 8, 16384 + 64, device=DEV))
    cache[where][:, :, 16383, 5] = value
    for step in (lib.softmax_tree_step, lib.dilution_tree_step):
        times = []
        for _ in range(4):
            start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            step(q, k, v, cache, tree)
            stop.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(stop))
        assert min(times) <= 0.3 + (1 if nodes <= 16 else 4) * 16384 * 0.25e-3, times
