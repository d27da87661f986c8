"""Caps far above the scores, which they then leave as they are: softmax_attention and softmax_tree_step, with bounds that count the
cap's error by the score and not by the cap (oracle/operators_oracle.py)."""

from __future__ import annotations

import pytest
import torch

from conftest import load_package
from oracle import operators_oracle as O
from test_gpu_masked import DEV, check, documents_of, inputs
from test_gpu_trees import TREE, case, within

pytestmark = pytest.mark.gpu
TYPES = [(torch.bfloat16, 16), (torch.bfloat16, 32), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 32)]


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("cap", [1.0, 1e4, 1e6, 1e20, 1e38])
def test_attention(cap, dtype, dim):
    check(inputs(1, 2, 1, 150, dim, dtype, q_scale=2.0), softcap=cap, documents=documents_of(1, 150, 60, seed=1, pad=9))


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("cap", [1.0, 1e4, 1e6, 1e20, 1e38])
def test_tree_steps(cap, dtype, dim):
    q, k, v, cache = case(1, 4, 2, len(TREE), dim, 150, dtype, q_scale=2.0)
    slopes = torch.tensor([0.5, 0.1, 0.01, 0.0], device=DEV)
    out, draft = load_package().softmax_tree_step(q, k, v, cache, TREE, softcap=cap, slopes=slopes)
    want, off, bids, bids_off = O.tree_nodes(q, k, v, cache["k"], cache["v"], 150, TREE, softcap=cap, slopes=slopes)
    within(out, want, off)
    before = cache["committed"].clone()
    load_package().tree_accept(cache, draft, [0, 1, 3])
    taken, far = (x[:, :, [0, 1, 3]][..., :150].unflatten(1, (2, 2)).sum((2, 3)) for x in (bids, bids_off))
    taken = taken + before[:, :, :150].double()
    within(cache["committed"][:, :, :150], taken, far + 2.0 ** -18 * taken + 1e-9)


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("cap", [1e4, 1e6])
def test_a_row_past_the_cap_beside_ordinary_ones(cap, dtype, dim):
    """One query in 40 has scores beyond the cap; its neighbours' stay as exact as without it."""
    q, k, v, dout = inputs(1, 2, 2, 200, dim, dtype)
    q[:, :, ::40] *= 8 * cap
    check((q, k, v, dout), softcap=cap)


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("cap", [1e4, 1e6])
def test_a_node_past_the_cap_beside_ordinary_ones(cap, dtype, dim):
    q, k, v, cache = case(1, 2, 2, len(TREE), dim, 150, dtype)
    q[:, :, 5] *= 8 * cap
    out, _ = load_package().softmax_tree_step(q, k, v, cache, TREE, softcap=cap)
    within(out, *O.tree_nodes(q, k, v, cache["k"], cache["v"], 150, TREE, softcap=cap)[:2])


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("cap", [1e-30, 1e-3])
def test_small_caps(cap, dtype, dim):
    """All weights alike: nothing is left of the scores."""
    check(inputs(1, 2, 1, 150, dim, dtype), softcap=cap, documents=documents_of(1, 150, 60, seed=1, pad=9))
