"""int64 arguments whose values do not fit 32 bits: a negative document is padding, a prefix past the row is the whole row, and parents and
paths outside the tree are what the documentation says, however large they are."""

from __future__ import annotations

import pytest
import torch

from conftest import load_package
from test_gpu_masked import DEV, call, inputs
from test_gpu_trees import case

pytestmark = pytest.mark.gpu
BIG = 1 << 32


@pytest.mark.parametrize("dim", [32, 64])
def test_documents_and_prefixes(dim):
    x = inputs(2, 2, 2, 150, dim, torch.bfloat16)
    docs = torch.arange(150, device=DEV).div(40, rounding_mode="floor").repeat(2, 1)
    docs[:, 100:] = -1
    far = torch.where(docs < 0, -BIG, docs)
    assert all(torch.equal(a, b) for a, b in zip(call(x, documents=docs), call(x, documents=far)))
    for prefix, same in (([BIG, -BIG], [150, 0]), ([BIG + 7, (1 << 31) + 5], [150, 150])):
        got, want = (call(x, prefix=torch.tensor(p, device=DEV)) for p in (prefix, same))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for prefix, same in ((1 << 40, 150), (-(1 << 40), 0)):
        assert all(torch.equal(a, b) for a, b in zip(call(x, prefix=prefix), call(x, prefix=same)))


def test_parents_and_paths():
    lib = load_package()
    q, k, v, cache = case(1, 2, 2, 5, 64, 100, torch.bfloat16)
    got, draft = lib.dilution_tree_step(q, k, v, cache, torch.tensor([BIG, BIG, BIG + 1, 2 - BIG, 3], device=DEV))
    want, _ = lib.dilution_tree_step(q, k, v, cache, [-1, -1, -1, -1, 3])
    assert torch.equal(got, want)
    lib.tree_accept(cache, draft, torch.tensor([-BIG + 3, BIG + 2], device=DEV))
    assert torch.equal(cache["k"][:, :, 100], k[:, :, 0]) and torch.equal(cache["k"][:, :, 101], k[:, :, 4])
