"""int64 arguments whose values do not fit 32 bits: a negative document is padding, a prefix past the row is the whole row, and parents and
paths outside the tree are what the documentation says, however large they are."""

from __future__ import annotations

import pytest
import torch

from test_gpu_masked import DEV, call, inputs

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
