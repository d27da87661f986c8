"""softmax_attention and softmax_tree_step with slopes of either sign: the bias is -slope |i - j| in every tile, masked or not, forward and backward.  Heads of
64 above 2560 tokens without documents have backward kernels of their own, which these lengths reach as well."""

from __future__ import annotations

import pytest
import torch

from conftest import load_package
from oracle import operators_oracle as O
from test_gpu_masked import DEV, TYPES, call, check, documents_of, inputs
from test_gpu_trees import CHAINS, TREE, case, check_accept, clone, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim", TYPES)
def test_slopes_of_both_signs(dtype, dim):
    check(inputs(2, 3, 3, 300, dim, dtype), slopes=torch.tensor([-0.25, 0.1, -2.0 ** -6], device=DEV))


@pytest.mark.parametrize("dtype,dim", TYPES)
def test_slopes_of_both_signs_with_every_mask(dtype, dim):
    check(inputs(2, 4, 2, 391, dim, dtype, q_scale=2.0), softcap=15.0, slopes=torch.tensor([-0.3, 0.1, -0.03, 0.01], device=DEV),
          documents=documents_of(2, 391, 90, seed=5, pad=20), prefix=torch.tensor([150, 77], device=DEV, dtype=torch.int32))


@pytest.mark.parametrize("dtype,dim", TYPES[:4])
@pytest.mark.parametrize("prefix", [100, 270])
def test_a_negative_slope_over_a_prefix(prefix, dtype, dim):
    """Keys on both sides of a query, and tiles of them without a mask."""
    check(inputs(1, 2, 1, 270, dim, dtype), slopes=torch.tensor([-0.125, 0.125], device=DEV),
          prefix=torch.tensor([prefix], device=DEV))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seq", [2561, 2900])
@pytest.mark.parametrize("options", [{}, {"slopes": [-0.02, 0.05]}, {"softcap": 12.0, "slopes": [0.02, -0.01], "prefix": 700}])
def test_long_rows_without_documents(options, seq, dim):
    options = dict(options)
    if "slopes" in options:
        options["slopes"] = torch.tensor(options["slopes"], device=DEV)
    if "prefix" in options:
        options["prefix"] = torch.tensor([options["prefix"]], device=DEV)
    check(inputs(1, 2, 1, seq, dim, torch.bfloat16, q_scale=2.0), **options)


def test_long_rows_repeat():
    x = inputs(1, 4, 2, 3333, 64, torch.bfloat16)
    slopes = torch.tensor([-0.01, 0.0, 0.02, 0.3], device=DEV)
    first = call(x, slopes=slopes)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call(x, slopes=slopes)))


def test_a_prefix_that_is_one_number():
    x = inputs(2, 2, 2, 200, 64, torch.bfloat16)
    want = call(x, prefix=torch.tensor([90, 90], device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(want, call(x, prefix=90)))
    assert load_package().softmax_attention(*x[:3], prefix=0).shape == x[0].shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_arguments_in_other_forms(dtype):
    """Slopes of other types and as a list, documents and prefixes that are views with strides."""
    x = inputs(2, 4, 2, 150, 64, torch.bfloat16)
    slopes = torch.tensor([-0.25, 0.125, 0.5, -0.0625], device=DEV)
    docs = documents_of(2, 150, 40, seed=3, pad=5)
    prefix = torch.tensor([20, 90], device=DEV)
    want = call(x, slopes=slopes, documents=docs, prefix=prefix)
    strided = torch.stack((docs, docs + 7), 2).transpose(0, 1).contiguous().transpose(0, 1)[..., 0]
    apart = torch.stack((prefix, prefix + 1), 1)[:, 0]
    assert not strided.is_contiguous() and not apart.is_contiguous()
    for some in (slopes.to(dtype), slopes.tolist(), slopes.to(dtype)[:, None].expand(4, 2)[:, 1]):
        assert all(torch.equal(a, b) for a, b in zip(want, call(x, slopes=some, documents=strided, prefix=apart)))


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("length", [0, 150, 5000])
def test_trees_with_slopes_of_both_signs(length, dtype, dim):
    """Over a cache: with a negative slope the first keys have the largest scores, which a scan comes to last."""
    q, k, v, cache = case(1, 4, 2, len(TREE), dim, length, dtype)
    slopes = torch.tensor([-0.25, 0.5, -0.001, 0.01], device=DEV)
    out, draft = load_package().softmax_tree_step(q, k, v, cache, TREE, slopes=slopes)
    want, off, bids, bids_off = O.tree_nodes(q, k, v, cache["k"], cache["v"], length, TREE, slopes=slopes)
    within(out, want, off)
    before, path = clone(cache), CHAINS["leaf"]
    load_package().tree_accept(cache, draft, path)
    check_accept(before, cache, k, v, bids, bids_off, [path], length)
