"""Ranges of the arguments of softmax_attention and the tree steps: what does not fit 32 bits is refused or held, never wrapped (no GPU
needed)."""

from __future__ import annotations

import pytest
import torch

from conftest import load_package
from test_operator_refusals import attend, caches, fake, message, tree


@pytest.mark.parametrize("cap", [1e-50, 1e-31, 2.5e38, 1e39, float("inf")])
def test_caps_that_32_bits_do_not_hold(cap):
    lib = load_package()
    q, k = fake(1, 4, 8, 64), fake(1, 2, 8, 64)
    with pytest.raises(ValueError, match="softcap"):
        lib.softmax_attention(q, k, k, softcap=cap)
    with pytest.raises(ValueError, match="softcap"):
        lib.softmax_tree_step(q, k, k, caches(), list(range(-1, 7)), softcap=cap)


@pytest.mark.parametrize("cap", [1e-40, 9e-31, 1.1e38, 2.5e38])
def test_caps_of_the_entries(cap):
    for rc in (attend(cap=cap), tree(softcap=cap)):
        assert rc == 1 and "cap" in message(rc)
