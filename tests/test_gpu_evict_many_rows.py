"""evict_cache over so many rows that a row's cluster moves its keys itself: one CTA a row, and clusters of two to eight whose CTAs move
places that others of them have written."""

from __future__ import annotations

import pytest
import torch

from test_gpu_evict import DEV, cache_of, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 16), (torch.float32, 128)])
@pytest.mark.parametrize("length,keep,recent,sinks", [(1, 1, 0, 0), (37, 20, 3, 2), (300, 299, 0, 0), (300, 1, 0, 0), (900, 333, 100, 4)])
@pytest.mark.parametrize("room", [0, 70])
def test_a_cta_a_row(length, keep, recent, sinks, room, dtype, dim):
    check(cache_of(10, 15, length, dim, dtype), keep, recent, sinks, capacity=keep + room)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 16)])
@pytest.mark.parametrize("batch,heads,length,keep", [(5, 8, 2049, 700), (5, 8, 1999, 1998), (19, 4, 3001, 1234), (4, 5, 2500, 2), (2, 19, 33000, 4001)])
def test_clusters(batch, heads, length, keep, dtype, dim):
    check(cache_of(batch, heads, length, dim, dtype), keep, min(keep, 20), 0, capacity=keep + 37)


@pytest.mark.parametrize("batch,heads,length,keep", [(10, 15, 300, 100), (5, 8, 3000, 1500)])
def test_equal_ranks(batch, heads, length, keep):
    cache = cache_of(batch, heads, length, 32, torch.bfloat16)
    cache["committed"] = torch.round(cache["committed"] * 2) / 2
    check(cache, keep, recent=3, sinks=1)
    cache["committed"].zero_()
    check(cache, keep)


def test_scores_in_place_of_the_demand():
    cache = cache_of(5, 8, 2100, 64, torch.bfloat16)
    scores = cache.pop("committed").flip(2).contiguous()
    assert scores.device.type == DEV
    check(cache, 999, scores=scores, capacity=1111)
