"""evict_cache: which keys stay, their order, ties, ranks that are not finite, and what the new cache holds."""

from __future__ import annotations

import pytest
import torch

from conftest import load_package, seeded
from oracle import operators_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def cache_of(batch, heads, length, dim, dtype, seed=0, room=5):
    shape = (batch, heads, length + room, dim)
    return dict(k=seeded(shape, seed).to(DEV, dtype), v=seeded(shape, seed + 1).to(DEV, dtype), len=length,
                committed=seeded(shape[:3], seed + 2).abs().to(DEV))


def same_bits(a, b):
    """Equal, NaN and the sign of zero included."""
    bits = torch.int16 if a.dtype == torch.bfloat16 else torch.int32
    return torch.equal(a.contiguous().view(bits), b.contiguous().view(bits))


def check(cache, keep, recent=0, sinks=0, scores=None, capacity=None):
    before = {x: y.clone() for x, y in cache.items() if isinstance(y, torch.Tensor)}
    length = cache["len"]
    kept = load_package().evict_cache(cache, keep, recent=recent, sinks=sinks, scores=scores, capacity=capacity)
    for x, y in before.items():
        assert same_bits(cache[x], y)
    ranks = (cache["committed"] if scores is None else scores)[:, :, :length]
    index = kept["index"]
    assert index.dtype == torch.int32
    assert torch.equal(index.long().cpu(), O.evicted(ranks.cpu(), keep, recent, sinks))
    rows = index.long()[..., None].expand(-1, -1, -1, cache["k"].shape[-1])
    for x in ("k", "v"):
        assert torch.equal(kept[x][:, :, :keep], torch.gather(cache[x], 2, rows)) and (kept[x][:, :, keep:] == 0).all()
        assert kept[x].shape[2] == (cache["k"].shape[2] if capacity is None else capacity)
    if "committed" in cache:
        assert same_bits(kept["committed"][:, :, :keep], torch.gather(cache["committed"], 2, index.long()))
        assert (kept["committed"][:, :, keep:] == 0).all()
    else:
        assert "committed" not in kept
    assert kept["len"] == keep and kept["evicted"] == length - keep
    return kept


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 16), (torch.bfloat16, 128), (torch.float32, 128)])
@pytest.mark.parametrize("length,keep,recent,sinks", [(1, 1, 0, 0), (2, 1, 0, 0), (2, 1, 1, 0), (100, 37, 0, 0), (100, 100, 0, 0),
                                                      (511, 200, 50, 4), (512, 1, 0, 1), (513, 512, 0, 0), (1025, 30, 30, 0),
                                                      (4099, 1000, 100, 4), (4099, 50, 25, 25)])
def test_sizes(dtype, dim, length, keep, recent, sinks):
    check(cache_of(2, 3, length, dim, dtype), keep, recent, sinks)


@pytest.mark.parametrize("length,keep", [(20000, 7777), (70001, 60000)])
def test_long_rows_in_clusters(length, keep):
    check(cache_of(1, 2, length, 16, torch.bfloat16), keep, recent=99, sinks=3, capacity=keep)


def test_a_row_too_long_to_be_held():
    cache = cache_of(1, 1, 400003, 16, torch.bfloat16)
    check(cache, 100001, recent=5, capacity=100001)


@pytest.mark.parametrize("length,keep", [(300, 100), (3000, 1500), (9000, 10)])
def test_equal_ranks_go_by_position(length, keep):
    cache = cache_of(2, 2, length, 32, torch.float32)
    cache["committed"] = torch.round(cache["committed"] * 2) / 2
    check(cache, keep, recent=3, sinks=1)
    cache["committed"].zero_()
    check(cache, keep)
    cache["committed"][:, :, ::2] = -0.0
    check(cache, keep)


def test_ranks_that_are_not_finite_and_negative_ones():
    cache = cache_of(1, 2, 2000, 32, torch.float32)
    c = cache["committed"]
    c -= 0.5
    c[0, 0, 5:40] = float("nan")
    c[0, 0, 60] = float("inf")
    c[0, 1, 100:1500] = float("-inf")
    c[0, 1, 7] = -float("nan")
    for keep in (1, 20, 35, 36, 37, 700):
        check(cache, keep)


def test_scores_of_a_softmax_layer():
    cache = cache_of(2, 2, 700, 64, torch.bfloat16)
    del cache["committed"]
    scores = seeded((2, 2, 700), 9).to(DEV)
    check(cache, 200, recent=10, scores=scores)
    check(cache, 200, scores=seeded((2, 700, 2), 9).to(DEV).transpose(1, 2))
    kept = check(cache, 300, scores=torch.cat((scores, torch.full((2, 2, 40), 99.0, device=DEV)), 2))
    assert kept["index"].max().item() < 700


def test_an_evicted_cache_is_evicted_again_and_counts():
    lib = load_package()
    cache = cache_of(1, 2, 900, 64, torch.bfloat16)
    once = lib.evict_cache(cache, 500)
    twice = lib.evict_cache(once, 100)
    assert twice["evicted"] == 800 and twice["len"] == 100
    assert torch.equal(twice["k"][:, :, :100], torch.gather(once["k"], 2, twice["index"].long()[..., None].expand(-1, -1, -1, 64)))


def test_recorded_and_on_another_stream():
    lib = load_package()
    cache = cache_of(2, 2, 5000, 64, torch.bfloat16)
    lib.evict_cache(cache, 1000)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = lib.evict_cache(cache, 1000, recent=10)
    for seed in (1, 2):
        cache["committed"].copy_(seeded(cache["committed"].shape, seed).to(DEV))
        graph.replay()
        assert torch.equal(kept["index"].long().cpu(), O.evicted(cache["committed"][:, :, :5000].cpu(), 1000, 10, 0))
    with torch.cuda.stream(torch.cuda.Stream()):
        other = lib.evict_cache(cache, 1000, recent=10)
    torch.cuda.synchronize()
    assert torch.equal(other["index"], kept["index"])
