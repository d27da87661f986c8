"""Trees of drafted tokens over a cache: softmax and dilution layers, the accepted branch, against 64 bits and against chains of
single steps."""

from __future__ import annotations

import pytest
import torch

from conftest import load_package, seeded
from oracle import operators_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"

TREE = [-1, 0, 0, 1, 1, 2, -1, 6, 3, 8, 9, 4]
CHAINS = {"leaf": [0, 1, 3, 8, 9, 10], "short": [6], "fork": [0, 2, 5]}


def case(batch, heads, kv_heads, nodes, dim, length, dtype, seed=0, room=9, q_scale=1.0):
    q = seeded((batch, heads, nodes, dim), seed, q_scale).to(DEV, dtype)
    k, v = (seeded((batch, kv_heads, nodes, dim), seed + s).to(DEV, dtype) for s in (1, 2))
    cap = length + nodes + room
    kc, vc = (seeded((batch, kv_heads, cap, dim), seed + s).to(DEV, dtype) for s in (3, 4))
    kc[:, :, length:] = float("nan")        # rows behind the last key are nobody's
    vc[:, :, length:] = float("nan")
    committed = seeded((batch, kv_heads, cap), seed + 5).abs().to(DEV) * 3
    return q, k, v, dict(k=kc, v=vc, len=length, committed=committed)


def clone(cache):
    return {x: y.clone() if isinstance(y, torch.Tensor) else y for x, y in cache.items()}


def random_tree(nodes, seed):
    g = torch.Generator().manual_seed(seed)
    return [int(torch.randint(-1, x, (1,), generator=g)) if x and torch.rand(1, generator=g) < 0.6 else x - 1 for x in range(nodes)]


def within(got, want, off):
    far = (got.double() - want).abs() - off
    assert torch.isfinite(got).all() and far.max().item() <= 1e-12, (far.max().item(), (got.double() - want).abs().max().item())


TYPES = [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float32, 128), (torch.bfloat16, 16),
         (torch.float32, 32)]


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("length", [0, 1, 63, 64, 200, 1111])
@pytest.mark.parametrize("options", [{}, {"softcap": 6.0, "slopes": True}])
def test_softmax_tree(length, options, dtype, dim):
    q, k, v, cache = case(2, 4, 2, len(TREE), dim, length, dtype, q_scale=2.0)
    options = dict(options)
    if options.get("slopes"):
        options["slopes"] = torch.tensor([0.5, 0.1, 0.01, 0.0], device=DEV)
    out, draft = load_package().softmax_tree_step(q, k, v, cache, torch.tensor(TREE, device=DEV), **options)
    want, off, bids, bids_off = O.tree_nodes(q, k, v, cache["k"], cache["v"], length, TREE, **options)
    within(out, want, off)
    # the accepted branch adds its attention weights, over the heads that share a key head
    path = CHAINS["leaf"]
    before = clone(cache)
    advanced = load_package().tree_accept(cache, draft, path)
    assert cache["len"] == length + len(path) and advanced is cache["committed"]
    check_accept(before, cache, k, v, bids, bids_off, [path] * 2, length)


def check_accept(before, cache, k, v, bids, bids_off, paths, length):
    batch, kv_heads = k.shape[:2]
    for b, path in enumerate(paths):
        a = len(path)
        for name, new in (("k", k), ("v", v)):
            assert torch.equal(cache[name][b, :, length:length + a], new[b][:, path])
            assert torch.equal(cache[name][b, :, :length], before[name][b, :, :length])
            assert cache[name][b, :, length + a:].isnan().all()
        at = list(range(length)) + [length + x for x in path]
        taken, off = (x[b][:, path][:, :, at].unflatten(0, (kv_heads, -1)).sum((1, 2)) for x in (bids, bids_off))
        taken[:, :length] += before["committed"][b, :, :length].double()
        within(cache["committed"][b, :, :length + a], taken, off + 2.0 ** -18 * taken + 1e-9)
        assert torch.equal(cache["committed"][b, :, length + a:], before["committed"][b, :, length + a:])


@pytest.mark.parametrize("dtype,dim", TYPES)
@pytest.mark.parametrize("length", [0, 1, 64, 130, 1111, 17000])
@pytest.mark.parametrize("chain", CHAINS)
def test_dilution_tree(length, chain, dtype, dim):
    q, k, v, cache = case(1, 3, 3, len(TREE), dim, length, dtype)
    out, draft = load_package().dilution_tree_step(q, k, v, cache, TREE)
    want, off, bids, bids_off = O.tree_nodes(q, k, v, cache["k"], cache["v"], length, TREE, committed=cache["committed"])
    within(out, want, off)
    before = clone(cache)
    load_package().tree_accept(cache, draft, CHAINS[chain])
    check_accept(before, cache, k, v, bids, bids_off, [CHAINS[chain]], length)


@pytest.mark.parametrize("nodes", [1, 2, 15, 16, 17, 33, 48, 64])
@pytest.mark.parametrize("dtype,dim", TYPES[:4])
def test_tree_sizes_and_a_tree_for_each_sequence(nodes, dtype, dim):
    trees = [random_tree(nodes, s) for s in (nodes, 100 + nodes)]
    q, k, v, cache = case(2, 2, 2, nodes, dim, 300, dtype)
    parents = torch.tensor(trees, device=DEV, dtype=torch.int32)
    out, _ = load_package().softmax_tree_step(q, k, v, cache, parents)
    within(out, *O.tree_nodes(q, k, v, cache["k"], cache["v"], 300, trees)[:2])
    out, draft = load_package().dilution_tree_step(q, k, v, cache, parents)
    want, off, bids, bids_off = O.tree_nodes(q, k, v, cache["k"], cache["v"], 300, trees, committed=cache["committed"])
    within(out, want, off)
    paths = []
    for tree in trees:                      # the branch of the last node, cut to one length
        path = [nodes - 1]
        while tree[path[0]] >= 0:
            path.insert(0, tree[path[0]])
        paths.append(path)
    a = min(len(p) for p in paths)
    paths = [p[:a] for p in paths]
    before = clone(cache)
    load_package().tree_accept(cache, draft, torch.tensor(paths, device=DEV))
    check_accept(before, cache, k, v, bids, bids_off, paths, 300)


@pytest.mark.parametrize("heads,kv_heads,nodes", [(16, 1, 30), (8, 2, 64), (6, 3, 5)])
@pytest.mark.parametrize("dtype,dim", TYPES[:3])
def test_many_rows_on_one_key_head(heads, kv_heads, nodes, dtype, dim):
    tree = random_tree(nodes, 7)
    q, k, v, cache = case(1, heads, kv_heads, nodes, dim, 500, dtype)
    out, draft = load_package().softmax_tree_step(q, k, v, cache, tree)
    want, off, bids, bids_off = O.tree_nodes(q, k, v, cache["k"], cache["v"], 500, tree)
    within(out, want, off)
    path = [nodes - 1]
    while tree[path[0]] >= 0:
        path.insert(0, tree[path[0]])
    before = clone(cache)
    load_package().tree_accept(cache, draft, path)
    check_accept(before, cache, k, v, bids, bids_off, [path], 500)


@pytest.mark.parametrize("dtype,dim", TYPES)
def test_a_branch_is_a_chain_of_decode_steps(dtype, dim):
    """Each node of a branch against dilution_decode_append_step on a copy of the cache, and the demand that both leave; the two
    differ by their roundings alone, 2 u of a bf16 output each."""
    lib = load_package()
    q, k, v, cache = case(2, 2, 2, len(TREE), dim, 257, dtype)
    single = clone(cache)
    for x in ("k", "v"):
        single[x] = torch.nan_to_num(single[x])
    single["committed"][:, :, 257:] = 0
    out, draft = lib.dilution_tree_step(q, k, v, cache, TREE)
    path = CHAINS["leaf"]
    _, off, _, bids_off = O.tree_nodes(q, k, v, cache["k"], cache["v"], 257, TREE, committed=cache["committed"])
    for x in path:
        y = lib.dilution_decode_append_step(*(t[:, :, x:x + 1].contiguous() for t in (q, k, v)), single)
        assert ((y[:, :, 0].double() - out[:, :, x].double()).abs() <= 2 * off[:, :, x] + 1e-12).all()
    lib.tree_accept(cache, draft, path)
    n = 257 + len(path)
    assert cache["len"] == single["len"] == n
    assert torch.equal(cache["k"][:, :, :n], single["k"][:, :, :n])
    # (a chain adds a demand and a bid at a time: 2^-24 of the demand for each)
    assert (cache["committed"][:, :, :n] - single["committed"][:, :, :n]).abs().max().item() <= 1e-4


@pytest.mark.parametrize("dtype,dim", TYPES[:4])
def test_a_round_after_a_prompt_and_an_eviction(dtype, dim):
    """Prompt, draft, accept, evict, draft again: the whole path of a serving loop."""
    lib = load_package()
    b, h, t = 1, 2, 320
    q, k, v = (seeded((b, h, t, dim), s).to(DEV, dtype) for s in range(3))
    prec = "bf16" if dtype == torch.bfloat16 else "ieee"
    _, aux = lib.dilution_attention_forward(q, k, v, dot_precision=prec, return_aux=True)
    cap = t + 64
    cache = dict(k=torch.zeros(b, h, cap, dim, device=DEV, dtype=dtype), v=torch.zeros(b, h, cap, dim, device=DEV, dtype=dtype),
                 len=t, committed=torch.zeros(b, h, cap, device=DEV))
    cache["k"][:, :, :t], cache["v"][:, :, :t], cache["committed"][:, :, :t] = k, v, aux["committed_total"]
    for turn in range(3):
        x = [seeded((b, h, len(TREE), dim), 30 + 3 * turn + s).to(DEV, dtype) for s in range(3)]
        out, draft = lib.dilution_tree_step(*x, cache, TREE)
        within(out, *O.tree_nodes(*x, cache["k"], cache["v"], cache["len"], TREE, committed=cache["committed"])[:2])
        lib.tree_accept(cache, draft, CHAINS["fork"])
        before = cache
        cache = lib.evict_cache(cache, cache["len"] - 50, recent=10, sinks=2)
        want = O.evicted(before["committed"][:, :, :before["len"]].cpu(), before["len"] - 50, 10, 2)
        assert torch.equal(cache["index"].long().cpu(), want)
        y = lib.dilution_decode_append_step(*(t_[:, :, :1].contiguous() for t_ in x), cache)
        assert torch.isfinite(y).all()
    assert cache["evicted"] == 150 and cache["len"] == t + 3 * (3 - 50 + 1)


def test_a_node_of_another_branch_may_hold_anything():
    for dtype, dim in TYPES:
        q, k, v, cache = case(1, 2, 2, len(TREE), dim, 100, dtype)
        lib = load_package()
        clean = [lib.softmax_tree_step(q, k, v, cache, TREE)[0], lib.dilution_tree_step(q, k, v, cache, TREE)[0]]
        k, v = k.clone(), v.clone()
        k[:, :, 6], v[:, :, 7] = float("nan"), float("inf")
        others = [x for x in range(len(TREE)) if x not in (6, 7)]
        got = [lib.softmax_tree_step(q, k, v, cache, TREE)[0], lib.dilution_tree_step(q, k, v, cache, TREE)[0]]
        for a, b in zip(clean, got):
            assert torch.equal(a[:, :, others], b[:, :, others])
            assert b[:, :, 6].isnan().all()


def test_parents_that_are_no_earlier_node_count_as_none():
    q, k, v, cache = case(1, 2, 2, 5, 64, 100, torch.bfloat16)
    wild = torch.tensor([3, 0, 2, 99, -7], device=DEV)
    out, _ = load_package().dilution_tree_step(q, k, v, cache, wild)
    want, _ = load_package().dilution_tree_step(q, k, v, cache, [-1, 0, -1, -1, -1])
    assert torch.equal(out, want)


def test_a_path_outside_the_tree_stays_inside_it():
    q, k, v, cache = case(1, 2, 2, 5, 64, 100, torch.bfloat16)
    _, draft = load_package().dilution_tree_step(q, k, v, cache, [-1, 0, 1, 2, 3])
    load_package().tree_accept(cache, draft, torch.tensor([-4, 99], device=DEV))
    assert torch.equal(cache["k"][:, :, 100], k[:, :, 0]) and torch.equal(cache["k"][:, :, 101], k[:, :, 4])


@pytest.mark.parametrize("dtype,dim", TYPES[:3])
def test_the_length_on_the_device_and_a_recorded_step(dtype, dim):
    lib = load_package()
    q, k, v, cache = case(2, 2, 2, len(TREE), dim, 200, dtype, room=400)
    softmax = {x: cache[x] for x in ("k", "v", "len")}
    pos = torch.tensor([200], device=DEV, dtype=torch.int32)
    recorded = dict(cache, pos_dev=pos, committed=cache["committed"].clone())
    path = torch.tensor(CHAINS["fork"], device=DEV)
    parents = torch.tensor(TREE, device=DEV)
    advanced = torch.zeros_like(cache["committed"])

    def step():
        a, _ = lib.softmax_tree_step(q, k, v, recorded, parents)
        b, draft = lib.dilution_tree_step(q, k, v, recorded, parents)
        held = recorded["len"]
        lib.tree_accept(recorded, draft, path, out=advanced)
        recorded["len"] = held
        return a, b

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for length in (200, 77, 0, 333):
        pos.fill_(length)
        with torch.no_grad():
            cache["k"][:, :, :length] = seeded((2, 2, length, dim), 60 + length).to(DEV, dtype)
            cache["v"][:, :, :length] = seeded((2, 2, length, dim), 61 + length).to(DEV, dtype)
        graph.replay()
        want, off, _, _ = O.tree_nodes(q, k, v, cache["k"], cache["v"], length, TREE)
        within(got[0], want, off)
        want, off, bids, _ = O.tree_nodes(q, k, v, cache["k"], cache["v"], length, TREE, committed=cache["committed"])
        within(got[1], want, off)
        assert torch.equal(cache["k"][:, :, length:length + 3], k[:, :, CHAINS["fork"]])
        taken = cache["committed"][:, :, :length].double() + bids[:, :, CHAINS["fork"], :length].sum(2)
        assert (advanced[:, :, :length].double() - taken).abs().max().item() <= 1e-4 if length else True
    assert softmax["len"] == 200


@pytest.mark.parametrize("dtype,dim", TYPES[:4])
def test_outputs_repeat_and_buffers_are_used(dtype, dim):
    lib = load_package()
    q, k, v, cache = case(2, 4, 4, 20, dim, 3000, dtype)
    tree = random_tree(20, 3)
    first, draft = lib.dilution_tree_step(q, k, v, cache, tree)
    out = torch.empty_like(q)
    scratch = torch.empty(1 << 24, device=DEV, dtype=torch.uint8)
    for _ in range(3):
        got, other = lib.dilution_tree_step(q, k, v, cache, tree, out=out, scratch=scratch)
        assert got is out and torch.equal(got, first) and torch.equal(draft["lse"], other["lse"])
    buf = torch.full_like(cache["committed"], -1.0)
    held = cache["committed"].clone()
    path = [0]
    while True:
        kids = [x for x in range(20) if tree[x] == path[-1]]
        if not kids:
            break
        path.append(kids[0])
    assert lib.tree_accept(dict(cache), draft, path, out=buf) is buf
    assert torch.equal(cache["committed"], held)
    assert (buf[:, :, 3000 + len(path):] == -1).all() and (buf[:, :, :3000] >= held[:, :, :3000]).all()
    assert lib.tree_accept(dict(cache), draft, [], out=buf) is buf and torch.equal(buf[:, :, :3000], held[:, :, :3000])


def test_two_streams_at_once():
    lib = load_package()
    cases = [case(4, 4, 4, 16, 64, 2000, torch.bfloat16, seed=s) for s in (0, 70)]
    tree = random_tree(16, 1)
    want = [lib.dilution_tree_step(q, k, v, cache, tree)[0] for q, k, v, cache in cases]
    torch.cuda.synchronize()
    got = []
    for q, k, v, cache in cases:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(lib.dilution_tree_step(q, k, v, cache, tree)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("nodes", [9, 20, 40, 64])
@pytest.mark.parametrize("dtype,dim", TYPES[:3])
@pytest.mark.parametrize("batch,heads,length", [(3, 11, 300), (1, 2, 16400)])
def test_caches_in_chunks(batch, heads, length, nodes, dtype, dim):
    """More heads, or more keys, than a step by clusters takes: the demand crosses kernels and chunks."""
    trees = [random_tree(nodes, s) for s in range(batch)]
    q, k, v, cache = case(batch, heads, heads, nodes, dim, length, dtype)
    parents = torch.tensor(trees, device=DEV, dtype=torch.int32)
    lib = load_package()
    out, draft = lib.dilution_tree_step(q, k, v, cache, parents)
    want, off, bids, bids_off = O.tree_nodes(q, k, v, cache["k"], cache["v"], length, trees, committed=cache["committed"])
    within(out, want, off)
    again, _ = lib.dilution_tree_step(q, k, v, cache, parents)
    assert torch.equal(out, again)
    before = clone(cache)
    lib.tree_accept(cache, draft, [0])
    check_accept(before, cache, k, v, bids, bids_off, [[0]] * batch, length)


@pytest.mark.parametrize("dim", [64, 128])
def test_a_recorded_step_in_chunks_beside_an_eager_one(dim):
    """40 heads: the step's launches start early behind one another, in a graph as on a stream."""
    lib = load_package()
    tree = random_tree(24, 5)
    q, k, v, cache = case(2, 20, 20, 24, dim, 900, torch.bfloat16)
    parents = torch.tensor(tree, device=DEV, dtype=torch.int32)
    want = lib.dilution_tree_step(q, k, v, cache, parents)[0]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = lib.dilution_tree_step(q, k, v, cache, parents)[0]
        graphs.append((graph, got))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for stream, (graph, got) in zip(streams, graphs):
            got.zero_()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        eager = lib.dilution_tree_step(q, k, v, cache, parents)[0]
        torch.cuda.synchronize()
        assert torch.equal(eager, want) and all(torch.equal(got, want) for _, got in graphs)


@pytest.mark.parametrize("dtype,dim", TYPES[:3])
def test_cached_keys_that_are_not_finite(dtype, dim):
    """A NaN key reaches its own head's rows alone, in either layer and on both of a dilution step's ways."""
    lib = load_package()
    for heads in (2, 40):
        q, k, v, cache = case(1, heads, heads, len(TREE), dim, 150, dtype)
        clean = [lib.softmax_tree_step(q, k, v, cache, TREE)[0], lib.dilution_tree_step(q, k, v, cache, TREE)[0]]
        cache["k"][0, 1, 77, 3] = float("nan")
        got = [lib.softmax_tree_step(q, k, v, cache, TREE)[0], lib.dilution_tree_step(q, k, v, cache, TREE)[0]]
        others = [h for h in range(heads) if h != 1]
        for a, b in zip(clean, got):
            assert b[0, 1].isnan().all() and torch.equal(a[:, others], b[:, others])


def test_strided_tokens_and_a_scratch_that_does_not_do():
    """Rows as a projection leaves them, (B, N, H, D); a scratch that is a view of fewer bytes than it counts is not used."""
    lib = load_package()
    q, k, v, cache = case(2, 4, 4, len(TREE), 64, 200, torch.bfloat16)
    want = lib.softmax_tree_step(q, k, v, cache, TREE)[0]
    strided = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    scratch = torch.zeros(16, device=DEV, dtype=torch.uint8).expand(1 << 20, 16)
    assert torch.equal(lib.softmax_tree_step(*strided, cache, TREE, scratch=scratch)[0], want)
    assert not scratch[0].any()
