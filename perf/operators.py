"""Operators around the attention layers of a model, as cases that can be timed.

    path "attend"  softmax attention of a training step or a prompt whose scores are capped by a tanh, lose a multiple
                   of the distance, and see a document's own tokens and a prefix: forward, or forward + backward
    path "tree"    softmax_tree_step: the drafted tokens of a tree (a single token is a tree of one) over a cache
    path "draft"   dilution_tree_step and tree_accept: the same for a dilution layer, whose nodes see the demand of
                   their ancestors, and the accepted branch's demand and rows into the cache
    path "evict"   evict_cache: the keys of a cache that were bid for least make room

Where `own` is false, `run` computes them from elementary torch operations in 32 bits; where it is true, it calls the
library.  Tensors are (batch, heads, seq, dim).
"""

from __future__ import annotations

import importlib
import math
import random

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp32": 4}
_EPS = 1e-9
_SLAB = 1 << 26          # scores that the plain forms hold at a time


def _package():
    return importlib.import_module("dilution-attention_b200")


def _attend(name, batch, heads, kv_heads, seq, dim, dtype, softcap=0.0, slopes=False, docs=0, prefix=0, grad=True):
    case = dict(path="attend", batch=batch, heads=heads, kv_heads=kv_heads, seq=seq, dim=dim, dtype=dtype, softcap=softcap,
                slopes=slopes, docs=docs, prefix=prefix, grad=grad)
    return dict(case, name=name) if name else case


def _tree(name, batch, heads, kv_heads, seq, dim, dtype, nodes, softcap=0.0, slopes=False):
    case = dict(path="tree", batch=batch, heads=heads, kv_heads=kv_heads, seq=seq, dim=dim, dtype=dtype, nodes=nodes,
                softcap=softcap, slopes=slopes)
    return dict(case, name=name) if name else case


def _draft(name, batch, heads, seq, dim, dtype, nodes, accepted):
    case = dict(path="draft", batch=batch, heads=heads, seq=seq, dim=dim, dtype=dtype, nodes=nodes, accepted=accepted)
    return dict(case, name=name) if name else case


def _evict(name, batch, heads, seq, dim, dtype, keep, recent, sinks):
    case = dict(path="evict", batch=batch, heads=heads, seq=seq, dim=dim, dtype=dtype, keep=keep, recent=recent, sinks=sinks)
    return dict(case, name=name) if name else case


def listed():
    return [
        # a training step of an alternating model's softmax layer on packed documents of 700 tokens on average
        _attend("train_packed_4k", 4, 16, 16, 4096, 64, "bf16", docs=700),
        # long-context training with capped scores, grouped keys and heads of 128
        _attend("train_cap_8k", 2, 16, 4, 8192, 128, "bf16", softcap=30.0),
        # a batch of short, ragged rows with a distance bias, all causal
        _attend("train_slopes_ragged", 8, 12, 12, 777, 64, "bf16", slopes=True),
        # a prompt whose first part sees itself whole, read once for a cache that follows: no gradient
        _attend("prompt_prefix", 1, 16, 8, 6001, 64, "bf16", slopes=True, prefix=1500, grad=False),
        # an fp32 model's parity run, everything at once
        _attend("train_fp32_small", 1, 4, 2, 301, 64, "fp32", softcap=20.0, slopes=True, docs=90, prefix=33),
        # serving with speculation: 16 sequences of 16K tokens, 32 drafted tokens each, keys shared by four heads
        _tree("tree_16x16k", 16, 16, 4, 16384, 64, "bf16", 32),
        # interactive generation of a model with capped scores and heads of 128: one token, an odd length
        _tree("token_one", 1, 16, 16, 3001, 128, "bf16", 1, softcap=50.0, slopes=True),
        # the dilution layers of a speculating model: 24 drafted tokens, 5 of them accepted
        _draft("draft_16x16k", 16, 16, 16384, 64, "bf16", 24, 5),
        # the same for one short sequence
        _draft("draft_one", 1, 16, 1001, 64, "bf16", 7, 3),
        # an fp32 cache and a tree of 40
        _draft("draft_fp32", 2, 8, 4099, 32, "fp32", 40, 6),
        # a batch of 64K-token caches down to a quarter
        _evict("evict_64k", 8, 16, 65536, 64, "bf16", 16384, 1024, 4),
        # one short fp32 cache down to what a context allows
        _evict("evict_small", 1, 8, 1777, 64, "fp32", 1024, 128, 0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _length(rng, lo, hi):
    """Lengths over their logarithm; a third of them multiples of 128."""
    n = _log_int(rng, lo, hi)
    return max(lo, n // 128 * 128) if n >= 256 and rng.random() < 0.34 else n


def _heads(rng, most):
    """(batch, heads, kv_heads) with at most `most` query rows."""
    heads = rng.choice([h for h in (1, 2, 4, 6, 8, 12, 16) if h <= max(1, most)])
    kv = heads if rng.random() < 0.5 else rng.choice([h for h in (1, 2, 4, 8) if heads % h == 0])
    return _log_int(rng, 1, max(1, min(32, most // heads))), heads, kv


def draw(rng):
    path = rng.choice(("attend", "attend", "attend", "tree", "tree", "draft", "draft", "evict"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    if path == "attend":
        dim = rng.choice((64, 64, 64, 128, 128, 32))
        seq = _length(rng, 1, 8192 if dtype == "bf16" else 2048)
        cells = (32 * 8192 ** 2 if dtype == "bf16" else 16 * 2048 ** 2) * 64 // max(dim, 64) // seq ** 2
        batch, heads, kv = _heads(rng, max(1, min(256, cells, (1 << 18) // seq)))
        docs = rng.choice((0, 0, _log_int(rng, 8, 2048)))
        return _attend(None, batch, heads, kv, seq, dim, dtype, softcap=rng.choice((0.0, 0.0, 15.0, 30.0, 50.0)),
                       slopes=rng.random() < 0.4, docs=docs, prefix=rng.choice((0, 0, seq // 3, seq // 7)),
                       grad=rng.random() < 0.7)
    dim = rng.choice((64, 64, 64, 128, 32))
    seq = _length(rng, 8, 65536)
    most = max(1, min(256, (1 << 29) // (seq * dim * _BYTES[dtype])))
    batch, heads, kv = _heads(rng, most)
    if path == "tree":
        nodes = rng.choice((1, 1, _log_int(rng, 2, 64)))
        return _tree(None, batch, heads, kv, seq, dim, dtype, nodes, softcap=rng.choice((0.0, 0.0, 20.0, 50.0)),
                     slopes=rng.random() < 0.4)
    if path == "draft":
        nodes = _log_int(rng, 1, 48)
        return _draft(None, batch, heads, seq, dim, dtype, nodes, rng.randint(1, min(nodes, 8)))
    keep = max(1, int(seq * rng.uniform(0.05, 1.0)))
    recent = rng.randint(0, keep // 4)
    return _evict(None, batch, heads, seq, dim, dtype, keep, recent, rng.choice((0, 0, min(4, keep - recent))))


def _normal(g, shape, dtype, scale=1.0):
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, scale, generator=g).to(dtype)


def _cache_tensor(g, shape, dtype):
    t = torch.empty(shape, device="cuda", dtype=dtype)
    for row in t:
        row.normal_(generator=g)
    return t


def _slopes(heads):
    """A geometric sequence over the heads, from 2^(-8 / heads) down to 2^-8."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")


def _documents(rng, batch, seq, mean):
    """Ids of documents of 1 to 2 mean - 1 tokens, one behind the other; a row may end in padding, whose id is -1."""
    rows = []
    for _ in range(batch):
        ids, doc = [], 0
        while len(ids) < seq:
            ids += [doc] * rng.randint(1, 2 * mean - 1)
            doc += 1
        pad = rng.randint(0, seq // 16)
        rows.append(ids[:seq - pad] + [-1] * pad)
    return torch.tensor(rows, dtype=torch.int32).cuda()


def _parents(rng, batch, nodes, accepted):
    """A tree for each sequence, parents in front of their children, and a branch of `accepted` nodes from the root."""
    parents, paths = [], []
    for _ in range(batch):
        path = sorted(rng.sample(range(nodes), accepted))
        row = [rng.randint(-1, i - 1) if rng.random() < 0.5 else i - 1 for i in range(nodes)]
        for a, i in enumerate(path):
            row[i] = path[a - 1] if a else -1
        parents.append(row)
        paths.append(path)
    return torch.tensor(parents, dtype=torch.int32).cuda(), torch.tensor(paths, dtype=torch.int32).cuda()


def _demand(g, shape, seq):
    """Position j of a prefix of seq tokens has collected about sum_{i >= j} 1 / (i + 1)."""
    pos = torch.arange(1, seq + 1, device="cuda", dtype=torch.float32)
    mean = torch.log(seq / pos) + 0.5 / pos
    out = torch.zeros(shape, device="cuda")
    out[..., :seq] = mean * torch.empty(*shape[:-1], seq, device="cuda").uniform_(0.5, 1.5, generator=g)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    b, h, t, d = case["batch"], case["heads"], case["seq"], case["dim"]
    dtype = _DTYPE[case["dtype"]]
    state = dict(case=case)
    if case["path"] == "attend":
        kv = case["kv_heads"]
        # capped models' scores are wide: a standard deviation of 3
        state["q"] = _normal(g, (b, h, t, d), dtype, 3.0 if case["softcap"] else 1.0)
        state["k"], state["v"] = (_normal(g, (b, kv, t, d), dtype) for _ in range(2))
        state["options"] = dict(softcap=case["softcap"] or None, slopes=_slopes(h) if case["slopes"] else None,
                                documents=_documents(rng, b, t, case["docs"]) if case["docs"] else None, prefix=None)
        if case["prefix"]:
            top = case["prefix"]
            state["options"]["prefix"] = torch.tensor([rng.randint(top // 2, top) for _ in range(b)], dtype=torch.int32).cuda()
        if case["grad"]:
            state["dout"] = _normal(g, (b, h, t, d), dtype, 1e-2)
            for name in "qkv":
                state[name].requires_grad_(True)
        return state
    if case["path"] == "evict":
        shape = (b, h, t, d)
        demand = _demand(g, shape[:-1], t)
        # keys that nobody has bid for since they came are alike
        demand[torch.empty(shape[:-1], device="cuda").uniform_(generator=g) < 0.1] = 0.0
        state["cache"] = dict(k=_cache_tensor(g, shape, dtype), v=_cache_tensor(g, shape, dtype), len=t, committed=demand)
        return state
    nodes = case["nodes"]
    kv = case.get("kv_heads", h)
    cap = t + 64
    state["q"] = _normal(g, (b, h, nodes, d), dtype, 3.0 if case.get("softcap") else 1.0)
    state["k"], state["v"] = (_normal(g, (b, kv, nodes, d), dtype) for _ in range(2))
    state["cache"] = dict(k=_cache_tensor(g, (b, kv, cap, d), dtype), v=_cache_tensor(g, (b, kv, cap, d), dtype), len=t)
    state["parents"], state["path"] = _parents(rng, b, nodes, case.get("accepted", 1))
    if case["path"] == "tree":
        state["options"] = dict(softcap=case["softcap"] or None, slopes=_slopes(h) if case["slopes"] else None)
    else:
        state["cache"]["committed"] = _demand(g, (b, h, cap), t)
        state["advanced"] = torch.zeros(b, h, cap, device="cuda")
    return state


# ---- the plain forms -------------------------------------------------------------------------
def _visible(documents, prefix, row, seq):
    """(seq, seq) truth values: the query of the row sees the key of the column."""
    pos = torch.arange(seq, device="cuda")
    see = pos[None, :] <= pos[:, None]
    if prefix is not None:
        see = see | (pos[None, :] < prefix[row])
    if documents is not None:
        ids = documents[row]
        see = see & (ids[:, None] == ids[None, :]) & (ids[:, None] >= 0)
    return see


def _plain_attend(state):
    case, opt = state["case"], state["options"]
    q, k, v = (state[x].detach() for x in "qkv")
    b, h, t, d = q.shape
    kv = k.shape[1]
    group, scale, cap = h // kv, 1.0 / math.sqrt(d), opt["softcap"]
    out = torch.empty_like(q)
    if case["grad"]:
        dq = torch.empty_like(q)
        dk, dv = (torch.zeros(b, kv, t, d, device="cuda") for _ in range(2))
    pos = torch.arange(t, device="cuda", dtype=torch.float32)
    far = (pos[:, None] - pos[None, :]).abs()
    slab = max(1, _SLAB // (t * t))
    for row in range(b):
        see = _visible(opt["documents"], opt["prefix"], row, t)
        for a in range(0, h, slab):
            heads = torch.arange(a, min(h, a + slab), device="cuda")
            qf, kf, vf = q[row, heads].float(), k[row, heads // group].float(), v[row, heads // group].float()
            z = scale * (qf @ kf.transpose(1, 2))
            if cap is not None:
                u = torch.tanh(z / cap)
                z = cap * u
            if opt["slopes"] is not None:
                z = z - opt["slopes"][heads, None, None] * far
            z = z.masked_fill(~see, -math.inf)
            top = z.amax(-1, keepdim=True)
            e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
            mass = e.sum(-1, keepdim=True)
            p = e / torch.where(mass == 0, 1.0, mass)
            out[row, heads] = (p @ vf).to(q.dtype)
            if case["grad"]:
                do = state["dout"][row, heads].float()
                dv[row].index_add_(0, heads // group, p.transpose(1, 2) @ do)
                dp = do @ vf.transpose(1, 2)
                dz = p * (dp - (p * dp).sum(-1, keepdim=True))
                if cap is not None:
                    dz = dz * (1.0 - u * u)
                dq[row, heads] = (scale * (dz @ kf)).to(q.dtype)
                dk[row].index_add_(0, heads // group, scale * (dz.transpose(1, 2) @ qf))
    return (out, dq, dk.to(q.dtype), dv.to(q.dtype)) if case["grad"] else out


def _lineage(parents):
    """(batch, nodes, nodes) of 0 and 1: the node of the row is the node of the column or comes from it."""
    n = parents.shape[1]
    step = (parents[:, :, None] == torch.arange(n, device="cuda")).float() + torch.eye(n, device="cuda")
    for _ in range(max(1, (n - 1).bit_length())):
        step = ((step @ step) > 0).float()
    return step


def _plain_bids(state, row, line):
    """Softmax of the nodes' scores over the cached keys and their lineage: (heads, nodes, length + nodes)."""
    case, cache, opt = state["case"], state["cache"], state.get("options", {})
    q, kn = state["q"][row].float(), state["k"][row].float()
    h, n, d = q.shape
    t, kv = case["seq"], kn.shape[0]
    keys = torch.cat((cache["k"][row, :, :t].float(), kn), 1)
    z = (q.view(kv, h // kv * n, d) @ keys.transpose(1, 2)).view(h, n, t + n) / math.sqrt(d)
    if opt.get("softcap") is not None:
        z = opt["softcap"] * torch.tanh(z / opt["softcap"])
    if opt.get("slopes") is not None:
        depth = line.sum(-1) - 1.0 + t
        at = torch.cat((torch.arange(t, device="cuda", dtype=torch.float32), depth))
        z = z - opt["slopes"][:, None, None] * (depth[:, None] - at[None, :])
    z[:, :, t:].masked_fill_(line == 0, -math.inf)
    e = torch.exp(z - z.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_tree(state):
    case, cache, q = state["case"], state["cache"], state["q"]
    line = _lineage(state["parents"])
    out = torch.empty_like(q)
    t = case["seq"]
    for row in range(case["batch"]):
        p = _plain_bids(state, row, line[row])
        vals = torch.cat((cache["v"][row, :, :t].float(), state["v"][row].float()), 1)
        kv, (h, n, m) = vals.shape[0], p.shape
        out[row] = (p.view(kv, h // kv * n, m) @ vals).view(h, n, -1).to(q.dtype)
    return out


def _plain_draft(state):
    case, cache, q = state["case"], state["cache"], state["q"]
    line = _lineage(state["parents"])
    t, n, a = case["seq"], case["nodes"], case["accepted"]
    out = torch.empty_like(q)
    advanced = state["advanced"]
    eye = torch.eye(n, device="cuda")
    for row in range(case["batch"]):
        p = _plain_bids(state, row, line[row])
        vals = torch.cat((cache["v"][row, :, :t].float(), state["v"][row].float()), 1)
        before = (line[row] - eye) @ p
        before[:, :, :t] += cache["committed"][row, :, None, :t]
        share = p / (before + p + _EPS)
        out[row] = ((share / (share.sum(-1, keepdim=True) + _EPS)) @ vals).to(q.dtype)
        path = state["path"][row].long()
        taken = p[:, path].sum(1)
        advanced[row, :, :t] = cache["committed"][row, :, :t] + taken[:, :t]
        advanced[row, :, t:t + a] = taken[:, t + path]
        cache["k"][row, :, t:t + a] = state["k"][row][:, path]
        cache["v"][row, :, t:t + a] = state["v"][row][:, path]
    return out, advanced, cache["k"][:, :, t:t + a], cache["v"][:, :, t:t + a]


def _plain_evict(state):
    case, cache = state["case"], state["cache"]
    t, keep, recent, sinks = case["seq"], case["keep"], case["recent"], case["sinks"]
    rank = cache["committed"][:, :, :t].clone()
    rank[:, :, :sinks] = math.inf
    rank[:, :, t - recent:] = math.inf
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :, :keep]
    index = torch.sort(best, dim=-1).values
    rows = index[..., None].expand(-1, -1, -1, cache["k"].shape[-1])
    return (torch.gather(cache["k"], 2, rows), torch.gather(cache["v"], 2, rows),
            torch.gather(cache["committed"], 2, index), index.int())


_PLAIN = {"attend": _plain_attend, "tree": _plain_tree, "draft": _plain_draft, "evict": _plain_evict}


def run(state):
    case = state["case"]
    if not own:
        return _PLAIN[case["path"]](state)
    lib = _package()
    if case["path"] == "attend":
        q, k, v = state["q"], state["k"], state["v"]
        out = lib.softmax_attention(q, k, v, **state["options"])
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), state["dout"])) if case["grad"] else out
    cache = state["cache"]
    cache["len"] = case["seq"]
    if case["path"] == "evict":
        kept = lib.evict_cache(cache, case["keep"], recent=case["recent"], sinks=case["sinks"], capacity=case["keep"])
        return kept["k"], kept["v"], kept["committed"], kept["index"]
    if case["path"] == "tree":
        out, _ = lib.softmax_tree_step(state["q"], state["k"], state["v"], cache, state["parents"], **state["options"])
        return out
    out, draft = lib.dilution_tree_step(state["q"], state["k"], state["v"], cache, state["parents"])
    lib.tree_accept(cache, draft, state["path"], out=state["advanced"])
    t, a = case["seq"], case["accepted"]
    return out, state["advanced"], cache["k"][:, :, t:t + a], cache["v"][:, :, t:t + a]


def work(case):
    """A product over the visible (query, key) pairs is 2 d flops a pair: 2 of them forward (q k^T, p v), 7 with the
    backward (q k^T again, dout v^T, dv, dq, dk).  Documents of 1 to 2 m - 1 tokens leave a query 2 m / 3 keys on
    average.  Bytes: each input and output once; a cache's rows and its demand once (written back where it advances)."""
    b, h, t, d = case["batch"], case["heads"], case["seq"], case["dim"]
    e = _BYTES[case["dtype"]]
    kv = case.get("kv_heads", h)
    if case["path"] == "attend":
        keys = (t + 1) / 2
        if case["prefix"]:
            keys += (0.75 * case["prefix"]) ** 2 / 2 / t
        if case["docs"]:
            keys = min(keys, max(1.0, 2 * case["docs"] / 3))
        pairs = b * h * t * keys
        rows = b * t * d * e * (2 * h + 2 * kv)
        if not case["grad"]:
            return {"bytes": rows, "flops": 4 * pairs * d}
        return {"bytes": 2 * rows, "flops": 14 * pairs * d}
    if case["path"] == "evict":
        return {"bytes": b * h * (4 * t + case["keep"] * (4 * d * e + 12)), "flops": 0}
    n = case["nodes"]
    nodes = b * n * d * e * (2 * h + 2 * kv)
    flops = 4 * b * h * n * (t + n) * d
    if case["path"] == "tree":
        return {"bytes": 2 * b * kv * t * d * e + nodes, "flops": flops}
    return {"bytes": b * h * t * (2 * d * e + 8) + nodes + 4 * b * h * case["accepted"] * d * e, "flops": flops}


# ---- the definitions in 64 bits -----------------------------------------------------------------
def _exact_attend(state):
    case, opt = state["case"], state["options"]
    q, k, v = (state[x].detach().double() for x in "qkv")
    b, h, t, d = q.shape
    group = h // k.shape[1]
    results = [torch.zeros_like(x) for x in (q, q, k, v)]
    i = torch.arange(t, device="cuda")[:, None]
    j = i.T
    for row in range(b):
        hidden = j > i
        if opt["prefix"] is not None:
            hidden = hidden & (j >= opt["prefix"][row])
        if opt["documents"] is not None:
            ids = opt["documents"][row]
            hidden = hidden | (ids[i] != ids[j]) | (ids[i] < 0)
        for head in range(h):
            leaves = [x.clone().requires_grad_(case["grad"]) for x in (q[row, head], k[row, head // group], v[row, head // group])]
            s = leaves[0] @ leaves[1].T * d ** -0.5
            if opt["softcap"] is not None:
                s = torch.tanh(s / opt["softcap"]) * opt["softcap"]
            if opt["slopes"] is not None:
                s = s - opt["slopes"][head].double() * (i - j).abs()
            w = torch.softmax(torch.where(hidden, -1e300, s), -1) * ~hidden
            o = w @ leaves[2]
            results[0][row, head] = o.detach()
            if case["grad"]:
                gq, gk, gv = torch.autograd.grad(o, leaves, state["dout"][row, head].double())
                results[1][row, head] = gq
                results[2][row, head // group] += gk
                results[3][row, head // group] += gv
    return tuple(results) if case["grad"] else results[0]


def _exact_nodes(state, dilute):
    """Node by node along its branch, as so many steps of single tokens would: (outputs, bids)."""
    case, cache, opt = state["case"], state["cache"], state.get("options", {})
    b, h, n, d = state["q"].shape
    t, kv = case["seq"], state["k"].shape[1]
    parents = state["parents"].tolist()
    out = torch.zeros(b, h, n, d, device="cuda", dtype=torch.float64)
    bids = []
    for row in range(b):
        share_of = torch.arange(h, device="cuda") // (h // kv)
        keys = torch.cat((cache["k"][row, :, :t], state["k"][row]), 1).double()
        vals = torch.cat((cache["v"][row, :, :t], state["v"][row]), 1).double()
        demand, mine, depth, chain = [], [], [], []
        for x in range(n):
            up = parents[row][x]
            chain.append((chain[up] if up >= 0 else []) + [x])
            depth.append(depth[up] + 1 if up >= 0 else 0)
            seen = torch.cat((torch.arange(t, device="cuda"), torch.tensor(chain[x], device="cuda") + t))
            q = state["q"][row, :, x].double()
            s = torch.stack([(keys[c] @ q[c * (h // kv):(c + 1) * (h // kv)].T).T for c in range(kv)]).view(h, t + n)[:, seen] * d ** -0.5
            if opt.get("softcap") is not None:
                s = torch.tanh(s / opt["softcap"]) * opt["softcap"]
            if opt.get("slopes") is not None:
                at = torch.cat((torch.arange(t, device="cuda"), t + torch.arange(len(chain[x]), device="cuda")))
                s = s - opt["slopes"].double()[:, None] * (t + depth[x] - at)
            p = torch.zeros(h, t + n, device="cuda", dtype=torch.float64)
            p[:, seen] = torch.softmax(s, -1)
            mine.append(p)
            w = p
            if dilute:
                if up >= 0:
                    had = demand[up] + mine[up]
                else:
                    had = torch.zeros_like(p)
                    had[:, :t] = cache["committed"][row, :, :t]
                demand.append(had)
                w = p / (had + p + _EPS)
                w = w / (w.sum(-1, keepdim=True) + _EPS)
            for c in range(kv):
                own_heads = share_of == c
                out[row, own_heads, x] = w[own_heads] @ vals[c]
        bids.append(torch.stack(mine, 1))
        del demand, mine
        if not dilute:
            bids.clear()
    return out, bids


def exact(case, seed):
    if case["path"] in ("tree", "draft") and case["batch"] * case["heads"] * case["nodes"] * case["seq"] > 1 << 28:
        return None
    state = prepare(case, seed)
    t = case["seq"]
    if case["path"] == "attend":
        return _exact_attend(state)
    cache = state["cache"]
    if case["path"] == "tree":
        return _exact_nodes(state, False)[0]
    if case["path"] == "draft":
        out, bids = _exact_nodes(state, True)
        advanced = torch.zeros_like(state["advanced"], dtype=torch.float64)
        a = case["accepted"]
        kept = [torch.zeros(*state["k"].shape[:2], a, case["dim"], device="cuda", dtype=torch.float64) for _ in range(2)]
        for row, p in enumerate(bids):
            path = state["path"][row].tolist()
            advanced[row, :, :t] = cache["committed"][row, :, :t].double()
            for x in path:
                advanced[row, :, :t] += p[:, x, :t]
            for at, key in enumerate(path):
                advanced[row, :, t + at] = sum(p[:, x, t + key] for x in path)
                for dst, src in zip(kept, (state["k"], state["v"])):
                    dst[row, :, at] = src[row, :, key].double()
        return out, advanced, *kept
    # whole numbers have one right answer: the order of (rank, position) pairs, one row at a time
    b, h = case["batch"], case["heads"]
    index = torch.empty(b, h, case["keep"], device="cuda", dtype=torch.int64)
    where = torch.arange(t, device="cuda")
    held = (where < case["sinks"]) | (where >= t - case["recent"])
    for row in range(b):
        for head in range(h):
            rank = cache["committed"][row, head, :t].double()
            others = where[~held]
            order = others[torch.argsort(-rank[others], stable=True)][:case["keep"] - int(held.sum())]
            index[row, head] = torch.cat((where[held], order)).sort().values
    pick = [torch.stack([torch.stack([x[r, c, index[r, c]] for c in range(h)]) for r in range(b)]).double()
            for x in (cache["k"], cache["v"], cache["committed"])]
    return *pick, index.int()
